// Binds the serving operators: paged rotary step, paged attention, 8-bit linear.
//
// Every check of types, sizes, strides and devices of a CUDA call is made here,
// in one native call (the Python side would take longer than a small kernel);
// what only the device knows (lengths, offsets, pages) is checked by the
// kernels, which leave a code in the error word.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <algorithm>
#include <cmath>
#include <cstdlib>
#include <functional>
#include <optional>
#include <utility>
#include <vector>

#include "../fp8/fp8.h"
#include "../paged/paged.h"
#include "ops.h"

namespace py = pybind11;

namespace {

using b200ar::paged::Batch;
using b200ar::paged::Half;
using b200ar::paged::Pool;
using OptTensor = std::optional<at::Tensor>;

constexpr int64_t kInt = 0x7fffffff;

#define VALUE_CHECK(cond, ...) \
  if (!(cond)) throw py::value_error(c10::str(__VA_ARGS__))
#define TYPE_CHECK(cond, ...) \
  if (!(cond)) throw py::type_error(c10::str(__VA_ARGS__))

cudaStream_t stream_of() { return at::cuda::getCurrentCUDAStream().stream(); }

bool aligned(const at::Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }

void check_device(const at::Tensor& t, const at::Tensor& like, const char* name) {
  VALUE_CHECK(t.device() == like.device(), name, " must be on ", like.device(), ", got ", t.device());
}

// Heads of d contiguous elements on 16-byte boundaries in every dimension before them; `written` ones must not
// share memory among themselves (each stride reaches over what the smaller ones span).
void check_heads(const at::Tensor& t, const char* name, bool written) {
  bool ok = t.stride(-1) == 1 && aligned(t);
  for (int64_t i = 0; i + 1 < t.dim(); ++i) {
    ok = ok && (t.size(i) <= 1 || (t.stride(i) % 8 == 0 && t.stride(i) >= 0));
    VALUE_CHECK(!written || t.size(i) <= 1 || t.stride(i) != 0, name, " is written and must not be expanded");
  }
  VALUE_CHECK(ok, name, " must have contiguous heads that start on 16-byte boundaries");
  if (!written || t.numel() == 0) return;
  int64_t span = t.size(-1), below = 0;  // elements that the dimensions with strides up to `below` span
  for (;;) {
    int64_t next = 0, at = -1;
    for (int64_t i = 0; i + 1 < t.dim(); ++i)
      if (t.size(i) > 1 && t.stride(i) > below && (at < 0 || t.stride(i) < next)) next = t.stride(i), at = i;
    if (at < 0) return;
    int64_t same = 0;
    for (int64_t i = 0; i + 1 < t.dim(); ++i) same += t.size(i) > 1 && t.stride(i) == next;
    VALUE_CHECK(next >= span && same == 1, name, " is written and its rows must not share memory");
    span += (t.size(at) - 1) * next;
    below = next;
  }
}

// Whether the address ranges of two tensors meet.
bool overlaps(const at::Tensor& a, const at::Tensor& b) {
  if (a.numel() == 0 || b.numel() == 0) return false;
  const auto span = [](const at::Tensor& t) {
    int64_t last = 0;
    for (int64_t i = 0; i < t.dim(); ++i) last += (t.size(i) - 1) * t.stride(i);
    const uintptr_t p = reinterpret_cast<uintptr_t>(t.data_ptr());
    return std::make_pair(p, p + (last + 1) * t.element_size());
  };
  const auto x = span(a), y = span(b);
  return x.first < y.second && y.first < x.second;
}

// Whether an element of a may be one of b; both have the same sizes and type. Dimension by dimension from the largest
// stride down: where both have the same, not below what the rest spans, only the two slices can meet whose distance is
// less than it. Other strides count as meeting.
bool share_memory(const at::Tensor& a, const at::Tensor& b) {
  if (!overlaps(a, b)) return false;
  struct Dim {
    int64_t size, a, b;
  };
  std::vector<Dim> dims;
  for (int64_t i = 0; i < a.dim(); ++i)
    if (a.size(i) > 1) dims.push_back({a.size(i), a.stride(i), b.stride(i)});
  std::sort(dims.begin(), dims.end(), [](const Dim& x, const Dim& y) { return x.a > y.a; });
  // Whether the dimensions from i on meet, b's `at` elements behind a's.
  const std::function<bool(size_t, int64_t)> meet = [&](size_t i, int64_t at) {
    int64_t span_a = 1, span_b = 1;
    for (size_t k = i; k < dims.size(); ++k) {
      span_a += (dims[k].size - 1) * dims[k].a;
      span_b += (dims[k].size - 1) * dims[k].b;
    }
    if (at >= span_a || -at >= span_b) return false;
    if (i == dims.size()) return true;
    if (dims[i].a != dims[i].b || dims[i].a < std::max(span_a, span_b) - (dims[i].size - 1) * dims[i].a) return true;
    const int64_t stride = dims[i].a, steps = at >= 0 ? at / stride : -((stride - 1 - at) / stride);
    const int64_t rest = at - steps * stride, last = dims[i].size - 1;
    return (std::abs(steps) <= last && meet(i + 1, rest)) ||
           (std::abs(steps + 1) <= last && meet(i + 1, rest - stride));
  };
  const int64_t bytes = reinterpret_cast<intptr_t>(b.data_ptr()) - reinterpret_cast<intptr_t>(a.data_ptr());
  return bytes % a.element_size() != 0 || meet(0, bytes / a.element_size());
}

Half half_of(const at::Tensor& t) {
  TYPE_CHECK(t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf,
             "paged ops take bfloat16 or float16, got ", t.scalar_type());
  return t.scalar_type() == at::kBFloat16 ? Half::kBf16 : Half::kFp16;
}

Pool pool_of(const at::Tensor& t, const at::Tensor& like, const at::Tensor& first, int64_t hkv, int64_t d,
             const char* name, bool written) {
  VALUE_CHECK(t.dim() == 4 && t.sizes() == first.sizes() && t.size(2) == hkv && t.size(3) == d, name,
              " must be [pages, page_size, ", hkv, ", ", d, "]");
  TYPE_CHECK(t.scalar_type() == like.scalar_type(), name, " must have the type of the input, ", like.scalar_type());
  check_device(t, like, name);
  VALUE_CHECK(t.size(0) >= 1 && t.size(0) < kInt && t.size(1) >= 1 && t.size(1) <= 65536, name,
              " must have pages of 1 to 65536 tokens");
  check_heads(t, name, written);
  for (int i = 0; i < 3; ++i) VALUE_CHECK(t.size(i) == 1 || t.stride(i) > 0, name, " must not be expanded");
  return Pool{t.data_ptr(), t.stride(0), t.stride(1), t.stride(2)};
}

// Types and shapes of the batch were checked when it was made (PagedBatch).
Batch batch_of(const at::Tensor& table, const at::Tensor& kv_len, const OptTensor& q_start, const at::Tensor& like,
               int64_t rows) {
  check_device(table, like, "the batch");
  const int64_t seqs = table.size(0);
  TORCH_CHECK(table.scalar_type() == at::kInt && kv_len.scalar_type() == at::kInt && kv_len.numel() == seqs &&
                  kv_len.device() == table.device() && table.size(1) < kInt && seqs < kInt && rows < kInt,
              "bad batch");
  Batch b{};
  if (q_start.has_value()) {
    TORCH_CHECK(q_start->scalar_type() == at::kInt && q_start->numel() == seqs + 1 &&
                    q_start->device() == table.device(),
                "bad batch");
    b.q_start = q_start->data_ptr<int>();
  } else {
    VALUE_CHECK(rows == seqs, "without q_start every sequence has one new token: ", seqs, " sequences, ", rows,
                " rows");
  }
  b.page_table = table.data_ptr<int>();
  b.kv_len = kv_len.data_ptr<int>();
  b.table_stride = table.stride(0);
  b.seqs = static_cast<int>(seqs);
  b.rows = static_cast<int>(rows);
  b.max_pages = static_cast<int>(table.size(1));
  return b;
}

int* err_of(const at::Tensor& err, const at::Tensor& like) {
  TORCH_CHECK(err.device() == like.device() && err.scalar_type() == at::kInt && err.numel() >= 1,
              "err must be a CUDA int32");
  return err.data_ptr<int>();
}

void check_head_dim(int64_t d) { VALUE_CHECK(d == 64 || d == 128, "head dimension must be 64 or 128, got ", d); }

b200ar::fp8::Type fp8_type(at::ScalarType t, bool wide, const char* name) {
  if (t == at::kBFloat16) return b200ar::fp8::Type::kBf16;
  if (t == at::kHalf) return b200ar::fp8::Type::kFp16;
  TYPE_CHECK(wide && t == at::kFloat, name, " must be bfloat16", wide ? ", float16 or float32" : " or float16");
  return b200ar::fp8::Type::kFp32;
}

void check_k(int64_t k) { VALUE_CHECK(k >= 1 && k % 16 == 0, "K must be a positive multiple of 16, got ", k); }

// [rows, K] with contiguous rows on 16-byte boundaries; copied if x is not laid out like that.
at::Tensor rows_2d(const at::Tensor& x) {
  const at::Tensor t = x.dim() == 2 ? x : x.reshape({-1, x.size(-1)});
  if ((t.size(1) <= 1 || t.stride(1) == 1) && aligned(t) && t.stride(0) >= 0 &&
      (t.size(0) <= 1 || t.stride(0) * t.element_size() % 16 == 0))
    return t;
  return t.clone(at::MemoryFormat::Contiguous);
}

}  // namespace

void register_serving_ops(py::module& m) {
  m.def(
      "qk_norm_rope_paged",
      [](const at::Tensor& qkv, const at::Tensor& table, const at::Tensor& kv_len, const OptTensor& q_start,
         const at::Tensor& cos_t, const at::Tensor& sin_t, const at::Tensor& k_pages, const at::Tensor& v_pages,
         int64_t hq, int64_t hkv, const OptTensor& q_gamma, const OptTensor& k_gamma, const OptTensor& q_out,
         const at::Tensor& err, double eps) {
        VALUE_CHECK(cos_t.dim() == 2, "the rotary table must be fp32 [positions, d / 2]");
        const int64_t d = 2 * cos_t.size(1);
        VALUE_CHECK(hq >= 1 && hkv >= 1 && hq <= 65535 && hkv <= 65535, "hq and hkv must be positive");
        VALUE_CHECK(qkv.dim() == 2 && qkv.size(1) == (hq + 2 * hkv) * d, "qkv must be [rows, (hq + 2 hkv) * ", d,
                    "]");
        const Half type = half_of(qkv);
        check_head_dim(d);
        b200ar::paged::RopeArgs a{};
        a.k = pool_of(k_pages, qkv, k_pages, hkv, d, "k_pages", true);
        a.v = pool_of(v_pages, qkv, k_pages, hkv, d, "v_pages", true);
        check_heads(qkv, "qkv", false);
        VALUE_CHECK(!share_memory(k_pages, v_pages), "k_pages and v_pages share memory");
        VALUE_CHECK(!overlaps(qkv, k_pages) && !overlaps(qkv, v_pages), "qkv overlaps the pools");
        const int64_t rows = qkv.size(0);
        a.batch = batch_of(table, kv_len, q_start, qkv, rows);
        for (const at::Tensor* t : {&cos_t, &sin_t})
          VALUE_CHECK(t->scalar_type() == at::kFloat && t->sizes() == cos_t.sizes() && t->is_contiguous() &&
                          t->device() == qkv.device() && t->size(0) < kInt && aligned(*t),
                      "the rotary table must be contiguous fp32 [positions, d / 2] on ", qkv.device());
        VALUE_CHECK(q_gamma.has_value() == k_gamma.has_value(), "give the norm weights of both q and k, or neither");
        if (q_gamma.has_value())
          for (const at::Tensor* t : {&*q_gamma, &*k_gamma})
            VALUE_CHECK(t->scalar_type() == qkv.scalar_type() && t->dim() == 1 && t->size(0) == d &&
                            t->is_contiguous() && t->device() == qkv.device() && aligned(*t),
                        "the norm weights must be [", d, "], of the type and on the device of qkv");
        const at::cuda::OptionalCUDAGuard guard(device_of(qkv));
        at::Tensor q;
        if (q_out.has_value()) {
          q = *q_out;
          VALUE_CHECK(q.dim() == 3 && q.size(0) == rows && q.size(1) == hq && q.size(2) == d &&
                          q.scalar_type() == qkv.scalar_type() && q.device() == qkv.device(),
                      "q_out must be [rows, hq, d], of the type and on the device of qkv");
          check_heads(q, "q_out", true);
          const bool in_place = q.data_ptr() == qkv.data_ptr() && (rows <= 1 || q.stride(0) == qkv.stride(0)) &&
                                (hq == 1 || q.stride(1) == d);
          VALUE_CHECK(in_place || !overlaps(q, qkv), "q_out overlaps qkv but is not its q part");
          VALUE_CHECK(!overlaps(q, k_pages) && !overlaps(q, v_pages), "q_out overlaps the pools");
        } else {
          q = at::empty({rows, hq, d}, qkv.options());
        }
        a.qkv = qkv.data_ptr();
        a.q_gamma = q_gamma.has_value() ? q_gamma->data_ptr() : nullptr;
        a.k_gamma = k_gamma.has_value() ? k_gamma->data_ptr() : nullptr;
        a.cos_t = cos_t.data_ptr<float>();
        a.sin_t = sin_t.data_ptr<float>();
        a.q_out = q.data_ptr();
        a.qkv_stride = qkv.stride(0);
        a.q_tok = q.stride(0);
        a.q_head = q.stride(1);
        a.err = err_of(err, qkv);
        a.rows = static_cast<int>(rows);
        a.hq = static_cast<int>(hq);
        a.hkv = static_cast<int>(hkv);
        a.positions = static_cast<int>(cos_t.size(0));
        a.num_pages = static_cast<int>(k_pages.size(0));
        a.page_size = static_cast<int>(k_pages.size(1));
        a.eps = static_cast<float>(eps);
        b200ar::paged::qk_norm_rope_paged(a, static_cast<int>(d), type, stream_of());
        return q;
      },
      "norms of q and k, rotary embedding and the write into a paged KV cache", py::arg("qkv"), py::arg("page_table"),
      py::arg("kv_len"), py::arg("q_start"), py::arg("cos_t"), py::arg("sin_t"), py::arg("k_pages"),
      py::arg("v_pages"), py::arg("hq"), py::arg("hkv"), py::arg("q_gamma"), py::arg("k_gamma"), py::arg("q_out"),
      py::arg("err"), py::arg("eps"));
  m.def(
      "paged_attention",
      [](const at::Tensor& q, const at::Tensor& k_pages, const at::Tensor& v_pages, const at::Tensor& table,
         const at::Tensor& kv_len, const OptTensor& q_start, const OptTensor& out_opt, const at::Tensor& err,
         std::optional<double> scale, bool causal, int64_t window) {
        VALUE_CHECK(q.dim() == 3, "q must be [rows, heads, d]");
        const int64_t rows = q.size(0), hq = q.size(1), d = q.size(2);
        const Half type = half_of(q);
        check_head_dim(d);
        VALUE_CHECK(k_pages.dim() == 4, "k_pages must be [pages, page_size, kv_heads, d]");
        const int64_t hkv = k_pages.size(2);
        VALUE_CHECK(hkv >= 1 && hq >= hkv && hq <= 65535 && hq % hkv == 0,
                    "query heads must be a multiple of the KV heads");
        VALUE_CHECK(k_pages.size(1) % 8 == 0, "the page size must be a multiple of 8, got ", k_pages.size(1));
        VALUE_CHECK(window >= 0 && (causal || window == 0),
                    "window must be 0 (all) or a number of positions, with causal attention");
        b200ar::paged::AttnArgs a{};
        a.scale = static_cast<float>(scale.has_value() ? *scale : 1.0 / std::sqrt(static_cast<double>(d)));
        VALUE_CHECK(std::isfinite(a.scale), "scale must be finite");
        a.k = pool_of(k_pages, q, k_pages, hkv, d, "k_pages", false);
        a.v = pool_of(v_pages, q, k_pages, hkv, d, "v_pages", false);
        for (const at::Tensor* t : {&k_pages, &v_pages})  // heads are counted in units of 64 values (pool_map())
          VALUE_CHECK(hkv == 1 || t->stride(2) % 64 == 0, "the pools' heads must be a multiple of 64 values apart");
        check_heads(q, "q", false);
        a.batch = batch_of(table, kv_len, q_start, q, rows);
        const at::cuda::OptionalCUDAGuard guard(device_of(q));
        at::Tensor out;
        a.o_head = d;
        if (out_opt.has_value()) {
          out = *out_opt;
          VALUE_CHECK(out.dim() == 2 && out.size(0) == rows && out.size(1) == hq * d &&
                          out.scalar_type() == q.scalar_type() && out.device() == q.device(),
                      "out must be [rows, hq * d], of the type and on the device of q");
          check_heads(out, "out", true);
          VALUE_CHECK(!overlaps(out, q) && !overlaps(out, k_pages) && !overlaps(out, v_pages),
                      "out overlaps an input");
        } else {
          out = at::empty({rows, hq * d}, q.options());
        }
        a.q = q.data_ptr();
        a.out = out.data_ptr();
        a.q_tok = q.stride(0);
        a.q_head = q.stride(1);
        a.o_tok = out.stride(0);
        a.err = err_of(err, q);
        a.rows = static_cast<int>(rows);
        a.hq = static_cast<int>(hq);
        a.hkv = static_cast<int>(hkv);
        a.num_pages = static_cast<int>(k_pages.size(0));
        a.page_size = static_cast<int>(k_pages.size(1));
        const int64_t capacity = std::min<int64_t>(table.size(1) * k_pages.size(1), 1 << 30);
        a.capacity = static_cast<int>(capacity);
        a.window = window >= capacity ? 0 : static_cast<int>(window);  // a window over every position hides nothing
        a.causal = causal;
        // From the caching allocator on this stream: concurrent calls, eager or captured, never share it.
        const at::Tensor workspace =
            at::empty({b200ar::paged::paged_attention_workspace(rows, a.hq, a.hkv, static_cast<int>(d))},
                      q.options().dtype(at::kFloat));
        b200ar::paged::paged_attention(a, static_cast<int>(d), type, workspace.data_ptr<float>(), stream_of());
        return out;
      },
      "attention of new tokens over a paged KV cache", py::arg("q"), py::arg("k_pages"), py::arg("v_pages"),
      py::arg("page_table"), py::arg("kv_len"), py::arg("q_start"), py::arg("out"), py::arg("err"), py::arg("scale"),
      py::arg("causal"), py::arg("window"));
  m.def(
      "quantize_fp8",
      [](const at::Tensor& x) {
        const b200ar::fp8::Type type = fp8_type(x.scalar_type(), true, "x");
        VALUE_CHECK(x.dim() >= 1, "x must be [..., K]");
        check_k(x.size(-1));
        const at::cuda::OptionalCUDAGuard guard(device_of(x));
        const at::Tensor x2 = rows_2d(x);
        const int64_t M = x2.size(0), K = x2.size(1), blocks = (K + 127) / 128;
        at::Tensor q = at::empty(x.sizes(), x.options().dtype(at::kFloat8_e4m3fn));
        at::Tensor scale = at::empty({blocks, M}, x.options().dtype(at::kFloat));
        b200ar::fp8::quantize(x2.data_ptr(), x2.stride(0), static_cast<uint8_t*>(q.data_ptr()),
                              scale.data_ptr<float>(), M, M, K, type, nullptr, 0, stream_of());
        std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end());
        shape.back() = blocks;
        std::vector<int64_t> strides(shape.size());
        strides.back() = M;
        for (int64_t i = static_cast<int64_t>(shape.size()) - 2, n = 1; i >= 0; --i) {
          strides[i] = n;
          n *= shape[i];
        }
        return std::make_pair(q, scale.as_strided(shape, strides));
      },
      "e4m3 values and a scale for each row and block of 128", py::arg("x"));
  m.def(
      "quantize_fp8_weight",
      [](const at::Tensor& w) {
        const b200ar::fp8::Type type = fp8_type(w.scalar_type(), true, "w");
        VALUE_CHECK(w.dim() == 2, "w must be [N, K]");
        check_k(w.size(1));
        const at::cuda::OptionalCUDAGuard guard(device_of(w));
        const at::Tensor w2 = rows_2d(w);
        const int64_t N = w2.size(0), K = w2.size(1);
        at::Tensor q = at::empty({N, K}, w.options().dtype(at::kFloat8_e4m3fn));
        at::Tensor scale = at::empty({(N + 127) / 128, (K + 127) / 128}, w.options().dtype(at::kFloat));
        b200ar::fp8::quantize_weight(w2.data_ptr(), w2.stride(0), static_cast<uint8_t*>(q.data_ptr()),
                                     scale.data_ptr<float>(), N, K, type, stream_of());
        return std::make_pair(q, scale);
      },
      "e4m3 values and a scale for each 128 x 128 block", py::arg("w"));
  m.def("linear_fp8_takes_pairs", &b200ar::fp8::linear_takes_pairs,
        "whether linear_fp8 runs these sizes on the kernel for many rows (tests)", py::arg("m"), py::arg("n"),
        py::arg("k"));
  m.def(
      "linear_fp8",
      [](const at::Tensor& x, const at::Tensor& w, const at::Tensor& w_scale, const OptTensor& out_opt,
         const OptTensor& x_scale, const OptTensor& like, const at::Tensor& err) {
        TYPE_CHECK(w.dim() == 2 && w.scalar_type() == at::kFloat8_e4m3fn && w.is_contiguous() && aligned(w),
                   "w_q must be contiguous float8_e4m3fn [N, K]");
        const int64_t N = w.size(0), K = w.size(1), blocks = (K + 127) / 128;
        check_k(K);
        VALUE_CHECK(N >= 1 && N % 8 == 0, "N must be a positive multiple of 8, got ", N);
        VALUE_CHECK(x.dim() >= 1 && x.size(-1) == K, "x must be [..., ", K, "]");
        VALUE_CHECK(w_scale.scalar_type() == at::kFloat && w_scale.is_contiguous() && w_scale.dim() == 2 &&
                        w_scale.size(0) == (N + 127) / 128 && w_scale.size(1) == blocks,
                    "w_scale must be contiguous fp32 [", (N + 127) / 128, ", ", blocks, "]");
        check_device(w, x, "w_q");
        check_device(w_scale, x, "w_scale");
        // The output's type: that of x, or with x_scale that of the empty tensor `like`.
        const at::ScalarType dtype = x_scale.has_value() ? like->scalar_type() : x.scalar_type();
        const b200ar::fp8::Type type = fp8_type(dtype, false, x_scale.has_value() ? "dtype" : "x");
        const at::cuda::OptionalCUDAGuard guard(device_of(x));
        const cudaStream_t s = stream_of();
        const int64_t M = x.numel() / K;
        at::Tensor out;
        if (out_opt.has_value()) {
          out = *out_opt;
          bool same = out.dim() == x.dim() && out.scalar_type() == dtype && out.size(-1) == N;
          for (int64_t i = 0; same && i + 1 < x.dim(); ++i) same = out.size(i) == x.size(i);
          VALUE_CHECK(same && out.device() == x.device(), "out must be ", dtype, " [..., ", N, "] on ", x.device());
        } else {
          std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end());
          shape.back() = N;
          out = at::empty(shape, x.options().dtype(dtype));
        }
        const at::Tensor out2 = out.dim() == 2 ? out : out.view({M, N});
        check_heads(out2, "out", true);
        VALUE_CHECK(!overlaps(out, x) && !overlaps(out, w) && !overlaps(out, w_scale) &&
                        !(x_scale.has_value() && overlaps(out, *x_scale)),
                    "out overlaps an input");
        b200ar::fp8::LinearArgs a{};
        a.w = static_cast<const uint8_t*>(w.data_ptr());
        a.sw = w_scale.data_ptr<float>();
        a.out = out2.data_ptr();
        a.ldo = out2.stride(0);
        a.M = M;
        a.N = N;
        a.K = K;
        a.err = err_of(err, x);
        at::Tensor x2, sx;
        if (x_scale.has_value()) {
          TYPE_CHECK(x.scalar_type() == at::kFloat8_e4m3fn, "with x_scale, x must be float8_e4m3fn");
          bool same = x_scale->dim() == x.dim() && x_scale->scalar_type() == at::kFloat && x_scale->size(-1) == blocks;
          for (int64_t i = 0; same && i + 1 < x.dim(); ++i) same = x_scale->size(i) == x.size(i);
          VALUE_CHECK(same && x_scale->device() == x.device(), "x_scale must be fp32 [..., ", blocks, "] on ",
                      x.device());
          x2 = x.reshape({M, K}).contiguous();
          if (!aligned(x2)) x2 = x2.clone();
          sx = x_scale->reshape({M, blocks}).t();
          if ((M > 1 && sx.stride(1) != 1) || sx.stride(0) < M) sx = sx.contiguous();
          a.x = static_cast<const uint8_t*>(x2.data_ptr());
          a.sx = sx.data_ptr<float>();
          a.lds = sx.stride(0);
        } else {
          x2 = rows_2d(x);
          a.raw = x2.data_ptr();
          a.ldx = x2.stride(0);
        }
        // From the caching allocator on this stream: concurrent calls, eager or captured, never share it.
        const int64_t bytes = b200ar::fp8::linear_scratch(a);
        at::Tensor scratch;
        if (bytes > 0) scratch = at::empty({bytes}, x.options().dtype(at::kByte));
        b200ar::fp8::linear(a, type, bytes > 0 ? scratch.data_ptr() : nullptr, s);
        return out;
      },
      "product of e4m3 operands with block scales; x is quantized unless it comes with its scales", py::arg("x"),
      py::arg("w_q"), py::arg("w_scale"), py::arg("out"), py::arg("x_scale"), py::arg("like"), py::arg("err"));
}
