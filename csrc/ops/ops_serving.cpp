// Binds the serving operators: paged rotary step, paged attention, 8-bit linear.
//
// Every check of types, sizes, strides and devices that keeps a kernel inside
// its tensors is made here; what only the device knows (lengths, offsets,
// pages) is checked by the kernels, which leave a code in the error word.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <algorithm>
#include <optional>

#include "../fp8/fp8.h"
#include "../paged/paged.h"
#include "ops.h"

namespace py = pybind11;

namespace {

using b200ar::paged::Batch;
using b200ar::paged::Half;
using b200ar::paged::Pool;

constexpr int64_t kInt = 0x7fffffff;

cudaStream_t stream_of() { return at::cuda::getCurrentCUDAStream().stream(); }

void check_device(const at::Tensor& t, const at::Tensor& like, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.device() == like.device(), name, " must be on ", like.device(), ", got ", t.device());
}

// [rows, heads, d] with any strides that keep 16-byte packets aligned.
void check_rows(const at::Tensor& t, const char* name) {
  TORCH_CHECK(t.dim() == 3 && t.size(0) <= kInt && t.size(1) <= 65535, name, " must be [rows, heads, d]");
  TORCH_CHECK(t.stride(2) == 1 && t.stride(1) % 8 == 0 && t.stride(0) % 8 == 0 && t.stride(0) >= 0 && t.stride(1) >= 0 &&
                  reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0,
              name, " must have contiguous heads that start on 16-byte boundaries");
}

Half half_of(const at::Tensor& t, const char* name) {
  TORCH_CHECK(t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf, name, " must be bfloat16 or float16");
  return t.scalar_type() == at::kBFloat16 ? Half::kBf16 : Half::kFp16;
}

Pool pool_of(const at::Tensor& t, const at::Tensor& like, const at::Tensor& first, int64_t hkv, int64_t d,
             const char* name) {
  check_device(t, like, name);
  TORCH_CHECK(t.scalar_type() == like.scalar_type(), name, " must have the type of the queries");
  TORCH_CHECK(t.dim() == 4 && t.size(2) == hkv && t.size(3) == d && t.sizes() == first.sizes(), name,
              " must be [pages, page_size, kv_heads, d]");
  TORCH_CHECK(t.size(0) >= 1 && t.size(0) < kInt && t.size(1) >= 1 && t.size(1) <= 65536, name,
              " must have pages of 1 to 65536 tokens");
  TORCH_CHECK(t.stride(3) == 1 && t.stride(2) % 8 == 0 && t.stride(1) % 8 == 0 && t.stride(0) % 8 == 0 &&
                  t.stride(0) >= 0 && t.stride(1) >= 0 && t.stride(2) >= 0 &&
                  reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0,
              name, " must have contiguous heads that start on 16-byte boundaries");
  for (int i = 0; i < 3; ++i) TORCH_CHECK(t.size(i) == 1 || t.stride(i) > 0, name, " must not be expanded");
  return Pool{t.data_ptr(), t.stride(0), t.stride(1), t.stride(2)};
}

Batch batch_of(const at::Tensor& table, const at::Tensor& kv_len, const std::optional<at::Tensor>& q_start,
               const at::Tensor& like, int64_t rows) {
  check_device(table, like, "page_table");
  check_device(kv_len, like, "kv_len");
  TORCH_CHECK(table.scalar_type() == at::kInt && table.dim() == 2 && (table.size(1) <= 1 || table.stride(1) == 1) &&
                  table.stride(0) >= 0 && table.size(0) < kInt && table.size(1) < kInt,
              "page_table must be int32 [sequences, pages] with contiguous rows");
  const int64_t seqs = table.size(0);
  TORCH_CHECK(kv_len.scalar_type() == at::kInt && kv_len.dim() == 1 && kv_len.size(0) == seqs &&
                  kv_len.is_contiguous(),
              "kv_len must be int32 [sequences]");
  Batch b{};
  if (q_start.has_value()) {
    check_device(*q_start, like, "q_start");
    TORCH_CHECK(q_start->scalar_type() == at::kInt && q_start->dim() == 1 && q_start->size(0) == seqs + 1 &&
                    q_start->is_contiguous(),
                "q_start must be int32 [sequences + 1]");
    b.q_start = q_start->data_ptr<int>();
  } else {
    TORCH_CHECK(rows == seqs, "without q_start every sequence has one new token: ", seqs, " sequences, ", rows,
                " rows");
  }
  b.page_table = table.data_ptr<int>();
  b.kv_len = kv_len.data_ptr<int>();
  b.table_stride = table.stride(0);
  b.seqs = static_cast<int>(seqs);
  b.max_pages = static_cast<int>(table.size(1));
  return b;
}

int* err_of(const at::Tensor& err, const at::Tensor& like) {
  check_device(err, like, "err");
  TORCH_CHECK(err.scalar_type() == at::kInt && err.numel() >= 1, "err must be a CUDA int32");
  return err.data_ptr<int>();
}

b200ar::fp8::Type fp8_type(const at::Tensor& t, bool wide, const char* name) {
  if (t.scalar_type() == at::kBFloat16) return b200ar::fp8::Type::kBf16;
  if (t.scalar_type() == at::kHalf) return b200ar::fp8::Type::kFp16;
  TORCH_CHECK(wide && t.scalar_type() == at::kFloat, name, " must be bfloat16", wide ? ", float16 or float32" : " or float16");
  return b200ar::fp8::Type::kFp32;
}

void check_rows_2d(const at::Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.dim() == 2 && (t.size(1) <= 1 || t.stride(1) == 1) &&
                  t.stride(0) * t.element_size() % 16 == 0 && t.stride(0) >= 0 &&
                  reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0,
              name, " must be a 2-D CUDA tensor with contiguous rows that start on 16-byte boundaries");
}

void check_codes(const at::Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.dim() == 2 && t.is_contiguous() && t.scalar_type() == at::kFloat8_e4m3fn &&
                  reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0,
              name, " must be a contiguous 2-D float8_e4m3fn CUDA tensor");
}

}  // namespace

void register_serving_ops(py::module& m) {
  m.def(
      "qk_norm_rope_paged",
      [](const at::Tensor& qkv, const at::Tensor& table, const at::Tensor& kv_len,
         const std::optional<at::Tensor>& q_start, const at::Tensor& cos_t, const at::Tensor& sin_t,
         at::Tensor& k_pages, at::Tensor& v_pages, const std::optional<at::Tensor>& q_gamma,
         const std::optional<at::Tensor>& k_gamma, at::Tensor& q_out, at::Tensor& err, double eps) {
        TORCH_CHECK(qkv.is_cuda() && qkv.dim() == 2, "qkv must be a CUDA tensor [rows, (hq + 2 hkv) * d]");
        const Half type = half_of(qkv, "qkv");
        check_rows(q_out, "q_out");
        check_device(q_out, qkv, "q_out");
        TORCH_CHECK(q_out.scalar_type() == qkv.scalar_type() && q_out.size(0) == qkv.size(0),
                    "q_out must have the type and the rows of qkv");
        TORCH_CHECK(k_pages.dim() == 4, "k_pages must be [pages, page_size, kv_heads, d]");
        const int64_t hq = q_out.size(1), d = q_out.size(2), hkv = k_pages.size(2);
        TORCH_CHECK(hq >= 1 && hkv >= 1 && qkv.size(1) == (hq + 2 * hkv) * d, "qkv must be [rows, (hq + 2 hkv) * d]");
        TORCH_CHECK((qkv.stride(1) == 1) && qkv.stride(0) % 8 == 0 && qkv.stride(0) >= 0 &&
                        reinterpret_cast<uintptr_t>(qkv.data_ptr()) % 16 == 0,
                    "qkv must have contiguous rows that start on 16-byte boundaries");
        b200ar::paged::RopeArgs a{};
        a.k = pool_of(k_pages, qkv, k_pages, hkv, d, "k_pages");
        a.v = pool_of(v_pages, qkv, k_pages, hkv, d, "v_pages");
        a.batch = batch_of(table, kv_len, q_start, qkv, qkv.size(0));
        for (const at::Tensor* t : {&cos_t, &sin_t}) {
          check_device(*t, qkv, "the rotary table");
          TORCH_CHECK(t->scalar_type() == at::kFloat && t->dim() == 2 && t->size(1) == d / 2 && t->is_contiguous() &&
                          t->size(0) < kInt && t->sizes() == cos_t.sizes(),
                      "the rotary table must be fp32 [positions, d / 2]");
        }
        TORCH_CHECK(q_gamma.has_value() == k_gamma.has_value(), "give the norm weights of both q and k, or neither");
        if (q_gamma.has_value())
          for (const at::Tensor* t : {&*q_gamma, &*k_gamma}) {
            check_device(*t, qkv, "the norm weights");
            TORCH_CHECK(t->scalar_type() == qkv.scalar_type() && t->numel() == d && t->is_contiguous() &&
                            reinterpret_cast<uintptr_t>(t->data_ptr()) % 16 == 0,
                        "the norm weights must be [d], of the type of qkv");
          }
        a.qkv = qkv.data_ptr();
        a.q_gamma = q_gamma.has_value() ? q_gamma->data_ptr() : nullptr;
        a.k_gamma = k_gamma.has_value() ? k_gamma->data_ptr() : nullptr;
        a.cos_t = cos_t.data_ptr<float>();
        a.sin_t = sin_t.data_ptr<float>();
        a.q_out = q_out.data_ptr();
        a.qkv_stride = qkv.stride(0);
        a.q_tok = q_out.stride(0);
        a.q_head = q_out.stride(1);
        a.err = err_of(err, qkv);
        a.rows = static_cast<int>(qkv.size(0));
        a.hq = static_cast<int>(hq);
        a.hkv = static_cast<int>(hkv);
        a.positions = static_cast<int>(cos_t.size(0));
        a.num_pages = static_cast<int>(k_pages.size(0));
        a.page_size = static_cast<int>(k_pages.size(1));
        a.eps = static_cast<float>(eps);
        const at::cuda::OptionalCUDAGuard guard(device_of(qkv));
        b200ar::paged::qk_norm_rope_paged(a, static_cast<int>(d), type, stream_of());
      },
      "norms of q and k, rotary embedding and the write into a paged KV cache", py::arg("qkv"), py::arg("page_table"),
      py::arg("kv_len"), py::arg("q_start"), py::arg("cos_t"), py::arg("sin_t"), py::arg("k_pages"),
      py::arg("v_pages"), py::arg("q_gamma"), py::arg("k_gamma"), py::arg("q_out"), py::arg("err"), py::arg("eps"));
  m.def(
      "paged_attention",
      [](const at::Tensor& q, const at::Tensor& k_pages, const at::Tensor& v_pages, const at::Tensor& table,
         const at::Tensor& kv_len, const std::optional<at::Tensor>& q_start, at::Tensor& out, at::Tensor& err,
         double scale, bool causal, int64_t window) {
        TORCH_CHECK(q.is_cuda(), "q must be a CUDA tensor");
        const Half type = half_of(q, "q");
        check_rows(q, "q");
        check_rows(out, "out");
        check_device(out, q, "out");
        TORCH_CHECK(out.scalar_type() == q.scalar_type() && out.sizes() == q.sizes(), "out must be like q");
        TORCH_CHECK(k_pages.dim() == 4, "k_pages must be [pages, page_size, kv_heads, d]");
        const int64_t hq = q.size(1), d = q.size(2), hkv = k_pages.size(2);
        TORCH_CHECK(hkv >= 1 && hq >= hkv && hq % hkv == 0, "query heads must be a multiple of the KV heads");
        TORCH_CHECK(k_pages.size(1) % 8 == 0, "the page size must be a multiple of 8");
        TORCH_CHECK(window >= 0 && window <= kInt && (causal || window == 0),
                    "window must be 0 (all) or a number of positions, with causal attention");
        b200ar::paged::AttnArgs a{};
        a.k = pool_of(k_pages, q, k_pages, hkv, d, "k_pages");
        a.v = pool_of(v_pages, q, k_pages, hkv, d, "v_pages");
        a.batch = batch_of(table, kv_len, q_start, q, q.size(0));
        a.q = q.data_ptr();
        a.out = out.data_ptr();
        a.q_tok = q.stride(0);
        a.q_head = q.stride(1);
        a.o_tok = out.stride(0);
        a.o_head = out.stride(1);
        a.err = err_of(err, q);
        a.rows = static_cast<int>(q.size(0));
        a.hq = static_cast<int>(hq);
        a.hkv = static_cast<int>(hkv);
        a.num_pages = static_cast<int>(k_pages.size(0));
        a.page_size = static_cast<int>(k_pages.size(1));
        const int64_t capacity = std::min<int64_t>(table.size(1) * k_pages.size(1), 1 << 30);
        a.capacity = static_cast<int>(capacity);
        a.window = window >= capacity ? 0 : static_cast<int>(window);  // a window over every position hides nothing
        a.causal = causal;
        a.scale = static_cast<float>(scale);
        const at::cuda::OptionalCUDAGuard guard(device_of(q));
        // From the caching allocator on this stream: concurrent calls, eager or captured, never share it.
        const at::Tensor workspace =
            at::empty({b200ar::paged::paged_attention_workspace(q.size(0), a.hq, a.hkv, static_cast<int>(d))},
                      q.options().dtype(at::kFloat));
        b200ar::paged::paged_attention(a, static_cast<int>(d), type, workspace.data_ptr<float>(), stream_of());
      },
      "attention of new tokens over a paged KV cache", py::arg("q"), py::arg("k_pages"), py::arg("v_pages"),
      py::arg("page_table"), py::arg("kv_len"), py::arg("q_start"), py::arg("out"), py::arg("err"), py::arg("scale"),
      py::arg("causal"), py::arg("window"));
  m.def(
      "quantize_fp8",
      [](const at::Tensor& x, at::Tensor& q, at::Tensor& scale) {
        check_rows_2d(x, "x");
        check_codes(q, "q");
        check_device(q, x, "q");
        check_device(scale, x, "scale");
        const int64_t M = x.size(0), K = x.size(1), blocks = (K + 127) / 128;
        TORCH_CHECK(q.sizes() == x.sizes(), "q must have the shape of x");
        TORCH_CHECK(scale.scalar_type() == at::kFloat && scale.dim() == 2 && scale.size(0) == blocks &&
                        scale.size(1) == M && (M <= 1 || scale.stride(1) == 1) && scale.stride(0) >= M,
                    "scale must be fp32 [ceil(K / 128), M]");
        const at::cuda::OptionalCUDAGuard guard(device_of(x));
        b200ar::fp8::quantize(x.data_ptr(), x.stride(0), static_cast<uint8_t*>(q.data_ptr()),
                              scale.data_ptr<float>(), scale.stride(0), M, K, fp8_type(x, true, "x"), nullptr, 0,
                              stream_of());
      },
      "e4m3 values and a scale for each row and block of 128", py::arg("x"), py::arg("q"), py::arg("scale"));
  m.def(
      "quantize_fp8_weight",
      [](const at::Tensor& w, at::Tensor& q, at::Tensor& scale) {
        check_rows_2d(w, "w");
        check_codes(q, "q");
        check_device(q, w, "q");
        check_device(scale, w, "scale");
        TORCH_CHECK(q.sizes() == w.sizes(), "q must have the shape of w");
        TORCH_CHECK(scale.scalar_type() == at::kFloat && scale.is_contiguous() && scale.dim() == 2 &&
                        scale.size(0) == (w.size(0) + 127) / 128 && scale.size(1) == (w.size(1) + 127) / 128,
                    "scale must be fp32 [ceil(N / 128), ceil(K / 128)]");
        const at::cuda::OptionalCUDAGuard guard(device_of(w));
        b200ar::fp8::quantize_weight(w.data_ptr(), w.stride(0), static_cast<uint8_t*>(q.data_ptr()),
                                     scale.data_ptr<float>(), w.size(0), w.size(1), fp8_type(w, true, "w"),
                                     stream_of());
      },
      "e4m3 values and a scale for each 128 x 128 block", py::arg("w"), py::arg("q"), py::arg("scale"));
  m.def(
      "linear_fp8",
      [](const at::Tensor& x, const std::optional<at::Tensor>& x_scale, const at::Tensor& w,
         const at::Tensor& w_scale, at::Tensor& out, at::Tensor& err) {
        check_codes(w, "w_q");
        TORCH_CHECK(x.dim() == 2, "x must be [M, K]");
        const int64_t M = x.size(0), K = x.size(1), N = w.size(0), blocks = (K + 127) / 128;
        check_device(w, x, "w_q");
        check_device(out, x, "out");
        check_device(w_scale, x, "w_scale");
        TORCH_CHECK(w.size(1) == K, "x and w_q must have the same K");
        TORCH_CHECK(w_scale.scalar_type() == at::kFloat && w_scale.is_contiguous() && w_scale.dim() == 2 &&
                        w_scale.size(0) == (N + 127) / 128 && w_scale.size(1) == blocks,
                    "w_scale must be fp32 [ceil(N / 128), ceil(K / 128)]");
        check_rows_2d(out, "out");
        TORCH_CHECK(out.size(0) == M && out.size(1) == N, "out must be [M, N]");
        const b200ar::fp8::Type type = fp8_type(out, false, "out");
        const at::cuda::OptionalCUDAGuard guard(device_of(x));
        const cudaStream_t s = stream_of();
        b200ar::fp8::LinearArgs a{};
        a.w = static_cast<const uint8_t*>(w.data_ptr());
        a.sw = w_scale.data_ptr<float>();
        a.out = out.data_ptr();
        a.ldo = out.stride(0);
        a.M = M;
        a.N = N;
        a.K = K;
        a.err = err_of(err, x);
        // Scratch from the caching allocator on this stream: concurrent calls, eager or captured, never share it.
        const b200ar::fp8::Scratch need = b200ar::fp8::linear_scratch(a);
        const auto bytes = x.options().dtype(at::kByte);
        const at::Tensor scratch = at::empty({need.floats * 4 + need.counters * 4}, bytes);
        a.workspace = static_cast<float*>(scratch.data_ptr());
        a.counters = reinterpret_cast<unsigned*>(a.workspace + need.floats);
        at::Tensor codes, scales;
        if (x_scale.has_value()) {
          check_codes(x, "x");
          check_device(*x_scale, x, "x_scale");
          TORCH_CHECK(x_scale->scalar_type() == at::kFloat && x_scale->dim() == 2 && x_scale->size(0) == blocks &&
                          x_scale->size(1) == M && (M <= 1 || x_scale->stride(1) == 1) && x_scale->stride(0) >= M,
                      "x_scale must be fp32 [ceil(K / 128), M]");
          a.x = static_cast<const uint8_t*>(x.data_ptr());
          a.sx = x_scale->data_ptr<float>();
          a.lds = x_scale->stride(0);
          if (M > 0 && need.counters) C10_CUDA_CHECK(cudaMemsetAsync(a.counters, 0, need.counters * 4, s));
        } else {
          check_rows_2d(x, "x");
          codes = at::empty({M, K}, bytes);
          scales = at::empty({blocks, M}, x.options().dtype(at::kFloat));
          a.x = codes.data_ptr<uint8_t>();
          a.sx = scales.data_ptr<float>();
          a.lds = M;
          a.early = true;
          b200ar::fp8::quantize(x.data_ptr(), x.stride(0), codes.data_ptr<uint8_t>(), scales.data_ptr<float>(), M, M,
                                K, fp8_type(x, false, "x"), a.counters, need.counters, s);
        }
        b200ar::fp8::linear(a, type, s);
      },
      "product of e4m3 operands with block scales; x is quantized unless it comes with its scales", py::arg("x"),
      py::arg("x_scale"), py::arg("w"), py::arg("w_scale"), py::arg("out"), py::arg("err"));
}
