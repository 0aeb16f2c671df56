"""Cases and plain forms of the serving operators: the rotary step that writes a
paged KV cache, attention over that cache, and the 8-bit linear layer.

Each operator has a plain form in elementary torch operations, the call a user
of the framework makes, and the same mathematics once more in 64 bits. Head
layouts are those of a tensor-parallel decoder with 64 query and 8 key-value
heads of 128 (all of it on one GPU, or 1/4 or 1/8 of it per rank), and of a
smaller one with heads of 64; the linear layers are its projections.

A batch is S sequences with `new` tokens each on top of `past` cached ones. The
lengths of a case follow from its plain values alone (see `lengths`).
"""

import math
import random

import torch

own = False

BLOCK = 128  # one scale for each 128 values along K (and 128 rows of a weight)
E4M3_MAX = 448.0
EPS = 1e-5
THETA = 500000.0
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ------------------------------------------------------------------ cases
def listed():
    return [
        # One conversation, one new token: rank 0 of 8, the smallest call of a decode step.
        _paged("rope_decode_1", "rope", 8, 1, 128, "bf16", 64, 1, (1, 1), (2048, 2048), norm=True),
        # A full decode batch on one GPU, no norm (a model without query and key norms), small pages.
        _paged("rope_decode_64", "rope", 64, 8, 64, "fp16", 16, 64, (1, 1), (1, 4000), norm=False),
        # Prompts of a batch in one step, ragged, some continued, two padding rows at the end.
        _paged("rope_prompts", "rope", 64, 8, 128, "bf16", 64, 5, (611, 2717), (0, 1500), norm=True, pad=2),
        # One conversation, one new token over 2048 cached ones on one rank of 8: latency.
        _paged("attention_decode_1", "attention", 8, 1, 128, "bf16", 64, 1, (1, 1), (2048, 2048)),
        # A full decode batch with contexts of all lengths: streaming the cache.
        _paged("attention_decode_64", "attention", 64, 8, 128, "bf16", 16, 64, (1, 1), (1, 4095)),
        # One chunk of a long prompt on one rank of 8: few heads, a long cache.
        _paged("attention_chunk_long", "attention", 8, 1, 128, "bf16", 128, 1, (512, 512), (32307, 32307)),
        # One large chunk with every head: the matrix products.
        _paged("attention_chunk_large", "attention", 64, 8, 128, "bf16", 64, 1, (4096, 4096), (4096, 4096)),
        # A mixed step: prompts' chunks and single tokens together, a sliding window, heads of 64, odd pages.
        _paged("attention_mixed", "attention", 16, 2, 64, "fp16", 24, 24, (1, 700), (0, 6000), window=1500, pad=3,
               ones=True),
        # One token through the gate-up projection of one rank of 8.
        _linear("linear_decode_1", "bf16", 1, 7168, 8192),
        # A decode batch through the down projection of one rank of 8.
        _linear("linear_decode_48", "bf16", 48, 8192, 3584),
        # Sizes that no tile and no block divides.
        _linear("linear_odd", "fp16", 333, 1288, 1040),
        # A prompt through the gate-up projection.
        _linear("linear_prompt", "bf16", 4093, 7168, 8192),
    ]


def _paged(name, op, hq, hkv, d, dtype, page, seqs, new, past, norm=False, window=0, pad=0, ones=False, shuffle=7):
    return {"name": name, "op": op, "hq": hq, "hkv": hkv, "d": d, "dtype": dtype, "page": page, "seqs": seqs,
            "new_lo": new[0], "new_hi": new[1], "past_lo": past[0], "past_hi": past[1], "norm": norm,
            "window": window, "pad": pad, "ones": ones, "shuffle": shuffle}


def _linear(name, dtype, m, n, k):
    return {"name": name, "op": "linear", "dtype": dtype, "m": m, "n": n, "k": k}


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the ranges that the listed ones stand for."""
    op = rng.choice(["rope", "attention", "attention", "linear"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if op == "linear":
        n, k = 8 * _log_int(rng, 64, 1280), 16 * _log_int(rng, 32, 512)
        case = _linear("", dtype, _log_int(rng, 1, 4096), n, k)
        del case["name"]
        return case
    hq, hkv = rng.choice([(64, 8), (16, 2), (8, 1), (8, 8), (12, 4), (7, 1), (32, 2)])
    d = rng.choice([64, 128])
    page = rng.choice([8, 16, 24, 32, 48, 64, 128, 256])
    shuffle = rng.randrange(1 << 20)
    kind = rng.choice(["decode", "chunk", "mixed"])
    if kind == "decode":
        seqs = _log_int(rng, 1, 96)
        hi = _log_int(rng, 16, 4096 if hkv == 8 else 16384)
        new, past = (1, 1), (0, hi)
    elif kind == "chunk":
        seqs = rng.randint(1, 3)
        hi = _log_int(rng, 2, 2048 if hq == 64 else 4096) // seqs + 1
        new, past = (max(1, hi // 2), hi), (0, _log_int(rng, 1, 4000 if hq == 64 else 16000))
    else:
        seqs = _log_int(rng, 2, 32)
        new, past = (1, _log_int(rng, 2, 400)), (0, _log_int(rng, 16, 4000))
    case = _paged("", op, hq, hkv, d, dtype, page, seqs, new, past, norm=rng.random() < 0.7,
                  window=rng.choice([0, 0, 0, _log_int(rng, 1, 4000)]), pad=rng.choice([0, 0, rng.randint(1, 9)]),
                  ones=kind == "mixed" and rng.random() < 0.5, shuffle=shuffle)
    if op == "rope":
        case["window"] = 0
    else:
        case["norm"] = False
    del case["name"]
    return case


def lengths(case):
    """(new tokens, tokens in the cache with them) of every sequence of a case."""
    rng = random.Random(case["shuffle"])
    new, total = [], []
    for i in range(case["seqs"]):
        n = rng.randint(case["new_lo"], case["new_hi"])
        if case["ones"] and i % 3:
            n = 1
        new.append(n)
        total.append(n + rng.randint(case["past_lo"], case["past_hi"]))
    return new, total


def _visible(n, total, window):
    """Positions that the n last of `total` positions may see, summed over the rows."""
    if not window:
        return n * (total - n) + n * (n + 1) // 2
    return sum(min(p + 1, window) for p in range(total - n, total))


def work(case):
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        scales = 4 * (-(-n // BLOCK)) * (-(-k // BLOCK))
        return {"bytes": 2 * m * k + n * k + scales + 2 * m * n, "flops": 2 * m * n * k}
    new, total = lengths(case)
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    rows = sum(new)
    if case["op"] == "rope":
        return {"bytes": 4 * rows * (hq + 2 * hkv) * d, "flops": rows * (hq + hkv) * d * (7 if case["norm"] else 3)}
    win = case["window"]
    cached = sum(min(t, n + win - 1) if win else t for n, t in zip(new, total))
    pairs = sum(_visible(n, t, win) for n, t in zip(new, total))
    return {"bytes": 4 * rows * hq * d + 4 * cached * hkv * d, "flops": 4 * pairs * hq * d}


# ------------------------------------------------------------------ inputs
def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        # Normed activations with a few channels that stand out, as a decoder has them.
        x = _randn(gen, m, k) * torch.exp(0.5 * _randn(gen, 1, k))
        w_q, w_scale = _quantize_weight(0.02 * _randn(gen, n, k))
        return {"case": case, "x": x.to(dtype), "w_q": w_q, "w_scale": w_scale}
    hq, hkv, d, page = case["hq"], case["hkv"], case["d"], case["page"]
    new, total = lengths(case)
    need = [-(-t // page) for t in total]
    # A pool with pages to spare, given to the sequences in no order; entries that are not used hold -1.
    pool = sum(need) + 3
    ids = list(range(pool))
    rng = random.Random(seed)
    rng.shuffle(ids)
    table = torch.full((case["seqs"], max(need) + 1), -1, dtype=torch.int32)
    at = 0
    for s, c in enumerate(need):
        table[s, :c] = torch.tensor(ids[at:at + c], dtype=torch.int32)
        at += c
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    rows = starts[-1] + case["pad"]
    state = {
        "case": case, "new": new, "total": total, "starts": starts, "rows": rows,
        "table": table.cuda(),
        "kv_len": torch.tensor(total, dtype=torch.int32).cuda(),
        # One new token everywhere and no padding: the decode form, which needs no row offsets.
        "q_start": None if max(new) == 1 and not case["pad"] else torch.tensor(starts, dtype=torch.int32).cuda(),
        "k_pages": _randn(gen, pool, page, hkv, d).to(dtype),
        "v_pages": _randn(gen, pool, page, hkv, d).to(dtype),
        # Rows behind the last sequence are left as they are, so the output buffer is part of the state.
        "out": torch.zeros(rows, hq * d, dtype=dtype, device="cuda"),
    }
    if case["op"] == "rope":
        state["qkv"] = _randn(gen, rows, (hq + 2 * hkv) * d).to(dtype)
        for g in ("q_gamma", "k_gamma"):
            state[g] = (1 + 0.1 * _randn(gen, d)).to(dtype) if case["norm"] else None
    else:
        state["q"] = _randn(gen, rows, hq, d).to(dtype)
    if own:
        from b200ar.ops.layers import RotaryTable
        from b200ar.ops.paged import PagedBatch

        state["batch"] = PagedBatch(state["table"], state["kv_len"], state["q_start"])
        if case["op"] == "rope":
            state["rot"] = RotaryTable(d, max(total), THETA, "cuda")
    return state


def _quantize_weight(w):
    """e4m3 values and one fp32 scale for each 128 x 128 block: amax / 448."""
    n, k = w.shape
    nb, kb = -(-n // BLOCK), -(-k // BLOCK)
    full = torch.zeros(nb * BLOCK, kb * BLOCK, device=w.device)
    full[:n, :k] = w
    full = full.view(nb, BLOCK, kb, BLOCK)
    amax = full.abs().amax(dim=(1, 3))
    scale = amax / torch.full_like(amax, E4M3_MAX)
    scale = torch.where(amax > 0, scale, torch.ones_like(scale))
    q = (full / scale[:, None, :, None]).clamp(-E4M3_MAX, E4M3_MAX)
    return q.view(nb * BLOCK, kb * BLOCK)[:n, :k].contiguous().to(torch.float8_e4m3fn), scale


# ------------------------------------------------------------------ one pass
def run(state):
    if own:
        return _run_own(state)
    return {"rope": _rope, "attention": _attention, "linear": _linear_plain}[state["case"]["op"]](state)


def _run_own(state):
    case = state["case"]
    if case["op"] == "linear":
        from b200ar.ops.fp8 import linear_fp8

        return linear_fp8(state["x"], state["w_q"], state["w_scale"])
    from b200ar.ops.paged import paged_attention, qk_norm_rope_paged

    if case["op"] == "rope":
        q = state["out"].view(-1, case["hq"], case["d"])
        qk_norm_rope_paged(state["qkv"], state["batch"], state["rot"], state["k_pages"], state["v_pages"],
                           case["hq"], case["hkv"], q_gamma=state["q_gamma"], k_gamma=state["k_gamma"], eps=EPS,
                           q_out=q)
        return [q, state["k_pages"], state["v_pages"]]
    return paged_attention(state["q"], state["k_pages"], state["v_pages"], state["batch"], window=case["window"],
                           out=state["out"])


def _row_index(state):
    """For every new token: its sequence and its position (long tensors)."""
    new = torch.tensor([0], device="cuda") if not state["new"] else state["kv_len"].new_tensor(state["new"]).long()
    used = state["starts"][-1]
    seq = torch.repeat_interleave(torch.arange(len(state["new"]), device="cuda"), new, output_size=used)
    first = state["kv_len"].long() - new
    begin = torch.cumsum(new, 0) - new
    return seq, torch.arange(used, device="cuda") - begin[seq] + first[seq]


def _rope(state):
    case = state["case"]
    hq, hkv, d, page = case["hq"], case["hkv"], case["d"], case["page"]
    used = state["starts"][-1]
    seq, pos = _row_index(state)
    x = state["qkv"][:used].float().view(used, hq + 2 * hkv, d)
    q, k, v = x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]
    if case["norm"]:
        q = q * torch.rsqrt((q * q).mean(-1, keepdim=True) + EPS) * state["q_gamma"].float()
        k = k * torch.rsqrt((k * k).mean(-1, keepdim=True) + EPS) * state["k_gamma"].float()
    inv = THETA ** (-torch.arange(0, d, 2, dtype=torch.float64, device="cuda") / d)
    angle = pos.double()[:, None] * inv
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def turn(t):
        a, b = t[..., :d // 2], t[..., d // 2:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)

    where = state["table"].long()[seq, pos // page]
    dtype = state["qkv"].dtype
    out = state["out"].view(-1, hq, d)
    out[:used] = turn(q).to(dtype)
    state["k_pages"][where, pos % page] = turn(k).to(dtype)
    state["v_pages"][where, pos % page] = v.to(dtype)
    return [out, state["k_pages"], state["v_pages"]]


def _attention(state):
    case = state["case"]
    hq, hkv, d, win = case["hq"], case["hkv"], case["d"], case["window"]
    out = state["out"].view(-1, hq, d)
    for s, (n, total) in enumerate(zip(state["new"], state["total"])):
        pages = state["table"][s, :-(-total // case["page"])].long()
        first = max(0, total - n - win + 1) if win else 0
        k = state["k_pages"][pages].view(-1, hkv, d)[first:total].float()
        v = state["v_pages"][pages].view(-1, hkv, d)[first:total].float()
        rows = slice(state["starts"][s], state["starts"][s + 1])
        at = torch.arange(total - n, total, device="cuda")[:, None]
        col = torch.arange(first, total, device="cuda")[None, :]
        hide = col > at
        if win:
            hide = hide | (col <= at - win)
        for h in range(hkv):
            heads = slice(h * (hq // hkv), (h + 1) * (hq // hkv))
            q = state["q"][rows, heads].float().transpose(0, 1)
            w = (q @ k[:, h].t()) * (1.0 / math.sqrt(d))
            w = w.masked_fill_(hide, float("-inf"))
            w = torch.exp(w - w.amax(-1, keepdim=True))
            o = (w @ v[:, h]) / w.sum(-1, keepdim=True)
            out[rows, heads] = o.transpose(0, 1).to(out.dtype)
    return state["out"]


def _linear_plain(state):
    x, w_q, w_scale = state["x"], state["w_q"], state["w_scale"]
    m, k = x.shape
    n = w_q.shape[0]
    kb = -(-k // BLOCK)
    full = torch.zeros(m, kb * BLOCK, device="cuda")
    full[:, :k] = x.float()
    full = full.view(m, kb, BLOCK)
    amax = full.abs().amax(-1, keepdim=True)
    scale = amax / torch.full_like(amax, E4M3_MAX)
    scale = torch.where(amax > 0, scale, torch.ones_like(scale))
    x_q = (full / scale).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    a = (x_q.float() * scale).view(m, kb * BLOCK)[:, :k]
    by_row = w_scale.repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]
    return (a @ (w_q.float() * by_row).t()).to(x.dtype)


# ------------------------------------------------------------------ 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    return {"rope": _exact_rope, "attention": _exact_attention, "linear": _exact_linear}[case["op"]](state)


def _exact_rope(state):
    case = state["case"]
    hq, hkv, d, page = case["hq"], case["hkv"], case["d"], case["page"]
    out = state["out"].double().view(-1, hq, d).clone()
    kp, vp = state["k_pages"].double(), state["v_pages"].double()
    freq = torch.tensor([THETA ** (-2.0 * i / d) for i in range(d // 2)], dtype=torch.float64, device="cuda")
    for s, (n, total) in enumerate(zip(state["new"], state["total"])):
        lo = state["starts"][s]
        heads = state["qkv"][lo:lo + n].double().reshape(n, -1, d)
        pos = torch.arange(total - n, total, device="cuda")
        # The pair (i, i + d/2) is one complex number, turned by the angle of its position.
        phase = torch.polar(torch.ones(n, d // 2, dtype=torch.float64, device="cuda"), pos[:, None] * freq)

        def turned(x, gamma):
            if gamma is not None:
                x = x / torch.sqrt(x.square().sum(-1, keepdim=True) / d + EPS) * gamma.double()
            z = torch.complex(x[..., :d // 2].contiguous(), x[..., d // 2:].contiguous()) * phase[:, None]
            return torch.cat([z.real, z.imag], -1)

        out[lo:lo + n] = turned(heads[:, :hq], state["q_gamma"])
        pages = state["table"][s].long()[torch.div(pos, page, rounding_mode="floor")]
        kp[pages, pos % page] = turned(heads[:, hq:hq + hkv], state["k_gamma"])
        vp[pages, pos % page] = heads[:, hq + hkv:]
    return [out, kp, vp]


def _exact_attention(state):
    case = state["case"]
    hq, hkv, d, win = case["hq"], case["hkv"], case["d"], case["window"]
    group = hq // hkv
    out = state["out"].double().view(-1, hq, d).clone()
    for s, (n, total) in enumerate(zip(state["new"], state["total"])):
        count = -(-total // case["page"])
        pages = state["table"][s, :count].long()
        for h in range(hkv):
            keys = state["k_pages"][pages, :, h].reshape(-1, d)[:total].double()
            vals = state["v_pages"][pages, :, h].reshape(-1, d)[:total].double()
            # A block of rows at a time, every head of the group: [rows, group, positions].
            for r0 in range(0, n, 512):
                r1 = min(n, r0 + 512)
                pos = total - n + torch.arange(r0, r1, device="cuda")
                end = total - n + r1
                begin = max(0, total - n + r0 - win + 1) if win else 0
                q = state["q"][state["starts"][s] + r0:state["starts"][s] + r1, h * group:(h + 1) * group].double()
                z = torch.einsum("rgd,cd->rgc", q, keys[begin:end]) / math.sqrt(d)
                back = pos[:, None] - torch.arange(begin, end, device="cuda")[None]
                seen = (back >= 0) & (back < win) if win else back >= 0
                z = torch.where(seen[:, None], z, torch.full_like(z, float("-inf")))
                p = torch.exp(z - torch.logsumexp(z, -1, keepdim=True))
                lo = state["starts"][s]
                out[lo + r0:lo + r1, h * group:(h + 1) * group] = torch.einsum("rgc,cd->rgd", p, vals[begin:end])
    return out.view(-1, hq * d)


def _exact_linear(state):
    x, w_q, w_scale = state["x"].double(), state["w_q"].double(), state["w_scale"].double()
    m, k = x.shape
    total = torch.zeros(m, w_q.shape[0], dtype=torch.float64, device="cuda")
    rows = torch.arange(w_q.shape[0], device="cuda") // BLOCK
    for b in range(-(-k // BLOCK)):
        xb, wb = x[:, b * BLOCK:(b + 1) * BLOCK], w_q[:, b * BLOCK:(b + 1) * BLOCK]
        top = xb.abs().amax(1)
        # The scale is part of the format: a number of 32 bits.
        s = torch.where(top > 0, top / E4M3_MAX, torch.ones_like(top)).float().double()
        q = (xb / s[:, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn).double()
        total += s[:, None] * (q @ wb.t()) * w_scale[rows, b][None]
    return total
