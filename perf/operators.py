"""The operators of a quantized decoder layer around its projections, as a serving loop calls them.

Four operators that belong together: the residual addition with RMSNorm and an
8-bit output, the e4m3 GEMM with one scale per block of 128, the write of new
keys and values into a paged cache, and the attention of one new token over that
cache. ``run`` computes one of them in plain 32-bit torch operations, or, where
``own`` is true, through ``cb200.ops``.

8-bit outputs are returned in the type that holds their numbers (float8_e4m3fn,
int8) with their scales beside them; int8 operands have to be equal.
"""

from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False

BLOCK = 128          # elements of K per scale (and weight rows per scale)
FP8_MAX = 448.0      # largest e4m3 value
NORM_FLOOR = 2.0 ** -100   # least quantization step of the norm's weighted row
QUANT_FLOOR = 1.0 / (448.0 * 512.0)  # least scale of the activation quantizer

_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32, "e4m3": torch.float8_e4m3fn}
_BYTES = {"bf16": 2, "f16": 2, "f32": 4, "e4m3": 1}


def _ops():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "cache-barrier_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from cb200 import ops

    return ops


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # the norm before a projection when one sequence decodes: latency
        {"name": "norm_int8_token", "op": "norm", "rows": 1, "H": 5120, "mode": "int8", "residual": True, "dtype": "bf16"},
        # the same norm feeding the block-scaled GEMM at a serving batch
        {"name": "norm_block_batch", "op": "norm", "rows": 77, "H": 5120, "mode": "fp8_block", "residual": True, "dtype": "bf16"},
        # a long prompt
        {"name": "norm_fp8_prompt", "op": "norm", "rows": 16384, "H": 8192, "mode": "fp8", "residual": True, "dtype": "f16"},
        # fused QKV projection of one token, operands already quantized by the norm
        {"name": "gemm_qkv_token", "op": "gemm", "M": 1, "N": 7168, "K": 5120, "dtype": "bf16", "bias": True, "dynamic": False},
        # down projection of a decode batch, quantized within the call
        {"name": "gemm_down_batch", "op": "gemm", "M": 32, "N": 5120, "K": 17408, "dtype": "bf16", "bias": False, "dynamic": True},
        # a chunk of a prompt through a ragged weight (edges inside a block of 128)
        {"name": "gemm_ragged_chunk", "op": "gemm", "M": 333, "N": 5000, "K": 5136, "dtype": "f16", "bias": True, "dynamic": False},
        # a long prompt through a square projection: arithmetic-bound
        {"name": "gemm_prompt", "op": "gemm", "M": 8192, "N": 8192, "K": 8192, "dtype": "bf16", "bias": False, "dynamic": False},
        # each sequence of a decode batch adds its token
        {"name": "append_batch", "op": "append", "T": 64, "Hkv": 8, "D": 128, "page": 16, "dtype": "bf16", "cache": "bf16"},
        # a prompt is written into an 8-bit cache
        {"name": "append_prompt_fp8", "op": "append", "T": 16384, "Hkv": 8, "D": 128, "page": 64, "dtype": "bf16", "cache": "e4m3"},
        # one short sequence: latency
        {"name": "attn_token", "op": "attn", "B": 1, "max_len": 999, "lens": "even", "Hkv": 8, "G": 5, "D": 128, "page": 16,
         "dtype": "bf16", "cache": "bf16"},
        # a batch of mixed lengths, one of them without any token, over an 8-bit cache
        {"name": "attn_mixed_fp8", "op": "attn", "B": 64, "max_len": 8191, "lens": "mixed", "Hkv": 4, "G": 6, "D": 256, "page": 32,
         "dtype": "f16", "cache": "e4m3"},
        # a few long contexts
        {"name": "attn_long", "op": "attn", "B": 8, "max_len": 65536, "lens": "even", "Hkv": 8, "G": 5, "D": 128, "page": 64,
         "dtype": "bf16", "cache": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "gemm", "append", "attn"])
    dtype = rng.choice(["bf16", "f16"])
    if op == "norm":
        H = _log(rng, 256, 16384)
        if rng.random() < 0.8:
            H = max(256, H // 16 * 16)
        rows = min(_log(rng, 1, 16384), 16384 * 8192 // H)
        return {"op": op, "rows": rows, "H": H, "mode": rng.choice(["int8", "fp8", "fp8_block"]), "residual": rng.random() < 0.7,
                "dtype": dtype}
    if op == "gemm":
        M = _log(rng, 1, 8192)
        N = _log(rng, 256, 17408)
        K = _log(rng, 256, 17408) // 16 * 16
        N = max(1, min(N, 8192 ** 3 // (M * K)))
        return {"op": op, "M": M, "N": N, "K": K, "dtype": dtype, "bias": rng.random() < 0.5, "dynamic": rng.random() < 0.5}
    Hkv = rng.choice([1, 2, 4, 5, 8])
    D = rng.choice([64, 128, 256])
    page = rng.choice([16, 32, 64, 128])
    cache = rng.choice([dtype, "e4m3"])
    if op == "append":
        T = min(_log(rng, 1, 16384), 16384 * 8 * 128 // (Hkv * D))
        return {"op": op, "T": T, "Hkv": Hkv, "D": D, "page": page, "dtype": dtype, "cache": cache}
    B = _log(rng, 1, 256)
    most = 8 * 65536 * 8 * 128 // (B * Hkv * D)
    return {"op": op, "B": B, "max_len": min(_log(rng, 1, 65536), max(1, most)), "lens": rng.choice(["even", "mixed"]), "Hkv": Hkv,
            "G": rng.choice([1, 2, 4, 5, 6, 8, 16]), "D": D, "page": page, "dtype": dtype, "cache": cache}


def _lengths(case):
    """The sequences' lengths: "even" lies in the upper quarter, "mixed" is spread over the logarithm and begins with an empty one."""
    B, top = case["B"], case["max_len"]
    if B == 1:
        return [top]
    if case["lens"] == "even":
        return [top - (top // 4) * i // (B - 1) for i in range(B)]
    return [0] + [max(1, int(round(top ** (i / (B - 1))))) for i in range(1, B)]


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) & 0x7FFFFFFF)


def _normal(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda", dtype=dtype)


def _activations(g, rows, width, dtype):
    """Hidden states: normal values with some channels ten times as large."""
    gain = 1.0 + 9.0 * (torch.rand(width, generator=g, device="cuda") < 0.01).float()
    return (_normal(g, rows, width) * gain).to(dtype)


def _blocks(t, size=BLOCK):
    """[rows, width] as [rows, blocks, size], padded with zeros."""
    pad = -t.shape[1] % size
    return torch.nn.functional.pad(t, (0, pad)).view(t.shape[0], -1, size)


def _weight(g, N, K):
    """A random [N, K] weight in e4m3 with one scale per 128 x 128 block."""
    w = _normal(g, N, K) * 0.02
    nb, kb = -(-N // BLOCK), -(-K // BLOCK)
    w = torch.nn.functional.pad(w, (0, kb * BLOCK - K, 0, nb * BLOCK - N)).view(nb, BLOCK, kb, BLOCK)
    s = (w.abs().amax(dim=(1, 3)) / FP8_MAX).clamp(min=QUANT_FLOOR)
    q = (w / s[:, None, :, None]).clamp(-FP8_MAX, FP8_MAX).to(torch.float8_e4m3fn)
    return q.view(torch.uint8).view(nb * BLOCK, kb * BLOCK)[:N, :K].contiguous().view(torch.float8_e4m3fn), s


def prepare(case, seed):
    g = _generator(seed)
    dt = _TYPES[case["dtype"]]
    if case["op"] == "norm":
        rows, H = case["rows"], case["H"]
        q_type = torch.int8 if case["mode"] == "int8" else torch.float8_e4m3fn
        scales = -(-H // BLOCK) if case["mode"] == "fp8_block" else 1
        return {"op": "norm", "mode": case["mode"], "eps": 1e-6, "x": _activations(g, rows, H, dt),
                "residual": _activations(g, rows, H, dt) if case["residual"] else None,
                "weight": (1.0 + 0.1 * _normal(g, H)).to(dt),
                "q": torch.empty(rows, H, dtype=q_type, device="cuda"),
                "s": torch.empty((rows, scales) if case["mode"] == "fp8_block" else (rows,), device="cuda"),
                "h": torch.empty(rows, H, dtype=dt, device="cuda") if case["residual"] else None}
    if case["op"] == "gemm":
        M, N, K = case["M"], case["N"], case["K"]
        w, w_scale = _weight(g, N, K)
        a = _activations(g, M, K, dt)
        state = {"op": "gemm", "dynamic": case["dynamic"], "w": w, "w_scale": w_scale,
                 "bias": _normal(g, N).to(dt) if case["bias"] else None,
                 "q": torch.empty(M, K, dtype=torch.float8_e4m3fn, device="cuda"),
                 "s": torch.empty(M, -(-K // BLOCK), device="cuda"),
                 "out": torch.empty(M, N, dtype=dt, device="cuda")}
        if case["dynamic"]:
            state["a"] = a
        else:
            state["aq"], state["a_scale"] = _quantize(a)
        return state
    Hkv, D, page = case["Hkv"], case["D"], case["page"]
    kind = _TYPES[case["cache"]]
    if case["op"] == "append":
        T = case["T"]
        pages = -(-T // page) + 3
        slots = torch.randperm(pages * page, generator=g, device="cuda")[:T].to(torch.int32)
    else:
        lens = _lengths(case)
        width = max(1, -(-max(lens) // page))
        used = sum(-(-n // page) for n in lens)
        pages = used + 3
    gain = 10.0 if kind == torch.float8_e4m3fn else 1.0  # stored values of about one once scaled back
    cache = [(_normal(g, pages, page, Hkv, D, dtype=torch.float16) * gain).to(kind) for _ in range(2)]
    scales = [0.05 + 0.1 * torch.rand(Hkv, generator=g, device="cuda") for _ in range(2)] if kind == torch.float8_e4m3fn else [None, None]
    state = {"op": case["op"], "k_cache": cache[0], "v_cache": cache[1], "k_scale": scales[0], "v_scale": scales[1]}
    if case["op"] == "append":
        return {**state, "k": _normal(g, T, Hkv, D).to(dt), "v": _normal(g, T, Hkv, D).to(dt), "slots": slots}
    order = random.Random(int(seed)).sample(range(len(lens)), len(lens))
    lens = [lens[i] for i in order]
    table = torch.zeros(len(lens), width, dtype=torch.int32)
    free = torch.randperm(pages, generator=torch.Generator().manual_seed(int(seed) & 0x7FFFFFFF)).to(torch.int32)
    at = 0
    for b, n in enumerate(lens):
        k = -(-n // page)
        table[b, :k] = free[at:at + k]
        at += k
    Hq = Hkv * case["G"]
    return {**state, "q": (_normal(g, len(lens), Hq, D) * 1.5).to(dt), "table": table.cuda(),
            "lens": torch.tensor(lens, dtype=torch.int32).cuda(), "scale": 1.0 / math.sqrt(D),
            "out": torch.empty(len(lens), Hq, D, dtype=dt, device="cuda"), "lse": torch.empty(len(lens), Hq, device="cuda")}


# ---------------------------------------------------------------------------
# the plain forms: 32 bits, rounded once at the end
# ---------------------------------------------------------------------------
def _const(like, value):
    return torch.full((), value, dtype=like.dtype, device=like.device)


def _quantize(a):
    """e4m3 with a scale per 128 elements of a row: scale = max(amax / 448, 1 / (448 * 512)), q = a / scale."""
    t = _blocks(a.float())
    amax = t.abs().amax(dim=2)
    s = torch.maximum(amax / _const(amax, FP8_MAX), _const(amax, QUANT_FLOOR))
    q = (t / s[:, :, None]).clamp(-FP8_MAX, FP8_MAX).to(torch.float8_e4m3fn)
    width = a.shape[1]
    return q.view(torch.uint8).view(a.shape[0], -1)[:, :width].contiguous().view(torch.float8_e4m3fn), s


def _plain_norm(x, weight, eps, residual, mode):
    """h = x + residual; r = 1 / sqrt(mean(h^2) + eps); u = h * weight; step = amax|u| / 127 or 448; q = u / step, scale = step * r.

    The row's factor r divides out of q, so q depends on u alone."""
    rows, H = x.shape
    h = x.float() if residual is None else x.float() + residual.float()
    r = 1.0 / torch.sqrt((h * h).mean(dim=1, keepdim=True) + eps)
    u = _blocks(h * weight.float(), BLOCK if mode == "fp8_block" else H)
    top = 127.0 if mode == "int8" else FP8_MAX
    amax = u.abs().amax(dim=2)
    step = torch.maximum(amax / _const(amax, top), _const(amax, NORM_FLOOR))
    v = u / step[:, :, None]
    if mode == "int8":
        q = torch.trunc(v + torch.copysign(_const(v, 0.5), v)).to(torch.int8).view(rows, -1)
    else:
        q = v.clamp(-FP8_MAX, FP8_MAX).to(torch.float8_e4m3fn).view(torch.uint8).view(rows, -1)[:, :H].contiguous().view(torch.float8_e4m3fn)
    s = step * r if mode == "fp8_block" else (step * r).view(rows)
    return q, s, None if residual is None else h.to(x.dtype)


def _spread(s, N, K):
    """Block scales [n, k] as one per element [N, K]."""
    return s.repeat_interleave(BLOCK, dim=1)[:, :K] if N is None else s.repeat_interleave(BLOCK, dim=0)[:N].repeat_interleave(BLOCK, dim=1)[:, :K]


def _plain_gemm(aq, a_scale, w, w_scale, bias, out_type):
    N, K = w.shape
    y = (aq.float() * _spread(a_scale, None, K)) @ (w.float() * _spread(w_scale, N, K)).t()
    if bias is not None:
        y = y + bias.float()
    return y.to(out_type)


def _plain_append(k, v, k_cache, v_cache, slots, k_scale, v_scale):
    at = slots.long()
    for new, cache, scale in ((k, k_cache, k_scale), (v, v_cache, v_scale)):
        t = new.float()
        if scale is not None:
            t = (t / scale[:, None]).clamp(-FP8_MAX, FP8_MAX)
        flat = cache.view(-1, *cache.shape[2:])
        if cache.dtype == torch.float8_e4m3fn:
            flat.view(torch.uint8)[at] = t.to(cache.dtype).view(torch.uint8)
        else:
            flat[at] = t.to(cache.dtype)
    return k_cache, v_cache


def _gather(cache, table, scale):
    """The pages of a table as [B, Hkv, L, D] in 32 bits."""
    raw = cache.view(torch.uint8)[table.long()].view(torch.float8_e4m3fn) if cache.dtype == torch.float8_e4m3fn else cache[table.long()]
    t = raw.float().flatten(1, 2).transpose(1, 2)
    return t if scale is None else t * scale[:, None, None]


def _plain_attention(q, k_cache, v_cache, table, lens, scale, k_scale, v_scale):
    """softmax(scale * q k^T) v over each sequence's tokens; a sequence without tokens gives zeros and a log sum of -inf."""
    B, Hq, D = q.shape
    Hkv = k_cache.shape[2]
    k = _gather(k_cache, table, k_scale)
    z = (q.float().view(B, Hkv, Hq // Hkv, D) @ k.transpose(2, 3)) * scale
    del k
    there = torch.arange(z.shape[3], device=z.device)[None, :] < lens[:, None]
    z = z.masked_fill(~there[:, None, None, :], -math.inf)
    m = z.amax(dim=3, keepdim=True)
    m = torch.where(m == -math.inf, _const(m, 0.0), m)
    e = torch.exp(z - m)
    del z
    total = e.sum(dim=3, keepdim=True)
    lse = (m + torch.log(total)).view(B, Hq)
    v = _gather(v_cache, table, v_scale).masked_fill(~there[:, None, :, None], 0.0)
    out = (e @ v) / torch.where(total == 0, _const(total, 1.0), total)
    return out.view(B, Hq, D).to(q.dtype), lse


def run(state):
    s = state
    if own:
        ops = _ops()
        if s["op"] == "norm":
            return ops.add_rmsnorm_quant(s["x"], s["weight"], s["eps"], residual=s["residual"], mode=s["mode"], q=s["q"], s=s["s"],
                                         h=s["h"])
        if s["op"] == "gemm":
            if s["dynamic"]:
                return ops.fp8_block_gemm_dynamic(s["a"], s["w"], s["w_scale"], q=s["q"], s=s["s"], out=s["out"], bias=s["bias"])
            return ops.fp8_block_gemm(s["aq"], s["w"], s["a_scale"], s["w_scale"], out=s["out"], bias=s["bias"])
        if s["op"] == "append":
            ops.paged_kv_append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["slots"], k_scale=s["k_scale"], v_scale=s["v_scale"])
            return s["k_cache"], s["v_cache"]
        ops.paged_decode_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lens"], scale=s["scale"], k_scale=s["k_scale"],
                                   v_scale=s["v_scale"], out=s["out"], lse=s["lse"])
        return s["out"], s["lse"]
    if s["op"] == "norm":
        return _plain_norm(s["x"], s["weight"], s["eps"], s["residual"], s["mode"])
    if s["op"] == "gemm":
        aq, a_scale = _quantize(s["a"]) if s["dynamic"] else (s["aq"], s["a_scale"])
        return _plain_gemm(aq, a_scale, s["w"], s["w_scale"], s["bias"], s["out"].dtype)
    if s["op"] == "append":
        return _plain_append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["slots"], s["k_scale"], s["v_scale"])
    return _plain_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lens"], s["scale"], s["k_scale"], s["v_scale"])


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    e = _BYTES[case["dtype"]]
    if case["op"] == "norm":
        n = case["rows"] * case["H"]
        scales = case["rows"] * (-(-case["H"] // BLOCK) if case["mode"] == "fp8_block" else 1)
        return {"bytes": n * (e + (2 * e if case["residual"] else 0) + 1) + 4 * scales + e * case["H"], "flops": 6 * n}
    if case["op"] == "gemm":
        M, N, K = case["M"], case["N"], case["K"]
        kb = -(-K // BLOCK)
        a = e * M * K if case["dynamic"] else M * K + 4 * M * kb
        return {"bytes": a + N * K + 4 * -(-N // BLOCK) * kb + e * M * N + (e * N if case["bias"] else 0), "flops": 2 * M * N * K}
    c = _BYTES[case["cache"]]
    if case["op"] == "append":
        n = 2 * case["T"] * case["Hkv"] * case["D"]
        return {"bytes": n * (e + c) + 4 * case["T"], "flops": n}
    tokens, Hq, D = sum(_lengths(case)), case["Hkv"] * case["G"], case["D"]
    return {"bytes": 2 * tokens * case["Hkv"] * D * c + 2 * case["B"] * Hq * D * e + 4 * case["B"] * Hq + 4 * case["B"],
            "flops": 4 * tokens * Hq * D}


# ---------------------------------------------------------------------------
# the same from the definitions, in 64 bits
# ---------------------------------------------------------------------------
def _per_block(t, size, top, floor):
    """(values over their block's step, steps) of a [rows, width] double tensor."""
    rows, width = t.shape
    n = -(-width // size)
    step = torch.zeros(rows, n, dtype=torch.float64, device=t.device)
    step.scatter_reduce_(1, (torch.arange(width, device=t.device) // size).expand(rows, width), t.abs(), "amax")
    step = (step / top).clamp(min=floor)
    return t / step.gather(1, (torch.arange(width, device=t.device) // size).expand(rows, width)), step


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        h = s["x"].double()
        if s["residual"] is not None:
            h = h + s["residual"].double()
        size = BLOCK if case["mode"] == "fp8_block" else case["H"]
        v, step = _per_block(h * s["weight"].double(), size, 127.0 if case["mode"] == "int8" else FP8_MAX, NORM_FLOOR)
        scale = step / ((h ** 2).sum(dim=1, keepdim=True) / case["H"] + s["eps"]).sqrt()
        return [None if case["mode"] == "int8" else v, scale if case["mode"] == "fp8_block" else scale[:, 0],
                None if s["residual"] is None else h]
    if case["op"] == "gemm":
        M, N, K = case["M"], case["N"], case["K"]
        kb = torch.arange(K, device="cuda") // BLOCK
        if case["dynamic"]:
            v, step = _per_block(s["a"].double(), BLOCK, FP8_MAX, QUANT_FLOOR)
            a = v.float().to(torch.float8_e4m3fn).double() * step[:, kb]
        else:
            a = s["aq"].double() * s["a_scale"].double()[:, kb]
        w = s["w"].double() * s["w_scale"].double()[torch.arange(N, device="cuda") // BLOCK][:, kb]
        y = torch.mm(a, w.T)
        return y if s["bias"] is None else y + s["bias"].double()
    if case["op"] == "append":
        caches = []
        for new, cache, scale in ((s["k"], s["k_cache"], s["k_scale"]), (s["v"], s["v_cache"], s["v_scale"])):
            t = cache.double().view(-1, case["Hkv"], case["D"])
            t[s["slots"].long()] = new.double() if scale is None else (new.double() / scale.double()[:, None]).clamp(-448.0, 448.0)
            caches.append(t.view(cache.shape))
        return caches
    B, Hq, D = s["q"].shape
    Hkv, G, page = case["Hkv"], case["G"], case["page"]
    if 4 * sum(_lengths(case)) * Hq * D > 4e12:
        return None
    out = torch.zeros(B, Hq, D, dtype=torch.float64, device="cuda")
    lse = torch.full((B, Hq), -math.inf, dtype=torch.float64, device="cuda")
    for b, n in enumerate(s["lens"].tolist()):
        if n == 0:
            continue
        t = torch.arange(n, device="cuda")
        row = s["table"][b].long()[t // page]
        k, v = (c.view(torch.uint8).view(-1, page, Hkv, D * c.element_size())[row, t % page].view(c.dtype).double()
                for c in (s["k_cache"], s["v_cache"]))
        if s["k_scale"] is not None:
            k, v = k * s["k_scale"].double()[:, None], v * s["v_scale"].double()[:, None]
        z = torch.einsum("hgd,lhd->hgl", s["q"][b].double().view(Hkv, G, D), k) * s["scale"]
        lse[b] = torch.logsumexp(z, dim=2).view(Hq)
        out[b] = torch.einsum("hgl,lhd->hgd", torch.softmax(z, dim=2), v).reshape(Hq, D)
    return [out, lse]
