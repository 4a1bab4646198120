"""The decoder layer of harness/decode_layer.py: every step's result against the formula
in 64 bits from the step's own inputs, over several tokens, and the graph's replay.

Tolerances: the norm's e4m3 rounding is 2^-4 of a value or half the least subnormal
(2^-10) of its scale, with 2^-18 for its fp32 sums and quotients; the products are those of
the block-scaled GEMM (2^-12 of the summed magnitudes S, one rounding of the 16-bit
output) and of the paged attention (probabilities rounded to the products' type,
u = 2^-8 for a bf16 cache and 2^-11 for e4m3, whose queries are rounded to 2^-11).
Dynamic entries quantize first: q * s is within 2^-4 |a| + 2^-10 s of a, where
s <= amax / 448 (1 + 2^-20) + 2^-17.
"""

import os
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
FP8 = torch.float8_e4m3fn
U16 = 2.0 ** -8


def _harness():
    sys.path.insert(0, os.path.join(ROOT, "cache-barrier_b200", "harness"))
    import decode_layer

    return decode_layer


def _wide(w):
    """(e4m3 weight, block scales) in 64 bits."""
    q, s = w
    N, K = q.shape
    return q.double() * s.double().repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]


def _rows(q, s):
    return q.double() * s.double().repeat_interleave(128, 1)[:, :q.shape[1]]


def _gemm_close(out, a, w, bias=None, a_err=None):
    wd = _wide(w)
    y, S = a @ wd.t(), a.abs() @ wd.abs().t()
    if bias is not None:
        y, S = y + bias.double(), S + bias.double().abs()
    tol = U16 * y.abs() + 2.0 ** -12 * S
    if a_err is not None:
        tol = tol + (a_err @ wd.abs().t()) * (1 + 2.0 ** -8 + 2.0 ** -12)
    assert torch.all((out.double() - y).abs() <= tol)


def _dynamic_error(a):
    """Largest |q * s - a| of the block quantization of a."""
    n = a.shape[1]
    t = torch.nn.functional.pad(a, (0, -n % 128)).view(a.shape[0], -1, 128).abs()
    s = (t.amax(2) / 448 * (1 + 2.0 ** -20) + 2.0 ** -17).repeat_interleave(128, 1)[:, :n]
    return 2.0 ** -4 * a.abs() * (1 + 2.0 ** -18) + 2.0 ** -10 * s


def _norm_close(q, s, h, w, eps):
    """h: the unrounded sum in 64 bits."""
    y = h / torch.sqrt((h * h).mean(1, keepdim=True) + eps) * w.double()
    step = s.double().repeat_interleave(128, 1)[:, :y.shape[1]]
    assert torch.all((_rows(q, s) - y).abs() <= (2.0 ** -4 + 2.0 ** -18) * y.abs() + 2.0 ** -10 * step)


@pytest.mark.parametrize("cache_dtype", [None, FP8])
@pytest.mark.parametrize("dims,lens", [(dict(hidden=512, heads=8, kv_heads=2, head_dim=64, inter=640), [0, 1, 15, 16, 77]),
                                       (dict(hidden=384, heads=5, kv_heads=5, head_dim=128, inter=400), [130])])
def test_every_step_of_the_layers(cuda_device, dims, lens, cache_dtype):
    H = _harness()
    from cb200 import ops

    d = H.Dims(**dims)
    B, D = len(lens), d.head_dim
    m = H.Decoder(d, 2, lens, 160, 16, cuda_device, cache_dtype=cache_dtype, seed=3)
    g = torch.Generator().manual_seed(5)
    for c in m.caches:  # what the cache held before
        for t in (c.k, c.v):
            old = torch.randn(t.shape, generator=g)
            if cache_dtype == FP8:
                t.view(torch.uint8).copy_((old * 16).to(FP8).view(torch.uint8))
            else:
                t.copy_(old.to(t.dtype))
    for token in range(3):
        x, residual, at = torch.randn(B, d.hidden, generator=g).to(torch.bfloat16).to(cuda_device), None, m.place()
        for i, (w, c) in enumerate(zip(m.layers, m.caches)):
            before = [t.view(torch.uint8).clone() for t in (c.k, c.v)]
            r = {}
            x_in, res_in = x, residual
            x, residual = m.layer(i, x, residual, at, r)
            h = x_in.double() + (0 if res_in is None else res_in.double())
            assert torch.all((r["h"].double() - h).abs() <= U16 * h.abs())
            _norm_close(r["q8"], r["s8"], h, w.norm_in, d.eps)
            _gemm_close(r["qkv"], _rows(r["q8"], r["s8"]), w.qkv, w.qkv_bias)
            # the cache: new rows in their slots, the rest as before
            for t, b4, new, sc in ((c.k, before[0], r["k"], c.k_scale), (c.v, before[1], r["v"], c.v_scale)):
                if cache_dtype == FP8:
                    new = (new.float() / sc[:, None]).clamp(-448, 448).to(FP8)
                b4.view(-1, *b4.shape[2:])[at.slots] = new.contiguous().view(torch.uint8).view(B, d.kv_heads, -1)
                assert torch.equal(t.view(torch.uint8), b4)
            # attention from what the cache now holds
            for b in range(B):
                n = lens[b] + token + 1
                t = torch.arange(n, device=cuda_device)
                rows = m.table[b].long()[t // 16] * 16 + t % 16
                k, v = (y.view(torch.uint8).view(-1, *b4.shape[2:])[rows].view(y.dtype).double() for y in (c.k, c.v))
                if cache_dtype == FP8:
                    k, v = k * c.k_scale.double()[:, None], v * c.v_scale.double()[:, None]
                q = r["q"][b].double().view(d.kv_heads, -1, D)
                z = torch.einsum("hgd,lhd->hgl", q, k) * D ** -0.5
                p = torch.softmax(z, 2)
                ref, A = (torch.einsum("hgl,lhd->hgd", p, y).reshape(-1, D) for y in (v, v.abs()))
                Z = (torch.einsum("hgd,lhd->hgl", q.abs(), k.abs()) * D ** -0.5).amax(2).reshape(-1, 1)
                dz = Z * (2.0 ** -16 + (2.0 ** -11 if cache_dtype == FP8 else 0)) + 2.0 ** -20
                u = 2.0 ** -11 if cache_dtype == FP8 else U16
                assert torch.all((r["attn"][b].double() - ref).abs() <= U16 * ref.abs() + (u + 2 * dz) * A)
            a = r["attn"].view(B, -1).double()
            _gemm_close(r["o"], a, w.o, a_err=_dynamic_error(a))
            h2 = r["o"].double() + r["h"].double()
            _norm_close(r["q8m"], r["s8m"], h2, w.norm_mid, d.eps)
            gu = torch.cat([r["gate"], r["up"]], 1)
            _gemm_close(gu, _rows(r["q8m"], r["s8m"]), w.gate_up)
            a = r["act"].double()
            _gemm_close(r["out"], a, w.down, a_err=_dynamic_error(a))
        m.lens.add_(1)
    assert ops.device_status(cuda_device) == 0


def test_replayed_steps_are_the_eager_ones(cuda_device):
    """A graph captured once follows lengths, pages and a sequence that fills up."""
    H = _harness()
    from cb200 import ops

    d = H.Dims(hidden=256, heads=4, kv_heads=2, head_dim=64, inter=384)
    lens, max_len = [3, 30, 0], 32
    eager, graphed = (H.Decoder(d, 2, lens, max_len, 16, cuda_device, seed=1) for _ in range(2))
    g = torch.Generator().manual_seed(2)
    xs = [torch.randn(3, d.hidden, generator=g).to(torch.bfloat16).to(cuda_device) for _ in range(2)]
    want = [eager.step(x).clone() for x in xs]
    x = xs[0].clone()
    graphed.step(x)  # workspaces exist before the capture
    graphed.lens.copy_(torch.tensor(lens, dtype=torch.int32))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = graphed.step(x)
    for t, ref in zip(xs, want):
        x.copy_(t)
        graph.replay()
        assert torch.equal(y, ref)
    full = graphed.place()
    assert graphed.lens.tolist() == [5, 32, 2] and (full.slots < 0).tolist() == [False, True, False] and full.held.tolist() == [6, 32, 3]
    for a, b in zip(eager.caches, graphed.caches):
        assert torch.equal(a.k, b.k) and torch.equal(a.v, b.v)
    assert ops.device_status(cuda_device) == 0
