"""Block-scaled FP8 GEMM (cb_fp8_block_gemm) against the formula in 64 bits.

Tolerance: with S[m, n] = sum_k |a_s a| |w_s w| (in 64 bits), the products of two
e4m3 values are exact, a tensor core adds the 128 of a block with at least 13
fraction bits below its largest addend, and the blocks are joined in fp32, so the
fp32 total is within 2^-12 S of exact. 16-bit outputs add one rounding (2^-8 or
2^-11 of the result).
"""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def _e4m3(v):
    return v.clamp(-448.0, 448.0).to(torch.float8_e4m3fn)


def _spread(s, n, size=128):
    return s.repeat_interleave(size, dim=-1)[..., :n]


def _make(B, M, N, K, seed):
    """Operands with every scale its own: a wrong scale index shows."""
    g = torch.Generator().manual_seed(seed)
    KB, NB = -(-K // 128), -(-N // 128)
    a = _e4m3(torch.randn(B, M, K, generator=g) * 60.0)
    w = _e4m3(torch.randn(B, N, K, generator=g) * 60.0)
    a_s = 0.001 * torch.exp2(torch.randint(-2, 3, (B, M, KB), generator=g).float()) * (1 + torch.rand(B, M, KB, generator=g))
    w_s = 0.001 * torch.exp2(torch.randint(-2, 3, (B, NB, KB), generator=g).float()) * (1 + torch.rand(B, NB, KB, generator=g))
    return a, w, a_s, w_s


def _exact(a, w, a_s, w_s, bias=None):
    K, N = a.shape[-1], w.shape[-2]
    ad = a.double() * _spread(a_s.double(), K)
    wd = w.double() * _spread(w_s.double(), K).repeat_interleave(128, dim=-2)[..., :N, :]
    y, S = ad @ wd.transpose(-1, -2), ad.abs() @ wd.abs().transpose(-1, -2)
    if bias is not None:
        b = bias.double()
        y = y + (b if b.dim() == 1 else b[:, None, :])
        S = S + (b if b.dim() == 1 else b[:, None, :]).abs()
    return y, S


def _close(out, y, S):
    d = (out.double().cpu() - y).abs()
    assert torch.all(d <= U[out.dtype] * y.abs() + 2.0 ** -12 * S), float((d / S).max())


def _squeeze(B, *ts):
    return [t[0] if B == 1 else t for t in ts]


@pytest.mark.parametrize("M", [1, 2, 7, 8, 9, 16, 17, 31, 33, 64, 65, 127, 130, 257, 300])
@pytest.mark.parametrize("N,K", [(256, 512), (200, 656), (1000, 2064)])
def test_sizes(cuda_device, M, N, K):
    from cb200 import ops
    a, w, a_s, w_s = _squeeze(1, *_make(1, M, N, K, M * 7 + N + K))
    out = ops.fp8_block_gemm(*(t.to(cuda_device) for t in (a, w, a_s, w_s)), out_dtype=torch.float32)
    _close(out, *_exact(a, w, a_s, w_s))


@pytest.mark.parametrize("N,K", [(1, 16), (1, 128), (3, 144), (127, 16), (128, 32), (129, 4112), (5000, 128), (16, 17408)])
@pytest.mark.parametrize("M", [1, 5, 40, 200])
def test_edges(cuda_device, M, N, K):
    from cb200 import ops
    a, w, a_s, w_s = _squeeze(1, *_make(1, M, N, K, M + 3 * N + K))
    out = ops.fp8_block_gemm(*(t.to(cuda_device) for t in (a, w, a_s, w_s)), out_dtype=torch.bfloat16)
    _close(out, *_exact(a, w, a_s, w_s))


@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("M,N,K", [(1, 7168, 5120), (4, 640, 17408), (24, 5120, 1024), (96, 1536, 2048), (513, 776, 1040)])
def test_types_and_bias(cuda_device, M, N, K, out_dtype):
    from cb200 import ops
    a, w, a_s, w_s = _squeeze(1, *_make(1, M, N, K, M + N))
    bias = torch.randn(N, generator=torch.Generator().manual_seed(1)).to(
        {torch.bfloat16: torch.bfloat16, torch.float16: torch.float16, torch.float32: torch.float32}[out_dtype])
    dev = [t.to(cuda_device) for t in (a, w, a_s, w_s)]
    out = ops.fp8_block_gemm(*dev, out_dtype=out_dtype, bias=bias.to(cuda_device))
    assert out.dtype == out_dtype
    _close(out, *_exact(a, w, a_s, w_s, bias))
    again = ops.fp8_block_gemm(*dev, out_dtype=out_dtype, bias=bias.to(cuda_device))
    assert torch.equal(again.view(torch.uint8), out.view(torch.uint8))  # the sums have one order


@pytest.mark.parametrize("B,M,N,K", [(1, 4500, 5000, 272), (1, 8000, 2560, 1040), (2, 1100, 8200, 128), (1, 300, 40000, 400),
                                     (1, 40000, 300, 1536)])
@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
def test_many_tiles(cuda_device, B, M, N, K, out_dtype):
    """Problems with many tiles, ragged in every direction; the reference runs in 64 bits on the device."""
    from cb200 import ops
    a, w, a_s, w_s = (t.to(cuda_device) for t in _squeeze(B, *_make(B, M, N, K, M)))
    bias = torch.randn(N, generator=torch.Generator().manual_seed(1)).to(cuda_device)
    out = ops.fp8_block_gemm(a, w, a_s, w_s, out_dtype=out_dtype, bias=bias)
    y, S = _exact(a, w, a_s, w_s, bias)
    assert torch.all((out.double() - y).abs() <= U[out_dtype] * y.abs() + 2.0 ** -12 * S)
    assert torch.equal(ops.fp8_block_gemm(a, w, a_s, w_s, out_dtype=out_dtype, bias=bias), out)
    odd = torch.full((*out.shape[:-1], N + 1), 3.0, dtype=out_dtype, device=cuda_device)  # rows off the 16-byte grid
    ops.fp8_block_gemm(a, w, a_s, w_s, out=odd[..., :N], bias=bias)
    assert torch.equal(odd[..., :N], out) and torch.all(odd[..., N] == 3.0)
    assert ops.device_status(cuda_device) == 0


@pytest.mark.parametrize("M,N,K", [(100, 333, 272), (300, 1001, 2064), (1300, 2049, 272), (1300, 2050, 272)])
@pytest.mark.parametrize("shift,pad", [(0, 0), (1, 1), (2, 6), (8, 8)])
@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_output_rows_of_any_alignment(cuda_device, M, N, K, shift, pad, out_dtype):
    """out starts `shift` elements into its storage, its rows N + pad apart; what lies between them is not touched."""
    from cb200 import ops
    a, w, a_s, w_s = _squeeze(1, *_make(1, M, N, K, M + N))
    store = torch.full((shift + M * (N + pad),), 7.0, dtype=out_dtype, device=cuda_device)
    out = store.as_strided((M, N), (N + pad, 1), shift)
    ops.fp8_block_gemm(*(t.to(cuda_device) for t in (a, w, a_s, w_s)), out=out)
    _close(out, *_exact(a, w, a_s, w_s))
    assert torch.all(store[:shift] == 7.0)
    if pad:
        gaps = store[shift:].view(M, N + pad)[:, N:]
        assert torch.all(gaps == 7.0)


@pytest.mark.parametrize("M", [1, 3, 20, 150])
def test_batches_and_strides(cuda_device, M):
    from cb200 import ops
    B, N, K = 3, 264, 528
    a, w, a_s, w_s = _make(B, M, N, K, M)
    bias = torch.randn(B, N, generator=torch.Generator().manual_seed(2))
    y, S = _exact(a, w, a_s, w_s, bias)

    def wide(t, pad):
        buf = torch.zeros(*t.shape[:-2], t.shape[-2] + 1, t.shape[-1] + pad, dtype=t.dtype, device=cuda_device)
        if t.element_size() == 1:
            buf.view(torch.uint8)[..., :t.shape[-2], :t.shape[-1]] = t.view(torch.uint8).to(cuda_device)
        else:
            buf[..., :t.shape[-2], :t.shape[-1]] = t.to(cuda_device)
        return buf[..., :t.shape[-2], :t.shape[-1]]

    obuf = torch.full((B, M + 2, N + 3), 5.0, dtype=torch.float16, device=cuda_device)
    out = ops.fp8_block_gemm(wide(a, 32), wide(w, 16), wide(a_s, 3), wide(w_s, 1), out=obuf[:, :M, :N],
                             bias=bias.to(cuda_device))
    _close(out, y, S)
    assert torch.all(obuf[:, M:] == 5.0) and torch.all(obuf[:, :, N:] == 5.0)
    out = ops.fp8_block_gemm(*(t.to(cuda_device) for t in (a, w, a_s, w_s)), bias=bias.to(cuda_device))
    _close(out, y, S)


@pytest.mark.parametrize("M,N,K", [(1, 512, 1024), (6, 136, 400), (77, 640, 5136), (260, 512, 1024)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_dynamic_is_quantize_then_gemm(cuda_device, M, N, K, dtype):
    from cb200 import ops
    _, w, _, w_s = _squeeze(1, *_make(1, M, N, K, M))
    a = torch.randn(M, K, generator=torch.Generator().manual_seed(9)).to(dtype).to(cuda_device)
    w, w_s = w.to(cuda_device), w_s.to(cuda_device)
    q, s = ops.quant_act_fp8_block(a)
    ref = ops.fp8_block_gemm(q, w, s, w_s, out_dtype=dtype)
    q2, s2 = torch.empty_like(q), torch.empty_like(s)
    out = ops.fp8_block_gemm_dynamic(a, w, w_s, q=q2, s=s2)
    assert out.dtype == dtype
    assert torch.equal(out.view(torch.int16), ref.view(torch.int16))
    assert torch.equal(q2.view(torch.uint8), q.view(torch.uint8)) and torch.equal(s2, s)
    _close(out, *_exact(q.cpu(), w.cpu(), s.cpu(), w_s.cpu()))


def test_nan_and_zero_operands_stay_in_their_rows(cuda_device):
    from cb200 import ops
    for M in (4, 150):
        a, w, a_s, w_s = _squeeze(1, *_make(1, M, 256, 1024, 1))
        y, S = _exact(a, w, a_s, w_s)
        a_s[1, 3] = float("nan")
        a.view(torch.uint8)[2] = 0
        out = ops.fp8_block_gemm(*(t.to(cuda_device) for t in (a, w, a_s, w_s)), out_dtype=torch.float32).cpu()
        assert torch.all(torch.isnan(out[1])) and torch.all(out[2] == 0)
        keep = [0] + list(range(3, M))
        _close(out[keep], y[keep], S[keep])


def test_split_order_does_not_depend_on_who_reduces(cuda_device):
    from cb200 import _lib as L
    from cb200 import ops
    for M, N, K in ((1, 384, 5120), (12, 512, 8192), (48, 640, 5120), (200, 256, 4096)):
        dev = [t.to(cuda_device) for t in _squeeze(1, *_make(1, M, N, K, M))]
        ref = ops.fp8_block_gemm(*dev, out_dtype=torch.float32)
        L.load().cb_debug_force_last_arriver(1)
        try:
            for _ in range(3):
                assert torch.equal(ops.fp8_block_gemm(*dev, out_dtype=torch.float32), ref)
        finally:
            L.load().cb_debug_force_last_arriver(0)
    assert ops.device_status(cuda_device) == 0


def test_graph_capture_and_streams(cuda_device):
    from cb200 import ops
    a, w, a_s, w_s = _squeeze(1, *_make(1, 16, 1024, 2048, 3))
    dev = [t.to(cuda_device) for t in (a, w, a_s, w_s)]
    ref = ops.fp8_block_gemm(*dev)
    out = torch.empty_like(ref)
    ops.fp8_block_gemm(*dev, out=out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        for _ in range(3):
            ops.fp8_block_gemm(*dev, out=out)
    for _ in range(4):
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ref)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = ops.fp8_block_gemm(*dev)
    side.synchronize()
    assert torch.equal(other, ref)


def test_empty_and_refusals(cuda_device):
    from cb200 import ops
    d = cuda_device
    a, w, a_s, w_s = (t.to(d) for t in _squeeze(1, *_make(1, 4, 128, 256, 1)))
    assert ops.fp8_block_gemm(a[:0], w, a_s[:0], w_s).shape == (0, 128)
    bf = torch.randn(4, 256, device=d).bfloat16()
    for bad in (
        lambda: ops.fp8_block_gemm(bf, w, a_s, w_s),
        lambda: ops.fp8_block_gemm(a, w, a_s[:, :1], w_s),
        lambda: ops.fp8_block_gemm(a, w, a_s, w_s[:, :1]),
        lambda: ops.fp8_block_gemm(a, w, a_s.double(), w_s),
        lambda: ops.fp8_block_gemm(a[:, :128], w, a_s[:, :1], w_s),
        lambda: ops.fp8_block_gemm(a, w, a_s, w_s, out=torch.empty(4, 127, device=d)),
        lambda: ops.fp8_block_gemm(a, w, a_s, w_s, out=torch.empty(4, 128, device=d, dtype=torch.int32)),
        lambda: ops.fp8_block_gemm(a, w, a_s, w_s, bias=torch.empty(127, device=d)),
        lambda: ops.fp8_block_gemm(a, w.cpu(), a_s, w_s),
        lambda: ops.fp8_block_gemm_dynamic(bf.float(), w, w_s),
        lambda: ops.fp8_block_gemm_dynamic(bf, w, w_s, q=torch.empty(4, 128, device=d, dtype=torch.float8_e4m3fn)),
        # K = 8 more than a multiple of 16, and rows off the 16-byte grid
        lambda: ops.fp8_block_gemm(a[:, :248], w[:, :248], a_s, w_s),
        lambda: ops.fp8_block_gemm(a[:, 8:248], w[:, 8:248], a_s, w_s),
    ):
        with pytest.raises(ValueError):
            bad()
