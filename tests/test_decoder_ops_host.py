"""Decoder-layer operators on a machine without a GPU: argument validation of the C
entries (no compute call is made), the torch layer's refusal of CPU tensors, and the
host packer of block-scaled FP8 weights."""

import ctypes

import numpy as np
import pytest
import torch

from cb200 import _lib as L
from cb200 import wformat as wf

F = ctypes.c_void_p(0x1000)  # never dereferenced: validation fails first


@pytest.fixture(scope="module")
def lib():
    return L.load()


def _st(*v):
    return (ctypes.c_int64 * len(v))(*v)


def _norm(lib, x=F, res=None, xd=L.CB_DTYPE_BF16, w=F, wd=L.CB_DTYPE_BF16, eps=1e-6, rows=4, H=256, xs=256, rs=256, mode=0,
          q=F, qs=256, s=F, ss=1, h=None, hs=256):
    return lib.cb_add_rmsnorm_quant(x, res, xd, w, wd, eps, rows, H, xs, rs, mode, q, qs, s, ss, h, hs, None)


def test_norm_validation(lib):
    assert _norm(lib, x=None, rows=0) == L.CB_OK
    assert _norm(lib, x=None, H=0) == L.CB_OK
    assert _norm(lib, rows=-1) == L.CB_ERR_INVALID_ARG
    assert _norm(lib, x=None) == L.CB_ERR_INVALID_ARG
    assert _norm(lib, mode=3) == L.CB_ERR_INVALID_ARG
    assert _norm(lib, h=F) == L.CB_ERR_INVALID_ARG  # a sum without a residual
    assert _norm(lib, eps=-1.0) == L.CB_ERR_INVALID_ARG
    assert _norm(lib, eps=float("nan")) == L.CB_ERR_INVALID_ARG
    assert _norm(lib, xd=L.CB_DTYPE_F32) == L.CB_ERR_DTYPE
    assert _norm(lib, wd=L.CB_DTYPE_I8) == L.CB_ERR_DTYPE
    assert _norm(lib, xs=255) == L.CB_ERR_STRIDE
    assert _norm(lib, qs=255) == L.CB_ERR_STRIDE
    assert _norm(lib, res=F, rs=255) == L.CB_ERR_STRIDE
    assert _norm(lib, res=F, h=F, hs=255) == L.CB_ERR_STRIDE
    assert _norm(lib, mode=L.CB_NORM_FP8_BLOCK, ss=1) == L.CB_ERR_STRIDE  # two blocks a row
    assert _norm(lib, rows=1 << 31) == L.CB_ERR_TOO_LARGE


def test_block_quantizer_validation(lib):
    def call(a=F, d=L.CB_DTYPE_F16, B=1, M=4, K=256, asm=256, q=F, qsm=256, s=F, ssm=2):
        return lib.cb_quant_act_fp8_block(a, d, B, M, K, 0, asm, q, 0, qsm, s, 0, ssm, None)

    assert call(a=None, M=0) == L.CB_OK
    assert call(a=None) == L.CB_ERR_INVALID_ARG
    assert call(K=-1) == L.CB_ERR_INVALID_ARG
    assert call(d=L.CB_DTYPE_F32) == L.CB_ERR_DTYPE
    assert call(asm=128) == L.CB_ERR_STRIDE
    assert call(ssm=1) == L.CB_ERR_STRIDE


def _gemm(lib, a=F, w=F, out=F, od=L.CB_DTYPE_BF16, bias=None, bd=0, B=1, M=4, N=256, K=256, st=None, ws=None, n=0):
    st = st or _st(0, 256, 0, 256, 0, 256, 0, 2, 0, 2, 0)
    return lib.cb_fp8_block_gemm(a, F, w, F, bias, bd, out, od, B, M, N, K, st, ws, n, None)


def test_block_gemm_validation(lib):
    assert _gemm(lib, a=None, M=0) == L.CB_OK
    assert _gemm(lib, a=None) == L.CB_ERR_INVALID_ARG
    assert _gemm(lib, M=-1) == L.CB_ERR_INVALID_ARG
    assert _gemm(lib, K=248) == L.CB_ERR_SHAPE
    assert _gemm(lib, K=0) == L.CB_ERR_SHAPE
    assert _gemm(lib, od=L.CB_DTYPE_I8) == L.CB_ERR_DTYPE
    assert _gemm(lib, bias=F, bd=L.CB_DTYPE_I8) == L.CB_ERR_DTYPE
    assert _gemm(lib, a=ctypes.c_void_p(0x1008)) == L.CB_ERR_ALIGNMENT
    assert _gemm(lib, st=_st(0, 264, 0, 256, 0, 256, 0, 2, 0, 2, 0)) == L.CB_ERR_ALIGNMENT
    assert _gemm(lib, st=_st(0, 128, 0, 256, 0, 256, 0, 2, 0, 2, 0)) == L.CB_ERR_STRIDE
    assert _gemm(lib, st=_st(0, 256, 0, 256, 0, 256, 0, 1, 0, 2, 0)) == L.CB_ERR_STRIDE
    assert _gemm(lib, st=_st(0, 256, 0, 256, 0, 256, 0, 2, 0, 1, 0)) == L.CB_ERR_STRIDE
    assert _gemm(lib, st=_st(0, 256, 0, 256, 0, -256, 0, 2, 0, 2, 0)) == L.CB_ERR_STRIDE
    assert _gemm(lib) == L.CB_ERR_WORKSPACE
    assert lib.cb_workspace_bytes(L.CB_OP_FP8_BLOCK, 1, 4, 256, 256) > 0


def test_append_validation(lib):
    def call(k=F, d=L.CB_DTYPE_BF16, c=L.CB_DTYPE_BF16, ks=None, T=4, heads=2, D=64, pages=8, page=16, st=None):
        st = st or _st(128, 64, 2048, 128, 64, 128, 64, 2048, 128, 64)
        return lib.cb_paged_kv_append(k, F, d, F, F, c, ks, None, F, 0, T, heads, D, pages, page, st, None, None)

    assert call(k=None, T=0) == L.CB_OK
    assert call(k=None) == L.CB_ERR_INVALID_ARG
    assert call(page=0) == L.CB_ERR_INVALID_ARG
    assert call(ks=F) == L.CB_ERR_INVALID_ARG  # scales without an e4m3 cache
    assert call(d=L.CB_DTYPE_F32) == L.CB_ERR_DTYPE
    assert call(c=L.CB_DTYPE_I8) == L.CB_ERR_DTYPE
    assert call(st=_st(128, 64, -2048, 128, 64, 128, 64, 2048, 128, 64)) == L.CB_ERR_STRIDE


def test_attention_validation(lib):
    def call(q=F, d=L.CB_DTYPE_BF16, c=L.CB_DTYPE_BF16, k=F, ks=None, B=2, Hq=8, Hkv=2, D=64, pages=8, page=16, width=4, st=None):
        st = st or _st(512, 64, 512, 64, 8, 4, 2048, 128, 64, 2048, 128, 64)
        return lib.cb_paged_decode_attention(q, d, k, F, c, ks, None, F, F, 0.1, F, None, B, Hq, Hkv, D, pages, page, width, st,
                                             None, 0, None)

    assert call(q=None, B=0) == L.CB_OK
    assert call(q=None) == L.CB_ERR_INVALID_ARG
    assert call(page=0) == L.CB_ERR_INVALID_ARG
    assert call(ks=F) == L.CB_ERR_INVALID_ARG
    assert call(D=32) == L.CB_ERR_SHAPE
    assert call(Hq=7) == L.CB_ERR_SHAPE
    assert call(Hkv=0) == L.CB_ERR_SHAPE
    assert call(c=L.CB_DTYPE_F16) == L.CB_ERR_DTYPE  # neither the queries' type nor e4m3
    assert call(k=ctypes.c_void_p(0x1008)) == L.CB_ERR_ALIGNMENT
    assert call(st=_st(512, 64, 512, 64, 8, 4, 2048, 130, 64, 2048, 128, 64)) == L.CB_ERR_ALIGNMENT
    assert call(st=_st(512, 64, 512, 64, 8, 4, -2048, 128, 64, 2048, 128, 64)) == L.CB_ERR_STRIDE
    assert call(width=1 << 30, page=1 << 20) == L.CB_ERR_TOO_LARGE
    assert call() == L.CB_ERR_WORKSPACE
    assert lib.cb_workspace_bytes(L.CB_OP_PAGED_ATTENTION, 0, 8, 2, 64) > 0
    assert lib.cb_workspace_bytes(L.CB_OP_PAGED_ATTENTION, 0, 1, 2, 64) == 0


def test_status_of_a_wrong_index():
    assert "outside the cache" in L.status_str(L.CB_ERR_DEVICE_INDEX)
    with pytest.raises(L.CbError):
        L.check("cb_workspace_status", L.CB_ERR_DEVICE_INDEX)


def test_ops_refuse_cpu_tensors():
    from cb200 import ops
    x = torch.zeros(2, 128, dtype=torch.bfloat16)
    f8 = torch.zeros(128, 128, dtype=torch.float8_e4m3fn)
    cache = torch.zeros(2, 16, 1, 64, dtype=torch.bfloat16)
    i32 = torch.zeros(2, dtype=torch.int32)
    for call in (lambda: ops.add_rmsnorm_quant(x, x[0]), lambda: ops.quant_act_fp8_block(x),
                 lambda: ops.fp8_block_gemm(f8, f8, torch.zeros(128, 1), torch.zeros(1, 1)),
                 lambda: ops.fp8_block_gemm_dynamic(x, f8, torch.zeros(1, 1)),
                 lambda: ops.paged_kv_append(cache[0, :2], cache[0, :2], cache, cache, i32),
                 lambda: ops.paged_decode_attention(cache[0, :2], cache, cache, i32[:, None], i32)):
        with pytest.raises(ValueError, match="CUDA"):
            call()


def test_e4m3_packing_matches_torch():
    """Every e4m3 value, the midpoints between neighbours, and values around them."""
    codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
    v = codes[~torch.isnan(codes)]
    s = torch.sort(v).values
    mid = (s[1:] + s[:-1]) / 2
    t = torch.cat([v, mid, mid * (1 + 2e-7), mid * (1 - 2e-7), torch.randn(5000) * 50, torch.tensor([1e-30, -1e-9, 448.0, -448.0])])
    want = t.clamp(-448.0, 448.0).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(wf._e4m3_bytes(t.numpy()), want)
    assert wf._e4m3_bytes(np.float32([1e9, -1e9])).tolist() == [0x7E, 0xFE]
    assert wf._e4m3_bytes(np.float32([np.nan]))[0] & 0x7F == 0x7F


@pytest.mark.parametrize("shape", [(128, 128), (200, 300), (2, 130, 16)])
def test_fp8_block_weights_round_trip(tmp_path, shape):
    w = torch.randn(*shape, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    p = wf.quantize_fp8_block(w)
    B = shape[0] if len(shape) == 3 else 1
    N, K = shape[-2:]
    assert p.w_nk.shape == (B, N, K) and p.scales.shape == (B, -(-N // 128), -(-K // 128))
    back = torch.from_numpy(p.w_nk).view(torch.float8_e4m3fn).float()
    s = torch.from_numpy(p.scales).repeat_interleave(128, 1)[:, :N].repeat_interleave(128, 2)[:, :, :K]
    # half a step of e4m3: 2^-4 of the value, or 2^-10 steps of the scale near zero
    assert torch.all((back * s - w.float().view(B, N, K)).abs() <= 2.0 ** -4 * w.float().view(B, N, K).abs() + s * 2.0 ** -10)
    path = str(tmp_path / "w.cbw")
    wf.save(path, {"gate": p})
    got = wf.load(path)["gate"]
    assert isinstance(got, wf.PackedFp8Block)
    assert np.array_equal(got.w_nk, p.w_nk) and np.array_equal(got.scales, p.scales)
    dev = wf.load(path, device="cpu")["gate"]
    assert dev.w_nk.dtype == torch.float8_e4m3fn and torch.equal(dev.scales, torch.from_numpy(p.scales))
    wf.save(path, {"gate": dev})
    assert np.array_equal(wf.load(path)["gate"].w_nk, p.w_nk)
