"""What paged attention loses against 64 bits, where it could lose more than fp32 does.

The probabilities enter their product as a leading and a remaining term of the products'
16-bit type, the leading one towards zero, so each is held to u = 2^-16 of itself (bf16:
2^-7 is left, of which 2^-9 is lost) or 2^-21 (f16, the type of e4m3 caches). With
A = sum_l p_l |v_l| and Z = max_l scale * sum_d |q_d k_d|, the scores are fp32 sums of
exact products (2^-16 Z off at most, 256 additions), the output within
(u + 2 dz) A of exact, dz = 2^-16 Z + 2^-20, and its own rounding comes on top.
Queries of bf16 over an e4m3 cache become f16 beside a power of two that puts the row's
largest value at 2^14: values down to 2^-28 of it keep all their bits.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

FP8 = torch.float8_e4m3fn
OUT = {torch.bfloat16: (2.0 ** -8, 2.0 ** -134), torch.float16: (2.0 ** -11, 2.0 ** -25)}


def _run(ops, q, k, v, page, device):
    """One sequence of k's length; k, v [L, Hkv, D]."""
    L, Hkv, D = k.shape
    pages = -(-L // page)

    def cache(t):
        raw = t.view(torch.uint8) if t.dtype == FP8 else t
        buf = torch.zeros(pages * page, Hkv, D, dtype=raw.dtype)
        buf[:L] = raw
        return buf.view(t.dtype).view(pages, page, Hkv, D).to(device)

    return ops.paged_decode_attention(q.to(device), cache(k), cache(v), torch.arange(pages, dtype=torch.int32, device=device)[None],
                                      torch.tensor([L], dtype=torch.int32, device=device)).double().cpu()


def _exact(q, k, v):
    """(out, A, Z) in 64 bits."""
    Hkv, D = k.shape[1:]
    qd, kd, vd = q[0].double().view(Hkv, -1, D), k.double(), v.double()
    scale = 1.0 / math.sqrt(D)
    p = torch.softmax(torch.einsum("hgd,lhd->hgl", qd, kd) * scale, dim=2)
    Z = (torch.einsum("hgd,lhd->hgl", qd.abs(), kd.abs()) * scale).amax(dim=2)
    out, A = (torch.einsum("hgl,lhd->hgd", p, x).reshape(1, -1, D) for x in (vd, vd.abs()))
    return out, A, Z.view(1, -1, 1)


def _check(out, q, k, v, u):
    ref, A, Z = _exact(q, k, v)
    rel, tiny = OUT[q.dtype]
    tol = rel * ref.abs() + tiny + (u + 2 * (2.0 ** -16 * Z + 2.0 ** -20)) * A
    err = (out - ref).abs()
    assert torch.all(err <= tol), float((err / tol).max())


@pytest.mark.parametrize("dtype,cache_dtype", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16), (torch.float16, FP8)])
@pytest.mark.parametrize("D,G", [(64, 3), (128, 8), (128, 13), (256, 4)])
def test_probabilities_keep_their_bits(cuda_device, D, G, dtype, cache_dtype):
    """Values of two signs that nearly cancel: the output is small beside what its terms lose."""
    from cb200 import ops
    g = torch.Generator().manual_seed(D + G)
    L, Hkv = 600, 2
    q = (torch.randn(1, Hkv * G, D, generator=g) * 0.3).to(dtype)
    k = (torch.randn(L, Hkv, D, generator=g) * 0.5).to(cache_dtype)
    sign = torch.where(torch.rand(L, Hkv, D, generator=g) < 0.5, 1.0, -1.0)
    v = (sign * 8.0).to(cache_dtype)
    _check(_run(ops, q, k, v, 16, cuda_device), q, k, v, 2.0 ** -16 if dtype == torch.bfloat16 else 2.0 ** -21)


def test_one_key_against_its_opposite(cuda_device):
    """Two tokens whose values cancel where their weights are equal: the output is the weights' difference."""
    from cb200 import ops
    D = 64
    for dtype, cache_dtype, u in ((torch.bfloat16, torch.bfloat16, 2.0 ** -16), (torch.float16, torch.float16, 2.0 ** -21),
                                  (torch.float16, FP8, 2.0 ** -21)):
        q = torch.zeros(1, 8, D, dtype=dtype)
        q[0, :, 0] = torch.tensor([2.0 ** -i for i in range(8)]).to(dtype)
        k, v = torch.zeros(2, 1, D), torch.ones(2, 1, D)
        k[0, 0, 0], v[1] = 1.0, -1.0
        k, v = k.to(cache_dtype), v.to(cache_dtype)
        _check(_run(ops, q, k, v, 16, cuda_device), q, k, v, u)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("gain", [1.0, 2.0 ** 60, 2.0 ** -60])
def test_small_query_values_beside_a_large_one(cuda_device, D, gain):
    """The row's largest value meets zeros; the scores come from values 2^-20 of it."""
    from cb200 import ops
    g = torch.Generator().manual_seed(D)
    L, Hkv, G = 40, 2, 5
    q = torch.randn(1, Hkv * G, D, generator=g) * 2.0 ** -20
    q[..., 7] = 1.5
    q = q.to(torch.bfloat16)
    k = torch.randn(L, Hkv, D, generator=g) * 100.0
    k[..., 7] = 0.0
    k, v = k.to(FP8), torch.randn(L, Hkv, D, generator=g).to(FP8)
    scale = torch.full((Hkv,), 2.0 ** 14, device=cuda_device)  # scores of about one
    pages = -(-L // 16)
    kc, vc = (torch.zeros(pages * 16, Hkv, D, dtype=torch.uint8) for _ in range(2))
    kc[:L], vc[:L] = k.view(torch.uint8), v.view(torch.uint8)
    kc, vc = (c.view(FP8).view(pages, 16, Hkv, D).to(cuda_device) for c in (kc, vc))
    out = ops.paged_decode_attention((q.float() * gain).to(torch.bfloat16).to(cuda_device), kc, vc,
                                     torch.arange(pages, dtype=torch.int32, device=cuda_device)[None],
                                     torch.tensor([L], dtype=torch.int32, device=cuda_device), k_scale=scale / gain)
    _check(out.double().cpu(), q, k.double() * 2.0 ** 14, v, 2.0 ** -21)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_infinite_values_stay_infinite(cuda_device, dtype):
    from cb200 import ops
    g = torch.Generator().manual_seed(5)
    q = torch.randn(1, 4, 64, generator=g).to(dtype)
    k, v = (torch.randn(90, 2, 64, generator=g).to(dtype) for _ in range(2))
    v[40, 0, 3], v[7, 1, 5], v[50, 1, 9] = float("inf"), -float("inf"), float("inf")
    v[51, 1, 9] = -float("inf")
    out = _run(ops, q, k, v, 16, cuda_device)
    p = torch.softmax(torch.einsum("hgd,lhd->hgl", q[0].double().view(2, 2, 64), k.double()) / 8.0, dim=2)
    ref = torch.einsum("hgl,lhd->hgd", p, v.double()).reshape(1, 4, 64)
    assert torch.equal(torch.isinf(out), torch.isinf(ref)) and torch.equal(torch.isnan(out), torch.isnan(ref))
    assert torch.equal(out[torch.isinf(ref)], ref[torch.isinf(ref)]) and int(torch.isinf(ref).sum()) == 4


@pytest.mark.parametrize("dtype,cache_dtype,top", [(torch.bfloat16, torch.bfloat16, 1e34), (torch.float16, torch.float16, 65504.0),
                                                   (torch.bfloat16, FP8, 448.0)])
def test_vanishing_weights_add_nothing(cuda_device, dtype, cache_dtype, top):
    """The first token holds all the weight and a small value; 20000 others are 2^-200 of it, with large values (whose
    plain sum fp32 still holds). Many sequences over the same pages, so that each CTA meets thousands of them."""
    from cb200 import ops
    L, D, Hkv, B, page = 20000, 64, 8, 64, 64
    q = torch.zeros(B, Hkv, D, dtype=dtype, device=cuda_device)
    q[..., 0] = 16.0
    k = torch.zeros(-(-L // page), page, Hkv, D)
    k[..., 0] = -70.0
    k[0, 0, :, 0] = 0.0
    v = torch.full(k.shape, top)
    v[0, 0] = 2.0 ** -6
    table = torch.arange(k.shape[0], dtype=torch.int32, device=cuda_device).expand(B, -1).contiguous()
    out = ops.paged_decode_attention(q, k.to(cache_dtype).to(cuda_device), v.to(cache_dtype).to(cuda_device), table,
                                     torch.full((B,), L, dtype=torch.int32, device=cuda_device))
    assert torch.all(out == 2.0 ** -6), float(out.float().max())
