"""Dimensions of size one: their stride is not a distance between anything, and frameworks
give any value there (torch: 1 for a transposed column). Such tensors are taken as what
they are, and a call that is refused has written nothing."""

import pytest
import torch

pytestmark = pytest.mark.gpu

FP8 = torch.float8_e4m3fn


def _fp8(g, *shape):
    return (torch.randn(*shape, generator=g) * 60.0).clamp(-448.0, 448.0).to(FP8)


def _odd(t, dim, stride=1):
    """t with another stride in its dimension `dim` of size one."""
    assert t.shape[dim] == 1
    s = list(t.stride())
    s[dim] = stride
    return t.as_strided(t.shape, s)


def _operands(M, N, K, d):
    g = torch.Generator().manual_seed(M + N + K)
    KB, NB = -(-K // 128), -(-N // 128)
    return [t.to(d) for t in (_fp8(g, M, K), _fp8(g, N, K), torch.rand(M, KB, generator=g), torch.rand(NB, KB, generator=g))]


@pytest.mark.parametrize("stride", [0, 1, 7])
@pytest.mark.parametrize("M,N", [(1, 300), (5, 1), (1, 1), (200, 1)])
def test_one_token_or_one_channel(cuda_device, M, N, stride):
    from cb200 import ops
    aq, w, a_s, w_s = _operands(M, N, 272, cuda_device)
    ref = ops.fp8_block_gemm(aq, w, a_s, w_s, out_dtype=torch.float32)
    a2, as2 = (_odd(t, 0, stride) if M == 1 else t for t in (aq, a_s))
    w2 = _odd(w, 0, stride) if N == 1 else w
    ws2 = _odd(w_s, 0, stride) if N <= 128 else w_s
    assert torch.equal(ops.fp8_block_gemm(a2, w2, as2, ws2, out_dtype=torch.float32), ref)


def test_one_batch_entry(cuda_device):
    from cb200 import ops
    ops3 = [t[None] for t in _operands(3, 130, 144, cuda_device)]
    ref = ops.fp8_block_gemm(*ops3, out_dtype=torch.float32)
    assert torch.equal(ops.fp8_block_gemm(*(_odd(t, 0, 5) for t in ops3), out_dtype=torch.float32), ref)


@pytest.mark.parametrize("M", [1, 4])
def test_dynamic_call(cuda_device, M):
    from cb200 import ops
    d = cuda_device
    _, w, _, w_s = _operands(M, 256, 512, d)
    a = torch.randn(M, 512, generator=torch.Generator().manual_seed(1)).bfloat16().to(d)
    ref = ops.fp8_block_gemm_dynamic(a, w, w_s)
    q_ref, s_ref = ops.quant_act_fp8_block(a)
    if M == 1:
        column = a.view(512, 1).t()
        assert column.stride() == (1, 1)
        q, s = (_odd(torch.zeros_like(t), 0) for t in (q_ref, s_ref))
        assert torch.equal(ops.fp8_block_gemm_dynamic(column, w, w_s, q=q, s=s), ref)
        assert torch.equal(q.view(torch.uint8), q_ref.view(torch.uint8)) and torch.equal(s, s_ref)
        assert torch.equal(ops.quant_act_fp8_block(column)[0].view(torch.uint8), q_ref.view(torch.uint8))
    # refused (rows of w off the 16-byte grid): q and s are as they were
    wide = torch.zeros(256, 520, dtype=torch.uint8, device=d).view(FP8)[:, :512]
    q, s = torch.full_like(q_ref.view(torch.uint8), 0x33), torch.full_like(s_ref, 7.0)
    with pytest.raises(ValueError):
        ops.fp8_block_gemm_dynamic(a, wide, w_s, q=q.view(FP8), s=s)
    assert bool((q == 0x33).all()) and bool((s == 7.0).all())


def _cache(g, pages, page, heads, D, dtype, d):
    t = torch.randn(pages, page, heads, D, generator=g)
    return (t.clamp(-448.0, 448.0).to(FP8) if dtype == FP8 else t.to(dtype)).to(d)


@pytest.mark.parametrize("dtype", [torch.bfloat16, FP8])
@pytest.mark.parametrize("pages,page,heads,dim", [(4, 16, 1, 2), (40, 1, 2, 1), (1, 64, 2, 0)])
def test_caches(cuda_device, pages, page, heads, dim, dtype):
    from cb200 import ops
    d, g, D = cuda_device, torch.Generator().manual_seed(pages), 64
    kc, vc = (_cache(g, pages, page, heads, D, dtype, d) for _ in range(2))
    q = torch.randn(1, heads, D, generator=g).bfloat16().to(d)
    table, lens = torch.arange(pages, dtype=torch.int32, device=d)[None], torch.tensor([pages * page - 3], dtype=torch.int32, device=d)
    ref = ops.paged_decode_attention(q, kc, vc, table, lens)
    for stride in (0, 1, 7):
        q2 = _odd(q, 0, stride)
        if heads == 1:
            q2 = _odd(q2, 1, stride)
        assert torch.equal(ops.paged_decode_attention(q2, _odd(kc, dim, stride), _odd(vc, dim, stride), _odd(table, 0, stride), lens), ref)
    k = torch.randn(1, heads, D, generator=g).bfloat16().to(d)
    slots = torch.tensor([5], dtype=torch.int32, device=d)
    k2, v2 = kc.clone(), vc.clone()
    ops.paged_kv_append(k, -k, k2, v2, slots)
    ops.paged_kv_append(_odd(k, 0, 3), _odd(-k, 0, 3), _odd(kc, dim, 3), _odd(vc, dim, 3), slots)
    bits = torch.uint8 if dtype == FP8 else torch.int16
    assert torch.equal(kc.view(bits), k2.view(bits)) and torch.equal(vc.view(bits), v2.view(bits))
    assert ops.device_status(d) == 0
