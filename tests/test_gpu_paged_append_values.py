"""Values that the append to an e4m3 cache rounds or saturates: every byte is that of the
fp32 quotient key / scale, to nearest even, saturated at 448, whatever the rows' alignment.
NaN keys alone become NaN."""

import pytest
import torch

pytestmark = pytest.mark.gpu

FP8 = torch.float8_e4m3fn


def _bytes(v):
    """fp32 -> e4m3 bytes; every NaN is 0x7F."""
    b = v.clamp(-448.0, 448.0).to(FP8).view(torch.uint8)
    return torch.where(torch.isnan(v), torch.full_like(b, 0x7F), b)


def _same(got, want):
    got = torch.where((got & 0x7F) == 0x7F, torch.full_like(got, 0x7F), got)
    assert torch.equal(got, want), f"{int((got != want).sum())} bytes differ"


def _append(ops, k, scale, heads, D):
    """The e4m3 rows that keys k [T, heads, D] become, as bytes; as keys and as values."""
    T = k.shape[0]
    kc, vc = (torch.zeros(-(-T // 16), 16, heads, D, dtype=torch.uint8, device=k.device).view(FP8) for _ in range(2))
    ops.paged_kv_append(k, k, kc, vc, torch.arange(T, device=k.device), scale, scale)
    kb, vb = (c.view(torch.uint8).view(-1, heads, D)[:T] for c in (kc, vc))
    assert torch.equal(kb, vb)
    return kb


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("aligned", [True, False])
def test_infinite_and_overflowing_keys_saturate(cuda_device, dtype, aligned):
    from cb200 import ops
    top = torch.finfo(dtype).max
    values = [float("inf"), -float("inf"), float("nan"), 0.0, -0.0, top, -top, top / 2, 60000.0, -60000.0, 448.0, -464.0, 465.0, 1.0,
              -1e-3, 2.0 ** -24]
    scales = torch.tensor([1.0, 0.05, 1e-3, 7.3, 2.0 ** -59, 2.0 ** -80, 2.0 ** 100], device=cuda_device)
    D = 64
    g = torch.Generator().manual_seed(0)
    k = torch.randn(len(values), len(scales), D, generator=g)
    for t, v in enumerate(values):
        k[t, :, t] = v  # one such element among ordinary ones ...
        k[t, :, 56:] = v  # ... and a vector of them
    store = torch.zeros(len(values), len(scales), D + (0 if aligned else 1), dtype=dtype, device=cuda_device)
    rows = store[:, :, :D] if aligned else store[:, :, 1:]
    rows.copy_(k.to(dtype))
    _same(_append(ops, rows, scales, len(scales), D), _bytes(rows.float() / scales[:, None]))


def _scales(n, seed):
    """Divisors over the ordinary range: random, with few bits, and next to powers of two."""
    g = torch.Generator().manual_seed(seed)
    m = 1.0 + torch.rand(n, generator=g)
    m[::4] = 1.0 + torch.randint(0, 16, (len(m[::4]),), generator=g) / 16.0
    m[1::8] = 2.0 - 2.0 ** -23 * torch.randint(1, 4, (len(m[1::8]),), generator=g)
    m[5::8] = 1.0 + 2.0 ** -23 * torch.randint(1, 4, (len(m[5::8]),), generator=g)
    return torch.ldexp(m, torch.randint(-30, 31, (n,), generator=g))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_every_16_bit_key_over_many_scales(cuda_device, dtype):
    """All bit patterns over 4096 scales: the quotient by reciprocal and remainder rounds as a division does."""
    from cb200 import ops
    heads, D = 256, 8
    k = torch.arange(65536, device=cuda_device).to(torch.int16).view(dtype).view(-1, 1, D).expand(-1, heads, D)
    for seed in range(16):
        s = _scales(heads, seed).to(cuda_device)
        _same(_append(ops, k, s, heads, D), _bytes(k.float() / s[:, None]))
