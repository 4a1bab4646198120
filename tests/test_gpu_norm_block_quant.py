"""Residual RMSNorm with 8-bit outputs (cb_add_rmsnorm_quant) and the per-128 e4m3
quantizer (cb_quant_act_fp8_block) against their formulas.

q depends on u = (x + residual) * weight alone, and every operation on the way
(one addition, one product, two divisions, one rounding) is a single correctly
rounded one, so q and the stored sum are compared bit for bit. A scale is
step / sqrt(mean(h^2) + eps): a thread adds at most 48 squares by fused multiply-add,
ten more additions join the threads, so the sum is within 58 * 2^-24 of exact, its
root within 29 * 2^-24, and the division by H, the addition, the root, the reciprocal
and the product with the step (itself one division) add 6 more: 35 * 2^-24 < 2.1e-6.
"""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

SCALE_RTOL = 2.1e-6


def _e4m3(v: torch.Tensor) -> torch.Tensor:
    return v.clamp(-448.0, 448.0).to(torch.float8_e4m3fn)


def _groups(u: torch.Tensor, size: int) -> torch.Tensor:
    pad = -u.shape[1] % size
    return torch.nn.functional.pad(u, (0, pad)).view(u.shape[0], -1, size)


def _reference(x, w, eps, res, mode):
    """(q as its numbers in fp32, scales in fp64, h or None), on the CPU."""
    h32 = x.float() if res is None else x.float() + res.float()
    u = h32 * w.float()
    size = 128 if mode == "fp8_block" else x.shape[1]
    g = _groups(u, size)
    top = torch.tensor(127.0 if mode == "int8" else 448.0)
    step = torch.maximum(g.abs().amax(dim=2) / top, torch.tensor(2.0 ** -100))
    v = g / step[:, :, None]
    if mode == "int8":
        q = torch.trunc(v + torch.copysign(torch.tensor(0.5), v))
    else:
        q = _e4m3(v).float()
    q = q.reshape(x.shape[0], -1)[:, :x.shape[1]]
    hd = x.double() if res is None else x.double() + res.double()
    ms = (hd * hd).mean(dim=1, keepdim=True)
    s = step.double() / torch.sqrt(ms + eps)
    return q, s if mode == "fp8_block" else s[:, 0], None if res is None else h32.to(x.dtype)


def _check(got, ref):
    q, s, h = (None if t is None else t.cpu() for t in got)
    rq, rs, rh = ref
    assert torch.equal(q.float(), rq)
    assert torch.all((s.double() - rs).abs() <= SCALE_RTOL * rs)
    if rh is None:
        assert h is None
    else:
        assert torch.equal(h.view(torch.int16), rh.view(torch.int16))


def _inputs(rows, H, dtype, w_dtype, seed, residual=True):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, H, generator=g) * 2.0).to(dtype)
    res = (torch.randn(rows, H, generator=g) * 3.0).to(dtype) if residual else None
    w = (1.0 + 0.2 * torch.randn(H, generator=g)).to(w_dtype)
    return x, w, res


def _dev(d, *ts):
    return [None if t is None else t.to(d) for t in ts]


@pytest.mark.parametrize("mode", ["int8", "fp8", "fp8_block"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,H", [(1, 1), (1, 5120), (3, 127), (5, 128), (9, 129), (7, 1000), (4, 1024), (300, 1032),
                                    (33, 8192), (2, 17408), (301, 4096), (2, 32768), (3, 32776), (2, 40001)])
def test_norm_matches_formula(cuda_device, rows, H, dtype, mode):
    from cb200 import ops
    x, w, res = _inputs(rows, H, dtype, dtype, rows * 13 + H)
    xd, wd, rd = _dev(cuda_device, x, w, res)
    _check(ops.add_rmsnorm_quant(xd, wd, 1e-6, residual=rd, mode=mode), _reference(x, w, 1e-6, res, mode))
    _check(ops.add_rmsnorm_quant(xd, wd, 1e-5, mode=mode), _reference(x, w, 1e-5, None, mode))


@pytest.mark.parametrize("mode", ["int8", "fp8", "fp8_block"])
@pytest.mark.parametrize("dtype,w_dtype", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32)])
@pytest.mark.parametrize("rows,H", [(1300, 1032), (1201, 4000), (2500, 8192), (1184, 16384), (5000, 2048), (3000, 512)])
def test_norm_many_rows(cuda_device, rows, H, dtype, w_dtype, mode):
    from cb200 import ops
    x, w, res = _inputs(rows, H, dtype, w_dtype, rows + H)
    x[rows // 2] *= 100.0  # a row of another scale in the middle of a CTA's rows
    xd, wd, rd = _dev(cuda_device, x, w, res)
    _check(ops.add_rmsnorm_quant(xd, wd, 1e-6, residual=rd, mode=mode, h=rd), _reference(x, w, 1e-6, res, mode))
    _check(ops.add_rmsnorm_quant(xd, wd, 1e-6, mode=mode), _reference(x, w, 1e-6, None, mode))


@pytest.mark.parametrize("w_dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("mode", ["int8", "fp8_block"])
def test_norm_weight_types(cuda_device, w_dtype, mode):
    from cb200 import ops
    x, w, res = _inputs(6, 2048, torch.bfloat16, w_dtype, 5)
    _check(ops.add_rmsnorm_quant(*_dev(cuda_device, x, w), 1e-6, residual=res.to(cuda_device), mode=mode),
           _reference(x, w, 1e-6, res, mode))


@pytest.mark.parametrize("mode", ["int8", "fp8", "fp8_block"])
@pytest.mark.parametrize("H,offset,pitch", [(512, 8, 640), (512, 3, 515), (260, 0, 272), (40000, 1, 40008)])
def test_norm_strided_rows_and_outputs(cuda_device, H, offset, pitch, mode):
    """Rows at any start and pitch, outputs with pitches of their own; what lies between the rows stays."""
    from cb200 import ops
    rows = 5
    x, w, res = _inputs(rows, H, torch.float16, torch.float16, H + offset)

    def spread(t, fill):
        buf = torch.full((rows, pitch + offset), fill, dtype=t.dtype)
        buf[:, offset:offset + H] = t
        return buf.to(cuda_device)

    bx, br = spread(x, 99.0), spread(res, 77.0)
    q_dtype = torch.int8 if mode == "int8" else torch.float8_e4m3fn
    bq = torch.zeros(rows, pitch + offset, dtype=torch.uint8, device=cuda_device)
    groups = -(-H // 128) if mode == "fp8_block" else 1
    bs = torch.full((rows, groups + 2), -1.0, device=cuda_device)
    s = bs[:, :groups] if mode == "fp8_block" else bs[:, 0]
    q = bq.view(q_dtype)[:, offset:offset + H]
    got = ops.add_rmsnorm_quant(bx[:, offset:offset + H], w.to(cuda_device), 1e-6, residual=br[:, offset:offset + H],
                                mode=mode, q=q, s=s, h=br[:, offset:offset + H])
    _check((got[0].contiguous() if mode == "int8" else bq[:, offset:offset + H].contiguous().view(q_dtype), got[1], got[2]),
           _reference(x, w, 1e-6, res, mode))
    assert torch.all(bq[:, :offset] == 0) and torch.all(bq[:, offset + H:] == 0)
    assert torch.all(bs[:, groups:] == -1.0)
    assert torch.all(br[:, :offset] == 77.0) and torch.all(br[:, offset + H:] == 77.0)
    assert torch.equal(bx[:, offset:offset + H].cpu(), x)


@pytest.mark.parametrize("mode", ["int8", "fp8", "fp8_block"])
def test_norm_special_rows(cuda_device, mode):
    """A zero row, a tiny row, a huge row, a zero weight, a NaN and an infinity: each stays in its row."""
    from cb200 import ops
    x, w, res = _inputs(6, 1024, torch.bfloat16, torch.float32, 3)
    x[1], res[1] = 0.0, 0.0
    x[2], res[2] = x[2] * 2.0 ** -110, 0.0
    x[3] = x[3] * 2.0 ** 50
    w[100] = 0.0
    xs = x.clone()
    xs[4, 7], xs[5, 900] = float("nan"), float("inf")
    q, s, h = (t.cpu() for t in ops.add_rmsnorm_quant(xs.to(cuda_device), w.to(cuda_device), 1e-6,
                                                      residual=res.to(cuda_device), mode=mode))
    rq, rs, rh = _reference(x, w, 1e-6, res, mode)
    assert torch.equal(q[:4].float(), rq[:4])
    assert torch.all((s[:4].double() - rs[:4]).abs() <= SCALE_RTOL * rs[:4])
    assert torch.all(q[1].float() == 0) and torch.all(s[1] > 0)
    assert torch.all(torch.isnan(s[4]))
    assert torch.isnan(h[4, 7]) and torch.isinf(h[5, 900])
    # the infinity's row: its scale (of the group that holds it) is NaN; no row takes part in another's
    assert torch.isnan(s[5, 900 // 128] if mode == "fp8_block" else s[5])


def test_norm_in_place_and_streams(cuda_device):
    from cb200 import ops
    x, w, res = _inputs(64, 5120, torch.bfloat16, torch.bfloat16, 11)
    ref = _reference(x, w, 1e-6, res, "fp8_block")
    side = torch.cuda.Stream()
    xd, wd, rd = _dev(cuda_device, x, w, res)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.add_rmsnorm_quant(xd, wd, 1e-6, residual=rd, mode="fp8_block", h=rd)
    side.synchronize()
    assert got[2] is rd
    _check(got, ref)
    got = ops.add_rmsnorm_quant(xd, wd, 1e-6, residual=res.to(cuda_device), mode="int8", h=xd)
    _check(got, _reference(x, w, 1e-6, res, "int8"))


def test_norm_feeds_the_int8_and_fp8_gemms(cuda_device):
    """The outputs are the other GEMMs' operands as they are."""
    from cb200 import ops
    x, w, res = _inputs(3, 1024, torch.bfloat16, torch.bfloat16, 4)
    g = torch.Generator().manual_seed(1)
    wt = torch.randint(-127, 128, (256, 1024), generator=g, dtype=torch.int32).to(torch.int8).to(cuda_device)
    ws = torch.rand(256, generator=g).to(cuda_device) * 0.01
    q, s, _ = ops.add_rmsnorm_quant(*_dev(cuda_device, x, w), 1e-6, residual=res.to(cuda_device), mode="int8")
    y = ops.w8a8_gemm(q, wt, s, ws, out_dtype=torch.float32)
    ref = (q.double() * s.double()[:, None]) @ (wt.double() * ws.double()[:, None]).t()
    assert torch.all((y.double() - ref).abs() <= 1e-6 * ref.abs().max())


def test_norm_empty_and_refusals(cuda_device):
    from cb200 import ops
    d = cuda_device
    x, w = torch.randn(4, 256, device=d).bfloat16(), torch.ones(256, device=d).bfloat16()
    q, s, h = ops.add_rmsnorm_quant(x[:0], w, mode="fp8_block")
    assert q.shape == (0, 256) and s.shape == (0, 2) and h is None
    for bad in (
        lambda: ops.add_rmsnorm_quant(x, w, mode="int4"),
        lambda: ops.add_rmsnorm_quant(x, w[:255]),
        lambda: ops.add_rmsnorm_quant(x.t(), w[:4]),
        lambda: ops.add_rmsnorm_quant(x.float(), w),
        lambda: ops.add_rmsnorm_quant(x, w, -1.0),
        lambda: ops.add_rmsnorm_quant(x, w, float("nan")),
        lambda: ops.add_rmsnorm_quant(x, w, residual=x[:3]),
        lambda: ops.add_rmsnorm_quant(x, w, residual=x.half()),
        lambda: ops.add_rmsnorm_quant(x, w, h=torch.empty_like(x)),
        lambda: ops.add_rmsnorm_quant(x, w, q=torch.empty(4, 256, dtype=torch.uint8, device=d)),
        lambda: ops.add_rmsnorm_quant(x, w, mode="fp8_block", s=torch.empty(4, device=d)),
        lambda: ops.add_rmsnorm_quant(x, w, s=torch.empty(3, device=d)),
        lambda: ops.add_rmsnorm_quant(x, w.cpu()),
        lambda: ops.add_rmsnorm_quant(x.expand(2, 4, 256)[0].as_strided((4, 256), (128, 1)), w),
        lambda: ops.quant_act_fp8_block(x.float()),
        lambda: ops.quant_act_fp8_block(x, s=torch.empty(4, 3, device=d)),
        lambda: ops.quant_act_fp8_block(x, q=torch.empty(4, 256, device=d)),
    ):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(1, 16), (1, 128), (3, 129), (33, 5136), (2, 5, 1000), (3, 7, 17), (2, 300, 256)])
def test_block_quantizer_bit_exact(cuda_device, shape, dtype):
    from cb200 import ops
    g = torch.Generator().manual_seed(sum(shape))
    a = (torch.randn(*shape, generator=g) * 3.0).to(dtype)
    a.view(-1, shape[-1])[0, : min(128, shape[-1])] = 0.0  # a group of zeros
    q, s = ops.quant_act_fp8_block(a.to(cuda_device))
    t = _groups(a.reshape(-1, shape[-1]).float(), 128)
    rs = torch.maximum(t.abs().amax(dim=2) / torch.tensor(448.0), torch.tensor(1.0 / (448.0 * 512.0)))
    rq = _e4m3(t / rs[:, :, None]).reshape(t.shape[0], -1)[:, :shape[-1]]
    assert np.array_equal(s.cpu().numpy().reshape(rs.shape).view(np.uint32), rs.numpy().view(np.uint32))
    assert torch.equal(q.cpu().float().reshape(rq.shape), rq.float())
    # a strided view gives the same
    wide = torch.zeros(*shape[:-1], shape[-1] + 5, dtype=dtype, device=cuda_device)
    wide[..., 3:3 + shape[-1]] = a.to(cuda_device)
    q2, s2 = ops.quant_act_fp8_block(wide[..., 3:3 + shape[-1]])
    assert torch.equal(q2.view(torch.uint8), q.view(torch.uint8)) and torch.equal(s2, s)
