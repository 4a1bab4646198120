"""Paged key-value cache: the append (cb_paged_kv_append, bit for bit) and the
attention of one new token (cb_paged_decode_attention) against the formulas in 64 bits.

Tolerance of the attention, with A = sum_l p_l |v_l| and Z = max_l scale * sum_d |q_d k_d|:
the probabilities are rounded to the products' 16-bit type (u = 2^-8 bf16, 2^-11 f16:
f16 for e4m3 caches), the scores are fp32 sums of exact products (at most 2^-16 Z
off, 256 additions), so each p is within (u + 2 * 2^-16 Z + 2^-20) and the output
within that times A, plus its own rounding (relative u, or half the type's
least subnormal); queries taken into f16 for an e4m3
cache are rounded to 2^-11 of each value, which moves a score by 2^-11 Z. The log
sum moves by at most the largest score error.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}  # half the least subnormal: the output rounding of a value near zero
FP8 = torch.float8_e4m3fn


def _cast(t, dtype):
    return t.clamp(-448.0, 448.0).to(FP8) if dtype == FP8 else t.to(dtype)


def _index(cache, page, slot):
    """cache[page, slot] for index tensors, for every type."""
    if cache.dtype == FP8:
        return cache.view(torch.uint8)[page, slot].view(FP8)
    return cache[page, slot]


class Case:
    """A batch over a shuffled cache whose unused slots hold NaN."""

    def __init__(self, lens, Hkv, G, D, page, dtype, cache_dtype, seed=0, layout="nhd", width=None, q_gain=1.0):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.Hkv, self.G, self.D, self.page = lens, Hkv, G, D, page
        B = len(lens)
        used = [-(-n // page) for n in lens]
        pages = sum(used) + 2
        order = torch.randperm(pages, generator=g)
        self.width = width or max(1, max(used))
        table = torch.full((B, self.width), 1 << 30, dtype=torch.int32)  # entries past the length are never read
        at = 0
        shape = (pages, page, Hkv, D)
        k, v = (_cast(torch.randn(shape, generator=g) * (3.0 if cache_dtype == FP8 else 1.0), cache_dtype) for _ in range(2))
        live = torch.zeros(pages, page, dtype=torch.bool)
        for b, n in enumerate(lens):
            ids = order[at:at + used[b]]
            table[b, :used[b]] = ids.to(torch.int32)
            at += used[b]
            for t in range(n):
                live[ids[t // page], t % page] = True
        for c in (k, v):
            if cache_dtype == FP8:
                c.view(torch.uint8)[~live] = 0x7F
            else:
                c[~live] = float("nan")
        self.k, self.v, self.table = k, v, table
        self.seq = torch.tensor(lens, dtype=torch.int32)
        self.q = (torch.randn(B, Hkv * G, D, generator=g) * q_gain).to(dtype)
        self.scales = [0.02 + 0.2 * torch.rand(Hkv, generator=g) for _ in range(2)] if cache_dtype == FP8 else [None, None]
        self.scale = 1.0 / math.sqrt(D)
        self.layout = layout

    def device(self, d):
        def place(c):
            if self.layout == "hnd":  # [pages, heads, page, D] storage
                buf = c.view(torch.uint8) if c.dtype == FP8 else c
                buf = buf.transpose(1, 2).contiguous().to(d)
                return (buf.view(FP8) if c.dtype == FP8 else buf).transpose(1, 2)
            return c.to(d)
        return (self.q.to(d), place(self.k), place(self.v), self.table.to(d), self.seq.to(d))

    def exact(self):
        """(out, lse, A, Z) in 64 bits."""
        B, Hq, D = self.q.shape
        out, A = torch.zeros(B, Hq, D, dtype=torch.float64), torch.zeros(B, Hq, D, dtype=torch.float64)
        lse, Z = torch.full((B, Hq), -math.inf, dtype=torch.float64), torch.zeros(B, Hq, dtype=torch.float64)
        for b, n in enumerate(self.lens):
            if n == 0:
                continue
            t = torch.arange(n)
            k, v = (_index(c, self.table[b].long()[t // self.page], t % self.page).double() for c in (self.k, self.v))
            if self.scales[0] is not None:
                k, v = k * self.scales[0].double()[:, None], v * self.scales[1].double()[:, None]
            q = self.q[b].double().view(self.Hkv, self.G, D)
            z = torch.einsum("hgd,lhd->hgl", q, k) * self.scale
            p = torch.softmax(z, dim=2)
            out[b], A[b] = (torch.einsum("hgl,lhd->hgd", p, x).reshape(Hq, D) for x in (v, v.abs()))
            lse[b] = torch.logsumexp(z, dim=2).reshape(Hq)
            Z[b] = (torch.einsum("hgd,lhd->hgl", q.abs(), k.abs()) * self.scale).amax(dim=2).reshape(Hq)
        return out, lse, A, Z

    def check(self, d, ops):
        args = self.device(d)
        lse = torch.full(self.q.shape[:2], 7.0, device=d)
        out = ops.paged_decode_attention(*args, k_scale=None if self.scales[0] is None else self.scales[0].to(d),
                                         v_scale=None if self.scales[1] is None else self.scales[1].to(d), lse=lse)
        ro, rl, A, Z = self.exact()
        fp8 = self.k.dtype == FP8
        dz = Z * (2.0 ** -16 + (2.0 ** -11 if fp8 else 0.0)) + 2.0 ** -20
        u = 2.0 ** -11 if fp8 else U[self.q.dtype]
        err = (out.double().cpu() - ro).abs()
        tol = U[self.q.dtype] * ro.abs() + TINY[self.q.dtype] + (u + 2 * dz)[:, :, None] * A
        assert torch.all(err <= tol), float((err / tol.clamp(min=1e-30)).max())
        live = torch.isfinite(rl)
        assert torch.equal(torch.isfinite(lse.cpu()), live)
        assert torch.all(lse.cpu()[~live] == -math.inf)
        assert torch.all((lse.double().cpu() - rl)[live].abs() <= (dz + 2.0 ** -20 * rl.abs())[live])
        return out


TYPES = [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16), (torch.bfloat16, FP8), (torch.float16, FP8)]


@pytest.mark.parametrize("dtype,cache_dtype", TYPES)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("G", [1, 5, 8, 11, 16, 19])
def test_heads_and_types(cuda_device, G, D, dtype, cache_dtype):
    from cb200 import ops
    Case([0, 1, 15, 16, 17, 64, 200], 2, G, D, 16, dtype, cache_dtype, seed=G + D).check(cuda_device, ops)
    assert ops.device_status(cuda_device) == 0


@pytest.mark.parametrize("page", [1, 5, 16, 24, 48, 64, 256])
@pytest.mark.parametrize("dtype,cache_dtype", TYPES[::3])
@pytest.mark.parametrize("layout", ["nhd", "hnd"])
def test_pages_and_layouts(cuda_device, page, dtype, cache_dtype, layout):
    from cb200 import ops
    Case([3, 63, 65, 130, 0, 257], 3, 4, 128, page, dtype, cache_dtype, seed=page, layout=layout, width=300).check(cuda_device, ops)
    assert ops.device_status(cuda_device) == 0


@pytest.mark.parametrize("lens", [[1], [0], [0, 0, 0], [64] * 7, [4097], [1] * 300, list(range(260)), [9000, 1, 1, 0, 700], [40000],
                                  [257, 256, 255, 320, 321] * 9])
@pytest.mark.parametrize("dtype,cache_dtype", [TYPES[0], TYPES[3]])
def test_lengths(cuda_device, lens, dtype, cache_dtype):
    from cb200 import ops
    case = Case(lens, 2, 3, 64, 32, dtype, cache_dtype, seed=len(lens))
    first = case.check(cuda_device, ops)
    assert torch.equal(case.check(cuda_device, ops), first)  # parts are joined in one order


@pytest.mark.parametrize("dtype,cache_dtype", TYPES)
def test_sharp_and_extreme_scores(cuda_device, dtype, cache_dtype):
    """Large queries (one key takes all the weight) and keys whose scores run over hundreds."""
    from cb200 import ops
    for gain in (1e-4, 20.0, 300.0):
        Case([1, 40, 500], 2, 5, 128, 16, dtype, cache_dtype, seed=8, q_gain=gain).check(cuda_device, ops)


def test_large_bf16_queries_over_fp8(cuda_device):
    """Queries beyond f16's range over an e4m3 cache: the scale brings the scores back."""
    from cb200 import ops
    case = Case([300, 17], 2, 4, 128, 16, torch.bfloat16, FP8, seed=2, q_gain=1.0)
    case.q = (case.q.float() * 2.0 ** 40).to(torch.bfloat16)
    case.scales[0] = case.scales[0] * 2.0 ** -40
    case.check(cuda_device, ops)
    case.q = (case.q.float() * 2.0 ** -90).to(torch.bfloat16)
    case.scales[0] = case.scales[0] * 2.0 ** 90
    case.check(cuda_device, ops)


def test_nan_and_infinity_in_the_cache_are_seen(cuda_device):
    from cb200 import ops
    case = Case([100, 100], 1, 2, 64, 16, torch.float16, torch.float16)
    page, slot = int(case.table[0, 50 // 16]), 50 % 16
    case.v[page, slot, 0, 3] = float("nan")
    q, k, v, table, lens = case.device(cuda_device)
    out = ops.paged_decode_attention(q, k, v, table, lens)
    assert torch.all(torch.isnan(out[0, :, 3]))
    assert not torch.any(torch.isnan(out[1])) and not torch.any(torch.isnan(out[0, :, :3]))
    case.k[page, slot, 0, :] = float("nan")
    q, k, v, table, lens = case.device(cuda_device)
    out = ops.paged_decode_attention(q, k, v, table, lens)
    assert torch.all(torch.isnan(out[0])) and not torch.any(torch.isnan(out[1]))


def test_wrong_pages_and_lengths_are_reported(cuda_device):
    """A page outside the cache counts as masked, a length outside the table is clamped; both are reported."""
    from cb200 import ops
    ops.device_status(cuda_device)
    case = Case([48, 32], 1, 2, 64, 16, torch.bfloat16, torch.bfloat16, seed=5)
    q, k, v, table, lens = case.device(cuda_device)
    ref = ops.paged_decode_attention(q, k, v, table, lens)
    assert ops.device_status(cuda_device) == 0
    wrong = table.clone()
    wrong[0, 2] = k.shape[0]  # the third page of sequence 0: its first 32 tokens remain
    out = ops.paged_decode_attention(q, k, v, wrong, lens)
    short = lens.clone()
    short[0] = 32
    assert torch.equal(out, ops.paged_decode_attention(q, k, v, table, short))
    assert ops.device_status(cuda_device) & 2
    wrong[0, 2] = -5
    assert torch.equal(ops.paged_decode_attention(q, k, v, wrong, lens), out)
    assert ops.device_status(cuda_device) & 2
    wrong[0] = -1  # no page at all: as an empty sequence
    lse = torch.zeros(2, 2, device=cuda_device)
    out = ops.paged_decode_attention(q, k, v, wrong, lens, lse=lse)
    assert torch.all(out[0] == 0) and torch.all(lse[0] == -math.inf) and torch.equal(out[1], ref[1])
    assert ops.device_status(cuda_device) & 2
    long = lens.clone()
    long[0], long[1] = 49, -1  # one past the table's three pages; a negative length
    out = ops.paged_decode_attention(q, k, v, table, long)
    assert torch.equal(out[0], ref[0]) and torch.all(out[1] == 0)
    assert ops.device_status(cuda_device) & 2
    assert ops.device_status(cuda_device) == 0


def test_strided_queries_and_outputs(cuda_device):
    from cb200 import ops
    case = Case([70, 0, 333], 2, 5, 128, 16, torch.bfloat16, torch.bfloat16, seed=4)
    q, k, v, table, lens = case.device(cuda_device)
    ref = ops.paged_decode_attention(q, k, v, table, lens)
    qkv = torch.zeros(3, 14, 131, dtype=q.dtype, device=cuda_device)  # rows off the 16-byte grid
    qkv[:, 1:11, 2:130] = q
    obuf = torch.full((3, 12, 130), 9.0, dtype=q.dtype, device=cuda_device)
    lbuf = torch.full((3, 13), 9.0, device=cuda_device)
    wide = torch.full((3, table.shape[1] + 3), 1 << 30, dtype=torch.int32, device=cuda_device)
    wide[:, :table.shape[1]] = table
    out = ops.paged_decode_attention(qkv[:, 1:11, 2:130], k, v, wide[:, :table.shape[1]], lens, out=obuf[:, 1:11, 1:129],
                                     lse=lbuf[:, :10])
    assert torch.equal(out, ref)
    assert torch.all(obuf[:, 0] == 9.0) and torch.all(obuf[:, 11] == 9.0) and torch.all(obuf[:, :, 0] == 9.0)
    assert torch.all(lbuf[:, 10:] == 9.0)


def test_offsets_past_32_bits(cuda_device):
    """Pages that lie more than 4 GiB into the cache, written by the append and read by the attention."""
    from cb200 import ops
    page, Hkv, D = 64, 8, 128
    pages = 33000  # 128 KiB each: 4.3 GB
    cache = torch.zeros(pages, page, Hkv, D, dtype=torch.bfloat16, device=cuda_device)
    g = torch.Generator().manual_seed(0)
    n = 100
    k = torch.randn(n, Hkv, D, generator=g).bfloat16().to(cuda_device)
    ids = torch.tensor([pages - 1, pages - 3], device=cuda_device)
    t = torch.arange(n, device=cuda_device)
    ops.paged_kv_append(k, k, cache, cache, ids[t // page] * page + t % page)
    assert torch.equal(cache[ids[t // page], t % page], k)
    q = torch.randn(1, Hkv, D, generator=g).bfloat16().to(cuda_device)
    out = ops.paged_decode_attention(q, cache, cache, ids.to(torch.int32)[None], torch.tensor([n], dtype=torch.int32, device=cuda_device))
    z = torch.einsum("hd,lhd->hl", q[0].double(), k.double()) / math.sqrt(D)
    ref = torch.einsum("hl,lhd->hd", torch.softmax(z, dim=1), k.double())
    A = torch.einsum("hl,lhd->hd", torch.softmax(z, dim=1), k.double().abs())
    assert torch.all((out[0].double() - ref).abs() <= 2.0 ** -8 * ref.abs() + (2.0 ** -8 + 2.0 ** -10) * A)


def test_graph_follows_lengths_and_streams(cuda_device):
    """A captured step appends and attends; the table and the lengths are read at replay."""
    from cb200 import ops
    case = Case([5, 80], 2, 4, 64, 16, torch.bfloat16, torch.bfloat16, seed=6, width=16)
    q, k, v, table, lens = case.device(cuda_device)
    table.clamp_(max=k.shape[0] - 1)
    new = torch.randn(2, 2, 64, device=cuda_device).bfloat16()
    slots = table[:, 0] * 16 + torch.tensor([5, 0], device=cuda_device, dtype=torch.int32)
    out = torch.empty_like(q)
    ops.paged_kv_append(new, new, k.clone(), v.clone(), slots)
    ops.paged_decode_attention(q, k, v, table, lens, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.paged_kv_append(new, new, k, v, slots)
        ops.paged_decode_attention(q, k, v, table, lens, out=out)
    for ls in ([6, 80], [6, 0], [1, 77]):
        lens.copy_(torch.tensor(ls, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            ref = ops.paged_decode_attention(q, k, v, table, lens)
        side.synchronize()
        assert torch.equal(out, ref)


# ---------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("cache_dtype", [torch.bfloat16, torch.float16, FP8])
@pytest.mark.parametrize("T,Hkv,D,page", [(1, 1, 64, 16), (7, 3, 128, 5), (40, 2, 256, 16), (5, 2, 20, 4), (1000, 8, 64, 64)])
def test_append_bit_exact(cuda_device, T, Hkv, D, page, dtype, cache_dtype):
    from cb200 import ops
    g = torch.Generator().manual_seed(T + D)
    k, v = ((torch.randn(T, Hkv, D, generator=g) * 2.0).to(dtype) for _ in range(2))
    k[0, 0, 0], v[-1, -1, -1] = 60000.0, -60000.0  # saturates an e4m3 cache
    pages = -(-T // page) + 2
    kc, vc = (_cast(torch.randn(pages, page, Hkv, D, generator=g), cache_dtype) for _ in range(2))
    scales = [0.1 + torch.rand(Hkv, generator=g) for _ in range(2)] if cache_dtype == FP8 else [None, None]
    slots = torch.randperm(pages * page, generator=g)[:T]
    slots[T // 2] = -1  # padding
    kd, vd = kc.to(cuda_device), vc.to(cuda_device)
    for index in (torch.int32, torch.int64):
        ops.paged_kv_append(k.to(cuda_device), v.to(cuda_device), kd, vd, slots.to(index).to(cuda_device),
                            *(None if s is None else s.to(cuda_device) for s in scales))
    for src, cache, got, s in ((k, kc, kd, scales[0]), (v, vc, vd, scales[1])):
        val = src.float() if s is None else src.float() / s[:, None]
        raw = (cache.view(torch.uint8) if cache_dtype == FP8 else cache).view(pages * page, Hkv, D)
        new = _cast(val, cache_dtype)
        keep = slots >= 0
        raw[slots[keep]] = (new.view(torch.uint8) if cache_dtype == FP8 else new)[keep]
        bits = torch.uint8 if cache_dtype == FP8 else torch.int16
        assert torch.equal(got.cpu().view(bits), cache.view(bits))


def test_append_strides_and_wrong_slots(cuda_device):
    from cb200 import ops
    ops.device_status(cuda_device)
    T, Hkv, D, page = 6, 2, 64, 4
    qkv = torch.randn(T, 3 * Hkv, D + 1, device=cuda_device).half()
    k, v = qkv[:, :Hkv, 1:], qkv[:, Hkv:2 * Hkv, 1:]
    store = torch.zeros(5, Hkv, page, D, dtype=torch.float16, device=cuda_device)  # [pages, heads, page, D]
    guard = torch.zeros(5, Hkv, page, D, dtype=torch.float16, device=cuda_device)
    kc, vc = store.transpose(1, 2), guard.transpose(1, 2)
    slots = torch.tensor([0, 19, 20, 7, 1 << 30, -3], dtype=torch.int32, device=cuda_device)  # 20 slots: two are wrong
    ops.paged_kv_append(k, v, kc, vc, slots)
    assert ops.device_status(cuda_device) & 2
    want_k, want_v = torch.zeros_like(kc), torch.zeros_like(vc)
    for t, s in ((0, 0), (1, 19), (3, 7)):
        want_k[s // page, s % page], want_v[s // page, s % page] = k[t], v[t]
    assert torch.equal(kc, want_k) and torch.equal(vc, want_v)
    assert ops.device_status(cuda_device) == 0


def test_refusals(cuda_device):
    from cb200 import ops
    d = cuda_device
    q = torch.zeros(2, 4, 64, device=d).bfloat16()
    kc = torch.zeros(3, 16, 2, 64, device=d).bfloat16()
    table, lens = torch.zeros(2, 2, dtype=torch.int32, device=d), torch.ones(2, dtype=torch.int32, device=d)
    k, slots = torch.zeros(5, 2, 64, device=d).bfloat16(), torch.zeros(5, dtype=torch.int32, device=d)
    one = torch.ones(2, device=d)
    attn, app = ops.paged_decode_attention, ops.paged_kv_append
    assert attn(q[:0], kc, kc, table[:0], lens[:0]).shape == (0, 4, 64)
    app(k[:0], k[:0], kc, kc, slots[:0])
    for bad in (
        lambda: attn(q.float(), kc, kc, table, lens),
        lambda: attn(q.half(), kc, kc, table, lens),
        lambda: attn(q[:, :3], kc, kc, table, lens),
        lambda: attn(q, kc, kc[:2], table, lens),
        lambda: attn(q, kc, kc.half(), table, lens),
        lambda: attn(q, kc, kc, table.long(), lens),
        lambda: attn(q, kc, kc, table, lens.long()),
        lambda: attn(q, kc, kc, table[:1], lens),
        lambda: attn(q, kc, kc, table, lens[:1]),
        lambda: attn(q, kc, kc, table, lens, k_scale=one),
        lambda: attn(q, kc, kc, table, lens, out=torch.empty(2, 4, 64, device=d)),
        lambda: attn(q, kc, kc, table, lens, lse=torch.empty(2, 3, device=d)),
        lambda: attn(q.cpu(), kc, kc, table, lens),
        lambda: attn(q, kc, kc, table.cpu(), lens),
        lambda: attn(q[..., :32], kc[..., :32], kc[..., :32], table, lens),  # D = 32
        lambda: attn(q, torch.zeros(12000, device=d).bfloat16().as_strided((3, 16, 2, 64), (4000, 129, 64, 1)), kc, table, lens),  # slots off the 16-byte grid
        lambda: app(k.float(), k.float(), kc, kc, slots),
        lambda: app(k, k[:4], kc, kc, slots),
        lambda: app(k, k, kc, kc, slots[:4]),
        lambda: app(k, k, kc, kc, slots.float()),
        lambda: app(k[:, :1], k[:, :1], kc, kc, slots),
        lambda: app(k, k, kc, kc, slots, k_scale=one),
        lambda: app(k, k, kc.view(torch.float8_e4m3fn)[..., :64], kc.view(torch.float8_e4m3fn)[..., :64], slots, k_scale=one[:1]),
    ):
        with pytest.raises(ValueError):
            bad()
