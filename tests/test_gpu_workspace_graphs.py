"""Several CUDA graphs of calls that join split work through a workspace: in any order, at
the same time, beside larger calls, and after a graph is gone."""

import time

import pytest
import torch

pytestmark = pytest.mark.gpu

FP8 = torch.float8_e4m3fn


class Gemm:
    """A block-scaled GEMM whose tiles are cut over K."""

    def __init__(self, d, M, N=1024, K=8192, seed=0):
        g = torch.Generator().manual_seed(seed + M)
        self.a, self.w = ((torch.randn(r, K, generator=g) * 60.0).clamp(-448.0, 448.0).to(FP8).to(d) for r in (M, N))
        self.a_s, self.w_s = (0.001 * (1.0 + torch.rand(r, K // 128, generator=g)).to(d) for r in (M, N // 128))
        self.out = torch.zeros(M, N, device=d)

    def __call__(self):
        from cb200 import ops
        ops.fp8_block_gemm(self.a, self.w, self.a_s, self.w_s, out=self.out)


class Attention:
    """One sequence over two heads, cut into many parts."""

    def __init__(self, d, L, D=128, seed=0):
        g = torch.Generator().manual_seed(seed + L)
        pages = -(-L // 64)
        self.q = torch.randn(1, 8, D, generator=g).bfloat16().to(d)
        self.k, self.v = (torch.randn(pages, 64, 2, D, generator=g).bfloat16().to(d) for _ in range(2))
        self.table = torch.arange(pages, dtype=torch.int32, device=d)[None]
        self.lens = torch.tensor([L], dtype=torch.int32, device=d)
        self.out = torch.zeros(1, 8, D, dtype=torch.bfloat16, device=d)

    def __call__(self):
        from cb200 import ops
        ops.paged_decode_attention(self.q, self.k, self.v, self.table, self.lens, out=self.out)


class W8A8:
    """The integer GEMM, whose workspace comes from Python."""

    def __init__(self, d, M, N=512, K=8192):
        g = torch.Generator().manual_seed(M)
        self.a = torch.randint(-127, 128, (M, K), generator=g).to(torch.int8).to(d)
        self.w = torch.randint(-127, 128, (N, K), generator=g).to(torch.int8).to(d)
        self.a_s, self.w_s = torch.rand(M, generator=g).to(d), torch.rand(N, generator=g).to(d)
        self.out = torch.zeros(M, N, dtype=torch.bfloat16, device=d)

    def __call__(self):
        from cb200 import ops
        ops.w8a8_gemm(self.a, self.w, self.a_s, self.w_s, out=self.out)


def _eager(call):
    call()
    torch.cuda.synchronize()
    ref = call.out.clone()
    call.out.zero_()
    return ref


def _capture(*calls, **kw):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, **kw):
        for call in calls:
            call()
    return graph


def _captures():
    from cb200 import ops
    return {k[2] for k in ops.POOL._bufs if k[2]}


@pytest.mark.parametrize("make", [lambda d: (Gemm(d, 1), Gemm(d, 2)), lambda d: (Gemm(d, 100), Gemm(d, 90)),
                                  lambda d: (Attention(d, 20000), Attention(d, 9000)), lambda d: (W8A8(d, 16), W8A8(d, 40)),
                                  lambda d: (Gemm(d, 5), Attention(d, 30000))])
def test_the_second_graph_is_replayed_first(cuda_device, make):
    from cb200 import ops
    calls = make(cuda_device)
    refs = [_eager(c) for c in calls]
    before = _captures()
    graphs = [_capture(c) for c in calls]
    assert len(_captures() - before) == 2
    assert ops.device_status(cuda_device) == 0  # graphs that have not run report nothing
    for i in (1, 0, 1, 1, 0):
        calls[i].out.zero_()
        graphs[i].replay()
        torch.cuda.synchronize()
        assert torch.equal(calls[i].out, refs[i])
    assert ops.device_status(cuda_device) == 0


def test_graphs_replayed_at_the_same_time(cuda_device):
    from cb200 import ops
    calls = [Gemm(cuda_device, 3, N=256), Gemm(cuda_device, 4, N=256), Attention(cuda_device, 40000), Attention(cuda_device, 41000)]
    refs = [_eager(c) for c in calls]
    graphs = [_capture(c, c, c) for c in calls]
    streams = [torch.cuda.Stream() for _ in calls]
    for _ in range(20):
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                for _ in range(5):
                    g.replay()
        torch.cuda.synchronize()
        for c, ref in zip(calls, refs):
            assert torch.equal(c.out, ref)
            c.out.zero_()
    assert ops.device_status(cuda_device) == 0


def test_small_call_before_a_large_one(cuda_device):
    """In one capture, and eagerly on the capture's own stream afterwards; memory handed out later is not written to."""
    from cb200 import ops
    d = cuda_device
    small, large, larger = Gemm(d, 1), Gemm(d, 100), Attention(d, 9000, D=256)
    refs = [_eager(c) for c in (small, large, larger)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        small()  # an eager workspace of that stream comes first
    side.synchronize()
    one = _capture(small, stream=side)
    both = _capture(small, large, larger, stream=side)
    with torch.cuda.stream(side):
        large()
        larger()
    side.synchronize()
    others = [torch.full((1 << 20,), 0x5A, dtype=torch.uint8, device=d) for _ in range(64)]
    for graph, calls in ((one, (small,)), (both, (small, large, larger)), (one, (small,))):
        for c in calls:
            c.out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for c in calls:
            assert torch.equal(c.out, refs[(small, large, larger).index(c)])
    assert all(bool((o == 0x5A).all()) for o in others)
    assert ops.device_status(d) == 0


def _gone(ids):
    from cb200 import _lib as L
    deadline = time.time() + 10.0
    while time.time() < deadline and any(L.load().cb_capture_live(i) for i in ids):
        time.sleep(0.01)
    return not any(L.load().cb_capture_live(i) for i in ids)


def test_a_graph_that_is_gone_gives_its_workspace_back(cuda_device):
    from cb200 import _lib as L
    from cb200 import ops
    call = Gemm(cuda_device, 1)
    ref = _eager(call)
    places = set()
    for _ in range(4):
        before = _captures()
        graph = _capture(call)
        new = _captures() - before
        assert len(new) == 1 and all(L.load().cb_capture_live(i) for i in new)
        (key,) = [k for k in ops.POOL._bufs if k[2] in new]
        places.add(ops.POOL._bufs[key][-1].data_ptr())
        call.out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(call.out, ref)
        del graph
        assert _gone(new)
        assert ops.device_status(cuda_device) == 0
        assert not (_captures() & new)
    assert len(places) == 1


def test_errors_of_a_replay_are_kept_until_they_are_read(cuda_device):
    from cb200 import ops
    d = cuda_device
    ops.device_status(d)
    cache = torch.zeros(2, 16, 1, 64, dtype=torch.bfloat16, device=d)
    k = torch.ones(1, 1, 64, dtype=torch.bfloat16, device=d)
    slots = torch.zeros(1, dtype=torch.int32, device=d)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.paged_kv_append(k, k, cache, cache, slots)
    graph.replay()
    assert ops.device_status(d) == 0
    for slot in (32, 1):  # outside the cache, then inside it
        slots.fill_(slot)
        graph.replay()
    assert ops.device_status(d) & 2
    assert ops.device_status(d) == 0
