"""An expired wait inside the block-scaled FP8 GEMM ends the call with a status.

The library's test hook (cb_debug_force_wait_timeout) makes one thread that issues MMAs
wait, with a 2 ms limit, on a workspace word that nothing sets, so the first block of
every CTA is never computed while the others are: the warps that hand over alternate
blocks, the epilogue, and the loads in flight all have to come to an end, the caller is
told, and the next call on the same workspace is right again.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu

HOOK_NS = 2_000_000  # 2 ms


def _operands(M, N, K, device):
    g = torch.Generator().manual_seed(M + N + K)
    KB, NB = -(-K // 128), -(-N // 128)
    a, w = ((torch.randn(r, K, generator=g) * 60.0).clamp(-448.0, 448.0).to(torch.float8_e4m3fn) for r in (M, N))
    a_s, w_s = (0.001 * (1.0 + torch.rand(r, KB, generator=g)) for r in (M, NB))
    return [t.to(device) for t in (a, w, a_s, w_s)]


# up to 64 tokens (16, 32 and 64 columns), one block or tile, whole tiles and parts of tiles;
# then 128 x 128 tiles, likewise
@pytest.mark.parametrize("M,N,K", [(1, 2048, 4096), (20, 640, 5120), (64, 1000, 8192), (64, 128, 128), (7, 256, 256), (3, 40000, 512),
                                   (100, 2000, 2048), (128, 1024, 8192), (1000, 1000, 8192), (70, 128, 128), (70, 128, 256)])
def test_expired_wait_ends_the_call(cuda_device, M, N, K):
    from cb200 import _lib as L
    from cb200 import ops
    lib, d = L.load(), cuda_device
    dev = _operands(M, N, K, d)
    ref = ops.fp8_block_gemm(*dev, out_dtype=torch.float32)
    assert ops.device_status(d) == 0
    lib.cb_debug_force_wait_timeout(HOOK_NS)
    try:
        ops.fp8_block_gemm(*dev, out_dtype=torch.float32)
        torch.cuda.synchronize()
    finally:
        lib.cb_debug_force_wait_timeout(0)
    assert ops.device_status(d) & 1
    assert ops.device_status(d) == 0  # read and cleared, the arrival counters with it
    assert torch.equal(ops.fp8_block_gemm(*dev, out_dtype=torch.float32), ref)
    assert ops.device_status(d) == 0


def test_expired_wait_of_the_dynamic_call(cuda_device):
    from cb200 import _lib as L
    from cb200 import ops
    lib, d = L.load(), cuda_device
    _, w, _, w_s = _operands(32, 1024, 4096, d)
    a = torch.randn(32, 4096, generator=torch.Generator().manual_seed(3)).bfloat16().to(d)
    ref = ops.fp8_block_gemm_dynamic(a, w, w_s)
    assert ops.device_status(d) == 0
    lib.cb_debug_force_wait_timeout(HOOK_NS)
    try:
        ops.fp8_block_gemm_dynamic(a, w, w_s)
        torch.cuda.synchronize()
    finally:
        lib.cb_debug_force_wait_timeout(0)
    assert ops.device_status(d) & 1
    assert torch.equal(ops.fp8_block_gemm_dynamic(a, w, w_s), ref)
    assert ops.device_status(d) == 0
