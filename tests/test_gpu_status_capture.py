"""The status block of a device when the first call that needs it is being captured.  Needs a B200."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_a_status_block_made_during_a_capture_is_its_own(cuda_device):
    """Two graphs of one memory pool: the second's capture makes the status block, and the first one's temporaries, which
    had the same pool before it, must not reach it."""
    from comfyui_b200 import moe_ops as M

    dev = cuda_device
    gen = torch.Generator(device=dev).manual_seed(1)
    x = torch.randn((40, 64), generator=gen, device=dev).bfloat16()
    w = torch.randn((2, 72, 64), generator=gen, device=dev).bfloat16()
    off = torch.tensor([0, 20, 40], dtype=torch.int32, device=dev)
    want = M.grouped_matmul(x, w, off)
    kept = dict(M._device_status)
    M._device_status.clear()                                   # as in a process that has made no call yet
    try:
        pool = torch.cuda.graph_pool_handle()
        first, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(first, pool=pool):
            total = sum(torch.full((4,), 7, dtype=torch.int32, device=dev).sum() for _ in range(64))
        with torch.cuda.graph(second, pool=pool):
            y = M.grouped_matmul(x, w, off)
        status = M.device_status(dev)
        for graph in (first, second, first):
            graph.replay()
            torch.cuda.synchronize()
            assert status.tolist() == [0] * 4
            # (a replay may overwrite the other graph's results, which lie in the same pool)
            assert torch.equal(y, want) if graph is second else total.item() == 64 * 28
        M.read_status(status)
        assert M.device_status(dev) is status and M.device_status(str(dev)) is status
    finally:
        M._device_status.clear()
        M._device_status.update(kept)
