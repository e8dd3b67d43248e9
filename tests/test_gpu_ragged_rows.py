"""Rows of no group and groups without rows at the sizes of the few-row kernels.  Needs a B200."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [1, 2, 5, 8, 9, 40, 300])
@pytest.mark.parametrize("zero", [0, 1])
def test_counts_of_a_single_group_without_offsets(cuda_device, rows, zero):
    """The C entry point takes one group without offsets: what counts leave out is zeroed, or stays, as with offsets."""
    from comfyui_b200 import _native as N
    from comfyui_b200 import moe_ops as M

    dev, n, k = cuda_device, 80, 272
    gen = torch.Generator(device=dev).manual_seed(rows)
    x = torch.randn((rows, k), generator=gen, device=dev).bfloat16()
    w, ws = M.quantize_weight_blocks_e4m3(torch.randn((n, k), generator=gen, device=dev))
    want = M.block_linear(x, w, ws)
    work = torch.empty(N.load().comfy_moe_block_workspace(rows, k), dtype=torch.uint8, device=dev)
    for used in {0, rows // 2, rows - 1, rows, rows + 3}:
        counts = torch.tensor([used], dtype=torch.int32, device=dev)
        out = torch.full((rows, n), 7.0, dtype=x.dtype, device=dev)
        M._call("comfy_moe_block_matmul", 0, x.data_ptr(), k, N.BF16, work.data_ptr(), w.data_ptr(), k, 0, ws.data_ptr(), 0, rows,
                1, n, k, None, counts.data_ptr(), None, zero, out.data_ptr(), n, M.device_status(dev).data_ptr())
        used = min(used, rows)
        assert torch.equal(out[:used], want[:used]) and (out[used:] == (0 if zero else 7)).all()
    M.read_status(M.device_status(dev))
