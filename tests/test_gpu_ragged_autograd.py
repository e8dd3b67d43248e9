"""Autograd around the products by expert and the block-scaled products: saved-tensor hooks, derivatives that are refused,
what a backward pass keeps.  Needs a B200."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def strided(t, before, behind):
    """The values of t as a slice of wider rows (and, for weights, of more rows), with NaN around them."""
    pad = (before, behind) if t.dim() == 2 else (before, behind, 0, 3)
    wide = torch.nn.functional.pad(t.float(), pad, value=float("nan")).to(t.dtype)
    return wide[..., :t.shape[-2], before:before + t.shape[-1]]


@pytest.mark.parametrize("pin", [False, True], ids=["pageable", "pinned"])
def test_strided_operands_saved_on_the_host(cuda_device, pin):
    """save_on_cpu hands back dense copies of strided operands: the gradients are those of the direct calls."""
    from comfyui_b200 import moe_ops as M

    dev, k, n = cuda_device, 136, 80
    gen = torch.Generator(device=dev).manual_seed(4)
    x = strided(torch.randn((201, k), generator=gen, device=dev).bfloat16(), 8, 512)
    w = strided(torch.randn((2, n, k), generator=gen, device=dev).bfloat16(), 8, 256)
    dy = torch.randn((201, n), generator=gen, device=dev).bfloat16()
    off = torch.tensor([0, 70, 201], dtype=torch.int32, device=dev)
    want = M.grouped_matmul_dgrad(dy, w, off), M.grouped_matmul_wgrad(dy, x, off)
    xg, wg = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    with torch.autograd.graph.save_on_cpu(pin_memory=pin):
        y = M.grouped_matmul(xg, wg, off)
    got = torch.autograd.grad(y, (xg, wg), dy)
    assert all(torch.equal(a, b) for a, b in zip(got, want))

    k = 272
    x = torch.randn((201, k), generator=gen, device=dev).bfloat16()
    wq, ws = M.quantize_weight_blocks_e4m3(torch.randn((2, n, k), generator=gen, device=dev))
    wide = strided(wq, 16, 240)
    assert not wide.is_contiguous()
    want = M.grouped_block_linear_dgrad(dy, wq, ws, off), M.block_linear_dgrad(dy, wq[1], ws[1])
    x.requires_grad_(True)
    with torch.autograd.graph.save_on_cpu(pin_memory=pin):
        ys = M.grouped_block_linear(x, wide, ws, off), M.block_linear(x, wide[1], ws[1])
    for y, expected in zip(ys, want):
        assert torch.equal(torch.autograd.grad(y, x, dy)[0], expected)
    M.read_status(M.device_status(dev))


def test_forward_mode_of_a_linear(cuda_device):
    """The tensor-level calls refuse a dual tensor; a Linear of the namespace composes, so its tangent is that of the weight."""
    from torch.autograd import forward_ad

    from comfyui_b200 import moe_ops as M
    from comfyui_b200 import ops

    dev, n, k = cuda_device, 48, 64
    gen = torch.Generator(device=dev).manual_seed(3)
    lin = ops.block_scaled_fp8_ops().Linear(k, n, device=dev, dtype=torch.bfloat16)
    w, ws = M.quantize_weight_blocks_e4m3(torch.randn((n, k), generator=gen, device=dev))
    lin.load_state_dict({"weight": w, "scale_weight": ws, "bias": torch.zeros(n, device=dev).bfloat16()}, strict=True)
    x = torch.randn((9, k), generator=gen, device=dev).bfloat16()
    along = torch.zeros_like(x)
    along[:, 5] = 1                                          # the tangent is then one column of the weight, rounded once
    with torch.no_grad(), forward_ad.dual_level():
        dual = forward_ad.make_dual(x, along)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            M.block_linear(dual, w, ws)
        got = forward_ad.unpack_dual(lin(dual)).tangent
    want = w.double()[:, 5] * ws.double()[0, 0]
    assert got is not None and ((got.double() - want).abs() <= 2.0 ** -7 * want.abs()).all()


def test_the_gradient_of_a_bias_alone(cuda_device):
    """out_features of 8 stay on the kernel where only the bias asks for a gradient, in the call and in a Linear."""
    from comfyui_b200 import moe_ops as M
    from comfyui_b200 import ops

    dev, n, k = cuda_device, 72, 272
    gen = torch.Generator(device=dev).manual_seed(8)
    x = torch.randn((50, k), generator=gen, device=dev).bfloat16()
    w, ws = M.quantize_weight_blocks_e4m3(torch.randn((n, k), generator=gen, device=dev))
    bias = torch.randn((n,), generator=gen, device=dev).bfloat16()
    dy = torch.randint(-3, 4, (50, n), generator=gen, device=dev).bfloat16()          # sums of whole numbers are exact
    want = M.block_linear(x, w, ws, bias)
    lin = ops.block_scaled_fp8_ops().Linear(k, n, device=dev, dtype=torch.bfloat16)
    lin.load_state_dict({"weight": w, "scale_weight": ws, "bias": bias}, strict=True)
    leaf = bias.clone().requires_grad_(True)
    for y, b in ((M.block_linear(x, w, ws, leaf), leaf), (lin(x), lin.bias)):
        assert torch.equal(y, want)
        assert torch.equal(torch.autograd.grad(y, b, dy)[0], dy.float().sum(0).bfloat16())


@pytest.mark.parametrize("reentrant", [False, True], ids=["hooks", "reentrant"])
def test_under_checkpointing(cuda_device, reentrant):
    """Recomputed operands, slices of a wider projection among them, give the gradients of the plain run bit for bit."""
    from torch.utils.checkpoint import checkpoint

    from comfyui_b200 import moe_ops as M

    dev, k, n = cuda_device, 144, 80
    gen = torch.Generator(device=dev).manual_seed(6)
    off = torch.tensor([0, 70, 70, 201], dtype=torch.int32, device=dev)
    x = torch.randn((201, k), generator=gen, device=dev).bfloat16().requires_grad_(True)
    w = torch.randn((3, 2 * n, k), generator=gen, device=dev).bfloat16().requires_grad_(True)
    v = torch.randn((3, k, n), generator=gen, device=dev).bfloat16().requires_grad_(True)
    wq, ws = M.quantize_weight_blocks_e4m3(torch.randn((64, k), generator=gen, device=dev))
    bias = torch.randn((64,), generator=gen, device=dev).bfloat16().requires_grad_(True)
    dy = torch.randn((201, 64), generator=gen, device=dev).bfloat16()

    def block(x, w, v):
        h = M.grouped_matmul(x, w, off)
        h = M.grouped_matmul(h[:, :n] * torch.sigmoid(h[:, n:]) + 0 * h[:, n:], v, off) + M.grouped_matmul(h[:, n:], v, off)
        return M.block_linear(h, wq, ws, bias)

    leaves = (x, w, v, bias)
    grads = []
    for run in (block, lambda *a: checkpoint(block, *a, use_reentrant=reentrant)):
        for t in leaves:
            t.grad = None
        run(x, w, v).backward(dy)
        grads.append([t.grad for t in leaves])
    assert all(torch.equal(a, b) and torch.isfinite(a).all() for a, b in zip(*grads))
    M.read_status(M.device_status(dev))
