"""Autograd around the products by expert, what needs no GPU: a recorder stands in for the C entry points."""
import pytest
import torch


class Recorder:
    """Calls of the C entry points as {name: arguments}; nothing is launched and no result is written."""

    def __init__(self):
        self.calls = {}

    def __call__(self, name, index, *args):
        self.calls[name] = args


@pytest.fixture
def recorder(monkeypatch):
    from comfyui_b200 import moe_ops as M

    rec = Recorder()
    monkeypatch.setattr(M, "_call", rec)
    monkeypatch.setattr(M, "_place", lambda first, *others: 0)
    monkeypatch.setattr(M, "device_status", lambda device: torch.zeros(4, dtype=torch.int32))
    return rec


def dense_copies():
    """What an offloading hook does: a dense copy when a tensor is saved, handed back in the backward pass."""
    kept = []

    def pack(t):
        kept.append(torch.empty(t.size(), dtype=t.dtype).copy_(t))
        return kept[-1]

    return torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t), kept


def test_gradients_read_the_strides_of_what_a_hook_hands_back(recorder):
    from comfyui_b200 import moe_ops as M

    k, n = 64, 80
    x = torch.zeros((11, 1024), dtype=torch.bfloat16)[:, :k].requires_grad_(True)
    w = torch.zeros((2, 96, 1024), dtype=torch.bfloat16)[:, :n, :k].requires_grad_(True)
    off = torch.tensor([0, 5, 11], dtype=torch.int32)
    dy = torch.zeros((11, n), dtype=torch.bfloat16)
    hooks, kept = dense_copies()
    with hooks:
        y = M.grouped_matmul(x, w, off)
    torch.autograd.grad(y, (x, w), dy)
    kx, kw = [t for t in kept if t.shape == x.shape][0], [t for t in kept if t.shape == w.shape][0]
    args = recorder.calls["comfy_moe_grouped_matmul_wgrad"]
    assert args[2:4] == (kx.data_ptr(), k)                                     # x and its row stride
    args = recorder.calls["comfy_moe_grouped_matmul_dgrad"]
    assert args[2:5] == (kw.data_ptr(), k, n * k)                              # w, its row and its group stride


def test_block_gradients_read_the_strides_of_what_a_hook_hands_back(recorder):
    from comfyui_b200 import moe_ops as M

    k, n = 64, 80
    x = torch.zeros((11, k), dtype=torch.bfloat16, requires_grad=True)
    w = torch.zeros((2, 96, 1024), dtype=torch.uint8).view(torch.float8_e4m3fn)[:, :n, :k]
    ws = torch.ones((2, 1, 1))
    off = torch.tensor([0, 5, 11], dtype=torch.int32)
    dy = torch.zeros((11, n), dtype=torch.bfloat16)
    for call, shape, step in ((lambda: M.grouped_block_linear(x, w, ws, off), w.shape, n * k),
                              (lambda: M.block_linear(x, w[1], ws[1]), w[1].shape, 1)):
        hooks, kept = dense_copies()
        with hooks:
            y = call()
        torch.autograd.grad(y, x, dy)
        kw = [t for t in kept if t.shape == shape][0]
        assert recorder.calls["comfy_moe_block_matmul"][4:7] == (kw.data_ptr(), k, step)


def test_what_a_hook_hands_back_unreadable_is_copied(recorder):
    """Transposed memory and odd addresses."""
    from comfyui_b200 import moe_ops as M

    k, n = 64, 80
    x = torch.zeros((11, k), dtype=torch.bfloat16, requires_grad=True)
    w = torch.zeros((2, n, k), dtype=torch.bfloat16, requires_grad=True)
    off = torch.tensor([0, 5, 11], dtype=torch.int32)

    def other_layout(t):
        if t.dim() == 3:
            return t.transpose(1, 2).contiguous().transpose(1, 2)
        buf = torch.zeros((t.numel() + 1,), dtype=t.dtype)[1:].view(t.shape)
        return buf.copy_(t)

    with torch.autograd.graph.saved_tensors_hooks(other_layout, lambda t: t):
        y = M.grouped_matmul(x, w, off)
    torch.autograd.grad(y, (x, w), torch.zeros((11, n), dtype=torch.bfloat16))
    for name, at, ld in (("comfy_moe_grouped_matmul_dgrad", 2, k), ("comfy_moe_grouped_matmul_wgrad", 2, k)):
        assert recorder.calls[name][at] % 16 == 0 and recorder.calls[name][at + 1] == ld


def test_forward_mode_derivatives_are_refused(recorder):
    """A result without a tangent would read as a derivative of zero."""
    from torch.autograd import forward_ad

    from comfyui_b200 import moe_ops as M
    from comfyui_b200 import torch_ops  # noqa: F401

    x, w = torch.zeros((11, 64), dtype=torch.bfloat16), torch.zeros((2, 48, 64), dtype=torch.bfloat16)
    off = torch.tensor([0, 5, 11], dtype=torch.int32)
    wq, ws, bias = w.to(torch.float8_e4m3fn), torch.ones((2, 1, 1)), torch.zeros(48, dtype=torch.bfloat16)
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))                          # noqa: E731
        for call in (lambda: M.grouped_matmul(dual(x), w, off), lambda: M.grouped_matmul(x, dual(w), off),
                     lambda: M.block_linear(dual(x), wq[0], ws[0]), lambda: M.block_linear(x, wq[0], ws[0], dual(bias)),
                     lambda: M.block_linear(x, wq[0], dual(ws[0])), lambda: M.grouped_block_linear(dual(x), wq, ws, off),
                     lambda: torch.ops.comfyui_b200.grouped_matmul(dual(x), w, off)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
            with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
                call()
        assert M.grouped_matmul(x, w, off).shape == (11, 48)                                 # no operand has a tangent
        assert M.block_linear(x, wq[0], ws[0], bias).shape == (11, 48)


def test_the_gradient_of_a_bias_alone_needs_no_product(recorder):
    """out_features of 8: the gradient of x would contract over them in steps of 16, that of the bias only adds up."""
    from comfyui_b200 import moe_ops as M

    x, bias = torch.zeros((11, 64), dtype=torch.bfloat16), torch.zeros(72, dtype=torch.bfloat16, requires_grad=True)
    w, ws = torch.zeros((72, 64), dtype=torch.bfloat16).to(torch.float8_e4m3fn), torch.ones((1, 1))
    dy = torch.arange(11.0)[:, None].expand(11, 72).bfloat16()
    y = M.block_linear(x, w, ws, bias)
    recorder.calls.clear()
    db, = torch.autograd.grad(y, bias, dy)
    assert (db == 55).all() and not recorder.calls
    with pytest.raises(ValueError, match="multiple of 16 for a gradient"):
        M.block_linear(x.clone().requires_grad_(True), w, ws, bias)


def test_a_frozen_operand_keeps_nothing_of_the_other(recorder):
    """The gradient of x reads w only, that of w x only: what is not read is not kept, and may be overwritten."""
    from comfyui_b200 import moe_ops as M
    from comfyui_b200 import torch_ops  # noqa: F401

    off, dy = torch.tensor([0, 5, 11], dtype=torch.int32), torch.zeros((11, 80), dtype=torch.bfloat16)
    leaf = lambda *shape: torch.zeros(shape, dtype=torch.bfloat16, requires_grad=True)        # noqa: E731
    for call in (M.grouped_matmul, torch.ops.comfyui_b200.grouped_matmul):
        for frozen in (0, 1):
            operands = [leaf(11, 64), leaf(2, 80, 64)]
            operands[frozen] = operands[frozen].detach()
            used = [t * 1 for t in operands]
            kept = []
            with torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append(t.shape) or t, lambda t: t):
                y = call(*used, off)
            assert used[1 - frozen].shape not in kept and used[frozen].shape in kept
            with torch.no_grad():
                used[1 - frozen].add_(1)
            torch.autograd.grad(y, operands[1 - frozen], dy)
    w, ws, bias = torch.zeros((80, 64), dtype=torch.bfloat16).to(torch.float8_e4m3fn), torch.ones((1, 1)), leaf(80)
    kept = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append(t.shape) or t, lambda t: t):
        y = M.block_linear(torch.zeros((11, 64), dtype=torch.bfloat16), w, ws, bias)
    assert not kept and (torch.autograd.grad(y, bias, dy + 1)[0] == 11).all()
