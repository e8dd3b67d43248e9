"""Products by expert and with block scales, what needs no GPU: refusals of the C entry points, the operators' shapes under
tracing, the block-scaled Linear's composition and checkpoint layout."""
import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from comfyui_b200 import _native, build

    build.build()
    return _native.load()


GOOD = ctypes.c_void_p(1 << 20)            # never read: every call here is refused, or has nothing to do, on the host
ODD = ctypes.c_void_p((1 << 20) + 8)


def matmul(lib, name="comfy_moe_grouped_matmul", x=GOOD, ld_x=64, w=GOOD, ld_w=64, step=64 * 32, dtype=0, rows=5, groups=2, n=32,
           k=64, offsets=GOOD, counts=None, zero=1, out=GOOD, ld_out=32, status=GOOD):
    return getattr(lib, name)(x, ld_x, w, ld_w, step, dtype, rows, groups, n, k, offsets, counts, zero, out, ld_out, status, None)


def test_grouped_matmul_refuses_on_the_host(lib):
    from comfyui_b200 import _native as N

    for bad, code in [(dict(x=None), N.EINVAL), (dict(x=ODD), N.EINVAL), (dict(out=ODD), N.EINVAL), (dict(w=None), N.EINVAL),
                      (dict(ld_x=60), N.EINVAL), (dict(ld_x=72 + 4), N.EINVAL), (dict(ld_out=24), N.EINVAL),
                      (dict(step=12), N.EINVAL), (dict(offsets=None), N.EINVAL), (dict(status=None), N.EINVAL),
                      (dict(rows=-1), N.EINVAL), (dict(n=0), N.EINVAL), (dict(k=-8), N.EINVAL),
                      (dict(n=33, ld_out=40), N.EUNSUPPORTED), (dict(k=60), N.EUNSUPPORTED), (dict(dtype=N.FP32), N.EUNSUPPORTED),
                      (dict(groups=N.RAGGED_MAX_GROUPS + 1), N.EUNSUPPORTED)]:
        assert matmul(lib, **bad) == code, bad
    assert matmul(lib, rows=0, x=None, out=None) == N.OK
    assert matmul(lib, "comfy_moe_grouped_matmul_dgrad", ld_x=24) == N.EINVAL           # rows of 32 elements
    call = lib.comfy_moe_grouped_matmul_wgrad
    good = [GOOD, 32, GOOD, 64, 0, 5, 2, 32, 64, GOOD, None, 0, GOOD, 64, 64 * 32, GOOD, None]
    for at, bad, code in [(0, None, N.EINVAL), (2, ODD, N.EINVAL), (11, N.FP16, N.EUNSUPPORTED), (12, None, N.EINVAL),
                          (13, 60, N.EINVAL), (14, 64 * 31, N.EINVAL), (15, None, N.EINVAL), (9, None, N.EINVAL)]:
        args = list(good)
        args[at] = bad
        assert call(*args) == code, at
    args = list(good)
    args[6] = 0
    assert call(*args) == N.OK


def test_block_products_refuse_on_the_host(lib):
    from comfyui_b200 import _native as N

    names = ["x", "ld_x", "dtype", "work", "w", "ld_w", "step", "scale", "transpose", "rows", "groups", "n", "k", "offsets",
             "counts", "bias", "zero", "out", "ld_out", "status", "stream"]
    good = dict(x=GOOD, ld_x=64, dtype=0, work=GOOD, w=GOOD, ld_w=64, step=0, scale=GOOD, transpose=0, rows=50, groups=1, n=32, k=64,
                offsets=None, counts=None, bias=None, zero=0, out=GOOD, ld_out=32, status=GOOD, stream=None)
    for bad, code in [(dict(x=None), N.EINVAL), (dict(work=None), N.EINVAL), (dict(work=ODD), N.EINVAL), (dict(scale=None), N.EINVAL),
                      (dict(ld_x=60), N.EINVAL), (dict(ld_w=72), N.EINVAL), (dict(bias=ODD), N.EINVAL), (dict(groups=2), N.EINVAL),
                      (dict(groups=2, offsets=GOOD, step=24), N.EINVAL), (dict(k=72, ld_x=72, ld_w=80), N.EUNSUPPORTED),
                      (dict(n=36, ld_out=40), N.EUNSUPPORTED), (dict(n=40, ld_out=64, ld_x=40, transpose=1), N.EUNSUPPORTED),
                      (dict(dtype=N.FP8_E4M3), N.EUNSUPPORTED), (dict(status=None), N.EINVAL), (dict(rows=-2), N.EINVAL)]:
        args = {**good, **bad}
        assert lib.comfy_moe_block_matmul(*[args[n] for n in names]) == code, bad
    assert lib.comfy_moe_block_matmul(*[{**good, "rows": 0}[n] for n in names]) == N.OK
    assert lib.comfy_moe_block_quantize(GOOD, 64, 0, 5, 60, GOOD, 64, GOOD, 5, None) == N.EUNSUPPORTED
    assert lib.comfy_moe_block_quantize(GOOD, 64, 0, 5, 64, GOOD, 64, GOOD, 4, None) == N.EINVAL
    assert lib.comfy_moe_block_quantize(None, 64, 0, 0, 64, None, 64, None, 0, None) == N.OK
    assert lib.comfy_moe_block_quantize_weight(GOOD, 64, 0, 0, 1, 32, 72, GOOD, GOOD, None) == N.EUNSUPPORTED
    assert lib.comfy_moe_block_quantize_weight(GOOD, 60, 0, 0, 1, 32, 64, GOOD, GOOD, None) == N.EINVAL
    assert lib.comfy_moe_block_workspace(3, 272) == 1024 + 3 * 3 * 4
    assert lib.comfy_moe_block_workspace(-1, 8) == 0


def test_cpu_tensors_are_refused():
    from comfyui_b200 import moe_ops as M

    x, w = torch.zeros((4, 64), dtype=torch.bfloat16), torch.zeros((2, 32, 64), dtype=torch.bfloat16)
    off = torch.zeros(3, dtype=torch.int32)
    wq, ws = w[0].to(torch.float8_e4m3fn), torch.ones((1, 1))
    for call in (lambda: M.grouped_matmul(x, w, off), lambda: M.grouped_matmul_dgrad(x[:, :32], w, off),
                 lambda: M.grouped_matmul_wgrad(x[:, :32], x, off), lambda: M.quantize_blocks_e4m3(x),
                 lambda: M.quantize_weight_blocks_e4m3(w), lambda: M.block_linear(x, wq, ws),
                 lambda: M.grouped_block_linear(x, wq[None], ws[None], off[:2])):
        with pytest.raises(ValueError, match="no CPU path"):
            call()


def test_operators_trace():
    from torch._subclasses.fake_tensor import FakeTensorMode

    from comfyui_b200 import torch_ops  # noqa: F401

    ops = torch.ops.comfyui_b200
    with FakeTensorMode():
        x, w = torch.empty((7, 64), dtype=torch.bfloat16), torch.empty((3, 32, 64), dtype=torch.bfloat16)
        off, dy = torch.empty(4, dtype=torch.int32), torch.empty((7, 32), dtype=torch.bfloat16)
        assert ops.grouped_matmul(x, w, off).shape == (7, 32)
        assert ops.grouped_matmul_dgrad(dy, w, off).shape == (7, 64)
        assert ops.grouped_matmul_wgrad(dy, x, off).shape == (3, 32, 64)
        wq, ws = torch.empty((32, 64), dtype=torch.float8_e4m3fn), torch.empty((1, 1))
        assert ops.block_linear(x.view(1, 7, 64), wq, ws).shape == (1, 7, 32)
        assert ops.grouped_block_linear(x, wq.expand(3, 32, 64), ws.expand(3, 1, 1), off).shape == (7, 32)


def _linear(n, k, bias=True, **kw):
    from comfyui_b200 import ops

    lin = ops.block_scaled_fp8_ops(**kw).Linear(k, n, bias=bias, dtype=torch.float32)
    g = torch.Generator().manual_seed(n + k)
    state = {"weight": torch.randn((n, k), generator=g).to(torch.float8_e4m3fn),
             "scale_weight": torch.rand(lin.scale_weight.shape, generator=g) + 0.5}
    if bias:
        state["bias"] = torch.randn((n,), generator=g)
    lin.load_state_dict(state, strict=True)
    return lin, state


def test_block_scaled_linear_on_the_host():
    """Layout of the checkpoint, the composition where no kernel runs, its gradient."""
    n, k = 200, 272
    lin, state = _linear(n, k)
    assert lin.weight.dtype == torch.float8_e4m3fn and lin.scale_weight.shape == (2, 3) and not lin.weight.requires_grad
    full = torch.empty((n, k))
    for i in range(n):
        for j in range(k):
            full[i, j] = state["weight"][i, j].float() * state["scale_weight"][i // 128, j // 128]
    x = torch.randn((2, 5, k), requires_grad=True)
    y = lin(x)
    torch.testing.assert_close(y, torch.nn.functional.linear(x, full, state["bias"]))
    gx, gb = torch.autograd.grad(y.sum(), (x, lin.bias))
    torch.testing.assert_close(gx, full.sum(0).expand(2, 5, k))
    torch.testing.assert_close(gb, torch.full((n,), 10.0))
    torch.testing.assert_close(lin.convert_weight(state["weight"].float()), full)


def test_block_scaled_linear_patches():
    """A model patcher's round trip: convert_weight, a change, set_weight with a seed; closures on the weight."""
    n, k = 130, 144
    lin, state = _linear(n, k, bias=False)
    from comfyui_b200 import ops

    back = lin.convert_weight(lin.weight.float())
    spread = torch.ones((256, 256)).view(2, 128, 2, 128).mul(state["scale_weight"][:, None, :, None]).view(256, 256)[:n, :k]
    lin.set_weight(back, seed=3)
    assert torch.equal(lin.weight.view(torch.uint8), ops.stochastic_rounding(back / spread, torch.float8_e4m3fn, 3).view(torch.uint8))
    back = lin.convert_weight(lin.weight.float())
    q = lin.set_weight(back * 1.01, seed=3, return_weight=True)
    assert q.dtype == torch.float8_e4m3fn and torch.equal(q.view(torch.uint8), lin.set_weight(back * 1.01, seed=3,
                                                                                           return_weight=True).view(torch.uint8))
    x = torch.randn((3, k))
    lin.weight_function = [lambda w: w * 2]
    torch.testing.assert_close(lin(x), torch.nn.functional.linear(x, 2 * back))


def test_models_take_the_namespace():
    from comfyui_b200 import ops
    from comfyui_b200.ldm.hidream.model import MOEFeedForwardSwiGLU

    m = MOEFeedForwardSwiGLU(256, 512, 4, 2, dtype=torch.float32, operations=ops.block_scaled_fp8_ops())
    keys = set(m.state_dict())
    assert {"experts.0.w1.weight", "experts.0.w1.scale_weight", "shared_experts.w2.scale_weight", "gate.weight"} <= keys
    with torch.no_grad():
        for name, p in m.named_parameters():
            p.copy_((0.1 * torch.randn(p.shape)).to(p.dtype) if not name.endswith("scale_weight") else torch.rand(p.shape))
        assert torch.isfinite(m(torch.randn((1, 9, 256)))).all()
