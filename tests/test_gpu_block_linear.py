"""e4m3 with block scales: the quantisers, the products, dense and by expert, and their gradients.  Needs a B200.

The quantisers are held to the bytes of the definition in 64 bits.  A product is held to the 64-bit product of the quantised
operands: one rounding of the result (half a step of its type) plus fp32 roundings: at most (terms + 3 per block) x 2^-23
of the sum of the products' magnitudes."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BLOCK = 128
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def blocks(n):
    return -(-n // BLOCK)


def quantised(x):
    """(q, scale) of rows x by the definition, in 64 bits; q as e4m3 values."""
    r, k = x.shape
    b = torch.nn.functional.pad(x.double(), (0, -k % BLOCK)).view(r, blocks(k), BLOCK)
    m = b.abs().amax(-1, keepdim=True).clamp(min=2.0 ** -100)
    q = (b * 448.0 / m).float().to(torch.float8_e4m3fn)
    return q.view(r, blocks(k) * BLOCK)[:, :k], (m / 448.0).squeeze(-1)


def quantised_weight(w):
    n, k = w.shape
    b = torch.nn.functional.pad(w.double(), (0, -k % BLOCK, 0, -n % BLOCK)).view(blocks(n), BLOCK, blocks(k), BLOCK)
    m = b.abs().amax((1, 3), keepdim=True).clamp(min=2.0 ** -100)
    q = (b * 448.0 / m).float().to(torch.float8_e4m3fn).view(blocks(n) * BLOCK, -1)[:n, :k]
    return q, (m / 448.0)[:, 0, :, 0]


def full(q, scale, rows):
    """The 64-bit values of e4m3 numbers with one scale for `rows` x 128 of them."""
    s = scale.double().repeat_interleave(BLOCK, -1)
    if rows > 1:
        s = s.repeat_interleave(rows, -2)
    return q.double() * s[..., :q.shape[-2], :q.shape[-1]]


def bytes_of(q):
    return q.contiguous().view(torch.uint8)


def spread(gen, dev, *shape):
    """Values over many magnitudes, with ties of the e4m3 grid among them."""
    x = torch.randn(shape, generator=gen, device=dev)
    return x * torch.exp2(torch.randint(-20, 12, shape[:-1] + (1,), generator=gen, device=dev).float())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("rows,cols", [(1, 16), (3, 128), (33, 144), (31, 1008), (257, 2560)])
def test_rows_quantised_to_the_byte(cuda_device, rows, cols, dtype):
    from comfyui_b200 import moe_ops as M

    gen = torch.Generator(device=cuda_device).manual_seed(rows + cols)
    x = spread(gen, cuda_device, rows, cols).clamp(-60000, 60000).to(dtype)
    q, scale = M.quantize_blocks_e4m3(x)
    want, want_scale = quantised(x)
    assert torch.equal(bytes_of(q), bytes_of(want))
    assert torch.equal(scale, want_scale.float())


def test_every_ratio_of_two_bf16_numbers(cuda_device):
    """x / m for all 8-bit significands of both: every tie of the grid, and every quotient next to one."""
    from comfyui_b200 import moe_ops as M

    sig = torch.arange(128, 256, device=cuda_device).double()
    x = torch.zeros((128, 16, BLOCK), device=cuda_device, dtype=torch.float64)
    x[:, 0, 0] = 256 * sig                                        # the maximum of a row's first block ...
    x[:, :, :] = torch.where(x == 0, sig[None, None, :] / (2.0 ** torch.arange(16, device=cuda_device))[None, :, None], x)
    x[:, :, 0] = (256 * sig)[:, None]                             # ... and of all others
    x = x.view(128, -1).bfloat16()
    q, scale = M.quantize_blocks_e4m3(x)
    want, want_scale = quantised(x)
    assert torch.equal(bytes_of(q), bytes_of(want)) and torch.equal(scale, want_scale.float())


@pytest.mark.parametrize("top", [1024, 1025, 1365, 1366, 1535, 1792, 1793, 2047], ids=str)
def test_every_significand_of_fp16(cuda_device, top):
    """x / m for all 11-bit significands of x over the powers of two that e4m3 covers, and both signs."""
    from comfyui_b200 import moe_ops as M

    dev = cuda_device
    sig = torch.arange(1024, 2048, device=dev).double()
    x = sig[None, :] / (2.0 ** torch.arange(19, device=dev).double())[:, None] * 4.0
    x = torch.cat([x, -x]).flatten()
    x = torch.nn.functional.pad(x, (0, -x.numel() % (BLOCK - 1))).view(-1, BLOCK - 1)
    x = torch.cat([torch.full((len(x), 1), 8.0 * top, device=dev, dtype=torch.float64), x.clamp(-8.0 * top, 8.0 * top)], 1).half()
    q, scale = M.quantize_blocks_e4m3(x)
    want, want_scale = quantised(x)
    assert torch.equal(bytes_of(q), bytes_of(want)) and torch.equal(scale, want_scale.float())


def test_fp32_rows(cuda_device):
    """fp32 values: the quotient's one rounding may move a value onto a border, by less than 2^-23 of it."""
    from comfyui_b200 import moe_ops as M

    gen = torch.Generator(device=cuda_device).manual_seed(5)
    x = spread(gen, cuda_device, 65, 272)
    q, scale = M.quantize_blocks_e4m3(x)
    _, want_scale = quantised(x)
    torch.testing.assert_close(scale.double(), want_scale, rtol=2.0 ** -24, atol=0)
    got, exact = full(q, scale, 1), x.double()
    # half a step of e4m3 (2^-4 of the value, at least 2^-10 of the scale), and the rounding of the quotient and the scale
    s = want_scale.repeat_interleave(BLOCK, -1)[:, :272]
    assert ((got - exact).abs() <= torch.maximum(2.0 ** -4 * exact.abs(), 2.0 ** -10 * s) * (1 + 2.0 ** -20)).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("shape", [(1, 16), (128, 128), (130, 272), (3, 200, 400)])
def test_weights_quantised_to_the_byte(cuda_device, shape, dtype):
    from comfyui_b200 import moe_ops as M

    gen = torch.Generator(device=cuda_device).manual_seed(sum(shape))
    w = (0.05 * torch.randn(shape, generator=gen, device=cuda_device)).to(dtype)
    q, scale = M.quantize_weight_blocks_e4m3(w)
    for i in range(shape[0] if len(shape) == 3 else 1):
        at = (i,) if len(shape) == 3 else ()
        want, want_scale = quantised_weight(w[at] if at else w)
        assert torch.equal(bytes_of(q[at] if at else q), bytes_of(want))
        assert torch.equal(scale[at] if at else scale, want_scale.float())


def test_blocks_of_zeros_tiny_and_not_finite_values(cuda_device):
    from comfyui_b200 import moe_ops as M

    x = torch.zeros((6, 256), device=cuda_device, dtype=torch.bfloat16)
    x[1, :] = 2.0 ** -120                                   # under the floor: the scale is the floor's, the values round to 0
    x[2, 5], x[2, 6] = float("nan"), 3.0
    x[3, 7], x[3, 8] = float("-inf"), 3.0
    x[4, 130], x[4, 131] = 3.3895313892515355e38, 1.0        # the largest bf16 number
    q, scale = M.quantize_blocks_e4m3(x)
    assert (q[:2].float() == 0).all() and (scale[:2] == 2.0 ** -100 / 448).all()
    assert torch.isnan(scale[2, 0]) and torch.isinf(scale[3, 0]) and torch.isfinite(scale[2:, 1]).all()
    assert torch.isnan(q[2, :128].float()).all() and (q[2, 128:].float() == 0).all()
    assert torch.isnan(q[3, 7].float()) and (q[3, 8:].float() == 0).all()
    assert q[4, 130].float() == 448 and q[4, 131].float() == 0
    gen = torch.Generator(device=cuda_device).manual_seed(1)
    w, ws = M.quantize_weight_blocks_e4m3(torch.randn((48, 256), generator=gen, device=cuda_device))
    y = M.block_linear(x, w, ws)
    assert (y[:2] == 0).all() and torch.isnan(y[2]).all() and not torch.isfinite(y[3]).any() and (y[5] == 0).all()


def product(x, w, ws, bias, dtype, transpose=False):
    """(64-bit product of the quantised operands, bound of its fp32 sums)."""
    q, s = quantised(x)
    a, b = full(q, s.float(), 1), full(w, ws, BLOCK)
    if not transpose:
        b = b.t()
    ref, mag = a @ b, a.abs() @ b.abs()
    if bias is not None:
        ref = ref + bias.double()
        mag = mag + bias.double().abs()
    return ref, mag


def close(got, ref, mag, terms, what):
    bound = HALF_STEP[got.dtype] * ref.abs() + (terms + 3 * blocks(terms)) * 2.0 ** -23 * mag + \
        2.0 ** -24 * (got.dtype == torch.float16)
    err = (got.double() - ref).abs()
    assert torch.isfinite(got.double()).all(), what
    assert (err <= bound).all(), f"{what}: {(err - bound).max().item():.3e} over at {(err > bound).sum().item()} places"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("n,k", [(16, 16), (128, 128), (144, 400), (264, 1040), (2064, 2560)])
@pytest.mark.parametrize("rows", [1, 2, 3, 8, 9, 16, 17, 33, 128, 300])
def test_dense(cuda_device, rows, n, k, dtype):
    from comfyui_b200 import moe_ops as M

    gen = torch.Generator(device=cuda_device).manual_seed(rows + n + k)
    x = torch.randn((rows, k), generator=gen, device=cuda_device).to(dtype)
    w, ws = M.quantize_weight_blocks_e4m3(0.05 * torch.randn((n, k), generator=gen, device=cuda_device))
    ws *= torch.rand(ws.shape, generator=gen, device=cuda_device) + 0.5      # blocks that differ, for a mixed-up scale to show
    bias = torch.randn((n,), generator=gen, device=cuda_device).to(dtype)
    for b in (None, bias):
        close(M.block_linear(x, w, ws, b), *product(x, w, ws, b, dtype), k, f"bias {b is not None}")
    if n % 16 == 0:
        dy = torch.randn((rows, n), generator=gen, device=cuda_device).to(dtype)
        close(M.block_linear_dgrad(dy, w, ws), *product(dy, w, ws, None, dtype, True), n, "dx")
    torch.cuda.synchronize()
    M.check_all_status()


@pytest.mark.parametrize("counts", [[1], [0, 2], [2, 0, 1], [0, 8], [9, 0, 5], [16], [3, 0, 130], [127, 128, 129, 1], [700, 0, 33, 515], [1] * 40],
                         ids=lambda c: "-".join(map(str, c))[:20])
@pytest.mark.parametrize("gap", [0, 1, 7])
@pytest.mark.parametrize("n,k", [(272, 400), (528, 1040)])
def test_by_expert(cuda_device, counts, n, k, gap):
    from comfyui_b200 import moe_ops as M

    dev = cuda_device
    gen = torch.Generator(device=dev).manual_seed(len(counts) + n)
    rows, g = sum(counts) + 2 * gap, len(counts)
    x = torch.randn((rows, k), generator=gen, device=dev).bfloat16()
    dy = torch.randn((rows, n), generator=gen, device=dev).bfloat16()
    w, ws = M.quantize_weight_blocks_e4m3(0.05 * torch.randn((g, n, k), generator=gen, device=dev))
    ws *= torch.rand(ws.shape, generator=gen, device=dev) + 0.5
    ends = [gap + sum(counts[:i]) for i in range(g + 1)]
    offsets = torch.tensor(ends, dtype=torch.int32, device=dev)
    y, dx = M.grouped_block_linear(x, w, ws, offsets), M.grouped_block_linear_dgrad(dy, w, ws, offsets)
    for i, (lo, hi) in enumerate(zip(ends[:-1], ends[1:])):
        close(y[lo:hi], *product(x[lo:hi], w[i], ws[i], None, x.dtype), k, f"y of group {i}")
        close(dx[lo:hi], *product(dy[lo:hi], w[i], ws[i], None, x.dtype, True), n, f"dx of group {i}")
    for t in (y, dx):
        assert (t[:gap] == 0).all() and (t[rows - gap:] == 0).all()
    out = torch.full_like(y, 7.0)
    M.grouped_block_linear(x, w, ws, offsets, out=out)
    assert torch.equal(out[gap:rows - gap], y[gap:rows - gap]) and (out[:gap] == 7).all() and (out[rows - gap:] == 7).all()
    # fewer rows than the offsets leave room for, with values that are not finite in what is left out
    most = torch.tensor([c // 2 for c in counts], dtype=torch.int32, device=dev)
    used = torch.zeros(rows, dtype=torch.bool, device=dev)
    for c, lo in zip(counts, ends):
        used[lo:lo + c // 2] = True
    x[~used] = float("nan")
    y2 = M.grouped_block_linear(x, w, ws, offsets, most)
    assert torch.equal(y2[used], y[used]) and (y2[~used] == 0).all()
    M.check_all_status()


def test_strides_and_shapes(cuda_device):
    from comfyui_b200 import moe_ops as M

    dev, n, k = cuda_device, 144, 272
    gen = torch.Generator(device=dev).manual_seed(3)
    x = torch.randn((2, 5, 7, k), generator=gen, device=dev).half()
    w, ws = M.quantize_weight_blocks_e4m3(torch.randn((n, k), generator=gen, device=dev))
    y = M.block_linear(x, w, ws)
    assert y.shape == (2, 5, 7, n) and torch.equal(y.view(-1, n), M.block_linear(x.view(-1, k), w, ws))
    wide = torch.full((70, k + 24), float("nan"), device=dev, dtype=torch.float16)
    wide[:, 8:8 + k] = x.view(-1, k)
    ww = torch.zeros((n, k + 32), device=dev, dtype=torch.uint8).view(torch.float8_e4m3fn)
    ww[:, 16:16 + k] = w
    out = torch.zeros((70, n + 16), device=dev, dtype=torch.float16)
    M.block_linear(wide[:, 8:8 + k], ww[:, 16:16 + k], ws, out=out[:, 8:8 + n])
    assert torch.equal(out[:, 8:8 + n], y.view(-1, n)) and (out[:, :8] == 0).all() and (out[:, 8 + n:] == 0).all()
    assert torch.equal(M.block_linear(x.transpose(1, 2), w, ws), y.transpose(1, 2))
    assert M.block_linear(x[:0], w, ws).shape == (0, 5, 7, n)
    assert torch.equal(M.block_linear(x[0, 0, 0], w, ws), M.block_linear(x[0, 0, :1], w, ws)[0])
    into = torch.empty_like(y)
    assert M.block_linear(x, w, ws, out=into) is into and torch.equal(into, y)


def test_gradients_through_autograd(cuda_device):
    from comfyui_b200 import moe_ops as M

    dev, n, k = cuda_device, 144, 272
    gen = torch.Generator(device=dev).manual_seed(3)
    x = torch.randn((33, k), generator=gen, device=dev).bfloat16()
    dy = torch.randn((33, n), generator=gen, device=dev).bfloat16()
    w, ws = M.quantize_weight_blocks_e4m3(torch.randn((3, n, k), generator=gen, device=dev))
    bias = torch.randn((n,), generator=gen, device=dev).bfloat16().requires_grad_(True)
    offsets = torch.tensor([1, 10, 10, 30], dtype=torch.int32, device=dev)
    want = M.block_linear_dgrad(dy, w[0], ws[0])
    want_g = M.grouped_block_linear_dgrad(dy, w, ws, offsets)
    x.requires_grad_(True)
    y = M.block_linear(x.view(3, 11, k), w[0], ws[0], bias)
    dx, db = torch.autograd.grad(y, (x, bias), dy.view(3, 11, n), retain_graph=True)
    assert torch.equal(dx, want)
    close(db[None], dy.double().sum(0)[None], dy.double().abs().sum(0)[None], 33, "bias")
    dx, = torch.autograd.grad(y.sum(), x)                                    # a gradient expanded from one number
    assert torch.equal(dx, M.block_linear_dgrad(torch.ones_like(dy), w[0], ws[0]))
    dx, = torch.autograd.grad(M.grouped_block_linear(x, w, ws, offsets), x, dy)
    assert torch.equal(dx, want_g) and (dx[:1] == 0).all() and (dx[30:] == 0).all()
    for call in (lambda: M.block_linear(x, w[0], ws[0]), lambda: M.grouped_block_linear(x, w, ws, offsets)):
        with pytest.raises(RuntimeError, match="differentiable once"):
            torch.autograd.grad(call(), x, dy, create_graph=True)
    # the gradient is that of the product with the quantised operands: <dx, u> = <q(dy) w, u> for any direction u
    u = torch.randn((33, k), generator=gen, device=dev, dtype=torch.float64)
    q, s = quantised(dy)
    along = ((u @ full(w[0], ws[0], BLOCK).t()) * full(q, s.float(), 1)).sum().item()
    assert abs((want.double() * u).sum().item() - along) <= 1.01 * 2.0 ** -8 * (want.double() * u).abs().sum().item()


def test_graph_replay_and_streams(cuda_device):
    from comfyui_b200 import moe_ops as M

    dev, n, k = cuda_device, 272, 656
    gen = torch.Generator(device=dev).manual_seed(3)
    x = torch.randn((200, k), generator=gen, device=dev).bfloat16()
    w, ws = M.quantize_weight_blocks_e4m3(torch.randn((3, n, k), generator=gen, device=dev))
    offsets = torch.tensor([0, 70, 71, 200], dtype=torch.int32, device=dev)
    call = lambda: (M.block_linear(x, w[1], ws[1]), M.grouped_block_linear(x, w, ws, offsets))        # noqa: E731
    want = call()
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for gr in graphs:
        with torch.cuda.graph(gr):
            outs.append(call())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for gr, st in zip(graphs, (torch.cuda.current_stream(), side)):
        with torch.cuda.stream(st):
            gr.replay()
    with torch.cuda.stream(side):
        outs.append(call())
    torch.cuda.synchronize()
    for o in outs:
        assert all(torch.equal(a, b) for a, b in zip(o, want))


def test_the_products_of_an_expert_layer_together(cuda_device):
    """Quantise, multiply by expert, SwiGLU, multiply back: against the same steps in 64 bits on the same routing."""
    from comfyui_b200 import moe_ops as M

    dev, e, dim, hidden, tokens = cuda_device, 4, 512, 768, 301
    gen = torch.Generator(device=dev).manual_seed(11)
    x = torch.randn((tokens, dim), generator=gen, device=dev).bfloat16()
    gate = torch.randn((e, dim), generator=gen, device=dev).bfloat16()
    w13, s13 = M.quantize_weight_blocks_e4m3(0.05 * torch.randn((e, 2 * hidden, dim), generator=gen, device=dev))
    w2, s2 = M.quantize_weight_blocks_e4m3(0.05 * torch.randn((e, dim, hidden), generator=gen, device=dev))
    idx, weight, block_counts, _, _ = M.gate_topk(x, gate)
    x_perm, row_map, counts, offsets = M.plan_permute(x, idx, block_counts, e)
    h = M.grouped_block_linear(x_perm, w13, s13, offsets, counts)
    h = torch.nn.functional.silu(h[:, :hidden]) * h[:, hidden:]
    y = M.combine(M.grouped_block_linear(h, w2, s2, offsets, counts), row_map, weight, None)
    # rounding points as above (bf16 after each product, silu, the product of the two, and in the combine)
    want = torch.zeros((tokens, dim), dtype=torch.float64, device=dev)
    for i in range(e):
        at, slot = (idx == i).nonzero(as_tuple=True)
        h13 = product(x[at], w13[i], s13[i], None, x.dtype)[0].bfloat16()
        hi = torch.nn.functional.silu(h13[:, :hidden]) * h13[:, hidden:]
        out = product(hi, w2[i], s2[i], None, x.dtype)[0].bfloat16().double()
        want.index_add_(0, at, out * weight[at, slot].bfloat16().double()[:, None])
    err = (y.double() - want).norm() / want.norm()
    # a rounding of h to bf16 that falls the other way may move its e4m3 value by one step (2^-3 of it): rare, so the
    # bound is that of the roundings that always happen: two products, the weighting and the sum, 2^-8 each
    assert err < 4 * 2.0 ** -8, err
    assert torch.isfinite(y).all()


def test_refusals(cuda_device):
    from comfyui_b200 import moe_ops as M

    dev = cuda_device
    x = torch.zeros((5, 64), device=dev, dtype=torch.bfloat16)
    w = torch.zeros((48, 64), device=dev, dtype=torch.uint8).view(torch.float8_e4m3fn)
    ws = torch.ones((1, 1), device=dev)
    off = torch.zeros(2, dtype=torch.int32, device=dev)
    for call, match in [
        (lambda: M.block_linear(x[:, :48], w, ws), "that fit"),
        (lambda: M.block_linear(x.float(), w, ws), "bf16 or fp16"),
        (lambda: M.block_linear(x, w.float(), ws), "e4m3"),
        (lambda: M.block_linear(x, w, ws.half()), "scales must be"),
        (lambda: M.block_linear(x, w, torch.ones((1, 2), device=dev)), "scales must be"),
        (lambda: M.block_linear(x[:, :56], w[:, :56], ws), "multiple of 16"),
        (lambda: M.block_linear(x, w[:44], ws), "of 8"),
        (lambda: M.block_linear(x, w, ws, torch.zeros(48, device=dev)), "bias must be"),
        (lambda: M.block_linear(x.cpu(), w, ws), "CUDA"),
        (lambda: M.block_linear(x, w, ws, out=torch.zeros((5, 40), device=dev, dtype=x.dtype)), "out must be"),
        (lambda: M.block_linear(x.clone().requires_grad_(True), w[:40], ws), "multiple of 16 for a gradient"),
        (lambda: M.block_linear_dgrad(torch.zeros((5, 40), device=dev, dtype=x.dtype), w[:40], ws), "multiple of 16"),
        (lambda: M.grouped_block_linear(x, w, ws, off), "that fit"),
        (lambda: M.grouped_block_linear(x, w[None], ws, off), "scales must be"),
        (lambda: M.grouped_block_linear(x, w[None], ws[None], off.long()), "int32"),
        (lambda: M.quantize_blocks_e4m3(x[:, :24]), "multiple of 16"),
        (lambda: M.quantize_blocks_e4m3(x.double()), "bf16, fp16 or fp32"),
        (lambda: M.quantize_weight_blocks_e4m3(x[0]), "w must be"),
    ]:
        with pytest.raises(ValueError, match=match):
            call()
    with pytest.raises(ValueError, match="frozen"):
        M.block_linear(x, w, ws.clone().requires_grad_(True))


def test_linear_of_the_namespace(cuda_device):
    """ops.block_scaled_fp8_ops: a Linear on the kernel, beside its composition; bias and input gradients; fallbacks."""
    from comfyui_b200 import moe_ops as M
    from comfyui_b200 import ops

    dev, n, k = cuda_device, 144, 272
    gen = torch.Generator(device=dev).manual_seed(3)
    lin = ops.block_scaled_fp8_ops().Linear(k, n, device=dev, dtype=torch.bfloat16)
    w, ws = M.quantize_weight_blocks_e4m3(torch.randn((n, k), generator=gen, device=dev))
    bias = torch.randn((n,), generator=gen, device=dev).bfloat16()
    lin.load_state_dict({"weight": w, "scale_weight": ws, "bias": bias}, strict=True)
    x = torch.randn((2, 9, k), generator=gen, device=dev).bfloat16().requires_grad_(True)
    y = lin(x)
    assert y.shape == (2, 9, n) and torch.equal(y, M.block_linear(x.detach(), w, ws, bias))
    dy = torch.randn(y.shape, generator=gen, device=dev).bfloat16()
    dx, db = torch.autograd.grad(y, (x, lin.bias), dy)
    assert torch.equal(dx.view(-1, k), M.block_linear_dgrad(dy.view(-1, n), w, ws))
    close(db[None], dy.double().sum((0, 1))[None], dy.double().abs().sum((0, 1))[None], 18, "bias")
    wide = torch.randn((2, 9, k + 3), generator=gen, device=dev).bfloat16()[..., 3:]          # rows that no kernel reads
    with torch.no_grad():
        assert torch.equal(lin(wide), lin(wide.contiguous()))
        f32 = lin(x.float())                                                                   # the composition
        assert f32.dtype == torch.float32
        torch.testing.assert_close(f32, x.float() @ full(w, ws, BLOCK).float().t() + bias.float(), rtol=1e-4, atol=1e-3)
        lin.weight_function = [lambda t: 0 * t]
        assert torch.equal(lin(x), bias.expand(2, 9, n))


def test_a_layer_of_the_namespace(cuda_device):
    """The mixture-of-experts module built with block-scaled Linears: finite, and near the layer with the weights scaled back."""
    from comfyui_b200 import moe_ops as M
    from comfyui_b200 import ops
    from comfyui_b200.ldm.hidream.model import MOEFeedForwardSwiGLU

    dev, dim, hidden = cuda_device, 512, 1024
    gen = torch.Generator(device=dev).manual_seed(5)
    layer = MOEFeedForwardSwiGLU(dim, hidden, 4, 2, dtype=torch.bfloat16, device=dev, operations=ops.block_scaled_fp8_ops())
    plain = MOEFeedForwardSwiGLU(dim, hidden, 4, 2, dtype=torch.bfloat16, device=dev, operations=ops.disable_weight_init)
    state, back = {}, {}
    for name, p in layer.state_dict().items():
        if name.endswith("scale_weight"):
            continue
        t = 0.05 * torch.randn(p.shape, generator=gen, device=dev)
        if p.dtype == torch.float8_e4m3fn:
            w, s = M.quantize_weight_blocks_e4m3(t)
            state[name], state[name.replace("weight", "scale_weight")] = w, s
            back[name] = full(w, s, BLOCK).bfloat16()
        else:
            state[name] = back[name] = t.bfloat16()
    layer.load_state_dict(state, strict=True)
    plain.load_state_dict(back, strict=True)
    x = torch.randn((2, 150, dim), generator=gen, device=dev).bfloat16()
    with torch.inference_mode():
        y, ref = layer(x), plain(x)
    # what differs is the rounding of each product's input to e4m3: 2^-4 of a value at most, a third of that in the mean
    # square (the error is spread evenly over a step, half a step at most), over two products in a row: 2^-4 / 3 x sqrt(2) < 0.03,
    # and as much again for the share that the non-linear product of the first two adds
    err = (y.double() - ref.double()).norm() / ref.double().norm()
    assert torch.isfinite(y).all() and err < 0.06, err


def test_registered_operators(cuda_device):
    from comfyui_b200 import moe_ops as M
    from comfyui_b200 import torch_ops  # noqa: F401

    dev, n, k = cuda_device, 144, 272
    gen = torch.Generator(device=dev).manual_seed(3)
    x = torch.randn((50, k), generator=gen, device=dev).bfloat16()
    w = torch.randn((2, n, k), generator=gen, device=dev).bfloat16()
    wq, ws = M.quantize_weight_blocks_e4m3(w)
    off = torch.tensor([0, 20, 50], dtype=torch.int32, device=dev)
    ops = torch.ops.comfyui_b200
    assert torch.equal(ops.grouped_matmul(x, w, off), M.grouped_matmul(x, w, off))
    assert torch.equal(ops.block_linear(x, wq[0], ws[0]), M.block_linear(x, wq[0], ws[0]))
    assert torch.equal(ops.grouped_block_linear(x, wq, ws, off), M.grouped_block_linear(x, wq, ws, off))
    x.requires_grad_(True)
    w.requires_grad_(True)
    got = torch.autograd.grad(ops.grouped_matmul(x, w, off).sum(), (x, w))
    want = torch.autograd.grad(M.grouped_matmul(x, w, off).sum(), (x, w))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("counts", [[17], [130], [0, 40, 100], [128, 1, 0, 60]], ids=str)
@pytest.mark.parametrize("n,k", [(144, 2688), (272, 4112), (16, 8192), (2064, 4112)])
def test_few_tiles_and_a_long_contraction(cuda_device, counts, n, k, dtype):
    from comfyui_b200 import moe_ops as M

    dev = cuda_device
    gen = torch.Generator(device=dev).manual_seed(n + k)
    rows, g = sum(counts) + 5, len(counts)
    x = torch.randn((rows, k), generator=gen, device=dev).to(dtype)
    w, ws = M.quantize_weight_blocks_e4m3(0.05 * torch.randn((g, n, k), generator=gen, device=dev))
    ws *= torch.rand(ws.shape, generator=gen, device=dev) + 0.5
    wt, wts = w.transpose(1, 2).contiguous(), ws.transpose(1, 2).contiguous()
    ends = [5 + sum(counts[:i]) for i in range(g + 1)]
    offsets = torch.tensor(ends, dtype=torch.int32, device=dev)
    bias = torch.randn((n,), generator=gen, device=dev).to(dtype)
    y, dx = M.grouped_block_linear(x, w, ws, offsets), M.grouped_block_linear_dgrad(x, wt, wts, offsets)
    for i, (lo, hi) in enumerate(zip(ends[:-1], ends[1:])):
        want = product(x[lo:hi], w[i], ws[i], None, dtype)
        close(y[lo:hi], *want, k, f"y of group {i}")
        close(dx[lo:hi], *want, k, f"dx of group {i}")
    assert (y[:5] == 0).all() and (dx[:5] == 0).all()
    close(M.block_linear(x, w[0], ws[0], bias), *product(x, w[0], ws[0], bias, dtype), k, "with a bias")
    again = [M.grouped_block_linear(x, w, ws, offsets) for _ in range(3)]
    assert all(torch.equal(a, y) for a in again)
    M.check_all_status()


def test_few_tiles_with_strides_padding_and_given_results(cuda_device):
    from comfyui_b200 import moe_ops as M

    dev, n, k = cuda_device, 272, 4112
    gen = torch.Generator(device=dev).manual_seed(9)
    offsets = torch.tensor([3, 60, 60, 110], dtype=torch.int32, device=dev)
    counts = torch.tensor([50, 1, 41], dtype=torch.int32, device=dev)
    x = torch.randn((120, k + 24), generator=gen, device=dev).bfloat16()[:, 8:8 + k]
    keep = torch.zeros(120, dtype=torch.bool, device=dev)
    for lo, hi in ((3, 53), (60, 101)):
        keep[lo:hi] = True
    x[~keep] = float("nan")
    w, ws = M.quantize_weight_blocks_e4m3(0.05 * torch.randn((3, n, k), generator=gen, device=dev))
    y = torch.full((120, n + 8), 7.0, dtype=torch.bfloat16, device=dev)
    M.grouped_block_linear(x, w, ws, offsets, counts, out=y[:, :n])
    for g, lo, hi in ((0, 3, 53), (2, 60, 101)):
        close(y[lo:hi, :n], *product(x[lo:hi], w[g], ws[g], None, x.dtype), k, f"y of group {g}")
    assert (y[~keep] == 7).all() and (y[:, n:] == 7).all()
    z = M.grouped_block_linear(x, w, ws, offsets, counts)
    assert torch.equal(z[keep], y[keep, :n]) and (z[~keep] == 0).all()
    M.check_all_status()
