"""Products grouped by expert and their gradients against 64-bit products, group by group.  Needs a B200.

Tolerance of an element: one rounding of the result (half a step of its type) plus the rounding of the fp32 sums, at most
terms x 2^-23 of the sum of the products' magnitudes (one fp32 rounding, or truncation, per term)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def make(dev, counts, k, n, dtype, seed=0, gap=0, scale=0.05):
    """Rows of len(counts) groups behind `gap` rows of nobody (and as many after them), weights, offsets."""
    gen = torch.Generator(device=dev).manual_seed(seed)
    rows = sum(counts) + 2 * gap
    x = torch.randn((rows, k), generator=gen, device=dev).to(dtype)
    w = (scale * torch.randn((len(counts), n, k), generator=gen, device=dev)).to(dtype)
    dy = torch.randn((rows, n), generator=gen, device=dev).to(dtype)
    ends = torch.tensor([gap] + [gap + sum(counts[:i + 1]) for i in range(len(counts))], dtype=torch.int32)
    return x, w, dy, ends.to(dev)


def by_group(x, w, ranges, rows, cols, product):
    """(64-bit result, bound of its fp32 sums) with zeros in the rows of no group."""
    ref = torch.zeros((rows, cols), dtype=torch.float64, device=x.device)
    mag = torch.zeros_like(ref)
    for g, (lo, hi) in enumerate(ranges):
        ref[lo:hi] = product(x[lo:hi].double(), w[g].double())
        mag[lo:hi] = product(x[lo:hi].double().abs(), w[g].double().abs())
    return ref, mag


def close(got, ref, mag, terms, what):
    bound = HALF_STEP[got.dtype] * ref.abs() + (terms * 2.0 ** -23) * mag + 2.0 ** -24 * (got.dtype == torch.float16)
    err = (got.double() - ref).abs()
    assert torch.isfinite(got.double()).all(), what
    assert (err <= bound).all(), f"{what}: {(err - bound).max().item():.3e} over at {(err > bound).sum().item()} places"


def check_all(dev, counts, k, n, dtype, seed=0, gap=0):
    from comfyui_b200 import moe_ops as M

    x, w, dy, offsets = make(dev, counts, k, n, dtype, seed, gap)
    ends = offsets.tolist()
    ranges = list(zip(ends[:-1], ends[1:]))
    y = M.grouped_matmul(x, w, offsets)
    close(y, *by_group(x, w, ranges, len(x), n, lambda a, b: a @ b.t()), k, "y")
    dx = M.grouped_matmul_dgrad(dy, w, offsets)
    close(dx, *by_group(dy, w, ranges, len(x), k, lambda a, b: a @ b), n, "dx")
    for out_dtype in (dtype, torch.float32):
        dw = M.grouped_matmul_wgrad(dy, x, offsets, out_dtype=out_dtype)
        assert dw.dtype == out_dtype and dw.shape == w.shape
        for g, (lo, hi) in enumerate(ranges):
            a, b = dy[lo:hi].double(), x[lo:hi].double()
            close(dw[g], a.t() @ b, a.abs().t() @ b.abs(), max(hi - lo, 1), f"dw[{g}]")
    torch.cuda.synchronize()
    M.check_all_status()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("k,n", [(8, 8), (64, 256), (72, 40), (200, 520), (1000, 1032)])
@pytest.mark.parametrize("counts", [[1], [0, 1, 0], [3, 0, 130], [127, 128, 129, 1], [64, 65, 63, 0]],
                         ids=lambda c: "-".join(map(str, c)))
def test_sizes(cuda_device, counts, k, n, dtype):
    check_all(cuda_device, counts, k, n, dtype)


@pytest.mark.parametrize("counts", [[700, 0, 1333, 15], [2500]], ids=["four", "one"])
def test_many_tiles(cuda_device, counts):
    check_all(cuda_device, counts, 2048, 2056, torch.bfloat16)


@pytest.mark.parametrize("groups,each,k,n", [(300, 3, 64, 72), (768, 1, 64, 72), (160, 90, 264, 264), (40, 300, 520, 776)])
def test_many_groups(cuda_device, groups, each, k, n):
    counts = [(g * 7 + 3) % (2 * each + 1) for g in range(groups)]
    check_all(cuda_device, counts, k, n, torch.bfloat16)


def test_rows_of_no_group_are_zero(cuda_device):
    check_all(cuda_device, [5, 0, 200], 64, 136, torch.bfloat16, gap=37)


def test_rows_of_no_group_stay_in_a_given_result(cuda_device):
    from comfyui_b200 import moe_ops as M

    x, w, dy, offsets = make(cuda_device, [5, 0, 200], 64, 136, torch.bfloat16, gap=37)
    out = torch.full((len(x), 136), 7.0, dtype=torch.bfloat16, device=cuda_device)
    assert M.grouped_matmul(x, w, offsets, out=out) is out
    ref = M.grouped_matmul(x, w, offsets)
    assert torch.equal(out[37:-37], ref[37:-37])
    assert (out[:37] == 7).all() and (out[-37:] == 7).all()
    dx = torch.full((len(x), 64), 7.0, dtype=torch.bfloat16, device=cuda_device)
    M.grouped_matmul_dgrad(dy, w, offsets, out=dx)
    assert (dx[:37] == 7).all() and (dx[-37:] == 7).all()


def test_counts_leave_padding_out(cuda_device):
    """Groups that begin on multiples of 128 with fewer rows than fit, as the routing plan lays them out."""
    from comfyui_b200 import moe_ops as M

    dev, k, n = cuda_device, 72, 136
    x, w, dy, _ = make(dev, [128, 256, 128], k, n, torch.bfloat16)
    offsets = torch.tensor([0, 128, 384, 512], dtype=torch.int32, device=dev)
    counts = torch.tensor([100, 129, 0], dtype=torch.int32, device=dev)
    ranges = [(0, 100), (128, 257), (384, 384)]
    used = torch.zeros(len(x), dtype=torch.bool, device=dev)
    for lo, hi in ranges:
        used[lo:hi] = True
    x[~used] = float("nan")                       # what stands in the padding must not be read into any result
    dy[~used] = float("inf")
    y = M.grouped_matmul(x, w, offsets, counts)
    close(y, *by_group(x, w, ranges, len(x), n, lambda a, b: a @ b.t()), k, "y")
    assert (y[~used] == 0).all()
    dx = M.grouped_matmul_dgrad(dy, w, offsets, counts)
    close(dx, *by_group(dy, w, ranges, len(x), k, lambda a, b: a @ b), n, "dx")
    dw = M.grouped_matmul_wgrad(dy, x, offsets, counts)
    for g, (lo, hi) in enumerate(ranges):
        a, b = dy[lo:hi].double(), x[lo:hi].double()
        close(dw[g], a.t() @ b, a.abs().t() @ b.abs(), max(hi - lo, 1), f"dw[{g}]")


@pytest.mark.parametrize("offsets,ranges", [
    ([0, 50, 20, 90], [(0, 50), (50, 50), (50, 90)]),             # a group that ends before it begins is empty
    ([0, 1000, 20, 90], [(0, 200), (200, 200), (200, 200)]),      # rows behind the buffer do not exist
    ([-5, 10, 10, 2000], [(0, 10), (10, 10), (10, 200)]),
])
def test_offsets_out_of_order_or_range(cuda_device, offsets, ranges):
    from comfyui_b200 import moe_ops as M

    x, w, dy, _ = make(cuda_device, [200, 0, 0], 64, 72, torch.bfloat16)
    off = torch.tensor(offsets, dtype=torch.int32, device=cuda_device)
    y = M.grouped_matmul(x, w, off)
    close(y, *by_group(x, w, ranges, 200, 72, lambda a, b: a @ b.t()), 64, "y")
    dw = M.grouped_matmul_wgrad(dy, x, off)
    for g, (lo, hi) in enumerate(ranges):
        a, b = dy[lo:hi].double(), x[lo:hi].double()
        close(dw[g], a.t() @ b, a.abs().t() @ b.abs(), max(hi - lo, 1), f"dw[{g}]")


def test_strided_operands(cuda_device):
    from comfyui_b200 import moe_ops as M

    dev, k, n = cuda_device, 72, 136
    x, w, dy, offsets = make(dev, [70, 131], k, n, torch.bfloat16)
    wide = lambda t, extra: torch.nn.functional.pad(t, (8, extra), value=float("nan"))[..., 8:-extra]   # noqa: E731
    xs, dys = wide(x, 16), wide(dy, 24)
    ws = torch.nn.functional.pad(w, (8, 8, 0, 3), value=float("nan"))[:, :n, 8:-8]
    assert not xs.is_contiguous() and not ws.is_contiguous()
    out = torch.zeros((len(x), n + 16), dtype=x.dtype, device=dev)
    M.grouped_matmul(xs, ws, offsets, out=out[:, 8:-8])
    assert torch.equal(out[:, 8:-8], M.grouped_matmul(x, w, offsets))
    assert (out[:, :8] == 0).all() and (out[:, -8:] == 0).all()
    assert torch.equal(M.grouped_matmul_dgrad(dys, ws, offsets), M.grouped_matmul_dgrad(dy, w, offsets))
    assert torch.equal(M.grouped_matmul_wgrad(dys, xs, offsets), M.grouped_matmul_wgrad(dy, x, offsets))
    dw = torch.zeros((2, n + 1, k + 8), dtype=torch.float32, device=dev)
    M.grouped_matmul_wgrad(dy, x, offsets, out=dw[:, :n, :k])
    assert torch.equal(dw[:, :n, :k], M.grouped_matmul_wgrad(dy, x, offsets, out_dtype=torch.float32))
    assert (dw[:, n] == 0).all() and (dw[:, :, k:] == 0).all()


def test_no_rows_and_no_groups(cuda_device):
    from comfyui_b200 import moe_ops as M

    dev = cuda_device
    x, w, dy, _ = make(dev, [0, 0], 64, 72, torch.bfloat16)
    offsets = torch.zeros(3, dtype=torch.int32, device=dev)
    assert M.grouped_matmul(x, w, offsets).shape == (0, 72)
    assert M.grouped_matmul_dgrad(dy, w, offsets).shape == (0, 64)
    assert (M.grouped_matmul_wgrad(dy, x, offsets) == 0).all()
    x = torch.ones((3, 64), dtype=torch.bfloat16, device=dev)
    assert (M.grouped_matmul(x, w[:0], offsets[:1]) == 0).all()
    assert (M.grouped_matmul(x, w, offsets) == 0).all()


def test_all_rows_of_no_group(cuda_device):
    """Every tile list empty: results are zeros, a given one is not touched, the weights' gradient is zero."""
    from comfyui_b200 import moe_ops as M

    x, w, dy, _ = make(cuda_device, [300, 0], 264, 136, torch.bfloat16)
    x[:], dy[:] = float("nan"), float("nan")
    for offsets, counts in (([0, 0, 0], None), ([300, 300, 300], None), ([7, 100, 300], [0, -3])):
        off = torch.tensor(offsets, dtype=torch.int32, device=cuda_device)
        cnt = None if counts is None else torch.tensor(counts, dtype=torch.int32, device=cuda_device)
        assert (M.grouped_matmul(x, w, off, cnt) == 0).all() and (M.grouped_matmul_dgrad(dy, w, off, cnt) == 0).all()
        assert (M.grouped_matmul_wgrad(dy, x, off, cnt) == 0).all()
        out = torch.full_like(dy, 7.0)
        assert (M.grouped_matmul(x, w, off, cnt, out=out) == 7).all()


def test_values_that_are_not_finite_stay_in_their_rows(cuda_device):
    from comfyui_b200 import moe_ops as M

    x, w, dy, offsets = make(cuda_device, [70, 70], 136, 72, torch.bfloat16)
    clean = M.grouped_matmul(x, w, offsets)
    x[3, 5], x[71, 0] = float("nan"), float("inf")
    y = M.grouped_matmul(x, w, offsets)
    rest = [r for r in range(140) if r not in (3, 71)]
    assert torch.isnan(y[3]).all() and not torch.isfinite(y[71]).any()
    assert torch.equal(y[rest], clean[rest])
    dw = M.grouped_matmul_wgrad(dy, x, offsets)
    assert torch.isnan(dw[0, :, 5]).all() and torch.isfinite(dw[0, :, :5]).all()
    assert torch.isfinite(dw[1, :, 1:]).all()


def test_gradients_through_autograd(cuda_device):
    from comfyui_b200 import moe_ops as M

    dev = cuda_device
    x, w, dy, offsets = make(dev, [70, 0, 131], 72, 136, torch.bfloat16, gap=5)
    want_dx, want_dw = M.grouped_matmul_dgrad(dy, w, offsets), M.grouped_matmul_wgrad(dy, x, offsets)
    x.requires_grad_(True)
    w.requires_grad_(True)
    y = M.grouped_matmul(x, w, offsets)
    dx, dw = torch.autograd.grad(y, (x, w), dy, retain_graph=True)
    assert torch.equal(dx, want_dx) and torch.equal(dw, want_dw) and (dw[1] == 0).all()
    # only one of the two; a gradient that is expanded from one number, and one that is transposed
    assert torch.equal(torch.autograd.grad(y, x, dy, retain_graph=True)[0], want_dx)
    ones = torch.ones_like(dy)
    got, = torch.autograd.grad(y.sum(), w, retain_graph=True)
    assert torch.equal(got, M.grouped_matmul_wgrad(ones, x.detach(), offsets))
    got, = torch.autograd.grad(y, x, dy.t().contiguous().t())
    assert torch.equal(got, want_dx)
    with torch.no_grad():
        assert not M.grouped_matmul(x, w, offsets).requires_grad
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(M.grouped_matmul(x, w, offsets), x, dy, create_graph=True)
    with pytest.raises(ValueError, match="out cannot be given"):
        M.grouped_matmul(x, w, offsets, out=torch.empty_like(dy))


def test_gradient_against_differences(cuda_device):
    """d/dt of <dy, y(x + t u, w + t v)> = <dx, u> + <dw, v>; y is bilinear, so the central difference in 64 bits is exact."""
    from comfyui_b200 import moe_ops as M

    x, w, dy, offsets = make(cuda_device, [40, 25], 64, 48, torch.float16)
    x.requires_grad_(True)
    w.requires_grad_(True)
    dx, dw = torch.autograd.grad(M.grouped_matmul(x, w, offsets), (x, w), dy)
    gen = torch.Generator(device=cuda_device).manual_seed(9)
    u = torch.randn(x.shape, generator=gen, device=cuda_device, dtype=torch.float64)
    v = torch.randn(w.shape, generator=gen, device=cuda_device, dtype=torch.float64)

    def along(t):
        a, b = x.detach().double() + t * u, w.detach().double() + t * v
        y = torch.cat([a[:40] @ b[0].t(), a[40:] @ b[1].t()])
        return (y * dy.double()).sum()

    want = (along(0.5) - along(-0.5)).item()
    got = ((dx.double() * u).sum() + (dw.double() * v).sum()).item()
    bound = 2.0 ** -11 * ((dx.double() * u).abs().sum() + (dw.double() * v).abs().sum()).item()
    assert abs(got - want) <= 1.01 * bound


def test_runs_are_alike_and_replay_from_a_graph(cuda_device):
    """The same bits every time, on another stream, from a graph replayed on new offsets, and two graphs at once."""
    from comfyui_b200 import moe_ops as M

    dev = cuda_device
    x, w, dy, offsets = make(dev, [300, 41, 0, 171], 264, 136, torch.bfloat16)
    call = lambda: (M.grouped_matmul(x, w, offsets), M.grouped_matmul_dgrad(dy, w, offsets),         # noqa: E731
                    M.grouped_matmul_wgrad(dy, x, offsets))
    want = call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    outs = []
    for gr in graphs:
        with torch.cuda.graph(gr):
            outs.append(call())
    other = torch.tensor([0, 12, 200, 400, 512], dtype=torch.int32, device=dev)
    first = offsets.clone()
    offsets.copy_(other)
    want2 = call()
    graphs[0].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs[0], want2))
    offsets.copy_(first)
    side.wait_stream(torch.cuda.current_stream())
    for gr, st in zip(graphs, (torch.cuda.current_stream(), side)):
        with torch.cuda.stream(st):
            gr.replay()
    torch.cuda.synchronize()
    for o in outs:
        assert all(torch.equal(a, b) for a, b in zip(o, want))


def test_backward_replays_from_a_graph(cuda_device):
    """Captured while no eager graph of the same leaves lives: PyTorch binds a leaf's accumulation to the stream of the first
    graph that is alive, and refuses to capture it on another one, whatever the operators in between."""
    from comfyui_b200 import moe_ops as M

    x, w, dy, offsets = make(cuda_device, [30, 41], 64, 72, torch.bfloat16)
    want = M.grouped_matmul_dgrad(dy, w, offsets), M.grouped_matmul_wgrad(dy, x, offsets)
    x.requires_grad_(True)
    w.requires_grad_(True)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        y = M.grouped_matmul(x, w, offsets)
        grads = torch.autograd.grad(y, (x, w), dy)
    for g in grads:
        g.zero_()
    gr.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(grads, want))


def test_refusals(cuda_device):
    from comfyui_b200 import moe_ops as M

    dev = cuda_device
    x, w, dy, off = make(dev, [5, 6], 64, 72, torch.bfloat16)
    for call, match in [
        (lambda: M.grouped_matmul(x, w[:, :, :56], off), "that fit"),
        (lambda: M.grouped_matmul(x.float(), w.float(), off), "bf16 or both fp16"),
        (lambda: M.grouped_matmul(x, w.half(), off), "bf16 or both fp16"),
        (lambda: M.grouped_matmul(x, w, off.long()), "int32"),
        (lambda: M.grouped_matmul(x, w, off[:2]), "int32 vector of 3"),
        (lambda: M.grouped_matmul(x, w, off, off), "int32 vector of 2"),
        (lambda: M.grouped_matmul(x.cpu(), w, off), "CUDA"),
        (lambda: M.grouped_matmul(x, w, off.cpu()), "CUDA"),
        (lambda: M.grouped_matmul(x[:, 1:57], w[:, :, :56], off), "16 bytes"),
        (lambda: M.grouped_matmul(x[:, :60], w[:, :, :60], off), "multiple of 8"),
        (lambda: M.grouped_matmul(x[:1].expand(11, 64), w, off), "rows must be contiguous"),
        (lambda: M.grouped_matmul(x, w[:1].expand(2, 72, 64), off), "groups must start"),
        (lambda: M.grouped_matmul(x, w, off, out=dy.float()), "out must be"),
        (lambda: M.grouped_matmul_wgrad(dy, x[:4], off), "need dy"),
        (lambda: M.grouped_matmul_wgrad(dy, x, off, out_dtype=torch.float16), "or fp32"),
    ]:
        with pytest.raises(ValueError, match=match):
            call()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("k,n", [(8, 8), (264, 1000), (2560, 6912)])
@pytest.mark.parametrize("counts,gap", [([1], 0), ([0, 1, 0, 1], 0), ([8], 0), ([5, 0, 4], 0), ([16], 0), ([0, 3, 0], 2), ([15, 1], 0)],
                         ids=str)
def test_few_rows(cuda_device, counts, gap, k, n, dtype):
    """The form that streams the weights for up to 16 rows, and the same call cut out of a longer batch."""
    from comfyui_b200 import moe_ops as M

    x, w, _, offsets = make(cuda_device, counts, k, n, dtype, gap=gap)
    ends = offsets.tolist()
    ranges = list(zip(ends[:-1], ends[1:]))
    ref = by_group(x, w, ranges, len(x), n, lambda a, b: a @ b.t())
    y = M.grouped_matmul(x, w, offsets)
    close(y, *ref, k, "y")
    long = torch.cat([x, torch.full((64, k), float("nan"), device=x.device, dtype=dtype)])
    close(M.grouped_matmul(long, w, offsets)[:len(x)], *ref, k, "y of a longer batch")
    if gap:
        out = torch.full((len(x), n), 7.0, dtype=dtype, device=x.device)
        M.grouped_matmul(x, w, offsets, out=out)
        assert torch.equal(out[gap:-gap], y[gap:-gap]) and (out[:gap] == 7).all() and (out[-gap:] == 7).all()
        assert (y[:gap] == 0).all() and (y[-gap:] == 0).all()
    most = torch.tensor([c // 2 for c in counts], dtype=torch.int32, device=x.device)
    half = M.grouped_matmul(x, w, offsets, most)
    for (lo, _), c in zip(ranges, counts):
        assert torch.equal(half[lo:lo + c // 2], y[lo:lo + c // 2]) and (half[lo + c // 2:lo + c] == 0).all()
    assert torch.equal(M.grouped_matmul(x, w, offsets), y)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("counts,k,n", [
    ([17], 4096, 136), ([0, 40, 100], 2056, 264), ([300, 0, 129], 1096, 1000),      # along k: the result
    ([17], 136, 4096), ([129, 0, 3, 40], 264, 1544),                                          # along n: the gradient of x
    ([4003], 520, 264), ([1500, 0, 1700], 264, 136), ([3000, 100, 0, 1], 72, 520), ([515, 509], 1000, 1032),   # the rows
], ids=str)
def test_few_tiles_and_a_long_contraction(cuda_device, counts, k, n, dtype):
    check_all(cuda_device, counts, k, n, dtype)


def test_few_tiles_run_alike_and_replay(cuda_device):
    from comfyui_b200 import moe_ops as M

    x, w, dy, offsets = make(cuda_device, [2000, 0, 1203], 4096, 136, torch.bfloat16)
    first = [M.grouped_matmul_dgrad(dy, w, offsets), M.grouped_matmul_wgrad(dy, x, offsets)]
    y = M.grouped_matmul(x[:90].contiguous(), w, offsets.clamp(max=90))
    stream = torch.cuda.Stream()
    small = x[:90].contiguous()
    few = offsets.clamp(max=90)
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        M.grouped_matmul(small, w, few)
    with torch.cuda.graph(graph, stream=stream):
        out = M.grouped_matmul(small, w, few)
        dw = M.grouped_matmul_wgrad(dy, x, offsets)
    for _ in range(3):
        out.fill_(float("nan"))
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, y) and torch.equal(dw, first[1])
    assert torch.equal(M.grouped_matmul_dgrad(dy, w, offsets), first[0])
    M.check_all_status()


@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_few_tiles_with_strides_padding_and_given_results(cuda_device, out_dtype):
    """Rows 16 apart in wider buffers, values that are not finite behind the groups, results in the middle of others."""
    from comfyui_b200 import moe_ops as M

    dev, k, n = cuda_device, 2056, 264
    gen = torch.Generator(device=dev).manual_seed(9)
    offsets = torch.tensor([2, 2900, 2900, 5900], dtype=torch.int32, device=dev)
    counts = torch.tensor([2801, 9, 2777], dtype=torch.int32, device=dev)
    ranges = [(2, 2803), (2900, 2900), (2900, 5677)]
    used = torch.zeros(6000, dtype=torch.bool, device=dev)
    for lo, hi in ranges:
        used[lo:hi] = True
    x = torch.randn((6000, 160), generator=gen, device=dev).bfloat16()[:, 8:144]
    dy = torch.randn((6000, n + 16), generator=gen, device=dev).bfloat16()[:, 8:8 + n]
    x[~used], dy[~used] = float("nan"), float("inf")
    dw = torch.full((3, n + 1, 144), 7.0, dtype=out_dtype, device=dev)
    M.grouped_matmul_wgrad(dy, x, offsets, counts, out=dw[:, :n, :136], out_dtype=out_dtype)
    for g, (lo, hi) in enumerate(ranges):
        a, b = dy[lo:hi].double(), x[lo:hi].double()
        close(dw[g, :n, :136], a.t() @ b, a.abs().t() @ b.abs(), max(hi - lo, 1), f"dw[{g}]")
    assert (dw[:, n] == 7).all() and (dw[:, :, 136:] == 7).all()
    few, most = torch.tensor([3, 60, 60, 110], dtype=torch.int32, device=dev), torch.tensor([50, 1, 41], dtype=torch.int32, device=dev)
    ranges = [(3, 53), (60, 60), (60, 101)]
    small = torch.randn((120, k + 24), generator=gen, device=dev).bfloat16()[:, 8:8 + k]
    w = (0.05 * torch.randn((3, n, k), generator=gen, device=dev)).bfloat16()
    keep = torch.zeros(120, dtype=torch.bool, device=dev)
    for lo, hi in ranges:
        keep[lo:hi] = True
    small[~keep] = float("nan")
    y = torch.full((120, n + 8), 7.0, dtype=torch.bfloat16, device=dev)
    M.grouped_matmul(small, w, few, most, out=y[:, :n])
    ref, mag = by_group(small, w, ranges, 120, n, lambda a, b: a @ b.t())
    close(y[keep, :n], ref[keep], mag[keep], k, "y")
    assert (y[~keep] == 7).all() and (y[:, n:] == 7).all()
    z = M.grouped_matmul(small, w, few, most)
    assert torch.equal(z[keep], y[keep, :n]) and (z[~keep] == 0).all()
    M.check_all_status()


def test_few_tiles_on_two_streams_at_once(cuda_device):
    from comfyui_b200 import moe_ops as M

    x, w, dy, offsets = make(cuda_device, [2000, 0, 1203], 4096, 136, torch.bfloat16)
    want = M.grouped_matmul_wgrad(dy, x, offsets)
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for i in range(12):
        stream = streams[i % 3]
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            got.append(M.grouped_matmul_wgrad(dy, x, offsets))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)
    M.check_all_status()
