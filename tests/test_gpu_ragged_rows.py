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


def ranges_of(offsets, counts, rows):
    """Rows of each group by the documented rule, from lists."""
    out, reach = [], 0
    for g in range(len(offsets) - 1):
        begin = reach = max(reach, min(max(offsets[g], 0), rows))
        reach = max(reach, min(max(offsets[g + 1], 0), rows))
        n = reach - begin
        out.append((begin, begin + (n if counts is None else min(n, max(counts[g], 0)))))
    return out


def layouts(groups, rows, seed):
    """(offsets, counts) as lists: spread, all in one group, padded, out of order, nobody's rows at both ends."""
    g = torch.Generator().manual_seed(seed)
    cut = torch.randint(0, rows + 1, (groups - 1,), generator=g).sort().values.tolist()
    yield [0] + cut + [rows], None
    at = int(torch.randint(0, groups, (1,), generator=g))
    yield [0] * (at + 1) + [rows] * (groups - at), None
    yield [0] + cut + [rows], torch.randint(-1, 3, (groups,), generator=g).tolist()
    yield torch.randint(-2, rows + 3, (groups + 1,), generator=g).tolist(), None
    ends = sorted(torch.randint(1, max(2, rows), (groups + 1,), generator=g).tolist())
    yield ends, None
    yield [rows] * (groups + 1), None


HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("rows", [1, 2, 3, 8, 9, 16, 17])
@pytest.mark.parametrize("groups", [2, 16, 17, 31, 32, 33, 64, 257, 768])
def test_few_rows_among_many_groups(cuda_device, groups, rows, dtype):
    """Every row by its own group's weight, whichever groups are empty; the tolerance is one rounding of the result plus one of
    fp32 for each term (and, with block scales, three for each block)."""
    from comfyui_b200 import moe_ops as M

    dev, n, k = cuda_device, 40, 144
    gen = torch.Generator(device=dev).manual_seed(groups + rows)
    x = torch.randn((rows, k), generator=gen, device=dev).to(dtype)
    w = (0.05 * torch.randn((groups, n, k), generator=gen, device=dev)).to(dtype)
    wq, ws = M.quantize_weight_blocks_e4m3(w)
    xq, xs = M.quantize_blocks_e4m3(x)
    spread = lambda s: s.double().repeat_interleave(128, -1)[..., :k]                           # noqa: E731
    operands = {"bf16 / fp16": (x.double(), w.double(), k),
                "block": (xq.double() * spread(xs), wq.double() * spread(ws).expand(groups, n, k), k + 3 * 2)}
    for offsets, counts in layouts(groups, rows, groups * 20 + rows):
        off = torch.tensor(offsets, dtype=torch.int32, device=dev)
        cnt = None if counts is None else torch.tensor(counts, dtype=torch.int32, device=dev)
        group_of = torch.full((rows,), -1)
        for g, (lo, hi) in enumerate(ranges_of(offsets, counts, rows)):
            group_of[lo:hi] = g
        used = (group_of >= 0).to(dev)
        for name, call in (("bf16 / fp16", lambda **kw: M.grouped_matmul(x, w, off, cnt, **kw)),
                           ("block", lambda **kw: M.grouped_block_linear(x, wq, ws, off, cnt, **kw))):
            a, b, terms = operands[name]
            b = b[group_of.clamp(min=0).to(dev)]
            ref, mag = torch.einsum("rk,rnk->rn", a, b), torch.einsum("rk,rnk->rn", a.abs(), b.abs())
            y = call()
            bound = HALF_STEP[dtype] * ref.abs() + terms * 2.0 ** -23 * mag + 2.0 ** -24 * (dtype == torch.float16)
            assert ((y.double() - ref).abs() <= bound)[used].all(), (name, offsets, counts)
            assert (y[~used] == 0).all()
            out = torch.full_like(y, 7.0)
            call(out=out)
            assert torch.equal(out[used], y[used]) and (out[~used] == 7).all()
    M.read_status(M.device_status(dev))


def device_time(call, calls=20):
    """Shortest time of a call in us, from replays of a graph of some."""
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for _ in range(calls):
            call()
    best = float("inf")
    for _ in range(8):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        graph.replay()
        b.record()
        b.synchronize()
        best = min(best, a.elapsed_time(b) * 1e3 / calls)
    return best


@pytest.mark.parametrize("rows", [1, 8])
def test_groups_without_rows_cost_little(cuda_device, rows):
    """The same weights are read whether 8 or 768 groups could have rows; what may grow is the look through the offsets."""
    from comfyui_b200 import moe_ops as M

    dev, n, k = cuda_device, 2048, 256
    gen = torch.Generator(device=dev).manual_seed(2)
    x = torch.randn((rows, k), generator=gen, device=dev).bfloat16()
    w = torch.randn((768, n, k), generator=gen, device=dev).bfloat16()
    wq, ws = M.quantize_weight_blocks_e4m3(w)
    times = {}
    for groups in (8, 768):
        ends = [min(g * rows // 8 if g <= 8 else rows, rows) for g in range(groups + 1)]
        off = torch.tensor(ends, dtype=torch.int32, device=dev)
        times[groups] = (device_time(lambda: M.grouped_matmul(x, w[:groups], off)),
                         device_time(lambda: M.grouped_block_linear(x, wq[:groups], ws[:groups], off)))
    print(times)
    assert all(many < 8 * few for few, many in zip(times[8], times[768])), times
