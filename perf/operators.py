"""What is measured of the grouped and of the block-scaled matrix products, and their plain forms.

Four operators, each through ``comfyui_b200.moe_ops``:

* ``experts``       y[r] = x[r] W[g(r)]^T: the rows of a routed batch, sorted by expert, against a stack of weights
                    (``grouped_matmul``); offsets live on the device;
* ``experts train`` the same with the gradients of x and of W;
* ``block``         y = x W^T + b, W in e4m3 with one fp32 scale for each 128 x 128 block, x quantised on the way with one
                    scale for each 128 elements of a row (``block_linear``); ``grad``: with the gradient of x as well;
* ``block experts`` both at once (``grouped_block_linear``).
"""
import math

import torch

own = False

DEV = "cuda"
BLOCK = 128
E4M3_MAX = 448.0
TINY = 2.0 ** -100        # smallest maximum a block is scaled by
_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # one token of a chat or of a preview, top 2 of 4 experts of the HiDream layer: weights are read once, latency counts
        dict(name="experts one token", op="experts", dtype="bf16", experts=4, tokens=1, top_k=2, k=2560, n=6912),
        # a short prompt through 8 wider experts
        dict(name="experts 75 tokens", op="experts", dtype="bf16", experts=8, tokens=75, top_k=2, k=2048, n=8192),
        # an image pair: 2 x 4096 tokens
        dict(name="experts 8192 tokens", op="experts", dtype="bf16", experts=4, tokens=8192, top_k=2, k=2560, n=6912),
        # a small fine-tuning step in half precision, top 1, sizes that are no multiple of a tile
        dict(name="experts train odd", op="experts train", dtype="fp16", experts=8, tokens=1003, top_k=1, k=1000, n=2056),
        # a training step of a block with 8 experts
        dict(name="experts train 8192 tokens", op="experts train", dtype="bf16", experts=8, tokens=8192, top_k=2, k=2048,
             n=8192),
        # one row through a projection: the adaptive norm's input, a single token
        dict(name="block one row", op="block", dtype="bf16", rows=1, k=2560, n=6912, bias=False, grad=False),
        # the text rows of an image pair through the second product of a feed-forward
        dict(name="block 768 rows", op="block", dtype="bf16", rows=768, k=6912, n=2560, bias=True, grad=False),
        # the image rows through the first product
        dict(name="block 8192 rows", op="block", dtype="bf16", rows=8192, k=2560, n=6912, bias=False, grad=False),
        # an adapter's training step through a frozen projection
        dict(name="block train 1999 rows", op="block", dtype="fp16", rows=1999, k=2560, n=2560, bias=True, grad=True),
        dict(name="block experts one token", op="block experts", dtype="bf16", experts=4, tokens=1, top_k=2, k=2560, n=6912,
             grad=False),
        dict(name="block experts 8192 tokens", op="block experts", dtype="bf16", experts=4, tokens=8192, top_k=2, k=2560,
             n=6912, grad=False),
        # an adapter's training step through frozen experts, odd rows
        dict(name="block experts train odd", op="block experts", dtype="bf16", experts=8, tokens=2051, top_k=1, k=2048,
             n=2064, grad=True),
    ]


def _between(rng, low, high, step=1):
    """A whole number between low and high, spread over the logarithm, a multiple of step."""
    v = math.exp(rng.uniform(math.log(low), math.log(high)))
    return max(step, int(round(v / step)) * step)


def draw(rng):
    op = rng.choice(["experts", "experts", "experts train", "block", "block", "block experts"])
    case = dict(op=op, dtype=rng.choice(["bf16", "bf16", "fp16"]))
    step = 8 if op in ("experts", "experts train") else 16
    case.update(k=_between(rng, 256, 8192, step), n=_between(rng, 256, 8192, step))
    rows = _between(rng, 1, 8192)
    if op == "block":
        case.update(rows=rows, bias=rng.random() < 0.5, grad=rng.random() < 0.3)
    else:
        top_k = rng.choice([1, 2])
        case.update(experts=rng.choice([2, 3, 4, 6, 8, 16]), tokens=max(1, rows // top_k), top_k=top_k)
        if op == "block experts":
            case["grad"] = rng.random() < 0.3
    return case


def _randn(gen, *shape):
    return torch.randn(shape, generator=gen, device=DEV, dtype=torch.float32)


def _routed(case, seed):
    """Rows of each expert for a router with a moderate preference among experts, as the routing kernels give them."""
    gen = torch.Generator().manual_seed(seed)
    logits = torch.randn((case["tokens"], case["experts"]), generator=gen)
    logits += 0.7 * torch.randn((1, case["experts"]), generator=gen)
    chosen = logits.topk(case["top_k"], dim=1).indices.flatten()
    counts = torch.bincount(chosen, minlength=case["experts"])
    offsets = torch.zeros(case["experts"] + 1, dtype=torch.int32)
    offsets[1:] = counts.cumsum(0)
    return offsets.to(DEV), int(counts.max())


def _rows(gen, rows, width, dtype):
    """Activations as they come out of a norm: unit variance, a few channels ten times larger."""
    x = _randn(gen, rows, width)
    x[:, :: 97] *= 10.0
    return x.to(dtype)


def _block_weight(gen, *shape):
    """An e4m3 weight with its 128 x 128 block scales, as a checkpoint holds them: (weight, scales)."""
    w = 0.02 * _randn(gen, *shape)
    n, k = shape[-2:]
    w = torch.nn.functional.pad(w, (0, -k % BLOCK, 0, -n % BLOCK))
    nb, kb = w.shape[-2] // BLOCK, w.shape[-1] // BLOCK
    blocks = w.view(*shape[:-2], nb, BLOCK, kb, BLOCK)
    scale = blocks.abs().amax(dim=(-3, -1)) / E4M3_MAX
    q = (blocks / scale[..., :, None, :, None]).clamp(-E4M3_MAX, E4M3_MAX).view(w.shape)
    return q[..., :n, :k].to(torch.float8_e4m3fn).contiguous(), scale.contiguous()


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    op, dtype, k, n = case["op"], _TYPES[case["dtype"]], case["k"], case["n"]
    s = {"op": op, "dtype": dtype, "k": k, "n": n, "grad": case.get("grad", op == "experts train"), "bias": None}
    if op == "block":
        rows = case["rows"]
        s["w"], s["scale"] = _block_weight(gen, n, k)
        if case["bias"]:
            s["bias"] = _randn(gen, n).to(dtype)
    else:
        rows, g = case["tokens"] * case["top_k"], case["experts"]
        s["offsets"], s["most"] = _routed(case, seed)
        if op == "block experts":
            s["w"], s["scale"] = _block_weight(gen, g, n, k)
        else:
            s["w"] = (0.02 * _randn(gen, g, n, k)).to(dtype)
    s["x"] = _rows(gen, rows, k, dtype)
    if s["grad"]:
        s["dy"] = _randn(gen, rows, n).to(dtype)
        s["x"].requires_grad_(True)
        if op == "experts train":
            s["w"].requires_grad_(True)
    return s


# ------------------------------------------------------------------------------------------------ the plain forms
def _blockwise(x):
    """x [R, K] in 32 bits as its e4m3 values times the scales of their blocks of 128."""
    r, k = x.shape
    b = torch.nn.functional.pad(x, (0, -k % BLOCK)).view(r, -1, BLOCK)
    top = b.abs().amax(dim=-1, keepdim=True).clamp(min=TINY)
    q = (b * 0.4375 / top * 1024.0).to(torch.float8_e4m3fn).float()      # b * 448 / top, without leaving the range
    return (q * (top / E4M3_MAX)).view(r, -1)[:, :k]


def _full_weight(w, scale):
    n, k = w.shape[-2:]
    return w.float() * scale.repeat_interleave(BLOCK, -2)[..., :n, :].repeat_interleave(BLOCK, -1)[..., :k]


def _places(s, rows):
    """(expert, place within the expert's rows) of every row."""
    r = torch.arange(rows, device=DEV, dtype=torch.int32)
    expert = torch.searchsorted(s["offsets"], r, right=True) - 1
    return expert, (r - s["offsets"][expert]).long()


def _padded(s, x, places):
    out = torch.zeros((s["w"].shape[0], s["most"], x.shape[1]), device=DEV, dtype=torch.float32)
    out[places] = x
    return out


def _plain(s):
    dtype, grad = s["dtype"], s["grad"]
    x, block = s["x"].detach().float(), s["op"].startswith("block")
    w = _full_weight(s["w"], s["scale"]) if block else s["w"].detach().float()
    if block:
        x = _blockwise(x)
    dy = s["dy"].float() if grad else None
    if block and grad:
        dy = _blockwise(dy)
    if s["op"] == "block":
        y = x @ w.t()
        if s["bias"] is not None:
            y = y + s["bias"].float()
        return (y.to(dtype), (dy @ w).to(dtype)) if grad else y.to(dtype)
    places = _places(s, x.shape[0])
    xp = _padded(s, x, places)
    y = torch.bmm(xp, w.transpose(1, 2))[places].to(dtype)
    if not grad:
        return y
    dyp = _padded(s, dy, places)
    dx = torch.bmm(dyp, w)[places].to(dtype)
    if block:
        return y, dx
    return y, dx, torch.bmm(dyp.transpose(1, 2), xp).to(dtype)


def run(state):
    s = state
    if not own:
        return _plain(s)
    from comfyui_b200 import moe_ops

    if s["op"] == "block":
        y = moe_ops.block_linear(s["x"], s["w"], s["scale"], s["bias"])
        leaves = [s["x"]]
    elif s["op"] == "block experts":
        y = moe_ops.grouped_block_linear(s["x"], s["w"], s["scale"], s["offsets"])
        leaves = [s["x"]]
    else:
        y = moe_ops.grouped_matmul(s["x"], s["w"], s["offsets"])
        leaves = [s["x"], s["w"]]
    if not s["grad"]:
        return y
    return (y.detach(), *torch.autograd.grad(y, leaves, s["dy"]))


def work(case):
    k, n, grad = case["k"], case["n"], case.get("grad", case["op"] == "experts train")
    wide = case["op"].startswith("block")
    if case["op"] == "block":
        rows, weights = case["rows"], 1
    else:
        rows = case["tokens"] * case["top_k"]
        weights = min(case["experts"], rows)
    wbytes = weights * n * k * (1 if wide else 2)
    moved, flops = 2 * rows * (k + n) + wbytes, 2.0 * rows * n * k
    if grad:
        moved += 2 * rows * (k + n)              # the output's gradient is read, x's is written; W is read once for both
        flops *= 2
        if not wide:
            moved += wbytes                      # W's gradient is written
            flops *= 1.5
    return {"bytes": moved, "flops": flops}


# ------------------------------------------------------------------------------------------------ in 64 bits
def _exact_blocks(x):
    out = torch.zeros_like(x, dtype=torch.float64)
    for j in range(0, x.shape[1], BLOCK):
        b = x[:, j:j + BLOCK].double()
        top = b.abs().max(dim=1, keepdim=True).values.clamp(min=TINY)
        out[:, j:j + BLOCK] = (b * E4M3_MAX / top).to(torch.float8_e4m3fn).double() * top / E4M3_MAX
    return out


def _exact_weight(w, scale):
    out = w.double()
    for i in range(scale.shape[-2]):
        for j in range(scale.shape[-1]):
            out[..., i * BLOCK:(i + 1) * BLOCK, j * BLOCK:(j + 1) * BLOCK] *= scale[..., i, j, None, None].double()
    return out


def exact(case, seed):
    s = prepare(case, seed)
    block, grad = s["op"].startswith("block"), s["grad"]
    w = _exact_weight(s["w"], s["scale"]) if block else s["w"].detach().double()
    x = _exact_blocks(s["x"].detach()) if block else s["x"].detach().double()
    dy = None
    if grad:
        dy = _exact_blocks(s["dy"]) if block else s["dy"].double()
    if s["op"] == "block":
        y = torch.matmul(x, w.t())
        if s["bias"] is not None:
            y += s["bias"].double()
        return (y, torch.matmul(dy, w)) if grad else y
    ends = s["offsets"].tolist()
    y = torch.zeros((x.shape[0], s["n"]), device=DEV, dtype=torch.float64)
    dx, dw = torch.zeros_like(x), None if block else torch.zeros_like(w)
    for g in range(w.shape[0]):
        rows = slice(ends[g], ends[g + 1])
        y[rows] = x[rows] @ w[g].t()
        if grad:
            dx[rows] = dy[rows] @ w[g]
            if not block:
                dw[g] = dy[rows].t() @ x[rows]
    if not grad:
        return y
    return (y, dx) if block else (y, dx, dw)
