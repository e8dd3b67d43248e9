"""The quantisers next to the borders between e4m3 values, held to the definition: nearest, ties to even, of the exact
quotient x * 448 / m.  Needs a B200.

The definition's quotient of two fp32 numbers is at least 2^-29 of itself away from a border that it is not equal to, so the
64-bit quotient (one rounding, 2^-53) lies on the same side; it is compared with the borders themselves, not rounded through
a type between."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BLOCK = 128


def grid(dev):
    """(the e4m3 magnitudes, the borders between them) in 64 bits."""
    codes = torch.arange(127, dtype=torch.uint8, device=dev)
    values = codes.view(torch.float8_e4m3fn).double()
    return values, (values[1:] + values[:-1]) / 2


def nearest(x, m):
    """Bytes of the e4m3 numbers nearest to x * 448 / m."""
    values, borders = grid(x.device)
    q = x.double().abs() * 448.0 / m.double()
    code = torch.searchsorted(borders, q)                                   # on a border: the value below it ...
    tie = borders[code.clamp(max=len(borders) - 1)] == q
    code = code + (tie & (code % 2 == 1))                                   # ... or the one above, whichever is even
    return (code + 128 * torch.signbit(x)).to(torch.uint8)


def next_to_borders(dev, rows, short, seed, share=1):
    """Rows [rows, 4 blocks] of fp32 numbers on the borders, and up to two steps of fp32 beside them, of maxima [rows, 4] of
    any magnitude, one for `share` rows; the maximum stands in each block's first place."""
    gen = torch.Generator(device=dev).manual_seed(seed)
    shape = (-(-rows // share), 4, 1)
    m = (1 + torch.rand(shape, generator=gen, device=dev, dtype=torch.float64)) * \
        2.0 ** torch.randint(-99, 127, shape, generator=gen, device=dev).double()
    m = m.float()
    if short:                                                               # of few digits: quotients that are borders
        m = (m.view(torch.int32) & -65536).view(torch.float32)
    m = m.repeat_interleave(share, 0)[:rows]
    borders = grid(dev)[1]
    b = borders[torch.randint(0, len(borders), (rows, 4, BLOCK), generator=gen, device=dev)]
    x = (b * m.double() / 448.0).float()
    step = torch.randint(-2, 3, x.shape, generator=gen, device=dev, dtype=torch.int32)
    x = (x.view(torch.int32) + step).view(torch.float32)
    if short:
        x = (x.view(torch.int32) & -4096).view(torch.float32)
    x = torch.minimum(x, m)
    x = torch.where(torch.rand(x.shape, generator=gen, device=dev) < 0.5, x, -x)
    x[:, :, 0] = m[:, :, 0]
    return x.view(rows, -1), m


@pytest.mark.parametrize("short", [False, True], ids=["all digits", "ties"])
def test_fp32_rows_next_to_every_border(cuda_device, short):
    from comfyui_b200 import moe_ops as M

    x, m = next_to_borders(cuda_device, 4000, short, 17 + short)
    q, scale = M.quantize_blocks_e4m3(x)
    want = nearest(x, m.expand(-1, -1, BLOCK).reshape(x.shape))
    assert torch.equal(q.view(torch.uint8), want)
    assert torch.equal(scale, (m.double() / 448.0).float().squeeze(-1))


def weight_maxima(w):
    n, k = w.shape
    return torch.nn.functional.pad(w, (0, 0, 0, -n % BLOCK)).view(-1, BLOCK, k // BLOCK, BLOCK).abs().amax((1, 3))


def check_weights(w):
    from comfyui_b200 import moe_ops as M

    tops = weight_maxima(w)
    q, scale = M.quantize_weight_blocks_e4m3(w)
    top = tops.repeat_interleave(BLOCK, 0)[:len(w)].repeat_interleave(BLOCK, 1)
    number = torch.isfinite(w) & ~torch.isnan(top)                          # (an infinity over an infinite maximum is NaN)
    assert torch.equal(torch.isnan(q.float()), ~number)
    assert torch.equal(q.view(torch.uint8)[number], nearest(w, top)[number])
    torch.testing.assert_close(scale, (tops.double() / 448.0).float(), rtol=0, atol=0, equal_nan=True)


@pytest.mark.parametrize("short", [False, True], ids=["all digits", "ties"])
def test_fp32_weights_next_to_every_border(cuda_device, short):
    w, m = next_to_borders(cuda_device, 700, short, 7 + short, share=BLOCK)
    assert torch.equal(weight_maxima(w), m[::BLOCK, :, 0])
    check_weights(w)


def test_fp32_weights_over_all_magnitudes(cuda_device):
    """Rows brought to the magnitude of their block's first one; where that leaves fp32, they hold infinities and zeros."""
    x, m = next_to_borders(cuda_device, 300, False, 5)
    first = m[::BLOCK]
    ratio = (first.repeat_interleave(BLOCK, 0)[:300] / m).expand(-1, -1, BLOCK).reshape(x.shape)
    check_weights((x.double() * ratio.double()).float())


def test_fp32_blocks_of_zeros_tiny_and_not_finite_values(cuda_device):
    from comfyui_b200 import moe_ops as M

    x = torch.zeros((6, 256), device=cuda_device)
    x[0, 3] = -0.0
    x[1] = -2.0 ** -120                                      # under the floor 2^-100: rounds to 0, and keeps its sign
    x[2, 5], x[2, 6] = float("nan"), 3.0
    x[3, 7], x[3, 8] = float("-inf"), -3.0
    x[4, 130], x[4, 131], x[4, 132] = 3.4028234663852886e38, 1.0, -1.0e-45        # the largest number, the smallest
    q, scale = M.quantize_blocks_e4m3(x)
    byte = q.view(torch.uint8)
    assert byte[0, 3] == 128 and (byte[1] == 128).all() and (scale[:2] == 2.0 ** -100 / 448).all()
    assert torch.isnan(q[2, :128].float()).all() and torch.isnan(scale[2, 0]) and (byte[2, 128:] == 0).all()
    assert torch.isnan(q[3, 7].float()) and torch.isinf(scale[3, 0]) and byte[3, 8] == 128 and byte[3, 9] == 0
    assert q[4, 130].float() == 448 and byte[4, 131] == 0 and byte[4, 132] == 128 and torch.isfinite(scale[4]).all()


@pytest.mark.parametrize("sign", [1, -1])
def test_every_ratio_of_bf16_significands(cuda_device, sign):
    """x / m for all 128 significands of both, powers of two among them, over every power of two that e4m3 covers."""
    from comfyui_b200 import moe_ops as M

    dev = cuda_device
    sig = torch.arange(128, 256, device=dev).double()
    x = (sig[:, None] / 2.0 ** torch.arange(20, device=dev).double()).flatten()          # 255 down to 2^-12
    x = sign * torch.nn.functional.pad(x, (0, -x.numel() % (BLOCK - 1)), value=1.0).view(-1, BLOCK - 1)
    alternate = torch.where(torch.arange(BLOCK - 1, device=dev) % 2 == 0, 1.0, -1.0)
    x = (x * alternate)[None].expand(128, -1, -1)
    m = (2 * sig)[:, None, None].expand(128, x.shape[1], 1)                             # a place of its own in every block
    rows = torch.cat([m, x], 2)
    for s in sig.tolist():
        assert (rows[0, :, 1:].abs() == s).any()
    rows, tops = rows.reshape(128, -1).bfloat16(), m.expand(-1, -1, BLOCK).reshape(128, -1)
    assert torch.equal(rows.view(128, -1, BLOCK).abs().amax(2).double(), m[:, :, 0])
    q, scale = M.quantize_blocks_e4m3(rows)
    assert torch.equal(q.view(torch.uint8), nearest(rows, tops))
    assert torch.equal(scale, (m[:, :, 0] / 448.0).float())
    q, scale = M.quantize_blocks_e4m3(rows.float())
    assert torch.equal(q.view(torch.uint8), nearest(rows, tops))
