"""The block-scaled Linear without the kernel: its composition, the model patcher's round trip, what the fused paths of the
models make of it."""
import pytest
import torch

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24, torch.float64: 2.0 ** -53}
N, K = 200, 272


def linear(scales, seed=0):
    """(Linear of N x K, its weight in 64 bits): e4m3 values, with the given scales dealt to the blocks."""
    from comfyui_b200 import ops

    g = torch.Generator().manual_seed(seed)
    lin = ops.block_scaled_fp8_ops().Linear(K, N, bias=False)
    lin.load_state_dict({"weight": (8 * torch.randn((N, K), generator=g)).to(torch.float8_e4m3fn),
                         "scale_weight": torch.tensor(scales)[torch.arange(6) % len(scales)].view(2, 3)}, strict=True)
    exact = torch.empty((N, K), dtype=torch.float64)
    for i in range(N):
        for j in range(K):
            exact[i, j] = lin.weight[i, j].double() * lin.scale_weight[i // 128, j // 128].double()
    return lin, exact


SCALES = [1.0057, 3.3e-6, 2.2e-8, 7.1e-5, 0.0123]           # in fp16 the second and the fourth lose digits, the third is 0


@pytest.mark.parametrize("dtype", [torch.float64, torch.float32, torch.bfloat16, torch.float16], ids=str)
def test_weights_are_scaled_back_with_one_rounding(dtype):
    lin, exact = linear(SCALES)
    plain = lin.weight.to(dtype)                                             # every e4m3 number is one of each type
    # half a step of the result, that of the fp32 product, and in fp16 half the smallest number
    bound = (HALF_STEP[dtype] + (dtype != torch.float64) * 2.0 ** -24) * exact.abs() + 2.0 ** -25 * (dtype == torch.float16)
    got = lin.convert_weight(plain)
    assert got.dtype == dtype and ((got.double() - exact).abs() <= bound * (1 + 2.0 ** -20)).all()
    assert torch.equal(lin.weight.to(dtype), plain)
    again = lin.convert_weight(plain, inplace=True)
    assert again is plain and torch.equal(again, got)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
def test_the_composition_against_64_bits(dtype):
    lin, exact = linear(SCALES, seed=1)
    x = torch.eye(K, dtype=dtype)                                            # picks single weights: no sum rounds
    got = lin(x).t().double()
    bound = (HALF_STEP[dtype] + 2.0 ** -24) * exact.abs() + 2.0 ** -25 * (dtype == torch.float16)
    assert ((got - exact).abs() <= bound * (1 + 2.0 ** -20)).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
def test_a_weight_is_set_through_scales_of_any_size(dtype):
    """set_weight divides by the scales in fp32: what convert_weight gave comes back as the e4m3 numbers it was made of, or as
    neighbours of theirs."""
    lin, _ = linear([1.0057, 7.1e-5, 0.0123] if dtype == torch.float16 else SCALES)
    q = lin.set_weight(lin.convert_weight(lin.weight.float()).to(dtype), seed=3, return_weight=True)
    assert q.dtype == torch.float8_e4m3fn
    got, want = q.double(), lin.weight.double()
    # the quotient is less than a step (2^-3 of the value, 2^-9 below 2^-6) from the number it came from: 2^-8 of it, or half the
    # smallest fp16 number over the scale, 2^-25 / 7.1e-5 = 0.22 x 2^-9; stochastic rounding then ends on it or next to it
    assert torch.isfinite(got).all()
    assert ((got - want).abs() <= torch.clamp(2.0 ** -3 * want.abs(), min=2.0 ** -9) * (1 + 2.0 ** -6)).all()


def test_no_fused_path_takes_the_weights_without_their_scales():
    """A module cast to bf16 as a whole holds e4m3 numbers in bf16: still nothing without the block scales."""
    from comfyui_b200 import ops

    cpu = torch.device("cpu")
    lin, exact = linear([0.5, 0.0078125])
    assert ops._linear_state(lin, cpu) is None
    lin.to(torch.bfloat16)
    assert lin.weight.dtype == torch.bfloat16
    for state in (ops._linear_state(lin, cpu), ops._biased_linear_state(lin, cpu)):
        assert state is None
    wide = ops.block_scaled_fp8_ops().Linear(256, 256, dtype=torch.bfloat16).to(torch.bfloat16)      # a shape for the projections
    assert ops._bias_linear_state(wide, cpu, 256) is None
    plain = ops.disable_weight_init.Linear(256, 256, dtype=torch.bfloat16)
    assert ops._bias_linear_state(plain, cpu, 256) is not None
    x = torch.eye(K, dtype=torch.bfloat16)
    assert torch.equal(lin(x).t().double(), exact)                           # powers of two: no rounding at all
