"""Sizes and results that the products by expert refuse before anything is launched; a recorder stands in for the C entry
points where Python decides, and the library itself is asked where it does."""
import ctypes

import pytest
import torch

GOOD = ctypes.c_void_p(1 << 20)            # never read: every call is refused on the host


@pytest.fixture
def calls(monkeypatch):
    from comfyui_b200 import moe_ops as M

    seen = []
    monkeypatch.setattr(M, "_call", lambda name, index, *args: seen.append(name))
    monkeypatch.setattr(M, "_place", lambda first, *others: 0)
    monkeypatch.setattr(M, "device_status", lambda device: torch.zeros(4, dtype=torch.int32))
    return seen


def meta(*shape, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype, device="meta")


def host(*shape, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype)


def test_sizes_beyond_int32_are_refused(calls):
    """The C entry points count in int32; ctypes would cut a row number down to it and compute a part."""
    from comfyui_b200 import moe_ops as M

    off, w, f8 = torch.zeros(2, dtype=torch.int32), meta(1, 16, 16), torch.float8_e4m3fn
    wq, ws = meta(16, 16, dtype=f8), meta(1, 1, dtype=torch.float32)
    many, wide = (1 << 32) + 8, 1 << 29
    for call in (lambda: M.grouped_matmul(meta(many, 16), w, off), lambda: M.grouped_matmul_dgrad(meta(many, 16), w, off),
                 lambda: M.grouped_matmul_wgrad(meta(many, 16), meta(many, 16), off), lambda: M.block_linear(meta(many, 16), wq, ws),
                 lambda: M.block_linear(meta(2, many, 16), wq, ws), lambda: M.block_linear_dgrad(meta(many, 16), wq, ws),
                 lambda: M.grouped_block_linear(meta(many, 16), wq[None], ws[None], off), lambda: M.quantize_blocks_e4m3(meta(many, 16)),
                 lambda: M.grouped_matmul(meta((1 << 31) - 8, 16), w, off),              # tiles of rows would pass the end
                 lambda: M.grouped_matmul(meta(1, wide), meta(1, 16, wide), off),
                 lambda: M.grouped_matmul(meta(1, 16), meta(1, wide, 16), off),
                 lambda: M.grouped_matmul_wgrad(meta(1, 16), meta(1, wide), off)):
        with pytest.raises(ValueError, match="at most 2147482624 rows"):
            call()
    long = 65535 * 128 + 16
    for call in (lambda: M.quantize_blocks_e4m3(meta(1, long)), lambda: M.quantize_weight_blocks_e4m3(meta(16, long)),
                 lambda: M.quantize_weight_blocks_e4m3(meta(long, 16)), lambda: M.quantize_weight_blocks_e4m3(meta(65536, 8, 16)),
                 lambda: M.block_linear(meta(1, long), meta(16, long, dtype=f8), meta(1, 65536, dtype=torch.float32))):
        with pytest.raises(ValueError, match="at most 65535 blocks"):
            call()
    assert not calls
    M.grouped_matmul(meta(2147482624, 16), w, off)
    M.quantize_blocks_e4m3(meta(1, long - 16))
    assert len(calls) == 2


def test_empty_features_and_offsets_are_refused(calls):
    from comfyui_b200 import moe_ops as M

    off = torch.zeros(2, dtype=torch.int32)
    for call in (lambda: M.grouped_matmul(meta(3, 0), meta(1, 16, 0), off), lambda: M.grouped_matmul(meta(3, 16), meta(1, 0, 16), off),
                 lambda: M.grouped_matmul_wgrad(meta(3, 0), meta(3, 16), off), lambda: M.grouped_matmul_wgrad(meta(3, 16), meta(3, 0), off)):
        with pytest.raises(ValueError, match="1 to 268435456 features"):
            call()
    with pytest.raises(ValueError, match="one element more"):
        M.grouped_matmul_wgrad(meta(3, 16), meta(3, 16), off[:0])
    assert not calls


def test_the_library_refuses_sizes_beyond_its_counters():
    from comfyui_b200 import _native as N
    from comfyui_b200 import build

    build.build()
    lib = N.load()
    rows, wide = N.RAGGED_MAX_ROWS + 1, N.RAGGED_MAX_FEATURES + 16
    for r, n, k in ((rows, 32, 64), (5, wide, 64), (5, 32, wide)):
        assert lib.comfy_moe_grouped_matmul(GOOD, k, GOOD, k, n * k, 0, r, 2, n, k, GOOD, None, 1, GOOD, n, GOOD, None) == N.EUNSUPPORTED
        assert lib.comfy_moe_grouped_matmul_dgrad(GOOD, n, GOOD, k, n * k, 0, r, 2, n, k, GOOD, None, 1, GOOD, k, GOOD, None) == N.EUNSUPPORTED
        assert lib.comfy_moe_grouped_matmul_wgrad(GOOD, n, GOOD, k, 0, r, 2, n, k, GOOD, None, 0, GOOD, k, n * k, GOOD, None) == N.EUNSUPPORTED
        assert lib.comfy_moe_block_matmul(GOOD, k, 0, GOOD, GOOD, k, 0, GOOD, 0, r, 1, n, k, None, None, None, 0, GOOD, n, GOOD,
                                          None) == N.EUNSUPPORTED
    long = N.MAX_SCALE_BLOCKS * N.SCALE_BLOCK + 16
    assert lib.comfy_moe_block_quantize(GOOD, 64, 0, rows, 64, GOOD, 64, GOOD, rows, None) == N.EUNSUPPORTED
    assert lib.comfy_moe_block_quantize(GOOD, long, 0, 5, long, GOOD, long, GOOD, 5, None) == N.EUNSUPPORTED
    for groups, n, k in ((1, 32, long), (1, long, 32), (N.MAX_SCALE_BLOCKS + 1, 32, 32)):
        assert lib.comfy_moe_block_quantize_weight(GOOD, k, n * k, 0, groups, n, k, GOOD, GOOD, None) == N.EUNSUPPORTED


def test_a_result_that_overlaps_an_operand_is_refused(calls):
    """Tiles of it would be written while others are still to be read."""
    from comfyui_b200 import moe_ops as M

    off = torch.zeros(2, dtype=torch.int32)
    x, w = torch.zeros((11, 64), dtype=torch.bfloat16), torch.zeros((1, 64, 64), dtype=torch.bfloat16)
    wq, ws = w.to(torch.float8_e4m3fn), torch.ones((1, 1, 1))
    rows = torch.zeros((40, 64), dtype=torch.bfloat16)
    dw = torch.zeros((1, 64, 64), dtype=torch.bfloat16)
    for call in (lambda: M.grouped_matmul(x, w, off, out=x), lambda: M.grouped_matmul_dgrad(x, w, off, out=x),
                 lambda: M.grouped_matmul(rows[:11], w, off, out=rows[10:21]), lambda: M.grouped_matmul(x, w, off, out=w[0, 3:14]),
                 lambda: M.grouped_matmul(rows.view(20, 128)[:5, :64], w, off, out=rows[:5]),
                 lambda: M.block_linear(x, wq[0], ws[0], out=x), lambda: M.block_linear_dgrad(x, wq[0], ws[0], out=x),
                 lambda: M.grouped_block_linear(x, wq, ws, off, out=x),
                 lambda: M.grouped_matmul_wgrad(dw[0, :11], x, off, out=dw)):
        with pytest.raises(ValueError, match="overlap an operand"):
            call()
    assert not calls
    wide = torch.zeros((11, 136), dtype=torch.bfloat16)                       # columns of one buffer, before and behind
    M.grouped_matmul(wide[:, :64], w, off, out=wide[:, 64:128])
    M.grouped_matmul(wide[:, 72:], w, off, out=wide[:, 8:72])
    M.grouped_matmul(rows[:11], w, off, out=rows[11:22])
    M.block_linear(wide[:, :64], wq[0], ws[0], out=wide[:, 72:])
    M.grouped_matmul(wide[3:4, 64:128], w, off, out=wide[3, :64][None])
    M.block_linear(wide[:, :64], wq[0], ws[0, :, :], out=wide[:, 64:128])
    M.grouped_matmul(wide[3, :64][None], w, off, out=wide[3:4, 64:128])
    assert len(calls) == 7
    with pytest.raises(ValueError, match="overlap an operand"):
        M.grouped_matmul(wide[:, :64], w, off, out=wide[:, 56:120])


def test_shapes_of_a_block_linear_are_checked(calls):
    """Leading dimensions of a given result are those of the rows; what cannot be read or written as rows is refused."""
    from comfyui_b200 import moe_ops as M

    n, k = 48, 64
    x, w, ws = host(2, 3, k), host(n, k, dtype=torch.float8_e4m3fn), host(1, 1, dtype=torch.float32)
    for call, match in ((lambda: M.block_linear(x, w, ws, out=host(3, 2, n)), "out must be of shape"),
                        (lambda: M.block_linear(x, w, ws, out=host(1, 6, n)), "out must be of shape"),
                        (lambda: M.block_linear(x, w, ws, out=host(2, 3, n + 8)), "out must be of shape"),
                        (lambda: M.block_linear(x[0, 0], w, ws, out=host(1, 1, n)), "out must be of shape"),
                        (lambda: M.block_linear(x, w, ws, out=host(3, 2, n).transpose(0, 1)), "equally far apart"),
                        (lambda: M.block_linear(host(), w, ws), "that fit"), (lambda: M.block_linear(x, w[0], ws), "that fit"),
                        (lambda: M.block_linear(host(0, 0), host(n, 0, dtype=w.dtype), ws), "that fit"),
                        (lambda: M.block_linear(x, w[None], ws), "that fit"), (lambda: M.block_linear(x[..., :48], w, ws), "that fit")):
        with pytest.raises(ValueError, match=match):
            call()
    assert not calls
    for rows, out in ((x, host(2, 3, n)), (x, host(6, n)), (x, host(2, 3, n + 8)[..., :n]), (x[0, 0], host(n)), (x[0, 0], host(1, n)),
                      (x[0], host(3, n)), (x[:0], host(0, 3, n))):
        assert M.block_linear(rows, w, ws, out=out) is out
    assert M.block_linear(x, w, ws).shape == (2, 3, n) and M.block_linear(x[0, 0], w, ws).shape == (n,)
    assert len(calls) == 9
