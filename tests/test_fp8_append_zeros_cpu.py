"""The oracle's rule for tokens that need no scale: they leave their block's to the others, whatever the calls they come in."""
import numpy as np
import pytest

from oracle import cache as orc


@pytest.mark.parametrize("odd", [0.0, np.nan, np.inf])
@pytest.mark.parametrize("at", [0, 7, 31])
def test_tokens_that_need_no_scale(odd, at):
    rng = np.random.default_rng(1)
    x = rng.standard_normal((1, 2, 32, 16)) * 0.003
    x[:, :, at] = odd
    fin = np.isfinite(x)
    outs = []
    for sizes in ([32], [1] * 32, [8, 1, 23], [31, 1]):
        codes, scale, n = np.zeros((1, 2, 32, 16), np.uint8), np.ones((1, 2, 1), np.float32), 0
        for m in sizes:
            orc.append_fp8(codes, scale, None, [n], x[:, :, n:n + m], 32)
            n += m
        for h in range(2):
            assert scale[0, h, 0] == orc.block_scale(np.abs(x[0, h][fin[0, h]]).max())
        have = orc.values(codes, scale)
        assert np.array_equal(np.isnan(have), ~fin)
        # half a step of a code, and half a step of a subnormal one for each scale it was re-encoded at (those at least double)
        tol = np.maximum(np.abs(x) * 2.0 ** -4, 3 * scale[..., None].astype(np.float64) * 2.0 ** -10)
        assert (np.abs(have - x)[fin] <= tol[fin]).all()
        outs.append(scale.copy())
    assert all(np.array_equal(o, outs[0]) for o in outs)


def test_blocks_without_a_value():
    codes, scale = np.full((1, 1, 64, 16), 0x31, np.uint8), np.ones((1, 1, 4), np.float32)
    orc.append_fp8(codes, scale, None, [0], np.zeros((1, 1, 5, 16)), 16)
    assert scale[0, 0, 0] == np.float32(2.0 ** -126) and (codes[0, 0, :5] == 0).all()
    orc.append_fp8(codes, scale, None, [5], np.full((1, 1, 1, 16), 448.0), 16)
    assert scale[0, 0, 0] == 1.0 and (codes[0, 0, :5] == 0).all() and (codes[0, 0, 5] == 0x7E).all()
    orc.append_fp8(codes, scale, None, [6], np.full((1, 1, 2, 16), np.nan), 16)
    assert scale[0, 0, 0] == 1.0 and (codes[0, 0, 5] == 0x7E).all() and (codes[0, 0, 6:8] == 0x7F).all()
