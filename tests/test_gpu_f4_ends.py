"""The 4-bit operators at the ends of their ranges: scales that saturate beside ones that do not, the smallest scales, activations and weights that are
very large, infinite or NaN, in each of the product's kernels.  Needs a B200: run with -m gpu."""
import numpy as np
import pytest

import lightnet_b200 as ln
from test_gpu_f4 import BLOCK, FMT, f32, narrow

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def be():
    b = ln.B200Backend(0)
    yield b
    b.close()


def same_as_defined(be, x, g, dtype, source):
    """Codes, scales and values of a narrowed tensor against the definition."""
    t = be.upload_f16(x.shape, x) if source == "f16" else be.upload_f32(x.shape, x)
    q = be.narrow_f4(t, g, dtype)
    codes, scales = be.download_f4(q)
    want_codes, want_scales, values = narrow(x, dtype, g)
    assert np.array_equal(scales, want_scales)
    assert np.array_equal(codes & 7, want_codes & 7)
    assert np.array_equal(be.download_f32(be.widen_f4(q)), values.astype(np.float32))
    return scales


@pytest.mark.parametrize("source", ["f32", "f16"])
@pytest.mark.parametrize("shape", [(1, 4096, 1, 1), (3, 333, 9, 11), (64, 48, 5, 5), (2, 1040, 7, 1)])
def test_saturated_scales_beside_others(be, shape, source):
    """g of a calibration on smaller values: which blocks' scales saturate differs from one to the next, in every order."""
    rng = np.random.default_rng(sum(shape))
    x = rng.normal(0, 1, shape)
    blocks = -(-shape[1] // 16)
    big = rng.random((shape[0], blocks) + shape[2:]) < 0.5
    big[0, :4, 0, 0] = (True, False, False, True)[: blocks]
    x = (x * np.where(np.repeat(big, 16, 1)[:, : shape[1]], 900.0, 1.0)).astype(np.float16).astype(np.float32)
    scales = same_as_defined(be, x, float(np.float32(4 / 2688)), ln.LN_F4, source)
    assert 0.3 < (scales == 126).mean() < 0.7


def test_quotients_next_to_a_border_at_the_smallest_scales(be):
    """Tensor scales of 2^-100 and a little more, block scales from 2^-9 on: values whose quotient by d lies next to the middle of two binary32 numbers at a
    border between two codes."""
    for extra in range(1, 40):
        g = float(np.float32((2 ** 23 + extra) * 2.0 ** -123))
        for s in (1, 2, 3, 5, 8, 9, 16, 40, 80, 126):  # codes of E4M3
            step = (s % 8 / 8 * 2.0 ** -6) if s < 8 else (1 + s % 8 / 8) * 2.0 ** (s // 8 - 7)
            d = np.float32(f32(step * g))
            x = np.zeros((1, 16 * 60, 1, 1), np.float32)
            x[0, ::16] = 6 * d
            near = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
            at = np.arange(16 * 60)[np.arange(16 * 60) % 16 != 0]
            v = (near[at % 7] * np.float64(d)).astype(np.float32)
            v = (v.view(np.uint32) + (at // 7 % 7 - 3).astype(np.uint32)).view(np.float32)
            x[0, at, 0, 0] = v * np.where(at % 2, 1, -1)
            scales = same_as_defined(be, x, g, ln.LN_F4, "f32")
            assert (scales == s).all()
