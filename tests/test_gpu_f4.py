"""Microscaled 4-bit tensors (LN_F4, LN_MX4) through the C ABI against a plain numpy restatement of their definition.

Codes, scales and widened values are compared exactly: every step that leads to them is one binary32 operation or a rounding to an
E4M3 / E2M1 / E8M0 value.  Products are compared with sums in 64 bits: a binary32 sum of n terms is off by at most about n half
steps of its largest partial sum, and the partial sums of one instruction (64 terms) are exact before they are aligned, so the bound
per output is (terms / 64 + 8) * 2^-23 * sum|x w| plus the activation's (a few 2^-23 of its value, times its slope, at most 1.1) and
half a step of the output type.  Needs a B200: run with -m gpu."""
import ctypes as C

import numpy as np
import pytest

import lightnet_b200 as ln

pytestmark = pytest.mark.gpu

LEVELS = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], np.float64)
BORDERS = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0]
TO_EVEN_ABOVE = [False, True, False, True, False, True, False]
E4M3 = np.array([m / 8 * 2.0 ** -6 for m in range(8)] + [(1 + m / 8) * 2.0 ** e for e in range(-6, 9) for m in range(8)][:-1])
BLOCK = {ln.LN_F4: 16, ln.LN_MX4: 32}
FMT = [ln.LN_F4, ln.LN_MX4]


@pytest.fixture(scope="module")
def be():
    b = ln.B200Backend(0)
    yield b
    b.close()


def f32(v):
    with np.errstate(over="ignore", invalid="ignore"):
        return np.asarray(v, np.float64).astype(np.float32).astype(np.float64)


def e4m3_code(v):
    """Nearest even, saturating; v >= 0, NaN is 0x7F."""
    v = np.asarray(v, np.float64)
    at = np.clip(np.searchsorted(E4M3, np.minimum(v, 448.0)), 1, len(E4M3) - 1)
    below, above = E4M3[at - 1], E4M3[at]
    up = (v - below > above - v) | ((v - below == above - v) & (at % 2 == 0))
    return np.where(np.isnan(v), 0x7F, np.where(v >= 448.0, 126, np.where(up, at, at - 1))).astype(np.int64)


def scale_value(dtype, code):
    if dtype == ln.LN_F4:
        return np.where(code == 0x7F, np.nan, E4M3[np.minimum(code, 126)])
    return np.where(code == 255, np.nan, np.ldexp(1.0, code.astype(np.int64) - 127))


def blocks_of(x, size):
    n, c, h, w = x.shape
    full = np.zeros((n, -(-c // size) * size, h, w))
    full[:, :c] = x
    return full.reshape(n, -1, size, h, w)


def narrow(x, dtype, g):
    """(codes [n, c, h, w], scale codes [n, blocks, h, w], values): g is a number or one per image (per filter)."""
    x = np.asarray(x, np.float32).astype(np.float64)
    g = np.broadcast_to(np.asarray(g, np.float64).reshape(-1, 1, 1, 1), (x.shape[0], 1, 1, 1))
    b = blocks_of(x, BLOCK[dtype])
    with np.errstate(all="ignore"):
        amax = np.abs(b).max(2)
        if dtype == ln.LN_F4:
            s = e4m3_code(f32(amax / f32(6.0 * g)))
            d = f32(scale_value(dtype, s) * g)
        else:
            bits = amax.astype(np.float32).view(np.uint32)
            field = (bits >> 23).astype(np.int64)
            s = np.where(np.isnan(amax), 255, np.maximum(field - 2, 0))
            d = scale_value(dtype, s)
        t = f32(b / d[:, :, None])
        t = np.where((d == 0)[:, :, None], 0.0, t)
        a = np.abs(t)
        code = np.zeros(a.shape, np.int64)
        for border, above in zip(BORDERS, TO_EVEN_ABOVE):
            code += (a >= border) if above else (a > border)
        values = LEVELS[code] * np.where(np.signbit(t), -1, 1) * d[:, :, None]
        values = f32(values)
    code |= np.signbit(t).astype(np.int64) << 3
    n, c, h, w = x.shape
    return code.reshape(n, -1, h, w)[:, :c], s, values.reshape(n, -1, h, w)[:, :c]


def inputs(rng, shape, zeros=True):
    """Values over a wide range of magnitudes from channel to channel, with blocks of zeros and exact ties."""
    x = rng.normal(0, 1, shape) * np.exp(rng.normal(0, 2, (1, shape[1], 1, 1)))
    x = np.where(rng.random(shape) < 0.2, np.round(x * 4) / 4, x)
    if zeros:
        x[:, :: 3] *= rng.random((shape[0], len(range(0, shape[1], 3)), shape[2], shape[3])) < 0.5
        x[0, : 32] = 0
    return x.astype(np.float32)


SHAPES = [(1, 1, 1, 1), (1, 4096, 1, 1), (3, 16, 5, 7), (2, 33, 9, 11), (5, 64, 1, 3), (1, 129, 13, 13), (2, 333, 7, 5), (130, 40, 1, 1), (1, 31, 40, 33), (2, 255, 19, 19),
          (131, 333, 1, 1), (37, 1111, 1, 1), (257, 96, 1, 1), (3, 17, 1, 1), (33, 16, 1, 1)]


@pytest.mark.parametrize("dtype", FMT)
@pytest.mark.parametrize("source", ["f32", "f16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_narrow_and_widen(be, shape, source, dtype):
    rng = np.random.default_rng(sum(shape) + dtype)
    x = inputs(rng, shape)
    if source == "f16":
        x = np.clip(x, -6e4, 6e4).astype(np.float16).astype(np.float32)
    for g in ([1.0] if dtype == ln.LN_MX4 else [float(np.float32(max(np.abs(x).max(), 1e-3) / 2688)), 0.25, float(np.float32(0.0371))]):
        t = be.upload_f16(shape, x) if source == "f16" else be.upload_f32(shape, x)
        q = be.narrow_f4(t, g, dtype)
        assert q.dtype == dtype and q.shape == shape and q.scale == np.float32(g)
        codes, scales = be.download_f4(q)
        want_codes, want_scales, values = narrow(x, dtype, g)
        assert np.array_equal(scales, want_scales)
        assert np.array_equal(codes & 7, want_codes & 7)
        assert np.array_equal(codes[(codes & 7) != 0] >> 3, want_codes[(codes & 7) != 0] >> 3)
        wide = be.widen_f4(q)
        assert np.array_equal(be.download_f32(wide), values.astype(np.float32))
        with np.errstate(over="ignore"):
            assert np.array_equal(be.download_f16(be.widen_f4(q, ln.LN_F16)), values.astype(np.float32).astype(np.float16).astype(np.float32))
        again = be.download_f4(be.narrow_f4(wide, g, dtype))  # (values that 4 bits hold come back as they are; a block's scale may be another)
        assert np.array_equal(narrow(values, dtype, g)[1], again[1])


@pytest.mark.parametrize("dtype", FMT)
@pytest.mark.parametrize("source", ["f32", "f16"])
def test_values_at_the_ends(be, dtype, source):
    """NaN, infinities, the largest and smallest values, negative zero: one block each, neighbours untouched."""
    b = BLOCK[dtype]
    rng = np.random.default_rng(5)
    x = rng.normal(0, 1, (1, 12 * b, 1, 1)).astype(np.float32)
    big = 65504.0 if source == "f16" else 3e38
    tiny = 6e-8 if source == "f16" else 1e-45
    x[0, 1 * b] = np.nan
    x[0, 3 * b + 2] = np.inf
    x[0, 5 * b + 1] = -np.inf
    x[0, 5 * b + 2] = np.nan
    x[0, 7 * b] = big
    x[0, 8 * b:9 * b] = tiny
    x[0, 9 * b:10 * b] = -0.0
    x[0, 10 * b: 11 * b] = -big
    t = be.upload_f16(x.shape, x) if source == "f16" else be.upload_f32(x.shape, x)
    x = be.download_f16(t) if source == "f16" else x
    for g in [1.0] if dtype == ln.LN_MX4 else [1.0, 2.0 ** -100, 2.0 ** 100, 1e-4]:
        q = be.narrow_f4(t, g, dtype)
        codes, scales = be.download_f4(q)
        want_codes, want_scales, values = narrow(x, dtype, g)
        assert np.array_equal(scales, want_scales)
        assert scales[0, 1, 0, 0] == scales[0, 5, 0, 0] == (0x7F if dtype == ln.LN_F4 else 0xFF)
        fine = np.repeat(scales.reshape(-1) != (0x7F if dtype == ln.LN_F4 else 0xFF), b).reshape(x.shape)
        assert np.array_equal((codes & 7)[fine], (want_codes & 7)[fine])
        wide = be.download_f32(be.widen_f4(q))
        assert np.array_equal(np.isnan(wide), ~fine)
        with np.errstate(over="ignore"):
            assert np.array_equal(wide[fine], values.astype(np.float32)[fine])


def act64(v, act):
    if act == "leaky":
        return np.maximum(v, 0.1 * v)
    if act == "relu":
        return np.maximum(v, 0)
    if act == "logistic":
        return 1 / (1 + np.exp(-v))
    if act == "swish":
        return v / (1 + np.exp(-v))
    if act == "mish":
        return v * np.tanh(np.logaddexp(v, 0))
    return v


def conv64(x, w, k, sx, sy, pad):
    n, c, h, wd = x.shape
    f = w.shape[0]
    oh, ow = max(h + 2 * pad - k, 0) // sy + 1, max(wd + 2 * pad - k, 0) // sx + 1
    full = np.zeros((n, c, max(h + 2 * pad, sy * (oh - 1) + k), max(wd + 2 * pad, sx * (ow - 1) + k)))
    full[:, :, pad:pad + h, pad:pad + wd] = x
    y = np.zeros((n, f, oh, ow))
    for r in range(k):
        for s in range(k):
            y += np.einsum("nchw,fc->nfhw", full[:, :, r:r + sy * (oh - 1) + 1:sy, s:s + sx * (ow - 1) + 1:sx], w[:, :, r, s], optimize=True)
    return y


# n, c, h, w, f, k, sx, sy, pad
CONV = [
    (1, 64, 1, 1, 64, 1, 1, 1, 0), (1, 4096, 1, 1, 512, 1, 1, 1, 0), (7, 1111, 1, 1, 777, 1, 1, 1, 0), (13, 100, 1, 1, 8, 1, 1, 1, 0), (129, 320, 1, 1, 200, 1, 1, 1, 0),
    (300, 1024, 1, 1, 1000, 1, 1, 1, 0), (1, 1, 1, 1, 1, 1, 1, 1, 0), (2, 17, 5, 9, 33, 1, 1, 1, 0), (1, 512, 19, 19, 255, 1, 1, 1, 0), (3, 64, 20, 13, 96, 3, 1, 1, 1),
    (1, 256, 13, 13, 512, 3, 1, 1, 1), (2, 128, 26, 30, 72, 3, 2, 2, 1), (2, 40, 15, 17, 40, 3, 2, 2, 1), (1, 96, 38, 38, 64, 3, 1, 1, 1), (2, 192, 9, 9, 320, 3, 1, 1, 1),
    (1, 33, 8, 9, 70, 5, 1, 1, 2), (1, 70, 11, 12, 50, 3, 1, 2, 1), (2, 48, 7, 7, 24, 3, 3, 3, 0), (1, 64, 3, 3, 64, 5, 1, 1, 0), (1, 48, 2, 2, 16, 3, 2, 2, 0),
    (8, 192, 1, 1, 40, 1, 1, 1, 0), (9, 4160, 1, 1, 100, 1, 1, 1, 0), (16, 320, 1, 1, 130, 1, 1, 1, 0), (17, 320, 1, 1, 130, 1, 1, 1, 0), (1, 96, 3, 5, 33, 1, 1, 1, 0), (2, 70, 2, 3, 65, 1, 1, 1, 0),
    (150, 64, 1, 1, 24, 1, 1, 1, 0), (131, 80, 1, 1, 40, 1, 1, 1, 0), (260, 64, 1, 1, 257, 1, 1, 1, 0), (4, 64, 1, 130, 130, 1, 2, 2, 0), (2, 80, 6, 10, 48, 2, 2, 2, 0), (1, 128, 30, 30, 128, 1, 2, 2, 0),
]


def run_conv(be, case, dtype, act, out_kind, seed=0, y_scale=1.0, reference=True):
    n, c, h, w, f, k, sx, sy, pad = case
    rng = np.random.default_rng(sum(case) + seed)
    x = inputs(rng, (n, c, h, w)) / 4
    wt = (rng.normal(0, np.sqrt(2.0 / (c * k * k)), (f, c, k, k)) * np.exp(rng.normal(0, 1, (f, 1, 1, 1)))).astype(np.float32)
    if f > 2:
        wt[1] = 0
    bias = rng.normal(0, 0.5, f).astype(np.float32)
    g = 1.0 if dtype == ln.LN_MX4 else float(np.float32(np.abs(x).max() / 2688 + 1e-6))
    gw = np.ones(f) if dtype == ln.LN_MX4 else np.where(np.abs(wt).max((1, 2, 3)) > 0, f32(np.abs(wt).max((1, 2, 3)).astype(np.float64) / 2688), 1.0)
    oh, ow = max(h + 2 * pad - k, 0) // sy + 1, max(w + 2 * pad - k, 0) // sx + 1
    q = be.narrow_f4(be.upload_f32(x.shape, x), g, dtype)
    packed = be.conv_weights_f4(be.upload_f32(wt.shape, wt), f, c, k, dtype)
    y = be.conv2d_bias_act_f4(q, packed, be.upload_f32((1, f, 1, 1), bias), (n, f, oh, ow), c, h, w, f, k, sx, sy, 1, pad, 1, act, y_scale, out_kind)
    if not reference:
        return y, None, None
    xv, wv = narrow(x, dtype, g)[2], narrow(wt, dtype, gw)[2]
    v = conv64(xv, wv, k, sx, sy, pad) + bias.astype(np.float64).reshape(1, f, 1, 1)
    size = conv64(np.abs(xv), np.abs(wv), k, sx, sy, pad) + np.abs(bias).reshape(1, f, 1, 1)
    ref = act64(v, act)
    bound = 1.1 * (c * k * k / 64 + 8) * 2.0 ** -23 * size + 16 * 2.0 ** -23 * np.abs(ref) + 1e-7
    return y, ref, bound


@pytest.mark.parametrize("dtype", FMT)
@pytest.mark.parametrize("case", CONV)
def test_convolution(be, case, dtype):
    for i, act in enumerate(["linear", "mish"]):
        y, ref, bound = run_conv(be, case, dtype, act, ln.LN_OUT_F32, i)
        got = be.download_f32(y)
        assert got.shape == ref.shape
        worst = np.max(np.abs(got - ref) / bound)
        assert worst <= 1, worst
    y, ref, bound = run_conv(be, case, dtype, "swish", ln.LN_OUT_F16)
    got = be.download_f16(y)
    assert np.array_equal(got, got.astype(np.float16).astype(np.float32))
    assert np.max(np.abs(got - ref) / (bound + 2.0 ** -11 * np.abs(ref) + 2.0 ** -25)) <= 1


@pytest.mark.parametrize("dtype", FMT)
@pytest.mark.parametrize("case", CONV)
def test_convolution_hands_4_bits_on(be, case, dtype):
    """The requantised output is the narrowed f32 output of the same convolution, code for code."""
    for act, ys in (("leaky", 0.003), ("logistic", 0.0004)):
        ys = 1.0 if dtype == ln.LN_MX4 else float(np.float32(ys))
        q, ref, _ = run_conv(be, case, dtype, act, ln.LN_OUT_Q, y_scale=ys)
        y, _, _ = run_conv(be, case, dtype, act, ln.LN_OUT_F32)
        assert q.dtype == dtype and q.scale == np.float32(ys)
        codes, scales = be.download_f4(q)
        want_codes, want_scales, values = narrow(be.download_f32(y), dtype, ys)
        assert np.array_equal(scales, want_scales)
        assert np.array_equal(codes & 7, want_codes & 7)
        assert np.array_equal(be.download_f32(be.widen_f4(q)), values.astype(np.float32))


@pytest.mark.parametrize("act", sorted(ln.ACTIVATIONS))
@pytest.mark.parametrize("exact", [False, True])
def test_activations(be, act, exact):
    be.set_exact_epilogue(exact)
    try:
        y, ref, bound = run_conv(be, (2, 64, 12, 12, 64, 3, 1, 1, 1), ln.LN_F4, act, ln.LN_OUT_F32)
        assert np.max(np.abs(be.download_f32(y) - ref) / bound) <= 1
    finally:
        be.set_exact_epilogue(False)


@pytest.mark.parametrize("dtype", FMT)
def test_nan_and_infinity_in_a_product(be, dtype):
    """A NaN in one pixel reaches the outputs whose taps read its block, and no other; an infinite value saturates (or is infinite)."""
    n, c, h, w, f = 1, 64, 9, 9, 64
    rng = np.random.default_rng(3)
    x = rng.normal(0, 1, (n, c, h, w)).astype(np.float32)
    wt = (np.abs(rng.normal(0, 0.1, (f, c, 3, 3))) + 0.01).astype(np.float32)
    bias = np.zeros(f, np.float32)
    x[0, 5, 4, 4] = np.nan
    x[0, 9, 0, 8] = np.inf
    g = 1.0 if dtype == ln.LN_MX4 else float(np.float32(4 / 2688))
    packed = be.conv_weights_f4(be.upload_f32(wt.shape, wt), f, c, 3, dtype)
    q = be.narrow_f4(be.upload_f32(x.shape, x), g, dtype)
    y = be.download_f32(be.conv2d_bias_act_f4(q, packed, be.upload_f32((1, f, 1, 1), bias), (n, f, h, w), c, h, w, f, 3, 1, 1, 1, 1, 1, "linear", 1.0, ln.LN_OUT_F32))
    nan = np.zeros((h, w), bool)
    nan[3:6, 3:6] = True
    assert np.array_equal(np.isnan(y), np.broadcast_to(nan, y.shape))
    near = np.zeros((h, w), bool)
    near[:2, 7:] = True
    if dtype == ln.LN_F4:
        assert np.isfinite(y[:, :, ~nan]).all()
    else:
        assert np.isfinite(y[:, :, ~nan & ~near]).all()


@pytest.mark.parametrize("tile", ["64", "128", "256", "128/64", "256/128", "256/64", "64*2", "128*4"])
@pytest.mark.parametrize("dtype", FMT)
def test_each_tile_of_filters(be, monkeypatch, dtype, tile):
    """Whatever a size would choose: outputs of all kinds, several tiles per SM, a last round in narrower ones, a k range
    split over several CTAs, filters that end inside a tile."""
    monkeypatch.setenv("LN_F4_BN", tile)
    for case in ((1, 512, 19, 19, 255, 1, 1, 1, 0), (131, 80, 1, 1, 40, 1, 1, 1, 0), (300, 1024, 1, 1, 1000, 1, 1, 1, 0), (2, 192, 9, 9, 320, 3, 1, 1, 1), (2, 128, 26, 30, 72, 3, 2, 2, 1),
                 (3, 70, 120, 119, 136, 1, 1, 1, 0), (2, 40, 75, 77, 300, 3, 1, 1, 1),
                 (1, 64, 150, 150, 200, 1, 1, 1, 0), (1, 200, 140, 141, 72, 3, 1, 1, 1), (1, 512, 13, 13, 300, 3, 1, 1, 1), (20, 4096, 1, 1, 264, 1, 1, 1, 0), (40, 2048, 1, 1, 257, 1, 1, 1, 0), (1, 96, 12, 13, 136, 5, 2, 2, 2)):
        y, ref, bound = run_conv(be, case, dtype, "mish", ln.LN_OUT_F32)
        wide = be.download_f32(y)
        assert np.max(np.abs(wide - ref) / bound) <= 1, case
        y, _, _ = run_conv(be, case, dtype, "mish", ln.LN_OUT_F16, reference=False)
        assert np.array_equal(be.download_f16(y), wide.astype(np.float16).astype(np.float32)), case
        ys = 1.0 if dtype == ln.LN_MX4 else 0.25
        q, _, _ = run_conv(be, case, dtype, "mish", ln.LN_OUT_Q, y_scale=ys, reference=False)
        assert np.array_equal(be.download_f32(be.widen_f4(q)), narrow(wide, dtype, ys)[2].astype(np.float32)), case


@pytest.mark.parametrize("case", [(2, 256, 1, 1, 48, 1, 1, 1, 0), (40, 256, 1, 1, 48, 1, 1, 1, 0), (1, 96, 9, 10, 48, 3, 1, 1, 1), (1, 96, 9, 10, 48, 3, 1, 2, 1)])
def test_the_range_of_power_of_two_scales(be, case):
    """LN_MX4 holds values of the whole range of binary32: blocks of very large and very small ones against weights of the other end."""
    n, c, h, w, f, k, sx, sy, pad = case
    rng = np.random.default_rng(sum(case))
    bias = np.zeros(f, np.float32)
    for px, pw in ((127, -40), (120, -120), (-122, 100), (-127, 126)):
        x = np.ldexp(rng.uniform(0.5, 1, (n, c, h, w)) * rng.choice([-1, 1], (n, c, h, w)), px - rng.integers(0, 4, (n, c, h, w))).astype(np.float32)
        wt = np.ldexp(rng.uniform(0.5, 1, (f, c, k, k)) * rng.choice([-1, 1], (f, c, k, k)), pw).astype(np.float32)
        q, packed = be.narrow_f4(be.upload_f32(x.shape, x), 1.0, ln.LN_MX4), be.conv_weights_f4(be.upload_f32(wt.shape, wt), f, c, k, ln.LN_MX4)
        oh, ow = (h + 2 * pad - k) // sy + 1, (w + 2 * pad - k) // sx + 1
        got = be.download_f32(be.conv2d_bias_act_f4(q, packed, be.upload_f32((1, f, 1, 1), bias), (n, f, oh, ow), c, h, w, f, k, sx, sy, 1, pad, 1, "linear", 1.0, ln.LN_OUT_F32))
        xv, wv = narrow(x, ln.LN_MX4, 1.0)[2], narrow(wt, ln.LN_MX4, np.ones(f))[2]
        ref, size = conv64(xv, wv, k, sx, sy, pad), conv64(np.abs(xv), np.abs(wv), k, sx, sy, pad)
        assert np.max(np.abs(got - ref) / (1.1 * (c * k * k / 64 + 8) * 2.0 ** -23 * size)) <= 1, (px, pw)


def test_more_tiles_than_any_network(be):
    """2^26 pixels and more: indexes of tiles, codes and scales at that size."""
    h, w, s = 8192, 8200, 64
    rng = np.random.default_rng(8)
    for dtype in FMT:
        x = rng.integers(-6, 7, (1, 1, h, w)).astype(np.float32)
        g = 1.0
        q = be.narrow_f4(be.upload_f32(x.shape, x), g, dtype)
        one, three = np.full((1, 1, 1, 1), 1.5, np.float32), rng.integers(-4, 5, (1, 1, 3, 3)).astype(np.float32)
        gw = 1.0 if dtype == ln.LN_MX4 else f32(np.abs(three).max((1, 2, 3)).astype(np.float64) / 2688)
        value = narrow(x[:, :, -s:], dtype, g)[2]
        assert np.array_equal(be.download_f32(be.widen_f4(q))[:, :, -s:], value)
        again = be.narrow_f4(be.widen_f4(q, ln.LN_F16), g, dtype)
        assert np.array_equal(be.download_f32(be.widen_f4(again))[:, :, -s:], value)
        del again
        b = be.zeros_f32((1, 1, 1, 1))
        y = be.download_f32(be.conv2d_bias_act_f4(q, be.conv_weights_f4(be.upload_f32(one.shape, one), 1, 1, 1, dtype), b, x.shape, 1, h, w, 1, 1, 1, 1, 1, 0, 1, "linear", 1.0, ln.LN_OUT_F32))
        assert np.allclose(y[:, :, -s:], value * 1.5, rtol=2.0 ** -21, atol=0)
        y = be.download_f32(be.conv2d_bias_act_f4(q, be.conv_weights_f4(be.upload_f32(three.shape, three), 1, 1, 3, dtype), b, x.shape, 1, h, w, 1, 3, 1, 1, 1, 1, 1, "linear", 1.0, ln.LN_OUT_F32))
        ref = conv64(value, narrow(three, dtype, gw)[2], 3, 1, 1, 1)[:, :, 1:]
        assert np.max(np.abs(y[:, :, 1 - s:] - ref)) <= 1.1 * 9 * 2.0 ** -23 * 9 * 6 * 4.0


def test_operators_together(be):
    """binary16 map -> 4 bits -> 1x1 -> 4 bits -> 3x3 -> binary16, twice on the same handles and again after other work: the same bits."""
    n, c, h, w, f = 2, 128, 20, 20, 64
    rng = np.random.default_rng(11)
    for dtype in FMT:
        g = 1.0 if dtype == ln.LN_MX4 else float(np.float32(4 / 2688))
        x = rng.normal(0, 1, (n, c, h, w)).astype(np.float32)
        w1 = rng.normal(0, np.sqrt(2 / c), (f, c, 1, 1)).astype(np.float32)
        w2 = rng.normal(0, np.sqrt(2 / (9 * f)), (2 * f, f, 3, 3)).astype(np.float32)
        t = be.upload_f16(x.shape, x)
        p1, p2 = be.conv_weights_f4(be.upload_f32(w1.shape, w1), f, c, 1, dtype), be.conv_weights_f4(be.upload_f32(w2.shape, w2), 2 * f, f, 3, dtype)
        b1, b2 = be.zeros_f32((1, f, 1, 1)), be.zeros_f32((1, 2 * f, 1, 1))

        def chain():
            y = be.conv2d_bias_act_f4(be.narrow_f4(t, g, dtype), p1, b1, (n, f, h, w), c, h, w, f, 1, 1, 1, 1, 0, 1, "leaky", g, ln.LN_OUT_Q)
            return y, be.conv2d_bias_act_f4(y, p2, b2, (n, 2 * f, h, w), f, h, w, 2 * f, 3, 1, 1, 1, 1, 1, "mish", 1.0, ln.LN_OUT_F16)

        runs = [chain() for _ in range(3)]
        got = [be.download_f16(r[1]) for r in runs]
        assert np.array_equal(got[0], got[1]) and np.array_equal(got[0], got[2])
        mid = be.download_f32(be.widen_f4(runs[0][0])).astype(np.float64)
        gw2 = 1.0 if dtype == ln.LN_MX4 else f32(np.abs(w2).max((1, 2, 3)).astype(np.float64) / 2688)
        wv = narrow(w2, dtype, gw2)[2]
        ref, size = act64(conv64(mid, wv, 3, 1, 1, 1), "mish"), conv64(np.abs(mid), np.abs(wv), 3, 1, 1, 1)
        assert np.max(np.abs(got[0] - ref) / (1.1 * (9 * f / 64 + 8) * 2.0 ** -23 * size + (2.0 ** -11 + 2.0 ** -19) * np.abs(ref) + 2e-7)) <= 1


def test_images_do_not_depend_on_the_batch(be):
    """An image has the same values alone and in a batch, to the rounding of the sums, whatever kernel a size leads to."""
    rng = np.random.default_rng(21)
    for dtype, (c, h, w, f, k) in ((ln.LN_F4, (96, 9, 11, 80, 3)), (ln.LN_MX4, (256, 13, 13, 64, 1)), (ln.LN_F4, (2048, 1, 1, 300, 1))):
        x = rng.normal(0, 1, (40, c, h, w)).astype(np.float32)
        wt = rng.normal(0, 0.05, (f, c, k, k)).astype(np.float32)
        g = 1.0 if dtype == ln.LN_MX4 else float(np.float32(5 / 2688))
        packed, bias = be.conv_weights_f4(be.upload_f32(wt.shape, wt), f, c, k, dtype), be.zeros_f32((1, f, 1, 1))

        def product(part):
            q = be.narrow_f4(be.upload_f32(part.shape, part), g, dtype)
            return be.download_f32(be.conv2d_bias_act_f4(q, packed, bias, (len(part), f, h, w), c, h, w, f, k, 1, 1, 1, k // 2, 1, "linear", 1.0, ln.LN_OUT_F32))

        whole = product(x)
        for lo, hi in ((0, 1), (39, 40), (3, 12), (0, 20)):
            assert np.allclose(product(x[lo:hi]), whole[lo:hi], rtol=0, atol=2.0 ** -20 * np.abs(whole).max())


def test_captured_and_replayed(be):
    """The operators on the backend's stream inside a captured graph: replays see what the input holds then."""
    torch = pytest.importorskip("torch")
    n, c, h, w, f = 2, 96, 14, 14, 72
    rng = np.random.default_rng(31)
    stream = torch.cuda.ExternalStream(be.stream)
    for dtype in FMT:
        g = 1.0 if dtype == ln.LN_MX4 else float(np.float32(5 / 2688))
        x = [rng.normal(0, 1, (n, c, h, w)).astype(np.float32) for _ in range(3)]
        w1, w2 = rng.normal(0, 0.1, (f, c, 1, 1)).astype(np.float32), rng.normal(0, 0.05, (f, f, 3, 3)).astype(np.float32)
        t = be.upload_f32(x[0].shape, x[0])
        p1, p2, b = be.conv_weights_f4(be.upload_f32(w1.shape, w1), f, c, 1, dtype), be.conv_weights_f4(be.upload_f32(w2.shape, w2), f, f, 3, dtype), be.zeros_f32((1, f, 1, 1))

        def chain():
            q = be.narrow_f4(t, g, dtype)
            y = be.conv2d_bias_act_f4(q, p1, b, (n, f, h, w), c, h, w, f, 1, 1, 1, 1, 0, 1, "leaky", g, ln.LN_OUT_Q)
            z = be.conv2d_bias_act_f4(y, p2, b, (n, f, h, w), f, h, w, f, 3, 1, 1, 1, 1, 1, "mish", g, ln.LN_OUT_Q)
            return q, y, z, be.widen_f4(z)

        want = []
        for v in x:
            t_view = torch.as_tensor(t, device="cuda")
            be.sync()
            t_view.copy_(torch.from_numpy(v))
            torch.cuda.synchronize()
            want.append(be.download_f32(chain()[3]))
        be.sync()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            kept = chain()  # (its memory comes from what the chains above gave back)
        for i in (1, 2, 0):
            t_view.copy_(torch.from_numpy(x[i]))
            torch.cuda.synchronize()
            with torch.cuda.stream(stream):
                graph.replay()
                graph.replay()
            assert np.array_equal(be.download_f32(kept[3]), want[i])
        be.sync()
        del graph


def test_two_backends_at_once():
    """Two threads, a context each: the same bits as one after the other."""
    import threading
    rng = np.random.default_rng(41)
    n, c, h, w, f = 3, 128, 26, 26, 160
    x = [rng.normal(0, 1, (n, c, h, w)).astype(np.float32) for _ in range(2)]
    wt = rng.normal(0, 0.05, (f, c, 3, 3)).astype(np.float32)
    bes = [ln.B200Backend(0) for _ in range(2)]
    try:
        def work(i, rounds):
            be, out = bes[i], []
            packed, b = be.conv_weights_f4(be.upload_f32(wt.shape, wt), f, c, 3, FMT[i]), be.zeros_f32((1, f, 1, 1))
            for _ in range(rounds):
                q = be.narrow_f4(be.upload_f32(x[i].shape, x[i]), 1.0, FMT[i])
                out.append(be.download_f32(be.conv2d_bias_act_f4(q, packed, b, (n, f, h, w), c, h, w, f, 3, 1, 1, 1, 1, 1, "swish", 1.0, ln.LN_OUT_F32)))
            return out

        alone = [work(i, 1)[0] for i in range(2)]
        got = [None, None]

        def run(i):
            got[i] = work(i, 20)

        threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        for i in range(2):
            assert got[i] is not None and all(np.array_equal(y, alone[i]) for y in got[i])
    finally:
        for b in bes:
            b.close()


def test_array_interface_shares_the_memory(be):
    torch = pytest.importorskip("torch")
    x = np.random.default_rng(1).normal(0, 1, (2, 37, 3, 5)).astype(np.float32)
    t, u = be.upload_f32(x.shape, x), be.upload_f16(x.shape, x)
    be.sync()
    a, b = torch.as_tensor(t, device="cuda"), torch.as_tensor(u, device="cuda")
    assert a.dtype == torch.float32 and np.array_equal(a.cpu().numpy(), x)
    assert b.dtype == torch.float16 and np.array_equal(b.cpu().numpy(), x.astype(np.float16))
    del t, u
    be.zeros_f32(x.shape)
    be.sync()
    assert np.array_equal(a.cpu().numpy(), x)
    q = be.narrow_f4(be.upload_f32(x.shape, x), 0.01)
    assert not hasattr(q, "__cuda_array_interface__")
    p, shape, s = C.c_void_p(), (C.c_int64 * 4)(), (C.c_int64 * 4)()
    assert be.lib.ln_tensor_device_data(q.h, C.byref(p), shape, s) == 5


def refused(kind, fn, *args):
    with pytest.raises(ln.BackendError) as e:
        fn(*args)
    assert e.value.kind == kind, str(e.value)


def test_refusals(be):
    x = np.ones((1, 32, 4, 4), np.float32)
    t = be.upload_f32(x.shape, x)
    q, m = be.narrow_f4(t, 0.01), be.narrow_f4(t, 1.0, ln.LN_MX4)
    for bad in (0.0, -1.0, float("nan"), float("inf"), 1e-35, 1e35):
        refused("argument", be.narrow_f4, t, bad)
        refused("argument", be.narrow_f4, t, bad, ln.LN_MX4)
    refused("argument", be.narrow_f4, t, 0.5, ln.LN_MX4)
    refused("argument", be.narrow_f4, t, 1.0, ln.LN_Q8)
    refused("argument", be.narrow_f4, q, 1.0)
    refused("argument", be.widen_f4, t)
    refused("argument", be.widen_f4, q, ln.LN_Q8)
    refused("argument", be.widen_q, q)
    refused("argument", be.widen_f16, q)
    refused("argument", be.download_f32, q)
    refused("argument", be.download_f4, t)
    wt = be.upload_f32((8, 32, 3, 3), np.ones((8, 32, 3, 3), np.float32))
    refused("shape", be.conv_weights_f4, wt, 8, 32, 1)
    refused("shape", be.conv_weights_f4, wt, 0, 32, 3)
    refused("unsupported", be.conv_weights_f4, wt, 1, 1 << 24, 64)
    refused("argument", be.conv_weights_f4, wt, 8, 32, 3, ln.LN_F8)
    refused("argument", be.conv_weights_f4, q, 8, 32, 3)
    w, wm = be.conv_weights_f4(wt, 8, 32, 3), be.conv_weights_f4(wt, 8, 32, 3, ln.LN_MX4)
    b = be.zeros_f32((1, 8, 1, 1))

    def conv(x=q, w=w, b=b, shape=(1, 8, 4, 4), c=32, h=4, wd=4, f=8, k=3, sx=1, sy=1, dil=1, pad=1, groups=1, act="linear", ys=0.01, out=ln.LN_OUT_Q):
        return be.conv2d_bias_act_f4(x, w, b, shape, c, h, wd, f, k, sx, sy, dil, pad, groups, act, ys, out)

    conv()
    conv(x=m, w=wm, ys=1.0)
    refused("argument", lambda: conv(x=t))
    refused("argument", lambda: conv(w=wm))
    refused("argument", lambda: conv(x=m, w=wm, ys=0.5))
    refused("argument", lambda: conv(ys=0.0))
    refused("argument", lambda: conv(out=ln.LN_OUT_ACC))
    refused("argument", lambda: conv(out=7))
    refused("unsupported", lambda: conv(groups=2))
    refused("unsupported", lambda: conv(dil=2))
    refused("unsupported", lambda: conv(act=17))
    refused("shape", lambda: conv(shape=(1, 8, 4, 5)))
    refused("shape", lambda: conv(c=16))
    refused("shape", lambda: conv(sx=0))
    refused("shape", lambda: conv(pad=-1))
    refused("shape", lambda: conv(b=be.zeros_f32((1, 9, 1, 1))))
    other = ln.B200Backend(0)
    try:
        refused("argument", other.narrow_f4, t, 1.0)
        refused("argument", other.widen_f4, q)
        refused("argument", lambda: conv(b=other.zeros_f32((1, 8, 1, 1))))
    finally:
        other.close()
    refused("argument", ln.GpuExecutableNetwork, be, "[net]\nwidth=32\nheight=32\nchannels=3\n[convolutional]\nfilters=8\nsize=1\nstride=1\nactivation=linear\n", 1, ln.LN_F4)
    refused("unsupported", be.narrow_f4, be.zeros_f32((1, (1 << 30) + 1, 1, 1)), 1.0)
    # a failed allocation is an error of the call, and the next one works
    be.debug_fail_alloc(1)
    refused("cuda", be.narrow_f4, t, 0.01)
    be.debug_fail_alloc(1)
    refused("cuda", conv)
    conv()
