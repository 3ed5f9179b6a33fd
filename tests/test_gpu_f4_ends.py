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


# shapes [n, c, h, w], kernel and strides that lead to each kernel of the product: up to 16 pixels, tensor cores (flat and under taps, with the k range
# split over a cluster), every other geometry
KERNELS = {"few": (3, 64, 1, 1, 1, 1, 1), "flat": (150, 64, 1, 1, 1, 1, 1), "taps": (1, 64, 9, 10, 3, 1, 1), "split": (20, 8192, 1, 1, 1, 1, 1), "any": (1, 64, 6, 7, 3, 1, 2)}
FAR = [-1e30, -3e38, -1e10, -1000.0, -180.0, -175.0, -174.0, -130.0, -104.0, -103.0, -100.0, -95.0, -90.0, -88.0, -87.5, -87.0, -86.5, -80.0, -61.0, -60.0, -59.5, -30.0,
       -1.0, -0.0, 0.5, 3.0, 25.0, 100.0, 1e10, 1e30, 3e38, -np.inf, np.inf]


def act64(v, act):
    with np.errstate(all="ignore"):
        if act == "linear":
            return v
        if act == "leaky":
            return np.maximum(v, f32(0.1) * v)
        if act == "relu":
            return np.maximum(v, 0)
        if act == "logistic":
            return 1 / (1 + np.exp(-v))
        limit = np.where(np.isposinf(v), np.inf, -0.0)
        got = v / (1 + np.exp(-v)) if act == "swish" else v * np.tanh(np.logaddexp(v, 0))
        return np.where(np.isinf(v), limit, got)


def product_of(be, kernel, dtype, act, bias, x=None, out=ln.LN_OUT_F32, wt=None):
    """A product with given biases: of zeros where there is no x, so that what goes into the activation is the bias itself."""
    n, c, h, w, k, sx, sy = KERNELS[kernel]
    f, pad = len(bias), k // 2
    oh, ow = (h + 2 * pad - k) // sy + 1, (w + 2 * pad - k) // sx + 1
    x = np.zeros((n, c, h, w), np.float32) if x is None else x
    wt = np.full((f, c, k, k), 0.01, np.float32) if wt is None else wt
    q, packed = be.narrow_f4(be.upload_f32(x.shape, x), 1.0, dtype), be.conv_weights_f4(be.upload_f32(wt.shape, wt), f, c, k, dtype)
    b = be.upload_f32((1, f, 1, 1), np.asarray(bias, np.float32))
    return be.conv2d_bias_act_f4(q, packed, b, (n, f, oh, ow), c, h, w, f, k, sx, sy, 1, pad, 1, act, 1.0, out)


@pytest.mark.parametrize("exact", [False, True])
@pytest.mark.parametrize("act", sorted(ln.ACTIVATIONS))
@pytest.mark.parametrize("kernel", sorted(KERNELS))
def test_activations_of_the_whole_range(be, kernel, act, exact):
    """Against 64 bits, relative to the value.  The fast exponentials take their argument times log2(e) in binary32: off by up to |v| half steps of 1.45,
    to -60 (for mish to -87); a few operations more; what is below 2^-126 is off by half a step of 2^-149 times v and up to e^20 more for the ratio of mish."""
    be.set_exact_epilogue(exact)
    try:
        v = np.asarray(FAR, np.float32).astype(np.float64)
        want = act64(v, act)
        for dtype in FMT:
            got = be.download_f32(product_of(be, kernel, dtype, act, FAR)).astype(np.float64)
            half = be.download_f16(product_of(be, kernel, dtype, act, FAR, out=ln.LN_OUT_F16)).astype(np.float64)
            for i, (a, r) in enumerate(zip(v, want)):
                with np.errstate(over="ignore"):
                    r16 = float(np.float16(r))
                if not np.isfinite(np.float32(r)):
                    assert np.array_equal(got[:, i], np.full_like(got[:, i], r)) and np.array_equal(half[:, i], np.full_like(half[:, i], r)), a
                    continue
                off = (min(abs(a), 87.0) + 16) * 2.0 ** -23 * abs(r) + 2.0 ** -149 * min(max(abs(a), 2), 200)
                assert np.max(np.abs(got[:, i] - r)) <= off, (dtype, a, r, got[0, i].ravel()[0])
                if np.isinf(r16):
                    assert np.array_equal(half[:, i], np.full_like(half[:, i], r16)), a
                else:
                    assert np.max(np.abs(half[:, i] - r)) <= off + 2.0 ** -11 * abs(r) + 2.0 ** -25, (dtype, a)
    finally:
        be.set_exact_epilogue(False)


@pytest.mark.parametrize("exact", [False, True])
@pytest.mark.parametrize("act", sorted(ln.ACTIVATIONS))
@pytest.mark.parametrize("kernel", sorted(KERNELS))
def test_nan_behind_every_activation(be, kernel, act, exact):
    """A NaN bias makes its filter's outputs NaN, a NaN in a pixel those of the pixels that its block reaches, and no others; a block handed on in 4 bits is NaN."""
    n, c, h, w, k, sx, sy = KERNELS[kernel]
    f, pad = 70, k // 2
    rng = np.random.default_rng(5)
    bias = rng.normal(0, 1, f).astype(np.float32)
    bias[3] = np.nan
    x = np.abs(rng.normal(0, 1, (n, c, h, w))).astype(np.float32)
    x[n // 2, 5, h // 2, w // 2] = np.nan
    hit = np.zeros((n, h + 2 * pad, w + 2 * pad), bool)
    hit[n // 2, h // 2 + pad, w // 2 + pad] = True
    oh, ow = (h + 2 * pad - k) // sy + 1, (w + 2 * pad - k) // sx + 1
    nan = np.zeros((n, f, oh, ow), bool)
    for r in range(k):
        for s in range(k):
            nan |= hit[:, None, r:r + sy * (oh - 1) + 1:sy, s:s + sx * (ow - 1) + 1:sx]
    nan[:, 3] = True
    be.set_exact_epilogue(exact)
    try:
        for dtype in FMT:
            for out, read in ((ln.LN_OUT_F32, be.download_f32), (ln.LN_OUT_F16, be.download_f16)):
                got = read(product_of(be, kernel, dtype, act, bias, x, out))
                assert np.array_equal(np.isnan(got), nan), (dtype, out)
            scales = be.download_f4(product_of(be, kernel, dtype, act, bias, x, ln.LN_OUT_Q))[1]
            size, none = BLOCK[dtype], 0x7F if dtype == ln.LN_F4 else 0xFF
            padded = np.zeros((n, -(-f // size) * size, oh, ow), bool)
            padded[:, :f] = nan
            assert np.array_equal(scales == none, padded.reshape(n, -1, size, oh, ow).any(2)), dtype
    finally:
        be.set_exact_epilogue(False)


@pytest.mark.parametrize("kernel", sorted(KERNELS))
def test_nan_and_infinity_among_the_weights(be, kernel):
    """A filter with a NaN has no other outputs than NaN, also where the tap that holds it lies outside the image, over an image of zeros, and in every
    kernel; an infinite weight saturates and makes none; the other filters do not change."""
    n, c, h, w, k, sx, sy = KERNELS[kernel]
    f = 40
    rng = np.random.default_rng(9)
    wt = rng.normal(0, 0.1, (f, c, k, k)).astype(np.float32)
    x = rng.normal(0, 1, (n, c, h, w)).astype(np.float32)
    bad = wt.copy()
    bad[7, 3, 0, 0] = np.nan
    bad[33, c - 1, k - 1, k - 1] = np.nan
    bad[12, 40, 0, 0] = np.inf
    rest = [i for i in range(f) if i not in (7, 33, 12)]
    for dtype in FMT:
        want = be.download_f32(product_of(be, kernel, dtype, "linear", np.ones(f), x, wt=wt))
        for data in (x, np.zeros_like(x)):
            got = be.download_f32(product_of(be, kernel, dtype, "linear", np.ones(f), data, wt=bad))
            assert np.isnan(got[:, [7, 33]]).all()
            assert not np.isnan(got[:, rest + [12]]).any()
        assert (got[:, rest + [12]] == 1).all()
        got = be.download_f32(product_of(be, kernel, dtype, "linear", np.ones(f), x, wt=bad))
        assert np.array_equal(got[:, rest], want[:, rest])


@pytest.mark.parametrize("kernel", sorted(KERNELS))
def test_a_replay_writes_no_memory_but_its_tensors(kernel):
    """A captured product that hands 4 bits on: with its tensors kept, a replay leaves what later calls put elsewhere."""
    torch = pytest.importorskip("torch")
    be = ln.B200Backend(0)
    n, c, h, w, k, sx, sy = KERNELS[kernel]
    f, pad = 70, k // 2
    oh, ow = (h + 2 * pad - k) // sy + 1, (w + 2 * pad - k) // sx + 1
    rng = np.random.default_rng(3)
    try:
        for dtype in FMT:
            wt = rng.normal(0, 0.1, (f, c, k, k)).astype(np.float32)
            x, packed, b = be.upload_f32((n, c, h, w), rng.normal(0, 1, (n, c, h, w))), be.conv_weights_f4(be.upload_f32(wt.shape, wt), f, c, k, dtype), be.zeros_f32((1, f, 1, 1))

            def call():
                q = be.narrow_f4(x, 1.0, dtype)
                return q, be.conv2d_bias_act_f4(q, packed, b, (n, f, oh, ow), c, h, w, f, k, sx, sy, 1, pad, 1, "mish", 1.0, ln.LN_OUT_Q)

            want = be.download_f4(call()[1])
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=torch.cuda.ExternalStream(be.stream)):
                kept = call()
            others, value = [], np.full((n, f, oh, ow), 7.0, np.float32)
            for size in (value, value[:, : f // 4], value[:, : f // 8]):
                others += [be.upload_f32(size.shape, size) for _ in range(4)]
            with torch.cuda.stream(torch.cuda.ExternalStream(be.stream)):
                graph.replay()
            be.sync()
            assert all((be.download_f32(t) == 7).all() for t in others)
            assert all(np.array_equal(a, r) for a, r in zip(be.download_f4(kept[1]), want))
            del graph, kept
    finally:
        be.close()


@pytest.mark.parametrize("tile", ["64", "128", "256", "128/64", "256/128", "256/64", "64*2", "128*4"])
def test_a_forced_tile_runs_where_it_can(be, monkeypatch, tile):
    """Sizes that each form of the tensor-core kernel takes: a cut last round wants more tiles than the 148 SMs and a last round whose units fit into one (76 x 2
    or 51 x 3 tiles: 4 and 5 behind the first round), a split wants few tiles and a long k range.  What ran is asked for: the form in two cases at least, and the
    outputs of the choice by size in all."""
    filters, narrow, parts = int(tile.split("/")[0].split("*")[0]), int(tile.split("/")[1]) if "/" in tile else 0, int(tile.split("*")[1]) if "*" in tile else 1
    rng, taken, rows = np.random.default_rng(2), 0, 76 if filters == 256 else 51
    cases = [(1, 70, 150, 147, 264, 3), (19000, 200, 1, 1, 258, 1), (1, 70, rows, 128, 264, 3), (rows * 128, 200, 1, 1, 264, 1)]
    for n, c, h, w, f, k in [(1, 320, 31, 33, 264, 3), (40, 2112, 1, 1, 257, 1)] if parts > 1 else cases:
        x, wt = rng.normal(0, 1, (n, c, h, w)).astype(np.float32), rng.normal(0, 0.05, (f, c, k, k)).astype(np.float32)
        for dtype in FMT:
            q, packed, b = be.narrow_f4(be.upload_f32(x.shape, x), 1.0, dtype), be.conv_weights_f4(be.upload_f32(wt.shape, wt), f, c, k, dtype), be.zeros_f32((1, f, 1, 1))

            def call():
                return be.download_f32(be.conv2d_bias_act_f4(q, packed, b, (n, f, h, w), c, h, w, f, k, 1, 1, 1, k // 2, 1, "linear", 1.0, ln.LN_OUT_F32))

            monkeypatch.setenv("LN_F4_BN", tile)
            got, ran = call(), be.debug_f4_plan()
            monkeypatch.delenv("LN_F4_BN")
            want = call()
            taken += ran == (filters, narrow, parts)
            assert np.max(np.abs(got - want)) <= 2.0 ** -20 * np.abs(want).max()
    assert taken >= 2 * len(FMT), taken


def test_which_kernel_a_size_runs_in(be):
    for kernel, tiles in (("few", False), ("any", False), ("flat", True), ("taps", True), ("split", True)):
        product_of(be, kernel, ln.LN_F4, "linear", np.zeros(70))
        filters, _, parts = be.debug_f4_plan()
        assert (filters > 0) == tiles and (parts > 1) == (kernel == "split"), kernel
    assert be.lib.ln_debug_f4_plan(None, None) == 5


@pytest.mark.parametrize("source", ["f32", "f16"])
def test_the_smallest_block_scales(be, source):
    """amax / (6 g) around 2^-10, where the scale becomes 0, and in the middle between two of the smallest scales, where |x / d| is up to 9: one block for each,
    with values of both signs down to nothing beside the largest."""
    at = [0.0, 2.0 ** -12, 0.999 * 2.0 ** -10, 2.0 ** -10, 1.001 * 2.0 ** -10] + [m * 2.0 ** -9 for m in (0.75, 1, 1.49, 1.5, 1.51, 2, 2.49, 2.5, 2.51, 3.5, 6.5, 7.4, 7.5, 7.6, 8.5)]
    x = np.zeros((2, 16 * len(at), 3, 1), np.float32)
    part = np.array([1, -1, 0.97, -0.9, 0.8, -0.7, 0.6, 0.5, -0.4, 0.3, 0.2, -0.1, 0.05, -0.01, 0.0, -0.0])
    for i, q in enumerate(at):
        x[:, 16 * i:16 * i + 16] = (6 * q * part).reshape(1, 16, 1, 1)
    if source == "f16":
        x = (x * 64).astype(np.float16).astype(np.float32)
    scales = same_as_defined(be, x, 64.0 if source == "f16" else 1.0, ln.LN_F4, source)
    assert (scales[:, :3] == 0).all() and (scales[:, 4] == 1).all() and scales.max() == 8
    q = be.narrow_f4(be.upload_f32(x.shape, x), 64.0 if source == "f16" else 1.0)
    codes = be.download_f4(q)[0]
    assert set(np.unique(codes[:, :48])) <= {0, 8}  # zeros of either sign
    assert not np.isnan(be.download_f32(be.widen_f4(q))).any()


@pytest.mark.parametrize("status", [1, 2, 3])
def test_a_wait_given_up_is_reported_once(be, status):
    """The word that such a kernel leaves in host memory: the next product, a download or ln_sync says so, and the context goes on."""
    x = np.random.default_rng(1).normal(0, 1, (1, 64, 9, 9)).astype(np.float32)

    def product():
        return product_of(be, "taps", ln.LN_F4, "leaky", np.ones(40), np.broadcast_to(x[:, :, :, :1], (1, 64, 9, 10)))

    want = be.download_f32(product())
    y, q = product(), be.narrow_f4(be.upload_f32(x.shape, x), 0.01)
    be.sync()
    for call in (product, be.sync, lambda: be.download_f32(y), lambda: be.download_f16(be.widen_f4(q, ln.LN_F16)), lambda: be.download_f4(q)):
        assert be.lib.ln_debug_set_status(be.ctx, status) == 0
        with pytest.raises(ln.BackendError) as e:
            call()
        assert e.value.kind == "timeout" and ("TMA producer", "MMA issuer", "epilogue")[status - 1] in str(e.value)
        call()
        assert np.array_equal(be.download_f32(product()), want)
    assert be.lib.ln_debug_set_status(be.ctx, 4) == be.lib.ln_debug_set_status(None, 0) == 5
