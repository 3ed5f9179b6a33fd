"""Performance cases of the microscaled 4-bit operators: narrowing, widening and the product (a convolution with bias and activation,
whose 1x1 form over [tokens, features, 1, 1] is the plain matrix product).

Two storage types, both with E2M1 elements (0, .5, 1, 1.5, 2, 3, 4, 6 and a sign) and a scale per block of channels:

  f4   blocks of 16 channels with an E4M3 scale s, one binary32 scale g per tensor (per filter for weights): value = code * s * g
       s = e4m3(amax / (6 g)), d = s * g, code = e2m1(x / d), both roundings to nearest even and saturating
  mx4  blocks of 32 channels with a scale 2^e, e = floor(log2(amax)) - 2: value = code * 2^e, code = e2m1(x / 2^e)

The divisions and products that lead to a code are binary32 operations: that is part of the definition, as it is for the 8-bit types.

A case has one of four kinds:

  narrow   a tensor of floating values to 4 bits and, since codes are compared as the values that they stand for, back
  widen    a 4-bit tensor to floating values
  product  a convolution of a 4-bit tensor with 4-bit weights, f32 or binary16 out
  chain    a binary16 map through narrow, a 1x1 convolution that hands 4 bits on (requantised in its epilogue) and a 3x3 one
"""
from __future__ import annotations

import math

import torch

own = False

LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
BLOCK = {"f4": 16, "mx4": 32}
SCALE_BYTES = {"f4": 1 / 16, "mx4": 1 / 32}
OUT_BYTES = {"f32": 4, "f16": 2}
MOST_VALUES = 64 * 128 * 76 * 76       # the largest listed tensor
MOST_FLOPS = 2 * 8192 * 4096 * 4096    # the largest listed product


def listed():
    return [
        # the activations of a single token in front of a product: launches are everything
        dict(name="narrow_token", kind="narrow", fmt="f4", src="f16", dst="f16", batch=1, channels=4096, height=1, width=1),
        # f32 maps of an odd size with a channel count that ends inside a block
        dict(name="narrow_odd_f32", kind="narrow", fmt="mx4", src="f32", dst="f32", batch=4, channels=333, height=45, width=37),
        # the benchmark's batch at the 76 x 76 stage of a detector
        dict(name="narrow_b64", kind="narrow", fmt="f4", src="f16", dst="f16", batch=64, channels=128, height=76, width=76),
        # one image's deepest map, back to f32 for a host that reads it
        dict(name="widen_map", kind="widen", fmt="mx4", dst="f32", batch=1, channels=1024, height=19, width=19),
        # a batch back to binary16 for the operators that have no 4-bit form
        dict(name="widen_b32", kind="widen", fmt="f4", dst="f16", batch=32, channels=256, height=76, width=76),
        # one token through a square projection: the weights are read, nothing else costs
        dict(name="product_token", kind="product", fmt="f4", out="f16", batch=1, channels=4096, height=1, width=1, filters=4096, k=1, stride=1, act="linear"),
        # a few tokens, odd feature counts
        dict(name="product_few_odd", kind="product", fmt="mx4", out="f32", batch=13, channels=1111, height=1, width=1, filters=777, k=1, stride=1, act="swish"),
        # the 3x3 layer of the single-layer sweep
        dict(name="product_3x3", kind="product", fmt="f4", out="f16", batch=16, channels=256, height=38, width=38, filters=512, k=3, stride=1, act="leaky"),
        # a down-sampling layer of the sweep
        dict(name="product_3x3_s2", kind="product", fmt="mx4", out="f16", batch=16, channels=128, height=104, width=104, filters=256, k=3, stride=2, act="mish"),
        # the convolution in front of a detection head: f32 out, 255 filters
        dict(name="product_head", kind="product", fmt="f4", out="f32", batch=16, channels=1024, height=19, width=19, filters=255, k=1, stride=1, act="linear"),
        # a large matrix product: 8192 tokens
        dict(name="product_matrix", kind="product", fmt="f4", out="f16", batch=8192, channels=4096, height=1, width=1, filters=4096, k=1, stride=1, act="swish"),
        # the operators as a detector uses them together
        dict(name="chain_b8", kind="chain", fmt="mx4", batch=8, channels=512, height=52, width=52, filters=256, act="leaky"),
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm."""
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    kind, fmt = rng.choice(["narrow", "widen", "product", "product", "product", "chain"]), rng.choice(["f4", "mx4"])
    floating = ["f16", "f32"]
    if kind in ("narrow", "widen"):
        if rng.random() < 0.4:  # tokens
            n, c, h, w = _spread(rng, 1, 8192), _spread(rng, 16, 8192), 1, 1
        else:
            n, c, h, w = _spread(rng, 1, 64), _spread(rng, 16, 1024), rng.randint(5, 104), rng.randint(5, 104)
        while n * c * h * w > MOST_VALUES:
            n, c = max(1, n // 2), max(16, c * 3 // 4)
        case = dict(kind=kind, fmt=fmt, dst=rng.choice(floating), batch=n, channels=c, height=h, width=w)
        return dict(case, src=rng.choice(floating)) if kind == "narrow" else case
    act = rng.choice(["linear", "leaky", "mish", "swish", "relu", "logistic"])
    if kind == "chain":
        n, c, h, w, f = _spread(rng, 1, 16), 32 * rng.randint(1, 16), rng.randint(7, 76), rng.randint(7, 76), 32 * rng.randint(1, 8)
        while 2 * n * h * w * (c * f + 18 * f * f) > MOST_FLOPS:
            n = max(1, n // 2)
        return dict(kind="chain", fmt=fmt, batch=n, channels=c, height=h, width=w, filters=f, act="leaky" if act == "logistic" else act)
    out = rng.choice(["f32", "f16", "f16"])
    if rng.random() < 0.5:  # tokens
        n, c, f = _spread(rng, 1, 8192), _spread(rng, 32, 8192), _spread(rng, 8, 8192)
        while 2 * n * c * f > MOST_FLOPS or n * f > MOST_VALUES:
            n = max(1, n // 2)
        return dict(kind="product", fmt=fmt, out=out, batch=n, channels=c, height=1, width=1, filters=f, k=1, stride=1, act=act)
    n, c, f = _spread(rng, 1, 32), _spread(rng, 16, 1024), _spread(rng, 8, 1024)
    h, w, k, stride = rng.randint(5, 104), rng.randint(5, 104), rng.choice([1, 3]), rng.choice([1, 1, 2])
    while n > 1 and (2 * n * h * w * c * f * k * k > MOST_FLOPS or n * h * w * max(c, f) > MOST_VALUES):
        n //= 2
    while 2 * n * h * w * c * f * k * k > MOST_FLOPS:
        h, w = max(5, h // 2), max(5, w // 2)
    return dict(kind="product", fmt=fmt, out=out, batch=n, channels=c, height=h, width=w, filters=f, k=k, stride=stride, act=act)


# ---- inputs -------------------------------------------------------------------------------------------------------------------


def _activations(case, g):
    """What a layer hands on: rectified normal values whose deviation differs from channel to channel, some channels ten times the others."""
    n, c, h, w = (case[k] for k in ("batch", "channels", "height", "width"))
    x = torch.randn((n, c, h, w), generator=g, device="cuda")
    gain = torch.exp(0.5 * torch.randn((1, c, 1, 1), generator=g, device="cuda"))
    gain = torch.where(torch.rand((1, c, 1, 1), generator=g, device="cuda") < 0.01, gain * 10, gain)
    return torch.where(x > 0, x, 0.1 * x) * gain


def _weights(f, c, k, g):
    return torch.randn((f, c, k, k), generator=g, device="cuda") * math.sqrt(2.0 / (c * k * k)), 0.1 * torch.randn((f,), generator=g, device="cuda")


def _tensor_scale(fmt, amax):
    """The scale that a calibration run gives a tensor: its largest block scale becomes 448."""
    return float(torch.tensor(amax / (6.0 * 448.0), dtype=torch.float32)) if fmt == "f4" else 1.0


def _inputs(case, seed):
    """Everything that the seed decides, as torch tensors on the GPU: the same for both forms and for exact()."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": case, "x": _activations(case, g)}
    fmt = case["fmt"]
    if case["kind"] == "chain":
        s["x"] = s["x"].half()
        f, c = case["filters"], case["channels"]
        s["w1"], s["b1"] = _weights(f, c, 1, g)
        s["w2"], s["b2"] = _weights(2 * f, f, 3, g)
        s["y_scale"] = _tensor_scale(fmt, 24.0)
    elif case["kind"] == "product":
        s["w"], s["b"] = _weights(case["filters"], case["channels"], case["k"], g)
    elif case["kind"] == "narrow" and case["src"] == "f16":
        s["x"] = s["x"].half()
    s["x_scale"] = _tensor_scale(fmt, float(s["x"].abs().max()))
    return s


# ---- the plain form -------------------------------------------------------------------------------------------------------------


def _pow2(e):
    """2^e in f32, from the bits, for whole e >= -126."""
    return ((e.clamp(min=-126) + 127) << 23).view(torch.float32)


def _plain_codes(t):
    """E2M1 codes, nearest even, saturating: the step is .5 below 2, 1 below 4, then 2; bit 3 is the sign."""
    a = t.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    v = (torch.round(a / step) * step).clamp(max=6.0)
    magnitude = torch.where(v < 2, 2 * v, torch.where(v < 4, v + 2, v / 2 + 4))
    return magnitude.to(torch.uint8) | (torch.signbit(t).to(torch.uint8) << 3)


def _plain_narrow(x, fmt, scale):
    """A tensor whose blocks run along dimension 1, in 4 bits: two codes per byte, and what a code of each block is multiplied by.
    `scale` is a number or one per row of dimension 0."""
    n, c = x.shape[:2]
    rest = x.shape[2:]
    pad = -c % BLOCK[fmt]
    x = x.float()
    if pad:
        x = torch.cat([x, x.new_zeros((n, pad) + rest)], 1)
    x = x.reshape((n, -1, BLOCK[fmt]) + rest)
    amax = x.abs().amax(2, keepdim=True)
    if fmt == "f4":
        scale = torch.as_tensor(scale, dtype=torch.float32, device=x.device)
        scale = scale.reshape((-1,) + (1,) * (x.dim() - 1))
        s = (amax / (6.0 * scale)).clamp(max=448.0)
        s = torch.where(scale > 0, s, torch.zeros_like(s))
        step = _pow2(torch.frexp(s)[1].clamp(min=-5) - 4)  # frexp: s in [2^(e-1), 2^e)
        d = torch.round(s / step) * step * scale
    else:
        d = _pow2(torch.frexp(amax)[1] - 3)
    codes = _plain_codes(torch.where(d > 0, x / d, torch.zeros_like(x))).reshape((n, -1) + rest)
    return codes[:, 0::2] | (codes[:, 1::2] << 4), d


def _plain_widen(four, c):
    """The first c channels of a 4-bit tensor, in f32."""
    packed, d = four
    codes = torch.stack([packed & 15, packed >> 4], 2).reshape((packed.shape[0], d.shape[1], -1) + packed.shape[2:])
    levels = torch.tensor(LEVELS + tuple(-v for v in LEVELS), device=packed.device)
    return (levels[codes.int()] * d).reshape((packed.shape[0], -1) + packed.shape[2:])[:, :c]


def _plain_weights(w, fmt):
    """Values of the weights: blocks run along the input channels of one tap; f4 has one scale per filter."""
    return _plain_widen(_plain_narrow(w, fmt, w.abs().amax((1, 2, 3)) / w.new_tensor(6.0 * 448.0) if fmt == "f4" else 1.0), w.shape[1])


def _plain_act(v, act):
    if act == "leaky":
        return torch.where(v > 0, v, 0.1 * v)
    if act == "relu":
        return v.clamp(min=0)
    if act == "logistic":
        return 1 / (1 + torch.exp(-v))
    if act == "swish":
        return v / (1 + torch.exp(-v))
    if act == "mish":
        e = torch.exp(v.clamp(max=20.0))
        u = e * (e + 2)
        return v * (u / (u + 2))
    return v


def _plain_conv(x, w, b, k, stride, act):
    """One product per tap over the shifted image."""
    n, c, h, wd = x.shape
    pad = k // 2
    oh, ow = (h + 2 * pad - k) // stride + 1, (wd + 2 * pad - k) // stride + 1
    if k > 1:
        full = x.new_zeros((n, h + 2 * pad, wd + 2 * pad, c))
        full[:, pad:pad + h, pad:pad + wd] = x.permute(0, 2, 3, 1)
    else:
        full = x.permute(0, 2, 3, 1)
    acc = None
    for r in range(k):
        for q in range(k):
            part = full[:, r:r + stride * (oh - 1) + 1:stride, q:q + stride * (ow - 1) + 1:stride].reshape(-1, c) @ w[:, :, r, q].t()
            acc = part if acc is None else acc.add_(part)
    return _plain_act(acc + b, act).reshape(n, oh, ow, -1).permute(0, 3, 1, 2)


def _as(x, kind):
    return x.half() if kind == "f16" else x.float()


def _run_plain(s):
    case, fmt = s["case"], s["case"]["fmt"]
    c = case["channels"]
    if case["kind"] == "narrow":
        return _as(_plain_widen(_plain_narrow(s["x"], fmt, s["x_scale"]), c), case["dst"])
    x = _plain_widen(s["x4"] if "x4" in s else _plain_narrow(s["x"], fmt, s["x_scale"]), c)
    if case["kind"] == "widen":
        return _as(x, case["dst"])
    if case["kind"] == "product":
        return _as(_plain_conv(x, s["wq"], s["b"], case["k"], case["stride"], case["act"]), case["out"])
    y = _plain_narrow(_plain_conv(x, s["w1q"], s["b1"], 1, 1, case["act"]), fmt, s["y_scale"])
    return _plain_conv(_plain_widen(y, case["filters"]), s["w2q"], s["b2"], 3, 1, case["act"]).half()


def _prepare_plain(s):
    """Weights are quantised once, and kept as the values that their codes stand for; a 4-bit input is in hand as codes and scales."""
    case, fmt = s["case"], s["case"]["fmt"]
    if case["kind"] == "product":
        s["wq"] = _plain_weights(s["w"], fmt)
    elif case["kind"] == "chain":
        s["w1q"], s["w2q"] = _plain_weights(s["w1"], fmt), _plain_weights(s["w2"], fmt)
    if case["kind"] in ("widen", "product"):
        s["x4"] = _plain_narrow(s.pop("x"), fmt, s["x_scale"])
    return s


# ---- the framework's operators ----------------------------------------------------------------------------------------------------


class _Session:
    """The one backend of the process."""

    backend = None

    @classmethod
    def get(cls):
        if cls.backend is None:
            import lightnet_b200 as ln

            cls.ln, cls.backend = ln, ln.B200Backend(0)
        return cls.ln, cls.backend


def _dtype(ln, kind):
    return {"f4": ln.LN_F4, "mx4": ln.LN_MX4, "f32": ln.LN_F32, "f16": ln.LN_F16}[kind]


def _prepare_own(s):
    case = s["case"]
    ln, be = _Session.get()
    dtype = _dtype(ln, case["fmt"])

    def packed(w, b):
        f, c, k, _ = w.shape
        return be.conv_weights_f4(be.from_device(w), f, c, k, dtype), be.from_device(b.reshape(1, f, 1, 1))

    own_state = {"case": case, "ln": ln, "be": be, "dtype": dtype, "x_scale": s["x_scale"], "y_scale": s.get("y_scale", 1.0)}
    if case["kind"] in ("narrow", "chain"):
        own_state["x"] = s["x"]  # (the array that the plain form takes: the framework's layout of it is made within the call)
    else:
        own_state["x"] = be.narrow_f4(s["x"], s["x_scale"], dtype)
    if case["kind"] == "product":
        own_state["w"] = packed(s["w"], s["b"])
    if case["kind"] == "chain":
        own_state["w1"], own_state["w2"] = packed(s["w1"], s["b1"]), packed(s["w2"], s["b2"])
    be.sync()
    return own_state


def _torch(t):
    return torch.as_tensor(t, device="cuda")


def _run_own(s):
    case, ln, be, dtype = s["case"], s["ln"], s["be"], s["dtype"]

    def conv(x, w, c, h, wd, f, k, stride, act, out):
        pad = k // 2
        oh, ow = (h + 2 * pad - k) // stride + 1, (wd + 2 * pad - k) // stride + 1
        kind = ln.LN_OUT_Q if out == case["fmt"] else (ln.LN_OUT_F16 if out == "f16" else ln.LN_OUT_F32)
        return be.conv2d_bias_act_f4(x, w[0], w[1], (case["batch"], f, oh, ow), c, h, wd, f, k, stride, stride, 1, pad, 1, act, s["y_scale"], kind)

    if case["kind"] == "narrow":
        return _torch(be.widen_f4(be.narrow_f4(s["x"], s["x_scale"], dtype), _dtype(ln, case["dst"])))
    if case["kind"] == "widen":
        return _torch(be.widen_f4(s["x"], _dtype(ln, case["dst"])))
    c, h, w, f = case["channels"], case["height"], case["width"], case["filters"]
    if case["kind"] == "product":
        return _torch(conv(s["x"], s["w"], c, h, w, f, case["k"], case["stride"], case["act"], case["out"]))
    y = conv(be.narrow_f4(s["x"], s["x_scale"], dtype), s["w1"], c, h, w, f, 1, 1, case["act"], case["fmt"])
    return _torch(conv(y, s["w2"], f, h, w, 2 * f, 3, 1, case["act"], "f16"))


# ---- what the tools call ------------------------------------------------------------------------------------------------------------


def prepare(case, seed):
    s = _inputs(case, seed)
    return _prepare_own(s) if own else _prepare_plain(s)


def run(state):
    return _run_own(state) if "be" in state else _run_plain(state)


def work(case):
    """Inputs, weights and results once, at their storage widths; operations of the products, two per multiply-add."""
    n, c, h, w = (case[k] for k in ("batch", "channels", "height", "width"))
    four = 0.5 + SCALE_BYTES[case["fmt"]]
    values = n * c * h * w
    if case["kind"] == "narrow":  # to 4 bits, and from there back
        return {"bytes": values * (OUT_BYTES[case["src"]] + 2 * four + OUT_BYTES[case["dst"]]), "flops": 0}
    if case["kind"] == "widen":
        return {"bytes": values * (four + OUT_BYTES[case["dst"]]), "flops": 0}
    f = case["filters"]
    if case["kind"] == "chain":
        pixels = n * h * w
        return {"bytes": pixels * (2 * c + 2 * 2 * f) + four * (c * f + 18 * f * f) + 4 * 3 * f, "flops": 2 * pixels * (c * f + 18 * f * f)}
    k, stride = case["k"], case["stride"]
    pixels = n * ((h + 2 * (k // 2) - k) // stride + 1) * ((w + 2 * (k // 2) - k) // stride + 1)
    return {"bytes": values * four + f * c * k * k * four + 4 * f + pixels * f * OUT_BYTES[case["out"]], "flops": 2 * pixels * f * c * k * k}


# ---- the definition in 64 bits ------------------------------------------------------------------------------------------------------


def _exact_narrow(x, fmt, scale):
    """Codes by counting the borders below a value, E4M3 scales from the table of all of them; the two divisions and the product
    that the definition has in binary32 are taken in 64 bits and rounded to binary32 (one rounding: 53 bits are more than 2 * 24 + 2)."""
    f32 = lambda v: v.float().double()  # noqa: E731
    n, c = x.shape[:2]
    rest = tuple(x.shape[2:])
    size = BLOCK[fmt]
    blocks = -(-c // size)
    full = torch.zeros((n, blocks * size) + rest, dtype=torch.float64, device=x.device)
    full[:, :c] = f32(x)
    full = full.reshape((n, blocks, size) + rest)
    amax = full.abs().max(2, keepdim=True).values
    if fmt == "f4":
        g = torch.as_tensor(scale, dtype=torch.float64, device=x.device).reshape((-1,) + (1,) * (full.dim() - 1))
        want = f32(amax / f32(6.0 * g)).nan_to_num(0.0)
        table = torch.tensor([m / 8 * 2.0 ** -6 for m in range(8)] + [(1 + m / 8) * 2.0 ** e for e in range(-6, 9) for m in range(8)][:-1],
                             dtype=torch.float64, device=x.device)  # 0 .. 448; an even index has an even mantissa
        at = torch.searchsorted(table, want.clamp(max=448.0).contiguous()).clamp(1, len(table) - 1)
        below, above = table[at - 1], table[at]
        up = (want - below > above - want) | ((want - below == above - want) & (at % 2 == 0))
        s = torch.where(want >= 448.0, torch.full_like(want, 448.0), torch.where(up, above, below))
        step, value_step = f32(s * g), s * g
    else:
        exponent = (amax.view(torch.int64) >> 52) - 1023 - 2  # of a normal number of 64 bits
        step = value_step = ((exponent.clamp(min=-127) + 1023) << 52).view(torch.float64)
    t = torch.where(step > 0, f32(full / step), torch.zeros_like(full))
    a = t.abs()
    code = torch.zeros_like(a, dtype=torch.int64)
    for border, even_above in ((0.25, False), (0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)):
        code += (a >= border) if even_above else (a > border)
    value = torch.tensor(LEVELS, dtype=torch.float64, device=x.device)[code] * torch.sign(t)
    return (value * value_step).reshape((n, blocks * size) + rest)[:, :c]


def _exact_conv(x, w, b, k, stride, act):
    cols = torch.nn.functional.unfold(x, k, padding=k // 2, stride=stride) if k > 1 or stride > 1 else x.flatten(2)
    oh, ow = (x.shape[2] + 2 * (k // 2) - k) // stride + 1, (x.shape[3] + 2 * (k // 2) - k) // stride + 1
    if oh * ow == 1:
        v = (cols[:, :, 0] @ w.flatten(1).t()).reshape(x.shape[0], -1, 1, 1)
    else:
        v = torch.stack([w.flatten(1) @ part for part in cols]).reshape(x.shape[0], -1, oh, ow)
    v = v + b.double().reshape(1, -1, 1, 1)
    if act == "leaky":
        return torch.maximum(v, 0.1 * v)
    if act == "relu":
        return torch.relu(v)
    if act == "logistic":
        return torch.sigmoid(v)
    if act == "swish":
        return v * torch.sigmoid(v)
    if act == "mish":
        return v * torch.tanh(torch.logaddexp(v, torch.zeros_like(v)))
    return v


def exact(case, seed):
    s = _inputs(case, seed)
    fmt = case["fmt"]
    x = s["x"]
    if case["kind"] in ("narrow", "widen"):
        return _exact_narrow(x, fmt, s["x_scale"])
    weights = lambda w: _exact_narrow(w, fmt, (w.double().abs().amax((1, 2, 3)) / (6.0 * 448.0)).float() if fmt == "f4" else 1.0)  # noqa: E731
    x = _exact_narrow(x, fmt, s["x_scale"])
    if case["kind"] == "product":
        return _exact_conv(x, weights(s["w"]), s["b"], case["k"], case["stride"], case["act"])
    y = _exact_conv(x, weights(s["w1"]), s["b1"], 1, 1, case["act"])
    return _exact_conv(_exact_narrow(y, fmt, s["y_scale"]), weights(s["w2"]), s["b2"], 3, 1, case["act"])
