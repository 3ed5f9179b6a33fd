"""Tensors that other libraries on the same GPU read: the order of their streams.  The work in front is held up by a kernel that spins for
some milliseconds, so that a read or a write in the wrong order meets the wrong values.  Needs a B200: run with -m gpu."""
import numpy as np
import pytest

import lightnet_b200 as ln

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

SPIN = 20_000_000  # cycles: 10 ms and more
SHAPE = (3, 40, 33, 35)


@pytest.fixture
def be():  # (of each test its own: which block an allocation takes is part of them)
    b = ln.B200Backend(0)
    yield b
    b.close()


def values(seed, shape=SHAPE):
    return np.random.default_rng(seed).integers(-6, 7, shape).astype(np.float32)


def address(t):
    return t.__cuda_array_interface__["data"][0]


@pytest.mark.parametrize("side", [False, True])
def test_a_reader_waits_for_what_made_the_tensor(be, side):
    x = values(1)
    own = torch.cuda.ExternalStream(be.stream)
    reader = torch.cuda.Stream() if side else torch.cuda.current_stream()
    old = be.upload_f32(SHAPE, values(2))
    where = address(old)
    t = be.upload_f32(SHAPE, x)
    be.sync()
    del old
    with torch.cuda.stream(own):
        torch.cuda._sleep(SPIN)
    y = be.widen_f4(be.narrow_f4(t, 1.0, ln.LN_MX4))  # (whole numbers up to 6 but 5, which ties to 4)
    if side:
        y.share(reader.cuda_stream)
    with torch.cuda.stream(reader):
        got = torch.as_tensor(y, device="cuda").clone()
    reader.synchronize()
    assert address(y) == where  # (where other values lay)
    assert np.array_equal(got.cpu().numpy(), np.where(np.abs(x) == 5, 4 * np.sign(x), x))


@pytest.mark.parametrize("side", [False, True])
def test_memory_is_used_again_behind_its_readers(be, side):
    x = values(3)
    reader = torch.cuda.Stream() if side else torch.cuda.current_stream()
    t = be.upload_f32(SHAPE, x)
    if side:
        t.share(reader.cuda_stream)
    view, where = torch.as_tensor(t, device="cuda"), address(t)
    with torch.cuda.stream(reader):
        torch.cuda._sleep(SPIN)
        got = view.clone()
    del view, t
    again = be.zeros_f32(SHAPE)
    assert address(again) == where
    assert not be.download_f32(again).any()
    reader.synchronize()
    assert np.array_equal(got.cpu().numpy(), x)


def test_released_while_a_graph_is_captured(be):
    """The block of a shared tensor that goes during a capture is not part of the graph, and serves again afterwards."""
    x = values(4)
    own = torch.cuda.ExternalStream(be.stream)
    three = [be.zeros_f32(SHAPE) for _ in range(3)]
    be.narrow_f4(three[0], 0.25)
    del three  # (memory for the two below and for the pass that is captured)
    fixed = be.upload_f32(SHAPE, x)
    shared = be.upload_f32(SHAPE, values(5))
    view, where = torch.as_tensor(shared, device="cuda"), address(shared)
    torch.cuda._sleep(SPIN)
    got = view.clone()
    be.sync()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=own):
        q = be.narrow_f4(fixed, 0.25)
        del view, shared
        y = be.widen_f4(q)
        assert torch.as_tensor(y, device="cuda").shape == SHAPE  # (asking for it is no error here)
        with pytest.raises(ln.BackendError) as e:
            y.share(0)
        assert e.value.kind == "unsupported"
        assert address(y) != where
    again = be.zeros_f32(SHAPE)
    assert address(again) == where
    assert np.array_equal(got.cpu().numpy(), values(5))
    with torch.cuda.stream(own):
        graph.replay()
    be.sync()
    want = be.download_f32(be.widen_f4(be.narrow_f4(fixed, 0.25)))
    assert np.array_equal(be.download_f32(y), want) and not be.download_f32(again).any()
    del graph


def test_share_refuses(be):
    t = be.upload_f32(SHAPE, values(6))
    t.share(be.stream)
    t.share()
    t.share(0)
    assert be.lib.ln_tensor_share(None, t.h, None) == be.lib.ln_tensor_share(be.ctx, None, None) == 5
    other = ln.B200Backend(0)
    try:
        assert be.lib.ln_tensor_share(other.ctx, t.h, None) == 5
    finally:
        other.close()
    with pytest.raises(AttributeError):
        be.narrow_f4(t, 0.5).__cuda_array_interface__


LAYOUTS = {
    "rows": lambda x: x,
    "channels last": lambda x: x.to(memory_format=torch.channels_last),
    "every other": lambda x: torch.stack([x, x + 1], -1)[..., 0],
    "turned": lambda x: x.permute(2, 3, 0, 1).contiguous().permute(2, 3, 0, 1),
    "columns": lambda x: x.transpose(2, 3).contiguous().transpose(2, 3),
    "odd start": lambda x: torch.cat([x.flatten()[:1], x.flatten()])[1:].reshape(x.shape),
}


@pytest.mark.parametrize("layout", sorted(LAYOUTS))
@pytest.mark.parametrize("kind", [torch.float32, torch.float16])
@pytest.mark.parametrize("shape", [(1, 1, 1, 1), (1, 4096, 1, 1), (3, 40, 7, 9), (130, 33, 1, 1), (2, 65, 13, 1), (1, 129, 1, 66), (5, 1, 64, 65), (2, 257, 19, 23)])
def test_a_tensor_from_device_memory(be, shape, kind, layout):
    x = torch.randn(shape, generator=torch.Generator("cuda").manual_seed(sum(shape)), device="cuda").to(kind)
    v = LAYOUTS[layout](x)
    assert torch.equal(v, x)
    t = be.from_device(v)
    assert t.shape == shape and t.dtype == (ln.LN_F32 if kind == torch.float32 else ln.LN_F16)
    got = be.download_f32(t) if kind == torch.float32 else be.download_f16(t)
    assert np.array_equal(got, x.float().cpu().numpy())


def test_broadcast_and_backward_strides(be):
    x = torch.arange(2 * 3 * 4 * 5, dtype=torch.float32, device="cuda").reshape(2, 3, 4, 5)
    wide = x[:, :1].expand(2, 70, 4, 5)
    assert np.array_equal(be.download_f32(be.from_device(wide)), wide.cpu().numpy())
    half = wide.half()[:, :1].expand(2, 70, 4, 5)
    assert np.array_equal(be.download_f16(be.from_device(half)), wide.cpu().numpy())
    back = be._out(be.lib.ln_tensor_from_device, x.data_ptr() + 4 * (x.numel() - 1), ln.LN_F32, ln._shape4(x.shape), ln._shape4([-s for s in x.stride()]), None)
    assert np.array_equal(be.download_f32(back), x.flip(0, 1, 2, 3).cpu().numpy())


def test_padding_channels_are_zero(be):
    """A binary16 convolution over memory that held NaN: the same as over an uploaded tensor."""
    n, c, h, w, f = 2, 40, 9, 10, 24
    rng = np.random.default_rng(7)
    x, wt = rng.normal(0, 1, (n, c, h, w)).astype(np.float16), rng.normal(0, 0.1, (f, c, 3, 3)).astype(np.float32)
    packed, b = be.conv_weights_f16(be.upload_f32(wt.shape, wt), f, c * 9), be.zeros_f32((1, f, 1, 1))

    def conv(t):
        return be.download_f16(be.conv2d_bias_act_f16(t, packed, b, (n, f, h, w), c, h, w, f, 3, 1, 1, 1, 1, 1, "leaky"))

    t = be.upload_f16(x.shape, x.astype(np.float32))
    want, where = conv(t), address(t)
    del t
    nan = be.upload_f16((n, 64, h, w), np.full((n, 64, h, w), np.nan, np.float32))
    assert address(nan) == where
    del nan
    t = be.from_device(torch.from_numpy(x).cuda())
    assert address(t) == where and np.array_equal(conv(t), want)


@pytest.mark.parametrize("side", [False, True])
@pytest.mark.parametrize("kind", [torch.float32, torch.float16])
def test_the_copy_lies_between_its_neighbours_on_the_stream(be, kind, side):
    x = torch.zeros(SHAPE, dtype=kind, device="cuda")
    new = torch.from_numpy(values(8)).cuda().to(kind)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream() if side else torch.cuda.current_stream()
    with torch.cuda.stream(stream):
        torch.cuda._sleep(SPIN)
        x.copy_(new)
        with torch.cuda.stream(torch.cuda.ExternalStream(be.stream)):
            torch.cuda._sleep(3 * SPIN)
        t = be.from_device(x, stream.cuda_stream if side else None)
        x.fill_(7)
    got = be.download_f32(t) if kind == torch.float32 else be.download_f16(t)
    assert np.array_equal(got, new.float().cpu().numpy())
    torch.cuda.synchronize()
    assert bool((x == 7).all())


@pytest.mark.parametrize("dtype", [ln.LN_F4, ln.LN_MX4])
@pytest.mark.parametrize("kind", [torch.float32, torch.float16])
def test_narrow_takes_an_array_on_the_gpu(be, kind, dtype):
    x = torch.from_numpy(np.random.default_rng(9).normal(0, 1, SHAPE).astype(np.float16)).cuda().to(kind)
    scale = 1.0 if dtype == ln.LN_MX4 else 0.002
    host = x.float().cpu().numpy()
    want = be.download_f4(be.narrow_f4(be.upload_f32(SHAPE, host) if kind == torch.float32 else be.upload_f16(SHAPE, host), scale, dtype))
    got = be.download_f4(be.narrow_f4(x, scale, dtype))
    assert all(np.array_equal(a, b) for a, b in zip(got, want))


def test_from_device_refuses(be):
    x = torch.zeros(SHAPE, device="cuda")
    one = ln._shape4((1, 1, 1, 1))

    def take(data=x.data_ptr(), dtype=ln.LN_F32, shape=SHAPE, strides=x.stride()):
        return be._out(be.lib.ln_tensor_from_device, data, dtype, ln._shape4(shape), ln._shape4(strides), None)

    def refused(kind, **what):
        with pytest.raises(ln.BackendError) as e:
            take(**what)
        assert e.value.kind == kind, str(e.value)

    take()
    host = np.zeros(SHAPE, np.float32)
    refused("argument", data=0)
    refused("argument", data=host.ctypes.data)
    refused("argument", data=torch.zeros(SHAPE).pin_memory().data_ptr())
    refused("argument", data=x.data_ptr() + 2)
    refused("argument", dtype=ln.LN_Q8)
    refused("argument", dtype=ln.LN_F4)
    refused("argument", strides=(1 << 36, 1, 1, 1))
    refused("argument", strides=(-(1 << 36), 1, 1, 1))
    refused("argument", strides=(1 << 62, 1 << 62, 1 << 62, 1 << 62))
    refused("shape", shape=(3, 0, 33, 35))
    refused("shape", shape=(3, -1, 33, 35))
    refused("shape", shape=(1 << 40, 1, 1, 1), strides=(0, 0, 0, 0))
    refused("unsupported", shape=(1 << 20, 1 << 20, 1, 1), strides=(0, 0, 0, 0))
    assert be.lib.ln_tensor_from_device(None, x.data_ptr(), ln.LN_F32, one, one, None, None) == 5
    with pytest.raises(ValueError):
        be.from_device(x.double())
    with pytest.raises(ValueError):
        be.from_device(x[0])
    be.debug_fail_alloc(1)
    refused("cuda")
    take()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.ExternalStream(be.stream)):
        refused("unsupported")
    del graph
    take()


@pytest.mark.parametrize("precision", [ln.LN_F32, ln.LN_F16, ln.LN_Q8])
def test_a_forward_waits_for_readers_of_the_last_one(be, precision):
    """Heads and layers that a network writes in place, eager and replayed: what another stream still reads is the forward that it asked about."""
    from lightnet_b200 import synth, zoo
    net, other = [ln.GpuExecutableNetwork(be, zoo.yolov3_tiny_cfg(160, 96), 2, precision) for _ in range(2)]
    blob = synth.he_weights(net.layers(), 3)
    images = [synth.uniform_images(2, 3, 96, 160, s) for s in range(6)]
    for n in (net, other):
        n.load_weights(blob)
        if precision == ln.LN_Q8:
            n.calibrate(images[0])
    want = []
    for x in images:
        other.forward(x)
        want.append([be.download_f32(other.head(k)) for k in range(other.num_heads())])
    read = []
    for x in images:
        net.forward(x)
        views = [torch.as_tensor(net.head(k), device="cuda") for k in range(net.num_heads())]
        torch.cuda._sleep(SPIN)
        read.append([v.clone() for v in views])
        del views
    torch.cuda.synchronize()
    if precision != ln.LN_F32:
        assert net.debug_replays() >= 3
    for got, ref in zip(read, want):
        assert all(np.array_equal(a.cpu().numpy(), b) for a, b in zip(got, ref))
    del net, other


def test_a_shared_f32_network_can_be_captured(be):
    """The forward of an f32 network makes its outputs anew, so heads that another stream may still read do not stand in the way of a capture."""
    from lightnet_b200 import synth, zoo
    net = ln.GpuExecutableNetwork(be, zoo.yolov3_tiny_cfg(160, 96), 1)
    net.load_weights(synth.he_weights(net.layers(), 3))
    x = synth.uniform_images(1, 3, 96, 160, 1)
    t = be.upload_f32(x.shape, x)
    held = []
    for _ in range(4):
        be._check(be.lib.ln_net_forward_device(net.h, t.h))
        held.append([torch.as_tensor(net.head(k), device="cuda") for k in range(net.num_heads())])
    want = [be.download_f32(net.head(k)) for k in range(net.num_heads())]
    views = held.pop()
    del held  # (memory for the forward that is captured)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.ExternalStream(be.stream)):
        be._check(be.lib.ln_net_forward_device(net.h, t.h))
    heads = [net.head(k) for k in range(net.num_heads())]
    with torch.cuda.stream(torch.cuda.ExternalStream(be.stream)):
        graph.replay()
    be.sync()
    for h, v, r in zip(heads, views, want):
        assert np.array_equal(be.download_f32(h), r) and np.array_equal(v.cpu().numpy(), r)
    del graph
