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
