"""Activations kept in 8 bits on a B200: the bytes of the torch form, SwiGLU from and to them."""
import pytest
import torch

from tilerl_b200 import tape as T
from tilerl_b200.ops import keep, native

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _odd(x, offset):
    return torch.empty(x.numel() + offset, device=DEV)[offset:].view(x.shape).copy_(x)


@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("shape", [(1,), (3, 4), (5, 127), (2, 3, 128), (7, 132), (4, 1001), (33, 5120), (9, 34816)])
def test_packed_rows_have_the_bytes_of_the_torch_form(shape, offset):
    g = torch.Generator().manual_seed(len(shape))
    x = torch.randn(shape, generator=g) * torch.exp(4 * torch.randn(shape, generator=g))
    before = native.launch_count
    kept = T.keep8(_odd(x, offset))
    back = kept.rows()
    assert native.launch_count == before + 2
    q, scale = keep.pack(x)
    assert torch.equal(kept.q.cpu(), q) and torch.equal(kept.scale.cpu(), scale) and torch.equal(back.cpu(), keep.unpack(q, scale))


def test_groups_out_of_range():
    x = torch.ones(7, 300)
    x[0, 3], x[1, 200], x[2], x[6, 299] = float("nan"), float("-inf"), 0.0, -float("nan")
    x[3, :128], x[4, :128], x[5, 7] = 1e-37, 1e-40, torch.finfo(torch.float32).max
    kept, (q, scale) = T.keep8(x.to(DEV)), keep.pack(x)
    assert torch.equal(kept.q.cpu(), q) and torch.allclose(kept.scale.cpu(), scale, rtol=0, atol=0, equal_nan=True)
    assert torch.allclose(kept.rows().cpu(), keep.unpack(q, scale), rtol=0, atol=0, equal_nan=True)
    assert T.keep8(torch.empty(0, 5, device=DEV)).rows().shape == (0, 5)


@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("shape", [(1, 2), (3, 10), (2, 5, 128), (7, 300), (40, 3000), (5, 34816)])
def test_swiglu_from_and_to_8_bits(shape, offset):
    """The result is SwiGLU of the pairs, the gradient that at what is kept.  Against 64 bits: exponential (2 ulp), its sum and quotient, two
    products: 8 roundings of a result; a gradient's sums have two terms of either sign, up to 1 + |g| times the product: 16 of that."""
    g = torch.Generator().manual_seed(shape[-1])
    x, up = torch.randn(shape, generator=g) * 2, torch.randn(*shape[:-1], shape[-1] // 2, generator=g)
    here, tape = _odd(x, offset), T.Tape()
    tape.watch(here)
    before = native.launch_count
    y = T.swiglu(tape, here, bits=8)
    grad = tape.backward(y, up.to(DEV))[id(here)].cpu()
    assert native.launch_count == before + 2
    a, b = x[..., 0::2].double(), x[..., 1::2].double()
    want = a * torch.sigmoid(a) * b
    assert ((y.cpu() - want).abs() <= want.abs() * 8 * 2 ** -24 + 1e-37).all()
    kept = keep.unpack(*keep.pack(x)).double()
    a, b = kept[..., 0::2], kept[..., 1::2]
    sig, e = torch.sigmoid(a), up.double()
    da, db = e * b * sig * (1 + a * (1 - sig)), e * a * sig
    assert ((grad[..., 0::2] - da).abs() <= (e * b * sig).abs() * (1 + a.abs()) * 16 * 2 ** -24 + 1e-37).all()
    assert ((grad[..., 1::2] - db).abs() <= db.abs() * 16 * 2 ** -24 + 1e-37).all()
    if shape[-1] > 2:                                    # a gradient of another shape is the torch form's matter, which refuses it
        wrong = T.Tape()
        wrong.watch(here)
        with pytest.raises(RuntimeError):
            wrong.backward(T.swiglu(wrong, here, bits=8), torch.ones(3, 7, 1 + shape[-1], device=DEV))


def test_segments_and_memory():
    """Layers of 4096 x 1024 rows: the inputs of the checkpointed ones take a quarter, and replays start from them."""
    g = torch.Generator(device=DEV).manual_seed(0)
    w = torch.ones(1024, device=DEV)
    fn = lambda t, z: T.add(t, z, T.rmsnorm(t, z, w, 1e-6))

    def run(bits):
        x = torch.randn(4096, 1024, generator=g, device=DEV)
        tape = T.Tape()
        tape.watch(w)
        torch.cuda.synchronize()
        start = torch.cuda.memory_allocated()
        for _ in range(8):
            x = tape.checkpoint(fn, x, params=(w,), bits=bits)
        held = torch.cuda.memory_allocated() - start
        return held, tape.backward(x, torch.ones_like(x))[id(w)]

    full, gw = run(32)
    g.manual_seed(0)
    small, gw8 = run(8)
    # (of eight inputs in fp32 the first is the caller's; the last output is there both times)
    assert small <= 1.05 * (4096 * 1024 * 4 + 8 * 4096 * 1024 * (1 + 4 / 128)) and full >= 8 * 4096 * 1024 * 4
    # a value is off by up to 1/254 of its group's largest, evenly: about 1 % of a unit-size value's gradient, over 4096 rows and eight layers
    assert float((gw - gw8).norm() / gw.norm()) < 0.01


def test_streams_and_graphs():
    x, up = torch.randn(50, 600, device=DEV), torch.randn(50, 300, device=DEV)

    def run(t):
        tape = T.Tape()
        tape.watch(t)
        y = T.swiglu(tape, t, bits=8)
        return y, tape.backward(y, up)[id(t)], T.keep8(t).rows()

    want = run(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(x)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    static = torch.zeros_like(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(static)
    static.copy_(x)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(want, out))


def test_offsets_past_32_bits():
    rows, width = 70000, 32768
    x = torch.zeros(rows, width, device=DEV)
    x[-3:] = torch.randn(3, width, generator=torch.Generator(device=DEV).manual_seed(0), device=DEV)
    x[0] = 2.0
    kept = T.keep8(x)
    q, scale = keep.pack(x[-3:].cpu())
    assert torch.equal(kept.q[-3:].cpu(), q) and torch.equal(kept.scale[-3:].cpu(), scale) and not any(p.any() for p in kept.q[1:-3].split(10000))
    back = kept.rows()
    assert torch.equal(back[-3:].cpu(), keep.unpack(q, scale)) and torch.equal(back[0], x[0])
    del back, kept
    tape = T.Tape()
    tape.watch(x)
    y = T.swiglu(tape, x, bits=8)
    grad = tape.backward(y, torch.ones_like(y))[id(x)]
    small = x[-3:].clone()
    one = T.Tape()
    one.watch(small)
    z = T.swiglu(one, small, bits=8)
    assert torch.equal(y[-3:], z) and torch.equal(grad[-3:], one.backward(z, torch.ones_like(z))[id(small)])


@pytest.mark.parametrize("shape", [(3, 8), (300, 3000), (5, 34816)])
def test_the_forward_pass_is_that_without_8_bits(shape):
    x = torch.randn(*shape, generator=torch.Generator(device=DEV).manual_seed(3), device=DEV) * 3
    assert torch.equal(T.swiglu(T.Tape(), x, bits=8), T.swiglu(T.Tape(), x))
