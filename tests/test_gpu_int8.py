"""Projections in 8-bit integers on a B200 against their definition in 64 bits."""
import dataclasses

import pytest
import torch

from tilerl_b200 import formats as F
from tilerl_b200 import tape as T
from tilerl_b200.ops import ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24                    # half a step of fp32; of bf16: 2^-8


@pytest.fixture(scope="module")
def ops():
    from tilerl_b200.ops.cuda import CudaOps
    return CudaOps(DEV)


def _weight(n, k, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    w = torch.randn(n, k, generator=g, device=DEV) * 0.02
    return F.quantize_int8(w * (0.2 + torch.rand(n, 1, generator=g, device=DEV)))


def _x(t, k, seed=1, dtype=torch.bfloat16):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(t, k, generator=g, device=DEV)
    return (x * (1 + 15 * (torch.rand(k, generator=g, device=DEV) < 0.05))).to(dtype)


def _norm_error(k):
    """Bound of a row's 1 / rms in fp32: a value's square and the sums over a vector of eight, 32 lanes, the groups of a lane and the lanes
    again (all of one sign: each sum half a step), the mean's division and eps, twice as much in the square as in its root; rsqrtf 2 ulp, and
    the product with the scale."""
    sums = 8 + 5 + -(-k // 8192) + 5 + 2
    return sums * U / 2 + 4 * U + U


def _ints(w):
    return w.w8.double()


# ---- rows ------------------------------------------------------------------------------------------------
def _quant(x, norm_w=None, eps=0.0, channels=None):
    from tilerl_b200.ops import gemm_int8
    t, k = x.shape
    rows = t if channels is None else 2 * t
    q = torch.full((rows, -(-k // 16) * 16), 99, dtype=torch.int8, device=DEV)
    s = torch.empty(t, device=DEV)
    gemm_int8.quant_rows(x, q, s, norm_w=norm_w, eps=eps, channels=channels)
    assert (q[:, k:] == 99).all()                    # what lies behind a row is left as it was
    return q[:, :k], s


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("t,k", [(1, 1), (3, 7), (2, 16), (5, 272), (1, 2048), (3, 2056), (2, 10240), (2, 10248), (3, 20488), (2, 65536), (2, 65551)])
def test_rows_give_the_integers_of_the_definition(t, k, dtype):
    x = _x(t, k, k, dtype)
    q, s = _quant(x)
    want, scale = F.quantize_act_int8(x)
    assert torch.equal(q, want) and torch.equal(s, scale)
    nw = torch.rand(k, device=DEV) + 0.5
    q, s = _quant(x, nw, 1e-6)
    want, plain = F._row_integers(x.float() * nw, F.INT8_MAX)
    assert torch.equal(q, want.to(torch.int8))
    exact = plain.double() / (x.double().square().mean(-1) + 1e-6).sqrt()
    assert ((s.double() - exact).abs() <= exact * _norm_error(k)).all()
    q, s = _quant(x, channels=nw)
    want, scale = F.quantize_grad_int16(x, nw)
    assert torch.equal(q.view(t, 2, k)[:, 0].int() * 256 + q.view(t, 2, k)[:, 1].int(), want) and torch.equal(s, scale)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_many_rows_one_after_the_other_and_long_ones_in_two_passes(dtype):
    for t, k in ((1500, 24), (1300, 2056), (700, 10264), (64, 10248), (67, 20487), (130, 34816), (3, 34816)):
        x, w = _x(t, k, k, dtype), torch.rand(k, device=DEV) + 0.5
        x[t // 2] = 0.0
        x[t - 1, k - 1] = float("nan")
        q, s = _quant(x, channels=w)
        want, scale = F.quantize_grad_int16(x, w)
        q = q.view(t, 2, k)
        assert torch.equal(q[:, 0].int() * 256 + q[:, 1].int(), want) and torch.equal(s.nan_to_num(-1.0), scale.nan_to_num(-1.0)) and torch.isnan(s[-1])
        q, s = _quant(x, w, 1e-6)
        want, _ = F._row_integers(x.float() * w, F.INT8_MAX)
        assert torch.equal(q, want.to(torch.int8)) and torch.isnan(s[-1]) and torch.isfinite(s[:-1]).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_off_every_boundary_and_apart(dtype):
    base = _x(9, 517, 3, dtype)
    for x in (base[:, 1:], base[::2, :515], base.flatten()[3:3 + 4 * 100].view(4, 100)):
        q, s = _quant(x)
        want, scale = F.quantize_act_int8(x)
        assert torch.equal(q, want) and torch.equal(s, scale)


def test_rows_of_zeros_tiny_huge_and_not_finite():
    x = torch.randn(8, 300, device=DEV)
    x[0] = 0.0
    x[1] *= 2.0 ** -126                              # (below what counts: zeros)
    x[2] *= 1e38 / x[2].abs().max()
    x[3, 299] = float("inf")
    x[4, 0] = float("nan")
    x[5, 7] = float("-inf")
    x[6] = -0.0
    q, s = _quant(x)
    want, scale = F.quantize_act_int8(x)
    assert torch.equal(q, want) and torch.equal(s.nan_to_num(-1.0), scale.nan_to_num(-1.0))
    assert torch.isnan(s[3:6]).all() and torch.isfinite(s[[0, 1, 2, 6, 7]]).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_weights_are_quantised_in_place(ops, dtype):
    w = torch.randn(37, 272, device=DEV).to(dtype)
    dst = F.INT8Tensor(torch.zeros(37, 272, dtype=torch.int8, device=DEV), torch.zeros(37, device=DEV))
    ops.quantize_int8_(w, dst)
    want = F.quantize_int8(w)
    assert torch.equal(dst.w8, want.w8) and torch.equal(dst.wscale, want.wscale)
    ops.quantize_int8_(w.t().contiguous().t(), dst)
    assert torch.equal(dst.w8, want.w8)


# ---- served ----------------------------------------------------------------------------------------------
def _check_served(ops, t, n, k, seed=0):
    w, x, nw = _weight(n, k, seed), _x(t, k, seed + 1), torch.rand(k, device=DEV) + 0.5
    q, s = F.quantize_act_int8(x)
    y = q.double() @ _ints(w).t() * s.double()[:, None] * w.wscale.double()
    res = _x(t, n, seed + 2)
    # fp32: the sum's rounding, the product of the scales, their product
    out = ops.linear_residual(x, w, res.clone())
    want = y + res.double()
    # (an addition of fp32 behind it, then bf16)
    assert ((out.double() - want).abs() <= want.abs() * 2.0 ** -8 * (1 + 2.0 ** -8) + (y.abs() * 3 + want.abs()) * U * 1.01).all()
    q, s = F._row_integers(x.float() * nw, F.INT8_MAX)
    s = s.double() / (x.double().square().mean(-1) + 1e-6).sqrt()
    y = q.double() @ _ints(w).t() * s[:, None] * w.wscale.double()
    e = _norm_error(k) + 3 * U
    out = ops.norm_linear(x, nw, w, 1e-6)
    assert out.shape == (t, n) and ((out.double() - y).abs() <= y.abs() * (2.0 ** -8 + 2 * e)).all()
    logits = ops.lm_head(x, nw, w, 1e-6)
    assert logits.dtype == torch.float32 and ((logits.double() - y).abs() <= y.abs() * e * 1.01).all()
    if n % 2 == 0:
        act = ops.norm_linear_swiglu(x, nw, w, 1e-6)
        gate, up = y[:, 0::2], y[:, 1::2]
        want = gate * torch.sigmoid(gate) * up
        # silu at a gate that is off by e moves by at most (1 + |gate|) e of itself; __expf is off by 2 + 1.2 |gate| ulp, the quotient by 2
        off = want.abs() * (2.0 ** -8 + 2 * ((2 + gate.abs()) * e + (6 + 1.2 * gate.abs()) * 2 * U + 2 * U)) + 1e-30
        assert act.shape == (t, n // 2) and ((act.double() - want).abs() <= off).all()


@pytest.mark.parametrize("t", [1, 2, 3, 4, 5, 8, 9, 16, 17, 31, 32, 33, 64, 65, 130, 257])
@pytest.mark.parametrize("n,k", [(2, 16), (130, 272), (1031, 1040)])
def test_products_of_all_numbers_of_rows(ops, t, n, k):
    _check_served(ops, t, n, k, seed=t)


@pytest.mark.parametrize("n,k", [(1, 16), (7, 48), (33, 64), (96, 4112), (255, 128), (256, 144), (513, 2048), (4098, 80), (5120, 17408), (20000, 512)])
def test_products_of_all_shapes(ops, n, k):
    for t in (1, 6, 24, 100, 300):
        _check_served(ops, t, n, k, seed=n)


@pytest.mark.parametrize("t", [1, 3, 40])
def test_adapters_over_served_integers(ops, t):
    n, k, r, scale = 386, 272, 8, 0.5
    g = torch.Generator(device=DEV).manual_seed(t)
    w, x, nw = _weight(n, k), _x(t, k), torch.rand(k, generator=g, device=DEV) + 0.5
    a, b = torch.randn(r, k, generator=g, device=DEV) / k ** 0.5, torch.randn(n, r, generator=g, device=DEV) * 0.1

    def adapter(h):
        """What the adapter adds, and the size of all that it adds up."""
        h, ad, bd = h.double(), a.double(), b.double()
        return h @ ad.t() @ bd.t() * scale, h.abs() @ ad.abs().t() @ bd.abs().t() * scale

    def room(y, delta, size, e):
        # the product's error, its rounding and the sum's to bf16; the adapter's sums of k and r terms, a rounding each, in fp32
        return (y.abs() + (y + delta).abs()) * 2.0 ** -8 * 1.01 + (y.abs() + size) * (e + (k + r + 8) * U) * 1.01
    q, s = F._row_integers(x.float() * nw, F.INT8_MAX)
    rstd = 1 / (x.double().square().mean(-1, keepdim=True) + 1e-6).sqrt()
    y = q.double() @ _ints(w).t() * (s.double()[:, None] * rstd) * w.wscale.double()
    delta, size = adapter(x.double() * rstd * nw.double())
    e = _norm_error(k) + 4 * U
    out = ops.norm_linear(x, nw, w, 1e-6, (a, b, scale)).double()
    assert ((out - y - delta).abs() <= room(y, delta, size, e)).all()
    act = ops.norm_linear_swiglu(x, nw, w, 1e-6, (a, b, scale)).double()
    gu, off = y + delta, room(y, delta, size, e)
    gate, up = gu[:, 0::2], gu[:, 1::2]
    silu = gate * torch.sigmoid(gate)
    # silu's slope is at most 1.1; its own error in fp32 and the result's rounding
    want = silu * up
    bound = off[:, 0::2] * 1.1 * (up.abs() + off[:, 1::2]) + silu.abs() * off[:, 1::2] + want.abs() * (2.0 ** -8 + (16 + 2 * gate.abs()) * 2 * U)
    assert ((act - want).abs() <= bound * 1.01 + 1e-30).all()
    q, s = F.quantize_act_int8(x)
    y = q.double() @ _ints(w).t() * s.double()[:, None] * w.wscale.double()
    delta, size = adapter(x)
    res = _x(t, n, 3)
    out = ops.linear_residual(x, w, res.clone(), (a, b, scale)).double()
    assert ((out - y - delta - res.double()).abs() <= room(y + res.double(), delta, size, 4 * U) + y.abs() * 4 * U).all()


@pytest.mark.parametrize("t", [1, 4, 20, 48, 300])
def test_one_row_has_the_same_bits_in_every_batch(ops, t):
    w, x, nw = _weight(386, 1168), _x(300, 1168), torch.rand(1168, device=DEV) + 0.5
    many = ops.norm_linear(x, nw, w, 1e-6).clone()
    some = ops.norm_linear(x[300 - t:], nw, w, 1e-6)
    assert torch.equal(some, many[300 - t:])


def test_sums_at_the_limits_of_32_bits(ops):
    k = 131072
    w = F.INT8Tensor(torch.full((3, k), 127, dtype=torch.int8, device=DEV), torch.ones(3, device=DEV))
    w.w8[1] = -127
    w.w8[2, ::2] = -128                              # (a file may hold it)
    x = torch.ones(33, k, device=DEV, dtype=torch.bfloat16)
    want = torch.tensor([127.0 * k, -127.0 * k, -0.5 * k], device=DEV, dtype=torch.float64)
    for t in (1, 33):
        got = ops.lm_head(x[:t], torch.ones(k, device=DEV), w, 0.0)
        assert ((got.double() - want).abs() <= want.abs() * (_norm_error(k) + 4 * U)).all()


def test_rows_that_are_not_finite_stay_among_themselves(ops):
    w, nw = _weight(130, 272), torch.ones(272, device=DEV)
    for t in (4, 40):
        x = _x(t, 272)
        clean = ops.norm_linear(x, nw, w, 1e-6).clone()
        x[1, 3], x[2, 5] = float("nan"), float("inf")
        got = ops.norm_linear(x, nw, w, 1e-6)
        others = [i for i in range(t) if i not in (1, 2)]
        assert torch.isnan(got[1:3]).all() and torch.equal(got[others], clean[others])
        x[:] = 0.0
        assert not ops.norm_linear(x, nw, w, 1e-6).any()


def test_strides_of_weights_rows_and_outputs(ops):
    from tilerl_b200.ops import gemm_int8
    big = _weight(140, 512)
    w = F.INT8Tensor(big.w8[3:133, 16:288], big.wscale[3:133].contiguous())
    solid = F.INT8Tensor(w.w8.contiguous(), w.wscale)
    for t in (3, 50, 200):
        x = _x(t, 300)[:, 8:280]
        out = torch.full((t, 141), 7.0, device=DEV, dtype=torch.bfloat16)
        gemm_int8.linear(ops, x, w, out[:, 5:135])
        want = torch.empty(t, 130, device=DEV, dtype=torch.bfloat16)
        gemm_int8.linear(ops, x.contiguous(), solid, want)
        assert torch.equal(out[:, 5:135], want) and (out[:, :5] == 7).all() and (out[:, 135:] == 7).all()
        res = _x(t, 150)[:, 3:133]
        gemm_int8.linear(ops, x, w, out[:, 5:135], residual=res, epi=gemm_int8.EPI_RESIDUAL)
        gemm_int8.linear(ops, x, solid, want, residual=res.contiguous(), epi=gemm_int8.EPI_RESIDUAL)
        assert torch.equal(out[:, 5:135], want)
        act = torch.full((t, 70), 7.0, device=DEV, dtype=torch.bfloat16)
        gemm_int8.linear(ops, x, w, act[:, 3:68], epi=gemm_int8.EPI_SWIGLU)
        want = torch.empty(t, 65, device=DEV, dtype=torch.bfloat16)
        gemm_int8.linear(ops, x, solid, want, epi=gemm_int8.EPI_SWIGLU)
        assert torch.equal(act[:, 3:68], want) and (act[:, :3] == 7).all() and (act[:, 68:] == 7).all()


@pytest.mark.parametrize("t", [1, 2, 3, 70])
def test_rows_that_are_the_residual_themselves(ops, t):
    """The output in the place of the rows that are multiplied, whole or in part."""
    from tilerl_b200.ops import gemm_int8
    w = _weight(1024, 1024)
    for _ in range(5):
        x = _x(t, 1024)
        want = ops.linear_residual(x.clone(), w, x.clone())
        assert torch.equal(ops.linear_residual(x, w, x), want)
    both = _x(t + 1, 1024)
    want = torch.empty(t, 1024, device=DEV, dtype=torch.bfloat16)
    gemm_int8.linear(ops, both[:t].clone(), w, want)
    gemm_int8.linear(ops, both[:t], w, both[1:])
    assert torch.equal(both[1:], want)


@pytest.mark.parametrize("t", [1, 3])
def test_rows_right_behind_the_output_go_in_one_launch(ops, t):
    """As small buffers of one allocator lie; a value further on they are the output's memory, and go in two."""
    from tilerl_b200.ops import gemm_int8, native
    n, k = 320, 256
    w, solid = _weight(n, k), _x(t, k)
    for epi, dtype, width in ((gemm_int8.EPI_STORE, torch.bfloat16, n), (gemm_int8.EPI_SWIGLU, torch.bfloat16, n // 2), (gemm_int8.EPI_STORE_F32, torch.float32, n)):
        want = torch.empty(t, width, device=DEV, dtype=dtype)
        gemm_int8.linear(ops, solid, w, want, epi=epi)
        size = want.element_size() * t * width
        for at, launches in ((size, 1), (size - 16, 2)):
            memory = torch.zeros(size + 2 * t * k, dtype=torch.int8, device=DEV)
            y, x = memory[:size].view(dtype).view(t, width), memory[at:at + 2 * t * k].view(torch.bfloat16).view(t, k)
            x.copy_(solid)
            before = native.launch_count
            gemm_int8.linear(ops, x, w, y, epi=epi)
            assert native.launch_count - before == launches and torch.equal(y, want)


def test_first_use_inside_a_capture():
    """Kernels that this process has not launched yet.  (The backend's buffers have their size already: it refuses to grow them in a capture.)"""
    import os
    import subprocess
    import sys
    code = """
import torch
from tilerl_b200 import formats as F, tape as T
from tilerl_b200.ops.cuda import CudaOps
ops = CudaOps()
ws = [F.quantize_int8(torch.randn(n, 1040, device="cuda")) for n in (386, 5120)]
xs = [torch.randn(t, 1040, device="cuda").bfloat16() for t in (1, 2, 33, 700)]
xf, up, nw = torch.randn(90, 1040, device="cuda"), torch.randn(90, 386, device="cuda"), torch.ones(1040, device="cuda")
ops.ws.get("proj", (700, 5120), torch.bfloat16), ops.ws.get("int8_rows", (700 * 1044,), torch.int8)
outs = []
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    for w in ws:
        for x in xs:
            outs.append(ops.norm_linear(x, nw, w, 1e-6).clone())
    tape = T.Tape()
    tape.watch(xf)
    y = T.linear(tape, xf, ws[0])
    outs += [y, tape.backward(y, up)[id(xf)]]
g.replay()
torch.cuda.synchronize()
want = [ops.norm_linear(x, nw, w, 1e-6).clone() for w in ws for x in xs]
tape = T.Tape()
tape.watch(xf)
y = T.linear(tape, xf, ws[0])
want += [y, tape.backward(y, up)[id(xf)]]
assert all(torch.equal(a, b) for a, b in zip(outs, want))
print("the same")
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=root, timeout=300)
    assert "the same" in r.stdout, r.stderr[-2000:]


def test_weights_that_were_just_written(ops):
    """Products load weights before they wait for the launch ahead of them; a weight's quantiser lets none start before its end."""
    for n, k, t in ((5120, 1024, 1), (4096, 4096, 1), (4096, 4096, 20), (8192, 2048, 300)):
        masters = [torch.randn(n, k, device=DEV) for _ in range(2)]
        want = [F.quantize_int8(m) for m in masters]
        w = F.INT8Tensor(torch.zeros(n, k, dtype=torch.int8, device=DEV), torch.zeros(n, device=DEV))
        x, nw = _x(t, k), torch.rand(k, device=DEV) + 0.5
        right = [ops.norm_linear(x, nw, v, 1e-6).clone() for v in want]
        torch.cuda.synchronize()
        for i in (0, 1, 0, 1, 0):
            ops.quantize_int8_(masters[i], w)
            assert torch.equal(ops.norm_linear(x, nw, w, 1e-6), right[i])


@pytest.mark.parametrize("t", [1, 3, 20, 300])
def test_weights_that_another_kernel_just_wrote(ops, t):
    """A copy, an operation in place: kernels that know nothing of the products behind them."""
    for n, k in ((5120, 1024), (4096, 4096), (8192, 2048)):
        two = [_weight(n, k, i) for i in range(2)]
        w = F.INT8Tensor(torch.zeros(n, k, dtype=torch.int8, device=DEV), torch.zeros(n, device=DEV))
        x, nw, up = _x(t, k), torch.rand(k, device=DEV) + 0.5, _x(t, n, 5, torch.float32)

        def gradient(v):
            tape = T.Tape()
            tape.watch(x)
            return tape.backward(T.linear(tape, x, v), up)[id(x)]
        right = [(ops.norm_linear(x, nw, v, 1e-6).clone(), T.linear(T.Tape(), x, v), gradient(v)) for v in two]
        other = ops.norm_linear(x, nw, F.INT8Tensor(-two[0].w8, two[0].wscale), 1e-6).clone()
        torch.cuda.synchronize()
        got = []
        for i in (0, 1, 0, 1):
            w.w8.zero_(), w.wscale.copy_(two[i].wscale), w.w8.copy_(two[i].w8)
            a = ops.norm_linear(x, nw, w, 1e-6).clone()
            w.w8.zero_(), w.w8.copy_(two[i].w8)
            b = T.linear(T.Tape(), x, w)
            w.w8.zero_(), w.w8.copy_(two[i].w8)
            got.append((i, a, b, gradient(w)))
        w.wscale.copy_(two[0].wscale), w.w8.copy_(two[0].w8), w.w8.neg_()
        assert torch.equal(ops.norm_linear(x, nw, w, 1e-6), other)
        for i, *outs in got:
            assert all(torch.equal(a, b) for a, b in zip(outs, right[i]))


def test_weights_and_outputs_past_32_bits_of_bytes(ops):
    """A weight of more than 2^31 bytes, and an output of as many values."""
    n, k = 20000, 110080
    w = F.INT8Tensor(torch.zeros(n, k, dtype=torch.int8, device=DEV), torch.rand(n, device=DEV) + 0.5)
    w.w8[-5:] = _weight(5, k).w8
    tail = F.INT8Tensor(w.w8[-5:], w.wscale[-5:])
    for t in (2, 40):
        x, nw = _x(t, k), torch.ones(k, device=DEV)
        got = ops.norm_linear(x, nw, w, 1e-6).clone()
        assert torch.equal(got[:, -5:], ops.norm_linear(x, nw, tail, 1e-6)) and not got[:, :-5].any()
    del w, got
    n, t = 34816, 65000
    w, x = _weight(n, 16), _x(t, 16)
    got = ops.norm_linear(x, torch.ones(16, device=DEV), w, 1e-6)
    part = got[-3:].clone()
    assert got.numel() > 2 ** 31 and torch.equal(part, ops.norm_linear(x[-3:].contiguous(), torch.ones(16, device=DEV), w, 1e-6))


def test_refusals(ops):
    from tilerl_b200.ops import gemm_int8
    w, x, y = _weight(32, 64), _x(2, 64), torch.empty(2, 32, device=DEV, dtype=torch.bfloat16)
    odd = F.INT8Tensor(w.w8[:, :40].contiguous(), w.wscale)
    with pytest.raises(ValueError, match="multiple of 16"):
        gemm_int8.linear(ops, x[:, :40], odd, y)
    with pytest.raises(ValueError, match="rows"):
        gemm_int8.linear(ops, x[:, :32], w, y)
    with pytest.raises(ValueError, match="rows"):
        gemm_int8.linear(ops, x.half(), w, y)
    with pytest.raises(ValueError, match="rows"):
        gemm_int8.linear(ops, x.t().contiguous().t(), w, y)
    with pytest.raises(ValueError, match="pairs"):
        gemm_int8.linear(ops, x, F.INT8Tensor(w.w8[:31], w.wscale[:31]), y, epi=gemm_int8.EPI_SWIGLU)
    for bad in (y[:1], y[:, :31], y.float(), y.cpu(), y.t().contiguous().t(), y[:1].expand(2, 32)):
        with pytest.raises(ValueError, match="output"):
            gemm_int8.linear(ops, x, w, bad)
    with pytest.raises(ValueError, match="residual"):
        gemm_int8.linear(ops, x, w, y, residual=y[:1], epi=gemm_int8.EPI_RESIDUAL)
    with pytest.raises(ValueError, match="residual"):
        gemm_int8.linear(ops, x, w, y, epi=gemm_int8.EPI_RESIDUAL)
    with pytest.raises(ValueError, match="norm"):
        gemm_int8.linear(ops, x, w, y, norm_w=torch.ones(63, device=DEV))
    wide = F.INT8Tensor(torch.zeros(1, 131088, dtype=torch.int8, device=DEV), torch.ones(1, device=DEV))
    with pytest.raises(ValueError, match="131072"):
        gemm_int8.linear(ops, torch.zeros(1, 131088, device=DEV), wide, torch.empty(1, 1, device=DEV, dtype=torch.bfloat16))
    gemm_int8.linear(ops, x[:0], w, y[:0])           # no tokens: nothing to do


# ---- trained -----------------------------------------------------------------------------------------------
def _check_trained(lead, n, k, dtype=torch.float32, seed=0):
    w = _weight(n, k, seed)
    t = 1
    for d in lead:
        t *= d
    x, up = _x(t, k, seed + 1, dtype).view(*lead, k), _x(t, n, seed + 2, torch.float32).view(*lead, n)
    tape = T.Tape()
    tape.watch(x)
    out = T.linear(tape, x, w, frozen=True)
    dx = tape.backward(out, up)[id(x)]
    q, s = F.quantize_act_int8(x)
    want = q.double() @ _ints(w).t() * s.double()[..., None] * w.wscale.double()
    assert out.shape == want.shape and out.dtype == torch.float32
    assert ((out.double() - want).abs() <= want.abs() * 3.01 * U).all()
    q, s = F.quantize_grad_int16(up, w.wscale)
    hi = (q + 128) >> 8
    high, low = (hi.double() @ _ints(w)) * 256, (q - hi * 256).double() @ _ints(w)
    want = (high + low) * s.double()[..., None]
    # both sums' roundings, that of their sum, the product
    off = (high.abs() + low.abs() + 2 * (high + low).abs()) * s.double()[..., None] * 1.01 * U
    assert dx.shape == x.shape and dx.dtype == torch.float32 and ((dx.double() - want).abs() <= off).all()


@pytest.mark.parametrize("n,k", [(1, 16), (7, 32), (130, 272), (129, 128), (1031, 1040), (256, 2048), (4098, 80), (300, 4112)])
def test_product_and_gradient(n, k):
    for lead in ((1,), (2, 3), (33,), (64,), (3, 50), (260,)):
        _check_trained(lead, n, k, seed=n)


def test_product_and_gradient_of_bf16_rows_and_one_row():
    _check_trained((3, 7), 130, 272, torch.bfloat16)
    _check_trained((), 130, 272)


def test_gradients_of_other_forms():
    w, x = _weight(130, 272), _x(6, 272, dtype=torch.float32)
    up = _x(6, 130, 4, torch.float32)

    def grad(g):
        tape = T.Tape()
        tape.watch(x)
        out = T.linear(tape, x, w)
        return tape.backward(out, g)[id(x)]
    want = grad(up)
    assert torch.equal(grad(up.t().contiguous().t()), want)
    assert torch.equal(grad(torch.cat([up, up], -1)[:, :130]), want)
    assert torch.equal(grad(up.double()), want)
    one = grad(torch.ones(1, 130, device=DEV).expand(6, 130))
    assert torch.equal(one[0], one[5])
    up[1], up[2, 3], up[3, 4] = 0.0, float("inf"), float("nan")
    got = grad(up)
    assert not got[1].any() and torch.isnan(got[2:4]).all() and torch.equal(got[[0, 4, 5]], want[[0, 4, 5]])


def test_gradient_against_differences():
    """On rows that lie on the grid the product is linear."""
    w = _weight(40, 48)
    x = torch.randint(-90, 90, (5, 48), device=DEV).float()
    x[:, 7] = 127.0
    up = _x(5, 40, 9, torch.float32)
    tape = T.Tape()
    tape.watch(x)
    dx = tape.backward(T.linear(tape, x, w), up)[id(x)]
    u = up.double() * w.wscale.double()
    off = (u.abs().amax(-1, keepdim=True) / 32512 * 0.51) * _ints(w).abs().sum(0)
    for at in ((0, 0), (2, 47), (4, 8)):
        hi, lo = x.clone(), x.clone()
        hi[at] += 9
        lo[at] -= 9
        a, b = T.linear(T.Tape(), hi, w).double(), T.linear(T.Tape(), lo, w).double()
        diff = ((a - b) * up.double()).sum() / 18
        room = off[at] + ((a.abs() + b.abs()) * up.double().abs()).sum() / 18 * 4 * U + dx[at].abs() * 8 * U
        assert abs(float(diff - dx[at])) <= float(room)


def test_adapters_and_checkpointed_layers_over_integers():
    from tilerl_b200.config import small_gpu
    from tilerl_b200.factory import build_model, make_ops
    cfg = dataclasses.replace(small_gpu(), quant="int8")
    dev_ops = make_ops(torch.device(DEV))
    m = build_model(cfg, DEV, seed=1, ops=dev_ops)
    assert isinstance(m.params["L0.gate_up"], F.INT8Tensor)
    m.add_lora(8)
    for k, v in m.lora.items():
        v[1].normal_(0, 0.02)
    ids = torch.randint(0, cfg.vocab, (2, 20), device=DEV)
    grads = []
    for again in (False, True):
        tape = T.Tape()
        tape.watch(*m.trainable().values())
        y = m.forward_dense(tape, ids, checkpoint_layers=again)
        got = tape.backward(y, torch.ones_like(y) * 1e-3)
        grads.append({k: got[id(v)] for k, v in m.trainable().items()})
    for k in grads[0]:
        assert torch.isfinite(grads[0][k]).all()
        assert float((grads[0][k] - grads[1][k]).norm()) <= 1e-3 * float(grads[0][k].norm()) + 1e-12, k


@pytest.mark.parametrize("trainer", [DEV, "cpu"])
def test_weights_that_did_not_move_keep_a_files_integers(trainer):
    """Packed again from masters and from a trainer, also one on another device, whose working type is bf16."""
    import types
    from tilerl_b200.config import get_config
    from tilerl_b200.models.hybrid import HybridModel, linear_names, random_master
    from tilerl_b200.parallel.resync import resync
    cfg = get_config("tiny-hybrid", "int8")
    g, master = torch.Generator().manual_seed(2), random_master(cfg, 3)
    for n in linear_names(cfg):
        shape = master[n].shape
        master[n] = F.INT8Tensor(torch.randint(-100, 100, shape, generator=g, dtype=torch.int8), torch.rand(shape[0], generator=g) * 1e-3 + 1e-5)
    m = HybridModel.from_master(cfg, master, device=DEV, keep_master=True)
    at = {n: m.params[n].w8.data_ptr() for n in linear_names(cfg)}
    weights = {n: w.to(trainer, torch.bfloat16) for n, w in m.params.items() if n.startswith("master.")}
    zero = types.SimpleNamespace(units=[0], unit_tensors=lambda i: weights, _prefetch=None, _drop=lambda u: None, device=torch.device("cpu"))
    for pack in (m.requantize_, lambda: resync(zero, m)):
        pack()
        for n in linear_names(cfg):
            assert torch.equal(m.params[n].w8.cpu(), master[n].w8) and torch.equal(m.params[n].wscale.cpu(), master[n].wscale) and m.params[n].w8.data_ptr() == at[n]
    weights["master.L0.down"][1] *= 3
    resync(zero, m)
    want = F.quantize_int8(weights["master.L0.down"].float())
    got = m.params["L0.down"]
    assert torch.equal(got.w8[1].cpu(), want.w8[1].cpu()) and torch.equal(got.wscale[1].cpu(), want.wscale[1].cpu()) and torch.equal(got.w8[2].cpu(), master["L0.down"].w8[2])


# ---- streams, graphs -----------------------------------------------------------------------------------------
def test_captured_and_replayed(ops):
    """Two captured products that share the backend's workspace, replayed one after the other over new rows; and a training pass."""
    wa, wb, nw = _weight(386, 272, 1), _weight(130, 272, 2), torch.rand(272, device=DEV) + 0.5
    for t in (1, 40):
        x = _x(t, 272)
        for w in (wa, wb):
            ops.norm_linear(x, nw, w, 1e-6), ops.norm_linear_swiglu(x, nw, w, 1e-6)
        outs, graphs = [torch.empty(t, 386, device=DEV, dtype=torch.bfloat16), torch.empty(t, 65, device=DEV, dtype=torch.bfloat16)], []
        torch.cuda.synchronize()
        for i in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                outs[i].copy_(ops.norm_linear(x, nw, wa, 1e-6) if i == 0 else ops.norm_linear_swiglu(x, nw, wb, 1e-6))
            graphs.append(g)
        for seed in (5, 6):
            x.copy_(_x(t, 272, seed))
            for g in graphs:
                g.replay()
            assert torch.equal(outs[0], ops.norm_linear(x, nw, wa, 1e-6))
            assert torch.equal(outs[1], ops.norm_linear_swiglu(x, nw, wb, 1e-6))


def test_captured_training_pass():
    w, x, up = _weight(130, 272), _x(9, 272, dtype=torch.float32), _x(9, 130, 3, torch.float32)

    def step():
        tape = T.Tape()
        tape.watch(x)
        out = T.linear(tape, x, w)
        return out, tape.backward(out, up)[id(x)]
    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out, dx = step()
    for seed in (7, 8):
        x.copy_(_x(9, 272, seed, torch.float32)), up.copy_(_x(9, 130, seed + 9, torch.float32))
        g.replay()
        a, b = step()
        assert torch.equal(a, out) and torch.equal(b, dx)


def test_two_threads_at_once_on_one_stream_and_on_two():
    """The kernels of a call hand each other its integers: no other call's."""
    import threading
    ws = [_weight(386, 1040, i) for i in range(2)]
    xs, ups = [_x(9 + i, 1040, i, torch.float32) for i in range(2)], [_x(9 + i, 386, i, torch.float32) for i in range(2)]

    def step(i):
        tape = T.Tape()
        tape.watch(xs[i])
        out = T.linear(tape, xs[i], ws[i])
        return out, tape.backward(out, ups[i])[id(xs[i])]
    want = [step(i) for i in range(2)]
    torch.cuda.synchronize()
    for streams in (None, [torch.cuda.Stream() for _ in range(2)]):
        wrong = []

        def work(i):
            with torch.cuda.stream(streams[i] if streams else torch.cuda.default_stream()):
                got = [step(i) for _ in range(200)]
                torch.cuda.current_stream().synchronize()
            wrong.extend(1 for g in got if not (torch.equal(g[0], want[i][0]) and torch.equal(g[1], want[i][1])))
        threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
        [t.start() for t in threads]
        [t.join() for t in threads]
        assert not wrong


def test_captured_training_passes_share_nothing():
    """Two captured passes of one thread, replayed at once on two streams."""
    w, x, up = _weight(386, 1040), [_x(30, 1040, i, torch.float32) for i in range(2)], _x(30, 386, 3, torch.float32)

    def step(i):
        tape = T.Tape()
        tape.watch(x[i])
        out = T.linear(tape, x[i], w)
        return out, tape.backward(out, up)[id(x[i])]
    want = [[t.clone() for t in step(i)] for i in range(2)]
    torch.cuda.synchronize()
    graphs, got = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for i in range(2):
        with torch.cuda.graph(graphs[i]):
            got.append(step(i))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        step(0)                                      # (and an eager one beside them)
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(got[i][0], want[i][0]) and torch.equal(got[i][1], want[i][1])


def test_on_another_stream(ops):
    w, nw = _weight(386, 1040), torch.rand(1040, device=DEV) + 0.5
    side = torch.cuda.Stream()
    for t in (1, 60):
        x = _x(t, 1040)
        want = ops.norm_linear(x, nw, w, 1e-6).clone()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            y = x * 0.5
            got = ops.norm_linear(y * 2, nw, w, 1e-6).clone()
            z = T.linear(T.Tape(), y, w)
        side.synchronize()
        assert torch.equal(got, want) and torch.equal(z, T.linear(T.Tape(), x * 0.5, w))


def test_many_calls_in_a_row_without_waiting(ops):
    """Each product reads what the one before it wrote, as a tick's do: kernels of consecutive launches are on the GPU together."""
    n = 1040
    w, nw = _weight(n, n), torch.rand(n, device=DEV) + 0.5
    for t in (1, 12, 70):
        x = _x(t, n)

        def chain(wait):
            y = x.clone()
            for _ in range(12):
                z = ops.norm_linear(y, nw, w, 1e-6)
                if wait:
                    torch.cuda.synchronize()
                y = ops.linear_residual(z, w, y)
                if wait:
                    torch.cuda.synchronize()
            return y
        want = chain(True)
        for _ in range(3):
            assert torch.equal(chain(False), want)


def test_a_run_of_them_together():
    """Prompt and captured decode ticks of a model in this format through the engine: its tokens are among those that the training forward
    over the same tokens finds largest.  (Attention and the recurrence round between the projections, and a value that lands on the other
    side of a half moves a step of 1 / 127; a token chosen by chance lies four deviations below the largest of 32768.)"""
    from tilerl_b200.config import small_gpu
    from tilerl_b200.engine import SamplingParams
    from tilerl_b200.factory import build_engine, build_model, make_ops
    cfg = dataclasses.replace(small_gpu(), quant="int8")
    dev_ops = make_ops(torch.device(DEV))
    m = build_model(cfg, DEV, seed=2, ops=dev_ops)
    eng = build_engine(m, dev_ops, blocks=64, slots=4, max_ctx=512)
    prompts = [list(range(7, 60)), list(range(300, 317)), [5, 6, 7]]
    res = eng.generate(prompts, SamplingParams(max_tokens=10, temperature=0.0))
    for p, r in zip(prompts, res):
        tokens = list(r.tokens)[-10:]
        logits = m.forward_dense(T.Tape(), torch.tensor([p + tokens], device=DEV))[0]
        for i, tok in enumerate(tokens):
            row = logits[len(p) - 1 + i].float()
            assert float(row.max() - row[tok]) <= 1.5 * float(row.std()), (i, tok)


def test_a_models_logits_against_the_reference_backend():
    from tilerl_b200.batch import Batch
    from tilerl_b200.config import small_gpu
    from tilerl_b200.factory import build_model, make_ops
    from tilerl_b200.kv import GdnStatePool, PagedKvPool
    from tilerl_b200.ops.backend import RefOps
    cfg = dataclasses.replace(small_gpu(), quant="int8")
    dev_ops = make_ops(DEV)
    m = build_model(cfg, DEV, seed=0, ops=dev_ops)
    toks = torch.randint(0, cfg.vocab, (24,), generator=torch.Generator().manual_seed(3)).tolist()
    outs = []
    for o, dt in ((dev_ops, torch.bfloat16), (RefOps(), torch.float32)):
        kv, st = PagedKvPool(cfg, 8, DEV, dtype=dt), GdnStatePool(cfg, 4, DEV, ring_dtype=torch.bfloat16)
        a = m.forward(Batch.build([dict(tokens=toks, start=0, blocks=[1, 2], slot=1)], DEV), o, kv, st).float().clone()
        b = m.forward(Batch.build([dict(tokens=[7], start=24, blocks=[1, 2], slot=1)], DEV), o, kv, st).float().clone()
        outs.append((a, b))
    # (a wrong epilogue, stride or scale shows as an error near 1)
    for a, b in zip(*outs):
        assert float((a - b).norm()) <= 0.25 * float(b.norm())
