"""Policy and preference losses on a B200 against their torch form in 64 bits on the CPU."""
import math

import pytest
import torch

from tilerl_b200 import tape as T
from tilerl_b200.ops import native

pytestmark = pytest.mark.gpu
DEV = "cuda"
NAN = float("nan")


def _inputs(rows, v, dtype, seed, offset=0):
    """Logits (on the GPU ``offset`` values off a 16-byte boundary), and what goes with them, fp32."""
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)
    logits, targets = (r(*rows, v) * 2), torch.randint(0, v, rows, generator=g)
    logits.scatter_(-1, targets[..., None], math.log(v) + r(*rows, 1))
    logits = logits.to(dtype)
    lp = torch.log_softmax(logits.double(), -1).gather(-1, targets[..., None])[..., 0]
    mask = torch.rand(rows, generator=g) < 0.7
    mask.view(-1)[0] = True
    here = torch.empty(logits.numel() + offset, dtype=dtype, device=DEV)[offset:].view(logits.shape).copy_(logits)
    return logits, here, targets, mask, r(rows[0]), (lp + 0.3 * r(*rows)).float(), (lp + 0.2 * r(*rows)).float()


def _adds(v):
    """fp32 roundings behind a sum of v exponentials: a thread's own sums (no form has fewer than 32 threads a row), the reductions over
    them, an exponential's own (2 ulp) and its argument's."""
    return min(v, v / 32 + 80) + 24


def _grad_bounds(lg, w, dw, v):
    """Of a gradient w (p - onehot): the weight's error, the probability's, the products' roundings."""
    p = torch.softmax(lg.double(), -1)
    half = {torch.float32: 0.0, torch.bfloat16: torch.finfo(torch.bfloat16).eps / 2}[lg.dtype]
    b = dw[..., None] + w.abs()[..., None] * (p * _adds(v) * 2 ** -24 + 2 ** -22)
    return b + half * (w.abs()[..., None] * 2 + b)


SHAPES = [((1,), 1, 0), ((3,), 2, 1), ((2, 5), 7, 0), ((4, 9), 320, 0), ((9,), 512, 0), ((5,), 513, 1), ((3,), 2049, 0), ((2,), 4096, 0), ((3, 3), 1023, 3), ((2, 2), 1024, 0), ((2, 2), 1025, 1), ((5,), 4099, 2), ((2, 3), 16384, 0),
          ((3,), 16391, 1), ((2, 2), 32768, 0), ((2,), 49999, 1), ((3,), 65540, 2), ((2, 2), 131072, 0), ((3,), 150001, 3), ((2,), 248320, 0), ((2,), 262144, 0), ((2,), 262145, 0),
          ((2,), 300007, 1)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,v,offset", SHAPES)
def test_policy_loss(rows, v, offset, dtype):
    """Vocabularies of every form of the kernels and one value to either side of their borders, rows that begin anywhere, rows that are not scored."""
    logits, here, targets, mask, adv, old, refs = _inputs(rows, v, dtype, v, offset)
    before = native.launch_count
    for kw in (dict(mask=mask, old_logprobs=old, ref_logprobs=refs, kl_coef=0.1, clip_eps_high=0.3), dict(old_logprobs=old), dict(mask=mask)):
        tape = T.Tape()
        tape.watch(here)
        dev = {k: t.to(DEV) if isinstance(t, torch.Tensor) else t for k, t in kw.items()}
        loss, terms = T.policy_loss(tape, here, targets.to(DEV), adv.to(DEV), scale=0.25, **dev)
        grad = tape.backward(loss)[id(here)].cpu()
        cpu = T.Tape()
        wide = logits.double()
        cpu.watch(wide)
        want, wants = T.policy_loss(cpu, wide, targets, adv, scale=0.25, **kw)
        wgrad = cpu.backward(want)[id(wide)]
        dlp = _adds(v) * 2 ** -24                        # a log-probability's error: the sum's relative one (and its rounding below)
        a = adv.double().abs().view(-1, *[1] * (len(rows) - 1)).expand(rows)
        slope = a * wants.ratio.double() + (0.1 * torch.exp(refs.double() - wants.logprobs.double()) if "kl_coef" in kw else 0.0)
        tol = lambda t: t.double().abs() * 2 ** -23 + 1e-30
        assert ((terms.logprobs.cpu() - wants.logprobs).abs() <= dlp + tol(wants.logprobs)).all()
        assert ((terms.ratio.cpu() - wants.ratio).abs() <= wants.ratio * dlp + tol(wants.ratio)).all()
        d = (refs.double() - wants.logprobs).abs()
        assert ((terms.kl.cpu() - wants.kl).abs() <= torch.expm1(d) * dlp + dlp * dlp + tol(wants.kl)).all()
        assert torch.equal(terms.clipped.cpu(), wants.clipped)
        assert abs(float(loss) - float(want)) <= float(0.25 * (slope * dlp).sum()) + abs(float(want)) * 2 ** -23
        assert grad.dtype == dtype and grad.shape == logits.shape
        dw = 0.25 * slope * dlp + wants.weights.double().abs() * 2 ** -23
        assert ((grad.double() - wgrad).abs() <= _grad_bounds(logits, wants.weights.double(), dw, v)).all()
        if "mask" in kw:
            assert not grad[~mask].any()
    assert native.launch_count > before and native.read_error()[0] == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("pairs,t,v,offset", [(1, 1, 1, 0), (2, 3, 5, 1), (3, 70, 320, 0), (1, 7, 4099, 1), (2, 5, 32768, 0), (1, 3, 49999, 3), (1, 2, 248320, 0)])
def test_preference_loss(pairs, t, v, offset, dtype):
    logits, here, targets, mask, _, _, refs = _inputs((2 * pairs, t), v, dtype, v + t, offset)
    mask[-1] = False                                     # a sequence without a scored token
    for kw in (dict(mask=mask, ref_logprobs=refs, beta=0.3, label_smoothing=0.1), dict(mask=mask, average=True, beta=2.0), dict(ref_logprobs=refs)):
        tape = T.Tape()
        tape.watch(here)
        dev = {k: x.to(DEV) if isinstance(x, torch.Tensor) else x for k, x in kw.items()}
        loss, terms = T.preference_loss(tape, here, targets.to(DEV), **dev)
        up = torch.tensor(0.5, device=DEV)
        grad = tape.backward(loss, up)[id(here)].cpu()
        cpu, wide = T.Tape(), logits.double()
        cpu.watch(wide)
        want, wants = T.preference_loss(cpu, wide, targets, **kw)
        wgrad = cpu.backward(want, torch.tensor(0.5, dtype=torch.float64))[id(wide)]
        beta, dlp = kw.get("beta", 0.1), _adds(v) * 2 ** -24
        dsum = t * dlp
        assert ((terms.logprobs.cpu() - wants.logprobs).abs() <= dsum + wants.logprobs.abs() * 2 ** -23).all()
        assert ((terms.margins.cpu() - wants.margins).abs() <= 2 * beta * dsum + wants.margins.abs() * 2 ** -23).all()
        assert abs(float(loss) - float(want)) <= 2 * beta * dsum + abs(float(want)) * 2 ** -23
        # a weight is beta / pairs times a sigmoid (halved), whose slope is a quarter at most
        most = 0.5 * beta / pairs
        w = torch.full(targets.shape, most, dtype=torch.float64)
        bound = _grad_bounds(logits, w, w * (beta * dsum + 2 ** -22), v)
        if dtype == torch.bfloat16:
            bound = bound * 2 + 2 * most * 2 ** -8       # (the gradient is rounded before and after it is halved)
        assert ((grad.double() - wgrad).abs() <= bound).all()
    assert native.read_error()[0] == 0


def test_rows_that_are_not_scored_are_not_looked_at():
    logits, here, targets, mask, adv, old, refs = _inputs((40,), 1003, torch.float32, 5)
    mask[20:] = False
    for at, x in ((21, NAN), (22, float("-inf")), (23, torch.finfo(torch.float32).min), (24, float("inf"))):
        here[at] = x
    old[20:], refs[20:], adv[20:], targets[20:] = NAN, float("inf"), NAN, 10 ** 12
    mask = mask.to(DEV)
    tape = T.Tape()
    tape.watch(here)
    loss, terms = T.policy_loss(tape, here, targets.to(DEV), adv.to(DEV), scale=1.0, mask=mask, old_logprobs=old.to(DEV), ref_logprobs=refs.to(DEV), kl_coef=0.1)
    grad = tape.backward(loss)[id(here)]
    assert torch.isfinite(loss) and torch.isfinite(grad).all() and not grad[20:].any() and not any(t[20:].any() for t in terms)
    loss, terms = T.policy_loss(tape, here, targets.to(DEV), adv.to(DEV), scale=1.0, mask=torch.zeros_like(mask))
    assert float(loss) == 0.0 and not tape.backward(loss)[id(here)].any()
    assert native.read_error()[0] == 0


@pytest.mark.parametrize("v", [40, 5000, 20000, 150000, 270000])
def test_infinities_and_nan_in_scored_rows(v):
    """As the torch form: words that cannot be (-inf, the type's lowest) count nothing, a NaN or +inf makes its row NaN and no other."""
    x = torch.randn(8, v, generator=torch.Generator().manual_seed(0))
    low = torch.finfo(torch.float32).min
    x[0, 1:], x[1, : v // 2], x[2, 3], x[3, v - 1], x[4], x[5, : v - 1] = float("-inf"), low, NAN, float("inf"), float("-inf"), low
    targets = torch.tensor([0, v - 1, 0, 0, 0, v - 1, 5, 6])
    sides = []
    for dev in ("cpu", DEV):
        lg, tape = x.to(dev), T.Tape()
        tape.watch(lg)
        loss, terms = T.policy_loss(tape, lg, targets.to(dev), torch.ones(8, device=dev), scale=1.0)
        sides.append([terms.logprobs.cpu(), terms.weights.cpu(), tape.backward(loss)[id(lg)].cpu(), loss.cpu()])
    for want, got in zip(*sides):
        assert torch.equal(want.isnan(), got.isnan())
        assert torch.allclose(want, got, rtol=1e-4, atol=1e-6, equal_nan=True)
    assert sides[1][0].isnan().tolist() == [False, False, True, True, True, False, False, False]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("v", [40, 900, 5000, 20001, 50000, 150000, 270000])
def test_rows_far_from_zero(v, dtype):
    """Logits of any finite size: masked words of -1e4 to the type's lowest in long runs, rows that lie at 1e6 or -1e30 as a whole, rows of nothing but the lowest
    value (all words alike).  Against 64 bits: a log-probability is off by its own rounding and that of the row's differences, 2^-22 of them, and by
    the sum's roundings."""
    g = torch.Generator().manual_seed(v)
    x = torch.randn(12, v, generator=g)
    low = torch.finfo(dtype).min
    x[0, : v - 3], x[1, 3:], x[2], x[3, : v // 2], x[4, : v // 2] = -1e10, low, low, -1e4, -1e30
    x[5] += 1e6
    x[6] -= 1e6
    x[7] = x[7] * 1e9
    x[8] = -1e30
    x[8, v // 3] = -1e30 * (1 - 2 ** -6)
    x[9] = 3e38
    x[10, : v - 1], x[10, v - 1] = low, -low
    x = x.to(dtype)
    targets = torch.tensor([v - 1, 2, 5, v - 1, v - 1, 7, 7, int(x[7].float().argmax()), v // 3, 1, v - 1, 3])
    wide, tape64 = x.double(), T.Tape()
    tape64.watch(wide)
    want, terms64 = T.policy_loss(tape64, wide, targets, torch.ones(12), scale=1.0)
    wgrad = tape64.backward(want)[id(wide)]
    here, tape = x.to(DEV), T.Tape()
    tape.watch(here)
    loss, terms = T.policy_loss(tape, here, targets.to(DEV), torch.ones(12, device=DEV), scale=1.0)
    grad = tape.backward(loss)[id(here)].cpu()
    spread = (wide.amax(-1) - wide.gather(-1, targets[:, None])[:, 0]).abs()
    assert ((terms.logprobs.cpu() - terms64.logprobs).abs() <= spread * 2 ** -22 + _adds(v) * 2 ** -24 + terms64.logprobs.abs() * 2 ** -23).all()
    bound = _grad_bounds(x, terms64.weights.double(), torch.zeros(12, dtype=torch.float64), v)
    assert torch.isfinite(grad).all() and ((grad.double() - wgrad).abs() <= bound).all()
    chosen = here.view(12, 1, v)
    tape.watch(chosen)
    pref, seen = T.preference_loss(tape, chosen, targets.to(DEV)[:, None])
    assert torch.allclose(seen.logprobs, terms.logprobs, rtol=2 ** -22, atol=_adds(v) * 2 ** -24)
    pgrad = tape.backward(pref)[id(chosen)].cpu().view(12, v).double()
    # the same rows with other weights (a sequence of one row each): their gradients are in the same proportion
    tg = torch.arange(12), targets
    share = pgrad[tg] / torch.where(wgrad[tg] == 0, 1.0, wgrad[tg])
    assert torch.isfinite(pgrad).all() and ((pgrad - wgrad * share[:, None]).abs() <= 2 * bound * share.abs()[:, None] + 2 ** -20 * (wgrad * share[:, None]).abs()
                                            + (wgrad[tg] == 0)[:, None]).all()


@pytest.mark.parametrize("v", [40, 5000, 20000, 150000, 270000])
def test_targets_outside_of_the_vocabulary(v):
    lg = torch.randn(4, v, generator=torch.Generator().manual_seed(0)).to(DEV)
    for t in (-1, v, 1 << 40):
        tape = T.Tape()
        tape.watch(lg)
        loss, terms = T.policy_loss(tape, lg, torch.tensor([0, t, 1, 2], device=DEV), torch.ones(4, device=DEV), scale=1.0)
        grad = tape.backward(loss)[id(lg)]
        assert loss.isnan() and terms.logprobs.isnan().tolist() == [False, True, False, False] and grad.isnan().any(-1).tolist() == [False, True, False, False]
        code, site, _, n = native.read_error()
        assert (code, site, n) == (2, 16, v)
    tape.watch(lg)
    pair = lg.view(4, 1, v)
    loss, _ = T.preference_loss(T.Tape(), pair, torch.tensor([[0], [v], [1], [2]], device=DEV))
    assert loss.isnan() and native.read_error()[0] == 2


def test_upstream_gradient_strides_streams_and_graphs():
    """A loss that is scaled further, logits that are a view, work on another stream, and a captured pass replayed on new inputs."""
    logits, here, targets, mask, adv, old, refs = _inputs((3, 6), 700, torch.float32, 9)
    dev = [t.to(DEV) for t in (targets, mask, adv, old, refs)]

    def run(lg, factor=None):
        tape = T.Tape()
        tape.watch(lg)
        loss, terms = T.policy_loss(tape, lg, dev[0], dev[2], scale=0.1, mask=dev[1], old_logprobs=dev[3], ref_logprobs=dev[4], kl_coef=0.1)
        if factor is not None:
            loss = T.scale(tape, loss, factor)
        return loss, tape.backward(loss)[id(lg)], terms.logprobs

    loss, grad, lp = run(here)
    assert torch.allclose(run(here, 3.0)[1], grad * 3, rtol=1e-6)
    wide = torch.zeros(3, 6, 800, device=DEV)
    wide[..., :700] = here
    view = wide[..., :700]
    assert not view.is_contiguous() and torch.equal(run(view)[1], grad)
    assert torch.equal(run(here.transpose(0, 1).contiguous().transpose(0, 1))[1], grad)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = run(here)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(other, (loss, grad, lp)))
    static = here.clone()
    with torch.cuda.stream(side):
        run(static)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(static, 2.0)
    static.copy_(here.flip(-1))
    graph.replay()
    again = run(here.flip(-1).contiguous(), 2.0)
    assert all(torch.equal(a, b) for a, b in zip(out, again))
    kept = grad.clone()
    here.zero_()                                          # the logits may be written into: the gradient is there
    assert torch.equal(grad, kept)


def test_the_same_bits_twice():
    for v in (320, 9000, 32768, 150000, 270000):
        logits, here, targets, mask, adv, old, refs = _inputs((2, 4), v, torch.bfloat16, 1)
        outs = []
        for _ in range(2):
            tape = T.Tape()
            tape.watch(here)
            loss, terms = T.policy_loss(tape, here, targets.to(DEV), adv.to(DEV), scale=0.1, mask=mask.to(DEV), old_logprobs=old.to(DEV))
            pair, _ = T.preference_loss(tape, here, targets.to(DEV), mask.to(DEV), refs.to(DEV))
            outs.append([loss, pair, tape.backward(loss)[id(here)], *terms])
        assert all(torch.equal(a, b) for a, b in zip(*outs))


def test_more_rows_than_blocks_run_at_a_time():
    """Persistent forms go through their rows in turn: every row as it is on its own, scored ones and others in any order."""
    for n, v in ((5000, 400), (900, 1500), (700, 20001), (200, 66000)):
        g = torch.Generator(device=DEV).manual_seed(n)
        lg = torch.randn(n, v, generator=g, device=DEV)
        tg = torch.randint(0, v, (n,), generator=g, device=DEV)
        mask = torch.rand(n, generator=g, device=DEV) < 0.6
        adv = torch.randn(n, generator=g, device=DEV)
        tape = T.Tape()
        tape.watch(lg)
        loss, terms = T.policy_loss(tape, lg, tg, adv, scale=1.0, mask=mask)
        grad = tape.backward(loss)[id(lg)]
        assert torch.equal(terms.logprobs == 0, ~mask) and not grad[~mask].any()
        for i in range(0, n, 61):
            one = T.Tape()
            row = lg[i:i + 1]
            one.watch(row)
            l1, t1 = T.policy_loss(one, row, tg[i:i + 1], adv[i:i + 1], scale=1.0, mask=mask[i:i + 1])
            assert torch.allclose(t1.logprobs, terms.logprobs[i:i + 1], rtol=1e-6) and torch.allclose(one.backward(l1)[id(row)][0], grad[i], rtol=1e-4, atol=1e-9)
        want = torch.log_softmax(lg[mask].double(), -1).gather(-1, tg[mask][:, None])[:, 0]
        assert torch.allclose(terms.logprobs[mask].double(), want, atol=1e-5)


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs in one process")
def test_losses_on_a_gpu_that_is_not_the_current_one():
    logits, here, targets, mask, adv, old, refs = _inputs((2, 4), 40000, torch.float32, 1)
    outs = []
    for dev in ("cuda:0", "cuda:1"):
        lg, tape = here.to(dev), T.Tape()
        tape.watch(lg)
        loss, _ = T.policy_loss(tape, lg, targets.to(dev), adv.to(dev), scale=0.1, mask=mask.to(dev))
        outs.append([loss.cpu(), tape.backward(loss)[id(lg)].cpu()])
    assert all(torch.equal(a, b) for a, b in zip(*outs))


def test_inputs_on_unlike_devices_are_refused():
    lg = torch.zeros(2, 5, device=DEV)
    for kw in (dict(targets=torch.zeros(2, dtype=torch.long)), dict(mask=torch.ones(2, dtype=torch.bool)), dict(advantages=torch.zeros(2)), dict(old_logprobs=torch.zeros(2))):
        with pytest.raises(ValueError):
            T.policy_loss(T.Tape(), **{**dict(logits=lg, targets=torch.zeros(2, dtype=torch.long, device=DEV), advantages=torch.zeros(2, device=DEV), scale=1.0), **kw})


def test_offsets_past_32_bits():
    """2.2e9 logits of which the first and the last rows are scored: as those rows on their own, zeros everywhere else."""
    n, v = 9000, 248320
    g = torch.Generator(device=DEV).manual_seed(0)
    lg = torch.empty(n, v, dtype=torch.bfloat16, device=DEV)
    some = torch.tensor([0, 1, n - 2, n - 1], device=DEV)
    rows = torch.randn(4, v, generator=g, device=DEV).bfloat16()
    lg[some] = rows
    lg[2:n - 2] = NAN
    targets, mask = torch.full((n,), -5, device=DEV), torch.zeros(n, dtype=torch.bool, device=DEV)
    targets[some], mask[some] = torch.tensor([0, v - 1, 7, v - 2], device=DEV), True
    adv = torch.randn(n, generator=g, device=DEV)
    for pref in (False, True):
        tape, one = T.Tape(), T.Tape()
        shape = (lambda t: t.view(2, n // 2, *t.shape[1:])) if pref else (lambda t: t)
        big, small = shape(lg), rows.view(2, 2, v) if pref else rows
        tape.watch(big), one.watch(small)
        if pref:
            loss, _ = T.preference_loss(tape, big, shape(targets), shape(mask))
            want, _ = T.preference_loss(one, small, targets[some].view(2, 2))
        else:
            loss, terms = T.policy_loss(tape, big, targets, adv, scale=0.25, mask=mask)
            want, alone = T.policy_loss(one, small, targets[some], adv[some], scale=0.25)
            assert torch.equal(terms.logprobs[some], alone.logprobs) and int(terms.logprobs.count_nonzero()) == 4
        assert torch.allclose(loss, want, rtol=1e-6)
        grad = tape.backward(loss)[id(big)].view(n, v)
        assert torch.equal(grad[some], one.backward(want)[id(small)].view(4, v))
        assert not any(part.any() for part in grad[2:n - 2].split(1000))
        del grad, tape, big


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("v,offset", [(5, 1), (700, 0), (4099, 3), (20000, 2), (33000, 0)])
def test_sums_of_rows_whose_target_is_nearly_certain(v, offset, dtype):
    """The target at 40, the others at 0: a log-probability of -(v - 1) e^-40.  What is left of it in 64 bits: 1e-16 a number near 1, and the words'
    mean, which is fp32 (6e-8 of 58, in binary places), times fp32's relative error of log2 e, 2^-24 at most: under 1e-12 a row.  The target's
    place goes through a vector, a thread's vectors, both ends of the row."""
    t = 96
    places = torch.tensor(sorted({*range(min(v, 24)), *range(max(0, v - 24), v), *torch.linspace(0, v - 1, 48).long().tolist()}))
    targets = places[torch.arange(2 * t) % len(places)].view(2, t).to(DEV)
    here = torch.zeros(2 * t * v + offset, dtype=dtype, device=DEV)[offset:].view(2, t, v)
    here.scatter_(-1, targets[..., None], 40.0)
    _, terms = T.preference_loss(T.Tape(), here, targets)
    want = -t * (v - 1) * math.exp(-40.0)
    assert ((terms.logprobs.double().cpu() - want).abs() <= t * 1e-12).all()


@pytest.mark.parametrize("v", [513, 33001])
def test_sums_of_rows_whose_target_is_far_from_the_mean(v):
    """The target at -80, the others at 0, whose exponentials are 1 exactly: what is left is what rows are given back for the mean of
    an exponential's error (under 2^-22 as the error is) and fp64's.  A relative error of fp32's log2 e (1.3e-8) in x would be 1e-6 a row."""
    t = 256
    here = torch.zeros(2, t, v, device=DEV)
    here[0, :, 3], here[1, :, 3] = -80.0, 40.0
    exact = torch.tensor([-80.0 - math.log(v - 1), -(v - 1) * math.exp(-40.0)], dtype=torch.float64)
    ref = exact.float()[:, None].expand(2, t).contiguous()
    _, terms = T.preference_loss(T.Tape(), here, torch.full((2, t), 3, device=DEV), ref_logprobs=ref.to(DEV), beta=0.5)
    off = (exact - ref[:, 0].double()) * t
    want = 0.5 * float(off[0] - off[1])
    assert abs(float(terms.margins) - want) <= 0.5 * t * 2 ** -22 / 4 + abs(want) * 2 ** -24


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("pairs,t,v,offset", [(3, 11, 17, 2), (2, 7, 512, 0), (1, 5, 513, 1), (2, 6, 1024, 0), (1, 9, 1025, 3), (3, 3, 2048, 0), (1, 7, 2049, 1), (2, 3, 4096, 0), (1, 3, 4096, 3), (1, 5, 4097, 0)])
def test_preference_loss_at_the_borders_of_its_short_rows(pairs, t, v, offset, dtype):
    """Rows of every number of threads that keep them in registers, and one value to either side."""
    test_preference_loss(pairs, t, v, offset, dtype)


@pytest.mark.parametrize("v", [11, 5000])
def test_one_row_without_dimensions_before_the_vocabulary(v):
    logits, here, targets, _, adv, old, refs = _inputs((1,), v, torch.float32, v)
    kw = dict(scale=1.0, kl_coef=0.1)
    whole, row = T.Tape(), T.Tape()
    whole.watch(here)
    loss, terms = T.policy_loss(whole, here, targets.to(DEV), adv.to(DEV), old_logprobs=old.to(DEV), ref_logprobs=refs.to(DEV), **kw)
    one = here[0].clone()
    row.watch(one)
    got, some = T.policy_loss(row, one, targets[0].to(DEV), adv[0].to(DEV), old_logprobs=old[0].to(DEV), ref_logprobs=refs[0].to(DEV), **kw)
    assert torch.equal(got, loss) and all(torch.equal(a, b[0]) and a.shape == () for a, b in zip(some, terms))
    assert torch.equal(row.backward(got)[id(one)], whole.backward(loss)[id(here)][0])


@pytest.mark.parametrize("pairs", [5, 7, 8, 9, 33])
@pytest.mark.parametrize("v", [40, 5000])
def test_losses_of_few_pairs_and_of_many(pairs, v):
    """Up to eight pairs' losses are added up where they are formed, more by a kernel of their own."""
    test_preference_loss(pairs, 3, v, 0, torch.float32)


@pytest.mark.parametrize("v,rows,launches", [(300, 64, 1), (300, 65, 2), (512, 57, 1), (700, 32, 1), (700, 33, 2), (1500, 16, 1), (1500, 17, 2), (4000, 8, 1), (4000, 9, 2),
                                             (4097, 5, 2)])
def test_policy_losses_of_few_rows_and_of_many(v, rows, launches):
    """Up to eight blocks of short rows add their losses up themselves, to either side of that."""
    test_policy_loss((rows,), v, 0, torch.float32)
    lg = torch.zeros(rows, v, device=DEV)
    off, _ = T.policy_loss(T.Tape(), lg, torch.zeros(rows, dtype=torch.long, device=DEV), torch.ones(rows, device=DEV), scale=0.5,
                           mask=torch.zeros(rows, dtype=torch.bool, device=DEV))
    assert float(off) == 0.0
    before = native.launch_count
    loss, _ = T.policy_loss(T.Tape(), lg, torch.zeros(rows, dtype=torch.long, device=DEV), torch.ones(rows, device=DEV), scale=0.5)       # (without a gradient)
    assert float(loss) == -0.5 * rows and native.launch_count == before + launches


@pytest.mark.parametrize("t", [255, 2500, 4096, 4097, 9000])
def test_preference_loss_of_long_sequences(t):
    """More tokens than a pair's block has threads."""
    test_preference_loss(2, t, 40, 0, torch.float32)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float64])
def test_targets_outside_of_the_vocabulary_in_the_torch_form(dtype):
    """Logits in types that the kernels do not take: a row without a number, as from the kernels, but for the error word."""
    lg = torch.randn(4, 30, generator=torch.Generator().manual_seed(0)).to(DEV, dtype)
    for t in (-1, 30, 1 << 40):
        tape = T.Tape()
        tape.watch(lg)
        loss, terms = T.policy_loss(tape, lg, torch.tensor([0, t, 1, 2], device=DEV), torch.ones(4, device=DEV), scale=1.0)
        grad = tape.backward(loss)[id(lg)]
        assert loss.isnan() and terms.logprobs.isnan().tolist() == [False, True, False, False] == grad.isnan().any(-1).tolist()
        loss, _ = T.preference_loss(T.Tape(), lg.view(4, 1, 30), torch.tensor([[0], [t], [1], [2]], device=DEV))
        assert loss.isnan()
    assert native.read_error()[0] == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("v", [600, 900, 2000, 4000, 4099, 40000])
def test_rows_of_few_words_that_can_be(v, dtype):
    """-inf everywhere but at three words, which few of a row's threads see, in rows that lie anywhere.  Against 64 bits, as rows far from zero."""
    g = torch.Generator().manual_seed(v)
    rows = [(level, place) for level in (0.0, -100.0, 100.0, -1e6, 1e6) for place in (0, 130, v // 2, v - 3)]
    x, targets = torch.full((len(rows), v), float("-inf")), torch.tensor([place + 1 for _, place in rows])
    for row, (level, place) in zip(x, rows):
        row[place:place + 3] = level + torch.randn(3, generator=g)
    x = x.to(dtype)
    wide, tape64 = x.double(), T.Tape()
    tape64.watch(wide)
    want, terms64 = T.policy_loss(tape64, wide, targets, torch.ones(len(rows)), scale=1.0)
    wgrad = tape64.backward(want)[id(wide)]
    here, tape = x.to(DEV), T.Tape()
    tape.watch(here)
    loss, terms = T.policy_loss(tape, here, targets.to(DEV), torch.ones(len(rows), device=DEV), scale=1.0)
    grad = tape.backward(loss)[id(here)].cpu()
    spread = (wide.amax(-1) - wide.gather(-1, targets[:, None])[:, 0]).abs()
    assert ((terms.logprobs.cpu() - terms64.logprobs).abs() <= spread * 2 ** -22 + _adds(v) * 2 ** -24 + terms64.logprobs.abs() * 2 ** -23).all()
    bound = _grad_bounds(x, terms64.weights.double(), torch.zeros(len(rows), dtype=torch.float64), v)
    assert torch.isfinite(grad).all() and ((grad.double() - wgrad).abs() <= bound).all() and not grad[x == float("-inf")].any()
    pairs = here.view(len(rows), 1, v)
    tape.watch(pairs)
    pref, seen = T.preference_loss(tape, pairs, targets.to(DEV)[:, None])
    pgrad = tape.backward(pref)[id(pairs)].view(len(rows), v).cpu()
    assert torch.isfinite(pref) and torch.isfinite(pgrad).all() and not pgrad[x == float("-inf")].any()
    assert torch.allclose(seen.logprobs, terms.logprobs, rtol=2 ** -22, atol=2 * _adds(v) * 2 ** -24)
    here.fill_(float("-inf"))                             # no word can be: no number
    tape.watch(here)
    loss, terms = T.policy_loss(tape, here, targets.to(DEV), torch.ones(len(rows), device=DEV), scale=1.0)
    assert loss.isnan() and terms.logprobs.isnan().all() and tape.backward(loss)[id(here)].isnan().all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("preference", [False, True])
def test_a_captured_backward_pass_of_an_eager_loss(preference, dtype):
    """Its gradient is multiplied in place, again at every replay, and its memory is the tape's, which lets go of it: refused.  Captured as a
    whole a pass gives the same at every replay."""
    logits, here, targets, mask, adv, _, _ = _inputs((2, 5), 900, dtype, 3)
    targets, adv, up = targets.to(DEV), adv.to(DEV), torch.tensor(0.5, device=DEV)

    def loss():
        tape = T.Tape()
        tape.watch(here)
        return tape, (T.preference_loss(tape, here, targets) if preference else T.policy_loss(tape, here, targets, adv, scale=1.0))[0]

    tape, l = loss()
    want = tape.backward(l, up)[id(here)].clone()
    for grad in (None, up):
        tape, l = loss()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            with pytest.raises(RuntimeError, match="captured with the forward pass"):
                tape.backward(l, grad)
            tape, l = loss()
            out = tape.backward(l, up)[id(here)]
        for _ in range(3):
            graph.replay()
            assert torch.equal(out, want)
    up.fill_(2.0)
    graph.replay()
    assert torch.equal(out, want * 4)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("v,offset", [(5, 1), (700, 0), (4096, 0), (4099, 3), (33000, 0)])
def test_gradients_of_targets_that_are_nearly_certain(v, offset, dtype):
    """The target's gradient is weight (p - 1), which is the others' share of the sum: relative to itself it has the roundings of that share's sum, of
    the quotient, the weight and the product (2^-24 each, 8 with what the weight is of), and the result's."""
    levels = torch.tensor([math.log((v - 1) / rest) for rest in (1e-1, 1e-3, 1e-5, 1e-7)])
    targets = torch.tensor([0, v - 1, v // 2, v // 3] * 2).view(2, 4)
    logits = torch.zeros(2, 4, v)
    logits.scatter_(-1, targets[..., None], levels[None, :, None].expand(2, 4, 1))
    logits = logits.to(dtype)
    here = torch.empty(logits.numel() + offset, dtype=dtype, device=DEV)[offset:].view(logits.shape).copy_(logits)
    tape, cpu, wide = T.Tape(), T.Tape(), logits.double()
    tape.watch(here), cpu.watch(wide)
    loss, _ = T.preference_loss(tape, here, targets.to(DEV), beta=0.5)
    want, _ = T.preference_loss(cpu, wide, targets, beta=0.5)
    grad, wgrad = tape.backward(loss)[id(here)].cpu().double(), cpu.backward(want)[id(wide)]
    # 64 bits of p - 1 leave 1e-16 of 1, 1e-9 of 1e-7
    got, exact = (t.gather(-1, targets[..., None]) for t in (grad, wgrad))
    half = 0.0 if dtype == torch.float32 else 2 ** -8
    assert ((got - exact).abs() <= exact.abs() * ((_adds(v) + 8) * 2 ** -24 + 2e-9 + half)).all()


@pytest.mark.parametrize("v", [9, 5000])
def test_margins_without_bounds(v):
    """A chosen or rejected word that cannot be (-inf): the side of the loss that has no share counts nothing, the other is infinite or 0."""
    inf = float("inf")
    for side, smooth, want in ((1, 0.0, 0.0), (1, 1.0, inf), (1, 0.5, inf), (0, 0.0, inf), (0, 1.0, 0.0), (0, 0.5, inf)):
        lg = torch.zeros(2, 3, v, device=DEV)
        lg[side, 1, 4] = -inf
        tape = T.Tape()
        tape.watch(lg)
        loss, terms = T.preference_loss(tape, lg, torch.full((2, 3), 4, device=DEV), beta=0.5, label_smoothing=smooth)
        assert float(loss) == want and float(terms.margins) == (inf if side else -inf)
        grad = tape.backward(loss)[id(lg)]
        assert torch.isfinite(grad).all() and bool(grad.any()) == (want == inf)
    lg[0, 0, 0] = NAN
    for smooth in (0.0, 0.5, 1.0):
        loss, terms = T.preference_loss(T.Tape(), lg, torch.full((2, 3), 4, device=DEV), label_smoothing=smooth)
        assert loss.isnan() and terms.margins.isnan().all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("v", [40, 900, 5000, 40000, 150000, 270000])
def test_targets_that_are_masked_with_a_low_value(v, dtype):
    """A target far below its row, with old and reference log-probabilities as low: the ratio is e to the minus of the other words' log-sum, of which
    64-bit numbers of that size keep something (2e-6 at 1e10) or nothing: at most 2, as a row's sum is of exponentials below the next power
    of two.  No weight but one of that size, no gradient without a number, and none of the target's p."""
    g = torch.Generator().manual_seed(v)
    x = torch.randn(6, v, generator=g).to(dtype)
    targets = torch.tensor([0, 1, 17, v // 2, v - 2, v - 1])
    for low in (-1e10, -1e30, torch.finfo(dtype).min):
        x[torch.arange(6), targets] = low
        same = x[torch.arange(6), targets].float().to(DEV)
        here, tape = x.to(DEV), T.Tape()
        tape.watch(here)
        loss, terms = T.policy_loss(tape, here, targets.to(DEV), torch.tensor([1.0, -1.0] * 3, device=DEV), scale=1.0, old_logprobs=same, ref_logprobs=same, kl_coef=0.1)
        grad = tape.backward(loss)[id(here)].cpu().double()
        rest = torch.logsumexp(x.double(), -1)
        assert torch.isfinite(loss) and (terms.logprobs.cpu() - same.cpu()).abs().le(same.cpu().abs() * 2 ** -23).all()
        assert (terms.ratio <= 2).all() and (terms.kl.abs() <= 1e6).all()
        if low == -1e10:
            assert torch.allclose(terms.ratio.cpu().double(), torch.exp(-rest), rtol=1e-5)
        w = terms.weights.cpu().double()
        p = torch.softmax(x.double(), -1)
        p[torch.arange(6), targets] -= 1.0
        assert torch.isfinite(w).all() and ((grad - w[:, None] * p).abs() <= _grad_bounds(x, w, w * 0, v)).all()
