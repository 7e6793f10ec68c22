"""Policy and preference losses, scoring and activations in 8 bits on the CPU: definitions, gradients, refusals."""
import gc
import math
import weakref

import pytest
import torch

from tilerl_b200 import tape as T
from tilerl_b200.ops import keep

NAN = float("nan")


def _logprob(row, t):
    m = max(row)
    return row[t] - m - math.log(sum(math.exp(x - m) for x in row))


def _policy(logits, targets, adv, scale, mask, old, ref, lo, hi, kl):
    """The definition in plain Python: loss, and terms of a row."""
    total, terms = 0.0, []
    for i, row in enumerate(logits):
        if not mask[i]:
            terms.append((0.0, 0.0, 0.0, False))
            continue
        lp = _logprob(row, targets[i])
        rho = math.exp(lp - old[i]) if old is not None else 1.0
        clip = min(max(rho, 1 - lo), 1 + hi)
        d = ref[i] - lp if ref is not None else 0.0
        k3 = math.exp(d) - d - 1
        total += -min(rho * adv[i], clip * adv[i]) + kl * k3
        terms.append((lp, rho, k3, (rho > 1 + hi and adv[i] > 0) or (rho < 1 - lo and adv[i] < 0)))
    return total * scale, terms


def _inputs(n, v, seed):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)
    logits, targets = r(n, v) * 2, torch.randint(0, v, (n,), generator=g)
    lp = torch.log_softmax(logits, -1).gather(-1, targets[:, None])[:, 0]
    mask = torch.rand(n, generator=g) < 0.7
    return logits, targets, mask, r(n), lp + 0.4 * r(n), lp + 0.3 * r(n)


@pytest.mark.parametrize("n,v,old,ref,kl,hi", [(1, 1, True, True, 0.1, None), (7, 2, True, False, 0.0, 0.4), (40, 11, True, True, 0.2, 0.28), (5, 300, False, True, 0.0, None),
                                             (6, 9, False, False, 0.0, None)])
def test_policy_loss_is_its_definition_and_the_gradient_its_differences(n, v, old, ref, kl, hi):
    """64 bits: the value to 1e-12; central differences with steps of 1e-6 leave 1e-9 of curvature and 1e-9 of rounding (no row's ratio lies
    within 1e-4 of the clipping's border, where there is no derivative)."""
    logits, targets, mask, adv, olds, refs = _inputs(n, v, n + v)
    mask[0] = True
    adv[-1] = 0.0
    kw = dict(scale=0.3, mask=mask, old_logprobs=olds if old else None, ref_logprobs=refs if ref else None, clip_eps=0.2, clip_eps_high=hi, kl_coef=kl)
    plain = lambda lg: _policy(lg.tolist(), targets.tolist(), adv.tolist(), 0.3, mask.tolist(), olds.tolist() if old else None, refs.tolist() if ref else None,
                               0.2, 0.2 if hi is None else hi, kl)
    tape = T.Tape()
    tape.watch(logits)
    loss, terms = T.policy_loss(tape, logits, targets, adv, **kw)
    want, rows = plain(logits)
    assert abs(float(loss) - want) < 1e-12 * max(1, abs(want))
    for got, k in ((terms.logprobs, 0), (terms.ratio, 1), (terms.kl, 2)):
        assert torch.allclose(got, torch.tensor([r[k] if m else 0.0 for r, m in zip(rows, mask)], dtype=torch.float64), atol=1e-12)
    assert terms.clipped.tolist() == [r[3] for r in rows]
    assert not old or all(abs(r[1] - e) > 1e-4 for r in rows for e in (0.8, 1.2, 1.4, 1.28))
    grad = tape.backward(loss)[id(logits)]
    for i in range(n):
        for c in range(min(v, 12)):
            up, down = logits.clone(), logits.clone()
            up[i, c] += 1e-6
            down[i, c] -= 1e-6
            # (without old ones the ratio is the constant 1, and the gradient that of the log-probability: minus weights times its slope)
            if old:
                slope = (plain(up)[0] - plain(down)[0]) / 2e-6
            else:
                f = lambda lg: _logprob(lg[i].tolist(), int(targets[i]))
                slope = -float(terms.weights[i]) * (f(up) - f(down)) / 2e-6
            assert abs(float(grad[i, c]) - slope) < 5e-8, (i, c)
    if not old and not ref:
        assert torch.allclose(terms.weights, torch.where(mask, adv * 0.3, 0.0))


def test_rows_that_are_not_scored_may_hold_anything():
    """NaN and infinite logits, targets of -100, unusable old ones: zeros come back; nothing scored at all: a loss of 0."""
    logits, targets, mask, adv, olds, refs = _inputs(12, 7, 3)
    mask[:6], mask[6:] = True, False
    logits[6], logits[7], logits[8] = NAN, float("-inf"), torch.finfo(torch.float64).min
    logits[9, 2] = float("inf")
    targets[6:], olds[6:], refs[6:], adv[6:] = -100, NAN, float("inf"), NAN
    tape = T.Tape()
    tape.watch(logits)
    loss, terms = T.policy_loss(tape, logits, targets, adv, scale=1.0, mask=mask, old_logprobs=olds, ref_logprobs=refs, kl_coef=0.1)
    short = T.policy_loss(T.Tape(), logits[:6], targets[:6], adv[:6], scale=1.0, old_logprobs=olds[:6], ref_logprobs=refs[:6], kl_coef=0.1)
    assert abs(float(loss) - float(short[0])) < 1e-14 * 12         # (the same terms, below 8 each, in another order: 12 x 8 x 2^-53)
    for got, want in zip(terms, short[1]):
        assert torch.equal(got[:6], want) and not got[6:].any()
    assert not tape.backward(loss)[id(logits)][6:].any()
    loss, _ = T.policy_loss(tape, logits, targets, adv, scale=1.0, mask=torch.zeros(12, dtype=torch.bool), old_logprobs=olds)
    assert float(loss) == 0.0
    lg = logits.view(2, 6, 7)
    tape.watch(lg)
    pair, terms = T.preference_loss(tape, lg, targets.view(2, 6), mask.view(2, 6), refs.view(2, 6))
    assert math.isfinite(float(pair)) and float(terms.logprobs[1]) == 0.0
    grad = tape.backward(pair)[id(lg)]
    assert torch.isfinite(grad).all() and grad[0].any() and not grad[1].any()


def test_unscored_values_at_the_ends_of_fp32_and_no_rows():
    lg = torch.full((2, 5), torch.finfo(torch.float32).min)
    lg[0, 1] = 0.0
    tape = T.Tape()
    tape.watch(lg)
    loss, terms = T.policy_loss(tape, lg, torch.tensor([1, 0]), torch.tensor([1.0, 1.0]), scale=1.0)
    assert terms.logprobs.tolist() == pytest.approx([0.0, -math.log(5)]) and torch.isfinite(tape.backward(loss)[id(lg)]).all()
    none = torch.zeros(0, 3, 5)
    loss, terms = T.policy_loss(T.Tape(), none, torch.zeros(0, 3, dtype=torch.long), torch.zeros(0), scale=1.0)
    assert float(loss) == 0.0 and terms.kl.shape == (0, 3)
    assert float(T.preference_loss(T.Tape(), none, torch.zeros(0, 3, dtype=torch.long))[0]) == 0.0
    empty = torch.zeros(2, 0, 5)
    assert float(T.preference_loss(T.Tape(), empty, torch.zeros(2, 0, dtype=torch.long))[0]) == pytest.approx(math.log(2))


@pytest.mark.parametrize("t,v,smooth,average,with_ref", [(1, 2, 0.0, False, True), (5, 7, 0.1, False, True), (4, 20, 0.3, True, True), (3, 6, 0.0, True, False)])
def test_preference_loss_is_its_definition_and_the_gradient_its_differences(t, v, smooth, average, with_ref):
    pairs = 3
    logits, targets, mask, _, _, refs = _inputs(2 * pairs * t, v, t * v)
    logits, targets, mask, refs = logits.view(-1, t, v), targets.view(-1, t), mask.view(-1, t), refs.view(-1, t)
    mask[0] = True
    mask[-1] = False

    def plain(lg):
        ratios, sums = [], []
        for i in range(2 * pairs):
            on = [j for j in range(t) if mask[i, j]]
            lps = [_logprob(lg[i, j].tolist(), int(targets[i, j])) for j in on]
            k = max(1, len(on)) if average else 1
            ratios.append(sum(lp - (float(refs[i, j]) if with_ref else 0.0) for lp, j in zip(lps, on)) / k)
            sums.append(sum(lps) / k)
        zs = [0.7 * (ratios[2 * p] - ratios[2 * p + 1]) for p in range(pairs)]
        sig = lambda z: 1 / (1 + math.exp(-z))
        return sum(-(1 - smooth) * math.log(sig(z)) - smooth * math.log(sig(-z)) for z in zs) / pairs, sums, zs

    tape = T.Tape()
    tape.watch(logits)
    loss, terms = T.preference_loss(tape, logits, targets, mask, refs if with_ref else None, beta=0.7, label_smoothing=smooth, average=average)
    want, sums, zs = plain(logits)
    assert abs(float(loss) - want) < 1e-12
    assert terms.logprobs.tolist() == pytest.approx(sums, abs=1e-12) and terms.margins.tolist() == pytest.approx(zs, abs=1e-12)
    grad = tape.backward(loss)[id(logits)]
    for i in range(2 * pairs):
        for j in range(t):
            for c in range(min(v, 4)):
                up, down = logits.clone(), logits.clone()
                up[i, j, c] += 1e-6
                down[i, j, c] -= 1e-6
                assert abs(float(grad[i, j, c]) - (plain(up)[0] - plain(down)[0]) / 2e-6) < 1e-8
    half, _ = T.preference_loss(T.Tape(), logits, targets, mask, refs if with_ref else None, beta=0.7, label_smoothing=smooth, average=average, scale=0.5 / pairs)
    assert float(half) == pytest.approx(want / 2, abs=1e-12)


def test_losses_refuse_what_they_do_not_take():
    lg, tg, adv = torch.zeros(2, 3, 5), torch.zeros(2, 3, dtype=torch.long), torch.zeros(2)
    ok = dict(scale=1.0)
    for bad in (dict(targets=tg[:, :2]), dict(targets=tg.float()), dict(advantages=torch.zeros(3)), dict(advantages=torch.zeros(2, dtype=torch.long)),
                dict(mask=torch.ones(2, 3)), dict(mask=torch.ones(2, dtype=torch.bool)), dict(old_logprobs=torch.zeros(2)), dict(ref_logprobs=tg),
                dict(kl_coef=0.1), dict(clip_eps=-0.1), dict(scale=NAN), dict(logits=tg), dict(logits=torch.zeros(2, 3, 0)), dict(clip_eps_high=-1.0)):
        with pytest.raises(ValueError):
            T.policy_loss(T.Tape(), **{**dict(logits=lg, targets=tg, advantages=adv), **ok, **bad})
    for bad in (dict(logits=torch.zeros(3, 3, 5), targets=torch.zeros(3, 3, dtype=torch.long)), dict(logits=lg[0], targets=tg[0]), dict(label_smoothing=1.5),
                dict(beta=NAN), dict(ref_logprobs=torch.zeros(2)), dict(mask=torch.ones(2, 3))):
        with pytest.raises(ValueError):
            T.preference_loss(T.Tape(), **{**dict(logits=lg, targets=tg), **bad})
    for f in (lambda t: T.policy_loss(t, lg, tg, adv, scale=1.0), lambda t: T.preference_loss(t, lg, tg)):
        with pytest.raises(ValueError):
            f(T.Tape(None, 2))
    h, w = torch.zeros(4, 6), torch.zeros(9, 6)
    for bad in (dict(w=torch.zeros(9, 5)), dict(targets=torch.zeros(3, dtype=torch.long)), dict(targets=torch.zeros(4)), dict(mask=torch.zeros(4)),
                dict(w=torch.zeros(9, 6, dtype=torch.long)), dict(h=torch.zeros(4, 6, dtype=torch.long)), dict(w=torch.zeros(0, 6))):
        with pytest.raises(ValueError):
            T.linear_logprobs(**{**dict(h=h, w=w, targets=torch.zeros(4, dtype=torch.long)), **bad})


def test_no_gradient_is_formed_where_none_is_wanted():
    lg = torch.randn(3, 5)
    tape = T.Tape()
    loss, _ = T.policy_loss(tape, lg, torch.zeros(3, dtype=torch.long), torch.ones(3), scale=1.0)
    assert not tape.nodes and math.isfinite(float(loss))


@pytest.mark.parametrize("rows,hidden,vocab", [((1,), 1, 1), ((2, 3), 7, 13), ((300,), 16, 40)])
def test_scoring_equals_log_softmax(rows, hidden, vocab):
    g = torch.Generator().manual_seed(hidden)
    h, w = torch.randn(*rows, hidden, generator=g, dtype=torch.float64), torch.randn(vocab, hidden, generator=g, dtype=torch.float64)
    tg, mask = torch.randint(0, vocab, rows, generator=g), torch.rand(rows, generator=g) < 0.5
    logp = torch.log_softmax(h @ w.t(), -1)
    lp, ent = T.linear_logprobs(h, w, tg, entropy=True)
    assert torch.allclose(lp, logp.gather(-1, tg[..., None])[..., 0], atol=1e-12)
    assert torch.allclose(ent, -(logp.exp() * logp).sum(-1), atol=1e-12)
    h[~mask], tg[~mask] = NAN, -1
    got = T.linear_logprobs(h, w, tg, mask=mask)
    assert torch.equal(got[mask], lp[mask]) and not got[~mask].any()
    assert T.linear_logprobs(h[:0], w, tg[:0]).shape == h[:0].shape[:-1]


# ---- 8 bits ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("shape", [(1,), (3, 127), (2, 2, 128), (4, 129), (1, 1000), (0, 5), (3, 0)])
def test_rows_in_8_bits(shape):
    """A value is off by half a step of its group at most: amax / 254, and fp32's roundings of the quotients, the product and the result (2^-22 of
    amax)."""
    x = torch.randn(shape, generator=torch.Generator().manual_seed(1)) * 3
    kept = T.keep8(x)
    back = kept.rows()
    assert kept.q.shape == back.shape == x.shape and kept.q.dtype == torch.int8 and kept.scale.shape == (*x.shape[:-1], -(-x.shape[-1] // 128))
    for a in range(0, shape[-1], 128):
        part, got = x[..., a:a + 128], back[..., a:a + 128]
        if part.numel():
            most = part.abs().amax(-1, keepdim=True)
            assert ((part - got).abs() <= most * (1 / 254 + 2 ** -22)).all()
            assert torch.equal(got.abs().amax(-1, keepdim=True), 127 * kept.scale[..., a // 128, None])


def test_groups_in_8_bits_that_are_out_of_range():
    x = torch.ones(6, 256)
    x[0, 3], x[1, 200], x[2] = NAN, float("-inf"), 0.0
    x[3, :128], x[4, :128] = 1e-37, 1e-40
    x[5, 7] = torch.finfo(torch.float32).max
    back = T.keep8(x).rows()
    assert back[0, :128].isnan().all() and (back[0, 128:] == 1).all() and back[1, 128:].isnan().all() and (back[1, :128] == 1).all()
    assert not back[2].any() and not back[3, :128].any() and not back[4, :128].any()
    assert torch.isfinite(back[5]).all() and float(back[5, 7]) == pytest.approx(torch.finfo(torch.float32).max, rel=1e-6)
    with pytest.raises(ValueError):
        T.keep8(x.double())
    with pytest.raises(ValueError):
        T.keep8(torch.tensor(1.0))


def _segment(w):
    return lambda tape, x: T.add(tape, x, T.swiglu(tape, T.linear(tape, T.rmsnorm(tape, x, torch.ones(x.shape[-1]), 1e-6), w)))


def test_segments_kept_in_8_bits_start_again_from_what_is_kept():
    """Three segments: the forward pass is the plain one, each segment's gradient that of the segment at what its packed input stands for, and no
    fp32 input of theirs is held but the watched one."""
    g = torch.Generator().manual_seed(0)
    ws = [torch.randn(80, 40, generator=g) * 0.2 for _ in range(3)]
    x0, up = torch.randn(5, 40, generator=g), torch.randn(5, 40, generator=g)
    tape, plain = T.Tape(), T.Tape()
    tape.watch(x0, *ws)
    xs, refs = [x0], []
    for w in ws:
        xs.append(tape.checkpoint(_segment(w), xs[-1], params=(w,), bits=8))
    y, want = xs[-1], x0
    for w in ws:
        want = plain.checkpoint(_segment(w), want, params=(w,))
    assert torch.equal(y, want)
    inputs = [x0] + [T.keep8(x).rows() for x in xs[1:-1]]
    refs = [weakref.ref(x) for x in xs[1:-1]]
    del xs, want
    gc.collect()
    assert all(r() is None for r in refs)
    got = tape.backward(y, up)
    for w, x in zip(reversed(ws), reversed(inputs)):
        one = T.Tape()
        one.watch(x, w)
        gs = one.backward(_segment(w)(one, x), up)
        assert torch.equal(got[id(w)], gs[id(w)])
        up = gs[id(x)]
    assert torch.equal(got[id(x0)], up)


def test_a_tensor_let_go_of_is_still_the_same_to_the_tape():
    """It may be read by further ops, watched again, and its number taken by another tensor."""
    x = torch.randn(4, 8)
    tape = T.Tape()
    tape.watch(x)
    h = T.scale(tape, x, 2.0)
    y = tape.checkpoint(lambda t, z: T.scale(t, z, 3.0), h, bits=8)
    z = T.add(tape, y, h)                     # h again, after the tape let go of it
    assert tape.wants(h)
    got = tape.backward(z, torch.ones_like(z))
    assert torch.equal(got[id(x)], torch.full_like(x, 8.0))
    tape = T.Tape()
    h = torch.randn(4, 8)
    y = tape.checkpoint(lambda t, z: T.scale(t, z, 3.0), h, bits=8)
    assert not tape.wants(h)
    tape.watch(h)
    assert torch.equal(tape.backward(y, torch.ones_like(y))[id(h)], torch.full_like(h, 3.0))
    tape = T.Tape()
    tape.watch(x)
    for _ in range(20):                       # tensors that come and go at the same addresses
        h = tape.checkpoint(lambda t, z: T.scale(t, z, 1.0), T.scale(tape, x, 1.0), bits=8)
        other = torch.randn(4, 8)
        assert not tape.wants(other)
        z = h
    assert torch.equal(tape.backward(z, torch.ones_like(z))[id(x)], torch.ones_like(x))


@pytest.mark.parametrize("shape", [(3, 10), (2, 5, 256), (7, 300)])
def test_swiglu_with_its_pairs_in_8_bits(shape):
    g = torch.Generator().manual_seed(2)
    gu, up = torch.randn(shape, generator=g), torch.randn(*shape[:-1], shape[-1] // 2, generator=g)
    sides = []
    for x, bits in ((gu, 8), (T.keep8(gu).rows(), 32)):
        tape = T.Tape()
        tape.watch(x)
        y = T.swiglu(tape, x, bits=bits)
        sides.append((y, tape.backward(y, up)[id(x)]))
    assert torch.equal(sides[0][0], T.swiglu(T.Tape(), gu)) and torch.equal(sides[0][1], sides[1][1])
    tape = T.Tape()
    tape.watch(up)
    h = T.scale(tape, gu, 1.0)
    seen = weakref.ref(h)
    y = T.swiglu(tape, h, bits=8)
    del h
    gc.collect()
    assert seen() is None
    for bad in (dict(bits=4), dict(gu=gu.double()), dict(gu=gu[..., :-1])):
        with pytest.raises(ValueError):
            T.swiglu(T.Tape(), **{**dict(gu=gu, bits=8), **bad})
    with pytest.raises(ValueError):
        T.Tape().checkpoint(lambda t, z: z, gu, bits=16)


def test_packed_bytes_by_hand():
    q, scale = keep.pack(torch.tensor([[127.0, -63.5, 0.4, 0.5, 1.5, -126.6]]))
    assert q.tolist() == [[127, -64, 0, 0, 2, -127]] and scale.tolist() == [[1.0]]        # ties go to the even one


def test_a_segment_that_hands_on_its_input():
    """What goes in is what comes out: the tape lets go of both, and the gradient goes on to the op that made it."""
    x = torch.randn(3, 200, generator=torch.Generator().manual_seed(1))
    tape = T.Tape()
    tape.watch(x)
    h = T.scale(tape, x, 2.0)
    y = tape.checkpoint(lambda t, z: z, h, bits=8)
    z = T.scale(tape, tape.checkpoint(lambda t, z: z, y, bits=8), 3.0)
    grads = tape.backward(z, torch.ones_like(z))
    assert torch.equal(grads[id(x)], torch.full_like(x, 6.0))


def test_targets_outside_of_the_vocabulary_in_the_torch_forms(monkeypatch):
    """Where an index out of range is no error (the torch forms on a GPU, for types and widths that the kernels do not take) nothing is indexed with one:
    its row has no number, in the losses and the log-probabilities, and no other row differs."""
    from tilerl_b200.ops import ref
    g = torch.Generator().manual_seed(0)
    logits, adv, mask = torch.randn(6, 9, generator=g, dtype=torch.float64), torch.randn(6, generator=g, dtype=torch.float64), torch.tensor([1, 1, 1, 0, 1, 1]).bool()
    targets, h, w = torch.tensor([0, 8, 3, 4, 5, 1]), torch.randn(6, 7, generator=g), torch.randn(9, 7, generator=g)

    def forms(tg):
        tape, pairs = T.Tape(), logits.view(2, 3, 9)
        tape.watch(logits, pairs)
        loss, terms = T.policy_loss(tape, logits, tg, adv, scale=0.5, mask=mask)
        grad = tape.backward(loss)[id(logits)]
        pref, seen = T.preference_loss(tape, pairs, tg.view(2, 3), mask.view(2, 3))
        return loss, terms, grad, pref, seen, tape.backward(pref)[id(pairs)], *T.linear_logprobs(h, w, tg, mask=mask, entropy=True)

    loss, terms, grad, pref, seen, pgrad, lp, ent = forms(targets)
    for bad in (-1, 9, 1 << 40):
        tg = targets.clone()
        tg[1], tg[3] = bad, bad                           # (row 3 is not scored)
        with pytest.raises((IndexError, RuntimeError)):
            forms(tg)
        with monkeypatch.context() as m:
            m.setattr(ref, "index_raises", lambda t: False)
            got = forms(tg)
        assert got[0].isnan() and got[1].logprobs.isnan().tolist() == [False, True] + [False] * 4 == got[2].isnan().any(-1).tolist()
        rest = [0, 2, 3, 4, 5]
        assert torch.equal(got[2][rest], grad[rest]) and torch.equal(got[1].logprobs[rest], terms.logprobs[rest]) and got[2][1].isnan().all()
        assert got[3].isnan() and got[4].logprobs.isnan().tolist() == [True, False] and got[5][mask.view(2, 3)].isnan().all() and not got[5][~mask.view(2, 3)].any()
        assert torch.equal(got[4].logprobs[1], seen.logprobs[1])
        assert got[6].isnan().tolist() == [False, True] + [False] * 4 and torch.equal(got[6][rest], lp[rest]) and torch.equal(got[7], ent)
    assert ref.within(targets, 9) == (targets, None)


@pytest.mark.parametrize("mask", [None, torch.zeros(4, 0, dtype=torch.bool)])
@pytest.mark.parametrize("average", [False, True])
def test_pairs_of_sequences_without_tokens(average, mask):
    """Log ratios of 0, sums as means: log 2 a pair."""
    tape, logits = T.Tape(), torch.zeros(4, 0, 5)
    tape.watch(logits)
    loss, terms = T.preference_loss(tape, logits, torch.zeros(4, 0, dtype=torch.long), mask, average=average)
    assert abs(float(loss) - math.log(2.0)) < 1e-6 and terms.logprobs.tolist() == [0.0] * 4 and terms.margins.tolist() == [0.0] * 2
    assert tape.backward(loss)[id(logits)].shape == (4, 0, 5)


def test_margins_without_bounds():
    """A chosen or rejected word that cannot be (-inf): the side of the loss that has no share counts nothing, the other is infinite or 0."""
    inf = float("inf")
    for side, smooth, want in ((1, 0.0, 0.0), (1, 1.0, inf), (1, 0.5, inf), (0, 0.0, inf), (0, 1.0, 0.0), (0, 0.5, inf)):
        lg = torch.zeros(2, 3, 9)
        lg[side, 1, 4] = -inf
        tape = T.Tape()
        tape.watch(lg)
        loss, terms = T.preference_loss(tape, lg, torch.full((2, 3), 4), beta=0.5, label_smoothing=smooth)
        assert float(loss) == want and float(terms.margins) == (inf if side else -inf)
        grad = tape.backward(loss)[id(lg)]
        assert torch.isfinite(grad).all() and bool(grad.any()) == (want == inf)
    lg[0, 0, 0] = NAN
    for smooth in (0.0, 0.5, 1.0):
        loss, terms = T.preference_loss(T.Tape(), lg, torch.full((2, 3), 4), label_smoothing=smooth)
        assert loss.isnan() and terms.margins.isnan().all()
