"""Scoring of tokens from hidden rows and the head on a B200 against 64 bits."""
import pytest
import torch

from tilerl_b200 import tape as T
from tilerl_b200.ops import native, score

pytestmark = pytest.mark.gpu
DEV = "cuda"
NAN = float("nan")


def _inputs(rows, hidden, vocab, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    h = torch.randn(*rows, hidden, generator=g, device=DEV).bfloat16()
    w = (torch.randn(vocab, hidden, generator=g, device=DEV) * 0.1).bfloat16()
    return h, w, torch.randint(0, vocab, rows, generator=g, device=DEV), torch.rand(rows, generator=g, device=DEV) < 0.6


def _exact(h, w, tg):
    logp = torch.log_softmax(h.double() @ w.double().t(), -1)
    return logp.gather(-1, tg[..., None])[..., 0], -(logp.exp() * logp).sum(-1)


def _bound(h, w):
    """What fp32 sums of the products may be off, a logit: the tensor cores cut each addition off at 2^-23 or so of the largest magnitude in
    play, for which a row's sum of |h w| stands: hidden / 16 additions of 16 terms at once, but never more than 2^-12 of it."""
    size = (h.double().abs() @ w.double().abs().t()).amax(-1)
    return size * min(h.shape[-1] / 16 + 2, 2 ** 11) * 2 ** -23 + 2e-6


@pytest.mark.parametrize("rows,hidden,vocab", [((1,), 8, 1), ((2, 3), 16, 7), ((5,), 64, 128), ((32,), 264, 8193), ((33,), 264, 8193), ((130,), 72, 129), ((3, 43), 256, 1000), ((257,), 128, 320), ((1,), 1024, 32768), ((300,), 520, 4099),
                                             ((2100,), 64, 700), ((33,), 5120, 9000)])
def test_scoring(rows, hidden, vocab):
    """One row, rows and words to either side of a tile, more rows than go through the words together, hidden sizes that end inside a k-block."""
    h, w, tg, mask = _inputs(rows, hidden, vocab, hidden + vocab)
    want, went = _exact(h, w, tg)
    before = native.launch_count
    lp, ent = T.linear_logprobs(h, w, tg, entropy=True)
    assert native.launch_count == before + 2 and score.takes(h, w)
    assert ((lp - want).abs() <= 2 * _bound(h, w) + want.abs() * 2 ** -23).all()
    # a logit's error moves the entropy by p (log p + H) of it, whose sum over the words is the deviation of log p: below 1 + log(vocab) here
    assert ((ent - went).abs() <= 10 * _bound(h, w) + went.abs() * 2 ** -22).all()
    assert torch.equal(T.linear_logprobs(h, w, tg), lp)
    got, gent = T.linear_logprobs(h.float(), w, tg, mask=mask, entropy=True)          # (the rows round to what they were)
    assert torch.equal(got, torch.where(mask, lp, 0.0)) and torch.equal(gent, torch.where(mask, ent, 0.0))
    assert native.read_error()[0] == 0


def test_rows_that_are_not_scored_are_not_looked_at():
    h, w, tg, mask = _inputs((600,), 128, 500, 0)
    mask[:300] = False
    want = torch.where(mask, T.linear_logprobs(h, w, tg), 0.0)
    h[~mask], tg[~mask] = NAN, 1 << 40
    for x in (h, h.float()):
        assert torch.equal(T.linear_logprobs(x, w, tg, mask=mask), want)
        lp, ent = T.linear_logprobs(x, w, tg, mask=torch.zeros_like(mask), entropy=True)
        assert not lp.any() and not ent.any()
    assert native.read_error()[0] == 0


def test_targets_outside_of_the_vocabulary_and_values_without_a_number():
    h, w, tg, _ = _inputs((4,), 64, 300, 1)
    for t in (-1, 300, 511, 1 << 40):
        tg[1] = t
        assert T.linear_logprobs(h, w, tg).isnan().tolist() == [False, True, False, False]
        code, site, _, n = native.read_error()
        assert (code, site, n) == (2, 17, 300)
    tg[1] = 0
    h[2, 5], w[7, 3] = NAN, 0.0
    lp, ent = T.linear_logprobs(h, w, tg, entropy=True)
    assert lp.isnan().tolist() == [False, False, True, False] == ent.isnan().tolist()
    h[2, 5] = 0.0
    w[7], h[:, 0] = 0.0, torch.tensor([2.0, -2.0, 0.5, 0.0], device=DEV)      # logits of +-inf: NaN for a row that has +inf, as softmax
    w[7, 0] = torch.finfo(torch.bfloat16).max
    logits = h.float() @ w.float().t()
    lp = T.linear_logprobs(h, w, tg)
    want = torch.log_softmax(logits, -1).gather(-1, tg[:, None])[:, 0]
    assert torch.equal(torch.isfinite(lp), torch.isfinite(want) & ~(logits == float("inf")).any(-1))


def test_forms_in_torch():
    """Hidden sizes that no copy can begin at, heads in fp32 (rounded, as the training head is), views, no rows."""
    h, w, tg, mask = _inputs((9,), 20, 50, 2)
    want, went = _exact(h, w, tg)
    lp, ent = T.linear_logprobs(h, w, tg, entropy=True, mask=mask)
    assert not score.takes(h, w)
    assert torch.allclose(lp.double(), torch.where(mask, want, 0.0), atol=1e-5) and torch.allclose(ent.double(), torch.where(mask, went, 0.0), atol=1e-5)
    h, w, tg, _ = _inputs((3, 50), 64, 400, 3)
    lp = T.linear_logprobs(h, w, tg)
    assert torch.equal(T.linear_logprobs(h, w.float(), tg), lp)
    wide = torch.zeros(3, 50, 65, device=DEV, dtype=torch.bfloat16)
    wide[..., 1:] = h
    assert torch.equal(T.linear_logprobs(wide[..., 1:], w, tg), lp)
    assert T.linear_logprobs(h[:0], w, tg[:0]).shape == (0, 50)


def test_calls_of_many_rows_streams_and_graphs(monkeypatch):
    h, w, tg, mask = _inputs((700,), 64, 900, 4)
    want = T.linear_logprobs(h, w, tg, mask=mask)
    monkeypatch.setattr(score, "ROWS", 256)
    assert torch.equal(T.linear_logprobs(h, w, tg, mask=mask), want)
    monkeypatch.undo()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = T.linear_logprobs(h, w, tg, mask=mask)
    side.synchronize()
    assert torch.equal(got, want)
    static, smask = torch.zeros_like(h), torch.zeros_like(mask)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = T.linear_logprobs(static, w, tg, mask=smask)
    static.copy_(h), smask.copy_(mask)
    graph.replay()
    assert torch.equal(out, want)
    for _ in range(50):                                   # the same bits every time
        assert torch.equal(T.linear_logprobs(h, w, tg, mask=mask), want)
    assert native.read_error()[0] == 0


@pytest.mark.parametrize("n", [1, 3, 20, 32, 33, 255, 300])
def test_masks_that_begin_anywhere(n):
    """The scored rows' places are counted from the mask's words or bytes, by where it begins: none, all, the first, the last, some."""
    h, w, tg, _ = _inputs((n,), 64, 300, n)
    lp, ent = T.linear_logprobs(h, w, tg, entropy=True)
    g = torch.Generator(device=DEV).manual_seed(n)
    for offset in range(4):
        mask = torch.zeros(n + offset, dtype=torch.bool, device=DEV)[offset:]
        for on in (mask, ~mask, torch.arange(n, device=DEV) == 0, torch.arange(n, device=DEV) == n - 1, torch.rand(n, generator=g, device=DEV) < 0.5):
            mask.copy_(on)
            for x in (h, h.float()):
                got, gent = T.linear_logprobs(x, w, tg, mask=mask, entropy=True)
                assert torch.equal(got, torch.where(on, lp, 0.0)) and torch.equal(gent, torch.where(on, ent, 0.0))


@pytest.mark.parametrize("vocab", [1, 31, 1024, 32768, 33001])
def test_few_rows_with_values_without_a_number(vocab):
    """Logits of infinity and NaN of a hidden row's, words on their own far above the others, in every block's part of the words."""
    w = torch.zeros(vocab, 16, device=DEV)
    w[:, 0] = 1.0
    places = sorted({0, vocab // 3, vocab // 2, vocab - 1})
    for k, c in enumerate(places):
        w[c, 1 + k] = 1.0
    h = torch.zeros(len(places) + 2, 16, device=DEV)
    for k in range(len(places)):
        h[k, 1 + k] = 60.0                    # the word is all of the row: e^-60 for each of the others
    h[-2, 0], h[-1, 0] = NAN, float("inf")
    tg = torch.tensor(places + [0, 0], device=DEV)
    lp, ent = T.linear_logprobs(h.bfloat16(), w.bfloat16(), tg, entropy=True)
    assert (lp[:-2].abs() <= 1e-15).all() and (ent[:-2].abs() <= 1e-15).all() if vocab > 1 else not lp[:-2].any()
    assert lp[-2:].isnan().all() and ent[-2:].isnan().all()


def test_targets_outside_of_the_vocabulary_in_the_torch_form():
    """As from the kernels, but for the error word: nothing is indexed with such a target."""
    for hidden, dtype in ((20, torch.bfloat16), (64, torch.float16), (64, torch.float64)):
        h, w, tg, _ = _inputs((300,), hidden, 50, 5)
        h = h.to(dtype)
        assert not score.takes(h, w)
        want, went = T.linear_logprobs(h, w, tg, entropy=True)
        for t in (-1, 50, 1 << 40):
            bad = tg.clone()
            bad[7], bad[299] = t, t
            lp, ent = T.linear_logprobs(h, w, bad, entropy=True)
            assert lp.isnan().nonzero()[:, 0].tolist() == [7, 299] and torch.equal(torch.where(lp.isnan(), want, lp), want) and torch.equal(ent, went)
    assert native.read_error()[0] == 0
