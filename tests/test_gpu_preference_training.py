"""The losses, the scoring and activations in 8 bits as training steps use them together, on a B200."""
import pytest
import torch

from tilerl_b200 import rl
from tilerl_b200 import tape as T
from tilerl_b200.config import small_gpu
from tilerl_b200.ops import native, ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def model():
    from tilerl_b200.factory import build_model, make_ops
    m = build_model(small_gpu(), DEV, seed=0, ops=make_ops(DEV))
    g = torch.Generator().manual_seed(0)
    for k in m.add_lora(rank=8, alpha=16.0):
        if k.endswith("lora_b"):
            m.params[k].copy_(torch.randn(m.params[k].shape, generator=g) * 0.02)
    return m


def _batch(model, n=4, t=70):
    g = torch.Generator().manual_seed(n)
    ids = torch.randint(0, model.cfg.vocab, (n, t), generator=g).to(DEV)
    slens = [t - 9 * i for i in range(n)]
    return ids, [20] * n, slens


def test_policy_step_against_its_composition(model):
    """Weights from log-probabilities and a weighted cross-entropy over the same logits, as separate ops: the logits' gradients agree to fp32, then
    round to bf16 before the products, where a last bit may fall the other way: half a step, 2^-8, of some."""
    ids, plens, slens = _batch(model)
    mask, targets = rl._scored_mask(ids, plens, slens).to(DEV), torch.roll(ids, -1, 1)
    adv = torch.tensor([1.0, -1.0, 0.5, 0.2], device=DEV)
    refs, ent = rl.sequence_logprobs(model, ids, plens, slens, adapters=False, entropy=True)
    old = rl.sequence_logprobs(model, ids, plens, slens)
    assert (refs[mask] < 0).all() and (ent[mask] > 0).all() and not refs[~mask].any()
    before = native.launch_count
    st = rl.policy_step(model, ids, plens, slens, adv.cpu(), None, old_logprobs=old, ref_logprobs=refs, kl_coef=0.2, max_norm=0.0, return_grads=True)
    assert native.launch_count > before
    n = float(mask.sum())

    def weights(lg):
        lp = ref.token_logprobs(lg.reshape(-1, lg.shape[-1]).double(), targets.reshape(-1)).view(ids.shape)
        rho = torch.exp(lp - old)
        free = ~(((rho > 1.2) & (adv[:, None] > 0)) | ((rho < 0.8) & (adv[:, None] < 0)))
        return ((adv[:, None] * rho * free - 0.2 * (1 - torch.exp(refs - lp))) * mask / n).float()

    loss, grads, _ = rl.forward_backward(model, ids, targets, weights, trainable=model.trainable())
    assert abs(st["loss"] - loss) < 1e-4 * abs(loss) and st["kl"] > 0
    for k, g in grads.items():
        assert float((st["grads"][k] - g).norm()) <= 2 ** -8 * float(g.norm()), k
    assert native.read_error()[0] == 0


def test_a_preference_run_with_layers_in_8_bits(model):
    """Reference from the scoring kernel, loss, checkpointed layers kept in 8 bits, AdamW over micro-batches of pairs."""
    from tilerl_b200.optim import AdamW
    g = torch.Generator().manual_seed(3)
    tokens = lambda n: torch.randint(0, model.cfg.vocab, (n,), generator=g).tolist()
    pairs = [(tokens(8), tokens(5 + i), tokens(9 - i)) for i in range(4)]
    ids = rl.pad_batch([p + c for p, a, b in pairs for c in (a, b)]).to(DEV)
    plens, slens = [8] * 8, [8 + len(c) for _, a, b in pairs for c in (a, b)]
    refs = rl.sequence_logprobs(model, ids, plens, slens, adapters=False)
    grads = [rl.preference_step(model, ids, plens, slens, None, ref_logprobs=refs, max_norm=0.0, return_grads=True, checkpoint_layers=True, activation_bits=b)["grads"]
             for b in (32, 8)]
    assert set(grads[0]) == set(grads[1]) and all(torch.isfinite(x).all() for x in grads[1].values())
    kept = {k: v.clone() for k, v in model.trainable().items()}
    loop = rl.preference_loop(model, pairs, AdamW(model.trainable(), lr=1e-3), steps=3, pairs_per_step=4, device=DEV, micro=2, checkpoint_layers=True,
                              activation_bits=8)
    ms = list(loop)
    assert all(m["tokens"] == sum(len(a) + len(b) for _, a, b in pairs) for m in ms) and any(not torch.equal(v, kept[k]) for k, v in model.trainable().items())
    for k, v in model.trainable().items():
        v.copy_(kept[k])
    assert native.read_error()[0] == 0


def test_swiglu_rows_are_let_go_of(model):
    """Without checkpointing the feed-forwards' rows are kept in 8 bits: the step holds less by most of three quarters of them."""
    ids, plens, slens = _batch(model, 4, 256)
    cfg, held = model.cfg, []
    for bits in (32, 8):
        tape = T.Tape()
        tape.watch(*model.trainable().values())
        torch.cuda.synchronize()
        start = torch.cuda.memory_allocated()
        lg = model.forward_dense(tape, ids, activation_bits=bits)
        torch.cuda.synchronize()
        held.append(torch.cuda.memory_allocated() - start)
        del lg, tape
    rows = ids.numel() * 2 * cfg.ffn * cfg.n_layers
    assert held[0] - held[1] >= 0.9 * rows * (4 - 1 - 4 / 128)


def test_a_policy_scored_as_its_own_reference():
    """Adapters that add nothing, a head whose logits reach 20: a row's log-probabilities are the reference's but for the order of two fp32 sums of
    ``hidden`` products, each addition off by 2^-23 of the row's sum of |h w| at most (hidden / 16 + 2 of them in either form), as scoring is tested."""
    from tilerl_b200.factory import build_model, make_ops
    m = build_model(small_gpu(), DEV, seed=1, ops=make_ops(DEV))
    m.add_lora(rank=4, alpha=8.0)
    head = m.params["embed" if m.cfg.tie_embeddings else "lm_head"]
    ids, plens, slens = _batch(m, 4, 70)
    tape = T.Tape()
    tape.enabled = False
    with torch.no_grad():
        h, w, _ = m.forward_dense(tape, ids, return_hidden=True)
        head.mul_(20.0 / float((h.bfloat16().float() @ w.float().t()).abs().max()))
        size = (h.bfloat16().double().abs() @ w.double().abs().t()).amax(-1)
    off = 4 * size * (h.shape[-1] / 16 + 2) * 2 ** -23 + 1e-5      # of a log-probability: its logit's and the sum's, in both forms
    assert float(off.max()) < 0.02
    mask = rl._scored_mask(ids, plens, slens).to(DEV)
    refs = rl.sequence_logprobs(m, ids, plens, slens, adapters=False)
    assert torch.equal(refs, rl.sequence_logprobs(m, ids, plens, slens))
    lg = m.forward_dense(T.Tape(), ids)
    assert 19.0 < float(lg.abs().max()) < 21.0
    _, terms = T.policy_loss(T.Tape(), lg, torch.roll(ids, -1, 1), torch.ones(4, device=DEV), scale=1.0, mask=mask, old_logprobs=refs, ref_logprobs=refs)
    d = (terms.logprobs - refs).abs()
    assert (d <= off).all() and (terms.kl <= off * off).all() and ((terms.ratio - 1).abs()[mask] <= 2 * off[mask]).all()
    st = rl.policy_step(m, ids, plens, slens, torch.ones(4), None, old_logprobs=refs, ref_logprobs=refs, kl_coef=0.1)
    assert st["kl"] <= float(off.max()) ** 2 and st["clipped"] == 0
    st = rl.preference_step(m, ids, plens, slens, None, ref_logprobs=refs, beta=0.1)
    assert abs(st["margin"]) <= 0.1 * float((off * mask).sum())
    # (each product of the chunked head is as long as that of the whole one)
    tape = T.Tape()
    _, lp = T.linear_cross_entropy(tape, h, w, torch.roll(ids, -1, 1), torch.zeros_like, chunk=100)
    assert ((lp - refs).abs()[mask] <= off[mask]).all()


def test_a_reference_with_a_quantised_head():
    """The head of a training forward may be quantised; its words are scored as what it stands for."""
    import dataclasses
    from tilerl_b200.factory import build_model, make_ops
    m = build_model(dataclasses.replace(small_gpu(), lm_head_quant="nvfp4"), DEV, seed=0, ops=make_ops(DEV))
    m.add_lora(rank=4, alpha=8.0)
    ids, plens, slens = _batch(m)
    tape = T.Tape()
    tape.enabled = False
    h, w, _ = m.forward_dense(tape, ids, return_hidden=True)
    assert hasattr(w, "wq")
    mask, targets = rl._scored_mask(ids, plens, slens).to(DEV), torch.roll(ids, -1, 1)
    want, went = T.linear_logprobs(h, w.dequant().to(DEV, torch.bfloat16), targets, mask=mask, entropy=True)
    got, gent = rl.sequence_logprobs(m, ids, plens, slens, adapters=False, entropy=True)
    assert torch.equal(got, want) and torch.equal(gent, went)
    st = next(iter(rl.preference_loop(m, [([1, 2], [3, 4, 5], [6, 7])], None, steps=1, device=DEV)))
    assert abs(st["margin"]) < 1e-3
