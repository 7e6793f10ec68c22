"""Preference training, reference policies and activations in 8 bits through the training loops, on the CPU."""
import json

import pytest
import torch

from helpers import autograd_forward, make_engine, rand_prompts
from tilerl_b200 import cli, rl
from tilerl_b200 import tape as T
from tilerl_b200.config import tiny, tiny_hybrid
from tilerl_b200.models.hybrid import HybridModel
from tilerl_b200.ops import keep
from tilerl_b200.optim import AdamW


def _adapters(model, seed=0, scale=0.05):
    g = torch.Generator().manual_seed(seed)
    for k in model.add_lora(rank=4, alpha=8.0):
        if k.endswith("lora_b"):
            model.params[k].copy_(torch.randn(model.params[k].shape, generator=g) * scale)
    return model


def _batch(cfg, seed=0):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, cfg.vocab, (4, 11), generator=g)
    return ids, [4, 4, 2, 2], [11, 9, 7, 3]


def _logprobs(model, ids, leaves=None):
    lg = autograd_forward(model, ids, leaves if leaves is not None else {k: v for k, v in model.trainable().items()})
    return torch.log_softmax(lg, -1).gather(-1, torch.roll(ids, -1, 1)[..., None])[..., 0]


def test_scored_tokens_and_base_model():
    model = _adapters(HybridModel.build_random(tiny_hybrid(), seed=4))
    ids, plens, slens = _batch(model.cfg)
    mask = rl._scored_mask(ids, plens, slens)
    lp, ent = rl.sequence_logprobs(model, ids, plens, slens, entropy=True, micro=3)
    want = torch.where(mask, _logprobs(model, ids), 0.0)
    assert torch.allclose(lp, want, atol=1e-4) and torch.equal(lp == 0, ~mask) and (ent[mask] > 0).all() and not ent[~mask].any()
    base = rl.sequence_logprobs(model, ids, plens, slens, adapters=False)
    plain = rl.sequence_logprobs(HybridModel.build_random(tiny_hybrid(), seed=4), ids, plens, slens)
    assert torch.equal(base, plain) and not torch.allclose(base, lp, atol=1e-3) and model.lora
    with pytest.raises(ValueError):
        rl.sequence_logprobs(model, ids[:0], [], [])


@pytest.mark.parametrize("micro,average,smooth", [(0, False, 0.0), (1, False, 0.2), (2, True, 0.0)])
def test_preference_step_gradients(micro, average, smooth):
    model = _adapters(HybridModel.build_random(tiny_hybrid(), seed=4))
    ids, plens, slens = _batch(model.cfg)
    refs = rl.sequence_logprobs(model, ids, plens, slens, adapters=False)
    st = rl.preference_step(model, ids, plens, slens, None, ref_logprobs=refs, beta=0.5, label_smoothing=smooth, average=average, micro=micro,
                            max_norm=0.0, return_grads=True)
    leaves = {k: v.detach().clone().requires_grad_(True) for k, v in model.trainable().items()}
    mask = rl._scored_mask(ids, plens, slens).float()
    gap = ((_logprobs(model, ids, leaves) - refs) * mask).sum(-1)
    if average:
        gap = gap / mask.sum(-1).clamp_min(1)
    z = 0.5 * (gap[0::2] - gap[1::2])
    loss = (-(1 - smooth) * torch.nn.functional.logsigmoid(z) - smooth * torch.nn.functional.logsigmoid(-z)).mean()
    assert abs(st["loss"] - float(loss.detach())) < 1e-5 and abs(st["margin"] - float(z.detach().mean())) < 1e-4 and st["accuracy"] == float((z > 0).float().mean())
    for k, g in zip(leaves, torch.autograd.grad(loss, list(leaves.values()))):
        assert torch.allclose(st["grads"][k], g, rtol=2e-3, atol=2e-6), k


def test_preference_step_refuses():
    model = HybridModel.build_random(tiny(), seed=1, keep_master=True)
    ids = torch.zeros(3, 5, dtype=torch.long)
    for kw in (dict(ids=ids), dict(ids=ids[:0]), dict(ids=ids[:2], fused_ce=True), dict(ids=ids[:2], tp_world=2)):
        with pytest.raises(ValueError):
            rl.preference_step(model, kw.pop("ids"), [1] * 3, [5] * 3, None, **kw)
    with pytest.raises(ValueError):
        next(rl.preference_loop(model, [], None, steps=1))
    with pytest.raises(ValueError):                       # no adapters to leave out
        next(rl.preference_loop(model, [([1], [2], [3])], None, steps=1))


def test_preference_loop_moves_adapters_from_the_base():
    model = HybridModel.build_random(tiny_hybrid(), seed=4)
    model.add_lora(rank=4, alpha=8.0)
    pairs = [([1, 2, 3], [4, 5], [6, 7, 8]), ([9, 1], [2], [3, 4, 5, 6]), ([5] * 4, [6] * 3, [])]
    before = {k: v.clone() for k, v in model.trainable().items()}
    ms = list(rl.preference_loop(model, pairs, AdamW(model.trainable(), lr=1e-3), steps=3, pairs_per_step=2, micro=1))
    assert len(ms) == 3 and abs(ms[0]["loss"] - 0.6931) < 1e-3 and abs(ms[0]["margin"]) < 1e-3          # (the base model to itself)
    assert all(torch.isfinite(torch.tensor(m["loss"])) for m in ms) and any(not torch.equal(v, before[k]) for k, v in model.trainable().items())


def test_grpo_with_a_kl_term_to_the_base_model():
    cfg = tiny_hybrid()
    eng = make_engine(cfg)
    _adapters(eng.model)
    kw = dict(steps=1, group=2, prompts_per_step=1, max_tokens=4, kl_coef=0.5)
    run = lambda **more: next(iter(rl.grpo_loop(eng, eng.model, rand_prompts(cfg, 1, 8), lambda p, c: float(c[0] % 7), None, **kw, **more)))
    plain, held = run(), run(reference="base")
    assert "kl" not in plain and held["kl"] > 0
    ids, plens, slens = _batch(cfg)
    refs, adv = rl.sequence_logprobs(eng.model, ids, plens, slens, adapters=False), torch.tensor([1.0, -1.0, 0.5, 0.0])
    st = rl.policy_step(eng.model, ids, plens, slens, adv, None, ref_logprobs=refs, kl_coef=0.3, max_norm=0.0, return_grads=True)
    leaves = {k: v.detach().clone().requires_grad_(True) for k, v in eng.model.trainable().items()}
    mask = rl._scored_mask(ids, plens, slens).float()
    lp = _logprobs(eng.model, ids, leaves)
    d = (refs - lp) * mask
    loss = ((-torch.exp(lp - lp.detach()) * adv[:, None] + 0.3 * (torch.exp(d) - d - 1)) * mask).sum() / mask.sum()
    assert abs(st["objective"] - float(loss.detach())) < 1e-5 and abs(st["kl"] - float(((torch.exp(d) - d - 1) * mask).sum().detach() / mask.sum())) < 1e-5
    for k, g in zip(leaves, torch.autograd.grad(loss, list(leaves.values()))):
        assert torch.allclose(st["grads"][k], g, rtol=2e-3, atol=2e-6), k
    with pytest.raises(ValueError):
        run(reference="other")


@pytest.mark.parametrize("checkpoint", [False, True])
def test_steps_with_activations_in_8_bits(checkpoint, monkeypatch):
    """The forward pass is the same; gradients have the bits of those of plain ops that go back at what packed rows stand for."""
    model = _adapters(HybridModel.build_random(tiny_hybrid(), seed=4))
    ids, plens, slens = _batch(model.cfg)
    step = lambda b: rl.policy_step(model, ids, plens, slens, torch.tensor([1.0, -1.0, 0.5, -0.25]), None, return_grads=True, max_norm=0.0,
                                    checkpoint_layers=checkpoint, activation_bits=b)
    full, small = step(32), step(8)
    assert full["loss"] == small["loss"] and any(not torch.equal(g, small["grads"][k]) for k, g in full["grads"].items())
    stands_for = lambda t: keep.unpack(*keep.pack(t))
    used = []

    def swiglu(tape, gu, bits=32):
        used.append(bits)
        out, _ = T._swiglu_torch(gu)
        _, back = T._swiglu_torch(stands_for(gu) if not checkpoint else gu)
        tape.record("swiglu", (gu,), (out,), back)
        return out

    def segment(tape, fn, x, params=(), bits=32):
        used.append(bits)
        tape.enabled, was = False, tape.enabled
        out = fn(tape, x)
        tape.enabled = was
        again = stands_for(x)

        def back(g):
            sub = T.Tape()
            sub.watch(again, *params)
            gs = sub.backward(fn(sub, again), g)
            return tuple(gs.get(id(t)) for t in (again, *params))
        tape.record("checkpoint", (x, *params), (out,), back)
        return out

    with monkeypatch.context() as m:
        m.setattr(T, "swiglu", swiglu)
        m.setattr(T.Tape, "checkpoint", segment)
        want = step(32)
    assert used
    for k, g in want["grads"].items():
        assert torch.equal(g, small["grads"][k]), k
    with pytest.raises(ValueError):
        model.forward_dense(T.Tape(), ids, activation_bits=16)


def test_train_preference_command(tmp_path, capsys, monkeypatch):
    monkeypatch.setenv("TRL_RUNS", str(tmp_path / "runs"))
    data = tmp_path / "pairs.jsonl"
    data.write_text("".join(json.dumps(dict(prompt=f"q{i}", chosen="yes", rejected="no, never")) + "\n" for i in range(3)))
    base = ["train", "--model", "tiny", "--device", "cpu", "--steps", "2", "--lora-rank", "2", "--preference", "--data", str(data)]
    assert cli.main(base + ["--beta", "0.2", "--checkpoint-layers", "--activation-bits", "8"]) == 0
    rows = [json.loads(ln) for ln in capsys.readouterr().out.splitlines() if ln.startswith("{")]
    assert [r["step"] for r in rows if "margin" in r] == [0, 1]
    assert cli.main(["train", "--model", "tiny", "--device", "cpu", "--rl", "--steps", "1", "--group", "2", "--prompts-per-step", "1", "--max-tokens", "3", "--lora-rank",
                     "2", "--kl-coef", "0.1", "--kl-reference", "base", "--allow-short-rollouts"]) == 0
    assert "\"kl\"" in capsys.readouterr().out
    data.write_text(json.dumps(dict(prompt="q", chosen="yes")) + "\n")
    for bad in (base, base[:-2], base + ["--rl"], base[:-3] + ["--kl-reference", "base"]):
        with pytest.raises(SystemExit):
            cli.main(bad + ["--force"])


def test_a_reference_with_a_quantised_head():
    """The head that a training forward takes may be quantised: its words are scored as what it stands for."""
    import dataclasses
    model = HybridModel.build_random(dataclasses.replace(tiny_hybrid(), lm_head_quant="nvfp4", tie_embeddings=False), seed=4)
    model.add_lora(rank=2)
    head = model.params["lm_head"]
    assert hasattr(head, "wq")
    ids, plens, slens = _batch(model.cfg)
    mask, tape = rl._scored_mask(ids, plens, slens), T.Tape()
    lp, ent = rl.sequence_logprobs(model, ids, plens, slens, adapters=False, entropy=True, micro=3)
    want = torch.log_softmax(model.forward_dense(tape, ids), -1)
    assert torch.allclose(lp, torch.where(mask, want.gather(-1, torch.roll(ids, -1, 1)[..., None])[..., 0], 0.0), atol=1e-5)
    assert torch.allclose(ent, torch.where(mask, -(want.exp() * want).sum(-1), 0.0), atol=1e-5)
    m = next(iter(rl.preference_loop(model, [([1, 2], [3, 4, 5], [6])], None, steps=1)))
    assert abs(m["margin"]) < 1e-4
    h = torch.zeros(2, head.shape[1])
    assert torch.equal(T.linear_logprobs(h, head, torch.tensor([0, 1])), T.linear_logprobs(h, head.dequant(), torch.tensor([0, 1])))
    for x, w in ((h[:, :-1], head), (h, None), (h, [[0.0]]), (h, head.to("meta"))):       # (another width, no weight, another device)
        with pytest.raises(ValueError):
            T.linear_logprobs(x, w, torch.tensor([0, 1]))


def test_adapters_stay_in_place_while_the_base_model_is_scored():
    """What other threads compute, and what is read of the adapters or added to them meanwhile, is as outside of the block."""
    import threading
    model = _adapters(HybridModel.build_random(tiny_hybrid(), seed=4))
    ids, plens, slens = _batch(model.cfg)
    run = lambda: rl.sequence_logprobs(model, ids, plens, slens)
    own, base, names, seen = run(), rl.sequence_logprobs(model, ids, plens, slens, adapters=False), set(model.trainable()), []
    with model.without_adapters():
        other = threading.Thread(target=lambda: seen.append(run()))
        other.start()
        other.join()
        assert torch.equal(run(), base) and set(model.trainable()) == names and all(".lora_" in k for k in names)
        with model.without_adapters():
            assert torch.equal(run(), base)
        assert torch.equal(run(), base)                   # (the inner block's end is not the outer one's)
        model.add_lora(rank=1, targets=["down"], seed=1)
        assert torch.equal(run(), base)
    assert torch.equal(seen[0], own)
    narrow = [k for k, v in model.lora.items() if v[0].shape[0] == 1]
    assert narrow and all(k.endswith("down") for k in narrow) and not torch.equal(run(), own)      # (added adapters are there)
    with pytest.raises(ZeroDivisionError):
        with model.without_adapters():
            1 / 0
    assert not torch.equal(run(), base)


def test_weights_that_a_sharded_trainer_holds_are_not_scored():
    from tilerl_b200.parallel.zero3 import Zero3
    whole, model = (HybridModel.build_random(tiny_hybrid(), seed=4, keep_master=True) for _ in range(2))
    Zero3(model)
    ids, plens, slens = _batch(model.cfg)
    with pytest.raises(ValueError, match="sharded trainer"):
        rl.sequence_logprobs(model, ids, plens, slens)
    assert (rl._reference_logprobs(whole, model, ids, plens, slens)[rl._scored_mask(ids, plens, slens)] < 0).all()
    adapted = _adapters(HybridModel.build_random(tiny_hybrid(), seed=4))
    base = rl.sequence_logprobs(adapted, ids, plens, slens, adapters=False)
    Zero3(adapted, mode="lora")                           # (the adapters alone: the base model is whole)
    with pytest.raises(ValueError, match="sharded trainer"):
        rl.sequence_logprobs(adapted, ids, plens, slens)
    assert torch.equal(rl.sequence_logprobs(adapted, ids, plens, slens, adapters=False), base)


def test_models_whose_forward_pass_keeps_32_bits_only():
    """A model of one's own, with the forward pass that training steps have always asked for."""
    class Own(HybridModel):
        def forward_dense(self, tape, ids, *, checkpoint_layers=False, positions=None, hook=None, cp=None, return_hidden=False):
            return super().forward_dense(tape, ids, checkpoint_layers=checkpoint_layers, positions=positions, hook=hook, cp=cp, return_hidden=return_hidden)

    model, own = (_adapters(cls.build_random(tiny_hybrid(), seed=4)) for cls in (HybridModel, Own))
    assert type(own) is Own
    ids, plens, slens = _batch(model.cfg)
    for fused in (False, True):
        want, got = (rl.policy_step(m, ids, plens, slens, torch.ones(4), None, return_grads=True, fused_ce=fused) for m in (model, own))
        assert want["loss"] == got["loss"] and all(torch.equal(g, got["grads"][k]) for k, g in want["grads"].items())
    with pytest.raises(TypeError):
        rl.policy_step(own, ids, plens, slens, torch.ones(4), None, activation_bits=8)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("watched", [True, False])
def test_a_segment_that_is_given_an_input_twice(bits, watched):
    """x^2 + 3 x from one tensor as two inputs, and a leaf that is an input and a parameter: gradients are not counted again."""
    g = torch.Generator().manual_seed(0)
    leaf, w = torch.randint(-127, 128, (3, 128), generator=g).float(), torch.randn(4, 128, generator=g)
    leaf[:, 0] = 127.0                                    # (whole steps of 1: what 8 bits stand for is the values)
    tape = T.Tape()
    tape.watch(leaf, w)
    x = leaf if watched else T.scale(tape, leaf, 1.0)

    def segment(tape, a, b, c):
        out = a * b
        tape.record("product", (a, b), (out,), lambda g: (g * b, g * a))
        return T.linear(tape, T.add(tape, out, T.scale(tape, a, 3.0)), c)

    y = tape.checkpoint(segment, x, x, w, params=(w,), bits=bits)
    up = torch.randn(3, 4, generator=g)
    grads = tape.backward(y, up)
    assert torch.allclose(grads[id(w)], up.t() @ (leaf * leaf + 3 * leaf), rtol=1e-5)
    assert torch.allclose(grads[id(leaf)], (up @ w) * (2 * leaf + 3), rtol=1e-4, atol=1e-2)
