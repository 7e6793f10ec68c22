"""Projections in 8-bit integers on the CPU: the format, the reference backend, the tape's op, checkpoints, shards, refusals."""
import dataclasses
import json

import pytest
import torch

from tilerl_b200 import formats as F
from tilerl_b200 import tape as T
from tilerl_b200.config import get_config
from tilerl_b200.models.hybrid import HybridModel, linear_names, random_master
from tilerl_b200.ops import ref
from tilerl_b200.ops.backend import RefOps


def _rows(t, k, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(t, k, generator=g)
    x[:, ::13] *= 9.0
    return x


def test_integers_are_the_nearest_and_the_largest_is_127():
    w = _rows(7, 48)
    w[3] = 0.0
    q = F.quantize_int8(w)
    assert q.w8.dtype == torch.int8 and q.wscale.dtype == torch.float32 and q.shape == (7, 48)
    amax = w.abs().amax(-1)
    assert torch.equal(q.w8.abs().amax(-1)[amax > 0], torch.full((6,), 127, dtype=torch.int8))
    # half a step, and the rounding of the quotient, the product and the scale (three halves of 2^-23 at 127 steps)
    step = amax.double() / 127
    assert ((q.dequant().double() - w.double()).abs() <= (step * (0.5 + 127 * 6 * 2.0 ** -24))[:, None]).all()
    assert q.wscale[3] == 0 and not q.w8[3].any()
    assert F.nbytes("int8", (7, 48)) == q.nbytes() == 7 * 48 + 28
    again = F.quantize_int8(q.dequant())
    assert torch.equal(again.w8, q.w8)


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_rows_with_an_infinity_or_nan_are_nan_as_a_whole(bad):
    x = _rows(3, 32)
    x[1, 5] = bad
    q, s = F.quantize_act_int8(x)
    assert torch.isnan(s[1]) and torch.isfinite(s[[0, 2]]).all() and not q[1].any()
    y = ref.linear_int8(x, F.quantize_int8(_rows(5, 32, 1)))
    assert torch.isnan(y[1]).all() and torch.isfinite(y[[0, 2]]).all()


def test_the_norms_factor_goes_into_the_scale_alone():
    x, w = _rows(5, 64), torch.rand(64) + 0.5
    q, s = F.quantize_act_int8(x, w, 1e-6)
    plain, _ = F.quantize_act_int8(x * w)
    assert torch.equal(q, plain)
    h = ref.rmsnorm(x, w, 1e-6)
    assert ((q.double() * s.double()[:, None] - h.double()).abs() <= h.abs().amax(-1, keepdim=True).double() / 127 * 0.501).all()


def test_products_in_16_bits_of_a_gradient():
    g = torch.Generator().manual_seed(3)
    up, w = torch.randn(4, 30, generator=g), F.quantize_int8(_rows(30, 16, 4))
    up[2] = 0.0
    q, s = F.quantize_grad_int16(up, w.wscale)
    assert int(q.abs().max()) == 32512
    u = up.double() * w.wscale.double()
    assert ((q.double() * s.double()[:, None] - u).abs() <= (u.abs().amax(-1) / 32512 * (0.5 + 32512 * 8 * 2.0 ** -24))[:, None]).all()
    # digits of 8 bits put together again
    hi = (q + 128) >> 8
    assert int(hi.abs().max()) <= 127 and int((q - 256 * hi).max()) <= 127 and int((q - 256 * hi).min()) >= -128
    want = u @ w.w8.double()
    off = (u.abs().amax(-1, keepdim=True) / 32512 * 0.51) * w.w8.double().abs().sum(0)
    assert ((ref.linear_int8_grad(up, w).double() - want).abs() <= off + want.abs() * 2.0 ** -20).all()


def test_tape_gradient_against_the_formula_and_differences():
    """On rows that lie on the grid the product is linear, so differences over whole steps are the gradient."""
    w = F.quantize_int8(_rows(12, 32, 5))
    g = torch.Generator().manual_seed(6)
    x = torch.randint(-90, 90, (2, 3, 32), generator=g).float()
    x[..., 7] = 127.0                                # the largest stays where it is
    up = torch.randn(2, 3, 12, generator=g)
    tape = T.Tape()
    tape.watch(x)
    out = T.linear(tape, x, w, frozen=True)
    assert out.shape == (2, 3, 12) and out.dtype == torch.float32
    dx = tape.backward(out, up)[id(x)]
    want = up.double() @ w.dequant().double()
    # half a 16-bit step of u for each channel
    off = ((up * w.wscale).double().abs().amax(-1, keepdim=True) / 32512 * 0.51) * w.w8.double().abs().sum(0) + want.abs() * 2.0 ** -20
    assert ((dx.double() - want).abs() <= off).all()
    for at in ((0, 0, 0), (1, 2, 31), (0, 1, 8)):
        hi, lo = x.clone(), x.clone()
        hi[at] += 5
        lo[at] -= 5
        diff = ((T.linear(T.Tape(), hi, w).double() - T.linear(T.Tape(), lo, w).double()) * up.double()).sum() / 10
        scale = (T.linear(T.Tape(), hi, w).double().abs() * up.double().abs()).sum() / 10
        assert abs(float(diff - dx[at])) <= float(off[at] + scale * 8 * 2.0 ** -23)


def test_adapters_over_integers():
    w, a, b = F.quantize_int8(_rows(8, 16, 7)), torch.randn(4, 16), torch.randn(8, 4)
    x, up = _rows(3, 16, 8), torch.randn(3, 8)
    tape = T.Tape()
    tape.watch(x, a, b)
    y = T.linear_lora(tape, x, w, True, a, b, 0.5)
    assert torch.allclose(y, ref.linear_int8(x, w) + x @ a.t() @ b.t() * 0.5, rtol=1e-5, atol=1e-5)
    grads = tape.backward(y, up)
    assert torch.allclose(grads[id(x)], ref.linear_int8_grad(up, w) + up @ b @ a * 0.5, rtol=1e-5, atol=1e-5)


@pytest.mark.parametrize("lead", [(), (0,), (2, 0)])
def test_rows_without_tokens_and_one_row(lead):
    w = F.quantize_int8(_rows(6, 16, 9))
    x = torch.randn(*lead, 16)
    tape = T.Tape()
    tape.watch(x)
    y = T.linear(tape, x, w)
    assert y.shape == (*lead, 6)
    assert tape.backward(y, torch.randn(*lead, 6))[id(x)].shape == x.shape


def test_refusals():
    with pytest.raises(ValueError, match="int8"):
        F.INT8Tensor(torch.zeros(4, 16), torch.zeros(4))
    with pytest.raises(ValueError, match="scales"):
        F.INT8Tensor(torch.zeros(4, 16, dtype=torch.int8), torch.zeros(3))
    with pytest.raises(ValueError, match=r"\[N, K\]"):
        F.quantize_int8(torch.zeros(4))
    from tilerl_b200.ops import gemm_int8
    w = F.quantize_int8(_rows(4, 16))
    assert not gemm_int8.takes(w)                    # (kernels read weights on a GPU)
    with pytest.raises(ValueError, match="INT8 products"):
        gemm_int8.linear(None, torch.zeros(2, 16), w, torch.zeros(2, 4))
    with pytest.raises(ValueError, match="quantize_"):
        gemm_int8.quantize_(torch.zeros(4, 16), w)


def _tiny(name="tiny"):
    return dataclasses.replace(get_config(name), quant="int8")


def test_reference_backend_serves_and_the_training_forward_gives_the_same_projection():
    cfg = _tiny()
    m = HybridModel.build_random(cfg, keep_master=False)
    assert all(isinstance(m.params[n], F.INT8Tensor) for n in linear_names(cfg))
    assert m.served_bytes() == sum(v.nbytes() if hasattr(v, "w8") else v.numel() * v.element_size() for v in m.params.values())
    ops = RefOps()
    w, nw = m.params["L0.qkv"], m.params["L0.norm1"] * 1.3
    x = _rows(5, cfg.hidden, 10)
    y = ops.norm_linear(x, nw, w, cfg.rms_eps)
    # the tape norms first: the same integers but where rounding puts a value on the other side of a half
    h = ref.rmsnorm(x, nw, cfg.rms_eps)
    z = T.linear(T.Tape(), h, w)
    step = h.abs().amax(-1, keepdim=True) / 127 * w.dequant().abs().amax(-1)
    assert ((y - z).abs() <= step * 3 + z.abs() * 1e-6).all()
    act = ops.norm_linear_swiglu(x, nw, m.params["L0.gate_up"], cfg.rms_eps)
    gu = ref.linear_int8(x, m.params["L0.gate_up"], nw, cfg.rms_eps)
    assert torch.equal(act, ref.swiglu(gu))


def test_training_model_has_gradients_and_requantises():
    cfg = _tiny()
    m = HybridModel.build_random(cfg, keep_master=True)
    before = m.params["L0.o"].w8.clone()
    m.params["master.L0.o"].mul_(-1)
    m.requantize_()
    assert torch.equal(m.params["L0.o"].w8, -before)
    lora = HybridModel.build_random(cfg)
    lora.add_lora(4)
    tape = T.Tape()
    tape.watch(*lora.trainable().values())
    y = lora.forward_dense(tape, torch.randint(0, cfg.vocab, (1, 9)))
    assert len(tape.backward(y)) == len(lora.trainable())


@pytest.mark.parametrize("leaf", ["L0.qkv", "L0.o", "L0.gate_up", "L0.down"])
def test_shards_hold_the_integers_of_the_whole(leaf):
    from tilerl_b200.parallel.mesh import shard_param
    cfg = _tiny()
    full = F.quantize_int8(random_master(cfg)[leaf])
    parts = [shard_param(cfg, leaf, full, r, 2) for r in range(2)]
    dense = [shard_param(cfg, leaf, full.dequant(), r, 2) for r in range(2)]
    for p, d in zip(parts, dense):
        assert isinstance(p, F.INT8Tensor) and torch.equal(p.dequant(), d) and p.w8.is_contiguous()


def test_checkpoints_keep_the_integers(tmp_path):
    from tilerl_b200.checkpoint import load_checkpoint, save_checkpoint
    cfg = _tiny()
    m = HybridModel.build_random(cfg)
    save_checkpoint(m, str(tmp_path))
    assert json.load(open(tmp_path / "config.json"))["quant"] == "int8"
    again = load_checkpoint(cfg, str(tmp_path))
    for n in linear_names(cfg):
        assert torch.equal(again.params[n].w8, m.params[n].w8) and torch.equal(again.params[n].wscale, m.params[n].wscale)


@pytest.mark.parametrize("scales", ["rows", "column", "one"])
def test_int8_files_are_taken_as_they_are(tmp_path, scales):
    """Projections of an exported file with its own scales: adopted by a model served in this format, decoded for any other."""
    from safetensors.torch import save_file
    from test_checkpoint import _hf_tensors
    from tilerl_b200.checkpoint import CheckpointError, load_checkpoint
    cfg = _tiny("tiny-hybrid")
    tensors = _hf_tensors(cfg, random_master(cfg, seed=3), "bf16")
    fn = str(tmp_path / "model.safetensors")
    g = torch.Generator().manual_seed(2)
    for k in [k for k in tensors if k.endswith("down_proj.weight") or k.endswith("gate_proj.weight") or k.endswith("up_proj.weight")]:
        n, kk = tensors[k].shape
        tensors[k] = torch.randint(-100, 100, (n, kk), generator=g, dtype=torch.int8)       # (no row reaches 127)
        s = torch.rand(n, generator=g) * 1e-3
        tensors[k + "_scale"] = {"rows": s, "column": s[:, None].contiguous(), "one": s[:1]}[scales]
    save_file(tensors, fn)
    m = load_checkpoint(cfg, str(tmp_path))
    down = next(k for k in tensors if k.endswith("layers.0.mlp.down_proj.weight"))
    assert torch.equal(m.params["L0.down"].w8, tensors[down])
    assert torch.equal(m.params["L0.down"].wscale, tensors[down + "_scale"].reshape(-1).expand(tensors[down].shape[0]))
    gate = down.replace("down", "gate")
    assert torch.equal(m.params["L0.gate_up"].w8[0::2], tensors[gate])
    dense = load_checkpoint(dataclasses.replace(cfg, quant="bf16"), str(tmp_path))
    assert torch.equal(dense.params["L0.down"].float(), m.params["L0.down"].dequant())
    del tensors[down + "_scale"]
    save_file(tensors, fn)
    with pytest.raises(CheckpointError, match="weight_scale"):
        load_checkpoint(cfg, str(tmp_path))


def test_resync_writes_integers():
    from tilerl_b200.parallel.resync import _store
    dst, src = F.quantize_int8(_rows(4, 16, 1)), F.quantize_int8(_rows(4, 16, 2))
    at = dst.w8.data_ptr()
    assert _store(dst, src) == 4 * 16 + 16 and torch.equal(dst.w8, src.w8) and torch.equal(dst.wscale, src.wscale) and dst.w8.data_ptr() == at


def test_a_run_of_them_together():
    """Prompt and decode ticks through the engine choose what the training forward over the same tokens finds largest: the rollout's
    projections are the trainer's."""
    from helpers import make_engine
    from tilerl_b200.engine import SamplingParams
    cfg = _tiny()
    eng = make_engine(cfg)
    prompt = [5, 17, 200, 31, 9, 77]
    got = eng.generate([prompt], SamplingParams(max_tokens=8, temperature=0.0))[0]
    tokens = list(getattr(got, "tokens", got))[-8:]
    logits = eng.model.forward_dense(T.Tape(), torch.tensor([prompt + tokens]))[0]
    for i, t in enumerate(tokens):
        row = logits[len(prompt) - 1 + i]
        assert float(row.max() - row[t]) <= 0.02 * float(row.std()), (i, t)


def test_weights_written_between_the_passes_are_refused():
    w, x = F.quantize_int8(_rows(8, 16)), _rows(3, 16, 1)
    tape = T.Tape()
    tape.watch(x)
    y = T.linear(tape, x, w)
    w.w8.neg_()
    with pytest.raises(RuntimeError, match="changed in place"):
        tape.backward(y)


def test_the_format_by_name_and_by_directory(tmp_path, capsys):
    from tilerl_b200.checkpoint import save_checkpoint
    from tilerl_b200.cli import main
    assert get_config("tiny", "int8").quant == "int8" and get_config("tiny").quant == "bf16"
    for bad in (("tiny", "int4"), ("deluvik-tiny", "int8")):
        with pytest.raises(ValueError, match="cannot be served"):
            get_config(*bad)
    save_checkpoint(HybridModel.build_random(_tiny()), str(tmp_path))
    assert get_config(str(tmp_path)) == _tiny()
    main(["serve", "--model", "qwen38-27b", "--dry-run", "--json", "--quant", "int8"])
    small = json.loads(capsys.readouterr().out)
    main(["serve", "--model", "qwen38-27b", "--dry-run", "--json", "--quant", "bf16"])
    large = json.loads(capsys.readouterr().out)
    assert small != large
    cfg = get_config("qwen38-27b", "int8")
    specs = F.weight_specs(cfg)
    assert specs["L0.gate_up"][1] == "int8" and F.nbytes("int8", (34816, 5120)) == 34816 * 5124
    from tilerl_b200.kernel_cost import prefill_rows
    assert prefill_rows(cfg, 100)


class _Elsewhere:
    """Memory of a backend on another device, as far as the checks look."""
    device = torch.device("cuda:1")

    def get_device(self):
        return 1


def _as_if_on_a_gpu(monkeypatch, n, k, buffer):
    """A weight that passes for one on a device, the products that would be launched, a backend with `buffer`."""
    import types
    from tilerl_b200.ops import gemm_int8
    w = F.quantize_int8(_rows(n, k))
    launched = []
    monkeypatch.setattr(gemm_int8, "_ready", lambda w: gemm_int8._Ready(w.w8, w.wscale, n, k, 0, k, 0, -1))
    monkeypatch.setattr(gemm_int8, "_product", lambda *a: launched.append(a))
    ops = types.SimpleNamespace(ws=types.SimpleNamespace(get=lambda name, shape, dtype: buffer))
    return w, ops, launched


def test_a_backend_on_another_device_is_refused(monkeypatch):
    from tilerl_b200.ops import gemm_int8
    w, ops, launched = _as_if_on_a_gpu(monkeypatch, 8, 16, _Elsewhere())
    x, y = torch.zeros(2, 16, dtype=torch.bfloat16), torch.zeros(2, 8, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="buffers on cuda:1"):
        gemm_int8.linear(ops, x, w, y)
    with pytest.raises(ValueError, match="buffers on cuda:1"):
        gemm_int8.linear(ops, x, w, y, residual=y, epi=gemm_int8.EPI_RESIDUAL)
    gemm_int8.linear(ops, x[:0], w, y[:0])
    assert not launched
    w, ops, launched = _as_if_on_a_gpu(monkeypatch, 8, 16, torch.zeros(99, dtype=torch.int8))
    gemm_int8.linear(ops, x, w, y)
    assert len(launched) == 1


def test_residuals_that_cross_the_output_are_refused(monkeypatch):
    """All pairs of views of one small buffer, against the elements that they consist of."""
    from tilerl_b200.ops import gemm_int8
    w, ops, launched = _as_if_on_a_gpu(monkeypatch, 3, 16, torch.zeros(99, dtype=torch.int8))
    x, buffer, seen = torch.zeros(4, 16, dtype=torch.bfloat16), torch.zeros(64, dtype=torch.bfloat16), set()
    for t in (1, 2, 4):
        views = [(s, ld) for ld in (3, 5, 8) for s in range(64 - (t - 1) * ld - 2)]
        place = {v: torch.tensor([v[0] + i * v[1] + j for i in range(t) for j in range(3)]) for v in views}
        for a in views[::3]:
            for b in views:
                y, res = (torch.as_strided(buffer, (t, 3), (ld, 1), s) for s, ld in (a, b))
                pa, pb = place[a], place[b]
                bad = bool(((pa[:, None] == pb[None]) & ~torch.eye(len(pa), dtype=torch.bool)).any())
                if a[1] != b[1] and t > 1 and not bad:
                    bad = None                       # (may be refused where the ranges cross)
                    if int(pa[-1]) < int(pb[0]) or int(pb[-1]) < int(pa[0]):
                        bad = False
                before = len(launched)
                try:
                    gemm_int8.linear(ops, x[:t], w, y, residual=res, epi=gemm_int8.EPI_RESIDUAL)
                    refused = False
                except ValueError as e:
                    assert "residual" in str(e)
                    refused = True
                assert refused == (len(launched) == before) and (bad is None or refused == bad), (t, a, b)
                seen.add((t, refused))
    assert len(seen) == 6


def test_parts_of_a_fused_projection_that_are_not_integers_leave_the_others_alone(tmp_path):
    """Exports that keep the recurrent layers' small projections in bf16."""
    from safetensors.torch import save_file
    from test_checkpoint import _hf_tensors
    from tilerl_b200.checkpoint import load_checkpoint
    cfg = _tiny("tiny-hybrid")
    tensors = _hf_tensors(cfg, random_master(cfg, seed=3), "bf16")
    g = torch.Generator().manual_seed(2)
    dense = ("in_proj_a", "in_proj_b", "k_proj", "up_proj")
    for k in [k for k in tensors if "_proj" in k and not any(d in k for d in dense)]:
        tensors[k] = torch.randint(-100, 100, tensors[k].shape, generator=g, dtype=torch.int8)      # (no row reaches 127)
        tensors[k + "_scale"] = torch.rand(len(tensors[k]), generator=g) * 1e-3 + 1e-5
    save_file(tensors, str(tmp_path / "model.safetensors"))
    m = load_checkpoint(cfg, str(tmp_path), keep_master=True)

    def whole(layer, *bases):
        return [(tensors[f"model.layers.{layer}.{b}.weight"], tensors.get(f"model.layers.{layer}.{b}.weight_scale")) for b in bases]

    def check(rows, scales, master, w, s):
        if s is not None:
            assert torch.equal(rows, w) and torch.equal(scales, s) and torch.equal(master, w * s[:, None])
        else:
            want = F.quantize_int8(w)
            assert torch.equal(rows, want.w8) and torch.equal(scales, want.wscale) and torch.equal(master, w.float())
    for name, parts in (("L0.in", whole(0, *("linear_attn.in_proj_" + n for n in ("qkv", "z", "a", "b")))),
                        ("L1.qkv", whole(1, *("self_attn." + n + "_proj" for n in "qkv")))):
        got, master, at = m.params[name], m.params["master." + name], 0
        for w, s in parts:
            here = slice(at, at + len(w))
            check(got.w8[here], got.wscale[here], master[here], w, s)
            at += len(w)
        assert at == len(got.w8) == len(master)
    got, master = m.params["L0.gate_up"], m.params["master.L0.gate_up"]
    for i, (w, s) in enumerate(whole(0, "mlp.gate_proj", "mlp.up_proj")):
        check(got.w8[i::2], got.wscale[i::2], master[i::2], w, s)
    half = load_checkpoint(cfg, str(tmp_path), keep_master=True, tp_rank=1, tp=2)
    from tilerl_b200.parallel.mesh import shard_param
    for name in ("L0.in", "L1.qkv", "L0.gate_up", "L0.out"):
        want = shard_param(cfg, name, m.params[name], 1, 2)
        assert torch.equal(half.params[name].w8, want.w8) and torch.equal(half.params[name].wscale, want.wscale)
        assert torch.equal(half.params["master." + name], shard_param(cfg, name, m.params["master." + name], 1, 2))


FORMATS = {"nvfp4": F.NVFP4Tensor, "fp8": F.FP8BlockTensor, "int8": F.INT8Tensor, "bf16": torch.Tensor}


@pytest.mark.parametrize("stored", ["nvfp4", "int8", "fp8", "bf16"])
def test_a_model_serves_the_format_that_its_configuration_names(tmp_path, stored):
    """Whatever the own dialect's file holds; bit for bit where it is the same."""
    from tilerl_b200.checkpoint import load_checkpoint, save_checkpoint
    from tilerl_b200.parallel.mesh import shard_param
    cfg = dataclasses.replace(get_config("tiny-hybrid"), quant=stored, lm_head_quant="nvfp4", tie_embeddings=False)
    m = HybridModel.build_random(cfg)
    save_checkpoint(m, str(tmp_path))
    dense = {n: m.params[n] if isinstance(m.params[n], torch.Tensor) else m.params[n].dequant() for n in linear_names(cfg)}
    if stored == "fp8":                              # (written in bf16)
        dense = {n: w.bfloat16().float() for n, w in dense.items()}
    for quant, kind in FORMATS.items():
        served = dataclasses.replace(cfg, quant=quant)
        for rank, tp in ((0, 1), (1, 2)):
            if quant == "fp8" and tp > 1:
                continue
            again = load_checkpoint(served, str(tmp_path), tp_rank=rank, tp=tp)
            assert isinstance(again.params["lm_head"], F.NVFP4Tensor)
            for n in linear_names(cfg):
                got = again.params[n]
                assert type(got) is kind, (quant, n)
                if quant == stored and stored != "fp8":
                    want = shard_param(cfg, n, m.params[n], rank, tp)
                elif quant == "fp8":
                    want = F.quantize_fp8_block(dense[n])
                elif stored in ("fp8", "bf16") and tp > 1:
                    continue                         # (dense values of this dialect are cut before they are quantised)
                else:
                    want = shard_param(cfg, n, {"nvfp4": F.quantize_nvfp4, "int8": F.quantize_int8, "bf16": lambda w: w}[quant](dense[n]), rank, tp)
                for field in {"nvfp4": ("wq", "tscale"), "fp8": ("w8", "wscale"), "int8": ("w8", "wscale"), "bf16": ("data",)}[quant]:
                    a, b = getattr(got, field), getattr(want, field)
                    assert torch.equal(a.view(torch.uint8) if a.element_size() == 1 else a, b.view(torch.uint8) if b.element_size() == 1 else b), (quant, n, field)


@pytest.mark.parametrize("quant", ["nvfp4", "fp8", "int8", "bf16"])
@pytest.mark.parametrize("name", ["tiny-hybrid", "small-gpu"])
def test_a_saved_models_directory_names_its_format(tmp_path, name, quant):
    from tilerl_b200.checkpoint import save_checkpoint
    cfg = get_config(name, quant)
    save_checkpoint(HybridModel(cfg, {"final_norm": torch.ones(cfg.hidden)}), str(tmp_path))
    assert get_config(str(tmp_path)) == cfg and get_config(str(tmp_path), "fp8").quant == "fp8"
    with open(tmp_path / "config.json") as f:
        j = json.load(f)
    j["quant"] = "of another day"
    with open(tmp_path / "config.json", "w") as f:
        json.dump(j, f)
    assert get_config(str(tmp_path)) == get_config(name)


def test_shards_of_dense_files_hold_the_integers_of_the_whole(tmp_path):
    """Rows cut along K before they are quantised would have a scale for each part."""
    from tilerl_b200.checkpoint import load_checkpoint, save_checkpoint
    from tilerl_b200.parallel.mesh import shard_param
    cfg = get_config("tiny-hybrid", "bf16")
    m = HybridModel.build_random(cfg)
    save_checkpoint(m, str(tmp_path))
    for rank in range(2):
        half = load_checkpoint(dataclasses.replace(cfg, quant="int8"), str(tmp_path), tp_rank=rank, tp=2)
        for n in linear_names(cfg):
            want = shard_param(cfg, n, F.quantize_int8(m.params[n]), rank, 2)
            assert torch.equal(half.params[n].w8, want.w8) and torch.equal(half.params[n].wscale, want.wscale), n


def _adopted(cfg, **kw):
    """A model whose integers came from a file: no row reaches 127."""
    g = torch.Generator().manual_seed(2)
    master = random_master(cfg, 3)
    for n in linear_names(cfg):
        shape = master[n].shape
        master[n] = F.INT8Tensor(torch.randint(-100, 100, shape, generator=g, dtype=torch.int8), torch.rand(shape[0], generator=g) * 1e-3 + 1e-5)
    return HybridModel.from_master(cfg, master, act_dtype=torch.float32, **kw)


def test_integers_that_training_left_alone_are_not_rounded_anew():
    cfg = _tiny("tiny-hybrid")
    m, before = _adopted(cfg, keep_master=True), _adopted(cfg).params
    m.requantize_()
    for n in linear_names(cfg):
        assert torch.equal(m.params[n].w8, before[n].w8) and torch.equal(m.params[n].wscale, before[n].wscale)
    moved = m.params["master.L0.down"]
    moved[3, 5] += 1.0
    m.requantize_()
    got, want, was = m.params["L0.down"], F.quantize_int8(moved), before["L0.down"]
    others = [i for i in range(len(moved)) if i != 3]
    assert torch.equal(got.w8[others], was.w8[others]) and torch.equal(got.wscale[others], was.wscale[others])
    assert torch.equal(got.w8[3], want.w8[3]) and got.wscale[3] == want.wscale[3]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("tp", [1, 2])
def test_resync_of_weights_that_did_not_move_keeps_their_integers(tp, dtype):
    import types
    from tilerl_b200.parallel.resync import resync
    cfg = _tiny("tiny-hybrid")
    trainer = _adopted(cfg, keep_master=True)
    weights = {n: w.to(dtype) for n, w in trainer.params.items() if n.startswith("master.")}
    zero = types.SimpleNamespace(units=[0], unit_tensors=lambda i: weights, _prefetch=None, _drop=lambda u: None, device=torch.device("cpu"))
    for rank in range(tp):
        rollout, before = (_adopted(cfg, tp_rank=rank, tp=tp) for _ in range(2))
        resync(zero, rollout)
        for n in linear_names(cfg):
            a, b = rollout.params[n], before.params[n]
            assert torch.equal(a.w8, b.w8) and torch.equal(a.wscale, b.wscale), n
    weights["master.L0.o" if "master.L0.o" in weights else "master.L0.out"].mul_(2)
    name = "L0.o" if "master.L0.o" in weights else "L0.out"
    resync(zero, rollout)
    from tilerl_b200.parallel.mesh import shard_param
    want = shard_param(cfg, name, F.quantize_int8(weights["master." + name].float()), rank, tp)
    assert torch.equal(rollout.params[name].w8, want.w8) and torch.equal(rollout.params[name].wscale, want.wscale)


def test_a_weight_that_the_kernels_do_not_read_is_named_as_the_cause():
    from tilerl_b200.ops import gemm_int8
    w = F.quantize_int8(_rows(37, 40))
    with pytest.raises(ValueError, match=r"quantize_ takes weights .*multiple of 16 values.*\(37, 40\)"):
        gemm_int8.quantize_(torch.zeros(37, 40), w)


def test_records_of_a_bench_name_a_format_that_is_not_the_models_own(tmp_path, monkeypatch, capsys):
    """Or the gate would measure one format against the other's best."""
    from tilerl_b200 import benchrec
    from tilerl_b200.cli import main
    monkeypatch.setenv("TRL_BENCH_STORE", str(tmp_path / "m.jsonl"))
    run = ["bench", "--model", "tiny", "--device", "cpu", "--prompt-len", "8", "--gen", "3", "--record"]
    for more in ([], ["--quant", "int8"], ["--quant", "bf16"]):
        assert main(run + more) == 0
    own, other, again = [r["shape"] for r in benchrec.load(str(tmp_path / "m.jsonl"))]
    assert "quant" not in own and other == dict(own, quant="int8") and again == own


@pytest.mark.parametrize("dialect", ["own", "export"])
def test_merges_go_by_what_the_integers_stand_for(tmp_path, dialect):
    from safetensors.torch import load_file, save_file
    from tilerl_b200.merge import merge_checkpoints
    w8, ws = ("p.w8", "p.wscale") if dialect == "own" else ("p.weight", "p.weight_scale")
    dense = [_rows(6, 32, i) for i in range(3)]
    dense[1][2], dense[2][2] = dense[0][2], dense[0][2]       # (a row that nobody moved)
    files = []
    for i, w in enumerate(dense):
        q = F.quantize_int8(w)
        q.w8[2], q.wscale[2] = torch.arange(32) - 9, 0.25      # (and that does not reach 127)
        (tmp_path / str(i)).mkdir()
        save_file({w8: q.w8, ws: q.wscale if dialect == "own" else q.wscale[:, None].contiguous(), "norm": torch.full((4,), float(i))},
                  str(tmp_path / str(i) / "model.safetensors"))
        files.append(q)
    merge_checkpoints(str(tmp_path / "0"), [str(tmp_path / "1"), str(tmp_path / "2")], str(tmp_path / "out"))
    got = load_file(str(tmp_path / "out" / "model.safetensors"))
    q = F.INT8Tensor(got[w8], got[ws])
    want = (files[1].dequant().double() + files[2].dequant().double()) / 2
    # half a step of the merged row, and fp32 sums of three terms
    step = want.abs().amax(-1, keepdim=True) / 127
    size = sum(f.dequant().double().abs() for f in files).amax(-1, keepdim=True)
    assert ((q.dequant().double() - want).abs() <= step * (0.5 + 127 * 6 * 2.0 ** -24) + size * 8 * 2.0 ** -24).all()
    assert torch.equal(q.w8[2], files[0].w8[2]) and q.wscale[2] == 0.25
    assert torch.equal(got["norm"], torch.full((4,), 1.5))
    if dialect == "export":                          # a dense base, tuned checkpoints in integers
        (tmp_path / "dense").mkdir()
        save_file({w8: dense[0]}, str(tmp_path / "dense" / "model.safetensors"))
        merge_checkpoints(str(tmp_path / "dense"), [str(tmp_path / "1"), str(tmp_path / "2")], str(tmp_path / "out"))
        got = load_file(str(tmp_path / "out" / "model.safetensors"))[w8]
        assert ((got.double() - want).abs() <= (size + dense[0].double().abs()) * 8 * 2.0 ** -24).all()
    (tmp_path / "other").mkdir()
    save_file({"norm": torch.zeros(4)}, str(tmp_path / "other" / "model.safetensors"))
    merge_checkpoints(str(tmp_path / "0"), [str(tmp_path / "other")], str(tmp_path / "out"))
    got = load_file(str(tmp_path / "out" / "model.safetensors"))
    assert torch.equal(got[w8], files[0].w8) and torch.equal(got[ws].reshape(-1), files[0].wscale)


@pytest.mark.parametrize("command", [["serve"], ["bench"], ["train", "--rl", "--reward", "mod7"]])
def test_dense_projections_are_refused_by_name_on_a_gpu(command, monkeypatch):
    """Before anything is built: no kernel of the GPU backend serves them."""
    from tilerl_b200 import cli, factory

    def reached(*a, **k):
        raise AssertionError("refused too late")
    for name in ("make_ops", "build_model", "build_engine"):
        monkeypatch.setattr(factory, name, reached)
    with pytest.raises(SystemExit, match="--quant bf16"):
        cli.main(command + ["--model", "small-gpu", "--quant", "bf16", "--device", "cuda"])
    with pytest.raises(AssertionError, match="too late"):
        cli.main(command + ["--model", "small-gpu", "--quant", "int8", "--device", "cpu"])


def test_a_training_run_in_another_format_is_another_run(tmp_path, capsys):
    """The same command asked twice is handed the finished manifest; with --quant it is not the same."""
    from tilerl_b200 import cli
    run = ["train", "--recipe", "grpo-tiny-smoke", "--device", "cpu", "--steps", "1", "--max-tokens", "4", "--prompt-len", "6", "--runs", str(tmp_path)]
    ids = []
    for more in ([], ["--quant", "int8"], ["--quant", "int8"], []):
        assert cli.main(run + more) == 0
        lines = [json.loads(l) for l in capsys.readouterr().out.splitlines() if l.startswith("{")]
        ids.append([l["run"] for l in lines if l.get("reused")])
    assert ids[:2] == [[], []] and len(ids[2]) == len(ids[3]) == 1 and ids[2] != ids[3]


def test_a_store_of_pages_tells_weights_apart_by_their_scales():
    """Twice as large a weight has the same integers."""
    from tilerl_b200.kv_tiers import weights_fingerprint
    cfg = _tiny("tiny-hybrid")
    a, b, c = (HybridModel.build_random(cfg) for _ in range(3))
    b.params["L0.down"].wscale.mul_(2)
    assert weights_fingerprint(a) == weights_fingerprint(c) != weights_fingerprint(b)


def test_a_rows_largest_value_has_the_low_digit_zero():
    """What keeps a gradient's sums of 131072 channels in 32 bits: low digits go down to -128, and so may a file's weights, but one of a row's
    digits is 0.  For every significand, at magnitudes up to the ends of the range."""
    m = torch.arange(1 << 23, dtype=torch.int32)
    for e in (18, 64, 126, 127, 128, 200, 253, 254):          # (the least that counts is 2^-110)
        v = (m + (e << 23)).view(torch.float32)
        q, s = F._row_integers(v[:, None], F.INT16_MAX)
        assert bool((q == 32512).all()) and bool(torch.isfinite(s).all())
        q, _ = F._row_integers(v[:, None], F.INT8_MAX)
        assert bool((q == 127).all())
    assert 131071 * 128 * 128 < 2 ** 31 and 131072 * 127 * 128 < 2 ** 31


def _tp_projections(rank, world):
    """Of two ranks: projections cut along their channels, projections cut along K with the sum over the ranks, and an engine."""
    import torch.distributed as dist
    from helpers import rand_prompts
    from tilerl_b200.engine import Engine, SamplingParams
    from tilerl_b200.kv import GdnStatePool, PagedKvPool
    from tilerl_b200.ops.backend import TPContext
    cfg = _tiny("tiny-hybrid")
    m = HybridModel.build_random(cfg, seed=1, tp_rank=rank, tp=world)
    ops = RefOps(TPContext(rank, world, dist.group.WORLD))
    x, nw = _rows(5, cfg.hidden, 3), torch.rand(cfg.hidden, generator=torch.Generator().manual_seed(4)) + 0.5
    act = ops.norm_linear_swiglu(x, nw, m.params["L0.gate_up"], cfg.rms_eps)
    out = ops.linear_residual(act, m.params["L0.down"], x)
    d = m.dims
    kv = PagedKvPool(cfg, 64, dtype=torch.float32, n_kv_heads=d.n_kv)
    st = GdnStatePool(cfg, 6, ring_dtype=torch.float32, n_v_heads=d.gdn_nv, n_k_heads=d.gdn_nk)
    eng = Engine(m, ops, kv, st)
    return act, out, [r.tokens for r in eng.generate(rand_prompts(cfg, 2, 24), SamplingParams(max_tokens=8))]


def test_two_ranks_serve_the_integers_of_one():
    from helpers import rand_prompts
    from tilerl_b200.parallel.mesh import shard_param
    from world_helpers import run_world
    cfg = _tiny("tiny-hybrid")
    whole = HybridModel.build_random(cfg, seed=1)
    x, nw = _rows(5, cfg.hidden, 3), torch.rand(cfg.hidden, generator=torch.Generator().manual_seed(4)) + 0.5
    got = run_world(2, _tp_projections)
    acts, outs, tokens = zip(*got)
    act = RefOps().norm_linear_swiglu(x, nw, whole.params["L0.gate_up"], cfg.rms_eps)
    assert torch.equal(torch.cat(acts, -1), act)
    # each rank's rows have a scale of their own; the sum of two fp32 products and the residual
    parts = [ref.linear_int8(a, shard_param(cfg, "L0.down", whole.params["L0.down"], r, 2)).double() for r, a in enumerate(acts)]
    want = parts[0] + parts[1] + x.double()
    room = (parts[0].abs() + parts[1].abs() + want.abs()) * 2 * 2.0 ** -24
    assert torch.equal(outs[0], outs[1]) and ((outs[0].double() - want).abs() <= room).all()
    assert tokens[0] == tokens[1]
    for prompt, toks in zip(rand_prompts(cfg, 2, 24), tokens[0]):
        toks = list(toks)[-8:]
        logits = whole.forward_dense(T.Tape(), torch.tensor([list(prompt) + toks]))[0]
        for i, t in enumerate(toks):                 # (a token chosen by chance lies some deviations below the largest)
            row = logits[len(prompt) - 1 + i]
            assert float(row.max() - row[t]) <= 0.2 * float(row.std()), (i, t)
