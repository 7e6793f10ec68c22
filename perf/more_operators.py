"""Operators of 8-bit integer projections: what is measured of them.

A model whose projections are kept in 8-bit integers, with a scale for each output channel, quantises the rows that go into a product
the same way, with a scale for each token.  Served, a tick's projections are such products of normed rows, with a residual added or
with SwiGLU over pairs of rows behind them; trained, the frozen weights' products and the gradients through them are on the tape.

Definitions, for rows x, weights wq (int8, one row an output channel) with scales ws, and a norm's weight g:
  rows in 8 bits:   t = x g (or x), m = max |t|, q = rint(t ((1 / m) 127)), s = m (1 / 127) r with r = rsqrt(mean x^2 + eps) (or 1);
                    a row of nothing but zeros has q = 0 and s = 0
  linear:           y = (q . wq) s ws, after a norm, or added to a residual
  gated:            the rows of wq are pairs (gate, up): y = gate / (1 + exp(-gate)) up
  train:            y = (q . wq) s ws of fp32 rows; the gradient takes the rounding of x for none: dx = (g ws) . wq, the rows u = g ws in
                    16 bits: m = max |u|, Q = rint(u ((1 / m) 32512)), dx = (Q . wq) m (1 / 32512)
What leads to integers, the products and quotients of t, m and q, is of 32 bits by definition, each rounded.
"""
import math

import torch

own = False

EPS = 1e-6
MOST8, MOST16 = 127.0, 32512.0
#: multiplications of the largest listed product: no drawn case has more
MOST_PRODUCT = 2000 * 34816 * 5120


def listed():
    return [
        # one token of a small model's attention projection: launches and host work count
        dict(name="linear-1-1024x5120", op="linear", tokens=1, n=5120, k=1024, residual=False),
        # one user's decode tick on the 27B model: the recurrent layers' fused input projection
        dict(name="linear-1-5120x16480", op="linear", tokens=1, n=16480, k=5120, residual=False),
        # a batch of 24 sequences decoding: the feed-forward's way back into the residual stream
        dict(name="linear-24-17408x5120-residual", op="linear", tokens=24, n=5120, k=17408, residual=True),
        # verify windows and short prompts riding in one tick, a projection off every tile
        dict(name="linear-133-2048x1999", op="linear", tokens=133, n=1999, k=2048, residual=False),
        # a prompt chunk of the 27B model
        dict(name="linear-2000-5120x16480", op="linear", tokens=2000, n=16480, k=5120, residual=False),
        # one user's decode tick: gate and up rows of the 27B model, the largest weight that a token reads
        dict(name="gated-1-5120x34816", op="gated", tokens=1, n=34816, k=5120),
        # a verify window of eight drafted tokens
        dict(name="gated-8-5120x34816", op="gated", tokens=8, n=34816, k=5120),
        # a ragged prompt of a small model
        dict(name="gated-301-1024x8192", op="gated", tokens=301, n=8192, k=1024),
        # a prompt chunk of the 27B model
        dict(name="gated-2000-5120x34816", op="gated", tokens=2000, n=34816, k=5120),
        # a short completion through a small model's projection, forward and gradient
        dict(name="train-37-1024x5120", op="train", tokens=37, n=5120, k=1024),
        # a micro-batch through the attention's output projection
        dict(name="train-1024-6144x5120", op="train", tokens=1024, n=5120, k=6144),
        # one sequence of a step through the widest frozen weight
        dict(name="train-2000-5120x34816", op="train", tokens=2000, n=34816, k=5120),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["linear", "linear", "gated", "train"])
    k = 16 * _log(rng, 4, 1088)
    n = 2 * _log(rng, 16, 17408) if op == "gated" else _log(rng, 32, 34816)
    tokens = _log(rng, 1, max(1, min(4096, MOST_PRODUCT // (n * k))))
    case = dict(op=op, tokens=tokens, n=n, k=k)
    return dict(case, residual=rng.random() < 0.4) if op == "linear" else case


# ---- what a program has in hand ------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    new = lambda *shape, dtype=torch.float32: torch.randn(*shape, generator=g, device="cuda", dtype=dtype)  # noqa: E731
    t, n, k = case["tokens"], case["n"], case["k"]
    st = dict(case=case, wq=torch.empty(n, k, dtype=torch.int8, device="cuda"), ws=torch.empty(n, device="cuda"))
    for rows in torch.arange(n, device="cuda").split(8192):
        # weights as random-init models have them, a channel's largest at 127
        w = new(len(rows), k).mul_(0.02)
        most = w.abs().amax(-1)
        st["wq"][rows] = torch.round(w * (MOST8 / most)[:, None]).to(torch.int8)
        st["ws"][rows] = most / MOST8
    # rows of the residual stream: a few channels far larger than the rest
    x = new(t, k) * (1 + 15 * (torch.rand(k, generator=g, device="cuda") < 0.01))
    if case["op"] == "train":
        st.update(x=x, up=new(t, n).mul_(0.01) * (1 + 15 * (torch.rand(t, 1, generator=g, device="cuda") < 0.1)))
    else:
        st.update(x=x.bfloat16())
        if case["op"] == "linear" and case["residual"]:
            st["residual"] = new(t, n, dtype=torch.bfloat16)
        else:
            st["norm"] = 1 + 0.1 * new(k)
    if own:
        _handle(st)
    return st


def _handle(st):
    """The backend and the weight as a program holds them."""
    if "w" not in st:
        from tilerl_b200.formats import INT8Tensor
        from tilerl_b200.ops.cuda import CudaOps
        st.update(ops=CudaOps(), w=INT8Tensor(st["wq"], st["ws"]))
    return st["ops"], st["w"]


# ---- plain forms -----------------------------------------------------------------------------------------
def _integers(t, most_int):
    """The integers of rows in fp32, and their rows' scales."""
    most = t.abs().amax(-1, keepdim=True)
    there = most > 0
    q = torch.where(there, torch.round(t * (torch.where(there, most, 1.0).reciprocal() * most_int)), 0.0)
    return q, most * torch.tensor(1.0 / most_int, dtype=torch.float32, device=t.device)


def _rows(st):
    x = st["x"].float()
    if "norm" not in st:
        return _integers(x, MOST8)
    q, s = _integers(x * st["norm"], MOST8)
    return q, s * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)


def _plain(st):
    op, wq, ws = st["case"]["op"], st["wq"].float(), st["ws"]
    q, s = _rows(st)
    y = (q @ wq.t()).mul_(s).mul_(ws)
    if op == "linear":
        return (y + st["residual"].float() if "residual" in st else y).bfloat16()
    if op == "gated":
        gate, up = y[:, 0::2], y[:, 1::2]
        return (gate / (1 + torch.exp(-gate)) * up).bfloat16()
    q, s = _integers(st["up"] * ws, MOST16)
    return dict(out=y, grad=(q @ wq).mul_(s))


def run(st):
    if not own:
        return _plain(st)
    op = st["case"]["op"]
    ops, w = _handle(st)
    if op == "gated":
        return ops.norm_linear_swiglu(st["x"], st["norm"], w, EPS)
    if op == "linear":
        if "residual" in st:
            return ops.linear_residual(st["x"], w, st["residual"].clone())      # (adds to the stream in place)
        return ops.norm_linear(st["x"], st["norm"], w, EPS)
    from tilerl_b200 import tape as T
    tape = T.Tape()
    tape.watch(st["x"])
    out = T.linear(tape, st["x"], w, frozen=True)
    return dict(out=out, grad=tape.backward(out, st["up"])[id(st["x"])])


# ---- what a pass cannot do without -----------------------------------------------------------------------
def work(case):
    """Of a training pass the weight is read for each direction: the loss stands between them."""
    t, n, k = case["tokens"], case["n"], case["k"]
    weight, product = n * k + 4 * n, 2 * t * n * k
    if case["op"] == "train":
        return {"bytes": 2 * weight + 8 * t * (n + k), "flops": 2 * product}
    if case["op"] == "gated":
        return {"bytes": weight + 2 * t * k + 4 * k + t * n, "flops": product}
    return {"bytes": weight + 2 * t * k + (2 * t * n if case["residual"] else 4 * k) + 2 * t * n, "flops": product}


# ---- in 64 bits, from the definitions ----------------------------------------------------------------------
def _codes(t, top):
    """What leads to the integers is of 32 bits by definition; the scale is not."""
    peak = t.abs().max(-1, keepdim=True).values
    factor = torch.reciprocal(peak.clamp_min(1e-30)) * top
    return torch.round(t * factor).double(), peak.double() / top


def exact(case, seed):
    st = prepare(case, seed)
    x, scales = st["x"].float(), st["ws"].double()
    weight = [part.double() for part in st["wq"].split(8192)]
    if "norm" in st:
        codes, unit = _codes(x * st["norm"], MOST8)
        unit = unit / (x.double().square().mean(-1, keepdim=True) + EPS).sqrt()
    else:
        codes, unit = _codes(x, MOST8)
    y = torch.cat([codes @ part.t() for part in weight], -1) * unit * scales
    if case["op"] == "linear":
        return y + st["residual"].double() if "residual" in st else y
    if case["op"] == "gated":
        return y[:, 0::2] * torch.sigmoid(y[:, 0::2]) * y[:, 1::2]
    codes, unit = _codes(st["up"] * st["ws"], MOST16)
    return dict(out=y, grad=sum(c @ part for c, part in zip(codes.split(8192, dim=-1), weight)) * unit)
