"""Operators of policy and preference training: what is measured of them.

A step of RL or preference training on a language model goes, beside its products, through the model's vocabulary: the clipped
policy loss with its KL term and the preference loss over pairs are formed from logits and give logits' gradients, and the frozen
policies that both compare with are scored, token by token, from hidden rows and the head.  What the step keeps between its passes is
kept in 8 bits where memory is short.

Definitions, for a row of logits x with target t:
  m = max x, s = sum exp(x - m), lp = x[t] - m - log s
  policy:      rho = exp(lp - old), u = min(rho A, clip(rho, 1 - lo, 1 + hi) A), kl = exp(d) - d - 1 with d = ref - lp,
               loss = scale * sum over scored rows of (-u + beta kl)
  preference:  S = sum (or mean) over a sequence's scored tokens of (lp - ref), z = beta (S_chosen - S_rejected),
               loss = scale * sum over pairs of (-(1 - e) log sigmoid(z) - e log sigmoid(-z))
  scoring:     x = h W^T; lp and the entropy log s - sum exp(x - m) (x - m) / s; 0 where a row is not scored
  kept rows:   groups of 128 values, scale = amax / 127, q = rint(x * (127 / amax)), both quotients and the product in 32 bits
Rows that are not scored have no gradient, whatever their logits and targets hold.
"""
import math

import torch

own = False

GROUP = 128
#: logits of the largest case, and multiplications of the largest scoring: no drawn case has more
MOST_LOGITS = 1024 * 248320
MOST_PRODUCT = 512 * 5120 * 248320


def listed():
    return [
        # one short completion of a byte-vocabulary model on its own: launches and host work count
        dict(name="policy-24x320", op="policy", seqs=1, tokens=24, vocab=320, dtype="fp32", scored=0.6, old=True, kl=0.05, hi=0.2),
        # a micro-batch of a small model's RL step, clipped further up than down, with the reference's KL
        dict(name="policy-4x512x32768", op="policy", seqs=4, tokens=512, vocab=32768, dtype="fp32", scored=0.8, old=True, kl=0.05, hi=0.28),
        # the 27B model's vocabulary: one sequence of completions at a time, logits as the tape has them
        dict(name="policy-1x1024x248320", op="policy", seqs=1, tokens=1024, vocab=248320, dtype="fp32", scored=1.0, old=True, kl=0.0, hi=0.2),
        # pairs of short answers, a vocabulary off every vector width, logits in the serving type
        dict(name="preference-2x100x49999-bf16", op="preference", pairs=2, tokens=100, vocab=49999, dtype="bf16", scored=0.5, beta=0.1, smooth=0.0, average=False),
        # a micro-batch of pairs as preference training takes it
        dict(name="preference-2x512x32768", op="preference", pairs=2, tokens=512, vocab=32768, dtype="fp32", scored=0.7, beta=0.1, smooth=0.1, average=False),
        # one token of one sequence: the smallest scoring, a pass over the head's weights
        dict(name="score-1-1024x32768", op="score", rows=1, hidden=1024, vocab=32768, scored=1.0, entropy=False),
        # the frozen reference of a small model over a batch, half of it prompt
        dict(name="score-4096-1024x32768", op="score", rows=4096, hidden=1024, vocab=32768, scored=0.5, entropy=True),
        # the 27B model's head over one completion
        dict(name="score-512-5120x248320", op="score", rows=512, hidden=5120, vocab=248320, scored=1.0, entropy=False),
        # one layer's input of a short sequence, kept and read back
        dict(name="keep-100x1024", op="keep", rows=100, width=1024),
        # the residual rows of a batch at the 27B model's width
        dict(name="keep-8192x5120", op="keep", rows=8192, width=5120),
        # feed-forward rows (gate and up interleaved) of the byte-vocabulary model, ragged in the last group
        dict(name="swiglu-300x1500", op="swiglu", rows=300, width=1500),
        # feed-forward rows of the 27B model
        dict(name="swiglu-2048x17408", op="swiglu", rows=2048, width=17408),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["policy", "policy", "preference", "score", "score", "keep", "swiglu"])
    scored = rng.choice([1.0, 0.8, 0.5, 0.2])
    if op in ("policy", "preference"):
        vocab = _log(rng, 300, 262144)
        seqs = rng.randint(1, 8)
        per = 2 if op == "preference" else 1
        tokens = _log(rng, 1, min(4096, MOST_LOGITS // (vocab * seqs * per)))
        both = dict(op=op, tokens=tokens, vocab=vocab, dtype=rng.choice(["fp32", "fp32", "bf16"]), scored=scored)
        if op == "policy":
            return dict(both, seqs=seqs, old=rng.random() < 0.8, kl=rng.choice([0.0, 0.05]), hi=rng.choice([0.2, 0.28]))
        return dict(both, pairs=seqs, beta=rng.choice([0.05, 0.1, 0.5]), smooth=rng.choice([0.0, 0.1]), average=rng.random() < 0.3)
    if op == "score":
        hidden = 8 * _log(rng, 8, 640)
        vocab = _log(rng, 300, 248320)
        rows = _log(rng, 1, min(8192, MOST_PRODUCT // (hidden * vocab)))
        return dict(op=op, rows=rows, hidden=hidden, vocab=vocab, scored=scored, entropy=rng.random() < 0.5)
    if op == "keep":
        width = 4 * _log(rng, 16, 2048)
        return dict(op=op, rows=_log(rng, 1, 8192 * 5120 // width), width=width)
    width = 4 * _log(rng, 16, 4352)
    return dict(op=op, rows=_log(rng, 1, min(32768, 2048 * 17408 // width)), width=width)


# ---- what a program has in hand ------------------------------------------------------------------------
def _lp64(logits, targets):
    """Log-probabilities of the targets in 64 bits, row by row of a sequence."""
    out = []
    for x, t in zip(logits.flatten(0, -2).split(256), targets.flatten().split(256)):
        x = x.double()
        out.append(x.gather(-1, t[:, None])[:, 0] - torch.logsumexp(x, -1))
    return torch.cat(out).view(targets.shape)


def _mask(case, shape, g):
    """The scored tokens: of each sequence the part after a prompt and before the padding (every sequence has one at least)."""
    n, t = shape
    length = torch.full((n,), t) if case["scored"] == 1.0 else torch.randint(max(1, t * 3 // 4), t + 1, (n,), generator=g)
    start = (length * (1 - case["scored"])).long().clamp(max=t - 1).minimum(length - 1)
    at = torch.arange(t)[None, :]
    return ((at >= start[:, None]) & (at < length[:, None])).cuda()


def prepare(case, seed):
    g, gc = torch.Generator(device="cuda").manual_seed(seed), torch.Generator().manual_seed(seed)
    new = lambda *shape, dtype=torch.float32: torch.randn(*shape, generator=g, device="cuda", dtype=dtype)  # noqa: E731
    st = dict(case=case)
    if case["op"] in ("policy", "preference"):
        n, t, v = case["seqs"] if case["op"] == "policy" else 2 * case["pairs"], case["tokens"], case["vocab"]
        # logits of a spread that trained heads have, the token that was taken among the likely ones
        logits = new(n, t, v).mul_(2.0)
        targets = torch.randint(0, v, (n, t), generator=g, device="cuda")
        logits.scatter_(-1, targets[..., None], math.log(v) + 2.0 + 1.5 * new(n, t, 1))
        if case["dtype"] == "bf16":
            logits = logits.bfloat16()
        lp = _lp64(logits, targets)
        st.update(logits=logits, targets=targets, mask=_mask(case, (n, t), gc))
        if case["op"] == "policy":
            st.update(advantages=new(n) + 0.3, scale=1.0 / float(st["mask"].sum()),
                      old=(lp + 0.15 * new(n, t)).float() if case["old"] else None, ref=(lp + 0.3 * new(n, t)).float() if case["kl"] else None)
        else:
            st.update(ref=(lp + 0.1 * new(n, t)).float())
    elif case["op"] == "score":
        # normed hidden rows and a head as random-init models have them
        st.update(h=new(case["rows"], case["hidden"]).bfloat16(), w=new(case["vocab"], case["hidden"], dtype=torch.bfloat16).mul_(0.02),
                  targets=torch.randint(0, case["vocab"], (case["rows"],), generator=g, device="cuda"),
                  mask=None if case["scored"] == 1.0 else torch.rand(case["rows"], generator=g, device="cuda") < case["scored"])
    elif case["op"] == "keep":
        # residual rows: a few channels far larger than the rest
        st.update(x=new(case["rows"], case["width"]) * (1 + 20 * (torch.rand(case["width"], generator=g, device="cuda") < 0.01)))
    else:
        st.update(x=new(case["rows"], 2 * case["width"]).mul_(1.4), up=new(case["rows"], case["width"]).mul_(0.01))
    return st


# ---- plain forms -----------------------------------------------------------------------------------------
def _softmax_parts(logits, targets, mask):
    """(e, s, lp): exponentials below the largest, their sums, log-probabilities in 64 bits; rows that are not scored as if all 0."""
    x = torch.where(mask[..., None], logits.float(), 0.0)
    m = x.amax(-1, keepdim=True)
    t = torch.where(mask, targets, 0)[..., None]
    e = torch.exp(x - m)
    s = e.sum(-1, keepdim=True)
    lp = (x.gather(-1, t) - m).double() - torch.log(s.double())
    return e, s, torch.where(mask, lp[..., 0], 0.0), t


def _logit_grad(e, s, t, weight, dtype):
    g = e.div_(s)
    g.scatter_add_(-1, t, torch.full_like(s, -1.0))
    return g.mul_(weight[..., None]).to(dtype)


def _policy(st):
    c, mask = st["case"], st["mask"]
    e, s, lp, t = _softmax_parts(st["logits"], st["targets"], mask)
    a = st["advantages"].double()[:, None].expand(lp.shape)
    rho = torch.ones_like(lp) if st["old"] is None else torch.exp(lp - st["old"])
    lo, hi = 0.2, c["hi"]
    u = torch.minimum(rho * a, rho.clamp(1 - lo, 1 + hi) * a)
    clipped = ((rho > 1 + hi) & (a > 0) | (rho < 1 - lo) & (a < 0)) & mask
    w = torch.where(clipped, 0.0, a * rho)
    kl = torch.zeros_like(lp)
    if st["ref"] is not None:
        d = st["ref"] - lp
        kl = torch.exp(d) - d - 1
        w = w - c["kl"] * (1 - torch.exp(d))
    zero = lambda z: torch.where(mask, z, 0.0)  # noqa: E731
    loss = (zero(c["kl"] * kl - u).sum() * st["scale"]).float()
    grad = _logit_grad(e, s, t, zero(w * st["scale"]).float(), st["logits"].dtype)
    return dict(loss=loss, logprobs=lp.float(), ratio=zero(rho).float(), kl=zero(kl).float(), clipped=clipped, grad=grad)


def _preference(st):
    c, mask = st["case"], st["mask"]
    e, s, lp, t = _softmax_parts(st["logits"], st["targets"], mask)
    count = mask.sum(-1).clamp_min(1).double() if c["average"] else torch.ones(mask.shape[0], dtype=torch.float64, device=mask.device)
    total = lp.sum(-1) / count
    ratio = torch.where(mask, lp - st["ref"], 0.0).sum(-1) / count
    z = c["beta"] * (ratio[0::2] - ratio[1::2])
    pairs, eps = z.shape[0], c["smooth"]
    soft = lambda y: torch.clamp_min(y, 0) + torch.log1p(torch.exp(-y.abs()))  # noqa: E731  (-log sigmoid(-y))
    loss = ((1 - eps) * soft(-z) + eps * soft(z)).sum() / pairs
    dz = (eps / (1 + torch.exp(-z)) - (1 - eps) / (1 + torch.exp(z))) / pairs
    side = torch.stack([-dz, dz], -1).flatten() * c["beta"] / count
    grad = _logit_grad(e, s, t, torch.where(mask, side[:, None], 0.0).float(), st["logits"].dtype)
    return dict(loss=loss.float(), logprobs=total.float(), margins=z.float(), grad=grad)


def _score(st):
    mask = torch.ones(st["h"].shape[0], dtype=torch.bool, device="cuda") if st["mask"] is None else st["mask"]
    x = st["h"].float() @ st["w"].float().t()
    m = x.amax(-1, keepdim=True)
    lp = (x.gather(-1, st["targets"][:, None]) - m)[:, 0]
    x = x.sub_(m)
    e = torch.exp(x)
    s = e.sum(-1)
    log_s = torch.log(s)
    out = dict(logprobs=torch.where(mask, lp - log_s, 0.0))
    if st["case"]["entropy"]:
        out["entropy"] = torch.where(mask, log_s - e.mul_(x).sum(-1) / s, 0.0)
    return out


def _kept(x):
    """The values that rows kept in 8 bits stand for."""
    rows, width = x.shape
    y = torch.nn.functional.pad(x, (0, -width % GROUP)).view(rows, -1, GROUP)
    most = y.abs().amax(-1, keepdim=True)
    q = torch.where(most > 0, torch.round(y * (127.0 / most)), 0.0)
    return (q * (most / 127.0)).view(rows, -1)[:, :width]


def _swiglu(gate, up):
    return gate / (1 + torch.exp(-gate)) * up


def _swiglu_grad(gate, up, g):
    sig = 1 / (1 + torch.exp(-gate))
    return torch.stack([g * up * sig * (1 + gate * (1 - sig)), g * gate * sig], -1).flatten(-2)


def run(st):
    c = st["case"]
    if own:
        from tilerl_b200 import tape as T
        if c["op"] in ("policy", "preference"):
            tape = T.Tape()
            tape.watch(st["logits"])
            if c["op"] == "policy":
                loss, terms = T.policy_loss(tape, st["logits"], st["targets"], st["advantages"], mask=st["mask"], scale=st["scale"], old_logprobs=st["old"],
                                            ref_logprobs=st["ref"], clip_eps=0.2, clip_eps_high=c["hi"], kl_coef=c["kl"])
                out = dict(loss=loss, logprobs=terms.logprobs, ratio=terms.ratio, kl=terms.kl, clipped=terms.clipped)
            else:
                loss, terms = T.preference_loss(tape, st["logits"], st["targets"], st["mask"], st["ref"], beta=c["beta"], label_smoothing=c["smooth"],
                                                average=c["average"])
                out = dict(loss=loss, logprobs=terms.logprobs, margins=terms.margins)
            out["grad"] = tape.backward(loss)[id(st["logits"])]
            return out
        if c["op"] == "score":
            got = T.linear_logprobs(st["h"], st["w"], st["targets"], mask=st["mask"], entropy=c["entropy"])
            return dict(logprobs=got[0], entropy=got[1]) if c["entropy"] else dict(logprobs=got)
        if c["op"] == "keep":
            return T.keep8(st["x"]).rows()
        tape = T.Tape()
        tape.watch(st["x"])
        y = T.swiglu(tape, st["x"], bits=8)
        return dict(out=y, grad=tape.backward(y, st["up"])[id(st["x"])])
    if c["op"] == "policy":
        return _policy(st)
    if c["op"] == "preference":
        return _preference(st)
    if c["op"] == "score":
        return _score(st)
    if c["op"] == "keep":
        return _kept(st["x"])
    x, kept = st["x"], _kept(st["x"])
    return dict(out=_swiglu(x[:, 0::2], x[:, 1::2]), grad=_swiglu_grad(kept[:, 0::2], kept[:, 1::2], st["up"]))


# ---- what a pass cannot do without -----------------------------------------------------------------------
def work(case):
    """Scored rows are about the share of the case's; the others are not read, and their gradients are zeros."""
    op, part = case["op"], case.get("scored", 1.0)
    if op in ("policy", "preference"):
        n = (case["seqs"] if op == "policy" else 2 * case["pairs"]) * case["tokens"]
        size = 4 if case["dtype"] == "fp32" else 2
        return {"bytes": int(n * case["vocab"] * size * (1 + part)) + n * 32, "flops": int(5 * n * case["vocab"] * part)}
    if op == "score":
        rows = max(1, int(case["rows"] * part))
        return {"bytes": 2 * case["hidden"] * (rows + case["vocab"]) + 16 * case["rows"], "flops": 2 * rows * case["hidden"] * case["vocab"]}
    if op == "keep":
        groups = case["rows"] * -(-case["width"] // GROUP)
        return {"bytes": 10 * case["rows"] * case["width"] + 8 * groups, "flops": 5 * case["rows"] * case["width"]}
    n, groups = case["rows"] * case["width"], case["rows"] * -(-2 * case["width"] // GROUP)
    return {"bytes": n * (8 + 4 + 2 + 2 + 4 + 8) + 8 * groups, "flops": 40 * n}


# ---- in 64 bits, from the definitions ----------------------------------------------------------------------
def _row64(x):
    x = x.double()
    low = x - x.max(-1, keepdim=True).values
    z = low.exp().sum(-1, keepdim=True)
    return low, z


def _exact_logits(st, case):
    """One sequence after the other: probabilities in 64 bits for all of it at once would not fit."""
    n = st["mask"].shape[0]
    lps = torch.zeros(st["mask"].shape, dtype=torch.float64, device="cuda")
    picked = []
    for i in range(n):
        picked.append(torch.nonzero(st["mask"][i])[:, 0])
        for at in picked[i].split(128):
            low, z = _row64(st["logits"][i, at])
            lps[i, at] = torch.gather(low, 1, st["targets"][i, at][:, None])[:, 0] - z[:, 0].log()
    weight = torch.zeros_like(lps)
    if case["op"] == "policy":
        adv, beta = st["advantages"].double(), case["kl"]
        rho, kl, clip, loss = (torch.zeros_like(lps) for _ in range(4))
        for i in range(n):
            at, a = picked[i], float(adv[i])
            r = (lps[i, at] - st["old"][i, at].double()).exp() if st["old"] is not None else torch.ones(len(at), dtype=torch.float64, device="cuda")
            rho[i, at] = r
            if a > 0:
                out = r > 1 + case["hi"]
                gain = torch.where(out, (1 + case["hi"]) * a, r * a)
            else:
                out = (r < 0.8) if a < 0 else torch.zeros_like(r, dtype=torch.bool)
                gain = torch.where(out, 0.8 * a, r * a)
            clip[i, at] = out.double()
            w = torch.where(out, 0.0, a * r)
            if st["ref"] is not None:
                d = st["ref"][i, at].double() - lps[i, at]
                kl[i, at] = torch.expm1(d) - d
                w = w + beta * torch.expm1(d)
            loss[i, at] = beta * kl[i, at] - gain
            weight[i, at] = w * st["scale"]
        out = dict(loss=loss.sum() * st["scale"], logprobs=lps, ratio=rho, kl=kl, clipped=clip > 0)
    else:
        sums, ratios, norm = [], [], []
        for i in range(n):
            k = max(1, len(picked[i])) if case["average"] else 1
            sums.append(lps[i].sum() / k)
            ratios.append((lps[i, picked[i]] - st["ref"][i, picked[i]].double()).sum() / k)
            norm.append(k)
        margins, losses = [], []
        for p in range(n // 2):
            z = case["beta"] * (ratios[2 * p] - ratios[2 * p + 1])
            margins.append(z)
            losses.append(-(1 - case["smooth"]) * torch.nn.functional.logsigmoid(z) - case["smooth"] * torch.nn.functional.logsigmoid(-z))
            slope = case["smooth"] * torch.sigmoid(z) - (1 - case["smooth"]) * torch.sigmoid(-z)
            for i, sign in ((2 * p, -1.0), (2 * p + 1, 1.0)):
                weight[i, picked[i]] = sign * slope * case["beta"] / norm[i] / (n // 2)
        out = dict(loss=torch.stack(losses).mean(), logprobs=torch.stack(sums), margins=torch.stack(margins))
    grad = torch.zeros(st["logits"].shape, dtype=torch.float64, device="cuda")
    for i in range(n):
        for at in picked[i].split(128):
            low, z = _row64(st["logits"][i, at])
            p = low.exp_().div_(z)
            p[torch.arange(len(at), device="cuda"), st["targets"][i, at]] -= 1.0
            grad[i, at] = p.mul_(weight[i, at][:, None])
    out["grad"] = grad
    return out


def _exact_kept(x):
    """Scale, quotient and product are of 32 bits by definition; what they stand for is not."""
    parts = []
    for block in x.split(GROUP, dim=-1):
        most = block.abs().max(-1, keepdim=True).values
        codes = torch.round(block * torch.where(most > 0, 127.0 / most, 0.0))
        parts.append(codes.double() * (most / 127.0).double())
    return torch.cat(parts, -1)


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] in ("policy", "preference"):
        return _exact_logits(st, case)
    if case["op"] == "score":
        n = st["h"].shape[0]
        lp, ent = (torch.zeros(n, dtype=torch.float64, device="cuda") for _ in range(2))
        at = torch.arange(n, device="cuda") if st["mask"] is None else torch.nonzero(st["mask"])[:, 0]
        for rows in at.split(512):
            x = torch.cat([st["h"][rows].double() @ part.double().t() for part in st["w"].split(16384)], -1)
            low, z = _row64(x)
            lp[rows] = torch.gather(low, 1, st["targets"][rows][:, None])[:, 0] - z[:, 0].log()
            ent[rows] = z[:, 0].log() - (low.exp() * low).sum(-1) / z[:, 0]
        return dict(logprobs=lp, entropy=ent) if case["entropy"] else dict(logprobs=lp)
    if case["op"] == "keep":
        return _exact_kept(st["x"])
    gate, up = st["x"][:, 0::2].double(), st["x"][:, 1::2].double()
    kept = _exact_kept(st["x"])
    a, b, g = kept[:, 0::2], kept[:, 1::2], st["up"].double()
    sig = torch.sigmoid(a)
    grad = torch.empty_like(kept)
    grad[:, 0::2] = g * b * (sig + a * sig * (1 - sig))
    grad[:, 1::2] = g * a * sig
    return dict(out=gate * torch.sigmoid(gate) * up, grad=grad)
