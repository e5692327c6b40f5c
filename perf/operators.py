"""Scoring and distillation of rows of logits: what is measured, and the operators' plain forms.

Three operators over the rows of a transducer's output layer (one row per lattice cell, R rows of V
entries, z = x / temperature, p = softmax(z), lse = logsumexp(z)):

  scores   token_logprobs: log p of M given tokens of a row (-1: no token, 0), the entropy of p, the K
           most probable entries (ties to the lowest index); backward through all three.
  distill  distill_loss: temperature^2 * KL(q || p) per row for a teacher's K top logits.  Without a
           tail q = softmax of the list; with one the list holds log-probabilities, the mass it leaves
           is one more class and so is the student's mass outside the list.  An index of -1 is absent.
  joint    joint_token_logprobs: the scores of x = h @ weight.T + bias, fp16 / bf16, forward only.

`run` computes them in elementary torch operations, or, where `own` is set, through the package.
"""
import math

import torch

own = False

_DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_LARGEST = 311449 * 1024  # logits of the largest listed case of the two stored-logits operators


def listed():
    return [
        # one step of a beam search: 4 utterances x 8 hypotheses, an output layer of 1024 entries
        dict(name="scores_step", op="scores", R=32, V=1024, dtype="f32", M=1, K=8, T=1.0, train=False, pad=0, mask=0.0),
        # a teacher's pass over a whole batch: 32 utterances, T in [100,250], U in [20,80]; blank and label
        # of every cell, entropy as a confidence, four alternatives
        dict(name="scores_lattice", op="scores", R=311449, V=1024, dtype="f32", M=2, K=4, T=1.0, train=False, pad=0,
             mask=0.0),
        # training on token scores with an entropy bonus, half-precision logits of 4096 word pieces
        dict(name="scores_train", op="scores", R=71387, V=4096, dtype="f16", M=2, K=4, T=1.0, train=True, pad=0, mask=0.0),
        # phonemes: odd short rows, the label scores trained
        dict(name="scores_phones", op="scores", R=600000, V=41, dtype="f32", M=2, K=3, T=1.0, train=True, pad=0, mask=0.0),
        # a vocabulary of an odd 50257 entries, some of them masked out, sampled at a temperature
        dict(name="scores_wide", op="scores", R=2048, V=50257, dtype="bf16", M=1, K=32, T=0.7, train=False, pad=0,
             mask=0.05),
        # the smallest batch there is: 4 utterances, 32 entries
        dict(name="distill_small", op="distill", R=737, V=32, dtype="f32", K=4, T=1.0, tail=True, reduction="mean", pad=0),
        # a whole batch against a teacher's 16 best entries per cell
        dict(name="distill_lattice", op="distill", R=311449, V=1024, dtype="f32", K=16, T=2.0, tail=False,
             reduction="mean", pad=0),
        # long utterances, a short vocabulary, the teacher collapsed to (blank, label, everything else)
        dict(name="distill_collapsed", op="distill", R=1513461, V=128, dtype="f32", K=2, T=1.0, tail=True,
             reduction="mean", pad=0),
        # logits in rows padded to a multiple of 64, an odd vocabulary, a loss per cell
        dict(name="distill_padded", op="distill", R=25841, V=4233, dtype="bf16", K=32, T=1.0, tail=True,
             reduction="none", pad=55),
        # one step of a greedy or beam search straight from the joint rows
        dict(name="joint_step", op="joint", R=8, V=1024, H=512, dtype="bf16", M=1, K=4, T=1.0),
        # a batch of hypotheses, 4096 word pieces
        dict(name="joint_beam", op="joint", R=512, V=4096, H=640, dtype="f16", M=1, K=8, T=1.0),
        # a teacher scoring a whole batch without storing its logits
        dict(name="joint_lattice", op="joint", R=311449, V=1024, H=512, dtype="bf16", M=2, K=8, T=1.0),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["scores", "distill", "joint"])
    if op == "joint":
        V, H = _log_int(rng, 32, 8192), 32 * rng.randint(2, 32)
        R = _log_int(rng, 1, max(1, min(311449, _LARGEST * 512 // (V * H))))
        return dict(op=op, R=R, V=V, H=H, dtype=rng.choice(["f16", "bf16"]), M=rng.randint(0, 3),
                    K=rng.randint(1, min(V, 16)), T=rng.choice([1.0, 0.8, 2.0]))
    V = _log_int(rng, 8, 50257)
    R = _log_int(rng, 1, max(1, min(1513461, _LARGEST // (2 * V))))
    case = dict(op=op, R=R, V=V, dtype=rng.choice(["f32", "f16", "bf16"]), T=rng.choice([1.0, 0.7, 2.0]),
                pad=rng.choice([0, 0, 0, (-V) % 64]))
    if op == "scores":
        case.update(M=rng.randint(0, 3), K=rng.randint(1, min(V // 2, 32)), train=rng.random() < 0.5,
                    mask=rng.choice([0.0, 0.0, 0.05]))
    else:
        case.update(K=rng.randint(1, min(V - 1, 64)), tail=rng.random() < 0.5, reduction=rng.choice(["mean", "none"]))
    return case


def _logits(R, V, gen, dtype, pad):
    """Rows as an output layer gives them: a spread of two nats, and in two thirds of the rows the blank
    (entry 0) with most of the mass.  With `pad` the rows are that much further apart than they are long."""
    buf = torch.empty((R, V + pad), dtype=dtype, device="cuda")
    step = max(1, (1 << 28) // (V + pad))
    for r in range(0, R, step):
        z = torch.randn((min(step, R - r), V + pad), device="cuda", generator=gen).mul_(2.0)
        z[:, 0] += (3.0 + math.log(V)) * (torch.rand(z.shape[0], device="cuda", generator=gen) < 0.66)
        buf[r:r + step] = z
    return buf[:, :V]


def _tokens(R, V, M, gen):
    """Blank first, then labels; one cell in fifty has no label."""
    t = torch.randint(0, V, (R, M), device="cuda", generator=gen, dtype=torch.int32)
    t[torch.rand((R, M), device="cuda", generator=gen) < 0.02] = -1
    t[:, :1] = 0
    return t


def _scale(case):
    """What multiplies the loss before its backward pass: a loss scaler's factor where gradients are fp16."""
    return 256.0 if case["dtype"] == "f16" else 1.0 / case["R"]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed) % (1 << 62))
    op, R, V, dt = case["op"], case["R"], case["V"], _DT[case["dtype"]]
    s = dict(case)
    if op == "joint":
        # Values of an 8-bit grid, as a quantised layer holds them: every sum of products is then exact in
        # 32 bits whatever its order, and the ranking of the alternatives is a fact of the inputs.
        H = case["H"]
        s["h"] = (torch.tanh(torch.randn((R, H), device="cuda", generator=gen)) * 128).round_().div_(128).to(dt)
        w = torch.randn((V, H), device="cuda", generator=gen) * (2.0 / (0.63 * math.sqrt(H)))
        s["weight"] = (w * 512).round_().clamp_(-255, 255).div_(512).to(dt)
        s["bias"] = (torch.randn(V, device="cuda", generator=gen) * 512).round_().clamp_(-255, 255).div_(512).to(dt)
        s["tokens"] = _tokens(R, V, case["M"], gen) if case["M"] else None
        return s
    x = _logits(R, V, gen, dt, case["pad"])
    if op == "scores":
        if case["mask"]:
            out = torch.rand(V, device="cuda", generator=gen) < case["mask"]
            out[0] = False
            x[:, out] = -math.inf
        s["tokens"] = _tokens(R, V, case["M"], gen) if case["M"] else None
        if case["train"]:
            x = x.detach().requires_grad_(True)
            g = lambda *shape: torch.randn(shape, device="cuda", generator=gen) * _scale(case)  # noqa: E731
            s["g_logprobs"] = g(R, case["M"]) if case["M"] else None
            s["g_entropy"] = g(R)
            s["g_top"] = g(R, case["K"])
    else:
        # the teacher: the same rows with another nat of noise, its best K of every row
        tops, idx = [], []
        step = max(1, (1 << 28) // V)
        for r in range(0, R, step):
            z = x[r:r + step].float()
            z = (z + torch.randn(z.shape, device="cuda", generator=gen)) / case["T"]
            v, i = z.topk(case["K"], dim=1)
            tops.append(v - torch.logsumexp(z, 1, keepdim=True) if case["tail"] else v * case["T"])
            idx.append(i.to(torch.int32))
        s["top"], s["index"] = torch.cat(tops), torch.cat(idx)
        if case["K"] > 2:  # lists cut short, as a teacher with a probability floor sends them
            s["index"][torch.rand(R, device="cuda", generator=gen) < 0.05, case["K"] - 1] = -1
        if case["reduction"] == "none":
            s["g"] = torch.rand(R, device="cuda", generator=gen) * _scale(case)
        else:
            s["g"] = torch.full((), _scale(case) * R, device="cuda")
        x = x.detach().requires_grad_(True)
    s["x"] = x
    return s


# ---- plain forms ---------------------------------------------------------------------------------
def _scores_plain(z, s):
    """z: (R, V) fp32 logits; ranks them, scores them, and where asked the gradient."""
    T, K, tok = s["T"], s["K"], s["tokens"]
    index = torch.sort(z, dim=1, descending=True, stable=True)[1][:, :K]
    z = z / T
    z = z - z.amax(1, keepdim=True)
    total = torch.exp(z).sum(1, keepdim=True)
    logp = z - torch.log(total)
    p = torch.exp(logp)
    plogp = torch.where(p > 0, p * logp, 0.0)
    entropy = -plogp.sum(1)
    out = {"entropy": entropy, "top_logprobs": logp.gather(1, index), "top_index": index.to(torch.int32)}
    if tok is not None:
        at, there = tok.clamp(min=0).long(), tok >= 0
        out["logprobs"] = torch.where(there, logp.gather(1, at), 0.0)
    if s.get("train"):
        d = -(plogp + p * entropy[:, None]) * s["g_entropy"][:, None] - p * s["g_top"].sum(1, keepdim=True)
        d.scatter_add_(1, index, s["g_top"])
        if tok is not None:
            g = torch.where(there, s["g_logprobs"], 0.0)
            d -= p * g.sum(1, keepdim=True)
            d.scatter_add_(1, at, g)
        out["dx"] = (d / T).to(s["x"].dtype)
    return out


def _distill_plain(s):
    x, T, idx = s["x"].detach(), s["T"], s["index"]
    z = x.float() / T
    there = idx >= 0
    at = idx.clamp(min=0).long()
    t = torch.where(there, s["top"], -math.inf)
    if s["tail"]:
        q = torch.exp(t)
        logq = t
        rest = (1.0 - torch.exp(t.double()).sum(1, keepdim=True)).clamp(min=0.0).float()  # 32 bits would leave noise
    else:
        t = t / T
        logq = t - torch.logsumexp(t, 1, keepdim=True)
        q = torch.exp(logq)
    lse = torch.logsumexp(z, 1, keepdim=True)
    terms = torch.where(there, q * (logq - (z.gather(1, at) - lse)), 0.0)
    loss = terms.sum(1)
    mass = q.sum(1, keepdim=True)
    d = None
    if s["tail"]:
        # entries outside the list: an absent index marks a spare column
        seen = torch.zeros((z.shape[0], z.shape[1] + 1), dtype=torch.bool, device=z.device)
        seen.scatter_(1, torch.where(there, at, z.shape[1]), True)
        others = z.masked_fill(seen[:, :-1], -math.inf)
        lse_r = torch.logsumexp(others, 1, keepdim=True)
        loss = loss + torch.where(rest > 0, rest * (torch.log(rest) - (lse_r - lse)), 0.0).squeeze(1)
        d = torch.exp(z - lse) * (mass + rest) - rest * torch.exp(others - lse_r)
    else:
        d = torch.exp(z - lse) * mass
    d.scatter_add_(1, at, torch.where(there, -q, 0.0))
    loss = loss * (T * T)
    if s["reduction"] == "mean":
        return {"loss": loss.mean(), "dx": (d * (T / x.shape[0] * s["g"])).to(x.dtype)}
    return {"loss": loss, "dx": (d * (T * s["g"][:, None])).to(x.dtype)}


def _named(out):
    return {k: v for k, v in sorted(out._asdict().items()) if v is not None and k != "lse"}


def run(state):
    s = state
    if own:
        import compactwarprnntloss_amd as pkg
        if s["op"] == "joint":
            return _named(pkg.joint_token_logprobs(s["h"], s["weight"], s["bias"], s["tokens"], top_k=s["K"],
                                                   entropy=True, temperature=s["T"]))
        if s["op"] == "distill":
            loss = pkg.distill_loss(s["x"], s["top"], s["index"], temperature=s["T"], tail=s["tail"],
                                    reduction=s["reduction"])
            dx, = torch.autograd.grad(loss, s["x"], s["g"])
            return {"loss": loss.detach(), "dx": dx}
        res = pkg.token_logprobs(s["x"], s["tokens"], top_k=s["K"], entropy=True, temperature=s["T"])
        out = _named(res)
        if s["train"]:
            pairs = [(res.entropy, s["g_entropy"]), (res.top_logprobs, s["g_top"])]
            if s["tokens"] is not None:
                pairs.append((res.logprobs, s["g_logprobs"]))
            out = {k: v.detach() for k, v in out.items()}
            out["dx"], = torch.autograd.grad([a for a, _ in pairs], s["x"], [b for _, b in pairs])
        return dict(sorted(out.items()))  # dx among them
    if s["op"] == "joint":
        z = s["h"].float() @ s["weight"].float().T + s["bias"].float()
        return dict(sorted(_scores_plain(z, s).items()))
    if s["op"] == "distill":
        return _distill_plain(s)
    return dict(sorted(_scores_plain(s["x"].detach().float(), s).items()))


def work(case):
    """Each input read once (a training pass reads the logits once more: the gradient of a row needs its
    sum first, and no cache holds the batch), each output written once; about eight operations a logit
    and direction besides the product of the joint form."""
    R, V, K, M = case["R"], case["V"], case["K"], case.get("M", 0)
    e = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "joint":
        H = case["H"]
        return {"bytes": e * (R * H + V * H + V) + R * (8 * M + 8 * K + 4), "flops": 2 * R * V * H + 8 * R * V}
    if case["op"] == "scores":
        nbytes = R * V * e + R * (8 * M + 8 * K + 4)
        if case["train"]:
            nbytes += 2 * R * V * e + R * (4 * M + 4 * K + 4)
        return {"bytes": nbytes, "flops": (2 if case["train"] else 1) * 8 * R * V}
    return {"bytes": 3 * R * V * e + R * (8 * K + 4), "flops": 2 * 8 * R * V}


# ---- the definition in 64 bits ---------------------------------------------------------------------
def _exact_rows_scores(z, tok, T, K, g):
    order = torch.argsort(-z, dim=1, stable=True)[:, :K]
    logp = torch.log_softmax(z / T, dim=1)
    p = logp.exp()
    contrib = torch.nan_to_num(p * logp, nan=0.0)
    H = -contrib.sum(1, keepdim=True)
    out = {"entropy": H[:, 0], "top_index": order.to(torch.int32), "top_logprobs": torch.gather(logp, 1, order)}
    present = None if tok is None else (tok >= 0).double()
    if tok is not None:
        out["logprobs"] = torch.nan_to_num(torch.gather(logp, 1, tok.long() * (tok >= 0)), neginf=-math.inf) * present
    if g is not None:
        # d log p_i / d x_v = ([v = i] - p_v) / T;  d H / d x_v = -p_v (log p_v + H) / T
        w = torch.zeros_like(z)
        rows = torch.arange(z.shape[0], device=z.device)
        for k in range(K):
            w[rows, order[:, k]] += g["top"][:, k].double()
        if tok is not None:
            for m in range(tok.shape[1]):
                w[rows, tok[:, m].long() * (tok[:, m] >= 0)] += g["lp"][:, m].double() * present[:, m]
        out["dx"] = (w - p * w.sum(1, keepdim=True) - (contrib + p * H) * g["ent"].double()[:, None]) / T
    return out


def _exact_rows_distill(x, top, idx, T, tail, g):
    z = x / T
    V = z.shape[1]
    there = idx >= 0
    t = top.double() if tail else top.double() / T
    t = t.masked_fill(~there, -math.inf)
    q = t.exp() if tail else torch.softmax(t, 1)
    spread = torch.zeros((z.shape[0], V + 1), dtype=torch.float64, device=z.device)
    listed_ = torch.zeros_like(spread)
    at = torch.where(there, idx.long(), torch.full_like(idx, V).long())
    rows = torch.arange(z.shape[0], device=z.device)
    for k in range(idx.shape[1]):
        spread[rows, at[:, k]] += q[:, k]
        listed_[rows, at[:, k]] = 1.0
    spread, listed_ = spread[:, :V], listed_[:, :V]
    logp = torch.log_softmax(z, 1)
    p = logp.exp()
    ent = torch.special.entr(q).sum(1)          # -sum q log q: the teacher's own entropy
    loss = -ent - (spread * logp).sum(1)
    target = spread
    if tail:
        rest = (1 - q.sum(1)).clamp(min=0)
        p_out = p * (1 - listed_)
        mass = p_out.sum(1)
        loss = loss - torch.special.entr(rest) - rest * mass.log()
        target = spread + rest[:, None] * p_out / mass[:, None]
    d = p * target.sum(1, keepdim=True) - target
    return {"loss": loss * T * T, "dx": d * T * g.double()[:, None]}


def exact(case, seed):
    s = prepare(case, seed)
    R, V = case["R"], case["V"]
    step = max(1, (1 << 25) // V)
    parts = []
    for r in range(0, R, step):
        cut = slice(r, min(R, r + step))
        pick = lambda k: None if s.get(k) is None else s[k][cut]  # noqa: E731
        if case["op"] == "distill":
            g = s["g"][cut] if case["reduction"] == "none" else (s["g"].double() / R).expand(cut.stop - r)
            parts.append(_exact_rows_distill(s["x"].detach()[cut].double(), s["top"][cut], s["index"][cut], case["T"],
                                             case["tail"], g))
            continue
        if case["op"] == "joint":
            z = torch.addmm(s["bias"].double(), s["h"][cut].double(), s["weight"].double().T)
        else:
            z = s["x"].detach()[cut].double()
        g = dict(lp=pick("g_logprobs"), ent=pick("g_entropy"), top=pick("g_top")) if case.get("train") else None
        parts.append(_exact_rows_scores(z, pick("tokens"), case["T"], case["K"], g))
    whole = {k: torch.cat([p[k] for p in parts]) for k in parts[0]}
    if case["op"] == "distill" and case["reduction"] == "mean":
        whole["loss"] = whole["loss"].mean()
        return whole
    return whole if case["op"] == "distill" else dict(sorted(whole.items()))
