"""Plain 64-bit restatements of the row operators (scores and distillation), for their tests: elementary
operations on float64 tensors, gradients by formula, and the bounds the fp32 kernels are held to."""
import math

import torch

EPS32 = 2.0 ** -24  # half a step of fp32, relative


def top_ref(x, k):
    """Indices of the k largest entries of each row, equal ones by ascending index (NaN as -inf)."""
    z = torch.nan_to_num(x.double(), nan=-math.inf, posinf=math.inf, neginf=-math.inf) + 0.0
    return torch.sort(z, dim=1, descending=True, stable=True)[1][:, :k]


def scores_ref(x, tokens, k, T):
    """dict(logp (R, V), p, entropy, lse, logprobs, top_index, top_logprobs) in float64."""
    z = x.double() / T
    m = z.amax(1, keepdim=True)
    empty = (m == -math.inf).squeeze(1)
    m = torch.where(m == -math.inf, 0.0, m)
    s = torch.exp(z - m).sum(1, keepdim=True)
    lse = (m + torch.log(s)).squeeze(1)
    # not z - lse: next to a maximum of 1e38 the sum's logarithm is lost even in 64 bits
    logp = torch.where((z == -math.inf) & ~torch.isnan(lse)[:, None], -math.inf, (z - m) - torch.log(s))
    p = torch.exp(logp)
    plogp = torch.where(p == 0, 0.0, p * logp)
    ent = torch.where(empty & ~torch.isnan(lse), 0.0, -plogp.sum(1))
    out = dict(logp=logp, p=p, entropy=ent, lse=lse)
    if tokens is not None:
        V = x.size(1)
        inside = (tokens >= 0) & (tokens < V)
        lp = logp.gather(1, torch.where(inside, tokens, 0).long())
        out["logprobs"] = torch.where(inside, lp, torch.where(tokens == -1, 0.0, math.nan))
    if k:
        idx = top_ref(x, k)
        out["top_index"] = idx
        out["top_logprobs"] = logp.gather(1, idx)
    return out


def scores_grad_ref(x, tokens, k, T, g_logprobs=None, g_entropy=None, g_lse=None, g_top=None):
    """(dx, scale): the gradient in float64 and what its error is measured against, element by element."""
    ref = scores_ref(x, tokens, k, T)
    R, V = x.shape
    logp, p = ref["logp"], ref["p"]
    w = torch.zeros((R, V), dtype=torch.float64, device=x.device)
    absw = torch.zeros_like(w)
    if tokens is not None and g_logprobs is not None:
        inside = (tokens >= 0) & (tokens < V)
        at = torch.where(inside, tokens, 0).long()
        for j in range(tokens.size(1)):
            g = torch.where(inside[:, j], g_logprobs[:, j].double(), 0.0)
            w.scatter_add_(1, at[:, j:j + 1], g[:, None])
            absw.scatter_add_(1, at[:, j:j + 1], g.abs()[:, None])
    if k and g_top is not None:
        for j in range(k):
            w.scatter_add_(1, ref["top_index"][:, j:j + 1], g_top[:, j:j + 1].double())
            absw.scatter_add_(1, ref["top_index"][:, j:j + 1], g_top[:, j:j + 1].double().abs())
    W, absW = w.sum(1, keepdim=True), absw.sum(1, keepdim=True)
    d = w - p * W
    scale = absw + p * absW
    if g_lse is not None:
        d = d + p * g_lse.double()[:, None]
        scale = scale + p * g_lse.double().abs()[:, None]
    if g_entropy is not None:
        pl = torch.where(p == 0, 0.0, p * logp)
        gh = g_entropy.double()[:, None]
        d = d - gh * (pl + p * ref["entropy"][:, None])
        scale = scale + gh.abs() * (pl.abs() + p * (1 + ref["entropy"][:, None]))
    d = torch.where((ref["lse"] == -math.inf)[:, None], 0.0, d)
    return d / T, torch.nan_to_num(scale) / T


def softmax_slack(V):
    """Relative error, in units of EPS32, of a sum of V exponentials formed in fp32: two roundings of every
    exponent (2 |t| ln 2 each way, weighted by p: at most about 2 log2 V), the exponential itself (2), and the
    chain of additions (8 per chunk of 1024 in a lane, one per chunk, 6 to 10 across lanes and waves)."""
    return 2 * math.log2(V + 1) + 2 + 8 + V / 1024 + 10


def distill_ref(x, top, index, T, tail):
    """(loss (R,), dx for unit gradients (R, V), scale (R, V)) in float64."""
    z = x.double() / T
    R, V = z.shape
    there = index >= 0
    at = torch.where(there, index, 0).long()
    lse = torch.logsumexp(z, 1, keepdim=True)
    logp = z - lse
    p = torch.exp(logp)
    t = torch.where(there, top.double(), -math.inf)
    if tail:
        q, logq = torch.exp(t), t
    else:
        t = t / T
        none = (t.amax(1, keepdim=True) == -math.inf)
        logq = torch.where(none, -math.inf, t - torch.logsumexp(t, 1, keepdim=True))
        q = torch.exp(logq)
    lp = logp.gather(1, at)
    loss = torch.where(there & (q > 0), q * (logq - lp), 0.0).sum(1)
    scale_loss = torch.where(there & (q > 0), q * (logq.abs() + lp.abs() + 1), 0.0).sum(1)
    spread = torch.zeros_like(z)
    hit = torch.zeros_like(z)
    for j in range(index.size(1)):
        spread.scatter_add_(1, at[:, j:j + 1], torch.where(there[:, j:j + 1], q[:, j:j + 1], 0.0))
        hit.scatter_add_(1, at[:, j:j + 1], there[:, j:j + 1].double())
    Q = q.sum(1, keepdim=True)
    d = p * Q - spread
    scale = p * Q + spread
    if tail:
        rest = (1 - Q).clamp(min=0)
        others = z.masked_fill(hit > 0, -math.inf)
        lse_r = torch.logsumexp(others, 1, keepdim=True)
        live = lse_r > -math.inf
        rest = torch.where(live, rest, 0.0)
        term = torch.where(rest > 0, rest * (torch.log(rest) - (lse_r - lse)), 0.0)
        loss = loss + term.squeeze(1)
        scale_loss = scale_loss + torch.where(rest > 0, rest * (torch.log(rest).abs() + (lse_r - lse).abs() + 1), 0.0).squeeze(1)
        pr = torch.where(live & (hit == 0), torch.exp(others - torch.where(live, lse_r, 0.0)), 0.0)
        d = p * (Q + rest) - spread - rest * pr
        scale = p * (Q + rest) + spread + rest * pr
    return loss * T * T, d * T, scale * T, scale_loss * T * T


def tiny(dtype):
    """Half the smallest step of the type: what rounding near zero may lose."""
    return {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -126}.get(dtype, 2.0 ** -126)


def half_step(dtype):
    return EPS32 if dtype == torch.float64 else torch.finfo(dtype).eps / 2
