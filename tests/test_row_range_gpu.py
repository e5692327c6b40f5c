"""Row operators on logits far from zero and at small temperatures: rows and chunks masked with finite constants,
shifted rows, m / T beyond what one fp32 number can hold beside the differences that matter."""
import math

import pytest
import torch

import compactwarprnntloss_amd as pkg
from tests.rowrefs import EPS32, half_step, scores_grad_ref, scores_ref, softmax_slack, tiny

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
LEVELS = [-1e6, -1e9, -1e10, -1e12, -1e20, -1e30]
# one group of lanes per row, one wave with one, two and three chunks, four and sixteen waves (with and without
# a second chunk of their own)
WIDTHS = [16, 41, 500, 1024, 2049, 2500, 4100, 9000, 20000]


def masked_rows(V, level, dtype, seed=0):
    """Ten rows: uniform at the level, the level in the first, last or every chunk but one, in all entries but
    one, in every other entry; nothing at the level; shifted by it where that leaves differences."""
    gen = torch.Generator(device=DEV).manual_seed(seed + V)
    x = torch.randn((10, V), device=DEV, generator=gen) * 2
    at = torch.arange(V, device=DEV)
    first = min(1024, V // 2)
    x[0] = level
    x[1, :first] = level
    x[2, V - first:] = level
    x[3, at != V // 2] = level
    x[4, at != V - 1] = level
    x[5, at != 0] = level
    x[6, ::2] = level
    x[7] = torch.where(at // 1024 % 4 == 0, level, x[7])  # all chunks of one of four waves
    x[7, V - 1] = 1.0
    x[8] += level / 1e3
    return x.to(dtype), gen


def slack_of(V):
    """softmax_slack and a third rounding of every exponent, where the maximum is subtracted first: ln 2 times the
    mean exponent, at most log2 V, in half steps."""
    return softmax_slack(V) + math.log2(V + 1)


def near(got, want, tol, what):
    fin = torch.isfinite(want)
    assert torch.equal(got[~fin].double(), want[~fin]), what
    err = (got.double() - want)[fin].abs() - tol[fin]
    assert not torch.isnan(got[fin]).any() and (err.numel() == 0 or float(err.max()) <= 0), (what, got, want)


def check_scores(x, T, gen, K=4, bits=40):
    """`bits`: how far below 2^-log2(V) a probability is held to its own size."""
    R, V = x.shape
    K = min(K, V)
    tok = torch.randint(0, V, (R, 3), device=DEV, dtype=torch.int32, generator=gen)
    tok[:, 0] = 0
    xr = x.to(torch.float32) if x.dtype == torch.float64 else x
    ref = scores_ref(xr, tok, K, T)
    x = x.detach().requires_grad_(True)
    out = pkg.token_logprobs(x, tok, top_k=K, entropy=True, temperature=T)
    slack = EPS32 * slack_of(V)
    assert torch.equal(out.top_index.long(), ref["top_index"])
    out_d = [t.detach() for t in out[:4]]
    near(out_d[2], ref["lse"], slack + EPS32 * ref["lse"].abs(), "lse")
    near(out_d[0], ref["logprobs"], slack + EPS32 * ref["logprobs"].abs(), "logprobs")
    near(out_d[3], ref["top_logprobs"], slack + EPS32 * ref["top_logprobs"].abs(), "top")
    near(out_d[1], ref["entropy"], slack * (2 + 2 * math.log2(V + 1)) + EPS32 * ref["entropy"].abs(), "entropy")
    g = [torch.randn(t.shape, device=DEV, generator=gen) for t in out_d]
    dx, = torch.autograd.grad([out.logprobs, out.entropy, out.lse, out.top_logprobs], x, g)
    want, scale = scores_grad_ref(xr, tok, K, T, *g)
    # as for ordinary logits (p to the slack of its sum and the roundings, here three, of its own exponent); what
    # the exponential flushes below 2^-126 is multiplied by at most a thousand / T
    rel = EPS32 * (2 * slack_of(V) + 3 * (math.log2(V + 1) + bits) + 3 + K)
    near(dx, want, half_step(x.dtype) * want.abs() + tiny(x.dtype) + 2.0 ** -126 * 1000 / T + rel * scale, "dx")


@pytest.mark.parametrize("T", [0.7, 1.0, 2.0])
@pytest.mark.parametrize("level", LEVELS)
@pytest.mark.parametrize("V", WIDTHS)
def test_scores_of_rows_masked_with_a_finite_constant(V, level, T):
    x, gen = masked_rows(V, level, torch.float32)
    check_scores(x, T, gen)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float64])
@pytest.mark.parametrize("level", [-1e6, -1e10, -1e30])
@pytest.mark.parametrize("V", [41, 1024, 2500, 9000])
def test_scores_of_masked_rows_of_other_types(V, level, dtype):
    x, gen = masked_rows(V, level, dtype, seed=1)
    check_scores(x, 1.0, gen)


@pytest.mark.parametrize("T", [1e-6, 1e-5, 1e-4])
@pytest.mark.parametrize("V", [16, 500, 1024, 2500, 9000, 20000])
def test_scores_at_small_temperatures(V, T):
    """Ordinary logits (one entry takes nearly everything), peaks, and rows whose entries differ by about T."""
    gen = torch.Generator(device=DEV).manual_seed(V)
    x = torch.randn((9, V), device=DEV, generator=gen) * 2
    x[1, V // 2] = 100.0
    x[2, V - 1] = 37.3
    x[3:6] = x[3:6] * T + torch.tensor([0.03, 5.0, -77.0], device=DEV)[:, None]
    x[6] = 19.0
    x[7] = torch.where(torch.arange(V, device=DEV) < V // 2, -4.0, x[7] * T + 3.0)
    check_scores(x, T, gen, bits=126)


@pytest.mark.parametrize("V", [41, 1024, 2500, 9000])
def test_scores_of_shifted_rows(V):
    """A constant added to a row changes nothing but lse: entries on a grid that the shifted row holds exactly."""
    gen = torch.Generator(device=DEV).manual_seed(V)
    base = torch.randint(-16, 17, (6, V), device=DEV, generator=gen).float() / 2
    plain = pkg.token_logprobs(base, top_k=3, entropy=True)
    for shift in (2.0 ** 10, 2.0 ** 15, 2.0 ** 16, 2.0 ** 20, -1e6, 2.0 ** 22):
        x = base + shift
        check_scores(x, 1.0, gen)
        out = pkg.token_logprobs(x, top_k=3, entropy=True)
        assert torch.equal(out.top_index, plain.top_index)
        tol = 2 * EPS32 * slack_of(V)
        assert float((out.top_logprobs - plain.top_logprobs).abs().max()) <= tol + 2 * EPS32 * 20
        assert float((out.entropy - plain.entropy).abs().max()) <= tol * (2 + 2 * math.log2(V + 1)) + 2 * EPS32 * 12


@pytest.mark.parametrize("V", [2049, 5000, 20000])
@pytest.mark.parametrize("base", [30.0, 1000.0, 20000.0, 40000.0])
def test_rows_whose_maximum_rises_from_chunk_to_chunk(V, base):
    """Sums measured against one maximum and moved to the next: the move loses nothing of what the products with
    the maxima were rounded by."""
    gen = torch.Generator(device=DEV).manual_seed(V)
    x = base + torch.randn((8, V), device=DEV, generator=gen) * 0.25
    x += 0.37 * (torch.arange(V, device=DEV) // 1024) / max(1, V // 1024)
    check_scores(x, 1.0, gen)


def distill_formula(x, top, index, T, tail):
    """(loss, dx, scale of dx, scale of the loss) of distill_loss in float64, every softmax next to its own maximum."""
    z = x.double() / T
    there = index >= 0
    at = torch.where(there, index, 0).long()
    m = z.amax(1, keepdim=True)
    s = torch.exp(z - m).sum(1, keepdim=True)
    logp = (z - m) - torch.log(s)
    p = torch.exp(logp)
    t = torch.where(there, top.double(), -math.inf)
    if tail:
        logq = t
    else:
        mt = t.amax(1, keepdim=True)
        logq = (t - mt) / T
        logq = logq - torch.log(torch.exp(logq).sum(1, keepdim=True))
    q = torch.exp(logq)
    lp = logp.gather(1, at)
    loss = torch.where(q > 0, q * (logq - lp), 0.0).sum(1)
    size = torch.where(q > 0, q * (logq.abs() + lp.abs() + 1), 0.0).sum(1)
    listed = torch.zeros_like(z).scatter_add_(1, at, there.double()) > 0
    spread = torch.zeros_like(z).scatter_add_(1, at, q)
    Q = q.sum(1, keepdim=True)
    d, scale = p * Q - spread, p * Q + spread
    if tail:
        rest = (1 - Q).clamp(min=0)
        mr = z.masked_fill(listed, -math.inf).amax(1, keepdim=True)
        er = torch.where(listed, 0.0, torch.exp(z - mr))
        sr = er.sum(1, keepdim=True)
        logpr = (mr - m) + torch.log(sr) - torch.log(s)
        loss = loss + (rest * (torch.log(rest) - logpr)).squeeze(1)
        size = size + (rest * (torch.log(rest).abs() + logpr.abs() + 1)).squeeze(1)
        d = p * (Q + rest) - spread - rest * er / sr
        scale = p * (Q + rest) + spread + rest * er / sr
    return loss * T * T, d * T, scale * T, size * T * T


def check_distill(x, T, tail, gen, K=3):
    R, V = x.shape
    index = torch.argsort(torch.rand((R, V), device=DEV, generator=gen), dim=1)[:, :K]
    index[:, 0] = torch.where((index == 0).any(1), index[:, 0], 0)  # entry 0 is listed in every row
    index = index.to(torch.int32)
    top = torch.randn((R, K), device=DEV, generator=gen)
    if tail:
        top = torch.log_softmax(torch.cat([top, torch.zeros((R, 1), device=DEV)], 1), 1)[:, :K].contiguous()
    xr = x.to(torch.float32) if x.dtype == torch.float64 else x
    want, d1, scale, size = distill_formula(xr, top, index, T, tail)
    x = x.detach().requires_grad_(True)
    loss = pkg.distill_loss(x, top, index, temperature=T, tail=tail, reduction="none")
    near(loss.detach(), want, EPS32 * (2 * slack_of(V) + 16 + K) * (size + T * T), "loss")
    g = torch.randn(R, device=DEV, generator=gen)
    dx, = torch.autograd.grad(loss, x, g)
    ref = d1 * g.double()[:, None]
    rel = EPS32 * (2 * slack_of(V) + 3 * (math.log2(V + 1) + 40) + 2 * K)
    near(dx, ref, half_step(x.dtype) * ref.abs() + tiny(x.dtype) + rel * scale * g.double().abs()[:, None], "dx")


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("T", [0.7, 1.0, 2.0])
@pytest.mark.parametrize("level", LEVELS)
@pytest.mark.parametrize("V", WIDTHS)
def test_distillation_of_rows_masked_with_a_finite_constant(V, level, T, tail):
    x, gen = masked_rows(V, level, torch.float32, seed=2)
    check_distill(x, T, tail, gen)


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float64])
@pytest.mark.parametrize("level", [-1e6, -1e10, -1e30])
@pytest.mark.parametrize("V", [41, 1024, 2500, 9000])
def test_distillation_of_masked_rows_of_other_types(V, level, dtype, tail):
    x, gen = masked_rows(V, level, dtype, seed=3)
    check_distill(x, 1.0, tail, gen)


@pytest.mark.parametrize("level", LEVELS)
@pytest.mark.parametrize("V", [16, 500, 2500, 9000, 20000])
def test_distillation_where_everything_unlisted_is_masked(V, level):
    """The student's mass outside the list, all of it at a finite constant: log p_r is about (level - max) / T."""
    gen = torch.Generator(device=DEV).manual_seed(V)
    x = torch.full((4, V), level, device=DEV)
    index = torch.stack([torch.randperm(V, device=DEV, generator=gen)[:3] for _ in range(4)]).to(torch.int32)
    x.scatter_(1, index.long(), torch.randn((4, 3), device=DEV, generator=gen))
    top = torch.log_softmax(torch.randn((4, 4), device=DEV, generator=gen), 1)[:, :3].contiguous()
    want, d1, scale, size = distill_formula(x, top, index, 1.0, True)
    x.requires_grad_(True)
    loss = pkg.distill_loss(x, top, index, tail=True, reduction="none")
    near(loss.detach(), want, EPS32 * (2 * slack_of(V) + 19) * (size + 1), "loss")
    dx, = torch.autograd.grad(loss.sum(), x)
    rel = EPS32 * (2 * slack_of(V) + 3 * (math.log2(V + 1) + 126) + 6)
    near(dx, d1, EPS32 * d1.abs() + 2 * tiny(torch.float32) + rel * scale, "dx")


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("T", [1e-6, 1e-5, 1e-4])
@pytest.mark.parametrize("V", [16, 1024, 2500, 9000])
def test_distillation_at_small_temperatures(V, T, tail):
    """Teacher values of about T (their own rounding is another matter), students as for the scores."""
    gen = torch.Generator(device=DEV).manual_seed(V)
    x = torch.randn((6, V), device=DEV, generator=gen) * 2
    x[1, V // 2] = 100.0
    x[2:4] = x[2:4] * T + torch.tensor([0.03, 5.0], device=DEV)[:, None]
    x[4] = 19.0
    index = torch.stack([torch.randperm(V, device=DEV, generator=gen)[:3] for _ in range(6)]).to(torch.int32)
    z = torch.randn((6, 4), device=DEV, generator=gen)
    top = (torch.log_softmax(z, 1) if tail else z * T)[:, :3].contiguous()
    want, d1, scale, size = distill_formula(x, top, index, T, tail)
    x.requires_grad_(True)
    loss = pkg.distill_loss(x, top, index, temperature=T, tail=tail, reduction="none")
    near(loss.detach(), want, EPS32 * (2 * slack_of(V) + 19) * (size + T * T), "loss")
    dx, = torch.autograd.grad(loss.sum(), x)
    rel = EPS32 * (2 * slack_of(V) + 3 * (math.log2(V + 1) + 126) + 6)
    near(dx, d1, EPS32 * d1.abs() + 2 * tiny(torch.float32) + rel * scale, "dx")


@pytest.mark.parametrize("level", [-1e9, -1e10, -1e30])
@pytest.mark.parametrize("R,V", [(40, 200), (30, 2500), (3000, 1300), (13000, 1100)])
def test_joint_scores_with_a_vocabulary_masked_by_the_bias(R, V, level):
    """Entries whose bias is a finite constant, a whole chunk of them among others: sums of products vanish beside it,
    and what is left is the rest of the vocabulary."""
    from tests.test_joint_scores_gpu import grid_problem
    h, w, b, z, gen = grid_problem(R, V, 128, torch.bfloat16, seed=V, bias="f32")
    cut = min(1024, V // 2)
    b[:cut] = level
    tok = torch.randint(cut, V, (R, 2), device=DEV, generator=gen, dtype=torch.int32)
    z[:, :cut] = -math.inf
    ref = scores_ref(z, tok, 5, 1.0)
    out = pkg.joint_token_logprobs(h, w, b, tok, top_k=5, entropy=True)
    slack = EPS32 * slack_of(V)
    assert torch.equal(out.top_index.long(), ref["top_index"])
    near(out.lse, ref["lse"], slack + EPS32 * ref["lse"].abs(), "lse")
    near(out.logprobs, ref["logprobs"], slack + EPS32 * ref["logprobs"].abs(), "logprobs")
    near(out.entropy, ref["entropy"], slack * (2 + 2 * math.log2(V + 1)) + EPS32 * ref["entropy"].abs(), "entropy")
