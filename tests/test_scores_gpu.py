"""token_logprobs against a plain 64-bit restatement: scores, ranking, gradients, masked rows, strides."""
import math

import pytest
import torch

import compactwarprnntloss_amd as pkg
from tests.rowrefs import EPS32, half_step, scores_grad_ref, scores_ref, softmax_slack, tiny, top_ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = [torch.float32, torch.float16, torch.bfloat16, torch.float64]


def make(R, V, dtype, seed=0, pad=0, spread=2.0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn((R, V + pad), device=DEV, generator=gen) * spread
    x[:, 0] += (3 + math.log(V)) * (torch.rand(R, device=DEV, generator=gen) < 0.6)
    return x.to(dtype)[:, :V], gen


def make_tokens(R, V, M, gen):
    t = torch.randint(0, V, (R, M), device=DEV, dtype=torch.int32, generator=gen)
    t[torch.rand((R, M), device=DEV, generator=gen) < 0.2] = -1
    return t


def check_scores(out, ref, V, K):
    slack = EPS32 * softmax_slack(V)

    def near(got, want, tol):
        want_f = torch.isfinite(want)
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(got[~want_f & ~torch.isnan(want)].double(), want[~want_f & ~torch.isnan(want)])
        err = (got.double() - want)[want_f].abs() - tol[want_f]
        assert err.numel() == 0 or float(err.max()) <= 0, float(err.max())

    near(out.lse, ref["lse"], slack + EPS32 * ref["lse"].abs())
    if out.logprobs is not None:
        want = ref["logprobs"].view(out.logprobs.shape)
        near(out.logprobs, want, slack + EPS32 * want.abs())
    if out.entropy is not None:
        # log2 S and U / S, the latter a mean of exponents of up to 2 log2 V: each as exact as the sum of V terms
        near(out.entropy, ref["entropy"], slack * (2 + 2 * math.log2(V + 1)) + EPS32 * ref["entropy"].abs())
    if K:
        assert out.top_index.dtype == torch.int32
        assert torch.equal(out.top_index.long(), ref["top_index"])
        near(out.top_logprobs, ref["top_logprobs"], slack + EPS32 * ref["top_logprobs"].abs())
    else:
        assert out.top_index is None and out.top_logprobs is None


SHAPES = [(1, 1, 1), (3, 2, 2), (5, 7, 3), (700, 32, 4), (17, 41, 3), (33, 64, 64), (9, 128, 8), (70, 128, 33), (6, 257, 5),
          (50, 500, 7), (50, 512, 20), (4, 1000, 8), (300, 1024, 4), (3, 1024, 64), (2, 1025, 16), (40, 2051, 1),
          (2, 4233, 8), (3, 8192, 64), (1100, 4100, 5), (1, 50257, 32), (5, 50257, 64)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("R,V,K", SHAPES)
def test_scores_match_the_definition(R, V, K, dtype):
    M = 1 + (R + V) % 5
    x, gen = make(R, V, dtype, seed=V)
    tok = make_tokens(R, V, M, gen)
    for T in (1.0, 0.7):
        xr = x.to(torch.float32) if dtype == torch.float64 else x  # 64-bit entries are rounded when read
        out = pkg.token_logprobs(x, tok, top_k=K, entropy=True, temperature=T)
        check_scores(out, scores_ref(xr, tok, K, T), V, K)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("R,V,K", SHAPES)
def test_gradients_match_the_formula(R, V, K, dtype):
    M = 1 + (R + V) % 5
    x, gen = make(R, V, dtype, seed=V + 1)
    tok = make_tokens(R, V, M, gen)
    T = 0.7 if V % 2 else 1.0
    x = x.detach().requires_grad_(True)
    out = pkg.token_logprobs(x, tok, top_k=K, entropy=True, temperature=T)
    g = [torch.randn(t.shape, device=DEV, generator=gen) for t in (out.logprobs, out.entropy, out.lse, out.top_logprobs)]
    dx, = torch.autograd.grad([out.logprobs, out.entropy, out.lse, out.top_logprobs], x, g)
    xr = x.detach().to(torch.float32) if dtype == torch.float64 else x.detach()
    want, scale = scores_grad_ref(xr, tok, K, T, *g)
    # p to the slack of its sum plus two roundings of its own exponent (|t| <= log2 V + 40 where p matters);
    # sums of up to M + K gradients; one rounding to the type
    rel = EPS32 * (2 * softmax_slack(V) + 2 * (math.log2(V + 1) + 40) + M + K)
    tol = half_step(dtype) * want.abs() + tiny(dtype) + rel * scale
    err = (dx.double() - want).abs() - tol
    assert dx.dtype == dtype and float(err.max()) <= 0, float(err.max())


@pytest.mark.parametrize("which", ["logprobs", "entropy", "lse", "top_logprobs"])
def test_each_output_has_its_own_gradient(which):
    x, gen = make(13, 77, torch.float32, seed=3)
    tok = make_tokens(13, 77, 2, gen)
    x.requires_grad_(True)
    out = pkg.token_logprobs(x, tok, top_k=3, entropy=True)
    g = torch.randn(getattr(out, which).shape, device=DEV, generator=gen)
    dx, = torch.autograd.grad(getattr(out, which), x, g)
    key = {"logprobs": "g_logprobs", "entropy": "g_entropy", "lse": "g_lse", "top_logprobs": "g_top"}[which]
    want, scale = scores_grad_ref(x.detach(), tok, 3, 1.0, **{key: g})
    assert float(((dx.double() - want).abs() - EPS32 * (want.abs() + 150 * scale)).max()) <= 0


def test_gradient_against_differences():
    """Central differences of the fp32 forward pass: step h = 2^-6 leaves h^2/6 times the third derivative
    (at most about 1 here) and the outputs' own error 4e-6 / h."""
    x, gen = make(2, 9, torch.float32, seed=5, spread=1.0)
    tok = torch.tensor([[0, 3], [8, -1]], device=DEV, dtype=torch.int32)
    g1, g2, g3 = (torch.randn(s, device=DEV, generator=gen) for s in ((2, 2), (2,), (2, 2)))
    x.requires_grad_(True)

    def total(z):
        o = pkg.token_logprobs(z, tok, top_k=2, entropy=True)
        return (o.logprobs.double() * g1).sum() + (o.entropy.double() * g2).sum() + (o.top_logprobs.double() * g3).sum()
    dx, = torch.autograd.grad(total(x), x)
    h = 2.0 ** -6
    for i in range(2):
        for v in range(9):
            e = torch.zeros_like(x)
            e[i, v] = h
            with torch.no_grad():
                d = (total(x + e) - total(x - e)) / (2 * h)
            bound = (g1.abs().sum() + g2.abs().sum() + g3.abs().sum()).item() * (4 * h * h + 4e-6 / h)
            assert abs(float(d) - float(dx[i, v])) <= bound


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [8, 41, 128, 500, 1024, 1031, 5000, 40000])
def test_ties_and_orders(V, dtype):
    """Equal values rank by index, whatever the order the row comes in."""
    gen = torch.Generator(device=DEV).manual_seed(V)
    ramp = torch.arange(V, device=DEV, dtype=torch.float32)
    rows = [torch.zeros(V, device=DEV), ramp, -ramp, ramp % 3, (V - ramp) % 7,
            torch.where(ramp % 2 == 0, 0.0, -0.0), torch.full((V,), -1e4, device=DEV),
            torch.randint(0, 3, (V,), device=DEV, generator=gen).float(),
            torch.where(ramp == V - 1, 1.0, 0.0), torch.where(ramp == 0, -1.0, 0.0)]
    x = torch.stack(rows).to(dtype)
    for K in sorted({1, 2, min(V, 8), min(V, 64)}):
        out = pkg.token_logprobs(x, top_k=K)
        assert torch.equal(out.top_index.long(), top_ref(x, K)), K


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [3, 41, 256, 1024, 1500, 5001])
def test_masked_infinite_and_nan_rows(V, dtype):
    x, gen = make(12, V, dtype, seed=V)
    x = x.clone()
    low = torch.finfo(dtype).min if dtype != torch.float64 else torch.finfo(torch.float32).min
    x[0] = -math.inf
    x[1, 1:] = -math.inf
    x[2, :-1] = -math.inf
    x[3] = low
    x[4, 1:] = low
    x[5, V // 2] = math.nan
    x[6] = math.nan
    x[7, V - 1] = math.inf
    x[8, 0] = math.inf
    x[8, V - 1] = math.nan
    x[9, ::2] = -math.inf
    x[10, :] = 0
    x[10, V // 3] = 300.0   # one entry takes everything
    tok = torch.zeros((12, 3), dtype=torch.int32, device=DEV)
    tok[:, 1] = V - 1
    tok[:, 2] = V // 2
    K = min(V, 6)
    xr = x.to(torch.float32) if dtype == torch.float64 else x
    x = x.requires_grad_(True)
    out = pkg.token_logprobs(x, tok, top_k=K, entropy=True)
    ref = scores_ref(xr, tok, K, 1.0)
    bad = torch.tensor([5, 6, 7, 8], device=DEV)
    for t in (out.logprobs, out.entropy, out.lse, out.top_logprobs):
        assert torch.isnan(t[bad]).all()
    fine = torch.tensor([0, 1, 2, 3, 4, 9, 10, 11], device=DEV)
    cut = type(out)(*[t[fine] for t in out])
    check_scores(cut, {k: v[fine] for k, v in ref.items()}, V, K)
    assert torch.equal(out.top_index.long(), top_ref(xr, K))
    assert float(out.entropy[0]) == 0 and float(out.lse[0]) == -math.inf
    g = torch.ones_like(out.entropy)
    dx, = torch.autograd.grad([out.logprobs, out.entropy], x, [torch.ones_like(out.logprobs), g])
    assert torch.isnan(dx[bad]).all()
    want, scale = scores_grad_ref(xr[fine], tok[fine], K, 1.0, torch.ones_like(out.logprobs)[fine], g[fine])
    # rows 1, 2, 9: entries of -inf have gradient 0 except where a token names them
    err = (dx[fine].double() - want).abs() - (half_step(dtype) * want.abs() + tiny(dtype) + EPS32 * 200 * (1 + scale))
    ok = torch.isfinite(want)
    assert float(err[ok].max()) <= 0
    assert (dx[0] == 0).all() == bool((want[0] == 0).all())


def test_tokens_outside_the_vocabulary_and_flags():
    x, _ = make(4, 40, torch.float32)
    tok = torch.tensor([[0, -1], [40, 1], [-2, 2], [39, 2 ** 31 - 1]], dtype=torch.int32, device=DEV)
    x.requires_grad_(True)
    out = pkg.token_logprobs(x, tok)
    nan = torch.isnan(out.logprobs)
    assert nan.tolist() == [[False, False], [True, False], [True, False], [False, True]]
    assert float(out.logprobs[0, 1]) == 0
    g = torch.ones_like(out.logprobs)
    dx, = torch.autograd.grad(out.logprobs, x, g)
    want, scale = scores_grad_ref(x.detach(), tok, 0, 1.0, g)
    assert float(((dx.double() - want).abs() - EPS32 * 200 * scale).max()) <= 0
    with pytest.raises(RuntimeError, match="label"):
        pkg.token_logprobs(x.detach(), tok, validate=True)
    pkg.token_logprobs(x.detach(), tok[:1].expand(4, 2).contiguous(), validate=True)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.float64])
@pytest.mark.parametrize("V,pad,shift", [(32, 32, 0), (41, 23, 0), (128, 1, 0), (1000, 24, 3), (1024, 8, 1), (5001, 7, 5)])
def test_strided_and_shifted_rows(V, pad, shift, dtype):
    """Rows any distance apart, starting anywhere; nothing outside a row is looked at (NaN lies there)."""
    R = 19
    gen = torch.Generator(device=DEV).manual_seed(V)
    buf = torch.full((R, V + pad + shift), math.nan, device=DEV, dtype=dtype)
    x = buf[:, shift:shift + V]
    x.copy_(torch.randn((R, V), device=DEV, generator=gen) * 2)
    x = x.detach().requires_grad_(True)
    tok = make_tokens(R, V, 2, gen)
    out = pkg.token_logprobs(x, tok, top_k=5, entropy=True)
    dense = x.detach().clone().requires_grad_(True)
    want = pkg.token_logprobs(dense, tok, top_k=5, entropy=True)
    xr = x.detach().float() if dtype == torch.float64 else x.detach()
    check_scores(out, scores_ref(xr, tok, 5, 1.0), V, 5)
    g = torch.randn(R, device=DEV, generator=gen)
    a, = torch.autograd.grad(out.entropy, x, g)
    b, = torch.autograd.grad(want.entropy, dense, g)
    assert a.is_contiguous() and torch.isfinite(a).all()
    assert float((a.double() - b.double()).abs().max()) <= 2 * half_step(dtype) * float(b.abs().max()) + 4e-6
    same = x.detach()[:1].expand(7, V)   # one row seen seven times
    o = pkg.token_logprobs(same, top_k=3)
    assert torch.equal(o.top_index, o.top_index[:1].expand(7, 3))


def test_no_rows_and_one_dimensional_tokens():
    x = torch.empty((0, 50), device=DEV, requires_grad=True)
    out = pkg.token_logprobs(x, torch.empty((0, 2), dtype=torch.int32, device=DEV), top_k=4, entropy=True)
    assert out.logprobs.shape == (0, 2) and out.top_index.shape == (0, 4) and out.entropy.shape == (0,)
    dx, = torch.autograd.grad(out.logprobs.sum(), x)
    assert dx.shape == (0, 50)
    x, gen = make(6, 50, torch.float32)
    tok = make_tokens(6, 50, 1, gen)
    a, b = pkg.token_logprobs(x, tok), pkg.token_logprobs(x, tok.view(6))
    assert b.logprobs.shape == (6,) and torch.equal(a.logprobs.view(6), b.logprobs)


def test_results_do_not_depend_on_the_number_of_waves_in_flight():
    """The same rows among few and among many: different kernels, the same ranking, scores within rounding;
    and twice the same call gives the same bits."""
    V = 20000
    x, gen = make(17000, V, torch.bfloat16, seed=9)
    tok = make_tokens(17000, V, 2, gen)
    many = pkg.token_logprobs(x, tok, top_k=9, entropy=True)
    again = pkg.token_logprobs(x, tok, top_k=9, entropy=True)
    for a, b in zip(many, again):
        assert torch.equal(a, b)
    for n in (3, 2000):
        few = pkg.token_logprobs(x[:n], tok[:n], top_k=9, entropy=True)
        assert torch.equal(few.top_index, many.top_index[:n])
        tol = EPS32 * softmax_slack(V) * 2
        assert float((few.lse - many.lse[:n]).abs().max()) <= tol + EPS32 * 2 * float(few.lse.abs().max())


def test_lattice_tokens_name_what_the_loss_walks_on():
    """Blank and label log-probabilities of every cell, fed back as log-probabilities: the loss of a lattice
    rebuilt from the pair equals the loss of the logits."""
    lx = torch.tensor([5, 1, 7], dtype=torch.int32, device=DEV)
    ly = torch.tensor([3, 0, 2], dtype=torch.int32, device=DEV)
    y = torch.tensor([[3, 4, 5], [1, 1, 1], [2, 2, 9]], dtype=torch.int32, device=DEV)
    R, V = 5 * 4 + 1 + 7 * 3, 12
    x, _ = make(R, V, torch.float32)
    tok = pkg.lattice_tokens(lx, y, ly, R, V)
    want = []
    for n in range(3):
        for _t in range(int(lx[n])):
            for u in range(int(ly[n]) + 1):
                want.append([0, int(y[n, u]) if u < int(ly[n]) else -1])
    assert tok.tolist() == want
    out = pkg.token_logprobs(x, tok, validate=True)
    sparse = torch.full((R, V), -50.0, device=DEV)
    sparse[:, 0] = out.logprobs[:, 0]
    rows = torch.arange(R, device=DEV)
    has = tok[:, 1] >= 0
    sparse[rows[has], tok[has, 1].long()] = out.logprobs[has, 1]
    a = pkg.transducer_loss(sparse, lx, y, ly, 0, "none")
    b = pkg.transducer_loss(x, lx, y, ly, 0, "none", fused_log_softmax=True)
    assert torch.allclose(a, b, rtol=1e-5, atol=1e-5)
