"""distill_loss against a plain 64-bit restatement."""
import math

import pytest
import torch

import compactwarprnntloss_amd as pkg
from tests.rowrefs import EPS32, distill_ref, half_step, softmax_slack, tiny

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = [torch.float32, torch.float16, torch.bfloat16, torch.float64]


def make(R, V, K, dtype, tail, T, seed=0, absent=0.1):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn((R, V), device=DEV, generator=gen) * 2
    x[:, 0] += (3 + math.log(V)) * (torch.rand(R, device=DEV, generator=gen) < 0.6)
    x = x.to(dtype)
    t = x.float() + torch.randn((R, V), device=DEV, generator=gen)
    top, idx = t.topk(K, dim=1)
    if tail:
        top = top / T - torch.logsumexp(t / T, 1, keepdim=True)
    idx = idx.to(torch.int32)
    idx[torch.rand((R, K), device=DEV, generator=gen) < absent] = -1
    return x, top, idx, gen


def check(x, top, idx, T, tail, gen, dtype):
    V = x.size(1)
    xr = x.detach().float() if dtype == torch.float64 else x.detach()
    want, d1, scale, scale_loss = distill_ref(xr, top, idx, T, tail)
    x = x.detach().requires_grad_(True)
    loss = pkg.distill_loss(x, top, idx, temperature=T, tail=tail, reduction="none")
    # log p to the slack of its sum, q and log q to a few roundings of numbers of their own size, K + 1 terms
    tol = EPS32 * (2 * softmax_slack(V) + 16 + idx.size(1)) * (scale_loss + T * T)
    assert float(((loss.double() - want).abs() - tol).max()) <= 0, float((loss.double() - want).abs().max())
    g = torch.randn(x.size(0), device=DEV, generator=gen)
    dx, = torch.autograd.grad(loss, x, g)
    ref = d1 * g.double()[:, None]
    rel = EPS32 * (2 * softmax_slack(V) + 2 * (math.log2(V + 1) + 40) + 2 * idx.size(1))
    tolg = half_step(dtype) * ref.abs() + tiny(dtype) + rel * scale * g.double().abs()[:, None]
    err = (dx.double() - ref).abs() - tolg
    assert dx.dtype == dtype and float(err.max()) <= 0, float(err.max())


SHAPES = [(1, 2, 1), (700, 32, 4), (17, 41, 3), (33, 64, 64), (9, 128, 2), (70, 128, 33), (6, 257, 5), (50, 512, 20),
          (4, 1000, 8), (300, 1024, 16), (2, 1025, 16), (40, 2051, 1), (2, 4233, 32), (1100, 4100, 5), (3, 50257, 64)]


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("R,V,K", SHAPES)
def test_loss_and_gradient_match_the_definition(R, V, K, dtype, tail):
    T = 2.0 if V % 2 else 1.0
    x, top, idx, gen = make(R, V, K, dtype, tail, T, seed=V)
    check(x, top, idx, T, tail, gen, dtype)


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("V", [6, 128, 1024, 3001])
def test_repeated_absent_and_complete_lists(V, tail):
    K = 6
    x, top, idx, gen = make(9, V, K, torch.float32, tail, 1.0, seed=V, absent=0.0)
    idx[0] = -1                       # an empty list
    idx[1, 1:] = -1                   # one entry
    idx[2, 3] = idx[2, 0]             # an index twice
    idx[3, :] = idx[3, 0]             # an index six times
    top[4] = -math.inf                # entries without mass
    top[5, 2] = -math.inf
    idx[6, 0] = V - 1
    idx[6, 1] = 0
    if tail:
        top[2:4] -= math.log(7.0)     # still a distribution where an index repeats
        top[6] -= math.log(3.0)
    check(x, top, idx, 1.0, tail, gen, torch.float32)
    x = x.requires_grad_(True)
    loss = pkg.distill_loss(x, top, idx, tail=tail, reduction="none")
    assert float(loss[0]) == 0
    dx, = torch.autograd.grad(loss.sum(), x)
    assert float(dx[0].abs().max()) <= (2.0 ** -22 if tail else 0)


def test_a_list_of_the_whole_vocabulary_is_the_full_divergence():
    V = 40
    gen = torch.Generator(device=DEV).manual_seed(2)
    x = (torch.randn((30, V), device=DEV, generator=gen) * 3).requires_grad_(True)
    t = torch.randn((30, V), device=DEV, generator=gen) * 3
    idx = torch.argsort(torch.rand((30, V), device=DEV, generator=gen), dim=1).to(torch.int32)
    logq = torch.log_softmax(t.double(), 1)
    want = (logq.exp() * (logq - torch.log_softmax(x.detach().double(), 1))).sum(1)
    dwant = torch.softmax(x.detach().double(), 1) - logq.exp()
    for tail in (False, True):
        val = (torch.log_softmax(t, 1) if tail else t).gather(1, idx.long())
        loss = pkg.distill_loss(x, val, idx, tail=tail, reduction="none")
        assert torch.allclose(loss.double(), want, atol=1e-5, rtol=1e-5)
        dx, = torch.autograd.grad(loss.sum(), x)
        assert float((dx.double() - dwant).abs().max()) <= EPS32 * 200


@pytest.mark.parametrize("V", [16, 1024, 6000])
def test_a_confident_student_keeps_its_tail(V):
    """The student's mass outside the list far below fp32's resolution of 1: log p_r still comes out."""
    gen = torch.Generator(device=DEV).manual_seed(V)
    x = torch.randn((8, V), device=DEV, generator=gen)
    x[:, 0] += torch.tensor([0.0, 5, 20, 40, 60, 90, 200, 1000], device=DEV)
    top = torch.full((8, 2), math.log(0.4), device=DEV)
    idx = torch.zeros((8, 2), dtype=torch.int32, device=DEV)
    idx[:, 1] = V - 1
    check(x, top, idx, 1.0, True, gen, torch.float32)


def test_masked_students():
    V = 50
    x, top, idx, gen = make(6, V, 4, torch.float32, True, 1.0, absent=0.0)
    x[0, :] = -math.inf
    keep = idx[1].long()
    x[1] = torch.where(torch.isin(torch.arange(V, device=DEV), keep), x[1], -math.inf)  # nothing outside the list
    x[2, idx[2, 0].long()] = -math.inf    # a listed entry the student cannot give
    x[3, V // 2] = math.nan
    x = x.requires_grad_(True)
    loss = pkg.distill_loss(x, top, idx, tail=True, reduction="none")
    assert float(loss[2]) == math.inf and math.isnan(float(loss[3]))
    q = top[1].double().exp()
    lp = torch.log_softmax(x.detach()[1, keep].double(), 0)
    assert abs(float(loss[1]) - float((q * (top[1].double() - lp)).sum())) <= 1e-5
    dx, = torch.autograd.grad(loss, x, torch.ones_like(loss))
    assert torch.isnan(dx[3]).all()
    assert torch.isfinite(dx[1]).all() and float(dx[1][torch.isinf(x.detach()[1])].abs().max()) == 0
    assert torch.isfinite(dx[2]).all() and torch.isfinite(dx[4:]).all()


def test_indices_outside_the_vocabulary():
    V = 50
    x, top, idx, gen = make(5, V, 4, torch.float32, False, 1.0, absent=0.0)
    good = idx.clone()
    idx[1, 2] = V
    idx[2, 0] = -2
    idx[3, 3] = 2 ** 31 - 1
    for tail in (False, True):
        xx = x.clone().requires_grad_(True)
        loss = pkg.distill_loss(xx, top, idx, tail=tail, reduction="none")
        assert torch.isnan(loss).tolist() == [False, True, True, True, False]
        dx, = torch.autograd.grad(loss, xx, torch.ones(5, device=DEV))
        assert float(dx[1:4].abs().max()) == 0 and torch.isfinite(dx).all()
        ref = pkg.distill_loss(xx, top, good, tail=tail, reduction="none")
        assert torch.equal(ref[[0, 4]], loss[[0, 4]])
    with pytest.raises(RuntimeError, match="label"):
        pkg.distill_loss(x, top, idx, validate=True)
    pkg.distill_loss(x, top, good, validate=True)


@pytest.mark.parametrize("R", [1, 500, 5000, 300001])
def test_reductions(R):
    x, top, idx, gen = make(R, 40, 3, torch.float32, True, 1.0)
    x.requires_grad_(True)
    rows = pkg.distill_loss(x, top, idx, tail=True, reduction="none")
    mean = pkg.distill_loss(x, top, idx, tail=True)
    total = pkg.distill_loss(x, top, idx, tail=True, reduction="sum")
    exact = rows.double().sum()
    assert abs(float(total) - float(exact)) <= EPS32 * abs(float(exact)) * 1.01
    assert abs(float(mean) - float(exact) / R) <= EPS32 * abs(float(exact) / R) * 1.01
    a, = torch.autograd.grad(mean * 3.0, x)
    b, = torch.autograd.grad(rows, x, torch.full((R,), 3.0 / R, device=DEV))
    assert torch.allclose(a, b, rtol=1e-6, atol=0)


def test_no_rows():
    x = torch.empty((0, 9), device=DEV, requires_grad=True)
    top, idx = torch.empty((0, 2), device=DEV), torch.empty((0, 2), dtype=torch.int32, device=DEV)
    assert pkg.distill_loss(x, top, idx, reduction="none").shape == (0,)
    s = pkg.distill_loss(x, top, idx, reduction="sum")
    assert float(s) == 0
    dx, = torch.autograd.grad(s, x)
    assert dx.shape == (0, 9)
    assert math.isnan(float(pkg.distill_loss(x, top, idx)))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V,pad,shift", [(32, 32, 0), (41, 23, 0), (1000, 24, 3), (5001, 7, 5)])
def test_strided_rows(V, pad, shift, dtype):
    x, top, idx, gen = make(19, V, 3, dtype, True, 1.0, seed=V)
    buf = torch.full((19, V + pad + shift), math.nan, device=DEV, dtype=dtype)
    buf[:, shift:shift + V] = x
    check(buf[:, shift:shift + V], top, idx, 1.0, True, gen, dtype)


def test_gradient_against_differences():
    x, top, idx, gen = make(2, 8, 2, torch.float32, True, 2.0, absent=0.0)
    x.requires_grad_(True)
    for tail in (False, True):
        f = lambda z: pkg.distill_loss(z, top, idx, temperature=2.0, tail=tail, reduction="sum")  # noqa: E731
        dx, = torch.autograd.grad(f(x), x)
        h = 2.0 ** -5
        for i in range(2):
            for v in range(8):
                e = torch.zeros_like(x)
                e[i, v] = h
                with torch.no_grad():
                    d = (f(x + e).double() - f(x - e).double()) / (2 * h)
                # third derivative of T^2 KL in x: below 1 / T; the sum's own error, 1e-6 a side
                assert abs(float(d) - float(dx[i, v])) <= h * h + 4e-6 / h


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("V", [40, 1024, 5000])
def test_rows_masked_with_the_lowest_value(V, dtype):
    """Entries at the type's lowest value are masked entries; a row of nothing else is uniform."""
    x, top, idx, gen = make(6, V, 3, dtype, False, 1.0, absent=0.0, seed=V)
    low = torch.finfo(dtype).min
    keep = torch.zeros((6, V), dtype=torch.bool, device=DEV).scatter_(1, idx.long(), True)
    x[1:4] = torch.where(keep[1:4], x[1:4], low)
    check(x[:4], top[:4], idx[:4], 1.0, False, gen, dtype)
    x[4] = low
    x.requires_grad_(True)
    loss = pkg.distill_loss(x, top, idx, reduction="none")
    q = torch.softmax(top[4].double(), 0)
    want = float((q * (q.log() + math.log(V))).sum())
    assert abs(float(loss[4]) - want) <= EPS32 * 100 * (1 + want)
    dx, = torch.autograd.grad(loss[4], x)
    ref = torch.full((V,), 1.0 / V, dtype=torch.float64, device=DEV).scatter_add_(0, idx[4].long(), -q)
    assert float((dx[4].double() - ref).abs().max()) <= half_step(dtype) + EPS32 * 100
    tailed = pkg.distill_loss(x, top - 20.0, idx, tail=True, reduction="none")
    dt, = torch.autograd.grad(tailed.sum(), x)
    assert torch.isfinite(dt[4]).all() and torch.isfinite(tailed[4])


def test_a_list_longer_than_the_vocabulary():
    x, top, idx, gen = make(50, 5, 5, torch.float32, True, 1.0, absent=0.0)
    long_top = torch.cat([top, top], 1) - math.log(2.0)
    long_idx = torch.cat([idx, idx], 1)
    check(x, long_top, long_idx, 1.0, True, gen, torch.float32)
    check(x, long_top, long_idx, 1.0, False, gen, torch.float32)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V,K", [(100003, 4), (70001, 1)])
def test_a_student_that_agrees_with_its_teacher(V, K, dtype):
    """The loss is far below the logarithms it is a difference of."""
    gen = torch.Generator(device=DEV).manual_seed(V)
    x = (torch.randn((64, V), device=DEV, generator=gen) * 0.25).to(dtype)
    t = x.double() + 0.02 * torch.randn((64, V), device=DEV, generator=gen).double()
    T = 2.0
    top, idx = torch.log_softmax(t / T, 1).topk(K, dim=1)
    top, idx = top.float(), idx.to(torch.int32)
    loss = pkg.distill_loss(x, top, idx, temperature=T, tail=True, reduction="none")
    want = distill_ref(x, top, idx, T, True)[0]
    # The listed mass is below 1e-3 and the row's sum enters by p_r - q_r only, so what is left are, for q_r near
    # 1: two logarithms of a mantissa in [1, 2) (1e-7 or 2 half steps each, log 2 of it after the change of base),
    # the move of the rest's sum to the maximum of all (2^d to 2, its product and the addition of the list 1
    # each), q_r as a number of 32 bits 1, and the sum of the terms 1: below 9 half steps, times T^2.
    assert float((loss.double() - want).abs().max()) <= 9 * EPS32 * T * T
    # (one fp32 number for a logarithm near 17 would be off by 16 half steps alone)


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("V", [32, 1024, 6000])
def test_a_student_with_nothing(V, tail):
    x, top, idx, _ = make(3, V, 2, torch.float32, tail, 1.0, absent=0.0)
    x[1] = -math.inf
    want = torch.zeros(V, device=DEV).double()
    want[idx[1].long()] = -(top[1].double().exp() if tail else torch.softmax(top[1].double(), 0))
    x.requires_grad_(True)
    loss = pkg.distill_loss(x, top, idx, tail=tail, reduction="none")
    assert float(loss[1]) == math.inf and torch.isfinite(loss[0]) and torch.isfinite(loss[2])
    dx, = torch.autograd.grad(loss, x, torch.ones_like(loss))
    # p = 0 everywhere leaves -q; q to its exponential, its sum and their quotient
    assert float((dx[1].double() - want).abs().max()) <= 16 * EPS32
