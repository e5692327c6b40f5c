"""distill_loss: the teacher's lists at the ends of what is allowed."""
import math

import pytest
import torch

import compactwarprnntloss_amd as pkg
from tests.rowrefs import EPS32, half_step, softmax_slack, tiny
from tests.test_row_range_gpu import distill_formula, near

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("T", [1e-6, 1e-5, 1e-3, 0.7, 3.0])
@pytest.mark.parametrize("base", [10.0, -300.0, 2.0e4, -1.0e9])
@pytest.mark.parametrize("V,K", [(40, 3), (600, 20), (5000, 33)])
def test_shares_of_a_teacher_far_from_zero(V, K, base, T):
    """Shares come from differences of the teacher's values, however large value / T is."""
    gen = torch.Generator(device=DEV).manual_seed(V)
    x = torch.randn((7, V), device=DEV, generator=gen) * T
    index = torch.stack([torch.randperm(V, device=DEV, generator=gen)[:K] for _ in range(7)]).to(torch.int32)
    top = base + torch.randn((7, K), device=DEV, generator=gen) * T
    want, d1, scale, size = distill_formula(x, top, index, T, False)
    x.requires_grad_(True)
    loss = pkg.distill_loss(x, top, index, temperature=T, reduction="none")
    # x / T is of ordinary size, so that the bounds are those of ordinary logits: three roundings of an exponent, q
    # and log q to 16 roundings of numbers of their own size, K terms
    slack = softmax_slack(V) + math.log2(V + 1)
    near(loss.detach(), want, EPS32 * (2 * slack + 16 + K) * (size + T * T), "loss")
    dx, = torch.autograd.grad(loss.sum(), x)
    rel = EPS32 * (2 * slack + 3 * (math.log2(V + 1) + 126) + 2 * K)
    near(dx, d1, EPS32 * d1.abs() + 2 * tiny(torch.float32) + rel * scale, "dx")


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("V", [16, 41, 1024, 2500, 9000, 20000])
def test_rows_without_a_list_do_not_count_whatever_is_in_them(V, tail):
    """An empty list marks a row that is not to be learned from: loss 0 and gradient 0 exactly, also where the row holds
    NaN, infinities or nothing, and the other rows' results stay what they are."""
    gen = torch.Generator(device=DEV).manual_seed(V)
    x = torch.randn((8, V), device=DEV, generator=gen)
    top = torch.randn((8, 5), device=DEV, generator=gen).log_softmax(1) - 0.1
    index = torch.stack([torch.randperm(V, device=DEV, generator=gen)[:5] for _ in range(8)]).to(torch.int32)
    want_x = x.clone().requires_grad_(True)
    want = pkg.distill_loss(want_x, top, index, tail=tail, reduction="none")
    d_want, = torch.autograd.grad(want.sum(), want_x)
    empty = torch.tensor([0, 1, 2, 3, 5, 6], device=DEV)
    index[empty] = -1
    x[1, V // 2] = math.nan
    x[2] = math.nan
    x[3, 0] = math.inf
    x[5] = -math.inf
    top[6] = math.nan  # what stands beside absent entries
    kept = torch.tensor([4, 7], device=DEV)
    x.requires_grad_(True)
    rows = pkg.distill_loss(x, top, index, tail=tail, reduction="none")
    assert (rows[empty] == 0).all() and torch.equal(rows[kept], want[kept])
    d, = torch.autograd.grad(rows.sum(), x)
    assert (d[empty] == 0).all() and torch.equal(d[kept], d_want[kept])
    for reduction, part in (("sum", 1), ("mean", 8)):
        loss = pkg.distill_loss(x, top, index, tail=tail, reduction=reduction)
        exact = float(want.detach()[kept].double().sum()) / part
        assert abs(float(loss.detach()) - exact) <= 2 * EPS32 * abs(exact)
        d, = torch.autograd.grad(loss, x)
        assert (d[empty] == 0).all() and torch.isfinite(d).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float64])
@pytest.mark.parametrize("T", [1e-6, 1e-3, 0.7, 1.0, 1.3])
@pytest.mark.parametrize("V", [16, 1024, 5000])
def test_listed_entries_masked_with_the_lowest_value(V, T, dtype):
    """q T^2 (log q - log p) of such an entry fits into fp32 although log p or T^2 log p does not: the loss is finite, with
    and without a tail, and where nothing but the lowest value is outside the list."""
    gen = torch.Generator(device=DEV).manual_seed(V)
    low = torch.finfo(torch.float32 if dtype == torch.float64 else dtype).min
    x = torch.randn((6, V), device=DEV, generator=gen).to(dtype)
    index = torch.stack([torch.randperm(V, device=DEV, generator=gen)[:3] for _ in range(6)]).to(torch.int32)
    x[torch.arange(3, device=DEV), index[:3, 1].long()] = low
    keep = torch.zeros((6, V), dtype=torch.bool, device=DEV).scatter_(1, index.long(), True)
    x[3:5] = torch.where(keep[3:5], x[3:5], low)
    z = torch.randn((6, 4), device=DEV, generator=gen)
    z[:, 1] -= 3.0  # the masked entry's share: a tenth at most in most rows
    slack = softmax_slack(V) + math.log2(V + 1)
    for tail in (False, True):
        top = (torch.log_softmax(z, 1) if tail else z * T)[:, :3].contiguous()
        want, d1, scale, size = distill_formula(x.float() if dtype == torch.float64 else x, top, index, T, tail)
        fits = torch.isfinite(want.float())
        assert int(fits.sum()) >= 5
        xg = x.clone().requires_grad_(True)
        loss = pkg.distill_loss(xg, top, index, temperature=T, tail=tail, reduction="none")
        near(loss.detach()[fits], want[fits], EPS32 * (2 * slack + 19) * (size + T * T)[fits], "loss")
        dx, = torch.autograd.grad(loss.sum(), xg)
        rel = EPS32 * (2 * slack + 3 * (math.log2(V + 1) + 126) + 6)
        near(dx, d1, half_step(dtype) * d1.abs() + 2 * tiny(dtype) + rel * scale, "dx")
