"""distill_loss: the teacher's lists at the ends of what is allowed."""
import math

import pytest
import torch

import compactwarprnntloss_amd as pkg
from tests.rowrefs import EPS32, softmax_slack, tiny
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
