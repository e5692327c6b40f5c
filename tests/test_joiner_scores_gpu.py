"""CompactJoiner.lattice_scores / step_scores as programs hold their joiners: mixed precision, tied weights, a
search scored step by step against the lattice."""
import pytest
import torch

import compactwarprnntloss_amd as pkg
from tests.rowrefs import EPS32, scores_ref, softmax_slack

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def setup(dtype, activation="tanh", H=96, V=61):
    torch.manual_seed(0)
    j = pkg.CompactJoiner(48, 40, H, V, activation=activation).to(DEV, dtype)
    lx = torch.tensor([9, 4, 1], dtype=torch.int32, device=DEV)
    ly = torch.tensor([3, 0, 5], dtype=torch.int32, device=DEV)
    y = torch.randint(1, V, (3, 5), dtype=torch.int32, device=DEV)
    e, p = torch.randn((3, 9, 48), device=DEV, dtype=dtype), torch.randn((3, 6, 40), device=DEV, dtype=dtype)
    return j, lx, ly, y, e, p


@pytest.mark.parametrize("half", [torch.bfloat16, torch.float16])
def test_scores_under_autocast(half):
    """fp32 parameters, 16-bit activations: the scores are those of the logits forward() gives there."""
    j, lx, ly, y, e, p = setup(torch.float32)
    with torch.autocast("cuda", dtype=half), torch.no_grad():
        logits = j(e, p, lx, ly)
        assert logits.dtype == half
        s = j.lattice_scores(e, p, lx, y, ly, top_k=4, entropy=True)
        one = j.step_scores(e[:, 0], p[:, 0], top_k=3)
    tok = pkg.lattice_tokens(lx, y, ly, logits.size(0), 61)
    ref = scores_ref(logits, tok, 4, 1.0)
    tol = EPS32 * (softmax_slack(61) + float(ref["logp"].abs().max()))
    assert float((s.logprobs.double() - ref["logprobs"]).abs().max()) <= tol
    assert torch.equal(s.top_index.long(), ref["top_index"])
    assert one.top_logprobs.shape == (3, 3) and torch.isfinite(one.top_logprobs).all()


def test_scores_of_a_weight_that_is_a_transposed_view():
    """An output layer tied to an embedding stored the other way round, as loss() takes it."""
    j, lx, ly, y, e, p = setup(torch.bfloat16)
    want = j.lattice_scores(e, p, lx, y, ly, top_k=4)
    step = j.step_scores(e[:, 0], p[:, 0], top_k=3)
    j.out.weight = torch.nn.Parameter(j.out.weight.detach().t().contiguous().t())
    assert not j.out.weight.is_contiguous()
    got = j.lattice_scores(e, p, lx, y, ly, top_k=4)
    assert torch.equal(got.logprobs, want.logprobs) and torch.equal(got.top_index, want.top_index)
    assert torch.equal(j.step_scores(e[:, 0], p[:, 0], top_k=3).top_logprobs, step.top_logprobs)
    assert torch.isfinite(j.loss(e, p, lx, y, ly))
