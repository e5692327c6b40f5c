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


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16, torch.float64])
@pytest.mark.parametrize("activation", ["tanh", "relu", None])
@pytest.mark.parametrize("R,H", [(1, 1), (3, 96), (700, 640), (257, 45), (0, 32)])
def test_rows_of_a_step_are_rows_of_the_lattice(R, H, activation, dtype):
    from compactwarprnntloss_amd.joiner import _join_rows
    gen = torch.Generator(device=DEV).manual_seed(R + H)
    f, g = ((torch.randn((R, H), device=DEV, generator=gen) * 2).to(dtype) for _ in range(2))
    got = _join_rows(f, g, activation)
    if R:
        one, none = torch.ones(R, dtype=torch.int32, device=DEV), torch.zeros(R, dtype=torch.int32, device=DEV)
        assert torch.equal(got, pkg.compact_join(f[:, None], g[:, None], one, none, activation, R))
    assert got.shape == (R, H) and got.dtype == dtype
    if R > 1:  # one frame and several hypotheses; operands off the 16-byte grid
        assert torch.equal(_join_rows(f[:1], g, activation), _join_rows(f[:1].expand(R, H).contiguous(), g, activation))
        flat = torch.zeros(R * H + 1, dtype=dtype, device=DEV)
        flat[1:] = f.reshape(-1)
        assert torch.equal(_join_rows(flat[1:].view(R, H), g, activation), got)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("activation", ["tanh", "relu", None])
def test_a_search_step_scores_what_the_lattice_scores(dtype, activation):
    """Projections on a grid where library products of any shape are exact: every cell scored on its own has the
    scores it has in the lattice."""
    j, lx, ly, y, e, p = setup(dtype, activation)
    with torch.no_grad():
        for w in (j.enc.weight, j.enc.bias, j.pred.weight):
            w.copy_((w * 64).round() / 64)
        e, p = (e * 4).round() / 4, (p * 4).round() / 4
    s = j.lattice_scores(e, p, lx, y, ly, top_k=4, entropy=True)
    tok = pkg.lattice_tokens(lx, y, ly, s.lse.numel(), 61)
    cells = [(n, t, u) for n in range(3) for t in range(int(lx[n])) for u in range(int(ly[n]) + 1)]
    frames = torch.stack([e[n, t] for n, t, _ in cells])
    states = torch.stack([p[n, u] for n, _, u in cells])
    one = j.step_scores(frames, states, tokens=tok, top_k=4, entropy=True)
    for a, b in zip(one, s):
        assert torch.equal(a, b)
