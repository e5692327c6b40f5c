"""joint_token_logprobs: scores straight from the joint rows, against a 64-bit product."""
import math

import pytest
import torch

import compactwarprnntloss_amd as pkg
from tests.rowrefs import EPS32, scores_ref, softmax_slack
from tests.test_scores_gpu import check_scores, make_tokens

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def grid_problem(R, V, H, dtype, seed=0, bias="same"):
    """h in multiples of 2^-7, weight and bias of 2^-9: every sum of products is a multiple of 2^-16 below
    2^8, exact in fp32 in any order, so that the ranking is a fact of the inputs."""
    gen = torch.Generator(device=DEV).manual_seed(seed)
    h = (torch.tanh(torch.randn((R, H), device=DEV, generator=gen)) * 128).round().div(128).to(dtype)
    w = (torch.randn((V, H), device=DEV, generator=gen) * (2 / (0.63 * math.sqrt(H))) * 512).round()
    w = w.clamp(-255, 255).div(512).to(dtype)
    b = (torch.randn(V, device=DEV, generator=gen) * 512).round().clamp(-255, 255).div(512)
    b = {"same": b.to(dtype), "f32": b, None: None}[bias]
    z = h.double() @ w.double().T
    if b is not None:
        z = z + b.double()
    assert float(z.abs().max()) < 128
    return h, w, b, z, gen


SHAPES = [(1, 32, 32, 1), (1, 1024, 512, 4), (5, 41, 64, 3), (8, 1000, 640, 8), (32, 33, 96, 33), (33, 1027, 128, 16),
          (64, 50, 1024, 8), (65, 4096, 640, 8), (512, 1024, 320, 4), (1000, 130, 160, 5), (1025, 257, 128, 4),
          (1100, 5000, 512, 8), (2000, 1024, 1024, 4), (3000, 129, 704, 2), (1500, 300, 1056, 3), (5000, 41, 256, 8),
          # large products: the walks with resident rows (their three kinds of shapes) and with streamed rows
          (3300, 4100, 512, 4), (12500, 1001, 704, 4), (12300, 1024, 1024, 2), (12101, 1003, 640, 8), (48001, 257, 192, 3),
          (13000, 1000, 96, 3), (12100, 1027, 1056, 4)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("R,V,H,K", SHAPES)
def test_scores_match_the_product(R, V, H, K, dtype):
    h, w, b, z, gen = grid_problem(R, V, H, dtype, seed=R + V, bias=["same", "f32", None][(R + H // 32) % 3])
    tok = make_tokens(R, V, 2, gen)
    for T in (1.0, 2.0):
        out = pkg.joint_token_logprobs(h, w, b, tok, top_k=K, entropy=True, temperature=T)
        check_scores(out, scores_ref(z, tok, K, T), V, K)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_ordinary_values_within_the_rounding_of_the_product(dtype):
    """fp32 accumulation of H products: an error of at most H 2^-24 sum |h w| in every logit (2^-23 where the
    matrix units round towards zero), the same in the log-probabilities twice over."""
    gen = torch.Generator(device=DEV).manual_seed(1)
    for R, V, H in ((7, 900, 512), (700, 1024, 640), (3000, 1000, 512)):
        h = torch.tanh(torch.randn((R, H), device=DEV, generator=gen)).to(dtype)
        w = (torch.randn((V, H), device=DEV, generator=gen) * 0.1).to(dtype)
        b = torch.randn(V, device=DEV, generator=gen).to(dtype)
        tok = make_tokens(R, V, 3, gen)
        out = pkg.joint_token_logprobs(h, w, b, tok, entropy=True)
        ref = scores_ref(h.double() @ w.double().T + b.double(), tok, 0, 1.0)
        slip = 2 * EPS32 * H * float((h.double().abs() @ w.double().abs().T).max())
        tol = 2 * slip + EPS32 * (softmax_slack(V) + ref["logprobs"].abs())
        assert float(((out.logprobs.double() - ref["logprobs"]).abs() - tol).max()) <= 0


def test_blocks_of_rows_give_the_same_scores():
    """More rows than a block of the workspace holds, and a workspace of a few rows only."""
    from compactwarprnntloss_amd import _lib
    R, V, H, K = 70000, 600, 128, 4
    h, w, b, z, gen = grid_problem(R, V, H, torch.bfloat16, seed=3)
    tok = make_tokens(R, V, 2, gen)
    out = pkg.joint_token_logprobs(h, w, b, tok, top_k=K, entropy=True)
    check_scores(out, scores_ref(z, tok, K, 1.0), V, K)
    assert _lib.load().cwr_joint_token_logprobs_workspace_bytes(R, V) < R * V * 4
    n = 700
    small = torch.empty(100 * 600 * 4, dtype=torch.uint8, device=DEV)
    lp, lse = torch.empty((n, 2), device=DEV), torch.empty(n, device=DEV)
    top, idx = torch.empty((n, K), device=DEV), torch.empty((n, K), dtype=torch.int32, device=DEV)
    rc = _lib.load().cwr_joint_token_logprobs(h.data_ptr(), w.data_ptr(), b.data_ptr(), _lib.BF16, _lib.BF16, n, H, V,
                                              tok.data_ptr(), 2, K, 1.0, lp.data_ptr(), None, lse.data_ptr(),
                                              top.data_ptr(), idx.data_ptr(), small.data_ptr(), small.numel(), None,
                                              torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    assert torch.equal(idx, out.top_index[:n])
    tol = 2 * EPS32 * softmax_slack(V)
    assert float((lp - out.logprobs[:n]).abs().max()) <= tol + 2 * EPS32 * float(lp.abs().max())


def test_masked_vocabulary_and_bad_tokens():
    h, w, b, z, gen = grid_problem(40, 200, 64, torch.bfloat16, bias="f32")
    b[::3] = -math.inf
    z[:, ::3] = -math.inf
    tok = torch.tensor([0, 1, -1, 199], dtype=torch.int32, device=DEV).repeat(10)[:, None].contiguous()
    out = pkg.joint_token_logprobs(h, w, b, tok, top_k=64, entropy=True, validate=True)
    check_scores(out, scores_ref(z, tok, 64, 1.0), 200, 64)
    with pytest.raises(RuntimeError, match="label"):
        pkg.joint_token_logprobs(h, w, b, tok + 1, validate=True)


def test_no_rows():
    h = torch.empty((0, 64), dtype=torch.float16, device=DEV)
    w = torch.zeros((10, 64), dtype=torch.float16, device=DEV)
    out = pkg.joint_token_logprobs(h, w, None, top_k=3, entropy=True)
    assert out.top_index.shape == (0, 3) and out.entropy.shape == (0,) and out.logprobs is None


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("activation", ["tanh", "relu", None])
def test_joiner_scores_agree_with_its_logits(dtype, activation):
    torch.manual_seed(0)
    j = pkg.CompactJoiner(48, 40, 96, 61, activation=activation).to(DEV, dtype)
    lx = torch.tensor([9, 4, 1], dtype=torch.int32, device=DEV)
    ly = torch.tensor([3, 0, 5], dtype=torch.int32, device=DEV)
    y = torch.randint(1, 61, (3, 5), dtype=torch.int32, device=DEV)
    e, p = torch.randn((3, 9, 48), device=DEV, dtype=dtype), torch.randn((3, 6, 40), device=DEV, dtype=dtype)
    s = j.lattice_scores(e, p, lx, y, ly, top_k=4, entropy=True)
    with torch.no_grad():
        h = pkg.compact_join(j.enc(e), j.pred(p), lx, ly, activation)
        z = h.double() @ j.out.weight.double().T + j.out.bias.double()
    R = z.size(0)
    tok = pkg.lattice_tokens(lx, y, ly, R, 61)
    ref = scores_ref(z, tok, 4, 1.0)
    tol = 1e-5 + (0 if dtype != torch.float32 else 1e-5)  # 96 products of size below 1 in fp32, twice over
    assert float((s.logprobs.double() - ref["logprobs"]).abs().max()) <= tol
    assert float((s.entropy.double() - ref["entropy"]).abs().max()) <= 4 * tol
    assert torch.equal(s.top_index.long(), ref["top_index"])
    one = j.step_scores(e[:, 0], p[:, 0], tokens=tok[[0, 36, 40], 1].contiguous(), top_k=4)
    rows = torch.tensor([0, 36, 40], device=DEV)
    # the step forms its row with library calls that round the sum to the type before the activation
    assert float((one.top_logprobs - s.top_logprobs[rows]).abs().max()) <= (0.15 if dtype == torch.bfloat16 else 1e-5)
    assert one.logprobs.shape == (3,)
