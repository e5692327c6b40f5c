"""The row operators' argument checks: in the C entry points, before any HIP call (no GPU needed), and in Python."""
import math

import pytest
import torch

import compactwarprnntloss_amd as pkg
from compactwarprnntloss_amd import _lib


def p(n):
    """A non-null, 256-byte aligned host address: validation never dereferences it."""
    return 0x10000 * n


def tokens_call(**kw):
    a = dict(x=p(1), dtype=0, R=10, V=40, stride=40, tokens=p(2), M=2, K=3, T=1.0, stat=p(3), lp=p(4), ent=p(5), lse=p(6),
             top=p(7), idx=p(8), status=p(9))
    a.update(kw)
    return _lib.load().cwr_token_logprobs(a["x"], a["dtype"], a["R"], a["V"], a["stride"], a["tokens"], a["M"], a["K"], a["T"],
                                          a["stat"], a["lp"], a["ent"], a["lse"], a["top"], a["idx"], a["status"], None)


def tokens_bwd(**kw):
    a = dict(x=p(1), dtype=0, R=10, V=40, stride=40, tokens=p(2), M=2, idx=p(3), K=3, T=1.0, stat=p(4), g1=p(5), g2=p(6),
             g3=p(7), g4=p(8), dx=p(9))
    a.update(kw)
    return _lib.load().cwr_token_logprobs_backward(a["x"], a["dtype"], a["R"], a["V"], a["stride"], a["tokens"], a["M"],
                                                   a["idx"], a["K"], a["T"], a["stat"], a["g1"], a["g2"], a["g3"], a["g4"],
                                                   a["dx"], None)


def distill_call(**kw):
    a = dict(x=p(1), dtype=0, R=10, V=40, stride=40, top=p(2), idx=p(3), K=3, T=1.0, tail=0, loss=p(4), stat=p(5), total=p(6),
             mean=p(7), ws=p(8), status=p(9))
    a.update(kw)
    return _lib.load().cwr_distill(a["x"], a["dtype"], a["R"], a["V"], a["stride"], a["top"], a["idx"], a["K"], a["T"],
                                   a["tail"], a["loss"], a["stat"], a["total"], a["mean"], a["ws"], a["status"], None)


def distill_bwd(**kw):
    a = dict(x=p(1), dtype=0, R=10, V=40, stride=40, top=p(2), idx=p(3), K=3, T=1.0, tail=1, stat=p(4), g=p(5), gs=1, dx=p(6))
    a.update(kw)
    return _lib.load().cwr_distill_backward(a["x"], a["dtype"], a["R"], a["V"], a["stride"], a["top"], a["idx"], a["K"],
                                            a["T"], a["tail"], a["stat"], a["g"], a["gs"], 1.0, a["dx"], None)


def joint_call(**kw):
    a = dict(h=p(1), w=p(2), b=p(3), bdt=0, dtype=2, R=10, H=64, V=40, tokens=p(4), M=2, K=3, T=1.0, lp=p(5), ent=p(6),
             lse=p(7), top=p(8), idx=p(9), ws=p(10), nb=1 << 20, status=p(11))
    a.update(kw)
    return _lib.load().cwr_joint_token_logprobs(a["h"], a["w"], a["b"], a["bdt"], a["dtype"], a["R"], a["H"], a["V"],
                                                a["tokens"], a["M"], a["K"], a["T"], a["lp"], a["ent"], a["lse"], a["top"],
                                                a["idx"], a["ws"], a["nb"], a["status"], None)


NULL, DTYPE, MODE, SHAPE, ALIGN, LARGE = 1, 2, 3, 4, 6, 8


@pytest.mark.parametrize("call", [tokens_call, tokens_bwd, distill_call, distill_bwd])
def test_checks_the_calls_on_logits_share(call):
    assert call(dtype=4) == DTYPE and call(dtype=-1) == DTYPE
    assert call(R=-1) == SHAPE and call(V=0) == SHAPE and call(stride=-1) == SHAPE and call(K=-1) == SHAPE
    assert call(V=1 << 28) == LARGE and call(K=65, V=100) == LARGE
    for T in (0.0, -1.0, math.inf, math.nan, 1e-7, 1e7):
        assert call(T=T) == SHAPE
    assert call(x=None) == NULL
    assert call(x=p(1) + 2) == ALIGN                 # fp32 off its 4-byte grid
    assert call(x=p(1) + 1, dtype=1) == ALIGN
    assert call(stat=p(4) + 8) == ALIGN


def test_checks_of_the_score_calls():
    assert tokens_call(M=-1) == SHAPE and tokens_call(M=65) == LARGE and tokens_call(K=41) == SHAPE
    assert tokens_call(tokens=None) == NULL and tokens_call(lp=None) == NULL
    assert tokens_call(top=None) == NULL and tokens_call(idx=None) == NULL
    assert tokens_call(tokens=p(2) + 1) == ALIGN and tokens_call(lse=p(6) + 2) == ALIGN and tokens_call(idx=p(8) + 2) == ALIGN
    assert tokens_bwd(stat=None) == NULL and tokens_bwd(dx=None) == NULL and tokens_bwd(idx=None) == NULL
    assert tokens_bwd(g2=p(6) + 2) == ALIGN and tokens_bwd(dx=p(9) + 2) == ALIGN
    assert tokens_call(R=0, x=None, tokens=None, lp=None, top=None, idx=None) == 0
    assert tokens_bwd(R=0, x=None, stat=None, dx=None, idx=None, tokens=None) == 0


def test_checks_of_the_distillation_calls():
    assert distill_call(K=0) == SHAPE and distill_call(tail=2) == MODE and distill_bwd(tail=-1) == MODE
    assert distill_call(top=None) == NULL and distill_call(idx=None) == NULL and distill_call(loss=None) == NULL
    assert distill_call(ws=None) == NULL and distill_call(ws=p(8) + 4) == ALIGN
    assert distill_bwd(gs=2) == SHAPE and distill_bwd(g=None) == NULL and distill_bwd(stat=None) == NULL
    assert distill_bwd(dx=None) == NULL and distill_bwd(dx=p(6) + 2) == ALIGN
    assert distill_call(R=0, x=None, top=None, idx=None, loss=None, total=None, mean=None, ws=None) == 0
    assert distill_bwd(R=0, x=None, top=None, idx=None, stat=None, g=None, dx=None) == 0
    assert _lib.load().cwr_distill_workspace_bytes() % 8 == 0


def test_checks_of_the_joint_call():
    assert joint_call(dtype=0) == DTYPE and joint_call(dtype=3) == DTYPE and joint_call(bdt=1) == DTYPE
    assert joint_call(bdt=1, b=None, R=0) == 0       # without a bias its type means nothing
    assert joint_call(H=48) == SHAPE and joint_call(H=0) == SHAPE and joint_call(H=1 << 30) == LARGE
    assert joint_call(w=None) == NULL and joint_call(ws=None) == NULL and joint_call(lp=None) == NULL
    assert joint_call(h=p(1) + 2) == ALIGN and joint_call(w=p(2) + 8) == ALIGN and joint_call(ws=p(10) + 16) == ALIGN
    assert joint_call(b=p(3) + 2) == ALIGN
    assert joint_call(nb=40 * 4 - 1) == SHAPE        # not one row of logits
    assert joint_call(M=65) == LARGE and joint_call(K=41) == SHAPE and joint_call(T=0.0) == SHAPE
    bytes_ = _lib.load().cwr_joint_token_logprobs_workspace_bytes
    assert bytes_(-1, 8) == 0 and bytes_(8, 0) == 0 and bytes_(3, 41) == 3 * 44 * 4
    assert bytes_(10 ** 9, 1024) <= 256 << 20 and bytes_(10 ** 9, 50257) == 4096 * 50260 * 4


def test_python_refuses_host_tensors():
    x = torch.zeros(3, 8)
    tok = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        pkg.token_logprobs(x, tok)
    with pytest.raises(RuntimeError, match="CUDA"):
        pkg.distill_loss(x, x[:, :2], torch.zeros((3, 2), dtype=torch.int32))
    with pytest.raises(RuntimeError, match="CUDA"):
        pkg.joint_token_logprobs(x.half(), x.half())
    with pytest.raises(RuntimeError, match="CUDA"):
        pkg.lattice_tokens(tok, tok, tok, 3, 8)


@pytest.mark.gpu
def test_python_refusals():
    dev = "cuda:0"
    x = torch.zeros((3, 8), device=dev)
    tok = torch.zeros(3, dtype=torch.int32, device=dev)
    bad = [lambda: pkg.token_logprobs(x[0], tok), lambda: pkg.token_logprobs(x.long(), tok), lambda: pkg.token_logprobs(x.t(), tok),
           lambda: pkg.token_logprobs(x[:, ::2], tok), lambda: pkg.token_logprobs(x, tok.long()),
           lambda: pkg.token_logprobs(x, tok[:2]), lambda: pkg.token_logprobs(x, tok.cpu()),
           lambda: pkg.token_logprobs(x, tok.expand(3, 3).t()[:, :2]), lambda: pkg.token_logprobs(x, top_k=9),
           lambda: pkg.token_logprobs(x, top_k=-1), lambda: pkg.token_logprobs(x, tok, temperature=0),
           lambda: pkg.token_logprobs(x, tok, temperature=math.nan),
           lambda: pkg.token_logprobs(x, torch.zeros((3, 65), dtype=torch.int32, device=dev)),
           lambda: pkg.token_logprobs(torch.zeros((3, 0), device=dev))]
    idx = torch.zeros((3, 2), dtype=torch.int32, device=dev)
    top = torch.zeros((3, 2), device=dev)
    bad += [lambda: pkg.distill_loss(x, top, idx.long()), lambda: pkg.distill_loss(x, top[:2], idx),
            lambda: pkg.distill_loss(x, top[:, :1], idx), lambda: pkg.distill_loss(x, top.cpu(), idx.cpu()),
            lambda: pkg.distill_loss(x, top.long(), idx), lambda: pkg.distill_loss(x, top, idx, temperature=-1),
            lambda: pkg.distill_loss(x, top[:, :0], idx[:, :0]),
            lambda: pkg.distill_loss(x, top.clone().requires_grad_(True), idx)]
    h, w = (torch.zeros(s, dtype=torch.float16, device=dev) for s in ((3, 32), (8, 32)))
    b = torch.zeros(8, dtype=torch.float16, device=dev)
    bad += [lambda: pkg.joint_token_logprobs(h.float(), w.float()), lambda: pkg.joint_token_logprobs(h, w.bfloat16()),
            lambda: pkg.joint_token_logprobs(h[:, :16].contiguous(), w[:, :16].contiguous()),
            lambda: pkg.joint_token_logprobs(h, w[:, :16]), lambda: pkg.joint_token_logprobs(h, w, b[:4]),
            lambda: pkg.joint_token_logprobs(h, w, b.bfloat16()), lambda: pkg.joint_token_logprobs(h, w.cpu()),
            lambda: pkg.joint_token_logprobs(h, w.clone().requires_grad_(True)),
            lambda: pkg.joint_token_logprobs(h[::2], w)]
    for i, f in enumerate(bad):
        with pytest.raises(RuntimeError):
            f()
            pytest.fail(f"call {i} was not refused")
    with pytest.raises(AssertionError):
        pkg.distill_loss(x, top, idx, reduction="max")
    with torch.no_grad():
        pkg.joint_token_logprobs(h, w.clone().requires_grad_(True))
