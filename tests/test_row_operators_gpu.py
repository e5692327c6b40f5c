"""The row operators as a program uses them: a teacher's pass, a student's training step next to the loss,
graphs, streams."""
import pytest
import torch

import compactwarprnntloss_amd as pkg
from compactwarprnntloss_amd import _lib, scores, workloads as wl

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def batch(dtype=torch.bfloat16, E=64, P=48, scale=0.15):
    cfg = wl.make_config(2, scale=scale)
    lx, ly = torch.from_numpy(cfg["lx"]).to(DEV), torch.from_numpy(cfg["ly"]).to(DEV)
    y = torch.from_numpy(cfg["y_padded"]).to(DEV) % 97
    gen = torch.Generator(device=DEV).manual_seed(0)
    e = torch.randn((cfg["N"], int(lx.max()), E), device=DEV, generator=gen).to(dtype)
    p = torch.randn((cfg["N"], int(ly.max()) + 1, P), device=DEV, generator=gen).to(dtype)
    return cfg["R"], lx, ly, y.contiguous(), e, p


@pytest.mark.parametrize("tail", [False, True])
def test_teacher_to_student_training_step(tail):
    """lattice_scores of a teacher -> distill_loss + transducer_loss on a student's logits: one backward pass whose
    parameter gradients are those of the two losses apart, and of the formula on float64 logits."""
    torch.manual_seed(1)
    R, lx, ly, y, e, p = batch()
    teacher = pkg.CompactJoiner(64, 48, 128, 97).to(DEV, torch.bfloat16)
    student = pkg.CompactJoiner(64, 48, 64, 97).to(DEV, torch.float32)
    s = teacher.lattice_scores(e, p, lx, y, ly, top_k=8, temperature=2.0, total_rows=R)
    assert s.top_logprobs.shape == (R, 8) and not s.top_logprobs.requires_grad

    def grads(a, b):
        student.zero_grad()
        logits = student(e.float(), p.float(), lx, ly, R)
        logits.retain_grad()
        total = 0.0
        if a:
            total = total + a * pkg.transducer_loss(logits, lx, y, ly, 0, "mean", fused_log_softmax=True)
        if b:
            total = total + b * pkg.distill_loss(logits, s.top_logprobs, s.top_index, temperature=2.0, tail=tail)
        total.backward()
        return logits, [q.grad.clone() for q in student.parameters()]
    logits, both = grads(1.0, 0.5)
    _, one = grads(1.0, 0)
    dl, two = grads(0, 0.5)
    for g, a, b in zip(both, one, two):
        assert float((g - a - b).abs().max()) <= 1e-5 * float(g.abs().max()) + 1e-7
    from tests.rowrefs import distill_ref
    _, d1, _, _ = distill_ref(dl.detach(), s.top_logprobs, s.top_index, 2.0, tail)
    want = d1 * (0.5 / R)
    assert float((dl.grad.double() - want).norm() / want.norm()) <= 2e-6


def _steps(x, tok, top, idx, h, w):
    """One forward and backward pass of each operator through the entry points, no autograd graph of x alive."""
    r = scores._run_scores(x, tok, 2, 4, True, 1.0, None, True)
    leaf = x.detach().requires_grad_(True)
    out = pkg.token_logprobs(leaf, tok, top_k=4, entropy=True)
    d1, = torch.autograd.grad([out.logprobs, out.entropy, out.top_logprobs], leaf,
                              [torch.ones_like(out.logprobs), torch.ones_like(out.entropy), torch.ones_like(out.top_logprobs)])
    loss = pkg.distill_loss(leaf, top, idx, tail=True)
    d2, = torch.autograd.grad(loss, leaf)
    j = pkg.joint_token_logprobs(h, w, None, tok, top_k=4)
    return [r[0], r[3], r[4], d1, loss.detach(), d2, j.logprobs, j.top_index]


@pytest.mark.parametrize("R,V", [(300, 41), (20000, 128), (70, 5001)])
def test_graph_replays_match_eager(R, V):
    gen = torch.Generator(device=DEV).manual_seed(R)

    def fresh():
        x = torch.randn((R, V), device=DEV, generator=gen) * 2
        tok = torch.randint(-1, V, (R, 2), device=DEV, generator=gen, dtype=torch.int32)
        top, idx = (x + torch.randn((R, V), device=DEV, generator=gen)).log_softmax(1).topk(5, dim=1)
        h = torch.randn((R, 64), device=DEV, generator=gen).to(torch.bfloat16)
        return x, tok, top, idx.to(torch.int32), h
    x, tok, top, idx, h = fresh()
    w = torch.randn((V, 64), device=DEV, generator=gen).to(torch.bfloat16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _steps(x, tok, top, idx, h, w)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = _steps(x, tok, top, idx, h, w)
    for _ in range(4):
        for dst, src in zip((x, tok, top, idx, h), fresh()):
            dst.copy_(src)
        graph.replay()
        torch.cuda.synchronize()
        want = _steps(x, tok, top, idx, h, w)   # eager work between the replays
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_calls_on_two_streams_do_not_disturb_each_other():
    gen = torch.Generator(device=DEV).manual_seed(0)
    a, b = (torch.randn((60000, 300), device=DEV, generator=gen) for _ in range(2))
    ta, tb = (torch.randint(0, 300, (60000, 2), device=DEV, generator=gen, dtype=torch.int32) for _ in range(2))
    tops = [t.topk(6, dim=1) for t in (a, b)]
    h = torch.randn((60000, 64), device=DEV, generator=gen).to(torch.float16)
    w = torch.randn((300, 64), device=DEV, generator=gen).to(torch.float16)

    def work(x, t, top):
        return _steps(x, t, top[0].log_softmax(1), top[1].to(torch.int32), h, w)
    want = [work(a, ta, tops[0]), work(b, tb, tops[1])]
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(3):
        with torch.cuda.stream(s1):
            g1 = work(a, ta, tops[0])
        with torch.cuda.stream(s2):
            g2 = work(b, tb, tops[1])
        torch.cuda.synchronize()
        for got, ref in zip((g1, g2), want):
            for p, q in zip(got, ref):
                assert torch.equal(p, q)


def test_a_graph_can_be_walked_twice_and_losses_changed_in_place():
    gen = torch.Generator(device=DEV).manual_seed(0)
    x = torch.randn((40, 70), device=DEV, generator=gen).requires_grad_(True)
    top, idx = torch.randn((40, 70), device=DEV, generator=gen).log_softmax(1).topk(5, dim=1)
    loss = pkg.distill_loss(x, top, idx.to(torch.int32), tail=True)
    a, = torch.autograd.grad(loss, x, retain_graph=True)
    b, = torch.autograd.grad(loss, x, retain_graph=True)
    assert torch.equal(a, b)
    loss *= 2.0
    c, = torch.autograd.grad(loss, x)
    assert torch.equal(c, 2 * a)
    out = pkg.token_logprobs(x, top_k=3, entropy=True)
    out.entropy.mul_(2.0)
    d, = torch.autograd.grad(out.entropy.sum(), x)
    e, = torch.autograd.grad(pkg.token_logprobs(x, entropy=True).entropy.sum(), x)
    assert torch.equal(d, 2 * e)


def test_rows_behind_the_last_and_neighbouring_memory_are_left_alone():
    """The entry points write their outputs and nothing else: guard rows around every one."""
    lib = _lib.load()
    R, V, K, M = 37, 45, 3, 2
    gen = torch.Generator(device=DEV).manual_seed(0)
    x = torch.randn((R, V), device=DEV, generator=gen)
    tok = torch.randint(0, V, (R, M), device=DEV, generator=gen, dtype=torch.int32)

    def guarded(rows, cols, dtype=torch.float32):
        t = torch.full((rows + 8, cols), 77, dtype=dtype, device=DEV)
        return t, t[4:]
    bufs = dict(stat=guarded(R, 4), lp=guarded(R, M), ent=guarded(R, 1), lse=guarded(R, 1), top=guarded(R, K),
                idx=guarded(R, K, torch.int32), dx=guarded(R, V), loss=guarded(R, 1), st4=guarded(R, 4), dd=guarded(R, V))
    ptr = {k: v[1].data_ptr() for k, v in bufs.items()}
    s = torch.cuda.current_stream().cuda_stream
    g = torch.ones((R, M), device=DEV)
    assert lib.cwr_token_logprobs(x.data_ptr(), 0, R, V, V, tok.data_ptr(), M, K, 1.0, ptr["stat"], ptr["lp"], ptr["ent"],
                                  ptr["lse"], ptr["top"], ptr["idx"], None, s) == 0
    assert lib.cwr_token_logprobs_backward(x.data_ptr(), 0, R, V, V, tok.data_ptr(), M, ptr["idx"], K, 1.0, ptr["stat"],
                                           g.data_ptr(), None, None, None, ptr["dx"], s) == 0
    assert lib.cwr_distill(x.data_ptr(), 0, R, V, V, ptr["top"], ptr["idx"], K, 1.0, 1, ptr["loss"], ptr["st4"], None, None,
                           None, None, s) == 0
    assert lib.cwr_distill_backward(x.data_ptr(), 0, R, V, V, ptr["top"], ptr["idx"], K, 1.0, 1, ptr["st4"], g.data_ptr(), 1,
                                    1.0, ptr["dd"], s) == 0
    torch.cuda.synchronize()
    for name, (whole, _) in bufs.items():
        assert (whole[:4] == 77).all() and (whole[4 + R:] == 77).all(), name
        assert not (whole[4:4 + R] == 77).any(), name
