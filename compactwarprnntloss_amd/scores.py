"""Scores of rows of logits, and distillation from a teacher's top logits.

`token_logprobs` gives, per row of a logit tensor such as the compact (sum_i T_i*(U_i+1), V) rows the
loss consumes, the log-probabilities of given tokens, the entropy and the most probable entries;
`distill_loss` pulls a student's rows towards a teacher's top entries.  Both read the logits once
(csrc/scores.hip, csrc/distill.hip) and are differentiable.  `lattice_tokens` names the (blank, label)
pair of every lattice cell, so that the two work next to `transducer_loss` on the same rows.

The reference has no counterpart; its callers run log_softmax on stored logits (test/test.py:19-20)."""
from __future__ import annotations

from typing import Any, NamedTuple, Optional

import torch

from . import _lib
from .loss import _DTYPES, _label_args, _raise_on_status, _stream_ptr

MAX_ROW_TOKENS = 64  # CWR_MAX_ROW_TOKENS


class TokenScores(NamedTuple):
    """What token_logprobs returns; fields that were not asked for are None."""
    logprobs: Optional[torch.Tensor]      # (R, M) fp32
    entropy: Optional[torch.Tensor]       # (R,) fp32
    lse: torch.Tensor                     # (R,) fp32
    top_logprobs: Optional[torch.Tensor]  # (R, K) fp32
    top_index: Optional[torch.Tensor]     # (R, K) int32


def _ptr(t: Optional[torch.Tensor]):
    return t.data_ptr() if t is not None else None


def _check_rows(x: torch.Tensor, temperature: float):
    if not x.is_cuda:
        raise RuntimeError("x must be a CUDA tensor")
    if x.dim() != 2:
        raise RuntimeError("x must be (R, V)")
    if x.dtype not in _DTYPES:
        raise RuntimeError(f"unsupported dtype {x.dtype}")
    if x.size(1) < 1:
        raise RuntimeError("x must have at least one entry per row")
    if x.size(1) > 1 and x.stride(1) != 1:
        raise RuntimeError("the entries of a row of x must be adjacent (rows may be any distance apart)")
    if not (1e-30 <= temperature <= 1e30):
        raise RuntimeError("temperature must be positive and finite")


def _check_tokens(tokens: Optional[torch.Tensor], R: int, device) -> Optional[torch.Tensor]:
    if tokens is None:
        return None
    if tokens.device != device:
        raise RuntimeError("tokens must be on the device of x")
    if tokens.dtype != torch.int32:
        raise RuntimeError("tokens must be torch::ScalarType::Int")
    if tokens.dim() not in (1, 2) or tokens.size(0) != R:
        raise RuntimeError("tokens must be (R,) or (R, M)")
    if not tokens.is_contiguous():
        raise RuntimeError("tokens must be contiguous")
    if tokens.dim() == 2 and not 1 <= tokens.size(1) <= MAX_ROW_TOKENS:
        raise RuntimeError(f"tokens must hold 1 to {MAX_ROW_TOKENS} tokens per row")
    return tokens.view(R, -1) if R else tokens.view(0, tokens.size(1) if tokens.dim() == 2 else 1)


def _check_top_k(top_k: int, V: int) -> int:
    if not 0 <= int(top_k) <= min(MAX_ROW_TOKENS, V):
        raise RuntimeError(f"top_k must lie between 0 and min({MAX_ROW_TOKENS}, V)")
    return int(top_k)


def _new_status(device) -> torch.Tensor:
    return torch.zeros(4, dtype=torch.int32, device=device)


class _TokenScores(torch.autograd.Function):
    @staticmethod
    def forward(ctx: Any, x, tokens, top_k, want_entropy, temperature, status):
        lib = _lib.load()
        R, V = x.shape
        dev = x.device
        M = tokens.size(1) if tokens is not None else 0
        need = ctx.needs_input_grad[0]

        def f32(*shape):
            return torch.empty(shape, dtype=torch.float32, device=dev)
        stat = f32(R, 2) if need else None
        logprobs = f32(R, M) if M else None
        entropy = f32(R) if want_entropy else None
        lse = f32(R)
        top = f32(R, top_k) if top_k else None
        index = torch.empty((R, top_k), dtype=torch.int32, device=dev) if top_k else None
        with torch.cuda.device(dev):
            rc = lib.cwr_token_logprobs(x.data_ptr(), _DTYPES[x.dtype], R, V, x.stride(0), _ptr(tokens), M, top_k,
                                        temperature, _ptr(stat), _ptr(logprobs), _ptr(entropy), lse.data_ptr(),
                                        _ptr(top), _ptr(index), _ptr(status), _stream_ptr(dev))
            _lib.check(rc, "cwr_token_logprobs")
        if index is not None:
            ctx.mark_non_differentiable(index)
        ctx.set_materialize_grads(False)
        if need:
            ctx.temperature = temperature
            ctx.save_for_backward(x, tokens, index, entropy, stat)
        return logprobs, entropy, lse, top, index

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx: Any, g_logprobs, g_entropy, g_lse, g_top, _g_index):
        x, tokens, index, entropy, stat = ctx.saved_tensors
        lib = _lib.load()
        R, V = x.shape
        dev = x.device
        grads = [g.to(torch.float32).contiguous() if g is not None else None for g in (g_logprobs, g_entropy, g_lse, g_top)]
        dx = torch.empty((R, V), dtype=x.dtype, device=dev)
        with torch.cuda.device(dev):
            rc = lib.cwr_token_logprobs_backward(
                x.data_ptr(), _DTYPES[x.dtype], R, V, x.stride(0), _ptr(tokens),
                tokens.size(1) if tokens is not None else 0, _ptr(index), index.size(1) if index is not None else 0,
                ctx.temperature, stat.data_ptr(), _ptr(entropy), *[_ptr(g) for g in grads], dx.data_ptr(),
                _stream_ptr(dev))
            _lib.check(rc, "cwr_token_logprobs_backward")
        return dx, None, None, None, None, None


def token_logprobs(x: torch.Tensor, tokens: Optional[torch.Tensor] = None, *, top_k: int = 0, entropy: bool = False,
                   temperature: float = 1.0, validate: bool = False) -> TokenScores:
    """Scores of the rows of logits x under softmax(x / temperature).

    x         (R, V) fp32, fp16, bf16 or fp64 logits (or log-probabilities); the entries of a row adjacent,
              rows any distance apart (a slice of a padded tensor is fine)
    tokens    (R,) or (R, M) int32, M <= 64: entries to score; -1 stands for no token (0, no gradient)
    top_k     number of most probable entries to return, <= 64, in descending order, equal ones by ascending
              index (NaN ranks with -inf)
    entropy   also return the entropy of each row
    validate  read the status word back (one synchronisation) and raise when a token lies outside
              [0, V); without it the log-probability of such a token is NaN and it gets no gradient

    Returns TokenScores(logprobs, entropy, lse, top_logprobs, top_index); logprobs has the shape of tokens.
    Differentiable in x through everything but top_index.  A row of nothing but -inf has log-probabilities
    -inf, entropy 0 and gradient 0; a row that holds NaN or +inf gives NaN."""
    temperature = float(temperature)
    _check_rows(x, temperature)
    R, V = x.shape
    rows = _check_tokens(tokens, R, x.device)
    status = _new_status(x.device) if validate else None
    logprobs, ent, lse, top, index = _TokenScores.apply(x, rows, _check_top_k(top_k, V), bool(entropy), temperature,
                                                        status)
    if validate:
        _raise_on_status(status, "token_logprobs")
    if tokens is not None and tokens.dim() == 1:
        logprobs = logprobs.view(R)
    return TokenScores(logprobs, ent, lse, top, index)


class _Distill(torch.autograd.Function):
    @staticmethod
    def forward(ctx: Any, x, top, index, temperature, tail, reduction, status):
        lib = _lib.load()
        R, V = x.shape
        dev = x.device
        need = ctx.needs_input_grad[0]
        loss = torch.empty(R, dtype=torch.float32, device=dev)
        stat = torch.empty((R, 4), dtype=torch.float32, device=dev) if need else None
        reduced = work = None
        if reduction != "none":
            reduced = torch.empty(2, dtype=torch.float32, device=dev)
            work = torch.empty(lib.cwr_distill_workspace_bytes(), dtype=torch.uint8, device=dev)
        with torch.cuda.device(dev):
            rc = lib.cwr_distill(x.data_ptr(), _DTYPES[x.dtype], R, V, x.stride(0), top.data_ptr(), index.data_ptr(),
                                 index.size(1), temperature, int(tail), loss.data_ptr(), _ptr(stat), _ptr(reduced),
                                 _ptr(work), _ptr(status), _stream_ptr(dev))
            _lib.check(rc, "cwr_distill")
        if need:
            ctx.temperature, ctx.tail, ctx.reduction = temperature, tail, reduction
            ctx.save_for_backward(x, top, index, stat)
        if reduction == "none":
            return loss
        return reduced[1 if reduction == "mean" else 0]

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx: Any, grad_out):
        x, top, index, stat = ctx.saved_tensors
        lib = _lib.load()
        R, V = x.shape
        dev = x.device
        go = grad_out.to(torch.float32).contiguous()
        stride = 1 if ctx.reduction == "none" else 0
        scale = 1.0 / R if ctx.reduction == "mean" and R else 1.0
        dx = torch.empty((R, V), dtype=x.dtype, device=dev)
        with torch.cuda.device(dev):
            rc = lib.cwr_distill_backward(x.data_ptr(), _DTYPES[x.dtype], R, V, x.stride(0), top.data_ptr(),
                                          index.data_ptr(), index.size(1), ctx.temperature, int(ctx.tail),
                                          stat.data_ptr(), go.data_ptr(), stride, scale, dx.data_ptr(), _stream_ptr(dev))
            _lib.check(rc, "cwr_distill_backward")
        return dx, None, None, None, None, None, None


def distill_loss(x: torch.Tensor, top_logits: torch.Tensor, top_index: torch.Tensor, *, temperature: float = 1.0,
                 tail: bool = False, reduction: Optional[str] = "mean", validate: bool = False) -> torch.Tensor:
    """temperature^2 * KL(teacher || student) per row, the student's softmax(x / temperature) against a teacher of
    which only the K best entries of a row are known.

    x           (R, V) student logits, as for token_logprobs
    top_logits  (R, K) the teacher's values, top_index (R, K) int32 the entries they belong to, K <= 64;
                an index of -1 is absent, a row whose list is empty has loss 0 and gradient 0
    tail        False: the teacher is softmax(top_logits / temperature) over the list.
                True: top_logits are log-probabilities at this temperature (token_logprobs(...,
                temperature=temperature).top_logprobs); the mass they leave is one more class, compared
                with the student's mass outside the list
    reduction   "mean" over the rows, "sum", or "none" / None for one loss per row
    validate    read the status word back (one synchronisation) and raise when an index lies outside
                [-1, V); without it the loss of such a row is NaN and its gradient 0

    Differentiable in x; the teacher gets no gradient."""
    assert reduction in ["mean", "sum", "none"] or reduction is None
    temperature = float(temperature)
    _check_rows(x, temperature)
    R, V = x.shape
    if top_logits.dim() != 2 or top_logits.shape != top_index.shape or top_index.size(0) != R:
        raise RuntimeError("top_logits and top_index must both be (R, K)")
    if not 1 <= top_index.size(1) <= MAX_ROW_TOKENS:
        raise RuntimeError(f"the teacher's lists must hold 1 to {MAX_ROW_TOKENS} entries")
    if top_index.dtype != torch.int32:
        raise RuntimeError("top_index must be torch::ScalarType::Int")
    if top_logits.dtype not in _DTYPES:
        raise RuntimeError(f"unsupported dtype {top_logits.dtype}")
    if top_logits.device != x.device or top_index.device != x.device:
        raise RuntimeError("top_logits and top_index must be on the device of x")
    if torch.is_grad_enabled() and top_logits.requires_grad:
        raise RuntimeError("the teacher gets no gradient: pass top_logits.detach()")
    status = _new_status(x.device) if validate else None
    loss = _Distill.apply(x, top_logits.to(torch.float32).contiguous(), top_index.contiguous(), temperature, bool(tail),
                          reduction if reduction in ("mean", "sum") else "none", status)
    if validate:
        _raise_on_status(status, "distill_loss")
    return loss


def lattice_tokens(lx: torch.Tensor, y: torch.Tensor, ly: torch.Tensor, total_rows: int, V: int,
                   blank: int = 0) -> torch.Tensor:
    """(total_rows, 2) int32: the blank and the label of every compact row, -1 where a row has no label (the
    last label position of a sequence) or belongs to no sequence: the `tokens` under which token_logprobs
    returns the pair of log-probabilities the loss walks on.

    lx, ly, y as for transducer_loss; total_rows = sum_i lx_i*(ly_i+1)."""
    for name, t in (("lx", lx), ("y", y), ("ly", ly)):
        if not t.is_cuda or t.dtype != torch.int32 or not t.is_contiguous():
            raise RuntimeError(f"{name} must be a contiguous CUDA int32 tensor")
    if lx.dim() != 1 or lx.shape != ly.shape or y.dim() not in (1, 2) or (y.dim() == 2 and y.size(0) != lx.size(0)):
        raise RuntimeError("lx, ly must be (N,), y (N, U) or concatenated")
    assert blank >= 0 and blank < V
    lib = _lib.load()
    dev = lx.device
    N, R = lx.numel(), int(total_rows)
    off = torch.empty(2 * (N + 1) + 2, dtype=torch.int64, device=dev)
    info = torch.empty((R, 2), dtype=torch.int32, device=dev)
    y_stride, y_len = _label_args(y)
    with torch.cuda.device(dev):
        stream = _stream_ptr(dev)
        rc = lib.cwr_offsets(lx.data_ptr(), ly.data_ptr(), N, R, off.data_ptr(), off[N + 1:].data_ptr(),
                             off[2 * (N + 1):].data_ptr(), stream)
        _lib.check(rc, "cwr_offsets")
        rc = lib.cwr_rowinfo(lx.data_ptr(), ly.data_ptr(), y.data_ptr(), y_stride, y_len, N, R, int(V), off.data_ptr(),
                             off[N + 1:].data_ptr(), info.data_ptr(), stream)
        _lib.check(rc, "cwr_rowinfo")
    label, owner = info[:, 0], info[:, 1]
    return torch.stack((torch.where(owner >= 0, int(blank), -1).to(torch.int32), label), dim=1)
