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


# The raw handle of a device's current stream: what torch.cuda.current_stream(device).cuda_stream returns,
# without building the Stream object in between (2 us, a tenth of a small call).
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


def _call(name: str, device: torch.device, *args):
    """Runs entry point `name` with `args` and the current stream of `device`, on that device."""
    fn = getattr(_lib.load(), name)
    index = device.index
    if torch.cuda.current_device() == index:
        rc = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _raw_stream(index))
    if rc:
        _lib.check(rc, name)


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
    if not (1e-6 <= temperature <= 1e6):
        raise RuntimeError("temperature must lie between 1e-6 and 1e6")


def _check_tokens(tokens: Optional[torch.Tensor], R: int, device) -> int:
    """Tokens per row M of a (R,) or (R, M) tensor of tokens, 0 for None."""
    if tokens is None:
        return 0
    if tokens.device != device:
        raise RuntimeError("tokens must be on the device of x")
    if tokens.dtype != torch.int32:
        raise RuntimeError("tokens must be torch::ScalarType::Int")
    dims = tokens.dim()
    if dims not in (1, 2) or tokens.size(0) != R:
        raise RuntimeError("tokens must be (R,) or (R, M)")
    if not tokens.is_contiguous():
        raise RuntimeError("tokens must be contiguous")
    M = tokens.size(1) if dims == 2 else 1
    if not 1 <= M <= MAX_ROW_TOKENS:
        raise RuntimeError(f"tokens must hold 1 to {MAX_ROW_TOKENS} tokens per row")
    return M


def _check_top_k(top_k: int, V: int) -> int:
    if not 0 <= int(top_k) <= min(MAX_ROW_TOKENS, V):
        raise RuntimeError(f"top_k must lie between 0 and min({MAX_ROW_TOKENS}, V)")
    return int(top_k)


def _new_status(device) -> torch.Tensor:
    return torch.zeros(4, dtype=torch.int32, device=device)


def _score_buffers(R: int, M: int, top_k: int, want_entropy: bool, dev):
    """(logprobs, entropy, lse, top_logprobs, top_index) to be written.  Sizes as separate arguments: half a
    microsecond less per tensor than a tuple, which a step of a search feels."""
    f32 = torch.float32
    logprobs = torch.empty(R, M, dtype=f32, device=dev) if M else None
    entropy = torch.empty(R, dtype=f32, device=dev) if want_entropy else None
    lse = torch.empty(R, dtype=f32, device=dev)
    top = index = None
    if top_k:
        top = torch.empty(R, top_k, dtype=f32, device=dev)
        index = torch.empty(R, top_k, dtype=torch.int32, device=dev)
    return logprobs, entropy, lse, top, index


def _run_scores(x, tokens, M, top_k, want_entropy, temperature, status, keep):
    """Binding of cwr_token_logprobs: (logprobs, entropy, lse, top_logprobs, top_index, stat)."""
    R, V = x.shape
    dev = x.device
    logprobs, entropy, lse, top, index = _score_buffers(R, M, top_k, want_entropy, dev)
    stat = torch.empty(R, 4, dtype=torch.float32, device=dev) if keep else None
    _call("cwr_token_logprobs", dev, x.data_ptr(), _DTYPES[x.dtype], R, V, x.stride(0), _ptr(tokens), M, top_k,
          temperature, _ptr(stat), _ptr(logprobs), _ptr(entropy), lse.data_ptr(), _ptr(top), _ptr(index), _ptr(status))
    return logprobs, entropy, lse, top, index, stat


class _TokenScores(torch.autograd.Function):
    @staticmethod
    def forward(ctx: Any, x, tokens, M, top_k, want_entropy, temperature, status):
        logprobs, entropy, lse, top, index, stat = _run_scores(x, tokens, M, top_k, want_entropy, temperature, status, True)
        if index is not None:
            ctx.mark_non_differentiable(index)
        ctx.set_materialize_grads(False)
        ctx.temperature, ctx.M = temperature, M
        ctx.save_for_backward(x, tokens, index, stat)
        return logprobs, entropy, lse, top, index

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx: Any, g_logprobs, g_entropy, g_lse, g_top, _g_index):
        x, tokens, index, stat = ctx.saved_tensors
        R, V = x.shape
        grads = [g if g is None else _rows_f32(g) for g in (g_logprobs, g_entropy, g_lse, g_top)]
        dx = torch.empty((R, V), dtype=x.dtype, device=x.device)
        _call("cwr_token_logprobs_backward", x.device, x.data_ptr(), _DTYPES[x.dtype], R, V, x.stride(0), _ptr(tokens),
              ctx.M, _ptr(index), index.size(1) if index is not None else 0,
              ctx.temperature, stat.data_ptr(), *[_ptr(g) for g in grads], dx.data_ptr())
        return dx, None, None, None, None, None, None


def _rows_f32(g: torch.Tensor) -> torch.Tensor:
    return g if g.dtype == torch.float32 and g.is_contiguous() else g.to(torch.float32).contiguous()


def token_logprobs(x: torch.Tensor, tokens: Optional[torch.Tensor] = None, *, top_k: int = 0, entropy: bool = False,
                   temperature: float = 1.0, validate: bool = False) -> TokenScores:
    """Scores of the rows of logits x under softmax(x / temperature).

    x         (R, V) fp32, fp16, bf16 or fp64 logits (or log-probabilities), fp64 rounded to fp32 when read; the
              entries of a row adjacent, rows any distance apart (a slice of a padded tensor is fine)
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
    M = _check_tokens(tokens, R, x.device)
    status = _new_status(x.device) if validate else None
    top_k = _check_top_k(top_k, V)
    if x.requires_grad and torch.is_grad_enabled():
        logprobs, ent, lse, top, index = _TokenScores.apply(x, tokens, M, top_k, bool(entropy), temperature, status)
    else:
        logprobs, ent, lse, top, index, _ = _run_scores(x, tokens, M, top_k, bool(entropy), temperature, status, False)
    if validate:
        _raise_on_status(status, "token_logprobs")
    if tokens is not None and tokens.dim() == 1:
        logprobs = logprobs.view(R)
    return TokenScores(logprobs, ent, lse, top, index)


def joint_token_logprobs(h: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
                         tokens: Optional[torch.Tensor] = None, *, top_k: int = 0, entropy: bool = False,
                         temperature: float = 1.0, validate: bool = False) -> TokenScores:
    """token_logprobs of the logits h @ weight.T + bias without storing them: h (R, H) joint rows (from
    compact_join, or one row per hypothesis of a search), weight (V, H), both fp16 or both bf16 with H a
    multiple of 32; bias (V,) in the same type or fp32, or None.  The product runs on the matrix cores with
    fp32 accumulation and is scored from fp32, a block of rows at a time (256 MiB of workspace at most, or 4096 rows).

    For a teacher's pass over a lattice and for the steps of a search: the scores carry no gradient, and a
    call that would need one is refused."""
    temperature = float(temperature)
    _check_rows(h, temperature)
    if h.dtype not in (torch.float16, torch.bfloat16) or weight.dtype != h.dtype:
        raise RuntimeError("h and weight must both be float16 or both be bfloat16")
    if weight.dim() != 2 or weight.size(1) != h.size(1) or weight.size(0) < 1:
        raise RuntimeError("weight must be (V, H) with the joint dimension H of the rows")
    if h.size(1) % 32 != 0:
        raise RuntimeError("the joint dimension must be a multiple of 32")
    dev = h.device
    if weight.device != dev or (bias is not None and bias.device != dev):
        raise RuntimeError("weight and bias must be on the device of h")
    if not h.is_contiguous() or not weight.is_contiguous():
        raise RuntimeError("h and weight must be contiguous")
    R, H = h.shape
    V = weight.size(0)
    if bias is not None and (bias.shape != (V,) or bias.dtype not in (h.dtype, torch.float32) or not bias.is_contiguous()):
        raise RuntimeError("bias must hold one value per vocabulary entry, in the type of h or fp32")
    if torch.is_grad_enabled() and (h.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad)):
        raise RuntimeError("joint_token_logprobs has no gradient: call it under torch.no_grad(), or use "
                           "token_logprobs on stored logits")
    M = _check_tokens(tokens, R, dev)
    top_k = _check_top_k(top_k, V)
    status = _new_status(dev) if validate else None
    logprobs, ent, lse, top, index = _score_buffers(R, M, top_k, entropy, dev)
    nbytes = _lib.load().cwr_joint_token_logprobs_workspace_bytes(R, V)
    work = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    _call("cwr_joint_token_logprobs", dev, h.data_ptr(), weight.data_ptr(), _ptr(bias),
          _DTYPES[bias.dtype] if bias is not None else _lib.F32, _DTYPES[h.dtype], R, H, V, _ptr(tokens), M, top_k,
          temperature, _ptr(logprobs), _ptr(ent), lse.data_ptr(), _ptr(top), _ptr(index), work.data_ptr(), nbytes,
          _ptr(status))
    if validate:
        _raise_on_status(status, "joint_token_logprobs")
    if tokens is not None and tokens.dim() == 1:
        logprobs = logprobs.view(R)
    return TokenScores(logprobs, ent, lse, top, index)


def _run_distill(x, top, index, temperature, tail, reduction, status, keep):
    """Binding of cwr_distill: (loss, stat)."""
    R, V = x.shape
    dev = x.device
    # what the backward pass needs and, under a reduction, its workspace and the rows' losses
    work_floats = _lib.load().cwr_distill_workspace_bytes() // 4
    buf = torch.empty(4 * R + (work_floats + R if reduction != "none" else 0), dtype=torch.float32, device=dev)
    base = buf.data_ptr()
    total = mean = work = None
    if reduction == "none":
        loss = torch.empty(R, dtype=torch.float32, device=dev)
        rows = loss.data_ptr()
    else:
        loss = torch.empty((), dtype=torch.float32, device=dev)
        work, rows = base + 16 * R, base + 16 * R + 4 * work_floats
        total, mean = (loss.data_ptr(), None) if reduction == "sum" else (None, loss.data_ptr())
    _call("cwr_distill", dev, x.data_ptr(), _DTYPES[x.dtype], R, V, x.stride(0), top.data_ptr(), index.data_ptr(),
          index.size(1), temperature, int(tail), rows, base if keep else None, total, mean, work, _ptr(status))
    return loss, buf


class _Distill(torch.autograd.Function):
    @staticmethod
    def forward(ctx: Any, x, top, index, temperature, tail, reduction, status):
        loss, stat = _run_distill(x, top, index, temperature, tail, reduction, status, True)
        ctx.temperature, ctx.tail, ctx.reduction = temperature, tail, reduction
        ctx.save_for_backward(x, top, index, stat)
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx: Any, grad_out):
        x, top, index, stat = ctx.saved_tensors
        R, V = x.shape
        go = _rows_f32(grad_out)
        stride = 1 if ctx.reduction == "none" else 0
        scale = 1.0 / R if ctx.reduction == "mean" and R else 1.0
        dx = torch.empty((R, V), dtype=x.dtype, device=x.device)
        _call("cwr_distill_backward", x.device, x.data_ptr(), _DTYPES[x.dtype], R, V, x.stride(0), top.data_ptr(),
              index.data_ptr(), index.size(1), ctx.temperature, int(ctx.tail), stat.data_ptr(), go.data_ptr(), stride,
              scale, dx.data_ptr())
        return dx, None, None, None, None, None, None


def distill_loss(x: torch.Tensor, top_logits: torch.Tensor, top_index: torch.Tensor, *, temperature: float = 1.0,
                 tail: bool = False, reduction: Optional[str] = "mean", validate: bool = False) -> torch.Tensor:
    """temperature^2 * KL(teacher || student) per row, the student's softmax(x / temperature) against a teacher of
    which only the K best entries of a row are known.

    x           (R, V) student logits, as for token_logprobs
    top_logits  (R, K) the teacher's values, top_index (R, K) int32 the entries they belong to, K <= 64;
                an index of -1 is absent, a row whose list is empty has loss 0 and gradient 0 whatever x holds
    tail        False: the teacher is softmax(top_logits / temperature) over the list.
                True: top_logits are log-probabilities at this temperature (token_logprobs(...,
                temperature=temperature).top_logprobs); the mass they leave is one more class, compared
                with the student's mass outside the list
    reduction   "mean" over the rows, "sum", or "none" / None for one loss per row
    validate    read the status word back (one synchronisation) and raise when an index lies outside
                [-1, V); without it the loss of such a row is NaN and its gradient 0

    A listed entry that the student has at -inf makes the loss infinite; the gradient takes its p as 0.

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
    reduction = reduction or "none"
    top = _rows_f32(top_logits.detach())
    if x.requires_grad and torch.is_grad_enabled():
        loss = _Distill.apply(x, top, top_index.contiguous(), temperature, bool(tail), reduction, status)
    else:
        loss, _ = _run_distill(x, top, top_index.contiguous(), temperature, bool(tail), reduction, status, False)
    if validate:
        _raise_on_status(status, "distill_loss")
    return loss


def lattice_tokens(lx: torch.Tensor, y: torch.Tensor, ly: torch.Tensor, total_rows: int, V: int,
                   blank: int = 0) -> torch.Tensor:
    """(total_rows, 2) int32: the blank and the label of every compact row, -1 where a row has no label (the
    last label position of a sequence, or a label outside [0, V)) or belongs to no sequence: the `tokens` under which token_logprobs
    returns the pair of log-probabilities the loss walks on.

    lx, ly, y as for transducer_loss; total_rows = sum_i lx_i*(ly_i+1)."""
    for name, t in (("lx", lx), ("y", y), ("ly", ly)):
        if not t.is_cuda or t.dtype != torch.int32 or not t.is_contiguous():
            raise RuntimeError(f"{name} must be a contiguous CUDA int32 tensor")
        if t.device != lx.device:
            raise RuntimeError(f"{name} must be on the device of lx")
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
