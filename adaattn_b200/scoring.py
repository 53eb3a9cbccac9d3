"""Log probabilities of given tokens, with entropy and top alternatives.

``token_logprobs`` reads the logits once (``ada_token_logprobs``) and writes a
few numbers per row, where log_softmax, its entropy and topk would each write
or read the whole vocabulary; its gradient reads them once more and writes
theirs (``ada_token_logprobs_bwd``).
"""

from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _lib
from .config import ShapeError
from .paged import _call, _device_of, _no_tangent


class TokenLogprobs(NamedTuple):
    """Per row of logits, float32 except top_tokens (int64); the last two are
    None without alternatives and carry no gradient."""

    logprobs: torch.Tensor
    entropy: torch.Tensor
    lse: torch.Tensor
    top_logprobs: Optional[torch.Tensor]
    top_tokens: Optional[torch.Tensor]


def _rows3(t: torch.Tensor) -> torch.Tensor:
    """[..., V] as [A, R, V] with a unit innermost stride, a view wherever the layout allows."""
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        t = t.contiguous()
    if t.dim() == 1:
        return t[None, None]
    if t.dim() == 2:
        return t[None]
    if t.dim() == 3:
        return t
    return t.reshape(t.shape[0], t.shape[1:-1].numel(), t.shape[-1])


def _grad_like(z3: torch.Tensor) -> torch.Tensor:
    """An empty tensor of z3's shape whose rows start like z3's relative to 32
    bytes, so that both are read and written in the same vectors. Rows of
    vocabulary-sized views (a padded matrix) stay padded in memory."""
    a, r, v = z3.shape
    unit = 32 // z3.element_size()
    ld = z3.stride(1) if r > 1 else z3.stride(0) if a > 1 else v
    if ld < v or ld > v + 1024 or (a > 1 and r > 1 and z3.stride(0) % unit != (r * ld) % unit):
        ld = (v + unit - 1) // unit * unit
    return torch.empty(a, r, ld, dtype=z3.dtype, device=z3.device)[..., :v]


def _forward(z3: torch.Tensor, tokens: torch.Tensor, top_k: int, ignore_index: int, with_stats: bool = False):
    """Each output in memory of its own: views of one buffer would share a
    version counter, and autograd refuse to change one in place beside another."""
    dev = z3.device
    rows = z3.shape[0] * z3.shape[1]
    lp = torch.empty(rows, dtype=torch.float32, device=dev)
    ent, lse = lp.new_empty(rows), lp.new_empty(rows)
    stats = lp.new_empty(rows, 2) if with_stats else None
    top_lp = torch.empty(rows, top_k, dtype=torch.float32, device=dev) if top_k else None
    top_id = torch.empty(rows, top_k, dtype=torch.int64, device=dev) if top_k else None
    _call("ada_token_logprobs", dev, _lib.load().ada_token_logprobs, _lib.packed(z3), _lib.packed(tokens),
          int(ignore_index), int(top_k), lp.data_ptr(), ent.data_ptr(), lse.data_ptr(), _lib.ptr(stats),
          _lib.ptr(top_lp), _lib.ptr(top_id))
    return lp, ent, lse, top_lp, top_id, stats


def token_logprobs_backward(logits: torch.Tensor, tokens: torch.Tensor, stats: torch.Tensor, entropy: torch.Tensor,
                            grad_logprobs: Optional[torch.Tensor] = None,
                            grad_entropy: Optional[torch.Tensor] = None, grad_lse: Optional[torch.Tensor] = None, *,
                            ignore_index: int = -100) -> torch.Tensor:
    """Gradient with respect to logits [A, R, V] (``ada_token_logprobs_bwd``):
    ``stats`` [A * R, 2] (row maximum and log of the sum of exp(z - maximum))
    and ``entropy`` as the forward computed them, upstream gradients [A * R]
    or None. Rows of a vocabulary that is no multiple of 16 bytes keep the
    logits' padding in memory."""
    if logits.dim() != 3:
        raise ShapeError(f"logits must be 3-D [A, R, V], got {logits.dim()}-D")
    rows = logits.shape[0] * logits.shape[1]
    ups = [None if g is None else g.float().contiguous() for g in (grad_logprobs, grad_entropy, grad_lse)]
    for name, t, shape in (("stats", stats, (rows, 2)), ("entropy", entropy, (rows,)), ("grad_logprobs", ups[0], (rows,)),
                           ("grad_entropy", ups[1], (rows,)), ("grad_lse", ups[2], (rows,))):
        if t is not None and (t.shape != shape or t.dtype != torch.float32):
            raise ShapeError(f"{name} must be float32 {list(shape)}, got {t.dtype} {list(t.shape)}")
    stats, entropy = stats.contiguous(), entropy.contiguous()
    dev = _device_of(logits, tokens, stats, entropy, *ups)
    _no_tangent("token_logprobs_backward", logits, stats, entropy, *ups)
    grad = _grad_like(logits)
    _call("ada_token_logprobs_bwd", dev, _lib.load().ada_token_logprobs_bwd, _lib.packed(logits),
          _lib.packed(tokens), int(ignore_index), stats.data_ptr(), entropy.data_ptr(),
          *(_lib.ptr(g) or None for g in ups), _lib.packed(grad))
    return grad


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, top_k, ignore_index):
        z3 = _rows3(logits)
        lp, ent, lse, top_lp, top_id, stats = _forward(z3, tokens, top_k, ignore_index, with_stats=True)
        ctx.save_for_backward(logits, tokens, stats, ent)
        ctx.ignore_index = ignore_index
        ctx.set_materialize_grads(False)
        if top_k:
            ctx.mark_non_differentiable(top_lp, top_id)
        return lp, ent, lse, top_lp, top_id

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g_lp, g_ent, g_lse, *_):
        if g_lp is None and g_ent is None and g_lse is None:
            return None, None, None, None
        logits, tokens, stats, ent = ctx.saved_tensors
        grad = token_logprobs_backward(_rows3(logits), tokens, stats, ent, g_lp, g_ent, g_lse,
                                       ignore_index=ctx.ignore_index)
        return (grad[0] if logits.dim() == 2 else grad.reshape(logits.shape)), None, None, None


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, *, top_k: int = 0,
                   ignore_index: int = -100) -> TokenLogprobs:
    """Scores of given tokens under softmax(logits) (``ada_token_logprobs``).

    logits [..., V] (fp32, fp16 or bf16; rows of any stride and alignment),
    tokens [...] int64 or int32. Per row: ``logprobs``, the log probability
    of the token (0 where it is ``ignore_index``, NaN where it is outside the
    vocabulary, which the library's status word records too); ``entropy`` and
    ``lse`` of the distribution; with ``top_k`` (up to 64) the largest log
    probabilities in order and their tokens, equal logits by lowest token.
    All arithmetic is fp32. A logit of -inf has probability 0; a row of
    nothing else, or one with +inf or NaN, gives NaN.

    logprobs, entropy and lse are differentiable with respect to the logits
    (once, in reverse mode; dual tensors are refused); the gradient has their dtype. An entropy gradient reaches ignored
    rows too.
    """
    dev = _device_of(logits, tokens)
    _no_tangent("token_logprobs", logits)
    if logits.dim() < 1:
        raise ShapeError("logits must be [..., V]")
    if logits.dtype not in (torch.float32, torch.float16, torch.bfloat16):
        raise TypeError(f"logits must be fp32, fp16 or bf16, got {logits.dtype}")
    if tokens.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"tokens must be int64 or int32, got {tokens.dtype}")
    lead = logits.shape[:-1]
    if tokens.shape != lead:
        raise ShapeError("tokens must have one entry per row of logits", expected_shape=tuple(lead),
                         actual_shape=tuple(tokens.shape))
    top_k = int(top_k)
    if not 0 <= top_k <= 64:
        raise ValueError(f"top_k must be in [0, 64], got {top_k}")
    if top_k > logits.shape[-1]:
        raise ValueError(f"top_k {top_k} exceeds the vocabulary of {logits.shape[-1]}")
    flat = tokens.reshape(-1)
    if not flat.is_contiguous():
        flat = flat.contiguous()
    if torch.is_grad_enabled() and logits.requires_grad:
        lp, ent, lse, top_lp, top_id = _TokenLogprobs.apply(logits, flat, top_k, int(ignore_index))
    else:
        lp, ent, lse, top_lp, top_id, _ = _forward(_rows3(logits), flat, top_k, int(ignore_index))
    if logits.dim() != 2:
        lp, ent, lse = lp.reshape(lead), ent.reshape(lead), lse.reshape(lead)
        if top_k:
            top_lp, top_id = top_lp.reshape(*lead, top_k), top_id.reshape(*lead, top_k)
    return TokenLogprobs(lp, ent, lse, top_lp, top_id)


__all__ = ["token_logprobs", "token_logprobs_backward", "TokenLogprobs"]
