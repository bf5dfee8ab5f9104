"""Verification of drafted tokens (speculative decoding): which of them stand
against the target model's probabilities, and the token that follows.

The reference has nothing of this kind.  ``generate.generate_paged`` drafts and
verifies with it; the target's probabilities of all drafted tokens come from one
model call, whose attention is ``PagedLayer.attend_tokens``."""

import torch

from . import _lib
from ._lib import check, dtype_code, ptr
from .ext import _require_device
from .paged import _call, _lens, _on, _pack_rows


def _probabilities(index, name, t, shape, dtype=None):
    """(B, n, V) tensor as C rows, copied only where its last dimension is
    strided -> (rows, tensor)."""
    _on(index, name, t)
    if t.dim() != 3 or tuple(t.shape) != shape or (dtype is not None and t.dtype != dtype):
        raise ValueError(f"{name} must be {shape}{f' {dtype}' if dtype is not None else ''}, got {tuple(t.shape)} {t.dtype}")
    if t.stride(2) != 1 and shape[2] > 1:
        t = t.contiguous()
    return _pack_rows(t.data_ptr(), t.stride(0), 0, t.stride(1)), t


def verify_drafts(target, draft, tokens, uniforms, n_draft=None):
    """How many of K <= 63 drafted tokens of each sequence stand, and the token
    that follows them -> (out (B, K + 1) of the tokens' type: the accepted tokens,
    the next one, then -1; accepted (B,) int32).

    ``target`` (B, K + 1, V) fp32, fp16 or bf16: the target's probabilities after
    i drafted tokens.  ``draft`` (B, K, V) of the same type: the probabilities that
    token i was drawn from, or None where tokens were not drawn (the largest one, a
    copy of earlier text).  ``tokens`` (B, K) int32 or int64, ``uniforms`` (B, K +
    1) fp32 random numbers in [0, 1), ``n_draft`` (B,) int32 on the device: only
    the first n_draft[b] tokens were drafted (default: all).

    Token i stands while uniforms[b, i] * draft(token) < target(token); one outside
    the vocabulary does not.  The next one is the first at which the running sum of
    the weights exceeds uniforms[b, K] times their sum, the weights being
    max(target - draft, 0) after a refused token (the target's own where that
    leaves nothing) and the target's after the last one: so tokens are distributed
    as the target's own.  It is -1 where the sum is not a positive number.
    Probabilities need not sum to one."""
    done = _lib.calls().verify(target, draft, tokens, uniforms, n_draft)
    if done is not NotImplemented:
        return done
    if not isinstance(target, torch.Tensor):
        raise TypeError(f"target must be a tensor, got {type(target).__name__}")
    _require_device(target)
    index = target.get_device()
    if target.dim() != 3 or target.shape[1] < 1 or target.shape[2] < 1:
        raise ValueError(f"target must be (B, K + 1, V), got {tuple(target.shape)}")
    B, K, V = target.shape[0], target.shape[1] - 1, target.shape[2]
    code = dtype_code(target.dtype)
    t_rows, t_held = _probabilities(index, "target", target, (B, K + 1, V))
    d_rows = None
    if draft is not None:
        d_rows, d_held = _probabilities(index, "draft", draft, (B, K, V), target.dtype)
    _on(index, "tokens", tokens)
    if tokens.dtype not in (torch.int32, torch.int64) or tokens.shape != (B, K):
        raise TypeError(f"tokens must be an int32 or int64 tensor of shape {(B, K)}, got {tuple(tokens.shape)} {tokens.dtype}")
    _on(index, "uniforms", uniforms)
    if uniforms.dtype != torch.float32 or uniforms.shape != (B, K + 1):
        raise TypeError(f"uniforms must be a float32 tensor of shape {(B, K + 1)}, got {tuple(uniforms.shape)} {uniforms.dtype}")
    tokens, uniforms = tokens.contiguous(), uniforms.contiguous()
    if n_draft is not None:
        n_draft = _lens("n_draft", n_draft, B, index)
    out = torch.empty((B, K + 1), dtype=tokens.dtype, device=target.device)
    accepted = torch.empty(B, dtype=torch.int32, device=target.device)
    n = _lib.load().fkv_verify_drafts_workspace(B, K, V)
    if n < 0:
        check(n, "fkv_verify_drafts_workspace")
    ws = torch.empty(n, dtype=torch.uint8, device=target.device)
    _call(index, "fkv_verify_drafts", t_rows, d_rows, code, B, K, V, ptr(tokens), int(tokens.dtype == torch.int64),
          ptr(uniforms), None if n_draft is None else ptr(n_draft), ptr(out), ptr(accepted), ptr(ws), n)
    return out, accepted
