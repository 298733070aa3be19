"""The gated delta rule over the C ABI: the token mixer's state, updated and read token by
token for decode and verify steps and in chunks for prefills, any mix of lengths in a call.
Device only."""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib
from ._lib import DeltaConfig, DeltaRows, call
from .heads import ST_DTYPE, require, require_device, scratch, stream_on
from .trellis import _ptr


def _rows(t: torch.Tensor, what: str, dtype, shape, device) -> int:
    """Token stride of (tokens, heads[, size]) rows whose tokens are contiguous blocks."""
    if t.dtype != dtype or t.shape != shape or t.device != device:
        raise ValueError(f"delta_rule: {what} must be a {dtype} tensor of shape {tuple(shape)} on {device}")
    strides = t.stride()
    if strides[1:] != ((shape[2], 1) if len(shape) == 3 else (1,)):
        size = 1
        for n, stride in zip(shape[:0:-1], strides[:0:-1]):  # (a size of 1 may have any stride)
            if stride != size and n > 1:
                raise ValueError(f"delta_rule: a token's {what} must be contiguous")
            size *= n
    return strides[0]


def _config(q, v, g, scale) -> DeltaConfig:
    return DeltaConfig(ST_DTYPE[q.dtype], q.shape[1], v.shape[1], q.shape[2], v.shape[2], int(g.dim() == 3),
                       q.shape[2] ** -0.5 if scale is None else scale)


def delta_rule(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, beta: torch.Tensor,
               state: torch.Tensor, *, starts: torch.Tensor | None = None, slots: torch.Tensor | None = None,
               dst: torch.Tensor | None = None, scale: float | None = None, out: torch.Tensor | None = None,
               ws: torch.Tensor | None = None) -> torch.Tensor:
    """S <- diag(exp(g)) S; u = beta (v - S^T k); S <- S + k u^T; out = scale S^T q, for every
    token in turn.

    q, k (T, heads_qk, dk) and v (T, heads_v, dv), f16 or bf16 (slices of packed rows work);
    g (T, heads_v) or (T, heads_v, dk) and beta (T, heads_v) f32; state (n_slots, heads_v, dk,
    dv) f32, updated in place. starts (n + 1) i32 are the sequences' first tokens (and the
    end; None: equal lengths, one sequence without slots either); slots (n) i32 each one's
    slot (None: sequence i has slot i), dst (n) i32 where its last state goes instead of its
    slot. A slot outside the state starts from zeros and stores nothing; one named by more
    than one sequence keeps its old state. scale: 1 / sqrt(dk) unless given."""
    if q.dim() != 3 or v.dim() != 3 or g.dim() not in (2, 3) or q.dtype not in (torch.float16, torch.bfloat16):
        raise ValueError("delta_rule: q and v must be (tokens, heads, size) in float16 or bfloat16, g (tokens, heads[, dk])")
    dev, dtype, (T, Hk, dk), (_, Hv, dv) = q.device, q.dtype, q.shape, v.shape
    if starts is not None and (starts.dim() != 1 or starts.numel() < 1):
        raise ValueError("delta_rule: starts must be (sequences + 1) int32")
    n = starts.numel() - 1 if starts is not None else 1 if slots is None else slots.numel()
    if starts is None and (T % n if n else T):
        raise ValueError("delta_rule: without starts the tokens must divide into the sequences")
    if state.dim() != 4:
        raise ValueError("delta_rule: state must be (slots, heads_v, dk, dv)")
    n_slots = state.shape[0]
    require(state, "delta_rule: state", torch.float32, (n_slots, Hv, dk, dv), dev)
    if starts is not None:
        require(starts, "delta_rule: starts", torch.int32, (n + 1,), dev)
    if slots is not None:
        require(slots, "delta_rule: slots", torch.int32, (n,), dev)
    if dst is not None:
        require(dst, "delta_rule: dst", torch.int32, (n,), dev)
    qk_shape, v_shape, g_shape = (T, Hk, dk), (T, Hv, dv), (T, Hv, dk) if g.dim() == 3 else (T, Hv)
    if out is None:
        out = v.new_empty(v_shape)
    x = DeltaRows(q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(), beta.data_ptr(), out.data_ptr(),
                  _rows(q, "q", dtype, qk_shape, dev), _rows(k, "k", dtype, qk_shape, dev), _rows(v, "v", dtype, v_shape, dev),
                  _rows(g, "g", torch.float32, g_shape, dev), _rows(beta, "beta", torch.float32, (T, Hv), dev),
                  _rows(out, "out", dtype, v_shape, dev))
    cfg = DeltaConfig(ST_DTYPE[dtype], Hk, Hv, dk, dv, len(g_shape) - 2, dk ** -0.5 if scale is None else scale)
    require_device(q, "delta_rule")
    need = _lib.lib().exl3_delta_workspace_size(C.byref(cfg), T, n)
    ws = scratch(ws, need, dev, "delta_rule")
    call("exl3_delta_rule", C.byref(cfg), C.byref(x), T, _ptr(starts), n, state.data_ptr(), n_slots,
         _ptr(slots), _ptr(dst), _ptr(ws), 0 if ws is None else ws.numel(), stream_on(dev))
    return out
