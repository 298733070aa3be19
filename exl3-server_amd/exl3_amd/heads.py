"""The norm of query and key heads with the position rotation behind it, over the C ABI.

head_norm(q, k) takes slices of a packed qkv row in place: only the values of a head have to
be adjacent. Serves the L2 norm of the delta rule's queries and keys (mode "l2"), and the
RMSNorm with weights and rotation of attention's (mode "rms"). Device only.
"""
from __future__ import annotations

import ctypes as C

import torch

from ._lib import NORM_L2, NORM_RMS, HeadNormConfig, HeadRows, call
from .trellis import _stream, _workspace

ST_DTYPE = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}  # exl3_st_dtype
MODES = {"rms": NORM_RMS, "l2": NORM_L2}


def require(t: torch.Tensor, what: str, dtype, shape, device) -> None:
    """t is a contiguous tensor of this dtype and shape on this device."""
    if t.dtype != dtype or t.shape != shape or not t.is_contiguous() or t.device != device:
        raise ValueError(f"{what} must be a contiguous {dtype} tensor of shape {tuple(shape)} on {device}")


# the current stream's handle of a device, without a Stream object for each call
_raw_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else None


def stream_on(device) -> int:
    return _raw_stream(device.index) if _raw_stream is not None else _stream()


def require_device(t: torch.Tensor, what: str) -> None:
    """t lives on the current GPU, whose stream and launches a call uses."""
    if t.device.type != "cuda" or t.device.index != torch.cuda.current_device():
        raise ValueError(f"{what}: tensors must be on the current device")


def scratch(ws: torch.Tensor | None, need: int, device, what: str) -> torch.Tensor | None:
    """The caller's workspace where it holds `need` bytes, else one of the allocator's (None for none)."""
    if ws is not None and (ws.device != device or ws.dtype != torch.uint8 or not ws.is_contiguous()):
        raise ValueError(f"{what}: ws must be a contiguous uint8 tensor on {device}")
    return _workspace(need, device) if need and (ws is None or ws.numel() < need) else ws


def _side(what, x, w, y, dtype, device):
    shape, xs, ys = x.shape, x.stride(), y.stride()
    if len(shape) != 3 or x.dtype != dtype or x.device != device or (shape[2] > 1 and xs[2] != 1):
        raise ValueError(f"head_norm: {what} must be (tokens, heads, head_dim) with adjacent values, of one dtype and device")
    if y.shape != shape or y.dtype != dtype or y.device != device or (shape[2] > 1 and ys[2] != 1):
        raise ValueError(f"head_norm: {what}'s output must have its shape, dtype and device")
    if w is not None:
        require(w, f"head_norm: {what}'s weight", dtype, (shape[2],), device)
    return HeadRows(x.data_ptr(), None if w is None else w.data_ptr(), y.data_ptr(), shape[1], xs[0], xs[1], ys[0], ys[1])


def head_norm(q: torch.Tensor, k: torch.Tensor | None = None, *, mode: str = "rms", eps: float = 1e-6,
              q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None,
              positions: torch.Tensor | None = None, inv_freq: torch.Tensor | None = None,
              interleaved: bool = False, q_out: torch.Tensor | None = None, k_out: torch.Tensor | None = None):
    """q (tokens, heads_q, d) and k (tokens, heads_k, d), f16 or bf16, normed over d and, given
    positions (tokens) i32 and inv_freq (R / 2) f32, rotated in their first R values. Returns
    (q_out, k_out) (or q_out alone without k); q_out=q, k_out=k work in place."""
    if mode not in MODES:
        raise ValueError("head_norm: mode must be 'rms' or 'l2'")
    if q.dtype not in (torch.float16, torch.bfloat16):
        raise ValueError("head_norm: q must be float16 or bfloat16")
    if q.dim() != 3 or (k is not None and (k.dim() != 3 or k.shape[0] != q.shape[0] or k.shape[2] != q.shape[2])):
        raise ValueError("head_norm: q and k must be (tokens, heads, head_dim) of the same tokens and head_dim")
    if (positions is None) != (inv_freq is None):
        raise ValueError("head_norm: the rotation needs both positions and inv_freq")
    if k is None and (k_weight is not None or k_out is not None):
        raise ValueError("head_norm: k_weight or k_out without k")
    T, _, d = q.shape
    rotate = 0
    if positions is not None:
        require(positions, "head_norm: positions", torch.int32, (T,), q.device)
        require(inv_freq, "head_norm: inv_freq", torch.float32, (inv_freq.numel(),), q.device)
        rotate = 2 * inv_freq.numel()
        if rotate > d:
            raise ValueError("head_norm: inv_freq has more than head_dim / 2 frequencies")
    q_out = torch.empty_like(q, memory_format=torch.contiguous_format) if q_out is None else q_out
    sides = [_side("q", q, q_weight, q_out, q.dtype, q.device)]
    if k is not None:
        k_out = torch.empty_like(k, memory_format=torch.contiguous_format) if k_out is None else k_out
        sides.append(_side("k", k, k_weight, k_out, q.dtype, q.device))
    require_device(q, "head_norm")
    cfg = HeadNormConfig(ST_DTYPE[q.dtype], MODES[mode], d, rotate, int(interleaved), eps)
    call("exl3_head_norm", C.byref(cfg), C.byref(sides[0]), C.byref(sides[1]) if k is not None else None, T,
         None if positions is None else positions.data_ptr(), None if inv_freq is None else inv_freq.data_ptr(), stream_on(q.device))
    return q_out if k is None else (q_out, k_out)
