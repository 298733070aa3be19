"""The choice of the next token from the head's logits over the C ABI: temperature, top-k,
top-p and min-p from given random numbers. Device only; nothing is read back."""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib
from ._lib import SampleConfig, call
from .heads import ST_DTYPE, require, require_device, scratch, stream_on
from .trellis import _ptr


def sample_tokens(logits: torch.Tensor, u: torch.Tensor, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0,
                  ids: torch.Tensor | None = None, probs: torch.Tensor | None = None,
                  ws: torch.Tensor | None = None):
    """(ids (rows) i32, probs (rows) f32): one token for each row of logits (rows, vocab), f16,
    bf16 or f32 (rows apart from each other, so an expanded row is refused), from u (rows) f32 in [0, 1).

    In a row's order (largest logit first, equal ones by id) the first top_k are kept, of those
    the fewest that hold top_p of their weight, of those the ones with at least min_p times the
    largest weight; always the first. The token is the first whose running weight exceeds u
    times the kept weight, its probability its share of that. Each parameter is a number or a
    (rows) tensor (f32; top_k i32); temperature <= 0 takes the largest logit, top_k <= 0, top_p
    >= 1 and min_p <= 0 keep all. -inf and NaN logits are never taken: a row without others
    gets id -1."""
    if logits.dim() != 2 or logits.dtype not in ST_DTYPE or (logits.shape[1] > 1 and logits.stride(1) != 1):
        raise ValueError("sample_tokens: logits must be (rows, vocab) with adjacent values, f16, bf16 or f32")
    dev, (rows, vocab) = logits.device, logits.shape
    require(u, "sample_tokens: u", torch.float32, (rows,), dev)
    cfg = SampleConfig(dtype=ST_DTYPE[logits.dtype])
    for name, value, dtype in (("temperature", temperature, torch.float32), ("top_k", top_k, torch.int32),
                               ("top_p", top_p, torch.float32), ("min_p", min_p, torch.float32)):
        if isinstance(value, torch.Tensor):
            require(value, f"sample_tokens: {name}", dtype, (rows,), dev)
            setattr(cfg, name + "s", value.data_ptr())
        else:
            setattr(cfg, name, value)
    if ids is None:
        ids = torch.empty(rows, dtype=torch.int32, device=dev)
    if probs is None:
        probs = torch.empty(rows, dtype=torch.float32, device=dev)
    require(ids, "sample_tokens: ids", torch.int32, (rows,), dev)
    require(probs, "sample_tokens: probs", torch.float32, (rows,), dev)
    require_device(logits, "sample_tokens")
    need = _lib.lib().exl3_sample_workspace_size(rows, vocab)
    ws = scratch(ws, need, dev, "sample_tokens")
    call("exl3_sample", C.byref(cfg), logits.data_ptr(), rows, vocab, logits.stride(0) if rows > 1 else vocab, u.data_ptr(),
         ids.data_ptr(), probs.data_ptr(), _ptr(ws), 0 if ws is None else ws.numel(), stream_on(dev))
    return ids, probs
