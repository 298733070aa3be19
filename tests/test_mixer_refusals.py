"""CPU tests of what exl3_head_norm, exl3_delta_rule and exl3_sample refuse before anything is
launched, through the C ABI (pointers that are never read) and through the Python entry points."""
import ctypes as C
import math

import pytest
import torch

from exl3_amd import _lib
from exl3_amd._lib import DeltaConfig, DeltaRows, HeadNormConfig, HeadRows, SampleConfig
from exl3_amd.delta import delta_rule
from exl3_amd.heads import head_norm
from exl3_amd.sampling import sample_tokens

INVALID, UNSUPPORTED, WORKSPACE = _lib.EXL3_ERR_INVALID, _lib.EXL3_ERR_UNSUPPORTED, _lib.EXL3_ERR_WORKSPACE


def with_(s, **kw):
    """A copy of a ctypes structure with some fields changed."""
    c = type(s).from_buffer_copy(s)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


HEADS = HeadNormConfig(0, 0, 128, 64, 0, 1e-6)
Q = HeadRows(0x100000, None, 0x200000, 4, 512, 128, 512, 128)
K = HeadRows(0x300000, 0x900000, 0x400000, 2, 256, 128, 256, 128)


def heads(cfg=HEADS, q=Q, k=K, tokens=8, pos=0x500000, inv=0x600000):
    L = _lib.lib()
    return L.exl3_head_norm(C.byref(cfg) if cfg else None, C.byref(q) if q else None, C.byref(k) if k else None, tokens,
                            pos, inv, None)


def test_head_norm_refusals():
    assert heads(cfg=None) == heads(q=None) == INVALID
    assert heads(cfg=with_(HEADS, dtype=2)) == heads(cfg=with_(HEADS, head_dim=0)) == UNSUPPORTED
    assert heads(cfg=with_(HEADS, head_dim=1025)) == UNSUPPORTED
    for bad in (dict(mode=2), dict(rotate_dims=130), dict(rotate_dims=63), dict(rotate_dims=-2), dict(eps=-1.0),
                dict(eps=math.nan)):
        assert heads(cfg=with_(HEADS, **bad)) == INVALID, bad
    assert heads(tokens=-1) == heads(tokens=2 ** 31) == INVALID
    for bad in (dict(heads=0), dict(heads=40000), dict(x=None), dict(y=None), dict(x=0x100001), dict(y_head=64),
                dict(y_token=511), dict(x_token=-512), dict(x_head=2 ** 40)):
        assert heads(q=with_(Q, **bad)) == INVALID, bad
    assert heads(pos=None) == heads(inv=None) == heads(pos=0x500002) == INVALID
    # outputs on inputs, on each other, on a weight
    for bad in (dict(y=0x100000 + 2), dict(y=0x100000, y_token=1024), dict(y=0x300000), dict(y=0x400000 + 4096 - 2),
                dict(y=0x900000)):
        assert heads(q=with_(Q, **bad)) == INVALID, bad
        assert b"overlap" in _lib.lib().exl3_last_error()
    # parts of one packed row may be in place; a part one value into the next may not
    packed = dict(x_token=1024, y_token=1024)
    q = with_(Q, x=0x100000, y=0x100000, **packed)
    k = with_(K, x=0x100000 + 1024 - 2, y=0x100000 + 1024 - 2, **packed)
    assert heads(q=q, k=k) == INVALID and b"overlap" in _lib.lib().exl3_last_error()
    # on the positions and frequencies; spans that 64 bits would not hold
    assert heads(pos=0x200000) == heads(inv=0x400000 + 8) == INVALID and b"positions" in _lib.lib().exl3_last_error()
    assert heads(q=with_(Q, x_token=2 ** 36), tokens=2 ** 31 - 1) == heads(q=with_(Q, y_token=2 ** 33), tokens=2 ** 20) == INVALID
    assert b"stride" in _lib.lib().exl3_last_error()
    assert heads(tokens=0) == _lib.EXL3_OK


DELTA = DeltaConfig(0, 2, 4, 128, 64, 1, 0.1)
ROWS = DeltaRows(0x10000000, 0x11000000, 0x12000000, 0x13000000, 0x14000000, 0x15000000, 256, 256, 256, 512, 4, 256)


def delta(cfg=DELTA, x=ROWS, tokens=64, starts=0x16000000, n=2, state=0x20000000, slots=3, src=None, dst=None,
          ws=0x30000000, nbytes=1 << 40):
    return _lib.lib().exl3_delta_rule(C.byref(cfg) if cfg else None, C.byref(x) if x else None, tokens, starts, n, state,
                                      slots, src, dst, ws, nbytes, None)


def test_delta_rule_refusals():
    assert delta(cfg=None) == delta(x=None) == INVALID
    for bad in (dict(dtype=2), dict(dk=32), dict(dk=96), dict(dv=8), dict(dv=65), dict(dv=272)):
        assert delta(cfg=with_(DELTA, **bad)) == UNSUPPORTED, bad
    for bad in (dict(heads_qk=0), dict(heads_qk=3), dict(heads_v=0), dict(heads_v=8192)):
        assert delta(cfg=with_(DELTA, **bad)) == INVALID, bad
    assert delta(tokens=-1) == delta(tokens=2 ** 31) == delta(n=-1) == delta(n=70000) == INVALID
    assert delta(starts=None, n=3) == INVALID and b"divide" in _lib.lib().exl3_last_error()
    assert delta(slots=0) == delta(state=None) == delta(state=0x20000004) == delta(starts=0x16000002) == INVALID
    for bad in (dict(q=None), dict(out=None), dict(q=0x10000001), dict(g=0x13000002), dict(q_token=255), dict(g_token=128),
                dict(out_token=255), dict(beta_token=3)):
        assert delta(x=with_(ROWS, **bad)) == INVALID, bad
    for bad in (dict(out=0x12000000), dict(out=0x10000000 + 100), dict(v=0x20000000), dict(out=0x20000000 + 64)):
        assert delta(x=with_(ROWS, **bad)) == INVALID and b"overlap" in _lib.lib().exl3_last_error(), bad
    # what a launch does not hold: tokens, heads of all sequences
    assert delta(tokens=2 ** 27 + 1) == delta(tokens=2 ** 20, cfg=with_(DELTA, heads_v=32), n=32769) == INVALID
    assert b"value heads" in _lib.lib().exl3_last_error()
    # the workspace on rows or the state
    for ws in (0x10000000, 0x13000000, 0x15000000 + 0x100, 0x20000000):
        assert delta(ws=ws) == INVALID and b"workspace" in _lib.lib().exl3_last_error(), hex(ws)
    assert delta(n=0) == _lib.EXL3_OK
    size = _lib.lib().exl3_delta_workspace_size
    assert size(C.byref(with_(DELTA, dk=32)), 64, 2) == 0
    # prefills need a workspace, single tokens none
    need = size(C.byref(DELTA), 64, 2)
    assert need > 0 and size(C.byref(DELTA), 64, 64) == 0
    assert delta(nbytes=need - 1) == delta(ws=None) == delta(ws=0x30000080) == WORKSPACE


SAMPLE = SampleConfig(dtype=0, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0)


def sample(cfg=SAMPLE, logits=0x1000, rows=2, vocab=100, stride=100, u=0x2000, ids=0x3000, probs=None, ws=0x100000,
           nbytes=1 << 30):
    return _lib.lib().exl3_sample(C.byref(cfg) if cfg else None, logits, rows, vocab, stride, u, ids, probs, ws, nbytes, None)


def test_sample_refusals():
    assert sample(cfg=None) == sample(logits=None) == sample(u=None) == sample(ids=None) == INVALID
    assert sample(cfg=with_(SAMPLE, dtype=3)) == UNSUPPORTED
    assert sample(rows=-1) == sample(rows=65536) == sample(vocab=0) == sample(vocab=2 ** 19 + 1, stride=2 ** 20) == INVALID
    assert sample(stride=99) == sample(logits=0x1001) == sample(u=0x2002) == sample(ids=0x3001) == sample(probs=0x4002) == INVALID
    assert sample(cfg=with_(SAMPLE, top_ks=0x5002)) == sample(cfg=with_(SAMPLE, dtype=2), logits=0x1002) == INVALID
    assert sample(stride=0) == sample(stride=-100) == INVALID
    need = _lib.lib().exl3_sample_workspace_size(2, 100)
    assert need > 0 and _lib.lib().exl3_sample_workspace_size(0, 100) == 0
    for bad in (dict(ids=0x1000), dict(ids=0x2004), dict(probs=0x3004), dict(ids=0x100100), dict(ws=0x1000), dict(logits=0x100000 - 4),
                dict(probs=0x1000 + 396)):
        assert sample(**bad) == INVALID and b"overlap" in _lib.lib().exl3_last_error(), bad
    assert sample(nbytes=need - 1) == sample(ws=None) == sample(ws=0x100080) == WORKSPACE
    assert sample(rows=0) == _lib.EXL3_OK


def test_python_refusals():
    h = lambda *s, dt=torch.float16: torch.zeros(s, dtype=dt)  # noqa: E731
    q, k = h(4, 2, 64), h(4, 1, 64)
    pos, inv = h(4, dt=torch.int32), h(16, dt=torch.float32)
    for bad in (lambda: head_norm(q, k, mode="layer"), lambda: head_norm(q.float()), lambda: head_norm(q, h(3, 1, 64)),
                lambda: head_norm(q, h(4, 1, 32)), lambda: head_norm(q, k, positions=pos), lambda: head_norm(q, k, inv_freq=inv),
                lambda: head_norm(q, k_out=k), lambda: head_norm(q, k, positions=pos.long(), inv_freq=inv),
                lambda: head_norm(q, k, positions=pos[:3], inv_freq=inv), lambda: head_norm(q, k, positions=pos, inv_freq=h(33, dt=torch.float32)),
                lambda: head_norm(q, k.bfloat16()), lambda: head_norm(q.transpose(1, 2)), lambda: head_norm(q, q_weight=h(32)),
                lambda: head_norm(q, q_out=h(4, 2, 32))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(ValueError, match="device"):
        head_norm(q, k)
    d = dict(q=h(6, 2, 64), k=h(6, 2, 64), v=h(6, 4, 32), g=h(6, 4, 64, dt=torch.float32), beta=h(6, 4, dt=torch.float32),
             state=h(3, 4, 64, 32, dt=torch.float32))
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    for bad in (dict(q=h(6, 2, 64, dt=torch.float32)), dict(k=h(6, 1, 64)), dict(v=h(5, 4, 32)), dict(g=h(6, 4)),
                dict(g=h(6, 4, 32, dt=torch.float32)), dict(beta=h(6, 2, dt=torch.float32)), dict(state=h(3, 4, 64, 32)),
                dict(state=h(4, 64, 32, dt=torch.float32)), dict(starts=i32(0, 6).long()), dict(starts=i32()),
                dict(starts=i32(0, 6), slots=i32(0, 1)), dict(slots=i32(0, 1, 2, 0)), dict(dst=i32(0, 1)),
                dict(out=h(6, 4, 64)), dict(q=h(6, 64, 2).transpose(1, 2))):
        with pytest.raises(ValueError):
            delta_rule(**{**d, **bad})
    with pytest.raises(ValueError, match="device"):
        delta_rule(**d)
    x, u = h(3, 50), h(3, dt=torch.float32)
    for bad in (dict(logits=h(50)), dict(logits=h(3, 50, dt=torch.float64)), dict(logits=h(50, 3).t()), dict(u=h(2, dt=torch.float32)),
                dict(u=u.double()), dict(temperature=h(3)), dict(top_k=h(3, dt=torch.int64)), dict(top_p=h(2, dt=torch.float32)),
                dict(ids=h(3, dt=torch.int64)), dict(probs=h(3))):
        with pytest.raises(ValueError):
            sample_tokens(**{**dict(logits=x, u=u), **bad})
    with pytest.raises(ValueError, match="device"):
        sample_tokens(x, u)
