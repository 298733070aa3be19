"""GPU tests of exl3_head_norm against its formula in 64 bits (tolerance derived in
mixer_cases.check_head_norm)."""
import pytest
import torch

from exl3_amd._lib import Exl3Error
from exl3_amd.heads import head_norm
from mixer_cases import check_head_norm, gen, normal

pytestmark = pytest.mark.gpu
EPS = 1e-6
TYPES = [torch.float16, torch.bfloat16]


def freqs(R, dev):
    return 10000.0 ** (-torch.arange(0, R, 2, device=dev, dtype=torch.float32) / max(R, 1))


def sides(seed, dev, T, Hq, Hk, d, dtype):
    g = gen(seed, dev)
    return normal(g, (T, Hq, d), dtype), normal(g, (T, Hk, d), dtype), normal(g, (d,), dtype, 0.2, 1.0), \
        normal(g, (d,), dtype, 0.2, 1.0)


# tokens, q heads, k heads, head size, rotated values
SHAPES = [(1, 64, 64, 128, 0), (1, 1, 1, 1, 0), (3, 5, 1, 128, 128), (17, 8, 2, 64, 32), (64, 64, 8, 128, 64),
          (5, 3, 3, 80, 20), (4, 2, 2, 96, 96), (7, 4, 4, 256, 128), (2, 3, 1, 512, 512), (3, 2, 1, 1024, 64),
          (5, 2, 2, 33, 32), (9, 7, 3, 100, 50), (300, 16, 16, 128, 128), (2, 1, 1, 8, 8), (2, 3, 2, 24, 16)]


@pytest.mark.parametrize("T,Hq,Hk,d,R", SHAPES)
@pytest.mark.parametrize("mode", ["rms", "l2"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
def test_formula(dev, T, Hq, Hk, d, R, mode, interleaved, dtype):
    q, k, wq, wk = sides(T + d, dev, T, Hq, Hk, d, dtype)
    pos = torch.arange(T, device=dev, dtype=torch.int32) * 977 if R else None
    inv = freqs(R, dev) if R else None
    a, b = head_norm(q, k, mode=mode, eps=EPS, q_weight=wq, k_weight=wk, positions=pos, inv_freq=inv,
                     interleaved=interleaved)
    check_head_norm(a, q, wq, mode, EPS, pos, inv, interleaved)
    check_head_norm(b, k, wk, mode, EPS, pos, inv, interleaved)
    # without weights, queries alone
    check_head_norm(head_norm(q, mode=mode, eps=EPS, positions=pos, inv_freq=inv, interleaved=interleaved), q, None,
                    mode, EPS, pos, inv, interleaved)


@pytest.mark.parametrize("dtype", TYPES)
def test_far_and_negative_positions(dev, dtype):
    q, k, _, _ = sides(3, dev, 6, 4, 2, 128, dtype)
    pos = torch.tensor([0, 1, -5, 1000003, 2 ** 31 - 1, -2 ** 31], device=dev, dtype=torch.int32)
    inv = freqs(128, dev)
    a, b = head_norm(q, k, eps=EPS, positions=pos, inv_freq=inv)
    # the last two: f64 angles of 31 bits times 24 are off by 2^-22 of a radian, within the bound's 32 2^-24
    check_head_norm(a, q, None, "rms", EPS, pos, inv)
    check_head_norm(b, k, None, "rms", EPS, pos, inv)


@pytest.mark.parametrize("d,R", [(128, 128), (64, 20), (50, 0)])
def test_strides_and_in_place(dev, d, R):
    g = gen(8, dev)
    T, Hq, Hk = 11, 6, 2
    pos, inv = (torch.arange(T, device=dev, dtype=torch.int32), freqs(R, dev)) if R else (None, None)
    kw = dict(eps=EPS, positions=pos, inv_freq=inv)
    for pad in (0, 8, 3):  # odd row lengths too: heads at 2-byte addresses
        row = normal(g, (T, (Hq + 2 * Hk) * d + pad), torch.float16)
        q, k = row[:, :Hq * d].view(T, Hq, d), row[:, Hq * d:(Hq + Hk) * d].view(T, Hk, d)
        a, b = head_norm(q, k, **kw)
        check_head_norm(a, q, None, "rms", EPS, pos, inv)
        check_head_norm(b, k, None, "rms", EPS, pos, inv)
        # heads outside tokens
        turned = q.transpose(0, 1).contiguous().transpose(0, 1)
        out = torch.empty_like(q.transpose(0, 1).contiguous()).transpose(0, 1)
        check_head_norm(head_norm(turned, q_out=out, **kw), q, None, "rms", EPS, pos, inv)
        # in place: the values' part of each row stays
        was = row.clone()
        head_norm(q, k, q_out=q, k_out=k, **kw)
        assert torch.equal(q, a) and torch.equal(k, b)
        assert torch.equal(row[:, (Hq + Hk) * d:], was[:, (Hq + Hk) * d:])


def test_extreme_values(dev):
    # a zero head stays zero under eps; the largest f16 values do not overflow; NaN keeps to its head
    x = torch.zeros((4, 2, 128), device=dev, dtype=torch.float16)
    x[1] = 65504.0
    x[2, 0, 5] = float("nan")
    x[2, 1] = 2.0 ** -24
    x[3, 1, 7] = float("inf")
    y = head_norm(x, eps=1e-6)
    assert bool((y[0] == 0).all())
    assert bool((y[1].float() - 1).abs().max() <= 2.0 ** -11)
    assert bool(y[2, 0].isnan().all()) and bool(y[2, 1].isfinite().all())
    check_head_norm(y[2:3, 1:], x[2:3, 1:], None, "rms", 1e-6)
    assert bool((y[3, 0] == 0).all()) and bool(y[3, 1, 7].isnan())


def test_no_tokens_and_refusals(dev):
    q, k, w, _ = sides(1, dev, 4, 2, 2, 128, torch.float16)
    assert head_norm(q[:0]).shape == (0, 2, 128)
    with pytest.raises(Exl3Error, match="overlap"):
        head_norm(q, k, k_out=q)
    with pytest.raises(Exl3Error, match="overlap"):
        head_norm(q[:3], q_out=q[1:])
    with pytest.raises(Exl3Error, match="overlap"):
        head_norm(q[:1], q_out=q[:1, :1].expand(1, 2, 128))
    with pytest.raises(Exl3Error, match="weight"):
        buf = torch.zeros(4 * 2 * 128, device=dev, dtype=torch.float16)
        head_norm(q, q_weight=buf[:128], q_out=buf.view(4, 2, 128))


def test_graph_replays(dev):
    q, k, w, _ = sides(2, dev, 33, 8, 4, 128, torch.float16)
    pos, inv = torch.arange(33, device=dev, dtype=torch.int32), freqs(128, dev)
    qo, ko = torch.empty_like(q), torch.empty_like(k)
    call = lambda: head_norm(q, k, q_weight=w, k_weight=w, positions=pos, inv_freq=inv, q_out=qo, k_out=ko)  # noqa: E731
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for i in range(3):
        q.copy_(normal(gen(50 + i, dev), q.shape, torch.float16))
        pos += 1000
        graph.replay()
        torch.cuda.synchronize()
        got = qo.clone(), ko.clone()
        call()
        assert torch.equal(got[0], qo) and torch.equal(got[1], ko)
