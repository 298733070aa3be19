"""GPU tests of the head norm, the delta rule and the sampler past 32-bit offsets: slots,
rows and tokens behind 2^31 elements of a buffer give what the same values give in a small
one, to the bit."""
import pytest
import torch

from exl3_amd.delta import delta_rule
from exl3_amd.heads import head_norm
from exl3_amd.sampling import sample_tokens
from mixer_cases import delta_inputs, gen, normal

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [1, 70])
def test_far_slots(dev, T):
    H, slots = 16, 9000  # 16 x 128 x 128 floats a slot: 2.36e9 floats
    x = delta_inputs(1, dev, T, H, H, 128, 128, True, 2)
    pool = torch.empty((slots, H, 128, 128), device=dev)
    pool[8999], pool[8500] = x["state"][0], 0
    small = x["state"].clone()
    want = delta_rule(x["q"], x["k"], x["v"], x["g"], x["beta"], small, slots=torch.tensor([0], device=dev, dtype=torch.int32))
    got = delta_rule(x["q"], x["k"], x["v"], x["g"], x["beta"], pool, slots=torch.tensor([8999], device=dev, dtype=torch.int32),
                     dst=torch.tensor([8500], device=dev, dtype=torch.int32))
    assert torch.equal(got, want) and torch.equal(pool[8500], small[0]) and torch.equal(pool[8999], x["state"][0])


def test_far_tokens(dev):
    # 160 tokens of rows 2^24 - 8 values apart
    T, H, stride = 160, 1, 2 ** 24 - 8
    x = delta_inputs(2, dev, T, H, H, 128, 128, False, 1)
    small = x["state"].clone()
    want = delta_rule(x["q"], x["k"], x["v"], x["g"], x["beta"], small)
    big = torch.empty(T * stride, device=dev, dtype=torch.float16).view(T, stride)

    def far(t, at):
        v = big[:, at:at + 128].view(T, H, 128)
        v.copy_(t)
        return v

    big_state = x["state"].clone()
    q, k, v, out = far(x["q"], 0), far(x["k"], 128), far(x["v"], 256), big[:, 512:640].view(T, H, 128)
    other = torch.empty((T, H, 128), device=dev, dtype=torch.float16)
    got = delta_rule(q, k, v, x["g"], x["beta"], big_state, out=other)
    assert torch.equal(got, want) and torch.equal(big_state, small)
    a, b = head_norm(q, k, q_out=out)
    c, d = head_norm(x["q"].contiguous(), x["k"].contiguous())
    assert torch.equal(a, c) and torch.equal(b, d)


def test_far_logits(dev):
    vocab, stride = 5000, 2 ** 30 + 16
    big = torch.empty(2 * stride + vocab, device=dev, dtype=torch.float16)
    x = normal(gen(3, dev), (3, vocab), torch.float16, 3.0)
    rows = big.as_strided((3, vocab), (stride, 1))
    rows.copy_(x)
    u = torch.tensor([0.1, 0.5, 0.9], device=dev)
    for kw in (dict(temperature=0.0), dict(top_k=50, top_p=0.9), dict()):
        (a, b), (c, d) = sample_tokens(rows, u, **kw), sample_tokens(x, u, **kw)
        assert torch.equal(a, c) and torch.equal(b, d)


def test_many_rows(dev):
    # more rows than workgroups at once, each with parameters of its own
    g = gen(4, dev)
    x, u = normal(g, (5000, 300), torch.float16, 2.0), torch.rand(5000, generator=g, device=dev)
    k = torch.randint(0, 40, (5000,), generator=g, device=dev, dtype=torch.int32)
    ids, probs = sample_tokens(x, u, top_k=k, top_p=0.9)
    for at in (0, 1777, 4999):
        a, b = sample_tokens(x[at:at + 1], u[at:at + 1], top_k=int(k[at]), top_p=0.9)
        assert torch.equal(a, ids[at:at + 1]) and torch.equal(b, probs[at:at + 1])


@pytest.mark.parametrize("interleaved", [False, True])
def test_many_heads(dev, interleaved):
    # results larger than the caches take stores of their own: the same bits as in small calls
    g = gen(5, dev)
    q, k = normal(g, (1000, 128, 128), torch.float16), normal(g, (1000, 16, 128), torch.float16)
    pos = torch.arange(1000, device=dev, dtype=torch.int32)
    inv = 10000.0 ** (-torch.arange(0, 128, 2, device=dev, dtype=torch.float32) / 128)
    kw = dict(inv_freq=inv, interleaved=interleaved)
    a, b = head_norm(q, k, positions=pos, **kw)
    for at in (0, 500, 999):
        c, d = head_norm(q[at:at + 1], k[at:at + 1], positions=pos[at:at + 1], **kw)
        assert torch.equal(a[at:at + 1], c) and torch.equal(b[at:at + 1], d)


def test_more_tokens_than_a_launch(dev):
    # 2^24 + 5 tokens of one head of 8, by both kernels (16-byte rows, and rows behind one value)
    T, d = 2 ** 24 + 5, 8
    x = normal(gen(6, dev), (T, 1, d), torch.float16)
    pos = torch.arange(T, device=dev, dtype=torch.int32)
    inv = torch.tensor([1.0, 0.5, 0.25, 0.125], device=dev)
    odd = torch.empty(T * d + 1, device=dev, dtype=torch.float16)[1:].view(T, 1, d)
    for interleaved, out in ((True, None), (False, None), (True, odd)):
        got = head_norm(x, positions=pos, inv_freq=inv, interleaved=interleaved, q_out=out)
        for a, b in ((0, 3), (2 ** 22 - 2, 2 ** 22 + 2), (2 ** 24 - 1, T)):
            part = torch.empty((b - a) * d + 1, device=dev, dtype=torch.float16)
            want = head_norm(x[a:b].contiguous(), positions=pos[a:b].contiguous(), inv_freq=inv, interleaved=interleaved,
                             q_out=part[1:].view(b - a, 1, d) if out is odd else None)
            assert torch.equal(got[a:b], want)


def test_workspaces_and_one_token_in_place(dev):
    g = gen(7, dev)
    x, u = normal(g, (3, 500), torch.float16), torch.tensor([0.1, 0.5, 0.9], device=dev)
    d = delta_inputs(8, dev, 64, 1, 1, 64, 64, False, 1)
    for ws in (torch.empty(1 << 22, dtype=torch.uint8), torch.empty(1 << 20, device=dev), torch.empty((1 << 23,), device=dev, dtype=torch.uint8)[::2]):
        with pytest.raises(ValueError, match="ws"):
            sample_tokens(x, u, ws=ws)
        with pytest.raises(ValueError, match="ws"):
            delta_rule(d["q"], d["k"], d["v"], d["g"], d["beta"], d["state"], ws=ws)
    # one token, whose stride says nothing, in place
    q = normal(g, (1, 4, 64), torch.float16)
    want = head_norm(q)
    other = q.as_strided((1, 4, 64), (7, 64, 1))
    assert torch.equal(head_norm(q, q_out=other), want) and torch.equal(q, want)
