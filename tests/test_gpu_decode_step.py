"""GPU test of the token mixer and the sampler as a decoder runs them, between its trellis
linears: qkv linear -> head norm (in place on the packed rows) -> delta rule -> o linear ->
head linear -> token, a ragged prefill first and single tokens after it, eagerly and as a
captured graph. Each operator's results are held to its formula in 64 bits on the inputs that
it got."""
import numpy as np
import pytest
import torch

from exl3_amd import _lib
from exl3_amd.delta import _config, delta_rule
from exl3_amd.heads import head_norm
from exl3_amd.sampling import sample_tokens
from exl3_amd.trellis import TrellisWeight, trellis_linear
from mixer_cases import check_delta, check_head_norm, choose64, delta64, gen, normal

pytestmark = pytest.mark.gpu
HIDDEN, HEADS, D, VOCAB = 512, 4, 128, 1024
EPS = 1e-6


def linear(g, inf, outf):
    words = torch.randint(-32768, 32768, (inf // 16, outf // 16, 64), dtype=torch.int16, generator=g, device=g.device)
    return TrellisWeight(words, normal(g, (inf,), torch.float16, 0.05, 1.0),
                         normal(g, (outf,), torch.float16, 0.05 * inf ** -0.5, inf ** -0.5), inf, outf, 4, 1)


class Model:
    def __init__(self, dev, n_slots):
        g = gen(31, dev)
        self.qkv, self.o, self.head = linear(g, HIDDEN, 3 * HEADS * D), linear(g, HEADS * D, HIDDEN), linear(g, HIDDEN, VOCAB)
        self.rate = torch.exp(torch.rand((HEADS, D), generator=g, device=dev) * 4 - 3)
        self.gates = normal(g, (HIDDEN, HEADS * (D + 1)), torch.float32, HIDDEN ** -0.5)
        self.embed = normal(g, (VOCAB, HIDDEN), torch.float16)
        self.state = torch.zeros((n_slots, HEADS, D, D), device=dev)

    def mix(self, ids, starts, slots, seen=None):
        """One mixer step over the tokens `ids`; `seen` collects what each operator got and gave."""
        x = self.embed[ids.long()]
        T, n = x.shape[0], HEADS * D
        row = trellis_linear(self.qkv, x)
        before = row.clone() if seen is not None else None
        q, k, v = (row[:, i * n:(i + 1) * n].view(T, HEADS, D) for i in range(3))
        head_norm(q, k, mode="l2", eps=EPS, q_out=q, k_out=k)
        gates = x.float() @ self.gates
        g = -self.rate * torch.nn.functional.softplus(gates[:, HEADS:].view(T, HEADS, D))
        beta = torch.sigmoid(gates[:, :HEADS]).contiguous()
        was = self.state.clone() if seen is not None else None
        o = delta_rule(q, k, v, g, beta, self.state, starts=starts, slots=slots)
        y = x + trellis_linear(self.o, o.view(T, n))
        if seen is not None:
            seen.append(dict(row=before, q=q, k=k, v=v, g=g, beta=beta, was=was, out=o))
        return y

    def step(self, ids, starts, slots, last, u, seen=None):
        y = self.mix(ids, starts, slots, seen)
        logits = trellis_linear(self.head, y[last])
        new, probs = sample_tokens(logits, u, temperature=0.8, top_k=50, top_p=0.95, min_p=0.01)
        if seen is not None:
            seen[-1].update(logits=logits, ids=new, probs=probs)
        return new


def ints(v, dev):
    return torch.tensor(v, device=dev, dtype=torch.int32)


def check(seen, starts, slots, u, state):
    n = HEADS * D
    T = seen["q"].shape[0]
    for i, name in enumerate(("q", "k")):
        check_head_norm(seen[name], seen["row"][:, i * n:(i + 1) * n].view(T, HEADS, D), None, "l2", EPS)
    assert torch.equal(seen["v"].reshape(T, n), seen["row"][:, 2 * n:])
    want, new, size, biggest = delta64(seen["q"], seen["k"], seen["v"], seen["g"], seen["beta"], seen["was"], starts, slots,
                                       slots, D ** -0.5)
    check_delta(seen["out"], state, want, new, size, biggest, starts, slots, D)
    x, uu = seen["logits"].float().cpu().numpy(), u.cpu().numpy()
    for r in range(len(uu)):
        want_id, prob = choose64(x[r], uu[r], float(np.float32(0.8)), 50, 0.95, 0.01)
        assert int(seen["ids"][r]) == want_id
        assert abs(float(seen["probs"][r]) - prob) <= prob * 2.0 ** -22 + 2.0 ** -44


def test_prefill_and_decode(dev):
    model = Model(dev, 5)
    lens, slots = [40, 5, 17], [3, 0, 4]
    starts = [0, 40, 45, 62]
    g = gen(32, dev)
    ids = torch.randint(0, VOCAB, (62,), generator=g, device=dev, dtype=torch.int32)
    u = torch.rand(3, generator=g, device=dev)
    seen = []
    ids = model.step(ids, ints(starts, dev), ints(slots, dev), torch.tensor([39, 44, 61], device=dev), u, seen)
    check(seen[-1], starts, slots, u, model.state)
    for _ in range(4):
        u = torch.rand(3, generator=g, device=dev)
        ids = model.step(ids, ints([0, 1, 2, 3], dev), ints(slots, dev), torch.arange(3, device=dev), u, seen)
        check(seen[-1], [0, 1, 2, 3], slots, u, model.state)


def test_captured_decode(dev):
    # the whole decode step as one graph, its tokens fed back, against the same steps eagerly
    slots, starts = ints([2, 0, 1], dev), ints([0, 1, 2, 3], dev)
    last = torch.arange(3, device=dev)
    first, g = ints([5, 900, 77], dev), gen(33, dev)
    us = [torch.rand(3, generator=g, device=dev) for _ in range(5)]
    eager, model = Model(dev, 3), Model(dev, 3)
    ids, u = first.clone(), us[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # libraries' first calls
        model.step(ids, starts, slots, last, u)
    torch.cuda.current_stream().wait_stream(side)
    model.state.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ids.copy_(model.step(ids, starts, slots, last, u))
    want = first.clone()
    ids.copy_(first)
    for i, ui in enumerate(us):
        u.copy_(ui)
        graph.replay()
        torch.cuda.synchronize()
        want = eager.step(want, starts, slots, last, ui)
        assert torch.equal(ids, want), i
        assert torch.equal(model.state, eager.state), i


def test_two_threads_on_streams_of_their_own(dev):
    # independent sequences, each on its own stream with its own workspaces, against one by one
    import threading
    inputs = []
    for seed in range(2):
        g = gen(40 + seed, dev)
        T = 130
        unit = lambda x: torch.nn.functional.normalize(x, dim=-1).half()  # noqa: E731
        inputs.append(dict(q=unit(normal(g, (T, 2, D))), k=unit(normal(g, (T, 2, D))), v=normal(g, (T, 2, D), torch.float16),
                           g=-torch.rand((T, 2), generator=g, device=dev), beta=torch.rand((T, 2), generator=g, device=dev),
                           state=normal(g, (1, 2, D, D), std=0.3)))
    need = _lib.lib().exl3_delta_workspace_size(_lib.C.byref(_config(inputs[0]["q"], inputs[0]["v"], inputs[0]["g"], None)), 130, 1)
    assert need > 0
    want = []
    for x in inputs:
        st = x["state"].clone()
        want.append((delta_rule(x["q"], x["k"], x["v"], x["g"], x["beta"], st), st))
    torch.cuda.synchronize()
    got, errors = [None, None], []

    def work(i):
        try:
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                x = inputs[i]
                for _ in range(10):
                    st = x["state"].clone()
                    out = delta_rule(x["q"], x["k"], x["v"], x["g"], x["beta"], st)
            s.synchronize()
            got[i] = out, st
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for (a, b), (c, d) in zip(got, want):
        assert torch.equal(a, c) and torch.equal(b, d)
