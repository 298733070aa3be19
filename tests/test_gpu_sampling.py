"""GPU tests of exl3_sample against the choice in 64 bits: ids equal, probabilities within an
f32 rounding and the integers' 2^-45 of the largest weight for each token of the row."""
import math

import numpy as np
import pytest
import torch

from exl3_amd._lib import Exl3Error
from exl3_amd.sampling import sample_tokens
from mixer_cases import choose64, gen, normal

pytestmark = pytest.mark.gpu
TYPES = [torch.float16, torch.bfloat16, torch.float32]


def check(logits, u, temp, k, p, min_p, **kw):
    ids, probs = sample_tokens(logits, u, temperature=temp, top_k=k, top_p=p, min_p=min_p, **kw)
    rows, vocab = logits.shape
    x, uu = logits.float().cpu().numpy(), u.cpu().numpy()
    one = lambda v, r: float(v[r]) if isinstance(v, torch.Tensor) else float(np.float32(v))  # noqa: E731
    for r in range(rows):
        want, prob = choose64(x[r], uu[r], one(temp, r), int(one(k, r)), one(p, r), one(min_p, r))
        assert int(ids[r]) == want, (r, int(ids[r]), want)
        # each weight is rounded by 2^-45 at most; the kept sum is 1 or more
        assert abs(float(probs[r]) - prob) <= prob * (2.0 ** -23 + vocab * 2.0 ** -45) + 2.0 ** -44, r
    return ids


def uniform(g, rows):
    return torch.rand(rows, generator=g, device=g.device)


@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (5, 7), (70, 100), (4, 2047), (4, 2049), (9, 32003), (2, 154880),
                                        (1, 262144), (1, 524288)])
@pytest.mark.parametrize("dtype", TYPES)
def test_sizes(dev, rows, vocab, dtype):
    g = gen(rows + vocab, dev)
    x = normal(g, (rows, vocab), dtype, 3.0)
    for temp, k, p, m in ((1.0, 0, 1.0, 0.0), (0.8, 40, 0.95, 0.0), (0.7, 0, 0.9, 0.0), (1.3, 1000, 0.98, 0.02),
                          (1.0, 0, 1.0, 0.1), (0.0, 0, 1.0, 0.0), (1.0, 1, 1.0, 0.0)):
        check(x, uniform(g, rows), temp, k, p, m)


def test_parameters_of_each_row(dev):
    g = gen(5, dev)
    rows, vocab = 64, 5003
    x = normal(g, (rows, vocab), torch.float16, 2.5)
    pick = lambda v: torch.tensor([v[i] for i in torch.randint(0, len(v), (rows,)).tolist()], device=dev)  # noqa: E731
    torch.manual_seed(0)
    for _ in range(3):
        check(x, uniform(g, rows), pick([0.0, -1.0, 1e-3, 0.5, 1.0, 3.0, 1e30]).float(), pick([0, -3, 1, 2, 50, vocab, 10 ** 9]).int(),
              pick([-1.0, 0.0, 1e-9, 0.3, 0.999, 1.0, 2.0]).float(), pick([-1.0, 0.0, 1e-12, 0.05, 1.0, 7.0]).float())


@pytest.mark.parametrize("u", [0.0, 0.5, 1.0 - 2.0 ** -24, 1.0, 3.0, -1.0])
@pytest.mark.parametrize("dtype", TYPES)
def test_equal_logits_and_ends_of_u(dev, u, dtype):
    # one bin, one logit: more ties than a list holds; every running weight is exact
    x = torch.full((2, 20001), 1.5, device=dev, dtype=dtype)
    uu = torch.full((2,), u, device=dev)
    n = 20001
    for k, p in ((0, 1.0), (7000, 1.0), (0, 0.25), (9000, 0.5), (3, 1.0)):
        ids, probs = sample_tokens(x, uu, top_k=k, top_p=p)
        kept = min(n, k) if k else n
        kept = math.ceil(p * kept)
        want = min(kept - 1, max(0, math.floor(u * kept)))
        assert ids.tolist() == [want, want]
        assert abs(float(probs[0]) - 1 / kept) <= 2.0 ** -23 / kept


def test_narrow_bins(dev):
    # many distinct logits in one bin of 1/64: the rounds over their bits, in f32 and on both
    # sides of zero, with ties across the row
    g = gen(9, dev)
    rows, vocab = 6, 40000
    x = normal(g, (rows, vocab), std=1e-3)
    x[2:4] = (x[2:4] * 1e5).round() / 1e5
    x[4:] += 100.0
    for k, p, m in ((0, 1.0, 0.0), (12345, 1.0, 0.0), (0, 0.6, 0.0), (30000, 0.7, 0.999)):
        check(x, uniform(g, rows), 1.0, k, p, m)
        check(x.half(), uniform(g, rows), 1.0, k, p, m)


@pytest.mark.parametrize("dtype", TYPES)
def test_masked_and_infinite(dev, dtype):
    g = gen(11, dev)
    inf, nan = math.inf, math.nan
    x = normal(g, (8, 3001), dtype, 2.0)
    x[0] = -inf
    x[1] = nan
    x[2] = -inf
    x[2, 2999] = -60000.0 if dtype == torch.float16 else -3e38
    x[3, ::2] = nan
    x[3, 1::4] = -inf
    x[4, [17, 2000, 2500]] = inf
    x[5] = nan
    x[5, 5] = inf
    x[6] = torch.finfo(dtype).min
    x[7, ::3] = -0.0
    x[7, 1::3] = 0.0
    x[7, 2::3] = -5.0
    for temp, k, p in ((1.0, 0, 1.0), (0.5, 2, 1.0), (2.0, 0, 0.5), (0.0, 0, 1.0)):
        ids = check(x, torch.tensor([0.3] * 4 + [0.5] + [0.9] * 3, device=dev), temp, k, p, 0.0)
        assert ids[:2].tolist() == [-1, -1] and int(ids[2]) == 2999 and int(ids[5]) == 5


def test_strides_streams_and_repeats(dev):
    g = gen(12, dev)
    wide = normal(g, (5, 4099), torch.float16, 3.0)
    u = uniform(g, 5)
    x = wide[:, 3:4003]
    want = check(x, u, 0.9, 100, 0.97, 0.0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got, _ = sample_tokens(x, u, temperature=0.9, top_k=100, top_p=0.97)
    side.synchronize()
    assert torch.equal(got, want)
    # one row for all: a stride of 0 is refused, one row alone takes any
    with pytest.raises(Exl3Error, match="stride"):
        from exl3_amd import _lib
        _lib.call("exl3_sample", _lib.C.byref(_lib.SampleConfig(dtype=0)), x.data_ptr(), 5, 4000, 0, u.data_ptr(),
                  got.data_ptr(), None, None, 0, None)
    with pytest.raises(Exl3Error, match="workspace"):
        from exl3_amd import _lib
        _lib.call("exl3_sample", _lib.C.byref(_lib.SampleConfig(dtype=0)), x.data_ptr(), 5, 4000, 4099, u.data_ptr(),
                  got.data_ptr(), None, None, 0, None)


def test_distribution(dev):
    # the same row for evenly spaced u: each token as often as its share says, to one in n
    n = 4000
    x = normal(gen(13, dev), (1, 50), torch.float32, 1.5)
    u = (torch.arange(n, device=dev) + 0.5) / n
    ids, probs = sample_tokens(x.expand(n, 50).contiguous(), u)
    share = torch.softmax(x[0].double(), 0)
    seen = torch.bincount(ids.long(), minlength=50).double() / n
    assert float((seen - share).abs().max()) <= 1.0 / n
    assert float((probs.double() - share[ids.long()]).abs().max()) <= 1e-7


def test_graph_replays(dev):
    g = gen(14, dev)
    x, u = normal(g, (8, 20011), torch.float16, 3.0), uniform(g, 8)
    ids, probs = torch.empty(8, device=dev, dtype=torch.int32), torch.empty(8, device=dev)
    from exl3_amd import _lib
    ws = torch.empty(_lib.lib().exl3_sample_workspace_size(8, 20011), device=dev, dtype=torch.uint8)
    call = lambda: sample_tokens(x, u, temperature=0.8, top_k=50, top_p=0.9, ids=ids, probs=probs, ws=ws)  # noqa: E731
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for i in range(4):
        x.copy_(normal(g, x.shape, torch.float16, 3.0))
        u.copy_(uniform(g, 8))
        graph.replay()
        torch.cuda.synchronize()
        got = ids.clone(), probs.clone()
        call()
        assert torch.equal(got[0], ids) and torch.equal(got[1], probs)


def test_rows_inside_each_other_are_refused(dev):
    x, u = normal(gen(11, dev), (1, 5003), torch.float16, 3.0), uniform(gen(12, dev), 9)
    for rows in (x.expand(9, 5003), x.flatten().as_strided((3, 4000), (500, 1))):
        with pytest.raises(Exl3Error, match="stride"):
            sample_tokens(rows, u[:len(rows)])
    # a single row's stride says nothing
    (a, b), (c, d) = sample_tokens(x.as_strided((1, 4000), (7, 1)), u[:1]), sample_tokens(x[:, :4000].contiguous(), u[:1])
    assert torch.equal(a, c) and torch.equal(b, d)


@pytest.mark.parametrize("temp", [1e-45, 1e-30, 1e-3, 1e30, math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("dtype", TYPES)
def test_extreme_temperatures(dev, temp, dtype):
    # from the largest logit alone to even shares of all that are not masked; NaN as 0
    g = gen(31, dev)
    x, u = normal(g, (4, 3001), dtype, 3.0), uniform(g, 4)
    x[1, 7], x[1, 2000] = math.inf, math.inf
    x[2, :1500] = -math.inf
    x[3, 11] = math.nan
    check(x, u, temp, 0, 1.0, 0.0)
    check(x, u, temp, 50, 0.9, 0.01)
