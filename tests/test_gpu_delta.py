"""GPU tests of exl3_delta_rule against the rule token by token in 64 bits (tolerance derived
in mixer_cases.check_delta)."""
import math

import pytest
import torch

from exl3_amd._lib import Exl3Error
from exl3_amd.delta import delta_rule
from mixer_cases import check_delta, delta64, delta_inputs, gen, normal

pytestmark = pytest.mark.gpu


def starts_of(lens, first=0):
    s = [first]
    for n in lens:
        s.append(s[-1] + n)
    return s


def ints(v, dev):
    return torch.tensor(v, device=dev, dtype=torch.int32)


def run(dev, lens, Hk=2, Hv=2, dk=128, dv=128, channel=True, dtype=torch.float16, packed=False, seed=0, first=0, tail=0,
        src=None, dst=None, n_slots=None, change=None, scale=None):
    starts = starts_of(lens, first)
    n = len(lens)
    n_slots = n + 2 if n_slots is None else n_slots
    x = delta_inputs(seed, dev, starts[-1] + tail, Hk, Hv, dk, dv, channel, n_slots, dtype, packed)
    if change:
        change(x)
    src = [(3 * i + 1) % n_slots if math.gcd(3, n_slots) == 1 else i for i in range(n)] if src is None else src
    used = src if dst is None else dst
    sc = dk ** -0.5 if scale is None else scale
    want, new, size, biggest = delta64(**x, starts=starts, src=src, dst=used, scale=sc)
    state, was = x["state"].clone(), x["state"].clone()
    out = torch.full((starts[-1] + tail, Hv, dv), 7.0, device=dev, dtype=dtype)
    delta_rule(x["q"], x["k"], x["v"], x["g"], x["beta"], state, starts=ints(starts, dev), slots=ints(src, dev),
               dst=None if dst is None else ints(dst, dev), out=out, scale=scale)
    # rows outside the sequences stay
    assert bool((out[:first] == 7).all()) and bool((out[starts[-1]:] == 7).all())
    check_delta(out, state, want, new, size, biggest, starts, used, dk)
    written = {used[i] for i in range(n) if not any(used[i] in (src[j], used[j]) for j in range(n) if j != i)}
    for s in set(range(n_slots)) - written:  # slots that nothing writes keep their bits
        assert torch.equal(state[s], was[s]), s
    return x, out, state


LENS = [[1], [2], [1, 1, 1], [4, 4], [16], [17], [31], [32], [33], [64], [65], [100, 1, 0, 37], [200], [0, 0, 5], [333, 64, 1, 128]]


@pytest.mark.parametrize("lens", LENS, ids=str)
@pytest.mark.parametrize("channel", [False, True])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_lengths(dev, lens, channel, dtype):
    run(dev, lens, channel=channel, dtype=dtype, seed=len(lens))


@pytest.mark.parametrize("Hk,Hv,dk,dv", [(1, 1, 64, 16), (3, 3, 64, 64), (2, 4, 128, 48), (1, 5, 128, 96), (4, 4, 64, 256),
                                         (1, 2, 128, 256), (5, 5, 128, 112)])
@pytest.mark.parametrize("lens", [[1, 1], [3, 40, 70]], ids=str)
@pytest.mark.parametrize("channel", [False, True])
def test_heads_and_sizes(dev, Hk, Hv, dk, dv, lens, channel):
    run(dev, lens, Hk, Hv, dk, dv, channel, packed=True, seed=Hv + dv, first=2, tail=3)


@pytest.mark.parametrize("lens", [[1] * 5, [40, 3, 0, 70, 33]], ids=str)
def test_slots(dev, lens):
    n = 5
    run(dev, lens, src=[4, 3, 2, 1, 0], dst=[5, 6, 7, 8, 9], n_slots=10)           # to other slots
    run(dev, lens, src=[4, -1, 2, 99, 0], dst=[5, 1, -1, 8, 100], n_slots=10)      # from zeros, and not stored
    run(dev, lens, src=[1, 1, 2, 3, 4], n_slots=6)                                 # one slot twice: kept
    run(dev, lens, src=[0, 0, 0, 3, 4], dst=[0, 1, 2, 3, 3], n_slots=6)            # forks; one target twice
    run(dev, lens, src=[0, 1, 2, 3, 4], dst=[1, 5, 0, 3, 4], n_slots=6)            # a slot that another reads
    run(dev, lens, src=list(range(n)), n_slots=3)


def test_decays_that_clear_and_keep(dev):
    # g = -inf clears a channel, very negative ones nearly; 0 keeps; chunks and steps agree with the rule
    def change(x):
        x["g"][::7] = -math.inf
        x["g"][3::11] = -500.0
        x["g"][5::13] = 0.0
        x["g"][40:] = -1e-4
        x["g"][60, :, ::2] = -80.0
    for lens in ([90], [1, 2, 87]):
        run(dev, lens, channel=True, change=change)

    def change_head(x):
        x["g"][::7] = -math.inf
        x["g"][3::11] = -500.0
        x["g"][5::13] = 0.0
        x["g"][45:] = -1e-4
    run(dev, [90], channel=False, change=change_head)


def test_strong_and_equal_keys(dev):
    # the same key over and over with beta 1 replaces the value each time: out = scale v (q = k)
    def change(x):
        x["k"][:] = x["k"][:1]
        x["q"][:] = x["k"]
        x["beta"][:] = 1.0
        x["g"][:] = 0.0
    x, out, _ = run(dev, [75], change=change, scale=1.0)
    k2 = x["k"][0].double().square().sum(-1)
    assert float((k2 - 1).abs().max()) < 2e-3  # f16 unit keys
    assert float((out.double() - x["v"].double()).abs().max()) < 5e-2

    def empty(x):
        x["beta"][:] = 0.0
    run(dev, [50], change=empty)


def test_special_values_stay_in_their_head_and_sequence(dev):
    x = delta_inputs(4, dev, 80, 2, 2, 128, 64, True, 2)
    st = x["state"].clone()
    clean = delta_rule(x["q"], x["k"], x["v"], x["g"], x["beta"], st, starts=ints([0, 40, 80], dev))
    v = x["v"].clone()
    v[50, 1, 3] = math.nan
    v[60, 1, 9] = math.inf
    st2 = x["state"].clone()
    out = delta_rule(x["q"], x["k"], v, x["g"], x["beta"], st2, starts=ints([0, 40, 80], dev))
    assert torch.equal(out[:40], clean[:40]) and torch.equal(out[:, 0], clean[:, 0]) and torch.equal(st2[0], st[0])
    # the tokens before it: the rule's values (a chunk with a NaN goes token by token, so the last
    # bits of its 16 columns' outputs may differ from the clean call's)
    part = {n: t[:50] if n != "state" else t for n, t in x.items()}
    want, new, size, biggest = delta64(**part, starts=[0, 40, 50], src=[0, 1], dst=[0, 1], scale=128 ** -0.5)
    bound = (2.0 ** -11 * (1 + 2.0 ** -10) * want.abs() + 2.0 ** -25
             + 8 * math.sqrt(144 * 11) * 2.0 ** -24 * size[..., None])  # check_delta's for 10 tokens
    assert bool(out[50:, 1, 3].isnan().all()) and bool(((out[40:50].double() - want[40:]).abs() <= bound[40:]).all())
    assert torch.equal(out[:, 1, 16:], clean[:, 1, 16:])


def test_unordered_starts_stay_in_bounds(dev):
    # starts that no caller should pass: clamped into the call's tokens, nothing else is touched
    x = delta_inputs(5, dev, 64, 1, 1, 64, 32, False, 4)
    buf = torch.zeros((64 + 2, 1, 32), device=dev, dtype=torch.float16)
    delta_rule(x["q"], x["k"], x["v"], x["g"], x["beta"], x["state"], starts=ints([-7, 50, 20, 1000], dev), out=buf[1:65])
    assert bool((buf[0] == 0).all()) and bool((buf[65] == 0).all()) and bool(buf.isfinite().all())


def test_equal_lengths_without_starts(dev):
    x = delta_inputs(6, dev, 12, 2, 2, 128, 128, True, 4)
    a, b = x["state"].clone(), x["state"].clone()
    slots = ints([2, 0, 3], dev)
    one = delta_rule(x["q"], x["k"], x["v"], x["g"], x["beta"], a, slots=slots)
    two = delta_rule(x["q"], x["k"], x["v"], x["g"], x["beta"], b, slots=slots, starts=ints([0, 4, 8, 12], dev))
    assert torch.equal(one, two) and torch.equal(a, b)
    a = x["state"].clone()
    whole = delta_rule(x["q"], x["k"], x["v"], x["g"], x["beta"], a)
    assert whole.shape == one.shape and torch.equal(a[1:], x["state"][1:])


def test_steps_continue_a_prefill(dev):
    # a prefill and then single tokens give what the whole sequence gives
    x = delta_inputs(7, dev, 140, 2, 4, 128, 128, True, 1)
    whole = x["state"].clone()
    out = delta_rule(x["q"], x["k"], x["v"], x["g"], x["beta"], whole)
    part = x["state"].clone()
    outs = []
    cut = [0, 100, 101, 102, 106, 140]
    for a, b in zip(cut, cut[1:]):
        outs.append(delta_rule(*(x[n][a:b] for n in ("q", "k", "v", "g", "beta")), part))
    want, new, size, biggest = delta64(**x, starts=[0, 140], src=[0], dst=[0], scale=128 ** -0.5)
    check_delta(out, whole, want, new, size, biggest, [0, 140], [0], 128)
    check_delta(torch.cat(outs), part, want, new, size, biggest, [0, 140], [0], 128)


def test_nothing_to_do_and_refusals(dev):
    x = delta_inputs(8, dev, 6, 2, 2, 128, 128, True, 3)
    args = [x[n] for n in ("q", "k", "v", "g", "beta", "state")]
    was = x["state"].clone()
    assert delta_rule(*[t[:0] for t in args[:5]], x["state"], starts=ints([0], dev)).shape == (0, 2, 128)
    delta_rule(*[t[:0] for t in args[:5]], x["state"], starts=ints([0, 0, 0], dev))
    assert torch.equal(was, x["state"])
    with pytest.raises(Exl3Error, match="overlap"):
        delta_rule(*args, out=x["v"])
    with pytest.raises(ValueError, match="divide"):
        delta_rule(*args, slots=ints([0, 1, 2, 0], dev))


@pytest.mark.parametrize("lens", [[1] * 6, [70, 3, 33]], ids=str)
def test_graph_replays_and_repeats(dev, lens):
    starts = starts_of(lens)
    n = len(lens)
    x = delta_inputs(9, dev, starts[-1], 2, 2, 128, 128, True, n)
    st, sl = ints(starts, dev), ints(list(range(n)), dev)
    out = torch.empty_like(x["v"])
    from exl3_amd import _lib
    from exl3_amd.delta import _config
    need = _lib.lib().exl3_delta_workspace_size(_lib.C.byref(_config(x["q"], x["v"], x["g"], None)), starts[-1], n)
    ws = torch.empty(max(need, 256), device=dev, dtype=torch.uint8)
    call = lambda state: delta_rule(x["q"], x["k"], x["v"], x["g"], x["beta"], state, starts=st, slots=sl, out=out, ws=ws)  # noqa: E731
    live, eager = x["state"].clone(), x["state"].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(live)
    torch.cuda.current_stream().wait_stream(side)
    live.copy_(eager)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(live)
    for i in range(4):
        x["v"].copy_(normal(gen(90 + i, dev), x["v"].shape, torch.float16))
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        call(eager)  # the states carry on from call to call on both sides
        assert torch.equal(got, out) and torch.equal(live, eager), i


@pytest.mark.parametrize("Hk,Hv,dv,lens", [(1, 2, 128, [1500]), (8, 8, 256, [300, 1, 77, 200, 64, 33]), (2, 2, 96, [129])], ids=str)
@pytest.mark.parametrize("channel", [False, True])
def test_long_sequences(dev, Hk, Hv, dv, lens, channel):
    # few workgroups (two column blocks each) and many (four)
    run(dev, lens, Hk, Hv, 128, dv, channel, seed=dv)


@pytest.mark.parametrize("dk", [64, 128])
@pytest.mark.parametrize("lens", [[1, 1, 1], [70, 33]], ids=str)
def test_rows_at_odd_addresses(dev, dk, lens):
    # rows of an odd number of values, beginning one value into a buffer: 2-byte addresses
    T, H = sum(lens), 2
    x = delta_inputs(12, dev, T, H, H, dk, 64, True, len(lens))
    starts = starts_of(lens)
    want, st = x["v"].clone(), x["state"].clone()
    delta_rule(x["q"], x["k"], x["v"], x["g"], x["beta"], st, starts=ints(starts, dev), out=want)

    def odd(t):
        n = t[0].numel()
        buf = torch.zeros(T * (n + 5) + 1, device=dev, dtype=t.dtype)[1:].view(T, n + 5)
        buf[:, :n] = t.flatten(1)
        return buf[:, :n].view(t.shape)

    out, st2 = odd(torch.zeros_like(want)), x["state"].clone()
    delta_rule(odd(x["q"]), odd(x["k"]), odd(x["v"]), odd(x["g"]), odd(x["beta"]), st2, starts=ints(starts, dev), out=out)
    assert torch.equal(out, want) and torch.equal(st, st2)


def test_columns_of_any_scale(dev):
    # columns are independent and scale exactly by powers of two (bf16, f32): to the bit, also in
    # the chunks' f16 pairs, whose scale is each column's own
    x = delta_inputs(13, dev, 100, 2, 2, 128, 64, True, 1, torch.bfloat16)
    by = torch.tensor([2.0 ** ((c % 5 - 2) * 12) for c in range(64)], device=dev)
    a, b = x["state"].clone(), x["state"] * by
    one = delta_rule(x["q"], x["k"], x["v"], x["g"], x["beta"], a)
    two = delta_rule(x["q"], x["k"], (x["v"].float() * by).to(torch.bfloat16), x["g"], x["beta"], b)
    assert torch.equal(one.float() * by, two.float()) and torch.equal(a * by, b)


def test_values_out_of_the_pairs_range(dev):
    # keys of 1000 and growing states: chunks that the matrix instructions do not take
    def large(x):
        x["k"][:] = (x["k"].float() * 1000).half()
        x["beta"][:] = 1e-6
    run(dev, [80], change=large)

    def growing(x):
        x["g"][:] = 0.005
    run(dev, [40], change=growing)
    run(dev, [40], change=growing, channel=False)

    def only_some(x):  # one chunk of three
        x["k"][40] = (x["k"][40].float() * 700).half()
        x["beta"][40] = 1e-6
    run(dev, [96], change=only_some)


def test_zero_and_tiny_inputs(dev):
    def zeros(x):
        for n in ("q", "k", "v", "state"):
            x[n][:] = 0
    x, out, state = run(dev, [50], change=zeros)
    assert bool((out == 0).all()) and bool((state[1] == 0).all())

    def tiny(x):
        x["v"][:] = (x["v"].float() * 1e-30).to(x["v"].dtype)
        x["state"][:] *= 1e-30
    run(dev, [50], change=tiny, dtype=torch.bfloat16)


@pytest.mark.parametrize("beta,k_scale,q_scale", [(1e-6, 1.0, 1.0), (1.0, 2.0 ** -12, 1.0), (1e-3, 2.0 ** -7, 2.0 ** -13),
                                                  (0.5, 1.0, 2.0 ** -30)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_small_writes_keep_their_precision(dev, beta, k_scale, q_scale, dtype):
    # from zeros, nothing forgotten: the state is a sum of 70 small products, so its error is held
    # to the state itself (not to the values, which are far larger), by check_delta's count of
    # roundings; small queries give outputs to half a step of their type
    scale = 2.0 ** 16
    if dtype == torch.float16 and q_scale < 2.0 ** -20:  # (f16 has no such queries: plain ones, whose results would overflow)
        q_scale = scale = 1.0
    x = delta_inputs(14, dev, 70, 1, 1, 128, 64, True, 1, dtype)
    x["g"][:], x["beta"][:], x["state"][:] = 0.0, beta, 0.0
    x["k"], x["q"] = (x["k"].float() * k_scale).to(dtype), (x["q"].float() * q_scale).to(dtype)
    want, new, _, _ = delta64(**x, starts=[0, 70], src=[0], dst=[0], scale=scale)
    st = x["state"].clone()
    out = delta_rule(x["q"], x["k"], x["v"], x["g"], x["beta"], st, scale=scale)
    rel = 4 * math.sqrt(128 + 16) * 2.0 ** -24 * math.sqrt(71)
    assert float((st.double() - new).norm() / new.norm()) <= rel
    # f16 results under 2^-14 are subnormals, 2^-24 apart: each off by up to 2^-25, n of them by
    # sqrt(n) 2^-25 in norm
    half, tiny = (2.0 ** -11, 2.0 ** -25) if dtype == torch.float16 else (2.0 ** -8, 0.0)
    assert float((out.double() - want).norm()) <= (half + 2 * rel) * float(want.norm()) + tiny * math.sqrt(out.numel())


# single tokens and short sequences beside long ones: each goes by its own length
MIXED = [[1] * 20 + [100], [100] + [3] * 20, [15, 16, 17, 1, 0, 31, 32, 33, 1, 1], [1] * 9 + [0] + [70] + [1] * 9 + [200], [7] * 12]


@pytest.mark.parametrize("lens", MIXED, ids=str)
@pytest.mark.parametrize("channel", [False, True])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_mixed_lengths(dev, lens, channel, dtype):
    run(dev, lens, channel=channel, dtype=dtype, seed=len(lens), first=3, tail=2)


@pytest.mark.parametrize("Hk,Hv,dk,dv", [(1, 3, 64, 16), (2, 4, 128, 48), (4, 4, 64, 256)])
def test_mixed_lengths_of_many_sequences(dev, Hk, Hv, dk, dv):
    run(dev, [1] * 300 + [40, 2] + [1] * 300 + [90], Hk, Hv, dk, dv, seed=dv, src=list(range(603)), n_slots=603)


def test_slots_between_long_and_short_sequences(dev):
    # sequences 0 and 3 are long: slots that a short one and a long one name, forks, zeros, targets elsewhere
    lens = [60, 1, 2, 90, 1, 1, 1, 0]
    run(dev, lens, src=[0, 0, 2, 3, 3, 5, 6, 7], n_slots=8)
    run(dev, lens, src=[0, 0, 0, 0, 4, 5, 6, 7], dst=[1, 2, 3, 8, 8, 9, 6, 10], n_slots=11)
    run(dev, lens, src=[1, 0, -1, 99, 4, 5, 6, 7], dst=[0, 1, 2, 3, -1, 9, 8, 7], n_slots=10)


def test_mixed_lengths_captured(dev):
    # the same graph over other lengths of the same total: a sequence goes from steps to chunks and back
    n, T, H = 12, 200, 2
    x = delta_inputs(21, dev, T, H, H, 128, 128, True, n)
    out, ws = torch.empty_like(x["v"]), torch.empty(1 << 22, device=dev, dtype=torch.uint8)
    all_lens = [[1] * 11 + [189], [100] + [9] * 10 + [10], [17] * 11 + [13], [0] * 10 + [100, 100]]
    starts, sl = ints(starts_of(all_lens[0]), dev), ints(list(range(n)), dev)
    call = lambda state: delta_rule(x["q"], x["k"], x["v"], x["g"], x["beta"], state, starts=starts, slots=sl, out=out, ws=ws)  # noqa: E731
    live, eager = x["state"].clone(), x["state"].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(live)
    torch.cuda.current_stream().wait_stream(side)
    live.copy_(eager)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(live)
    for lens in all_lens:
        assert sum(lens) == T
        starts.copy_(ints(starts_of(lens), dev))
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        before = eager.clone()
        call(eager)
        assert torch.equal(got, out) and torch.equal(live, eager), lens
        want, new, size, biggest = delta64(x["q"], x["k"], x["v"], x["g"], x["beta"], before, starts_of(lens), list(range(n)),
                                           list(range(n)), 128 ** -0.5)
        check_delta(got, live, want, new, size, biggest, starts_of(lens), list(range(n)), 128)
