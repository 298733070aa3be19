"""The token mixer's and the sampler's operators that are timed: the per-head norm of queries
and keys with their rotation, the gated delta rule and the choice of a token from the head's
logits, over the calls that a decode step, a speculative verify step, a prefill and a ragged
batch make.

Heads are 64 of 128 values (the qkv linear's 24,576 = 3 x 64 x 128) or fewer where a model is
sharded over GPUs or shares its query and key heads; the vocabulary is the head linear's
154,880, and smaller ones. Activations are N(0, 1) rows as a linear gives them, queries and
keys of the delta rule have unit norm, decays come from a softplus with a learned rate.
"""
import math
import os
import sys

import torch

own = False

sys.path.insert(0, os.path.join(os.getcwd(), "exl3-server_amd"))

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
NORM_EPS = 1e-6


def listed():
    return [
        # a single sequence's decode step: q and k of one packed qkv row, to unit norm
        dict(name="norm_l2_t1", kind="norm", T=1, Hq=64, Hk=64, d=128, mode="l2", rot=0, inter=False, far=0, dtype="f16"),
        # a batch of decode steps of an attention layer with shared key heads, far in its context
        dict(name="norm_rms_rot_t64", kind="norm", T=64, Hq=64, Hk=8, d=128, mode="rms", rot=64, inter=True,
             far=1000000, dtype="bf16"),
        # a prefill chunk: norm with weights and the rotation of whole heads
        dict(name="norm_rms_rot_t2048", kind="norm", T=2048, Hq=64, Hk=64, d=128, mode="rms", rot=128, inter=False,
             far=0, dtype="f16"),
        # one token of one sequence: latency
        dict(name="delta_step_n1", kind="delta", lens="1", Hk=64, Hv=64, dk=128, dv=128, channel=True, dtype="f16"),
        # a decode step of 64 sequences: the states' traffic
        dict(name="delta_step_n64", kind="delta", lens=",".join(["1"] * 64), Hk=64, Hv=64, dk=128, dv=128,
             channel=True, dtype="f16"),
        # a verify step of 8 sequences with 3 drafted tokens each, on one of 4 GPUs
        dict(name="delta_verify_n8", kind="delta", lens=",".join(["4"] * 8), Hk=16, Hv=16, dk=128, dv=128,
             channel=True, dtype="f16"),
        # a 2048-token prefill chunk of one sequence
        dict(name="delta_prefill_2048", kind="delta", lens="2048", Hk=64, Hv=64, dk=128, dv=128, channel=True,
             dtype="f16"),
        # a ragged batch of prefills and single tokens with one decay a head and shared q/k heads
        dict(name="delta_ragged_n7", kind="delta", lens="700,1,64,333,1001,1,17", Hk=16, Hv=32, dk=128, dv=128,
             channel=False, dtype="bf16"),
        # the next token of one sequence from the head's logits
        dict(name="sample_r1", kind="sample", rows=1, vocab=154880, dtype="f16", temp=0.8, k=40, p=0.95, minp=0.0,
             spread=3.0, banned=0),
        # a batch of 8, nucleus only
        dict(name="sample_r8", kind="sample", rows=8, vocab=154880, dtype="f16", temp=1.0, k=0, p=0.9, minp=0.0,
             spread=3.0, banned=0),
        # a batch of 64 in f32 with every filter, part of the vocabulary masked by a grammar
        dict(name="sample_r64_f32", kind="sample", rows=64, vocab=154880, dtype="f32", temp=0.7, k=1000, p=0.98,
             minp=0.02, spread=3.0, banned=100000),
        # a large batch over a smaller, odd vocabulary, no filter: the whole distribution
        dict(name="sample_r200_all", kind="sample", rows=200, vocab=32003, dtype="bf16", temp=1.2, k=0, p=1.0,
             minp=0.0, spread=2.0, banned=0),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))


def draw(rng):
    kind = rng.choice(["norm", "delta", "delta", "delta", "sample", "sample"])
    if kind == "norm":
        d = rng.choice([64, 80, 96, 128, 128, 128, 192, 256])
        Hk = rng.choice([1, 2, 4, 5, 8, 16, 32, 64])
        Hq = Hk * rng.choice([1, 1, 2, 4, 8])
        most = max(1, 4096 * 8192 // (d * (Hq + Hk)))
        return dict(kind=kind, T=_log_int(rng, 1, min(4096, most)), Hq=Hq, Hk=Hk, d=d, mode=rng.choice(["rms", "l2"]),
                    rot=rng.choice([0, d // 4 * 2, d]), inter=rng.random() < 0.5, far=_log_int(rng, 1, 1000000),
                    dtype=rng.choice(["f16", "bf16"]))
    if kind == "delta":
        Hk = rng.choice([1, 2, 4, 5, 8, 16, 32])
        c = dict(kind=kind, lens="", Hk=Hk, Hv=Hk * rng.choice([1, 1, 1, 2]), dk=rng.choice([64, 128, 128, 128]),
                 dv=rng.choice([64, 128, 128, 128, 96, 256]), channel=rng.random() < 0.6,
                 dtype=rng.choice(["f16", "f16", "bf16"]))
        form = rng.choice(["step", "verify", "prefill", "ragged"])
        heads = 64 * 128 * 128 / (c["Hv"] * c["dk"] * c["dv"])
        if form == "step":
            lens = [1] * _log_int(rng, 1, 60 * min(4.0, heads))
        elif form == "verify":
            lens = [rng.randint(2, 8)] * _log_int(rng, 1, 24 * min(4.0, heads))
        elif form == "prefill":
            lens = [_log_int(rng, 20, 1800 * min(2.0, heads))]
        else:
            left, lens = int(1800 * min(2.0, heads)), []
            while left > 0 and len(lens) < 24:
                lens.append(min(left, _log_int(rng, 1, 1200)))
                left -= lens[-1]
        c["lens"] = ",".join(map(str, lens))
        return c
    vocab = _log_int(rng, 1000, 200000)
    rows = _log_int(rng, 1, min(128, max(1, 64 * 154880 // vocab)))
    return dict(kind=kind, rows=rows, vocab=vocab, dtype=rng.choice(["f16", "bf16", "f32"]),
                temp=rng.choice([0.0, 0.3, 0.7, 1.0, 1.0, 1.3]), k=rng.choice([0, 0, 1, 20, 50, 500, vocab // 2]),
                p=rng.choice([1.0, 1.0, 0.5, 0.9, 0.95, 0.99]), minp=rng.choice([0.0, 0.0, 0.01, 0.1]),
                spread=rng.choice([1.0, 2.0, 3.0, 4.0]), banned=rng.choice([0, 0, vocab // 3]))


# --- inputs, from the seed alone ------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 6271 + 29)
    return g


def _normal(g, shape, std=1.0, mean=0.0, dtype=torch.float32):
    return (torch.randn(shape, generator=g, device="cuda") * std + mean).to(dtype)


def _uniform(g, shape, lo=0.0, hi=1.0):
    return torch.rand(shape, generator=g, device="cuda") * (hi - lo) + lo


def _norm_inputs(c, g):
    T, Hq, Hk, d, dt = c["T"], c["Hq"], c["Hk"], c["d"], TYPES[c["dtype"]]
    # one packed row a token, as the qkv linear writes it: queries, keys, and values behind them
    rows = _normal(g, (T, (Hq + 2 * Hk) * d), dtype=dt)
    t = dict(q=rows[:, :Hq * d].view(T, Hq, d), k=rows[:, Hq * d:(Hq + Hk) * d].view(T, Hk, d),
             q_weight=None, k_weight=None, positions=None, inv_freq=None)
    if c["mode"] == "rms":
        t["q_weight"], t["k_weight"] = _normal(g, (d,), 0.2, 1.0, dt), _normal(g, (d,), 0.2, 1.0, dt)
    if c["rot"]:
        t["inv_freq"] = 10000.0 ** (-torch.arange(0, c["rot"], 2, device="cuda", dtype=torch.float32) / c["rot"])
        if c["T"] > 64 or not c["far"]:
            t["positions"] = torch.arange(T, device="cuda", dtype=torch.int32) + c["far"]
        else:
            t["positions"] = torch.randint(0, c["far"] + 1, (T,), generator=g, device="cuda", dtype=torch.int32)
    return t


def _delta_inputs(c, g):
    lens = [int(x) for x in c["lens"].split(",")]
    T, n, Hk, Hv, dk, dv, dt = sum(lens), len(lens), c["Hk"], c["Hv"], c["dk"], c["dv"], TYPES[c["dtype"]]
    unit = lambda x: (x / x.square().sum(-1, keepdim=True).sqrt()).to(dt)  # noqa: E731
    rate = torch.exp(_uniform(g, (Hv, dk) if c["channel"] else (Hv,), -4.0, 2.0))  # memories of a token to hundreds
    soft = torch.log1p(torch.exp(_normal(g, (T, Hv, dk) if c["channel"] else (T, Hv), 1.0, -1.0)))
    starts = torch.zeros(n + 1, dtype=torch.int32)
    starts[1:] = torch.cumsum(torch.tensor(lens), 0)
    return dict(q=unit(_normal(g, (T, Hk, dk))), k=unit(_normal(g, (T, Hk, dk))),
                v=_normal(g, (T, (Hv + 1) * dv), dtype=dt)[:, :Hv * dv].view(T, Hv, dv),
                g=-rate * soft, beta=torch.sigmoid(_normal(g, (T, Hv))),
                state=_normal(g, (n + 2, Hv, dk, dv), 0.3), starts=starts.cuda(),
                slots=torch.randperm(n + 2, generator=g, device="cuda")[:n].to(torch.int32))


def _sample_inputs(c, g):
    logits = _normal(g, (c["rows"], c["vocab"]), c["spread"])
    if c["banned"]:
        logits[:, :c["banned"]].masked_fill_(_uniform(g, (c["rows"], c["banned"])) < 0.9, -math.inf)
    one = lambda v, s: (v * _uniform(g, (c["rows"],), 1 - s, 1 + s)).float()  # noqa: E731
    return dict(logits=logits.to(TYPES[c["dtype"]]), u=_uniform(g, (c["rows"],)),
                temperature=one(c["temp"], 0.1), top_k=torch.full((c["rows"],), c["k"], device="cuda", dtype=torch.int32),
                top_p=one(c["p"], 0.0), min_p=one(c["minp"], 0.1))


def _inputs(c, seed):
    return {"norm": _norm_inputs, "delta": _delta_inputs, "sample": _sample_inputs}[c["kind"]](c, _gen(seed))


def prepare(case, seed):
    return case, _inputs(case, seed)


# --- one pass -------------------------------------------------------------------------

def run(state):
    case, t = state
    if own:
        return _own(case, t)
    return {"norm": _plain_norm, "delta": _plain_delta, "sample": _plain_sample}[case["kind"]](case, t)


def _own(case, t):
    if case["kind"] == "norm":
        from exl3_amd.heads import head_norm
        return head_norm(t["q"], t["k"], mode=case["mode"], eps=NORM_EPS, q_weight=t["q_weight"],
                         k_weight=t["k_weight"], positions=t["positions"], inv_freq=t["inv_freq"],
                         interleaved=case["inter"])
    if case["kind"] == "delta":
        from exl3_amd.delta import delta_rule
        out = delta_rule(t["q"], t["k"], t["v"], t["g"], t["beta"], t["state"], starts=t["starts"], slots=t["slots"])
        return out, t["state"]
    from exl3_amd.sampling import sample_tokens
    return sample_tokens(t["logits"], t["u"], temperature=t["temperature"], top_k=t["top_k"], top_p=t["top_p"],
                         min_p=t["min_p"])


def _plain_norm(c, t):
    return _plain_heads(c, t, t["q"], t["q_weight"]), _plain_heads(c, t, t["k"], t["k_weight"])


def _plain_heads(c, t, x, w):
    y = x.float()
    s = y.square().mean(-1, keepdim=True) if c["mode"] == "rms" else y.square().sum(-1, keepdim=True)
    y = y / torch.sqrt(s + NORM_EPS)
    if w is not None:
        y = y * w.float()
    if c["rot"]:
        R = c["rot"]
        angle = t["positions"].double()[:, None, None] * t["inv_freq"].double()  # far positions: 64 bits
        cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
        a, b = (y[..., 0:R:2], y[..., 1:R:2]) if c["inter"] else (y[..., :R // 2], y[..., R // 2:R])
        a, b = a * cos - b * sin, b * cos + a * sin
        turned = torch.stack((a, b), -1).flatten(-2) if c["inter"] else torch.cat((a, b), -1)
        y = torch.cat((turned, y[..., R:]), -1)
    return y.to(x.dtype)


def _plain_delta(c, t):
    """In chunks of C tokens, all sequences side by side (padded with tokens that change nothing);
    the states of a chunk follow from those before it, so the chunks are a loop."""
    starts, T, rep = t["starts"].long(), t["q"].shape[0], c["Hv"] // c["Hk"]
    n, dk = starts.numel() - 1, c["dk"]
    lens = [int(x) for x in c["lens"].split(",")]
    C = max(1, min(32, max(lens), int(math.sqrt(2 ** 26 / (n * c["Hv"] * dk)))))
    L = -(-max(lens) // C) * C
    at = starts[:-1, None] + torch.arange(L, device="cuda")
    real = at < starts[1:, None]
    at = at.clamp(max=T - 1)

    def rows(x, fill=0.0):  # (T, H, ...) -> (n, H, L, ...) in f32
        x = torch.where(real.view(n, L, *([1] * (x.dim() - 1))), x[at].float(), fill)
        return x.movedim(2, 1)

    q, k = (rows(t[x]).repeat_interleave(rep, 1) for x in ("q", "k"))
    v, beta = rows(t["v"]), rows(t["beta"])
    g = rows(t["g"])
    g = g if c["channel"] else g[..., None]
    S = t["state"][t["slots"].long()]
    out = torch.empty((n, c["Hv"], L, c["dv"]), device="cuda")
    low = torch.ones((C, C), device="cuda", dtype=torch.bool).tril()
    eye = torch.eye(C, device="cuda")
    for s in range(0, L, C):
        qc, kc, vc, bc = (x[:, :, s:s + C] for x in (q, k, v, beta))
        G = torch.cumsum(g[:, :, s:s + C].double(), 2)  # long sums whose differences count: 64 bits
        ratio = torch.where(low[:, :, None], G[:, :, :, None] - G[:, :, None], -math.inf).exp().float()
        if c["channel"]:
            kr = ratio * kc[:, :, None]
            A = (kr @ kc[..., None])[..., 0].tril(-1)
            B = (kr @ qc[..., None])[..., 0]
        else:
            A = (ratio[..., 0] * (kc @ kc.mT)).tril(-1)
            B = ratio[..., 0] * (qc @ kc.mT)
        decay, left = G.exp().float(), (G[:, :, -1:] - G).exp().float()
        X = bc[..., None] * (vc - (kc * decay) @ S)
        N = bc[..., None] * A
        U = X[:, :, :1]
        for i in range(1, C):  # forward substitution of (I + N) U = X
            U = torch.cat((U, X[:, :, i:i + 1] - N[:, :, i:i + 1, :i] @ U), 2)
        out[:, :, s:s + C] = (qc * decay) @ S + B @ U
        S = decay[:, :, -1, :, None] * S + (kc * left).mT @ U
    t["state"][t["slots"].long()] = S
    out = (out * dk ** -0.5).movedim(1, 2)[real]
    return out.to(t["q"].dtype), t["state"]


def _plain_sample(c, t):
    x, order = torch.sort(t["logits"].double(), dim=-1, descending=True, stable=True)  # borders: 64 bits
    temp = t["temperature"].double()[:, None]
    w = torch.where(x > -math.inf, ((x - x[:, :1]) / temp).exp(), 0.0)
    rank = torch.arange(x.shape[1], device="cuda")
    k = t["top_k"].long()[:, None]
    w = torch.where((k <= 0) | (rank < k), w, 0.0)
    run_, p = torch.cumsum(w, -1), t["top_p"].double()[:, None]
    w = torch.where((p >= 1) | (rank == 0) | (run_ - w < p * run_[:, -1:]), w, 0.0)
    w = torch.where((w >= t["min_p"].double()[:, None]) | (rank == 0), w, 0.0)
    run_ = torch.cumsum(w, -1)
    at = (run_ <= t["u"].double()[:, None] * run_[:, -1:]).sum(-1, keepdim=True)
    greedy = temp <= 0
    at = torch.where(greedy, 0, at)
    prob = torch.where(greedy, 1.0, w.gather(1, at) / run_[:, -1:])
    return order.gather(1, at)[:, 0].int(), prob[:, 0].float()


# --- what a pass cannot do without ----------------------------------------------------

def work(case):
    c = case
    size = {"f16": 2, "bf16": 2, "f32": 4}[c["dtype"]]
    if c["kind"] == "norm":
        n = c["T"] * (c["Hq"] + c["Hk"]) * c["d"]
        return dict(bytes=2 * size * n + 4 * c["T"] * bool(c["rot"]), flops=n * (4 + 3 * c["rot"] / c["d"]))
    if c["kind"] == "delta":
        lens = [int(x) for x in c["lens"].split(",")]
        T, S = sum(lens), c["Hv"] * c["dk"] * c["dv"]
        b = size * T * 2 * (c["Hk"] * c["dk"] + c["Hv"] * c["dv"]) + 4 * T * c["Hv"] * (1 + (c["dk"] if c["channel"] else 1))
        return dict(bytes=b + 8 * S * len(lens), flops=7 * T * S)
    n = c["rows"] * c["vocab"]
    return dict(bytes=size * n + 28 * c["rows"], flops=4 * n)


# --- the same results in 64 bits ------------------------------------------------------

def exact(case, seed):
    c, t = case, _inputs(case, seed)
    return {"norm": _exact_norm, "delta": _exact_delta, "sample": _exact_sample}[c["kind"]](c, t)


def _exact_norm(c, t):
    def one(x, w):
        z = x.double()
        power = torch.linalg.vector_norm(z, dim=-1, keepdim=True) ** 2 / (c["d"] if c["mode"] == "rms" else 1)
        z = z * (power + NORM_EPS) ** -0.5 * (1 if w is None else w.double())
        if c["rot"]:
            R = c["rot"]
            pairs = z[..., :R].unflatten(-1, (R // 2, 2) if c["inter"] else (2, R // 2))
            pairs = pairs if c["inter"] else pairs.mT
            turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                               t["positions"].double()[:, None, None] * t["inv_freq"].double())
            pairs = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
            z[..., :R] = (pairs if c["inter"] else pairs.mT).flatten(-2)
        return z
    return one(t["q"], t["q_weight"]), one(t["k"], t["k_weight"])


def _exact_delta(c, t):
    """Token by token, as the rule is defined; the sequences that still have a token side by side."""
    lens = [int(x) for x in c["lens"].split(",")]
    first = t["starts"][:-1].long()
    rep, slots = c["Hv"] // c["Hk"], t["slots"].long()
    out = torch.zeros((sum(lens), c["Hv"], c["dv"]), dtype=torch.float64, device="cuda")
    state = t["state"].double()
    for i in range(max(lens)):
        on = torch.tensor([j for j, n in enumerate(lens) if n > i], device="cuda")
        at, S = first[on] + i, state[slots[on]]
        a = torch.exp(t["g"][at].double())
        S = S * (a[..., None] if c["channel"] else a[..., None, None])
        k, q = (torch.repeat_interleave(t[x][at].double(), rep, dim=1)[..., None] for x in ("k", "q"))
        u = t["beta"][at].double()[..., None] * (t["v"][at].double() - (k * S).sum(-2))
        S = S + k * u[..., None, :]
        out[at] = (q * S).sum(-2) / math.sqrt(c["dk"])
        state[slots[on]] = S
    return out, state


def _exact_sample(c, t):
    probs = []
    for r in range(c["rows"]):
        x, temp = t["logits"][r].double(), float(t["temperature"][r])
        if temp <= 0:
            probs.append(1.0)
            continue
        keep = torch.argsort(-x, stable=True)
        keep = keep[x[keep] > -math.inf]
        if c["k"] > 0:
            keep = keep[:c["k"]]
        p = torch.softmax(x[keep] / temp, 0)
        if float(t["top_p"][r]) < 1:
            before = torch.cat((p.new_zeros(1), torch.cumsum(p, 0)[:-1]))
            p = p[before < float(t["top_p"][r])]
        p = p[p >= float(t["min_p"][r]) * p[0]]
        run_ = torch.cumsum(p / p.sum(), 0)
        at = int(torch.searchsorted(run_, t["u"][r].double(), right=True).clamp(max=len(p) - 1))
        probs.append(float(p[at] / p.sum()))
    return None, torch.tensor(probs, dtype=torch.float64)
