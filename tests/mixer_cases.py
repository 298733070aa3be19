"""Plain 64-bit forms of the head norm, the gated delta rule and the token choice, and the
inputs that their tests share. Written from the formulas; tensors on any device."""
import math

import numpy as np
import torch

HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}  # half a step
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}  # half a subnormal step
U32 = 2.0 ** -24


def gen(seed, device):
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    return g


def normal(g, shape, dtype=torch.float32, std=1.0, mean=0.0):
    return (torch.randn(shape, generator=g, device=g.device) * std + mean).to(dtype)


# --- head norm --------------------------------------------------------------------------

def head_norm64(x, w, mode, eps, positions=None, inv_freq=None, interleaved=False):
    """(y, the sum of the two magnitudes a rotated value is made of) in f64."""
    z = x.double()
    s = (z * z).mean(-1, keepdim=True) if mode == "rms" else (z * z).sum(-1, keepdim=True)
    z = z / torch.sqrt(s + eps)
    if w is not None:
        z = z * w.double()
    size = z.abs()
    if inv_freq is not None and inv_freq.numel():
        half, R = inv_freq.numel(), 2 * inv_freq.numel()
        ang = positions.double()[:, None, None] * inv_freq.double()
        c, s = torch.cos(ang), torch.sin(ang)
        p = torch.arange(half, device=x.device)
        ia, ib = (2 * p, 2 * p + 1) if interleaved else (p, p + half)
        a, b = z[..., ia], z[..., ib]
        z, size = z.clone(), size.clone()
        z[..., ia], z[..., ib] = a * c - b * s, b * c + a * s
        size[..., ia] = size[..., ib] = a.abs() + b.abs()
    return z, size


def check_head_norm(got, x, w, mode, eps, positions=None, inv_freq=None, interleaved=False):
    """One rounding of the element type over f32 arithmetic: the sum of squares is off by at
    most d 2^-24 of itself, half of that in its root; the root, quotient, two products, the
    rotation's two and its sum, and the cosine and sine (2 ulp, their angle 2^-22 of a
    radian) are within 32 2^-24 of the magnitudes that meet in a value."""
    want, size = head_norm64(x, w, mode, eps, positions, inv_freq, interleaved)
    d = x.shape[-1]
    bound = HALF[x.dtype] * want.abs() * (1 + 2.0 ** -10) + TINY[x.dtype] + (d / 2 + 32) * U32 * size
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), float((off / bound).max())


# --- gated delta rule -------------------------------------------------------------------

def unit(x, dtype):
    return (x / x.square().sum(-1, keepdim=True).sqrt()).to(dtype)


def delta_inputs(seed, device, T, Hk, Hv, dk, dv, channel, n_slots, dtype=torch.float16, packed=False):
    g = gen(seed, device)
    q, k = unit(normal(g, (T, Hk, dk)), dtype), unit(normal(g, (T, Hk, dk)), dtype)
    v = normal(g, (T, Hv, dv), dtype)
    if packed:  # slices of one row a token, with something behind them
        row = torch.cat([q.flatten(1), k.flatten(1), v.flatten(1), normal(g, (T, 24), dtype)], 1)
        n = Hk * dk
        q, k, v = row[:, :n].view(T, Hk, dk), row[:, n:2 * n].view(T, Hk, dk), row[:, 2 * n:2 * n + Hv * dv].view(T, Hv, dv)
    rate = torch.exp(torch.rand((Hv, dk) if channel else (Hv,), generator=g, device=device) * 6 - 4)
    soft = torch.nn.functional.softplus(normal(g, (T, Hv, dk) if channel else (T, Hv), std=1.0, mean=-1.0))
    return dict(q=q, k=k, v=v, g=-rate * soft, beta=torch.sigmoid(normal(g, (T, Hv))),
                state=normal(g, (n_slots, Hv, dk, dv), std=0.3))


def delta64(q, k, v, g, beta, state, starts, src, dst, scale):
    """(out, state, what the sizes of the values were) in f64, token by token. out is None where no
    sequence has the row. `src` / `dst` are lists; slots named by several sequences keep theirs."""
    T, Hk, dk = q.shape
    Hv, dv, n = v.shape[1], v.shape[2], len(starts) - 1
    q, k = (x.double().repeat_interleave(Hv // Hk, 1) for x in (q, k))
    a = torch.exp(g.double())
    a = a if a.dim() == 3 else a[..., None]
    out = torch.full((T, Hv, dv), math.nan, dtype=torch.float64, device=q.device)
    size = torch.zeros((T, Hv), dtype=torch.float64, device=q.device)
    old, new = state.double(), state.double().clone()
    biggest = torch.zeros((n, Hv), dtype=torch.float64, device=q.device)
    ok = lambda s: 0 <= s < state.shape[0]  # noqa: E731
    for i in range(n):
        S = old[src[i]].clone() if ok(src[i]) else torch.zeros((Hv, dk, dv), dtype=torch.float64, device=q.device)
        big = S.square().sum((1, 2)).sqrt()
        for t in range(starts[i], starts[i + 1]):
            S = S * a[t][:, :, None]
            u = beta[t].double()[:, None] * (v[t].double() - torch.matmul(k[t][:, None], S)[:, 0])
            S = S + k[t][:, :, None] * u[:, None]
            out[t] = scale * torch.matmul(q[t][:, None], S)[:, 0]
            big = torch.maximum(big, S.square().sum((1, 2)).sqrt() + v[t].double().square().sum(1).sqrt())
            size[t] = big * q[t].square().sum(1).sqrt() * abs(scale)
        biggest[i] = big
        others = [s for j in range(n) if j != i for s in (src[j], dst[j])]
        if ok(dst[i]) and dst[i] not in others:
            new[dst[i]] = S
    return out, new, size, biggest


def check_delta(got, state, want, new, size, biggest, starts, dst, dk):
    """Roundings of random sign: a token's update adds an error of at most 4 sqrt(dk + 16)
    2^-24 of the head's state and value (the dot over dk, the product and the sums; four
    standard deviations), and does not grow older ones (unit keys, decays and beta at most
    1), so after T tokens it is sqrt(T) of that. An output is a product with the query on
    top, and one rounding to its type."""
    n = len(starts) - 1
    for i in range(n):
        T = starts[i + 1] - starts[i]
        rel = 4 * math.sqrt(dk + 16) * U32 * math.sqrt(T + 1)
        if 0 <= dst[i] < state.shape[0]:
            off = (state[dst[i]].double() - new[dst[i]]).square().sum((1, 2)).sqrt()
            assert bool((off <= rel * biggest[i] + 1e-37).all()), (i, float((off / biggest[i]).max()), rel)
        rows = slice(starts[i], starts[i + 1])
        if T:
            o, w = got[rows].double(), want[rows]
            bound = HALF[got.dtype] * (1 + 2.0 ** -10) * w.abs() + TINY[got.dtype] + 2 * rel * size[rows][..., None]
            off = (o - w).abs()
            assert bool((off <= bound).all()), (i, float((off / bound).max()))


# --- token choice -----------------------------------------------------------------------

def choose64(x, u, temp, k, p, min_p):
    """(id, probability, the least distance of u's goal and top-p's to a running weight) of one
    row in f64. x a numpy row."""
    x = x.astype(np.float64)
    ids = np.flatnonzero(~np.isnan(x) & (x > -np.inf))
    if not len(ids):
        return -1, 0.0
    order = ids[np.argsort(-x[ids], kind="stable")]
    if not temp > 0:
        return int(order[0]), 1.0
    s = x[order]
    with np.errstate(invalid="ignore", over="ignore"):
        t = np.where(s == s[0], 0.0, (s[0] - s) / np.float64(temp))
        if s[0] == np.inf:  # those of +inf share the row, at an infinite temperature too (inf / inf above)
            t[s != s[0]] = np.inf
    w = np.exp(-t)
    w[w < 2.0 ** -45] = 0.0
    keep = len(w)
    if k > 0:
        keep = min(keep, k)
    if p < 1:
        total = w[:keep].sum()
        keep = int(np.argmax(np.cumsum(w[:keep]) >= np.float64(np.float32(p)) * total)) + 1
    above = int((w[:keep] >= np.float64(np.float32(min_p))).sum())
    w = w[:max(1, min(keep, above))]
    run = np.cumsum(w)
    over = np.flatnonzero(run > np.float64(u) * run[-1])
    at = over[0] if len(over) else np.flatnonzero(w > 0)[-1]
    return int(order[at]), float(w[at] / run[-1])
