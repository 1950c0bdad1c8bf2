"""Attention over packed sequences in 64 bits, with and without the roundings that the kernels make, and the limits that follow from them.

A bound per element adds what can go wrong at worst, over every key, row and head of a sum: several times the value itself where a key head sums 64
query heads.  Roundings to bf16 are independent of one another and their sum grows with the root of their number, so the NORM of a result's error is
known far more closely: it is what the same roundings cost in 64 bits.  `run(.., rounded=True)` makes them where the kernels do - the
probabilities before P V, ctx, the probabilities and dS before their products, the results - and a result is within its limit if its error's norm is
at most
    1.1 x that of the rounded run over a whole tensor, 2 x over the rows of a tile of 128 and one head      (other bits, as many roundings)
  + 4 P x the norm of the result, P the most by which fp32 scores move a probability: (D + 16) 2^-24 of the largest sum of a score's magnitudes.
lse is fp32 all the way, with a bound per row: the score (D + 4 roundings of at most 2^-24 of the sum of magnitudes), the factors log2 e, ln 2 and the scale
(8 of the value), a sum over n keys (n)."""
import math

import torch

TILE = 128
WHOLE, BLOCK = 1.1, 2.0


def bf16(x):
    return x.float().to(torch.bfloat16).double()


def visible(n, left, right, mask, device):
    i = torch.arange(n, device=device)
    gap = i[None, :] - i[:, None]
    see = torch.ones((n, n), dtype=torch.bool, device=device)
    if left >= 0:
        see &= gap >= -left
    if right >= 0:
        see &= gap <= right
    return see if mask is None else see & (mask != 0)[None, :]


def reach(i, n, left, right):
    """keys inside row i's window, masked ones among them"""
    return (n - 1 if right < 0 else min(i + right, n - 1)) - (0 if left < 0 else max(i - left, 0)) + 1


def from_probabilities(n, left, right, device):
    """rows whose tile takes delta from the probabilities: its first or last row reaches at most 64 keys"""
    out = torch.zeros(n, dtype=torch.bool, device=device)
    for a in range(0, n, TILE):
        e = min(a + TILE, n)
        out[a:e] = min(reach(a, n, left, right), reach(e - 1, n, left, right)) <= 64
    return out


def lagging(s, see):
    """The running maximum that is taken off the scores of each tile of 64 keys (in log2), and the last one: rows in groups of 32, left as it is while no row
    of the group outgrows it by more than 2^20.  P is rounded beside it, so which bits of a probability are lost depends on it."""
    n = s.shape[0]
    rows = -(-n // 32) * 32
    x = torch.full((rows, n), -math.inf, dtype=s.dtype, device=s.device)
    x[:n] = torch.where(see, s / math.log(2.0), -math.inf)
    m, used = torch.full((rows,), -1e30, dtype=s.dtype, device=s.device), []
    for a in range(0, n, 64):
        top = x[:, a:a + 64].amax(1)
        grown = (top > m + 20).view(-1, 32).any(1).repeat_interleave(32)
        m = torch.where(grown, torch.maximum(m, top), m)
        used.append(m[:n, None].expand(n, min(64, n - a)))
    return torch.cat(used, 1), m[:n, None]


def run(q, k, v, dctx, lens, left, right, mask, scale, rounded=False, plant=None, noise=0.0):
    """{ctx, lse, dq, dk, dv, lse_tol, moved}; moved is P above.  noise: what fp32 may move a probability by, at random.
    plant, for tests of the limits: ("step", row, head): 64 rows of one query head are missing in dk and dv; ("head", h): all of its rows are; ("delta",): no
    delta; ("ctx delta",): delta from the stored ctx everywhere; ("max",): lse without its sum; ("lag",): the sums of the first 64 keys are not
    scaled when the maximum grows."""
    what = plant[0] if plant else None
    (T, H, D), Hk, dev = q.shape, k.shape[1], q.device
    G = H // Hk
    z = lambda *s: torch.zeros(s, dtype=torch.float64, device=dev)  # noqa: E731
    r = {"ctx": z(T, H, D), "lse": z(H, T) - math.inf, "dq": z(T, H, D), "dk": z(T, Hk, D), "dv": z(T, Hk, D), "lse_tol": z(H, T), "moved": 0.0}
    rnd = bf16 if rounded else (lambda x: x)
    gen = torch.Generator(device=dev).manual_seed(1)
    a = 0
    for n in lens:
        e = a + n
        if n == 0:
            continue
        mk = None if mask is None else mask[a:e]
        see = visible(n, left, right, mk, dev)
        exact_delta = from_probabilities(n, left, right, dev)[:, None]
        for h in range(H):
            Q, K, V, dO = q[a:e, h].double(), k[a:e, h // G].double(), v[a:e, h // G].double(), dctx[a:e, h].double()
            s = (Q @ K.t() * scale).masked_fill(~see, -math.inf)
            top = s.amax(1, keepdim=True)
            there = top > -math.inf
            m, last = lagging(s, see)
            s2 = torch.where(see, s / math.log(2.0), -math.inf)
            w, back = torch.exp2(s2 - m), torch.exp2(m - last)
            if what == "lag":
                back[:, :64] = 1.0
            w = w * (1 + noise * torch.randn(w.shape, generator=gen, dtype=w.dtype, device=dev)) if noise else w
            total = (w * back).sum(1, keepdim=True)
            lse = torch.where(there, (last + torch.log2(total)) * math.log(2.0), top)
            o = torch.where(there, (rnd(w) * back) @ V / torch.where(there, total, 1.0), 0.0)
            o_stored = rnd(o)
            sizes = (Q.abs() @ K.abs().t() * scale).masked_fill(~see, 0.0).amax(1)
            r["ctx"][a:e, h], r["lse"][h, a:e] = o_stored, (top if what == "max" else lse)[:, 0]
            r["lse_tol"][h, a:e] = 2.0 ** -24 * ((D + 4) * sizes + 8 * (lse[:, 0].abs() + torch.where(there, top, 0.0)[:, 0].abs()) + n + 32)
            r["moved"] = max(r["moved"], (D + 16) * 2.0 ** -24 * float(sizes.max()))
            p = torch.where(see, torch.exp(s - torch.where(there, lse, 0.0)), 0.0)
            p = p * (1 + noise * torch.randn(p.shape, generator=gen, dtype=p.dtype, device=dev)) if noise else p
            dp = dO @ V.t()
            delta = (p * dp).sum(1, keepdim=True)
            if rounded:
                stored = (dO * o_stored).sum(1, keepdim=True)
                delta = stored if what == "ctx delta" else torch.where(exact_delta, delta, stored)
            if what == "delta":
                delta = torch.zeros_like(delta)
            ds, pr = rnd(p * (dp - delta)), rnd(p)
            r["dq"][a:e, h] = rnd(ds @ K * scale)
            if what == "head" and h == plant[1]:
                continue
            if what == "step" and h == plant[2]:
                ds[plant[1]:plant[1] + 64], pr[plant[1]:plant[1] + 64] = 0.0, 0.0
            r["dk"][a:e, h // G] += ds.t() @ Q * scale
            r["dv"][a:e, h // G] += pr.t() @ dO
        a = e
    r["dk"], r["dv"] = rnd(r["dk"]), rnd(r["dv"])
    return r


def beyond(got, val, emu, lens):
    """what of `got` is outside its limits: [(tensor, sequence's first row, tile, head, error / limit)]"""
    bad, moved = [], 4 * val["moved"]
    off = (got["lse"].double() - val["lse"]).abs() / val["lse_tol"]
    off = torch.where(val["lse"] == -math.inf, torch.where(got["lse"].double() == val["lse"], 0.0, math.inf), off)
    if not bool((off[:, :sum(lens)] <= 1.0).all()):
        bad.append(("lse", 0, 0, 0, float(off[:, :sum(lens)].max())))
    for name in ("ctx", "dq", "dk", "dv"):
        if name not in got:
            continue
        err, due, size = got[name].double() - val[name], emu[name] - val[name], val[name]
        lim = WHOLE * due.norm() + moved * size.norm()
        if not bool(err.norm() <= lim):
            bad.append((name, "all", "all", "all", float(err.norm() / lim)))
        a = 0
        for n in lens:
            for t in range(a, a + n, TILE):
                rows = slice(t, min(t + TILE, a + n))
                if (rows.stop - rows.start) * size.shape[2] < 512:  # (too few for a norm to be near what it is on average)
                    continue
                of = lambda x: x[rows].pow(2).sum((0, 2)).sqrt()  # noqa: E731
                lim = BLOCK * of(due) + moved * of(size)
                worse = of(err) / lim.clamp(min=1e-300)
                for h in (~(worse <= 1.0)).nonzero().flatten().tolist():
                    bad.append((name, a, (t - a) // TILE, h, float(worse[h])))
            a += n
    return bad


def inputs(lens, H, Hk, D, masked, seed, spread, device):
    g = torch.Generator(device=device).manual_seed(seed)
    T = sum(lens)
    r = lambda h, by=1.0: (torch.randn((T, h, D), generator=g, device=device) * by).to(torch.bfloat16)  # noqa: E731
    mask = (torch.rand(T, generator=g, device=device) >= masked).to(torch.int32) if masked else None
    off = torch.tensor([0] + list(torch.tensor(lens).cumsum(0)), dtype=torch.int32, device=device)
    return r(H, spread), r(Hk, spread), r(Hk), r(H), mask, off
