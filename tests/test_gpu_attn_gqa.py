"""ops.attn_gqa_fwd / attn_gqa_bwd (cocodr_attn_gqa_*) against the definition in 64 bits.

Tolerances are bounds per element, from the roundings that the kernels make: the probabilities and dS go to bf16 for the matrix pipe and the
results are stored in bf16 (each off by at most half a step, U = 2^-8 of the value), delta is taken from the stored ctx, and what is computed in
fp32 - scores, exponentials, sums - moves a probability by less than P32 of itself: a score is a sum of at most 128 products (128 x 2^-24 of the
sum of their magnitudes, which stays below 64 here), the exponential and the log-sum-exp add a few 2^-23 of numbers below 64."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -8
P32 = 64 * 128 * 2.0 ** -24 + 64 * 8 * 2.0 ** -23


def visible(n, left, right, mask):
    i = torch.arange(n, device="cuda")
    gap = i[None, :] - i[:, None]
    see = torch.ones((n, n), dtype=torch.bool, device="cuda")
    if left >= 0:
        see &= gap >= -left
    if right >= 0:
        see &= gap <= right
    if mask is not None:
        see &= (mask != 0)[None, :]
    return see


def reference(q, k, v, dctx, lens, left, right, mask, scale):
    """(values, bounds) in 64 bits: ctx, lse, dq, dk, dv of all rows, those of no sequence 0 and -inf"""
    T, H, D = q.shape
    Hk = k.shape[1]
    G = H // Hk
    z = lambda *s: torch.zeros(s, dtype=torch.float64, device="cuda")  # noqa: E731
    val = {"ctx": z(T, H, D), "lse": z(H, T) - math.inf, "dq": z(T, H, D), "dk": z(T, Hk, D), "dv": z(T, Hk, D)}
    tol = {n: torch.zeros_like(x) for n, x in val.items()}
    tol["lse"] = z(H, T)
    a = 0
    for n in lens:
        e = a + n
        if n == 0:
            continue
        mk = None if mask is None else mask[a:e]
        see = visible(n, left, right, mk)
        dead = torch.zeros(n, dtype=torch.bool, device="cuda") if mk is None else mk == 0
        for h in range(H):
            Q, K, V, dO = q[a:e, h].double(), k[a:e, h // G].double(), v[a:e, h // G].double(), dctx[a:e, h].double()
            K, V = K.masked_fill(dead[:, None], 0.0), V.masked_fill(dead[:, None], 0.0)
            s = (Q @ K.t() * scale).masked_fill(~see, -math.inf)
            lse = torch.logsumexp(s, 1)
            p = torch.where(see, torch.exp(s - lse[:, None]), 0.0)
            o = p @ V
            dp = dO @ V.t()
            delta = (dO * o).sum(1, keepdim=True)
            ds = torch.where(see, p * (dp - delta), 0.0)
            val["ctx"][a:e, h], val["lse"][h, a:e] = o, lse
            val["dq"][a:e, h] = ds @ K * scale
            val["dk"][a:e, h // G] += ds.t() @ Q * scale
            val["dv"][a:e, h // G] += p.t() @ dO
            o_off = (U + P32) * (p @ V.abs()) + U * o.abs()
            d_off = (dO.abs() * o_off).sum(1, keepdim=True)
            ds_off = U * ds.abs() + p * (d_off + 2 * P32 * (dO.abs() @ V.abs().t() + delta.abs()))
            tol["ctx"][a:e, h] = o_off
            tol["lse"][h, a:e] = P32 * (1 + lse.abs())
            tol["dq"][a:e, h] = ds_off @ K.abs() * scale
            tol["dk"][a:e, h // G] += ds_off.t() @ Q.abs() * scale
            tol["dv"][a:e, h // G] += (U + P32) * (p.t() @ dO.abs())
        a = e
    for name in ("dq", "dk", "dv"):
        tol[name] += U * val[name].abs()
    for name in ("ctx", "dq", "dk", "dv"):
        tol[name] += 1e-30
    return val, tol


def assert_within(name, got, val, tol):
    got = got.double()
    assert torch.equal(torch.isfinite(got), torch.isfinite(val)), name
    fin = torch.isfinite(val)
    worst = ((got - val).abs() / tol.clamp(min=1e-37))[fin]
    assert worst.numel() == 0 or worst.max().item() <= 1.0, (name, worst.max().item())
    assert torch.equal(got[~fin], val[~fin]), name


def make(lens, H, Hk, D, tail=0, seed=0, fused=True, spread=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    T = sum(lens) + tail
    off = torch.tensor([0] + list(torch.tensor(lens).cumsum(0)), dtype=torch.int32, device="cuda")
    r = lambda *s: torch.randn(s, generator=g, device="cuda").to(torch.bfloat16)  # noqa: E731
    if fused:
        qkv = r(T, (H + 2 * Hk) * D) * spread
        q, k, v = (x.unflatten(1, (-1, D)) for x in qkv.split((H * D, Hk * D, Hk * D), 1))
    else:
        q, k, v = r(H, T, D).transpose(0, 1) * spread, r(T, Hk, D), r(T, Hk, D)
    return q, k, v, r(T, H, D), off


# lens, query heads, key heads, head size, causal, (left, right), share of keys masked out, rows behind, fused
CASES = [
    ([1], 1, 1, 64, False, (-1, -1), 0, 0, True),
    ([1, 1, 1, 2, 3], 2, 1, 128, True, (-1, -1), 0, 0, True),
    ([0, 5, 0, 0, 64, 1, 0], 2, 2, 64, False, (-1, -1), 0, 3, True),
    ([31, 32, 33, 63, 64, 65, 127, 128, 129], 4, 2, 64, True, (-1, -1), 0, 0, True),
    ([31, 32, 33, 63, 64, 65, 127, 128, 129], 4, 1, 128, False, (-1, -1), 0, 5, True),
    ([257, 300], 3, 3, 80, True, (-1, -1), 0, 0, False),
    ([200, 77], 6, 2, 96, False, (-1, -1), 0.3, 0, False),
    ([129, 64], 2, 1, 8, True, (-1, -1), 0.2, 1, True),
    ([100, 31], 2, 2, 16, False, (7, 3), 0, 0, True),
    ([513], 4, 4, 64, False, (64, 64), 0, 0, True),
    ([700, 130, 1], 4, 1, 128, True, (100, 0), 0.1, 2, True),
    ([400], 2, 1, 128, False, (0, 0), 0, 0, True),
    ([400, 65], 2, 1, 64, False, (0, 500), 0.5, 0, True),
    ([333, 260], 2, 2, 128, False, (-1, 20), 0, 0, False),
    ([333, 260], 2, 1, 64, False, (20, -1), 0.9, 0, False),
    ([1100], 8, 2, 128, True, (-1, -1), 0, 0, True),
    ([40] * 70 + [3] * 70, 1, 1, 64, True, (-1, -1), 0, 9, True),   # more than 64 sequences: the search for a tile's sequence takes two steps
    ([5] * 256, 1, 1, 32, True, (-1, -1), 0.1, 0, True),             # 256: the most that are numbered without gaps
    ([130, 5] * 128 + [1], 1, 1, 32, False, (-1, -1), 0, 3, True),
    ([2] * 4200, 1, 1, 32, False, (-1, -1), 0, 0, True),            # ... three
    ([256, 128], 32, 8, 72, True, (-1, -1), 0, 0, True),
]


# long and few sequences: tiles in the order of their work, the heads of a group summed in parts, one sequence far longer than the rest
CASES += [
    ([1500, 3, 0, 700, 64, 129], 8, 2, 64, True, (-1, -1), 0, 7, True),
    ([3, 1500, 0, 129, 700, 64], 4, 1, 128, False, (-1, -1), 0.1, 0, True),
    ([64, 1300, 600], 8, 1, 64, False, (-1, 40), 0, 0, False),
    ([600, 0, 1300], 4, 2, 128, False, (40, -1), 0.3, 2, True),
    ([1000, 1000, 1000], 2, 2, 128, True, (-1, -1), 0.2, 0, True),
    ([257] * 63 + [300], 1, 1, 16, True, (-1, -1), 0, 0, True),
    ([1900, 1], 8, 1, 32, True, (900, -1), 0, 0, True),
    ([300], 64, 1, 64, False, (-1, -1), 0, 0, True),                 # the 64 query heads of one key head in up to 8 parts
    ([2100], 1, 1, 128, False, (-1, -1), 0.1, 5, True),              # one head's 33 tiles of queries in two parts
    ([2500], 2, 1, 64, True, (-1, -1), 0.3, 0, True),
    ([1800, 60], 1, 1, 80, False, (1500, 300), 0, 9, False),
    ([3, 2200], 2, 2, 32, False, (-1, 700), 0.6, 0, True),
    ([1500, 90], 6, 2, 72, True, (-1, -1), 0, 0, True),              # three heads: parts begin inside a head
    ([700, 40], 32, 1, 128, True, (-1, -1), 0.1, 0, False),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{len(c[0])}x{max(c[0])}-h{c[1]}k{c[2]}d{c[3]}-{'causal' if c[4] else 'full'}{c[5]}-m{c[6]}")
def test_forward_and_backward(case):
    from cocodr_amd import ops
    lens, H, Hk, D, causal, window, masked, tail, fused = case
    q, k, v, dctx, off = make(lens, H, Hk, D, tail, seed=len(lens) + D, fused=fused)
    mask = None
    if masked:
        g = torch.Generator(device="cuda").manual_seed(7)
        mask = (torch.rand(q.shape[0], generator=g, device="cuda") >= masked).to(torch.int32) * 5
        mask[off[-2]:off[-1]] = 0  # the last sequence sees nothing at all
    how = dict(causal=causal, window=window, mask=mask)
    ctx, lse = ops.attn_gqa_fwd(q, k, v, off, **how)
    dq, dk, dv = ops.attn_gqa_bwd(q, k, v, ctx, dctx, lse, off, **how)
    val, tol = reference(q, k, v, dctx, lens, window[0], 0 if causal else window[1], mask, D ** -0.5)
    for name, got in (("ctx", ctx), ("lse", lse), ("dq", dq), ("dk", dk), ("dv", dv)):
        assert_within(name, got, val[name], tol[name])
    again = ops.attn_gqa_bwd(q, k, v, ctx, dctx, lse, off, **how)
    assert all(torch.equal(x, y) for x, y in zip((dq, dk, dv), again))


def test_peaked_scores_and_a_scale_of_its_own():
    """scores of several hundred: the running maximum moves by more than it may be left standing, and most probabilities vanish"""
    from cocodr_amd import ops
    lens, H, Hk, D = [300, 190], 2, 1, 64
    q, k, v, dctx, off = make(lens, H, Hk, D, seed=3, spread=4.0)
    ctx, lse = ops.attn_gqa_fwd(q, k, v, off, scale=0.25)
    val, tol = reference(q, k, v, dctx, lens, -1, -1, None, 0.25)
    # the scores are up to 16 times those that P32 counts (q and k 4 times as large, the scale twice: sums of magnitudes below 2048)
    more = 32
    assert_within("lse", lse, val["lse"], tol["lse"] * more)
    assert_within("ctx", ctx, val["ctx"], tol["ctx"] + (more * P32) * v.double().abs().amax())


def test_masked_rows_may_hold_anything_and_tokens_behind_do_not_count():
    from cocodr_amd import ops
    lens, H, Hk, D = [90, 200, 17], 4, 2, 64
    q, k, v, dctx, off = make(lens, H, Hk, D, tail=40, seed=5, fused=False)
    mask = torch.ones(q.shape[0], dtype=torch.int32, device="cuda")
    mask[20:50] = 0
    mask[100] = 0
    base = ops.attn_gqa_fwd(q, k, v, off, mask=mask)
    grads = ops.attn_gqa_bwd(q, k, v, base[0], dctx, base[1], off, mask=mask)
    bad = mask == 0
    bad[sum(lens):] = True
    k2, v2 = k.clone(), v.clone()
    k2[bad], v2[bad] = float("nan"), float("inf")
    got = ops.attn_gqa_fwd(q, k2, v2, off, mask=mask)
    assert torch.equal(got[0], base[0]) and torch.equal(got[1], base[1])
    g2 = ops.attn_gqa_bwd(q, k2, v2, base[0], dctx, base[1], off, mask=mask)
    assert all(torch.equal(x, y) for x, y in zip(grads, g2))
    assert float(grads[1][20:50].abs().max()) == 0 and float(grads[2][20:50].abs().max()) == 0


def test_rows_of_no_sequence():
    """zeros in fresh results, untouched in those that the caller gave - also views of one fused gradient"""
    from cocodr_amd import ops
    lens, H, Hk, D = [30, 140], 2, 1, 64
    q, k, v, dctx, off = make(lens, H, Hk, D, tail=70, seed=6)
    off = off + 9  # nine rows in front, too
    ctx, lse = ops.attn_gqa_fwd(q, k, v, off, causal=True)
    grads = ops.attn_gqa_bwd(q, k, v, ctx, dctx, lse, off, causal=True)
    outside = torch.ones(q.shape[0], dtype=torch.bool, device="cuda")
    outside[9:179] = False
    for t in (ctx,) + grads:
        assert torch.count_nonzero(t[outside]) == 0 and torch.isfinite(t.float()).all()
    assert (lse[:, outside] == -math.inf).all() and torch.isfinite(lse[:, ~outside]).all()
    buf = torch.full((q.shape[0], H, D), 7.0, dtype=torch.bfloat16, device="cuda")
    c2, _ = ops.attn_gqa_fwd(q, k, v, off, causal=True, out=buf)
    assert c2 is buf and (buf[outside] == 7).all() and torch.equal(buf[~outside], ctx[~outside])
    fused = torch.full((q.shape[0], (H + 2 * Hk) * D), 3.0, dtype=torch.bfloat16, device="cuda")
    views = tuple(x.unflatten(1, (-1, D)) for x in fused.split((H * D, Hk * D, Hk * D), 1))
    ops.attn_gqa_bwd(q, k, v, ctx, dctx, lse, off, causal=True, out=views)
    assert (fused[outside] == 3).all() and all(torch.equal(x[~outside], y[~outside]) for x, y in zip(views, grads))


def test_row_offsets_behind_two_gib():
    """a token stride that carries the last rows past 2^31 elements"""
    from cocodr_amd import ops
    T, D, ld = 600, 64, 1 << 22
    big = torch.zeros((T * ld,), dtype=torch.bfloat16, device="cuda")
    q, k, v = (torch.as_strided(big, (T, 1, D), (ld, D, 1), o) for o in (0, 64, 128))
    sq, sk, sv, dctx, off = make([T], 1, 1, D, seed=8, fused=False)
    q.copy_(sq), k.copy_(sk), v.copy_(sv)
    a, b = ops.attn_gqa_fwd(q, k, v, off, causal=True), ops.attn_gqa_fwd(sq, sk, sv, off, causal=True)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    ga, gb = (ops.attn_gqa_bwd(*t, a[0], dctx, a[1], off, causal=True) for t in ((q, k, v), (sq, sk, sv)))
    assert all(torch.equal(x, y) for x, y in zip(ga, gb))


def test_head_major_tensors_and_heads_that_share_their_memory():
    """[heads, T, dim] tensors seen as [T, heads, dim], and keys and values whose heads (or rows) are one in memory"""
    from cocodr_amd import ops
    q, k, v, dctx, off = make([90, 230], 4, 2, 64, seed=15, fused=False)
    turn = lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)  # noqa: E731
    want = ops.attn_gqa_fwd(q, k, v, off, causal=True)
    grads = ops.attn_gqa_bwd(q, k, v, want[0], dctx, want[1], off, causal=True)
    ctx = turn(torch.empty_like(dctx))
    got = ops.attn_gqa_fwd(turn(q), turn(k), turn(v), off, causal=True, out=ctx)
    assert got[0] is ctx and torch.equal(ctx, want[0]) and torch.equal(got[1], want[1])
    outs = tuple(turn(torch.empty(t.shape, dtype=torch.bfloat16, device="cuda")) for t in (q, k, v))
    ops.attn_gqa_bwd(turn(q), turn(k), turn(v), ctx, turn(dctx), want[1], off, causal=True, out=outs)
    assert all(torch.equal(x, y) for x, y in zip(outs, grads))
    for one in (k[:, :1].expand(-1, 2, -1), k[:1].expand(320, -1, -1)):
        a, b = (ops.attn_gqa_fwd(q, t, v, off, causal=True) for t in (one, one.contiguous()))
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        ga, gb = (ops.attn_gqa_bwd(q, t, v, a[0], dctx, a[1], off, causal=True) for t in (one, one.contiguous()))
        assert all(torch.equal(x, y) for x, y in zip(ga, gb))


@pytest.mark.parametrize("stride", [7, 8, 1 << 24, 1 << 31])
def test_a_single_row_with_any_stride(stride):
    """what stands between the rows of one row does not count, whatever a view says it is"""
    from cocodr_amd import ops
    q, k, v, dctx, off = make([1], 4, 2, 128, seed=14, fused=False)
    q, k, v, dctx = (t.contiguous() for t in (q, k, v, dctx))
    odd = [torch.as_strided(t, t.shape, (stride, 128, 1)) for t in (q, k, v, dctx)]
    a, b = ops.attn_gqa_fwd(q, k, v, off), ops.attn_gqa_fwd(*odd[:3], off)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    ga, gb = (ops.attn_gqa_bwd(*t[:3], a[0], t[3], a[1], off) for t in ((q, k, v, dctx), odd))
    assert all(torch.equal(x, y) for x, y in zip(ga, gb))


def test_another_stream_and_a_captured_graph():
    from cocodr_amd import ops
    lens, H, Hk, D = [100, 260, 3], 4, 2, 128
    q, k, v, dctx, off = make(lens, H, Hk, D, seed=9)
    want = ops.attn_gqa_fwd(q, k, v, off, causal=True)
    want += ops.attn_gqa_bwd(q, k, v, want[0], dctx, want[1], off, causal=True)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = ops.attn_gqa_fwd(q, k, v, off, causal=True)
        got += ops.attn_gqa_bwd(q, k, v, got[0], dctx, got[1], off, causal=True)
    s.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.attn_gqa_fwd(q, k, v, off, causal=True)
        out += ops.attn_gqa_bwd(q, k, v, out[0], dctx, out[1], off, causal=True)
    for seed in (11, 12, 13):
        q2, k2, v2, d2, _ = make(lens, H, Hk, D, seed=seed)
        for t, x in ((q, q2), (k, k2), (v, v2), (dctx, d2)):
            t.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        eager = ops.attn_gqa_fwd(q, k, v, off, causal=True)
        eager += ops.attn_gqa_bwd(q, k, v, eager[0], dctx, eager[1], off, causal=True)
        assert all(torch.equal(x, y) for x, y in zip(out, eager))


def test_gradient_against_differences():
    """directional differences of the forward in 64 bits of the same definition: the gradient is that of the function, not only of its formula"""
    from cocodr_amd import ops
    lens, H, Hk, D = [50, 21], 2, 1, 32
    q, k, v, dctx, off = make(lens, H, Hk, D, seed=10, fused=False)
    ctx, lse = ops.attn_gqa_fwd(q, k, v, off, causal=True)
    grads = ops.attn_gqa_bwd(q, k, v, ctx, dctx, lse, off, causal=True)
    _, tol = reference(q, k, v, dctx, lens, -1, 0, None, D ** -0.5)
    f = lambda a, b, c: (reference(a, b, c, dctx, lens, -1, 0, None, D ** -0.5)[0]["ctx"] * dctx.double()).sum()  # noqa: E731
    base = [t.double() for t in (q, k, v)]
    for n, name in enumerate(("dq", "dk", "dv")):
        d = torch.randn(base[n].shape, generator=torch.Generator(device="cuda").manual_seed(n), device="cuda", dtype=torch.float64)
        h = 1e-5
        up, down = list(base), list(base)
        up[n], down[n] = base[n] + h * d, base[n] - h * d
        slope = (f(*up) - f(*down)) / (2 * h)  # off by h^2 third derivatives: far below the gradients' own bound
        got = (grads[n].double() * d).sum()
        assert (got - slope).abs() <= (tol[name] * d.abs()).sum()


def test_refusals_on_the_device():
    from cocodr_amd import ops
    q, k, v, dctx, off = make([64], 4, 2, 64, seed=1, fused=False)
    with pytest.raises(ValueError, match="multiple of kv_heads"):
        ops.attn_gqa_fwd(q[:, :3], k, v, off)
    with pytest.raises(ValueError, match="dtype"):
        ops.attn_gqa_fwd(q.half(), k, v, off)
    with pytest.raises(ValueError, match="shape"):
        ops.attn_gqa_fwd(q, k, v[:32], off)
    with pytest.raises(ValueError, match="k: expected shape"):
        ops.attn_gqa_fwd(q, k[:63], v[:63], off)
    with pytest.raises(ValueError, match="k: expected shape"):
        ops.attn_gqa_fwd(q, k[:, :, :32], v, off)
    with pytest.raises(ValueError, match="adjacent"):
        ops.attn_gqa_fwd(q, k.transpose(1, 2).contiguous().transpose(1, 2), v, off)
    with pytest.raises(ValueError, match="16-byte"):
        ops.attn_gqa_fwd(torch.empty(64 * 4 * 64 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(64, 4, 64), k, v, off)
    with pytest.raises(ValueError, match="multiples of 8"):
        ops.attn_gqa_fwd(torch.empty((64, 4, 65), dtype=torch.bfloat16, device="cuda")[:, :, :64], k, v, off)
    with pytest.raises(ValueError, match="seq_off"):
        ops.attn_gqa_fwd(q, k, v, off.long())
    with pytest.raises(ValueError, match="causal"):
        ops.attn_gqa_fwd(q, k, v, off, causal=True, window=(3, 3))
    with pytest.raises(ValueError, match="window"):
        ops.attn_gqa_fwd(q, k, v, off, window=(-2, 0))
    with pytest.raises(ValueError, match="scale"):
        ops.attn_gqa_fwd(q, k, v, off, scale=-1.0)
    with pytest.raises(ValueError, match="mask"):
        ops.attn_gqa_fwd(q, k, v, off, mask=torch.ones(63, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError, match="apart"):
        ops.attn_gqa_fwd(q, k, v, off, out=torch.empty((64, 1, 64), dtype=torch.bfloat16, device="cuda").expand(64, 4, 64))
    ctx, lse = ops.attn_gqa_fwd(q, k, v, off)
    with pytest.raises(ValueError, match="lse"):
        ops.attn_gqa_bwd(q, k, v, ctx, dctx, lse.t().contiguous(), off)
    with pytest.raises(ValueError, match="GPU"):
        ops.attn_gqa_bwd(q, k, v, ctx, dctx.cpu(), lse, off)
