"""ops.embed_fwd / embed_bwd (cocodr_embed_*) and ops.dropout_fwd / dropout_bwd (cocodr_dropout_*) against their definitions in 64 bits.

One rounding to the result's type is off by at most half a step: 2^-8 of the value in bf16, 2^-24 in fp32; the scaling multiplies in fp32 (2^-24
more).  A sum of c rows in fp32 is off by at most c 2^-24 of the sum of their magnitudes."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def ids_of(kind, n, V, seed, dtype=torch.int32):
    g = np.random.default_rng(seed)
    if kind == "one":
        x = np.full(n, V // 2)
    elif kind == "text":
        x = np.minimum((np.exp(g.random(n) * np.log(V + 1)) - 1).astype(np.int64), V - 1)
    elif kind == "distinct":
        x = g.permutation(max(n, V))[:n] % V
    elif kind == "two":
        x = np.where(g.random(n) < 0.7, 0, V - 1)
    else:  # padding of all kinds among the others
        x = g.integers(-3, V + 3, n)
    return torch.tensor(x, dtype=dtype, device="cuda")


@pytest.mark.parametrize("table,out", [(torch.float32, torch.bfloat16), (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float32, torch.float32)])
@pytest.mark.parametrize("n,V,H,idt", [(1, 1, 8, torch.int32), (7, 100, 768, torch.int64), (300, 50, 776, torch.int32), (2050, 997, 64, torch.int64), (33, 5, 4096, torch.int32)])
def test_embed_fwd(n, V, H, idt, table, out):
    from cocodr_amd import ops
    E = torch.randn((V, H), generator=torch.Generator(device="cuda").manual_seed(n), device="cuda").to(table)
    ids = ids_of("pads", n, V, n, idt)
    got = ops.embed_fwd(ids, E, scale=27.7128, out_dtype=out)
    ok = (ids >= 0) & (ids < V)
    s = float(np.float32(27.7128))
    want = torch.where(ok[:, None], E.double()[ids.clamp(0, V - 1).long()] * s, 0.0)
    assert got.dtype == out and got.shape == (n, H)
    assert ((got.double() - want).abs() <= want.abs() * (HALF[out] + 2.0 ** -23)).all()
    assert torch.equal(ops.embed_fwd(ids.view(1, n, 1), E, scale=27.7128, out_dtype=out).view(n, H), got)


BWD = [("text", 1, 1, 8), ("one", 1, 2, 8), ("one", 3, 9, 8), ("text", 64, 3, 64), ("one", 64, 4, 768), ("one", 65, 4, 768), ("one", 5000, 10, 520), ("one", 40000, 9, 64), ("two", 9000, 1025, 1032),
       ("text", 8192, 30522, 768), ("pads", 777, 40, 40), ("pads", 20000, 100, 16), ("distinct", 4096, 5000, 128), ("text", 33333, 2000, 264), ("two", 140000, 2, 8)]


@pytest.mark.parametrize("kind,n,V,H", BWD)
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_embed_bwd(kind, n, V, H, dt):
    from cocodr_amd import ops
    ids = ids_of(kind, n, V, n, torch.int64 if n % 2 else torch.int32)
    dout = torch.randn((n, H), generator=torch.Generator(device="cuda").manual_seed(n), device="cuda").to(dt)
    ok = (ids >= 0) & (ids < V)
    at = ids[ok].long()
    s = 0.5
    want = torch.zeros((V, H), dtype=torch.float64, device="cuda").index_put_((at,), dout[ok].double() * s, accumulate=True)
    size = torch.zeros((V, H), dtype=torch.float64, device="cuda").index_put_((at,), dout[ok].double().abs() * s, accumulate=True)
    count = torch.bincount(at, minlength=V).double()
    tol = size * (count[:, None] + 2) * 2.0 ** -24
    got = ops.embed_bwd(dout, ids, V, scale=s)
    assert ((got.double() - want).abs() <= tol).all()
    assert torch.equal(got, ops.embed_bwd(dout, ids, V, scale=s))  # the same bits
    base = torch.randn((V, H), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    acc = base.clone()
    assert ops.embed_bwd(dout, ids, V, scale=s, out=acc, accumulate=True) is acc
    assert ((acc.double() - base.double() - want).abs() <= tol + (base.abs().double() + want.abs()) * 2.0 ** -23).all()
    assert torch.equal(acc[count == 0], base[count == 0])
    out = torch.full((V, H), float("nan"), device="cuda")
    assert torch.equal(ops.embed_bwd(dout, ids, V, scale=s, out=out), got)


def test_embed_without_tokens():
    from cocodr_amd import ops
    ids = torch.empty((0,), dtype=torch.int32, device="cuda")
    assert ops.embed_fwd(ids, torch.ones((4, 16), device="cuda")).shape == (0, 16)
    dout = torch.empty((0, 16), dtype=torch.bfloat16, device="cuda")
    assert torch.count_nonzero(ops.embed_bwd(dout, ids, 5, out=torch.ones((5, 16), device="cuda"))) == 0
    kept = torch.ones((5, 16), device="cuda")
    assert (ops.embed_bwd(dout, ids, 5, out=kept, accumulate=True) == 1).all()
    nowhere = torch.full((300,), -1, dtype=torch.int32, device="cuda")
    assert torch.count_nonzero(ops.embed_bwd(torch.ones((300, 16), device="cuda"), nowhere, 5)) == 0


def test_embed_rows_behind_four_gib():
    """a table whose last rows lie past 2^32 bytes and past 2^31 elements"""
    from cocodr_amd import ops
    V, H = 530000, 4096
    E = torch.zeros((V, H), dtype=torch.bfloat16, device="cuda")
    ids = torch.tensor([V - 1, 0, V - 2, V - 1], dtype=torch.int32, device="cuda")
    E[V - 1], E[V - 2] = 2.0, 3.0
    got = ops.embed_fwd(ids, E, scale=2.0)
    assert [float(x) for x in got[:, -1]] == [4.0, 0.0, 6.0, 4.0]
    del E
    g = ops.embed_bwd(torch.ones((4, H), dtype=torch.bfloat16, device="cuda"), ids, V)
    assert [float(g[i, -1]) for i in (0, 1, V - 2, V - 1)] == [1.0, 0.0, 1.0, 2.0]


def keep_of(dm, n):
    """the mask's definition (include/cocodr.h "Dropout"), in numpy"""
    pair = np.arange((n + 1) // 2, dtype=np.uint32)
    w = pair ^ np.uint32(dm.k0)
    w ^= w >> np.uint32(16); w *= np.uint32(0x7feb352d); w ^= w >> np.uint32(15); w *= np.uint32(0x846ca68b); w ^= w >> np.uint32(16)
    w ^= np.uint32(dm.k1)
    u = np.stack([w & np.uint32(0xffff), w >> np.uint32(16)], 1).reshape(-1)[:n]
    return torch.tensor(u >= dm.threshold, device="cuda")


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n,at", [(1, 0), (2, 1), (7, 0), (8, 0), (9, 3), (255, 1), (256 * 768, 0), (100003, 0), (100003, 5), (33 << 15, 0)])
@pytest.mark.parametrize("p", [0.1, 0.5])
def test_dropout(n, at, dt, p):
    """at: how many elements into a tensor the (contiguous) view begins: not every view is 16-byte aligned"""
    from cocodr_amd import ops
    g = torch.Generator(device="cuda").manual_seed(n + at)
    x, r = (torch.randn(n + at, generator=g, device="cuda").to(dt)[at:] for _ in range(2))
    dm = ops.dropout_mask(p, 1234567, n, 3, ops.KIND_FFN_OUT)
    keep, scale = keep_of(dm, n), float(dm.scale)
    want = torch.where(keep, x.double() * scale, 0.0)
    got = ops.dropout_fwd(x, dm)
    assert ((got.double() - want).abs() <= want.abs() * (HALF[dt] + 2.0 ** -23)).all()
    assert torch.equal(got, ops.dropout_bwd(x, dm))
    sum_ = ops.dropout_fwd(x, dm, residual=r)
    w2 = want + r.double()
    assert ((sum_.double() - w2).abs() <= w2.abs() * HALF[dt] + (want.abs() + r.double().abs()) * 2.0 ** -23).all()
    assert torch.equal(sum_[~keep], r[~keep])
    assert torch.equal(ops.dropout_fwd(x, ops.dropout_mask(0.0, 1, 1, 0, 0)), x)


def test_dropout_matches_the_fused_site():
    """the GEMM epilogue that drops the dense output and adds the residual (EPI_ADD) and the operator draw the same mask"""
    from cocodr_amd import _native as N, ops
    g = torch.Generator(device="cuda").manual_seed(0)
    a, w = (torch.randn(s, generator=g, device="cuda").to(torch.bfloat16) for s in ((96, 64), (128, 64)))
    r = torch.zeros((96, 128), dtype=torch.bfloat16, device="cuda")
    dm = ops.dropout_mask(0.2, 99, 5, 2, ops.KIND_ATTN_OUT)
    fused = ops.gemm(a, w, epi=N.EPI_ADD, r=r, drop=dm)
    own = ops.dropout_fwd(ops.gemm(a, w), dm)
    assert torch.equal(fused == 0, own == 0)


def test_dropout_gradient_against_differences():
    from cocodr_amd import ops
    x = torch.randn((31, 65), generator=torch.Generator(device="cuda").manual_seed(2), device="cuda")
    dm = ops.dropout_mask(0.3, 5, 6, 0, ops.KIND_EMBED)
    dy = torch.randn_like(x)
    d = torch.randn_like(x)
    up, down = ops.dropout_fwd(x + d, dm), ops.dropout_fwd(x - d, dm)
    slope = ((up.double() - down.double()) * dy.double()).sum() / 2  # linear: the step may be large
    got = (ops.dropout_bwd(dy, dm).double() * d.double()).sum()
    assert (got - slope).abs() <= 8 * 2.0 ** -24 * ((x.abs() + d.abs()).double() * dy.abs().double()).sum() * float(dm.scale)


def test_embed_gradient_against_differences():
    from cocodr_amd import ops
    V, H, n = 23, 24, 90
    ids = ids_of("pads", n, V, 4)
    g = torch.Generator(device="cuda").manual_seed(3)
    E, d = (torch.randn((V, H), generator=g, device="cuda") for _ in range(2))
    dy = torch.randn((n, H), generator=g, device="cuda")
    f = lambda t: ops.embed_fwd(ids, t, scale=3.0, out_dtype=torch.float32).double()  # noqa: E731
    slope = ((f(E + d) - f(E - d)) * dy.double()).sum() / 2
    got = (ops.embed_bwd(dy, ids, V, scale=3.0).double() * d.double()).sum()
    assert (got - slope).abs() <= 64 * 2.0 ** -24 * 3.0 * (dy.abs().double().sum(1) * 10).sum()


def test_streams_and_graphs():
    from cocodr_amd import ops
    V, H, n = 500, 136, 9000
    ids, other = ids_of("text", n, V, 1), ids_of("text", n, V, 2)
    dout = torch.randn((n, H), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").to(torch.bfloat16)
    E = torch.randn((V, H), generator=torch.Generator(device="cuda").manual_seed(2), device="cuda")
    dm = ops.dropout_mask(0.1, 1, 2, 3, ops.KIND_EMBED)
    step = lambda: (ops.dropout_fwd(ops.embed_fwd(ids, E), dm), ops.embed_bwd(ops.dropout_bwd(dout, dm), ids, V))  # noqa: E731
    want = step()
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        got = step()
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(4):
        ids.copy_(other if k % 2 == 0 else ids_of("one", n, V, 0))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step()))


def test_refusals():
    from cocodr_amd import _native as N, ops
    ids = torch.zeros(4, dtype=torch.int32, device="cuda")
    E = torch.zeros((10, 16), device="cuda")
    for bad in (lambda: ops.embed_fwd(ids.short(), E), lambda: ops.embed_fwd(ids, E.half()), lambda: ops.embed_fwd(ids, E, out_dtype=torch.float16),
                lambda: ops.embed_fwd(ids, E[:, :12].contiguous()), lambda: ops.embed_fwd(ids, E.t()), lambda: ops.embed_fwd(ids.cpu(), E),
                lambda: ops.embed_fwd(ids, E, scale=float("inf")), lambda: ops.embed_bwd(E[:3], ids, 10), lambda: ops.embed_bwd(E[:4], ids, 0),
                lambda: ops.embed_bwd(E[:4], ids, 10, accumulate=True), lambda: ops.embed_bwd(E[:4], ids, 10, out=E[:9]),
                lambda: ops.embed_bwd(E[:4], ids, 10, out=E.bfloat16()), lambda: ops.dropout_fwd(E.half(), ops.dropout_mask(0.1, 1, 1, 0, 0)),
                lambda: ops.dropout_fwd(E, ops.dropout_mask(0.1, 1, 1, 0, 0), residual=E[:9]), lambda: ops.dropout_fwd(E, N.DropoutMask(1, 2, 65536, 1.0)),
                lambda: ops.dropout_fwd(E.t(), ops.dropout_mask(0.1, 1, 1, 0, 0)), lambda: ops.dropout_bwd(E.cpu(), ops.dropout_mask(0.1, 1, 1, 0, 0))):
        with pytest.raises(ValueError):
            bad()
