"""The first layer of a decoder as a user would write it with ops: embedding * scale -> dropout -> fused Q | K | V projection -> attention with grouped
heads over packed sequences -> output projection -> dropout + residual, and back to the gradients of both weights and the table - against the same
layer in 64 bits (torch autograd, the same dropout masks), eager and replayed from a captured graph.

Tolerance, in norm: eleven results lie one behind the other on the longest way (embedding, dropout, projection, probabilities, ctx; then dy, dctx, dS,
dq | dk | dv, dx and the embedding's gradient), each rounded to bf16, off by at most U = 2^-8 of itself.  A stage hands an error on about as it
hands on the signal (random matrices, means over keys); 2 allows for the softmax, whose gradient is a difference: 11 x 2 x U."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -8
TOL = 11 * 2 * U
V, H, Hq, Hk, D = 500, 256, 4, 2, 64
LENS, TAIL = [1, 200, 33, 0, 128, 310], 8   # 672 + 8 rows
SCALE = H ** 0.5


def inputs(seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    T = sum(LENS) + TAIL
    ids = torch.randint(0, V, (T,), generator=g, device="cuda", dtype=torch.int32)
    ids[-TAIL:] = -1
    mask = (torch.rand(T, generator=g, device="cuda") >= 0.1).to(torch.int32)
    return dict(ids=ids, mask=mask, table=r(V, H) * 0.05, wqkv=(r((Hq + 2 * Hk) * D, H) / H ** 0.5).to(torch.bfloat16),
                wo=(r(H, Hq * D) / H ** 0.5).to(torch.bfloat16), dout=r(T, H).to(torch.bfloat16))


def masks(ops):
    return ops.dropout_mask(0.1, 11, 3, 0, 1), ops.dropout_mask(0.1, 11, 3, 1, 1)


def layer(ops, N, t, off, how):
    d0, d1 = masks(ops)
    T = t["ids"].numel()
    heads = lambda x: tuple(y.unflatten(1, (-1, D)) for y in x.split((Hq * D, Hk * D, Hk * D), 1))  # noqa: E731
    x = ops.dropout_fwd(ops.embed_fwd(t["ids"], t["table"], scale=SCALE), d0)
    qkv = ops.gemm(x, t["wqkv"])
    ctx, lse = ops.attn_gqa_fwd(*heads(qkv), off, **how)
    out = ops.dropout_fwd(ops.gemm(ctx.view(T, Hq * D), t["wo"]), d1, residual=x)
    dy = ops.dropout_bwd(t["dout"], d1)
    dwo = ops.gemm(dy, ctx.view(T, Hq * D), trans_a=True, trans_b=True, out_f32=True)
    dctx = ops.gemm(dy, t["wo"], trans_b=True)
    dqkv = torch.zeros_like(qkv)  # (the rows behind the last sequence are left as they are)
    ops.attn_gqa_bwd(*heads(qkv), ctx, dctx.view(T, Hq, D), lse, off, out=heads(dqkv), **how)
    dwqkv = ops.gemm(dqkv, x, trans_a=True, trans_b=True, out_f32=True)
    dx = ops.gemm(dqkv, t["wqkv"], trans_b=True, epi=N.EPI_ADD, r=t["dout"])
    return out, dwo, dwqkv, ops.embed_bwd(ops.dropout_bwd(dx, d0), t["ids"], V, scale=SCALE)


def reference(ops, t, how):
    keep = [ops.dropout_fwd(torch.ones((t["ids"].numel(), H), device="cuda"), d).double() for d in masks(ops)]
    table, wqkv, wo = (t[n].double().requires_grad_() for n in ("table", "wqkv", "wo"))
    there = (t["ids"] >= 0).double()[:, None]
    x = table[t["ids"].clamp(min=0).long()] * there * SCALE * keep[0]
    q, k, v = (y.unflatten(1, (-1, D)) for y in (x @ wqkv.t()).split((Hq * D, Hk * D, Hk * D), 1))
    parts, a = [], 0
    for n in LENS:
        i = torch.arange(n, device="cuda")
        see = (i[None, :] <= i[:, None]) & (how["mask"][a:a + n] != 0)[None, :] & (i[:, None] - i[None, :] <= how["window"][0])
        heads = []
        for h in range(Hq):
            s = (q[a:a + n, h] @ k[a:a + n, h // (Hq // Hk)].t() * D ** -0.5).masked_fill(~see, -1e300)
            p = torch.where(see, torch.softmax(s, 1), 0.0)  # (a row that sees nothing: zeros)
            heads.append(p @ v[a:a + n, h // (Hq // Hk)])
        parts.append(torch.stack(heads, 1).flatten(1))
        a += n
    ctx = torch.cat(parts + [torch.zeros((TAIL, Hq * D), dtype=torch.float64, device="cuda")])
    out = (ctx @ wo.t()) * keep[1] + x
    out.backward(t["dout"].double())
    return out.detach(), wo.grad, wqkv.grad, table.grad


def close(got, want):
    for name, x, y in zip(("out", "dwo", "dwqkv", "dtable"), got, want):
        off = (x.double() - y).norm() / y.norm()
        assert off <= TOL, (name, off.item())


def test_a_decoder_layer_and_its_gradients():
    from cocodr_amd import _native as N, ops
    t = inputs(1)
    off = torch.tensor([0] + list(torch.tensor(LENS).cumsum(0)), dtype=torch.int32, device="cuda")
    how = dict(causal=True, window=(150, -1), mask=t["mask"])
    close(layer(ops, N, t, off, how), reference(ops, t, how))
    # the same from a captured graph, with new inputs and eager work between the replays
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = layer(ops, N, t, off, how)
    for seed in (2, 3, 4):
        for name, x in inputs(seed).items():
            t[name].copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in res]
        eager = layer(ops, N, t, off, how)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, eager)), seed
        close(got, reference(ops, t, how))


def test_two_layers_at_once_on_two_streams():
    """nothing is shared between calls: workspaces are each call's own"""
    from cocodr_amd import _native as N, ops
    ts = [inputs(5), inputs(6)]
    off = torch.tensor([0] + list(torch.tensor(LENS).cumsum(0)), dtype=torch.int32, device="cuda")
    hows = [dict(causal=True, window=(150, -1), mask=t["mask"]) for t in ts]
    want = [layer(ops, N, t, off, how) for t, how in zip(ts, hows)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [None, None]
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = layer(ops, N, ts[i], off, hows[i])
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
