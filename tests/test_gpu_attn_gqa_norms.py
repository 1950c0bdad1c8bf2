"""ops.attn_gqa_fwd / attn_gqa_bwd against 64 bits in norm, over each result and over each tile and head of it, with the limits of attn_gqa_oracle (derived
there; tests/test_attn_gqa_norms_cpu.py shows what they see)."""
import pytest
import torch

import attn_gqa_oracle as A

pytestmark = pytest.mark.gpu

# sequences, query heads, key heads, head size, causal, window, share of keys masked out, spread of q and k, scale
PLAIN = [
    ([300], 64, 1, 64, False, (-1, -1), 0, 1, None),                 # the 64 query heads of one key head in up to 8 parts
    ([1500], 4, 1, 128, False, (-1, -1), 0, 1, None),
    ([2048], 8, 2, 128, True, (-1, -1), 0, 1, None),
    ([2048, 2048, 700], 8, 2, 64, True, (-1, -1), 0.1, 1, None),
    ([700, 40], 6, 2, 72, True, (-1, -1), 0, 1, None),               # three heads: parts begin inside a head
    ([128] * 6, 4, 4, 64, False, (-1, -1), 0, 1, None),
    ([20, 256, 100, 33] * 5, 4, 4, 64, False, (-1, -1), 0.1, 1, None),
    ([200, 77] * 135, 1, 1, 64, True, (-1, -1), 0, 1, None),         # more than 256 sequences
    ([2, 3, 4, 5, 6, 8, 11, 20] * 12, 4, 2, 64, True, (-1, -1), 0, 1, None),   # delta from the probabilities ..
    ([500], 4, 2, 128, True, (2, -1), 0, 1, None),                   # .. here, too
    ([900, 513], 4, 4, 64, False, (64, 64), 0.2, 1, None),
    ([1300], 4, 1, 128, True, (333, -1), 0, 1, None),
    ([700], 2, 1, 8, False, (-1, 100), 0, 1, None),
    ([1000, 300], 2, 1, 32, True, (-1, -1), 0, 1, None),
    ([600], 4, 2, 80, False, (-1, -1), 0.3, 1, None),
    ([600, 257], 4, 2, 96, True, (-1, -1), 0, 1, None),
]
# scores of several hundred: the running maximum grows by far more than it may lag behind, and delta is what is left of large numbers
PEAKED = [(lens, 2, 1, D, causal, window, masked, 6, 0.25) for D in (64, 128)
          for lens, causal, window, masked in (([300, 190], False, (-1, -1), 0), ([520], True, (-1, -1), 0), ([700], False, (150, 90), 0.2))]
LONG = [([8192], 1, 1, 128, True, (-1, -1), 0, 1, None), ([8191], 2, 1, 64, False, (-1, -1), 0.1, 1, None), ([5000, 3, 6145], 1, 1, 64, False, (1000, 64), 0, 1, None)]


@pytest.mark.parametrize("case", PLAIN + PEAKED + LONG, ids=lambda c: f"{len(c[0])}x{max(c[0])}-h{c[1]}k{c[2]}d{c[3]}-{'causal' if c[4] else 'full'}{c[5]}-m{c[6]}-x{c[7]}")
def test_norms(case):
    from cocodr_amd import ops
    lens, H, Hk, D, causal, window, masked, spread, scale = case
    q, k, v, dctx, mask, off = A.inputs(lens, H, Hk, D, masked, 3, spread, "cuda")
    how = dict(causal=causal, window=window, mask=mask, scale=scale)
    ctx, lse = ops.attn_gqa_fwd(q, k, v, off, **how)
    dq, dk, dv = ops.attn_gqa_bwd(q, k, v, ctx, dctx, lse, off, **how)
    a = (q, k, v, dctx, lens, window[0], 0 if causal else window[1], mask, D ** -0.5 if scale is None else scale)
    val, emu = A.run(*a), A.run(*a, rounded=True)
    rel = {n: (float((g.double() - val[n]).norm() / val[n].norm()), float((emu[n] - val[n]).norm() / val[n].norm())) for n, g in (("ctx", ctx), ("dq", dq), ("dk", dk), ("dv", dv))}
    print(rel, flush=True)
    assert A.beyond(dict(ctx=ctx, lse=lse, dq=dq, dk=dk, dv=dv), val, emu, lens) == []
