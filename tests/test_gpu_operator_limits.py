"""Sizes at and behind the limits of the operators for decoder and long-document backbones: they are taken, or refused with a ValueError."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("window", [(1 << 32, -1), (-1, 1 << 32), ((1 << 32) + 3, 3), (-(1 << 32), 0), ((1 << 31), -1)])
def test_windows_that_32_bits_cannot_hold(window):
    """2^32 is not 0: cut to 32 bits it would be"""
    from cocodr_amd import ops
    t = torch.randn((8, 2, 64), generator=torch.Generator(device="cuda").manual_seed(0), device="cuda").to(torch.bfloat16)
    off = torch.tensor([0, 8], dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="32 bits"):
        ops.attn_gqa_fwd(t, t, t, off, window=window)
    ctx, lse = ops.attn_gqa_fwd(t, t, t, off)
    with pytest.raises(ValueError, match="32 bits"):
        ops.attn_gqa_bwd(t, t, t, ctx, t, lse, off, window=window)


def test_more_heads_than_32_bits_count():
    from cocodr_amd import ops
    t = torch.ones((8,), dtype=torch.bfloat16, device="cuda").expand(1, (1 << 32) + 4, 8)  # (one head's memory)
    with pytest.raises(ValueError, match="32 bits"):
        ops.attn_gqa_fwd(t, t[:, :2], t[:, :2], torch.tensor([0, 1], dtype=torch.int32, device="cuda"))


@pytest.mark.parametrize("vocab", [(1 << 32) + 5, 1 << 31, -(1 << 32) + 5])
def test_a_vocabulary_that_32_bits_cannot_hold(vocab):
    """refused before the table of that many rows is allocated"""
    from cocodr_amd import ops
    with pytest.raises(ValueError, match="32 bits"):
        ops.embed_bwd(torch.ones((3, 8), device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda"), vocab)


def test_a_lookup_of_more_rows_than_a_launch_has_workgroups():
    """2^24 rows of 4104 columns, of which a workgroup would take one: 138 GB of results"""
    from cocodr_amd import ops
    n, H = (1 << 24) + 3, 4104
    if torch.cuda.mem_get_info()[0] < n * H * 2 + (1 << 33):
        pytest.skip("needs 146 GB of free device memory")
    table = torch.arange(5 * H, device="cuda").remainder(251).view(5, H).to(torch.bfloat16)
    ids = torch.arange(n, device="cuda", dtype=torch.int32).remainder(7)  # (5 and 6: padding)
    got = ops.embed_fwd(ids, table)
    for a in (0, 1 << 23, (1 << 24) - 2000, n - 2000):
        part = ids[a:a + 2000].long()
        want = torch.where((part < 5)[:, None], table[part.clamp(max=4)], torch.zeros((), dtype=torch.bfloat16, device="cuda"))
        assert torch.equal(got[a:a + 2000], want), a
    for col in (0, 2051, H - 1):  # every row
        assert torch.equal(got[:, col].float(), torch.where(ids < 5, table[ids.clamp(max=4).long(), col].float(), 0.0))
    del got
    torch.cuda.empty_cache()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("sign", [1, -1])
def test_scores_at_the_end_of_their_range(D, sign):
    """all of a row's scores 2^24 or -2^24: each key counts the same, ctx is the mean of v.  Equal scores give equal probabilities, at most 2 times too
    large or small all together (half of 2^24's step): what is left are the roundings of P and ctx, 2^-8 each, and n 2^-24 of the sums.
    lse is the score + log n = 5.3, off by at most 0.7 where log2 of the sum is added (half of the step at 2^24.5), 1.5 by scale log2 e, 0.5 by ln 2 and 1
    at the end: below 10 in all.  Values near 2^92 do not overflow on the way"""
    from cocodr_amd import ops
    n, H = 200, 2
    q = torch.full((n, H, D), 2.0 ** 9, dtype=torch.bfloat16, device="cuda")
    k = torch.full((n, 1, D), sign * 2.0 ** 9, dtype=torch.bfloat16, device="cuda")
    v = (torch.rand((n, 1, D), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda") * 2.0 ** 92).to(torch.bfloat16)
    off = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    ctx, lse = ops.attn_gqa_fwd(q, k, v, off, scale=64.0 / D)
    assert ((lse.double() - sign * 2.0 ** 24).abs() <= 10).all()
    want = v.double().mean(0, keepdim=True).expand(n, H, D)
    assert ((ctx.double() - want).abs() <= want * (2 * 2.0 ** -8 + 2.0 ** -14)).all()
