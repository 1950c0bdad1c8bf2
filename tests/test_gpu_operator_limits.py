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
