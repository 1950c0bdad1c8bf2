"""The limits of attn_gqa_oracle see the mistakes that sums in parts and a running maximum can make.  All of it runs in 64 bits on the CPU; the mistakes are
planted in the oracle."""
import pytest

import attn_gqa_oracle as A

# sequences, query heads, key heads, head size, window, spread of q and k, scale
HEADS64 = ([300], 64, 1, 64, (-1, -1), 1.0, 0.125)
LONG = ([1500], 4, 1, 128, (-1, -1), 1.0, 128 ** -0.5)
CAUSAL = ([700, 40], 6, 2, 72, (-1, 0), 1.0, 72 ** -0.5)
SHORT = ([2, 3, 4, 5, 6, 8, 11, 20] * 12, 4, 2, 64, (-1, 0), 1.0, 0.125)
NEAR = ([500], 4, 2, 128, (2, 0), 1.0, 128 ** -0.5)
PEAKED = ([300, 190], 2, 1, 64, (-1, -1), 6.0, 0.25)


def three(case, **how):
    lens, H, Hk, D, (left, right), spread, scale = case
    q, k, v, dctx, mask, _ = A.inputs(lens, H, Hk, D, 0.0, 3, spread, "cpu")
    go = lambda **x: A.run(q, k, v, dctx, lens, left, right, mask, scale, **x)  # noqa: E731
    return go(), go(rounded=True), go(rounded=True, **how), lens


@pytest.mark.parametrize("case", [HEADS64, CAUSAL, SHORT, NEAR, PEAKED], ids=["64 heads", "causal", "short", "near", "peaked"])
def test_other_bits_of_the_same_roundings_are_within(case):
    """probabilities moved at random by what fp32 does to them round to other neighbours here and there"""
    val, emu, got, lens = three(case, noise=2.0 ** -18)
    assert A.beyond(got, val, emu, lens) == []


@pytest.mark.parametrize("case,plant,where", [
    (HEADS64, ("step", 64, 17), {"dk", "dv"}), (HEADS64, ("head", 40), {"dk", "dv"}), (HEADS64, ("delta",), {"dq", "dk"}),
    (LONG, ("step", 704, 1), {"dk", "dv"}), (LONG, ("delta",), {"dq", "dk"}),
    (CAUSAL, ("step", 128, 4), {"dk", "dv"}), (CAUSAL, ("head", 2), {"dk", "dv"}), (CAUSAL, ("delta",), {"dq", "dk"}),
    (SHORT, ("ctx delta",), {"dq", "dk"}), (NEAR, ("ctx delta",), {"dq", "dk"}), (SHORT, ("max",), {"lse"}),
    (PEAKED, ("max",), {"lse"}), (PEAKED, ("lag",), {"ctx", "lse"}), (PEAKED, ("step", 64, 0), {"dk", "dv"})], ids=lambda x: str(x)[:24])
def test_planted_mistakes_are_beyond(case, plant, where):
    val, emu, got, lens = three(case, plant=plant)
    assert {b[0] for b in A.beyond(got, val, emu, lens)} >= where


def test_the_scores_of_the_peaked_case_are_several_hundred():
    """... so that the running maximum grows by more than 2^20 from tile to tile"""
    lens, H, Hk, D, _, spread, scale = PEAKED
    q, k, *_ = A.inputs(lens, H, Hk, D, 0.0, 3, spread, "cpu")
    s = q[:300, 0].double() @ k[:300, 0].double().t() * scale
    assert s.max() > 250
    tops = [s[:, a:a + 64].amax(1) for a in range(0, 300, 64)]
    assert int((tops[1] - tops[0] > 20).sum()) > 50
