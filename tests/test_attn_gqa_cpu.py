"""What cocodr_attn_gqa_fwd / _bwd refuse before they launch anything (host arithmetic: no GPU is needed), and what ops refuses."""
import ctypes as C

import pytest
import torch

from test_abi_cpu import lib  # noqa: F401  (the module's fixture: builds and loads the library)


def args(**over):
    from cocodr_amd import _native as N
    a = dict(q=4096, k=4096, v=4096, seq_off=4096, mask=0, q_row=512, q_head=64, k_row=256, k_head=64, v_row=256, v_head=64, o_row=512, o_head=64,
             do_row=512, do_head=64, dq_row=512, dq_head=64, dk_row=256, dk_head=64, dv_row=256, dv_head=64, T=100, B=3, heads=8, kv_heads=4,
             dim=64, left=-1, right=-1, scale=0.125)
    a.update(over)
    return N.AttnGqaArgs(**a)


COMMON = [
    (dict(q=0), b"null pointer"), (dict(seq_off=0), b"null pointer"), (dict(T=0), b"T=0"), (dict(T=1 << 30), b"2^30"), (dict(B=0), b"B=0"),
    (dict(heads=6), b"multiple of kv_heads"), (dict(kv_heads=0), b"multiple of kv_heads"), (dict(dim=136), b"head size"), (dict(dim=60), b"head size"),
    (dict(dim=0), b"head size"), (dict(scale=0.0), b"scale"), (dict(scale=float("nan")), b"scale"), (dict(scale=float("inf")), b"scale"),
    (dict(left=-2), b"window"), (dict(right=1 << 30), b"window"), (dict(k=4104), b"16-byte"), (dict(q_row=513), b"multiples of 8"),
    (dict(v_row=1 << 23), b"2^23"), (dict(k_head=-64), b"multiples of 8"), (dict(T=(1 << 30) - 1, heads=1 << 12), b"one launch"),
]


@pytest.mark.parametrize("over,says", COMMON, ids=lambda x: str(x))
def test_refused_in_both_directions(lib, over, says):  # noqa: F811
    a, big = args(**over), 1 << 40
    assert lib.cocodr_attn_gqa_fwd(C.byref(a), 4096, 4096, 0, None) == -1 and says in lib.cocodr_last_error()
    assert lib.cocodr_attn_gqa_bwd(C.byref(a), 4096, 4096, 4096, 4096, 4096, 4096, 0, 4096, big, None) == -1 and says in lib.cocodr_last_error()


def test_outputs_that_overlap_or_are_missing(lib):  # noqa: F811
    fwd = lambda ctx=4096, lse=4096, **over: lib.cocodr_attn_gqa_fwd(C.byref(args(**over)), ctx, lse, 0, None)  # noqa: E731
    assert fwd(ctx=0) == -1 and fwd(lse=0) == -1 and fwd(ctx=4098) == -1
    assert fwd(o_head=0) == -1 and b"apart" in lib.cocodr_last_error()
    assert fwd(o_row=448) == -1 and b"apart" in lib.cocodr_last_error()  # the last head of a row would reach into the next row
    bwd = lambda p=(4096,) * 6, floats=1 << 30, ws=4096, **over: lib.cocodr_attn_gqa_bwd(C.byref(args(**over)), *p, 0, ws, floats, None)  # noqa: E731
    for i in range(6):
        assert bwd(p=tuple(0 if j == i else 4096 for j in range(6))) == -1
    for over in (dict(dq_head=0), dict(dk_row=8), dict(dv_row=192), dict(do_row=4)):
        assert bwd(**over) == -1, over
    a = args()
    need = lib.cocodr_attn_gqa_bwd_workspace_floats(C.byref(a))
    assert need >= 2 * 100 * 8
    assert bwd(ws=4104) == -1 and b"workspace" in lib.cocodr_last_error()
    # few tiles with many steps: room for the parts of dk and dv, 2 x 128 x 64 floats a tile and part; none for short ones
    a = args(T=4096, B=3, heads=32, kv_heads=8)
    assert lib.cocodr_attn_gqa_bwd_workspace_floats(C.byref(a)) >= 2 * 4096 * 32 + 2 * (4096 // 128 + 3) * 8 * 2 * 128 * 64
    assert lib.cocodr_attn_gqa_bwd_workspace_floats(C.byref(args(T=32, B=1))) == 2 * 32 * 8
    assert bwd(floats=need - 1) == -3 and b"workspace" in lib.cocodr_last_error() and bwd(ws=0) == -3


def test_ops_refuse_tensors_of_the_host():
    from cocodr_amd import ops
    t = torch.zeros((8, 2, 64), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="GPU"):
        ops.attn_gqa_fwd(t, t, t, torch.tensor([0, 8], dtype=torch.int32))
