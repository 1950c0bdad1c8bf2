"""Where the limits of cocodr_attn_gqa_* lie: the last size that is taken and the first that is refused (host arithmetic: no GPU is needed)."""
import ctypes as C

import pytest

from test_abi_cpu import lib  # noqa: F401  (the module's fixture: builds and loads the library)
from test_attn_gqa_cpu import args


@pytest.mark.parametrize("T,heads,taken,refused", [(200, 16, (1 << 20) - 2, (1 << 20) - 1), (127, 1, (1 << 24) - 1, 1 << 24), (1 << 20, 8, (1 << 21) - 8193, (1 << 21) - 8192)])
def test_workgroups_of_one_launch(lib, T, heads, taken, refused):  # noqa: F811
    """256 work-items each, and a launch counts them in 32 bits.  A size that is taken comes as far as the workspace, which is missing here."""
    size = lambda B: dict(T=T, B=B, heads=heads, kv_heads=heads, k_row=512, v_row=512, dk_row=512, dv_row=512)  # noqa: E731
    bwd = lambda a: lib.cocodr_attn_gqa_bwd(C.byref(a), 4096, 4096, 4096, 4096, 4096, 4096, 0, None, 0, None)  # noqa: E731
    wide = dict(q_row=1024, k_row=1024, v_row=1024, o_row=1024, do_row=1024, dq_row=1024, dk_row=1024, dv_row=1024)
    assert bwd(args(**dict(size(taken), **wide))) == -3, lib.cocodr_last_error()
    a = args(**dict(size(refused), **wide))
    assert bwd(a) == -1 and b"one launch" in lib.cocodr_last_error()
    assert lib.cocodr_attn_gqa_fwd(C.byref(a), 4096, 4096, 0, None) == -1 and b"one launch" in lib.cocodr_last_error()
