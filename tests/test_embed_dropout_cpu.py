"""What cocodr_embed_fwd / _bwd and cocodr_dropout_fwd / _bwd refuse before they launch anything (host arithmetic: no GPU is needed)."""
import ctypes as C

import pytest

from test_abi_cpu import lib  # noqa: F401  (the module's fixture: builds and loads the library)

P = 4096  # a pointer that is never followed


@pytest.mark.parametrize("over,says", [(dict(n=-1), b"n=-1"), (dict(n=1 << 30), b"2^30"), (dict(vocab=0), b"vocab=0"), (dict(H=12), b"width"), (dict(H=0), b"width"),
                                       (dict(ids=0), b"null"), (dict(a=0), b"null"), (dict(b=0), b"null"), (dict(a=P + 8), b"16-byte"),
                                       (dict(b=P + 4), b"16-byte"), (dict(scale=float("nan")), b"scale"), (dict(scale=float("inf")), b"scale")], ids=str)
def test_embed_refusals(lib, over, says):  # noqa: F811
    a = dict(ids=P, a=P, b=P, n=100, H=768, vocab=1000, scale=1.0)
    a.update(over)
    assert lib.cocodr_embed_fwd(a["ids"], 0, a["a"], 1, a["b"], 0, a["n"], a["H"], a["vocab"], a["scale"], None) == -1 and says in lib.cocodr_last_error()
    assert lib.cocodr_embed_bwd(a["a"], 0, a["ids"], 0, a["b"], a["n"], a["H"], a["vocab"], a["scale"], 0, P, 1 << 40, None) == -1
    assert says in lib.cocodr_last_error()


def test_embed_workspace(lib):  # noqa: F811
    need = lib.cocodr_embed_bwd_workspace_bytes(8192, 768, 30522)
    assert need >= 4 * (2 * 30522 + 2 * 8192) and lib.cocodr_embed_bwd_workspace_bytes(-1, 768, 1) == 0
    call = lambda ws, size: lib.cocodr_embed_bwd(P, 0, P, 0, P, 8192, 768, 30522, 1.0, 0, ws, size, None)  # noqa: E731
    assert call(P, need - 1) == -3 and b"workspace" in lib.cocodr_last_error()
    assert call(0, need) == -3 and call(P + 4, need) == -3


def test_dropout_refusals(lib):  # noqa: F811
    from cocodr_amd import _native as N
    ok, all_ = N.DropoutMask(1, 2, 6554, 1.1), N.DropoutMask(1, 2, 65536, 1.0)
    fwd = lambda x=P, r=None, out=P, n=100, f32=0, dm=ok: lib.cocodr_dropout_fwd(x, r, out, n, f32, C.byref(dm) if dm else None, None)  # noqa: E731
    bwd = lambda x=P, out=P, n=100, f32=0, dm=ok: lib.cocodr_dropout_bwd(x, out, n, f32, C.byref(dm) if dm else None, None)  # noqa: E731
    for call in (fwd, bwd):
        assert call(dm=None) == -1 and call(dm=all_) == -1 and call(x=0) == -1 and call(out=0) == -1
        assert call(n=(1 << 33) + 1) == -1 and b"2^32 pairs" in lib.cocodr_last_error()
        assert call(x=P + 1) == -1 and call(out=P + 2, f32=1) == -1
        assert call(x=0, out=0, n=0) == 0
    assert fwd(r=P + 1) == -1
