"""Calls of the vocabulary operators that have to be refused, or that go another
way on the host; no GPU is needed."""

from __future__ import annotations

import ctypes

from dabsn_b200 import _native

NULL = ctypes.c_void_p(0)


# ---------------------------------------------------------------------------
# Tensors without memory of their own
# ---------------------------------------------------------------------------
def test_null_pointers_are_refused():
    """A wrapper subclass (a DTensor) and a tensor under functionalize have a
    null data pointer; nothing may be launched with one.  1 stands for an
    address: the call is refused before it is used."""
    lib = _native.load()
    f = ctypes.c_float

    def scores(x=1, t=1, lp=1, ent=1, values=None, ids=None, k=0):
        return lib.dabsn_token_scores_fwd(0, 4, 10, 10, x, t, -100, f(1.0), k, lp, ent, None,
                                          values, ids, NULL)

    def scores_back(x=16, t=1, st=1, ent=1, dx=16):
        return lib.dabsn_token_scores_bwd(0, 4, 10, 10, x, t, -100, f(1.0), st, ent, None, None,
                                          dx, 10, NULL)

    def distill(x=16, ids=1, tl=1, ws=1):
        return lib.dabsn_distill_fwd(0, 4, 10, 10, x, 0, 2, ids, tl, -100, f(1.0), f(1.0), 1, ws,
                                     None, None, None, 0, NULL)

    def distill_back(x=16, ws=1, up=1, dx=16):
        return lib.dabsn_distill_bwd(0, 4, 10, 10, x, 2, ws, f(1.0), f(1.0), 1, up, 0, 0, dx, 10,
                                     NULL)

    def lookup(t=1, w=1, out=1):
        return lib.dabsn_embedding_fwd(0, 0, 4, 10, 8, t, w, 8, f(1.0), out, NULL)

    def table(t=1, g=1, dw=1, ws=1):
        return lib.dabsn_embedding_bwd(0, 0, 4, 10, 8, t, -1, g, f(1.0), dw, ws, 1 << 30, NULL)

    for call, names in ((scores, ("x", "t", "lp", "ent")), (scores_back, ("t", "st", "ent")),
                        (distill, ("x", "ids", "tl", "ws")), (distill_back, ("ws", "up")),
                        (lookup, ("t", "w", "out")), (table, ("t", "g", "dw", "ws"))):
        for name in names:
            assert call(**{name: None}) == 4, (call.__name__, name)
            assert b"null pointer" in lib.dabsn_last_error(), (call.__name__, name)
    for call in (scores_back, distill_back):  # the two share their 16-byte phase
        assert call(x=None, dx=16) == 4 and b"null pointer" in lib.dabsn_last_error()
        assert call(x=16, dx=None) == 4 and b"null pointer" in lib.dabsn_last_error()
    assert scores(k=2, values=None, ids=1) == 4 and scores(k=2, values=1, ids=None) == 4
    assert b"null pointer" in lib.dabsn_last_error()
