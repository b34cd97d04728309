"""Calls of the vocabulary operators that have to be refused, or that go another
way on the host; no GPU is needed."""

from __future__ import annotations

import contextlib
import ctypes
import threading

import pytest
import torch
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

import dabsn_b200
from dabsn_b200 import _native, ops

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


# ---------------------------------------------------------------------------
# Forward-mode derivatives and tracing
# ---------------------------------------------------------------------------
def _written(values):
    """A result as the kernels give one: allocated by torch, written through
    its address."""
    out = torch.empty(values.shape, dtype=values.dtype)
    values = values.detach().contiguous()
    ctypes.memmove(out.data_ptr(), values.data_ptr(), values.numel() * values.element_size())
    return out


@pytest.fixture
def host(monkeypatch):
    """The operators with their kernels replaced by the same sums on the CPU."""
    off = torch._C._DisableTorchDispatch  # a kernel's work is out of torch's sight

    def quiet(f):
        def run(*args, **kw):
            state = torch._C._get_tracing_state()
            torch._C._set_tracing_state(None)
            try:
                with off(), torch.no_grad():
                    values = f(*args, **kw)
            finally:
                torch._C._set_tracing_state(state)
            return values

        return run

    def scores(logits, tokens, top_k, temperature, ignore_index, with_stats=True):
        logp = quiet(lambda: torch.log_softmax(logits / temperature, -1))()
        lp = _written(quiet(lambda: logp.gather(1, tokens[:, None])[:, 0].contiguous())())
        ent = _written(quiet(lambda: -(logp.exp() * logp).sum(-1))())
        return lp, ent, None, None, torch.zeros(len(tokens), 2)

    def distill(logits, ids, tl, temperature, weight, ignore_index, reduction, gradient=False):
        q = quiet(lambda: torch.softmax(tl / temperature, -1))()
        logp = quiet(lambda: torch.log_softmax(logits / temperature, -1))()
        loss = quiet(lambda: (q * (q.log() - logp.gather(1, ids))).sum(-1).mean())()
        return _written(loss), torch.zeros(1), torch.zeros_like(logits) if gradient else None

    def lookup(tokens, weight, scale, dtype):
        return _written(quiet(lambda: (weight[tokens] * scale).to(dtype))())

    monkeypatch.setattr(ops, "token_scores_forward", scores)
    monkeypatch.setattr(ops, "distill_forward", distill)
    monkeypatch.setattr(ops, "embedding_forward", lookup)
    monkeypatch.setattr(ops, "capture_id", lambda device: 0)
    monkeypatch.setattr(ops, "embedding_backward", lambda t, g, *a: _written(
        quiet(lambda: torch.zeros(5, 3).index_add_(0, t, g))()))
    ids = torch.tensor([[1, 2], [0, 1], [2, 1]])
    t = torch.tensor([1, 0, 2])
    tl = torch.tensor([[0.0, 1.0], [2.0, 1.0], [0.5, 0.5]])
    return {
        "token_log_probs": lambda x: dabsn_b200.token_log_probs(x[:3], t).log_prob,
        "distillation_loss": lambda x: dabsn_b200.distillation_loss(x[:3], ids, tl),
        "embedding": lambda x: dabsn_b200.embedding(t, x),
    }


NAMES = ["token_log_probs", "distillation_loss", "embedding"]


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("name", NAMES)
def test_forward_mode_is_refused(host, name, grad):
    x = torch.randn(5, 3).requires_grad_(grad)
    want = host[name](x)
    with forward_ad.dual_level():
        assert torch.equal(host[name](x), want)  # no tangent: as without
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            host[name](dual)
        with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
            host[name](dual)
    with pytest.raises(RuntimeError):
        torch.func.jvp(host[name], (x.detach(),), (torch.ones_like(x),))


def test_forward_mode_of_the_teacher_and_of_a_reverse_is_refused(host):
    x = torch.randn(3, 4)
    ids, tl = torch.tensor([[1], [0], [2]]), torch.zeros(3, 1)
    with forward_ad.dual_level():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            dabsn_b200.distillation_loss(x, ids, forward_ad.make_dual(tl, torch.ones_like(tl)))
    w = torch.randn(5, 3, requires_grad=True)
    out = host["embedding"](w)
    (g,) = torch.autograd.grad(out, w, torch.ones_like(out), retain_graph=True)
    assert g.sum(-1).tolist() == [3.0, 3.0, 3.0, 0.0, 0.0]
    with forward_ad.dual_level():
        up = forward_ad.make_dual(torch.ones_like(out), torch.ones_like(out))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.autograd.grad(out, w, up)


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("name", NAMES)
def test_a_traced_call_computes(host, name, grad):
    """torch.jit.trace records the operator, not the allocation of its result."""
    traced = torch.jit.trace(host[name], (torch.randn(5, 3).requires_grad_(grad),))
    for seed in range(3):
        x = torch.randn(5, 3, generator=torch.Generator().manual_seed(seed))
        assert torch.equal(traced(x).detach(), host[name](x))


@pytest.mark.parametrize("pre_dispatch", [False, True])
@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("name", NAMES)
def test_make_fx_is_refused(host, name, grad, pre_dispatch):
    x = torch.randn(5, 3).requires_grad_(grad)
    with pytest.raises(RuntimeError, match="make_fx"):
        make_fx(host[name], pre_dispatch=pre_dispatch)(x)
    host[name](x)


def test_make_fx_of_a_reverse_is_refused(host):
    w = torch.randn(5, 3, requires_grad=True)
    out = host["embedding"](w)
    with pytest.raises(RuntimeError, match="make_fx"):
        make_fx(lambda g: torch.autograd.grad(out, w, g)[0])(torch.ones_like(out))


# ---------------------------------------------------------------------------
# What the kernels can only record
# ---------------------------------------------------------------------------
def test_the_device_status_can_be_raised(monkeypatch):
    codes, waits = [8, 0], []
    monkeypatch.setattr(_native, "device_status", lambda reset=False: codes.pop(0))
    monkeypatch.setattr(torch.cuda, "synchronize", lambda: waits.append(1))
    monkeypatch.setattr(torch.cuda, "device", contextlib.nullcontext)
    with pytest.raises(RuntimeError, match="outside"):
        dabsn_b200.raise_on_device_status()
    dabsn_b200.raise_on_device_status()
    assert len(waits) == 2
    for name in NAMES:
        text = getattr(dabsn_b200, name).__doc__
        assert "dabsn_b200.raise_on_device_status()" in text
        assert "next synchronisation" not in " ".join(text.split())


def test_rows_too_long_for_alternatives_are_refused():
    """The scans for alternatives step 512 elements at a time through 32-bit
    indices, which a row of nearly 2^31 would carry past the largest."""
    lib = _native.load()

    def scores(V, k):
        return lib.dabsn_token_scores_fwd(0, 0, V, V, None, None, -100, ctypes.c_float(1.0), k,
                                          *([None] * 6))

    assert scores(2 ** 31 - 2, 1) and b"alternatives" in lib.dabsn_last_error()
    assert scores(2 ** 31 - 512, 1) and scores(2 ** 31 - 513, 1) == 0
    assert scores(2 ** 31 - 2, 0) == 0
    assert 2 ** 31 - 513 + 512 < 2 ** 31  # the largest index that the scans form


def test_the_capture_is_that_of_the_logits_device(monkeypatch):
    """A call on another device than the current one asks that device's stream."""
    class Lib:
        @staticmethod
        def dabsn_capture_id(stream):
            return {10: 0, 11: 7}[stream]

    monkeypatch.setattr(_native, "load", lambda: Lib)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch.cuda, "device", contextlib.nullcontext)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda i: 10 + i, raising=False)
    assert ops.capture_id(torch.device("cuda", 0)) == 0
    assert ops.capture_id(torch.device("cuda", 1)) == 7


def test_make_fx_in_another_thread_refuses_nothing_here(host):
    """Only the thread that traces is refused."""
    x, seen = torch.randn(5, 3), []

    def other():
        seen.append(host["embedding"](x))

    def traced(z):
        thread = threading.Thread(target=other)
        thread.start()
        thread.join()
        return z + 1

    make_fx(traced)(x)
    assert len(seen) == 1 and torch.equal(seen[0], host["embedding"](x))


def test_upstream_gradients_with_a_pending_sign():
    """The imaginary part of one conjugate number is a contiguous view with its
    sign still to be turned."""
    pending = torch.tensor([1.0 + 2.0j]).conj().imag
    dense = ops._dense_f32(pending)
    assert (ctypes.c_float * 1).from_address(dense.data_ptr())[0] == -2.0
    assert pending.is_neg() and pending.is_contiguous()
    wide = torch.tensor([[1.0 + 2.0j, 3.0 + 4.0j]]).conj().imag
    dense = ops._dense(wide)
    assert list((ctypes.c_float * 2).from_address(dense.data_ptr())) == [-2.0, -4.0]
    assert ops._dense_f32(None) is None
    plain = torch.randn(3)
    assert ops._dense_f32(plain) is plain
    assert ops._dense_f32(plain.double()).dtype == torch.float32
