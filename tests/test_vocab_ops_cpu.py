"""What the vocabulary operators refuse, before anything is launched."""

from __future__ import annotations

import ctypes

import pytest
import torch

import dabsn_b200
from dabsn_b200 import _native, ops


def _logits(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


def test_shapes_are_checked():
    x = _logits(4, 10)
    with pytest.raises(ValueError, match="tokens"):
        dabsn_b200.token_log_probs(x, torch.zeros(3, dtype=torch.int64))
    with pytest.raises(ValueError, match="teacher_tokens"):
        dabsn_b200.distillation_loss(x, torch.zeros(3, 2, dtype=torch.int64), torch.zeros(4, 2))
    with pytest.raises(ValueError, match="teacher_logits"):
        dabsn_b200.distillation_loss(x, torch.zeros(4, 2, dtype=torch.int64), torch.zeros(4))
    with pytest.raises(ValueError, match="differ"):
        dabsn_b200.distillation_loss(x, torch.zeros(4, 2, dtype=torch.int64), torch.zeros(4, 3))
    with pytest.raises(ValueError, match="at least one entry"):
        dabsn_b200.distillation_loss(x, torch.zeros(4, 0, dtype=torch.int64), torch.zeros(4, 0))
    with pytest.raises(ValueError, match="reduction"):
        dabsn_b200.distillation_loss(x, torch.zeros(4, 2, dtype=torch.int64), torch.zeros(4, 2),
                                     reduction="median")
    with pytest.raises(ValueError, match="vocabulary"):
        dabsn_b200.token_log_probs(_logits(4, 0), torch.zeros(4, dtype=torch.int64))
    with pytest.raises(ValueError, match="weight"):
        dabsn_b200.embedding(torch.zeros(3, dtype=torch.int64), torch.zeros(5))
    with pytest.raises(ValueError, match="padding_idx"):
        dabsn_b200.embedding(torch.zeros(3, dtype=torch.int64), torch.zeros(5, 4), padding_idx=5)


def test_cpu_tensors_are_refused():
    ids = torch.zeros(4, dtype=torch.int64)
    with pytest.raises(TypeError, match="CUDA"):
        dabsn_b200.token_log_probs(_logits(4, 10), ids)
    with pytest.raises(TypeError, match="CUDA"):
        dabsn_b200.distillation_loss(_logits(4, 10), ids[:, None], torch.zeros(4, 1))
    with pytest.raises(TypeError, match="CUDA"):
        dabsn_b200.embedding(ids, torch.zeros(5, 4))


@pytest.mark.parametrize("t", [0.0, -1.0, float("inf"), float("nan"), 1e-45, 1e39, 9e-7, 1.1e6])
def test_temperatures(t):
    with pytest.raises(ValueError, match="temperature"):
        ops._temperature(t)


def test_ids_must_be_integers():
    with pytest.raises(TypeError, match="int64 or int32"):
        ops._int_rows(torch.zeros(4), (4,), "tokens")
    assert ops._int_rows(torch.zeros(4, dtype=torch.int32), (4,), "t").dtype == torch.int64


NULL = ctypes.c_void_p(0)


def test_entry_points_check_sizes_before_launching():
    """The C entry points refuse what their kernels do not cover; nothing is
    launched, so null pointers are never read."""
    lib = _native.load()
    f = ctypes.c_float

    def scores(dtype=0, rows=4, V=10, ld=10, t=1.0, k=0):
        return lib.dabsn_token_scores_fwd(dtype, rows, V, ld, NULL, NULL, -100, f(t), k,
                                          *([NULL] * 6))

    assert scores(rows=0) == 0
    assert scores(rows=-1) and scores(V=0) and scores(ld=9) and scores(V=2 ** 31 - 1, ld=2 ** 31)
    assert scores(dtype=2) and scores(t=0.0) and scores(t=float("nan"))
    assert scores(k=11) and scores(V=1000, ld=1000, k=129) and scores(k=-1)

    def distill(dtype=0, teacher=0, rows=4, V=10, ld=10, K=2, t=1.0, x=16, dx=None, ldd=10,
                result=None):
        return lib.dabsn_distill_fwd(dtype, rows, V, ld, x, teacher, K, NULL, NULL, -100, f(t), f(1.0), 1,
                                     NULL, NULL, result, dx, ldd, NULL)

    assert distill(rows=0) == 0
    assert distill(K=0) and distill(K=257) and distill(dtype=7) and distill(t=float("inf"))
    assert distill(teacher=2) and distill(V=0) and distill(ld=9) and distill(rows=2 ** 31)
    assert distill(dx=16) and b"result" in lib.dabsn_last_error()
    assert distill(dx=8, result=16) and b"phase" in lib.dabsn_last_error()
    assert distill(dx=32, result=16, ldd=9) and distill(dx=32, result=16, ldd=11)

    def reverse(ld=10, ldd=10, x=0, dx=0, unless_one=0, stride=0):
        return lib.dabsn_distill_bwd(0, 4, 10, ld, x, 2, NULL, f(1.0), f(1.0), 1, NULL, stride,
                                     unless_one, dx, ldd, NULL)

    assert reverse(ld=9) and reverse(ldd=9) and reverse(ldd=11) and reverse(x=16, dx=4)
    assert reverse(unless_one=1, stride=1)
    assert lib.dabsn_token_scores_bwd(0, 4, 10, 10, 16, NULL, -100, f(1.0), *([NULL] * 4), 4, 10,
                                      NULL)
    assert lib.dabsn_distill_workspace(100, 5) >= 100 * 5 * 12
    assert lib.dabsn_distill_workspace(-1, 5) == 0

    def lookup(w=0, o=0, N=4, V=10, D=8, ldw=8):
        return lib.dabsn_embedding_fwd(w, o, N, V, D, NULL, NULL, ldw, f(1.0), NULL, NULL)

    assert lookup(N=0) == 0
    assert lookup(w=3) and lookup(o=3) and lookup(D=0) and lookup(V=0) and lookup(ldw=7)
    assert lookup(N=2 ** 31)
    need = lib.dabsn_embedding_bwd_workspace(1000, 50, 8)
    assert need > 0 and lib.dabsn_embedding_bwd_workspace(-1, 50, 8) == 0
    assert lib.dabsn_embedding_bwd(0, 0, 1000, 50, 8, NULL, -1, NULL, f(1.0), NULL, NULL,
                                   need - 1, NULL)
    assert b"workspace" in lib.dabsn_last_error()
