"""Calls that the vocabulary operators' documentation allows and that lie at the
edges of their kernels.

Tolerances count FP32 half steps as in test_gpu_vocab_ops.py, whose helpers and
64-bit definitions these tests use.
"""

from __future__ import annotations

import math

import pytest
import torch

from test_gpu_vocab_ops import (BF16, F32, U, _distill_reference, _half_step,  # noqa: F401
                                _logits, _near, _tokens, lib)

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------
# A teacher's rows that were ignored
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,V,K", [(7, 60, 5), (9, 1001, 20), (460, 8191, 9), (6, 40001, 33)])
def test_distilling_from_scores_with_ignored_rows(lib, rows, V, K, dtype):
    """token_log_probs marks a row whose token it ignores with id -1 and -inf;
    such a row lists nothing for distillation_loss."""
    teacher = _logits(rows, V, dtype, 1)
    tokens = _tokens(rows, V, 1)
    tokens[0] = -100
    tokens[rows - 1] = -100
    t = lib.token_log_probs(teacher, tokens, top_k=K)
    ignored = (tokens == -100).cpu()
    assert (t.top_tokens.cpu()[ignored] == -1).all() and int(ignored.sum()) == 3

    x = _logits(rows, V, dtype, 2)
    ids = torch.where(t.top_tokens == -1, -100, t.top_tokens)
    loss, size, grad, gsize, live, C = _distill_reference(x, ids, t.top_log_probs, 2.0)
    assert torch.equal(live, ~ignored)
    ltol = U * C * size * 2
    gtol = _half_step(dtype) * grad.abs() + 2 * U * C[:, None] * gsize + 1e-37
    plain = lib.distillation_loss(x, t.top_tokens, t.top_log_probs, temperature=2.0,
                                  reduction="none")
    _near(plain, loss, ltol)
    leaf = x.detach().requires_grad_()
    mean = lib.distillation_loss(leaf, t.top_tokens, t.top_log_probs, temperature=2.0)
    n = rows - 3
    _near(mean, loss.sum() / n, (ltol.sum() + U * size.sum()) / n + U * loss.sum().abs() / n)
    (dx,) = torch.autograd.grad(mean, leaf)
    _near(dx, grad / n, gtol / n + 1e-37)
    assert float(dx[ignored.cuda()].abs().max()) == 0.0


def test_an_id_of_minus_one_with_a_logit_is_outside(lib):
    """Only -inf makes an entry of id -1 absent."""
    from dabsn_b200 import _native

    _native.device_status(reset=True)
    x = _logits(3, 50, F32, 1)
    ids = torch.tensor([[-1, 3], [-1, 3], [2, -2]], device="cuda")
    tl = torch.tensor([[-math.inf, 1.0], [0.0, 1.0], [0.0, -math.inf]], device="cuda")
    loss = lib.distillation_loss(x, ids, tl, reduction="none")
    assert loss.isnan().tolist() == [False, True, True]
    assert _native.device_status(reset=True) == 8
