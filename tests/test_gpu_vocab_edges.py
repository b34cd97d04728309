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


# ---------------------------------------------------------------------------
# Ids outside the vocabulary
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,V", [(6, 60), (6, 9000), (450, 9000), (6, 40001)])
def test_gradients_of_lists_with_a_bad_id(lib, rows, V, dtype):
    """A list that names a token outside [0, V) has a NaN loss and a NaN
    gradient, also where no id of it is valid and where the student's row is
    masked throughout; the other rows are as if it were not there."""
    from dabsn_b200 import _native

    x = _logits(rows, V, dtype, 3)
    x[3] = -math.inf
    ids = torch.arange(4, device="cuda").repeat(rows, 1)
    tl = torch.randn(rows, 4, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    ids[0, 2] = V
    ids[1] = -5
    ids[3, 0] = V + 7
    bad = torch.tensor([0, 1, 3], device="cuda")
    rest = torch.tensor([r for r in range(rows) if r not in (0, 1, 3)], device="cuda")
    leaf = x.detach().requires_grad_()
    up = torch.linspace(0.5, 2.0, rows, device="cuda")
    none = lib.distillation_loss(leaf, ids, tl, reduction="none")
    total = lib.distillation_loss(leaf, ids, tl, reduction="sum")
    assert none[bad].isnan().all() and not none[rest].isnan().any() and total.isnan()
    grads = [torch.autograd.grad(none, leaf, up)[0],
             torch.autograd.grad(total, leaf, retain_graph=True)[0],
             torch.autograd.grad(total, leaf, torch.tensor(0.5, device="cuda"))[0]]
    good = ids.clone()
    good[bad] = -100
    a = lib.distillation_loss(leaf, good, tl, reduction="none")
    b = lib.distillation_loss(leaf, good, tl, reduction="sum")
    want = [torch.autograd.grad(a, leaf, up)[0],
            torch.autograd.grad(b, leaf, retain_graph=True)[0],
            torch.autograd.grad(b, leaf, torch.tensor(0.5, device="cuda"))[0]]
    for got, ref in zip(grads, want):
        assert got[bad].isnan().all()
        assert torch.equal(got[rest], ref[rest])
    # an upstream gradient of zero takes the row out
    up0 = up.clone()
    up0[bad] = 0.0
    none = lib.distillation_loss(leaf, ids, tl, reduction="none")
    (dx,) = torch.autograd.grad(none, leaf, up0)
    assert float(dx[bad].abs().max()) == 0.0 and torch.equal(dx[rest], want[0][rest])
    assert _native.device_status(reset=True) == 8


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V", [60, 9000])
def test_gradients_of_a_bad_token(lib, V, dtype):
    """Its log-probability is NaN and so is that gradient; its entropy does not
    depend on the token."""
    from dabsn_b200 import _native

    x = _logits(5, V, dtype, 4)
    x[4] = -math.inf
    tokens = torch.tensor([3, V, -7, 5, V + 1], device="cuda")
    bad = [1, 2, 4]
    leaf = x.detach().requires_grad_()
    out = lib.token_log_probs(leaf, tokens, temperature=0.9)
    up = torch.linspace(0.5, 1.5, 5, device="cuda")
    fine = lib.token_log_probs(leaf, tokens.clamp(0, V - 1), temperature=0.9)
    (g,) = torch.autograd.grad(out.log_prob, leaf, up, retain_graph=True)
    (want,) = torch.autograd.grad(fine.log_prob, leaf, up, retain_graph=True)
    assert out.log_prob.isnan().tolist() == [False, True, True, False, True]
    assert g[bad].isnan().all() and torch.equal(g[[0, 3]], want[[0, 3]])
    (h,) = torch.autograd.grad(out.entropy, leaf, up, retain_graph=True)
    (hwant,) = torch.autograd.grad(fine.entropy, leaf, up, retain_graph=True)
    assert torch.equal(h, hwant)
    (both,) = torch.autograd.grad([out.log_prob, out.entropy], leaf, [up, up], retain_graph=True)
    assert both[bad].isnan().all() and not both[[0, 3]].isnan().any()
    # an upstream gradient of zero takes the log-probability out
    up0 = up.clone()
    up0[bad] = 0.0
    (some,) = torch.autograd.grad([out.log_prob, out.entropy], leaf, [up0, up])
    assert torch.equal(some[bad], hwant[bad])
    assert _native.device_status(reset=True) == 8


def test_nan_of_a_teacher_with_a_masked_student(lib):
    """NaN among the teacher's logits makes the listed tokens' gradient NaN,
    whatever the student's row holds."""
    for rows, V in ((4, 60), (4, 9000), (450, 9000)):
        x = _logits(rows, V, F32, 1)
        x[1] = -math.inf
        ids = torch.arange(6, device="cuda").repeat(rows, 1)
        tl = torch.zeros(rows, 6, device="cuda")
        tl[1, 2] = math.nan
        leaf = x.detach().requires_grad_()
        loss = lib.distillation_loss(leaf, ids, tl, reduction="none")
        total = lib.distillation_loss(leaf, ids, tl, reduction="sum")
        assert loss.isnan().tolist() == [r == 1 for r in range(rows)]
        for grad in (torch.autograd.grad(loss, leaf, torch.ones_like(loss))[0],
                     torch.autograd.grad(total, leaf, retain_graph=True)[0],
                     torch.autograd.grad(total, leaf, torch.tensor(2.0, device="cuda"))[0]):
            assert grad[1, :6].isnan().all() and float(grad[1, 6:].abs().max()) == 0.0
            rest = [r for r in range(rows) if r != 1]
            assert not grad[rest].isnan().any()


# ---------------------------------------------------------------------------
# Loops that only large calls go round
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V,pad,offset", [(4099, 5, 3), (4104, 0, 0), (2057, 1, 1)])
def test_distillation_of_many_rows_with_gaps(lib, V, pad, offset, dtype):
    """A CTA of the one-pass gradient takes every 444th row: rows without a loss
    between two that have one, several in a row, and at either end."""
    rows, K, T = 2011, 7, 1.5
    x = _logits(rows, V, dtype, V, pad=pad, offset=offset)
    gen = torch.Generator().manual_seed(V)
    ids = torch.randint(0, V, (rows, K), generator=gen)
    tl = torch.randn(rows, K, generator=gen) * 2.0
    ids[::3] = -100
    for first in (5, 17, 200, 443):
        ids[first::444] = -100  # nothing at all for this CTA
    for first in (7, 100):
        ids[first + 444] = ids[first + 888] = -100  # two in a row, between others
    ids[0], ids[444], ids[1332] = 1, 2, 3
    ids, tl = ids.cuda(), tl.cuda()
    loss, size, grad, gsize, live, C = _distill_reference(x, ids, tl, T)
    n = int(live.sum())
    assert 0 < n < rows
    ltol = U * C * size * 2
    gtol = _half_step(dtype) * grad.abs() + 2 * U * C[:, None] * gsize + 1e-37
    plain = lib.distillation_loss(x, ids, tl, temperature=T, reduction="none")
    _near(plain, loss, ltol)
    leaf = x.detach().requires_grad_()
    got = lib.distillation_loss(leaf, ids, tl, temperature=T)
    _near(got, loss.sum() / n, (ltol.sum() + U * size.sum()) / n + U * loss.sum().abs() / n)
    (dx,) = torch.autograd.grad(got, leaf, retain_graph=True)
    _near(dx, grad / n, gtol / n + 1e-37)
    # the reverse from the logits, over the same rows
    (half,) = torch.autograd.grad(got, leaf, torch.tensor(0.5, device="cuda"))
    _near(half, grad / n * 0.5, gtol / n * 0.51 + 1e-37)


@pytest.mark.parametrize("N,V", [(600011, 37), (600011, 900), (262145, 70001), (786432, 70001)])
def test_embedding_gradient_of_many_tokens(lib, N, V):
    """More tokens than 256 sort blocks rank in one step, one to three digits;
    sums of small whole numbers are exact."""
    g = torch.Generator().manual_seed(N + V)
    tokens = (torch.rand(N, generator=g) ** 3 * V).long().clamp(max=V - 1)
    go = torch.randint(-4, 5, (N, 8), generator=g).float()
    w = torch.zeros(V, 8, device="cuda", requires_grad=True)
    (dw,) = torch.autograd.grad(lib.embedding(tokens.cuda(), w), w, go.cuda())
    assert torch.equal(dw.cpu(), torch.zeros(V, 8).index_add_(0, tokens, go))


@pytest.mark.parametrize("D", [515, 1029, 2056])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_embedding_runs_over_column_tiles(lib, D, dtype):
    """Tokens whose positions cover whole pieces of the sums, in tables wider
    than a tile of columns; whole numbers, exact."""
    runs = [63, 1, 9000, 64, 65, 127, 129, 192, 2, 1, 62, 300, 33, 33, 1000]
    for many in (1, 4):  # below and above 32768 positions
        sizes = runs * many
        V = 2 * len(sizes) + 1
        g = torch.Generator().manual_seed(D)
        tokens = torch.cat([torch.full((n,), 2 * i + 1) for i, n in enumerate(sizes)])
        tokens = tokens[torch.randperm(len(tokens), generator=g)]
        go = torch.randint(-4, 5, (len(tokens), D), generator=g).float()
        w = torch.zeros(V, D, device="cuda", requires_grad=True)
        out = lib.embedding(tokens.cuda(), w, dtype=dtype)
        (dw,) = torch.autograd.grad(out, w, go.cuda().to(dtype))
        assert torch.equal(dw.cpu(), torch.zeros(V, D).index_add_(0, tokens, go))


# ---------------------------------------------------------------------------
# Tensors that are not what a kernel can read
# ---------------------------------------------------------------------------
def test_tensors_without_memory_are_refused(lib):
    """Under functionalize a tensor's data pointer is null."""
    x = _logits(4, 50, F32, 1)
    t = torch.arange(4, device="cuda")
    for call in (lambda z: lib.token_log_probs(z, t).log_prob,
                 lambda z: lib.distillation_loss(z, t[:, None], torch.zeros(4, 1, device="cuda")),
                 lambda z: lib.embedding(t, z)):
        with pytest.raises(RuntimeError, match="null pointer"):
            torch.func.functionalize(call)(x)


# ---------------------------------------------------------------------------
# Tracing and forward mode, with the kernels themselves
# ---------------------------------------------------------------------------
def _calls(lib):
    t = torch.tensor([4, 0, 49, 7], device="cuda")
    ids = torch.tensor([[1, 2], [3, 4], [5, 6], [0, 49]], device="cuda")
    tl = torch.linspace(-1, 1, 8, device="cuda").view(4, 2)
    return (lambda z: lib.token_log_probs(z, t, top_k=2).log_prob + 0,
            lambda z: lib.distillation_loss(z, ids, tl) + 0,
            lambda z: lib.embedding(t % 4, z) + 0)


def test_traced_and_compiled_calls_compute(lib):
    x, y = _logits(4, 50, F32, 1), _logits(4, 50, F32, 2)
    for call in _calls(lib):
        traced = torch.jit.trace(call, (x,))
        assert torch.equal(traced(y), call(y)) and torch.equal(traced(x), call(x))
        torch._dynamo.reset()
        compiled = torch.compile(call, backend="eager")
        assert torch.equal(compiled(y), call(y))
        a, b = y.clone().requires_grad_(), y.clone().requires_grad_()
        (got,) = torch.autograd.grad(compiled(a).sum(), a)
        (want,) = torch.autograd.grad(call(b).sum(), b)
        assert torch.equal(got, want)


def test_forward_mode_is_refused(lib):
    x = _logits(4, 50, F32, 1)
    for call in _calls(lib):
        with torch.autograd.forward_ad.dual_level():
            dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call(dual)
        with pytest.raises(RuntimeError):
            torch.func.jvp(call, (x,), (torch.ones_like(x),))


def test_the_status_of_another_stream_is_raised(lib):
    """raise_on_device_status waits for work that is still queued on a stream of
    its own."""
    w = torch.randn(5, 16, device="cuda")
    bad, good = torch.tensor([1, 5], device="cuda"), torch.tensor([1, 4], device="cuda")
    lib.embedding(good, w)
    lib.raise_on_device_status()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(100_000_000)
        lib.embedding(bad, w)
    with pytest.raises(RuntimeError, match="outside"):
        lib.raise_on_device_status()
    lib.raise_on_device_status()
    lib.embedding(bad, w)
    with pytest.raises(RuntimeError, match="outside"):
        lib.raise_on_device_status(0)


# ---------------------------------------------------------------------------
# Counted launches
# ---------------------------------------------------------------------------
def _kernels_of(call):
    """Kernels in a graph of the call, and how many the library counted."""
    from cuda.bindings import runtime as rt

    from dabsn_b200 import ops

    graph = torch.cuda.CUDAGraph(keep_graph=True)
    before = ops.LAUNCH_COUNT["n"]
    with torch.cuda.graph(graph):
        call()
    counted = ops.LAUNCH_COUNT["n"] - before
    raw = rt.cudaGraph_t(graph.raw_cuda_graph())
    err, _, total = rt.cudaGraphGetNodes(raw, 0)
    assert err == rt.cudaError_t.cudaSuccess
    if total == 0:
        return 0, counted
    err, nodes, total = rt.cudaGraphGetNodes(raw, total)
    assert err == rt.cudaError_t.cudaSuccess
    kinds = [rt.cudaGraphNodeGetType(node)[1] for node in nodes[:total]]
    return sum(k == rt.cudaGraphNodeType.cudaGraphNodeTypeKernel for k in kinds), counted


@pytest.mark.parametrize("n,V", [(0, 9), (1, 9), (64, 9), (65, 9), (96, 9), (97, 300),
                                 (8192, 300), (8193, 9), (8193, 255), (8193, 256), (8193, 65535),
                                 (40000, 65536), (40000, 1009)])
def test_launches_of_the_embedding(lib, n, V):
    from dabsn_b200 import ops

    t = torch.zeros(n, dtype=torch.int64, device="cuda")
    w = torch.zeros(V, 8, device="cuda")
    g = torch.zeros(n, 8, device="cuda")
    for call in (lambda: ops.embedding_forward(t, w, 1.0, F32),
                 lambda: ops.embedding_backward(t, g, V, 1.0, None, F32)):
        call()
        kernels, counted = _kernels_of(call)
        assert kernels == counted


@pytest.mark.parametrize("rows", [0, 3])
def test_launches_of_scores_and_distillation(lib, rows):
    from dabsn_b200 import ops

    x, t = _logits(rows, 40, F32, 1), torch.zeros(rows, dtype=torch.int64, device="cuda")
    ids, tl = t[:, None].contiguous(), torch.zeros(rows, 1, device="cuda")
    for k in (0, 3):
        lp, h, _, _, stats = ops.token_scores_forward(x, t, k, 1.0, -100)
        kernels, counted = _kernels_of(lambda: ops.token_scores_forward(x, t, k, 1.0, -100))
        assert kernels == counted
        kernels, counted = _kernels_of(
            lambda: ops.token_scores_backward(x, t, 1.0, -100, stats, h, lp, h))
        assert kernels == counted
    for reduction in ("none", "sum"):
        def forward(reduction=reduction):
            return ops.distill_forward(x, ids, tl, 1.0, 1.0, -100, reduction, reduction == "sum")

        loss, ws, _ = forward()
        kernels, counted = _kernels_of(forward)
        assert kernels == counted
        kernels, counted = _kernels_of(
            lambda: ops.distill_backward(x, ws, 1, 1.0, 1.0, False, loss))
        assert kernels == counted


def test_make_fx_is_refused(lib):
    from torch.fx.experimental.proxy_tensor import make_fx

    x = _logits(4, 50, F32, 1)
    for call in _calls(lib):
        for pre_dispatch in (False, True):
            with pytest.raises(RuntimeError, match="make_fx"):
                make_fx(call, pre_dispatch=pre_dispatch)(x)
        leaf = x.clone().requires_grad_()
        out = call(leaf)
        with pytest.raises(RuntimeError, match="make_fx"):  # on the engine's thread
            make_fx(lambda g: torch.autograd.grad(out, leaf, g)[0])(torch.ones_like(out))


def test_a_gradient_with_a_pending_sign(lib):
    """An upstream gradient that is the imaginary part of a conjugate: for one
    number a contiguous view whose sign is still to be turned."""
    x = _logits(1, 50, F32, 1)
    t = torch.tensor([4], device="cuda")

    def log_prob(z):
        return lib.token_log_probs(z, t).log_prob

    def column(z):
        return lib.embedding(t * 0, z[:, :1])

    for f in (log_prob, column):
        a = x.clone().requires_grad_()
        out = f(a)
        up = torch.complex(torch.zeros_like(out), torch.full_like(out, 2.0)).detach().conj().imag
        assert up.is_neg() and up.is_contiguous()
        (want,) = torch.autograd.grad(out, a, torch.full_like(out, -2.0), retain_graph=True)
        (got,) = torch.autograd.grad(out, a, up)
        assert torch.equal(got, want) and float(want.abs().max()) > 0
