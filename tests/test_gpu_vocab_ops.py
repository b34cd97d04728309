"""Token log-probabilities, distillation from top logits and the scaled
embedding against their definitions in 64 bits.

Tolerances, from the arithmetic.  u = 2^-24 is FP32's half step.  A row's sums
of V exponentials run over at most V / 32 terms in sequence, then over fewer
than 64 merges, so their relative error is at most u (V / 32 + 64), to which an
exponential adds 2 ulp and the rounding of its argument (u |x - m| / T, a few
times): C = V / 32 + 64 + 8 max |x - m| / T counts them in units of u.  An
output held in a type is off by half its step once more (u for FP32, 2^-9 of
BF16's 8-bit significand, taken as finfo.eps / 2).  Sums of n gradient rows in
FP32 are off by u n times the sum of their magnitudes.
"""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def lib():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    import dabsn_b200
    from dabsn_b200 import _native

    _native.device_status(reset=True)
    return dabsn_b200


def _half_step(dtype):
    return torch.finfo(dtype).eps / 2


def _logits(rows, V, dtype, seed, *, kind="normal", pad=0, offset=0):
    """[rows, V] on the GPU; `pad` columns behind each row and `offset`
    elements before the first make the rows start anywhere."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, V, generator=g) * 3.0
    if kind == "ties":
        x = torch.randint(-2, 3, (rows, V), generator=g).float()
    elif kind == "flat":
        x = torch.zeros(rows, V)
    elif kind == "far":
        x = x + 1000.0
    elif kind == "falling":
        x = x.sort(dim=-1, descending=True).values
    elif kind == "rising":
        x = x.sort(dim=-1).values
    elif kind in ("masked", "lowest"):
        low = -math.inf if kind == "masked" else torch.finfo(dtype).min
        keep = torch.rand(rows, V, generator=g) < 0.05
        keep[0] = False  # nothing left
        if rows > 1:
            keep[1] = False
            keep[1, V // 2] = True  # one left
        x = x.to(dtype).float().masked_fill(~keep, low)
    elif kind == "clustered":
        # columns that one thread of a strided sweep reads together are the
        # large ones
        high = (torch.arange(V) // 8) % 256 < 7
        x = torch.where(high, x.abs() + 50.0, x - 50.0)
    store = torch.full((rows * (V + pad) + offset,), float("nan"), dtype=dtype, device="cuda")
    view = store[offset:].view(rows, V + pad)[:, :V]
    view.copy_(x.to(dtype))
    return view


def _score_reference(x, tokens, T, ignore):
    """Definitions in 64 bits, on the CPU: log p, entropy and rows' C."""
    z = x.double().cpu() / T
    empty = (z == -math.inf).all(-1)
    m = z.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    logp = z - m - torch.log(torch.exp(z - m).sum(-1, keepdim=True))
    logp = torch.where(empty[:, None], torch.full_like(logp, -math.inf), logp)
    p = torch.exp(logp)
    ent = -(p * torch.where(p > 0, logp, torch.zeros_like(logp))).sum(-1)
    live = tokens.cpu() != ignore
    gap = (m - torch.where(z < m - 160, m, z)).amax(-1)
    C = z.shape[-1] / 32 + 64 + 8 * gap
    return logp, p, torch.where(live, ent, torch.zeros_like(ent)), live, empty, C


def _tokens(rows, V, seed, ignored=True):
    g = torch.Generator().manual_seed(seed + 1)
    t = torch.randint(0, V, (rows,), generator=g)
    if ignored and rows > 2:
        t[rows // 2] = -100
    return t.cuda()


SCORE_CASES = [
    (1, 1, "normal", 0, 0), (1, 2, "normal", 0, 0), (3, 7, "normal", 0, 0),
    (5, 17, "ties", 3, 1), (4, 60, "masked", 0, 0), (6, 64, "normal", 64, 0),
    (9, 515, "ties", 1, 5), (3, 1000, "lowest", 0, 0), (4, 1001, "masked", 0, 3),
    (3, 1023, "flat", 0, 0), (7, 4099, "normal", 5, 0), (2, 8192, "rising", 0, 0),
    (2, 8200, "falling", 8, 0), (3, 32000, "normal", 0, 0), (4, 32771, "masked", 0, 0),
    (2, 32771, "far", 2, 7), (3, 33000, "flat", 0, 0), (300, 4096, "normal", 0, 0),
    (2, 163840, "clustered", 0, 0), (1, 200003, "normal", 0, 0), (700, 100, "ties", 0, 0),
]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,V,kind,pad,offset", SCORE_CASES)
def test_token_log_probs(lib, rows, V, kind, pad, offset, dtype):
    T = 1.0 if V % 2 else 0.75
    x = _logits(rows, V, dtype, V + rows, kind=kind, pad=pad, offset=offset)
    tokens = _tokens(rows, V, V)
    k = min(V, 20 if V > 100 else 7)
    leaf = x.detach().requires_grad_()
    out = lib.token_log_probs(leaf, tokens, top_k=k, temperature=T)
    logp, p, ent, live, empty, C = _score_reference(x, tokens, T, -100)
    at = tokens.cpu().clamp(min=0)
    lp = torch.where(live, logp.gather(1, at[:, None]).squeeze(1), torch.zeros(rows).double())
    assert out.log_prob.dtype == F32 and out.entropy.dtype == F32
    _near(out.log_prob, lp, U * (C + 4 * lp.abs()), inf_below=-3e38)
    _near(out.entropy, ent, U * C * (2 + math.log(V)))

    # the alternatives: the same ids, ties to the lowest
    order = torch.sort(x.float().cpu(), dim=-1, descending=True, stable=True).indices[:, :k]
    assert torch.equal(out.top_tokens.cpu(),
                       torch.where(live[:, None], order, torch.full_like(order, -1)))
    top = torch.where(live[:, None], logp.gather(1, order), torch.full_like(logp[:, :k], -math.inf))
    _near(out.top_log_probs, top, U * (C[:, None] + 4 * top.abs()), inf_below=-3e38)

    # the reverse of both numbers
    gen = torch.Generator().manual_seed(V + 3)
    g = torch.randn(rows, generator=gen)
    h = torch.randn(rows, generator=gen)
    for gl, he in ((g, h), (g, None), (None, h)):
        outs = [o for o, w in ((out.log_prob, gl), (out.entropy, he)) if w is not None]
        ups = [w.cuda() for w in (gl, he) if w is not None]
        (dx,) = torch.autograd.grad(outs, leaf, ups, retain_graph=True)
        G = (torch.zeros(rows) if gl is None else gl).double()[:, None]
        Hh = (torch.zeros(rows) if he is None else he).double()[:, None]
        lz = torch.where(p > 0, logp, torch.zeros_like(logp))
        hit = torch.zeros_like(p).scatter_(1, at[:, None], 1.0)
        exact = (G * (hit - p) - Hh * p * (lz + ent[:, None])) / T
        exact[empty | ~live] = 0.0
        size = (p * (G.abs() + Hh.abs() * (lz.abs() + ent[:, None] + 1)) + G.abs() * hit) / T
        assert dx.dtype == dtype and dx.shape == x.shape
        _near(dx, exact, _half_step(dtype) * exact.abs() + 2 * U * C[:, None] * size + 1e-37)


def _near(got, want, tol, inf_below=None):
    got, want = got.detach().double().cpu(), want.double()
    if inf_below is not None:  # FP32 overflows to -inf where 64 bits do not
        want = torch.where(want < inf_below, torch.full_like(want, -math.inf), want)
        got = torch.where(got < inf_below, torch.full_like(got, -math.inf), got)
    finite = torch.isfinite(want)
    assert torch.equal(got[~finite], want[~finite])
    tol = torch.as_tensor(tol).double().expand_as(want)
    bad = (got - want).abs()[finite] - tol[finite]
    assert not torch.isnan(got[finite]).any()
    if bad.numel():
        i = int(bad.argmax())
        assert float(bad.max()) <= 0, (got[finite][i], want[finite][i], tol[finite][i])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V,pad,offset", [(60, 1, 3), (300, 0, 0), (5000, 3, 1), (40001, 0, 0)])
def test_token_log_probs_few_left(lib, V, pad, offset, dtype):
    """0, 1, ... logits left by a mask, around the number asked for: those
    first, then the masked ids in order; the same of one shared value."""
    k = 20
    x = _logits(2 * k + 4, V, dtype, V, kind="flat", pad=pad, offset=offset)
    g = torch.Generator().manual_seed(V)
    for r in range(2 * k + 4):
        left = torch.randperm(V, generator=g)[: r // 2].cuda()
        x[r] = -math.inf if r % 2 else -7.0
        x[r, left] = torch.randn(len(left), generator=g).to(dtype).cuda()
    out = lib.token_log_probs(x, _tokens(2 * k + 4, V, 1, ignored=False), top_k=k)
    order = torch.sort(x.float().cpu(), dim=-1, descending=True, stable=True).indices[:, :k]
    assert torch.equal(out.top_tokens.cpu(), order)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_token_log_probs_top_k_range(lib, dtype):
    for V, k in ((128, 128), (130, 1), (5000, 128), (40000, 128), (60, 60)):
        x = _logits(3, V, dtype, k, kind="ties" if V == 5000 else "normal")
        out = lib.token_log_probs(x, _tokens(3, V, 1, ignored=False), top_k=k)
        order = torch.sort(x.float().cpu(), dim=-1, descending=True, stable=True).indices[:, :k]
        assert torch.equal(out.top_tokens.cpu(), order), (V, k)


def test_token_log_probs_non_finite_rows(lib):
    x = _logits(4, 600, F32, 3)
    x[0, 5] = math.nan
    x[1, 7] = math.inf
    x[2, 100:] = -math.inf
    out = lib.token_log_probs(x, _tokens(4, 600, 2, ignored=False), top_k=3)
    assert out.log_prob[:2].isnan().all() and out.entropy[:2].isnan().all()
    assert out.top_log_probs[:2].isnan().all()
    assert ((out.top_tokens >= 0) & (out.top_tokens < 600)).all()
    assert not out.entropy[2:].isnan().any()


def test_zeros_of_either_sign_tie(lib):
    x = torch.full((1, 300), -1.0, device="cuda")
    x[0, 10], x[0, 4], x[0, 200] = 0.0, -0.0, 0.0
    out = lib.token_log_probs(x, torch.zeros(1, dtype=torch.int64, device="cuda"), top_k=4)
    assert out.top_tokens[0].tolist() == [4, 10, 200, 0]


def test_token_log_probs_shapes_and_int32(lib):
    x = _logits(12, 50, BF16, 1).view(3, 4, 50)
    t = _tokens(12, 50, 4, ignored=False).view(3, 4)
    a = lib.token_log_probs(x, t, top_k=2)
    b = lib.token_log_probs(x, t.int(), top_k=2)
    assert a.log_prob.shape == (3, 4) and a.top_tokens.shape == (3, 4, 2)
    assert torch.equal(a.log_prob, b.log_prob) and torch.equal(a.top_tokens, b.top_tokens)
    one = lib.token_log_probs(x[1, 2], t[1, 2])
    assert one.log_prob.shape == () and one.top_tokens is None and one.top_log_probs is None
    assert torch.equal(one.log_prob, a.log_prob[1, 2])
    none = lib.token_log_probs(x[:0], t[:0], top_k=2)
    assert none.log_prob.shape == (0, 4) and none.top_tokens.shape == (0, 4, 2)
    # columns apart: copied to rows
    y = x.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(lib.token_log_probs(y, t).log_prob, a.log_prob)
    # one row for all tokens.  Its copies start at other alignments, so their
    # sums run in another order: each is within u C (2 + log V) of the entropy
    # (C = V / 32 + 64 + 8 max gap <= 170, the gap being below 13), and two
    # of them within twice that.
    wide = x[:1, :1].expand(3, 4, 50)
    _near(lib.token_log_probs(wide, t).entropy, a.entropy[0, 0].expand(3, 4).cpu(),
          2 * U * 170 * (2 + math.log(50)))


def test_bad_token_is_reported(lib):
    from dabsn_b200 import _native

    _native.device_status(reset=True)
    x = _logits(3, 40, F32, 1)
    out = lib.token_log_probs(x, torch.tensor([0, 40, 3], device="cuda"))
    assert out.log_prob.isnan().tolist() == [False, True, False]
    with pytest.raises(RuntimeError, match="outside"):
        _native.raise_on_device_status()
    w = torch.randn(5, 16, device="cuda", requires_grad=True)
    e = lib.embedding(torch.tensor([1, 5, -1, 4], device="cuda"), w)
    assert e.isnan().all(-1).tolist() == [False, True, True, False]
    (dw,) = torch.autograd.grad(e, w, torch.ones_like(e))
    assert dw.sum(-1).tolist() == [0.0, 16.0, 0.0, 0.0, 16.0]
    with pytest.raises(RuntimeError, match="outside"):
        _native.raise_on_device_status()
    loss = lib.distillation_loss(x, torch.tensor([[1], [2], [40]], device="cuda"),
                                 torch.zeros(3, 1, device="cuda"), reduction="none")
    assert loss.isnan().tolist() == [False, False, True]
    with pytest.raises(RuntimeError, match="outside"):
        _native.raise_on_device_status()
    assert _native.device_status() == 0


# ---------------------------------------------------------------------------
# Distillation
# ---------------------------------------------------------------------------
DISTILL_CASES = [
    (1, 1, 1, "normal", 0, 0), (2, 5, 3, "normal", 0, 0), (5, 60, 8, "normal", 0, 0),
    (6, 64, 33, "masked", 2, 0), (4, 1001, 64, "normal", 0, 3), (3, 8200, 1, "lowest", 8, 0),
    (7, 4099, 100, "far", 5, 0), (3, 32000, 64, "normal", 0, 0), (2, 32771, 256, "flat", 0, 1),
    (300, 4096, 16, "normal", 0, 0), (1, 128003, 128, "normal", 0, 0), (900, 70, 5, "ties", 0, 0),
    (2, 700001, 4, "normal", 0, 0), (500, 33000, 3, "normal", 0, 0),
    (301, 4099, 7, "normal", 5, 3), (460, 8191, 5, "masked", 1, 1), (451, 1025, 40, "ties", 0, 0),
]


def _teacher(rows, V, K, seed, dtype=F32):
    g = torch.Generator().manual_seed(seed + 2)
    ids = torch.randint(0, V, (rows, K), generator=g)  # the same id twice, now and then
    logits = torch.randn(rows, K, generator=g) * 2.0
    drop = torch.rand(rows, K, generator=g) < 0.2
    ids[drop] = -100
    if rows > 2:
        ids[2] = -100  # lists nothing
    if rows > 3:
        logits[3, : (K + 1) // 2] = -math.inf
    if rows > 4:
        logits[4] = -math.inf
    return ids.cuda(), logits.to(dtype).cuda()


def _distill_reference(x, ids, tl, T, low=-math.inf):
    logp, p, _, _, empty, C = _score_reference(x, torch.zeros(x.shape[0]), T, -100)
    ids, tl = ids.cpu(), tl.double().cpu()
    t = torch.where(ids != -100, tl / T, torch.full_like(tl, -math.inf))
    live = (t > -math.inf).any(-1)
    m = t.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    e = torch.exp(t - m)
    q = torch.where(live[:, None], e / e.sum(-1, keepdim=True), torch.zeros_like(e))
    at = ids.clamp(min=0)
    lp = logp.gather(1, at)
    term = torch.where(q > 0, q * (torch.log(torch.where(q > 0, q, 1.0)) - lp),
                       torch.zeros_like(q))
    size = torch.where(q > 0, q * (torch.log(torch.where(q > 0, q, 1.0)).abs() + lp.abs() + 1),
                       torch.zeros_like(q))
    loss = T * T * term.sum(-1)
    merged = torch.zeros_like(p).scatter_add_(1, at, q)
    grad = T * (p - merged)
    grad[~live | empty] = 0.0
    return loss, T * T * size.sum(-1), grad, T * (p + merged), live, C


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,V,K,kind,pad,offset", DISTILL_CASES)
def test_distillation(lib, rows, V, K, kind, pad, offset, dtype):
    T = 2.0 if K % 2 else 1.0
    x = _logits(rows, V, dtype, V + K, kind=kind, pad=pad, offset=offset)
    ids, tl = _teacher(rows, V, K, V, dtype if K % 3 else F32)
    loss, size, grad, gsize, live, C = _distill_reference(x, ids, tl, T)
    ltol = U * C * size * 2
    gtol = _half_step(dtype) * grad.abs() + 2 * U * C[:, None] * gsize + 1e-37
    plain = lib.distillation_loss(x, ids, tl, temperature=T, reduction="none")
    assert plain.dtype == F32 and plain.shape == (rows,)
    finite = loss < 1e30
    _near(plain.cpu()[finite], loss[finite], ltol[finite])
    assert (plain.cpu()[~finite] > 1e30).all()
    n = max(1, int(live.sum()))
    for reduction, share in (("mean", 1.0 / n), ("sum", 1.0)):
        leaf = x.detach().requires_grad_()
        got = lib.distillation_loss(leaf, ids, tl, temperature=T, reduction=reduction)
        without = lib.distillation_loss(x, ids, tl, temperature=T, reduction=reduction)
        if finite.all():
            want = loss.sum() * share
            _near(got, want, (ltol.sum() + U * (size.sum())) * share + U * want.abs())
            _near(without, want, (ltol.sum() + U * (size.sum())) * share + U * want.abs())
        (dx,) = torch.autograd.grad(got, leaf, retain_graph=True)
        assert dx.dtype == dtype
        _near(dx, grad * share, gtol * share + 1e-37)
        # another upstream gradient, and the first one again
        (half,) = torch.autograd.grad(got, leaf, torch.tensor(-0.3, device="cuda"),
                                      retain_graph=True)
        _near(half, grad * share * -0.3, gtol * share * 0.3 * 1.01 + 1e-37)
        (again,) = torch.autograd.grad(got, leaf)
        assert torch.equal(again, dx)
    # a factor known beforehand: a power of two changes no digit
    leaf = x.detach().requires_grad_()
    got4 = lib.distillation_loss(leaf, ids, tl, temperature=T, weight=0.25, reduction="sum")
    assert torch.equal(got4, got.detach() * 0.25)
    for up in (1.0, 0.5):
        (dx4,) = torch.autograd.grad(got4, leaf, torch.tensor(up, device="cuda"),
                                     retain_graph=True)
        _near(dx4, grad * 0.25 * up, gtol * 0.25 * up + 1e-37)
    leaf = x.detach().requires_grad_()
    w = torch.randn(rows, generator=torch.Generator().manual_seed(5))
    got = lib.distillation_loss(leaf, ids, tl, temperature=T, reduction="none")
    assert torch.equal(lib.distillation_loss(x, ids, tl, temperature=T, weight=2.0,
                                             reduction="none"), got.detach() * 2.0)
    (dx,) = torch.autograd.grad(got, leaf, w.cuda())
    _near(dx, grad * w.double()[:, None], gtol * w.double().abs()[:, None] * 1.01 + 1e-37)


@pytest.mark.parametrize("rows,V", [(4, 60), (4, 9000), (450, 9000)])
def test_distillation_of_non_finite_numbers(lib, rows, V):
    """Each row by itself: NaN or +inf of the teacher, NaN of the student, all
    logits of the student masked, one listed token masked."""
    x = _logits(rows, V, F32, 1)
    ids = torch.arange(6, device="cuda").repeat(rows, 1)
    tl = torch.randn(rows, 6, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    tl[0, 2] = math.nan
    tl[1, 3] = math.inf
    x[2, V - 1] = math.nan
    x[3] = -math.inf
    if rows > 4:
        x[4, 5] = -math.inf
    leaf = x.detach().requires_grad_()
    loss = lib.distillation_loss(leaf, ids, tl, reduction="none")
    assert loss[:3].isnan().all() and loss[3] == math.inf
    total = lib.distillation_loss(leaf, ids, tl, reduction="sum")
    for grad in (torch.autograd.grad(loss, leaf, torch.ones_like(loss))[0],
                 torch.autograd.grad(total, leaf)[0]):
        assert grad[0, :6].isnan().any() and grad[1, :6].isnan().any()
        assert grad[2].isnan().all()
        assert float(grad[3].abs().max()) == 0.0
        if rows > 4:
            assert loss[4] == math.inf and torch.isfinite(grad[4:]).all()
            assert torch.isfinite(loss[5:]).all()


def test_refusals(lib):
    x, t = _logits(3, 200, F32, 1), _tokens(3, 200, 1)
    ids, tl = _teacher(3, 200, 4, 1)
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        lib.token_log_probs(x.half(), t)
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        lib.distillation_loss(x.double(), ids, tl)
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        lib.distillation_loss(x, ids, tl.half())
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        lib.embedding(t.clamp(min=0), torch.zeros(200, 8, device="cuda"), dtype=torch.float16)
    with pytest.raises(TypeError, match="int64 or int32"):
        lib.token_log_probs(x, t.float())
    with pytest.raises(TypeError, match="int64 or int32"):
        lib.embedding(t.short(), torch.zeros(200, 8, device="cuda"))
    with pytest.raises(ValueError, match="top_k"):
        lib.token_log_probs(x, t, top_k=129)
    with pytest.raises(ValueError, match="top_k"):
        lib.token_log_probs(x[:, :7], t.clamp(max=6), top_k=8)
    with pytest.raises(ValueError, match="entries"):
        lib.distillation_loss(x, ids.repeat(1, 65), tl.repeat(1, 65))
    with pytest.raises(ValueError, match="temperature"):
        lib.distillation_loss(x, ids, tl, temperature=0.0)
    with pytest.raises(ValueError, match="same device"):
        lib.token_log_probs(x, t.cpu())
    with pytest.raises(ValueError, match="same device"):
        lib.embedding(t.cpu(), torch.zeros(200, 8, device="cuda"))


def test_distillation_of_nothing(lib):
    x = _logits(3, 40, BF16, 1).requires_grad_()
    ids = torch.full((3, 2), -100, device="cuda")
    loss = lib.distillation_loss(x, ids, torch.zeros(3, 2, device="cuda"))
    (dx,) = torch.autograd.grad(loss, x)
    assert float(loss) == 0.0 and float(dx.abs().max()) == 0.0
    none = lib.distillation_loss(x[:0], ids[:0], torch.zeros(0, 2, device="cuda"))
    assert float(none) == 0.0
    (dx,) = torch.autograd.grad(none, x)
    assert float(dx.abs().max()) == 0.0


# ---------------------------------------------------------------------------
# Embedding
# ---------------------------------------------------------------------------
EMBED_CASES = [
    (1, 1, 1), (3, 2, 8), (7, 5, 17), (64, 60, 128), (100, 1009, 515), (257, 300, 64),
    (4099, 1009, 72), (5000, 257, 33), (20000, 70000, 16), (33000, 40, 24), (9000, 32000, 264),
]


@pytest.mark.parametrize("wdtype,odtype", [(F32, F32), (F32, BF16), (BF16, BF16), (BF16, F32)])
@pytest.mark.parametrize("N,V,D", EMBED_CASES)
def test_embedding(lib, N, V, D, wdtype, odtype):
    g = torch.Generator().manual_seed(N + V)
    # few tokens take most positions, some take none
    tokens = (torch.rand(N, generator=g) ** 4 * V).long().clamp(max=V - 1)
    weight = torch.randn(V, D, generator=g).to(wdtype)
    pad_idx, scale = (V // 2 - V if V > 1 else None), 1.75
    leaf = weight.cuda().requires_grad_()
    out = lib.embedding(tokens.cuda(), leaf, scale=scale, padding_idx=pad_idx, dtype=odtype)
    want = weight.double()[tokens] * scale
    _near(out, want, (_half_step(odtype) + U) * 1.01 * want.abs())
    go = torch.randn(N, D, generator=g).to(odtype)
    (dw,) = torch.autograd.grad(out, leaf, go.cuda(), retain_graph=True)
    (dw2,) = torch.autograd.grad(out, leaf, go.cuda())
    assert torch.equal(dw, dw2)
    part = go.double()
    if pad_idx is not None:
        part = part * (tokens != pad_idx % V)[:, None]
    want = torch.zeros(V, D).double().index_add_(0, tokens, part) * scale
    size = torch.zeros(V, D).double().index_add_(0, tokens, part.abs()) * scale
    n = torch.bincount(tokens, minlength=V).double()[:, None]
    assert dw.dtype == wdtype
    _near(dw, want, _half_step(wdtype) * 1.01 * want.abs() + U * (n + 1) * size)


RUNS = [
    [1], [64], [65, 1], [32, 32, 32], [31, 1, 64, 2, 95, 33], [1, 63, 1, 64, 1, 65],
    [16, 32, 16, 32, 64], [200], [31, 97, 1, 1, 30], [5] * 41, [128, 128, 127, 129],
    [40000], [63, 1, 40000, 64, 65, 127, 129, 192, 2], [33] * 1200, [64] * 520 + [1],
    [1, 62, 2, 62, 130] * 140,
]


@pytest.mark.parametrize("D", [8, 21, 72])
@pytest.mark.parametrize("runs", RUNS, ids=lambda r: f"{len(r)}runs{sum(r)}")
def test_embedding_runs(lib, runs, D):
    """Numbers of positions per token that begin and end at every place of the
    pieces that the sums are cut into, absent tokens between them; the sums of
    small whole numbers are exact."""
    g = torch.Generator().manual_seed(len(runs))
    V = 2 * len(runs) + 1
    tokens = torch.cat([torch.full((n,), 2 * i + 1) for i, n in enumerate(runs)])
    tokens = tokens[torch.randperm(len(tokens), generator=g)]
    go = torch.randint(-8, 9, (len(tokens), D), generator=g).float()
    for dtype in (F32, BF16):
        w = torch.zeros(V, D, device="cuda", requires_grad=True)
        out = lib.embedding(tokens.cuda(), w, dtype=dtype)
        (dw,) = torch.autograd.grad(out, w, go.cuda().to(dtype))
        want = torch.zeros(V, D).index_add_(0, tokens, go)
        assert torch.equal(dw.cpu(), want)


def test_embedding_views_and_shapes(lib):
    table = torch.randn(50, 40, device="cuda")
    t = torch.randint(0, 50, (3, 4), device="cuda")
    for w in (table[:, :32], table[:, 3:35], table[5:45, :17], table.t()[:40]):
        leaf = w.detach().requires_grad_()
        ids = t % w.shape[0]
        out = lib.embedding(ids.int(), leaf)
        assert torch.equal(out, w[ids])
        go = torch.randn(3, 4, w.shape[1], device="cuda")
        (dw,) = torch.autograd.grad(out, leaf, go)
        want = torch.zeros(w.shape).double().index_add_(0, ids.cpu().reshape(-1),
                                                       go.cpu().double().reshape(12, -1))
        _near(dw, want, U * 13 * (want.abs() + 12 * 5))
    out = lib.embedding(t[:0], leaf)
    assert out.shape == (0, 4, leaf.shape[1])
    (dw,) = torch.autograd.grad(out, leaf, torch.zeros_like(out))
    assert float(dw.abs().max()) == 0.0


# ---------------------------------------------------------------------------
# Differences, a run of them together, streams and graphs
# ---------------------------------------------------------------------------
def test_gradients_against_differences(lib):
    """Central differences of the definitions in 64 bits along a direction v:
    (f(x + e v) - f(x - e v)) / 2 e is off by e^2 f''' / 6 (below 1e-7 of the
    sum of |v| for e = 1e-4) and by 1e-16 f / e = 1e-11."""
    V, rows, K = 97, 5, 6
    x = _logits(rows, V, F32, 11)
    tokens = _tokens(rows, V, 3, ignored=False)
    ids, tl = _teacher(rows, V, K, 5)
    gen = torch.Generator().manual_seed(0)
    v = torch.randn(rows, V, generator=gen).double()
    leaf = x.detach().requires_grad_()
    out = lib.token_log_probs(leaf, tokens, temperature=0.7)
    loss = lib.distillation_loss(leaf, ids, tl, temperature=1.5, reduction="sum")

    def score(z):
        logp = torch.log_softmax(z / 0.7, -1)
        return (logp.gather(1, tokens.cpu()[:, None]).sum()
                - 0.3 * (torch.exp(logp) * logp).sum())

    def distill(z):
        logp = torch.log_softmax(z / 1.5, -1)
        t = torch.where(ids.cpu() != -100, tl.double().cpu() / 1.5, -math.inf)
        total = 0.0
        for r in range(rows):
            if (t[r] > -math.inf).any():
                q = torch.softmax(t[r], -1)
                keep = q > 0
                lp = logp[r, ids.cpu()[r].clamp(min=0)[keep]]
                total = total + 2.25 * (q[keep] * (torch.log(q[keep]) - lp)).sum()
        return total

    (a,) = torch.autograd.grad(out.log_prob.sum() + 0.3 * out.entropy.sum(), leaf)
    (b,) = torch.autograd.grad(loss, leaf)
    e = 1e-4
    z = x.double().cpu()
    for f, grad in ((score, a), (distill, b)):
        want = float(f(z + e * v) - f(z - e * v)) / (2 * e)
        got = float((grad.double().cpu() * v).sum())
        size = float((grad.double().cpu() * v).abs().sum())
        assert abs(got - want) <= 1e-7 * float(v.abs().sum()) + 200 * U * size


def test_scoring_then_distilling_through_the_table(lib):
    """A teacher's top logits feed a student whose table is looked up and read
    out: the losses and every gradient against 64 bits."""
    V, D, N, K = 203, 48, 37, 9
    gen = torch.Generator().manual_seed(9)
    table = torch.randn(V, D, generator=gen)
    tokens = torch.randint(0, V, (N,), generator=gen)
    teacher_logits = torch.randn(N, V, generator=gen).cuda()
    teacher = lib.token_log_probs(teacher_logits, tokens.cuda(), top_k=K)
    leaf = table.cuda().requires_grad_()
    hidden = lib.embedding(tokens.cuda(), leaf, scale=0.25)
    logits = hidden @ leaf.detach().t()
    loss = lib.distillation_loss(logits, teacher.top_tokens, teacher.top_log_probs,
                                 temperature=2.0)
    scores = lib.token_log_probs(logits, tokens.cuda())
    total = loss - 0.1 * scores.log_prob.mean() - 0.01 * scores.entropy.mean()
    (dw,) = torch.autograd.grad(total, leaf)

    ref = table.double().requires_grad_()
    z = ref[tokens] * 0.25 @ table.double().t()
    top = torch.topk(torch.log_softmax(teacher_logits.double().cpu(), -1), K)
    assert torch.equal(teacher.top_tokens.cpu(), top.indices)
    q = torch.softmax(top.values / 2.0, -1)
    logp2 = torch.log_softmax(z / 2.0, -1).gather(1, top.indices)
    logp = torch.log_softmax(z, -1)
    want = (4.0 * (q * (torch.log(q) - logp2)).sum(-1).mean()
            - 0.1 * logp.gather(1, tokens[:, None]).mean()
            + 0.01 * (torch.exp(logp) * logp).sum(-1).mean())
    (dref,) = torch.autograd.grad(want, ref)
    # the logits of the FP32 product are off by at most D u sum |h w| (about
    # 1e-5 here), which moves losses and gradients by as much, relatively
    assert abs(float(total) - float(want)) <= 1e-4 * abs(float(want))
    assert float((dw.double().cpu() - dref).abs().max()) <= 1e-4 * float(dref.abs().max())


def test_on_another_stream_and_in_a_graph(lib):
    V, rows, K, D = 3001, 40, 5, 24
    x = _logits(rows, V, BF16, 2)
    tokens = _tokens(rows, V, 2)
    ids, tl = _teacher(rows, V, K, 3)
    table = torch.randn(V, D, device="cuda")
    go = torch.randn(rows, D, device="cuda")
    words = tokens.clamp(min=0)

    def step():
        leaf = x.detach().requires_grad_()
        s = lib.token_log_probs(leaf, tokens, top_k=K)
        loss = lib.distillation_loss(leaf, ids, tl)
        (dx,) = torch.autograd.grad(s.log_prob.sum() + s.entropy.sum() + loss, leaf)
        w = table.detach().requires_grad_()
        e = lib.embedding(words, w)
        (dw,) = torch.autograd.grad(e, w, go)
        return s.log_prob.detach(), s.top_tokens, loss.detach(), dx, e.detach(), dw

    want = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step()
        graphs.append((graph, outs))
    x.copy_(_logits(rows, V, BF16, 77))
    want2 = [t.clone() for t in step()]
    for graph, outs in graphs + graphs[::-1]:
        graph.replay()
        for a, b in zip(outs, want2):
            assert torch.equal(a, b)
    assert not torch.equal(want[0], want2[0])


def test_reverse_captured_without_its_forward(lib):
    """A graph that holds a reverse alone, replayed with other upstream
    gradients: every replay starts from the saved logits, whatever the replay
    before it left behind."""
    x = _logits(400, 2000, BF16, 4)
    ids, tl = _teacher(400, 2000, 6, 4)
    # a reverse runs on its forward's stream, so that one is the capture's
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        leaf = x.detach().requires_grad_()
        loss = lib.distillation_loss(leaf, ids, tl)
    up = torch.ones((), device="cuda")
    want = {}
    for w in (1.0, 0.5, -3.0):
        a = x.detach().requires_grad_()
        (want[w],) = torch.autograd.grad(lib.distillation_loss(a, ids, tl), a,
                                         torch.tensor(w, device="cuda"))
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        (dx,) = torch.autograd.grad(loss, leaf, up, retain_graph=True)
    for w in (1.0, 0.5, 1.0, -3.0, 1.0):
        up.fill_(w)
        graph.replay()
        assert torch.equal(dx, want[w]), w
    # the eager graph still has its reverse
    torch.cuda.synchronize()
    (again,) = torch.autograd.grad(loss, leaf)
    torch.cuda.synchronize()
    assert torch.equal(again, want[1.0])


def test_changed_logits_are_refused_in_the_reverse(lib):
    x = _logits(3, 50, F32, 1)
    for loss in (lambda z: lib.token_log_probs(z, _tokens(3, 50, 1)).log_prob.sum(),
                 lambda z: lib.distillation_loss(z, *_teacher(3, 50, 2, 1))):
        base = x.detach().requires_grad_()
        z = base * 1.0
        out = loss(z)
        z.mul_(2.0)
        with pytest.raises(RuntimeError, match="modified"):
            torch.autograd.grad(out, base)


def test_calls_on_two_streams_at_once(lib):
    """Calls that overlap share nothing: their results are those of calls in a
    row."""
    xs = [_logits(300, 9000, BF16, s) for s in (1, 2)]
    tokens = _tokens(300, 9000, 1)
    ids, tl = _teacher(300, 9000, 5, 1)
    w = torch.randn(500, 64, device="cuda")
    words = torch.randint(0, 500, (20000,), device="cuda")
    go = torch.randn(20000, 64, device="cuda")

    def step(x):
        leaf = x.detach().requires_grad_()
        s = lib.token_log_probs(leaf, tokens, top_k=30)
        loss = lib.distillation_loss(leaf, ids, tl)
        (dx,) = torch.autograd.grad(s.entropy.sum() + loss, leaf)
        table = w.detach().requires_grad_()
        (dw,) = torch.autograd.grad(lib.embedding(words, table), table, go * x[0, 0].float())
        return [s.log_prob.detach(), s.top_tokens, loss.detach(), dx, dw]

    want = [step(x) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = [[], []]
    for _ in range(3):
        for i, (x, stream) in enumerate(zip(xs, streams)):
            with torch.cuda.stream(stream):
                got[i] = step(x)
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        for u, v in zip(a, b):
            assert torch.equal(u, v)


def test_second_derivatives_are_refused(lib):
    x = _logits(2, 30, F32, 1).requires_grad_()
    out = lib.token_log_probs(x, _tokens(2, 30, 1))
    (dx,) = torch.autograd.grad(out.log_prob.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()


def test_offsets_beyond_32_bits(lib):
    """Rows whose elements lie past 2^31: the last row as if it were alone (V a
    multiple of 8, so that both start on a 16-byte boundary and sum alike)."""
    V, rows = 65544, 33000
    x = torch.zeros(rows, V, dtype=BF16, device="cuda")
    x[-1] = _logits(1, V, BF16, 1)[0]
    t = torch.full((rows,), -100, device="cuda")
    t[-1] = 77
    ids, tl = _teacher(1, V, 7, 2)
    lists = torch.full((rows, 7), -100, device="cuda")
    lists[-1] = ids[0]
    tlog = torch.zeros(rows, 7, device="cuda")
    tlog[-1] = tl[0]
    a = lib.token_log_probs(x, t, top_k=4)
    b = lib.token_log_probs(x[-1:].clone(), t[-1:], top_k=4)
    for u, v in zip(a, b):
        assert torch.equal(u[-1:], v)
    leaf = x.requires_grad_()
    loss = lib.distillation_loss(leaf, lists, tlog)
    (dx,) = torch.autograd.grad(loss, leaf)
    one = x.detach()[-1:].clone().requires_grad_()
    loss1 = lib.distillation_loss(one, ids, tl)
    (d1,) = torch.autograd.grad(loss1, one)
    assert float(loss) == float(loss1)
    assert torch.equal(dx[-1:], d1) and float(dx[:-1].abs().max()) == 0.0
