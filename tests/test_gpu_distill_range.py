"""Distillation from a teacher's top logits (GPU) over the range its arguments may take: rows of padding
with any student, temperatures from 1e-30, operands of any distribution.

The operands are small integers, so that every logit is a sum of integers below 2^24 and exact in fp32
in whatever order and with whatever cutting it is formed. What is left are roundings that do not grow
with 1 / T: an exponent (x - c) / T carries three of its own size (8 U with the constants beside it),
ex2 errs by 2^-22, a sum of exponentials is formed over fewer than 64 additions in a row, expf and logf
are off by two units."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16]


def _rows(n, V, d, k, dtype, seed, near=True):
    """Integer operands; each teacher row keeps the k largest logits of an integer student of its own,
    near the student's (near) or not."""
    g = torch.Generator().manual_seed(seed)
    W = torch.randint(-3, 4, (V, d), generator=g).float()
    h = torch.randint(-2, 3, (n, d), generator=g).float()
    t = h + (torch.rand(n, d, generator=g) < 0.05).float() if near else torch.randint(-2, 3, (n, d), generator=g).float()
    values, ids = (t @ W.T).topk(k)
    return dict(student=h.to(DEV, dtype), values=values.to(DEV), ids=ids.to(DEV), index=None, weight=W.to(DEV, dtype),
                row_weight=(0.5 + torch.rand(n, generator=g)).to(DEV))


def _formula(a, T):
    """kl, gradient and agreement in 64 bits, and the bounds of the first two (see above)."""
    T = float(torch.tensor(T, dtype=torch.float32))
    h, W, w = a["student"].double(), a["weight"].double(), a["row_weight"].double()
    live = (a["ids"] >= 0) & (a["values"] > -math.inf)
    some = live.any(1, keepdim=True)
    v, ids = torch.where(live, a["values"].double(), -math.inf), a["ids"].clamp_min(0)
    v = torch.where(some, (v - v.max(1, keepdim=True).values) / T, -math.inf)
    lq = torch.where(live, v - torch.where(some, v.logsumexp(1, keepdim=True), 0.0), -math.inf)
    q = torch.where(live, lq.exp(), 0.0)
    s = h @ W.T
    y = (s - s.max(1, keepdim=True).values) / T
    lp = y.log_softmax(1)
    lpk = lp.gather(1, ids)
    taken = q > 0
    kl = torch.where(taken, q * (lq - lpk), 0.0).sum(1)
    zerr = 2.0 ** -22 + 64 * U
    step = 16 * U * (1 + lq.abs()) * (lq - lpk).abs() + 8 * U * (lq.abs() + lpk.abs() + 1) + zerr
    klb = torch.where(taken, q * step, 0.0).sum(1)
    qs = torch.zeros_like(lp).scatter_add_(1, ids, q)
    c = (w / T)[:, None]
    Qp = q.sum(1, keepdim=True) * lp.exp()
    diff = c * (Qp - qs)
    half = 2.0 ** -8 if a["student"].dtype == torch.bfloat16 else U
    lqs = torch.where(taken, 16 * U * (1 + lq.abs()), 0.0).max(1, keepdim=True).values
    # exponentials below 2^-126 are 0, and the largest of a row is 2^-60 or more: 2^-66 of p
    dd = c * 2.0 ** -66 + c * (Qp * (zerr + 8 * U * lp.abs().clamp_max(1e3) + lqs) + qs * (lqs + zerr)) + diff.abs() * half
    grad = diff @ W
    gb = (dd + diff.abs() * W.shape[0] * 2.0 ** -23) @ W.abs() + half * grad.abs()
    top = torch.where(live, a["values"].double(), -math.inf).argmax(1, keepdim=True)
    agree = some[:, 0] & (s.argmax(1) == ids.gather(1, top)[:, 0])
    return kl, grad, agree, klb, gb


def _check(a, T):
    from orthrus_training_b200.objective import FusedLinearTopKKL

    student = a["student"].detach().requires_grad_()
    total, kl, agree = FusedLinearTopKKL.apply(student, a["values"], a["ids"], a["index"], a["weight"], 4096,
                                               a["row_weight"], T)
    total.backward()
    grad = student.grad
    want_kl, want_grad, want_agree, klb, gb = _formula(a, T)
    assert torch.isfinite(kl).all() and torch.isfinite(grad).all()
    assert ((kl.double() - want_kl).abs() <= klb).all(), ((kl.double() - want_kl).abs() / klb).max()
    assert ((grad.double() - want_grad).abs() <= gb).all(), ((grad.double() - want_grad).abs() / gb).max()
    assert torch.equal(agree, want_agree)
    return total, kl, grad


@pytest.mark.parametrize("T", [1.0, 0.3, 0.02])
@pytest.mark.parametrize("dtype", DTYPES)
def test_padding_rows_of_low_logits_are_nothing(dtype, T):
    """Rows whose teacher kept nothing (no ids, ids past the vocabulary, an index out of range), all of
    whose logits lie near -240: kl 0 and gradient 0, beside rows that kept something."""
    from orthrus_training_b200 import _lib, ops

    n, m = 300, 200
    a = _rows(n, 900, 64, 6, dtype, seed=1)
    a["student"][:, 0] = 2
    a["weight"][:, 0] = -120
    a["values"], a["ids"] = a["values"][:m] - 240, a["ids"][:m].clone()
    a["index"] = torch.arange(n, device=DEV) % m
    a["ids"][10:20] = -1
    a["index"][30:40] = 12
    _lib.device_error(0)
    clean = ops.lmhead_topk_kl(**a, temperature=T)
    none = (a["ids"] < 0).all(1)[a["index"]]
    assert _lib.device_error(0) == 0 and 10 <= int(none.sum()) < n
    a["ids"][15:20] = 900
    a["index"][35:40] = torch.tensor([m, -1, 2 ** 40, m + 1, -2 ** 40], device=DEV)
    got = ops.lmhead_topk_kl(**a, temperature=T)
    assert _lib.device_error(0) == _lib.ERR_BOUNDS
    for total, kl, agree, grad, _, _ in (clean, got):
        assert (kl[none] == 0).all() and (grad[none] == 0).all() and not agree[none].any()
        assert torch.isfinite(total) and torch.isfinite(kl).all() and torch.isfinite(grad).all()
        assert (grad[~none] != 0).any()


@pytest.mark.parametrize("V", [900, 5003])  # the gradient's product in one and in several parts
@pytest.mark.parametrize("dtype", DTYPES)
def test_padding_rows_of_any_student_are_nothing(dtype, V):
    """What stands in the student's row has no effect where the teacher kept nothing: NaN and
    infinities there leave kl and gradient 0, and the other rows as they are."""
    from orthrus_training_b200 import ops

    a = _rows(300, V, 64, 6, dtype, seed=2)
    a["ids"][5:280:3] = -1
    none = (a["ids"] < 0).all(1)
    clean = ops.lmhead_topk_kl(**a)
    for junk in (math.nan, math.inf, -math.inf, torch.finfo(dtype).max):
        a["student"][none] = junk
        for x, y in zip(ops.lmhead_topk_kl(**a)[:4], clean[:4]):
            assert torch.equal(x, y)
    assert (clean[1][none] == 0).all() and (clean[3][none] == 0).all() and (clean[3][~none] != 0).any()


@pytest.mark.parametrize("dtype,T", [(t, T) for t in DTYPES for T in (1e-2, 1e-3, 1e-5)] +
                         [(torch.float32, T) for T in (1e-8, 1e-30)])
def test_teacher_ties_at_low_temperatures(dtype, T):
    """Equal kept logits share the teacher's mass however large the logits are beside the temperature: a
    student with the same ties has kl 0 and no gradient but of roundings."""
    a = _rows(200, 700, 64, 4, dtype, seed=3)
    W = a["weight"]
    W[1::2] = W[::2]  # every logit stands twice
    values, ids = (a["student"].double() @ W.double().T).sort(dim=1, descending=True, stable=True)
    a["values"], a["ids"] = values[:, :4].float(), ids[:, :4].contiguous()
    _check(a, T)


@pytest.mark.parametrize("T", [1e-6, 1e-7, 1e-8, 1e-12, 1e-30])
@pytest.mark.parametrize("near", [True, False])
@pytest.mark.parametrize("dtype", DTYPES)
def test_low_temperatures(dtype, near, T):
    """The lowest temperatures the loss takes, where a logit over T has no fraction left: softmax is one
    entry or a tie, kl the largest logit's distance over T, everything finite."""
    a = _rows(300, 700, 64, 5, dtype, seed=4, near=near)
    a["ids"][7] = -1
    _, _, grad = _check(a, T)
    assert (grad[7] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_low_temperatures_beside_large_logits(dtype):
    """Rows whose largest logit is far above, at, or far below every kept one, in one tile."""
    a = _rows(300, 700, 64, 5, dtype, seed=5)
    a["student"][::5] *= 64
    a["student"][1::5] *= -32
    for T in (1.0, 1e-3, 1e-9):
        _check(a, T)


@pytest.mark.parametrize("kind", ["one", "integers", "positive"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [256, 1024, 8192])
def test_operands_of_any_distribution(dtype, d, kind):
    """Logits of one product, of many small integers, and of one sign: the sums are exact, so kl is right
    to its own roundings at any width."""
    g = torch.Generator().manual_seed(d)
    n, V, k = 200, 600, 4
    W = torch.randint(-4, 5, (V, d), generator=g).float()
    h = torch.zeros(n, d)
    if kind == "integers":
        h = torch.randint(-1, 2, (n, d), generator=g).float() * (torch.rand(n, d, generator=g) < 64 / d)
    elif kind == "positive":
        W, h = W.abs(), (torch.rand(n, d, generator=g) < 32 / d).float()
    else:
        h.scatter_(1, torch.randint(0, d, (n, 1), generator=g), 16.0)
    ids = torch.randint(0, V, (n, k), generator=g)
    a = dict(student=h.to(DEV, dtype), values=torch.randint(0, 3, (n, k), generator=g).float().to(DEV), ids=ids.to(DEV),
             index=None, weight=W.to(DEV, dtype), row_weight=torch.ones(n, device=DEV))
    _check(a, 1.0)


@pytest.mark.parametrize("d", [64, 768, 1024, 4096])
@pytest.mark.parametrize("kind", ["normal", "positive", "same"])
def test_kl_of_sums_that_are_cut(kind, d):
    """The tensor cores' adder cuts where fp32 rounds: every 16 products up to a unit of the partial sum, half
    of one on average, which is d / 32 units of a logit whose partial sums grow evenly to it, halved for
    their growth. The loss measures and puts back what was cut: in sum over the rows it is off by no more
    than a quarter of the like."""
    from orthrus_training_b200 import ops

    g = torch.Generator().manual_seed(d)
    n, V, k = 512, 5003, 32
    W, t = torch.randn(V, d, generator=g) * 3 / math.sqrt(d), torch.randn(n, d, generator=g)
    h = t if kind == "same" else 0.6 * t + 0.4 * torch.randn(n, d, generator=g)
    if kind == "positive":
        W, t, h = W.abs(), t.abs(), h.abs()
    W, t, h = W.to(DEV).bfloat16(), t.to(DEV).bfloat16(), h.to(DEV).bfloat16()
    values, ids = (t.double() @ W.double().T).topk(k)
    values = values.float()
    kl = ops.lmhead_topk_kl(h, values, ids, None, W, need_grad=False)[1].double()
    lq, s = values.double().log_softmax(1), h.double() @ W.double().T
    q, p = lq.exp(), s.softmax(1)
    want = (q * (lq - s.log_softmax(1).gather(1, ids))).sum(1)
    slope = (p * s).sum(1) - (q * s.gather(1, ids)).sum(1)  # of kl by a common part of the logits
    # roundings of kl itself, of either sign: log q, the exponents, log z, the sums (see the top)
    noise = (8 * U * (q * lq.abs()).sum(1) + 8 * U * (q * s.log_softmax(1).gather(1, ids).abs()).sum(1) + 2.0 ** -22).sum()
    noise = noise / math.sqrt(n)
    assert (kl - want).sum().abs() <= d / 64 * 2 * U / 4 * slope.abs().sum() + noise
