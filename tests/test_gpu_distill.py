"""Distillation from a teacher's top logits through the LM head (GPU): value, gradient, statistics and
refusals against the formula in 64 bits, differences of the loss, and the training paths that use it.

Tolerances are bounds on the roundings. A logit is a sum of d exact (bf16) or once rounded (fp32)
products in fp32, off by at most (d + 1) 2^-23 times the sum of its terms' sizes (2^-23: an adder may
cut instead of round). A log-probability inherits at most two logit errors, over the temperature,
plus a few roundings of its own size."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24


def _mods():
    from orthrus_training_b200 import objective, ops

    return objective, ops


def _inputs(n, m, V, d, k, dtype, seed=0, scale=3.0, shift=0.45, pad=0.0, dup=False, index="sorted"):
    g = torch.Generator().manual_seed(seed)
    W = (torch.randn(V, d, generator=g) * scale / math.sqrt(d)).to(dtype)
    teacher = torch.randn(m, d, generator=g)
    idx = torch.randint(0, m, (n,), generator=g)
    if index == "sorted":
        idx = idx.sort().values
    elif index is None:
        idx = torch.arange(n)
    student = ((1 - shift) * teacher[idx] + shift * torch.randn(n, d, generator=g)).to(dtype)
    logits = teacher.to(dtype).double() @ W.double().T
    kk = min(k, V)
    values, ids = logits.topk(kk)
    lse = logits.logsumexp(1)
    if k > kk:
        values = torch.nn.functional.pad(values, (0, k - kk), value=-math.inf)
        ids = torch.nn.functional.pad(ids, (0, k - kk), value=-1)
    if dup:  # an id kept twice
        ids[:, -1] = ids[:, 0]
    if pad:
        gone = torch.rand(m, k, generator=g) < pad
        gone[0] = True  # a row that kept nothing
        values, ids = values.masked_fill(gone, -math.inf), ids.masked_fill(gone, -1)
    w = 0.2 + torch.rand(n, generator=g)
    dev = lambda t: t.to(DEV)  # noqa: E731
    return dict(student=dev(student), values=dev(values.float()), ids=dev(ids),
                index=None if index is None else dev(idx), weight=dev(W), row_weight=dev(w)), dev(lse.float())


def _formula(a, T, lse=None):
    """kl, total, grad, agree and the bounds of kl and grad in 64 bits."""
    h, W, w = a["student"].double(), a["weight"].double(), a["row_weight"].double()
    idx = a["index"] if a["index"] is not None else torch.arange(h.shape[0], device=DEV)
    live = (a["ids"] >= 0) & (a["values"] > -math.inf)
    v = torch.where(live, a["values"].double(), -math.inf) / T
    norm = v.logsumexp(1, keepdim=True) if lse is None else lse.double()[:, None]
    norm = torch.where(live.any(1, keepdim=True), norm, 0.0)
    lq, live, ids = (v - norm)[idx], live[idx], a["ids"].clamp_min(0)[idx]
    q = torch.where(live, lq.exp(), 0.0)
    s = h @ W.T / T
    lp = s.log_softmax(1)
    kl = torch.where(live, q * (lq - lp.gather(1, ids)), 0.0).sum(1)
    Q = q.sum(1, keepdim=True)
    qs = torch.zeros_like(lp).scatter_add_(1, ids, q)
    c = (w / T)[:, None]
    diff = c * (Q * lp.exp() - qs)
    # bounds
    d, half = h.shape[1], (2.0 ** -8 if h.dtype == torch.bfloat16 or a["student"].dtype == torch.bfloat16 else U)
    logit = (h.abs() @ W.abs().T) * (d + 1) * 2.0 ** -23 / T + s.abs() * 4 * U
    E = 2 * logit.max(1, keepdim=True).values + 16 * U + 4 * U * (lp.abs() * lp.exp()).sum(1, keepdim=True)
    kept = torch.where(live, q, 0.0)
    size = torch.where(live, lq.abs() + lp.gather(1, ids).abs() + v[idx].abs(), 0.0)
    klb = (kept * (E + 16 * U * (1 + size))).sum(1)
    dd = c * (Q * lp.exp() * (E + 32 * U * (1 + s.abs())) + qs * 32 * U * (1 + torch.where(live, size, 0.0).max(1, keepdim=True).values))
    dd = dd + diff.abs() * (half + lp.shape[1] * 2.0 ** -23)
    grad = diff @ W
    gb = dd @ W.abs() + half * grad.abs()
    top = torch.where(live, a["values"][idx].double(), -math.inf).argmax(1, keepdim=True)
    agree = live.any(1) & (s.argmax(1) == ids.gather(1, top)[:, 0])
    return kl, (kl * w).sum(), grad, agree, klb, gb


def _check(a, T=1.0, lse=None, chunk=4096):
    objective, _ = _mods()
    student = a["student"].detach().requires_grad_()
    total, kl, agree = objective.FusedLinearTopKKL.apply(student, a["values"], a["ids"], a["index"], a["weight"],
                                                         chunk, a["row_weight"], T, lse)
    total.backward()
    want_kl, want_total, want_grad, want_agree, klb, gb = _formula(a, T, lse)
    assert ((kl.double() - want_kl).abs() <= klb).all(), ((kl.double() - want_kl).abs() / klb).max()
    tb = (klb * a["row_weight"].double()).sum() + 64 * U * (want_kl.abs() * a["row_weight"].double()).sum()
    assert (total.double() - want_total).abs() <= tb
    grad = student.grad
    assert grad.dtype == a["student"].dtype
    assert ((grad.double() - want_grad).abs() <= gb).all(), ((grad.double() - want_grad).abs() / gb).max()
    # agreement may turn only where the two largest logits are nearer than their errors: not here
    assert torch.equal(agree, want_agree)
    return total, kl, grad


SIZES = [(1, 1, 1, 8, 1), (5, 3, 7, 24, 3), (130, 60, 1000, 64, 16), (300, 300, 1030, 256, 64), (70, 9, 5003, 100, 33),
         (129, 200, 2048, 1024, 128), (40, 40, 300, 72, 1024)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,m,V,d,k", SIZES)
def test_sizes(dtype, n, m, V, d, k):
    a, lse = _inputs(n, m, V, d, k, dtype, seed=n + V)
    _check(a)
    _check(a, 1.0, lse)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", ["padded", "twice", "unordered", "rows", "soft", "sharp", "far", "same", "chunks"])
def test_kinds(dtype, kind):
    n, m, V, d, k = 150, 80, 1500, 128, 20
    opts = {"padded": dict(pad=0.4), "twice": dict(dup=True), "unordered": dict(index="any"), "rows": dict(index=None),
            "far": dict(shift=1.0, scale=60.0), "same": dict(shift=0.0)}.get(kind, {})
    a, _ = _inputs(n, n if kind == "rows" else m, V, d, k, dtype, seed=3, **opts)
    _check(a, {"soft": 4.0, "sharp": 0.25}.get(kind, 1.0), chunk=128 if kind == "chunks" else 4096)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_largest_logit_far_above_the_kept_ones(dtype):
    """The student's mass sits hundreds of nats above every kept logit in some rows."""
    a, _ = _inputs(300, 300, 900, 64, 8, dtype, seed=4, index=None)
    a["weight"][5] = 0
    a["weight"][5, 0] = 50.0
    a["student"][:, 0] = 0
    a["student"][::7, 0] = 8.0   # logit 400 at index 5
    a["student"][3::7, 0] = -8.0
    a["ids"][a["ids"] == 5] = 6
    _check(a)


def test_rows_without_teacher_entries_are_nothing():
    for dtype in (torch.float32, torch.bfloat16):
        a, _ = _inputs(140, 140, 700, 64, 4, dtype, index=None)
        a["ids"][10:135] = -1
        total, kl, grad = _check(a)
        assert (kl[10:135] == 0).all() and (grad[10:135] == 0).all() and (grad[:10] != 0).any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_padding_values_are_never_read(dtype):
    """Whatever stands in a padded entry (NaN, infinities, an id of -1 with a large value) has no effect."""
    a, _ = _inputs(60, 60, 700, 64, 8, dtype, index=None)
    a["ids"][:, 3] = -1
    clean = _check(a)
    for junk in (math.nan, math.inf, -math.inf, 1e30):
        a["values"][:, 3] = junk
        for x, y in zip(_check(a), clean):
            assert torch.equal(x, y)


def test_per_offset_sums_and_no_gradient():
    _, ops = _mods()
    for dtype in (torch.float32, torch.bfloat16):
        a, _ = _inputs(200, 90, 1000, 64, 16, dtype, seed=8)
        offsets = torch.randint(0, 5, (200,), device=DEV)
        args = (a["student"], a["values"], a["ids"], a["index"], a["weight"], a["row_weight"], offsets, 5)
        total, kl, agree, grad, kbo, abo = ops.lmhead_topk_kl(*args)
        again = ops.lmhead_topk_kl(*args, need_grad=False)
        assert again[3] is None and torch.equal(again[0], total) and torch.equal(again[1], kl)
        assert torch.equal(abo, torch.bincount(offsets, weights=agree.double(), minlength=5).long())
        want = torch.bincount(offsets, weights=kl.double(), minlength=5)
        assert ((kbo.double() - want).abs() <= 200 * U * torch.bincount(offsets, weights=kl.double().abs())).all()


def test_gradient_is_the_slope_of_the_loss():
    """Central differences of the loss in 64 bits along random directions, at fp32 inputs."""
    a, _ = _inputs(6, 6, 200, 32, 10, torch.float32, seed=9, index=None)
    _, _, grad = _check(a, 1.5)
    g = torch.Generator().manual_seed(1)
    for _ in range(4):
        v = torch.randn(6, 32, generator=g).to(DEV).double()
        eps = 1e-4

        def loss(sign):
            b = dict(a, student=a["student"].double() + sign * eps * v)
            return _formula(b, 1.5)[1]

        slope = (loss(1) - loss(-1)) / (2 * eps)
        # third derivatives: logits move by at most eps |v| |W|, so the remainder is below 1e-6
        assert (slope - (grad.double() * v).sum()).abs() <= 1e-6 * 200 + 1e-4 * grad.abs().max()


def test_full_width_equals_the_whole_teacher():
    """With every logit kept, the loss is FusedLinearForwardKL's."""
    objective, _ = _mods()
    n, m, V, d = 180, 70, 1000, 64
    for dtype in (torch.float32, torch.bfloat16):
        a, _ = _inputs(n, m, V, d, 4, dtype, seed=12)
        g = torch.Generator().manual_seed(2)
        teacher = torch.randn(m, d, generator=g).to(DEV, dtype)
        values, ids, lse = objective.teacher_top_logits(teacher, a["weight"], V, chunk_rows=32)
        s1 = a["student"].detach().requires_grad_()
        s2 = a["student"].detach().requires_grad_()
        t1, kl1, ag1 = objective.FusedLinearTopKKL.apply(s1, values, ids, a["index"], a["weight"], 4096, a["row_weight"])
        t2, kl2, ag2 = objective.FusedLinearForwardKL.apply(s2, teacher, a["index"], a["weight"], 4096, False,
                                                            a["row_weight"])
        (2.0 * t1).backward()
        (2.0 * t2).backward()
        # both are within the bound of their logits' errors of the same number
        bound = _formula(dict(a, values=values, ids=ids), 1.0)
        assert ((kl1 - kl2).double().abs() <= 4 * bound[4]).all()
        assert torch.equal(ag1, ag2)
        assert ((s1.grad - s2.grad).double().abs() <= 2 * 2 * bound[5] + 2.0 ** -7 * s2.grad.double().abs()).all()


def test_teacher_top_logits():
    objective, _ = _mods()
    for dtype in (torch.float32, torch.bfloat16):
        for m, V, d in ((1, 50, 8), (77, 3001, 100)):
            g = torch.Generator().manual_seed(m)
            h, W = torch.randn(m, d, generator=g).to(DEV, dtype), torch.randn(V, d, generator=g).to(DEV, dtype)
            values, ids, lse = objective.teacher_top_logits(h, W, 20, 2.0, chunk_rows=32)
            s = h.double() @ W.double().T
            tol = ((h.double().abs() @ W.double().abs().T) * (d + 1) * 2.0 ** -23).max()
            assert ((values.double() - s.topk(20).values).abs() <= tol).all()
            assert ((values.double() - s.gather(1, ids)).abs() <= tol).all()
            assert ((lse.double() - (s / 2.0).logsumexp(1)).abs() <= tol + 40 * U * (1 + lse.double().abs())).all()


def test_capture_repeats_and_streams():
    """The same call gives the same bits, twice, on another stream and replayed on new inputs."""
    objective, _ = _mods()
    a, _ = _inputs(300, 300, 2000, 128, 16, torch.bfloat16, index=None)
    b, _ = _inputs(300, 300, 2000, 128, 16, torch.bfloat16, seed=5, index=None)

    def call(x):
        s = x["student"].detach().requires_grad_()
        total, kl, agree = objective.FusedLinearTopKKL.apply(s, x["values"], x["ids"], x["index"], x["weight"], 256,
                                                             x["row_weight"])
        (g,) = torch.autograd.grad(total, s)
        return total.detach(), kl, agree, g

    first, other = call(a), call(b)
    assert all(torch.equal(x, y) for x, y in zip(first, call(a)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(a)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = call(a)
        for inputs, want in ((a, first), (b, other)):
            for key in ("student", "values", "ids", "weight", "row_weight"):
                a[key].copy_(inputs[key].clone())
            graph.replay()
            assert all(torch.equal(x, y) for x, y in zip(out, want))
    torch.cuda.current_stream().wait_stream(side)


def test_out_of_range_entries_are_reported_and_left_out():
    from orthrus_training_b200 import _lib

    objective, ops = _mods()
    for dtype in (torch.float32, torch.bfloat16):
        a, _ = _inputs(20, 20, 500, 64, 4, dtype)
        a["index"] = torch.arange(20, device=DEV)
        a["ids"][2] = -1
        a["index"][3] = 2  # padding instead of an index out of range
        clean = ops.lmhead_topk_kl(**a)
        assert _lib.device_error(0) == 0
        a["index"][3] = 20
        a["ids"][2] = 500
        got = ops.lmhead_topk_kl(**a)
        assert _lib.device_error(0) == _lib.ERR_BOUNDS
        for x, y in zip(got[:4], clean[:4]):
            assert torch.equal(x, y)


def test_no_rows():
    _, ops = _mods()
    a, _ = _inputs(1, 1, 50, 16, 4, torch.bfloat16)
    total, kl, agree, grad, kbo, abo = ops.lmhead_topk_kl(
        a["student"][:0], a["values"], a["ids"], a["index"][:0], a["weight"], a["row_weight"][:0],
        a["index"][:0], 3)
    assert total == 0 and kl.shape == (0,) and grad.shape == (0, 16) and (kbo == 0).all() and (abo == 0).all()


def test_refusals():
    _, ops = _mods()
    a, lse = _inputs(10, 6, 50, 16, 4, torch.float32)
    for bad in (dict(temperature=0.0), dict(temperature=math.nan), dict(weight=a["weight"].bfloat16()),
                dict(student=a["student"].half(), weight=a["weight"].half()), dict(ids=a["ids"][:, :3]),
                dict(values=a["values"][:, :0], ids=a["ids"][:, :0]), dict(index=a["index"][:9]), dict(index=None),
                dict(row_weight=a["row_weight"][:3]), dict(teacher_lse=lse[:2]), dict(student=a["student"][:, :8]),
                dict(values=torch.zeros(6, 1025, device=DEV), ids=torch.zeros(6, 1025, dtype=torch.int64, device=DEV)),
                dict(ids=a["ids"].cpu())):
        with pytest.raises(ValueError):
            ops.lmhead_topk_kl(**dict(a, **bad))


def _tiny():
    """A two-layer bf16 model of 1024 tokens whose twins differ from the frozen view."""
    from __graft_entry__ import _tiny_config
    from orthrus_training_b200.modeling_orthrus import OrthrusLM, copy_diff_from_ar, freeze_to_diffusion

    torch.manual_seed(0)
    with torch.device(DEV):
        model = OrthrusLM(_tiny_config()).to(torch.bfloat16)
    copy_diff_from_ar(model)
    with torch.no_grad():
        for name, p in model.named_parameters():
            if "_diff." in name and "norm" not in name:
                p.add_(torch.randn_like(p) * 0.004)
    freeze_to_diffusion(model)
    return model


def test_orthrus_loss_from_top_logits():
    """With as many logits as the vocabulary has, the loss of the whole teacher; with fewer, the
    formula's on the same states, and gradients in every trainable weight."""
    from orthrus_training_b200.objective import (FusedLinearTopKKL, SupervisedLayout, model_states, orthrus_loss,
                                                 sample_anchors, teacher_top_logits)
    from orthrus_training_b200.synthetic import packed_rows

    model = _tiny()
    V, K = model.config.vocab_size, model.config.block_size
    ids, mask = packed_rows(2, 256, V - 1, seed=3, ids="uniform", doc="short")
    ids, mask = ids.to(DEV), mask.to(DEV)
    anchors, valid = sample_anchors(mask, K, 4, torch.Generator(device=DEV).manual_seed(1))
    whole, stats = orthrus_loss(model, ids, mask, anchors, valid, 4096, gamma=8.0)
    kept, kstats = orthrus_loss(model, ids, mask, anchors, valid, 4096, gamma=8.0, teacher_topk=V)
    # the two read the same logits from different products (fp32 sums of 256 terms): 2^-16 of the loss
    assert (whole - kept).abs() <= 2.0 ** -12 * (whole.abs() + 2.0 ** -8)
    assert int(stats["tokens"]) == int(kstats["tokens"]) and set(stats) == set(kstats)
    loss, _ = orthrus_loss(model, ids, mask, anchors, valid, 4096, teacher_topk=16)
    loss.backward()
    with torch.no_grad():
        layout = SupervisedLayout(mask, anchors, valid, K, 0.0)
        student, teacher = model_states(model, ids, anchors)
        top = teacher_top_logits(teacher.flatten(0, 1)[layout.positions], model.lm_head.weight, 16)
        rows = student.reshape(-1, student.shape[-1])[layout.student_rows]
        total, _, _ = FusedLinearTopKKL.apply(rows, top[0], top[1], layout.index, model.lm_head.weight, 4096)
        assert torch.equal(loss.detach(), total / layout.count.float().clamp_min(1e-6))
    for name, p in model.named_parameters():
        if "_diff." in name:
            assert p.grad is not None and torch.isfinite(p.grad).all(), name
    assert any((p.grad != 0).any() for n, p in model.named_parameters() if "_diff." in n)


def test_trainer_steps_on_top_logits():
    from orthrus_training_b200.synthetic import packed_rows
    from orthrus_training_b200.train_step import Trainer

    model = _tiny()
    trainer = Trainer(model, num_anchors=4, kl_chunk_size=256, total_steps=4, teacher_topk=8)
    before = [p.detach().clone() for p in trainer.params]
    for step in range(2):
        ids, mask = packed_rows(2, 256, model.config.vocab_size - 1, seed=step, ids="uniform", doc="short")
        out = trainer.step([(ids.to(DEV), mask.to(DEV))])
        assert torch.isfinite(out["loss"]) and not bool(out["skipped"])
    assert any(not torch.equal(p, q) for p, q in zip(trainer.params, before))


@pytest.mark.parametrize("n,V,d,chunk", [(600, 8001, 100, 4096), (300, 4000, 33, 4096), (97, 1009, 513, 4096),
                                         (600, 2500, 257, 256), (33, 20011, 7, 4096)])
def test_fp32_product_tiles(n, V, d, chunk):
    """Every tile size of the fp32 products, with and without parts of the long axis, ragged in all three."""
    a, lse = _inputs(n, 40, V, d, 9, torch.float32, seed=n)
    _check(a, 1.5, lse, chunk=chunk)
