"""Cases of the vocabulary-row operators, for timing and comparing them: the top logits of rows, sampling
from rows with given uniforms, and distillation from a teacher's top logits through the LM head.

`run(state)` computes one pass, in plain torch operations, or with the package's operators where `own`
is true. `exact(case, seed)` gives the same outputs in 64 bits from the definitions.

Definitions (x a row of V logits; entries that are -inf or NaN are not candidates; T a temperature):

  topk     the k largest candidates in descending order, the lower index first among equals, padded
           with (-inf, -1), and lse = log sum exp(x / T) over the candidates (-inf if there are none).
  sample   w_i = exp((x_i - max x) / T). Kept are the candidates with x_i >= the top_k-th largest value
           (0: all); of these the prefix in (descending value, ascending index) order whose mass
           before the entry is at most top_p of their total (1: all); and of these the ones with
           w_i >= min_p. The token is the first kept index whose running sum of kept weights, in index
           order, exceeds u times their total. T below 1e-5: the first largest entry. No candidates: -1.
  distill  q_j = softmax over a teacher row's kept logits v_j / T (or exp(v_j / T - lse) with the
           teacher's own normaliser), p = softmax(W h / T); per student row r with teacher row
           index[r], kl_r = sum_j q_j (log q_j - log p_{id_j}); total = sum_r w_r kl_r, and its
           gradient with respect to h. Entries with id -1 or value -inf are padding.
"""

import math

import torch

own = False

VOCAB = 151936  # the benchmark model's vocabulary; its hidden size is 1024, its blocks have 32 rows


def listed():
    return [
        # the last rows of two prompts at the test model's vocabulary: the smallest call
        dict(name="topk_2x1024_k8", op="topk", rows=2, vocab=1024, k=8, dtype="float32", temperature=1.0,
             pitch=0, masked=0.0),
        # one 32-row block's teacher logits kept for distillation
        dict(name="topk_32x151936_k64", op="topk", rows=32, vocab=VOCAB, k=64, dtype="float32", temperature=1.0,
             pitch=0, masked=0.0),
        # a chunk of teacher logits as the LM head writes them, at the training step's width
        dict(name="topk_1024x151936_k64", op="topk", rows=1024, vocab=VOCAB, k=64, dtype="float32", temperature=1.0,
             pitch=0, masked=0.0),
        # bf16 logits (many equal values) of an odd vocabulary inside a wider buffer, a third masked out
        dict(name="topk_333x50257_k300_bf16", op="topk", rows=333, vocab=50257, k=300, dtype="bfloat16",
             temperature=2.0, pitch=50304, masked=0.33),
        # one token of one sequence with the generation defaults: a call where latency counts
        dict(name="sample_1x151936", op="sample", rows=1, vocab=VOCAB, dtype="float32", temperature=0.7, top_k=20,
             top_p=0.8, min_p=0.0, per_row=False, masked=0.0),
        # a serving batch that filters by nucleus alone: the border can lie anywhere in the vocabulary
        dict(name="sample_256x151936_top_p", op="sample", rows=256, vocab=VOCAB, dtype="float32", temperature=1.0,
             top_k=0, top_p=0.95, min_p=0.0, per_row=False, masked=0.0),
        # every position of 32 blocks of 32 rows, bf16, each row with its own knobs (greedy rows among them)
        dict(name="sample_1024x151936_rows", op="sample", rows=1024, vocab=VOCAB, dtype="bfloat16", temperature=1.0,
             top_k=50, top_p=0.9, min_p=0.05, per_row=True, masked=0.0),
        # an odd vocabulary under a grammar mask, filtered by min-p alone
        dict(name="sample_77x32003_min_p", op="sample", rows=77, vocab=32003, dtype="float32", temperature=1.3,
             top_k=0, top_p=1.0, min_p=0.05, per_row=False, masked=0.9),
        # the exact-parity type at the test model's size
        dict(name="distill_90x1024x256_f32", op="distill", rows=90, teacher_rows=60, vocab=1024, hidden=256, k=16,
             dtype="float32", temperature=1.0, full_mass=False, padded=0.0),
        # a small micro-batch of the benchmark model
        dict(name="distill_512x151936x1024", op="distill", rows=512, teacher_rows=300, vocab=VOCAB, hidden=1024, k=32,
             dtype="bfloat16", temperature=1.0, full_mass=False, padded=0.0),
        # an odd vocabulary, softened, with the teacher's own normaliser and rows that kept fewer logits
        dict(name="distill_1999x50257x768", op="distill", rows=1999, teacher_rows=1500, vocab=50257, hidden=768, k=16,
             dtype="bfloat16", temperature=2.0, full_mass=True, padded=0.25),
        # the benchmark's training step: 8 rows of 32 blocks, 31 supervised positions each
        dict(name="distill_7936x151936x1024", op="distill", rows=7936, teacher_rows=6000, vocab=VOCAB, hidden=1024,
             k=64, dtype="bfloat16", temperature=1.0, full_mass=False, padded=0.0),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["topk", "sample", "distill"])
    dtype = rng.choice(["float32", "bfloat16"])
    vocab = VOCAB if rng.random() < 0.3 else _log_int(rng, 1000, VOCAB)
    if op == "topk":
        return dict(op=op, rows=_log_int(rng, 1, 1024), vocab=vocab, k=_log_int(rng, 1, 512), dtype=dtype,
                    temperature=rng.choice([1.0, 2.0, 0.5]), pitch=vocab + 13 if rng.random() < 0.3 else 0,
                    masked=rng.choice([0.0, 0.0, 0.5]))
    if op == "sample":
        mode = rng.choice(["plain", "top_k", "top_p", "min_p", "all"])
        return dict(op=op, rows=_log_int(rng, 1, 1024), vocab=vocab, dtype=dtype,
                    temperature=round(rng.uniform(0.3, 1.5), 3),
                    top_k=_log_int(rng, 1, 500) if mode in ("top_k", "all") else 0,
                    top_p=round(rng.uniform(0.3, 0.99), 3) if mode in ("top_p", "all") else 1.0,
                    min_p=round(rng.uniform(0.01, 0.3), 3) if mode in ("min_p", "all") else 0.0,
                    per_row=mode == "all", masked=rng.choice([0.0, 0.0, 0.8]))
    if dtype == "float32":  # parity runs are small
        rows, vocab, hidden = _log_int(rng, 64, 600), _log_int(rng, 1000, 8000), 8 * _log_int(rng, 8, 64)
    else:
        hidden = 8 * _log_int(rng, 16, 128)
        rows = _log_int(rng, 64, 6000)
    return dict(op=op, rows=rows, teacher_rows=max(1, int(rows * rng.uniform(0.3, 1.0))), vocab=vocab, hidden=hidden,
                k=_log_int(rng, 1, 128), dtype=dtype, temperature=rng.choice([1.0, 1.0, 2.0]),
                full_mass=rng.random() < 0.3, padded=rng.choice([0.0, 0.0, 0.3]))


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _logits(case, g):
    """Rows as a language model gives them: a wide bulk of small logits and a few dozen large ones."""
    R, V = case["rows"], case["vocab"]
    pitch = max(case.get("pitch", 0), V)
    x = torch.randn(R, pitch, device="cuda", generator=g) * 2.0
    n = min(48, V // 4)
    heads = torch.randint(0, V, (R, n), device="cuda", generator=g)
    lift = 6.0 + 6.0 * torch.rand(R, n, device="cuda", generator=g)
    x.scatter_add_(1, heads, lift)
    if case["masked"] > 0:
        x.masked_fill_(torch.rand(R, pitch, device="cuda", generator=g) < case["masked"], -math.inf)
    return x.to(getattr(torch, case["dtype"]))[:, :V]


def prepare(case, seed):
    g = _generator(seed)
    dev = "cuda"
    if case["op"] == "topk":
        return dict(case=case, logits=_logits(case, g))
    if case["op"] == "sample":
        R = case["rows"]
        s = dict(case=case, logits=_logits(case, g), u=torch.rand(R, device=dev, generator=g))
        for key in ("temperature", "top_k", "top_p", "min_p"):
            s[key] = case[key]
        if case["per_row"]:  # each request its own knobs; one in eight is greedy, some filters off
            t = case["temperature"] * (0.5 + torch.rand(R, device=dev, generator=g))
            s["temperature"] = torch.where(torch.rand(R, device=dev, generator=g) < 0.125, torch.zeros_like(t), t)
            k = (case["top_k"] * (0.2 + 1.8 * torch.rand(R, device=dev, generator=g))).to(torch.int32) + 1
            s["top_k"] = torch.where(torch.rand(R, device=dev, generator=g) < 0.25, torch.zeros_like(k), k)
            p = case["top_p"] + (1 - case["top_p"]) * torch.rand(R, device=dev, generator=g)
            s["top_p"] = torch.where(torch.rand(R, device=dev, generator=g) < 0.25, torch.ones_like(p), p)
            m = case["min_p"] * torch.rand(R, device=dev, generator=g)
            s["min_p"] = torch.where(torch.rand(R, device=dev, generator=g) < 0.5, torch.zeros_like(m), m)
        return s
    n, m, V, d, k = case["rows"], case["teacher_rows"], case["vocab"], case["hidden"], case["k"]
    dtype, T = getattr(torch, case["dtype"]), case["temperature"]
    weight = (torch.randn(V, d, device=dev, generator=g) * (3.0 / math.sqrt(d))).to(dtype)
    teacher = torch.randn(m, d, device=dev, generator=g)
    index = torch.randint(0, m, (n,), device=dev, generator=g).sort().values
    student = (0.9 * teacher[index] + 0.45 * torch.randn(n, d, device=dev, generator=g)).to(dtype)
    values = torch.empty(m, k, device=dev)
    ids = torch.empty(m, k, dtype=torch.int64, device=dev)
    lse = torch.empty(m, device=dev)
    for r in range(0, m, 1024):  # the teacher's logits, a chunk of rows at a time
        logits = (teacher[r : r + 1024].to(dtype) @ weight.T).float()
        values[r : r + 1024], ids[r : r + 1024] = logits.topk(k)
        lse[r : r + 1024] = torch.logsumexp(logits / T, -1)
    if case["padded"] > 0:  # rows of which fewer logits were kept (at least one)
        short = torch.rand(m, device=dev, generator=g) < case["padded"]
        keep = 1 + (torch.rand(m, device=dev, generator=g) * (k - 1)).long()
        pad = short[:, None] & (torch.arange(k, device=dev)[None] >= keep[:, None])
        values, ids = values.masked_fill(pad, -math.inf), ids.masked_fill(pad, -1)
    return dict(case=case, student=student, values=values, ids=ids, index=index, weight=weight,
                row_weight=0.2 + 0.8 * torch.rand(n, device=dev, generator=g),
                lse=lse if case["full_mass"] else None)


def _plain_topk(x, k, T):
    x = x.float()
    x = torch.where(torch.isnan(x), -math.inf, x)
    values, ids = torch.sort(x, dim=1, descending=True, stable=True)
    if x.shape[1] < k:
        more = k - x.shape[1]
        values = torch.cat([values, values.new_full((x.shape[0], more), -math.inf)], 1)
        ids = torch.cat([ids, ids.new_full((x.shape[0], more), -1)], 1)
    top = values[:, :1]
    total = torch.exp(((x - top) / T).double()).sum(1)
    lse = torch.where(top[:, 0] == -math.inf, -math.inf, (top[:, 0].double() / T + torch.log(total))).float()
    values, ids = values[:, :k].contiguous(), ids[:, :k]
    return values, torch.where(values == -math.inf, -1, ids), lse


def _column(v, like):
    """A knob as a [R, 1] column in 64 bits; it is given in 32 bits, as the operator takes it."""
    if not torch.is_tensor(v):
        v = torch.full((like.shape[0],), float(v), device=like.device)
    return v.float().double()[:, None]


def _plain_sample(x, u, temperature, top_k, top_p, min_p):
    V = x.shape[1]
    x = x.double()
    x = torch.where(torch.isnan(x), -math.inf, x)
    T, k, p, m = (_column(v, x) for v in (temperature, top_k, top_p, min_p))
    ordered, order = torch.sort(x, dim=1, descending=True, stable=True)
    none = ordered[:, :1] == -math.inf
    w = torch.exp((ordered - ordered[:, :1]) / T.clamp_min(1e-5))
    w = torch.where(ordered == -math.inf, 0.0, w)
    kth = ordered.gather(1, torch.where((k < 1) | (k > V), V, k).long() - 1)
    w = torch.where(ordered >= kth, w, 0.0)
    before = torch.cumsum(w, 1) - w
    kept = (w > 0) & ((p >= 1) | (before <= p * w.sum(1, keepdim=True))) & (w >= m)
    w = torch.zeros_like(w).scatter_(1, order, torch.where(kept, w, 0.0))
    running = torch.cumsum(w, 1)
    token = (running <= u.double()[:, None] * running[:, -1:]).sum(1, keepdim=True).clamp_max(V - 1)
    token = torch.where(T < 1e-5, order[:, :1], token)
    return torch.where(none, -1, token)[:, 0]


def _plain_distill(student, values, ids, index, weight, row_weight, T, lse):
    h, W = student.float(), weight.float()
    pad = (ids < 0) | (values == -math.inf)
    logq = torch.where(pad, -math.inf, values / T)
    logq = logq - (torch.logsumexp(logq, 1, keepdim=True) if lse is None else lse[:, None])
    logq, at = logq[index], ids.clamp_min(0)[index]
    q = torch.exp(logq)
    s = (h @ W.T) / T
    top = s.max(1, keepdim=True).values
    e = torch.exp(s - top)
    z = e.sum(1, keepdim=True)
    logp = (s.gather(1, at) - top) - torch.log(z)
    kl = torch.where(q > 0, q * (logq - logp), 0.0).sum(1)
    diff = (e / z * q.sum(1, keepdim=True)).scatter_add_(1, at, -q)
    grad = (diff * (row_weight / T)[:, None]) @ W
    return dict(total=(kl * row_weight).sum(), kl_rows=kl, grad=grad.to(student.dtype))


def run(state):
    case = state["case"]
    if own:
        from orthrus_training_b200 import objective, ops

        if case["op"] == "topk":
            return ops.topk_rows(state["logits"], case["k"], case["temperature"])
        if case["op"] == "sample":
            return ops.sample_logits(state["logits"], state["u"], state["temperature"], state["top_k"],
                                     state["top_p"], state["min_p"])
        # the third output, the rows' top-1 agreement, is a comparison of neighbouring logits
        # that the order of a sum can turn, so it is not compared here
        student = state["student"].detach().requires_grad_()
        total, kl_rows, _ = objective.FusedLinearTopKKL.apply(
            student, state["values"], state["ids"], state["index"], state["weight"], 8192, state["row_weight"],
            case["temperature"], state["lse"])
        total.backward()
        return dict(total=total.detach(), kl_rows=kl_rows, grad=student.grad)
    if case["op"] == "topk":
        return _plain_topk(state["logits"], case["k"], case["temperature"])
    if case["op"] == "sample":
        return _plain_sample(state["logits"], state["u"], state["temperature"], state["top_k"], state["top_p"],
                             state["min_p"])
    return _plain_distill(state["student"], state["values"], state["ids"], state["index"], state["weight"],
                          state["row_weight"], case["temperature"], state["lse"])


def work(case):
    size = 2 if case["dtype"] == "bfloat16" else 4
    R, V = case["rows"], case["vocab"]
    if case["op"] == "topk":  # every logit read once; an exponential and a sum each
        return {"bytes": R * V * size + R * (case["k"] * 12 + 4), "flops": 3.0 * R * V}
    if case["op"] == "sample":
        return {"bytes": R * V * size + R * (4 + 8), "flops": 3.0 * R * V}
    d, k, m = case["hidden"], case["k"], case["teacher_rows"]
    # the logits and their gradient's product with the LM head: two products of rows x vocab x hidden
    return {"bytes": V * d * size + 2 * R * d * size + m * k * 12 + R * 16, "flops": 4.0 * R * V * d}


def _exact_sample(state):
    """Row by row from the definition: the kept set as a truth value per token, then the walk in index order."""
    R, V = state["logits"].shape
    knob = [_column(state[key], state["logits"])[:, 0].tolist() for key in ("temperature", "top_k", "top_p", "min_p")]
    tokens = []
    for r in range(R):
        T, k, p, m = (v[r] for v in knob)
        x = state["logits"][r].double().nan_to_num(nan=-math.inf, posinf=math.inf, neginf=-math.inf)
        top, first = x.max(0)
        if T < 1e-5 or top == -math.inf:
            tokens.append(torch.where(top == -math.inf, -1, (x == top).int().argmax()))
            continue
        w = ((x - top) / T).exp()
        if 1 <= k < V:
            w = w * (x >= torch.topk(x, int(k)).values[-1])
        kept = w >= m
        if p < 1:
            order = torch.argsort(-x, stable=True)
            mass = torch.cat([w.new_zeros(1), w[order].cumsum(0)])
            outside = order[mass[:-1] > p * mass[-1]]
            kept[outside] = False
        w = w * kept
        c = w.cumsum(0)
        tokens.append(torch.searchsorted(c, state["u"][r].double() * c[-1], right=True).clamp_max(V - 1))
    return torch.stack([t.reshape(()).long() for t in tokens])


def exact(case, seed):
    state = prepare(case, seed)
    T = case.get("temperature")
    if case["op"] == "sample":
        return _exact_sample(state)
    if case["op"] == "topk":
        x = state["logits"].double()
        values = x.topk(min(case["k"], x.shape[1]), dim=1).values
        values = torch.nn.functional.pad(values, (0, case["k"] - values.shape[1]), value=-math.inf)
        return values, None, torch.logsumexp(x / T, 1)
    h = state["student"].double().requires_grad_()
    W, ids, index = state["weight"].double(), state["ids"], state["index"]
    logp = torch.log_softmax(h @ W.T / T, 1)
    kl = []
    v = state["values"].double() / T
    live = ids[index] >= 0
    norm = v.logsumexp(1) if state["lse"] is None else state["lse"].double()
    lq = (v - norm[:, None])[index]
    for j in range(case["k"]):  # one kept logit of every row at a time
        at = ids[index, j].clamp_min(0)[:, None]
        lqj = torch.where(live[:, j], lq[:, j], 0.0)
        kl.append(torch.where(live[:, j], lqj.exp() * (lqj - logp.gather(1, at)[:, 0]), 0.0))
    kl = torch.stack(kl).sum(0)
    total = (kl * state["row_weight"].double()).sum()
    (grad,) = torch.autograd.grad(total, h)
    return dict(total=total.detach(), kl_rows=kl.detach(), grad=grad)
