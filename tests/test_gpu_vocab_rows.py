"""The row operators over vocabulary logits (GPU): top logits and sampling against plain 64-bit forms.

Values, ids and tokens are compared exactly. A value is one of the inputs. A token rests on sums that
the operator forms exactly from weights of 42 or more fractional bits: it can differ from the 64-bit
form only for a uniform within about 1e-11 of a border, out of the 2^24 a uniform can take."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.float32, torch.bfloat16]


def _ops():
    from orthrus_training_b200 import ops

    return ops


def _rows(kind, R, V, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(R, V, generator=g) * 2.5
    if kind == "equal":
        x = torch.full((R, V), 1.25)
    elif kind == "two":  # two values, so every border falls among equals
        x = torch.where(torch.rand(R, V, generator=g) < 0.3, 2.0, 1.0)
    elif kind == "ascending":
        x = x.sort(1).values
    elif kind == "descending":
        x = x.sort(1, descending=True).values
    elif kind == "masked":
        x = x.masked_fill(torch.rand(R, V, generator=g) < 0.9, -math.inf)
    elif kind == "lowest":  # a mask of the type's lowest value leaves numbers, not holes
        x = torch.where(torch.rand(R, V, generator=g) < 0.9, torch.finfo(dtype).min, x)
    elif kind == "nan":
        x = x.masked_fill(torch.rand(R, V, generator=g) < 0.5, math.nan)
    elif kind == "zeros":
        x = torch.where(torch.rand(R, V, generator=g) < 0.5, -0.0, 0.0)
    elif kind == "peaked":
        x[:, V // 2] = 60.0
    return x.to(dtype).to(DEV)


KINDS = ["normal", "equal", "two", "ascending", "descending", "masked", "lowest", "nan", "zeros", "peaked"]


def _topk64(x, k, T):
    x = x.double()
    x = torch.where(torch.isnan(x), -math.inf, x)
    v, i = torch.sort(x, dim=1, descending=True, stable=True)
    pad = max(0, k - x.shape[1])
    v = torch.nn.functional.pad(v, (0, pad), value=-math.inf)[:, :k]
    i = torch.nn.functional.pad(i, (0, pad), value=-1)[:, :k]
    return v, torch.where(v == -math.inf, -1, i), torch.logsumexp(x / T, 1)


def _check_topk(x, k, T):
    values, ids, lse = _ops().topk_rows(x, k, T)
    v, i, want = _topk64(x, k, T)
    assert values.dtype == torch.float32 and ids.dtype == torch.int64 and lse.dtype == torch.float32
    assert torch.equal(values.double(), v)
    assert torch.equal(ids, i)
    fine = torch.isfinite(want)
    assert torch.equal(lse[~fine].double(), want[~fine])
    # the exponent (x - max) / T is rounded twice and ex2 errs by 2^-22; each weighs in with its
    # probability (terms at distance d count e^-d, and d e^-d < 0.4); the sum of positive fp32
    # numbers over a thread's entries adds at most n 2^-24 (n <= 1000); one rounding at the end
    V = x.shape[1]
    tol = 2 ** -22 * 3 + (V / 512 + 10) * 2 ** -24 + want.abs() * 2 ** -23
    assert ((lse.double() - want).abs() <= tol)[fine].all(), (lse.double() - want).abs().max()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [1, 2, 7, 33, 1000, 1024, 5003, 32003, 151936, 2 ** 20])
def test_topk_sizes(dtype, V):
    for k in sorted({1, min(V, 5), 64, 1024}):
        _check_topk(_rows("normal", 3, V, dtype, seed=V + k), k, 1.0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", KINDS)
def test_topk_kinds(dtype, kind):
    for V in (600, 20011):
        for k in (1, 17, 500):
            _check_topk(_rows(kind, 4, V, dtype, seed=k), k, 0.7)


@pytest.mark.parametrize("dtype", DTYPES)
def test_topk_few_candidates_and_infinities(dtype):
    x = torch.full((5, 3001), -math.inf, device=DEV, dtype=dtype)
    x[1, 2999] = -5.0
    x[2, [0, 7, 3000]] = torch.tensor([1.0, math.nan, 1.0], device=DEV, dtype=dtype)
    x[3, 100] = math.inf
    x[3, 50] = 3.0
    x[4] = math.nan
    _check_topk(x, 4, 1.0)
    assert _ops().topk_rows(x, 4)[1].tolist() == [[-1] * 4, [2999, -1, -1, -1], [0, 3000, -1, -1],
                                                  [100, 50, -1, -1], [-1] * 4]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("start", [0, 1, 2, 3, 5, 7])
def test_topk_views(dtype, start):
    """Rows at any alignment and pitch, repeated rows (pitch 0), and no row at all."""
    base = _rows("normal", 6, 4111, dtype)
    _check_topk(base[::2, start : start + 4000], 40, 1.0)
    _check_topk(base[1:2, start:].expand(3, -1), 3, 1.0)
    values, ids, lse = _ops().topk_rows(base[:0], 7)
    assert values.shape == (0, 7) and ids.shape == (0, 7) and lse.shape == (0,)


def _sample64(x, u, temperature, top_k, top_p, min_p):
    """The definition, row by row."""
    out = []
    R, V = x.shape

    def knob(v, r):
        return float(v[r].float()) if torch.is_tensor(v) else float(torch.tensor(float(v), dtype=torch.float32))

    for r in range(R):
        T, k, p, m = (knob(v, r) for v in (temperature, top_k, top_p, min_p))
        row = x[r].double()
        row = torch.where(torch.isnan(row), -math.inf, row)
        order = torch.argsort(row, descending=True, stable=True)
        top = row[order[0]]
        if top == -math.inf:
            out.append(-1)
            continue
        if T < 1e-5:
            out.append(int(order[0]))
            continue
        w = torch.where(row == top, 1.0, torch.exp((row - top) / T))
        w = torch.where(row == -math.inf, 0.0, w)
        if 1 <= k < V:
            w = torch.where(row >= row[order[int(k) - 1]], w, 0.0)
        if p < 1:
            c = torch.cumsum(w[order], 0)
            before = c - w[order]
            drop = order[before > p * c[-1]]
            w[drop] = 0.0
        w = torch.where(w >= m, w, 0.0)
        c = torch.cumsum(w, 0)
        uu = min(max(float(u[r]), 0.0), 1 - 2.0 ** -53) if not math.isnan(float(u[r])) else 0.0
        out.append(int((c <= uu * c[-1]).sum()))
    return torch.tensor(out, device=x.device)


FILTERS = [dict(), dict(top_k=1), dict(top_k=40), dict(top_p=0.9), dict(top_p=0.2), dict(min_p=0.1),
           dict(top_k=300, top_p=0.8, min_p=0.02), dict(top_k=5000, top_p=0.999)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [1, 2, 7, 33, 1000, 5003, 32003, 151936, 2 ** 20])
def test_sample_sizes(dtype, V):
    g = torch.Generator().manual_seed(V)
    x = _rows("normal", 6, V, dtype, seed=V)
    for f in FILTERS:
        u = torch.rand(6, generator=g).to(DEV)
        args = dict(dict(temperature=0.9, top_k=0, top_p=1.0, min_p=0.0), **f)
        assert torch.equal(_ops().sample_logits(x, u, **args), _sample64(x, u, **args)), (V, f)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", KINDS)
def test_sample_kinds(dtype, kind):
    g = torch.Generator().manual_seed(5)
    for V in (600, 20011):
        x = _rows(kind, 8, V, dtype, seed=V)
        for f in FILTERS:
            for T in (0.3, 1.7):
                u = torch.rand(8, generator=g).to(DEV)
                args = dict(dict(temperature=T, top_k=0, top_p=1.0, min_p=0.0), **f)
                assert torch.equal(_ops().sample_logits(x, u, **args), _sample64(x, u, **args)), (V, f, T)


@pytest.mark.parametrize("dtype", DTYPES)
def test_sample_rows_of_their_own_knobs(dtype):
    """Per-row knobs, greedy rows, empty rows, +inf entries and uniforms at and past their ends."""
    R, V = 64, 9001
    g = torch.Generator().manual_seed(1)
    x = _rows("normal", R, V, dtype)
    x[3] = -math.inf
    x[4] = math.nan
    x[5, 77] = math.inf
    x[6, [70, 8000]] = math.inf
    u = torch.rand(R, generator=g)
    u[6] = 0.5
    u[7:12] = torch.tensor([0.0, 1 - 2.0 ** -24, 1.0, -0.5, math.nan])
    u = u.to(DEV)
    t = (0.2 + torch.rand(R, generator=g)).to(DEV)
    t[20:24] = 0.0
    k = torch.randint(0, 60, (R,), generator=g).to(DEV)
    k[30], k[31] = V, 10 ** 6
    p = (0.1 + torch.rand(R, generator=g)).to(DEV)  # some at or above 1: off
    m = (torch.rand(R, generator=g) * 0.2).to(DEV)
    got = _ops().sample_logits(x, u, t, k, p, m)
    assert torch.equal(got, _sample64(x, u, t, k, p, m))
    assert got[3] == -1 and got[4] == -1 and got[5] == 77
    assert torch.equal(got[20:24], x[20:24].float().argmax(1))


def test_sample_draws_follow_the_distribution():
    """A grid of uniforms picks each token as often as its share of the filtered distribution says:
    the count of n evenly spaced points in an interval of length q is q n, give or take one."""
    V, n = 53, 100_000
    x = _rows("normal", 1, V, torch.float32)
    u = ((torch.arange(n, dtype=torch.float64) + 0.5) / n).float().to(DEV)
    got = _ops().sample_logits(x.expand(n, V), u, 0.8, 20, 0.9, 0.01)
    w = torch.softmax(x[0].double() / 0.8, 0)
    w = torch.where(x[0] >= x[0].topk(20).values[-1], w, 0.0)
    s, order = w.sort(descending=True)
    w[order[(s.cumsum(0) - s) > 0.9 * s.sum()]] = 0.0
    w = torch.where(w >= 0.01 * w.max(), w, 0.0)
    counts = torch.bincount(got, minlength=V).double()
    # the uniforms are rounded to fp32: up to 2^-25 n = 0.003 of a point more at each end
    assert ((counts - n * w / w.sum()).abs() <= 1.01).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_row_does_not_depend_on_the_others(dtype):
    """Every row of a batch gives what it gives alone, in a view of another alignment and on replay."""
    R, V = 40, 33333
    x = _rows("normal", R, V, dtype)
    u = torch.rand(R, generator=torch.Generator().manual_seed(2)).to(DEV)
    ops = _ops()
    whole = ops.sample_logits(x, u, 1.0, 0, 0.95, 0.0)
    wide = torch.zeros(R, V + 3, dtype=dtype, device=DEV)
    wide[:, 1 : V + 1] = x
    assert torch.equal(ops.sample_logits(wide[:, 1 : V + 1], u, 1.0, 0, 0.95, 0.0), whole)
    for r in (0, 17, 39):
        assert torch.equal(ops.sample_logits(x[r : r + 1], u[r : r + 1], 1.0, 0, 0.95, 0.0), whole[r : r + 1])


def test_capture_and_streams():
    """Both operators replay in a graph on new inputs, and follow the current stream."""
    ops = _ops()
    R, V = 5, 151936
    x, u = _rows("normal", R, V, torch.float32), torch.rand(R, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.topk_rows(x, 50), ops.sample_logits(x, u, 0.8, 50, 0.9)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            values, ids, lse = ops.topk_rows(x, 50)
            token = ops.sample_logits(x, u, 0.8, 50, 0.9)
        for seed in (3, 4):
            x.copy_(_rows("normal", R, V, torch.float32, seed))
            u.copy_(torch.rand(R, generator=torch.Generator().manual_seed(seed)).to(DEV))
            graph.replay()
            want = ops.topk_rows(x, 50)
            assert torch.equal(values, want[0]) and torch.equal(ids, want[1]) and torch.equal(lse, want[2])
            assert torch.equal(token, ops.sample_logits(x, u, 0.8, 50, 0.9))
    torch.cuda.current_stream().wait_stream(side)


def test_refusals():
    ops = _ops()
    x, u = torch.zeros(2, 8, device=DEV), torch.zeros(2, device=DEV)
    for k in (0, 1025):
        with pytest.raises(ValueError):
            ops.topk_rows(x, k)
    for t in (0.0, -1.0, math.nan, math.inf):
        with pytest.raises(ValueError):
            ops.topk_rows(x, 2, t)
    with pytest.raises(ValueError):
        ops.topk_rows(x.half(), 2)
    with pytest.raises(ValueError):
        ops.topk_rows(x.t(), 2)
    with pytest.raises(ValueError):
        ops.topk_rows(x[0], 2)
    with pytest.raises(ValueError):
        ops.topk_rows(torch.zeros(1, 2 ** 20 + 1, device=DEV), 2)  # a row longer than the operators take
    for bad in (u[:1], u.double(), u.cpu()):
        with pytest.raises(ValueError):
            ops.sample_logits(x, bad)
    for knobs in (dict(temperature=-0.1), dict(temperature=math.nan), dict(top_k=-1), dict(top_p=0.0),
                  dict(top_p=1.5), dict(min_p=-0.1), dict(min_p=1.1), dict(top_p=u[:1]), dict(min_p=u.cpu())):
        with pytest.raises(ValueError):
            ops.sample_logits(x, u, **knobs)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [5003, 151936])
def test_sample_wide_rows(dtype, V):
    """Rows that keep thousands of entries: nuclei and min-p at high temperatures, top-k beyond a list."""
    g = torch.Generator().manual_seed(V + 1)
    x = _rows("normal", 12, V, dtype, seed=V)
    x[10, : V // 2] = 1.0  # half a row of equals
    x[11, 1::2] = -math.inf
    for T in (1.5, 6.0, 40.0):
        for f in (dict(top_p=0.5), dict(top_p=0.95), dict(top_p=0.9999), dict(min_p=0.001), dict(min_p=0.5),
                  dict(top_p=0.8, min_p=0.3), dict(top_k=3000), dict(top_k=3000, top_p=0.9, min_p=0.01)):
            u = torch.rand(12, generator=g).to(DEV)
            args = dict(dict(temperature=T, top_k=0, top_p=1.0, min_p=0.0), **f)
            assert torch.equal(_ops().sample_logits(x, u, **args), _sample64(x, u, **args)), (T, f)


def test_sample_more_wide_rows_than_have_lists():
    """Rows past the 2048 wide ones of a call are gone over one by one: the same tokens."""
    R, V = 2100, 4099
    x = _rows("normal", R, V, torch.float32)
    u = torch.rand(R, generator=torch.Generator().manual_seed(3)).to(DEV)
    args = (4.0, 0, 0.9, 0.0)
    whole = _ops().sample_logits(x, u, *args)
    assert torch.equal(whole[:1050], _ops().sample_logits(x[:1050], u[:1050], *args))
    assert torch.equal(whole[1050:], _ops().sample_logits(x[1050:], u[1050:], *args))
    assert torch.equal(whole[:20], _sample64(x[:20], u[:20], *args))


def test_sample_wide_rows_replay():
    """The wide rows' launches in a graph: their number is counted anew on every replay."""
    R, V = 9, 151936
    x, u = _rows("normal", R, V, torch.float32), torch.rand(R, device=DEV)
    temperature = torch.full((R,), 3.0, device=DEV)
    args = (temperature, 0, 0.95, 0.0)
    _ops().sample_logits(x, u, *args)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        token = _ops().sample_logits(x, u, *args)
    for seed, sharp in ((1, 0), (2, 4), (3, 9)):  # that many rows are not wide
        x.copy_(_rows("normal", R, V, torch.float32, seed))
        temperature.fill_(3.0)[:sharp] = 0.2
        graph.replay()
        assert torch.equal(token, _sample64(x, u, *args))


def test_sample_tail_of_lost_weights():
    """A peak over a million entries whose weights round to nothing: a top-p near 1 asks for more than
    the entries' own weights hold, which keeps them all."""
    V = 2 ** 20
    x = torch.full((2, V), -29.9, device=DEV)
    x[0, 5] = x[1, V - 1] = 0.0
    p = 1 - 2.0 ** -24
    got = _ops().sample_logits(x, torch.tensor([0.5, 0.25], device=DEV), 1.0, 0, p, 0.0)
    assert got.tolist() == [5, V - 1]


def test_sample_knobs_beyond_their_ranges():
    """Per-row knobs are not checked: NaN and low temperatures are greedy, +inf weighs all candidates
    alike, top-k past 32 bits is off, top-p at or below 0 keeps the first, NaN filters are off."""
    R, V = 8, 1000
    x = _rows("normal", R, V, torch.float32)
    x[1, 10:] = -math.inf
    u = torch.full((R,), 0.55, device=DEV)
    nan = math.nan
    t = torch.tensor([nan, math.inf, -1.0, 1.0, 1.0, 1.0, 1.0, 1.0], device=DEV)
    k = torch.tensor([0, 0, 0, 2 ** 32 + 1, -2 ** 40, 0, 0, 0], device=DEV)
    p = torch.tensor([1.0, 1.0, 1.0, 1.0, 1.0, 0.0, -1.0, nan], device=DEV)
    m = torch.tensor([0.0, 0.0, 0.0, 0.0, 0.0, 0.0, 0.0, nan], device=DEV)
    got = _ops().sample_logits(x, u, t, k, p, m)
    best = x.argmax(1)
    off = _ops().sample_logits(x, u)
    want = [best[0], 5, best[2], off[3], off[4], best[5], best[6], off[7]]
    assert got.tolist() == [int(w) for w in want]


def test_temperature_range():
    ops = _ops()
    x = _rows("normal", 2, 50, torch.float32)
    for t in (1e-31, 1e31):
        with pytest.raises(ValueError):
            ops.topk_rows(x, 2, t)
    for t in (1e-30, 1e30):
        lse = ops.topk_rows(x, 2, t)[2].double()
        want = torch.logsumexp(x.double() / t, 1)
        assert ((lse - want).abs() <= want.abs() * 2 ** -22 + 2 ** -20).all()


def _small_model():
    from transformers import Qwen3Config

    from orthrus_training_b200.modeling_orthrus import OrthrusLM, copy_diff_from_ar

    cfg = Qwen3Config(vocab_size=1009, hidden_size=128, intermediate_size=256, num_hidden_layers=2,
                      num_attention_heads=4, num_key_value_heads=2, head_dim=32, rms_norm_eps=1e-6,
                      rope_theta=1e4, tie_word_embeddings=True, max_position_embeddings=512)
    cfg.rope_parameters = {"rope_theta": 1e4, "rope_type": "default"}
    cfg.block_size, cfg.mask_token_id = 8, 1008
    torch.manual_seed(0)
    with torch.device(DEV):
        model = OrthrusLM(cfg)
    copy_diff_from_ar(model)
    return model


def test_generate_draws_with_sample_logits():
    """The AR view's sampled generation: each token is the draw from the logits of the sequence up to
    it, the same seed gives the same tokens, and top_k = 1 decodes greedily."""
    ops = _ops()
    model = _small_model()
    prompt = torch.randint(0, 1000, (1, 9), generator=torch.Generator().manual_seed(1)).to(DEV)
    sampler = ops.SamplingParams(0.9, top_k=0, top_p=0.97, seed=11, min_p=0.01)
    out = model.generate(prompt, max_new_tokens=12, use_diffusion_mode=False, sampler=sampler)
    assert torch.equal(out, model.generate(prompt, max_new_tokens=12, use_diffusion_mode=False, sampler=sampler))
    assert out.shape == (1, 21) and torch.equal(out[:, :9], prompt)
    g = torch.Generator(DEV).manual_seed(11)
    for i in range(9, 21):
        with torch.inference_mode():
            logits = model(input_ids=out[:, :i], use_cache=False).logits[0, -1:]
        u = torch.rand(1, device=DEV, generator=g)
        w = torch.softmax(logits[0].double() / 0.9, 0)
        token = ops.sample_logits(logits.float().contiguous(), u, 0.9, 0, 0.97, 0.01)
        assert token.item() == out[0, i].item() and w[token.item()] >= 0.01 * w.max()
    greedy = model.generate(prompt, max_new_tokens=12, use_diffusion_mode=False)
    one = model.generate(prompt, max_new_tokens=12, use_diffusion_mode=False,
                         sampler=ops.SamplingParams(1.0, top_k=1, top_p=1.0, seed=3))
    assert torch.equal(one, greedy)
    with pytest.raises(ValueError):
        model.generate(prompt, max_new_tokens=4, sampler=sampler)
    with pytest.raises(ValueError):
        ops.sample_candidates(torch.zeros(1, 1009, device=DEV), ops.SamplingParams(1.0, min_p=0.1))
