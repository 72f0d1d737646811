"""The operators for drafted tokens (tree plans, tree attention over the 4-bit
cache, logit rules and picks, the end of a step) against plain restatements
(drafts_ref.py).

Tolerances.  Integers and moved bytes are equal.  Adjusted logits: the same
fp32 operations, each rounded, are the same bits in fp32, and in 16 bits after
one more rounding.  Attention: those of test_gpu_serving.py, whose arithmetic
it shares: with u the output type's half unit, t half of its smallest
subnormal, w the half unit of the probabilities (2^-11 for 16-bit activations,
2^-21 for fp32) and e = 2^-20 * (largest scale * sum |q k|), |out - ref| <= u
|ref| + t + (w + 4 e + 2^-19) * sum p |v| + 2^-33 sum |v|, |lse - ref| <= 2 e +
2^-19 (1 + |ref|)."""
import math

import numpy as np
import pytest
import torch

import drafts_ref as D
import serving_ref as R
from test_gpu_serving import DTYPES, HALF_UNIT, SMALLEST, _attend_case, _gen

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def S():
    from sili__new_b200 import serving
    return serving


def _dev(x, dtype=torch.int32):
    return torch.as_tensor(np.asarray(x)).to(dtype).cuda()


def _starts(counts, first=0):
    return np.concatenate([[first], first + np.cumsum(counts)]).astype(np.int64)


# ── plans ────────────────────────────────────────────────────────────────────
@pytest.mark.parametrize("counts,first,extra,window", [
    ([], 0, 3, 0), ([1], 0, 0, 0), ([1, 0, 7, 64], 0, 5, 0), ([65, 3, 130], 2, 300, 0), ([256, 1, 200], 0, 1, 0),
    ([33, 64, 5], 0, 2, 4), ([255, 12], 0, 0, 70), ([1] * 700, 0, 0, 0), ([2, 0, 0], 0, 0, 1)])
def test_draft_tree(S, counts, first, extra, window):
    rng = np.random.default_rng(sum(counts) + window)
    starts = _starts(counts, first)
    tokens = int(starts[-1]) + extra
    parents = np.full(tokens, -1)
    for r, n in enumerate(counts):
        parents[starts[r]:starts[r + 1]] = D.random_tree(n, rng, chain=r % 3 == 0)[:n]
    lens = rng.integers(0, 9000, len(counts)) + np.asarray(counts, int)
    words = max(-(-max(counts, default=0) // 64), 1)
    got = S.draft_tree(_dev(parents), _dev(starts), _dev(lens), max(counts, default=0), window)
    masks, positions = D.draft_tree(parents, starts, lens, tokens, words, window)
    assert got.masks.shape == (tokens, words)
    np.testing.assert_array_equal(got.masks.cpu().numpy(), masks)
    np.testing.assert_array_equal(got.positions.cpu().numpy(), positions)


def test_draft_tree_rows_that_are_none(S):
    """Parents out of place take their descendants with them; rows past the masks' bits; a step that lacks rows."""
    parents = [-1, 0, 2, 2, 1, -5, 5, 0, 9, 8] + [-1] + list(range(69)) + [-1, 0, 1]
    starts, lens = [0, 10, 80, 90], [30, 71, 14]
    got = S.draft_tree(_dev(parents), _dev(starts), _dev(lens), 10)
    masks, positions = D.draft_tree(parents, starts, lens, 83, 1, 0)
    np.testing.assert_array_equal(got.masks.cpu().numpy(), masks)
    np.testing.assert_array_equal(got.positions.cpu().numpy(), positions)
    assert [int(m) for m in got.masks[:10, 0]] == [1, 3, 0, 0, 19, 0, 0, 129, 0, 0]
    assert (got.masks[74:80] == 0).all() and got.positions[80:83].tolist() == [4, 5, 6]     # 14 - 10 committed


# ── attention ────────────────────────────────────────────────────────────────
def _tree_case(committed, counts, h, hk, dim, page, dtype, seed, extra_rows=0, words=None, kind="tree", spare_width=0,
               scale_q=1.5):
    lens = [c + n for c, n in zip(committed, counts)]
    q, codes, scales, table, lens, starts = _attend_case(lens, counts, h, hk, dim, page, dtype, seed, extra_rows=extra_rows,
                                                         spare_width=spare_width, scale_q=scale_q)
    rng = np.random.default_rng(seed)
    tokens = q.shape[0]
    words = words or max(-(-max(counts) // 64), 1)
    if kind == "any":           # not a tree's: any bits, rows without one among them
        masks = rng.integers(-2 ** 63, 2 ** 63, (tokens, words)) & rng.integers(-2 ** 63, 2 ** 63, (tokens, words))
        masks[rng.random(tokens) < 0.25] = 0
    else:
        parents = np.full(tokens, -1)
        for r, n in enumerate(counts):
            parents[starts[r]:starts[r + 1]] = D.random_tree(n, rng, chain=kind == "chain")[:n]
        masks, _ = D.draft_tree(parents, starts, lens.cpu().numpy(), tokens, words, 0)
    return q, codes, scales, table, lens, starts, torch.from_numpy(masks).cuda()


def _check_tree(S, case, dtype, window=0, scale=None, most_new=None):
    q, codes, scales, table, lens, starts, masks = case
    sc = 1 / math.sqrt(q.shape[2]) if scale is None else scale
    out, lse = S.tree_attention(q, codes, scales, table, lens, _dev(starts), masks, most_new=most_new, scale=scale,
                                window=window, return_lse=True)
    S.check_attention()
    ref, ref_lse, spread, size, total = D.tree_attention(q, codes, scales, table, lens.cpu().numpy(), starts, masks, sc, window)
    out, lse = out.double().cpu().numpy(), lse.double().cpu().numpy()
    w = 2.0 ** -21 if dtype == torch.float32 else 2.0 ** -11
    e = 2.0 ** -20 * size
    empty = np.isinf(ref_lse)
    assert (np.isinf(lse) == empty).all() and (out[empty] == 0).all()
    ok = ~empty
    assert (np.abs(lse[ok] - ref_lse[ok]) <= 2 * e[ok] + 2.0 ** -19 * (1 + np.abs(ref_lse[ok]))).all()
    bound = HALF_UNIT[dtype] * np.abs(ref) + SMALLEST[dtype] + (w + 4 * e[..., None] + 2.0 ** -19) * spread + 2.0 ** -33 * total
    worst = (np.abs(out - ref) / np.maximum(bound, 1e-30))[ok].max(initial=0.0)
    assert worst <= 1.0, worst


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("committed,counts,h,hk,dim,page", [
    ([0], [1], 1, 1, 64, 16), ([1, 0, 15], [1, 5, 16], 4, 2, 128, 16), ([700, 3, 64], [8, 0, 24], 8, 2, 128, 16),
    ([333, 48], [9, 33], 3, 3, 256, 48), ([1000, 1, 260], [7, 64, 40], 8, 2, 64, 64), ([530], [20], 20, 4, 128, 128),
    ([77, 200], [65, 130], 5, 1, 128, 32), ([127, 128, 129], [1, 2, 3], 10, 1, 64, 16), ([250], [256], 2, 1, 64, 16)])
def test_tree_attention(S, dtype, committed, counts, h, hk, dim, page):
    case = _tree_case(committed, counts, h, hk, dim, page, dtype, sum(committed) + dim, extra_rows=3, spare_width=2)
    _check_tree(S, case, dtype, most_new=max(counts))
    _check_tree(S, case, dtype, most_new=1)     # a wrong hint changes nothing


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("h,hk,dim,page", [(8, 2, 128, 16), (6, 1, 64, 48), (2, 1, 256, 32)])
def test_tree_attention_any_masks(S, dtype, h, hk, dim, page):
    """Bits that make no tree, rows without one, more words than there are rows."""
    case = _tree_case([300, 0, 31, 5], [50, 70, 3, 130], h, hk, dim, page, dtype, 3, extra_rows=2, words=4, kind="any")
    _check_tree(S, case, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("window", [1, 4, 37, 150, 100000])
def test_tree_attention_window(S, dtype, window):
    case = _tree_case([400, 20, 0], [30, 40, 33], 8, 2, 128, 16, dtype, window)
    _check_tree(S, case, dtype, window=window)


@pytest.mark.parametrize("dtype", DTYPES)
def test_tree_attention_edges(S, dtype):
    """Missing pages, a table too narrow, lengths below the rows' number, large and negative scales, no requests."""
    case = _tree_case([90, 200, 40], [20, 40, 12], 8, 2, 128, 16, dtype, 5, scale_q=4.0)
    q, codes, scales, table, lens, starts, masks = case
    table[0, 2], table[1, 14] = -1, 1 << 29
    _check_tree(S, case, dtype)
    _check_tree(S, case, dtype, scale=-0.05)
    _check_tree(S, case, dtype, scale=0.0)
    _check_tree(S, (q, codes, scales, table[:, :6], *case[4:]), dtype)
    few = torch.tensor([7, 0, -3], dtype=torch.int32, device="cuda")
    few_case = (q, codes, scales, table, few, starts, masks)
    _check_tree(S, few_case, dtype)
    out = S.tree_attention(q, codes, scales, table[:0], lens[:0], _dev([0]), masks)
    assert (out == 0).all()
    assert S.tree_attention(q[:0], codes, scales, table[:0], lens[:0], _dev([0]), masks[:0]).shape == (0, 8, 128)


@pytest.mark.parametrize("dtype", DTYPES)
def test_tree_attention_step_that_lacks_rows(S, dtype):
    """Rows past the step's arrays are left out and move no other row."""
    q, codes, scales, table, lens, starts, masks = case = _tree_case([90, 50], [20, 40], 8, 2, 64, 16, dtype, 6)
    _check_tree(S, (q[:45], codes, scales, table, lens, starts, masks[:45]), dtype)
    whole = S.tree_attention(q, codes, scales, table, lens, _dev(starts), masks, most_new=40)
    part = S.tree_attention(q[:45], codes, scales, table, lens, _dev(starts), masks[:45].clone(), most_new=40)
    assert torch.equal(whole[:45], part)
    assert case[0] is q


def test_a_chain_is_a_prompt(S):
    """Rows that each follow the one before see what cache_attention's rows see: the same kernel, the same bits."""
    case = _tree_case([300, 0, 77], [20, 6, 1], 8, 2, 128, 16, torch.float32, 8, kind="chain")
    q, codes, scales, table, lens, starts, masks = case
    for window in (0, 40):
        a = S.tree_attention(q, codes, scales, table, lens, _dev(starts), masks, window=window, return_lse=True)
        b = S.cache_attention(q, codes, scales, table, lens, starts=_dev(starts), window=window, return_lse=True)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("dtype", DTYPES)
def test_tree_attention_nan_reaches_its_readers_only(S, dtype):
    case = _tree_case([100, 90], [40, 12], 8, 2, 128, 16, dtype, 9, kind="any")
    q, codes, scales, table, lens, starts, masks = case
    clean = S.tree_attention(q, codes, scales, table, lens, _dev(starts), masks)
    # V of request 0, kv head 1, its drafted row 7 (key 107), values 32..63; K of request 1's committed key 5, kv head 0
    scales[table[0, 6].long(), 1, 1, 11, 1] = 0xFF
    scales[table[1, 0].long(), 0, 0, 5, 0] = 0xFF
    got = S.tree_attention(q, codes, scales, table, lens, _dev(starts), masks)
    some = masks[:, 0] != 0
    want = torch.zeros_like(got, dtype=torch.bool)
    sees = (masks[:40, 0] >> 7 & 1).bool()
    want[:40][sees, 4:, 32:64] = True
    want[40:][some[40:], :4] = True
    assert torch.equal(torch.isnan(got), want) and torch.equal(got[~want], clean[~want])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_tree_attention_is_deterministic_across_streams_and_graphs(S, dtype):
    case = _tree_case([4000, 900, 17], [40, 64, 3], 32, 8, 128, 16, dtype, 10)
    q, codes, scales, table, lens, starts, masks = case
    starts = _dev(starts)

    def call(out=None):
        return S.tree_attention(q, codes, scales, table, lens, starts, masks, most_new=64, out=out)

    first = call()
    for _ in range(3):
        assert torch.equal(first, call())
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        other = call()
    side.synchronize()
    assert torch.equal(first, other)
    graphs, outs = [], []
    for _ in range(2):
        out, graph = torch.empty_like(first), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call(out)
        graphs.append(graph)
        outs.append(out)
    for _ in range(2):
        for out in outs:
            out.zero_()
        torch.cuda.synchronize()
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
        other = call()
        torch.cuda.synchronize()
        assert torch.equal(first, outs[0]) and torch.equal(first, outs[1]) and torch.equal(first, other)
    # lengths and masks are read on the device: a replay follows them
    lens.sub_(11)
    masks.bitwise_and_(masks.roll(1, 0))
    graphs[0].replay()
    assert torch.equal(outs[0], call())


def test_tree_attention_offsets_pass_32_bits(S):
    """Pages whose code bytes lie past 4 GB."""
    n_pages, page, hk, dim = 4500, 1024, 8, 128
    codes = torch.zeros(n_pages, 2, hk, page, dim // 2, dtype=torch.uint8, device="cuda")
    scales = torch.full((n_pages, 2, hk, page, dim // 32), 100, dtype=torch.uint8, device="cuda")
    small, small_scales = R.random_cache(2, hk, page, dim, _gen(4))
    codes[4490:4492], scales[4490:4492] = small, small_scales
    q = torch.randn(24, 8, dim, generator=_gen(5), device="cuda").half()
    masks = torch.from_numpy(D.draft_tree(D.random_tree(24, np.random.default_rng(1)), [0, 24], [1100], 24, 1, 0)[0]).cuda()
    lens, starts = _dev([1100]), _dev([0, 24])
    got = S.tree_attention(q, codes, scales, _dev([[4490, 4491]]), lens, starts, masks)
    want = S.tree_attention(q, small, small_scales, _dev([[0, 1]]), lens, starts, masks)
    assert torch.equal(got, want)


# ── logits ───────────────────────────────────────────────────────────────────
def _rules(requests, rows, vocab, rng, history=0, drafted=None, biases=0, masked=False, starts=None):
    q = {}
    if history:
        q["history"] = rng.integers(-2, vocab + 2, (requests, history)).astype(np.int32)
        q["history"][:, ::3] = rng.integers(0, min(7, vocab), q["history"][:, ::3].shape)      # some many times
        q["history_lens"] = rng.integers(-1, history + 3, requests).astype(np.int32)
        q["prompt_lens"] = rng.integers(-1, history + 1, requests).astype(np.int32)
    for name, lo, hi in (("repetition", 0.8, 1.6), ("presence", -0.3, 1.0), ("frequency", -0.1, 0.5), ("temperature", 0.2, 1.5)):
        q[name] = rng.uniform(lo, hi, requests).astype(np.float32)
    q["temperature"][::4] = 0.0
    if biases:
        q["bias_tokens"] = rng.integers(-1, vocab + 1, (requests, biases)).astype(np.int32)
        q["bias_values"] = (rng.normal(size=(requests, biases)) * 3).astype(np.float32)
    if masked:
        words = rng.integers(-2 ** 31, 2 ** 31, (rows, -(-vocab // 32))).astype(np.int32)
        words[::3] = -1
        words[4::5] = 0
        q["allowed"] = words
    if drafted is not None:
        q["drafted"], q["masks"] = drafted
    return q


def _logit_case(counts, vocab, dtype, seed, extra=0, history=0, biases=0, masked=False, tree=False, stride=0):
    rng = np.random.default_rng(seed)
    starts = None if counts is None else _starts(counts, 1 if extra else 0)
    rows = 6 if counts is None else int(starts[-1]) + extra
    requests = 6 if counts is None else len(counts)
    x = (rng.normal(size=(rows, vocab + stride)) * 4).astype(np.float32)
    x = torch.from_numpy(x).to(dtype)[:, :vocab] if stride else torch.from_numpy(x).to(dtype)
    drafted = None
    if tree:
        words = max(-(-max(counts) // 64), 1)
        masks = rng.integers(-2 ** 63, 2 ** 63, (rows, words)) & rng.integers(-2 ** 63, 2 ** 63, (rows, words))
        tokens = rng.integers(-1, vocab + 1, rows).astype(np.int32)
        tokens[::2] = rng.integers(0, min(5, vocab), len(tokens[::2]))
        drafted = tokens, masks
    return x, starts, _rules(requests, rows, vocab, rng, history, drafted, biases, masked, starts)


def _on_gpu(starts, rules):
    d = {k: torch.from_numpy(np.ascontiguousarray(v)).cuda() for k, v in rules.items()}
    if starts is not None:
        d["starts"] = _dev(starts)
    return d


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("counts,vocab,kw", [
    (None, 1, {}), (None, 31, dict(history=3, masked=True)), (None, 1000, dict(history=200, biases=9, masked=True)),
    ([3, 0, 1, 5], 8191, dict(history=40, extra=2, tree=True, biases=70, masked=True)),
    ([20, 9], 8192, dict(history=900, tree=True)), ([66, 130], 999, dict(history=50, tree=True, masked=True, stride=13)),
    (None, 20011, dict(history=5000, biases=400)), ([1, 1], 40000, dict(masked=True, stride=3)), ([2, 7], 16384, dict())])
def test_logit_rules(S, dtype, counts, vocab, kw):
    x, starts, rules = _logit_case(counts, vocab, dtype, vocab, **kw)
    y, of = D.adjust(x.float().numpy(), starts, rules)
    g = _on_gpu(starts, rules)
    xs = torch.empty(x.shape[0], x.stride(0), dtype=dtype, device="cuda")[:, :vocab].copy_(x)
    want = torch.from_numpy(y).to(dtype)
    got = S.adjust_logits(xs, **g)
    assert torch.equal(got.cpu(), want)
    np.testing.assert_array_equal(S.pick_tokens(xs, **g).cpu().numpy(), D.pick(y, of))
    # an output of another alignment, then in place
    out = torch.full((x.shape[0], vocab + 5), 7.0, dtype=dtype, device="cuda")
    assert S.adjust_logits(xs, **g, out=out[:, 1:vocab + 1]).data_ptr() == out[:, 1:].data_ptr()
    assert torch.equal(out[:, 1:vocab + 1].cpu(), want) and (out[:, 0] == 7).all() and (out[:, vocab + 1:] == 7).all()
    assert S.adjust_logits(xs, **g, out=xs) is xs and torch.equal(xs.cpu(), want)


@pytest.mark.parametrize("dtype", DTYPES)
def test_logit_rules_alone(S, dtype):
    """Each part without the others."""
    x, starts, rules = _logit_case([4, 3], 3001, dtype, 2, history=90, biases=20, masked=True, tree=True)
    g = _on_gpu(starts, rules)
    parts = [(), ("repetition",), ("history", "history_lens", "repetition"),
             ("history", "history_lens", "prompt_lens", "presence"), ("history", "history_lens", "frequency"),
             ("drafted", "masks", "frequency"), ("drafted", "masks", "repetition", "presence"),
             ("bias_tokens", "bias_values"), ("temperature",), ("allowed",), ("allowed", "temperature")]
    for names in parts:
        y, of = D.adjust(x.float().numpy(), starts, {n: rules[n] for n in names})
        some = {n: g[n] for n in names}
        assert torch.equal(S.adjust_logits(x.cuda(), starts=g["starts"], **some).cpu(), torch.from_numpy(y).to(dtype)), names
        np.testing.assert_array_equal(S.pick_tokens(x.cuda(), starts=g["starts"], **some).cpu().numpy(), D.pick(y, of))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [5, 8200, 70001])
def test_pick_ties_infinities_and_nan(S, dtype, vocab):
    x = torch.full((9, vocab), -2.0)
    x[0] = -math.inf                                   # nothing
    x[1, vocab - 1] = 3.0
    x[2, 1:] = 0.0                                     # the first of equals, -0 and 0 alike
    x[2, 1] = -0.0
    x[3, 2], x[3, 3] = math.nan, math.inf              # NaN is above all
    x[4, vocab // 2:] = math.inf
    x[5] = -math.inf
    x[5, vocab - 2] = torch.finfo(dtype).min           # the lowest value is still a value
    x[6, 0], x[6, 4] = 1.0, 1.0
    x[7] = math.nan
    x[8, 3] = math.nan                                 # but not where the mask does not allow it
    allowed = torch.full((9, -(-vocab // 32)), -1, dtype=torch.int32)
    allowed[8, 0] &= ~8
    allowed[8, -1] &= (1 << (vocab % 32)) - 1 if vocab % 32 else -1
    got = S.pick_tokens(x.to(dtype).cuda(), allowed=allowed.cuda()).tolist()
    assert got == [-1, vocab - 1, 1, 2, vocab // 2, vocab - 2, 0, 0, 0]
    # a row of equals whose order a temperature's rounding makes: neighbours in fp32 that the quotient joins
    if dtype == torch.float32:
        y = torch.ones(1, vocab)
        y[0, 3] = 1.0 + 2.0 ** -23
        for heat in (1.0, 0.7, 1.3, 3.0):
            q = np.asarray(y.numpy() / np.float32(heat))[0]
            assert S.pick_tokens(y.cuda(), temperature=torch.tensor([heat], device="cuda")).item() == int(q.argmax())


def test_pick_agrees_with_adjusted_rows(S):
    """The pick is the adjusted row's argmax, near-equal values included (temperatures join neighbours)."""
    g = _gen(7)
    base = torch.randint(0, 40, (64, 20000), generator=g, device="cuda").float()
    x = torch.nextafter(base, torch.full_like(base, math.inf)) * (torch.rand(base.shape, generator=g, device="cuda") < 0.5) + \
        base * (torch.rand(base.shape, generator=g, device="cuda") < 0.5)
    heat = torch.rand(64, generator=g, device="cuda") * 3 + 0.1
    history = torch.randint(0, 20000, (64, 500), generator=g, device="cuda", dtype=torch.int32)
    rules = dict(temperature=heat, history=history, history_lens=torch.full((64,), 500, dtype=torch.int32, device="cuda"),
                 repetition=torch.full((64,), 0.999, device="cuda"))
    y = S.adjust_logits(x, **rules)
    top = y.amax(1, keepdim=True)
    at = torch.where(y == top, torch.arange(y.shape[1], device="cuda"), y.shape[1]).amin(1)
    assert torch.equal(S.pick_tokens(x, **rules).long(), at)


def test_logits_many_rows_streams_and_graphs(S):
    """More row groups than a grid's second axis has, another stream, a graph whose replay follows its inputs."""
    x = torch.randn(70001, 40, generator=_gen(1), device="cuda")
    assert torch.equal(S.pick_tokens(x).long(), x.argmax(1))
    assert torch.equal(S.adjust_logits(x, temperature=torch.full((70001,), 0.5, device="cuda")), x / 0.5)
    x = torch.randn(5, 60000, generator=_gen(2), device="cuda").bfloat16()
    heat = torch.full((5,), 0.7, device="cuda")
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    want, best = S.adjust_logits(x, temperature=heat), S.pick_tokens(x, temperature=heat)
    with torch.cuda.stream(side):
        assert torch.equal(S.adjust_logits(x, temperature=heat), want)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        y, b = S.adjust_logits(x, temperature=heat), S.pick_tokens(x, temperature=heat)
    graph.replay()
    assert torch.equal(y, want) and torch.equal(b, best)
    x.copy_(x.flip(1))
    graph.replay()
    assert torch.equal(y, want.flip(1)) and torch.equal(b, S.pick_tokens(x, temperature=heat))


def test_logits_offsets_pass_32_bits(S):
    x = torch.zeros(17000, 131072, dtype=torch.bfloat16, device="cuda")       # 2.2e9 elements, 4.5 GB
    at = (torch.arange(17000, device="cuda") * 977) % 131072
    x[torch.arange(17000, device="cuda"), at] = 1.0
    assert torch.equal(S.pick_tokens(x).long(), at)
    S.adjust_logits(x, temperature=torch.full((17000,), 0.5, device="cuda"), out=x)
    assert float(x.amax()) == 2.0 and torch.equal(S.pick_tokens(x).long(), at)


# ── the end of a step ────────────────────────────────────────────────────────
def _settle_case(counts, committed, page, seed, extra=0, first=0, chain=False, agree=0.7):
    rng = np.random.default_rng(seed)
    starts = _starts(counts, first)
    tokens = int(starts[-1]) + extra
    parents, drafted = np.full(tokens, -1), rng.integers(0, 50, tokens)
    picked = rng.integers(-1, 50, tokens)
    for r, n in enumerate(counts):
        a = int(starts[r])
        parents[a:a + n] = D.random_tree(n, rng, chain)[:n]
        for i in range(n):
            children = [j for j in range(i + 1, n) if parents[a + j] == i]
            if children and rng.random() < agree:
                picked[a + i] = drafted[a + children[int(rng.integers(len(children)))]]
    lens = np.asarray(committed) + np.asarray(counts, int)
    used = -(-lens // page)
    width = int(used.max(initial=0)) + 1
    n_pages = int(used.sum()) + 4
    perm = rng.permutation(n_pages)
    table = np.full((len(counts), width), -1)
    at = 0
    for r, u in enumerate(used):
        table[r, :u] = perm[at:at + u]
        at += u
    ring = np.full(n_pages, -7)
    taken = int(rng.integers(0, 5 * n_pages))
    ring[(taken + np.arange(n_pages - at)) % n_pages] = perm[at:]
    return starts, tokens, parents, drafted, picked, lens, table, ring, np.array([taken, taken + n_pages - at]), n_pages


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("counts,committed,page,hk,dim,layers,kw", [
    ([1], [0], 16, 1, 64, 1, {}), ([8, 0, 1, 20], [33, 5, 0, 100], 16, 2, 128, 3, dict(extra=4, first=2)),
    ([64, 30, 64], [10, 47, 300], 16, 3, 256, 2, {}), ([256, 200], [7, 20], 48, 2, 64, 2, dict(chain=True, agree=1.0)),
    ([300], [3], 16, 1, 64, 1, dict(chain=True, agree=1.0)), ([12, 9], [40, 17], 16, 2, 128, 130, {}),
    ([3] * 1300, [14] * 1300, 16, 1, 64, 1, {})])
def test_settle_drafts(S, wide, counts, committed, page, hk, dim, layers, kw):
    starts, tokens, parents, drafted, picked, lens, table, ring, pool, n_pages = _settle_case(counts, committed, page, sum(counts), **kw)
    if len(counts) > 2:
        table[2, -2:] = -1                              # pages that lack
    caches = [R.random_cache(n_pages, hk, page, dim, _gen(i)) for i in range(layers)]
    path, kept, token, out = D.accept(drafted, parents, picked, starts, lens, tokens)
    want = [[x.cpu().numpy().copy() for x in c] for c in caches]
    for w in want:
        D.move(w, table, starts, lens, path, kept, page)
    new_ring, new_pool = D.trim(lens, out, table, ring, pool, page)
    held, table_before = _dev(ring), _dev(table)
    objects = [S.KVCache4.__new__(S.KVCache4) for _ in caches]
    for o, (c, b) in zip(objects, caches):
        o.codes, o.scales = c, b
    dev_table = _dev(table)
    a = S.settle_drafts(_dev(drafted), _dev(parents), _dev(picked, torch.int64 if wide else torch.int32), _dev(starts),
                        _dev(lens), dev_table, objects if wide else caches, held, _dev(pool, torch.int64))
    np.testing.assert_array_equal(a.path.cpu().numpy(), path)
    np.testing.assert_array_equal(a.kept.cpu().numpy(), kept)
    np.testing.assert_array_equal(a.token.cpu().numpy(), token)
    np.testing.assert_array_equal(a.lens.cpu().numpy(), out)
    np.testing.assert_array_equal(held.cpu().numpy(), new_ring)
    assert a.pool.tolist() == new_pool and torch.equal(dev_table, table_before)
    for (c, b), (wc, wb) in zip(caches, want):
        np.testing.assert_array_equal(c.cpu().numpy(), wc)
        np.testing.assert_array_equal(b.cpu().numpy(), wb)
    # the same inputs write the same values again, but for the caches
    again = S.settle_drafts(_dev(drafted), _dev(parents), _dev(picked), _dev(starts), _dev(lens), dev_table,
                            [R.random_cache(n_pages, hk, page, dim, _gen(0))], held, _dev(pool, torch.int64))
    assert all(torch.equal(x, y) for x, y in zip(a, again)) and np.array_equal(held.cpu().numpy(), new_ring)


def test_settle_step_that_lacks_rows_and_has_no_root(S):
    parents, drafted = [-1, 0, 1, 2, 0, 0, -1, 0, 1, 2], [5, 6, 7, 8, 1, 2, 9, 3, 4, 5]
    picked = [6, 7, 8, 9, 6, 7, 3, 4, 5, 6]
    starts, lens = [0, 4, 6, 12], [24, 12, 26]          # the last request lacks two rows
    codes, scales = R.random_cache(5, 1, 16, 64, _gen(1))
    table = _dev([[0, 1], [2, -1], [3, 4]])
    ring, pool = S.page_pool(5)
    a = S.settle_drafts(_dev(drafted), _dev(parents), _dev(picked), _dev(starts), _dev(lens), table, [(codes, scales)], ring,
                        _dev([5, 5], torch.int64))
    assert a.path.tolist() == [0, 1, 2, 3, -1, -1, 0, 1, 2, 3]
    assert a.kept.tolist() == [4, 0, 4] and a.token.tolist() == [9, -1, 6] and a.lens.tolist() == [24, 10, 24]
    assert a.pool.tolist() == [5, 5]


def test_settle_on_a_graph_and_another_stream(S):
    starts, tokens, parents, drafted, picked, lens, table, ring, pool, n_pages = _settle_case([20, 31], [40, 9], 16, 4)
    codes, scales = R.random_cache(n_pages, 2, 16, 128, _gen(3))
    start = codes.clone(), scales.clone()
    held = _dev(ring)
    args = [_dev(drafted), _dev(parents), _dev(picked), _dev(starts), _dev(lens), _dev(table), [(codes, scales)], held,
            _dev(pool, torch.int64)]
    first = S.settle_drafts(*args)
    moved, ring_after = codes.clone(), held.clone()
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        a = S.settle_drafts(*args)
    for replay in (graph.replay, lambda: S.settle_drafts(*args)):
        codes.copy_(start[0])
        scales.copy_(start[1])
        held.copy_(_dev(ring))
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            replay()
        side.synchronize()
        assert torch.equal(codes, moved) and torch.equal(held, ring_after)
        assert all(torch.equal(x, y) for x, y in zip(a, first))


# ── all of it together ───────────────────────────────────────────────────────
class _Toy:
    """Two attention layers over 4-bit caches between an embedding and a head, greedy."""

    def __init__(self, S, dtype, requests, pages, page=16, hidden=128, h=4, hk=2, dim=64, vocab=97):
        g = _gen(11)
        self.S, self.h, self.hk, self.dim, self.page, self.dtype, self.vocab = S, h, hk, dim, page, dtype, vocab
        rand = lambda *s: torch.randn(*s, generator=g, device="cuda", dtype=torch.float64)  # noqa: E731
        self.embed, self.head = rand(vocab, hidden), rand(hidden, vocab)
        self.w = [(rand(hidden, (h + 2 * hk) * dim) / 12, rand(h * dim, hidden) / 8) for _ in range(2)]
        self.caches = [S.KVCache4(pages, page, hk, dim) for _ in range(2)]
        self.ring, self.pool = S.page_pool(pages)
        self.table = torch.full((requests, pages), -1, dtype=torch.int32, device="cuda")
        self.lens = torch.zeros(requests, dtype=torch.int32, device="cuda")
        self.cos, self.sin = S.rotary_table(4096, dim)
        self.rep = torch.full((requests,), 1.2, device="cuda")
        self.pres = torch.full((requests,), 0.5, device="cuda")

    def layers(self, tokens, t, positions, attend):
        S, x = self.S, self.embed[tokens.clamp(min=0).long()]
        for (w, o), c in zip(self.w, self.caches):
            y = (x @ w).to(self.dtype).view(len(tokens), -1, self.dim)
            q, k, v = y[:, :self.h], y[:, self.h:self.h + self.hk], y[:, self.h + self.hk:]
            q = S.cache_append(k, v, c.codes, c.scales, t.slots, cos=self.cos, sin=self.sin, positions=positions, q=q)
            x = x + attend(q, c).double().flatten(1) @ o
        return (x @ self.head).float()

    def tables(self, fresh, rows):
        t = self.S.page_tables(self.lens, fresh, self.table, self.ring, self.pool, self.page, rows)
        assert t.status.tolist() == [0, 0, 0]
        return t

    def prompt(self, prompts):
        fresh = _dev([len(p) for p in prompts])
        tokens = _dev(sum(prompts, []))
        t = self.tables(fresh, len(tokens))
        self.layers(tokens, t, t.positions, lambda q, c: self.S.cache_attention(q, c.codes, c.scales, self.table, t.lens,
                                                                                 starts=t.starts, most_new=max(map(len, prompts))))
        self.lens, self.pool = t.lens, t.pool


def test_drafted_decoding_gives_the_tokens_of_plain_decoding(S, dtype=torch.float32):
    """Prompts, then steps of drafted trees (plans, append, tree attention, picks under penalties, acceptance), against
    the same model that decodes a token a step.  Drafts are partly the plain run's own tokens, so some are accepted."""
    prompts, steps = [[3, 14, 15, 92, 65], [35, 8], [9] * 17], 24
    plain, n = _Toy(S, dtype, 3, 40), 3
    plain.prompt([p[:-1] for p in prompts])
    told = [list(p) for p in prompts]
    ones = torch.ones(n, dtype=torch.int32, device="cuda")
    margin = math.inf
    for _ in range(steps + 12):
        t = plain.tables(ones, n)
        logits = plain.layers(_dev([x[-1] for x in told]), t, t.positions, lambda q, c: S.cache_attention(
            q, c.codes, c.scales, plain.table, t.lens))
        history = torch.zeros(n, 200, dtype=torch.int32, device="cuda")
        for r, x in enumerate(told):
            history[r, :len(x)] = _dev(x)
        # (of a prompt the last token is the first step's root, and so on the path: in both runs it counts as output)
        rules = dict(history=history, history_lens=_dev([len(x) for x in told]), prompt_lens=_dev([len(p) - 1 for p in prompts]),
                     repetition=plain.rep, presence=plain.pres)
        two = S.adjust_logits(logits, **rules).topk(2, 1).values
        margin = min(margin, float((two[:, 0] - two[:, 1]).min()))
        for r, v in enumerate(S.pick_tokens(logits, **rules).tolist()):
            told[r].append(v)
        plain.lens, plain.pool = t.lens, t.pool
    assert margin > 1e-3      # no pick of the plain run hangs on a rounding

    toy, rng = _Toy(S, dtype, n, 40), np.random.default_rng(5)
    toy.prompt([p[:-1] for p in prompts])
    got, accepted, stepped = [list(p) for p in prompts], 0, 0
    while min(len(g) - len(p) for g, p in zip(got, prompts)) < steps:
        counts = [int(c) for c in rng.integers(1, 40, n)]
        starts = _starts(counts)
        rows = int(starts[-1]) + 3
        parents, drafted = np.full(rows, -1), np.full(rows, -1)
        for r, c in enumerate(counts):
            tree = D.random_tree(c, rng)
            depth = [0]
            for i in range(1, c):
                depth.append(depth[tree[i]] + 1)
            for i in range(c):
                at = len(got[r]) - 1 + depth[i]
                right = i == 0 or (rng.random() < 0.6 and at < len(told[r]))
                drafted[starts[r] + i] = told[r][at] if right else rng.integers(0, toy.vocab)
            parents[starts[r]:starts[r] + c] = tree
        parents, drafted = _dev(parents), _dev(drafted)
        t = toy.tables(_dev(counts), rows)
        tree = S.draft_tree(parents, t.starts, t.lens, max(counts))
        logits = toy.layers(drafted, t, tree.positions, lambda q, c: S.tree_attention(
            q, c.codes, c.scales, toy.table, t.lens, t.starts, tree.masks, most_new=max(counts)))
        history = torch.zeros(n, 200, dtype=torch.int32, device="cuda")
        for r, x in enumerate(got):
            history[r, :len(x) - 1] = _dev(x[:-1])
        # the step's root is the last token: it stands on the path, not in the history
        picked = S.pick_tokens(logits, starts=t.starts, history=history, history_lens=_dev([len(x) - 1 for x in got]),
                               prompt_lens=_dev([len(p) - 1 for p in prompts]), drafted=drafted, masks=tree.masks,
                               repetition=toy.rep, presence=toy.pres)
        end = S.settle_drafts(drafted, parents, picked, t.starts, t.lens, toy.table, toy.caches, toy.ring, t.pool)
        toy.lens, toy.pool = end.lens, end.pool
        path, kept, token = end.path.tolist(), end.kept.tolist(), end.token.tolist()
        for r in range(n):
            rows_of = [path[starts[r] + j] for j in range(kept[r])]
            got[r] += [int(drafted[starts[r] + i]) for i in rows_of[1:]] + [token[r]]
            accepted += kept[r] - 1
        stepped += n
        held = sorted(p for r in range(n) for p in toy.table[r, :-(-int(toy.lens[r]) // toy.page)].tolist())
        assert len(set(held)) == len(held) == int(toy.pool[0] - toy.pool[1]) + 40
        free = [int(toy.ring[i % 40]) for i in range(int(toy.pool[0]), int(toy.pool[1]))]
        assert sorted(held + free) == list(range(40))
    assert accepted > stepped // 4
    for r in range(n):
        m = min(len(got[r]), len(told[r]))
        assert got[r][:m] == told[r][:m]


# ── the kernel of many 16-bit rows ───────────────────────────────────────────
def _own_kernel(dtype, dim, h, hk, most_new):
    from sili__new_b200 import _cuda
    code = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}[dtype]
    return _cuda.kv4_tree_attention_workspace(code, dim, h, hk, most_new) != _cuda.kv4_attention_workspace()


def test_which_calls_have_a_kernel_of_their_own():
    assert not _own_kernel(torch.float32, 128, 32, 8, 64) and not _own_kernel(torch.bfloat16, 256, 32, 8, 64)
    assert not _own_kernel(torch.float16, 64, 8, 8, 32) and _own_kernel(torch.float16, 64, 8, 8, 33)
    assert _own_kernel(torch.bfloat16, 128, 32, 8, 9) and not _own_kernel(torch.bfloat16, 128, 32, 8, 8)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("h,hk,dim,page,most,longest", [(8, 2, 64, 16, 60, 200), (4, 2, 128, 48, 64, 150), (20, 4, 64, 32, 51, 90)])
def test_many_short_trees(S, dtype, h, hk, dim, page, most, longest):
    """A CTA's run goes over many segments of one or two units, of one row tile or two."""
    rng = np.random.default_rng(most)
    counts = [int(c) for c in rng.integers(0, most + 1, 70)]
    counts[3], counts[7] = most, 1
    committed = [int(c) for c in rng.integers(0, longest, 70)]
    assert _own_kernel(dtype, dim, h, hk, most)
    case = _tree_case(committed, counts, h, hk, dim, page, dtype, most, extra_rows=4)
    _check_tree(S, case, dtype, most_new=most)
    _check_tree(S, case, dtype, most_new=most, window=25)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("counts,h,hk,dim", [([130], 2, 1, 128), ([256, 3, 200], 8, 8, 64), ([33, 40], 4, 4, 128)])
def test_trees_over_long_caches(S, dtype, counts, h, hk, dim):
    """Segments that many CTAs share."""
    assert _own_kernel(dtype, dim, h, hk, max(counts))
    case = _tree_case([6000, 2500, 3000][:len(counts)], counts, h, hk, dim, 64, dtype, 4)
    _check_tree(S, case, dtype, most_new=max(counts))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("size", [1e-4, 30.0, 3000.0])
def test_tree_query_sizes(S, dtype, size):
    """Flat to one-hot softmaxes, maxima that move late; rows of very different sizes in one tile."""
    case = _tree_case([900, 90], [40, 36], 8, 2, 128, 16, dtype, 13, scale_q=size)
    _check_tree(S, case, dtype)
    _check_tree(S, case, dtype, scale=-0.3 / size)
    q = case[0].clone()
    q[::3] *= 2.0 ** -12
    _check_tree(S, (q, *case[1:]), dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_tree_sums_of_long_runs_hold(S, dtype):
    """Runs of more units than a row's sums stay in tensor memory for (fp16): V is the same in every key, so the output is V.
    |out - V| <= u |V| + 2^-11 |V| (probabilities rounded) + 2^-19 |V| (fp32 sums)."""
    from test_gpu_serving_long import _one_v
    keys, hk, d, n = 420000, 8, 64, 40
    assert _own_kernel(dtype, d, hk, hk, n) and keys * hk // 128 // 148 > 128
    codes, scales, want = _one_v(keys, hk, d, 3)
    table = torch.arange(codes.shape[0], dtype=torch.int32, device="cuda")[None]
    masks = torch.from_numpy(D.draft_tree(D.random_tree(n, np.random.default_rng(2)), [0, n], [keys], n, 1, 0)[0]).cuda()
    q = (torch.randn(n, hk, d, generator=_gen(1), device="cuda") * 0.3).to(dtype)
    args = (codes, scales, table, _dev([keys]), _dev([0, n]), masks)
    out, lse = S.tree_attention(q, *args, return_lse=True)
    S.check_attention()
    off = out.double() / want[None] - 1
    assert float(off.abs().max()) <= HALF_UNIT[dtype] + 2.0 ** -11 + 2.0 ** -19
    assert abs(float(off.mean())) <= 2.0 ** -12
    # each row's lse against the kernel for single rows (fp32 sums of the same probabilities in another order)
    few = S.tree_attention(q[:3], codes, scales, table, _dev([keys]), _dev([0, n]), masks[:3].clone(), most_new=1, return_lse=True)[1]
    assert float((few - lse[:3]).abs().max()) <= 2.0 ** -18 * (1 + float(few.abs().max()))


@pytest.mark.parametrize("counts,h,hk,dim", [([40, 12], 32, 8, 64), ([30, 20], 8, 4, 128)])
def test_a_tree_wait_that_runs_out_is_reported(S, counts, h, hk, dim):
    """Every role's first wait gives up: the rows are NaN, the status says so, and the next call is whole again."""
    from sili__new_b200 import _cuda
    q, codes, scales, table, lens, starts, masks = _tree_case([700, 300], counts, h, hk, dim, 16, torch.bfloat16, dim)
    assert _own_kernel(torch.bfloat16, dim, h, hk, max(counts))

    def call():
        return S.tree_attention(q, codes, scales, table, lens, _dev(starts), masks, most_new=max(counts), return_lse=True)

    S.check_attention()
    want, want_lse = call()
    S.check_attention()
    try:
        _cuda.kv4_attention_wait_limit(polls=0)
        out, lse = call()
        torch.cuda.synchronize()
    finally:
        _cuda.kv4_attention_wait_limit()
    assert torch.isnan(out).all() and torch.isnan(lse).all()
    with pytest.raises(RuntimeError, match="gave up"):
        S.check_attention()
    S.check_attention()
    again, again_lse = call()
    S.check_attention()
    assert torch.equal(again, want) and torch.equal(again_lse, want_lse)
