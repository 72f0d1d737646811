"""The serving operators (page tables, rotary positions, 4-bit cache append
and read, attention over the cache) against plain restatements
(serving_ref.py).

Tolerances.  Integers, codes and scale bytes are equal.  Rotary: two products
and a sum rounded once each in fp32, so 2^-23 (|a| + |b|) (|cos|, |sin| <= 1
times the table's gain), then the output type's half unit.  Attention: with u
the output type's half unit (and t half of its smallest subnormal), w the half unit of the probabilities' type (2^-11
for 16-bit activations, 2^-21 for fp32, whose probabilities and queries are
kept in two halves), and e = 2^-20 * (largest scale * sum |q k|) the error of
a logit (exact products, fp32 sums of at most 256 terms): |out - ref| <= u
|ref| + t + (w + 4 e + 2^-19) * sum p |v| + 2^-33 sum |v| (a half's subnormals: probabilities are at least 2^8 at the
row's largest, so what a half cannot hold is below 2^-25 / 2^8 of it), |lse - ref| <= 2 e + 2^-19 * (1 +
|ref|)."""
import math

import numpy as np
import pytest
import torch

import serving_ref as R

pytestmark = pytest.mark.gpu
HALF_UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
SMALLEST = {torch.float32: 2.0 ** -150, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def S():
    from sili__new_b200 import serving
    return serving


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


# ── page tables ──────────────────────────────────────────────────────────────
def _tables_case(requests, most, page, seed, free, width=None, chunk=40):
    rng = np.random.default_rng(seed)
    cached = rng.integers(0, most + 1, requests).astype(np.int32)
    cached[rng.random(requests) < 0.2] = 0
    fresh = rng.integers(0, 3, requests).astype(np.int32)
    fresh[rng.random(requests) < 0.2] = rng.integers(1, chunk + 1)
    have = -(-cached.astype(np.int64) // page)
    if width is None:
        width = int((-(-(cached.astype(np.int64) + fresh) // page)).max(initial=0)) + 2
    n_pages = int(have.sum()) + free
    perm = rng.permutation(n_pages).astype(np.int32)
    table = np.full((requests, width), -1, np.int32)
    at = 0
    for r in range(requests):
        n = min(have[r], width)
        table[r, :n] = perm[at:at + n]
        at += n
    ring = np.full(max(n_pages, 1), -7, np.int32)
    taken = int(rng.integers(0, 10 * n_pages + 1))
    ring[(taken + np.arange(free)) % len(ring)] = perm[n_pages - free:]
    return cached, fresh, table, ring, np.array([taken, taken + free], np.int64)


@pytest.mark.parametrize("requests,most,page,free,width,short", [
    (0, 10, 16, 3, 4, 0), (1, 0, 16, 9, None, 0), (1, 31, 16, 9, None, 5), (37, 200, 16, 400, None, 0),
    (300, 1000, 64, 3000, None, 0), (300, 1000, 7, 20, None, 0), (300, 1000, 64, 900, 6, 0), (64, 50, 1, 4000, None, 17),
    (4096, 90, 16, 9000, None, 0), (4097, 90, 16, 9000, None, 0), (9001, 40, 32, 100, None, 1000)])
def test_page_tables(S, requests, most, page, free, width, short):
    cached, fresh, table, ring, pool = _tables_case(requests, most, page, requests + page, free, width)
    total = max(int(fresh.sum()) + 9 - short, 0)
    want = R.page_tables(cached, fresh, table, ring, pool, page, total)
    dev = [torch.from_numpy(a).cuda() for a in (cached, fresh, table, ring, pool)]
    for _ in range(2):      # the same inputs again write the same values
        p = S.page_tables(*dev, page, total)
        got = dict(table=dev[2], starts=p.starts, lens=p.lens, slots=p.slots, positions=p.positions, pool=p.pool,
                   status=p.status)
        for name, w in want.items():
            np.testing.assert_array_equal(got[name].cpu().numpy(), w, err_msg=name)


def test_page_tables_negative_lengths_and_strided_table(S):
    cached = torch.tensor([-5, 16, 3], dtype=torch.int32, device="cuda")
    fresh = torch.tensor([2, -1, 14], dtype=torch.int32, device="cuda")
    wide = torch.full((3, 9), -1, dtype=torch.int32, device="cuda")
    wide[1, 0], wide[2, 0] = 5, 6
    ring, pool = S.page_pool(4)
    p = S.page_tables(cached, fresh, wide[:, :4], ring, pool, 16, 16)
    assert p.starts.tolist() == [0, 2, 2, 16] and p.lens.tolist() == [2, 16, 17]
    assert wide.tolist() == [[0] + [-1] * 8, [5] + [-1] * 8, [6, 1] + [-1] * 7]
    assert p.slots.tolist() == [0, 1] + [6 * 16 + i for i in range(3, 16)] + [16]
    assert p.pool.tolist() == [2, 4] and p.status.tolist() == [0, 0, 0]


def test_pages_go_round(S):
    """Many steps of admissions, growth and release: no page is ever held twice."""
    rng = np.random.default_rng(3)
    n, page, pages = 23, 16, 90
    ring, pool = S.page_pool(pages)
    table = torch.full((n, 12), -1, dtype=torch.int32, device="cuda")
    lens = torch.zeros(n, dtype=torch.int32, device="cuda")
    for step in range(60):
        fresh = torch.from_numpy(rng.integers(0, 9, n).astype(np.int32)).cuda()
        fresh = torch.minimum(fresh, 12 * page - lens)
        p = S.page_tables(lens, fresh, table, ring, pool, page, 256)
        assert p.status.tolist() == [0, 0, 0]
        pool, lens = p.pool, p.lens
        held = table[table >= 0].tolist()
        assert len(set(held)) == len(held) == int(pool[0] - pool[1]) + pages
        assert len(held) == int(((lens + page - 1) // page).sum())
        done = torch.from_numpy(rng.random(n) < 0.3).cuda() | (lens > 150)
        pool = S.release_pages(done, lens, table, ring, pool, page)
        assert int((lens[done] != 0).sum()) == 0 and int((table[done] >= 0).sum()) == 0


def test_release_passes_over_lacking_pages(S):
    ring = torch.arange(8, dtype=torch.int32, device="cuda")
    pool = torch.tensor([7, 8], dtype=torch.int64, device="cuda")
    table = torch.tensor([[3, -1, 4], [5, 6, -1]], dtype=torch.int32, device="cuda")
    lens = torch.tensor([40, 20], dtype=torch.int32, device="cuda")
    out = S.release_pages(torch.tensor([True, False], device="cuda"), lens, table, ring, pool, 16)
    assert out.tolist() == [7, 10] and ring.tolist()[:2] == [3, 4]
    assert table.tolist() == [[-1, -1, -1], [5, 6, -1]] and lens.tolist() == [0, 20]


# ── rotary ───────────────────────────────────────────────────────────────────
def test_rotary_table(S):
    for scaling in (None, {"type": "linear", "factor": 4.0}, {"type": "base", "factor": 8.0},
                    {"type": "yarn", "factor": 16.0, "original": 4096},
                    {"type": "wavelength", "factor": 8.0, "original": 8192}):
        inv, gain = S.rotary_frequencies(64, 10000.0, scaling)
        cos, sin = S.rotary_table(70001, 64, scaling=scaling)
        at = np.array([0, 1, 2, 777, 70000])
        ang = at[:, None] * inv[None, :]
        # a double angle, cosine and sine, rounded once to fp32
        np.testing.assert_allclose(cos[at].cpu().double().numpy(), np.cos(ang) * np.float32(gain), rtol=0, atol=2e-7 * gain)
        np.testing.assert_allclose(sin[at].cpu().double().numpy(), np.sin(ang) * np.float32(gain), rtol=0, atol=2e-7 * gain)


def _rotary_bound(x, dtype):
    m = np.abs(x)
    return 2.0 ** -22 * (m + np.abs(x).max(-1, keepdims=True)) + HALF_UNIT[dtype] * 1.5 * (m + 1e-30)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("tokens,h,hk,dim,rot,offset", [
    (1, 1, 1, 2, 2, 0), (5, 3, 1, 64, 64, 0), (7, 32, 8, 128, 64, 0), (33, 4, 2, 80, 20, 0), (2, 5, 5, 100, 6, 1),
    (260, 6, 2, 256, 256, 0), (3, 40, 8, 128, 128, 3), (9, 2, 1, 48, 16, 0)])
def test_rotary(S, dtype, layout, tokens, h, hk, dim, rot, offset):
    g = _gen(tokens + dim)
    cos, sin = S.rotary_table(500, rot)
    # slices of one row, off a 16-byte boundary where offset says so
    rows = torch.randn(tokens, offset + (h + hk) * dim + 5, generator=g, device="cuda").to(dtype)
    q = rows[:, offset:offset + h * dim].view(tokens, h, dim)
    k = rows[:, offset + h * dim:offset + (h + hk) * dim].view(tokens, hk, dim)
    pos = torch.randint(0, 500, (tokens,), generator=g, device="cuda", dtype=torch.int32)
    got = S.rotary(q, k, cos, sin, pos, layout=layout)
    back = S.rotary_backward(q, k, cos, sin, pos.long(), layout=layout)
    c, s, p = cos.double().cpu().numpy(), sin.double().cpu().numpy(), pos.cpu().numpy()
    for sign, outs in ((1.0, got), (-1.0, back)):
        for x, o in zip((q, k), outs):
            x = x.double().cpu().numpy()
            want = R.turn(x, c, s, p, layout, sign)
            assert o.shape == x.shape and o.dtype == dtype
            assert (np.abs(o.double().cpu().numpy() - want) <= _rotary_bound(want, dtype)
                    + 2.0 ** -22 * np.abs(x).max(-1, keepdims=True)).all()
    # in place, k left out
    only = q.clone()
    o, none = S.rotary(only, None, cos, sin, pos, layout=layout, q_out=only)
    assert none is None and o is only and torch.equal(only, got[0])


def test_rotary_padding_and_past_the_table(S):
    cos, sin = S.rotary_table(8, 32)
    x = torch.randn(4, 2, 64, device="cuda")
    pos = torch.tensor([-1, 7, 8, 1 << 40], device="cuda")
    q, _ = S.rotary(x, None, cos, sin, pos)
    assert (q[0] == 0).all() and torch.isfinite(q[1]).all() and torch.isnan(q[2:]).all()
    assert S.rotary(x[:0], None, cos, sin, pos[:0])[0].shape == (0, 2, 64)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rotary_gradient(S, layout):
    """autograd = the formula's transpose, and = differences (the operator is
    linear, so a difference is exact to its rounding)."""
    g = _gen(5)
    cos, sin = S.rotary_table(64, 32)
    pos = torch.randint(0, 64, (6,), generator=g, device="cuda")
    q = torch.randn(6, 3, 64, generator=g, device="cuda", requires_grad=True)
    k = torch.randn(6, 1, 64, generator=g, device="cuda", requires_grad=True)
    wq, wk = torch.randn(6, 3, 64, generator=g, device="cuda"), torch.randn(6, 1, 64, generator=g, device="cuda")
    a, b = S.rotary(q, k, cos, sin, pos, layout=layout)
    ((a * wq).sum() + (b * wk).sum()).backward()
    c, s, p = cos.double().cpu().numpy(), sin.double().cpu().numpy(), pos.cpu().numpy()
    for x, w in ((q, wq), (k, wk)):
        want = R.turn(w.double().cpu().numpy(), c, s, p, layout, -1.0)
        assert (np.abs(x.grad.double().cpu().numpy() - want) <= 2.0 ** -21 * (np.abs(want).max() + 1)).all()
    for e in (0, 5, 16, 31, 40):
        d = torch.zeros_like(q)
        d[2, 1, e] = 1.0
        with torch.no_grad():
            up = S.rotary(q + d, None, cos, sin, pos, layout=layout)[0]
            dn = S.rotary(q - d, None, cos, sin, pos, layout=layout)[0]
        diff = float(((up - dn).double() * wq.double()).sum() / 2)
        assert abs(diff - float(q.grad[2, 1, e])) <= 2.0 ** -19 * 64
    # only one of the two outputs used
    q.grad = None
    S.rotary(q, k, cos, sin, pos, layout=layout)[0].sum().backward()
    assert q.grad is not None


# ── the cache ────────────────────────────────────────────────────────────────
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("tokens,h,hk,dim,rot,page", [
    (1, 4, 1, 64, 64, 16), (3, 8, 2, 128, 128, 16), (70, 6, 3, 128, 32, 48), (19, 4, 4, 256, 128, 64),
    (5, 2, 1, 64, 16, 5), (2, 1, 1, 256, 0, 16)])
def test_append_and_read(S, dtype, layout, tokens, h, hk, dim, rot, page):
    g = _gen(tokens * dim + rot)
    x = torch.randn(tokens, (h + 2 * hk) * dim, generator=g, device="cuda")
    x *= torch.exp(2 * torch.randn(tokens, 1, generator=g, device="cuda"))
    x = x.to(dtype)
    q, k, v = (x[:, a * dim:b * dim].view(tokens, b - a, dim) for a, b in ((0, h), (h, h + hk), (h + hk, h + 2 * hk)))
    n_pages = -(-2 * tokens // page)
    slots = torch.randperm(n_pages * page, generator=g, device="cuda")[:tokens]
    slots[tokens // 2:tokens // 2 + 1] = -1 if tokens > 1 else slots[:1]
    codes = torch.full((n_pages, 2, hk, page, dim // 2), 0xA5, dtype=torch.uint8, device="cuda")
    scales = torch.full((n_pages, 2, hk, page, dim // 32), 0x5A, dtype=torch.uint8, device="cuda")
    want_c, want_s = codes.cpu().numpy(), scales.cpu().numpy()
    kr = k.float().cpu().numpy()
    if rot:
        cos, sin = S.rotary_table(300, rot)
        pos = torch.randint(0, 300, (tokens,), generator=g, device="cuda", dtype=torch.int32)
        qo = S.cache_append(k, v, codes, scales, slots, cos=cos, sin=sin, positions=pos, layout=layout, q=q)
        assert torch.equal(qo, S.rotary(q, None, cos, sin, pos, layout=layout)[0])
        kr = R.turn(kr, cos.cpu().numpy(), sin.cpu().numpy(), pos.cpu().numpy(), layout)
    else:
        assert S.cache_append(k, v, codes, scales, slots) is None
    for w, val in ((0, kr), (1, v.float().cpu().numpy())):
        c, b = R.quantise(val)
        for t, s in enumerate(slots.tolist()):
            if s >= 0:
                want_c[s // page, w, :, s % page], want_s[s // page, w, :, s % page] = c[t], b[t]
    np.testing.assert_array_equal(scales.cpu().numpy(), want_s)
    np.testing.assert_array_equal(codes.cpu().numpy(), want_c)
    for dt in DTYPES:
        kk, vv = S.cache_read(codes, scales, slots, dtype=dt)
        for w, o in ((0, kk), (1, vv)):
            for t, s in enumerate(slots.tolist()):
                want = R.values(want_c[s // page, w, :, s % page], want_s[s // page, w, :, s % page]) if s >= 0 else 0.0
                np.testing.assert_array_equal(o[t].double().cpu().numpy(), np.broadcast_to(want, (hk, dim)))


def test_append_extremes(S):
    """Zeros, tiny and huge groups, every rounding midpoint, infinities and NaN poison their group alone."""
    n = 64
    v = torch.zeros(n, 1, 64, device="cuda")
    v[1] = 1e-30
    v[2] = 3.0e38
    v[3, 0, :32] = torch.tensor([6.0] + [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.25, -0.75, -5.0, 0.2499999, -0.1]
                                + [0.0] * 19, device="cuda")
    v[4, 0, 3], v[5, 0, 40], v[6, 0, 0] = float("inf"), float("nan"), float("-inf")
    v[7] = 2.0 ** -17
    v[8:] = torch.exp2(torch.linspace(-30, 20, n - 8, device="cuda"))[:, None, None] * torch.randn(
        n - 8, 1, 64, generator=_gen(1), device="cuda")
    codes = torch.zeros(4, 2, 1, 16, 32, dtype=torch.uint8, device="cuda")
    scales = torch.zeros(4, 2, 1, 16, 2, dtype=torch.uint8, device="cuda")
    slots = torch.arange(n, device="cuda")
    S.cache_append(v, v, codes, scales, slots)
    c, b = R.quantise(v.cpu().numpy())
    for w in (0, 1):
        np.testing.assert_array_equal(scales[:, w, 0].reshape(n, 2).cpu().numpy(), b[:, 0])
        np.testing.assert_array_equal(codes[:, w, 0].reshape(n, 32).cpu().numpy(), c[:, 0])
    k, _ = S.cache_read(codes, scales, slots)
    bad = torch.isnan(k[:, 0])
    assert bad[4, :32].all() and bad[5, 32:].all() and bad[6, :32].all() and int(bad.sum()) == 96
    # slots past the cache are passed over
    before = codes.clone()
    S.cache_append(v[:3] + 1, v[:3] + 1, codes, scales, torch.tensor([64, -1, 1 << 40], device="cuda"))
    assert torch.equal(before, codes)
    assert (S.cache_read(codes, scales, torch.tensor([64, -9], device="cuda"))[0] == 0).all()


def test_codes_are_the_layers_codes(S):
    """A group with scale 1 holds fp4_quantize_array's codes."""
    import sili__new_b200 as pkg
    x = torch.randn(1, 1, 64, generator=_gen(2), device="cuda").clamp(-5.9, 5.9)
    x[0, 0, 0] = x[0, 0, 32] = 6.0
    codes = torch.zeros(1, 2, 1, 16, 32, dtype=torch.uint8, device="cuda")
    scales = torch.zeros(1, 2, 1, 16, 2, dtype=torch.uint8, device="cuda")
    S.cache_append(x, x, codes, scales, torch.zeros(1, dtype=torch.int64, device="cuda"))
    got = codes[0, 0, 0, 0].cpu().numpy()
    want = np.asarray(pkg.fp4_quantize_array(x.cpu().numpy().reshape(-1))).reshape(-1)
    np.testing.assert_array_equal(np.stack([got & 15, got >> 4], -1).reshape(-1), want)


# ── attention ────────────────────────────────────────────────────────────────
def _attend_case(lens, new, h, hk, dim, page, dtype, seed, extra_rows=0, spare_width=0, scale_q=1.5):
    g = _gen(seed)
    lens = np.asarray(lens)
    used = -(-np.maximum(lens, 0) // page)
    n_pages = int(used.sum()) + 3
    codes, scales = R.random_cache(n_pages, hk, page, dim, g)
    width = int(used.max(initial=0)) + spare_width
    table = torch.full((len(lens), max(width, 1)), 1 << 30, dtype=torch.int32, device="cuda")
    perm = torch.randperm(n_pages, generator=g, device="cuda").int()
    at = 0
    for r, u in enumerate(used):
        table[r, :u] = perm[at:at + u]
        # keys past the end: NaN scales in the last page's unused rows
        if lens[r] % page:
            scales[perm[at + u - 1].long(), :, :, lens[r] % page:] = 0xFF
        at += u
    starts = np.concatenate([[0], np.cumsum(new)])
    tokens = int(starts[-1]) + extra_rows
    q = (torch.randn(tokens, h, dim + 8, generator=g, device="cuda") * scale_q).to(dtype)[..., :dim]
    return q, codes, scales, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), starts


def _check_attention(S, case, dtype, window=0, scale=None, decode=False, most_new=None):
    q, codes, scales, table, lens, starts = case
    d = q.shape[2]
    sc = 1 / math.sqrt(d) if scale is None else scale
    out, lse = S.cache_attention(q, codes, scales, table, lens,
                                 starts=None if decode else torch.tensor(starts, dtype=torch.int32, device="cuda"),
                                 most_new=most_new, scale=scale, window=window, return_lse=True)
    ref, ref_lse, spread, size, total = R.attention(q, codes, scales, table, lens.cpu().numpy(), starts, sc, window, q.shape[0])
    out, lse = out.double().cpu().numpy(), lse.double().cpu().numpy()
    w = 2.0 ** -21 if dtype == torch.float32 else 2.0 ** -11
    e = 2.0 ** -20 * size
    empty = np.isinf(ref_lse)
    assert (np.isinf(lse) == empty).all() and (out[empty] == 0).all()
    ok = ~empty
    assert (np.abs(lse - ref_lse)[ok] <= (2 * e + 2.0 ** -19 * (1 + np.abs(ref_lse)))[ok]).all()
    bound = HALF_UNIT[dtype] * np.abs(ref) + SMALLEST[dtype] + (w + 4 * e[..., None] + 2.0 ** -19) * spread + 2.0 ** -33 * total
    worst = (np.abs(out - ref) / np.maximum(bound, 1e-30))[ok].max(initial=0.0)
    assert worst <= 1.0, worst


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens,h,hk,dim,page", [
    ([1], 1, 1, 64, 16), ([0, 1, 15, 16, 17], 4, 2, 128, 16), ([700, 3, 0, 64, 65, 128], 8, 2, 128, 16),
    ([333, 48, 49], 3, 3, 256, 48), ([5000, 1, 260], 16, 2, 64, 64), ([1030], 32, 8, 128, 128),
    ([77, 200], 20, 1, 128, 32), ([300, 5], 40, 1, 64, 16)])
def test_attention_decode(S, dtype, lens, h, hk, dim, page):
    case = _attend_case(lens, [1] * len(lens), h, hk, dim, page, dtype, sum(lens) + dim, spare_width=2)
    _check_attention(S, case, dtype, decode=True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens,new,h,hk,dim,page,window", [
    ([1], [1], 2, 1, 64, 16, 0), ([40, 130, 7], [3, 1, 7], 4, 2, 128, 16, 0), ([150, 0, 65], [130, 0, 64], 4, 1, 64, 16, 0),
    ([90, 33], [90, 2], 3, 3, 256, 32, 20), ([300, 64, 129], [20, 1, 129], 8, 2, 128, 48, 1),
    ([260], [260], 6, 2, 128, 64, 100), ([520, 300], [200, 300], 4, 2, 128, 16, 0)])
def test_attention_prompt(S, dtype, lens, new, h, hk, dim, page, window):
    case = _attend_case(lens, new, h, hk, dim, page, dtype, sum(lens) + window)
    _check_attention(S, case, dtype, window=window)
    _check_attention(S, case, dtype, window=window, most_new=1)     # a wrong hint changes nothing


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lens,new,h,hk,dim,page,window", [
    ([700, 130, 20], [500, 100, 20], 32, 8, 128, 16, 0), ([641, 0, 300], [641, 0, 300], 28, 4, 64, 48, 0),
    ([900, 257], [500, 130], 32, 8, 128, 64, 70), ([260, 5, 400], [255, 5, 360], 32, 1, 128, 128, 0),
    ([300, 310], [300, 300], 40, 40, 64, 16, 129)])
def test_attention_long_prompt(S, dtype, lens, new, h, hk, dim, page, window):
    """Enough 16-bit rows for the tensor-memory kernel; odd groups, ragged ends, windows, queries before the keys."""
    case = _attend_case(lens, new, h, hk, dim, page, dtype, sum(lens) + window, extra_rows=3)
    assert case[0].shape[0] * h >= 74 * 256
    _check_attention(S, case, dtype, window=window)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_attention_long_prompt_edges(S, dtype):
    """Requests with fewer keys than queries, missing pages, NaN in K and V of single keys, large and negative scales."""
    case = _attend_case([300, 420, 200], [330, 300, 7], 32, 8, 128, 16, dtype, 21, scale_q=4.0)
    q, codes, scales, table, lens, starts = case
    table[1, 3], table[1, 20] = -1, 1 << 29
    _check_attention(S, case, dtype)
    _check_attention(S, case, dtype, scale=-0.05)
    _check_attention(S, case, dtype, scale=0.0)
    starts32 = torch.tensor(starts, dtype=torch.int32, device="cuda")
    clean = S.cache_attention(q, codes, scales, table, lens, starts=starts32)
    # V of request 1's key 250, kv head 3, values 64..95: seen by queries at positions >= 250 (row 330 + 130 on)
    scales[table[1, 15].long(), 1, 3, 10, 2] = 0xFF
    got = S.cache_attention(q, codes, scales, table, lens, starts=starts32)
    bad = torch.isnan(got)
    want = torch.zeros_like(bad)
    want[330 + 130:630, 12:16, 64:96] = True
    assert torch.equal(bad, want) and torch.equal(got[~bad], clean[~bad])
    # K of the same key: its readers' rows are NaN as a whole, no other row changes
    scales[table[1, 15].long(), 0, 3, 10, 0] = 0xFF
    got = S.cache_attention(q, codes, scales, table, lens, starts=starts32)
    want[330 + 130:630, 12:16] = True
    assert torch.equal(torch.isnan(got), want) and torch.equal(got[~want], clean[~want])


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_window_decode(S, dtype):
    case = _attend_case([900, 30, 64, 1], [1] * 4, 8, 2, 128, 16, dtype, 11)
    for window in (1, 16, 33, 5000):
        _check_attention(S, case, dtype, window=window, decode=True)


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_rows_that_see_nothing(S, dtype):
    """Requests with fewer keys than queries (their first queries see none),
    rows past the last request, pages that are not there, no requests."""
    case = _attend_case([3, 70, 40], [6, 2, 40], 4, 2, 128, 16, dtype, 12, extra_rows=5)
    case[3][1, 1:3] = -1
    case[3][2, :] = -1
    _check_attention(S, case, dtype)
    q, codes, scales, table, lens, _ = case
    out = S.cache_attention(q, codes, scales, table[:0], lens[:0], starts=torch.zeros(1, dtype=torch.int32, device="cuda"))
    assert (out == 0).all()
    empty = S.cache_attention(q[:0], codes, scales, table[:0], lens[:0])
    assert empty.shape == (0, 4, 128)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", [1e-4, 30.0, 3000.0])
def test_attention_query_sizes(S, dtype, size):
    """Flat to one-hot softmaxes; queries far from 1 in both directions."""
    case = _attend_case([400, 90], [1, 1], 4, 2, 128, 16, dtype, 13, scale_q=size)
    _check_attention(S, case, dtype, decode=True)
    case = _attend_case([200], [70], 4, 2, 128, 16, dtype, 14, scale_q=size)
    _check_attention(S, case, dtype)
    _check_attention(S, case, dtype, scale=-0.3 / size)


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_nan_reaches_its_readers_only(S, dtype):
    case = _attend_case([100, 100], [1, 1], 4, 2, 128, 16, dtype, 15)
    q, codes, scales, table, lens, starts = case
    scales[table[0, 2].long(), 1, 0, 5, 1] = 0xFF       # V of request 0, kv head 0, token 37, values 32..63
    out = S.cache_attention(q, codes, scales, table, lens)
    bad = torch.isnan(out)
    assert bad[0, :2, 32:64].all() and int(bad.sum()) == 64


def test_attention_is_deterministic_across_streams_and_graphs(S):
    case = _attend_case([4000, 900, 17], [1] * 3, 32, 8, 128, 16, torch.bfloat16, 16)
    q, codes, scales, table, lens, _ = case
    first = S.cache_attention(q, codes, scales, table, lens)
    for _ in range(3):
        assert torch.equal(first, S.cache_attention(q, codes, scales, table, lens))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        other = S.cache_attention(q, codes, scales, table, lens)
    side.synchronize()
    assert torch.equal(first, other)
    graph = torch.cuda.CUDAGraph()
    out = torch.empty_like(first)
    with torch.cuda.graph(graph):
        S.cache_attention(q, codes, scales, table, lens, out=out)
    for _ in range(2):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(first, out)
    # the lengths are read on the device: a replay follows them
    lens.copy_(torch.tensor([100, 1, 900], dtype=torch.int32))
    table[2, :] = table[0, :]
    graph.replay()
    assert torch.equal(out, S.cache_attention(q, codes, scales, table, lens))


def test_long_cache_offsets_pass_32_bits(S):
    """Pages whose code bytes lie past 4 GB."""
    n_pages, page, hk, dim = 4500, 1024, 8, 128        # 2.4 GB each of K and V codes
    codes = torch.zeros(n_pages, 2, hk, page, dim // 2, dtype=torch.uint8, device="cuda")
    scales = torch.zeros(n_pages, 2, hk, page, dim // 32, dtype=torch.uint8, device="cuda")
    g = _gen(20)
    assert codes.numel() > 1 << 32
    k = torch.randn(40, hk, dim, generator=g, device="cuda")
    slots = torch.arange(40, device="cuda") + (n_pages - 1) * page
    S.cache_append(k, k, codes, scales, slots)
    kk, _ = S.cache_read(codes, scales, slots)
    assert float((kk - k).abs().max()) < 1.0 and float(kk.abs().max()) > 1
    table = torch.full((1, 1), n_pages - 1, dtype=torch.int32, device="cuda")
    lens = torch.tensor([40], dtype=torch.int32, device="cuda")
    q = torch.randn(1, 8, dim, generator=g, device="cuda")
    got = S.cache_attention(q, codes, scales, table, lens)
    small = codes[-1:].clone(), scales[-1:].clone()
    table.zero_()
    assert torch.equal(got, S.cache_attention(q, *small, table, lens))


# ── refusals ─────────────────────────────────────────────────────────────────
def test_refusals(S):
    cos, sin = S.rotary_table(16, 32)
    pos = torch.zeros(2, dtype=torch.int32, device="cuda")
    c = S.KVCache4(2, 16, 2, 64)
    x = torch.randn(2, 2, 64, device="cuda")
    slots = torch.zeros(2, dtype=torch.int64, device="cuda")
    lens = torch.ones(2, dtype=torch.int32, device="cuda")
    table = torch.zeros(2, 2, dtype=torch.int32, device="cuda")
    ring, pool = S.page_pool(4)
    for bad in (lambda: S.rotary(x.double(), None, cos, sin, pos),
                lambda: S.rotary(x, None, cos, sin, pos[:1]),
                lambda: S.rotary(x, None, cos, sin, pos.float()),
                lambda: S.rotary(x, None, cos, sin, pos, layout="pairs"),
                lambda: S.rotary(x[..., :16], None, cos, sin, pos),
                lambda: S.rotary(x.transpose(1, 2), None, cos, sin, pos),
                lambda: S.rotary(x, x.half(), cos, sin, pos),
                lambda: S.rotary(x, None, cos.cpu(), sin.cpu(), pos),
                lambda: S.rotary(x, None, cos, sin, pos, q_out=x[:, :1]),
                lambda: S.cache_append(x, x[:1], c.codes, c.scales, slots),
                lambda: S.cache_append(x[:, :1], x[:, :1], c.codes, c.scales, slots),
                lambda: S.cache_append(x, x, c.codes, c.scales, slots.int()),
                lambda: S.cache_append(x, x, c.codes, c.scales, slots, cos=cos),
                lambda: S.cache_append(x, x, c.codes, c.scales, slots, q=x),
                lambda: S.cache_append(x, x, c.codes.int(), c.scales, slots),
                lambda: S.cache_append(x, x, c.codes, c.scales[..., :1], slots),
                lambda: S.cache_append(x, x, c.codes, c.scales, slots, cos=cos[:, :4].contiguous(),
                                       sin=sin[:, :4].contiguous(), positions=pos),
                lambda: S.cache_read(c.codes, c.scales, slots, dtype=torch.float64),
                lambda: S.cache_attention(x.double(), c.codes, c.scales, table, lens),
                lambda: S.cache_attention(x[:, :1], c.codes, c.scales, table, lens),
                lambda: S.cache_attention(x, c.codes, c.scales, table.long(), lens),
                lambda: S.cache_attention(x, c.codes, c.scales, table[:1], lens),
                lambda: S.cache_attention(x[:1], c.codes, c.scales, table, lens),
                lambda: S.cache_attention(x, c.codes, c.scales, table, lens, window=-1),
                lambda: S.cache_attention(x, c.codes, c.scales, table, lens, starts=lens),
                lambda: S.cache_attention(x.cpu(), c.codes, c.scales, table, lens),
                lambda: S.page_tables(lens.long(), lens, table, ring, pool, 16, 4),
                lambda: S.page_tables(lens, lens, table, ring, pool, 0, 4),
                lambda: S.page_tables(lens, lens, table, ring, pool, 16, -1),
                lambda: S.page_tables(lens, lens, table[:, :1].expand(2, 2), ring, pool, 16, 4),
                lambda: S.release_pages(lens, lens, table, ring, pool, 16),
                lambda: S.KVCache4(2, 20, 2, 64),
                lambda: S.KVCache4(2, 16, 2, 96)):
        with pytest.raises(ValueError):
            bad()
    cache8 = torch.zeros(2, 2, 2, 8, 32, dtype=torch.uint8, device="cuda")
    with pytest.raises(ValueError):     # pages of 8 can be written and read, not attended over
        S.cache_attention(x, cache8, torch.zeros(2, 2, 2, 8, 2, dtype=torch.uint8, device="cuda"), table, lens)
    # the C entries refuse by themselves
    from sili__new_b200 import _cuda
    with pytest.raises(ValueError):
        _cuda.rotary_ptr(0, 0, 1, 1, 0, 1, 1, 1, 0, 0, 0, 0, 0, 0, 0, 1, 64, 32, cos.data_ptr(), sin.data_ptr(), 16,
                         pos.data_ptr(), False, False, False, 0)
    with pytest.raises(ValueError):
        _cuda.kv4_attention_ptr(0, x.data_ptr(), 128, 64, 2, 2, 96, c.codes.data_ptr(), c.scales.data_ptr(), 2, 16, 2,
                                table.data_ptr(), 2, 2, lens.data_ptr(), 2, 0, 1, 1.0, 0, x.data_ptr(), 0, 0, 0)


def test_served_block_example(S):
    """The example's prompts, decoding, release and reuse over folded sparse projections (fp32 throughout)."""
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "serve_folded_attention.py")
    spec = importlib.util.spec_from_file_location("serve_folded_attention", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    block, worst = mod.main(["--check", "--decode", "8"])
    assert block.lens.tolist() == [37 + 9, 30 + 4, 0, 64 + 9]
    held = block.table[block.table >= 0].tolist()
    assert len(held) == len(set(held)) == sum(-(-n // 16) for n in block.lens.tolist())
    assert worst <= 2e-6        # fp32: a few units of 2^-24 in logits of size ~10 and in the sums


def test_rotary_wide_heads_off_alignment(S):
    """More pairs than a CTA of the aligned path has threads."""
    g = _gen(30)
    cos, sin = S.rotary_table(9, 1000)
    x = torch.randn(3, 2 * 1024 + 1, generator=g, device="cuda")[:, 1:].view(3, 2, 1024)
    pos = torch.tensor([0, 3, 8], device="cuda")
    for layout in ("half", "interleaved"):
        got = S.rotary(x, None, cos, sin, pos, layout=layout)[0]
        assert torch.equal(got, S.rotary(x.contiguous(), None, cos, sin, pos, layout=layout)[0])
    with pytest.raises(ValueError):
        S.rotary(torch.zeros(3, 1, 1026, device="cuda"), None, cos, sin, pos)


def test_check_attention_is_quiet(S):
    S.check_attention()


@pytest.mark.parametrize("dtype", DTYPES)
def test_append_turns_q_in_place(S, dtype):
    g = _gen(31)
    cos, sin = S.rotary_table(64, 128)
    pos = torch.randint(0, 64, (50,), generator=g, device="cuda")
    q = torch.randn(50, 41, 128, generator=g, device="cuda").to(dtype)
    k = torch.randn(50, 3, 128, generator=g, device="cuda").to(dtype)
    c = S.KVCache4(4, 16, 3, 128)
    slots = torch.arange(50, device="cuda")
    want = S.cache_append(k, k, c.codes, c.scales, slots, cos=cos, sin=sin, positions=pos, q=q)
    assert S.cache_append(k, k, c.codes, c.scales, slots, cos=cos, sin=sin, positions=pos, q=q, q_out=q) is q
    assert torch.equal(q, want)


def test_attention_without_a_hint(S):
    """most_new left out: the mean number of queries picks the kernel, the result stays."""
    case = _attend_case([300, 40, 77], [40, 1, 1], 8, 2, 128, 16, torch.bfloat16, 32)
    _check_attention(S, case, torch.bfloat16)
    _check_attention(S, case, torch.bfloat16, most_new=40)
