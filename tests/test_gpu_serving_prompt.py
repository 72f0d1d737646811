"""The long-prompt attention kernel at the masks, scales and pages where it can
go wrong.  Every case asks the library whether it runs there; bounds as in
test_gpu_serving.py."""
import numpy as np
import pytest
import torch

from test_gpu_serving import _attend_case, _check_attention

pytestmark = pytest.mark.gpu
HALVES = [torch.float16, torch.bfloat16]


def _case(lens, new, h, hk, dim, page, dtype, seed, **more):
    from sili__new_b200 import _cuda
    case = _attend_case(lens, new, h, hk, dim, page, dtype, seed, **more)
    q = case[0]
    hint = -(-q.shape[0] // len(lens))        # what a call without most_new goes by
    code = {torch.float16: 1, torch.bfloat16: 2}[dtype]
    assert _cuda.kv4_attention_long_prompt(code, dim, q.shape[0], h, hk, hint)
    return case


def _attend(case, **more):
    from sili__new_b200 import serving
    q, codes, scales, table, lens, starts = case
    return serving.cache_attention(q, codes, scales, table, lens,
                                   starts=torch.tensor(starts, dtype=torch.int32, device="cuda"), **more)


def test_which_kernel():
    from sili__new_b200 import _cuda
    takes = _cuda.kv4_attention_long_prompt
    assert takes(2, 128, 1 << 20, 32, 8, 1 << 20) and takes(1, 64, 1 << 20, 8, 8, 1 << 20)
    assert not takes(0, 128, 1 << 20, 32, 8, 1 << 20)         # fp32
    assert not takes(2, 256, 1 << 20, 32, 8, 1 << 20)
    assert not takes(2, 128, 1 << 20, 32, 8, 1)               # one query a request
    assert not takes(2, 128, 8, 32, 8, 8)                     # few rows
    for bad in ((2, 128, -1, 32, 8, 1), (2, 128, 1, 32, 5, 1), (2, 128, 1, 0, 1, 1), (2, 128, 1, 32, 8, -1)):
        with pytest.raises(ValueError):
            takes(*bad)


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("lens,new,h,hk,dim,page,window", [
    ([800, 130, 20], [620, 100, 20], 32, 8, 128, 16, 0), ([900, 357], [500, 230], 32, 8, 128, 64, 70),
    ([700, 65], [640, 64], 32, 8, 128, 48, 1), ([1300], [641], 32, 8, 128, 128, 129), ([1800], [1216], 16, 4, 128, 1024, 0),
    ([700, 300], [650, 300], 28, 4, 64, 48, 300), ([530, 540], [520, 530], 20, 20, 128, 16, 0),
    ([1400, 5], [1290, 5], 16, 16, 64, 32, 64)])
def test_lengths_windows_and_head_layouts(dtype, lens, new, h, hk, dim, page, window):
    _check_attention(_serving(), _case(lens, new, h, hk, dim, page, dtype, sum(lens) + window, extra_rows=3), dtype,
                     window=window)


def _serving():
    from sili__new_b200 import serving
    return serving


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("h,hk,dim", [(32, 8, 128), (28, 4, 64)])
def test_missing_pages_scales_and_rows_without_keys(dtype, h, hk, dim):
    """The first request has fewer keys than queries, the second misses pages inside and at its end, the third all."""
    case = _case([300, 430, 350], [390, 300, 300], h, hk, dim, 16, dtype, 21, scale_q=4.0)
    table = case[3]
    table[1, 3], table[1, 20], table[1, 26] = -1, 1 << 29, -7
    table[2, :] = -1
    for more in (dict(), dict(scale=-0.05), dict(scale=0.0), dict(window=40), dict(scale=2.5, window=17)):
        _check_attention(_serving(), case, dtype, **more)


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("h,hk,dim,page", [(32, 8, 128, 16), (28, 4, 64, 32)])
@pytest.mark.parametrize("window", [0, 90])
def test_a_scale_that_is_no_number_reaches_its_readers_only(dtype, h, hk, dim, page, window):
    """NaN in V reaches one group of 32 values of the queries that see its key, in K their whole rows, and nothing else
    changes by a bit."""
    group = h // hk
    case = _case([300, 420, 200], [400, 300, 200], h, hk, dim, page, dtype, 22)
    scales, table = case[2], case[3]
    clean = _attend(case, window=window)
    assert not torch.isnan(clean).any()
    want = torch.zeros_like(clean, dtype=torch.bool)

    def spoil(request, key, head, kv, part):
        """NaN into (K or V) part of one key of one kv head; `want` marks who sees it."""
        scales[table[request, key // page].long(), kv, head, key % page, part] = 0xFF
        n, length, first = (400, 300, 0), (300, 420, 400), (200, 200, 700)
        n, length, first = (n, length, first)[request]
        for i in range(n):
            pos = length - n + i
            if key <= pos and (not window or key > pos - window):
                at = slice(32 * part, 32 * part + 32) if kv else slice(None)
                want[first + i, head * group:(head + 1) * group, at] = True

    for at in ((1, 250, hk - 1, 1, dim // 32 - 1), (1, 251, hk - 1, 1, 0), (0, 0, 0, 1, 1), (2, 199, 1, 1, 0), (2, 64, 2, 1, 1),
               (1, 127, 0, 1, 0), (1, 128, 0, 1, 1), (1, 250, 1, 0, 0), (2, 63, 0, 0, 1)):
        spoil(*at)
        got = _attend(case, window=window)
        assert torch.equal(torch.isnan(got), want), at
        assert torch.equal(got[~want], clean[~want]), at


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("size", [1e-4, 30.0, 3000.0])
def test_query_sizes(dtype, size):
    """Flat to one-hot softmaxes: the running maximum stays, or moves often."""
    case = _case([900], [700], 32, 8, 128, 32, dtype, 23, scale_q=size)
    _check_attention(_serving(), case, dtype)
    _check_attention(_serving(), case, dtype, scale=-0.3 / size)


def test_repeats_streams_and_graphs():
    case = _case([900, 300], [640, 100], 32, 8, 128, 16, torch.bfloat16, 24)
    first, lse = _attend(case, return_lse=True)
    again, lse2 = _attend(case, return_lse=True)
    assert torch.equal(first, again) and torch.equal(lse, lse2)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        other = _attend(case)
    side.synchronize()
    assert torch.equal(first, other)


@pytest.mark.parametrize("prompt", [True, False])
def test_a_whole_step_in_a_graph(prompt):
    """Tables, append and attention captured together; replays follow the lengths on the device."""
    from sili__new_b200 import _cuda, serving as S
    g = torch.Generator(device="cuda").manual_seed(25)
    h, hk, dim, page, rows = 32, 8, 128, 16, 704 if prompt else 8
    most = rows if prompt else 2
    assert _cuda.kv4_attention_long_prompt(2, dim, rows, h, hk, most) == prompt
    qkv = torch.randn(rows, (h + 2 * hk) * dim, generator=g, device="cuda").bfloat16()
    q, k, v = (x.view(rows, -1, dim) for x in qkv.split([h * dim, hk * dim, hk * dim], 1))
    cos, sin = S.rotary_table(4096, dim)

    class Step:
        def __init__(self):
            self.cache = S.KVCache4(200, page, hk, dim)
            self.ring, self.pool = S.page_pool(200)
            self.table = torch.full((3, 100), -1, dtype=torch.int32, device="cuda")
            self.lens, self.fresh = (torch.zeros(3, dtype=torch.int32, device="cuda") for _ in range(2))

        def __call__(self):
            c = self.cache
            t = S.page_tables(self.lens, self.fresh, self.table, self.ring, self.pool, page, rows)
            y = S.cache_append(k, v, c.codes, c.scales, t.slots, cos=cos, sin=sin, positions=t.positions, q=q)
            out = S.cache_attention(y, c.codes, c.scales, self.table, t.lens, starts=t.starts, most_new=most)
            self.lens.copy_(t.lens)
            self.pool.copy_(t.pool)
            return out

    eager, captured = Step(), Step()
    captured()                                  # (nothing is new: nothing changes)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = captured()
    for fresh in ((600, 4, 100), (0, 1, 300), (700, 0, 4)) if prompt else ((2, 1, 2), (1, 1, 1), (2, 0, 2)):
        for s in (eager, captured):
            s.fresh.copy_(torch.tensor(fresh, dtype=torch.int32))
        want = eager()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        assert torch.equal(captured.table, eager.table) and torch.equal(captured.lens, eager.lens)
        assert torch.equal(captured.cache.codes, eager.cache.codes) and torch.equal(captured.pool, eager.pool)
    assert np.array_equal(eager.lens.cpu().numpy(), np.array([1300, 5, 404] if prompt else [5, 2, 5]))
