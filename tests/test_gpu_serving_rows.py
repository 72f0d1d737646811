"""Attention over the 4-bit cache where a step brought more tokens than q has
rows: page tables keep counting the tokens beyond max_tokens, so the last
requests' rows are cut, and what is there keeps its positions."""
import math

import numpy as np
import pytest
import torch

import serving_ref as R
from test_gpu_serving import DTYPES, HALF_UNIT, SMALLEST, _attend_case

pytestmark = pytest.mark.gpu


def _check_cut(lens, new, rows, h, hk, dim, page, dtype, window, most_new=None):
    """The first `rows` rows of a case of sum(new) rows, against the whole case's in 64 bits; bounds as in
    test_gpu_serving.py."""
    from sili__new_b200 import serving
    q, codes, scales, table, lens_, starts = _attend_case(lens, new, h, hk, dim, page, dtype, sum(lens) + rows)
    scale = 1 / math.sqrt(dim)
    out, lse = serving.cache_attention(q[:rows], codes, scales, table, lens_,
                                       starts=torch.tensor(starts, dtype=torch.int32, device="cuda"),
                                       most_new=most_new, window=window, return_lse=True)
    ref, ref_lse, spread, size, total = (x[:rows] for x in R.attention(q, codes, scales, table, lens, starts, scale,
                                                                       window, q.shape[0]))
    out, lse = out.double().cpu().numpy(), lse.double().cpu().numpy()
    w = 2.0 ** -21 if dtype == torch.float32 else 2.0 ** -11
    e = 2.0 ** -20 * size
    empty = np.isinf(ref_lse)
    assert (np.isinf(lse) == empty).all() and (out[empty] == 0).all()
    ok = ~empty
    assert (np.abs(lse[ok] - ref_lse[ok]) <= (2 * e + 2.0 ** -19 * (1 + np.abs(ref_lse)))[ok]).all()
    bound = HALF_UNIT[dtype] * np.abs(ref) + SMALLEST[dtype] + (w + 4 * e[..., None] + 2.0 ** -19) * spread \
        + 2.0 ** -33 * total
    assert (np.abs(out - ref) <= np.maximum(bound, 1e-30))[ok].all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens,new,rows,h,hk,dim,page,window", [
    ([40, 130, 7], [3, 9, 7], 8, 4, 2, 128, 16, 0),          # the second is cut, the third has no row
    ([300], [200], 3, 4, 1, 64, 16, 0), ([90, 60], [90, 60], 100, 3, 3, 256, 32, 20),
    ([500, 33], [20, 30], 21, 8, 2, 128, 48, 1), ([5], [9], 6, 2, 1, 64, 16, 0)])
def test_cut_requests_keep_their_positions(dtype, lens, new, rows, h, hk, dim, page, window):
    _check_cut(lens, new, rows, h, hk, dim, page, dtype, window)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lens,new,rows,window", [
    ([500, 900, 30], [400, 500, 30], 700, 0), ([500, 900], [400, 500], 700, 100), ([1000], [1000], 641, 0)])
def test_cut_long_prompts_keep_their_positions(dtype, lens, new, rows, window):
    assert rows * 4 // 256 * 8 >= 74        # 16-bit rows enough for the long-prompt kernel
    _check_cut(lens, new, rows, 32, 8, 128, 16, dtype, window)


def test_a_step_with_more_tokens_than_rows():
    """Through the step's own calls: the rows that fit are the same as in a step that holds all tokens."""
    from sili__new_b200 import serving as S
    g = torch.Generator(device="cuda").manual_seed(3)
    fresh = torch.tensor([5, 20, 9], dtype=torch.int32, device="cuda")
    x = torch.randn(34, 4, 64, generator=g, device="cuda")
    outs = []
    for rows in (34, 17):
        cache = S.KVCache4(8, 16, 2, 64)
        ring, pool = S.page_pool(8)
        table = torch.full((3, 4), -1, dtype=torch.int32, device="cuda")
        cos, sin = S.rotary_table(64, 64)
        t = S.page_tables(torch.zeros_like(fresh), fresh, table, ring, pool, 16, rows)
        assert t.status.tolist() == [0, 34 - rows, 0]
        q = S.cache_append(x[:rows, :2], x[:rows, 2:], cache.codes, cache.scales, t.slots, cos=cos, sin=sin,
                           positions=t.positions, q=x[:rows])
        outs.append(S.cache_attention(q, cache.codes, cache.scales, table, t.lens, starts=t.starts))
    # (the cut moves the even split of the work, so sums may be joined in another order)
    assert float((outs[0][:17] - outs[1]).abs().max()) <= 1e-5 * float(outs[0].abs().max())
