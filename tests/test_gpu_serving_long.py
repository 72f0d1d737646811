"""Attention over long caches: the sums of hundreds of thousands of keys.

V is the same in every key, so the output is V whatever the probabilities are:
what it falls short by is the sums' own error.  |out - V| <= u |V| (the
output's half unit) + 2^-11 |V| (probabilities rounded to halves; their sum is
not) + 2^-19 |V| (fp32 sums), as in test_gpu_serving.py."""
import numpy as np
import pytest
import torch

import serving_ref as R

pytestmark = pytest.mark.gpu


def _one_v(keys, hk, d, seed, page=64):
    g = torch.Generator(device="cuda").manual_seed(seed)
    pages = -(-keys // page)
    codes = torch.randint(0, 256, (pages, 2, hk, page, d // 2), generator=g, device="cuda", dtype=torch.uint8)
    scales = torch.randint(90, 115, (pages, 2, hk, page, d // 32), generator=g, device="cuda", dtype=torch.uint8)
    value = torch.randint(88, 120, (hk, 1, d // 32), generator=g, device="cuda", dtype=torch.uint8)
    codes[:, 1], scales[:, 1] = 0x22, value                                  # 1 x the group's scale
    want = (value.int() << 7).short().view(torch.float16).double()[:, 0].repeat_interleave(32, -1)
    return codes, scales, want


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("keys,new,h,hk,d,window", [
    (262144, 704, 32, 8, 128, 0), (262131, 700, 28, 4, 64, 0), (65536, 1184, 32, 4, 64, 0), (40000, 704, 32, 8, 128, 0), (262144, 704, 32, 8, 128, 100000)])
def test_long_prompt_sums_hold(dtype, keys, new, h, hk, d, window):
    from sili__new_b200 import _cuda, serving as S
    assert _cuda.kv4_attention_long_prompt(1, d, new, h, hk, new)
    codes, scales, want = _one_v(keys, hk, d, keys)
    g = torch.Generator(device="cuda").manual_seed(1)
    table = torch.arange(codes.shape[0], dtype=torch.int32, device="cuda")[None]
    lens = torch.tensor([keys], dtype=torch.int32, device="cuda")
    starts = torch.tensor([0, new], dtype=torch.int32, device="cuda")
    q = (torch.randn(new, h, d, generator=g, device="cuda") * 0.3).to(dtype)
    out, lse = S.cache_attention(q, codes, scales, table, lens, starts=starts, most_new=new, window=window, return_lse=True)
    again = S.cache_attention(q, codes, scales, table, lens, starts=starts, most_new=new, window=window)
    S.check_attention()
    assert torch.equal(out, again)
    off = out.double().view(new, hk, h // hk, d) / want[None, :, None] - 1
    u = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[dtype]
    assert float(off.abs().max()) <= u + 2.0 ** -11 + 2.0 ** -19
    # most of that allowance is for roundings of either sign: their mean over many elements is none
    assert abs(float(off.mean())) <= 2.0 ** -12
    # the rows' own lse against the split kernel's (fp32 sums of the same probabilities in another order)
    few = S.cache_attention(q[-3:], codes, scales, table, lens, starts=torch.tensor([0, 3], dtype=torch.int32, device="cuda"),
                            most_new=3, window=window, return_lse=True)[1]
    assert float((few - lse[-3:]).abs().max()) <= 2.0 ** -18 * (1 + float(few.abs().max()))


def test_long_prompt_sums_move_with_the_maximum():
    """Keys whose logits grow along the cache, then fall: sums set aside stand over other maxima than the last."""
    from sili__new_b200 import _cuda, serving as S
    keys, new, h, hk, d, page = 20000, 9472, 2, 2, 64, 16
    g = torch.Generator(device="cuda").manual_seed(2)
    assert _cuda.kv4_attention_long_prompt(1, d, new, h, hk, new)
    codes, scales = R.random_cache(-(-keys // page), hk, page, d, g)
    codes[:, 0] = 0x22
    at = torch.arange(keys, device="cuda").view(-1, page)
    grow = 60 + 2 * ((at % 9000) // 180)                   # K: from 2^-7.4 up to 28, twice
    scales[:, 0] = grow[:, None, :, None].to(torch.uint8)
    table = torch.arange(codes.shape[0], dtype=torch.int32, device="cuda")[None]
    lens = torch.tensor([keys], dtype=torch.int32, device="cuda")
    q = torch.randn(new, h, d, generator=g, device="cuda").half()
    out, lse = S.cache_attention(q, codes, scales, table, lens, starts=torch.tensor([0, new], dtype=torch.int32, device="cuda"),
                                 most_new=new, return_lse=True)
    for row in (0, 1, 777, 4000, new - 1):
        n = keys - new + row + 1
        ref, ref_lse, spread, size, total = R.attention(q[row:row + 1], codes, scales, table, [n], [0, 1], d ** -0.5, 0, 1)
        e = 2.0 ** -20 * size
        bound = 2.0 ** -11 * np.abs(ref) + 2.0 ** -25 + (2.0 ** -11 + 4 * e[..., None] + 2.0 ** -19) * spread + 2.0 ** -33 * total
        assert (np.abs(out[row].double().cpu().numpy() - ref[0]) <= bound[0]).all()
        assert (np.abs(lse[row].double().cpu().numpy() - ref_lse[0]) <= 2 * e[0] + 2.0 ** -19 * (1 + np.abs(ref_lse[0]))).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("requests,h,hk,d", [(300, 1, 1, 128), (310, 12, 1, 64), (160, 20, 1, 128), (160, 4, 1, 256)])
def test_long_decode_sums_hold(dtype, requests, h, hk, d):
    """More segments than CTAs, of more keys than a warp's sums take in at once (the requests share their pages)."""
    from sili__new_b200 import serving as S
    keys = 1000001 if d == 128 and h == 1 else 300001
    codes, scales, want = _one_v(keys, hk, d, keys + h)
    g = torch.Generator(device="cuda").manual_seed(3)
    table = torch.arange(codes.shape[0], dtype=torch.int32, device="cuda").repeat(requests, 1)
    lens = torch.full((requests,), keys, dtype=torch.int32, device="cuda")
    lens[5], lens[77] = 0, 200000
    q = (torch.randn(requests, h, d, generator=g, device="cuda") * 0.3).to(dtype)
    out, lse = S.cache_attention(q, codes, scales, table, lens, return_lse=True)
    assert torch.equal(out, S.cache_attention(q, codes, scales, table, lens))
    assert (out[5] == 0).all() and torch.isinf(lse[5]).all()
    there = torch.arange(requests, device="cuda") != 5
    off = out.double()[there].view(-1, hk, h // hk, d) / want[None, :, None] - 1
    u = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}[dtype]
    w = 2.0 ** -21 if dtype == torch.float32 else 2.0 ** -11
    assert float(off.abs().max()) <= u + w + 2.0 ** -19
    assert abs(float(off.mean())) <= 2.0 ** -12
    # a request by itself is split over all CTAs, in other parts
    for r in (0, 77, requests - 1):
        one, one_lse = S.cache_attention(q[r:r + 1], codes, scales, table[r:r + 1], lens[r:r + 1], return_lse=True)
        assert float((one_lse - lse[r:r + 1]).abs().max()) <= 2.0 ** -18 * (1 + float(one_lse.abs().max()))
        assert float((one - out[r:r + 1]).abs().max()) <= (2 * u + 2.0 ** -19) * float(want.max())


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("h,d", [(1, 64), (9, 128)])
def test_long_decode_sums_move_with_the_maximum(dtype, h, d):
    from sili__new_b200 import serving as S
    keys, requests, page = 290000, 300, 80
    g = torch.Generator(device="cuda").manual_seed(4)
    codes, scales = R.random_cache(-(-keys // page), 1, page, d, g)
    codes[:, 0] = 0x22
    at = torch.arange(codes.shape[0], device="cuda")[:, None] * page + torch.arange(page, device="cuda")
    grow = 60 + 2 * ((at % 150000) // 3000)                # K: from 2^-7.4 up to 28, twice
    scales[:, 0] = grow[:, None, :, None].to(torch.uint8)
    table = torch.arange(codes.shape[0], dtype=torch.int32, device="cuda").repeat(requests, 1)
    lens = torch.full((requests,), keys, dtype=torch.int32, device="cuda")
    q = torch.randn(requests, h, d, generator=g, device="cuda").to(dtype)
    out, lse = S.cache_attention(q, codes, scales, table, lens, return_lse=True)
    for r in (0, 150, requests - 1):
        ref, ref_lse, spread, size, total = R.attention(q[r:r + 1], codes, scales, table[r:r + 1], [keys], [0, 1], d ** -0.5, 0, 1)
        e = 2.0 ** -20 * size
        u, w, least = (2.0 ** -24, 2.0 ** -21, 2.0 ** -150) if dtype == torch.float32 else (2.0 ** -11, 2.0 ** -11, 2.0 ** -25)
        bound = u * np.abs(ref) + least + (w + 4 * e[..., None] + 2.0 ** -19) * spread + 2.0 ** -33 * total
        assert (np.abs(out[r].double().cpu().numpy() - ref[0]) <= bound[0]).all()
        assert (np.abs(lse[r].double().cpu().numpy() - ref_lse[0]) <= 2 * e[0] + 2.0 ** -19 * (1 + np.abs(ref_lse[0]))).all()
