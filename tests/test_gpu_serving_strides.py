"""Strides of axes of length one, which no address depends on."""
import pytest
import torch

from test_gpu_serving import DTYPES

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,h,hk", [(1, 4, 2), (5, 1, 1), (1, 1, 1)])
def test_strides_of_single_tokens_and_heads_do_not_count(dtype, tokens, h, hk):
    """One token's row of an odd width, and one head with an odd stride: the same results as of contiguous copies."""
    from sili__new_b200 import serving as S
    dim = 64
    g = torch.Generator(device="cuda").manual_seed(tokens + h)

    def odd(heads):
        x = torch.randn(tokens, heads, dim, generator=g, device="cuda").to(dtype)
        return x, torch.as_strided(x.clone(), x.shape, (x.stride(0) if tokens > 1 else 8191, dim if heads > 1 else 77, 1))

    (q, qs), (k, ks), (v, vs) = odd(h), odd(hk), odd(hk)
    cos, sin = S.rotary_table(64, 64)
    pos = torch.arange(tokens, device="cuda")
    slots = torch.arange(tokens, device="cuda")
    table = torch.arange(tokens, dtype=torch.int32, device="cuda")[:, None] * 0
    lens = torch.full((tokens,), tokens, dtype=torch.int32, device="cuda")
    got = []
    for a, b, c in ((q, k, v), (qs, ks, vs)):
        cache = S.KVCache4(1, 16, hk, dim)
        r = torch.as_strided(torch.empty_like(q), q.shape, a.stride())
        y = S.cache_append(b, c, cache.codes, cache.scales, slots, cos=cos, sin=sin, positions=pos, q=a, q_out=r)
        z, _ = S.rotary(a, None, cos, sin, pos)
        got.append((cache.codes, cache.scales, y, z, S.cache_attention(y, cache.codes, cache.scales, table, lens)))
    for x, y in zip(*got):
        assert torch.equal(x, y)
