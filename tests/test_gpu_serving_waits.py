"""The long-prompt attention kernel's bounded waits: when one runs out, its
rows are NaN, the status says so, and the next call is whole again."""
import pytest
import torch

from test_gpu_serving import _attend_case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("limits", [dict(polls=0), dict(output_polls=0)])
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 32)])
def test_a_wait_that_runs_out_is_reported(limits, dim, page):
    """`polls`: every role's first wait gives up; `output_polls`: the softmax warps' last one alone, when the threads that
    issue the products may have left already."""
    from sili__new_b200 import _cuda, serving
    q, codes, scales, table, lens, starts = _attend_case([700, 300], [640, 260], 32, 8, dim, page, torch.bfloat16, dim)
    assert q.shape[0] * 4 // 256 * 8 >= 74       # rows enough for the long-prompt kernel
    starts = torch.tensor(starts, dtype=torch.int32, device="cuda")

    def call():
        return serving.cache_attention(q, codes, scales, table, lens, starts=starts, most_new=640, return_lse=True)

    serving.check_attention()
    want, want_lse = call()
    serving.check_attention()
    try:
        _cuda.kv4_attention_wait_limit(**limits)
        out, lse = call()
        torch.cuda.synchronize()
    finally:
        _cuda.kv4_attention_wait_limit()
    assert torch.isnan(out).all() and torch.isnan(lse).all()
    with pytest.raises(RuntimeError, match="gave up"):
        serving.check_attention()
    serving.check_attention()
    again, again_lse = call()
    serving.check_attention()
    assert torch.equal(again, want) and torch.equal(again_lse, want_lse)
