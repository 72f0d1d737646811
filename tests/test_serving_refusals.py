"""What the serving calls refuse before they look for a device (no GPU)."""
import pytest
import torch
from torch.autograd import forward_ad

from sili__new_b200 import serving as S


@pytest.fixture
def calls():
    """Each call by the name of the input that takes part in it, as a function of that input."""
    x = torch.zeros(2, 2, 64)
    cos, pos = torch.zeros(4, 16), torch.zeros(2, dtype=torch.int32)
    codes, scales = torch.zeros(2, 2, 2, 16, 32, dtype=torch.uint8), torch.zeros(2, 2, 2, 16, 2, dtype=torch.uint8)
    slots = torch.zeros(2, dtype=torch.int64)
    table, lens = torch.zeros(2, 2, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    turn = dict(cos=cos, sin=cos, positions=pos)
    return x, {"append k": lambda a: S.cache_append(a, x, codes, scales, slots),
               "append v": lambda a: S.cache_append(x, a, codes, scales, slots),
               "append q": lambda a: S.cache_append(x, x, codes, scales, slots, q=a, **turn),
               "attention q": lambda a: S.cache_attention(a, codes, scales, table, lens)}


@pytest.mark.parametrize("which", ["append k", "append v", "append q", "attention q"])
def test_a_gradient_that_would_be_lost_is_refused(calls, which):
    x, by_name = calls
    call = by_name[which]
    with pytest.raises(ValueError, match="no gradient"):
        call(x.clone().requires_grad_())
    with forward_ad.dual_level(), pytest.raises(ValueError, match="no gradient"):
        call(forward_ad.make_dual(x, torch.ones_like(x)))
    # not asked for: the call goes on (to the next refusal here)
    with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):
        call(x.clone().requires_grad_())
    with pytest.raises(ValueError, match="CUDA"):
        call(x)


def test_outputs_whose_rows_share_elements_are_refused():
    """Several rows would be written to one place, in no order."""
    x, cos, pos = torch.zeros(4, 3, 64), torch.zeros(4, 16), torch.zeros(4, dtype=torch.int32)
    codes, scales = torch.zeros(2, 2, 3, 16, 32, dtype=torch.uint8), torch.zeros(2, 2, 3, 16, 2, dtype=torch.uint8)
    slots = torch.zeros(4, dtype=torch.int64)
    turn = dict(cos=cos, sin=cos, positions=pos)
    flat = torch.zeros(4096)
    for strides in ((0, 64, 1), (192, 0, 1), (192, 32, 1), (64, 128, 1), (100, 64, 1), (64, 64, 1)):
        out = flat.as_strided(x.shape, strides)
        for call in (lambda o: S.rotary(x, None, cos, cos, pos, q_out=o), lambda o: S.rotary(x, x, cos, cos, pos, k_out=o),
                     lambda o: S.rotary_backward(x, x, cos, cos, pos, k_out=o),
                     lambda o: S.cache_append(x, x, codes, scales, slots, q=x, q_out=o, **turn)):
            with pytest.raises(ValueError, match="share elements"):
                call(out)
    # rows apart from one another, tokens or heads outermost, and axes of length one: on to the next refusal
    for shape, strides in ((x.shape, (192, 64, 1)), (x.shape, (300, 70, 1)), (x.shape, (64, 256, 1)), (x.shape, (65, 700, 1)),
                           ((1, 3, 64), (0, 64, 1)), ((4, 1, 64), (64, 0, 1)), ((4, 1, 64), (64, 1, 1)), ((0, 3, 64), (0, 0, 1))):
        y, p = torch.zeros(shape), pos[:shape[0]]
        with pytest.raises(ValueError, match="CUDA"):
            S.rotary(y, None, cos, cos, p, q_out=flat.as_strided(shape, strides))


def test_a_table_that_asks_for_a_gradient_is_refused():
    x, cos, pos = torch.zeros(2, 2, 64), torch.zeros(4, 16), torch.zeros(2, dtype=torch.int32)
    codes, scales = torch.zeros(2, 2, 2, 16, 32, dtype=torch.uint8), torch.zeros(2, 2, 2, 16, 2, dtype=torch.uint8)
    slots = torch.zeros(2, dtype=torch.int64)
    learned = cos.clone().requires_grad_()
    for c, s in ((learned, cos), (cos, learned)):
        for call in (lambda: S.rotary(x, None, c, s, pos), lambda: S.rotary(x.clone().requires_grad_(), x, c, s, pos),
                     lambda: S.rotary_backward(x, None, c, s, pos),
                     lambda: S.cache_append(x, x, codes, scales, slots, cos=c, sin=s, positions=pos)):
            with pytest.raises(ValueError, match="no gradient"):
                call()
            with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):
                call()
