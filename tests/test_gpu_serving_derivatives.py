"""Second derivatives and tangents through the rotary kernel."""
import numpy as np
import pytest
import torch
from torch.autograd import forward_ad

import serving_ref as R

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rotary_second_derivative_and_tangent(layout):
    """The gradient of |turned back gradient|^2 / 2 through y^2: with y = R x and g = 2 R^T y = 2 x, it is 4 x (R keeps
    lengths); each turn is off by at most 2^-22 of the pair's size (two products and a sum), of which there are four."""
    from sili__new_b200 import serving as S
    g = torch.Generator(device="cuda").manual_seed(7)
    cos, sin = S.rotary_table(64, 32)
    pos = torch.randint(0, 64, (9,), generator=g, device="cuda")
    q, k = (torch.randn(9, h, 64, generator=g, device="cuda", requires_grad=True) for h in (3, 1))
    y, z = S.rotary(q, k, cos, sin, pos, layout=layout)
    dq, dk = torch.autograd.grad((y ** 2).sum() + (z ** 2).sum(), (q, k), create_graph=True)
    ddq, ddk = torch.autograd.grad((dq ** 2).sum() / 2 + (dk ** 2).sum() / 2, (q, k))
    for x, d in ((q, ddq), (k, ddk)):
        assert float((d - 4 * x).detach().abs().max()) <= 16 * 2.0 ** -22 * float(x.detach().abs().max()) * 2
    t = torch.randn_like(q)
    with forward_ad.dual_level():
        out, _ = S.rotary(forward_ad.make_dual(q.detach(), t), None, cos, sin, pos, layout=layout)
        p, got = forward_ad.unpack_dual(out)
    assert torch.equal(p, y.detach())
    want = R.turn(t.double().cpu().numpy(), cos.double().cpu().numpy(), sin.double().cpu().numpy(), pos.cpu().numpy(), layout)
    assert (np.abs(got.double().cpu().numpy() - want) <= 2.0 ** -21 * float(t.abs().max())).all()
