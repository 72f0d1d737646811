"""Derivatives of rotary past the first gradient, with a plain turn in place of
the kernel (no GPU): the operator is linear, so a gradient of its gradient is
the turn itself and a tangent turns as its value does."""
import pytest
import torch
from torch.autograd import forward_ad

from sili__new_b200 import serving as S


def _plain(x, cos, sin, positions, layout, inverse):
    half = cos.shape[1]
    at = torch.arange(half)
    a, b = (at, at + half) if layout == "half" else (2 * at, 2 * at + 1)
    c, s = cos[positions.long()][:, None, :].to(x.dtype), sin[positions.long()][:, None, :].to(x.dtype)
    if inverse:
        s = -s
    out = x.clone()
    out[..., a], out[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    return out


@pytest.fixture
def case(monkeypatch):
    """(q, k, and a plain differentiable turn of both); the kernel's call works on data alone, as raw pointers do."""
    def raw(who, q, k, cos, sin, positions, layout, inverse, q_out, k_out):
        assert q_out is None and k_out is None
        with torch.no_grad():
            return tuple(None if x is None else _plain(x.detach(), cos, sin, positions, layout, inverse) for x in (q, k))
    monkeypatch.setattr(S, "_turn", raw)
    g = torch.Generator().manual_seed(0)
    q, k = torch.randn(5, 3, 16, generator=g).double(), torch.randn(5, 1, 16, generator=g).double()
    cos, sin = torch.randn(9, 4, generator=g), torch.randn(9, 4, generator=g)
    pos = torch.tensor([0, 8, 3, 3, 1])
    return q, k, (cos, sin, pos)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("call,inverse", [("rotary", False), ("rotary_backward", True)])
def test_gradient_of_a_gradient(case, layout, call, inverse):
    q, k, table = case
    got = []
    for turn in (lambda a, b: getattr(S, call)(a, b, *table, layout=layout),
                 lambda a, b: tuple(_plain(x, *table, layout, inverse) for x in (a, b))):
        a, b = q.clone().requires_grad_(), k.clone().requires_grad_()
        y, z = turn(a, b)
        loss = (y ** 3).sum() + (z ** 3).sum() + (y[:, :1] * z).sum()
        da, db = torch.autograd.grad(loss, (a, b), create_graph=True)
        assert da.requires_grad and db.requires_grad
        penalty = (da ** 2).sum() + (db ** 2).sum()
        got.append((da, db, *torch.autograd.grad(penalty + (a ** 2).sum(), (a, b))))
    for x, y in zip(*got):
        torch.testing.assert_close(x, y, rtol=1e-12, atol=1e-12)


@pytest.mark.parametrize("with_k", [True, False])
def test_only_one_gradient(case, with_k):
    q, k, table = case
    a = q.clone().requires_grad_()
    y, z = S.rotary(a, k if with_k else None, *table)
    (da,) = torch.autograd.grad((y ** 2).sum(), a, create_graph=True)
    (dda,) = torch.autograd.grad((da ** 2).sum(), a)
    a2 = q.clone().requires_grad_()
    (db,) = torch.autograd.grad((_plain(a2, *table, "half", False) ** 2).sum(), a2, create_graph=True)
    (ddb,) = torch.autograd.grad((db ** 2).sum(), a2)
    torch.testing.assert_close(dda, ddb, rtol=1e-12, atol=1e-12)
    assert (z is None) == (not with_k)


@pytest.mark.parametrize("duals", ["q", "k", "both"])
def test_tangents(case, duals):
    q, k, table = case
    tq, tk = torch.randn_like(q), torch.randn_like(k)
    with forward_ad.dual_level():
        a = forward_ad.make_dual(q, tq) if duals != "k" else q
        b = forward_ad.make_dual(k, tk) if duals != "q" else k
        y, z = S.rotary(a, b, *table)
        for out, x, t, dual in ((y, q, tq, duals != "k"), (z, k, tk, duals != "q")):
            p, got = forward_ad.unpack_dual(out)
            torch.testing.assert_close(p, _plain(x, *table, "half", False), rtol=0, atol=0)
            want = _plain(t, *table, "half", False) if dual else torch.zeros_like(x)
            torch.testing.assert_close(torch.zeros_like(x) if got is None else got, want, rtol=0, atol=0)
        if duals != "k":
            y, z = S.rotary(a, None, *table)
            assert z is None
            torch.testing.assert_close(forward_ad.unpack_dual(y).tangent, _plain(tq, *table, "half", False), rtol=0, atol=0)
        with pytest.raises(ValueError, match="output array"):
            S.rotary(a, b, *table, q_out=torch.empty_like(q))


def test_a_call_without_derivatives_stays_raw(case):
    q, k, table = case
    y, z = S.rotary(q, k, *table)
    assert not y.requires_grad and not z.requires_grad
    with torch.no_grad():
        assert not S.rotary(q.clone().requires_grad_(), k, *table)[0].requires_grad
