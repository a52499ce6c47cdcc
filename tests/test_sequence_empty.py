"""Batches, sequences and channels of which there are none."""

import pytest
import torch

from mpgcn_amd import ops

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def _stale(*shape):
    """Leaves NaN in the memory that the next tensor of this shape gets."""
    torch.full(shape, float("nan"), device=DEV)


@pytest.mark.parametrize("B,L,D,G", [(0, 3, 4, 2), (2, 0, 4, 2), (2, 3, 0, 2), (0, 0, 0, 1)])
def test_scan_of_nothing(B, L, D, G):
    N = 5
    t = dict(u=torch.zeros(B, L, D, device=DEV), delta=torch.zeros(B, L, D, device=DEV), A=torch.zeros(D, N, device=DEV),
             B=torch.ones(B, L, G, N, device=DEV), C=torch.ones(B, L, G, N, device=DEV),
             skip=torch.ones(D, device=DEV), state=torch.ones(B, D, N, device=DEV))
    leaves = [v.requires_grad_() for v in t.values()]
    y, h = ops.selective_scan(**t, delta_softplus=True, return_state=True)
    assert y.shape == (B, L, D) and h.shape == (B, D, N)
    for v in leaves:
        _stale(*v.shape), _stale(*v.shape)
    got = dict(zip(t, torch.autograd.grad([y, h], leaves, [torch.ones_like(y), torch.ones_like(h)])))
    for k, v in t.items():
        assert got[k].shape == v.shape and bool((got[k] == (1 if k == "state" else 0)).all()), k


@pytest.mark.parametrize("B,L,D", [(0, 3, 4), (2, 0, 4), (2, 3, 0)])
def test_conv_of_nothing(B, L, D):
    x, w, b, s = (torch.ones(*n, device=DEV).requires_grad_() for n in ((B, L, D), (D, 3), (D,), (B, 2, D)))
    y, last = ops.short_conv(x, w, b, state=s, return_state=True)
    assert y.shape == (B, L, D) and torch.equal(last, torch.ones(B, 2, D, device=DEV))
    for v in (x, w, b, s):
        _stale(*v.shape), _stale(*v.shape)
    gx, gw, gb, gs = torch.autograd.grad([y, last], [x, w, b, s], [torch.ones_like(y), torch.ones_like(last)])
    assert gx.shape == x.shape and not gw.any() and not gb.any() and torch.equal(gs, torch.ones_like(s))


def test_steps_and_norms_of_nothing():
    z = lambda *s: torch.ones(*s, device=DEV)
    for B, D in ((0, 4), (2, 0)):
        assert ops.short_conv_step(z(B, D), z(B, 2, D), z(D, 3))[0].shape == (B, D)
        assert ops.selective_scan_step(z(B, D), z(B, D), z(D, 4), z(B, 4), z(B, 4), z(B, D, 4))[0].shape == (B, D)
    x, w, s, q = (v.requires_grad_() for v in (z(0, 6), z(6), z(6), z(6)))
    y, h = ops.norm_gate_residual(x, gate=z(0, 6), post_weight=w, residual=z(0, 6), scale=s, pre_weight=q)
    _stale(3, 6), _stale(3, 6)
    for v, g in zip((x, w, s, q), torch.autograd.grad([y, h], [x, w, s, q], [z(0, 6), z(0, 6)])):
        assert g.shape == v.shape and not g.any()
    with pytest.raises(ValueError):
        ops.norm_gate_residual(z(3, 0), post_weight=z(0))
