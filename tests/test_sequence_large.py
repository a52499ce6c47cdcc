"""Calls whose work items pass 32 bits or whose channels fill more than one
grid's limit. Each is compared where its parts can be told apart."""

import pytest
import torch

from mpgcn_amd import ops

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def _rn(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator(DEV).manual_seed(seed), device=DEV)


def test_conv_of_very_many_sequences():
    """2^30 sequences of one token: over 2^32 pieces of four channels. The rows
    are one row repeated, so the input takes no memory; the output takes 80 GiB."""
    B, D = 2 ** 30 - 1, 20
    if torch.cuda.mem_get_info()[0] < 100 * 2 ** 30:
        pytest.skip("needs 100 GiB of free memory")
    x, w, b = _rn(1, 1, 1, D), _rn(2, D, 4), _rn(3, D)
    want = ops.short_conv(x, w, b)[0, 0]
    y = ops.short_conv(x.expand(B, 1, D), w, b)[:, 0]
    for part in y.split(2 ** 27):
        assert bool((part == want).all())
    del y, part
    torch.cuda.empty_cache()


def test_conv_of_very_many_channels():
    """Gradients of 2^26 channels: more column sums than one launch may have
    threads for, more channel groups than 65536."""
    D = 2 ** 26 + 4
    x, dy, b = (_rn(s, 1, 1, D) for s in (4, 5, 6))
    w = _rn(7, D, 4)
    for t in (x, w, b):
        t.requires_grad_()
    y = ops.short_conv(x, w, b[0, 0])
    got = torch.autograd.grad(y, [x, w, b], dy)
    x, w, b, y = (t.detach() for t in (x, w, b, y))
    x1, b1, d1 = x[0, 0], b[0, 0], dy[0, 0]
    s = w[:, 3].double() * x1 + b1
    sg = torch.sigmoid(s)
    # the sum's three roundings, and some of the sigmoid's and its slope's, relative to the terms
    mag = (w[:, 3] * x1).abs() + b1.abs() + 1
    assert bool(((y[0, 0] - s * sg).abs() <= 24 * 2.0 ** -24 * (s.abs() + mag)).all())
    ds = d1 * (sg + s * sg * (1 - sg))
    tol = 24 * 2.0 ** -24 * d1.abs() * mag
    for g, f in ((got[0][0, 0], w[:, 3]), (got[1][:, 3], x1), (got[2][0, 0], torch.ones_like(x1))):
        assert bool(((g - ds * f).abs() <= tol * f.abs()).all())
    assert not got[1][:, :3].any()


def test_scan_of_very_many_channels():
    """2^22 channels of 64 states, one token: 2^28 column sums of dA."""
    D, N = 2 ** 22 + 8, 64
    u, delta, dy = (_rn(s, 1, 1, D) for s in (8, 9, 10))
    A, m, c = -_rn(11, D, N).abs(), _rn(12, 1, 1, 1, N), _rn(13, 1, 1, 1, N)
    h = torch.full((1, D, N), 0.5, device=DEV)
    A.requires_grad_()
    y = ops.selective_scan(u, delta, A, m, c, delta_softplus=True, state=h)
    gA = torch.autograd.grad(y, A, dy)[0]
    dt = torch.nn.functional.softplus(delta[0, 0].double()).unsqueeze(1)
    want = (dy[0, 0].unsqueeze(1) * c[0, 0, 0]) * dt * torch.exp(dt * A.detach()) * 0.5
    assert bool(((gA - want).abs() <= 64 * 2.0 ** -24 * want.abs() + 1e-37).all())


def test_scans_refuse_more_channels_than_a_launch_holds():
    D = 2 ** 26
    u, A, m = torch.zeros(1, 1, D, device=DEV), torch.zeros(D, 1, device=DEV), torch.zeros(1, 1, 1, device=DEV)
    with pytest.raises(ValueError, match="channels"):
        ops.selective_scan(u, u, A, m, m)
    with pytest.raises(ValueError, match="channels"):
        ops.selective_scan_step(u[0], u[0], A, m[0], m[0], A.view(1, D, 1))
