"""The scan where the decay of a segment leaves the range of float32."""

import pytest
import torch

import sequence_oracle as oracle
from mpgcn_amd import ops

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def _inputs(seed, L, D, N):
    g = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g).to(DEV)
    return dict(u=rn(1, L, D), delta=rn(1, L, D).abs() * 0.1, A=-torch.exp(0.3 * rn(D, N)), B=rn(1, L, 1, N),
                C=rn(1, L, 1, N))



@pytest.mark.parametrize("N", [4, 13, 16, 24])
def test_growing_steps_leave_an_empty_state_empty(N):
    """400 tokens whose steps grow by e^6 and more each and whose inputs are
    zero: the state stays zero, however the time axis is cut."""
    t = _inputs(1, 700, 24, N)
    t["A"] = t["A"].clamp(max=-1)
    t["u"][:, :400] = 0
    t["delta"][:, :400] = -6
    y, last = ops.selective_scan(**t, return_state=True)
    ref = oracle.scan(**t, softplus=False)
    r = oracle.scan_roundings(700, N)
    oracle.within(y, *ref["y"], r, "y")
    oracle.within(last, *ref["last"], r, "last")


@pytest.mark.parametrize("N", [4, 13, 16, 24])
def test_growing_steps_leave_an_empty_adjoint_empty(N):
    """The same backwards: no inputs, so states of zero throughout, and no
    gradient behind token 300, where the steps grow. (A state that decays below
    the range before it grows again would not do: its exact value is that of the
    summed exponents, which neither 32 nor 64 bits can follow step by step.)"""
    t = _inputs(2, 700, 24, N)
    t["A"] = t["A"].clamp(max=-1)
    t["u"].zero_()
    t["delta"][:, 300:] = -6
    dy = torch.randn(1, 700, 24, generator=torch.Generator().manual_seed(3)).to(DEV)
    dy[:, 300:] = 0
    ref = oracle.scan(**t, softplus=False, dy=dy)
    leaves = {k: v.requires_grad_() for k, v in t.items()}
    y = ops.selective_scan(**t)
    r = oracle.scan_roundings(700, N)
    for name, got in zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy)):
        more = 24 if name in ("B", "C") else 1400 if name == "A" else 0
        oracle.within(got, *ref[name], r + more, name)


def test_a_segments_decay_past_the_range():
    """A state of 1e-30 grows by e^100 over the first segment and shrinks again:
    it stays in the range, the segment's decay does not."""
    t = _inputs(4, 48, 8, 16)
    t["A"].fill_(-1)
    t["u"].zero_()
    t["delta"][:, :16] = -6.25
    t["state"] = torch.full((1, 8, 16), 1e-30, device=DEV)
    y, last = ops.selective_scan(**t, return_state=True)
    ref = oracle.scan(**t, softplus=False)
    # an exponent is off by 2 of its own roundings, the segment's by as much of their sum: 100 log2(e)
    r = oracle.scan_roundings(48, 16) + 4 * 145
    oracle.within(y, *ref["y"], r, "y")
    oracle.within(last, *ref["last"], r, "last")
