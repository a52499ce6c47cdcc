"""The scan where decays, states and steps leave the range of float32, over
sequences that are cut into segments and in whole ones."""

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


@pytest.mark.parametrize("softplus", [True, False])
@pytest.mark.parametrize("L,at", [(20, 10), (700, 350)])
@pytest.mark.parametrize("N", [3, 13, 16, 21])
def test_an_infinite_step_is_not_seen_before_it(N, L, at, softplus):
    """Tokens before an infinite step have the outputs and, where no loss comes
    from behind it, the gradients of the sequence that ends there, also where the
    states do not fill their lanes. From that step on a channel is not finite."""
    t = _inputs(5, L, 12, N)
    if softplus:
        t["delta"] = t["delta"] - 3
    t["delta"][:, at] = float("inf")
    dy = torch.randn(1, L, 12, generator=torch.Generator().manual_seed(6)).to(DEV)
    dy[:, at:] = 0
    cut = {k: v[:, :at] if k != "A" else v for k, v in t.items()}
    ref = oracle.scan(**cut, softplus=softplus, dy=dy[:, :at])
    leaves = {k: v.requires_grad_() for k, v in t.items()}
    y = ops.selective_scan(**t, delta_softplus=softplus)
    r = oracle.scan_roundings(at, N)
    oracle.within(y[:, :at], *ref["y"], r, "y")
    assert not torch.isfinite(y[:, at:]).any()
    got = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy)))
    for name in ("u", "delta", "B", "C"):
        oracle.within(got[name][:, :at], *ref[name], r + (12 if name in ("B", "C") else 0), name)


@pytest.mark.parametrize("N", [3, 13, 16, 21])
def test_a_token_with_an_infinite_step(N):
    t = _inputs(7, 1, 12, N)
    t = {k: v.abs() if k in ("u", "B", "C") else v for k, v in t.items()}
    t["delta"][:, 0, 5] = float("inf")
    t["state"] = torch.ones(1, 12, N, device=DEV)
    ref = oracle.scan(**t, softplus=False)
    one = {k: v if k in ("A", "state") else v[:, 0] for k, v in t.items()}
    y, s = ops.selective_scan_step(**one)
    assert y[0, 5] == float("inf") and (s[0, 5] == float("inf")).all()
    rest = [i for i in range(12) if i != 5]
    oracle.within(y[:, rest], ref["y"][0][:, 0, rest], ref["y"][1][:, 0, rest], oracle.scan_roundings(1, N), "y")
    oracle.within(s[:, rest], ref["last"][0][:, rest], ref["last"][1][:, rest], oracle.scan_roundings(1, N), "state")


@pytest.mark.parametrize("D,size", [(64, 2e18), (2560, 3e17), (16384, 1.2e17)])
def test_norms_of_large_values(D, size):
    """Rows whose root mean square stays below 1.8e19 / sqrt(D)."""
    g = torch.Generator().manual_seed(8)
    x = torch.where(torch.rand(3, D, generator=g) < 0.5, -size, size).to(DEV)
    w, q = torch.randn(D, generator=g).to(DEV), torch.randn(D, generator=g).to(DEV)
    r = oracle.norm_roundings(D)
    oracle.within(ops.norm_gate_residual(x, post_weight=w), *oracle.norm(x, None, w)["y"], r, "y")
    y, h = ops.norm_gate_residual(x * 0, post_weight=w, residual=x, pre_weight=q)
    ref = oracle.norm(x * 0, None, w, x, None, q)
    oracle.within(h, *ref["h"], r, "h")
    oracle.within(y, *ref["y"], r, "y")
