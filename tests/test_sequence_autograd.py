"""The sequence operators beside the rest of autograd on the GPU: states that
change under a graph that saved them, forward-mode derivatives, tracing."""

import pytest
import torch
import torch.autograd.forward_ad as fwad

from mpgcn_amd import ops

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
NAMES = ["short_conv", "short_conv_step", "selective_scan", "selective_scan_step", "norm_gate_residual"]


def _rn(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(DEV)


def _scan(L, seed=0):
    return dict(u=_rn(seed, 2, L, 8), delta=_rn(seed + 1, 2, L, 8), A=-_rn(seed + 2, 8, 4).abs(),
                B=_rn(seed + 3, 2, L, 4), C=_rn(seed + 4, 2, L, 4))


def _step_of(t):
    return {k: v if k == "A" else v[:, 0] for k, v in t.items()}


@pytest.mark.parametrize("L", [4, 20])
def test_a_step_over_a_saved_state_is_noticed(L):
    """A graph that saved the state it started from refuses its backward once a
    step has overwritten that state, as it does on the CPU."""
    t, w = _scan(L), _rn(9, 8, 3).requires_grad_()
    t["A"].requires_grad_()
    conv, h = _rn(10, 2, 2, 8), _rn(11, 2, 8, 4)
    for run, step, state in (
            (lambda: ops.short_conv(t["u"], w, state=conv), lambda: ops.short_conv_step(t["u"][:, 0], conv, w), conv),
            (lambda: ops.selective_scan(**t, state=h, delta_softplus=True),
             lambda: ops.selective_scan_step(**_step_of(t), state=h, delta_softplus=True), h)):
        y = run()
        before = state._version
        with torch.no_grad():
            step()
        assert state._version > before
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()


def test_only_the_state_that_is_written_counts_as_changed():
    t, w = _scan(1), _rn(9, 8, 3)
    for s, step in ((_rn(10, 2, 2, 8), lambda s, o: ops.short_conv_step(t["u"][:, 0], s, w, state_out=o)),
                    (_rn(11, 2, 8, 4), lambda s, o: ops.selective_scan_step(**_step_of(t), state=s, state_out=o))):
        out = torch.empty_like(s)
        before = s._version, out._version
        step(s, out)
        assert s._version == before[0] and out._version > before[1]
        with torch.inference_mode():
            held = s.clone()
            step(held, None)
        want = held.clone()
        step(want, None)
        step(held, None)  # a state made in inference mode, outside of it
        assert torch.equal(held, want)


def _forms():
    """name -> (call of its tensors, the tensors)."""
    t = _scan(5)
    w, h = _rn(21, 8, 3), _rn(22, 2, 8, 4)
    x, z = _rn(23, 2, 5, 8), _rn(24, 2, 5, 8)
    return {
        "short_conv": (lambda x, w, b, s: ops.short_conv(x, w, b, state=s), (x, w, w[:, 0], _rn(25, 2, 2, 8))),
        "short_conv_step": (lambda x, s, w: ops.short_conv_step(x, s, w)[0], (x[:, 0], _rn(25, 2, 2, 8), w)),
        "selective_scan": (lambda u, d, A, B, C, k, b, s: ops.selective_scan(
            u, d, A, B, C, k, delta_bias=b, delta_softplus=True, state=s), (*t.values(), w[:, 0], w[:, 1], h)),
        "selective_scan_step": (lambda u, d, A, B, C, s: ops.selective_scan_step(u, d, A, B, C, s)[0],
                                (*_step_of(t).values(), h)),
        "norm_gate_residual": (lambda x, z, p, r, s, q: ops.norm_gate_residual(
            x, gate=z, post_weight=p, residual=r, scale=s, pre_weight=q)[0], (x, z, w[:, 0], x, w[:, 1], w[:, 2])),
    }


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_is_refused(name, grad):
    """No tangent is dropped in silence, whichever input carries it."""
    call, args = _forms()[name]
    with torch.set_grad_enabled(grad):
        for i, a in enumerate(args):
            with fwad.dual_level():
                dual = fwad.make_dual(a, torch.ones_like(a))
                with pytest.raises(RuntimeError, match="forward-mode"):
                    call(*args[:i], dual, *args[i + 1:])
    with pytest.raises(RuntimeError):
        torch.func.jvp(call, args, tuple(torch.ones_like(a) for a in args))


@pytest.mark.parametrize("name", ["short_conv", "selective_scan", "norm_gate_residual"])
def test_forward_mode_over_the_gradient_is_refused(name):
    call, args = _forms()[name]
    leaf = args[0].clone().requires_grad_()
    y = call(leaf, *args[1:])
    with fwad.dual_level():
        dy = fwad.make_dual(torch.ones_like(y), torch.ones_like(y))
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.autograd.grad(y, leaf, dy)


@pytest.mark.parametrize("name", NAMES)
def test_tracing_is_refused(name):
    """A trace would hold the outputs as constants."""
    call, args = _forms()[name]
    with torch.no_grad(), pytest.raises(RuntimeError, match="traced"):
        torch.jit.trace(call, tuple(args), check_trace=False)
