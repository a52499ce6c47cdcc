"""The sequence operators beside the rest of autograd on the GPU: states that
change under a graph that saved them."""

import pytest
import torch

from mpgcn_amd import ops

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


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
