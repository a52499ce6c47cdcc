"""What a call of the sequence operators does when it fails on the way: the
error reaches the caller, and nothing is done twice."""

import pytest
import torch

from mpgcn_amd import ops

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def _calls(b, d):
    """Every whole-sequence call on inputs of b rows that cost no memory; their
    outputs of b x d would."""
    row = torch.randn(1, 1, d, device=DEV)
    x, w, A = row.expand(b, 1, d), torch.randn(d, 4, device=DEV), -torch.rand(d, 4, device=DEV)
    m = torch.randn(1, 1, 4, device=DEV).expand(b, 1, 4)
    return {"short_conv": lambda: ops.short_conv(x, w),
            "selective_scan": lambda: ops.selective_scan(x, x, A, m, m, delta_softplus=True),
            "norm_gate_residual": lambda: ops.norm_gate_residual(x, post_weight=w[:, 0].contiguous())}


@pytest.mark.parametrize("name", ["short_conv", "selective_scan", "norm_gate_residual"])
def test_out_of_memory_is_met_once(name):
    """An output of 2 TiB: asked for once, and the error is the allocator's."""
    call = _calls(2 ** 29, 1024)[name]
    before = torch.cuda.memory_stats()["num_ooms"]
    with pytest.raises(torch.cuda.OutOfMemoryError):
        call()
    assert torch.cuda.memory_stats()["num_ooms"] == before + 1


@pytest.mark.parametrize("name", ["short_conv_step", "selective_scan_step"])
def test_a_token_is_applied_once_beside_an_old_error(name):
    """An error that an unrelated runtime call left behind is reported after the
    launch. The token has been applied by then, and is not applied again."""
    g = torch.Generator().manual_seed(5)
    rn = lambda *s: torch.randn(*s, generator=g).to(DEV)
    x = rn(3, 8)
    if name == "short_conv_step":
        w, state = rn(8, 3), rn(3, 2, 8)
        step = lambda s: ops.short_conv_step(x, s, w)
    else:
        A, m, state = -rn(8, 4).abs(), rn(3, 4), rn(3, 8, 4)
        step = lambda s: ops.selective_scan_step(x, x, A, m, m, s, delta_softplus=True)
    once = state.clone()
    step(once)
    torch.cuda.synchronize()
    torch.cuda.cudart().cudaHostUnregister(0)  # no such registration: refused by the host
    try:
        step(state)
    except RuntimeError:
        pass
    torch.cuda.synchronize()
    assert torch.equal(state, once)
