"""Sequence operators on the CPU: the plain definitions against the 64-bit
oracle, the oracle's gradients against differences, and every refusal."""

import pytest
import torch

import sequence_oracle as oracle
from mpgcn_amd import ops

g = torch.Generator().manual_seed(5)


def randn(*shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g).to(dtype)


def scan_inputs(B, L, D, N, G, dtype=torch.float32):
    return dict(u=randn(B, L, D, dtype=dtype), delta=randn(B, L, D, dtype=dtype),
                A=-torch.exp(randn(D, N)), B=randn(B, L, G, N, dtype=dtype), C=randn(B, L, G, N, dtype=dtype))


# ---- definitions and gradients ----------------------------------------------

@pytest.mark.parametrize("L", [0, 1, 2, 9])
@pytest.mark.parametrize("K", [2, 3, 4])
@pytest.mark.parametrize("carried,lengths", [(False, None), (True, [9, 0, 1])])
def test_short_conv_definition(L, K, carried, lengths):
    B, D = 3, 5
    x, w, b = randn(B, L, D), randn(D, K), randn(D)
    s = randn(B, K - 1, D) if carried else None
    n = None if lengths is None else torch.tensor(lengths).clamp(max=L)
    leaves = [t.requires_grad_() for t in (x, w, b, s) if t is not None]
    y, last = ops.short_conv(x, w, b, state=s, lengths=n, return_state=True)
    dy, dl = randn(B, L, D), randn(B, K - 1, D)
    ref = oracle.conv(x, w, b, s, n, True, dy, dl)
    r = oracle.conv_roundings(K) + 2 * B * L
    oracle.within(y, *ref["y"], r, "y")
    assert torch.equal(last.double(), ref["last"][0])
    torch.autograd.backward([y, last], [dy, dl])
    for name, t in zip(("x", "weight", "bias", "state"), leaves):
        oracle.within(t.grad, *ref[name], r, name)


@pytest.mark.parametrize("L", [0, 1, 7])
@pytest.mark.parametrize("softplus", [True, False])
@pytest.mark.parametrize("carried,lengths", [(False, None), (True, [7, 0, 2])])
def test_selective_scan_definition(L, softplus, carried, lengths):
    B, D, N, G = 3, 6, 3, 2
    i = scan_inputs(B, L, D, N, G)
    skip, bias = randn(D), randn(D)
    s = randn(B, D, N) if carried else None
    n = None if lengths is None else torch.tensor(lengths).clamp(max=L)
    leaves = dict(i, skip=skip, delta_bias=bias, **({"state": s} if carried else {}))
    for t in leaves.values():
        t.requires_grad_()
    y, last = ops.selective_scan(**i, skip=skip, delta_bias=bias, delta_softplus=softplus, state=s, lengths=n,
                                 return_state=True)
    dy, dl = randn(B, L, D), randn(B, D, N)
    ref = oracle.scan(**i, skip=skip, delta_bias=bias, softplus=softplus, state=s, lengths=n, dy=dy, dlast=dl)
    r = oracle.scan_roundings(L, N) + 2 * B * L + D
    oracle.within(y, *ref["y"], r, "y")
    oracle.within(last, *ref["last"], r, "last")
    through = [(v, d) for v, d in ((y, dy), (last, dl)) if v.requires_grad]  # no token, no state: constants
    if through:
        torch.autograd.backward(*zip(*through))
    for name, t in leaves.items():
        oracle.within(torch.zeros_like(t) if t.grad is None else t.grad, *ref[name], r, name)


NORMS = [dict(post=True), dict(gate=True, post=True), dict(res=True, pre=True),
         dict(gate=True, post=True, res=True, scale=True, pre=True), dict(post=True, res=True),
         dict(gate=True, res=True, scale=True, pre=True)]


@pytest.mark.parametrize("parts", NORMS)
@pytest.mark.parametrize("D", [1, 7, 64])
def test_norm_definition(parts, D):
    shape = (2, 3, D)
    t = dict(x=randn(*shape), gate=randn(*shape) if parts.get("gate") else None,
             post=randn(D) if parts.get("post") else None, residual=randn(*shape) if parts.get("res") else None,
             scale=randn(D) if parts.get("scale") else None, pre=randn(D) if parts.get("pre") else None)
    for v in t.values():
        if v is not None:
            v.requires_grad_()
    out = ops.norm_gate_residual(t["x"], gate=t["gate"], post_weight=t["post"], residual=t["residual"],
                                 scale=t["scale"], pre_weight=t["pre"])
    both = parts.get("res") and parts.get("pre")
    out = dict(zip(("y", "h"), out)) if both else {"h" if parts.get("res") else "y": out}
    d = {k: randn(*shape) for k in out}
    ref = oracle.norm(**t, dy=d.get("y"), dh=d.get("h"))
    r = oracle.norm_roundings(D) + 6
    for k, v in out.items():
        oracle.within(v, *ref[k], r, k)
    torch.autograd.backward(list(out.values()), [d[k] for k in out])
    for k, v in t.items():
        if v is not None:
            oracle.within(v.grad, *ref[k], r, k)


def test_definitions_pass_gradcheck():
    f64 = torch.float64

    def r(*s):
        return torch.randn(*s, generator=g, dtype=f64).requires_grad_()

    n = torch.tensor([4, 0, 2])
    torch.autograd.gradcheck(
        lambda x, w, b, s: ops.short_conv(x, w, b, state=s, lengths=n, return_state=True),
        (r(3, 4, 2), r(2, 3), r(2), r(3, 2, 2)))
    torch.autograd.gradcheck(
        lambda u, d, A, B, C, k, b, s: ops.selective_scan(u, d, A, B, C, k, delta_bias=b, delta_softplus=True,
                                                          state=s, lengths=n, return_state=True),
        (r(3, 4, 2), r(3, 4, 2), r(2, 2), r(3, 4, 1, 2), r(3, 4, 1, 2), r(2), r(2), r(3, 2, 2)))
    torch.autograd.gradcheck(
        lambda x, z, a, h, s, b: ops.norm_gate_residual(x, gate=z, post_weight=a, residual=h, scale=s, pre_weight=b),
        (r(2, 5), r(2, 5), r(5), r(2, 5), r(5), r(5)))


@pytest.mark.parametrize("what", ["conv", "scan", "norm"])
def test_oracle_gradients_against_differences(what):
    """The oracle's hand-written gradients against central differences of its
    own outputs, step 1e-6: off by the third derivative times 1e-12 and by
    2^-53 / 1e-6 of the outputs, both under 1e-6 of the magnitude."""
    n = torch.tensor([4, 0, 3])
    if what == "conv":
        t = dict(x=randn(3, 4, 2), weight=randn(2, 3), bias=randn(2), state=randn(3, 2, 2))
        fn = lambda t, **d: oracle.conv(**t, lengths=n, **d)
        outs, dn = ("y", "last"), ("dy", "dlast")
    elif what == "scan":
        t = dict(scan_inputs(3, 4, 4, 2, 2), skip=randn(4), delta_bias=randn(4), state=randn(3, 4, 2))
        fn = lambda t, **d: oracle.scan(**t, lengths=n, **d)
        outs, dn = ("y", "last"), ("dy", "dlast")
    else:
        t = dict(x=randn(3, 5), gate=randn(3, 5), post=randn(5), residual=randn(3, 5), scale=randn(5), pre=randn(5))
        fn = lambda t, **d: oracle.norm(**t, **d)
        outs, dn = ("y", "h"), ("dy", "dh")
    t = {k: v.double() for k, v in t.items()}
    base = fn(t)
    d = {a: randn(*base[o][0].shape).double() for a, o in zip(dn, outs)}
    ref = fn(t, **d)

    def loss(t):
        o = fn(t)
        return sum((o[k][0] * d[a]).sum() for a, k in zip(dn, outs))

    for name, v in t.items():
        num = torch.zeros_like(v)
        for i in range(v.numel()):
            e = torch.zeros_like(v).view(-1)
            e[i] = 1e-6
            e = e.view_as(v)
            num.view(-1)[i] = (loss({**t, name: v + e}) - loss({**t, name: v - e})) / 2e-6
        assert ((num - ref[name][0]).abs() <= 1e-6 * (1 + ref[name][1])).all(), name


# ---- the step forms and a run over calls ------------------------------------

def test_steps_continue_a_prompt():
    B, L, D, N, K = 2, 6, 4, 3, 3
    i = scan_inputs(B, L, D, N, 1)
    x, w, b = randn(B, L, D), randn(D, K), randn(D)
    whole = ops.short_conv(x, w, b)
    y, cs = ops.short_conv(x[:, :4], w, b, return_state=True)
    ys = [y] + [ops.short_conv_step(x[:, t], cs, w, b)[0].unsqueeze(1) for t in (4, 5)]
    torch.testing.assert_close(torch.cat(ys, 1), whole, rtol=0, atol=1e-6)
    kw = dict(delta_softplus=True)
    whole, end = ops.selective_scan(**i, **kw, return_state=True)
    y, hs = ops.selective_scan(**{k: v[:, :4] if k != "A" else v for k, v in i.items()}, **kw, return_state=True)
    ys = [y]
    for t in (4, 5):
        y, same = ops.selective_scan_step(i["u"][:, t], i["delta"][:, t], i["A"], i["B"][:, t], i["C"][:, t], hs, **kw)
        assert same is hs
        ys.append(y.unsqueeze(1))
    torch.testing.assert_close(torch.cat(ys, 1), whole, rtol=0, atol=1e-5)
    torch.testing.assert_close(hs, end, rtol=0, atol=1e-5)
    out = torch.empty_like(hs)
    kept = hs.clone()
    _, got = ops.selective_scan_step(i["u"][:, 0], i["delta"][:, 0], i["A"], i["B"][:, 0], i["C"][:, 0], hs,
                                     state_out=out)
    assert got is out and torch.equal(hs, kept)


def test_padding_is_not_read():
    n = torch.tensor([2, 0])
    i = scan_inputs(2, 5, 4, 3, 1)
    x, w = randn(2, 5, 4), randn(4, 3)
    clean = ops.short_conv(x, w, lengths=n), ops.selective_scan(**i, lengths=n, delta_softplus=True)
    for t in (x, i["u"], i["delta"], i["B"], i["C"]):
        t[0, 2:], t[1] = float("nan"), float("inf")
    soiled = ops.short_conv(x, w, lengths=n), ops.selective_scan(**i, lengths=n, delta_softplus=True)
    for a, b in zip(clean, soiled):
        assert torch.equal(a, b)


# ---- refusals ---------------------------------------------------------------

def test_short_conv_refusals():
    x, w = randn(2, 5, 4), randn(4, 3)
    for err, args, kw in [
        (TypeError, (x.half(), w), {}),
        (TypeError, (x.long(), w), {}),
        (ValueError, (x[0], w), {}),
        (ValueError, (x, randn(5, 3)), {}),
        (ValueError, (x, randn(4, 1)), {}),
        (ValueError, (x, randn(4, 5)), {}),
        (TypeError, (x, w.long()), {}),
        (ValueError, (x, w, randn(3)), {}),
        (ValueError, (x, w), dict(activation="relu")),
        (ValueError, (x, w), dict(state=randn(2, 3, 4))),
        (TypeError, (x, w), dict(state=randn(2, 2, 4, dtype=torch.bfloat16))),
        (TypeError, (x, w), dict(lengths=torch.ones(2))),
        (ValueError, (x, w), dict(lengths=torch.ones(3, dtype=torch.int32))),
    ]:
        with pytest.raises(err):
            ops.short_conv(*args, **kw)
    s = randn(2, 2, 4)
    with pytest.raises(ValueError):
        ops.short_conv_step(x, s, w)
    with pytest.raises(ValueError):
        ops.short_conv_step(x[:, 0], s[:, :1], w)
    with pytest.raises(ValueError):
        ops.short_conv_step(x[:, 0], randn(4, 2, 2).permute(1, 2, 0)[..., :4], w)
    buf = randn(2 * 2 * 4 + 1)
    with pytest.raises(ValueError):
        ops.short_conv_step(x[:, 0], buf[:-1].view(2, 2, 4), w, state_out=buf[1:].view(2, 2, 4))
    with pytest.raises(RuntimeError):
        ops.short_conv_step(x[:, 0], s, w.clone().requires_grad_())


def test_selective_scan_refusals():
    i = scan_inputs(2, 5, 6, 3, 2)
    for err, kw in [
        (TypeError, dict(u=i["u"].half())),
        (ValueError, dict(u=i["u"][0])),
        (TypeError, dict(delta=i["delta"].bfloat16())),
        (ValueError, dict(delta=i["delta"][:, :4])),
        (ValueError, dict(A=randn(5, 3))),
        (ValueError, dict(A=randn(6, 65))),
        (ValueError, dict(A=randn(6, 0))),
        (ValueError, dict(A=randn(6, 4))),
        (TypeError, dict(B=i["B"].bfloat16())),
        (TypeError, dict(C=None)),
        (ValueError, dict(B=randn(2, 5, 4, 3), C=randn(2, 5, 4, 3))),
        (ValueError, dict(C=randn(2, 5, 3, 3))),
        (ValueError, dict(skip=randn(5))),
        (ValueError, dict(delta_bias=randn(6, 1))),
        (ValueError, dict(state=randn(2, 6, 4))),
        (TypeError, dict(state=randn(2, 6, 3, dtype=torch.bfloat16))),
        (TypeError, dict(lengths=torch.ones(2, dtype=torch.int16))),
    ]:
        with pytest.raises(err):
            ops.selective_scan(**{**i, **kw})
    wide = torch.empty(1, 1, 2 ** 26, device="meta")
    with pytest.raises(ValueError):
        ops.selective_scan(wide, wide, wide.view(-1, 1), wide[..., :1], wide[..., :1])
    s = dict(u=i["u"][:, 0], delta=i["delta"][:, 0], A=i["A"], B=i["B"][:, 0], C=i["C"][:, 0])
    with pytest.raises(ValueError):
        ops.selective_scan_step(**s, state=randn(2, 6, 4))
    with pytest.raises(TypeError):
        ops.selective_scan_step(**s, state=randn(2, 6, 3, dtype=torch.bfloat16))
    with pytest.raises(RuntimeError):
        ops.selective_scan_step(**{**s, "A": s["A"].clone().requires_grad_()}, state=randn(2, 6, 3))


def test_norm_refusals():
    x, w = randn(3, 8), randn(8)
    for err, kw in [
        (ValueError, {}),
        (ValueError, dict(gate=x)),
        (ValueError, dict(pre_weight=w)),
        (ValueError, dict(post_weight=w, scale=w)),
        (ValueError, dict(post_weight=randn(7))),
        (ValueError, dict(post_weight=w, eps=0.0)),
        (ValueError, dict(post_weight=w, eps=float("nan"))),
        (ValueError, dict(post_weight=w, eps=1e-40)),
        (ValueError, dict(post_weight=w, gate=randn(2, 8))),
        (TypeError, dict(post_weight=w, gate=x.bfloat16())),
        (TypeError, dict(post_weight=w, residual=x.half())),
        (ValueError, dict(post_weight=w, residual=x[:2])),
    ]:
        with pytest.raises(err):
            ops.norm_gate_residual(x, **kw)
    with pytest.raises(TypeError):
        ops.norm_gate_residual(x.half(), post_weight=w)
    with pytest.raises(ValueError):
        ops.norm_gate_residual(randn(1, 16385), post_weight=randn(16385))
