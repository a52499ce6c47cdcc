"""Sequence operators on the GPU: the HIP kernels against the 64-bit oracle of
the same inputs, at the sizes, strides and masks where they can go wrong."""

import pytest
import torch

import sequence_oracle as oracle
from mpgcn_amd import ops

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF, F = torch.bfloat16, torch.float32


def gen(seed):
    return torch.Generator().manual_seed(seed)


def rn(g, *shape, dtype=F, scale=1.0):
    return (torch.randn(*shape, generator=g) * scale).to(dtype).to(DEV)


def grads(outs, douts, leaves):
    return torch.autograd.grad(outs, leaves, douts, allow_unused=True)


# ---- short convolution ------------------------------------------------------

def conv_case(seed, dtype, B, L, D, K, carried, lengths, bias=True, view=False):
    g = gen(seed)
    x = rn(g, B, L, 2 * D + 3, dtype=dtype)[..., 1:D + 1] if view else rn(g, B, L, D, dtype=dtype)
    w, b = rn(g, D, K), rn(g, D) if bias else None
    s = rn(g, B, K - 1, D, dtype=dtype) if carried else None
    n = None
    if lengths:
        n = torch.randint(0, L + 1, (B,), generator=g).to(lengths)
        n[0] = 0
        n = n.to(DEV)
    return x, w, b, s, n


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("B,L,D,K,carried,lengths,bias", [
    (1, 1, 1, 2, False, None, True),
    (2, 1, 64, 4, True, None, True),
    (3, 2, 24, 4, True, torch.int32, False),
    (5, 7, 32, 4, False, None, True),
    (2, 16, 33, 3, True, torch.int64, True),
    (2, 17, 520, 2, True, torch.int32, True),
    (1, 301, 8, 4, False, None, False),
    (300, 5, 16, 4, True, torch.int64, True),
    (2, 0, 8, 3, True, None, True),
])
def test_short_conv(dtype, B, L, D, K, carried, lengths, bias):
    x, w, b, s, n = conv_case(B * 100 + L, dtype, B, L, D, K, carried, lengths, bias)
    g = gen(1)
    dy, dl = rn(g, B, L, D, dtype=dtype), rn(g, B, K - 1, D, dtype=dtype)
    leaves = [t.requires_grad_() for t in (x, w, b, s) if t is not None]
    names = [k for k, t in zip(("x", "weight", "bias", "state"), (x, w, b, s)) if t is not None]
    y, last = ops.short_conv(x, w, b, state=s, lengths=n, return_state=True)
    ref = oracle.conv(x, w, b, s, n, True, dy, dl)
    r = oracle.conv_roundings(K)
    oracle.within(y, *ref["y"], r, "y")
    assert torch.equal(last.detach().cpu().double(), ref["last"][0])
    for name, got in zip(names, grads([y, last], [dy, dl], leaves)):
        oracle.within(got, *ref[name], r + (2 * B * L if name in ("weight", "bias") else 0), name)
    # without a gradient the same kernel gives the same bits, and no activation is the sum itself
    with torch.no_grad():
        assert torch.equal(ops.short_conv(x, w, b, state=s, lengths=n), y)
        lin = ops.short_conv(x, w, b, state=s, lengths=n, activation=None)
    oracle.within(lin, *oracle.conv(x, w, b, s, n, False)["y"], r, "linear")


@pytest.mark.parametrize("dtype", [BF, F])
def test_short_conv_views(dtype):
    """Slices with odd strides and bases, expanded batches, permuted time."""
    x, w, b, s, n = conv_case(3, dtype, 3, 20, 40, 4, True, torch.int32, view=True)
    r = oracle.conv_roundings(4)
    oracle.within(ops.short_conv(x, w, b, state=s, lengths=n), *oracle.conv(x, w, b, s, n)["y"], r)
    e = x[:1].expand(3, 20, 40)
    oracle.within(ops.short_conv(e, w, b), *oracle.conv(e, w, b)["y"], r)
    t = x.transpose(0, 1)  # batch and time change places
    oracle.within(ops.short_conv(t, w, b), *oracle.conv(t, w, b)["y"], r)
    c = x.transpose(1, 2)  # channels not contiguous
    w2 = rn(gen(4), 20, 3)
    oracle.within(ops.short_conv(c, w2), *oracle.conv(c, w2)["y"], r)
    v = x.detach().clone().requires_grad_()
    ops.short_conv(v.expand(2, 3, 20, 40)[1], w, b).float().sum().backward()
    oracle.within(v.grad, *oracle.conv(v, w, b, dy=torch.ones_like(v))["x"], r)


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("B,D,K", [(1, 1, 2), (1, 1024, 4), (7, 33, 3), (256, 96, 4)])
def test_short_conv_step(dtype, B, D, K):
    g = gen(B + D)
    x, w, b, s = rn(g, B, 3 * D, dtype=dtype)[:, D:2 * D], rn(g, D, K), rn(g, D), rn(g, B, K - 1, D, dtype=dtype)
    ref = oracle.conv(x.unsqueeze(1), w, b, s)
    out = torch.full_like(s, float("nan"))
    y, same = ops.short_conv_step(x, s, w, b, state_out=out)
    assert same is out
    oracle.within(y.unsqueeze(1), *ref["y"], oracle.conv_roundings(K))
    assert torch.equal(out.cpu().double(), ref["last"][0])
    y2, same = ops.short_conv_step(x, s, w, b)  # in place
    assert same is s and torch.equal(y2, y) and torch.equal(s, out)


# ---- selective scan ---------------------------------------------------------

def scan_case(seed, dtype, B, L, D, N, G, carried, lengths, skip=True, bias=True):
    g = gen(seed)
    t = dict(u=rn(g, B, L, D, dtype=dtype), delta=rn(g, B, L, D, dtype=dtype),
             A=-torch.exp(rn(g, D, N)), B=rn(g, B, L, G, N, dtype=dtype), C=rn(g, B, L, G, N, dtype=dtype),
             skip=rn(g, D) if skip else None, delta_bias=rn(g, D) - 2 if bias else None,
             state=rn(g, B, D, N) if carried else None)
    n = None
    if lengths:
        n = torch.randint(0, L + 1, (B,), generator=g).to(lengths)
        n[0] = 0
        n = n.to(DEV)
    return t, n


def check_scan(t, n, dtype, softplus=True, with_state=True):
    B, L, D = t["u"].shape
    N = t["A"].shape[1]
    g = gen(2)
    dy, dl = rn(g, B, L, D, dtype=dtype), rn(g, B, D, N)
    leaves = {k: v.requires_grad_() for k, v in t.items() if v is not None}
    out = ops.selective_scan(**t, lengths=n, delta_softplus=softplus, return_state=with_state)
    y, last = out if with_state else (out, None)
    ref = oracle.scan(**t, softplus=softplus, lengths=n, dy=dy, dlast=dl if with_state else None)
    r = oracle.scan_roundings(L, N)
    oracle.within(y, *ref["y"], r, "y")
    got = grads([y, last] if with_state else [y], [dy, dl] if with_state else [dy], list(leaves.values()))
    if with_state:
        oracle.within(last, *ref["last"], r, "last")
    for name, v in zip(leaves, got):
        more = D if name in ("B", "C") else 2 * B * L if name in ("A", "skip", "delta_bias") else 0
        oracle.within(v, *ref[name], r + more, name)
    with torch.no_grad():
        assert torch.equal(ops.selective_scan(**t, lengths=n, delta_softplus=softplus), y)


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("B,L,D,N,G,carried,lengths", [
    (1, 1, 1, 1, 1, False, None),
    (2, 1, 64, 16, 1, True, None),
    (3, 7, 32, 16, 1, False, None),        # two sequences a wave, one left over
    (9, 14, 32, 16, 1, True, torch.int32),
    (2, 33, 66, 13, 2, True, torch.int64),
    (2, 25, 200, 16, 1, False, None),      # a channel block that is not full
    (1, 40, 8, 5, 4, True, torch.int32),
    (3, 9, 5, 3, 1, True, torch.int32),
    (2, 19, 48, 24, 1, False, torch.int64),
    (1, 21, 36, 64, 3, True, None),
    (2, 12, 7, 33, 1, True, torch.int32),
    (1, 300, 64, 16, 1, True, None),
    (130, 3, 4, 4, 1, False, torch.int32),
])
def test_selective_scan(dtype, B, L, D, N, G, carried, lengths):
    check_scan(*scan_case(B * 1000 + L, dtype, B, L, D, N, G, carried, lengths), dtype)


@pytest.mark.parametrize("softplus,skip,bias,with_state", [
    (False, True, True, True), (True, False, True, False), (True, True, False, True), (False, False, False, False)])
def test_selective_scan_parts(softplus, skip, bias, with_state):
    t, n = scan_case(11, F, 2, 18, 40, 16, 1, False, torch.int32, skip, bias)
    if not softplus:  # a step size as it is: positive, as the decay needs
        t["delta"] = t["delta"].abs() * 0.1
        if bias:
            t["delta_bias"] = t["delta_bias"].abs() * 0.05
    check_scan(t, n, F, softplus, with_state)


def test_selective_scan_only_state_gradient():
    """A loss on the final state alone: no gradient arrives for y."""
    t, _ = scan_case(12, F, 2, 11, 24, 8, 1, True, None)
    leaves = {k: v.requires_grad_() for k, v in t.items()}
    _, last = ops.selective_scan(**t, delta_softplus=True, return_state=True)
    dl = rn(gen(3), *last.shape)
    ref = oracle.scan(**t, softplus=True, dlast=dl)
    for name, v in zip(leaves, grads([last], [dl], list(leaves.values()))):
        more = 24 if name in ("B", "C") else 44 if name in ("A", "delta_bias") else 0
        oracle.within(v, *ref[name], oracle.scan_roundings(11, 8) + more, name)


@pytest.mark.parametrize("dtype", [BF, F])
def test_selective_scan_views(dtype):
    """dt, B and C as slices of one projection's output, u as a half of another."""
    g = gen(21)
    B, L, D, N = 3, 13, 48, 16
    xz, dbc = rn(g, B, L, 2 * D, dtype=dtype), rn(g, B, L, D + 2 * N + 1, dtype=dtype)
    t = dict(u=xz[..., D:], delta=dbc[..., :D], A=-torch.exp(rn(g, D, N)), B=dbc[..., D:D + N],
             C=dbc[..., D + N:D + 2 * N])
    ref = oracle.scan(t["u"], t["delta"], t["A"], t["B"].unsqueeze(2), t["C"].unsqueeze(2))
    oracle.within(ops.selective_scan(**t, delta_softplus=True), *ref["y"], oracle.scan_roundings(L, N))
    p = {k: v if k == "A" else v.transpose(0, 1) for k, v in t.items()}
    ref = oracle.scan(p["u"], p["delta"], p["A"], p["B"].unsqueeze(2), p["C"].unsqueeze(2))
    oracle.within(ops.selective_scan(**p, delta_softplus=True), *ref["y"], oracle.scan_roundings(B, N))


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("B,D,N,G", [(1, 1, 1, 1), (1, 1024, 16, 1), (5, 33, 13, 3), (64, 96, 64, 2), (3, 40, 20, 1)])
def test_selective_scan_step(dtype, B, D, N, G):
    t, _ = scan_case(B + D, dtype, B, 1, D, N, G, True, None)
    ref = oracle.scan(**t)
    one = {k: v if k in ("A", "skip", "delta_bias") else v[:, 0] for k, v in t.items() if k != "state"}
    s = t["state"]
    out = torch.full_like(s, float("nan"))
    y, same = ops.selective_scan_step(**one, state=s, delta_softplus=True, state_out=out)
    assert same is out
    oracle.within(y.unsqueeze(1), *ref["y"], oracle.scan_roundings(1, N))
    oracle.within(out, *ref["last"], oracle.scan_roundings(1, N))
    y2, same = ops.selective_scan_step(**one, state=s, delta_softplus=True)
    assert same is s and torch.equal(y2, y) and torch.equal(s, out)


def test_extreme_decays_and_padding():
    """Step sizes of 0 and far beyond exp's range, NaN and infinities behind the
    sequences' ends, an infinite decay: finite where the formula is."""
    t, _ = scan_case(31, F, 3, 20, 32, 16, 1, True, None)
    n = torch.tensor([20, 4, 0], device=DEV)
    t["delta"][0, :5] = -200.0
    t["delta"][0, 5:9] = 1000.0
    t["delta"][0, 9] = -3e38
    t["delta"][0, 10] = float("-inf")
    t["A"][3] = -1e30
    clean = {k: v.clone() for k, v in t.items()}
    for k in ("u", "delta", "B", "C"):
        t[k][1, 4:] = float("nan")
        t[k][2] = float("inf")
    y, last = ops.selective_scan(**t, lengths=n, delta_softplus=True, return_state=True)
    ref = oracle.scan(**clean, lengths=n)
    oracle.within(y, *ref["y"], oracle.scan_roundings(20, 16) + 4000, "y")
    oracle.within(last, *ref["last"], oracle.scan_roundings(20, 16) + 4000, "last")
    leaves = [t[k].requires_grad_() for k in ("u", "delta", "B", "C", "A", "state")]
    y = ops.selective_scan(**t, lengths=n, delta_softplus=True)
    got = grads([y], [torch.ones_like(y)], leaves)
    for k, v in zip(("u", "delta", "B", "C", "A", "state"), got):
        assert torch.isfinite(v).all(), k
        if k in ("u", "delta", "B", "C"):
            assert not v[1, 4:].any() and not v[2].any(), k
    x, w = rn(gen(5), 3, 20, 32), rn(gen(6), 32, 4)
    want = ops.short_conv(x, w, lengths=n, return_state=True)
    x[1, 4:], x[2] = float("nan"), float("inf")
    for a, b in zip(want, ops.short_conv(x, w, lengths=n, return_state=True)):
        assert torch.equal(a, b)


def test_lengths_are_held_to_the_range():
    t, _ = scan_case(32, F, 3, 6, 8, 4, 1, False, None)
    n = torch.tensor([-5, 99, 1 << 40], device=DEV)
    want = torch.tensor([0, 6, 6], device=DEV)
    assert torch.equal(ops.selective_scan(**t, lengths=n), ops.selective_scan(**t, lengths=want))
    x, w = rn(gen(7), 3, 6, 8), rn(gen(8), 8, 3)
    for a, b in zip(ops.short_conv(x, w, lengths=n, return_state=True),
                    ops.short_conv(x, w, lengths=want, return_state=True)):
        assert torch.equal(a, b)


# ---- norms ------------------------------------------------------------------

@pytest.mark.parametrize("dtype,res", [(BF, None), (F, None), (BF, BF), (BF, F), (F, F), (F, BF)])
@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("R,D", [(1, 1), (3, 8), (70, 32), (5, 33), (9, 512), (4, 520), (3, 1025), (2, 2560),
                                 (2, 4096), (3, 4100), (300, 5128), (2, 8200), (2, 16384)])
def test_norm(dtype, res, gate, R, D):
    g = gen(R * D)
    modes = [dict(post=True)] if res is None else [dict(post=True, scale=True, pre=True), dict(pre=True),
                                                   dict(post=True)]
    for m in modes:
        t = dict(x=rn(g, R, D, dtype=dtype), gate=rn(g, R, D, dtype=dtype) if gate else None,
                 post=rn(g, D) if m.get("post") else None,
                 residual=None if res is None else rn(g, R, D, dtype=res, scale=2.0),
                 scale=rn(g, D) if m.get("scale") else None, pre=rn(g, D) if m.get("pre") else None)
        leaves = {k: v.requires_grad_() for k, v in t.items() if v is not None}
        out = ops.norm_gate_residual(t["x"], gate=t["gate"], post_weight=t["post"], residual=t["residual"],
                                     scale=t["scale"], pre_weight=t["pre"])
        both = res is not None and m.get("pre")
        out = dict(zip(("y", "h"), out)) if both else {"y" if res is None else "h": out}
        d = {k: rn(g, R, D, dtype=v.dtype) for k, v in out.items()}
        ref = oracle.norm(**t, dy=d.get("y"), dh=d.get("h"))
        r = oracle.norm_roundings(D)
        for k, v in out.items():
            oracle.within(v, *ref[k], r, k)
        got = grads(list(out.values()), list(d.values()), list(leaves.values()))
        for k, v in zip(leaves, got):
            oracle.within(v, *ref[k], r + (R if k in ("post", "scale", "pre") else 0), k)


def test_norm_shapes_views_and_missing_gradients():
    g = gen(41)
    big = rn(g, 4, 6, 100, dtype=BF)
    x, z = big[..., 3:43], big[..., 50:90]
    w, r = rn(g, 40), rn(g, 4, 6, 40)
    y = ops.norm_gate_residual(x, gate=z, post_weight=w)
    assert y.shape == x.shape
    oracle.within(y, *oracle.norm(x, z, w)["y"], oracle.norm_roundings(40))
    # batch and time change places: the rows have no single stride
    oracle.within(ops.norm_gate_residual(x.transpose(0, 1), post_weight=w),
                  *oracle.norm(x.transpose(0, 1), None, w)["y"], oracle.norm_roundings(40))
    x = x.detach().clone().requires_grad_()
    for which in (0, 1):  # only one of the two outputs is used
        out = ops.norm_gate_residual(x, residual=r, pre_weight=w)
        d = rn(g, 4, 6, 40, dtype=out[which].dtype)
        ref = oracle.norm(x, residual=r, pre=w, **{("dy", "dh")[which]: d})
        oracle.within(grads([out[which]], [d], [x])[0], *ref["x"], oracle.norm_roundings(40))
    assert ops.norm_gate_residual(x[:0], post_weight=w).shape == (0, 6, 40)
    zero = torch.zeros(2, 40, device=DEV)
    assert not ops.norm_gate_residual(zero, post_weight=w).any()


# ---- together, and as programs use them -------------------------------------

def block(p, x, state=None):
    """norm -> projection -> conv -> scan -> gated norm -> projection."""
    D, N = p["D"], p["N"]
    res, x = x, ops.norm_gate_residual(x, post_weight=p["n0"])
    xz = x @ p["w_in"]
    u, z = xz[..., :D], xz[..., D:]
    step = x.dim() == 2
    if state is None:
        u = ops.short_conv(u, p["taps"], p["cbias"])
    elif step:
        u, _ = ops.short_conv_step(u, state["conv"], p["taps"], p["cbias"])
    else:
        u, state["conv"] = ops.short_conv(u, p["taps"], p["cbias"], return_state=True)
    dbc = u @ p["w_x"]
    kw = dict(skip=p["skip"], delta_bias=p["dbias"], delta_softplus=True)
    a = (u, dbc[..., :D], p["A"], dbc[..., D:D + N], dbc[..., D + N:])
    if state is None:
        y = ops.selective_scan(*a, **kw)
    elif step:
        y, _ = ops.selective_scan_step(*a, state["scan"], **kw)
    else:
        y, state["scan"] = ops.selective_scan(*a, **kw, return_state=True)
    y = ops.norm_gate_residual(y, gate=z, post_weight=p["n1"])
    return ops.norm_gate_residual(y @ p["w_out"], residual=res, scale=p["ls"], pre_weight=p["n2"])


def block_params(dtype, D=32, N=16, H=24):
    g = gen(51)
    return dict(D=D, N=N, n0=rn(g, H), w_in=rn(g, H, 2 * D, dtype=dtype, scale=0.2), taps=rn(g, D, 4, scale=0.5),
                cbias=rn(g, D), w_x=rn(g, D, D + 2 * N, dtype=dtype, scale=0.2), A=-torch.exp(rn(g, D, N)),
                skip=rn(g, D), dbias=rn(g, D) - 2, n1=rn(g, D), w_out=rn(g, D, H, dtype=dtype, scale=0.2),
                ls=rn(g, H), n2=rn(g, H))


def test_prompt_then_steps_equals_the_whole():
    p = block_params(F)
    x = rn(gen(52), 3, 12, 24)
    with torch.no_grad():
        y, h = block(p, x)
        st = {}
        y1, h1 = block(p, x[:, :9], st)
        ys, hs = [y1], [h1]
        for t in range(9, 12):
            a, b = block(p, x[:, t], st)
            ys.append(a.unsqueeze(1))
            hs.append(b.unsqueeze(1))
    # the same sums in another order: products of up to 56 terms, 12 steps
    torch.testing.assert_close(torch.cat(ys, 1), y, rtol=1e-4, atol=1e-4)
    torch.testing.assert_close(torch.cat(hs, 1), h, rtol=1e-4, atol=1e-4)


def test_block_gradients_against_the_definitions_on_cpu():
    p = block_params(F)
    x = rn(gen(53), 3, 12, 24)
    dy = rn(gen(54), 3, 12, 24)

    def run(p, x, dy):
        p = {k: v.detach().clone().requires_grad_() if torch.is_tensor(v) else v for k, v in p.items()}
        x = x.detach().clone().requires_grad_()
        y, h = block(p, x)
        leaves = {"x": x, **{k: v for k, v in p.items() if torch.is_tensor(v)}}
        return dict(zip(leaves, grads([y, h], [dy, dy], list(leaves.values()))))

    got = run(p, x, dy)
    ref = run({k: v.cpu().double() if torch.is_tensor(v) else v for k, v in p.items()}, x.cpu().double(),
              dy.cpu().double())
    for k, v in got.items():
        scale = float(ref[k].abs().max())
        assert float((v.cpu().double() - ref[k]).abs().max()) <= 1e-4 * scale, k


def test_same_call_same_bits():
    t, n = scan_case(61, BF, 70, 9, 32, 16, 1, True, torch.int32)
    x, w, b, s, m = conv_case(62, BF, 70, 9, 32, 4, True, torch.int32)
    leaves = [v.requires_grad_() for v in t.values()] + [v.requires_grad_() for v in (x, w, b, s)]
    z, nw = rn(gen(63), 70, 9, 32, dtype=BF).requires_grad_(), rn(gen(64), 32).requires_grad_()

    def run():
        y = ops.selective_scan(**t, lengths=n, delta_softplus=True)
        c = ops.short_conv(x, w, b, state=s, lengths=m)
        o = ops.norm_gate_residual(y, gate=z, post_weight=nw)
        return [y, c, o, *grads([c, o], [torch.ones_like(c), torch.ones_like(o)], leaves + [z, nw])]

    for a, b2 in zip(run(), run()):
        assert torch.equal(a, b2)


def test_other_stream():
    t, n = scan_case(71, BF, 4, 50, 64, 16, 1, True, torch.int32)
    want = ops.selective_scan(**t, lengths=n, delta_softplus=True)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        u = t["u"] * 1
        got = ops.selective_scan(**{**t, "u": u}, lengths=n, delta_softplus=True)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)


def test_captured_step_and_prompt():
    p = block_params(BF)
    g = gen(81)
    x1, xs = rn(g, 4, 24, dtype=BF), rn(g, 4, 10, 24, dtype=BF)
    st = dict(conv=rn(g, 4, 3, 32, dtype=BF), scan=rn(g, 4, 32, 16))
    with torch.no_grad():
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            block(p, x1, {k: v.clone() for k, v in st.items()})
            block(p, xs)
        torch.cuda.current_stream().wait_stream(side)
        cap = {k: v.clone() for k, v in st.items()}
        one, two = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(one):
            ys = block(p, x1, cap)[0]
        with torch.cuda.graph(two):
            yp = block(p, xs)[0]
        eager = {k: v.clone() for k, v in st.items()}
        for k in cap:
            cap[k].copy_(st[k])
        for i in range(4):
            x1.copy_(rn(g, 4, 24, dtype=BF))
            xs.copy_(rn(g, 4, 10, 24, dtype=BF))
            one.replay()
            two.replay()
            a, b = block(p, x1, eager)[0], block(p, xs)[0]
            torch.cuda.synchronize()
            assert torch.equal(ys, a) and torch.equal(yp, b), i
            assert all(torch.equal(cap[k], eager[k]) for k in cap), i


def test_captured_training_step():
    p = {k: v.requires_grad_() if torch.is_tensor(v) else v for k, v in block_params(BF).items()}
    leaves = [v for v in p.values() if torch.is_tensor(v)]
    g = gen(82)
    x, dy = rn(g, 4, 10, 24, dtype=BF), rn(g, 4, 10, 24, dtype=BF)

    def step():
        y, h = block(p, x)
        return grads([y, h], [dy, dy], leaves)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(4):
        x.copy_(rn(g, 4, 10, 24, dtype=BF))
        dy.copy_(rn(g, 4, 10, 24, dtype=BF))
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b), i


def test_capture_with_a_live_eager_graph_is_refused():
    """Refused on the host, in the forward: nothing of it is queued."""
    w = rn(gen(91), 32)
    wb = w.to(BF)
    for leaf, cast in ((w.requires_grad_(), False), (wb.requires_grad_(), True)):
        x = rn(gen(92), 4, 32)
        alive = ops.norm_gate_residual(x, post_weight=leaf)  # holds the leaf on this stream
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match="eager autograd graph"):
            with torch.cuda.graph(graph):
                ops.norm_gate_residual(x, post_weight=leaf)
        del alive
    torch.cuda.synchronize()


def test_argument_devices_are_checked():
    x, w = rn(gen(93), 2, 5, 8), rn(gen(94), 8, 3)
    with pytest.raises(ValueError):
        ops.short_conv(x, w.cpu())
    with pytest.raises(ValueError):
        ops.short_conv(x, w, lengths=torch.tensor([1, 2]))
    with pytest.raises(ValueError):
        ops.norm_gate_residual(x, post_weight=w[:, 0].cpu())
    with pytest.raises(TypeError):
        ops.norm_gate_residual(x.double(), post_weight=w[:, 0])


def test_second_derivatives_are_refused():
    """First gradients under create_graph are the usual ones; differentiating
    them again raises instead of giving zeros."""
    x, w = rn(gen(95), 2, 5, 8).requires_grad_(), rn(gen(96), 8, 3).requires_grad_()
    t, _ = scan_case(97, F, 2, 5, 8, 4, 1, False, None)
    u = t["u"].requires_grad_()
    for leaf, fn in ((x, lambda: ops.short_conv(x, w)),
                     (u, lambda: ops.selective_scan(**t)),
                     (x, lambda: ops.norm_gate_residual(x, gate=x * 2, post_weight=w[:, 0]))):
        plain = torch.autograd.grad(fn().square().sum(), leaf)[0]
        kept = torch.autograd.grad(fn().square().sum(), leaf, create_graph=True)[0]
        assert torch.equal(plain, kept)
        with pytest.raises(RuntimeError, match="second derivative"):
            kept.sum().backward()


@pytest.mark.parametrize("dtype", [BF, F])
def test_gradients_reach_only_what_asks(dtype):
    """Any one leaf alone, the others constants."""
    t, n = scan_case(98, dtype, 3, 9, 16, 5, 1, True, torch.int32)
    ref = oracle.scan(**t, lengths=n, dy=torch.ones(3, 9, 16))
    for name in t:
        one = {k: v.detach().clone().requires_grad_(k == name) for k, v in t.items()}
        y = ops.selective_scan(**one, lengths=n, delta_softplus=True)
        y.backward(torch.ones_like(y))
        oracle.within(one[name].grad, *ref[name], oracle.scan_roundings(9, 5) + 54, name)
        assert all(v.grad is None for k, v in one.items() if k != name)


def test_converted_arguments():
    """Weights of another type and channels that are not contiguous take the
    long way round, gradients included."""
    x, w = rn(gen(99), 2, 8, 6).transpose(1, 2).requires_grad_(), rn(gen(100), 8, 3, dtype=BF).requires_grad_()
    y = ops.short_conv(x, w)
    dy = rn(gen(101), 2, 6, 8)
    ref = oracle.conv(x, w.float(), dy=dy)
    oracle.within(y, *ref["y"], oracle.conv_roundings(3))
    gx, gw = grads([y], [dy], [x, w])
    oracle.within(gx, *ref["x"], oracle.conv_roundings(3))
    assert gw.dtype == BF
    oracle.within(gw, *ref["weight"], oracle.conv_roundings(3) + 24)


def test_offsets_beyond_32_bits():
    """Sequences 2^31 elements apart, and more than 2^31 elements in one tensor."""
    pool = torch.empty(2 ** 31 + 4096, device=DEV, dtype=BF)
    far = pool.as_strided((2, 6, 32), (2 ** 31 + 8, 64, 1))
    near = rn(gen(110), 2, 6, 32, dtype=BF)
    far.copy_(near)
    # bit for bit; the raw steps (no softplus) grow some states past the range, where the formula gives NaN
    same = lambda a, b: torch.testing.assert_close(a, b, rtol=0, atol=0, equal_nan=True)
    w = rn(gen(111), 32, 4)
    assert torch.equal(ops.short_conv(far, w), ops.short_conv(near, w))
    t, _ = scan_case(112, BF, 2, 6, 32, 16, 1, False, None)
    same(ops.selective_scan(**{**t, "u": far, "delta": far}), ops.selective_scan(**{**t, "u": near, "delta": near}))
    step = pool.as_strided((3, 6, 8), (64, 2 ** 28, 1))  # tokens too far apart for lane offsets: a copy
    step.copy_(near[:1, :, :8].expand(3, 6, 8))
    t, _ = scan_case(113, BF, 3, 6, 8, 4, 1, False, None)
    same(ops.selective_scan(**{**t, "u": step}), ops.selective_scan(**{**t, "u": step.contiguous()}))
    rows = pool.as_strided((2, 40), (2 ** 31 + 8, 1))
    rows.copy_(near[:, 0].repeat(1, 2)[:, :40])
    pw = rn(gen(114), 40)
    assert torch.equal(ops.norm_gate_residual(rows, post_weight=pw),
                       ops.norm_gate_residual(rows.contiguous(), post_weight=pw))
    del far, step, rows
    # one tensor of 2^31 + elements: its end equals the end computed alone
    L = 2 ** 31 // 32 + 64
    x = pool[: L * 32].view(1, L, 32)
    x.normal_()
    y, last = ops.short_conv(x, w, return_state=True)
    tail, last2 = ops.short_conv(x[:, -50:].contiguous(), w, return_state=True)
    assert torch.equal(y[:, -40:], tail[:, -40:]) and torch.equal(last, last2)
    del y
    n = ops.norm_gate_residual(x[0], post_weight=w[:, 0])
    assert torch.equal(n[-70:], ops.norm_gate_residual(x[0, -70:].contiguous(), post_weight=w[:, 0]))


def test_long_sequence_equals_its_parts():
    """65 k tokens in one call, in segments, against two calls that hand the
    state over: the same recurrence from other segment starts."""
    t, _ = scan_case(120, F, 1, 65536, 40, 16, 1, True, None)
    kw = dict(delta_softplus=True, return_state=True)
    y, h = ops.selective_scan(**t, **kw)
    cut = 33333
    part = lambda a, b: {k: v[:, a:b] if k in ("u", "delta", "B", "C") else v for k, v in t.items()}
    y1, h1 = ops.selective_scan(**part(0, cut), **kw)
    y2, h2 = ops.selective_scan(**{**part(cut, None), "state": h1}, **kw)
    # states forget within some hundred steps: 4 roundings a step of them
    mag = float(y.abs().max())
    assert float((torch.cat([y1, y2], 1) - y).abs().max()) <= 4 * 1000 * 2.0 ** -24 * mag
    assert float((h2 - h).abs().max()) <= 4 * 1000 * 2.0 ** -24 * float(h.abs().max())


@pytest.mark.parametrize("dtype,B,L,D,N,lengths", [
    (BF, 2, 700, 96, 16, torch.int32), (F, 1, 1500, 33, 13, None), (BF, 3, 530, 24, 8, torch.int64),
    (F, 2, 600, 40, 40, torch.int32)])
def test_selective_scan_in_segments(dtype, B, L, D, N, lengths):
    """Few long sequences: the time axis is cut, ends fall inside segments."""
    check_scan(*scan_case(B + L, dtype, B, L, D, N, 1, True, lengths), dtype)


def test_only_the_last_state_has_a_gradient():
    """Both without segments and in them; skip and C see none of it."""
    for L in (9, 700):
        t, n = scan_case(130 + L, F, 2, L, 24, 16, 1, True, torch.int32)
        dl = rn(gen(131), 2, 24, 16)
        leaves = {k: v.requires_grad_() for k, v in t.items()}
        _, last = ops.selective_scan(**t, lengths=n, delta_softplus=True, return_state=True)
        got = dict(zip(leaves, grads([last], [dl], list(leaves.values()))))
        ref = oracle.scan(**t, softplus=True, lengths=n, dy=torch.zeros(2, L, 24, device=DEV), dlast=dl)
        r = oracle.scan_roundings(L, 16)
        for name in ("u", "delta", "A", "B", "delta_bias", "state"):
            more = 24 if name == "B" else 4 * L if name in ("A", "delta_bias") else 0
            oracle.within(got[name], *ref[name], r + more, name)
        for name in ("C", "skip"):
            assert got[name] is None or not got[name].any(), name


def test_broadcast_inputs_and_gradients():
    """Inputs that repeat (strides of 0), one tensor in two places, an expanded
    gradient: what autograd adds up is the sum over the repeats."""
    g = gen(140)
    t, _ = scan_case(141, F, 1, 1, 24, 16, 1, False, None)
    u, delta = rn(g, 3, 12, 24).requires_grad_(), rn(g, 1, 12, 24).requires_grad_()
    Bm, s = rn(g, 3, 1, 1, 16).requires_grad_(), rn(g, 1, 24, 16).requires_grad_()
    full = lambda: dict(u=u, delta=delta.expand(3, 12, 24), A=t["A"], B=Bm.expand(3, 12, 1, 16),
                        C=Bm.expand(3, 12, 1, 16), state=s.expand(3, 24, 16))
    y = ops.selective_scan(**full(), delta_softplus=True)
    got = torch.autograd.grad(y.sum(), [u, delta, Bm, s])
    clean = {k: v.detach().clone().requires_grad_() for k, v in full().items()}
    y2 = ops.selective_scan(**clean, delta_softplus=True)
    d = dict(zip(clean, torch.autograd.grad(y2, list(clean.values()), torch.ones_like(y2))))
    assert torch.equal(y, y2) and torch.equal(got[0], d["u"])
    both = (d["B"].double() + d["C"].double()).sum(1, keepdim=True)
    for a, b, n in ((got[1], d["delta"].double().sum(0, keepdim=True), 3),
                    (got[2], both, 24), (got[3], d["state"].double().sum(0, keepdim=True), 3)):
        # n - 1 roundings of sums no larger than the sum of magnitudes, taken as n times the largest term
        assert float((a.double() - b).abs().max()) <= n * n * 2.0 ** -24 * max(float(v.abs().max()) for v in d.values())
    row = rn(g, 24).requires_grad_()
    w = rn(g, 24, 4)
    x = row.expand(2, 9, 24)
    assert torch.equal(ops.short_conv(x, w), ops.short_conv(x.contiguous(), w))
    y = ops.norm_gate_residual(x, gate=x, post_weight=w[:, 0])
    assert torch.equal(y, ops.norm_gate_residual(x.contiguous(), gate=x.contiguous(), post_weight=w[:, 0]))
    assert torch.equal(torch.autograd.grad(y.sum(), row)[0] != 0, torch.ones(24, dtype=torch.bool, device=DEV))


def test_inference_mode():
    t, n = scan_case(142, BF, 2, 20, 32, 16, 1, True, torch.int32)
    x, w = t["u"], rn(gen(143), 32, 4)
    want = (ops.short_conv(x, w), ops.selective_scan(**t, lengths=n), ops.norm_gate_residual(x, post_weight=w[:, 0]))
    with torch.inference_mode():
        got = (ops.short_conv(x, w), ops.selective_scan(**t, lengths=n),
               ops.norm_gate_residual(x, post_weight=w[:, 0]))
        state = torch.zeros(2, 3, 32, device=DEV, dtype=BF)
        y, same = ops.short_conv_step(x[:, 0], state, w)
    assert same is state and torch.equal(y, want[0][:, 0])
    for a, b in zip(got, want):
        torch.testing.assert_close(a, b, rtol=0, atol=0, equal_nan=True)


def test_two_streams_at_once():
    """The same calls side by side on two streams give what they give alone."""
    t, _ = scan_case(144, BF, 1, 4000, 96, 16, 1, False, None)
    leaves = {k: v.requires_grad_() for k, v in t.items() if v is not None}
    dy = rn(gen(145), 1, 4000, 96, dtype=BF)

    def run():
        y = ops.selective_scan(**t, delta_softplus=True)
        return [y, *torch.autograd.grad(y, list(leaves.values()), dy)]

    want = run()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(run())
    torch.cuda.synchronize()
    for o in outs:
        for a, b in zip(o, want):
            assert torch.equal(a, b)
