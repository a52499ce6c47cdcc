"""Definitions of the sequence operators in 64 bits, gradients by hand, and for
every result a magnitude: the same formula with all terms taken absolutely.
A computation in f32 that adds the same terms is off by no more than the
number of roundings on the longest path times 2^-24 of that magnitude, and an
output of fewer bits by half a step of its own on top (``within``)."""

import torch

U32 = 2.0 ** -24


def within(got, ref, mag, roundings, name=""):
    """got (any type) against ref +- (half a step of got's type + roundings u mag)."""
    ref, mag = ref.detach().cpu(), mag.detach().cpu()
    half = torch.finfo(got.dtype).eps / 2
    tiny = torch.finfo(got.dtype).tiny  # below it steps are absolute
    soft = roundings * U32 * mag
    tol = half * (ref.abs() + soft) + soft + tiny
    err = (got.detach().cpu().double() - ref).abs()
    bad = ~(err <= tol)
    assert got.shape == ref.shape, (name, got.shape, ref.shape)
    assert not bad.any(), (
        f"{name}: {int(bad.sum())} of {bad.numel()} off, worst {float((err / tol).nan_to_num(1e30).max()):.3g} "
        f"times the tolerance at {tuple(bad.nonzero()[0].tolist())}")


def _d(t):
    return None if t is None else t.detach().cpu().double()


def live(lengths, B, L):
    if lengths is None:
        return torch.ones(B, L, 1, dtype=torch.bool)
    return (torch.arange(L) < lengths.cpu().clamp(0, L).unsqueeze(1)).unsqueeze(-1)


def conv(x, weight, bias=None, state=None, lengths=None, silu=True, dy=None, dlast=None):
    """-> dict of (ref, mag)."""
    x, weight, bias, state, dy, dlast = map(_d, (x, weight, bias, state, dy, dlast))
    B, L, D = x.shape
    K = weight.shape[1]
    ok = live(lengths, B, L)
    n = torch.full((B,), L) if lengths is None else lengths.cpu().clamp(0, L).long()
    full = torch.zeros(B, K - 1 + L, D, dtype=torch.double)
    full[:, K - 1:] = torch.where(ok, x, torch.zeros((), dtype=torch.double))
    if state is not None:
        full[:, :K - 1] = state
    acc, mag = torch.zeros(B, L, D, dtype=torch.double), torch.zeros(B, L, D, dtype=torch.double)
    for k in range(K):
        acc += full[:, k:k + L] * weight[:, k]
        mag += (full[:, k:k + L] * weight[:, k]).abs()
    if bias is not None:
        acc, mag = acc + bias, mag + bias.abs()
    sg = torch.sigmoid(acc)
    okd = ok.double()
    y = (acc * sg if silu else acc) * okd
    at = n.view(B, 1) + torch.arange(K - 1)
    rows = torch.arange(B).view(B, 1)
    last = full[rows, at]
    out = {"y": (y, (mag + y.abs()) * okd), "last": (last, torch.zeros_like(last))}
    if dy is None and dlast is None:
        return out
    dy = torch.zeros_like(acc) if dy is None else dy
    slope = sg + acc * sg * (1 - sg) if silu else torch.ones_like(acc)
    ds, mds = dy * slope * okd, dy.abs() * (1.1 + mag) * okd
    dfull, mfull = torch.zeros_like(full), torch.zeros_like(full)
    for k in range(K):
        dfull[:, k:k + L] += ds * weight[:, k]
        mfull[:, k:k + L] += mds * weight[:, k].abs()
    if dlast is not None:
        for b in range(B):
            dfull[b, at[b]] += dlast[b]
            mfull[b, at[b]] += dlast[b].abs()
    out["x"] = (dfull[:, K - 1:] * okd, mfull[:, K - 1:] * okd)
    out["state"] = (dfull[:, :K - 1], mfull[:, :K - 1])
    out["bias"] = (ds.sum((0, 1)), mds.sum((0, 1)))
    out["weight"] = tuple(torch.stack([(a * b[:, k:k + L]).sum((0, 1)) for k in range(K)], dim=1)
                          for a, b in ((ds, full), (mds, full.abs())))
    return out


def conv_roundings(K):
    return 4 * K + 24  # K products and sums, sigmoid of a few, its slope


def scan(u, delta, A, B, C, skip=None, delta_bias=None, softplus=True, state=None, lengths=None, dy=None, dlast=None):
    """B, C: (batch, L, G, N) -> dict of (ref, mag)."""
    u, delta, A, B, C, skip, delta_bias, state, dy, dlast = map(
        _d, (u, delta, A, B, C, skip, delta_bias, state, dy, dlast))
    nb, L, D = u.shape
    G, N = B.shape[2:]
    ok = live(lengths, nb, L)
    zero = torch.zeros((), dtype=torch.double)
    raw = torch.where(ok, delta, zero) + (0 if delta_bias is None else delta_bias)
    dt = torch.logaddexp(raw, zero.expand_as(raw)) if softplus else raw
    dt = torch.where(ok, dt, zero)
    u = torch.where(ok, u, zero)
    Bd, Cd = (torch.where(ok.unsqueeze(-1), t, zero).repeat_interleave(D // G, dim=2) for t in (B, C))
    h = torch.zeros(nb, D, N, dtype=torch.double) if state is None else state
    m = h.abs()
    before, mbefore, y, ym = [], [], [], []
    for t in range(L):
        before.append(h)
        mbefore.append(m)
        a, x = torch.exp(dt[:, t, :, None] * A), (dt[:, t] * u[:, t]).unsqueeze(-1) * Bd[:, t]
        h, m = a * h + x, a * m + x.abs()
        y.append((h * Cd[:, t]).sum(-1))
        ym.append((m * Cd[:, t].abs()).sum(-1))
    y, ym = (torch.stack(v, 1) if v else torch.zeros(nb, 0, D, dtype=torch.double) for v in (y, ym))
    if skip is not None:
        y, ym = y + skip * u, ym + (skip * u).abs()
    out = {"y": (y, ym), "last": (h, m)}
    if dy is None and dlast is None:
        return out
    dy = torch.zeros_like(u) if dy is None else torch.where(ok, dy, zero)
    g = torch.zeros(nb, D, N, dtype=torch.double) if dlast is None else dlast
    gm = g.abs()
    names = ("u", "delta", "B", "C")
    r = {k: [] for k in names}
    dA, dAm = torch.zeros_like(A), torch.zeros_like(A)

    def group(v):
        return v.view(nb, G, D // G, N).sum(2)

    for t in range(L - 1, -1, -1):
        a = torch.exp(dt[:, t, :, None] * A)
        du = (dt[:, t] * u[:, t]).unsqueeze(-1)
        back, backm = a * before[t], a * mbefore[t]
        now, nowm = back + du * Bd[:, t], backm + (du * Bd[:, t]).abs()
        dyt = dy[:, t].unsqueeze(-1)
        g, gm = g + dyt * Cd[:, t], gm + (dyt * Cd[:, t]).abs()
        r["C"].append((group(dyt * now), group(dyt.abs() * nowm)))
        r["B"].append((group(g * du), group(gm * du.abs())))
        into, intom = (g * Bd[:, t]).sum(-1), (gm * Bd[:, t].abs()).sum(-1)
        r["u"].append((dt[:, t] * into, dt[:, t].abs() * intom))
        r["delta"].append((u[:, t] * into + (g * back * A).sum(-1),
                           u[:, t].abs() * intom + (gm * backm * A.abs()).sum(-1)))
        dA = dA + (g * back * dt[:, t, :, None]).sum(0)
        dAm = dAm + (gm * backm * dt[:, t, :, None].abs()).sum(0)
        g, gm = g * a, gm * a

    def stack(k, i, shape):
        v = [e[i] for e in reversed(r[k])]
        return torch.stack(v, 1) if v else torch.zeros(shape, dtype=torch.double)

    for k in names:
        shape = (nb, 0, D) if k in ("u", "delta") else (nb, 0, G, N)
        out[k] = [stack(k, 0, shape), stack(k, 1, shape)]
    if skip is not None:
        out["u"] = [out["u"][0] + skip * dy, out["u"][1] + (skip * dy).abs()]
    slope = (torch.sigmoid(raw) if softplus else torch.ones_like(raw)) * ok.double()
    out["delta"] = [v * slope for v in out["delta"]]
    out["delta_bias"] = tuple(v.sum((0, 1)) for v in out["delta"])
    out["A"] = (dA, dAm)
    out["skip"] = ((dy * u).sum((0, 1)), (dy * u).abs().sum((0, 1)))
    out["state"] = (g, gm)
    return out


def scan_roundings(L, N):
    # four a step along the recurrence (decay, its argument, product, sum), N
    # for the sum over states, step size and decay's argument: a relative error
    # of some 16 u in dt A, weighed by exp(-|dt A|), stays under 64 u in all
    return 4 * L + N + 64


def norm(x, gate=None, post=None, residual=None, scale=None, pre=None, eps=1e-5, dy=None, dh=None):
    """-> dict of (ref, mag); absent results are left out."""
    x, gate, post, residual, scale, pre, dy, dh = map(_d, (x, gate, post, residual, scale, pre, dy, dh))
    one = torch.ones(x.shape[-1], dtype=torch.double)
    sg = torch.sigmoid(gate) if gate is not None else None
    p0 = x * gate * sg if gate is not None else x
    inv1 = 1 / torch.sqrt((p0 ** 2).mean(-1, keepdim=True) + eps) if post is not None else torch.ones_like(x[..., :1])
    n1 = p0 * inv1
    w1, s = one if post is None else post, one if scale is None else scale
    p = n1 * w1
    out = {}
    if residual is None:
        out["y"] = (p, p.abs())
    else:
        h, hm = residual + s * p, residual.abs() + (s * p).abs()
        out["h"] = (h, hm)
        if pre is not None:
            inv2 = 1 / torch.sqrt((h ** 2).mean(-1, keepdim=True) + eps)
            # an error in h reaches y directly and through the row's norm
            shift = inv2 ** 2 * (h.abs() * hm).mean(-1, keepdim=True)
            n2, n2m = h * inv2, hm * inv2 + h.abs() * inv2 * shift
            out["y"] = (n2 * pre, n2m * pre.abs())
    if dy is None and dh is None:
        return out
    flat = tuple(range(x.dim() - 1))
    if residual is None:
        d, dm = dy, dy.abs()
    else:
        d = torch.zeros_like(x) if dh is None else dh
        dm = d.abs()
        if pre is not None:
            t = (torch.zeros_like(x) if dy is None else dy) * pre
            dot, dotm = (t * n2).mean(-1, keepdim=True), (t.abs() * n2m).mean(-1, keepdim=True)
            out["pre"] = ((t / pre * n2).sum(flat), ((t / pre).abs() * n2m).sum(flat))
            d = d + inv2 * (t - n2 * dot)
            dm = dm + inv2 * (1 + shift) * (t.abs() + 2 * n2m * dotm)
        out["residual"] = (d, dm)
        if scale is not None:
            out["scale"] = ((d * p).sum(flat), (dm * p.abs()).sum(flat))
        d, dm = d * s, dm * s.abs()
    if post is not None:
        out["post"] = ((d * n1).sum(flat), (dm * n1.abs()).sum(flat))
        q, qm = d * w1, dm * w1.abs()
        d = inv1 * (q - n1 * (q * n1).mean(-1, keepdim=True))
        dm = inv1 * (qm + n1.abs() * (qm * n1.abs()).mean(-1, keepdim=True))
    out["x"] = (d, dm)
    if gate is not None:
        si = gate * sg
        out["x"] = (d * si, dm * si.abs())
        slope, slopem = sg + si * (1 - sg), sg + (si * (1 - sg)).abs()
        out["gate"] = (d * x * slope, dm * x.abs() * slopem)
    return out


def norm_roundings(D):
    # a mean of D squares or products, added in any order (at most D roundings;
    # lanes and chunks make it D / 64 + 32, the plain form pairwise), and the
    # factors of both norms and the gate
    return D / 64 + 96
