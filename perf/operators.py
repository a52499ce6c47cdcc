"""Timed cases of the sequence-mixing operators: short causal convolution,
selective state space scan, and the norms around a block with its gate and
residual scale — each for whole sequences, for training and, where a state is
carried, for one new token.

``run`` with ``own`` false computes the plain form from elementary torch
operations in 32 bits; with ``own`` true it makes the calls a user makes of
``mpgcn_amd.ops``. ``exact`` states the same results from the definitions in
64 bits, gradients by the adjoint recurrences rather than by autograd.
"""

from __future__ import annotations

import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "f32": torch.float32}
_EPS = 1e-5
# work bounds of a drawn case, in elements: B*L*D and B*L*D*N
_MAX_ELEMS = 1 << 26
_MAX_STATES = 900_000_000


def listed():
    return [
        # one new token of one sequence: nothing but latency
        dict(name="conv_step_one", op="conv", mode="step", dtype="bf16", B=1, L=1, D=1024, K=4),
        # training over every OD pair's weekly window (batch 32, 47 regions, hidden 32)
        dict(name="conv_train_od", op="conv", mode="train", dtype="f32", B=70688, L=7, D=32, K=4,
             bias=True, state=False, lengths=False),
        # a long prompt at a generic model width
        dict(name="conv_prompt_long", op="conv", mode="prompt", dtype="bf16", B=1, L=16384, D=4096, K=4,
             bias=True, state=False, lengths=False),
        # one new token of one sequence, and of a served batch of them
        dict(name="scan_step_one", op="scan", mode="step", dtype="bf16", B=1, L=1, D=1024, N=16, G=1),
        dict(name="scan_step_batch", op="scan", mode="step", dtype="bf16", B=256, L=1, D=4096, N=16, G=1),
        # training over every OD pair's window at the flagship's 256 regions (batch 4, hidden 32)
        dict(name="scan_train_od", op="scan", mode="train", dtype="bf16", B=262144, L=7, D=32, N=16, G=1,
             state=False, lengths=False),
        # ordinary training: few sequences of middle length
        dict(name="scan_train_mid", op="scan", mode="train", dtype="bf16", B=2, L=1024, D=1536, N=16, G=1,
             state=False, lengths=False),
        # the largest: one long prompt, whose time axis has to fill the card
        dict(name="scan_prompt_long", op="scan", mode="prompt", dtype="bf16", B=1, L=16384, D=2048, N=16, G=1,
             state=True, lengths=False),
        # a padded batch of odd sizes in two groups, one row without a token
        dict(name="scan_train_ragged", op="scan", mode="train", dtype="f32", B=3, L=389, D=198, N=13, G=2,
             state=True, lengths=True),
        # the block's norms for one token: latency again
        dict(name="norm_one", op="norm", mode="prompt", dtype="bf16", R=1, D=1024,
             gate=True, post=True, residual="f32", scale=True, pre=True),
        # training: norms on both sides of a block, float32 residual stream
        dict(name="norm_train", op="norm", mode="train", dtype="bf16", R=8192, D=2560,
             gate=False, post=True, residual="f32", scale=True, pre=True),
        # training: the gated norm behind the scan, narrow rows in the flagship's number
        dict(name="norm_train_od", op="norm", mode="train", dtype="bf16", R=1835008, D=32,
             gate=True, post=True, residual="", scale=False, pre=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["conv", "scan", "scan", "norm"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if op == "norm":
        D = _log(rng, 16, 8192)
        post = rng.random() < 0.7
        res = rng.choice(["", "f32", dtype]) if post else rng.choice(["f32", dtype])
        return dict(op=op, mode=rng.choice(["prompt", "train"]), dtype=dtype,
                    R=_log(rng, 1, max(1, _MAX_ELEMS // D)), D=D, gate=rng.random() < 0.5, post=post,
                    residual=res, scale=bool(res) and rng.random() < 0.5,
                    pre=bool(res) and (not post or rng.random() < 0.7))
    mode = rng.choice(["step", "prompt", "train", "train"])
    if op == "conv":
        D, K = _log(rng, 16, 6144), rng.choice([2, 3, 4, 4])
        if mode == "step":
            return dict(op=op, mode=mode, dtype=dtype, B=_log(rng, 1, 512), L=1, D=D, K=K)
        L = _log(rng, 1, 16384)
        return dict(op=op, mode=mode, dtype=dtype, B=_log(rng, 1, max(1, _MAX_ELEMS // (D * L))), L=L, D=D, K=K,
                    bias=rng.random() < 0.7, state=rng.random() < 0.4, lengths=rng.random() < 0.4)
    G = rng.choice([1, 1, 1, 2, 4])
    D, N = G * _log(rng, 16, 4096 // G), rng.choice([4, 8, 13, 16, 16, 16, 24, 32, 64])
    if mode == "step":
        return dict(op=op, mode=mode, dtype=dtype, B=_log(rng, 1, max(1, min(512, _MAX_ELEMS // (D * N)))), L=1,
                    D=D, N=N, G=G)
    # the plain form goes step by step over the length
    L = min(_log(rng, 1, 16384 if mode == "prompt" else 2048), max(1, _MAX_STATES // (2 * D * N)))
    return dict(op=op, mode=mode, dtype=dtype, B=_log(rng, 1, max(1, _MAX_STATES // (2 * D * N * L))), L=L, D=D,
                N=N, G=G, state=rng.random() < 0.4, lengths=rng.random() < 0.4)


# ---- inputs -----------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt = _DT[case["dtype"]]

    def randn(*shape, dtype=torch.float32, scale=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)

    def rand(*shape):
        return torch.rand(*shape, generator=g, device="cuda")

    s = dict(case=case)
    train = case["mode"] == "train"
    if case["op"] == "norm":
        R, D = case["R"], case["D"]
        s["x"] = randn(R, D, dtype=dt)
        s["gate"] = randn(R, D, dtype=dt) if case["gate"] else None
        s["post_weight"] = 1 + randn(D, scale=0.1) if case["post"] else None
        s["residual"] = randn(R, D, dtype=_DT[case["residual"]], scale=2.0) if case["residual"] else None
        s["scale"] = 0.5 + randn(D, scale=0.1) if case["scale"] else None
        s["pre_weight"] = 1 + randn(D, scale=0.1) if case["pre"] else None
        s["leaves"] = ["x", "gate", "post_weight", "residual", "scale", "pre_weight"]
        s["douts"] = []
        if train:
            if case["pre"] or not case["residual"]:
                s["douts"].append(randn(R, D, dtype=dt))
            if case["residual"]:
                s["douts"].append(randn(R, D, dtype=_DT[case["residual"]]))
    elif case["op"] == "conv":
        B, L, D, K = (case[k] for k in "BLDK")
        shape = (B, D) if case["mode"] == "step" else (B, L, D)
        s["x"] = randn(*shape, dtype=dt)
        s["weight"] = (rand(D, K) * 2 - 1) / math.sqrt(K)
        s["bias"] = randn(D, scale=0.1) if case.get("bias", True) else None
        s["state"] = (randn(B, K - 1, D, dtype=dt)
                      if case["mode"] == "step" or case["state"] else None)
        if case["mode"] == "step":
            s["state_out"] = torch.empty_like(s["state"])
        s["leaves"] = ["x", "weight", "bias", "state"]
        s["douts"] = [randn(*shape, dtype=dt)] if train else []
    else:
        B, L, D, N, G = (case[k] for k in "BLDNG")
        step = case["mode"] == "step"
        lead = (B,) if step else (B, L)
        s["u"] = torch.nn.functional.silu(randn(*lead, D)).to(dt)
        s["delta"] = randn(*lead, D, dtype=dt, scale=0.5)
        s["B"] = randn(*lead, G, N, dtype=dt)
        s["C"] = randn(*lead, G, N, dtype=dt)
        s["A"] = -(torch.arange(1, N + 1, device="cuda") * torch.exp(randn(D, N, scale=0.1)))
        s["skip"] = 1 + randn(D, scale=0.1)
        # softplus(delta_bias) spread over 1e-3 .. 1e-1
        first = torch.exp(rand(D) * math.log(100.0) + math.log(1e-3))
        s["delta_bias"] = first + torch.log(-torch.expm1(-first))
        s["state"] = randn(B, D, N) if step or case["state"] else None
        if step:
            s["state_out"] = torch.empty_like(s["state"])
        s["leaves"] = ["u", "delta", "A", "B", "C", "skip", "delta_bias", "state"]
        s["douts"] = [randn(B, L, D, dtype=dt), randn(B, D, N, scale=0.1)] if train else []
    if case.get("lengths"):
        n = torch.randint(1, case["L"] + 1, (case["B"],), generator=g, device="cuda", dtype=torch.int32)
        n[0] = case["L"]
        n[-1] = 0 if case["B"] > 1 else case["L"]
        s["lengths"] = n
    else:
        s["lengths"] = None
    s["leaves"] = [k for k in s["leaves"] if s[k] is not None]
    if train:
        for k in s["leaves"]:
            s[k].requires_grad_(True)
    return s


# ---- one pass ---------------------------------------------------------------

def run(state):
    case = state["case"]
    train = case["mode"] == "train"
    with torch.set_grad_enabled(train):
        outs = (_own if own else _plain)(state)
        if not train:
            return outs
        through = [v for v in outs.values() if v.requires_grad]
        grads = torch.autograd.grad(through, [state[k] for k in state["leaves"]], state["douts"])
    res = {k: v.detach() for k, v in outs.items()}
    res.update(("d_" + k, v) for k, v in zip(state["leaves"], grads))
    return res


def _own(s):
    from mpgcn_amd import ops

    case = s["case"]
    if case["op"] == "norm":
        out = ops.norm_gate_residual(s["x"], gate=s["gate"], post_weight=s["post_weight"], residual=s["residual"],
                                     scale=s["scale"], pre_weight=s["pre_weight"], eps=_EPS)
        if case["pre"]:
            return {"y": out[0], "h": out[1]}
        return {"h" if case["residual"] else "y": out}
    if case["op"] == "conv":
        if case["mode"] == "step":
            y, st = ops.short_conv_step(s["x"], s["state"], s["weight"], s["bias"], state_out=s["state_out"])
            return {"y": y, "state": st}
        if case["mode"] == "train":
            return {"y": ops.short_conv(s["x"], s["weight"], s["bias"], state=s["state"], lengths=s["lengths"])}
        y, st = ops.short_conv(s["x"], s["weight"], s["bias"], state=s["state"], lengths=s["lengths"],
                               return_state=True)
        return {"y": y, "state": st}
    if case["mode"] == "step":
        y, st = ops.selective_scan_step(s["u"], s["delta"], s["A"], s["B"], s["C"], s["state"], s["skip"],
                                        delta_bias=s["delta_bias"], delta_softplus=True, state_out=s["state_out"])
        return {"y": y, "state": st}
    y, st = ops.selective_scan(s["u"], s["delta"], s["A"], s["B"], s["C"], s["skip"], delta_bias=s["delta_bias"],
                               delta_softplus=True, state=s["state"], lengths=s["lengths"], return_state=True)
    return {"y": y, "state": st}


def _valid(s, L):
    """(B, L, 1) truth values of the tokens that count, or None for all."""
    if s["lengths"] is None:
        return None
    return (torch.arange(L, device="cuda") < s["lengths"].unsqueeze(1)).unsqueeze(-1)


def _plain(s):
    case = s["case"]
    dt = _DT[case["dtype"]]
    f = {k: (v.float() if torch.is_tensor(v) and v.is_floating_point() else v) for k, v in s.items()}
    if case["op"] == "norm":
        p = f["x"]
        if case["gate"]:
            p = p * (f["gate"] * torch.sigmoid(f["gate"]))
        if case["post"]:
            p = p * torch.rsqrt((p * p).mean(-1, keepdim=True) + _EPS) * f["post_weight"]
        if not case["residual"]:
            return {"y": p.to(dt)}
        h = f["residual"] + (p * f["scale"] if case["scale"] else p)
        out = {"h": h.to(_DT[case["residual"]])}
        if case["pre"]:
            y = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + _EPS) * f["pre_weight"]
            out = {"y": y.to(dt), "h": out["h"]}
        return out
    if case["op"] == "conv":
        B, L, D, K = (case[k] for k in "BLDK")
        x = f["x"].view(B, L, D)
        ok = _valid(s, L)
        if ok is not None:
            x = torch.where(ok, x, torch.zeros((), device="cuda"))
        before = f["state"] if f["state"] is not None else x.new_zeros(B, K - 1, D)
        xp = torch.cat([before, x], dim=1)
        acc = sum(xp[:, k:k + L] * f["weight"][:, k] for k in range(K))
        if f["bias"] is not None:
            acc = acc + f["bias"]
        y = acc * torch.sigmoid(acc)
        if ok is not None:
            y = torch.where(ok, y, torch.zeros((), device="cuda"))
        y = y.to(dt)
        if case["mode"] == "train":
            return {"y": y}
        if s["lengths"] is None:
            st = xp[:, L:]
        else:
            at = s["lengths"].long().unsqueeze(1) + torch.arange(K - 1, device="cuda")
            st = xp.gather(1, at.unsqueeze(-1).expand(B, K - 1, D))
        st = st.to(dt)
        if case["mode"] == "step":
            return {"y": y.view(B, D), "state": s["state_out"].copy_(st)}
        return {"y": y, "state": st}
    B, L, D, N, G = (case[k] for k in "BLDNG")
    u, delta = f["u"].view(B, L, D), f["delta"].view(B, L, D) + f["delta_bias"]
    Bm, Cm = f["B"].view(B, L, G, N), f["C"].view(B, L, G, N)
    step = torch.clamp(delta, min=0) + torch.log1p(torch.exp(-delta.abs()))
    ok = _valid(s, L)
    if ok is not None:
        step = torch.where(ok, step, torch.zeros((), device="cuda"))
    # (B, L, D, N): decay and input of every state, then the recurrence
    decay = torch.exp(step.unsqueeze(-1) * f["A"])
    drive = ((step * u).view(B, L, G, D // G, 1) * Bm.unsqueeze(3)).view(B, L, D, N)
    h = f["state"] if f["state"] is not None else u.new_zeros(B, D, N)
    hs = []
    for a, x in zip(decay.unbind(1), drive.unbind(1)):
        h = a * h + x
        hs.append(h)
    del decay, drive
    hs = torch.stack(hs, dim=1).view(B, L, G, D // G, N)
    y = (hs * Cm.unsqueeze(3)).sum(-1).view(B, L, D) + f["skip"] * u
    if ok is not None:
        y = torch.where(ok, y, torch.zeros((), device="cuda"))
    y = y.to(dt)
    if case["mode"] == "step":
        return {"y": y.view(B, D), "state": s["state_out"].copy_(h)}
    return {"y": y, "state": h}


# ---- the work that no form can do without -----------------------------------

def work(case):
    e = 2 if case["dtype"] == "bf16" else 4
    train = case["mode"] == "train"
    if case["op"] == "norm":
        n = case["R"] * case["D"]
        er = {"": 0, "f32": 4, "bf16": 2}[case["residual"]]
        ins = e + (e if case["gate"] else 0) + er
        outs = (e if case["pre"] or not er else 0) + er
        per = 4 * case["gate"] + 4 * case["post"] + 2 * bool(er) + 4 * case["pre"]
        # training reads the outputs' gradients too and writes the inputs'
        return {"bytes": n * (ins + outs) * (2 if train else 1), "flops": n * per * (3 if train else 1)}
    B, L, D = case["B"], case["L"], case["D"]
    n = B * L * D
    if case["op"] == "conv":
        K = case["K"]
        st = B * (K - 1) * D * e * (2 if case["mode"] == "step" else 1 if case.get("state") else 0)
        return {"bytes": n * e * (4 if train else 2) + st + D * (K + 1) * 4 * (2 if train else 1),
                "flops": n * (2 * K + 4) * (3 if train else 1)}
    N, G = case["N"], case["G"]
    st = B * D * N * 4 * (2 if case["mode"] == "step" or case.get("state") else 1)
    bc = 2 * B * L * G * N * e
    return {"bytes": (n * e * 3 + bc) * (2 if train else 1) + st * (2 if train else 1) + D * (N + 2) * 4,
            "flops": n * N * (22 if train else 7) + n * 10}


# ---- the definition in 64 bits ----------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    train = case["mode"] == "train"
    w = {k: (v.detach().double() if torch.is_tensor(v) and v.is_floating_point() else v) for k, v in s.items()}
    dout = [d.double() for d in s["douts"]]
    with torch.no_grad():
        out = {"norm": _exact_norm, "conv": _exact_conv, "scan": _exact_scan}[case["op"]](case, w, dout, train)
    res = out[0]
    if train:
        res.update(("d_" + k, out[1][k]) for k in s["leaves"])
    return res


def _rms_back(x, inv, weight, dy):
    """Gradients of x * inv * weight, inv = rsqrt(mean(x^2) + eps)."""
    t = dy * weight
    dx = inv * (t - x * inv * inv * (t * x).mean(-1, keepdim=True))
    return dx, (dy * x * inv).sum(0)


def _exact_norm(case, w, dout, train):
    gate_s = 1 / (1 + torch.exp(-w["gate"])) if case["gate"] else None
    x1 = w["x"] * w["gate"] * gate_s if case["gate"] else w["x"]
    p, inv1 = x1, None
    if case["post"]:
        inv1 = 1 / torch.sqrt((x1 ** 2).sum(-1, keepdim=True) / case["D"] + _EPS)
        p = x1 * inv1 * w["post_weight"]
    res = {}
    if not case["residual"]:
        res["y"] = p
    else:
        h = w["residual"] + (w["scale"] * p if case["scale"] else p)
        if case["pre"]:
            inv2 = 1 / torch.sqrt((h ** 2).sum(-1, keepdim=True) / case["D"] + _EPS)
            res["y"] = h * inv2 * w["pre_weight"]
        res["h"] = h
    if not train:
        return res, None
    gr = {}
    if case["residual"]:
        dh = dout[-1]
        if case["pre"]:
            more, gr["pre_weight"] = _rms_back(h, inv2, w["pre_weight"], dout[0])
            dh = dh + more
        gr["residual"] = dh
        dp = dh
        if case["scale"]:
            gr["scale"] = (dh * p).sum(0)
            dp = dh * w["scale"]
    else:
        dp = dout[0]
    if case["post"]:
        dp, gr["post_weight"] = _rms_back(x1, inv1, w["post_weight"], dp)
    gr["x"] = dp
    if case["gate"]:
        gr["x"] = dp * w["gate"] * gate_s
        gr["gate"] = dp * w["x"] * (gate_s + w["gate"] * gate_s * (1 - gate_s))
    return res, gr


def _exact_conv(case, w, dout, train):
    B, L, D, K = (case[k] for k in "BLDK")
    x = w["x"].view(B, L, D)
    lens = w["lengths"].tolist() if w["lengths"] is not None else None
    live = x.new_ones(B, L, 1)
    if lens is not None:
        live = (torch.arange(L, device=x.device).expand(B, L) < w["lengths"].view(B, 1)).unsqueeze(-1).double()
    x = x * live
    full = x.new_zeros(B, K - 1 + L, D)
    full[:, K - 1:] = x
    if w["state"] is not None:
        full[:, :K - 1] = w["state"]
    win = full.unfold(1, K, 1)  # (B, L, D, K)
    acc = torch.zeros_like(x)
    for k in range(K):
        acc += win[..., k] * w["weight"][:, k]
    if w["bias"] is not None:
        acc += w["bias"]
    sg = 1 / (1 + torch.exp(-acc))
    res = {"y": (acc * sg * live).view(w["x"].shape)}
    if not train:
        if lens is None:
            res["state"] = full[:, L:].clone()
        else:
            pick = w["lengths"].long().view(B, 1) + torch.arange(K - 1, device=x.device)
            res["state"] = full[torch.arange(B, device=x.device).view(B, 1), pick]
        return res, None
    ds = dout[0] * live * (sg + acc * sg * (1 - sg))
    dfull = torch.zeros_like(full)
    for k in range(K):
        dfull[:, k:k + L] += ds * w["weight"][:, k]
    gr = {"x": dfull[:, K - 1:] * live, "state": dfull[:, :K - 1], "bias": ds.sum((0, 1)),
          "weight": torch.stack([(ds * win[..., k]).sum((0, 1)) for k in range(K)], dim=1)}
    return res, gr


def _exact_scan(case, w, dout, train):
    B, L, D, N, G = (case[k] for k in "BLDNG")
    per = D // G
    u, raw = w["u"].view(B, L, D), w["delta"].view(B, L, D) + w["delta_bias"]
    Bm, Cm = w["B"].view(B, L, G, 1, N), w["C"].view(B, L, G, 1, N)
    A = w["A"].view(G, per, N)
    dt = torch.logaddexp(raw, torch.zeros_like(raw))
    live = u.new_ones(B, L, 1)
    if w["lengths"] is not None:
        live = (torch.arange(L, device=u.device).expand(B, L) < w["lengths"].view(B, 1)).unsqueeze(-1).double()
    dt = (dt * live).view(B, L, G, per, 1)
    ug = u.view(B, L, G, per, 1)
    h0 = w["state"].view(B, G, per, N) if w["state"] is not None else u.new_zeros(B, G, per, N)
    hist, h = [], h0
    y = u.new_zeros(B, L, G, per)
    for t in range(L):
        if train:
            hist.append(h)
        h = torch.exp(dt[:, t] * A) * h + dt[:, t] * ug[:, t] * Bm[:, t]
        y[:, t] = (h * Cm[:, t]).sum(-1)
    y = (y.view(B, L, D) + w["skip"] * u) * live
    res = {"y": y.view(w["u"].shape), "state": h.reshape(B, D, N)}
    if not train:
        return res, None
    dy = (dout[0] * live).view(B, L, G, per, 1)
    g = dout[1].view(B, G, per, N)
    du, ddt = u.new_zeros(B, L, G, per), u.new_zeros(B, L, G, per)
    dB, dC = torch.zeros_like(Bm[:, :, :, 0]), torch.zeros_like(Bm[:, :, :, 0])
    dA = torch.zeros_like(A)
    for t in range(L - 1, -1, -1):
        a, prev = torch.exp(dt[:, t] * A), hist.pop()
        now = a * prev + dt[:, t] * ug[:, t] * Bm[:, t]
        dC[:, t] = (dy[:, t] * now).sum(2)
        g = g + dy[:, t] * Cm[:, t]
        into = (g * Bm[:, t]).sum(-1)
        dB[:, t] = (g * dt[:, t] * ug[:, t]).sum(2)
        du[:, t] = into * dt[:, t, ..., 0]
        back = g * a * prev
        ddt[:, t] = into * ug[:, t, ..., 0] + (back * A).sum(-1)
        dA += (back * dt[:, t]).sum(0)
        g = g * a
    draw_ = ddt.view(B, L, D) * live / (1 + torch.exp(-raw))
    dyf = dy.reshape(B, L, D)
    gr = {"u": du.view(B, L, D) + w["skip"] * dyf, "delta": draw_, "A": dA.view(D, N),
          "B": dB.view(w["B"].shape), "C": dC.view(w["C"].shape), "skip": (dyf * u).sum((0, 1)),
          "delta_bias": draw_.sum((0, 1)), "state": g.reshape(B, D, N)}
    return res, gr
