"""Eager (pure-PyTorch) implementations of the core ops.

These serve two roles:
  1. CPU execution path (this framework runs end-to-end without a GPU, e.g. the
     16-region plumbing config of BASELINE.json).
  2. The reference math for unit tests of the HIP kernels.

The BDGCN layer here uses the *factored* algorithm (see ``bdgcn_layer_eager``):
algebraically identical to the reference's K^2-pair formulation (MPGCN.py:24-50)
but with K mode-1 + K mode-2 axis products instead of K^2 of each — a ~3x FLOP
reduction at K = 3. The HIP path implements the same factorization.

Derivation. The reference computes, for every support pair (o, s):
    Z_{o,s}[b,m,d,l] = sum_c Gd[s,c,d] * (sum_n Go[o,n,m] * X[b,n,c,l])
then concatenates over (o, s) on the channel axis and projects:
    H[b,m,d,h] = sum_{o,s,l} Z_{o,s}[b,m,d,l] * W[(o*K+s)*C + l, h]        (+ bias, act)
Since the destination-axis product and the projection are both linear, swap them:
    U_o[b,m,c,l]   = sum_n Go[o,n,m] * X[b,n,c,l]                  (K mode-1 products)
    V_s[b,m,c,h]   = sum_{o,l} U_o[b,m,c,l] * W[(o*K+s)*C + l, h]  (one flat GEMM)
    H[b,m,d,h]     = sum_{s,c} Gd[s,c,d] * V_s[b,m,c,h]            (K mode-2 products)
which is exactly H above, term for term.
"""

from __future__ import annotations

import torch


def reorder_projection_weight(W: torch.Tensor, S: int, C: int) -> torch.Tensor:
    """(C*S*S, H) reference-layout W -> (S*C, S*H) factored-layout Wre.

    Reference row index k = (o*S + s)*C + l (concat order of MPGCN.py:28-44);
    Wre[o*C + l, s*H + h] = W[(o*S + s)*C + l, h].
    """
    H = W.shape[1]
    return W.view(S, S, C, H).permute(0, 2, 1, 3).reshape(S * C, S * H)


def mode1_apply(X: torch.Tensor, G: torch.Tensor) -> torch.Tensor:
    """Origin-axis graph product. X:(B,N,N,C), G:(S,N,N) or (B,S,N,N).

    U[b,m,d,o,l] = sum_n G[(b,)o,n,m] X[b,n,d,l]; output layout (B, N, N, S, C)
    so that (o, l) is the contiguous trailing pair the projection GEMM consumes.
    """
    if G.dim() == 3:
        return torch.einsum("onm,bndl->bmdol", G, X)
    return torch.einsum("bonm,bndl->bmdol", G, X)


def mode2_apply(V: torch.Tensor, G: torch.Tensor) -> torch.Tensor:
    """Destination-axis graph product summed over supports.

    V:(B,N,N,S,H), G:(S,N,N) or (B,S,N,N);
    Y[b,m,d,h] = sum_{s,c} G[(b,)s,c,d] V[b,m,c,s,h].
    """
    if G.dim() == 3:
        return torch.einsum("scd,bmcsh->bmdh", G, V)
    return torch.einsum("bscd,bmcsh->bmdh", G, V)


def bdgcn_layer_eager(
    X: torch.Tensor,
    Go: torch.Tensor,
    Gd: torch.Tensor,
    W: torch.Tensor,
    bias: torch.Tensor | None,
    activation: str = "relu",
) -> torch.Tensor:
    """Full 2-D GCN layer (factored algorithm). See module docstring.

    X: (B, N, N, C); Go/Gd: (S, N, N) static or (B, S, N, N) dynamic;
    W: (C*S*S, H) in the reference's concat layout; bias: (H,) or None.
    """
    S = Go.shape[-3]
    C = X.shape[-1]
    B, N = X.shape[0], X.shape[1]
    Hdim = W.shape[1]

    U = mode1_apply(X, Go)  # (B, N, N, S, C)
    Wre = reorder_projection_weight(W, S, C)
    V = (U.reshape(B * N * N, S * C) @ Wre).view(B, N, N, S, Hdim)
    Y = mode2_apply(V, Gd)
    if bias is not None:
        Y = Y + bias
    if activation == "relu":
        Y = torch.relu(Y)
    elif activation not in (None, "none", "linear"):
        raise ValueError(f"unsupported activation {activation!r}")
    return Y


def lstm_forward_eager(
    x: torch.Tensor,
    w_ih: torch.Tensor,
    w_hh: torch.Tensor,
    b_ih: torch.Tensor,
    b_hh: torch.Tensor,
    h0: torch.Tensor | None = None,
    c0: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Single-layer batch-first LSTM, torch gate order (i, f, g, o).

    x: (R, T, I); w_ih: (4H, I); w_hh: (4H, H). Returns (out (R,T,H), h_T, c_T).
    Matches nn.LSTM(num_layers=1, batch_first=True) numerics.
    """
    R, T, _ = x.shape
    Hd = w_hh.shape[1]
    h = x.new_zeros(R, Hd) if h0 is None else h0
    c = x.new_zeros(R, Hd) if c0 is None else c0
    bias = b_ih + b_hh
    outs = []
    for t in range(T):
        gates = x[:, t, :] @ w_ih.t() + h @ w_hh.t() + bias
        i, f, g, o = gates.chunk(4, dim=1)
        i, f, o = torch.sigmoid(i), torch.sigmoid(f), torch.sigmoid(o)
        g = torch.tanh(g)
        c = f * c + i * g
        h = o * torch.tanh(c)
        outs.append(h)
    return torch.stack(outs, dim=1), h, c


# ---- sequence operators -----------------------------------------------------
# The definitions of mpgcn_amd/ops/sequence.py in elementary operations: f32
# (f64 for f64 inputs) inside, rounded once to the output's type.


def _wide(*tensors):
    dt = torch.float64 if any(t is not None and t.dtype == torch.float64 for t in tensors) else torch.float32
    return [None if t is None else t.to(dt) for t in tensors]


def valid_tokens(lengths: torch.Tensor | None, L: int) -> torch.Tensor | None:
    """(B, L, 1) truth values of the tokens before each sequence's end."""
    if lengths is None:
        return None
    return (torch.arange(L, device=lengths.device) < lengths.unsqueeze(1)).unsqueeze(-1)


def short_conv_eager(x, weight, bias, state, lengths, silu):
    """-> (y (B, L, D), final state (B, K-1, D)), both of x's type."""
    B, L, D = x.shape
    K = weight.shape[1]
    xw, w, b, s = _wide(x, weight, bias, state)
    zero = xw.new_zeros(())
    ok = valid_tokens(lengths, L)
    if ok is not None:
        xw = torch.where(ok, xw, zero)
    xp = torch.cat([xw.new_zeros(B, K - 1, D) if s is None else s, xw], dim=1)
    acc = sum(xp[:, k:k + L] * w[:, k] for k in range(K))
    if b is not None:
        acc = acc + b
    y = acc * torch.sigmoid(acc) if silu else acc
    if ok is not None:
        y = torch.where(ok, y, zero)
    if lengths is None:
        last = xp[:, L:]
    else:
        at = lengths.clamp(0, L).long().unsqueeze(1) + torch.arange(K - 1, device=x.device)
        last = xp.gather(1, at.unsqueeze(-1).expand(B, K - 1, D))
    return y.to(x.dtype), last.to(x.dtype).contiguous()


def selective_scan_eager(u, delta, A, B, C, skip, delta_bias, softplus, state, lengths):
    """B, C: (batch, L, G, N) -> (y (batch, L, D) of u's type, final state (batch, D, N))."""
    nb, L, D = u.shape
    G, N = B.shape[2], B.shape[3]
    uw, dw, Aw, Bw, Cw, sk, db, h = _wide(u, delta, A, B, C, skip, delta_bias, state)
    zero = uw.new_zeros(())
    step = dw if db is None else dw + db
    if softplus:
        step = step.clamp(min=0) + torch.log1p(torch.exp(-step.abs()))
    ok = valid_tokens(lengths, L)
    if ok is not None:
        step, uw = torch.where(ok, step, zero), torch.where(ok, uw, zero)
        Bw, Cw = (torch.where(ok.unsqueeze(-1), t, zero) for t in (Bw, Cw))
    h = uw.new_zeros(nb, D, N) if h is None else h.clone()
    ys = []
    for t in range(L):
        dt = step[:, t].unsqueeze(-1)
        Bt, Ct = (v[:, t].repeat_interleave(D // G, dim=1) for v in (Bw, Cw))
        h = torch.exp(dt * Aw) * h + dt * uw[:, t].unsqueeze(-1) * Bt
        ys.append((h * Ct).sum(-1))
    y = torch.stack(ys, dim=1) if ys else uw.new_zeros(nb, 0, D)
    if sk is not None:
        y = y + sk * uw
    return y.to(u.dtype), h


def norm_gate_residual_eager(x, gate, post_weight, residual, scale, pre_weight, eps):
    """-> (y or None, h or None)."""
    p, g, w1, r, s, w2 = _wide(x, gate, post_weight, residual, scale, pre_weight)
    if g is not None:
        p = p * (g * torch.sigmoid(g))
    if w1 is not None:
        p = p * torch.rsqrt((p * p).mean(-1, keepdim=True) + eps) * w1
    if r is None:
        return p.to(x.dtype), None
    h = r + (p if s is None else p * s)
    y = None
    if w2 is not None:
        y = (h * torch.rsqrt((h * h).mean(-1, keepdim=True) + eps) * w2).to(x.dtype)
    return y, h.to(residual.dtype)
