"""Operators that mix a sequence over time, and the norms around such a block.

    y        = short_conv(x, weight, bias)                      # few taps, causal
    y        = selective_scan(u, delta, A, B, C, skip)          # state space scan
    y        = norm_gate_residual(y, gate=z, post_weight=w)     # norm of y * silu(z)
    n, h     = norm_gate_residual(o, residual=r, scale=s, pre_weight=w)

Whole sequences are (batch, length, channels) with the channels contiguous;
batch and time may have any stride, so slices of one projection's output go in
without a copy. ``lengths`` (batch,) int32 or int64 on the same device gives
the valid tokens of a right-padded batch, zero included; values outside
[0, length] are held to it. What is past them is never read into a result:
outputs and gradients there are zero and the state is the one at the end.

``state``/``return_state`` carry a sequence over calls, and the ``_step`` forms
take one new token per sequence: they update ``state`` in place (or write
``state_out``) and have no gradient.

Activations are bf16 or f32 (f64 on CPU, for reference runs). Parameters are
the f32 masters; another floating type is converted. Sums, states and norms
are f32, each output is rounded once. Gradients of parameters and of B and C
are added in a fixed order: the same call gives the same bits. On a GPU
forward-mode derivatives and calls inside torch.jit.trace are refused.

Work is queued on the current stream of the inputs' device. On a GPU the HIP
kernels run; on CPU the definitions in mpgcn_amd/ops/eager.py.

A training call may be captured into a graph. It is refused during capture if
an eager graph of the same leaves is still alive on another stream, since the
captured backward would have to wait for that stream.
"""

from __future__ import annotations

import torch
from mpgcn_amd import ops as _ops
from mpgcn_amd.ops import eager

_MAX_STATES = 64
_MAX_NORM_D = 16384
_MIN_EPS = torch.finfo(torch.float32).tiny
_MAX_SCAN_D = (1 << 26) - 4  # where every channel is a group: a wave each in one launch
_MAX_STEP = 1 << 26  # elements between tokens that the scan's 32-bit lane offsets allow


def _on_gpu(t) -> bool:
    return isinstance(t, torch.Tensor) and t.is_cuda


# ---- argument checks --------------------------------------------------------

def _check_act(t: torch.Tensor, name: str, shape, like: torch.Tensor | None = None) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor")
    if shape is not None and t.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    if like is None:
        if t.dtype not in (torch.bfloat16, torch.float32) and not (t.dtype == torch.float64 and not t.is_cuda):
            raise TypeError(f"{name} must be bf16 or f32, got {t.dtype}")
    else:
        if t.dtype != like.dtype:
            raise TypeError(f"{name} must be {like.dtype}, got {t.dtype}")
        if t.device != like.device:
            raise ValueError(f"{name} must be on {like.device}, got {t.device}")


def _param(t: torch.Tensor | None, name: str, shape, like: torch.Tensor) -> torch.Tensor | None:
    """A parameter in the kernels' form: f32 (f64 beside f64), contiguous."""
    if t is None:
        return None
    if t.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    if not t.is_floating_point():
        raise TypeError(f"{name} must be a floating-point tensor")
    if t.device != like.device:
        raise ValueError(f"{name} must be on {like.device}, got {t.device}")
    want = torch.float64 if like.dtype == torch.float64 else torch.float32
    if t.dtype != want:
        t = t.to(want)
    return t.contiguous()


def _rows(t: torch.Tensor | None) -> torch.Tensor | None:
    """Channels contiguous; a copy only where they are not."""
    if t is None or t.stride(-1) == 1 or t.shape[-1] == 1:
        return t
    return t.contiguous()


def _check_lengths(lengths, batch: int, like: torch.Tensor):
    if lengths is None:
        return None
    if lengths.dtype not in (torch.int32, torch.int64):
        raise TypeError("lengths must be int32 or int64")
    if lengths.shape != (batch,):
        raise ValueError(f"lengths must have shape ({batch},), got {tuple(lengths.shape)}")
    if lengths.device != like.device:
        raise ValueError(f"lengths must be on {like.device}, got {lengths.device}")
    return lengths.contiguous()


def _check_carried(t: torch.Tensor, name: str, shape, dtype, like: torch.Tensor) -> None:
    if t.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if t.device != like.device:
        raise ValueError(f"{name} must be on {like.device}, got {t.device}")


def _state_pair(state, state_out, shape, dtype, like):
    """The state read and the one written by a step: the same or apart."""
    _check_carried(state, "state", shape, dtype, like)
    if not state.is_contiguous():
        raise ValueError("state must be contiguous")
    if state_out is None or state_out is state:
        return state
    _check_carried(state_out, "state_out", shape, dtype, like)
    if not state_out.is_contiguous():
        raise ValueError("state_out must be contiguous")
    a, b = state.data_ptr(), state_out.data_ptr()
    if a != b and abs(a - b) < state.numel() * state.element_size():
        raise ValueError("state_out overlaps state without being the same")
    return state_out


def _no_grad_only(name: str, *tensors) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError(f"{name} has no gradient: call it under torch.no_grad()")


def _check_capture(*tensors) -> None:
    """Refuse a training call inside a capture whose backward could not be
    captured: a leaf that an eager graph still holds on another stream."""
    if not (torch.is_grad_enabled() and torch.cuda.is_current_stream_capturing()):
        return
    ext = _ops.get_ext()
    seen, todo = set(), []
    for t in tensors:
        if t is None or not t.requires_grad:
            continue
        if t.grad_fn is not None:
            todo.append(t.grad_fn)
        elif ext.accumulates_elsewhere(t):
            raise RuntimeError(_LIVE_GRAPH)
    while todo:
        fn = todo.pop()
        if fn is None or fn in seen:
            continue
        seen.add(fn)
        leaf = getattr(fn, "variable", None)
        if isinstance(leaf, torch.Tensor) and ext.accumulates_elsewhere(leaf):
            raise RuntimeError(_LIVE_GRAPH)
        todo.extend(f for f, _ in fn.next_functions)


_LIVE_GRAPH = ("a leaf of this call is held by an eager autograd graph on another stream: drop that graph "
               "(its loss and outputs) before capturing a training step")


# ---- short causal convolution -----------------------------------------------


def _check_taps(weight, D: int) -> int:
    if not isinstance(weight, torch.Tensor) or weight.dim() != 2 or weight.shape[0] != D:
        raise ValueError(f"weight must have shape ({D}, K)")
    K = weight.shape[1]
    if not 2 <= K <= 4:
        raise ValueError(f"weight must have 2 to 4 taps, got {K}")
    return K


def _check_activation(activation) -> bool:
    if activation not in ("silu", None, "none"):
        raise ValueError("activation must be 'silu' or None")
    return activation == "silu"


def short_conv(x, weight, bias=None, *, state=None, lengths=None, activation="silu", return_state=False):
    """Causal convolution over time, one filter per channel:

        y[b, t, d] = act(bias[d] + sum_k weight[d, k] x[b, t - K + 1 + k, d])

    x: (B, L, D); weight: (D, K), K in 2..4, the last tap on the newest input;
    bias: (D,). state: (B, K-1, D) of x's type, the inputs before the first
    (zeros if None). Returns y, or (y, state after the last valid token).
    """
    silu = _check_activation(activation)
    if _on_gpu(x):
        out = _ops.get_ext().short_conv_direct(x, weight, bias, state, lengths, silu, return_state)
        if out is not None:
            return out
    _check_act(x, "x", None)
    if x.dim() != 3:
        raise ValueError(f"x must be (batch, length, channels), got {tuple(x.shape)}")
    B, _, D = x.shape
    K = _check_taps(weight, D)
    weight = _param(weight, "weight", (D, K), x)
    bias = _param(bias, "bias", (D,), x)
    if state is not None:
        _check_carried(state, "state", (B, K - 1, D), x.dtype, x)
    lengths = _check_lengths(lengths, B, x)
    if not x.is_cuda:
        y, last = eager.short_conv_eager(x, weight, bias, state, lengths, silu)
        return (y, last) if return_state else y
    x = _rows(x)
    state = None if state is None else state.contiguous()
    _check_capture(x, weight, bias, state)
    return _ops.get_ext().short_conv_direct(x, weight, bias, state, lengths, silu, return_state, prepared=True)


def short_conv_step(x, state, weight, bias=None, *, activation="silu", state_out=None):
    """short_conv of one new token per sequence. x: (B, D); state: (B, K-1, D)
    contiguous. Returns (y (B, D), the new state): written over ``state``, or to
    ``state_out`` if given."""
    silu = _check_activation(activation)
    if _on_gpu(x):
        res = _ops.get_ext().short_conv_step_direct(x, state, state_out, weight, bias, silu)
        if res is not None:
            return res
    _check_act(x, "x", None)
    if x.dim() != 2:
        raise ValueError(f"x must be (batch, channels), got {tuple(x.shape)}")
    B, D = x.shape
    K = _check_taps(weight, D)
    _no_grad_only("short_conv_step", x, state, weight, bias, state_out)
    weight = _param(weight, "weight", (D, K), x)
    bias = _param(bias, "bias", (D,), x)
    out = _state_pair(state, state_out, (B, K - 1, D), x.dtype, x)
    if not x.is_cuda:
        y, last = eager.short_conv_eager(x.unsqueeze(1), weight, bias, state, None, silu)
        out.copy_(last)
        return y.squeeze(1), out
    return _ops.get_ext().short_conv_step(_rows(x), state, out, weight, bias, silu), out


# ---- selective state space scan ---------------------------------------------


def _check_scan(u, delta, A, B, C, lead):
    """Shapes and types that the scan and its step share; B and C with groups."""
    _check_act(u, "u", None)
    if u.dim() != len(lead) + 1:
        raise ValueError(f"u must be ({', '.join(lead)}, channels), got {tuple(u.shape)}")
    D = u.shape[-1]
    if D > _MAX_SCAN_D:
        raise ValueError(f"u must have at most {_MAX_SCAN_D} channels, got {D}")
    _check_act(delta, "delta", u.shape, u)
    if not isinstance(A, torch.Tensor) or A.dim() != 2 or A.shape[0] != D:
        raise ValueError(f"A must have shape ({D}, N)")
    N = A.shape[1]
    if not 1 <= N <= _MAX_STATES:
        raise ValueError(f"A must have 1 to {_MAX_STATES} states a channel, got {N}")
    out = []
    for name, t in (("B", B), ("C", C)):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a tensor")
        if t.dim() == u.dim():
            t = t.unsqueeze(-2)
        if t.dim() != u.dim() + 1 or t.shape[:-2] != u.shape[:-1] or t.shape[-1] != N:
            raise ValueError(f"{name} must be ({', '.join(lead)}, groups, {N}), got {tuple(t.shape)}")
        _check_act(t, name, None, u)
        out.append(t)
    G = out[0].shape[-2]
    if out[1].shape != out[0].shape:
        raise ValueError("B and C must have the same shape")
    if G < 1 or D % G:
        raise ValueError(f"the groups ({G}) must divide the channels ({D})")
    return _param(A, "A", (D, N), u), out[0], out[1]


def _state_dtype(u):
    return torch.float64 if u.dtype == torch.float64 else torch.float32


def selective_scan(u, delta, A, B, C, skip=None, *, delta_bias=None, delta_softplus=False, state=None, lengths=None,
                   return_state=False):
    """Linear recurrence whose step size, input and output maps depend on the token:

        dt = softplus(delta + delta_bias)            (as it is without delta_softplus)
        h_t[d, n] = exp(dt A[d, n]) h_{t-1}[d, n] + dt u_t[d] B_t[g, n]
        y_t[d] = sum_n C_t[g, n] h_t[d, n] + skip[d] u_t[d]

    u, delta: (B, L, D); A: (D, N), N up to 64; B, C: (B, L, N) or (B, L, G, N),
    group g of D / G channels sharing one row; skip, delta_bias: (D,). From a
    step of +inf on its channel's outputs are inf or NaN.
    state: (B, D, N) f32, h before the first token (zeros if None). Returns y,
    or (y, f32 state after the last valid token).
    """
    softplus = bool(delta_softplus)
    if _on_gpu(u):
        out = _ops.get_ext().selective_scan_direct(u, delta, A, B, C, skip, delta_bias, state, lengths, softplus,
                                                   return_state)
        if out is not None:
            return out
    A, B, C = _check_scan(u, delta, A, B, C, ("batch", "length"))
    nb, _, D = u.shape
    N = A.shape[1]
    skip = _param(skip, "skip", (D,), u)
    delta_bias = _param(delta_bias, "delta_bias", (D,), u)
    if state is not None:
        _check_carried(state, "state", (nb, D, N), _state_dtype(u), u)
    lengths = _check_lengths(lengths, nb, u)
    if not u.is_cuda:
        y, last = eager.selective_scan_eager(u, delta, A, B, C, skip, delta_bias, softplus, state, lengths)
        return (y, last) if return_state else y
    u, delta, B, C = (t.contiguous() if t.shape[1] > 1 and t.stride(1) >= _MAX_STEP else _rows(t)
                      for t in (u, delta, B, C))
    state = None if state is None else state.contiguous()
    _check_capture(u, delta, A, B, C, skip, delta_bias, state)
    return _ops.get_ext().selective_scan_direct(u, delta, A, B, C, skip, delta_bias, state, lengths, softplus,
                                                return_state, prepared=True)


def selective_scan_step(u, delta, A, B, C, state, skip=None, *, delta_bias=None, delta_softplus=False,
                        state_out=None):
    """selective_scan of one new token per sequence. u, delta: (B, D); B, C:
    (B, N) or (B, G, N); state: (B, D, N) f32 contiguous. Returns (y (B, D), the
    new state): written over ``state``, or to ``state_out`` if given."""
    softplus = bool(delta_softplus)
    if _on_gpu(u):
        res = _ops.get_ext().selective_scan_step_direct(u, delta, A, B, C, state, state_out, skip, delta_bias, softplus)
        if res is not None:
            return res
    A, B, C = _check_scan(u, delta, A, B, C, ("batch",))
    nb, D = u.shape
    _no_grad_only("selective_scan_step", u, delta, A, B, C, state, skip, delta_bias, state_out)
    skip = _param(skip, "skip", (D,), u)
    delta_bias = _param(delta_bias, "delta_bias", (D,), u)
    out = _state_pair(state, state_out, (nb, D, A.shape[1]), _state_dtype(u), u)
    if not u.is_cuda:
        y, last = eager.selective_scan_eager(u.unsqueeze(1), delta.unsqueeze(1), A, B.unsqueeze(1), C.unsqueeze(1),
                                             skip, delta_bias, softplus, state, None)
        out.copy_(last)
        return y.squeeze(1), out
    return _ops.get_ext().selective_scan_step(_rows(u), _rows(delta), A, _rows(B), _rows(C), state, out, skip,
                                              delta_bias, softplus), out


# ---- norms around a block ---------------------------------------------------


def norm_gate_residual(x, *, gate=None, post_weight=None, residual=None, scale=None, pre_weight=None, eps=1e-5):
    """Root-mean-square norms after a block and before the next, with the
    block's gate, residual and residual scale, in one pass:

        p = x * silu(gate)                                      (gate)
        p = p / sqrt(mean(p^2) + eps) * post_weight             (post_weight)
        h = residual + scale * p                                (residual, scale)
        y = h / sqrt(mean(h^2) + eps) * pre_weight              (pre_weight)

    x, gate: (..., D) of one type, D up to 16384; residual: (..., D) bf16 or f32,
    which need not be x's type; post_weight, scale, pre_weight: (D,). Parts left
    out are skipped: one norm at least, and scale and pre_weight only with a
    residual. h feeds the second norm unrounded. Squares are summed in f32: a row
    whose root mean square passes 1.8e19 / sqrt(D) overflows the sum and is
    normed to zeros. Returns p without a residual, h without pre_weight, else
    (y, h): p and y of x's type, h of the residual's.
    """
    if _on_gpu(x):
        out = _ops.get_ext().block_norm_direct(x, gate, post_weight, residual, scale, pre_weight, eps)
        if out is not None:
            return out
    _check_act(x, "x", None)
    if x.dim() < 1:
        raise ValueError("x must have a channel axis")
    D = x.shape[-1]
    if not 1 <= D <= _MAX_NORM_D:
        raise ValueError(f"x must have 1 to {_MAX_NORM_D} channels, got {D}")
    if post_weight is None and pre_weight is None:
        raise ValueError("post_weight or pre_weight is needed")
    if residual is None and (scale is not None or pre_weight is not None):
        raise ValueError("scale and pre_weight need a residual")
    if not eps >= _MIN_EPS:
        raise ValueError(f"eps must be at least {_MIN_EPS:.3g} (a normal float32), got {eps}")
    if gate is not None:
        _check_act(gate, "gate", x.shape, x)
    if residual is not None:
        _check_act(residual, "residual", x.shape)
        if residual.device != x.device:
            raise ValueError(f"residual must be on {x.device}, got {residual.device}")
        if (residual.dtype == torch.float64) != (x.dtype == torch.float64):
            raise TypeError("residual must be f64 where x is, and only there")
    post = _param(post_weight, "post_weight", (D,), x)
    scale = _param(scale, "scale", (D,), x)
    pre = _param(pre_weight, "pre_weight", (D,), x)
    eps = float(eps)
    if not x.is_cuda:
        y, h = eager.norm_gate_residual_eager(x, gate, post, residual, scale, pre, eps)
        return (y, h) if y is not None and h is not None else h if y is None else y
    x, gate, residual = _rows(x), _rows(gate), _rows(residual)
    _check_capture(x, gate, post, residual, scale, pre)
    return _ops.get_ext().block_norm_direct(x, gate, post, residual, scale, pre, eps, prepared=True)
