"""SelectiveEncoder: a state space temporal encoder beside the LSTM.

Maps each OD pair's scalar sequence to the hidden state after its last step,
as TemporalEncoder (models/mpgcn.py) does, with one mixing block:

    u, z  = in_proj(x)                       per step, (R, T, H) each
    v     = silu(short_conv(u))
    delta, B, C = x_proj(v)
    y     = selective_scan(v, delta, A, B, C) + skip v
    o     = out_proj(norm(y silu(z)))        from the last step on: all it needs
    h     = norm(u + scale o)

Its state is the last taps - 1 values of u and an (H, states) f32 scan state a
sequence, so a served model can take one new observation at a time (``start``,
``step``) at a cost that does not grow with the window.
"""

from __future__ import annotations

import math

import torch
from torch import nn

from mpgcn_amd.ops import (
    linear_act,
    norm_gate_residual,
    selective_scan,
    selective_scan_step,
    short_conv,
    short_conv_step,
)


class SelectiveEncoder(nn.Module):
    def __init__(self, input_size: int, hidden_size: int, state_size: int = 16, taps: int = 4):
        super().__init__()
        if input_size != 1:
            raise ValueError("SelectiveEncoder supports input_size=1 (OD-flow scalar)")
        if not 1 <= state_size <= 64:
            raise ValueError("state_size must be 1 to 64")
        if not 2 <= taps <= 4:
            raise ValueError("taps must be 2 to 4")
        H, N = hidden_size, state_size
        self.hidden_size, self.state_size, self.taps = H, N, taps
        self.in_proj = nn.Linear(1, 2 * H)
        self.conv_weight = nn.Parameter(torch.empty(H, taps))
        self.conv_bias = nn.Parameter(torch.zeros(H))
        self.x_proj = nn.Linear(H, H + 2 * N, bias=False)
        self.A_log = nn.Parameter(torch.log(torch.arange(1, N + 1, dtype=torch.float32)).repeat(H, 1))
        self.skip = nn.Parameter(torch.ones(H))
        self.delta_bias = nn.Parameter(torch.empty(H))
        self.gate_norm = nn.Parameter(torch.ones(H))
        self.out_proj = nn.Linear(H, H)
        self.residual_scale = nn.Parameter(torch.ones(H))
        self.out_norm = nn.Parameter(torch.ones(H))
        nn.init.uniform_(self.conv_weight, -1 / math.sqrt(taps), 1 / math.sqrt(taps))
        with torch.no_grad():
            # first step sizes spread evenly over the decades from 1e-2 to 1:
            # windows here are days, not thousands of tokens
            dt = torch.exp(torch.rand(H) * math.log(100.0) + math.log(1e-2))
            self.delta_bias.copy_(dt + torch.log(-torch.expm1(-dt)))

    def _project(self, rows: torch.Tensor, layer: nn.Linear) -> torch.Tensor:
        return linear_act(rows, layer.weight.to(rows.dtype), layer.bias, relu=False)

    def _inputs(self, x: torch.Tensor):
        """(R, T) -> u, z (R, T, H), views of one projection."""
        uz = self._project(x.reshape(-1, 1).contiguous(), self.in_proj).view(*x.shape, 2 * self.hidden_size)
        return uz[..., : self.hidden_size], uz[..., self.hidden_size:]

    def _maps(self, v: torch.Tensor):
        """delta, A, B, C of the scan, views of one projection."""
        H, N = self.hidden_size, self.state_size
        m = self._project(v.reshape(-1, H), self.x_proj).view(*v.shape[:-1], H + 2 * N)
        return m[..., :H], -torch.exp(self.A_log), m[..., H:H + N], m[..., H + N:]

    def _leave(self, y: torch.Tensor, u: torch.Tensor, z: torch.Tensor) -> torch.Tensor:
        """(R, H) of one step each: gate, norm, projection, residual, norm."""
        o = self._project(norm_gate_residual(y, gate=z, post_weight=self.gate_norm), self.out_proj)
        return norm_gate_residual(o, residual=u, scale=self.residual_scale, pre_weight=self.out_norm)[0]

    def _run(self, x: torch.Tensor, keep: bool):
        u, z = self._inputs(x)
        conv = short_conv(u, self.conv_weight, self.conv_bias, return_state=keep)
        v, conv_state = conv if keep else (conv, None)
        scan = selective_scan(v, *self._maps(v), self.skip, delta_bias=self.delta_bias, delta_softplus=True,
                              return_state=keep)
        y, scan_state = scan if keep else (scan, None)
        h = self._leave(y[:, -1], u[:, -1], z[:, -1])
        return (h, (conv_state, scan_state)) if keep else h

    def forward(self, x: torch.Tensor, T: int | None = None) -> torch.Tensor:
        """x: (R, T) scalar sequences -> (R, hidden) after the last step.
        T: logical length when x rows are padded (as for TemporalEncoder)."""
        return self._run(x if T is None or T == x.shape[1] else x[:, :T], False)

    @torch.no_grad()
    def start(self, x: torch.Tensor):
        """-> (hidden state after x (R, T), state to go on from)."""
        return self._run(x, True)

    @torch.no_grad()
    def step(self, x: torch.Tensor, state) -> torch.Tensor:
        """One new value per sequence, x: (R,), updating ``state`` in place."""
        conv_state, scan_state = state
        u, z = self._inputs(x)
        v, _ = short_conv_step(u, conv_state, self.conv_weight, self.conv_bias)
        delta, A, B, C = self._maps(v)
        y, _ = selective_scan_step(v, delta, A, B, C, scan_state, self.skip, delta_bias=self.delta_bias,
                                   delta_softplus=True)
        return self._leave(y, u, z)

    def extra_repr(self) -> str:
        return f"hidden={self.hidden_size}, states={self.state_size}, taps={self.taps}"
