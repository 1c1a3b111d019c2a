"""A policy's sequence memory on the GPU, of the operators in marlsoccer.sequence.

The reference's policy sees three stacked frames and nothing before them. SequenceMemory is a
residual block beside them: it takes the normalised observations of every agent and returns them with
what the memory adds, so the actor and critic behind it stay as they are:

    u, z = in_proj(x);  u = silu(short_conv(u));  rate, B, C = x_proj(u)
    y = x + out_proj(ssm_scan(u, rate, B, C) * silu(z))

    agent = Agent(memory=SequenceMemory())        # DeviceRollout and evaluate then carry its state
    y, state = agent.memory(x, starts, state)     # whole sequences (T, R, 66), for the update
    y = agent.memory.step(x, state, starts)       # one step (R, 66), the state renewed in place
"""
from __future__ import annotations

import math

import torch
import torch.nn as nn

from .sequence import short_conv, short_conv_step, ssm_scan, ssm_step


class SequenceMemory(nn.Module):
    """width: features in and out (66, an observation); channels: of the memory; states: for each
    channel (1..64); conv: steps the convolution sees (2..4); rank: of the rates' projection."""

    def __init__(self, width: int = 66, channels: int = 128, states: int = 16, conv: int = 4, rank: int | None = None):
        super().__init__()
        self.width, self.channels, self.states, self.conv = width, channels, states, conv
        self.rank = max(1, math.ceil(width / 16)) if rank is None else rank
        self.in_proj = nn.Linear(width, 2 * channels, bias=False)
        self.conv_weight = nn.Parameter(torch.randn(channels, conv) * conv ** -0.5)
        self.conv_bias = nn.Parameter(torch.zeros(channels))
        self.x_proj = nn.Linear(channels, self.rank + 2 * states, bias=False)
        self.rate_proj = nn.Linear(self.rank, channels, bias=False)
        # softplus(rate_bias) is log-uniform in [1e-3, 1e-1]: memories of 10 to 1,000 steps
        rate = torch.exp(torch.rand(channels) * math.log(100.0) + math.log(1e-3))
        self.rate_bias = nn.Parameter(rate + torch.log(-torch.expm1(-rate)))
        self.A_log = nn.Parameter(torch.log(torch.arange(1, states + 1).float()).repeat(channels, 1))
        self.skip = nn.Parameter(torch.ones(channels))
        self.out_proj = nn.Linear(channels, width, bias=False)
        with torch.no_grad():
            self.out_proj.weight.mul_(0.1)  # near the identity at first

    def init_state(self, rows: int, device=None, dtype: torch.dtype = torch.float32) -> tuple:
        """Zero state of `rows` rows: the convolution's inputs (of the activations' dtype) and the
        scan's states (float32)."""
        return (torch.zeros((rows, self.conv - 1, self.channels), dtype=dtype, device=device),
                torch.zeros((rows, self.channels, self.states), dtype=torch.float32, device=device))

    def _rates(self, u):
        r, B, C = self.x_proj(u).split((self.rank, self.states, self.states), dim=-1)
        return self.rate_proj(r), B, C

    def forward(self, x, starts=None, state=None):
        """x (T, R, width); starts (T, R) bool: row r begins an episode at step t (the rollout's dones);
        state: init_state's or a call's (None: zeros; the convolution's is taken in the type that x is
        projected to, so a bfloat16 rollout's state replays in float32 too). Returns y (T, R, width) and
        the state after."""
        conv_state, scan_state = (None, None) if state is None else state
        u, z = self.in_proj(x).chunk(2, dim=-1)
        if conv_state is not None:
            conv_state = conv_state.to(u.dtype)
        u, conv_state = short_conv(u, self.conv_weight, self.conv_bias, conv_state, starts, "silu", return_state=True)
        rate, B, C = self._rates(u)
        y, scan_state = ssm_scan(u, rate, -torch.exp(self.A_log), B, C, D=self.skip, z=z, delta_bias=self.rate_bias,
                                 state=scan_state, starts=starts, return_state=True)
        return x + self.out_proj(y), (conv_state, scan_state)

    @torch.no_grad()
    def step(self, x, state, starts=None):
        """One step: x (R, width), starts (R,); both tensors of `state` are renewed in place."""
        u, z = self.in_proj(x).chunk(2, dim=-1)
        u = short_conv_step(u, state[0], self.conv_weight, self.conv_bias, starts=starts, activation="silu")
        rate, B, C = self._rates(u)
        y = ssm_step(state[1], u, rate, -torch.exp(self.A_log), B, C, D=self.skip, z=z, delta_bias=self.rate_bias, starts=starts)
        return x + self.out_proj(y)
