"""Queries that read the tokens of several fixations.

``FixationReader`` is a pre-norm cross-attention block on the package's kernels: layer norm of the
queries and of the states, rotary positions on (fixation, row, column), and attention of the
queries to the states. In training it is called with the states; a serving program projects the
states of each new fixation once (``project``), keeps keys and values in its own buffers, and calls
the block with them and the number of states that each image has so far.
"""
from __future__ import annotations

import math

import torch
import torch.nn as nn

from .attention import cross_attention
from .norm import LayerNorm
from .rotary import AxialRotary

__all__ = ["FixationReader", "fixation_positions"]


def fixation_positions(coords, fixations, first=0, device="cuda"):
    """``[F * N, 3]`` positions (fixation number, row, column) of the tokens of ``fixations``
    fixations, fixation by fixation, from a sensor's ``SamplingCoords`` of N token centres."""
    rowcol = torch.as_tensor(coords.cartesian_rowcol).to(device=device, dtype=torch.float32)
    number = torch.arange(first, first + fixations, device=device, dtype=torch.float32)
    n = rowcol.shape[0]
    return torch.cat([number.repeat_interleave(n)[:, None], rowcol.repeat(fixations, 1)], 1)


class FixationReader(nn.Module):
    """``x + W_o attention(norm(x), norm(states))`` with rotary positions on the keys (and on the
    queries that have one).

    ``sections``: pairs per axis of a head (fixation number, row, column), by default a quarter of
    the pairs and the rest in two halves. ``base`` and ``scale`` as in ``AxialRotary``; by default row and
    column, in [-1, 1], turn by 2 pi at most, and fixations, counted in whole numbers, by one radian each (whole
    turns would tell none apart). ``kv_heads`` < ``heads`` shares key heads.
    """

    def __init__(self, dim, state_dim, heads, head_dim=64, kv_heads=None, sections=None, base=100.0, device="cuda",
                 scale=None):
        super().__init__()
        kv_heads = heads if kv_heads is None else kv_heads
        if heads % kv_heads:
            raise ValueError(f"FixationReader: {heads} heads over {kv_heads} key heads")
        if sections is None:
            row = (head_dim // 2 - head_dim // 8) // 2
            sections = (head_dim // 2 - 2 * row, row, row)
        if scale is None:
            scale = (1.0, 2 * math.pi, 2 * math.pi) if len(sections) == 3 else 2 * math.pi
        self.dim, self.state_dim, self.heads, self.kv_heads, self.head_dim = dim, state_dim, heads, kv_heads, head_dim
        self.norm, self.state_norm = LayerNorm(dim, device=device), LayerNorm(state_dim, device=device)
        self.to_q = nn.Linear(dim, heads * head_dim, bias=False, device=device)
        self.to_kv = nn.Linear(state_dim, 2 * kv_heads * head_dim, bias=False, device=device)
        self.to_out = nn.Linear(heads * head_dim, dim, device=device)
        self.rotary = AxialRotary(head_dim, sections, base=base, scale=scale, device=device)

    def project(self, states, positions):
        """Keys and values ``[B, S, kv_heads, head_dim]`` of ``states [B, S, state_dim]`` at ``positions
        [S, 3]`` or ``[B, S, 3]``."""
        b, s, _ = states.shape
        kv = self.to_kv(self.state_norm(states)).view(b, s, 2, self.kv_heads, self.head_dim)
        return self.rotary(kv[:, :, 0], positions), kv[:, :, 1]

    def forward(self, x, states=None, positions=None, keys=None, values=None, x_positions=None, kv_lengths=None,
                mask=None):
        """``x [B, L, dim]`` reads ``states`` at ``positions``, or the ``keys`` and ``values`` that ``project``
        gave. ``x_positions [L, 3]`` or ``[B, L, 3]`` turns the queries too; ``kv_lengths`` and ``mask`` as
        in ``cross_attention``."""
        if (states is None) == (keys is None) or (keys is None) != (values is None):
            raise ValueError("FixationReader: either states with positions, or keys and values")
        if states is not None:
            if positions is None:
                raise ValueError("FixationReader: states without positions")
            keys, values = self.project(states, positions)
        b, n, _ = x.shape
        q = self.to_q(self.norm(x)).view(b, n, self.heads, self.head_dim)
        if x_positions is not None:
            q = self.rotary(q, x_positions)
        read = cross_attention(q, keys, values, kv_lengths=kv_lengths, mask=mask)
        return x + self.to_out(read.reshape(b, n, self.heads * self.head_dim))
