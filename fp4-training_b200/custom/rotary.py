"""What stands between the (stacked) q / k / v projections and the attention core: rotary positions
with several axes, and the RMS norm of every query and key head with that rotation in the same pass.

The reference has neither: its blocks add a learned position embedding once (models/vit.py:50-56) and
use q and k as projected (models/transformer_block.py:89-95).  Normalised heads bound the attention
scores whatever the projections' precision does to the size of q and k; rotary positions need no
parameters and go on to images and videos larger than those trained on.

Tensors are [batch, tokens, heads, head_dim] (or [tokens, heads, head_dim]) with any strides, so views
of a stacked projection's output go in as they are; results are contiguous.  float32 and bfloat16;
everything is computed in fp32 and rounded once."""
from __future__ import annotations

import math

import torch
from torch import nn

from backend._ext import ext as _ext


_NO_TABLE = (None, None, 0, False)


class RotaryPositions(nn.Module):
    """Rotary positions with one or several axes (a text's index; an image's row and column; a video's
    frame, row and column).

    sections: how many pairs of a head each axis turns; they fill the first 2 * sum(sections)
      elements of a head and the others are passed through.
    spectrum: "axis" gives every axis its own frequencies base^(-j / sections[a]); "shared" runs
      base^(-p / sum(sections)) over all pairs, whichever axis they belong to.
    order: "blocks" lays the axes' pairs out one axis after the other, "cycled" in turn (an axis
      drops out of the cycle when its pairs are used up).
    layout: "half" pairs element p with p + sum(sections), "interleaved" 2p with 2p + 1.
    frequencies: radians per position of every pair, in place of base and spectrum (scaled contexts).

    positions are integers, [tokens, axes] or [batch, tokens, axes] ([tokens] will do with one axis),
    negative ones included; angles are exact modulo one turn for all of them."""

    def __init__(self, head_dim, sections, base=10000.0, layout="half", order="blocks", spectrum="axis", frequencies=None,
                 device=None):
        super().__init__()
        sections = [int(s) for s in ([sections] if isinstance(sections, int) else sections)]
        pairs = sum(sections)
        if head_dim % 2 or not 2 <= head_dim <= 512:
            raise ValueError(f"head_dim must be even, 2 to 512, got {head_dim}")
        if not sections or min(sections) < 1 or 2 * pairs > head_dim:
            raise ValueError(f"sections {sections} must be positive and turn at most head_dim / 2 = {head_dim // 2} pairs")
        if layout not in ("half", "interleaved") or order not in ("blocks", "cycled") or spectrum not in ("axis", "shared"):
            raise ValueError(f"unknown layout {layout!r}, order {order!r} or spectrum {spectrum!r}")
        self.head_dim, self.sections, self.layout = head_dim, tuple(sections), layout
        if order == "blocks":
            axis = [a for a, n in enumerate(sections) for _ in range(n)]
        else:
            axis = [a for j in range(max(sections)) for a, n in enumerate(sections) if j < n]
        if frequencies is None:
            if not (base > 0.0 and math.isfinite(base)):
                raise ValueError("base must be positive and finite")
            nth, frequencies = [0] * len(sections), []
            for p, a in enumerate(axis):
                frequencies.append(base ** -(nth[a] / sections[a] if spectrum == "axis" else p / pairs))
                nth[a] += 1
        else:
            frequencies = [float(f) for f in frequencies]
            if len(frequencies) != pairs or not all(math.isfinite(f) for f in frequencies):
                raise ValueError(f"frequencies must be {pairs} finite numbers")
        # turns per position as a 64-bit fixed-point fraction: integer multiples wrap modulo one turn
        turns = []
        for f in frequencies:
            v = round(math.fmod(f / (2.0 * math.pi), 1.0) * 2.0 ** 64) % 2 ** 64
            turns.append(v - 2 ** 64 if v >= 2 ** 63 else v)
        self.register_buffer("turns", torch.tensor(turns, dtype=torch.int64, device=device), persistent=False)
        self.register_buffer("axis", torch.tensor(axis, dtype=torch.int32, device=device), persistent=False)

    @property
    def table(self):
        buffers = self._buffers     # a third of an attribute's time; a replica of the module has attributes only
        try:
            turns, axis = buffers["turns"], buffers["axis"]
        except KeyError:
            turns, axis = self.turns, self.axis
        return turns, axis, len(self.sections), self.layout == "interleaved"

    def _check(self, x):
        if x.shape[-1] != self.head_dim:
            raise ValueError(f"head_dim {x.shape[-1]} is not this module's {self.head_dim}")

    def forward(self, *x, positions):
        """rotary(q, k, positions=p) -> (q', k'), or rotary(x, positions=p) -> x'."""
        if len(x) not in (1, 2):
            raise ValueError("RotaryPositions takes one or two tensors")
        self._check(x[0])
        y = _ext().rotary_call(x[0], x[1] if len(x) == 2 else None, positions, *self.table)
        return tuple(y) if len(x) == 2 else y[0]

    def extra_repr(self):
        return f"head_dim={self.head_dim}, sections={self.sections}, layout={self.layout!r}"


class FusedQKNorm(nn.Module):
    """RMS norm of every query and key head over its head_dim elements with one weight vector each
    for queries and keys, and the rotation of `rotary` (a RotaryPositions, or None) in the same pass.
    The backward pass recomputes the norms from q and k; nothing else is kept."""

    def __init__(self, head_dim, rotary=None, eps=1e-6, device=None, dtype=None):
        super().__init__()
        if head_dim % 2 or not 2 <= head_dim <= 512:
            raise ValueError(f"head_dim must be even, 2 to 512, got {head_dim}")
        if rotary is not None and rotary.head_dim != head_dim:
            raise ValueError(f"the rotary positions are for head_dim {rotary.head_dim}, not {head_dim}")
        if not eps >= 0.0:
            raise ValueError("eps must not be negative")
        self.head_dim, self.eps, self.rotary = head_dim, eps, rotary
        self.q_weight = nn.Parameter(torch.ones(head_dim, device=device, dtype=dtype))
        self.k_weight = nn.Parameter(torch.ones(head_dim, device=device, dtype=dtype))

    def forward(self, q, k, positions=None):
        if q.shape[-1] != self.head_dim:
            raise ValueError(f"head_dim {q.shape[-1]} is not this module's {self.head_dim}")
        table = _NO_TABLE if self.rotary is None else self.rotary.table
        params = self._parameters
        try:
            q_weight, k_weight = params["q_weight"], params["k_weight"]
        except KeyError:            # parametrized, pruned or replicated: attributes that are no parameters
            q_weight, k_weight = self.q_weight, self.k_weight
        return tuple(_ext().qk_norm_call(q, k, q_weight, k_weight, positions, *table, self.eps))

    def extra_repr(self):
        return f"head_dim={self.head_dim}, eps={self.eps}"
