"""Keys that mark their tiles: the float64 attention of rows whose every element
tells whether the keys of one 32-key tile were counted, and how often.

A request's token g has the value 1 in latent dimension (g // 32) % 512 and 0 in
the others, and the queries have no latent part, so scores come from the 64 rope
values alone: an output element is the share of its tile (of every 512th tile) in
the row's softmax.

Bound, relative to the element.  A probability is rounded to bf16 (2^-8), and the
sum is of the rounded ones: the quotient of two sums of positive terms each off by
u at most is off by (1 + u) / (1 - u); the output is rounded to bf16.  u = 2^-8 +
2^-10: the scores (64 products in fp32, 2^-23 of their magnitudes' sum, below 300,
a step, times sm log2 e = 0.06: 1.4e-4), the reference point's difference (below
200: 2^-17), and the fp32 sums (a step 2^-23 of the sum, 16 keys a step, 131072
keys over 256 workgroups and their join: below 2.7e-4) stay within 2^-10.
"""

from __future__ import annotations

import torch

TILE, DIMS = 32, 512
_U = 2.0 ** -8 + 2.0 ** -10
BOUND = (1 + _U) / (1 - _U) * (1 + 2.0 ** -8) - 1


def marks(n: int, device=None) -> torch.Tensor:
    """Marked latent dimension of tokens 0 .. n - 1."""
    return torch.arange(n, device=device) // TILE % DIMS


def shares(q_rope: torch.Tensor, k_rope: torch.Tensor, pos: torch.Tensor, count: torch.Tensor | None = None) -> torch.Tensor:
    """[rows, 512] float64 of queries [rows, 64] at positions pos [rows] over
    keys [n, 64]; count [n]: how often each key counts (None: once)."""
    n = k_rope.shape[0]
    s = q_rope.double() @ k_rope.double().T * 576 ** -0.5
    s = s.masked_fill(torch.arange(n, device=s.device) > pos[:, None], float("-inf"))
    w = torch.exp(s - s.amax(-1, keepdim=True).clamp_min(-1e300))
    if count is not None:
        w = w * count
    out = torch.zeros(s.shape[0], DIMS, dtype=torch.float64, device=s.device)
    out.index_add_(1, marks(n, s.device), w)
    return out / w.sum(-1, keepdim=True).clamp_min(1e-300)


def worst(got: torch.Tensor, ref: torch.Tensor) -> float:
    """The largest error over the bound (infinite where a 0 is not a 0)."""
    err = (got.double() - ref).abs()
    return float((err / (BOUND * ref)).nan_to_num(nan=0.0, posinf=float("inf")).max())
