"""What a shared block needs around and inside it, between two reads of the update stack: the norms before and after the
block with its gate, dropout and residual scale, dropout on its own, and the gated feed-forward product.

    block_norm      u = w n(x),  n(v) = v / sqrt(mean(v^2) + eps)
    block_residual  out = x + s g m b, with b = w n(y) (or y); and, given the next block's norm, u = w' n(out)
    dropout         out = m x
    gated_ffn       y = (act(x Wg^T) * (x Wu^T)) Wd^T

The read cell forms a block's input (cell.combine), the caller's block turns it into a proposal with these operators, and
`DattnStack.write` stores the difference: h = block_residual(x, f(block_norm(x, w)), ...) is what `write(s, h, x)` and
`combine(h, ...)` take.  Rows are bf16 or fp32 as everywhere in this package, arithmetic is fp32 with one rounding per
result, and there is no CPU or eager path: inputs the kernels cannot take raise.  The reference's models run these as
separate PyTorch operations between their reads (looped_transformer.py, the block the reads sit between).
"""
from __future__ import annotations

import torch
from torch import nn

from . import _lib

__all__ = ["block_norm", "block_residual", "dropout", "gated_ffn", "FeedForwardBlock"]

_ACTS = {"silu": 0, "gelu": 1}


def block_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6) -> torch.Tensor:
    """weight * x / sqrt(mean(x^2) + eps) over the last dimension, differentiable (once) in both. `weight` (d,) in x's type or
    fp32."""
    return _lib.torch_ops().block_norm(x, weight, eps)


def _threshold(what, p):
    t = int(float(p) * 65536 + 0.5) if 0.0 <= float(p) < 1.0 else -1
    if not 0 <= t <= 65535:
        raise ValueError(f"loopback_b200.{what}: need 0 <= p < 1 (to the nearest 1 / 65536), got {p}")
    return t


def _rng_args(what, rng):
    """(device pair or None, seed, offset)"""
    if isinstance(rng, torch.Tensor):
        return rng, 0, 0
    if rng is None:
        raise ValueError(f"loopback_b200.{what}: dropout needs rng = (seed, offset)")
    seed, offset = (int(v) for v in rng)
    wrap = lambda v: (v & (1 << 64) - 1) - (1 << 64 if v >> 63 & 1 else 0)  # noqa: E731  any 64-bit pattern
    return None, wrap(seed), wrap(offset)


def dropout(x: torch.Tensor, p: float, rng) -> torch.Tensor:
    """Each element is kept with probability 1 - p (p to the nearest 1 / 65536) and scaled by the inverse of what is kept on
    average, else replaced by 0 (also where it is infinite or NaN). The mask is never stored: the backward draws the same
    numbers again.

    rng = (seed, offset), two 64-bit integers: a pair of Python integers, or a contiguous int64 tensor of two on x's
    device, read when the kernel runs (a captured graph draws new numbers on every replay if the offset is advanced in
    between; the backward uses the pair its forward used). The same pair gives the same mask for the same element count."""
    return _lib.torch_ops().dropout(x, _threshold("dropout", p), *_rng_args("dropout", rng))


def block_residual(x: torch.Tensor, y: torch.Tensor, weight=None, *, gate=None, scale=1.0, next_weight=None,
                   eps: float = 1e-6, p: float = 0.0, rng=None):
    """The end of a block in one pass over its rows: out = x + scale * gate * dropout(norm(y)), and, given `next_weight`, the
    norm the next block starts with. Returns out, or (out, norm of out).

    x, y         the residual stream and the block's output, one shape and type
    weight       (d,) of the norm after the block; None: no such norm, y itself is added
    gate         None, (d,) per channel, (..., 1) per token or x's shape
    scale        a number, or a tensor of one element (learned)
    next_weight  (d,) of the norm of out; its statistics come from out before it is rounded to its storage type
    p, rng       dropout of the (normed) block output, as in `dropout`, drawn over x's elements; without `weight`, what y holds
                 where it is dropped reaches neither the results nor a gradient
    Per-channel parameters are in x's type or fp32, gates per token or element in x's. Differentiable (once) in every tensor."""
    t = _threshold("block_residual", p) if p else 0
    pair, seed, offset = _rng_args("block_residual", rng) if t else (None, 0, 0)
    learned, scale = (scale, 1.0) if isinstance(scale, torch.Tensor) else (None, scale)
    got = _lib.torch_ops().block_residual(x, y, weight, gate, learned, scale, next_weight, eps, t, pair, seed, offset)
    return got[0] if next_weight is None else (got[0], got[1])


def gated_ffn(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor, act: str = "silu") -> torch.Tensor:
    """(act(x w_gate^T) * (x w_up^T)) w_down^T, differentiable (once) in every tensor.

    x (..., d), w_gate and w_up (f, d), w_down (d, f), all bf16 (the products run on the tensor cores in bf16 with fp32
    accumulation; h and the result, and in the backward the two gradients behind the product, are each rounded once),
    contiguous weights, d and f multiples of 8. act: "silu" or "gelu" (with erf). Both projections, the activation and the
    product are one launch. With gradients h and two factors of 24 bits are kept: 8 bytes per token and column of f."""
    if act not in _ACTS:
        raise ValueError(f"loopback_b200.gated_ffn: act is one of {sorted(_ACTS)}, got {act!r}")
    return _lib.torch_ops().gated_ffn(x, w_gate, w_up, w_down, _ACTS[act])


class FeedForwardBlock(nn.Module):
    """A feed-forward block between two reads, on the operators above:

        out = x + scale * gate * dropout(norm_after(ffn(norm(x))))

    `post_norm` adds the norm after the block, `gate` a learned vector per channel (ones at first), `scale` the residual
    scale (a number; a learned one with `learn_scale`), `p` the dropout of the branch, applied in training. Its result is
    the proposal `cell.combine` takes and the first argument of `DattnStack.write`."""

    def __init__(self, dim: int, hidden: int, act: str = "silu", *, post_norm: bool = False, gate: bool = False, scale: float = 1.0,
                 learn_scale: bool = False, p: float = 0.0, eps: float = 1e-6, device=None, dtype=torch.bfloat16):
        super().__init__()
        if act not in _ACTS:
            raise ValueError(f"loopback_b200.FeedForwardBlock: act is one of {sorted(_ACTS)}, got {act!r}")
        if dim < 1 or hidden < 1 or dim % 8 or hidden % 8:
            raise ValueError(f"loopback_b200.FeedForwardBlock: dim and hidden are multiples of 8, got {dim} and {hidden}")
        _threshold("FeedForwardBlock", p)
        make = dict(device=device, dtype=dtype)
        self.act, self.p, self.eps = act, float(p), float(eps)
        self.norm = nn.Parameter(torch.ones(dim, **make))
        self.norm_after = nn.Parameter(torch.ones(dim, **make)) if post_norm else None
        self.gate = nn.Parameter(torch.ones(dim, **make)) if gate else None
        self.scale = nn.Parameter(torch.full((1,), float(scale), device=device)) if learn_scale else float(scale)
        self.w_gate = nn.Parameter(torch.empty(hidden, dim, **make))
        self.w_up = nn.Parameter(torch.empty(hidden, dim, **make))
        self.w_down = nn.Parameter(torch.empty(dim, hidden, **make))
        self.reset_parameters()

    def reset_parameters(self):
        with torch.no_grad():
            for w in (self.w_gate, self.w_up, self.w_down):
                w.normal_(0.0, w.shape[1] ** -0.5)

    def forward(self, x: torch.Tensor, normed=None, next_weight=None, rng=None):
        """out, or (out, norm of out by `next_weight`). `normed`: norm(x), where the previous block already formed it (its
        `next_weight` was this block's `norm`). `rng`: see `dropout`; needed in training with p > 0."""
        u = block_norm(x, self.norm, self.eps) if normed is None else normed
        y = gated_ffn(u, self.w_gate, self.w_up, self.w_down, self.act)
        return block_residual(x, y, self.norm_after, gate=self.gate, scale=self.scale, next_weight=next_weight, eps=self.eps,
                              p=self.p if self.training else 0.0, rng=rng)
