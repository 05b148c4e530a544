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
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import check, dtype_code
from .fused_dattn import _require_cuda

__all__ = ["block_norm", "block_residual", "dropout", "gated_ffn"]

GATE_NONE, GATE_TOKEN, GATE_CHANNEL, GATE_FULL = range(4)

_current_device, _raw_stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream


def _call(x, what, fn, *args):
    """fn(*args, stream) on x's device, on its current stream. A decode step is bound by what the host does per call, so this
    avoids the guard and the Stream object where x's device is the current one."""
    dev = x.get_device()
    if dev == _current_device():
        rc = fn(*args, _raw_stream(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, _raw_stream(dev))
    check(rc, what)


def _p(t):
    return None if t is None else t.data_ptr()


def _require_rows(x, what):
    if not x.is_cuda:
        _require_cuda(x, what)
    if x.dim() == 0 or x.shape[-1] == 0:
        raise RuntimeError(f"loopback_b200.{what}: rows need a last dimension of at least one column, got shape {tuple(x.shape)}")


def _same_device(what, ref, *tensors):
    dev = ref.device
    for t in tensors:
        if t is not None and t.device != dev:
            raise RuntimeError(f"loopback_b200.{what}: a tensor is on {t.device}, the rows are on {dev}")


def _scratch(d, dev):
    return torch.empty(_lib.lib().lb_block_scratch_bytes(d), dtype=torch.uint8, device=dev)


def _channel_params(what, x, d, *params):
    """The per-channel parameters in one storage type the kernels take: the rows' or, where they are fp32 or differ, fp32."""
    kind, cast = None, False
    for p in params:
        if p is not None:
            if p.shape != (d,):
                raise RuntimeError(f"loopback_b200.{what}: a per-channel parameter has shape {tuple(p.shape)}, rows have {d} columns")
            cast = cast or (p.dtype != kind and kind is not None) or (p.dtype != x.dtype and p.dtype != torch.float32)
            kind = p.dtype
    if cast:
        params = [p if p is None else p.float() for p in params]
    return [p if p is None else p.contiguous() for p in params]


# --------------------------------------------------------------------------------------------------------------
# the norm before a block
# --------------------------------------------------------------------------------------------------------------
def _norm_forward(x, w, eps, save):
    d = x.shape[-1]
    n_tok = x.numel() // d
    u = torch.empty_like(x)
    r = torch.empty(n_tok, dtype=torch.float32, device=x.device) if save else None
    _call(x, "block norm", _lib.lib().lb_norm_fwd, x.data_ptr(), w.data_ptr(), u.data_ptr(), _p(r), n_tok, d, eps,
          dtype_code(x.dtype), dtype_code(w.dtype))
    return u, r


class _BlockNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, eps):
        u, r = _norm_forward(x, w, eps, True)
        ctx.save_for_backward(x, w, r)
        return u

    @staticmethod
    @once_differentiable
    def backward(ctx, du):
        x, w, r = ctx.saved_tensors
        d = x.shape[-1]
        du = du.contiguous()
        dx = torch.empty_like(x) if ctx.needs_input_grad[0] else None
        dw = torch.empty_like(w) if ctx.needs_input_grad[1] else None
        scratch = _scratch(d, x.device) if dw is not None else None
        _call(x, "block norm backward", _lib.lib().lb_norm_bwd, x.data_ptr(), w.data_ptr(), r.data_ptr(), du.data_ptr(), _p(dx),
              _p(dw), _p(scratch), x.numel() // d, d, dtype_code(x.dtype), dtype_code(w.dtype))
        return dx, dw, None


def block_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6) -> torch.Tensor:
    """weight * x / sqrt(mean(x^2) + eps) over the last dimension, differentiable in both. `weight` (d,) in x's type or
    fp32."""
    _require_rows(x, "block_norm")
    _same_device("block_norm", x, weight)
    (w,) = _channel_params("block_norm", x, x.shape[-1], weight)
    x = x.contiguous()
    if (x.requires_grad or w.requires_grad) and torch.is_grad_enabled():
        return _BlockNorm.apply(x, w, float(eps))
    return _norm_forward(x, w, float(eps), False)[0]


# --------------------------------------------------------------------------------------------------------------
# dropout
# --------------------------------------------------------------------------------------------------------------
def _threshold(what, p):
    t = int(float(p) * 65536 + 0.5) if 0.0 <= float(p) < 1.0 else -1
    if not 0 <= t <= 65535:
        raise ValueError(f"loopback_b200.{what}: need 0 <= p < 1 (to the nearest 1 / 65536), got {p}")
    return t


def _rng_args(what, x, rng):
    """(device pair or None, seed, offset)"""
    if isinstance(rng, torch.Tensor):
        if rng.dtype != torch.int64 or rng.shape != (2,) or not rng.is_contiguous():
            raise RuntimeError(f"loopback_b200.{what}: rng must be a contiguous int64 tensor (seed, offset) or a pair of integers")
        _same_device(what, x, rng)
        return rng, 0, 0
    if rng is None:
        raise ValueError(f"loopback_b200.{what}: dropout needs rng = (seed, offset)")
    seed, offset = (int(v) for v in rng)
    wrap = lambda v: (v & (1 << 64) - 1) - (1 << 64 if v >> 63 & 1 else 0)  # noqa: E731  any 64-bit pattern
    return None, wrap(seed), wrap(offset)


def _dropout_launch(x, threshold, rng, seed, offset, used):
    out = torch.empty_like(x)
    _call(x, "dropout", _lib.lib().lb_dropout, x.data_ptr(), out.data_ptr(), threshold, _p(rng), seed, offset, _p(used), x.numel(),
          dtype_code(x.dtype))
    return out


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, threshold, rng, seed, offset):
        used = None if rng is None else torch.empty_like(rng)
        out = _dropout_launch(x, threshold, rng, seed, offset, used)
        ctx.save_for_backward(used)
        ctx.args = threshold, seed, offset
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        (used,) = ctx.saved_tensors
        threshold, seed, offset = ctx.args
        return _dropout_launch(g.contiguous(), threshold, used, seed, offset, None), None, None, None, None


def dropout(x: torch.Tensor, p: float, rng) -> torch.Tensor:
    """Each element is kept with probability 1 - p (p to the nearest 1 / 65536) and scaled by the inverse of what is kept on
    average, else replaced by 0 (also where it is infinite or NaN). The mask is never stored: the backward draws the same
    numbers again.

    rng = (seed, offset), two 64-bit integers: a pair of Python integers, or a contiguous int64 tensor of two on x's
    device, read when the kernel runs (a captured graph draws new numbers on every replay if the offset is advanced in
    between; the backward uses the pair its forward used). The same pair gives the same mask for the same element count."""
    _require_cuda(x, "dropout")
    t = _threshold("dropout", p)
    pair, seed, offset = _rng_args("dropout", x, rng)
    x = x.contiguous()
    if x.requires_grad and torch.is_grad_enabled():
        return _Dropout.apply(x, t, pair, seed, offset)
    return _dropout_launch(x, t, pair, seed, offset, None)


# --------------------------------------------------------------------------------------------------------------
# the end of a block
# --------------------------------------------------------------------------------------------------------------
def _wcode(x, w, gate, kind, next_w):
    for t in (w, next_w, gate if kind == GATE_CHANNEL else None):
        if t is not None:
            return dtype_code(t.dtype)
    return dtype_code(x.dtype)


def _residual_forward(x, y, w, gate, scale_t, next_w, args, save):
    kind, scale, eps, threshold, rng, seed, offset = args
    d = x.shape[-1]
    n_tok, dev = x.numel() // d, x.device
    out = torch.empty_like(x)
    u = torch.empty_like(x) if next_w is not None else None
    ry = torch.empty(n_tok, dtype=torch.float32, device=dev) if save and w is not None else None
    ro = torch.empty(n_tok, dtype=torch.float32, device=dev) if save and next_w is not None else None
    used = torch.empty_like(rng) if save and rng is not None else None
    _call(x, "block residual", _lib.lib().lb_residual_fwd, x.data_ptr(), y.data_ptr(), _p(w), _p(gate), kind, _p(scale_t), scale,
          _p(next_w), out.data_ptr(), _p(u), _p(ry), _p(ro), threshold, _p(rng), seed, offset, _p(used), n_tok, d, eps,
          dtype_code(x.dtype), _wcode(x, w, gate, kind, next_w))
    return out, u, ry, ro, used


class _BlockResidual(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, y, w, gate, scale_t, next_w, args):
        out, u, ry, ro, used = _residual_forward(x, y, w, gate, scale_t, next_w, args, True)
        ctx.save_for_backward(x, y, w, gate, scale_t, next_w, ry, ro, used)
        ctx.args = args
        ctx.set_materialize_grads(False)
        return (out, u) if u is not None else out

    @staticmethod
    @once_differentiable
    def backward(ctx, g_out, g_u=None):
        x, y, w, gate, scale_t, next_w, ry, ro, used = ctx.saved_tensors
        kind, scale, _, threshold, _, seed, offset = ctx.args
        if g_out is None and g_u is None:
            return (None,) * 7
        d, dev = x.shape[-1], x.device
        g_out = None if g_out is None else g_out.contiguous()
        g_u = None if g_u is None else g_u.contiguous()
        grads = [torch.empty_like(t) if t is not None and need else None
                 for t, need in zip((x, y, w, gate, scale_t, next_w), ctx.needs_input_grad)]
        dx, dy, dw, dgate, dscale, dnext = grads
        sums = dw is not None or dscale is not None or dnext is not None or (dgate is not None and kind == GATE_CHANNEL)
        scratch = _scratch(d, dev) if sums else None
        _call(x, "block residual backward", _lib.lib().lb_residual_bwd, x.data_ptr(), y.data_ptr(), _p(w), _p(gate), kind,
              _p(scale_t), scale, _p(next_w), _p(ry), _p(ro), threshold, _p(used), seed, offset, _p(g_out), _p(g_u), _p(dx), _p(dy),
              _p(dw), _p(dgate), _p(dscale), _p(dnext), _p(scratch), x.numel() // d, d, dtype_code(x.dtype),
              _wcode(x, w, gate, kind, next_w))
        return (*grads, None)


def block_residual(x: torch.Tensor, y: torch.Tensor, weight=None, *, gate=None, scale=1.0, next_weight=None,
                   eps: float = 1e-6, p: float = 0.0, rng=None):
    """The end of a block in one pass over its rows: out = x + scale * gate * dropout(norm(y)), and, given `next_weight`, the
    norm the next block starts with. Returns out, or (out, norm of out).

    x, y         the residual stream and the block's output, one shape and type
    weight       (d,) of the norm after the block; None: no such norm, y itself is added
    gate         None, (d,) per channel, (..., 1) per token or x's shape
    scale        a number, or a tensor of one element (learned)
    next_weight  (d,) of the norm of out; its statistics come from out before it is rounded to its storage type
    p, rng       dropout of the (normed) block output, as in `dropout`, drawn over x's elements
    Per-channel parameters are in x's type or fp32, gates per token or element in x's. Differentiable in every tensor."""
    _require_rows(x, "block_residual")
    _same_device("block_residual", x, y, weight, gate, next_weight)
    if y.shape != x.shape or y.dtype != x.dtype:
        raise RuntimeError(f"loopback_b200.block_residual: x is {tuple(x.shape)} {x.dtype}, y is {tuple(y.shape)} {y.dtype}")
    d = x.shape[-1]
    kind = GATE_NONE
    if gate is not None:
        kind = (GATE_CHANNEL if gate.shape == (d,) else GATE_FULL if gate.shape == x.shape else
                GATE_TOKEN if gate.shape == x.shape[:-1] + (1,) else None)
        if kind is None:
            raise RuntimeError(f"loopback_b200.block_residual: a gate of shape {tuple(gate.shape)} is neither per channel, per "
                               f"token nor per element of {tuple(x.shape)}")
        if kind != GATE_CHANNEL and gate.dtype != x.dtype:
            raise RuntimeError(f"loopback_b200.block_residual: a gate per token or element has the rows' type, got {gate.dtype}")
    w, next_w, channel_gate = _channel_params("block_residual", x, d, weight, next_weight, gate if kind == GATE_CHANNEL else None)
    gate = channel_gate if kind == GATE_CHANNEL else None if gate is None else gate.contiguous()
    scale_t = None
    if isinstance(scale, torch.Tensor):
        if scale.numel() != 1:
            raise RuntimeError("loopback_b200.block_residual: a learned scale has one element")
        _same_device("block_residual", x, scale)
        scale_t, scale = scale.float(), 1.0
    t = _threshold("block_residual", p)
    pair, seed, offset = _rng_args("block_residual", x, rng) if t else (None, 0, 0)
    x, y = x.contiguous(), y.contiguous()
    args = kind, float(scale), float(eps), t, pair, seed, offset
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, y, w, gate, scale_t, next_w)):
        return _BlockResidual.apply(x, y, w, gate, scale_t, next_w, args)
    out, u = _residual_forward(x, y, w, gate, scale_t, next_w, args, False)[:2]
    return out if u is None else (out, u)


# --------------------------------------------------------------------------------------------------------------
# the gated feed-forward product
# --------------------------------------------------------------------------------------------------------------
_ACTS = {"silu": 0, "gelu": 1}
_FFN_FORWARD, _FFN_BACKWARD, _FFN_INFERENCE = 0, 1, 2


def _ffn_workspace(x, n_tok, d, f, kind):
    dev = x.get_device()
    if dev == _current_device():
        nbytes = _lib.lib().lb_ffn_workspace_bytes(n_tok, d, f, kind)
    else:
        with torch.cuda.device(dev):
            nbytes = _lib.lib().lb_ffn_workspace_bytes(n_tok, d, f, kind)
    if nbytes == 0:
        raise RuntimeError("loopback_b200.gated_ffn: " + _lib.lib().lb_last_error_string().decode("utf-8", "replace"))
    return torch.empty(nbytes, dtype=torch.uint8, device=x.device), nbytes


def _ffn_forward(x, wg, wu, wd, act, save):
    d, f = x.shape[-1], wg.shape[0]
    n_tok = x.numel() // d
    y = torch.empty_like(x)
    h = kept = None
    if save:
        h = torch.empty((n_tok, f), dtype=x.dtype, device=x.device)
        kept = torch.empty(_lib.lib().lb_ffn_kept_bytes(n_tok, f), dtype=torch.uint8, device=x.device)
    ws, nbytes = _ffn_workspace(x, n_tok, d, f, _FFN_FORWARD if save else _FFN_INFERENCE)
    _call(x, "gated ffn", _lib.lib().lb_ffn_fwd, x.data_ptr(), wg.data_ptr(), wu.data_ptr(), wd.data_ptr(), y.data_ptr(), _p(h),
          _p(kept), ws.data_ptr(), nbytes, n_tok, d, f, act, _lib.LB_DTYPE_BF16)
    return y, h, kept


class _GatedFFN(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, wg, wu, wd, act):
        y, h, kept = _ffn_forward(x, wg, wu, wd, act, True)
        ctx.save_for_backward(x, wg, wu, wd, h, kept)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, wg, wu, wd, h, kept = ctx.saved_tensors
        d, f = x.shape[-1], wg.shape[0]
        n_tok = x.numel() // d
        dy = dy.contiguous()
        need = ctx.needs_input_grad
        dx = torch.empty_like(x) if need[0] else None
        dgu = torch.empty((2, f, d), dtype=x.dtype, device=x.device) if need[1] or need[2] else None
        dwd = torch.empty_like(wd) if need[3] else None
        ws, nbytes = _ffn_workspace(x, n_tok, d, f, _FFN_BACKWARD)
        _call(x, "gated ffn backward", _lib.lib().lb_ffn_bwd, x.data_ptr(), wg.data_ptr(), wu.data_ptr(), wd.data_ptr(),
              h.data_ptr(), kept.data_ptr(), dy.data_ptr(), _p(dx), _p(dgu), _p(dwd), ws.data_ptr(), nbytes, n_tok, d, f,
              _lib.LB_DTYPE_BF16)
        return dx, dgu[0] if need[1] else None, dgu[1] if need[2] else None, dwd, None


def gated_ffn(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor, act: str = "silu") -> torch.Tensor:
    """(act(x w_gate^T) * (x w_up^T)) w_down^T, differentiable in every tensor.

    x (..., d), w_gate and w_up (f, d), w_down (d, f), all bf16 (the products run on the tensor cores in bf16 with fp32
    accumulation; h and the result, and in the backward the two gradients behind the product, are each rounded once),
    contiguous weights, d and f multiples of 8. act: "silu" or "gelu" (with erf). Both projections, the activation and the
    product are one launch. With gradients h and two factors of 24 bits are kept: 8 bytes per token and column of f."""
    _require_rows(x, "gated_ffn")
    _same_device("gated_ffn", x, w_gate, w_up, w_down)
    if act not in _ACTS:
        raise ValueError(f"loopback_b200.gated_ffn: act is one of {sorted(_ACTS)}, got {act!r}")
    d = x.shape[-1]
    if w_gate.dim() != 2 or w_gate.shape[1] != d or w_up.shape != w_gate.shape or w_down.shape != w_gate.shape[::-1]:
        raise RuntimeError(f"loopback_b200.gated_ffn: rows have {d} columns, weights are {tuple(w_gate.shape)}, "
                           f"{tuple(w_up.shape)}, {tuple(w_down.shape)}; expected (f, d), (f, d), (d, f)")
    if not x.dtype == w_gate.dtype == w_up.dtype == w_down.dtype == torch.bfloat16:
        raise RuntimeError(f"loopback_b200.gated_ffn: the products run in bf16, got rows of {x.dtype} and weights of "
                           f"{w_gate.dtype}, {w_up.dtype}, {w_down.dtype}")
    if not (w_gate.is_contiguous() and w_up.is_contiguous() and w_down.is_contiguous()):
        raise RuntimeError("loopback_b200.gated_ffn: weights must be contiguous")
    x = x.contiguous()
    if torch.is_grad_enabled() and (x.requires_grad or w_gate.requires_grad or w_up.requires_grad or w_down.requires_grad):
        return _GatedFFN.apply(x, w_gate, w_up, w_down, _ACTS[act])
    return _ffn_forward(x, w_gate, w_up, w_down, _ACTS[act], False)[0]
