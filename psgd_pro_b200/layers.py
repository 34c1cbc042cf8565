"""Operators of the model whose parameters KronWhiten trains, as hand-written sm_100a kernels (no counterpart in the
reference, whose models run on torch's own operators):

  residual_norm          the joint between two blocks: the norm after a block, dropout, gate, scaled residual add and
                         the norm before the next block in one pass, with its backward pass
  dropout                counter-based: the mask is a function of (seed, offset, element) and is never stored
  linear_cross_entropy   the loss of a large vocabulary from the last hidden states and the head's weight, with both
                         gradients, without ever keeping the logits

Tensors are CUDA fp32, bf16 or fp16; arithmetic, statistics and sums are fp32 and each output is rounded once. Work is
enqueued on the current stream of the inputs' device; outputs and workspaces come from torch's allocator on that stream.
The functions take part in autograd; the *_forward / *_grad forms are the same launches for callers that hold the
gradients themselves (KronWhiten.step_math takes them as they come). Argument errors raise RuntimeError at the call.
A target that is no class is found on the device: it counts as ignored, and the next linear_cross_entropy (or
check_errors()) raises, as for the operators of psgd_pro_b200.ops."""
import ctypes
from typing import NamedTuple, Optional

import torch
from torch import Tensor

from . import _capi, ops
from ._capi import check
from .ops import check_errors, reset_errors

__all__ = ["dropout", "dropout_grad", "residual_norm", "residual_norm_forward", "residual_norm_grad",
           "linear_cross_entropy", "linear_cross_entropy_grad", "ResidualNormGrads", "check_errors", "reset_errors"]

_TYPES = {torch.float32: _capi.PSGD_F32, torch.bfloat16: _capi.PSGD_BF16, torch.float16: _capi.PSGD_F16}
_NORMS = {"rms": _capi.PSGD_NORM_RMS, "layer": _capi.PSGD_NORM_LAYER}
_REDUCTIONS = {"none": _capi.PSGD_REDUCE_NONE, "mean": _capi.PSGD_REDUCE_MEAN, "sum": _capi.PSGD_REDUCE_SUM}
DEFAULT_PIECE_BYTES = 4 << 30


def _fail(text):
    raise RuntimeError(f"psgd_pro_b200.layers: {text}")


def _elements(t, name):
    code = _TYPES.get(t.dtype)
    if code is None or not t.is_cuda:
        _fail(f"{name} must be an fp32, bf16 or fp16 CUDA tensor")
    return code


def _like(t, ref, name, shape=None):
    if t.dtype != ref.dtype or t.device != ref.device:
        _fail(f"{name} must have the type and device of the first argument")
    if shape is not None and t.shape != shape:
        _fail(f"{name} must have the shape {tuple(shape)}")


def _ptr(t):
    return None if t is None else t.data_ptr()


def _stream(t):
    return torch.cuda.current_stream(t.device).cuda_stream


class _On:
    """Makes the tensor's device current for the launches inside."""
    __slots__ = ("index", "before")

    def __init__(self, t):
        self.index = t.get_device()

    def __enter__(self):
        self.before = torch.cuda.current_device()
        if self.before != self.index:
            torch.cuda.set_device(self.index)

    def __exit__(self, *_):
        if self.before != self.index:
            torch.cuda.set_device(self.before)
        return False


# ---- dropout --------------------------------------------------------------------------------------------------------
def _generator(p, seed, offset, device):
    """(threshold, scale, seed, offset, rng pointer) of a mask."""
    if not 0.0 <= p <= 1.0:
        _fail("the dropout probability must lie in [0, 1]")
    threshold = int(round(p * 65536))
    scale = 65536.0 / (65536 - threshold) if threshold < 65536 else 0.0
    if isinstance(seed, Tensor):
        if seed.dtype != torch.int64 or seed.device != device or seed.numel() != 2 or not seed.is_contiguous():
            _fail("a seed tensor must hold two contiguous int64 values (seed, offset) on the inputs' device")
        return threshold, scale, 0, 0, seed.data_ptr()
    return threshold, scale, seed & 0xFFFFFFFFFFFFFFFF, offset & 0xFFFFFFFFFFFFFFFF, None


def _dropout(x, p, seed, offset, residual):
    code = _elements(x, "x")
    threshold, scale, seed, offset, rng = _generator(p, seed, offset, x.device)
    x = x.contiguous()
    if residual is not None:
        _like(residual, x, "residual", x.shape)
        residual = residual.contiguous()
    out = torch.empty_like(x)
    spec = _capi.Dropout(x.data_ptr(), _ptr(residual), out.data_ptr(), x.numel(), code, threshold, scale, seed, offset, rng)
    with _On(x):
        check(_capi.lib().psgd_dropout(ctypes.byref(spec), _stream(x)), "psgd_dropout")
    return out


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, p, seed, offset, residual):
        ctx.mask = (p, seed, offset)
        return _dropout(x, p, seed, offset, residual)

    @staticmethod
    def backward(ctx, dy):
        dx = dropout_grad(dy, *ctx.mask) if ctx.needs_input_grad[0] else None
        return dx, None, None, None, dy if ctx.needs_input_grad[4] else None


def dropout(x: Tensor, p: float, seed, offset: int = 0, residual: Optional[Tensor] = None) -> Tensor:
    """[residual +] x with each element kept with probability 1 - p and scaled by its inverse, or zero.

    Element i (in row-major order) is kept when 16-bit field i % 8 of the Philox4x32-10 output for counter
    (i / 8, offset) under the 64-bit key `seed` is at least T = round(65536 p), whatever the type, shape or strides; the scale
    is 1 / (1 - T / 65536), so p has a resolution of 2^-16. The same (seed, offset) gives the same mask: take another
    offset for each use and step. seed may instead be an int64 CUDA tensor (seed, offset), read by the kernel, so that a
    captured CUDA graph draws another mask at each replay; it must not change before the backward pass has run."""
    if torch.is_grad_enabled() and (x.requires_grad or (residual is not None and residual.requires_grad)):
        return _Dropout.apply(x, p, seed, offset, residual)
    return _dropout(x, p, seed, offset, residual)


def dropout_grad(dy: Tensor, p: float, seed, offset: int = 0) -> Tensor:
    """Gradient of dropout's x for the gradient dy of its output (a residual's gradient is dy itself)."""
    return _dropout(dy, p, seed, offset, None)


# ---- the joint between two blocks ------------------------------------------------------------------------------------
class ResidualNormGrads(NamedTuple):
    """Gradients of residual_norm's inputs; None where the input (or, for rms norms, the bias) is not there."""
    dx: Tensor
    dy: Tensor
    dweight: Optional[Tensor]
    dbias: Optional[Tensor]
    dpost_weight: Optional[Tensor]
    dpost_bias: Optional[Tensor]
    dgate: Optional[Tensor]


def _rows(t, d, name):
    """t as rows of d elements with a unit stride inside (a copy only where its strides allow no such view)."""
    if t.dim() != 2:
        t = t.reshape(-1, d)
    if t.stride(1) != 1 and d > 1 or t.stride(0) < d and t.shape[0] > 1:
        t = t.contiguous()
    return t


def _joint_spec(x, y, norm, post_norm, weight, bias, post_weight, post_bias, gate, scale, eps, dropout_p, seed, offset):
    """(spec, rows, tensors to keep until the launch) of a joint of x (the residual, or its output) and y."""
    code = _elements(x, "x")
    if x.dim() < 1 or x.shape[-1] < 1 or x.shape[-1] > _capi.JOINT_MAX_D:
        _fail(f"rows must have 1 to {_capi.JOINT_MAX_D} elements")
    if norm not in _NORMS:
        _fail("norm must be 'rms' or 'layer'")
    _like(y, x, "y", x.shape)
    d = x.shape[-1]
    params, kept = None, []
    for t, name in ((weight, "weight"), (bias, "bias"), (post_weight, "post_weight"), (post_bias, "post_bias")):
        if t is None:
            continue
        _elements(t, name)
        if t.shape != (d,) or t.device != x.device:
            _fail(f"{name} must hold {d} values on the inputs' device")
        if params is None:
            params = t.dtype
        if t.dtype != params or params not in (x.dtype, torch.float32):
            _fail("weights and biases must share one type: that of x, or fp32")
    if not post_norm and (post_weight is not None or post_bias is not None):
        _fail("post_weight and post_bias need post_norm")
    if norm == "rms" and (bias is not None or post_bias is not None):
        _fail("an rms norm has no bias")
    if not eps > 0.0:
        _fail("eps must be positive")
    vectors = [t if t is None or t.is_contiguous() else t.contiguous() for t in (weight, bias, post_weight, post_bias)]
    x2, y2 = _rows(x, d, "x"), _rows(y, d, "y")
    rows = x2.shape[0]
    gates = 0
    if gate is not None:
        _like(gate, x, "gate")
        gates = _gates(gate, x, rows)
        gate = gate.contiguous()
    threshold, keep, seed, offset, rng = _generator(dropout_p, seed, offset, x.device)
    s = _capi.Joint()
    s.x, s.y, s.ld_x, s.ld_y = x2.data_ptr(), y2.data_ptr(), x2.stride(0), y2.stride(0)
    s.weight, s.bias, s.post_weight, s.post_bias = (_ptr(t) for t in vectors)
    s.gate, s.gates, s.rows, s.d, s.dtype = _ptr(gate), gates, rows, d, code
    s.param_dtype = _TYPES[params or torch.float32]
    s.kind, s.post, s.scale, s.eps = _NORMS[norm], int(post_norm), scale, eps
    s.threshold, s.keep_scale, s.seed, s.offset, s.rng = threshold, keep, seed, offset, rng
    return s, rows, (x2, y2, vectors, gate)


def _gates(gate, x, rows):
    """How many rows of d the gate has: its leading dimensions are the first dimensions of x (ones after them), so that
    each of its rows serves consecutive rows of x; for a two-dimensional gate, any number that divides them."""
    d = x.shape[-1]
    if gate.dim() < 1 or gate.shape[-1] != d:
        _fail(f"gate must have rows of {d} values")
    lead, count = tuple(gate.shape[:-1]), gate.numel() // d
    if gate.dim() <= 2:
        if count >= 1 and (rows == 0 or rows % count == 0):
            return count
    elif gate.dim() == x.dim():
        k = len(lead)
        while k and lead[k - 1] == 1:
            k -= 1
        if lead[:k] == tuple(x.shape[:k]) and count:
            return count
    _fail("gate must be (d), (g, d) with g dividing the rows, or x's shape with ones after its first dimensions")


def residual_norm_forward(x: Tensor, y: Tensor, *, norm: str = "rms", post_norm: bool = False, weight=None, bias=None,
                          post_weight=None, post_bias=None, gate=None, scale: float = 1.0, eps: float = 1e-6,
                          dropout_p: float = 0.0, seed=0, offset: int = 0):
    """(out, normed, stats) of residual_norm; stats (rows, 4) in fp32 is what residual_norm_grad needs besides out and y."""
    s, rows, keep = _joint_spec(x, y, norm, post_norm, weight, bias, post_weight, post_bias, gate, scale, eps, dropout_p,
                                seed, offset)
    out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    normed = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    stats = torch.empty(rows, 4, dtype=torch.float32, device=x.device)
    s.out, s.normed, s.stats = out.data_ptr(), normed.data_ptr(), stats.data_ptr()
    with _On(x):
        check(_capi.lib().psgd_joint_forward(ctypes.byref(s), _stream(x)), "psgd_joint_forward")
    return out, normed, stats


def residual_norm_grad(d_out: Optional[Tensor], d_normed: Optional[Tensor], out: Tensor, y: Tensor, stats: Tensor, *,
                       norm: str = "rms", post_norm: bool = False, weight=None, bias=None, post_weight=None,
                       post_bias=None, gate=None, scale: float = 1.0, eps: float = 1e-6, dropout_p: float = 0.0, seed=0,
                       offset: int = 0) -> ResidualNormGrads:
    """Gradients of residual_norm's inputs from those of its outputs (None: zero), its output `out`, its input y and the
    stats of the forward call with the same options."""
    s, rows, keep = _joint_spec(out, y, norm, post_norm, weight, bias, post_weight, post_bias, gate, scale, eps, dropout_p,
                                seed, offset)
    if stats.shape != (rows, 4) or stats.dtype != torch.float32 or stats.device != out.device or not stats.is_contiguous():
        _fail("stats must be what residual_norm_forward returned")
    d, device = s.d, out.device
    pd = next((t.dtype for t in (weight, bias, post_weight, post_bias) if t is not None), torch.float32)
    ups = []
    for t, name in ((d_out, "d_out"), (d_normed, "d_normed")):
        if t is not None:
            _like(t, out, name, out.shape)
            t = _rows(t, d, name)
        ups.append(t)
    s.stats, s.d_out, s.d_normed = stats.data_ptr(), _ptr(ups[0]), _ptr(ups[1])
    s.ld_d_out, s.ld_d_normed = (d if t is None else t.stride(0) for t in ups)
    layer = s.kind == _capi.PSGD_NORM_LAYER

    def vector(there):
        make = torch.empty if rows else torch.zeros
        return make(d, dtype=pd, device=device) if there else None

    dx, dy = (torch.empty(out.shape, dtype=out.dtype, device=device) for _ in range(2))
    dweight, dbias, dpw, dpb = (vector(b) for b in (True, layer, post_norm, post_norm and layer))
    dgate = None if gate is None else (torch.empty if rows else torch.zeros)(gate.shape, dtype=gate.dtype, device=device)
    s.dx, s.dy, s.dgate = dx.data_ptr(), dy.data_ptr(), _ptr(dgate)
    s.dweight, s.dbias, s.dpost_weight, s.dpost_bias = (_ptr(t) for t in (dweight, dbias, dpw, dpb))
    with _On(out):
        L = _capi.lib()
        size = L.psgd_joint_workspace(ctypes.byref(s))
        check(min(size, 0), "psgd_joint_workspace")
        ws = torch.empty(max(size, 16), dtype=torch.uint8, device=device)
        check(L.psgd_joint_backward(ctypes.byref(s), ws.data_ptr(), size, _stream(out)), "psgd_joint_backward")
    return ResidualNormGrads(dx, dy, dweight if weight is not None else None, dbias if bias is not None else None,
                             dpw if post_weight is not None else None, dpb if post_bias is not None else None, dgate)


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, y, weight, bias, post_weight, post_bias, gate, options):
        out, normed, stats = residual_norm_forward(x, y, weight=weight, bias=bias, post_weight=post_weight,
                                                   post_bias=post_bias, gate=gate, **options)
        ctx.save_for_backward(out, y, stats, weight, bias, post_weight, post_bias, gate)
        ctx.options = options
        ctx.set_materialize_grads(False)
        return out, normed

    @staticmethod
    def backward(ctx, d_out, d_normed):
        out, y, stats, weight, bias, post_weight, post_bias, gate = ctx.saved_tensors
        if d_out is None and d_normed is None:
            return (None,) * 8
        g = residual_norm_grad(d_out, d_normed, out, y, stats, weight=weight, bias=bias, post_weight=post_weight,
                               post_bias=post_bias, gate=gate, **ctx.options)
        return (*(t if need else None for t, need in zip(g, ctx.needs_input_grad)), None)


def residual_norm(x: Tensor, y: Tensor, *, norm: str = "rms", post_norm: bool = False, weight=None, bias=None,
                  post_weight=None, post_bias=None, gate=None, scale: float = 1.0, eps: float = 1e-6,
                  dropout_p: float = 0.0, seed=0, offset: int = 0):
    """(out, normed): out = x + scale * gate * dropout(post(y)) and normed = pre(out), where x is the residual stream, y a
    block's output, post the norm after the block (post_norm; otherwise y itself) and pre the norm before the next one.

    norm 'rms': a / sqrt(mean a^2 + eps) * weight; 'layer': (a - mean) / sqrt(var + eps) * weight + bias, for both norms.
    x, y: (..., d), d at most 8192, any strides (rows with a unit stride are read in place). weight, bias, post_weight,
    post_bias: (d), or None for ones and zeros, all of x's type or all fp32. gate: (d), (g, d), or x's shape with ones after
    its first dimensions, each row serving as many consecutive rows of x; its gradient sums over them. scale: the
    residual scale. Dropout as in dropout(), over the elements of x in row-major order."""
    options = dict(norm=norm, post_norm=post_norm, scale=scale, eps=eps, dropout_p=dropout_p, seed=seed, offset=offset)
    tensors = (x, y, weight, bias, post_weight, post_bias, gate)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        return _ResidualNorm.apply(*tensors, options)
    return residual_norm_forward(x, y, weight=weight, bias=bias, post_weight=post_weight, post_bias=post_bias, gate=gate,
                                 **options)[:2]


# ---- the loss of a large vocabulary ----------------------------------------------------------------------------------
def _lce(h, w, target, grads, grad, ignore_index, label_smoothing, z_loss, reduction, piece_bytes):
    code = _elements(h, "h")
    if reduction not in _REDUCTIONS:
        _fail("reduction must be 'none', 'mean' or 'sum'")
    if w.dim() != 2 or h.dim() < 1 or h.shape[-1] != w.shape[1] or w.shape[0] < 1 or w.shape[1] < 1:
        _fail("h (..., d) and w (v, d) must share d")
    _like(w, h, "w")
    if target.shape != h.shape[:-1] or target.dtype != torch.int64 or target.device != h.device:
        _fail("target must hold one int64 value for each row of h, on its device")
    if not 0.0 <= label_smoothing <= 1.0:
        _fail("label_smoothing must lie in [0, 1]")
    v, d = w.shape
    h2, w2, t = _rows(h, d, "h"), _rows(w, d, "w"), target.contiguous()
    n = h2.shape[0]
    none = reduction == "none"
    if grad is not None:
        if grad.dtype != torch.float32 or grad.device != h.device or grad.shape != (target.shape if none else ()):
            _fail("grad must be fp32 on the inputs' device: a scalar, or one value for each row with reduction 'none'")
        grad = grad.contiguous()
    loss = torch.empty(target.shape if none else (), dtype=torch.float32, device=h.device)
    dh = torch.empty(h.shape, dtype=h.dtype, device=h.device) if grads else None
    dw = torch.empty(w.shape, dtype=w.dtype, device=h.device) if grads else None
    if n == 0:
        for x in (loss, dw):
            if x is not None:
                x.zero_()
        return loss, dh, dw
    s = _capi.Lce()
    s.h, s.w, s.target, s.grad, s.loss, s.dh, s.dw = (_ptr(x) for x in (h2, w2, t, grad, loss, dh, dw))
    s.ld_h, s.ld_w, s.n, s.d, s.v, s.dtype = max(h2.stride(0), d), max(w2.stride(0), d), n, d, v, code
    s.reduction, s.grads, s.ignore_index = _REDUCTIONS[reduction], int(grads), ignore_index
    s.label_smoothing, s.z_loss, s.piece_bytes = label_smoothing, z_loss, piece_bytes
    with _On(h), ops._call(h) as err:
        L = _capi.lib()
        size = L.psgd_lce_workspace(ctypes.byref(s))
        check(min(size, 0), "psgd_lce_workspace")
        ws = torch.empty(size, dtype=torch.uint8, device=h.device)
        s.workspace, s.workspace_bytes = ws.data_ptr(), size
        check(L.psgd_lce(ctypes.byref(s), err.data_ptr(), _stream(h)), "psgd_lce")
    return loss, dh, dw


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, h, w, target, options):
        ctx.options = options
        ctx.save_for_backward(h, w, target)
        return _lce(h, w, target, False, None, **options)[0]

    @staticmethod
    def backward(ctx, grad):
        h, w, target = ctx.saved_tensors
        _, dh, dw = _lce(h, w, target, True, grad.float(), **ctx.options)
        return dh if ctx.needs_input_grad[0] else None, dw if ctx.needs_input_grad[1] else None, None, None


def linear_cross_entropy(h: Tensor, w: Tensor, target: Tensor, *, ignore_index: int = -100, label_smoothing: float = 0.0,
                         z_loss: float = 0.0, reduction: str = "mean", piece_bytes: int = DEFAULT_PIECE_BYTES) -> Tensor:
    """Cross entropy of the logits h w^T against target, in fp32, plus z_loss times the squared log-normaliser:

        lse = log sum_v exp(l_v);  loss = (1 - s) (lse - l_target) + s (lse - mean_v l_v) + z_loss lse^2

    h (..., d), w (v, d) of one type; target (...) int64. Rows whose target is ignore_index have loss 0 and touch nothing
    (not even with NaN in h); 'mean' divides by the number of the others (0 when there is none). reduction 'none' keeps
    target's shape.

    Under autograd the forward call keeps h, w and target only, and the backward call forms the loss again with both
    gradients; where the gradient is wanted in any case linear_cross_entropy_grad does all in one (the same kernels, a
    quarter fewer operations). piece_bytes bounds what is kept of the vocabulary's probabilities at a time (16 bits each,
    fp32: 80 bits); tokens are taken in pieces of that size."""
    options = dict(ignore_index=ignore_index, label_smoothing=label_smoothing, z_loss=z_loss, reduction=reduction,
                   piece_bytes=piece_bytes)
    if torch.is_grad_enabled() and (h.requires_grad or w.requires_grad):
        return _LinearCrossEntropy.apply(h, w, target, options)
    return _lce(h, w, target, False, None, **options)[0]


def linear_cross_entropy_grad(h: Tensor, w: Tensor, target: Tensor, *, grad: Optional[Tensor] = None,
                              ignore_index: int = -100, label_smoothing: float = 0.0, z_loss: float = 0.0,
                              reduction: str = "mean", piece_bytes: int = DEFAULT_PIECE_BYTES):
    """(loss, dh, dw): the loss and the gradients of h and w for the upstream gradient `grad` (fp32; default ones)."""
    return _lce(h, w, target, True, grad, ignore_index, label_smoothing, z_loss, reduction, piece_bytes)
