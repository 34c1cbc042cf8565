"""Operators of the model whose parameters KronWhiten trains, as hand-written sm_100a kernels (no counterpart in the
reference, whose models run on torch's own operators):

  residual_norm          the joint between two blocks: the norm after a block, dropout, gate, scaled residual add and
                         the norm before the next block in one pass, with its backward pass
  dropout                counter-based: the mask is a function of (seed, offset, element) and is never stored
  linear_cross_entropy   the loss of a large vocabulary from the last hidden states and the head's weight, with both
                         gradients, without ever keeping the logits

Tensors are CUDA fp32, bf16 or fp16; arithmetic, statistics and sums are fp32 and each output is rounded once (the
gradients of 16-bit losses also carry the rounding of an operand: linear_cross_entropy). Work is enqueued on the current
stream of the inputs' device; outputs and workspaces come from torch's allocator on that stream.
The functions take part in autograd (once: second derivatives and forward mode raise); the *_forward / *_grad forms are the
same launches for callers that hold the gradients themselves (KronWhiten.step_math takes them as they come) and that
autograd does not see. Argument errors raise RuntimeError at the call.
A target that is no class is found on the device: it counts as ignored, and later linear_cross_entropy calls (and
check_errors(), which waits) raise until reset_errors(), as for the operators of psgd_pro_b200.ops."""
import ctypes
import threading
from typing import NamedTuple, Optional

import torch
from torch import Tensor
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _capi
from ._capi import check

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
    if t.dtype != ref.dtype or not t.is_cuda or t.get_device() != ref.get_device():
        _fail(f"{name} must have the type and device of the first argument")
    if shape is not None and t.shape != shape:
        _fail(f"{name} must have the shape {tuple(shape)}")


def _ptr(t):
    return None if t is None else t.data_ptr()


def _launch(device, fn, *args):
    """fn(*args, stream) with `device` current, on its current stream (asked for by its raw handle: the Stream object
    costs thirty times as much, and these calls are as short as their host code)."""
    if torch._C._cuda_getDevice() == device:
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(device))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(device))
    if rc != 0:
        check(rc, fn.__name__)


def _new(t):
    """An uninitialised contiguous tensor like t."""
    return torch.empty_like(t) if t.is_contiguous() else torch.empty_like(t, memory_format=torch.contiguous_format)


def _differentiated(*tensors):
    """Whether autograd has to see the call: a gradient will be asked for, or an input carries a forward-mode tangent, which a
    launch of its own would drop without a word (the autograd functions have no forward-mode formula and raise)."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        return True
    return forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


# ---- dropout --------------------------------------------------------------------------------------------------------
def _generator(p, seed, offset, x):
    """(threshold, scale, seed, offset, rng pointer) of a mask."""
    if not 0.0 <= p <= 1.0:
        _fail("the dropout probability must lie in [0, 1]")
    threshold = int(round(p * 65536))
    scale = 65536.0 / (65536 - threshold) if threshold < 65536 else 0.0
    if isinstance(seed, Tensor):
        if seed.dtype != torch.int64 or seed.device != x.device or seed.numel() != 2 or not seed.is_contiguous():
            _fail("a seed tensor must hold two contiguous int64 values (seed, offset) on the inputs' device")
        return threshold, scale, 0, 0, seed.data_ptr()
    return threshold, scale, int(seed) & 0xFFFFFFFFFFFFFFFF, int(offset) & 0xFFFFFFFFFFFFFFFF, None


def _dropout(x, p, seed, offset, residual):
    code = _elements(x, "x")
    threshold, scale, seed, offset, rng = _generator(p, seed, offset, x)
    if not x.is_contiguous():
        x = x.contiguous()
    at = None
    if residual is not None:
        _like(residual, x, "residual", x.shape)
        residual = residual.contiguous()
        at = residual.data_ptr()
    out = torch.empty_like(x)
    spec = _capi.Dropout(x.data_ptr(), at, out.data_ptr(), x.numel(), code, threshold, scale, seed, offset, rng)
    _launch(x.get_device(), _capi.lib().psgd_dropout, ctypes.byref(spec))
    return out


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, p, seed, offset, residual):
        # (a seed tensor is saved as one, so that a change of it before the backward pass raises there)
        ctx.mask = (p, None if isinstance(seed, Tensor) else seed, offset)
        ctx.save_for_backward(seed if isinstance(seed, Tensor) else None)
        return _dropout(x, p, seed, offset, residual)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        dx = None
        if ctx.needs_input_grad[0]:
            p, seed, offset = ctx.mask
            rng, = ctx.saved_tensors
            dx = dropout_grad(dy, p, seed if rng is None else rng, offset)
        return dx, None, None, None, dy if ctx.needs_input_grad[4] else None


def dropout(x: Tensor, p: float, seed, offset: int = 0, residual: Optional[Tensor] = None) -> Tensor:
    """[residual +] x with each element kept with probability 1 - p and scaled by its inverse, or zero.

    Element i (in row-major order) is kept when 16-bit field i % 8 of the Philox4x32-10 output for counter
    (i / 8, offset) under the 64-bit key `seed` is at least T = round(65536 p), whatever the type, shape or strides; the scale
    is 1 / (1 - T / 65536), so p has a resolution of 2^-16. The same (seed, offset) gives the same mask: take another
    offset for each use and step. seed may instead be an int64 CUDA tensor (seed, offset), read by the kernel, so that a
    captured CUDA graph draws another mask at each replay; it must not change before the backward pass has run (autograd
    raises where it sees a change in place)."""
    if _differentiated(x, residual):
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


def _rows(t, d):
    """(t, stride of its rows): t as rows of d elements with a unit stride inside (a copy only where its strides allow no
    such view)."""
    if t.is_contiguous():
        return t, d
    if t.dim() != 2:
        t = t.reshape(-1, d)
    if (t.stride(1) != 1 and d > 1) or (t.stride(0) < d and t.shape[0] > 1):
        t = t.contiguous()
    return t, max(t.stride(0), d)


def _joint_spec(x, y, norm, post_norm, weight, bias, post_weight, post_bias, gate, scale, eps, dropout_p, seed, offset):
    """(spec, rows, type of the parameters, tensors to keep until the launch) of a joint of x (the residual, or its output)
    and y."""
    dtype, device, shape = x.dtype, x.get_device(), x.shape
    code, kind = _TYPES.get(dtype), _NORMS.get(norm)
    if code is None or device < 0:
        _fail("x must be an fp32, bf16 or fp16 CUDA tensor")
    if kind is None:
        _fail("norm must be 'rms' or 'layer'")
    d = shape[-1] if shape else 0
    if not 1 <= d <= _capi.JOINT_MAX_D:
        _fail(f"rows must have 1 to {_capi.JOINT_MAX_D} elements")
    if y.dtype != dtype or y.shape != shape or y.get_device() != device:
        _fail("y must have the type, shape and device of the first argument")
    if not post_norm and (post_weight is not None or post_bias is not None):
        _fail("post_weight and post_bias need post_norm")
    if kind == 0 and (bias is not None or post_bias is not None):
        _fail("an rms norm has no bias")
    if not eps > 0.0:
        _fail("eps must be positive")
    params, pointers, kept = None, [None] * 4, []
    for k, t in enumerate((weight, bias, post_weight, post_bias)):
        if t is None:
            continue
        if params is None:
            params = t.dtype
        if t.dtype != params or (params != dtype and params != torch.float32) or t.get_device() != device or \
                t.dim() != 1 or t.numel() != d:
            _fail(f"weights and biases must hold {d} values of one type, that of x or fp32, on the inputs' device")
        if not t.is_contiguous():
            t = t.contiguous()
            kept.append(t)
        pointers[k] = t.data_ptr()
    (x, ld_x), (y, ld_y) = _rows(x, d), _rows(y, d)
    rows, gates, gate_at = x.numel() // d, 0, None
    if gate is not None:
        if gate.dtype != dtype or gate.get_device() != device:
            _fail("gate must have the type and device of the first argument")
        gates = _gates(gate, shape, rows)
        gate = gate.contiguous()
        gate_at = gate.data_ptr()
    threshold, keep, seed, offset, rng = _generator(dropout_p, seed, offset, x) if dropout_p else (0, 1.0, 0, 0, None)
    s = _capi.Joint(x.data_ptr(), y.data_ptr(), None, None, None, *pointers, gate_at, None, None, None, None, None, None,
                    None, None, None, ld_x, ld_y, d, d, rows, gates, d, code, _TYPES[params or torch.float32], kind,
                    post_norm, scale, eps, threshold, keep, seed, offset, rng)
    return s, rows, params or torch.float32, (x, y, kept, gate)


def _gates(gate, shape, rows):
    """How many rows of d the gate has: its leading dimensions are the first dimensions of x (ones after them), so that
    each of its rows serves consecutive rows of x; for a two-dimensional gate, any number that divides them."""
    d = shape[-1]
    if gate.dim() < 1 or gate.shape[-1] != d:
        _fail(f"gate must have rows of {d} values")
    lead, count = tuple(gate.shape[:-1]), gate.numel() // d
    if gate.dim() <= 2:
        if count >= 1 and (rows == 0 or rows % count == 0):
            return count
    elif gate.dim() == len(shape):
        k = len(lead)
        while k and lead[k - 1] == 1:
            k -= 1
        if lead[:k] == tuple(shape[:k]) and count:
            return count
    _fail("gate must be (d), (g, d) with g dividing the rows, or x's shape with ones after its first dimensions")


def residual_norm_forward(x: Tensor, y: Tensor, *, norm: str = "rms", post_norm: bool = False, weight=None, bias=None,
                          post_weight=None, post_bias=None, gate=None, scale: float = 1.0, eps: float = 1e-6,
                          dropout_p: float = 0.0, seed=0, offset: int = 0):
    """(out, normed, stats) of residual_norm; stats (rows, 4) in fp32 is what residual_norm_grad needs besides out and y."""
    s, rows, _, keep = _joint_spec(x, y, norm, post_norm, weight, bias, post_weight, post_bias, gate, scale, eps, dropout_p,
                                   seed, offset)
    out, normed = _new(x), _new(x)
    stats = x.new_empty((rows, 4), dtype=torch.float32)
    s.out, s.normed, s.stats = out.data_ptr(), normed.data_ptr(), stats.data_ptr()
    _launch(x.get_device(), _capi.lib().psgd_joint_forward, ctypes.byref(s))
    return out, normed, stats


def residual_norm_grad(d_out: Optional[Tensor], d_normed: Optional[Tensor], out: Tensor, y: Tensor, stats: Tensor, *,
                       norm: str = "rms", post_norm: bool = False, weight=None, bias=None, post_weight=None,
                       post_bias=None, gate=None, scale: float = 1.0, eps: float = 1e-6, dropout_p: float = 0.0, seed=0,
                       offset: int = 0) -> ResidualNormGrads:
    """Gradients of residual_norm's inputs from those of its outputs (None: zero), its output `out`, its input y and the
    stats of the forward call with the same options. The stats are those of the sum before its rounding to `out`, which is
    what the second norm is formed again from here: a 16-bit residual stream whose mean is far above its deviation has the
    gradients of that rounding."""
    s, rows, pd, keep = _joint_spec(out, y, norm, post_norm, weight, bias, post_weight, post_bias, gate, scale, eps,
                                    dropout_p, seed, offset)
    d, device, shape = s.d, out.get_device(), out.shape
    if stats.shape != (rows, 4) or stats.dtype != torch.float32 or stats.get_device() != device or not stats.is_contiguous():
        _fail("stats must be what residual_norm_forward returned")
    s.stats = stats.data_ptr()
    if d_out is not None:
        _like(d_out, out, "d_out", shape)
        d_out, s.ld_d_out = _rows(d_out, d)
        s.d_out = d_out.data_ptr()
    if d_normed is not None:
        _like(d_normed, out, "d_normed", shape)
        d_normed, s.ld_d_normed = _rows(d_normed, d)
        s.d_normed = d_normed.data_ptr()
    layer = s.kind == _capi.PSGD_NORM_LAYER

    def vector(there, like):
        if not there:
            return None
        if rows and like is not None:
            return _new(like)
        return (out.new_empty if rows else out.new_zeros)((d,), dtype=pd)

    dx, dy = _new(out), _new(out)
    dweight, dbias = vector(True, weight), vector(layer, bias)
    dpw, dpb = vector(post_norm, post_weight), vector(post_norm and layer, post_bias)
    dgate = None if gate is None else _new(gate) if rows else torch.zeros_like(gate)
    s.dx, s.dy, s.dgate = dx.data_ptr(), dy.data_ptr(), _ptr(dgate)
    s.dweight, s.dbias, s.dpost_weight, s.dpost_bias = dweight.data_ptr(), _ptr(dbias), _ptr(dpw), _ptr(dpb)
    L = _capi.lib()
    size = L.psgd_joint_workspace(ctypes.byref(s))
    if size < 0:
        check(size, "psgd_joint_workspace")
    ws = out.new_empty((size + 16,), dtype=torch.uint8)
    _launch(device, L.psgd_joint_backward, ctypes.byref(s), ws.data_ptr(), size)
    return ResidualNormGrads(dx, dy, dweight if weight is not None else None, dbias if bias is not None else None,
                             dpw if post_weight is not None else None, dpb if post_bias is not None else None, dgate)


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, y, weight, bias, post_weight, post_bias, gate, options):
        out, normed, stats = residual_norm_forward(x, y, weight=weight, bias=bias, post_weight=post_weight,
                                                   post_bias=post_bias, gate=gate, **options)
        rng = options["seed"] if options["dropout_p"] and isinstance(options["seed"], Tensor) else None
        ctx.save_for_backward(out, y, stats, weight, bias, post_weight, post_bias, gate, rng)
        ctx.options = dict(options, seed=0) if rng is not None else options
        ctx.set_materialize_grads(False)
        return out, normed

    @staticmethod
    @once_differentiable
    def backward(ctx, d_out, d_normed):
        out, y, stats, weight, bias, post_weight, post_bias, gate, rng = ctx.saved_tensors
        if d_out is None and d_normed is None:
            return (None,) * 8
        options = ctx.options if rng is None else dict(ctx.options, seed=rng)
        g = residual_norm_grad(d_out, d_normed, out, y, stats, weight=weight, bias=bias, post_weight=post_weight,
                               post_bias=post_bias, gate=gate, **options)
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
    if _differentiated(*tensors):
        return _ResidualNorm.apply(*tensors, options)
    return residual_norm_forward(x, y, weight=weight, bias=bias, post_weight=post_weight, post_bias=post_bias, gate=gate,
                                 **options)[:2]


# ---- the loss of a large vocabulary ----------------------------------------------------------------------------------
class _ErrorWords:
    """A word of pinned host memory for each device, which the kernels write when something is wrong and the host reads
    at any time, without a copy or an event: the calls that follow (or check_errors) raise."""

    def __init__(self):
        self.words, self.lock = {}, threading.Lock()

    def get(self, device):
        w = self.words.get(device)
        if w is None:
            with self.lock:  # (one word a device, whichever thread asks first: kernels keep its address)
                w = self.words.get(device)
                if w is None:
                    t = torch.zeros(1, dtype=torch.int32).pin_memory()
                    w = self.words[device] = (t, ctypes.c_int.from_address(t.data_ptr()), t.data_ptr())
        if w[1].value:
            _fail(f"an earlier linear_cross_entropy reported: {_capi.describe_err(w[1].value)}")
        return w[2]

    def check(self):
        for device in list(self.words):
            torch.cuda.synchronize(device)
            self.get(device)

    def reset(self):
        for device, w in list(self.words.items()):
            torch.cuda.synchronize(device)
            w[1].value = 0


_ERRORS = _ErrorWords()


def check_errors():
    """Waits for the devices' work and raises RuntimeError if a kernel of this module reported an error."""
    _ERRORS.check()


def reset_errors():
    """Waits and clears what was reported, so that later calls run again."""
    _ERRORS.reset()


def _lce(h, w, target, need, grad, ignore_index, label_smoothing, z_loss, reduction, piece_bytes):
    dtype, index, shape = h.dtype, h.get_device(), h.shape
    code, kind = _TYPES.get(dtype), _REDUCTIONS.get(reduction)
    if code is None or index < 0:
        _fail("h must be an fp32, bf16 or fp16 CUDA tensor")
    if kind is None:
        _fail("reduction must be 'none', 'mean' or 'sum'")
    if w.dim() != 2 or not shape or shape[-1] != w.shape[1] or w.numel() == 0:
        _fail("h (..., d) and w (v, d) must share d")
    if w.dtype != dtype or w.get_device() != index:
        _fail("w must have the type and device of h")
    if target.shape != shape[:-1] or target.dtype != torch.int64 or target.get_device() != index:
        _fail("target must hold one int64 value for each row of h, on its device")
    if not 0.0 <= label_smoothing <= 1.0:
        _fail("label_smoothing must lie in [0, 1]")
    v, d = w.shape
    if max(target.numel(), v, d) > _capi.LCE_MAX:
        _fail(f"h and w may have up to {_capi.LCE_MAX} rows, each of as many elements")
    if grad is not None:
        if grad.dtype != torch.float32 or grad.get_device() != index or grad.shape != (() if kind else target.shape):
            _fail("grad must be fp32 on the inputs' device: a scalar, or one value for each row with reduction 'none'")
        grad = grad.contiguous()
    (h, ld_h), (w, ld_w), target = _rows(h, d), _rows(w, d), target.contiguous()
    n = target.numel()
    loss = target.new_empty(() if kind else target.shape, dtype=torch.float32)
    dh = h.new_empty(shape) if need[0] else None
    dw = torch.empty_like(w) if need[1] and ld_w == d else w.new_empty((v, d)) if need[1] else None
    if n == 0:
        for x in (loss, dw):
            if x is not None:
                x.zero_()
        return loss, dh, dw
    err = _ERRORS.get(index)
    s = _capi.Lce(h.data_ptr(), w.data_ptr(), target.data_ptr(), _ptr(grad), loss.data_ptr(), _ptr(dh), _ptr(dw), None, ld_h,
                  ld_w, ignore_index, 0, piece_bytes, n, d, v, code, kind, need[0] or need[1], label_smoothing, z_loss)
    L = _capi.lib()
    size = L.psgd_lce_workspace(ctypes.byref(s))
    if size < 0:
        check(size, "psgd_lce_workspace")
    ws = h.new_empty((size,), dtype=torch.uint8)
    s.workspace, s.workspace_bytes = ws.data_ptr(), size
    _launch(index, L.psgd_lce, ctypes.byref(s), err)
    return loss, dh, dw


class _LinearCrossEntropy(torch.autograd.Function):
    """A scalar loss forms its gradients in the forward pass (6 N V D operations for everything; the backward pass then
    only scales them, if the upstream gradient is not one). Losses by row, whose upstream gradients are not known yet, and
    fp16, where a gradient before the upstream scale may be below the type's range, form them in the backward pass
    (8 N V D)."""

    @staticmethod
    def forward(ctx, h, w, target, options):
        ctx.options, ctx.grads = options, None
        ctx.early = options["reduction"] != "none" and h.dtype != torch.float16
        ctx.save_for_backward(h, w, target)
        loss, *grads = _lce(h, w, target, ctx.needs_input_grad[:2] if ctx.early else (False, False), None, **options)
        if ctx.early:
            ctx.grads = grads
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        grads = ctx.grads
        ctx.grads = None  # they are the caller's now: a second pass (retain_graph) forms its own, in the same way
        if grads is None:
            h, w, target = ctx.saved_tensors
            _, *grads = _lce(h, w, target, ctx.needs_input_grad[:2], None if ctx.early else grad, **ctx.options)
        if ctx.early:
            for t in grads:
                if t is not None and t.numel():
                    _launch(t.get_device(), _capi.lib().psgd_lce_scale, t.data_ptr(), _TYPES[t.dtype], t.numel(), grad.data_ptr())
        return *grads, None, None


def linear_cross_entropy(h: Tensor, w: Tensor, target: Tensor, *, ignore_index: int = -100, label_smoothing: float = 0.0,
                         z_loss: float = 0.0, reduction: str = "mean", piece_bytes: int = DEFAULT_PIECE_BYTES) -> Tensor:
    """Cross entropy of the logits h w^T against target, in fp32, plus z_loss times the squared log-normaliser:

        lse = log sum_v exp(l_v);  loss = (1 - s) (lse - l_target) + s (lse - mean_v l_v) + z_loss lse^2

    h (..., d), w (v, d) of one type; target (...) int64. Rows whose target is ignore_index have loss 0 and touch nothing
    (not even with NaN in h); 'mean' divides by the number of the others (0 when there is none). reduction 'none' keeps
    target's shape.

    Precision: losses are fp32 whatever the type (logits from tensor-core sums of at most 1024 products, added in fp32). The
    gradients of 16-bit inputs are products of operands of that type: d loss / d l is rounded to it once (and before that
    the exponentials to fp16), which adds about 1e-3 (bf16; fp16: 2e-4) to the 1.7e-3 (2e-4) of the gradients' own rounding, in the
    2-norm. Calls of up to 2^20 products n v d, where it costs nothing, have three bf16 limbs there instead, as fp32 inputs
    do (about 1e-6).

    Under autograd a scalar loss (mean, sum) of bf16 or fp32 inputs that require gradients forms them at once and holds
    them for the backward pass, which multiplies them by an upstream gradient other than one (and rounds them once more, if it
    is no power of two); otherwise the backward pass forms loss and gradients again. Evaluation belongs under
    torch.no_grad(). piece_bytes bounds what is kept of the vocabulary's probabilities at a time (16 bits each; fp32: 80
    bits); tokens are taken in pieces of that size (of 256 at least)."""
    options = dict(ignore_index=ignore_index, label_smoothing=label_smoothing, z_loss=z_loss, reduction=reduction,
                   piece_bytes=piece_bytes)
    if _differentiated(h, w):
        return _LinearCrossEntropy.apply(h, w, target, options)
    return _lce(h, w, target, (False, False), None, **options)[0]


def linear_cross_entropy_grad(h: Tensor, w: Tensor, target: Tensor, *, grad: Optional[Tensor] = None,
                              ignore_index: int = -100, label_smoothing: float = 0.0, z_loss: float = 0.0,
                              reduction: str = "mean", piece_bytes: int = DEFAULT_PIECE_BYTES):
    """(loss, dh, dw): the loss and the gradients of h and w for the upstream gradient `grad` (fp32; default ones)."""
    return _lce(h, w, target, (True, True), grad, ignore_index, label_smoothing, z_loss, reduction, piece_bytes)
