"""Operators of a classification head of the caller's own making, on the HIP path.

The model's own head is fixed (1024 -> 512 -> 256 -> k with BatchNorm, model/pointnet.py:174-190) and its loss takes
stored log-probabilities (main_1v.py:270, `training.nll_loss`).  For another head on the pooled feature - wider, deeper,
regularised, with many classes - there are

* `linear`                 y = act(x W^T + b) + residual,
* `dropout`                counter-based, its mask a function of (seed, offset, position) that is never stored,
* `linear_cross_entropy`   the loss of softmax(x W^T + b) without the logits ever being stored whole,

each differentiable once through torch.autograd, in float32, bfloat16 and float16.  Every tensor of a call has one type
and lies on one GPU; sums and row statistics are 32-bit.  Calls run on the current stream of the tensors' device and can be
captured into a graph; take the gradients of a captured step with `torch.autograd.grad`, whose results are the graph's own,
and let go of eager results of the same leaves (a kept loss) first: torch's engine would wait for their stream in the middle
of the capture.
"""
from __future__ import annotations

import functools

import torch
from torch.autograd.function import once_differentiable

from . import _lib

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_ACTIVATIONS = {None: 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}
_REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}


def _refuse(x, name, like, shape):
    """Raises what is wrong with an argument that `_fits` does not take."""
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{name}: expected a tensor, got {type(x).__name__}")
    if not x.is_cuda:
        raise RuntimeError(f"{name} is on {x.device}: pointnetgpd_amd runs on MI355X only (there is no CPU path)")
    if x.layout != torch.strided:
        raise TypeError(f"{name}: expected a dense tensor, got layout {x.layout}")
    if x.dtype not in _TYPES:
        raise TypeError(f"{name}: expected float32, bfloat16 or float16, got {x.dtype}")
    if like is not None and x.device != like.device:
        raise RuntimeError(f"{name} is on {x.device}, the input on {like.device}")
    if like is not None and x.dtype != like.dtype:
        raise TypeError(f"{name} is {x.dtype}, the input {like.dtype}")
    raise ValueError(f"{name}: expected shape {tuple(shape)}, got {tuple(x.shape)}")


def _fits(x, like=None, shape=None):
    return isinstance(x, torch.Tensor) and x.is_cuda and x.layout == torch.strided and x.dtype in _TYPES and \
        (like is None or (x.dtype == like.dtype and x.device == like.device)) and (shape is None or x.shape == shape)


def _require(x, name, like=None, shape=None):
    if not _fits(x, like, shape):
        _refuse(x, name, like, shape)


def _rows(t, cols):
    """(tensor whose memory is rows of `cols` dense elements, distance of two rows): a view where the strides allow it, else
    a copy."""
    if t.is_contiguous():
        return t, cols
    t2 = t.reshape(-1, cols)
    if cols == 1 or t2.stride(1) == 1:
        if t2.shape[0] <= 1:
            return t2, cols
        if t2.stride(0) >= cols:
            return t2, t2.stride(0)
    return t2.contiguous(), cols


def _aligned(t, ld, size):
    """Whether rows start at 16-byte addresses, whole 16-byte chunks and at most 2^23 bytes apart."""
    return t.data_ptr() % 16 == 0 and ld * size % 16 == 0 and ld * size <= 1 << 23


def _vector(t):
    return t if t is None or t.is_contiguous() else t.contiguous()


def _ptr(t):
    return None if t is None else t.data_ptr()


# Handles without Python objects around them: torch.cuda.device / current_stream cost more than a small kernel's launch, above
# all when the forward pass (the caller's thread) and the backward pass (autograd's) take turns in them.
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
    (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _call(fn, t, *args):
    """fn(*args, stream) on t's device and its current stream."""
    index = t.get_device()
    if _current_device() == index:
        rc = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _raw_stream(index))
    if rc:
        _lib.check(rc)


@functools.lru_cache(maxsize=4096)
def _linear_bytes(kind, M, N, K, backward, aligned):
    return _lib.load().pngpd_linear_workspace_bytes(kind, M, N, K, backward, aligned)


@functools.lru_cache(maxsize=4096)
def _loss_bytes(kind, T, V, D, backward, aligned):
    return _lib.load().pngpd_linear_cross_entropy_workspace_bytes(kind, T, V, D, backward, aligned)


def _workspace(nbytes, like):
    return torch.empty(nbytes, dtype=torch.uint8, device=like.device) if nbytes else None


def _wants_grad(*tensors):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _plain(t):
    """Without a pending negation (a lazy view of a complex tensor's part)."""
    return t.resolve_neg() if t is not None and t.is_neg() else t


def _once(backward):
    """once_differentiable, whose wrapper is skipped where no graph of the gradient is asked for."""
    wrapped = once_differentiable(backward)

    def call(ctx, *grads):
        return wrapped(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)

    return call


# ---- linear ---------------------------------------------------------------------------------------------------------------

def _linear_forward(x, weight, bias, residual, act, keep):
    lib = _lib.load()
    N, K = weight.shape
    x2, ldx = _rows(x, K)
    w2, ldw = _rows(weight, K)
    M = x.numel() // K
    kind, size = _TYPES[x.dtype], x.element_size()
    y = x.new_empty(x.shape[:-1] + (N,))
    z = x.new_empty((M, N)) if keep and act else None
    r2, ldr = (None, N) if residual is None else _rows(residual, N)
    b = _vector(bias)
    nbytes = _linear_bytes(kind, M, N, K, 0, _aligned(x2, ldx, size) and _aligned(w2, ldw, size))
    ws = _workspace(nbytes, x)
    _call(lib.pngpd_linear_forward, x, kind, M, N, K, x2.data_ptr(), ldx, w2.data_ptr(), ldw, _ptr(b), act, _ptr(r2), ldr,
          y.data_ptr(), _ptr(z), _ptr(ws), nbytes)
    return y, z


class LinearFunction(torch.autograd.Function):
    """autograd bridge of `linear`: pngpd_linear_forward / pngpd_linear_backward."""

    @staticmethod
    def forward(ctx, x, weight, bias, residual, act):
        need = ctx.needs_input_grad
        y, z = _linear_forward(x, weight, bias, residual, act, need[0] or need[1] or need[2])
        ctx.act = act
        ctx.save_for_backward(x, weight, z)
        return y

    @staticmethod
    @_once
    def backward(ctx, dy):
        lib = _lib.load()
        x, weight, z = ctx.saved_tensors
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        dy = _plain(dy)
        if not (need_x or need_w or need_b):
            return None, None, None, dy if need_r else None, None
        N, K = weight.shape
        x2, ldx = _rows(x, K)
        w2, ldw = _rows(weight, K)
        d2, ld_dy = _rows(dy, N)
        M = x.numel() // K
        kind, size = _TYPES[x.dtype], x.element_size()
        dx = x.new_empty(x.shape) if need_x else None
        dw = x.new_empty((N, K)) if need_w else None
        db = x.new_empty(N) if need_b else None
        nbytes = _linear_bytes(kind, M, N, K, 1, _aligned(x2, ldx, size) and _aligned(w2, ldw, size) and _aligned(d2, ld_dy, size))
        ws = _workspace(nbytes, x)
        _call(lib.pngpd_linear_backward, x, kind, M, N, K, d2.data_ptr(), ld_dy, _ptr(z), x2.data_ptr(), ldx, w2.data_ptr(), ldw,
              ctx.act, _ptr(dx), _ptr(dw), _ptr(db), _ptr(ws), nbytes)
        return dx, dw, db, dy if need_r else None, None


def linear(x, weight, bias=None, activation=None, residual=None):
    """act(x W^T + b) + residual: x [..., K], weight [N, K], bias [N], residual and result [..., N].

    activation: None, "relu", "gelu" (the error function's), "gelu_tanh" or "silu".  For 16-bit types the sums are 32-bit
    and the result is rounded once; in training the pre-activation is kept in the tensors' type."""
    if activation not in _ACTIVATIONS:
        raise ValueError(f"activation: expected one of {list(_ACTIVATIONS)}, got {activation!r}")
    _require(x, "x")
    _require(weight, "weight", x)
    if weight.dim() != 2 or weight.shape[0] < 1 or weight.shape[1] < 1:
        raise ValueError(f"weight: expected [N, K], got {tuple(weight.shape)}")
    N, K = weight.shape
    if x.dim() < 1 or x.shape[-1] != K:
        raise ValueError(f"x: expected [..., {K}], got {tuple(x.shape)}")
    if bias is not None:
        _require(bias, "bias", x, (N,))
    if residual is not None:
        _require(residual, "residual", x, x.shape[:-1] + (N,))
    x, weight, bias, residual = _plain(x), _plain(weight), _plain(bias), _plain(residual)
    act = _ACTIVATIONS[activation]
    if _wants_grad(x, weight, bias, residual):
        return LinearFunction.apply(x, weight, bias, residual, act)
    return _linear_forward(x, weight, bias, residual, act, False)[0]


# ---- dropout --------------------------------------------------------------------------------------------------------------

def _dropout_call(x, residual, p, seed, offset, rng):
    lib = _lib.load()
    n = x.numel()
    cols = x.shape[-1] if x.dim() else 1
    if x.is_contiguous() and (residual is None or residual.is_contiguous()):
        x2, ldx, r2, ldr = x, cols, residual, cols
    else:
        x2, ldx = _rows(x, cols)
        r2, ldr = (None, cols) if residual is None else _rows(residual, cols)
    y = x.new_empty(x.shape)
    if n:
        _call(lib.pngpd_dropout, x, _TYPES[x.dtype], n // cols, cols, x2.data_ptr(), ldx, _ptr(r2), ldr, y.data_ptr(), p, seed,
              offset, _ptr(rng))
    return y


class DropoutFunction(torch.autograd.Function):
    """autograd bridge of `dropout`: the backward pass is the same call on the gradient."""

    @staticmethod
    def forward(ctx, x, residual, p, seed, offset, rng):
        ctx.args = (p, seed, offset)
        if rng is not None:
            ctx.save_for_backward(rng)
        return _dropout_call(x, residual, p, seed, offset, rng)

    @staticmethod
    @_once
    def backward(ctx, dy):
        saved = ctx.saved_tensors
        dy = _plain(dy)
        need_x, need_r = ctx.needs_input_grad[:2]
        dx = _dropout_call(dy, None, *ctx.args, saved[0] if saved else None) if need_x else None
        return dx, dy if need_r else None, None, None, None, None


def dropout(x, p, seed, offset=0, residual=None):
    """residual + keep x / (1 - p), element i of x (in row-major order) kept when its 32 random bits are at least p 2^32.

    The bits are a function of (seed, offset, i) alone: the same arguments drop the same elements, on any strides and in the
    backward pass, and no mask is stored.  Give every layer and step a (seed, offset) of its own.  seed: an int, or an int64
    GPU tensor of two elements {seed, offset}, which the kernel reads when it runs: a captured graph draws a new mask
    whenever the tensor is changed between replays.  It must keep its values until the backward pass has run."""
    _require(x, "x")
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"p: expected a probability, got {p}")
    if residual is not None:
        _require(residual, "residual", x, x.shape)
    rng = None
    if isinstance(seed, torch.Tensor):
        if seed.dtype != torch.int64 or seed.numel() != 2 or seed.device != x.device or not seed.is_contiguous():
            raise ValueError("seed: expected an int, or a dense int64 tensor of two elements on x's device")
        if offset != 0:
            raise ValueError("offset: the seed tensor holds it")
        rng, seed = seed, 0
    seed, offset = int(seed) & (2 ** 64 - 1), int(offset) & (2 ** 64 - 1)
    x, residual = _plain(x), _plain(residual)
    if _wants_grad(x, residual):
        return DropoutFunction.apply(x, residual, p, seed, offset, rng)
    return _dropout_call(x, residual, p, seed, offset, rng)


# ---- linear + cross entropy -----------------------------------------------------------------------------------------------

def _loss_forward(x, weight, bias, target, ignore_index, label_smoothing, reduction):
    lib = _lib.load()
    V, D = weight.shape
    x2, ldx = _rows(x, D)
    w2, ldw = _rows(weight, D)
    T = x.numel() // D
    kind, size = _TYPES[x.dtype], x.element_size()
    loss = torch.empty(x.shape[:-1] if reduction == 0 else (), dtype=torch.float32, device=x.device)
    lse = torch.empty(T, dtype=torch.float32, device=x.device)
    b = _vector(bias)
    nbytes = _loss_bytes(kind, T, V, D, 0, _aligned(x2, ldx, size) and _aligned(w2, ldw, size))
    ws = _workspace(nbytes, x)
    _call(lib.pngpd_linear_cross_entropy_forward, x, kind, T, V, D, x2.data_ptr(), ldx, w2.data_ptr(), ldw, _ptr(b),
          target.data_ptr(), ignore_index, label_smoothing, reduction, loss.data_ptr(), lse.data_ptr(), _ptr(ws), nbytes)
    return loss, lse


class LinearCrossEntropyFunction(torch.autograd.Function):
    """autograd bridge of `linear_cross_entropy`: pngpd_linear_cross_entropy_forward / _backward."""

    @staticmethod
    def forward(ctx, x, weight, bias, target, ignore_index, label_smoothing, reduction):
        loss, lse = _loss_forward(x, weight, bias, target, ignore_index, label_smoothing, reduction)
        ctx.args = (ignore_index, label_smoothing, reduction)
        ctx.save_for_backward(x, weight, bias, target, lse)
        return loss

    @staticmethod
    @_once
    def backward(ctx, dloss):
        lib = _lib.load()
        x, weight, bias, target, lse = ctx.saved_tensors
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        V, D = weight.shape
        x2, ldx = _rows(x, D)
        w2, ldw = _rows(weight, D)
        T = x.numel() // D
        kind, size = _TYPES[x.dtype], x.element_size()
        dloss = _plain(dloss).contiguous()
        dx = x.new_empty(x.shape) if need_x else None
        dw = x.new_empty((V, D)) if need_w else None
        db = x.new_empty(V) if need_b else None
        b = _vector(bias)
        nbytes = _loss_bytes(kind, T, V, D, 1, _aligned(x2, ldx, size) and _aligned(w2, ldw, size))
        ws = _workspace(nbytes, x)
        _call(lib.pngpd_linear_cross_entropy_backward, x, kind, T, V, D, x2.data_ptr(), ldx, w2.data_ptr(), ldw, _ptr(b),
              target.data_ptr(), *ctx.args, lse.data_ptr(), dloss.data_ptr(), _ptr(dx), _ptr(dw), _ptr(db), _ptr(ws), nbytes)
        return dx, dw, db, None, None, None, None


def linear_cross_entropy(x, weight, target, bias=None, ignore_index=-100, label_smoothing=0.0, reduction="mean"):
    """F.cross_entropy(F.linear(x, weight, bias), target) without the logits: x [..., D], weight [V, D], target [...] of
    whole numbers, bias [V] -> float32 loss, a scalar for reduction "mean" (over the rows that are not ignored) and "sum",
    [...] for "none".

    Rows with target == ignore_index have loss 0 and no gradient, whatever values they hold.  Another target outside [0, V)
    makes the loss NaN and gives its row no gradient, as `training.nll_loss` does.  A class is masked by a bias of -inf."""
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction: expected one of {list(_REDUCTIONS)}, got {reduction!r}")
    _require(x, "x")
    _require(weight, "weight", x)
    if weight.dim() != 2 or weight.shape[0] < 1 or weight.shape[1] < 1:
        raise ValueError(f"weight: expected [V, D], got {tuple(weight.shape)}")
    V, D = weight.shape
    if x.dim() < 1 or x.shape[-1] != D:
        raise ValueError(f"x: expected [..., {D}], got {tuple(x.shape)}")
    if bias is not None:
        _require(bias, "bias", x, (V,))
    if not isinstance(target, torch.Tensor) or target.dtype.is_floating_point or target.dtype.is_complex or \
            target.dtype == torch.bool:
        raise TypeError("target: expected a tensor of whole numbers")
    if target.device != x.device:
        raise RuntimeError(f"target is on {target.device}, the input on {x.device}")
    if target.shape != x.shape[:-1]:
        raise ValueError(f"target: expected shape {tuple(x.shape[:-1])}, got {tuple(target.shape)}")
    label_smoothing = float(label_smoothing)
    if not 0.0 <= label_smoothing <= 1.0:
        raise ValueError(f"label_smoothing: expected a number in [0, 1], got {label_smoothing}")
    if target.dtype != torch.int64:
        target = target.to(torch.int64)
    target = _vector(target)
    x, weight, bias = _plain(x), _plain(weight), _plain(bias)
    args = (int(ignore_index), label_smoothing, _REDUCTIONS[reduction])
    if _wants_grad(x, weight, bias):
        return LinearCrossEntropyFunction.apply(x, weight, bias, target, *args)
    return _loss_forward(x, weight, bias, target, *args)[0]
