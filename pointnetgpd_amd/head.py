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


def _require(x, name, like=None, shape=None):
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{name}: expected a tensor, got {type(x).__name__}")
    if not x.is_cuda:
        raise RuntimeError(f"{name} is on {x.device}: pointnetgpd_amd runs on MI355X only (there is no CPU path)")
    if x.layout != torch.strided:
        raise TypeError(f"{name}: expected a dense tensor, got layout {x.layout}")
    if like is None:
        if x.dtype not in _TYPES:
            raise TypeError(f"{name}: expected float32, bfloat16 or float16, got {x.dtype}")
    else:
        if x.device != like.device:
            raise RuntimeError(f"{name} is on {x.device}, the input on {like.device}")
        if x.dtype != like.dtype:
            raise TypeError(f"{name} is {x.dtype}, the input {like.dtype}")
    if shape is not None and tuple(x.shape) != tuple(shape):
        raise ValueError(f"{name}: expected shape {tuple(shape)}, got {tuple(x.shape)}")


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


def _count(t, cols):
    return t.numel() // cols


def _aligned(size, *matrices):
    """Whether all (tensor, distance of rows) start at 16-byte addresses with rows of whole 16-byte chunks apart."""
    return int(all(t.data_ptr() % 16 == 0 and ld * size % 16 == 0 and ld * size <= 1 << 23 for t, ld in matrices))


def _vector(t):
    return t if t is None or t.is_contiguous() else t.contiguous()


def _ptr(t):
    return None if t is None else t.data_ptr()


def _workspace(nbytes, dev):
    return torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None


# the stream's handle without a Stream object around it; torch.cuda.device / current_stream cost more than a small kernel's
# launch, above all when the forward pass (the caller's thread) and the backward pass (autograd's) take turns in them
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
    (lambda index: torch.cuda.current_stream(index).cuda_stream)


class _OnDevice:
    """Makes a device the current one for the calls inside, if it is not."""
    __slots__ = ("index", "before")

    def __init__(self, index):
        self.index = index

    def __enter__(self):
        self.before = torch.cuda.current_device()
        if self.before != self.index:
            torch.cuda.set_device(self.index)
        return _raw_stream(self.index)

    def __exit__(self, *exc):
        if self.before != self.index:
            torch.cuda.set_device(self.before)


@functools.lru_cache(maxsize=4096)
def _linear_bytes(*sizes):
    return _lib.load().pngpd_linear_workspace_bytes(*sizes)


@functools.lru_cache(maxsize=4096)
def _loss_bytes(*sizes):
    return _lib.load().pngpd_linear_cross_entropy_workspace_bytes(*sizes)


def _wants_grad(*tensors):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _conj_free(*tensors):
    return [t.resolve_neg() if t is not None and t.is_neg() else t for t in tensors]


# ---- linear ---------------------------------------------------------------------------------------------------------------

def _linear_forward(x, weight, bias, residual, act, keep):
    lib = _lib.load()
    N, K = weight.shape
    x2, ldx = _rows(x, K)
    w2, ldw = _rows(weight, K)
    M = _count(x, K)
    dev, kind = x.device, _TYPES[x.dtype]
    y = torch.empty(x.shape[:-1] + (N,), dtype=x.dtype, device=dev)
    z = torch.empty((M, N), dtype=x.dtype, device=dev) if keep and act else None
    r2, ldr = _rows(residual, N) if residual is not None else (None, N)
    b = _vector(bias)
    nbytes = _linear_bytes(kind, M, N, K, 0, _aligned(x.element_size(), (x2, ldx), (w2, ldw)))
    with _OnDevice(dev.index) as stream:
        ws = _workspace(nbytes, dev)
        _lib.check(lib.pngpd_linear_forward(kind, M, N, K, _ptr(x2), ldx, _ptr(w2), ldw, _ptr(b), act, _ptr(r2), ldr, _ptr(y),
                                            _ptr(z), _ptr(ws), nbytes, stream))
    return y, z


class LinearFunction(torch.autograd.Function):
    """autograd bridge of `linear`: pngpd_linear_forward / pngpd_linear_backward."""

    @staticmethod
    def forward(ctx, x, weight, bias, residual, act):
        y, z = _linear_forward(x, weight, bias, residual, act, any(ctx.needs_input_grad[:3]))
        ctx.act = act
        ctx.save_for_backward(x, weight, z)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        lib = _lib.load()
        x, weight, z = ctx.saved_tensors
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        dy, = _conj_free(dy)
        if not (need_x or need_w or need_b):
            return None, None, None, dy if need_r else None, None
        N, K = weight.shape
        dev, kind = x.device, _TYPES[x.dtype]
        x2, ldx = _rows(x, K)
        w2, ldw = _rows(weight, K)
        d2, ld_dy = _rows(dy, N)
        M = _count(x, K)
        dx = torch.empty(x.shape, dtype=x.dtype, device=dev) if need_x else None
        dw = torch.empty((N, K), dtype=x.dtype, device=dev) if need_w else None
        db = torch.empty(N, dtype=x.dtype, device=dev) if need_b else None
        nbytes = _linear_bytes(kind, M, N, K, 1,
                                                  _aligned(x.element_size(), (x2, ldx), (w2, ldw), (d2, ld_dy)))
        with _OnDevice(dev.index) as stream:
            ws = _workspace(nbytes, dev)
            _lib.check(lib.pngpd_linear_backward(kind, M, N, K, _ptr(d2), ld_dy, _ptr(z), _ptr(x2), ldx, _ptr(w2), ldw, ctx.act,
                                                 _ptr(dx), _ptr(dw), _ptr(db), _ptr(ws), nbytes, stream))
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
    x, weight, bias, residual = _conj_free(x, weight, bias, residual)
    act = _ACTIVATIONS[activation]
    if _wants_grad(x, weight, bias, residual):
        return LinearFunction.apply(x, weight, bias, residual, act)
    return _linear_forward(x, weight, bias, residual, act, False)[0]


# ---- dropout --------------------------------------------------------------------------------------------------------------

def _dropout_call(x, residual, p, seed, offset, rng):
    lib = _lib.load()
    dev = x.device
    y = torch.empty(x.shape, dtype=x.dtype, device=dev)
    if x.numel() == 0:
        return y
    cols = x.shape[-1] if x.dim() else 1
    if x.is_contiguous() and (residual is None or residual.is_contiguous()):
        # one long row would pass the size limit: the rows stay those of the tensor
        x2, ldx, r2, ldr = x, cols, residual, cols
    else:
        x2, ldx = _rows(x, cols)
        r2, ldr = _rows(residual, cols) if residual is not None else (None, cols)
    with _OnDevice(dev.index) as stream:
        _lib.check(lib.pngpd_dropout(_TYPES[x.dtype], x.numel() // cols, cols, _ptr(x2), ldx, _ptr(r2), ldr, _ptr(y), p, seed,
                                     offset, _ptr(rng), stream))
    return y


class DropoutFunction(torch.autograd.Function):
    """autograd bridge of `dropout`: the backward pass is the same call on the gradient."""

    @staticmethod
    def forward(ctx, x, residual, p, seed, offset, rng):
        ctx.args = (p, seed, offset)
        ctx.save_for_backward(rng)
        return _dropout_call(x, residual, p, seed, offset, rng)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        rng, = ctx.saved_tensors
        dy, = _conj_free(dy)
        dx = _dropout_call(dy, None, *ctx.args, rng) if ctx.needs_input_grad[0] else None
        return dx, dy if ctx.needs_input_grad[1] else None, None, None, None, None


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
    x, residual = _conj_free(x, residual)
    if _wants_grad(x, residual):
        return DropoutFunction.apply(x, residual, p, seed, offset, rng)
    return _dropout_call(x, residual, p, seed, offset, rng)


# ---- linear + cross entropy -----------------------------------------------------------------------------------------------

class LinearCrossEntropyFunction(torch.autograd.Function):
    """autograd bridge of `linear_cross_entropy`: pngpd_linear_cross_entropy_forward / _backward."""

    @staticmethod
    def forward(ctx, x, weight, bias, target, ignore_index, label_smoothing, reduction):
        loss, lse = _loss_forward(x, weight, bias, target, ignore_index, label_smoothing, reduction)
        ctx.args = (ignore_index, label_smoothing, reduction)
        ctx.save_for_backward(x, weight, bias, target, lse)
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss):
        lib = _lib.load()
        x, weight, bias, target, lse = ctx.saved_tensors
        ignore_index, label_smoothing, reduction = ctx.args
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        V, D = weight.shape
        dev, kind = x.device, _TYPES[x.dtype]
        x2, ldx = _rows(x, D)
        w2, ldw = _rows(weight, D)
        T = _count(x, D)
        dloss = _conj_free(dloss)[0].to(torch.float32).contiguous()
        dx = torch.empty(x.shape, dtype=x.dtype, device=dev) if need_x else None
        dw = torch.empty((V, D), dtype=x.dtype, device=dev) if need_w else None
        db = torch.empty(V, dtype=x.dtype, device=dev) if need_b else None
        nbytes = _loss_bytes(
            kind, T, V, D, 1, _aligned(x.element_size(), (x2, ldx), (w2, ldw)))
        b = _vector(bias)
        with _OnDevice(dev.index) as stream:
            ws = _workspace(nbytes, dev)
            _lib.check(lib.pngpd_linear_cross_entropy_backward(
                kind, T, V, D, _ptr(x2), ldx, _ptr(w2), ldw, _ptr(b), _ptr(target), ignore_index, label_smoothing, reduction,
                _ptr(lse), _ptr(dloss), _ptr(dx), _ptr(dw), _ptr(db), _ptr(ws), nbytes, stream))
        return dx, dw, db, None, None, None, None


def _loss_forward(x, weight, bias, target, ignore_index, label_smoothing, reduction):
    lib = _lib.load()
    V, D = weight.shape
    dev, kind = x.device, _TYPES[x.dtype]
    x2, ldx = _rows(x, D)
    w2, ldw = _rows(weight, D)
    T = _count(x, D)
    loss = torch.empty(x.shape[:-1] if reduction == 0 else (), dtype=torch.float32, device=dev)
    lse = torch.empty(T, dtype=torch.float32, device=dev)
    nbytes = _loss_bytes(
        kind, T, V, D, 0, _aligned(x.element_size(), (x2, ldx), (w2, ldw)))
    b = _vector(bias)
    with _OnDevice(dev.index) as stream:
        ws = _workspace(nbytes, dev)
        _lib.check(lib.pngpd_linear_cross_entropy_forward(kind, T, V, D, _ptr(x2), ldx, _ptr(w2), ldw, _ptr(b), _ptr(target),
                                                          ignore_index, label_smoothing, reduction, _ptr(loss), _ptr(lse),
                                                          _ptr(ws), nbytes, stream))
    return loss, lse


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
    if tuple(target.shape) != tuple(x.shape[:-1]):
        raise ValueError(f"target: expected shape {tuple(x.shape[:-1])}, got {tuple(target.shape)}")
    label_smoothing = float(label_smoothing)
    if not 0.0 <= label_smoothing <= 1.0:
        raise ValueError(f"label_smoothing: expected a number in [0, 1], got {label_smoothing}")
    target = target.detach().to(torch.int64).contiguous()
    x, weight, bias = _conj_free(x, weight, bias)
    args = (int(ignore_index), label_smoothing, _REDUCTIONS[reduction])
    if _wants_grad(x, weight, bias):
        return LinearCrossEntropyFunction.apply(x, weight, bias, target, *args)
    return _loss_forward(x, weight, bias, target, *args)[0]
