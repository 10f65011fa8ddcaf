"""Operators of a classification head of the caller's own making, on the HIP path.

The model's own head is fixed (1024 -> 512 -> 256 -> k with BatchNorm, model/pointnet.py:174-190) and its loss takes
stored log-probabilities (main_1v.py:270, `training.nll_loss`).  For another head on the pooled feature - wider, deeper,
regularised, with many classes - there are

* `linear`                 y = act(x W^T + b) + residual,
* `dropout`                counter-based, its mask a function of (seed, offset, position) that is never stored,
* `linear_cross_entropy`   the loss of softmax(x W^T + b) without the logits having to be stored whole,

each differentiable once through torch.autograd, in float32, bfloat16 and float16.  Every tensor of a call has one type
and lies on one GPU; sums and row statistics are 32-bit.  Calls run on the current stream of the tensors' device and can be
captured into a graph; take the gradients of a captured step with `torch.autograd.grad`, whose results are the graph's own,
and let go of eager results of the same leaves (a kept loss) first: torch's engine would wait for their stream in the middle
of the capture, so the backward pass raises there.  Forward-mode differentiation is refused.
"""
from __future__ import annotations

import torch

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


def _plain(t):
    """Without a pending negation (a lazy view of a complex tensor's part)."""
    return t.resolve_neg() if t is not None and t.is_neg() else t


# ---- linear ---------------------------------------------------------------------------------------------------------------

def linear(x, weight, bias=None, activation=None, residual=None):
    """act(x W^T + b) + residual: x [..., K], weight [N, K], bias [N], residual and result [..., N].

    activation: None, "relu", "gelu" (the error function's), "gelu_tanh" or "silu".  For 16-bit types the sums are 32-bit
    and the result is rounded once; in training the pre-activation is kept, and its gradient handed to the products, in the
    tensors' type (dx and dW are off as those of torch's own 16-bit autograd are: 0.0024 of their norm in bfloat16)."""
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
    return _lib.load_head().linear(_plain(x), _plain(weight), _plain(bias), _plain(residual), _ACTIVATIONS[activation])


# ---- dropout --------------------------------------------------------------------------------------------------------------

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
    return _lib.load_head().dropout(_plain(x), _plain(residual), p, seed, offset, rng)


# ---- linear + cross entropy -----------------------------------------------------------------------------------------------

def linear_cross_entropy(x, weight, target, bias=None, ignore_index=-100, label_smoothing=0.0, reduction="mean", keep_logits=True):
    """F.cross_entropy(F.linear(x, weight, bias), target) without the logits: x [..., D], weight [V, D], target [...] of
    whole numbers, bias [V] -> float32 loss, a scalar for reduction "mean" (over the rows that are not ignored) and "sum",
    [...] for "none".

    Rows with target == ignore_index have loss 0 and no gradient, whatever values they hold.  Another target outside [0, V)
    makes the loss NaN and gives its row no gradient, as `training.nll_loss` does.  A class is masked by a bias of -inf, or a
    large negative one.

    The logits are formed in pieces, in the backward pass again.  Where that is quicker, and one piece holds them all (256 MiB in
    x's type, or as much as x and weight take), they are kept in 32 bits instead; keep_logits=False never keeps them (at most
    eight classes always do: 16 or 32 bytes a row)."""
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
    return _lib.load_head().linear_cross_entropy(_plain(x), _plain(weight), target.contiguous(), _plain(bias), int(ignore_index),
                                                 label_smoothing, _REDUCTIONS[reduction], bool(keep_logits) or V <= 8)
