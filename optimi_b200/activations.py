"""Activations kept in 8 bits for the backward pass, and the operators that read them there.

With gradient release no gradient outlives its step, and what bounds a batch is the activations the forward
pass keeps.  Here they are kept as int8 codes with one shared power of two for every 32 neighbouring
channels of a token (8.25 bits a value instead of 16 or 32), and the backward pass works on the codes:

* `compress` / `decompress`: a tensor to that form and back.  Restored values are exact in their type; what is
  lost is lost in the rounding to codes, at most half a step: 1/127 of the group's largest magnitude.
* `rms_norm`: residual addition and RMS norm; the normalised row leaves in 8 bits beside the output, and the
  backward pass needs nothing else of the forward pass.
* `linear`: a linear layer that keeps its input in 8 bits (or shares the norm's) and takes its weight gradient straight
  from the codes (`weight_gradient`).
* `checkpoint`: recomputation of a block in the backward pass from inputs kept in 8 bits.
* `prepare_for_compressed_activations` / `remove_compressed_activations`: the `nn.Linear` and `nn.RMSNorm`
  layers of a model do this by themselves, as `prepare_for_gradient_release` does for the step.

Forward results are those of the plain layers; gradients are those of the plain formulas with the kept
activation in place of the original.  CUDA tensors only, like the optimizers.
"""

from __future__ import annotations

from collections import OrderedDict
from collections.abc import Callable, Sequence
from typing import Any, NamedTuple
from warnings import warn

import torch
import torch.utils.checkpoint
from torch import Tensor, nn

from . import _lib

__all__ = [
    "CompressedActivation", "RMSNormOutput", "compress", "decompress", "rms_norm", "linear", "weight_gradient", "checkpoint",
    "prepare_for_compressed_activations", "remove_compressed_activations",
]  # fmt: skip

GROUP = 32  # channels that share an exponent byte

_PREPARED_ATTR = "_compressed_activation_modules"
_KEPT_ATTR = "_optimi_kept_activation"


class CompressedActivation:
    """An activation in 8 bits: `codes` (int8, one row per token, the row pitch a multiple of 32 bytes), `exponents`
    (uint8, one per token and group of 32 channels), the `shape` and `dtype` of what they stand for.

    A value is ``code * 2**(exponent - 127)``; exponent 0 is a group of zeros, 255 a group that held an infinity or a
    NaN and reads back as NaNs.  `channel_scale`, where given, multiplies the last dimension (a norm's weight).
    """

    __slots__ = ("_codes", "_exponents", "_buffer", "shape", "dtype", "channel_scale")

    def __init__(self, codes: Tensor, exponents: Tensor, shape, dtype: torch.dtype, channel_scale: Tensor | None = None):
        shape = torch.Size(shape)
        if dtype not in _lib.DTYPE_CODE:
            raise ValueError(f"unsupported activation dtype {dtype} (float32, bfloat16 and float16 are)")
        if len(shape) == 0:
            raise ValueError("an activation has at least one dimension")
        cols = shape[-1]
        rows = _rows(shape)
        padded = -(-cols // GROUP) * GROUP
        if codes.dtype != torch.int8 or codes.dim() != 2 or codes.shape[0] != rows or codes.shape[1] < padded:
            raise ValueError(f"codes must be int8 with {rows} rows of at least {padded} values")
        if exponents.dtype != torch.uint8 or exponents.dim() != 2 or exponents.shape[0] != rows or exponents.shape[1] < padded // GROUP:
            raise ValueError(f"exponents must be uint8 with {rows} rows of at least {padded // GROUP} values")
        if codes.device != exponents.device:
            raise ValueError(f"codes are on {codes.device} and exponents on {exponents.device}")
        if rows and cols:
            if codes.stride(1) != 1 or (exponents.shape[1] > 1 and exponents.stride(1) != 1) or (rows > 1 and codes.stride(0) % GROUP) or codes.data_ptr() % 16:
                raise ValueError("rows of codes and exponents must be contiguous, codes 16-byte aligned with a pitch that is a multiple of 32")
            if rows > 1 and (codes.stride(0) < padded or exponents.stride(0) < padded // GROUP):
                raise ValueError("rows of codes and exponents must not overlap")
        if channel_scale is not None and (channel_scale.shape != shape[-1:] or channel_scale.dtype != dtype or channel_scale.device != codes.device):
            raise ValueError(f"channel_scale must be a {dtype} tensor of {cols} values on {codes.device}")
        self._codes, self._exponents, self._buffer = codes, exponents, None
        self.shape, self.dtype, self.channel_scale = shape, dtype, channel_scale

    @classmethod
    def _of(cls, tensors: Sequence[Tensor], shape, dtype, channel_scale=None) -> CompressedActivation:
        """From what `_tensors` gives: two tensors, or one buffer that holds the codes, then the exponents; no checks."""
        self = object.__new__(cls)
        self._codes, self._exponents, self._buffer = (*tensors, None) if len(tensors) == 2 else (None, None, tensors[0])
        self.shape, self.dtype, self.channel_scale = shape, dtype, channel_scale
        return self

    def _tensors(self) -> tuple[Tensor, ...]:
        """What holds the codes and exponents."""
        return (self._codes, self._exponents) if self._buffer is None else (self._buffer,)

    @property
    def codes(self) -> Tensor:
        if self._buffer is None:
            return self._codes
        rows, groups = _rows(self.shape), -(-self.shape[-1] // GROUP)
        return self._buffer[: rows * groups * GROUP].view(torch.int8).view(rows, groups * GROUP)

    @property
    def exponents(self) -> Tensor:
        if self._buffer is None:
            return self._exponents
        rows, groups = _rows(self.shape), -(-self.shape[-1] // GROUP)
        return self._buffer[rows * groups * GROUP : rows * groups * (GROUP + 1)].view(rows, groups)

    @property
    def device(self) -> torch.device:
        return (self._codes if self._buffer is None else self._buffer).device

    @property
    def nbytes(self) -> int:
        """Bytes of the codes and exponents."""
        return self.codes.numel() + self.exponents.numel()

    def decompress(self) -> Tensor:
        return decompress(self)

    def __repr__(self) -> str:
        return f"CompressedActivation(shape={tuple(self.shape)}, dtype={self.dtype}, device={self.device}, nbytes={self.nbytes})"


class RMSNormOutput(NamedTuple):
    """What `rms_norm` returns: the normalised `output`, the updated `residual` (None if none was given) and, where it was
    kept, the 8-bit form of the output (`saved`, for `linear`)."""

    output: Tensor
    residual: Tensor | None
    saved: CompressedActivation | None


# ---------------------------------------------------------------------------------------------
# operators: checks of arguments, autograd nodes and kernel calls are in csrc/activations_host.cpp
# ---------------------------------------------------------------------------------------------


def _rows(shape) -> int:
    rows = 1
    for n in shape[:-1]:
        rows *= n
    return rows


def compress(x: Tensor) -> CompressedActivation:
    """`x` (float32, bfloat16 or float16; any shape with at least one dimension) in 8 bits.  Takes no part in autograd."""
    return CompressedActivation._of((_lib.HOST.compress(x),), x.shape, x.dtype)


def decompress(saved: CompressedActivation) -> Tensor:
    """The activation `saved` stands for, its `channel_scale` applied."""
    return _lib.HOST.decompress(saved._tensors(), saved.shape, saved.dtype, saved.channel_scale)


def weight_gradient(grad: Tensor, saved: CompressedActivation) -> Tensor:
    """Gradient of a linear layer's weight, ``grad^T @ saved`` summed over all tokens: (outputs, channels), in `grad`'s type.

    `grad` (bfloat16 or float16) has the leading dimensions of `saved.shape`.  The kept activation goes to the tensor
    cores as it is (its values are exact in 16 bits); sums are held in 32 bits.  Takes no part in autograd.
    """
    return _lib.HOST.weight_gradient(grad, saved._tensors(), saved.shape, saved.dtype, saved.channel_scale)


def rms_norm(x: Tensor, weight: Tensor | None = None, residual: Tensor | None = None, *, eps: float | None = None,
             compress: bool = False) -> RMSNormOutput:  # fmt: skip
    """Root-mean-square norm of ``h = x + residual`` over the last dimension, ``h / sqrt(mean(h**2) + eps) * weight``.

    The sum is rounded to `x`'s type before it is normalised, and is returned as the new residual.  `eps` defaults to
    float32's machine epsilon, 2**-23, for all three types, as in `torch.nn.RMSNorm`.  Where gradients are wanted the normalised
    row is kept in 8 bits: the backward pass reads it, and `linear` can share it (`saved`).  `compress=True` keeps it without
    gradients too.
    """
    output, new_residual, buffer = _lib.HOST.rms_norm(x, weight, residual, eps, compress)
    if buffer is None:
        return RMSNormOutput(output, new_residual, None)
    saved = CompressedActivation._of((buffer,), x.shape, x.dtype, None if weight is None else weight.detach())
    return RMSNormOutput(output, new_residual, saved)


def linear(x: Tensor, weight: Tensor, bias: Tensor | None = None, *, saved: CompressedActivation | None = None) -> Tensor:
    """`torch.nn.functional.linear` that keeps its input in 8 bits for the weight gradient instead of `x` itself.

    `saved`: the 8-bit form of `x` where there is one already (`rms_norm`'s, or one `compress(x)` shared by several
    layers); else `x` is compressed here, where the weight needs a gradient.  bfloat16 and float16; under autocast
    the arguments are cast as `torch.nn.functional.linear` casts them.
    """
    if saved is None:
        return _lib.HOST.linear(x, weight, bias, (), (), None, None)
    return _lib.HOST.linear(x, weight, bias, saved._tensors(), saved.shape, saved.dtype, saved.channel_scale)


# ---------------------------------------------------------------------------------------------
# recomputation from 8 bits
# ---------------------------------------------------------------------------------------------


def _pack(t: Tensor):
    # An activation, not a mask, table or parameter: it has a history.  A leaf is held by the user anyway.
    if t.requires_grad and not t.is_leaf and t.dtype in _lib.DTYPE_CODE and t.dim() > 0 and t.numel() > 0:
        return compress(t)
    return t


def _unpack(kept):
    return decompress(kept) if isinstance(kept, CompressedActivation) else kept


def checkpoint(function: Callable, *args: Any, **kwargs: Any):
    """`torch.utils.checkpoint.checkpoint(function, *args, use_reentrant=False, **kwargs)` whose differentiable inputs are kept in
    8 bits: the backward pass restores them and runs `function` again.

    Inputs that carry no history (masks, tables, parameters, leaves) are kept as they are.
    """
    if kwargs.pop("use_reentrant", False):
        raise ValueError("checkpoint: use_reentrant=True is not supported")
    with torch.autograd.graph.saved_tensors_hooks(_pack, _unpack):
        return torch.utils.checkpoint.checkpoint(function, *args, use_reentrant=False, **kwargs)


# ---------------------------------------------------------------------------------------------
# models
# ---------------------------------------------------------------------------------------------


class _Kept:
    """A norm's 8-bit row, on the norm's output, and what tells whether that is still the tensor it was.

    The row is shared only where saved tensors take the way they took in the norm: a block that is run again in the backward
    pass gets the output of a norm outside as a tensor of its own, without the row, and has to save the same both times.
    """

    __slots__ = ("saved", "version", "address", "shape", "hook")

    def __init__(self, saved: CompressedActivation, y: Tensor):
        self.saved, self.version, self.address, self.shape = saved, y._version, y.data_ptr(), y.shape
        self.hook = _lib.HOST.saving_hook()

    def __reduce__(self):
        # a copy or a file of the output has no part in it (and loads with weights_only)
        return OrderedDict, ()


def _kept(x: Tensor) -> CompressedActivation | None:
    """The 8-bit form a norm attached to this very tensor, unless the tensor was written to or given other memory since."""
    kept = getattr(x, _KEPT_ATTR, None)
    if type(kept) is not _Kept or (kept.version, kept.address, kept.shape) != (x._version, x.data_ptr(), x.shape):
        return None
    return kept.saved if kept.hook is _lib.HOST.saving_hook() else None


class _CompressedLinear(nn.Linear):
    def forward(self, x: Tensor) -> Tensor:
        casts = torch.is_autocast_enabled("cuda")
        dtype = torch.get_autocast_dtype("cuda") if casts else self.weight.dtype
        if not (torch.is_grad_enabled() and self.weight.requires_grad and dtype in (torch.bfloat16, torch.float16)) or torch.jit.is_tracing():
            return super().forward(x)
        if casts and not all(t.is_floating_point() and t.dtype != torch.float64 for t in (x, self.weight)):  # autocast leaves these alone
            return super().forward(x)
        return linear(x, self.weight, self.bias, saved=_kept(x) if x.dtype == dtype else None)


class _CompressedRMSNorm(nn.RMSNorm):
    def forward(self, x: Tensor) -> Tensor:
        w = self.weight
        if not torch.is_grad_enabled() or not (x.requires_grad or (w is not None and w.requires_grad)):
            return super().forward(x)
        if torch.is_autocast_enabled("cuda") or torch.jit.is_tracing() or x.dtype not in _lib.DTYPE_CODE or (w is not None and w.dtype != x.dtype):
            return super().forward(x)
        out = rms_norm(x, w, eps=self.eps)
        y = out.output
        setattr(y, _KEPT_ATTR, _Kept(out.saved, y))
        return y


def prepare_for_compressed_activations(model: nn.Module) -> nn.Module:
    """Makes the `nn.Linear` and `nn.RMSNorm` layers of `model` keep their activations in 8 bits while gradients are recorded.

    A linear layer that follows such a norm directly shares the norm's 8-bit row, unless only one of the two is in a block that is
    recomputed; every other one compresses its own input, so that layers which share an input that no such norm made keep it
    once each (`linear` with one `compress(x)` for all of them does not).  What is written to a norm's output past autograd
    (`.data`, raw pointers) is not seen by the row.  Layers of other types, subclasses of these two, norms over more than the last dimension, linear layers that
    compute in float32 and norms under autocast or with a weight of another type stay as they are, and so does every layer
    in float64 or under `torch.jit.trace`.  Parameters and `state_dict` do not change, nor do forward results beyond a norm's last bit.  Works
    with gradient release, gradient accumulation and autocast.
    """
    if hasattr(model, _PREPARED_ATTR):
        raise ValueError("Model is already prepared for compressed activations.")
    changed = []
    for module in model.modules():
        if type(module) is nn.Linear:
            module.__class__ = _CompressedLinear
        elif type(module) is nn.RMSNorm and len(module.normalized_shape) == 1:
            module.__class__ = _CompressedRMSNorm
        else:
            continue
        changed.append(module)
    object.__setattr__(model, _PREPARED_ATTR, changed)
    return model


def remove_compressed_activations(model: nn.Module) -> None:
    """Gives the layers that `prepare_for_compressed_activations` changed their own forward back."""
    changed = getattr(model, _PREPARED_ATTR, None)
    if changed is None:
        warn("`model` does not have any compressed activations to remove.")
        return
    for module in changed:
        if type(module) is _CompressedLinear:
            module.__class__ = nn.Linear
        elif type(module) is _CompressedRMSNorm:
            module.__class__ = nn.RMSNorm
    delattr(model, _PREPARED_ATTR)
