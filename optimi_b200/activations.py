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

from collections.abc import Callable, Sequence
from typing import Any, NamedTuple
from warnings import warn

import torch
import torch.nn.functional as F
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
            if codes.stride(1) != 1 or exponents.stride(1) != 1 or (rows > 1 and codes.stride(0) % GROUP) or codes.data_ptr() % 16:
                raise ValueError("rows of codes and exponents must be contiguous, codes 16-byte aligned with a pitch that is a multiple of 32")
            if rows > 1 and (codes.stride(0) < padded or exponents.stride(0) < padded // GROUP):
                raise ValueError("rows of codes and exponents must not overlap")
        if channel_scale is not None and (channel_scale.shape != shape[-1:] or channel_scale.dtype != dtype or channel_scale.device != codes.device):
            raise ValueError(f"channel_scale must be a {dtype} tensor of {cols} values on {codes.device}")
        self._codes, self._exponents, self._buffer = codes, exponents, None
        self.shape, self.dtype, self.channel_scale = shape, dtype, channel_scale

    @classmethod
    def _of(cls, tensors: Sequence[Tensor], shape, dtype, channel_scale=None) -> CompressedActivation:
        """From what `_tensors` gave, or one buffer of `_buffer_bytes` that holds the codes, then the exponents; no checks."""
        self = object.__new__(cls)
        self._codes, self._exponents, self._buffer = (*tensors, None) if len(tensors) == 2 else (None, None, tensors[0])
        self.shape, self.dtype, self.channel_scale = shape, dtype, channel_scale
        return self

    def _tensors(self) -> tuple[Tensor, ...]:
        """What holds the codes and exponents, to be kept with `ctx.save_for_backward`."""
        return (self._codes, self._exponents) if self._buffer is None else (self._buffer,)

    def _layout(self) -> tuple[int, int, int, int]:
        """Addresses and pitches of codes and exponents."""
        if self._buffer is None:
            c, e = self._codes, self._exponents
            return c.data_ptr(), c.stride(0), e.data_ptr(), e.stride(0)
        rows, groups = _rows(self.shape), -(-self.shape[-1] // GROUP)
        at = self._buffer.data_ptr()
        return at, groups * GROUP, at + rows * groups * GROUP, groups

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
# calls of the kernels
# ---------------------------------------------------------------------------------------------


def _rows(shape) -> int:
    rows = 1
    for n in shape[:-1]:
        rows *= n
    return rows


def _check(name: str, what: str, t: Tensor, like: Tensor | None = None) -> None:
    if not t.is_cuda:
        raise RuntimeError(f"{name}: `{what}` lives on {t.device}; optimi_b200 takes CUDA tensors only (there is no CPU path)")
    if t.dtype not in _lib.DTYPE_CODE:
        raise RuntimeError(f"{name}: `{what}` has unsupported dtype {t.dtype} (float32, bfloat16 and float16 are)")
    if like is not None and (t.device != like.device or t.dtype != like.dtype):
        raise RuntimeError(f"{name}: `{what}` ({t.dtype}, {t.device}) does not match {like.dtype} on {like.device}")


def _as_rows(t: Tensor) -> Tensor:
    """`t` as a matrix of its last dimension whose rows are contiguous and do not overlap: itself where that holds, else a copy."""
    if t.is_neg():  # a lazily negated view: its memory holds the opposite
        t = t.detach().resolve_neg()
    if t.dim() != 2:
        t = t.detach().reshape(_rows(t.shape), t.shape[-1])
    if t.is_contiguous():
        return t
    if t.shape[1] != 1 and t.stride(1) != 1 or t.shape[0] > 1 and t.stride(0) < t.shape[1]:
        t = t.detach().contiguous()
    return t


def _ptr(t: Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _stream(device: torch.device) -> int:
    # torch.cuda.current_stream(device).cuda_stream without the Stream object around it (2 us of a 15 us call)
    return torch._C._cuda_getCurrentRawStream(device.index)


def _call(fn, device: torch.device, *args) -> None:
    """Calls entry point `fn` with `args` and the current stream of `device`, that device being current."""
    if torch.cuda.current_device() == device.index:
        rc = fn(*args, _stream(device))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, _stream(device))
    if rc:
        _lib.check(rc)


def _dense_like(t: Tensor) -> Tensor:
    """A new contiguous tensor of `t`'s shape and type."""
    return torch.empty_like(t) if t.is_contiguous() else torch.empty(t.shape, dtype=t.dtype, device=t.device)


def _buffer_bytes(rows: int, cols: int) -> tuple[int, int]:
    """Bytes of codes and exponents in one buffer, and where 4-byte values may follow them."""
    n = rows * -(-cols // GROUP) * (GROUP + 1)
    return n, -(-n // 16) * 16


def compress(x: Tensor) -> CompressedActivation:
    """`x` (float32, bfloat16 or float16; any shape with at least one dimension) in 8 bits.  Takes no part in autograd."""
    _check("compress", "x", x)
    if x.dim() == 0:
        raise RuntimeError("compress: `x` must have at least one dimension")
    m = _as_rows(x)
    rows, cols = m.shape
    device = x.device
    saved = CompressedActivation._of((torch.empty(_buffer_bytes(rows, cols)[0], dtype=torch.uint8, device=device),), x.shape, x.dtype)
    _call(_lib.LIB.optimi_b200_compress, device, m.data_ptr(), m.stride(0), rows, cols, _lib.DTYPE_CODE[x.dtype], *saved._layout())
    return saved


def decompress(saved: CompressedActivation) -> Tensor:
    """The activation `saved` stands for, its `channel_scale` applied."""
    device = saved.device
    if device.type != "cuda":
        raise RuntimeError(f"decompress: `saved` lives on {device}; optimi_b200 takes CUDA tensors only (there is no CPU path)")
    out = torch.empty(saved.shape, dtype=saved.dtype, device=device)
    scale = None if saved.channel_scale is None else saved.channel_scale.detach().contiguous()
    _call(_lib.LIB.optimi_b200_decompress, device, *saved._layout(), _ptr(scale), _rows(saved.shape), saved.shape[-1],
          _lib.DTYPE_CODE[saved.dtype], out.data_ptr())  # fmt: skip
    return out


def weight_gradient(grad: Tensor, saved: CompressedActivation) -> Tensor:
    """Gradient of a linear layer's weight, ``grad^T @ saved`` summed over all tokens: (outputs, channels), in `grad`'s type.

    `grad` (bfloat16 or float16) has the leading dimensions of `saved.shape`.  The kept activation goes to the tensor
    cores as it is (its values are exact in 16 bits); sums are held in 32 bits.
    """
    name = "weight_gradient"
    _check(name, "grad", grad)
    if grad.dtype == torch.float32:
        raise RuntimeError(f"{name}: `grad` is float32; bfloat16 and float16 are supported")
    if saved.dtype != grad.dtype or saved.device != grad.device:
        raise RuntimeError(f"{name}: `saved` ({saved.dtype}, {saved.device}) does not match `grad` ({grad.dtype}, {grad.device})")
    if grad.dim() == 0 or _rows(grad.shape) != _rows(saved.shape):
        raise RuntimeError(f"{name}: `grad` {tuple(grad.shape)} and `saved` {tuple(saved.shape)} have different numbers of tokens")
    m = _as_rows(grad.detach())
    rows, outputs = m.shape
    channels = saved.shape[-1]
    device, code = grad.device, _lib.DTYPE_CODE[grad.dtype]
    pitch = -(-outputs // 8) * 8
    copied = m.data_ptr() % 16 != 0 or (m.stride(0) if rows > 1 else outputs) % 8 != 0  # the kernel loads rows that begin on 16 bytes
    stride = pitch if copied or rows <= 1 else m.stride(0)
    dw = torch.empty((outputs, channels), dtype=grad.dtype, device=device)
    scale = None if saved.channel_scale is None else saved.channel_scale.detach().contiguous()
    need = _lib.LIB.optimi_b200_weight_gradient_workspace_bytes(rows, outputs, channels)
    workspace = torch.empty(need, dtype=torch.uint8, device=device) if need else None
    if copied:
        source, m = m, torch.empty((rows, pitch), dtype=grad.dtype, device=device)
        _call(_lib.LIB.optimi_b200_align_rows, device, source.data_ptr(), source.stride(0), rows, outputs, code, m.data_ptr(), pitch)
    _call(_lib.LIB.optimi_b200_weight_gradient, device, m.data_ptr(), stride, *saved._layout(), _ptr(scale), rows, outputs, channels,
          code, dw.data_ptr(), _ptr(workspace), need)  # fmt: skip
    return dw


def _norm_forward(x: Tensor, weight: Tensor | None, residual: Tensor | None, eps: float, keep: bool):
    """(output, sum, buffer): the buffer holds the 8-bit form of the normalised rows and, behind it, their 1 / rms."""
    m = _as_rows(x)
    r = None if residual is None else _as_rows(residual)
    rows, cols = m.shape
    device = x.device
    y = _dense_like(x)
    h = None if r is None else _dense_like(x)
    buffer = None
    kept = (None, 0, None, 0, None)
    if keep:
        _, after = _buffer_bytes(rows, cols)
        buffer = torch.empty(after + 4 * rows, dtype=torch.uint8, device=device)
        at, groups = buffer.data_ptr(), -(-cols // GROUP)
        kept = (at, groups * GROUP, at + rows * groups * GROUP, groups, at + after)
    _call(_lib.LIB.optimi_b200_rms_norm, device, m.data_ptr(), m.stride(0), _ptr(r), 0 if r is None else r.stride(0), _ptr(weight),
          rows, cols, eps, _lib.DTYPE_CODE[x.dtype], y.data_ptr(), _ptr(h), *kept)  # fmt: skip
    return y, h, buffer


class _RMSNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps, kept):
        w = None if weight is None else weight.contiguous()
        y, h, buffer = _norm_forward(x, w, residual, eps, True)
        kept.append(buffer)
        ctx.save_for_backward(buffer, weight)
        ctx.set_materialize_grads(False)
        return y, h

    @staticmethod
    def backward(ctx, grad, grad_sum):
        _refuse_double_backward("rms_norm")
        buffer, weight = ctx.saved_tensors
        need_x, need_w, need_r = ctx.needs_input_grad[:3]
        if grad is None:  # only the residual was used: it passes through
            dw = torch.zeros_like(weight) if need_w else None
            return grad_sum if need_x else None, dw, grad_sum if need_r else None, None, None
        g = _as_rows(grad)
        s = None if grad_sum is None else _as_rows(grad_sum)
        w = None if weight is None else weight.contiguous()
        rows, cols = g.shape
        dx = _dense_like(grad) if need_x or need_r else None
        dw = torch.empty_like(w) if need_w else None
        code = _lib.DTYPE_CODE[grad.dtype]
        need = _lib.LIB.optimi_b200_rms_norm_backward_workspace_bytes(rows, cols, code) if need_w else 0
        workspace = torch.empty(need, dtype=torch.uint8, device=grad.device) if need else None
        at, groups = buffer.data_ptr(), -(-cols // GROUP)
        _call(_lib.LIB.optimi_b200_rms_norm_backward, grad.device, g.data_ptr(), g.stride(0), _ptr(s), 0 if s is None else s.stride(0),
              at, groups * GROUP, at + rows * groups * GROUP, groups, at + _buffer_bytes(rows, cols)[1], _ptr(w), rows, cols,
              code, _ptr(dx), _ptr(dw), _ptr(workspace), need)  # fmt: skip
        return dx if need_x else None, dw, dx if need_r else None, None, None


def _refuse_double_backward(name: str) -> None:
    # gradients are recorded inside a backward pass only under create_graph=True, and these kernels' would come out as constants
    if torch.is_grad_enabled():
        raise RuntimeError(f"{name}: differentiating the backward pass (create_graph=True) is not supported")


def rms_norm(x: Tensor, weight: Tensor | None = None, residual: Tensor | None = None, *, eps: float | None = None,
             compress: bool = False) -> RMSNormOutput:  # fmt: skip
    """Root-mean-square norm of ``h = x + residual`` over the last dimension, ``h / sqrt(mean(h**2) + eps) * weight``.

    The sum is rounded to `x`'s type before it is normalised, and is returned as the new residual.  `eps` defaults to
    the type's machine epsilon, as in `torch.nn.RMSNorm`.  Where gradients are wanted the normalised row is kept in 8 bits:
    the backward pass reads it, and `linear` can share it (`saved`).  `compress=True` keeps it without gradients too.
    """
    name = "rms_norm"
    _check(name, "x", x)
    if x.dim() == 0:
        raise RuntimeError(f"{name}: `x` must have at least one dimension")
    if weight is not None:
        _check(name, "weight", weight, x)
        if weight.shape != x.shape[-1:]:
            raise RuntimeError(f"{name}: `weight` {tuple(weight.shape)} does not match the last dimension of `x` {tuple(x.shape)}")
    if residual is not None:
        _check(name, "residual", residual, x)
        if residual.shape != x.shape:
            raise RuntimeError(f"{name}: `residual` {tuple(residual.shape)} does not match `x` {tuple(x.shape)}")
    eps = torch.finfo(x.dtype).eps if eps is None else float(eps)
    if not eps >= 0:
        raise ValueError(f"{name}: eps={eps} must not be negative")
    wants_grad = torch.is_grad_enabled() and (
        x.requires_grad or (weight is not None and weight.requires_grad) or (residual is not None and residual.requires_grad)
    )
    if wants_grad:
        kept: list[Tensor] = []
        y, h = _RMSNorm.apply(x, weight, residual, eps, kept)
        buffer = kept[0]
    else:
        w = None if weight is None else weight.detach().contiguous()
        y, h, buffer = _norm_forward(x, w, residual, eps, compress)
    saved = None if buffer is None else CompressedActivation._of((buffer,), x.shape, x.dtype, None if weight is None else weight.detach())
    return RMSNormOutput(y, h, saved)


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, saved):
        out = F.linear(x, weight, bias)
        ctx.shape = x.shape
        ctx.keeps_weight = ctx.needs_input_grad[0]
        keep = [weight] if ctx.keeps_weight else []
        if ctx.needs_input_grad[1]:
            if saved is None:
                saved = compress(x)
            keep += [saved.channel_scale, *saved._tensors()]
        ctx.save_for_backward(*keep)
        return out

    @staticmethod
    def backward(ctx, grad):
        _refuse_double_backward("linear")
        kept = list(ctx.saved_tensors)
        dx = dw = db = None
        if ctx.keeps_weight:
            dx = grad @ kept.pop(0)
        if ctx.needs_input_grad[1]:
            scale, *tensors = kept
            dw = weight_gradient(grad, CompressedActivation._of(tensors, ctx.shape, grad.dtype, scale))
        if ctx.needs_input_grad[2]:
            db = grad.reshape(-1, grad.shape[-1]).sum(0)
        return dx, dw, db, None


def linear(x: Tensor, weight: Tensor, bias: Tensor | None = None, *, saved: CompressedActivation | None = None) -> Tensor:
    """`torch.nn.functional.linear` that keeps its input in 8 bits for the weight gradient instead of `x` itself.

    `saved`: the 8-bit form of `x` where there is one already (`rms_norm`'s, or one `compress(x)` shared by several
    layers); else `x` is compressed here, once the weight needs a gradient.  bfloat16 and float16; under autocast
    the arguments are cast as `torch.nn.functional.linear` casts them.
    """
    name = "linear"
    if torch.is_autocast_enabled("cuda") and x.is_cuda:
        dtype = torch.get_autocast_dtype("cuda")
        x, weight, bias = x.to(dtype), weight.to(dtype), None if bias is None else bias.to(dtype)
    _check(name, "x", x)
    _check(name, "weight", weight, x)
    if bias is not None:
        _check(name, "bias", bias, x)
    if x.dtype == torch.float32:
        raise RuntimeError(f"{name}: float32 is not supported (bfloat16 and float16 are); use torch.nn.functional.linear")
    if x.dim() == 0 or weight.dim() != 2 or x.shape[-1] != weight.shape[1]:
        raise RuntimeError(f"{name}: `x` {tuple(x.shape)} and `weight` {tuple(weight.shape)} do not match")
    if bias is not None and bias.shape != weight.shape[:1]:
        raise RuntimeError(f"{name}: `bias` {tuple(bias.shape)} does not match `weight` {tuple(weight.shape)}")
    if saved is not None and (_rows(saved.shape), saved.shape[-1], saved.dtype, saved.device) != (_rows(x.shape), x.shape[-1], x.dtype, x.device):
        raise RuntimeError(f"{name}: `saved` ({tuple(saved.shape)}, {saved.dtype}, {saved.device}) does not stand for `x` "
                           f"({tuple(x.shape)}, {x.dtype}, {x.device})")  # fmt: skip
    if not torch.is_grad_enabled():
        return F.linear(x, weight, bias)
    with torch.autocast("cuda", enabled=False):
        return _Linear.apply(x, weight, bias, saved)


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


def _kept(x: Tensor) -> CompressedActivation | None:
    """The 8-bit form a norm attached to this very tensor, unless the tensor was written to or given other memory since."""
    kept = getattr(x, _KEPT_ATTR, None)
    return kept[0] if kept is not None and kept[1:] == (x._version, x.data_ptr(), x.shape) else None


class _CompressedLinear(nn.Linear):
    def forward(self, x: Tensor) -> Tensor:
        casts = torch.is_autocast_enabled("cuda")
        dtype = torch.get_autocast_dtype("cuda") if casts else self.weight.dtype
        if not (torch.is_grad_enabled() and self.weight.requires_grad and dtype in (torch.bfloat16, torch.float16)):
            return super().forward(x)
        return linear(x, self.weight, self.bias, saved=_kept(x) if x.dtype == dtype else None)


class _CompressedRMSNorm(nn.RMSNorm):
    def forward(self, x: Tensor) -> Tensor:
        w = self.weight
        if not torch.is_grad_enabled() or not (x.requires_grad or (w is not None and w.requires_grad)):
            return super().forward(x)
        if torch.is_autocast_enabled("cuda") or (w is not None and w.dtype != x.dtype):
            return super().forward(x)
        out = rms_norm(x, w, eps=self.eps)
        y = out.output
        setattr(y, _KEPT_ATTR, (out.saved, y._version, y.data_ptr(), y.shape))
        return y


def prepare_for_compressed_activations(model: nn.Module) -> nn.Module:
    """Makes the `nn.Linear` and `nn.RMSNorm` layers of `model` keep their activations in 8 bits while gradients are recorded.

    A linear layer that follows such a norm directly shares the norm's 8-bit row; every other one compresses its own
    input.  Layers of other types, subclasses of these two, norms over more than the last dimension, linear layers that
    compute in float32 and norms under autocast or with a weight of another type stay as they are.  Parameters and
    `state_dict` do not change, nor do forward results beyond a norm's last bit.  Works with gradient release, gradient
    accumulation and autocast.
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
