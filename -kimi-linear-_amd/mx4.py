"""Weights in 4 bits: the layers' projections for serving, as functions on the
gfx950 kernels and as a module.

A matrix ``[N, K]`` in this form is ``data``, ``torch.float4_e2m1fn_x2 [N, K / 2]``
-- values 0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives, two a byte, the lower
half first -- and ``scale``, ``torch.float8_e8m0fnu [N, K / 32]``, a power of two
for each 32 values along a row (the OCP microscaling format MXFP4).  Both may
come as ``torch.uint8`` of the same bytes.

* :func:`mx4_quantize` -- a matrix to that form;
* :func:`mx4_dequantize` -- and back in 16 bits;
* :func:`mx4_linear` -- x W^T with W in that form, for one row of x or many;
* :class:`Mx4Linear` -- the module around it, which ``KimiDeltaAttention`` and
  ``LatentAttention`` take in the places of their projections
  (``quantize_mx4_``).

HIP tensors only, fp16 or bf16 activations, forward only, no fallback: anything
else raises :class:`KdaError`, as do calls under a trace, ``vmap`` or
forward-mode differentiation.  Calls are asynchronous on torch's current
stream and may be captured.
"""

from __future__ import annotations

import torch
import torch.nn as nn

from . import _native
from .kda import KdaError, _check_tensor
from .mla import _ACT, _activations, _native_call, _no_grad, _on_device, _refuse_transforms

GROUP = 32
_DATA = (torch.float4_e2m1fn_x2, torch.uint8)
_SCALE = (torch.float8_e8m0fnu, torch.uint8)


def _even_rows(x, align=16):
    """x with contiguous channels, aligned rows and one stride between them; copied if it has not."""
    def rows():
        try:
            return x.view(-1, x.shape[-1])
        except RuntimeError:
            return None
    r = rows() if x.stride(-1) == 1 or x.shape[-1] == 1 else None
    if r is not None and r.data_ptr() % align == 0 and (r.shape[0] <= 1 or r.stride(0) * r.element_size() % align == 0
                                                        and 0 <= r.stride(0) <= 2 ** 22):
        return x
    return x.clone(memory_format=torch.contiguous_format)


def _check_mx4(data, scale, names=("data", "scale")):
    for name, x, types in zip(names, (data, scale), (_DATA, _SCALE)):
        _check_tensor(name, x)
        if x.dtype not in types:
            raise KdaError(f"{name} must be {types[0]} or uint8, got {x.dtype}")
    if data.dim() < 1 or scale.dim() != data.dim() or data.shape[-1] == 0 or data.shape[-1] != GROUP // 2 * scale.shape[-1] or (
            data.shape[:-1] != scale.shape[:-1]):
        raise KdaError(f"{names[0]} must be [.., K / 2] and {names[1]} [.., K / {GROUP}], K a multiple of {GROUP}; got "
                       f"{tuple(data.shape)} and {tuple(scale.shape)}")


def _packed(x):
    """Contiguous and aligned as the kernels read it."""
    x = x.detach().view(torch.uint8).contiguous()
    return x if x.data_ptr() % 16 == 0 else x.clone()


def mx4_quantize(w):
    """``w [.., K]`` (fp16, bf16 or fp32, K a multiple of 32) as ``(data, scale)``.

    A group's power is the least 2^e (e from -126) that leaves its largest
    magnitude at most 7, so no value is off by more than half the format's
    widest step; the quotients, which are exact, go to the nearest value, ties
    to the even one, above 6 to 6.  A group with a value that is not finite has
    the scale NaN, and reads back as NaN."""
    try:
        got = _native.host().mx4_quantize(w)
    except TypeError:
        got = None
    if got is not None:
        return got
    _refuse_transforms("mx4_quantize", w)
    _check_tensor("w", w)
    if w.device.type != "cuda":
        raise KdaError(f"the 4-bit kernels need HIP tensors (got w on {w.device}); there is no CPU path")
    if w.dtype not in (*_ACT, torch.float32):
        raise KdaError(f"w must be float16, bfloat16 or float32, got {w.dtype}")
    if w.dim() < 1 or w.shape[-1] == 0 or w.shape[-1] % GROUP != 0:
        raise KdaError(f"w must be [.., K], K a multiple of {GROUP}; got {tuple(w.shape)}")
    _no_grad("mx4_quantize", w)
    return _native_call("mx4_quantize", _even_rows(w.detach()))


def mx4_dequantize(data, scale, dtype=torch.bfloat16):
    """The matrix ``[.., K]`` that ``data`` and ``scale`` stand for, each value rounded once to ``dtype`` (fp16 or
    bf16; exact in bf16 for scales from 2^-125 to 2^125, in fp16 from 2^-23 to 2^13).  Past ``dtype``'s range that is
    infinity, which :func:`mx4_quantize` makes of finite values beyond 1.75 2^127 (fp16: 1.75 2^15): taken as 2^128 (2^16)."""
    try:
        out = _native.host().mx4_dequantize(data, scale, dtype)
    except (TypeError, AttributeError):
        out = None
    if out is not None:
        return out
    _refuse_transforms("mx4_dequantize", data, scale)
    _check_mx4(data, scale)
    if data.device.type != "cuda":
        raise KdaError(f"the 4-bit kernels need HIP tensors (got data on {data.device}); there is no CPU path")
    if dtype not in _ACT:
        raise KdaError(f"dtype must be float16 or bfloat16, got {dtype}")
    _on_device(data.device, scale=scale)
    return _native_call("mx4_dequantize", _packed(data), _packed(scale), dtype)


def mx4_linear(x, weight, weight_scale, bias=None, residual=None):
    """``x [.., K]`` times the transpose of a weight ``[N, K]`` in 4 bits, ``[.., N]`` in x's type.

    Sums are fp32, with the weight's values in x's type (exact in bf16 for
    scales from 2^-125 to 2^125, in fp16 from 2^-23 to 2^13; others are rounded, which beyond the type's range is infinity); ``bias [N]`` is
    added before the one rounding.  ``residual [.., N]``: the sum of it and the
    rounded product, as a residual stream adds it.  x may have any strides;
    rows that are not 16-byte aligned are copied.  Forward only."""
    return _linear(x, weight, weight_scale, bias, residual, None)


def _linear(x, weight, weight_scale, bias, residual, out):
    """:func:`mx4_linear`, into ``out`` [.., N], contiguous and apart from the inputs, where it is given."""
    try:
        y = _native.host().mx4_linear(x, weight, weight_scale, bias, residual, out)
    except TypeError:
        y = None
    if y is not None:
        return y
    _refuse_transforms("mx4_linear", x, weight, weight_scale, bias, residual)
    _check_tensor("x", x)
    if torch.is_autocast_enabled("cuda") and x.device.type == "cuda" and x.dtype.is_floating_point:
        x = x.to(torch.get_autocast_dtype("cuda"))      # as a projection in 16 bits is run under autocast
    _activations("x", x)
    _check_mx4(weight, weight_scale, ("weight", "weight_scale"))
    N = weight.shape[0]
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != 2 * weight.shape[1]:
        raise KdaError(f"shapes do not fit: x {tuple(x.shape)} [.., K], weight {tuple(weight.shape)} [N, K / 2]")
    for name, t, shape in (("bias", bias, (N,)), ("residual", residual, (*x.shape[:-1], N))):
        if t is not None:
            _check_tensor(name, t)
            if tuple(t.shape) != shape:
                raise KdaError(f"{name} must be {list(shape)}, got {tuple(t.shape)}")
    _on_device(x.device, weight=weight, weight_scale=weight_scale, bias=bias, residual=residual)
    _no_grad("mx4_linear", x, bias, residual)
    y = _general(x, weight, weight_scale, bias, residual)
    return y if out is None else out.copy_(y)


def _general(x, weight, weight_scale, bias, residual):
    bias = None if bias is None else bias.detach().to(x.dtype).contiguous()
    alike = residual is None or residual.dtype == x.dtype
    with torch.autocast("cuda", enabled=False):
        y = _native_call("mx4_linear", _even_rows(x.detach()), _packed(weight), _packed(weight_scale), bias,
                         _even_rows(residual.detach()) if residual is not None and alike else None, None)
    return y if alike else residual + y


class Mx4Linear(nn.Module):
    """``nn.Linear`` for serving, its weight in 4 bits.

    Buffers ``weight`` and ``weight_scale`` (``torch.uint8``, so that
    ``module.to(dtype)`` leaves them as they are) and ``bias`` or None.  Make it
    from a trained module with :meth:`from_linear`."""

    def __init__(self, in_features, out_features, bias=False, device=None, dtype=None):
        super().__init__()
        if in_features <= 0 or in_features % GROUP != 0:
            raise KdaError(f"in_features must be a multiple of {GROUP}, got {in_features}")
        self.in_features, self.out_features = in_features, out_features
        self.register_buffer("weight", torch.zeros(out_features, in_features // 2, dtype=torch.uint8, device=device))
        self.register_buffer("weight_scale", torch.full((out_features, in_features // GROUP), 127, dtype=torch.uint8,
                                                        device=device))
        self.register_buffer("bias", torch.zeros(out_features, device=device, dtype=dtype) if bias else None)

    @classmethod
    @torch.no_grad()
    def from_linear(cls, linear):
        """The 4-bit form of an ``nn.Linear`` on a HIP device.  A module that does more than the product with its
        weight and the bias (an adapter, a hook, a forward of its own) is refused: it would lose that."""
        if (type(linear) is not nn.Linear or linear._forward_hooks or linear._forward_pre_hooks or "forward" in linear.__dict__):
            raise KdaError(f"only a plain nn.Linear has a 4-bit form; got {type(linear).__name__} with hooks, a forward of its "
                           "own or another type")
        w = linear.weight
        data, scale = mx4_quantize(w)
        with torch.inference_mode(False), torch.no_grad():
            new = cls(linear.in_features, linear.out_features, linear.bias is not None, device=w.device, dtype=w.dtype)
            new.weight.copy_(data.view(torch.uint8))
            new.weight_scale.copy_(scale.view(torch.uint8))
            if linear.bias is not None:
                new.bias.copy_(linear.bias.detach())
        return new.train(linear.training)

    def forward(self, x):
        return mx4_linear(x, self.weight, self.weight_scale, self.bias)

    def extra_repr(self):
        return f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}"


def _plain_mx4(mod):
    """Whether a module is an :class:`Mx4Linear` as written here, without hooks or a forward of its own."""
    return (type(mod) is Mx4Linear and not mod._forward_hooks and not mod._forward_pre_hooks
            and "forward" not in mod.__dict__ and not nn.modules.module._has_any_global_hook())
