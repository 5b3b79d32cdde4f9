"""Latent attention: the full-attention mixer between the KDA layers
(``kimi_linear/mla.py``), as functions on the gfx950 kernels.

A token's keys and values come from one latent vector of ``rank`` channels and
a few position channels that all heads share.

* :func:`mla_expanded` -- keys and values already expanded per head, for
  prompts and training (differentiable);
* :func:`mla_absorbed` -- in the latent space over the cache itself, for
  decoding: single tokens, or a few at once;
* :func:`mla_cache_append` -- new rows written behind the cached ones, the
  latent part RMS-normalised on the way if asked, in 16 bits, 8 or 4;
* :func:`mla_cache_read` -- an 8- or 4-bit cache back in 16 bits.

A cache is ``[B, S, rank + P]``: one row a token, latent then position
channels.  In 16 bits it has the activations' type; in 8 bits it is
``torch.float8_e4m3fn`` with ``cache_scale`` fp32 ``[B, S, 2]``, a scale for a
row's latent and one for its position part; in 4 bits ``torch.float4_e2m1fn_x2
[B, S, (rank + P) / 2]``, two channels a byte, with ``cache_scale``
``torch.float8_e8m0fnu [B, S, 8]``: a power of two for each 128 latent channels,
then one for the position part (bytes beyond it are not read).  ``lengths``, ``starts`` and
``counts`` are integer tensors ``[B]`` on the device; the kernels read them, so
a captured graph follows them.  A length to read by counts as 0 below 0 and as
S above it; rows to append that a length puts outside the cache are dropped.

Softmax weights are operands of 16 bits, off by up to half a step of the type
(2^-8 of themselves in bf16, 2^-11 in fp16); in fp16 one below 2^-29 of its row's
largest has fewer bits, and below 2^-40 none.  (Over an 8-bit cache that goes for a weight times its row's scale,
in 4 bits its group's, and in bf16 nothing is left below 2^-126 of the largest.)  Scores may be of any size that fp32 holds; a
weight is as exact as its score, to 2^-24 of that.  (Over 8 and 4 bits, what a workgroup has of a sequence is gone over
twice where a row's largest score there is past 66.)

HIP tensors only, fp16 or bf16 activations, no fallback: anything else raises
:class:`KdaError`, as do calls under a trace, ``vmap`` or forward-mode differentiation.  Calls are asynchronous on torch's current stream and may be
captured.  Views are read in place where their channels are contiguous and
their rows 16-byte aligned, and copied otherwise.
"""

from __future__ import annotations

import math

import torch
from torch.autograd import forward_ad
from torch.utils._python_dispatch import _disable_current_modes

from . import _native
from .kda import KdaError, _check_tensor

RANKS = (128, 256, 512)
POSITION_DIMS = (0, 32, 64)
HEAD_DIMS = (64, 128)
_ACT = (torch.float16, torch.bfloat16)
_FOUR = torch.float4_e2m1fn_x2


_FAR = 2 ** 23          # elements between tokens from which a tile's offsets pass 32 bits


def _rows(x, tiled=False):
    """x with contiguous channels and 16-byte aligned rows, and tokens that are not far apart where they are
    loaded in tiles; copied if it has not."""
    n = 16 // x.element_size()
    if (x.stride(-1) == 1 or x.shape[-1] <= 1) and x.data_ptr() % 16 == 0 and all(
            s % n == 0 for s, m in zip(x.stride()[:-1], x.shape[:-1]) if m > 1) and not (
            tiled and x.shape[1] > 1 and x.stride(1) >= _FAR):
        return x
    return x.clone(memory_format=torch.contiguous_format)


def _counts(name, x, B, device):
    if x is None:
        return None
    _check_tensor(name, x)
    if tuple(x.shape) != (B,) or x.dtype not in (torch.int32, torch.int64):
        raise KdaError(f"{name} must be an int32 or int64 tensor of shape [{B}]; got {x.dtype} {tuple(x.shape)}")
    _on_device(device, **{name: x})
    if x.dtype == torch.int64:
        x = x.clamp(-2 ** 31, 2 ** 31 - 1)
    return x.to(torch.int32).contiguous()


def _on_device(device, **tensors):
    for name, x in tensors.items():
        if x is not None and x.device != device:
            raise KdaError(f"{name} must be on {device}, got {x.device}")


def _activations(name, x):
    _check_tensor(name, x)
    if x.device.type != "cuda":
        raise KdaError(f"the latent-attention kernels need HIP tensors (got {name} on {x.device}); there is no CPU path")
    if x.dtype not in _ACT:
        raise KdaError(f"{name} must be float16 or bfloat16, got {x.dtype}")


def _positive(name, x):
    x = float(x)
    if not (math.isfinite(x) and x > 0):
        raise KdaError(f"{name} must be positive and finite, got {x}")
    return x


def _no_grad(what, *tensors):
    if torch.is_grad_enabled() and any(x is not None and x.requires_grad for x in tensors):
        raise KdaError(f"{what} is forward-only: call it under torch.no_grad() or detach the inputs")


def _refuse_transforms(name, *tensors):
    """A trace would record an output's memory without the kernel that fills it, and a transformed tensor or a
    subclass that dispatches for itself has no memory that the kernels could read."""
    if _native.host().traced():
        raise KdaError(f"{name} cannot be traced (make_fx, torch.export, torch.jit.trace, fake tensors): "
                       "keep the call out of the traced region")
    for x in tensors:
        if isinstance(x, torch.Tensor) and (torch._C._functorch.is_functorch_wrapped_tensor(x)
                                            or type(x).__torch_dispatch__ is not torch.Tensor.__torch_dispatch__):
            raise KdaError(f"{name} takes plain tensors: no vmap or other transform, no subclass that dispatches for itself")
        if isinstance(x, torch.Tensor) and forward_ad._current_level >= 0 and forward_ad.unpack_dual(x).tangent is not None:
            raise KdaError(f"{name} has no forward-mode derivative")


def _native_call(name, *args):
    """The native call on arguments already checked and laid out.  A dispatch mode that only looks on (one that
    counts operations, say) does not see it."""
    with _disable_current_modes():
        got = getattr(_native.host(), name)(*args)
    if got is None or got is False:
        raise KdaError(f"{name}: no kernel for these arguments (sizes beyond the kernels' limits, an output that "
                       "overlaps an input, or tensor subclasses)")
    return got


# ---- expanded ---------------------------------------------------------------

def mla_expanded(q, k_nope, k_pe, v, lengths=None, starts=None, scale=None):
    """Causal attention over expanded keys and values.

    ``q [B, T, H, N + P]``, ``k_nope [B, S, H, N]``, ``k_pe [B, S, P]`` (None if
    P = 0), ``v [B, S, H, N]``, N 64 or 128, P 0, 32 or 64; ``scale`` defaults
    to ``(N + P) ** -0.5``.  Returns ``o [B, T, H, N]``:

        o_t = sum_j softmax_j(scale q_t . [k_nope_j | k_pe_j]) v_j,
        j < lengths[b],  j <= starts[b] + t

    ``lengths`` (default S) are the tokens each sequence has: rows of k and v
    from there on are never read.  ``starts`` (default S - T) is the position
    of query 0, of either sign.  A query whose position is ``lengths[b]`` or more does not
    exist, and one below 0 or of an empty sequence sees no key: both give zeros
    (and zero gradients).  A key or value that is not finite may reach the
    queries of up to 127 positions before its own.

    Differentiable in q, k_nope, k_pe and v (once); gradients have the inputs'
    types, are the same from run to run, and zero in rows past ``lengths``.  In a
    captured backward pass the inputs must have no eager graph alive on the
    default stream (its outputs deleted, or made on another stream): refused."""
    try:
        o = _native.host().mla_expanded(q, k_nope, k_pe, v, lengths, starts, q.shape[-1] ** -0.5 if scale is None else scale)
    except (TypeError, AttributeError, ZeroDivisionError):      # an argument of no type a common call has
        o = None
    if o is not None:
        return o
    _refuse_transforms("mla_expanded", q, k_nope, k_pe, v, lengths, starts)
    _activations("q", q)
    _check_tensor("k_nope", k_nope)
    _check_tensor("v", v)
    if q.dim() != 4 or k_nope.dim() != 4 or v.dim() != 4:
        raise KdaError(f"q, k_nope and v must be [B, tokens, H, D]; got {tuple(q.shape)}, {tuple(k_nope.shape)}, "
                       f"{tuple(v.shape)}")
    B, T, H, D = q.shape
    S, N = k_nope.shape[1], k_nope.shape[3]
    if k_pe is not None:
        _check_tensor("k_pe", k_pe)
        if k_pe.dim() == 3 and k_pe.shape[2] == 0:
            k_pe = None
    P = 0 if k_pe is None else k_pe.shape[-1]
    if N not in HEAD_DIMS or P not in POSITION_DIMS:
        raise KdaError(f"no kernel for head dimension {N} and position dimension {P} (N in {HEAD_DIMS}, P in {POSITION_DIMS})")
    if tuple(k_nope.shape) != (B, S, H, N) or tuple(v.shape) != (B, S, H, N) or D != N + P or (
            k_pe is not None and tuple(k_pe.shape) != (B, S, P)):
        raise KdaError(f"shapes do not fit: q {tuple(q.shape)} [B, T, H, N + P], k_nope {tuple(k_nope.shape)} and "
                       f"v {tuple(v.shape)} [B, S, H, N], k_pe {None if k_pe is None else tuple(k_pe.shape)} [B, S, P]")
    _on_device(q.device, k_nope=k_nope, k_pe=k_pe, v=v)
    for name, x in (("k_nope", k_nope), ("v", v), ("k_pe", k_pe)):
        if x is not None and not x.dtype.is_floating_point:
            raise KdaError(f"{name} must be a floating tensor, got {x.dtype}")
    lengths, starts = _counts("lengths", lengths, B, q.device), _counts("starts", starts, B, q.device)
    scale = _positive("scale", D ** -0.5 if scale is None else scale)
    q = _rows(q, tiled=True)
    k_nope, v = _rows(k_nope.to(q.dtype), tiled=True), _rows(v.to(q.dtype), tiled=True)
    k_pe = None if k_pe is None else _rows(k_pe.to(q.dtype), tiled=True)
    return _native_call("mla_expanded", q, k_nope, k_pe, v, lengths, starts, scale)


# ---- the cache --------------------------------------------------------------

def _check_cache(cache, cache_scale, rank, B, D, act):
    _check_tensor("cache", cache)
    if rank not in RANKS or D - rank not in POSITION_DIMS:
        raise KdaError(f"no kernel for rank {rank} and position dimension {D - rank} "
                       f"(rank in {RANKS}, position dimension in {POSITION_DIMS})")
    width = D // 2 if cache.dtype == _FOUR else D
    if cache.dim() != 3 or cache.shape[0] != B or cache.shape[2] != width:
        raise KdaError(f"cache must be [B, S, rank + P{' over 2' if width != D else ''}] = [{B}, S, {width}]; got {tuple(cache.shape)}")
    if cache.dtype == _FOUR:
        if not isinstance(cache_scale, torch.Tensor) or cache_scale.dtype != torch.float8_e8m0fnu or tuple(
                cache_scale.shape) != (B, cache.shape[1], 8):
            raise KdaError(f"a 4-bit cache needs cache_scale, float8_e8m0fnu [B, S, 8] = [{B}, {cache.shape[1]}, 8]")
    elif cache.dtype == torch.float8_e4m3fn:
        if not isinstance(cache_scale, torch.Tensor) or cache_scale.dtype != torch.float32 or tuple(
                cache_scale.shape) != (B, cache.shape[1], 2):
            raise KdaError(f"an 8-bit cache needs cache_scale, float32 [B, S, 2] = [{B}, {cache.shape[1]}, 2]")
    elif cache.dtype != act:
        raise KdaError(f"cache must be {act} (the activations' type), float8_e4m3fn or float4_e2m1fn_x2, got {cache.dtype}")
    elif cache_scale is not None:
        raise KdaError("cache_scale belongs to an 8- or 4-bit cache only")


def _check_layout(**tensors):
    """The cache and its scales are used in place, so their layout has to fit as it is."""
    for name, x in tensors.items():
        if x is None:
            continue
        n = 8 if x.dtype in (torch.float32, torch.float8_e8m0fnu) else 16          # bytes
        if x.stride(-1) != 1 or x.data_ptr() % n != 0 or any(
                s * x.element_size() % n != 0 for s, m in zip(x.stride()[:-1], x.shape[:-1]) if m > 1):
            raise KdaError(f"{name} needs contiguous channels and aligned rows (16 bytes; a row's scales 8); "
                           f"got strides {x.stride()}")


def mla_absorbed(q, cache, lengths, rank, scale, cache_scale=None):
    """Attention in the latent space: ``q [B, T, H, rank + P]``, its first
    ``rank`` channels taken through each head's key up-projection, over the
    cache ``[B, S, rank + P]`` itself.  Returns ``o [B, T, H, rank]`` (which the
    value up-projection takes to the heads' values):

        o_t = sum_j softmax_j(scale q_t . cache_j) cache_j[:rank],
        j <= lengths[b] - T + t

    ``lengths [B]`` counts a sequence's tokens with the T new ones, which are
    its last (append them first); cache rows from there on are never read.  A
    row that sees no key (an idle slot, or ``lengths[b] < T``) gives zeros.  A value of a 4-bit cache is taken in q's
    type by a score in bf16, where one past the type's range (scales of 2^126 and 2^127) is infinity.  A
    cached row that is not finite may reach the up to T - 1 queries before its own.
    ``scale`` is that of the expanded form, ``(N + P) ** -0.5``; ``cache_scale``
    of the tokens as :func:`mla_cache_append` writes it (positive, from 2^-60).
    Ranks 128, 256, 512, P 0, 32, 64; cache rows less than 2^23 elements apart.
    Forward only."""
    try:
        o = _native.host().mla_absorbed(q, cache, lengths, rank, scale, cache_scale)
    except TypeError:
        o = None
    if o is not None:
        return o
    _refuse_transforms("mla_absorbed", q, cache, lengths, cache_scale)
    _activations("q", q)
    if q.dim() != 4:
        raise KdaError(f"q must be [B, T, H, rank + P]; got {tuple(q.shape)}")
    _check_cache(cache, cache_scale, rank, q.shape[0], q.shape[3], q.dtype)
    _on_device(q.device, cache=cache, cache_scale=cache_scale)
    _no_grad("mla_absorbed", q, cache, cache_scale)
    lengths = _counts("lengths", lengths, q.shape[0], q.device)
    if lengths is None:
        raise KdaError("lengths is needed: an integer tensor [B] on the device")
    _check_layout(cache=cache, cache_scale=cache_scale)
    return _native_call("mla_absorbed", _rows(q.detach()), cache.detach(), lengths, rank, _positive("scale", scale),
                        cache_scale)


def mla_cache_append(x, cache, lengths, rank, cache_scale=None, counts=None, norm_weight=None, eps=1e-6):
    """Write ``x [B, T, rank + P]`` into the cache, in place: row t of sequence b
    to cache row ``lengths[b] + t`` for ``t < counts[b]`` (default T).  Rows that
    would fall below 0, at or past S are dropped, every other row of the cache is left
    as it is; ``lengths`` itself does not change.

    With ``norm_weight [rank]`` (x's type, or taken in fp32) the latent part is
    RMS-normalised first, in fp32.  Values are rounded once to the cache's type.  In 8 bits a row's
    latent part and its position part each get the scale max|x| / 448 (at
    least 2^-60, written to ``cache_scale``; 1 where P = 0) and x / scale is
    rounded to the nearest e4m3 value.  In 4 bits each 128 channels of the latent
    part, and the position part, get the least power of two (at least 2^-60) that
    leaves their largest magnitude at most 7, the quotients, which are exact, go
    to the nearest e2m1 value, ties to the even one, above 6 to 6, and the norm's
    mean is summed in 64 bits.  A row with a value that is not finite
    reads back as not finite.  x must not overlap the cache, nor rows of the
    cache each other.  Forward only."""
    try:
        if _native.host().mla_append(x, cache, lengths, rank, cache_scale, counts, norm_weight, eps):
            return
    except TypeError:
        pass
    _refuse_transforms("mla_cache_append", x, cache, lengths, cache_scale, counts, norm_weight)
    _activations("x", x)
    if x.dim() != 3:
        raise KdaError(f"x must be [B, T, rank + P]; got {tuple(x.shape)}")
    B, T, D = x.shape
    _check_cache(cache, cache_scale, rank, B, D, x.dtype)
    _on_device(x.device, cache=cache, cache_scale=cache_scale, norm_weight=norm_weight)
    _no_grad("mla_cache_append", x, cache, cache_scale, norm_weight)
    if norm_weight is not None:
        _check_tensor("norm_weight", norm_weight)
        if norm_weight.numel() != rank:
            raise KdaError(f"norm_weight must have {rank} values; got {tuple(norm_weight.shape)}")
        norm_weight = norm_weight.detach().reshape(rank)
        norm_weight = _rows(norm_weight if norm_weight.dtype == x.dtype else norm_weight.float())
    lengths, counts = _counts("lengths", lengths, B, x.device), _counts("counts", counts, B, x.device)
    if lengths is None:
        raise KdaError("lengths is needed: an integer tensor [B] on the device")
    _check_layout(cache=cache, cache_scale=cache_scale)
    _native_call("mla_append", _rows(x.detach()), cache, lengths, rank, cache_scale, counts, norm_weight, float(eps))


def mla_cache_read(cache, cache_scale, rank, dtype=torch.bfloat16, tokens=None, lengths=None):
    """The first ``tokens`` (default all) rows of an 8- or 4-bit cache in 16 bits:
    ``[B, tokens, rank + P]`` of value x scale, rounded once.  Rows at or past
    ``lengths[b]`` are zeros, and not read.  Forward only."""
    try:
        out = _native.host().mla_read(cache, cache_scale, rank, dtype, cache.shape[1] if tokens is None else tokens,
                                      lengths)
    except (TypeError, AttributeError, IndexError):
        out = None
    if out is not None:
        return out
    _refuse_transforms("mla_cache_read", cache, cache_scale, lengths)
    _check_tensor("cache", cache)
    if dtype not in _ACT:
        raise KdaError(f"dtype must be float16 or bfloat16, got {dtype}")
    if cache.device.type != "cuda":
        raise KdaError(f"the latent-attention kernels need HIP tensors (got cache on {cache.device}); there is no CPU path")
    if cache.dtype not in (torch.float8_e4m3fn, _FOUR) or cache.dim() != 3:
        raise KdaError(f"cache must be float8_e4m3fn [B, S, rank + P] or float4_e2m1fn_x2 [B, S, (rank + P) / 2]; "
                       f"got {cache.dtype} {tuple(cache.shape)}")
    _check_cache(cache, cache_scale, rank, cache.shape[0], cache.shape[2] * (2 if cache.dtype == _FOUR else 1), dtype)
    _on_device(cache.device, cache_scale=cache_scale)
    n = cache.shape[1] if tokens is None else int(tokens)
    if not 0 <= n <= cache.shape[1]:
        raise KdaError(f"tokens must be between 0 and {cache.shape[1]}, got {tokens}")
    _check_layout(cache=cache, cache_scale=cache_scale)
    return _native_call("mla_read", cache, cache_scale, rank, dtype, n, _counts("lengths", lengths, cache.shape[0], cache.device))
