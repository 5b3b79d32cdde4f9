"""A latent-attention layer: the full-attention layer between the KDA layers
(``kimi_linear/mla.py``), around the kernels of :mod:`kimi_linear_amd.mla`.

    q = W_q x                      per head [N | P]
    [c | p] = W_down x             latent (rank channels) and position channels
    c <- RMSNorm(c)
    [k | v] = W_up c               per head, N channels each
    out = W_o attention(q, [k | p], v)

The position channels carry no rotation.  The layer has the call
protocol of ``KimiDeltaAttention``, so the two mix in one stack and in
``KdaGraphedDecoder``:

* ``layer(x)``: the whole sequence, through the expanded form; under grad mode
  differentiable, without a cache or state;
* ``layer(x, use_cache=True)``: the same, with the state
  ``{"latent", "scale", "lengths", "tokens"}``: the cache ``[B, max_tokens,
  rank + P]`` in 16 or 8 bits and its scales, the tokens held per sequence on
  the device and, as all sequences grow together, on the host;
* ``layer(x, state=state, use_cache=True)``: continues it, in place: one token
  through the absorbed form (the key and value up-projections applied to q and
  to the output), several through the expanded form over the cached latents.
  The absorbed form takes ``kv_up`` for the product with its weight: where the
  module does more (an adapter, a hook, a bias, a forward of its own) one token
  goes through the expanded form too, which calls the module;
* ``layer.decode_step_(x, state)``: one token.

A cache that would overflow raises :class:`KdaError` before anything is written.
"""

from __future__ import annotations

from types import SimpleNamespace

import torch
import torch.nn as nn

from . import _native
from .kda import KdaError
from .layer import _plain_weight
from .mla import mla_absorbed, mla_cache_append, mla_cache_read, mla_expanded


def latent_attn_config(**kw) -> SimpleNamespace:
    """A config object with the fields :class:`LatentAttention` reads; keyword
    overrides go into ``latent_attn_config`` except ``hidden_size`` and ``rms_norm_eps``."""
    la = dict(num_heads=16, head_dim=128, position_dim=64, rank=512, cache_bits=16, max_tokens=4096, proj_bias=False)
    top = dict(hidden_size=2048, rms_norm_eps=1e-6)
    for k, v in kw.items():
        (top if k in top else la)[k] = v
    return SimpleNamespace(latent_attn_config=la, **top)


class LatentAttention(nn.Module):
    """The latent-attention layer; see the module's docstring."""

    def __init__(self, config):
        super().__init__()
        la, d = config.latent_attn_config, config.hidden_size
        self.num_heads, self.head_dim = la["num_heads"], la["head_dim"]
        self.position_dim, self.rank = la["position_dim"], la["rank"]
        self.cache_bits, self.max_tokens = la["cache_bits"], la["max_tokens"]
        if self.cache_bits not in (8, 16):
            raise KdaError(f"cache_bits must be 8 or 16, got {self.cache_bits}")
        self.eps = config.rms_norm_eps
        H, N, P, R = self.num_heads, self.head_dim, self.position_dim, self.rank
        bias = la.get("proj_bias", False)
        self.q_proj = nn.Linear(d, H * (N + P), bias=bias)
        self.kv_down = nn.Linear(d, R + P, bias=bias)
        self.kv_norm = nn.Parameter(torch.ones(R))
        self.kv_up = nn.Linear(R, H * 2 * N, bias=False)         # per head: N key rows, then N value rows
        self.o_proj = nn.Linear(H * N, d, bias=bias)
        self.scale = (N + P) ** -0.5
        self._up = None            # (key, W_k [H, N, R], W_v [H, R, N], weight) for the absorbed form

    def _up_weights(self):
        """The up-projections as the absorbed form takes them, per head ``W_k [H, N, R]`` and ``W_v [H, R, N]``:
        copies of ``kv_up.weight``, made again (in place, so that a captured step sees them) when it changes.
        After writes through ``.data`` call :meth:`refresh_fused_weight`.  The key holds the weight's address, so
        the weight copied from is kept too: no other can come to lie there."""
        w = self.kv_up.weight
        key = _native.host().params_key([w])
        if self._up is not None and self._up[0] == key:
            return self._up[1], self._up[2]
        H, N, R = self.num_heads, self.head_dim, self.rank
        with torch.inference_mode(False), torch.no_grad():      # (normal tensors, which a later call may refill)
            per_head = w.detach().view(H, 2 * N, R)
            old = self._up
            if old is not None and old[1].dtype == w.dtype and old[1].device == w.device:
                wk, wv = old[1], old[2]
                wk.copy_(per_head[:, :N])
                wv.copy_(per_head[:, N:].transpose(1, 2))
            else:
                wk, wv = per_head[:, :N].clone(), per_head[:, N:].transpose(1, 2).clone(memory_format=torch.contiguous_format)
        self._up = (key, wk.detach(), wv.detach(), w.detach())
        return self._up[1], self._up[2]

    def refresh_fused_weight(self) -> None:
        """Make the absorbed form's copies again."""
        if self._up is not None:
            self._up = (None, *self._up[1:])
        if self._absorbs():
            self._up_weights()

    def _unmodified(self, method):
        """Whether the method is the one written here, not a subclass's, the instance's or a later replacement."""
        return getattr(type(self), method) is _METHODS[method] and method not in self.__dict__

    def _absorbs(self, x=None):
        """Whether ``kv_up`` is just the product with its weight, which the absorbed form splits."""
        return _plain_weight(self.kv_up, *(() if x is None else (x,))) is not None

    def _weight_buffers(self):
        """What a captured step reads beside the parameters."""
        return [w.data_ptr() for w in self._up_weights()] if self._absorbs() else []

    # ------------------------------------------------------------ the cache
    def new_state(self, B: int, device, dtype) -> dict:
        """An empty state for B sequences; of normal tensors under inference mode too, so that a later call
        outside it can go on with the state."""
        shape = (B, self.max_tokens, self.rank + self.position_dim)
        eight = self.cache_bits == 8
        with torch.inference_mode(False):
            return {"latent": torch.empty(shape, device=device, dtype=torch.float8_e4m3fn if eight else dtype),
                    "scale": torch.empty(B, self.max_tokens, 2, device=device) if eight else None,
                    "lengths": torch.zeros(B, dtype=torch.int32, device=device), "tokens": 0}

    def _room(self, state, T):
        held, most = state["tokens"], state["latent"].shape[1]
        if held + T > most:
            raise KdaError(f"the latent cache holds {held} of at most {most} tokens a sequence; {T} more do not fit")

    def _append(self, c, state):
        """Appends c, ``kv_down``'s output, whose type (x's, or autocast's) is the cache's."""
        mla_cache_append(c, state["latent"], state["lengths"], self.rank, cache_scale=state["scale"],
                         norm_weight=self.kv_norm, eps=self.eps)
        state["lengths"].add_(c.shape[1])

    # ------------------------------------------------------------ the two forms
    def _expanded(self, x, rows, lengths=None, starts=None):
        """Attention of x's queries over latent rows [B, S, rank + P], normalised already."""
        B, T, _ = x.shape
        H, N, R = self.num_heads, self.head_dim, self.rank
        kv = self.kv_up(rows[..., :R]).view(B, rows.shape[1], H, 2 * N)
        o = mla_expanded(self.q_proj(x).view(B, T, H, N + self.position_dim), kv[..., :N],
                         rows[..., R:] if self.position_dim else None, kv[..., N:], lengths=lengths, starts=starts,
                         scale=self.scale)
        return self.o_proj(o.reshape(B, T, H * N))

    def _norm(self, c):
        f = c.float()
        return (f * torch.rsqrt(f.square().mean(-1, keepdim=True) + self.eps) * self.kv_norm.float()).to(c.dtype)

    def _absorbed(self, x, state):
        B, T, _ = x.shape
        H, N, R = self.num_heads, self.head_dim, self.rank
        wk, wv = self._up_weights()
        q = self.q_proj(x).view(B * T, H, N + self.position_dim)
        qa = torch.bmm(q[..., :N].transpose(0, 1), wk).transpose(0, 1)               # [B T, H, R]
        q = torch.cat([qa, q[..., N:]], -1).view(B, T, H, R + self.position_dim)
        o = mla_absorbed(q, state["latent"], state["lengths"], R, self.scale, cache_scale=state["scale"])
        o = torch.bmm(o.view(B * T, H, R).transpose(0, 1), wv).transpose(0, 1)       # [B T, H, N]
        return self.o_proj(o.reshape(B, T, H * N))

    # ------------------------------------------------------------ public API
    def forward(self, x, state=None, use_cache=False):
        """x ``[B, T, d]`` -> ``[B, T, d]``, with ``use_cache`` (out, state)."""
        if torch.is_grad_enabled() and (x.requires_grad or any(p.requires_grad for p in self.parameters())):
            if use_cache or state is not None:
                raise KdaError("the training path takes no cache or state: run cached calls under torch.no_grad()")
            return self._whole(x)
        if not use_cache:
            if state is not None:
                raise KdaError("a state needs use_cache=True")
            return self._whole(x)
        T = x.shape[1]
        if state is not None:
            self._room(state, T)
            if T == 1 and state["tokens"] > 0:
                return self.decode_step_(x, state), state
        c = self.kv_down(x)
        if state is None:
            state = self.new_state(x.shape[0], x.device, c.dtype)
            self._room(state, T)
        self._append(c, state)
        state["tokens"] += T
        return self._expanded(x, self._held(state, state["tokens"], c.dtype)), state

    def _whole(self, x):
        c = self.kv_down(x)
        return self._expanded(x, torch.cat([self._norm(c[..., :self.rank]), c[..., self.rank:]], -1))

    def _held(self, state, n, dtype):
        """The cache's first n rows in 16 bits."""
        if self.cache_bits == 8:
            return mla_cache_read(state["latent"], state["scale"], self.rank, dtype=dtype, tokens=n)
        return state["latent"][:, :n]

    def _step(self, x, state, n=None):
        """One token, unchecked: the captured part of a decode step.  ``n``: the tokens held with it, by which the
        expanded form is cut to the rows that there are; a captured step, whose count moves, expands all of the
        cache and takes the count from the device."""
        c = self.kv_down(x)
        self._append(c, state)
        if self._absorbs(x):
            return self._absorbed(x, state)
        if n is not None:
            return self._expanded(x, self._held(state, n, c.dtype))
        rows = self._held(state, state["latent"].shape[1], c.dtype)
        return self._expanded(x, rows, lengths=state["lengths"], starts=state["lengths"] - 1)

    @torch.no_grad()
    def decode_step_(self, x, state):
        """One token x ``[B, 1, d]`` -> ``[B, 1, d]``; the state is updated in place."""
        if x.dim() != 3 or x.shape[1] != 1:
            raise KdaError(f"decode_step_ takes one token, got x of shape {tuple(x.shape)}")
        self._room(state, 1)
        out = self._step(x, state, state["tokens"] + 1)
        state["tokens"] += 1
        return out


_METHODS = {n: getattr(LatentAttention, n) for n in ("decode_step_",)}
