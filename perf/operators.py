"""Latent attention and its cache: the calls programs make of them, with sizes.

A token's keys and values come from one latent vector c (``rank`` channels) and
a few position channels p that all heads share.  Four operators:

* ``expanded``: attention over keys and values already expanded per head, a
  key being its head's own channels and the shared position channels; causal,
  the first query at position ``start``, a sequence's tokens ending at its
  length; ``expanded_train`` adds the gradients of q, k_nope, k_pe and v;
* ``absorbed``: attention in the latent space over the cache itself, whose
  rows are key and (their first ``rank`` channels) value of every head, in 16
  bits or in 8 bits with two scales a token;
* ``append``: new rows written into the cache behind each sequence, the latent
  part RMS-normalised on the way, quantised where the cache holds 8 bits;
* ``requant``: rows written into an 8-bit cache, and the cache read back in 16
  bits, as the next piece of a long prompt reads what the pieces before it left.

``run`` computes them in plain torch where ``own`` is false and calls the
package where it is true; ``exact`` is the definition in float64.
"""

from __future__ import annotations

import functools

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
DEV = "cuda"
F8 = torch.float8_e4m3fn
EPS = 1e-6


def listed():
    return [
        # one user's next token, a short context: launch latency
        absorbed("decode_one", 1, 1, 16, 200, 512, 64, "bf16"),
        # a serving batch's next token, contexts of all lengths and an idle slot
        absorbed("decode_batch", 64, 1, 16, 4096, 512, 64, "bf16", ragged=True),
        # one user's next token in a long document
        absorbed("decode_long", 1, 1, 16, 32768, 512, 64, "f16"),
        # a serving batch over a cache in 8 bits
        absorbed("decode_8bit", 64, 1, 16, 8192, 512, 64, "bf16", bits=8, ragged=True),
        # five tokens verified at once in a smaller model, an odd number of heads
        absorbed("verify", 8, 5, 20, 1501, 256, 32, "f16"),
        # one prompt of any length
        expanded("prompt", "expanded", 1, 1000, 0, 16, 128, 64, "f16"),
        # a piece of a long prompt over what the cache holds already
        expanded("prompt_piece", "expanded", 1, 2048, 14336, 16, 128, 64, "bf16"),
        # a training step of one layer's attention
        expanded("train", "expanded_train", 4, 2048, 0, 16, 128, 64, "bf16"),
        # a small model's padded batch in training
        expanded("train_small", "expanded_train", 4, 203, 0, 8, 64, 32, "f16", ragged=True),
        # a serving batch's next token written into a cache in 8 bits
        cache("append", "append", 64, 1, 1024, 512, 64, "bf16", bits=8),
        # prompts written into a cache in 16 bits, ragged
        cache("append_prompt", "append", 4, 2000, 4096, 512, 64, "f16", bits=16),
        # prompts written in 8 bits and read back for the next piece
        cache("requant", "requant", 4, 2048, 8192, 512, 64, "bf16", bits=8),
    ]


def absorbed(name, B, T, H, S, R, P, dtype, bits=16, ragged=False):
    return {"name": name, "kind": "absorbed", "B": B, "T": T, "H": H, "S": S, "R": R, "P": P, "dtype": dtype,
            "bits": bits, "ragged": ragged}


def expanded(name, kind, B, T, prefix, H, N, P, dtype, ragged=False):
    return {"name": name, "kind": kind, "B": B, "T": T, "S": T + prefix, "H": H, "N": N, "P": P, "V": N,
            "dtype": dtype, "ragged": ragged}


def cache(name, kind, B, T, S, R, P, dtype, bits):
    return {"name": name, "kind": kind, "B": B, "T": T, "S": S, "R": R, "P": P, "dtype": dtype, "bits": bits}


def _log_int(rng, lo, hi):
    """A whole number in [lo, hi], spread evenly over its logarithm."""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(["absorbed", "absorbed", "absorbed8", "expanded", "expanded_train", "append", "requant"])
    dtype = rng.choice(["f16", "bf16"])
    if kind.startswith("absorbed"):
        R, P = rng.choice([(512, 64), (512, 64), (256, 32), (128, 64), (512, 0)])
        B = _log_int(rng, 1, 64)
        S = _log_int(rng, 1, min(32768, 2 * 64 * 4096 // B))
        T = 1 if rng.random() < 0.6 else rng.randint(2, 6)
        T = min(T, S)
        c = absorbed("", B, T, rng.choice([4, 8, 16, 16, 20]), S, R, P, dtype, 8 if kind.endswith("8") else 16,
                     rng.random() < 0.5)
    elif kind.startswith("expanded"):
        N, P = rng.choice([(128, 64), (128, 64), (64, 32), (64, 64), (128, 0)])
        B, H = _log_int(rng, 1, 4), rng.choice([3, 8, 16])
        T = _log_int(rng, 1, 2048)
        prefix = 0 if kind == "expanded_train" or rng.random() < 0.5 else _log_int(rng, 1, 8192 // B)
        c = expanded("", kind, B, T, prefix, H, N, P, dtype, rng.random() < 0.5)
    else:
        R, P = rng.choice([(512, 64), (256, 32), (128, 64), (512, 0)])
        B, S = _log_int(rng, 1, 64), _log_int(rng, 16, 8192)
        S = min(S, 65536 // B)
        c = cache("", kind, B, _log_int(rng, 1, S), S, R, P, dtype, 8 if kind == "requant" else rng.choice([8, 16]))
    del c["name"]
    return c


# ---- what a case fixes ------------------------------------------------------

def _lengths(c):
    """Tokens each sequence holds (after the call's own): all of S, or spread from S down, the last of four
    or more sequences an idle slot."""
    B, S = c["B"], c["S"]
    if not c.get("ragged"):
        return [S] * B
    n = [S - b * S // B for b in range(B)]
    if B >= 4:
        n[-1] = 0
    return n


def _held(c):
    """Rows the cache holds before an append, and how many of the T new rows each sequence brings."""
    B, T, S = c["B"], c["T"], c["S"]
    held = [(b * (S - T)) // B for b in range(B)]
    if c["kind"] == "append" and T > 1:
        return held, [T - b * T // (2 * B) for b in range(B)]
    return held, [T] * B


def _visible(c):
    """(query, key) pairs of one head that the causal mask leaves, and query rows that exist."""
    T, S = c["T"], c["S"]
    pairs = 0
    for n in _lengths(c):
        start = n - T if c["kind"] == "absorbed" else S - T
        lo, hi = max(0, -start), min(T, n - start)        # queries whose position is in [0, n)
        if hi > lo:
            pairs += (hi - lo) * (start + 1) + (hi * (hi - 1) - lo * (lo - 1)) // 2
    return pairs


def work(c):
    B, T, S = c["B"], c["T"], c["S"]
    if c["kind"] == "absorbed":
        H, R, P = c["H"], c["R"], c["P"]
        row = (R + P) * c["bits"] // 8 + (8 if c["bits"] == 8 else 0)
        return {"bytes": sum(_lengths(c)) * row + B * T * H * (2 * R + P) * 2, "flops": _visible(c) * H * 2 * (2 * R + P)}
    if c["kind"].startswith("expanded"):
        H, D, P, V = c["H"], c["N"] + c["P"], c["P"], c["V"]
        q, k, pe, v = B * T * H * D * 2, B * S * H * c["N"] * 2, B * S * P * 2, B * S * H * V * 2
        o = B * T * H * V * 2
        if c["kind"] == "expanded":
            return {"bytes": q + k + pe + v + o, "flops": _visible(c) * H * 2 * (D + V)}
        return {"bytes": 2 * (q + k + pe + v) + 2 * o, "flops": _visible(c) * H * 2 * (4 * D + 3 * V)}
    D = c["R"] + c["P"]
    row = D * c["bits"] // 8 + (8 if c["bits"] == 8 else 0)
    rows = sum(_held(c)[1])
    back = 0 if c["kind"] == "append" else B * S * (row + D * 2)
    return {"bytes": rows * (D * 2 + row) + back, "flops": rows * D * 4}


# ---- inputs -----------------------------------------------------------------

def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _quantise(x, R):
    """x [..., R + P] fp32 as e4m3 with two scales a row: amax / 448 of its latent and of its position part."""
    parts, scales = [], []
    for part in (x[..., :R], x[..., R:]):
        if part.shape[-1] == 0:
            scales.append(torch.ones_like(x[..., :1]))
            parts.append(part.to(F8))
            continue
        s = part.abs().amax(-1, keepdim=True).clamp_min(448 * 2.0 ** -60) / 448
        parts.append((part / s).clamp(-448, 448).to(F8))
        scales.append(s)
    return torch.cat([p.view(torch.uint8) for p in parts], -1).view(F8), torch.cat(scales, -1)


def _dequantise(data, scales, R):
    s = torch.cat([scales[..., :1].expand(*data.shape[:-1], R),
                   scales[..., 1:].expand(*data.shape[:-1], data.shape[-1] - R)], -1)
    return data.to(torch.float32) * s


def prepare(c, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = DTYPES[c["dtype"]]
    B, T, S = c["B"], c["T"], c["S"]

    def rand(*shape, std=1.0):
        return torch.randn(*shape, device=DEV, generator=g) * std

    s = {"case": c}
    if c["kind"].startswith("expanded"):
        H, N, P, V = c["H"], c["N"], c["P"], c["V"]
        # one product of the latents gives a head's keys and values side by side
        kv = rand(B, S, H, N + V).to(dt)
        s.update(q=rand(B, T, H, N + P).to(dt), k_nope=kv[..., :N], v=kv[..., N:],
                 k_pe=rand(B, S, P).to(dt) if P else None,
                 lengths=_int32(_lengths(c)) if c["ragged"] else None, scale=(N + P) ** -0.5)
        if c["kind"] == "expanded_train":
            s["do"] = rand(B, T, H, V).to(dt)
            for n in ("q", "k_nope", "v", "k_pe"):
                if s[n] is not None:
                    s[n] = s[n].detach().requires_grad_()
    elif c["kind"] == "absorbed":
        H, R, P = c["H"], c["R"], c["P"]
        rows = rand(B, S, R + P)
        s.update(q=rand(B, T, H, R + P, std=2.0 * R ** -0.5 * 128 ** 0.5).to(dt), lengths=_int32(_lengths(c)),
                 scale=(128 + P) ** -0.5)
        s["cache"], s["cache_scale"] = _quantise(rows, R) if c["bits"] == 8 else (rows.to(dt), None)
    else:
        R, P = c["R"], c["P"]
        held, counts = _held(c)
        rows = rand(B, S, R + P)
        s.update(x=rand(B, T, R + P, std=1.7).to(dt), weight=(1 + rand(R, std=0.1)).to(dt), lengths=_int32(held),
                 counts=_int32(counts))
        s["cache"], s["cache_scale"] = _quantise(rows, R) if c["bits"] == 8 else (rows.to(dt), None)
    return s


# ---- one pass ---------------------------------------------------------------

def run(s):
    return _own(s) if own else _plain(s)


@functools.cache
def _package():
    from __graft_entry__ import load_package
    return load_package()


def _own(s):
    kda, c = _package(), s["case"]
    if c["kind"].startswith("expanded"):
        o = kda.mla_expanded(s["q"], s["k_nope"], s["k_pe"], s["v"], lengths=s["lengths"], scale=s["scale"])
        if c["kind"] == "expanded":
            return o
        wrt = [s[n] for n in ("q", "k_nope", "v", "k_pe") if s[n] is not None]
        return [o.detach(), *torch.autograd.grad(o, wrt, s["do"])]
    if c["kind"] == "absorbed":
        return kda.mla_absorbed(s["q"], s["cache"], s["lengths"], c["R"], s["scale"], cache_scale=s["cache_scale"])
    kda.mla_cache_append(s["x"], s["cache"], s["lengths"], c["R"], cache_scale=s["cache_scale"],
                         counts=s["counts"], norm_weight=s["weight"], eps=EPS)
    if c["kind"] == "requant":
        return kda.mla_cache_read(s["cache"], s["cache_scale"], c["R"], dtype=s["x"].dtype)
    return [s["cache"]] + ([s["cache_scale"]] if c["bits"] == 8 else [])


def _mask(c, T, S, dev):
    """[B, T, S] truth values: the keys each query sees."""
    n = torch.tensor(_lengths(c), device=dev)[:, None]
    start = n - T if c["kind"] == "absorbed" else torch.full_like(n, S - T)
    pos = start + torch.arange(T, device=dev)
    j = torch.arange(S, device=dev)
    return (j <= pos[..., None]) & (j < n[..., None]) & (pos < n)[..., None]


def _softmax(scores, mask):
    """exp(s - max) / sum over the keys that the mask leaves; zeros in a row it leaves none."""
    scores = scores.masked_fill(~mask, -torch.inf)
    top = scores.amax(-1, keepdim=True).nan_to_num(neginf=0.0)
    e = torch.exp(scores - top)
    return e / e.sum(-1, keepdim=True).clamp_min(torch.finfo(e.dtype).tiny)


@torch.no_grad()
def _plain(s):
    c = s["case"]
    f = torch.float32
    if c["kind"].startswith("expanded"):
        return _attend(c, s, f)
    if c["kind"] == "absorbed":
        rows = s["cache"].to(f) if c["bits"] == 16 else _dequantise(s["cache"], s["cache_scale"], c["R"])
        scores = torch.matmul(s["q"].to(f).flatten(1, 2), rows.transpose(1, 2)) * s["scale"]       # [B, T H, S]
        mask = _mask(c, c["T"], c["S"], DEV).repeat_interleave(c["H"], 1)
        o = torch.matmul(_softmax(scores, mask), rows[..., : c["R"]])
        return o.to(s["q"].dtype).unflatten(1, (c["T"], c["H"]))
    R, T, dt = c["R"], c["T"], s["x"].dtype
    x = s["x"].to(f)
    lat = x[..., :R] * torch.rsqrt(x[..., :R].square().mean(-1, keepdim=True) + EPS) * s["weight"].to(f)
    x = torch.cat([lat, x[..., R:]], -1)
    t = torch.arange(T, device=DEV)
    at = s["lengths"][:, None] + t                                    # [B, T]
    b, t = torch.nonzero((t < s["counts"][:, None]) & (at < c["S"]), as_tuple=True)
    at = at[b, t].long()
    if c["bits"] == 16:
        s["cache"][b, at] = x[b, t].to(dt)
        return [s["cache"]]
    data, scales = _quantise(x, R)
    s["cache"].view(torch.uint8)[b, at] = data.view(torch.uint8)[b, t]
    s["cache_scale"][b, at] = scales[b, t]
    if c["kind"] == "requant":
        return _dequantise(s["cache"], s["cache_scale"], R).to(dt)
    return [s["cache"], s["cache_scale"]]


def _attend(c, s, f):
    """The expanded form and, in training, its gradients, in the type f."""
    T, S = c["T"], c["S"]

    def heads(x):
        return x.detach().to(f).transpose(1, 2)                       # [B, H, tokens, channels]

    q, v = heads(s["q"]), heads(s["v"])
    k = heads(s["k_nope"])
    if c["P"]:
        k = torch.cat([k, s["k_pe"].detach().to(f)[:, None].expand(-1, c["H"], -1, -1)], -1)
    mask = _mask(c, T, S, q.device)[:, None]
    p = _softmax(torch.matmul(q, k.transpose(2, 3)) * s["scale"], mask)
    o = torch.matmul(p, v)

    def out(x):
        return x.transpose(1, 2).to(s["q"].dtype if f == torch.float32 else f)

    if c["kind"] == "expanded":
        return out(o)
    do = heads(s["do"])
    dv = torch.matmul(p.transpose(2, 3), do)
    dp = torch.matmul(do, v.transpose(2, 3))
    ds = p * (dp - (do * o).sum(-1, keepdim=True)) * s["scale"]
    dq, dk = torch.matmul(ds, k), torch.matmul(ds.transpose(2, 3), q)
    got = [out(o), out(dq), out(dk[..., : c["N"]]), out(dv)]
    if c["P"]:
        got.append(out(dk[..., c["N"]:].sum(1, keepdim=True)).squeeze(2))
    return got


# ---- the definition in 64 bits ----------------------------------------------

def _e4m3(x):
    """x (float64) to the nearest e4m3 value, ties to the even one: steps of 2^-3 of the leading bit, of 2^-9
    below 2^-6, at most 448."""
    exp = torch.frexp(x).exponent.to(torch.float64) - 1
    step = torch.exp2(exp.clamp_min(-6.0) - 3)
    return (torch.round(x / step) * step).clamp(-448, 448)


@torch.no_grad()
def exact(c, seed):
    s = prepare(c, seed)
    d = torch.float64
    if c["kind"].startswith("expanded"):
        return _exact_expanded(c, s)
    lengths = _lengths(c)
    if c["kind"] == "absorbed":
        R, T = c["R"], c["T"]
        o = torch.zeros(c["B"], T, c["H"], R, device=DEV, dtype=d)
        for b, n in enumerate(lengths):
            if n == 0:
                continue
            rows = s["cache"][b, :n].to(d)
            if c["bits"] == 8:
                rows[:, :R] *= s["cache_scale"][b, :n, :1].to(d)
                rows[:, R:] *= s["cache_scale"][b, :n, 1:].to(d)
            for t in range(T):
                seen = n - T + t + 1
                if seen > 0:
                    w = torch.softmax(s["q"][b, t].to(d) @ rows[:seen].T * s["scale"], -1)
                    o[b, t] = w @ rows[:seen, :R]
        return o
    R, S = c["R"], c["S"]
    held, counts = _held(c)
    data, scales = s["cache"].to(d), None if c["bits"] == 16 else s["cache_scale"].to(d)
    for b, (at, n) in enumerate(zip(held, counts)):
        n = min(n, S - at)
        x = s["x"][b, :n].to(d)
        x[:, :R] /= torch.sqrt((x[:, :R] ** 2).mean(1, keepdim=True) + EPS)
        x[:, :R] *= s["weight"].to(d)
        if c["bits"] == 8:
            for i, (lo, hi) in enumerate(((0, R), (R, R + c["P"]))):
                if hi > lo:
                    scales[b, at:at + n, i] = x[:, lo:hi].abs().amax(1).clamp_min(448 * 2.0 ** -60) / 448
                    x[:, lo:hi] = _e4m3(x[:, lo:hi] / scales[b, at:at + n, i, None])
                else:
                    scales[b, at:at + n, i] = 1
        data[b, at:at + n] = x
    if c["kind"] == "requant":
        data[..., :R] *= scales[..., :1]
        data[..., R:] *= scales[..., 1:]
        return data
    return [data] + ([scales] if c["bits"] == 8 else [])


def _exact_expanded(c, s):
    """One head at a time, by softmax and autograd in float64."""
    T, S, H, N = c["T"], c["S"], c["H"], c["N"]
    names = [n for n in ("q", "k_nope", "v", "k_pe") if s[n] is not None]
    train = c["kind"] == "expanded_train"
    o = torch.zeros(c["B"], T, H, c["V"], device=DEV, dtype=torch.float64)
    grads = {n: torch.zeros(s[n].shape, device=DEV, dtype=torch.float64) for n in names}
    for b, n in enumerate(_lengths(c)):
        n_q = min(T, n - (S - T))             # queries that exist, at positions S - T on
        if n_q <= 0:
            continue
        hidden = torch.ones(n_q, n, device=DEV, dtype=torch.bool).triu(S - T + 1)
        for h in range(H):
            x = {"q": s["q"][b, :n_q, h], "k_nope": s["k_nope"][b, :n, h], "v": s["v"][b, :n, h]}
            if "k_pe" in names:
                x["k_pe"] = s["k_pe"][b, :n]
            x = {m: t.detach().double().requires_grad_(train) for m, t in x.items()}
            with torch.set_grad_enabled(train):
                a = x["q"][:, :N] @ x["k_nope"].T
                if "k_pe" in names:
                    a = a + x["q"][:, N:] @ x["k_pe"].T
                y = torch.softmax((a * s["scale"]).masked_fill(hidden, -torch.inf), 1) @ x["v"]
            o[b, :n_q, h] = y.detach()
            if train:
                got = torch.autograd.grad(y, [x[m] for m in names], s["do"][b, :n_q, h].double())
                for m, t in zip(names, got):
                    if m == "k_pe":
                        grads[m][b, :n] += t
                    else:
                        grads[m][b, : t.shape[0], h] += t
    return [o, *(grads[m] for m in names)] if train else o
