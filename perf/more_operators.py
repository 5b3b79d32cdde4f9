"""Decoding in 4 bits: the calls programs make of the 4-bit operators, with sizes.

Numbers are e2m1 values (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives), two a
byte, the lower half first, with a power of two for each group, stored as its
exponent plus 127.  The group's exponent is the smallest that leaves the
largest magnitude at most 7, so that quotients are exact and nothing but the
format's own rounding takes part.

* ``linear``: x W^T with W in groups of 32 along its rows, from one row of x (a
  decode step) to a prompt; with a residual added where a layer does;
* ``repack``: a weight quantised, and read back in 16 bits;
* ``absorbed``: latent attention over a cache whose rows hold 4 bits a channel
  and eight bytes of scales, one for each 128 latent channels and one for the
  position channels;
* ``step``: a decode step's new rows written into such a cache, RMS-normalised
  on the way, and the attention over it;
* ``requant``: rows written, and the cache read back in 16 bits, as the next
  piece of a long prompt reads what the pieces before it left.

``run`` computes them in plain torch where ``own`` is false and calls the
package where it is true; ``exact`` is the definition in float64.
"""

from __future__ import annotations

import functools

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
DEV = "cuda"
EPS = 1e-6
LEAST_WEIGHT, LEAST_CACHE = -126, -60            # the smallest exponents of the two kinds of groups


def listed():
    return [
        # a layer's output projection for one user's next token, with the residual stream
        linear("proj_token", 1, 2048, 2048, "bf16", residual=True),
        # the joined q, k and v projections of a serving batch
        linear("proj_batch", 16, 6144, 2048, "f16"),
        # one token through a wide projection: a read of the weight
        linear("wide_token", 1, 28672, 8192, "bf16"),
        # several sequences' tokens verified at once, an odd number of rows
        linear("proj_verify", 53, 6160, 4096, "f16"),
        # a prompt through the joined projections
        linear("proj_prompt", 4000, 6144, 2048, "bf16"),
        # a weight converted when a model is loaded, and checked against itself
        repack("repack", 8192, 8192, "bf16"),
        # one layer's small projection: launch latency
        repack("repack_small", 576, 2048, "f16"),
        # one user's next token in a long document
        absorbed("attend_long", "absorbed", 1, 1, 16, 65536, 512, 64, "f16"),
        # five tokens verified at once in a smaller model, an odd number of heads
        absorbed("attend_verify", "absorbed", 8, 5, 20, 1501, 256, 32, "f16"),
        # a serving batch's next token, contexts of all lengths and an idle slot
        absorbed("step_batch", "step", 64, 1, 16, 8192, 512, 64, "bf16", ragged=True),
        # prompts written and read back for their next piece
        cache("requant", 4, 2048, 8192, 512, 64, "bf16"),
        # one short prompt of a smaller model
        cache("requant_small", 1, 203, 512, 256, 32, "f16"),
    ]


def linear(name, M, N, K, dtype, residual=False, bias=False):
    return {"name": name, "kind": "linear", "M": M, "N": N, "K": K, "dtype": dtype, "residual": residual, "bias": bias}


def repack(name, N, K, dtype):
    return {"name": name, "kind": "repack", "N": N, "K": K, "dtype": dtype}


def absorbed(name, kind, B, T, H, S, R, P, dtype, ragged=False):
    return {"name": name, "kind": kind, "B": B, "T": T, "H": H, "S": S, "R": R, "P": P, "dtype": dtype, "ragged": ragged}


def cache(name, B, T, S, R, P, dtype):
    return {"name": name, "kind": "requant", "B": B, "T": T, "S": S, "R": R, "P": P, "dtype": dtype}


def _log_int(rng, lo, hi):
    """A whole number in [lo, hi], spread evenly over its logarithm."""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "linear", "repack", "absorbed", "absorbed", "step", "requant"])
    dtype = rng.choice(["f16", "bf16"])
    if kind == "linear":
        K, N = 32 * _log_int(rng, 1, 256), _log_int(rng, 16, 16384)
        M = min(_log_int(rng, 1, 4096), 4000 * 6144 * 2048 // (N * K))
        c = linear("", M, N, K, dtype, rng.random() < 0.3, rng.random() < 0.3)
    elif kind == "repack":
        c = repack("", _log_int(rng, 1, 8192), 32 * _log_int(rng, 1, 256), dtype)
    elif kind == "requant":
        R, P = rng.choice([(512, 64), (256, 32), (128, 64), (512, 0)])
        B, S = _log_int(rng, 1, 64), _log_int(rng, 16, 8192)
        S = min(S, 32768 // B)
        c = cache("", B, _log_int(rng, 1, S), S, R, P, dtype)
    else:
        R, P = rng.choice([(512, 64), (512, 64), (256, 32), (128, 64), (512, 0)])
        B = _log_int(rng, 1, 64)
        S = _log_int(rng, 1, min(65536, 64 * 4160 // B))
        T = min(S, 1 if rng.random() < 0.6 else rng.randint(2, 6))
        c = absorbed("", kind, B, T, rng.choice([4, 8, 16, 16, 20]), S, R, P, dtype, rng.random() < 0.5)
    del c["name"]
    return c


# ---- what a case fixes ------------------------------------------------------

def _lengths(c):
    """Tokens each sequence holds (after the call's own): all of S, or spread from S down, the last of four
    or more sequences an idle slot."""
    B, S = c["B"], c["S"]
    if not c["ragged"]:
        return [S] * B
    n = [S - b * S // B for b in range(B)]
    if B >= 4:
        n[-1] = 0
    return n


def _held(c):
    """Rows the cache holds before an append (below 0: the new rows are dropped)."""
    if c["kind"] == "step":
        return [n - c["T"] if n else -1 for n in _lengths(c)]
    return [(b * (c["S"] - c["T"])) // c["B"] for b in range(c["B"])]


def _visible(c):
    """(query, key) pairs of one head that the causal mask leaves."""
    T, pairs = c["T"], 0
    for n in _lengths(c):
        start = n - T
        lo = max(0, -start)
        if n > 0 and T > lo:
            pairs += (T - lo) * (start + 1) + (T * (T - 1) - lo * (lo - 1)) // 2
    return pairs


def work(c):
    if c["kind"] == "linear":
        M, N, K = c["M"], c["N"], c["K"]
        extra = (2 * M * N if c["residual"] else 0) + (2 * N if c["bias"] else 0)
        return {"bytes": N * K // 2 + N * K // 32 + 2 * M * (K + N) + extra, "flops": 2 * M * N * K}
    if c["kind"] == "repack":
        n = c["N"] * c["K"]
        return {"bytes": 2 * (2 * n + n // 2 + n // 32), "flops": 2 * n}
    B, T, R, P = c["B"], c["T"], c["R"], c["P"]
    row, new = (R + P) // 2 + 8, B * T * (2 * (R + P) + (R + P) // 2 + 8)
    if c["kind"] == "requant":
        return {"bytes": new + B * c["S"] * (row + 2 * (R + P)), "flops": B * T * (R + P) * 4}
    more = new if c["kind"] == "step" else 0
    return {"bytes": sum(_lengths(c)) * row + B * T * c["H"] * (2 * R + P) * 2 + more,
            "flops": _visible(c) * c["H"] * 2 * (2 * R + P)}


# ---- the format -------------------------------------------------------------

def _encode(x, group, least):
    """x [..., n] as bytes [..., n / 2] and the groups' exponents + 127, [..., n / group]; the type of x (fp32 or
    more) holds every step exactly."""
    g = x.unflatten(-1, (-1, group))
    top = g.abs().amax(-1)
    m, e = torch.frexp(top)
    e = torch.where(top > 0, e - 3 + (m > 0.875), least).clamp(least, 127)
    y = torch.ldexp(g, -e[..., None].to(g.dtype))
    a = y.abs()
    step = 0.5 + 0.5 * (a >= 2).to(a.dtype) + (a >= 4).to(a.dtype)
    a = (torch.round(a / step) * step).clamp(max=6)
    code = torch.where(a <= 2, 2 * a, torch.where(a <= 4, a + 2, 7.0)).to(torch.uint8) + 8 * (y < 0).to(torch.uint8)
    code = code.flatten(-2)
    return code[..., 0::2] + 16 * code[..., 1::2], (e + 127).to(torch.uint8)


def _decode(data, dtype):
    """The e2m1 values [..., n] of bytes [..., n / 2]."""
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=dtype, device=data.device)
    table = torch.cat([table, -table])
    return table[torch.stack([data & 15, data >> 4], -1).flatten(-2).int()]


def _powers(e, dtype):
    return torch.ldexp(torch.ones((), dtype=dtype, device=e.device), e.to(dtype) - 127)


def _weight(data, e, dtype):
    return (_decode(data, dtype).unflatten(-1, (-1, 32)) * _powers(e, dtype)[..., None]).flatten(-2)


def _encode_rows(x, R):
    """Cache rows x [..., R + P]: bytes, and the eight bytes of scales (those without a group: 2^0)."""
    lat, e = _encode(x[..., :R], 128, LEAST_CACHE)
    scales = torch.full((*x.shape[:-1], 8), 127, dtype=torch.uint8, device=x.device)
    scales[..., : R // 128] = e
    if x.shape[-1] == R:
        return lat, scales
    pos, e = _encode(x[..., R:], x.shape[-1] - R, LEAST_CACHE)
    scales[..., R // 128] = e[..., 0]
    return torch.cat([lat, pos], -1), scales


def _rows(data, scales, R, dtype):
    """Cache rows [..., R + P] of their bytes and scales."""
    D = 2 * data.shape[-1]
    s = _powers(scales[..., : R // 128 + 1], dtype)
    s = torch.cat([s[..., :-1].repeat_interleave(128, -1), s[..., -1:].expand(*s.shape[:-1], D - R)], -1)
    return _decode(data, dtype) * s


# ---- inputs -----------------------------------------------------------------

def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def prepare(c, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = DTYPES[c["dtype"]]

    def rand(*shape, std=1.0):
        return torch.randn(*shape, device=DEV, generator=g) * std

    s = {"case": c}
    if c["kind"] in ("linear", "repack"):
        N, K = c["N"], c["K"]
        # weights of a trained layer: rows of different size, most entries near zero
        w = rand(N, K, std=K ** -0.5) * torch.exp2(rand(N, 1, std=0.7))
        if c["kind"] == "repack":
            return {**s, "w": w.to(dt)}
        data, e = _encode(w, 32, LEAST_WEIGHT)
        s.update(weight=data.view(torch.float4_e2m1fn_x2), scale=e.view(torch.float8_e8m0fnu),
                 # activations: some channels much larger than the others
                 x=(rand(1, c["M"], K) * torch.exp2(rand(K, std=1.0))).to(dt),
                 bias=rand(N).to(dt) if c["bias"] else None,
                 residual=rand(1, c["M"], N, std=4.0).to(dt) if c["residual"] else None)
        return s
    B, T, S, R, P = c["B"], c["T"], c["S"], c["R"], c["P"]
    data, e = _encode_rows(rand(B, S, R + P), R)
    s.update(cache=data.view(torch.float4_e2m1fn_x2), cache_scale=e.view(torch.float8_e8m0fnu))
    if c["kind"] != "absorbed":
        s.update(x=rand(B, T, R + P, std=1.7).to(dt), weight=(1 + rand(R, std=0.1)).to(dt), held=_int32(_held(c)))
    if c["kind"] != "requant":
        s.update(q=rand(B, T, c["H"], R + P, std=2.0 * R ** -0.5 * 128 ** 0.5).to(dt), lengths=_int32(_lengths(c)),
                 scale=(128 + P) ** -0.5)
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
    kind = c["kind"]
    if kind == "linear":
        return kda.mx4_linear(s["x"], s["weight"], s["scale"], bias=s["bias"], residual=s["residual"])
    if kind == "repack":
        return kda.mx4_dequantize(*kda.mx4_quantize(s["w"]), dtype=s["w"].dtype)
    if kind != "absorbed":
        kda.mla_cache_append(s["x"], s["cache"], s["held"], c["R"], cache_scale=s["cache_scale"],
                             norm_weight=s["weight"], eps=EPS)
    if kind == "requant":
        return kda.mla_cache_read(s["cache"], s["cache_scale"], c["R"], dtype=s["x"].dtype)
    return kda.mla_absorbed(s["q"], s["cache"], s["lengths"], c["R"], s["scale"], cache_scale=s["cache_scale"])


@torch.no_grad()
def _plain(s):
    c, f = s["case"], torch.float32
    kind = c["kind"]
    if kind == "linear":
        w = _weight(s["weight"].view(torch.uint8), s["scale"].view(torch.uint8), f)
        y = torch.matmul(s["x"].to(f), w.T)
        if s["bias"] is not None:
            y = y + s["bias"].to(f)
        y = y.to(s["x"].dtype)
        return y if s["residual"] is None else (s["residual"].to(f) + y.to(f)).to(y.dtype)
    if kind == "repack":
        return _weight(*_encode(s["w"].to(f), 32, LEAST_WEIGHT), f).to(s["w"].dtype)
    data, scales, R = s["cache"].view(torch.uint8), s["cache_scale"].view(torch.uint8), c["R"]
    if kind != "absorbed":
        x = s["x"].to(f)
        # (the mean in 64 bits: a value next to a border of the format should not go by the order of a sum)
        rstd = torch.rsqrt(s["x"][..., :R].double().square().mean(-1, keepdim=True) + EPS).to(f)
        new, e = _encode_rows(torch.cat([x[..., :R] * rstd * s["weight"].to(f), x[..., R:]], -1), R)
        at = s["held"][:, None] + torch.arange(c["T"], device=DEV)
        b, t = torch.nonzero((s["held"][:, None] >= 0) & (at < c["S"]), as_tuple=True)
        at = at[b, t].long()
        data[b, at], scales[b, at] = new[b, t], e[b, t]
    rows = _rows(data, scales, R, f)
    if kind == "requant":
        return rows.to(s["x"].dtype)
    scores = torch.matmul(s["q"].to(f).flatten(1, 2), rows.transpose(1, 2)) * s["scale"]       # [B, T H, S]
    n = s["lengths"][:, None]
    pos = n - c["T"] + torch.arange(c["T"], device=DEV)
    mask = torch.arange(c["S"], device=DEV) <= pos[..., None]
    scores = scores.masked_fill(~mask.repeat_interleave(c["H"], 1), -torch.inf)
    e = torch.exp(scores - scores.amax(-1, keepdim=True).nan_to_num(neginf=0.0))
    p = e / e.sum(-1, keepdim=True).clamp_min(torch.finfo(f).tiny)
    return torch.matmul(p, rows[..., :R]).to(s["q"].dtype).unflatten(1, (c["T"], c["H"]))


# ---- the definition in 64 bits ----------------------------------------------

_VALUES = [0, 0.5, 1, 1.5, 2, 3, 4, 6]


def _nearest(x, group, least):
    """x (float64) [n, k] to the nearest value 2^e v of its group, e the smallest power that leaves at most 7."""
    v = torch.tensor(_VALUES, dtype=torch.float64, device=x.device)
    borders = (v[1:] + v[:-1]) / 2
    y = x.reshape(x.shape[0], -1, group)
    top = y.abs().amax(2, keepdim=True)
    unit = torch.exp2(torch.ceil(torch.log2(top / 7)).clamp_min(least))
    unit = torch.where(top > 7 * unit, 2 * unit, torch.where((top <= 3.5 * unit) & (unit > 2.0 ** least), unit / 2, unit))
    a = (y / unit).abs().contiguous()
    up, down = torch.bucketize(a, borders, right=True), torch.bucketize(a, borders, right=False)
    code = torch.where(up == down, up, torch.where(up % 2 == 0, up, down))       # between two: the even one
    return (torch.sign(y) * v[code] * unit).reshape(x.shape)


def _values(data, scales, groups):
    """Stored bytes [n, k / 2] and scales as float64 [n, k]; groups: the channels of each scale."""
    v = torch.tensor(_VALUES + [-x for x in _VALUES], dtype=torch.float64, device=data.device)
    out = torch.empty(data.shape[0], 2 * data.shape[1], dtype=torch.float64, device=data.device)
    out[:, 0::2], out[:, 1::2] = v[(data % 16).int()], v[(data // 16).int()]
    at = 0
    for i, n in enumerate(groups):
        out[:, at:at + n] *= torch.exp2(scales[:, i:i + 1].double() - 127)
        at += n
    return out


@torch.no_grad()
def exact(c, seed):
    s = prepare(c, seed)
    if c["kind"] == "linear":
        data, e = s["weight"].view(torch.uint8), s["scale"].view(torch.uint8)
        y = torch.empty(1, c["M"], c["N"], dtype=torch.float64, device=DEV)
        for n in range(0, c["N"], 4096):
            w = _values(data[n:n + 4096], e[n:n + 4096], [32] * (c["K"] // 32))
            y[0, :, n:n + 4096] = s["x"][0].double() @ w.T
        for name in ("bias", "residual"):
            if s[name] is not None:
                y += s[name].double()
        return y
    if c["kind"] == "repack":
        return _nearest(s["w"].double(), 32, LEAST_WEIGHT)
    B, R, P, T = c["B"], c["R"], c["P"], c["T"]
    groups = [128] * (R // 128) + [P]
    new = None
    if c["kind"] != "absorbed":
        x = s["x"].double().flatten(0, 1)
        lat = x[:, :R] / torch.sqrt((x[:, :R] ** 2).mean(1, keepdim=True) + EPS) * s["weight"].double()
        new = [_nearest(lat, 128, LEAST_CACHE)] + ([_nearest(x[:, R:], P, LEAST_CACHE)] if P else [])
        new = torch.cat(new, 1).view(B, T, R + P)
    back = torch.empty(B, c["S"], R + P, dtype=torch.float64, device=DEV) if c["kind"] == "requant" else None
    o = None if back is not None else torch.zeros(B, T, c["H"], R, dtype=torch.float64, device=DEV)
    for b in range(B):
        rows = _values(s["cache"][b].view(torch.uint8), s["cache_scale"][b].view(torch.uint8), groups)
        if new is not None and _held(c)[b] >= 0:
            at = _held(c)[b]
            n = min(T, c["S"] - at)
            rows[at:at + n] = new[b, :n]
        if back is not None:
            back[b] = rows
            continue
        for t in range(T):
            seen = _lengths(c)[b] - T + t + 1
            if seen > 0:
                w = torch.softmax(s["q"][b, t].double() @ rows[:seen].T * s["scale"], -1)
                o[b, t] = w @ rows[:seen, :R]
    return o if back is None else back
