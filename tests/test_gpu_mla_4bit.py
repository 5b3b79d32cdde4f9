"""Latent attention over a cache in 4 bits, against its formulas in float64.

The attention's bounds are those of the other widths (``test_gpu_mla``): the
cache's values are exact in both activation types and their powers enter in
fp32, so a score has the roundings of one over a 16-bit cache, and a weight one
rounding to the type.  What is written has one answer, and is compared bit by bit.
"""

from __future__ import annotations

import pytest
import torch
from test_gpu_mla import ABSORBED, BF16, CACHE, F16, SHARED, absorbed_ref, close, half_step, i32, rand
from test_gpu_mla import dequantised as dequantised8, quantised as quantised8
from test_gpu_mx4 import definition, raw

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
FOUR, E8M0 = torch.float4_e2m1fn_x2, torch.float8_e8m0fnu
VALUES = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def quantised(x, R):
    """Rows [.., R + P] as the cache holds them, by the definition."""
    parts, scales = [], torch.full((*x.shape[:-1], 8), 127, dtype=torch.uint8, device=x.device)
    for lo, hi, n in ((0, R, 128), (R, x.shape[-1], x.shape[-1] - R)):
        if hi > lo:
            code, e = definition(x[..., lo:hi], n, -60)
            parts.append(code)
            scales[..., lo // 128:lo // 128 + (hi - lo) // n] = e.to(torch.uint8)
    code = torch.cat(parts, -1)
    return (code[..., 0::2] + 16 * code[..., 1::2]).to(torch.uint8).view(FOUR), scales.view(E8M0)


def dequantised(cache, scale, R):
    data, e = raw(cache), raw(scale).double()
    v = torch.tensor(VALUES + [-x for x in VALUES], dtype=torch.float64, device=data.device)
    v = v[torch.stack([data % 16, data // 16], -1).flatten(-2).long()]
    p = torch.where(e == 255, torch.nan, torch.exp2(e - 127))
    P = v.shape[-1] - R
    return v * torch.cat([p[..., :R // 128].repeat_interleave(128, -1), p[..., R // 128:R // 128 + 1].expand(*p.shape[:-1], P)], -1)


def poison(cache, scale, lengths):
    """Unwritten memory: any bytes, and scales that are NaN."""
    for b, n in enumerate(lengths):
        raw(cache)[b, max(n, 0):] = 0x7f
        raw(scale)[b, max(n, 0):] = 0xff


@pytest.mark.parametrize("case", ABSORBED + SHARED, ids=lambda c: "-".join(map(str, c[:6])) + "-" + str(c[6])[6:])
def test_absorbed(kda_pkg, case):
    B, T, H, S, R, P, dtype, lengths = case
    q = rand(B, T, H, R + P, seed=1, dtype=dtype, std=R ** -0.5 * 12)
    rows = rand(B, S, R + P, seed=2, dtype=torch.float32)
    rows[..., R:] *= 3
    cache, scale = quantised(rows, R)
    held = dequantised(cache, scale, R)
    poison(cache, scale, lengths)
    got = kda_pkg.mla_absorbed(q, cache, i32(lengths), R, (128 + P) ** -0.5, cache_scale=scale)
    want, bound = absorbed_ref(q, held, lengths, R, (128 + P) ** -0.5)
    close("o", got, want, bound)
    assert torch.equal(got, kda_pkg.mla_absorbed(q, cache, i32(lengths), R, (128 + P) ** -0.5, cache_scale=scale))


@pytest.mark.parametrize("R,P", [(128, 0), (128, 32), (128, 64), (256, 0), (256, 32), (256, 64), (512, 0), (512, 32), (512, 64)])
@pytest.mark.parametrize("S", [1, 15, 17, 64, 65, 130])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_absorbed_every_width(kda_pkg, R, P, S, dtype):
    """All widths at lengths around a unit and a window; one head, and heads that fill two row tiles in part."""
    for H, T in ((1, 1), (19, 1), (3, 2)):
        q = rand(2, T, H, R + P, seed=3, dtype=dtype, std=R ** -0.5 * 12)
        cache, scale = quantised(rand(2, S, R + P, seed=4, dtype=torch.float32), R)
        lengths = [S, S // 2]
        held = dequantised(cache, scale, R)
        poison(cache, scale, lengths)
        got = kda_pkg.mla_absorbed(q, cache, i32(lengths), R, 0.09, cache_scale=scale)
        close("o", got, *absorbed_ref(q, held, lengths, R, 0.09))


@pytest.mark.parametrize("S", [300, 3000])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("R,P", [(128, 32), (256, 64), (512, 64)])
def test_absorbed_scales_of_any_size(kda_pkg, R, P, S, dtype):
    """Powers that differ from token to token and from group to group, rows of zeros among them: every group's
    channels keep their precision, whatever the others' size."""
    rows = rand(1, S, R + P, seed=5, dtype=torch.float32) * torch.logspace(-5, 1, S, device=DEV)[None, :, None]
    rows[:, ::7] = 0
    for g in range(R // 128):
        rows[..., 128 * g:128 * g + 128] *= 2.0 ** (-9 * g)
    rows[:, ::5, :128] = 0
    rows[:, 1::5, R:] = 0
    q = rand(1, 1, 16, R + P, seed=6, dtype=dtype, std=0.5)
    for x in (rows, rows * 2.0 ** -13):
        cache, scale = quantised(x, R)
        got = kda_pkg.mla_absorbed(q, cache, i32([S]), R, 0.1, cache_scale=scale)
        want, bound = absorbed_ref(q, dequantised(cache, scale, R), [S], R, 0.1)
        close("o", got, want, bound)


def test_absorbed_small_groups_in_bf16(kda_pkg):
    """Channels 2^-40 of the others' size come out as exactly as theirs, relative to themselves."""
    S, R, P = 700, 512, 64
    rows = rand(2, S, R + P, seed=7, dtype=torch.float32)
    rows[..., 128:256] *= 2.0 ** -40
    cache, scale = quantised(rows, R)
    q = rand(2, 1, 16, R + P, seed=8, dtype=BF16, std=0.5)
    got = kda_pkg.mla_absorbed(q, cache, i32([S, S - 1]), R, 0.1, cache_scale=scale).double()
    want, bound = absorbed_ref(q, dequantised(cache, scale, R), [S, S - 1], R, 0.1)
    assert ((got - want).abs() <= bound)[..., 128:256].all()
    close("o", got, want, bound)


@pytest.mark.parametrize("S", [40, 3000])
def test_absorbed_largest_scales(kda_pkg, S):
    """The largest power there is, 2^127, beside others: its group's denominator is 2^-127 of its sums, a number
    below the normal ones, which is no zero.  (Queries of zeros: every weight is alike.)"""
    R, P = 512, 64
    cache, scale = quantised(rand(2, S, R + P, seed=12, dtype=torch.float32), R)
    raw(cache).bitwise_and_(0x99)                        # 0 and 0.5, of either sign
    raw(scale)[..., 0], raw(scale)[..., 1], raw(scale)[..., 2] = 254, 253, 0
    q = torch.zeros(2, 1, 16, R + P, dtype=BF16, device=DEV)
    got = kda_pkg.mla_absorbed(q, cache, i32([S, S - 3]), R, 0.1, cache_scale=scale)
    held = dequantised(cache, scale, R)[..., :R]
    want = torch.stack([held[0].mean(0), held[1, :S - 3].mean(0)])[:, None, None]
    # one rounding of the output; the weights are 1, the sums of halves exact, and the denominator has the 22 bits
    # of a number of that size, as 1 / it and their product have 24 or more
    close("o", got, want.expand(2, 1, 16, R), half_step(BF16) * (1 + 2.0 ** -8) * want.abs().expand(2, 1, 16, R))


@pytest.mark.parametrize("S", [100, 2000])
def test_absorbed_not_finite(kda_pkg, S):
    """A NaN scale reaches every channel of the queries that see its row, and no other sequence; behind the
    length none."""
    R, P = 256, 32
    cache, scale = quantised(rand(3, S, R + P, seed=9, dtype=torch.float32), R)
    q = rand(3, 1, 5, R + P, seed=10, dtype=BF16, std=0.5)
    lengths = [S, S - 20, S]
    want = kda_pkg.mla_absorbed(q, cache, i32(lengths), R, 0.1, cache_scale=scale)
    for at, byte in ((S // 2, 0), (S // 3, 1), (S // 2, 2)):
        bad = raw(scale).clone()
        bad[0, at, byte] = 255
        bad[1, S - 20:] = 255
        got = kda_pkg.mla_absorbed(q, cache, i32(lengths), R, 0.1, cache_scale=bad.view(E8M0))
        assert not torch.isfinite(got[0]).any(), byte
        assert torch.equal(got[1:], want[1:])


def test_absorbed_far_scores(kda_pkg):
    """Scores far from zero, all alike but one: their softmax, not the rounding of their size."""
    R, P, S = 128, 32, 200
    rows = torch.zeros(1, S, R + P, device=DEV)
    rows[..., R] = 4.0
    rows[..., :R] = rand(1, S, R, seed=11, dtype=torch.float32)
    cache, scale = quantised(rows, R)
    for size in (1e4, -1e4, 3e4):
        q = torch.zeros(1, 1, 4, R + P, dtype=F16, device=DEV)
        q[..., R] = size
        got = kda_pkg.mla_absorbed(q, cache, i32([S]), R, 1.0, cache_scale=scale)
        want = dequantised(cache, scale, R)[:, :, :R].mean(1)
        close("o", got, want[:, None, None].expand(1, 1, 4, R), (half_step(F16) * 2 + 1e-6) * want.abs() + 2.0 ** -12)


def test_absorbed_far_rows(kda_pkg):
    """A cache past 2^32 bytes: rows of zeros but for some."""
    R, P = 512, 64
    S = 2 ** 32 // ((R + P) // 2) + 5000
    cache = torch.zeros(1, S, (R + P) // 2, dtype=torch.uint8, device=DEV)
    scale = torch.full((1, S, 8), 127, dtype=torch.uint8, device=DEV)
    at = torch.tensor([0, 1000, S // 2, S - 3001, S - 1], device=DEV)
    some, e = quantised(rand(5, R + P, seed=12, dtype=torch.float32) * 3, R)
    cache[0, at], scale[0, at] = raw(some), raw(e)
    q = rand(1, 1, 4, R + P, seed=13, dtype=BF16, std=0.7)
    got = kda_pkg.mla_absorbed(q, cache.view(FOUR), i32([S]), R, 1.0, cache_scale=scale.view(E8M0))
    c = dequantised(some, e, R)
    s = q[0, 0].double() @ c.T                               # every other score is 0
    top = s.amax(1, keepdim=True).clamp_min(0)
    w = torch.exp(s - top)
    w = w / (w.sum(1, keepdim=True) + (S - 5) * torch.exp(-top))
    close("o", got[0, 0], w @ c[:, :R], (half_step(BF16) + 4e-4) * (w @ c[:, :R].abs()) + half_step(BF16) * (w @ c[:, :R]).abs())


@pytest.mark.parametrize("norm", [None, "same", "f32"])
@pytest.mark.parametrize("case", CACHE, ids=lambda c: "-".join(map(str, c[:5])) + "-" + str(c[5])[6:])
def test_append(kda_pkg, case, norm):
    B, T, S, R, P, dtype, lengths, counts = case
    x = rand(B, T, R + P, seed=21, dtype=dtype, std=2.0)
    x[:, -1, R // 2:] = 0
    x[0, 0] = 0
    w = None if norm is None else rand(R, seed=22, dtype=dtype if norm == "same" else torch.float32)
    cache, scale = quantised(rand(B, S, R + P, seed=23, dtype=torch.float32), R)
    old, old_scale = raw(cache).clone(), raw(scale).clone()
    out = kda_pkg.mla_cache_append(x, cache, i32(lengths), R, cache_scale=scale,
                                   counts=None if counts is None else i32(counts), norm_weight=w, eps=1e-5)
    assert out is None
    y = x.float()
    if norm is not None:                     # the kernel's own roundings: the mean in 64 bits, two products in 32
        rstd = torch.rsqrt(x[..., :R].double().square().mean(-1, keepdim=True) + torch.tensor(1e-5).double().item()).float()
        y = torch.cat([y[..., :R] * rstd * w.float(), y[..., R:]], -1)
    want, want_scale = quantised(y, R)
    touched = torch.zeros(B, S, dtype=torch.bool, device=DEV)
    for b in range(B):
        for t in range(T if counts is None else counts[b]):
            at = lengths[b] + t
            if not (0 <= lengths[b] and at < S):
                continue
            touched[b, at] = True
            assert torch.equal(raw(scale)[b, at], raw(want_scale)[b, t])
            got, ref = raw(cache)[b, at], raw(want)[b, t]
            zero = torch.stack([ref % 16 % 8 == 0, ref // 16 % 8 == 0], -1)      # (zeros may have either sign)
            same = torch.stack([got % 16 == ref % 16, got // 16 == ref // 16], -1)
            size = torch.stack([got % 8 == ref % 8, got // 16 % 8 == ref // 16 % 8], -1)
            assert (same | zero).all() and size.all()
    assert torch.equal(raw(cache)[~touched], old[~touched])
    assert torch.equal(raw(scale)[~touched], old_scale[~touched])


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("B,S,R,P,n", [(1, 1, 128, 0, None), (3, 77, 512, 64, [77, 0, 13]), (2, 300, 256, 32, None),
                                       (2, 9, 256, 0, [-3, 100]), (1, 40, 512, 0, [39]), (1, 21, 128, 64, [20])])
def test_read(kda_pkg, B, S, R, P, n, dtype):
    cache, scale = quantised(rand(B, S, R + P, seed=31, dtype=torch.float32), R)
    want = dequantised(cache, scale, R).to(dtype)
    if n is not None:
        for b in range(B):
            want[b, max(n[b], 0):] = 0
        poison(cache, scale, n)
    lengths = None if n is None else i32(n)
    got = kda_pkg.mla_cache_read(cache, scale, R, dtype=dtype, lengths=lengths)
    assert torch.equal(got, want)
    assert torch.equal(kda_pkg.mla_cache_read(cache, scale, R, dtype=dtype, tokens=S // 2, lengths=lengths), want[:, :S // 2])


def test_strided_caches(kda_pkg):
    """Caches and scales that are parts of larger buffers, read, written and attended to in place."""
    B, S, R, P = 3, 90, 256, 64
    cache, scale = quantised(rand(B, S, R + P, seed=33, dtype=torch.float32), R)
    big, bigs = torch.full((B, 2 * S, 208), 0x77, dtype=torch.uint8, device=DEV), torch.full((S, B, 24), 255, dtype=torch.uint8, device=DEV)
    c, s = big[:, ::2, 32:192].view(FOUR), bigs[..., 8:16].transpose(0, 1).view(E8M0)
    raw(c).copy_(raw(cache))
    raw(s).copy_(raw(scale))
    q, lengths = rand(B, 1, 16, R + P, seed=34, dtype=F16, std=0.5), i32([S, 5, 41])
    assert torch.equal(kda_pkg.mla_absorbed(q, c, lengths, R, 0.1, cache_scale=s),
                       kda_pkg.mla_absorbed(q, cache, lengths, R, 0.1, cache_scale=scale))
    assert torch.equal(kda_pkg.mla_cache_read(c, s, R), kda_pkg.mla_cache_read(cache, scale, R))
    x = rand(B, 4, R + P, seed=35, dtype=F16)
    for a, b in ((c, s), (cache, scale)):
        kda_pkg.mla_cache_append(x, a, lengths, R, cache_scale=b)
    assert torch.equal(raw(c), raw(cache)) and torch.equal(raw(s), raw(scale))
    assert (big[:, 1::2] == 0x77).all() and (big[:, :, :32] == 0x77).all() and (big[:, :, 192:] == 0x77).all()
    assert (bigs[..., :8] == 255).all() and (bigs[..., 16:] == 255).all()


def test_not_finite_rows(kda_pkg):
    """What is not finite reads back as NaN in its group of channels; its neighbours do not notice."""
    R, P = 256, 32
    x = rand(1, 5, R + P, seed=36, dtype=BF16)
    x[0, 1, 3], x[0, 2, R + 1], x[0, 3, 200] = float("inf"), float("nan"), -float("inf")
    cache = torch.zeros(1, 5, (R + P) // 2, dtype=torch.uint8, device=DEV).view(FOUR)
    scale = torch.zeros(1, 5, 8, dtype=torch.uint8, device=DEV).view(E8M0)
    kda_pkg.mla_cache_append(x, cache, i32([0]), R, cache_scale=scale)
    got = kda_pkg.mla_cache_read(cache, scale, R).isnan()
    want = torch.zeros_like(got)
    want[0, 1, :128], want[0, 2, R:], want[0, 3, 128:R] = True, True, True
    assert torch.equal(got, want)


def test_run_together(kda_pkg):
    """A prompt in two pieces read back for the expanded form, then tokens appended and attended to, captured and
    replayed with other work between; every step against the formula over what the cache holds."""
    B, H, P, R, S, dtype = 2, 4, 64, 256, 96, BF16
    w = rand(R, seed=43, dtype=dtype, std=0.1) + 1
    cache = torch.full((B, S, (R + P) // 2), 0x7f, device=DEV, dtype=torch.uint8).view(FOUR)
    scale = torch.full((B, S, 8), 255, device=DEV, dtype=torch.uint8).view(E8M0)
    lengths = torch.zeros(B, dtype=torch.int32, device=DEV)
    for piece, T in enumerate((40, 23)):
        x = rand(B, T, R + P, seed=50 + piece, dtype=dtype, std=1.5)
        kda_pkg.mla_cache_append(x, cache, lengths, R, cache_scale=scale, norm_weight=w)
        lengths += T
        n = int(lengths[0])
        rows = kda_pkg.mla_cache_read(cache, scale, R, dtype=dtype, tokens=n, lengths=lengths)
        assert torch.equal(rows.double(), dequantised(cache, scale, R)[:, :n])
        y = x.double()
        y[..., :R] *= torch.rsqrt(y[..., :R].square().mean(-1, keepdim=True) + 1e-6) * w.double()
        # half of the widest step of a group, whose largest magnitude is over 3.5 steps' unit
        top = torch.cat([y[..., :R].unflatten(-1, (-1, 128)).abs().amax(-1).repeat_interleave(128, -1),
                         y[..., R:].abs().amax(-1, keepdim=True).expand(B, T, P)], -1)
        assert ((rows[:, n - T:].double() - y).abs() <= top * (1 / 3.5 + 1e-6)).all()
    x_in, q_in = torch.zeros(B, 1, R + P, dtype=dtype, device=DEV), torch.zeros(B, 1, H, R + P, dtype=dtype, device=DEV)

    def step():
        kda_pkg.mla_cache_append(x_in, cache, lengths, R, cache_scale=scale, norm_weight=w)
        lengths.add_(1)
        return kda_pkg.mla_absorbed(q_in, cache, lengths, R, 0.07, cache_scale=scale)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    lengths.sub_(1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = step()
    for t in range(6):
        x_in.copy_(rand(B, 1, R + P, seed=70 + t, dtype=dtype, std=1.5))
        q_in.copy_(rand(B, 1, H, R + P, seed=80 + t, dtype=dtype, std=0.6))
        graph.replay()
        torch.cuda.synchronize()
        n = lengths.tolist()
        assert n == [64 + t] * B
        want, bound = absorbed_ref(q_in, dequantised(cache, scale, R).nan_to_num(), n, R, 0.07)
        close("o", o, want, bound)
        assert torch.equal(o, kda_pkg.mla_absorbed(q_in, cache, lengths, R, 0.07, cache_scale=scale))


def test_refusals(kda_pkg):
    R, P, S = 128, 32, 8
    cache, scale = quantised(rand(1, S, R + P, seed=90, dtype=torch.float32), R)
    q, x, n = rand(1, 1, 2, R + P, seed=91, dtype=F16), rand(1, 2, R + P, seed=92, dtype=F16), i32([3])
    wide = torch.zeros(1, S, 100, dtype=torch.uint8, device=DEV)
    bad = [
        lambda: kda_pkg.mla_absorbed(q, cache, n, R, 0.1),                                   # no scales
        lambda: kda_pkg.mla_absorbed(q, cache, n, R, 0.1, cache_scale=raw(scale)),           # of another type
        lambda: kda_pkg.mla_absorbed(q, cache, n, R, 0.1, cache_scale=scale[..., :2]),
        lambda: kda_pkg.mla_absorbed(q, cache, n, R, 0.1, cache_scale=torch.ones(1, S, 2, device=DEV)),
        lambda: kda_pkg.mla_absorbed(q, raw(cache), n, R, 0.1, cache_scale=scale),
        lambda: kda_pkg.mla_absorbed(q[..., :-8], cache, n, R, 0.1, cache_scale=scale),
        lambda: kda_pkg.mla_absorbed(q, wide[..., 2:82].view(FOUR), n, R, 0.1, cache_scale=scale),      # rows not aligned
        lambda: kda_pkg.mla_absorbed(q, cache, n, 192, 0.1, cache_scale=scale),
        lambda: kda_pkg.mla_cache_append(x, cache, n, R),
        lambda: kda_pkg.mla_cache_append(x, cache[:, :1].expand(1, S, 80), n, R, cache_scale=scale),
        lambda: kda_pkg.mla_cache_append(x, cache, n, R, cache_scale=scale[:, :1].expand(1, S, 8)),
        lambda: kda_pkg.mla_cache_read(cache, scale, R, dtype=torch.float32),
        lambda: kda_pkg.mla_cache_read(cache, scale.view(torch.uint8), R),
        lambda: kda_pkg.mla_cache_read(cache, scale, R, tokens=S + 1),
        lambda: kda_pkg.mla_cache_read(raw(cache), scale, R),
    ]
    before = raw(cache).clone()
    for i, call in enumerate(bad):
        with pytest.raises(kda_pkg.KdaError):
            call()
            pytest.fail(f"call {i} was answered")
    assert torch.equal(raw(cache), before)


@pytest.mark.parametrize("top", [66, 67, 100, 125])
@pytest.mark.parametrize("B,T,H,S,R,P", [(1, 1, 16, 2, 512, 64), (2, 3, 5, 130, 128, 32), (3, 1, 16, 3000, 512, 64), (40, 1, 16, 700, 256, 0)])
def test_absorbed_scales_far_apart(kda_pkg, B, T, H, S, R, P, top):
    """Powers of one group from 2^-60, which rows of zeros have, to 2^125: the softmax's denominator goes by the scores
    alone.  (Queries of zeros but where the powers are ordinary, so that scores are of like size.)"""
    g = torch.Generator(device=DEV).manual_seed(100 + S)
    cache, scale = quantised(rand(B, S, R + P, seed=101, dtype=torch.float32), R)
    any_of = torch.tensor([67, 67, 127, top + 127], dtype=torch.uint8, device=DEV)
    raw(scale)[..., :R // 128] = any_of[torch.randint(0, 4, (B, S, R // 128), generator=g, device=DEV)]
    raw(scale)[:, :2, 0] = torch.tensor([67, top + 127], dtype=torch.uint8, device=DEV)
    q = rand(B, T, H, R + P, seed=102, dtype=BF16, std=0.5)
    q[..., :R] = 0
    lengths = [max(S - 7 * b, 0) for b in range(B)]
    held = dequantised(cache, scale, R)
    got = kda_pkg.mla_absorbed(q, cache, i32(lengths), R, 0.1, cache_scale=scale)
    close("o", got, *absorbed_ref(q, held, lengths, R, 0.1))


@pytest.mark.parametrize("S", [2, 90, 2500])
def test_absorbed_zeros_beside_large_rows(kda_pkg, S):
    """Rows as they are appended, half of them zeros: of equal weights the output is half of the others' mean."""
    R, P = 256, 32
    x = rand(1, S, R + P, seed=103, dtype=BF16) * 2.0 ** 90
    x[:, ::2] = 0
    cache = torch.zeros(1, S, (R + P) // 2, dtype=torch.uint8, device=DEV).view(FOUR)
    scale = torch.zeros(1, S, 8, dtype=torch.uint8, device=DEV).view(E8M0)
    kda_pkg.mla_cache_append(x, cache, i32([0]), R, cache_scale=scale)
    q = torch.zeros(1, 1, 4, R + P, dtype=BF16, device=DEV)
    got = kda_pkg.mla_absorbed(q, cache, i32([S]), R, 1.0, cache_scale=scale)
    close("o", got, *absorbed_ref(q, dequantised(cache, scale, R), [S], R, 1.0))


@pytest.mark.parametrize("late", [False, True])
@pytest.mark.parametrize("dtype,a,b", [(BF16, 60, 43), (BF16, -60, 43), (BF16, 60, 65), (BF16, -60, 65), (BF16, 20, 7), (BF16, 17, 0),
                                       (BF16, -17, 0), (F16, 15, 14), (F16, -15, 14), (F16, 12, 10)], ids=str)
@pytest.mark.parametrize("B,T,H,S", [(1, 1, 16, 100), (2, 3, 4, 1000), (70, 1, 16, 600)])
def test_absorbed_far_scores_and_scales(kda_pkg, B, T, H, S, dtype, a, b, late):
    """Scores of up to 2^126 in size over rows of different powers: the keys that share the largest share the weight,
    whatever their powers.  late: the far scores come behind keys whose scores are zero."""
    R, P = 128, 32
    g = torch.Generator(device=DEV).manual_seed(104)
    cache, scale = quantised(rand(B, S, R + P, seed=105, dtype=torch.float32), R)
    lo, hi = (-10, 10) if dtype == F16 else (-50, 50)
    raw(scale)[..., 0] = (torch.randint(lo, hi, (B, S), generator=g, device=DEV) + 127).to(torch.uint8)
    raw(scale)[..., 1] = b + 127
    raw(cache)[..., R // 2:] = 0
    raw(cache)[..., R // 2] = torch.randint(2, 8, (B, S), generator=g, device=DEV, dtype=torch.uint8)       # 1 to 6
    if late:
        raw(cache)[:, :S // 2, R // 2] = 0
    q = torch.zeros(B, T, H, R + P, dtype=dtype, device=DEV)
    q[..., R] = float((1 if a > 0 else -1) * 2.0 ** abs(a))
    got = kda_pkg.mla_absorbed(q, cache, i32([S] * B), R, 0.125, cache_scale=scale)
    close("o", got, *absorbed_ref(q, dequantised(cache, scale, R), [S] * B, R, 0.125))


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("B,T,H,S", [(1, 1, 16, 100), (2, 3, 20, 700), (70, 1, 16, 600), (1, 2, 16, 20000), (600, 1, 4, 130)])
def test_absorbed_scores_of_all_sizes_in_a_tile(kda_pkg, B, T, H, S, dtype, bits):
    """Heads of one row tile whose scores are small, large and of either sign, over parts of a sequence whose scores
    are near zero, past 66 and past 200, and powers that differ.  One channel makes the scores: products are exact."""
    R, P = 128, 32
    g = torch.Generator(device=DEV).manual_seed(120 + S)
    size = torch.tensor([0.0, 1.0, -1.0, 5.0, -5.0, 10.0, -10.0, 20.0, 30.0, -40.0], dtype=torch.float64, device=DEV)
    q = torch.zeros(B, T, H, R + P, dtype=dtype, device=DEV)
    q[..., R] = size[torch.randint(0, len(size), (B, T, H), generator=g, device=DEV)].to(dtype)
    rows = rand(B, S, R + P, seed=121, dtype=torch.float32) * torch.exp2(torch.randint(-8, 5, (B, S, 1), generator=g, device=DEV).float())
    rows[..., R:] = 0
    step = torch.tensor([1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=DEV)[torch.randint(0, 6, (B, S), generator=g, device=DEV)]
    at = torch.arange(S, device=DEV) * 5 // S                        # fifths: far, near zero, far the other way, further, near zero
    rows[..., R] = step * torch.tensor([1.0, 2.0 ** -6, -1.0, 2.0, 0.0], device=DEV)[at]
    if bits == 4:
        cache, scale = quantised(rows, R)
        held = dequantised(cache, scale, R)
    else:
        cache, scale = quantised8(rows, R)
        held = dequantised8(cache, scale, R)
    lengths = [max(S - 3 * (b % 40), 0) for b in range(B)]
    got = kda_pkg.mla_absorbed(q, cache, i32(lengths), R, 1.0, cache_scale=scale)
    close("o", got, *absorbed_ref(q, held, lengths, R, 1.0))
