"""Latent attention and its cache against their formulas in float64.

Bounds are per element, from the roundings the kernels make: u is half a step
of the activation type (``finfo.eps / 2``), E the relative error of a softmax
weight from fp32 scores and exponentials.  A score's sum of D products in fp32
is off by at most D 2^-24 times the sum of their magnitudes; at these tests'
D <= 576 and magnitudes (below 60 after scaling) that is 2e-3 in the worst
case and 2^-24 sqrt(D) 60 = 9e-5 where roundings are independent; the
exponential adds 2^-22.  E = 4e-4.

* forward: weights rounded to the type (u), sums in fp32, output rounded (u):
  |o - o'| <= (u + E) sum p |v| + u |o|
* dv: the same with |do|.  ds = p (dp - delta): rounded (u), delta from the
  rounded o (u sum |do o|), dp's fp32 sum (2^-20 sum |do v| covers 128 terms):
  |dds| <= (u + 2E) |ds| + p (u sum |do o| + 2^-20 sum |do v|), and dq and dk
  are sums of it against |k| and |q|, rounded once (u).
"""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
E = 4e-4
F8 = torch.float8_e4m3fn
BF16, F16 = torch.bfloat16, torch.float16


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def rand(*shape, seed, dtype=torch.float64, std=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(*shape, device=DEV, generator=g, dtype=torch.float64) * std).to(dtype)


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def close(name, got, want, bound):
    """Every element within its bound (plus the smallest step of a 16-bit type)."""
    assert got.shape == want.shape, (name, got.shape, want.shape)
    assert torch.isfinite(got.double()).all(), f"{name} is not finite"
    off = (got.double() - want).abs() - bound - 2.0 ** -24
    worst = off.max().item() if off.numel() else -1.0
    assert worst <= 0, f"{name}: {worst:.3e} over its bound, {int((off > 0).sum())} of {off.numel()} elements"


# ---- the formulas -----------------------------------------------------------

def mask_of(T, S, lengths, starts):
    n = torch.tensor(lengths, device=DEV).clamp(0, S)[:, None]
    pos = torch.tensor(starts, device=DEV)[:, None] + torch.arange(T, device=DEV)
    return (torch.arange(S, device=DEV) <= pos[..., None]) & (torch.arange(S, device=DEV) < n[..., None]) & (
        pos < n)[..., None]                                                      # [B, T, S]


def weights(s, mask):
    s = s.masked_fill(~mask, -torch.inf)
    e = torch.exp(s - s.amax(-1, keepdim=True).nan_to_num(neginf=0.0))
    return e / e.sum(-1, keepdim=True).clamp_min(1e-300)


def expanded_ref(q, kn, pe, v, lengths, starts, scale, d_o=None):
    """(o, its bound) and, with d_o, {gradient: (value, bound)}; all [B, tokens, ...] in float64."""
    u = half_step(q.dtype)
    B, T, H, _ = q.shape
    S, N = kn.shape[1], kn.shape[3]
    mask = mask_of(T, S, lengths, starts)[:, None]
    keep = (torch.arange(S, device=DEV) < torch.tensor(lengths, device=DEV)[:, None])[:, :, None, None]
    Q = q.double().transpose(1, 2)
    K = torch.where(keep, kn.double(), 0).transpose(1, 2)
    V = torch.where(keep, v.double(), 0).transpose(1, 2)
    if pe is not None:
        Pe = torch.where(keep[..., 0], pe.double(), 0)
        K = torch.cat([K, Pe[:, None].expand(B, H, S, pe.shape[-1])], -1)
    p = weights(Q @ K.transpose(2, 3) * scale, mask)
    o = p @ V
    bound = (u + E) * (p @ V.abs()) + u * o.abs()
    if d_o is None:
        return o.transpose(1, 2), bound.transpose(1, 2)
    dO = torch.where(mask.any(-1)[..., None], d_o.double().transpose(1, 2), 0)
    dp = dO @ V.transpose(2, 3)
    ds = p * (dp - (dO * o).sum(-1, keepdim=True))
    e_ds = (u + 2 * E) * ds.abs() + p * (u * (dO * o).abs().sum(-1, keepdim=True)
                                         + 2.0 ** -20 * (dO.abs() @ V.abs().transpose(2, 3)))
    e_ds = e_ds + 2.0 ** -30 * ds.abs().amax((-1, -2), keepdim=True)     # fp16: ds far below the largest of its wave
    dv, e_dv = p.transpose(2, 3) @ dO, (u + E) * (p.transpose(2, 3) @ dO.abs())
    dq, e_dq = scale * ds @ K, scale * e_ds @ K.abs()
    dk, e_dk = scale * ds.transpose(2, 3) @ Q, scale * e_ds.transpose(2, 3) @ Q.abs()

    def out(x, e):
        return x.transpose(1, 2), (e + u * x.abs()).transpose(1, 2)

    grads = {"q": out(dq, e_dq), "k_nope": out(dk[..., :N], e_dk[..., :N]), "v": out(dv, e_dv)}
    if pe is not None:
        x, e = dk[..., N:].sum(1), e_dk[..., N:].sum(1)
        grads["k_pe"] = (x, e + u * x.abs())
    return o.transpose(1, 2), bound.transpose(1, 2), grads


def absorbed_ref(q, rows, lengths, rank, scale):
    u = half_step(q.dtype)
    B, T, H, D = q.shape
    S = rows.shape[1]
    mask = mask_of(T, S, lengths, [n - T for n in lengths])
    rows = torch.where((torch.arange(S, device=DEV) < torch.tensor(lengths, device=DEV)[:, None])[..., None],
                       rows.double(), 0)
    p = weights(torch.einsum("bthd,bsd->bhts", q.double(), rows) * scale, mask[:, None])
    o = (p @ rows[:, None, :, :rank]).transpose(1, 2)
    return o, (u + E) * (p @ rows[:, None, :, :rank].abs()).transpose(1, 2) + u * o.abs()


def quantised(x, rank):
    """x [B, S, D] float as the 8-bit cache holds it."""
    scale = torch.stack([x[..., :rank].float().abs().amax(-1),
                         x[..., rank:].float().abs().amax(-1) if x.shape[-1] > rank else
                         torch.full(x.shape[:2], 448.0, device=DEV)], -1).clamp_min(448 * 2.0 ** -60)
    scale = scale / torch.full_like(scale, 448.0)        # (by a Python number torch multiplies with its rounded inverse)
    each = torch.cat([scale[..., :1].expand(*x.shape[:2], rank), scale[..., 1:].expand(*x.shape[:2], x.shape[-1] - rank)], -1)
    return (x.float() / each).clamp(-448, 448).to(F8), scale


def dequantised(data, scale, rank):
    return torch.cat([data[..., :rank].double() * scale[..., :1].double(),
                      data[..., rank:].double() * scale[..., 1:].double()], -1)


# ---- expanded ---------------------------------------------------------------

def inputs(B, T, S, H, N, P, dtype, seed=0):
    return (rand(B, T, H, N + P, seed=seed, dtype=dtype), rand(B, S, H, N, seed=seed + 1, dtype=dtype),
            rand(B, S, P, seed=seed + 2, dtype=dtype) if P else None, rand(B, S, H, N, seed=seed + 3, dtype=dtype))


EXPANDED = [
    # B, T, S, H, N, P, dtype, lengths, starts
    (1, 1, 1, 1, 128, 64, BF16, None, None),
    (2, 1, 300, 3, 128, 64, F16, [300, 77], [299, 76]),          # one new token each, of two lengths
    (1, 65, 65, 2, 64, 32, BF16, None, None),
    (2, 200, 200, 3, 128, 64, F16, [200, 131], None),            # a padded batch
    (3, 70, 190, 2, 64, 64, BF16, [190, 0, 130], [120, 0, 60]),  # pieces of prompts and an empty slot
    (1, 33, 500, 1, 128, 0, F16, None, None),
    (1, 300, 300, 2, 64, 0, BF16, None, None),
    (1, 129, 257, 5, 128, 32, BF16, None, [100]),                # queries end before the keys do
    (2, 40, 16, 2, 64, 64, F16, None, None),                     # more queries than keys: the first see none
    (1, 600, 600, 16, 128, 64, BF16, None, None),
    (1, 1, 5000, 2, 128, 64, BF16, None, None),                  # few rows over many keys: shared among workgroups
    (2, 70, 2100, 3, 64, 32, F16, [2100, 40], [2030, 0]),
    (3, 9, 1300, 2, 128, 0, BF16, [0, 600, 1300], [0, 591, 1291]),
    (4, 700, 700, 24, 64, 32, F16, None, None),                  # enough rows for the widest workgroups
]


@pytest.mark.parametrize("case", EXPANDED, ids=lambda c: "-".join(map(str, c[:6])) + "-" + str(c[6])[6:])
def test_expanded_forward_and_gradients(kda_pkg, case):
    B, T, S, H, N, P, dtype, lengths, starts = case
    q, kn, pe, v = inputs(B, T, S, H, N, P, dtype)
    n, st = lengths or [S] * B, starts or [S - T] * B
    for b in range(B):                       # what the kernels must not read
        for x in (kn, v, pe):
            if x is not None:
                x[b, n[b]:] = float("nan")
    d_o = rand(B, T, H, N, seed=9, dtype=dtype)
    leaves = [x.requires_grad_() for x in (q, kn, pe, v) if x is not None]
    kw = dict(lengths=None if lengths is None else i32(lengths), starts=None if starts is None else i32(starts))
    o = kda_pkg.mla_expanded(q, kn, pe, v, **kw)
    grads = torch.autograd.grad(o, leaves, d_o)
    with torch.no_grad():
        assert torch.equal(o, kda_pkg.mla_expanded(q, kn, pe, v, **kw))
        want, bound, ref = expanded_ref(q, kn, pe, v, n, st, (N + P) ** -0.5, d_o)
    close("o", o, want, bound)
    names = [m for m, x in (("q", q), ("k_nope", kn), ("k_pe", pe), ("v", v)) if x is not None]
    for m, g in zip(names, grads):
        close("d" + m, g, *ref[m])


# Each of the backward's tilings (rows or keys a workgroup, how the waves share them), at lengths that end inside one.
TILINGS = [
    (1, 300, 300, 2, 128, 64, F16, [299], None),                 # 64 rows and keys
    (2, 333, 700, 3, 128, 32, BF16, [700, 411], [367, 78]),
    (1, 1100, 1100, 5, 128, 64, BF16, None, None),
    (1, 270, 270, 1, 128, 0, F16, None, None),
    (4, 520, 520, 16, 128, 64, BF16, [520, 519, 1, 300], None),  # 128 rows, their keys shared
    (4, 520, 520, 16, 64, 32, F16, [520, 0, 129, 384], None),    # 128 rows
    (2, 1030, 1030, 16, 64, 64, BF16, None, None),
    (8, 300, 300, 16, 128, 64, F16, [300, 1, 0, 257, 256, 255, 299, 33], None),
    (16, 300, 300, 16, 128, 64, BF16, [300, 1, 0, 257, 256, 255, 299, 33] * 2, None),   # 256 rows
]


@pytest.mark.parametrize("case", TILINGS, ids=lambda c: "-".join(map(str, c[:6])) + "-" + str(c[6])[6:])
def test_expanded_tilings(kda_pkg, case):
    test_expanded_forward_and_gradients(kda_pkg, case)


def test_expanded_gradients_against_differences(kda_pkg):
    """The directional derivative of sum(o w) in each input, by central differences of the float64 formula."""
    B, T, S, H, N, P = 1, 40, 56, 2, 64, 32
    q, kn, pe, v = inputs(B, T, S, H, N, P, BF16, seed=20)
    w = rand(B, T, H, N, seed=30, dtype=BF16)
    leaves = [x.requires_grad_() for x in (q, kn, pe, v)]
    grads = torch.autograd.grad(kda_pkg.mla_expanded(q, kn, pe, v), leaves, w)
    base = [x.detach().double() for x in (q, kn, pe, v)]

    def value(xs):
        K = torch.cat([xs[1], xs[2][:, :, None].expand(B, S, H, P)], -1).transpose(1, 2)
        p = weights(xs[0].transpose(1, 2) @ K.transpose(2, 3) * (N + P) ** -0.5, mask_of(T, S, [S], [S - T])[:, None])
        return ((p @ xs[3].transpose(1, 2)).transpose(1, 2) * w.double()).sum()

    _, _, ref = expanded_ref(*(x.detach() for x in (q, kn, pe, v)), [S], [S - T], (N + P) ** -0.5, w)
    for i, m in enumerate(("q", "k_nope", "k_pe", "v")):
        d = rand(*base[i].shape, seed=40 + i)
        up, down = list(base), list(base)
        up[i], down[i] = base[i] + 1e-5 * d, base[i] - 1e-5 * d
        slope = (value(up) - value(down)).item() / 2e-5
        got = (grads[i].double() * d).sum().item()
        # each element's bound against |d|, and the differences' own error (third derivatives, 1e-10, and roundings, 1e-9)
        assert abs(got - slope) <= (ref[m][1] * d.abs()).sum().item() + 1e-6, m


def test_expanded_small_fp16_gradients(kda_pkg):
    """Gradients a loss scale has left near fp16's smallest: ds is 2^-24 and below, its sums are not."""
    q, kn, pe, v = inputs(1, 256, 256, 2, 64, 32, F16, seed=50)
    d_o = rand(1, 256, 2, 64, seed=51, dtype=F16, std=2.0 ** -9)
    leaves = [x.requires_grad_() for x in (q, kn, pe, v)]
    grads = torch.autograd.grad(kda_pkg.mla_expanded(q, kn, pe, v), leaves, d_o)
    _, _, ref = expanded_ref(*(x.detach() for x in leaves), [256], [0], 96 ** -0.5, d_o)
    for m, g in zip(("q", "k_nope", "k_pe", "v"), grads):
        close("d" + m, g, *ref[m])


@pytest.mark.parametrize("B,T,H,N,P,dtype", [(1, 2, 3, 128, 0, BF16), (1, 33, 3, 64, 64, BF16), (2, 128, 2, 128, 64, F16)])
def test_expanded_few_tokens(kda_pkg, B, T, H, N, P, dtype):
    """Of few values no single rounding may dominate: the weights and ds keep 16 bits or more, so what is left of
    an output's error is its own rounding (relative, in the 2-norm) and less than 2^-12 in bf16 (a weight kept to
    2^-17, o and its rounding to 2^-17, a sum's cancellation below 2^5), 2^-14 in fp16 (E, as above, is 2^-11)."""
    q, kn, pe, v = inputs(B, T, T, H, N, P, dtype, seed=60)
    d_o = rand(B, T, H, N, seed=64, dtype=dtype)
    leaves = [x.requires_grad_() for x in (q, kn, pe, v) if x is not None]
    o = kda_pkg.mla_expanded(q, kn, pe, v)
    grads = torch.autograd.grad(o, leaves, d_o)
    with torch.no_grad():
        want, _, ref = expanded_ref(q, kn, pe, v, [T] * B, [0] * B, (N + P) ** -0.5, d_o)
    ref = {"o": (want, None), **ref}
    names = ["o"] + [m for m, x in (("q", q), ("k_nope", kn), ("k_pe", pe), ("v", v)) if x is not None]
    for m, got in zip(names, (o, *grads)):
        r = ref[m][0]
        off, own = (((x.double() - r).norm() / r.norm()).item() for x in (got, r.to(dtype)))
        assert off <= own + (2.0 ** -12 if dtype is BF16 else 2.0 ** -14), (m, off, own)


def test_expanded_views_streams_and_types(kda_pkg):
    B, T, H, N, P = 2, 90, 3, 128, 64
    kv = rand(B, T, H, 2 * N, seed=60, dtype=BF16)
    wide = rand(B, T, 700, seed=61, dtype=BF16)
    q = rand(B, H, T, N + P, seed=62, dtype=BF16).transpose(1, 2)
    kn, v, pe = kv[..., :N], kv[..., N:], wide[..., 512:512 + P]
    want = kda_pkg.mla_expanded(q.contiguous(), kn.contiguous(), pe.contiguous(), v.contiguous())
    assert torch.equal(kda_pkg.mla_expanded(q, kn, pe, v), want)
    # unaligned rows and reversed channels are copied first; 64-bit lengths are taken too
    odd = rand(B, T, P + 1, seed=61, dtype=BF16)
    odd[..., 1:] = pe
    assert torch.equal(kda_pkg.mla_expanded(q, kn, odd[..., 1:], v, lengths=torch.full((B,), T, device=DEV)), want)
    # one sequence for all: batch stride 0
    one = kda_pkg.mla_expanded(q, kn[:1].expand(B, T, H, N), pe[:1].expand(B, T, P), v[:1].expand(B, T, H, N))
    assert torch.equal(one[0], want[0])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = kda_pkg.mla_expanded(q, kn, pe, v)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(other, want)
    # fp32 keys are taken in q's type, as under mixed precision; their gradient comes back in fp32
    k32 = kn.float().contiguous().requires_grad_()
    o = kda_pkg.mla_expanded(q, k32, pe, v)
    assert torch.equal(o, want)
    assert torch.autograd.grad(o.float().sum(), k32)[0].dtype == torch.float32


def test_expanded_is_differentiated_once(kda_pkg):
    q, kn, pe, v = (x.requires_grad_() for x in inputs(1, 20, 20, 2, 64, 32, BF16, seed=90))
    o = kda_pkg.mla_expanded(q, kn, pe, v)
    first = torch.autograd.grad(o.float().square().sum(), (q, kn, pe, v), create_graph=True)
    with pytest.raises(RuntimeError):            # torch's own word for it: v is not in first's graph
        torch.autograd.grad(first[0].float().sum(), v)
    with pytest.raises(RuntimeError, match="once"):
        first[0].float().sum().backward()
    # an input changed after the forward is noticed
    leaf = v.detach().clone()
    o = kda_pkg.mla_expanded(q, kn, pe, leaf)
    leaf.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        o.float().sum().backward()
    # a gradient of another layout or shared by broadcasting
    o = kda_pkg.mla_expanded(q, kn, pe, v)
    a = torch.autograd.grad(o, v, torch.ones_like(o), retain_graph=True)[0]
    b = torch.autograd.grad(o, v, torch.ones(1, 1, 1, 1, dtype=BF16, device=DEV).expand_as(o))[0]
    assert torch.equal(a, b)


def test_expanded_empty(kda_pkg):
    q, kn, pe, v = inputs(2, 0, 5, 2, 64, 32, BF16)
    leaves = [x.requires_grad_() for x in (q, kn, pe, v)]
    o = kda_pkg.mla_expanded(q, kn, pe, v)
    assert o.shape == (2, 0, 2, 64)
    for g in torch.autograd.grad(o.sum(), leaves):
        assert (g == 0).all()
    q, kn, pe, v = inputs(2, 7, 0, 2, 64, 32, BF16)
    assert (kda_pkg.mla_expanded(q, kn, pe, v) == 0).all()


def test_expanded_far_offsets(kda_pkg):
    """A batch stride past 2^32 bytes."""
    H, N, T, far = 1, 64, 20, 2 ** 31 + 2 ** 20
    store = torch.empty(far + T * H * N, dtype=BF16, device=DEV)
    kn = store.as_strided((2, T, H, N), (far, H * N, N, 1))
    src = rand(2, T, H, N, seed=70, dtype=BF16)
    kn.copy_(src)
    q, v = rand(2, T, H, N, seed=71, dtype=BF16), rand(2, T, H, N, seed=72, dtype=BF16)
    assert torch.equal(kda_pkg.mla_expanded(q, kn, None, v), kda_pkg.mla_expanded(q, src, None, v))


def test_expanded_captured(kda_pkg):
    """Forward and backward in a graph whose lengths change between replays, beside eager work."""
    B, T, H, N, P = 2, 150, 2, 64, 32
    q, kn, pe, v = inputs(B, T, T, H, N, P, BF16, seed=80)
    d_o = rand(B, T, H, N, seed=84, dtype=BF16)
    leaves = [x.requires_grad_() for x in (q, kn, pe, v)]
    lengths = i32([T, T])

    def step():
        o = kda_pkg.mla_expanded(q, kn, pe, v, lengths=lengths)
        return [o.detach(), *torch.autograd.grad(o, leaves, d_o)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for n in ([150, 150], [1, 100], [0, 64], [150, 149]):
        lengths.copy_(i32(n))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, step()):
            assert torch.equal(a, b), n


def test_expanded_capture_beside_an_eager_graph(kda_pkg):
    """An eager graph of the same leaves, on the default stream, that lives when a backward pass is captured:
    refused, as the engine would end the process; with it deleted, or of other leaves, the capture is fine."""
    q, kn, pe, v = inputs(1, 70, 70, 2, 64, 32, F16, seed=85)
    d_o = rand(1, 70, 2, 64, seed=89, dtype=F16)
    leaves = [x.requires_grad_() for x in (q, kn, pe, v)]

    def grads(xs):
        return torch.autograd.grad(kda_pkg.mla_expanded(*xs), xs, d_o)

    want = grads(leaves)
    others = [x.detach().clone().requires_grad_() for x in leaves]
    kept = kda_pkg.mla_expanded(*leaves)
    torch.cuda.synchronize()
    with pytest.raises(kda_pkg.KdaError, match="default stream"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            grads(leaves)
    for xs in (others, leaves):
        if xs is leaves:
            assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(kept, leaves, d_o), want))
            del kept
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = grads(xs)
        for _ in range(3):
            for g in got:
                g.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want))


# ---- absorbed ---------------------------------------------------------------

ABSORBED = [
    # B, T, H, S, R, P, dtype, lengths
    (1, 1, 16, 1, 512, 64, BF16, [1]),
    (1, 1, 16, 200, 512, 64, F16, [199]),
    (3, 1, 16, 70, 512, 64, BF16, [70, 0, 33]),
    (5, 1, 7, 1000, 256, 32, F16, [1000, 1, 999, 0, 517]),        # shared among workgroups, an idle slot
    (2, 3, 5, 2000, 128, 0, BF16, [2000, 2]),                     # several tokens; the second has fewer than T
    (2, 6, 20, 777, 512, 64, F16, [777, 500]),
    (70, 1, 16, 600, 128, 64, BF16, [(37 * b) % 601 for b in range(70)]),
    (1100, 1, 4, 520, 128, 32, F16, [(211 * b) % 521 for b in range(1100)]),   # one workgroup a sequence
    (1, 1, 64, 5000, 512, 64, BF16, [4999]),                      # four row tiles
    (1, 2, 16, 9000, 256, 64, BF16, [8999]),
    (2, 1, 16, 30000, 512, 0, F16, [30000, 12345]),
]


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("case", ABSORBED, ids=lambda c: "-".join(map(str, c[:6])) + "-" + str(c[6])[6:])
def test_absorbed(kda_pkg, case, bits):
    B, T, H, S, R, P, dtype, lengths = case
    q = rand(B, T, H, R + P, seed=1, dtype=dtype, std=R ** -0.5 * 12)
    rows = rand(B, S, R + P, seed=2, dtype=torch.float32)
    rows[..., R:] *= 3
    cache, scale = (rows.to(dtype), None) if bits == 16 else quantised(rows, R)
    held = cache.double() if bits == 16 else dequantised(cache, scale, R)
    for b in range(B):                       # unwritten memory
        if bits == 16:
            cache[b, lengths[b]:] = float("nan")
        else:
            cache.view(torch.uint8)[b, lengths[b]:] = 0x7f
            scale[b, lengths[b]:] = float("nan")
    got = kda_pkg.mla_absorbed(q, cache, i32(lengths), R, (128 + P) ** -0.5, cache_scale=scale)
    want, bound = absorbed_ref(q, held, lengths, R, (128 + P) ** -0.5)
    close("o", got, want, bound)
    assert torch.equal(got, kda_pkg.mla_absorbed(q, cache, i32(lengths), R, (128 + P) ** -0.5, cache_scale=scale))


# Row tiles cut one by one, the most of them, and one more.
SHARED = [
    (64, 1, 16, 600, 128, 64, BF16, [600] + [1] * 63),
    (64, 1, 16, 4096, 256, 32, F16, [(997 * b) % 4097 for b in range(64)]),
    (65, 1, 16, 4096, 256, 32, F16, [(997 * b) % 4097 for b in range(65)]),
    (9, 5, 20, 900, 128, 0, BF16, [900, 899, 0, 5, 3, 128, 129, 640, 17]),       # 63 row tiles
    (60, 1, 16, 2048, 128, 64, BF16, 60 * [2048]),
]


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("case", SHARED, ids=lambda c: "-".join(map(str, c[:6])) + "-" + str(c[6])[6:])
def test_absorbed_shared(kda_pkg, case, bits):
    test_absorbed(kda_pkg, case, bits)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_absorbed_8bit_scales_of_any_size(kda_pkg, dtype):
    """Scales from 2^-60 (rows of zeros) over six orders of magnitude: weights keep their precision."""
    S, R, P = 300, 128, 32
    rows = rand(1, S, R + P, seed=5, dtype=torch.float32) * torch.logspace(-5, 1, S, device=DEV)[None, :, None]
    rows[:, ::7] = 0
    cache, scale = quantised(rows, R)
    q = rand(1, 1, 16, R + P, seed=6, dtype=dtype, std=0.5)
    got = kda_pkg.mla_absorbed(q, cache, i32([S]), R, 0.1, cache_scale=scale)
    want, bound = absorbed_ref(q, dequantised(cache, scale, R), [S], R, 0.1)
    close("o", got, want, bound)
    tiny = rows * 1e-4                       # every value is small: so is the output, at the same relative error
    cache, scale = quantised(tiny, R)
    got = kda_pkg.mla_absorbed(q, cache, i32([S]), R, 0.1, cache_scale=scale)
    want, bound = absorbed_ref(q, dequantised(cache, scale, R), [S], R, 0.1)
    close("o", got, want, bound)


def test_absorbed_far_rows(kda_pkg):
    """A cache past 2^32 bytes: rows of zeros but for some, so the softmax has a closed form."""
    R, P = 512, 64
    S = 2 ** 32 // ((R + P) * 2) + 5000
    cache = torch.zeros(1, S, R + P, dtype=BF16, device=DEV)
    at = torch.tensor([0, 1000, S // 2, S - 3001, S - 1], device=DEV)
    some = rand(5, R + P, seed=7, dtype=BF16)
    cache[0, at] = some
    q = rand(1, 1, 4, R + P, seed=8, dtype=BF16, std=0.7)
    got = kda_pkg.mla_absorbed(q, cache, i32([S]), R, 1.0)[0, 0]
    s = q[0, 0].double() @ some.double().T
    w = torch.exp(s)
    den = w.sum(1, keepdim=True) + (S - 5)
    p = w / den
    want, u = p @ some[:, :R].double(), half_step(BF16)
    close("o", got, want, (u + E) * (p @ some[:, :R].double().abs()) + u * want.abs())


def test_absorbed_views_streams_and_graph(kda_pkg):
    B, H, S, R, P = 4, 16, 900, 128, 64
    store = rand(B + 1, S + 30, R + P + 64, seed=11, dtype=BF16)
    cache = store[1:, 10:S + 10, :R + P]
    q = rand(B, H, 1, R + P, seed=12, dtype=BF16).transpose(1, 2)
    n = [900, 0, 451, 32]
    want = kda_pkg.mla_absorbed(q.contiguous(), cache.contiguous(), i32(n), R, 0.05)
    lengths = i32(n)
    assert torch.equal(kda_pkg.mla_absorbed(q, cache, lengths, R, 0.05), want)
    assert torch.equal(kda_pkg.mla_absorbed(q, cache, lengths.long(), R, 0.05), want)
    # lengths out of range count as S and 0
    assert torch.equal(kda_pkg.mla_absorbed(q, cache, i32([5000, -7, 451, 32]), R, 0.05), want)
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for s in streams:                        # calls at once, each with a workspace of its own
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(kda_pkg.mla_absorbed(q, cache, lengths, R, 0.05))
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(g, want) for g in got)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        kda_pkg.mla_absorbed(q, cache, lengths, R, 0.05)
    torch.cuda.current_stream().wait_stream(side)
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    outs = []
    for g in graphs:
        with torch.cuda.graph(g):
            outs.append(kda_pkg.mla_absorbed(q, cache, lengths, R, 0.05))
    for n in ([900, 0, 451, 32], [1, 900, 0, 700], [0, 0, 0, 0], [33, 64, 65, 899]):
        lengths.copy_(i32(n))
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        want = kda_pkg.mla_absorbed(q, cache, lengths, R, 0.05)
        assert all(torch.equal(o, want) for o in outs), n


def test_absorbed_is_the_expanded_form(kda_pkg):
    """The two forms of one attention: up-projections applied to the latents, or to q and o."""
    B, S, H, N, P, R = 2, 130, 8, 128, 64, 256
    cache = rand(B, S, R + P, seed=13, dtype=F16)
    wk, wv = rand(H, N, R, seed=14, dtype=F16, std=R ** -0.5), rand(H, N, R, seed=15, dtype=F16, std=R ** -0.5)
    q = rand(B, 1, H, N + P, seed=16, dtype=F16)
    lat = cache[..., :R].double()
    kn = torch.einsum("bsr,hnr->bshn", lat, wk.double()).to(F16)
    v = torch.einsum("bsr,hnr->bshn", lat, wv.double()).to(F16)
    full = kda_pkg.mla_expanded(q, kn, cache[..., R:].contiguous(), v)
    qa = torch.cat([torch.einsum("bthn,hnr->bthr", q[..., :N].double(), wk.double()).to(F16), q[..., N:]], -1)
    o = kda_pkg.mla_absorbed(qa, cache, i32([S, S]), R, (N + P) ** -0.5)
    absorbed = torch.einsum("bthr,hnr->bthn", o.double(), wv.double())
    # intermediate roundings of keys, values, queries and outputs (2^-11 each) move scores of size <= 6 and values of size <= 5
    assert (full.double() - absorbed).abs().max().item() <= 2.0 ** -11 * (6 * 4 * 2 + 4) * 2


# ---- the cache --------------------------------------------------------------

CACHE = [
    # B, T, S, R, P, dtype, lengths, counts
    (1, 1, 1, 512, 64, BF16, [0], None),
    (64, 1, 100, 512, 64, F16, [b % 101 for b in range(64)], None),          # some at the end: dropped
    (3, 50, 120, 256, 32, BF16, [0, 100, 70], [50, 50, 13]),
    (2, 37, 64, 128, 0, F16, [5, 27], [0, 37]),
    (2, 9, 30, 512, 0, BF16, [-4, 2 ** 31 - 5], None),                       # held rows that cannot be
]


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("case", CACHE, ids=lambda c: "-".join(map(str, c[:5])) + "-" + str(c[5])[6:])
def test_append(kda_pkg, case, bits, norm):
    B, T, S, R, P, dtype, lengths, counts = case
    x = rand(B, T, R + P, seed=21, dtype=dtype, std=2.0)
    x[:, -1, R // 2:] = 0
    x[0, 0] = 0
    w = rand(R, seed=22, dtype=dtype) if norm else None
    before = rand(B, S, R + P, seed=23, dtype=torch.float32)
    cache, scale = (before.to(dtype), None) if bits == 16 else quantised(before, R)
    raw = torch.int16 if bits == 16 else torch.uint8
    old, old_scale = cache.clone(), None if scale is None else scale.clone()
    out = kda_pkg.mla_cache_append(x, cache, i32(lengths), R, cache_scale=scale,
                                   counts=None if counts is None else i32(counts), norm_weight=w, eps=1e-5)
    assert out is None
    y = x.double()
    if norm:
        y[..., :R] = y[..., :R] * torch.rsqrt(y[..., :R].square().mean(-1, keepdim=True) + 1e-5) * w.double()
    touched = torch.zeros(B, S, dtype=torch.bool, device=DEV)
    for b in range(B):
        for t in range(T if counts is None else counts[b]):
            at = lengths[b] + t
            if not (0 <= lengths[b] and at < S):
                continue
            touched[b, at] = True
            if bits == 16:
                if norm:                                # fp32 arithmetic (2^-21), rounded once
                    close("row", cache[b, at], y[b, t], (half_step(dtype) + 2.0 ** -21) * y[b, t].abs())
                else:
                    assert torch.equal(cache[b, at], x[b, t])
            else:
                want, s = quantised(y[b, t][None, None], R)
                if not norm:                            # the same divisions: the same bits
                    assert torch.equal(scale[b, at], s[0, 0])
                    assert torch.equal(cache.view(torch.uint8)[b, at], want.view(torch.uint8)[0, 0])
                else:                                   # half a step of e4m3, 2^-4, of 2^-9 below its normal range
                    assert ((scale[b, at] - s[0, 0]).abs() <= 2.0 ** -21 * s[0, 0]).all()
                    got = dequantised(cache[b:b + 1, at:at + 1], scale[b:b + 1, at:at + 1], R)[0, 0]
                    step = torch.cat([s[0, 0, :1].expand(R), s[0, 0, 1:].expand(P)]).double() * 2.0 ** -10
                    close("row", got, y[b, t], (2.0 ** -4 + 2.0 ** -20) * y[b, t].abs() + step)
    keep = ~touched
    assert torch.equal(cache.view(raw)[keep], old.view(raw)[keep])
    if scale is not None:
        assert torch.equal(scale[keep], old_scale[keep])


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("B,S,R,P,n", [(1, 1, 128, 0, None), (3, 77, 512, 64, [77, 0, 13]), (2, 300, 256, 32, None)])
def test_read(kda_pkg, B, S, R, P, n, dtype):
    cache, scale = quantised(rand(B, S, R + P, seed=31, dtype=torch.float32), R)
    want = dequantised(cache, scale, R).to(torch.float32).to(dtype)     # the product of an e4m3 value and a scale, in fp32
    if n is not None:
        for b in range(B):
            want[b, n[b]:] = 0
            cache.view(torch.uint8)[b, n[b]:] = 0x7f
    got = kda_pkg.mla_cache_read(cache, scale, R, dtype=dtype, lengths=None if n is None else i32(n))
    assert torch.equal(got, want)
    assert torch.equal(kda_pkg.mla_cache_read(cache, scale, R, dtype=dtype, tokens=S // 2,
                                              lengths=None if n is None else i32(n)), want[:, :S // 2])


def test_not_finite_rows(kda_pkg):
    """A row with an infinity or a NaN reads back as not finite; its neighbours do not notice."""
    R, P = 128, 32
    x = rand(1, 4, R + P, seed=32, dtype=BF16)
    x[0, 1, 3], x[0, 2, R + 1] = float("inf"), float("nan")
    cache, scale = torch.zeros(1, 4, R + P, dtype=F8, device=DEV), torch.ones(1, 4, 2, device=DEV)
    kda_pkg.mla_cache_append(x, cache, i32([0]), R, cache_scale=scale)
    got = torch.isfinite(kda_pkg.mla_cache_read(cache, scale, R).float())
    assert got[0, 0].all() and got[0, 3].all()
    assert not got[0, 1, :R].any() and got[0, 1, R:].all() and got[0, 2, :R].all() and not got[0, 2, R:].any()


@pytest.mark.parametrize("bits", [16, 8])
def test_run_together(kda_pkg, bits):
    """A prompt in two pieces through the expanded form, then tokens through the absorbed one, captured; every
    step against the formula over what the cache holds."""
    B, H, N, P, R, S, dtype = 2, 4, 128, 64, 256, 96, BF16
    scale = (N + P) ** -0.5
    wk, wv = rand(H, N, R, seed=41, dtype=dtype, std=R ** -0.5), rand(H, N, R, seed=42, dtype=dtype, std=R ** -0.5)
    w = rand(R, seed=43, dtype=dtype, std=0.1) + 1
    cache = torch.full((B, S, R + P), 0x7f if bits == 8 else -1, device=DEV, dtype=torch.uint8 if bits == 8 else torch.int16)
    cache = cache.view(F8 if bits == 8 else dtype)
    scales = torch.full((B, S, 2), float("nan"), device=DEV) if bits == 8 else None
    lengths = torch.zeros(B, dtype=torch.int32, device=DEV)

    def held():
        return cache.double() if bits == 16 else dequantised(cache, scales, R)

    for piece, T in enumerate((40, 23)):
        x = rand(B, T, R + P, seed=50 + piece, dtype=dtype, std=1.5)
        q = rand(B, T, H, N + P, seed=60 + piece, dtype=dtype)
        kda_pkg.mla_cache_append(x, cache, lengths, R, cache_scale=scales, norm_weight=w)
        starts = lengths.clone()
        lengths += T
        n = int(lengths[0])
        rows = cache[:, :n] if bits == 16 else kda_pkg.mla_cache_read(cache, scales, R, dtype=dtype, tokens=n, lengths=lengths)
        kn = torch.einsum("bsr,hnr->bshn", rows[..., :R].float(), wk.float()).to(dtype)
        v = torch.einsum("bsr,hnr->bshn", rows[..., :R].float(), wv.float()).to(dtype)
        o = kda_pkg.mla_expanded(q, kn, rows[..., R:], v, lengths=lengths, starts=starts)
        close("piece", o, *expanded_ref(q, kn, rows[..., R:], v, [n] * B, [n - T] * B, scale))
    x_in, q_in = torch.zeros(B, 1, R + P, dtype=dtype, device=DEV), torch.zeros(B, 1, H, R + P, dtype=dtype, device=DEV)

    def step():
        kda_pkg.mla_cache_append(x_in, cache, lengths, R, cache_scale=scales, norm_weight=w)
        lengths.add_(1)
        return kda_pkg.mla_absorbed(q_in, cache, lengths, R, scale, cache_scale=scales)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    lengths.sub_(1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for t in range(5):
        x_in.copy_(rand(B, 1, R + P, seed=70 + t, dtype=dtype))
        q_in.copy_(rand(B, 1, H, R + P, seed=80 + t, dtype=dtype, std=0.7))
        graph.replay()
        n = int(lengths[0])
        assert n == 64 + t
        close("token", out, *absorbed_ref(q_in, held(), [n] * B, R, scale))


# ---- a token that takes nearly all of the weight ----------------------------

@pytest.mark.parametrize("gap", [16.0, 20.0])
@pytest.mark.parametrize("B,T,S,at", [(1, 1, 4097, 0), (1, 70, 4097, 1000), (2, 300, 300, 0), (1, 20, 20, 0), (4, 520, 520, 3)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_expanded_sink(kda_pkg, dtype, B, T, S, at, gap):
    """One key scores `gap` nats above all others and its values are zero in half of the channels: what the others
    leave there, each with a weight of 2^-23 to 2^-29, is kept to the types' precision."""
    H, N, P, scale = 2, 64, 32, 0.1
    q, kn, pe, v = inputs(B, T, S, H, N, P, dtype, seed=70)
    q, kn, pe, v = 0.3 * q, 0.3 * kn, 0.3 * pe, 30 * v.abs() + 30
    q[..., 0], kn[..., 0], kn[:, at, :, 0] = 8.0, 0.0, gap / (8 * scale)
    v[:, at, :, ::2] = 0
    d_o = rand(B, T, H, N, seed=75, dtype=dtype)
    leaves = [x.requires_grad_() for x in (q, kn, pe, v)]
    o = kda_pkg.mla_expanded(q, kn, pe, v, scale=scale)
    grads = torch.autograd.grad(o, leaves, d_o)
    with torch.no_grad():
        want, bound, ref = expanded_ref(q, kn, pe, v, [S] * B, [S - T] * B, scale, d_o)
    close("o", o, want, bound)
    for m, g in zip(("q", "k_nope", "k_pe", "v"), grads):
        close("d" + m, g, *ref[m])


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("gap", [16.0, 20.0])
@pytest.mark.parametrize("B,T,H,S,at", [(1, 1, 16, 4097, 0), (3, 2, 4, 400, 130), (70, 1, 16, 1000, 7)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_absorbed_sink(kda_pkg, dtype, B, T, H, S, at, gap, bits):
    R, P, scale = 128, 32, 0.1
    q = rand(B, T, H, R + P, seed=76, dtype=dtype, std=0.01)
    rows = rand(B, S, R + P, seed=77, dtype=torch.float32)
    rows[..., :R] = 30 * rows[..., :R].abs() + 30
    q[..., R], rows[..., R], rows[:, at, R] = 8.0, 0.0, gap / (8 * scale)
    rows[:, at, :R:2] = 0
    cache, sc = (rows.to(dtype), None) if bits == 16 else quantised(rows, R)
    held = cache.double() if bits == 16 else dequantised(cache, sc, R)
    got = kda_pkg.mla_absorbed(q, cache, i32([S] * B), R, scale, cache_scale=sc)
    close("o", got, *absorbed_ref(q, held, [S] * B, R, scale))


# ---- scores far from zero ---------------------------------------------------

def steps(shape, at):
    """1, 1 + 2^-7 .. 2 - 2^-7 along dimension `at`, in a shuffled order: what a bf16 mantissa holds."""
    n = shape[at]
    m = 1 + (torch.arange(n, device=DEV, dtype=torch.float64) * 37 % 128) / 128
    return m.view([-1 if d == at else 1 for d in range(len(shape))]).expand(shape)


FAR = [(BF16, -60, 43), (BF16, 60, 43), (BF16, -60, 66), (BF16, 60, 66), (F16, 15, 14), (F16, -15, 14), (F16, -12, 10),
       (BF16, 17, 0), (BF16, -17, 0)]


# (one magnitude a type for the widest workgroups)
FAR_EXPANDED = [(*shape, *far) for shape in ((1, 20, 20, 2), (2, 300, 300, 3), (1, 70, 2100, 2), (2, 150, 400, 1)) for far in FAR]
FAR_EXPANDED += [(8, 520, 520, 16, *far) for far in FAR if far[2] in (43, 14)]


@pytest.mark.parametrize("B,T,S,H,dtype,a,b", FAR_EXPANDED, ids=lambda x: str(x)[6:] if isinstance(x, torch.dtype) else str(x))
def test_expanded_far_scores(kda_pkg, B, T, S, H, dtype, a, b):
    """Scores of one sign and up to 2^126 in size, all far from zero: finite, so a row's largest takes the weight,
    shared evenly by the keys that have it.  The products are exact, and weights other than these below 2^-700."""
    N, P = 64, 32
    q, kn, pe, v = inputs(B, T, S, H, N, P, dtype, seed=90)
    q.zero_()
    q[..., 0] = float((1 if a > 0 else -1) * 2.0 ** abs(a))
    kn[..., 0] = (steps((B, S, H), 1) * 2.0 ** b).to(dtype)
    d_o = rand(B, T, H, N, seed=95, dtype=dtype)
    leaves = [x.requires_grad_() for x in (q, kn, pe, v)]
    o = kda_pkg.mla_expanded(q, kn, pe, v, scale=1.0)
    grads = torch.autograd.grad(o, leaves, d_o)
    with torch.no_grad():
        want, bound, ref = expanded_ref(q, kn, pe, v, [S] * B, [S - T] * B, 1.0, d_o)
    close("o", o, want, bound)
    for m, g in zip(("q", "k_nope", "k_pe", "v"), grads):
        r, e = ref[m]
        if torch.finfo(dtype).max < 1e5:                 # fp16: a bound past its largest value allows any
            inside = (r.abs() + e) < torch.finfo(dtype).max
            g, r, e = torch.where(inside, g.double(), 0), torch.where(inside, r, 0), torch.where(inside, e, 0)
        close("d" + m, g, r, e)


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("dtype,a,b", FAR, ids=lambda x: str(x)[6:] if isinstance(x, torch.dtype) else str(x))
@pytest.mark.parametrize("B,T,H,S", [(1, 1, 16, 100), (2, 3, 4, 1000), (70, 1, 16, 600)])
def test_absorbed_far_scores(kda_pkg, B, T, H, S, dtype, a, b, bits):
    R, P = 128, 32
    q = torch.zeros(B, T, H, R + P, dtype=dtype, device=DEV)
    q[..., R] = float((1 if a > 0 else -1) * 2.0 ** abs(a))
    rows = rand(B, S, R + P, seed=96, dtype=torch.float32)
    rows[..., R:] = 0
    rows[..., R] = (steps((B, S), 1) * 2.0 ** b).float()
    rows[..., 0] = 8.0                       # one latent scale: its logarithm is part of an 8-bit cache's scores
    cache, sc = (rows.to(dtype), None) if bits == 16 else quantised(rows, R)
    held = cache.double() if bits == 16 else dequantised(cache, sc, R)
    got = kda_pkg.mla_absorbed(q, cache, i32([S] * B), R, 1.0, cache_scale=sc)
    want, bound = absorbed_ref(q, held, [S] * B, R, 1.0)
    close("o", got, want, bound)


# ---- first queries before the first key -------------------------------------

@pytest.mark.parametrize("T,S", [(40, 16), (150, 20), (700, 90), (300, 299), (1200, 1100)])
def test_expanded_negative_starts_are_the_default(kda_pkg, T, S):
    """starts = S - T given is starts left out, in the output and the gradients, where that is below 0."""
    xs = [x.requires_grad_() for x in inputs(2, T, S, 2, 64, 32, BF16, seed=110)]
    d_o = rand(2, T, 2, 64, seed=115, dtype=BF16)

    def call(starts):
        o = kda_pkg.mla_expanded(*xs, starts=starts)
        return [o, *torch.autograd.grad(o, xs, d_o)]

    want = call(None)
    assert (want[0][:, :T - S] == 0).all() and (want[0][:, T - S:] != 0).any()
    for given in (i32([S - T] * 2), i32([S - T] * 2).long()):
        assert all(torch.equal(a, b) for a, b in zip(call(given), want))


@pytest.mark.parametrize("B,T,S,lengths,starts", [(3, 40, 16, [16, 9, 0], [-24, -3, -1]), (2, 300, 200, [200, 77], [-150, -299]),
                                                  (4, 70, 1100, [1100, 30, 1100, 5], [-1, -64, 1030, -2 ** 31])])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_expanded_negative_starts(kda_pkg, B, T, S, lengths, starts, dtype):
    H, N, P = 2, 64, 32
    q, kn, pe, v = inputs(B, T, S, H, N, P, dtype, seed=120)
    d_o = rand(B, T, H, N, seed=125, dtype=dtype)
    leaves = [x.requires_grad_() for x in (q, kn, pe, v)]
    o = kda_pkg.mla_expanded(q, kn, pe, v, lengths=i32(lengths), starts=i32(starts))
    grads = torch.autograd.grad(o, leaves, d_o)
    with torch.no_grad():
        want, bound, ref = expanded_ref(q, kn, pe, v, lengths, starts, (N + P) ** -0.5, d_o)
    close("o", o, want, bound)
    for m, g in zip(("q", "k_nope", "k_pe", "v"), grads):
        close("d" + m, g, *ref[m])


# ---- what looks on, and what would record -----------------------------------

def test_traces_and_transforms_are_refused(kda_pkg):
    """A trace would hold the outputs' memory without the kernels: every call under one raises, as do batching and
    forward-mode transforms; a mode that only looks on changes nothing."""
    import torch.autograd.forward_ad as fwd
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx
    from torch.utils.flop_counter import FlopCounterMode
    R, P = 128, 32
    q, kn, pe, v = inputs(1, 20, 20, 2, 64, 32, BF16, seed=130)
    qa, x, n = rand(1, 1, 2, R + P, seed=131, dtype=BF16), rand(1, 3, R + P, seed=132, dtype=BF16), i32([20])
    cache = rand(1, 40, R + P, seed=133, dtype=BF16)
    f8, sc = quantised(cache.float(), R)
    calls = {"expanded": (lambda t: kda_pkg.mla_expanded(t, kn, pe, v), q),
             "absorbed": (lambda t: kda_pkg.mla_absorbed(t, cache, n, R, 0.1), qa),
             "append": (lambda t: kda_pkg.mla_cache_append(t, cache, n, R) or t, x),
             "read": (lambda t: kda_pkg.mla_cache_read(t, sc, R), f8)}
    before = cache.clone()
    for name, (call, arg) in calls.items():
        with pytest.raises(kda_pkg.KdaError):
            make_fx(call)(arg)
        with pytest.raises(kda_pkg.KdaError):
            make_fx(call, pre_dispatch=True)(arg)
        with pytest.raises(kda_pkg.KdaError):
            torch.jit.trace(call, arg, check_trace=False)
        with pytest.raises(kda_pkg.KdaError):
            with FakeTensorMode(allow_non_fake_inputs=True):
                call(arg)
        with pytest.raises(kda_pkg.KdaError):
            torch.vmap(call)(torch.stack([arg, arg]))
        if name != "read":
            with fwd.dual_level(), pytest.raises(kda_pkg.KdaError):
                call(fwd.make_dual(arg, torch.ones_like(arg)))
            with pytest.raises(kda_pkg.KdaError):
                torch.func.grad(lambda t: call(t).float().sum())(arg)
    assert torch.equal(cache, before)
    leaf = q.clone().requires_grad_()
    o = kda_pkg.mla_expanded(leaf, kn, pe, v)
    with pytest.raises(kda_pkg.KdaError, match="traced"):
        make_fx(lambda g: torch.autograd.grad(o, leaf, g, retain_graph=True))(torch.ones_like(o))
    want, grad = o.detach(), torch.autograd.grad(o, leaf, torch.ones_like(o))[0]
    with FlopCounterMode(display=False):
        o = kda_pkg.mla_expanded(leaf, kn, pe, v)
        assert torch.equal(o, want) and torch.equal(torch.autograd.grad(o, leaf, torch.ones_like(o))[0], grad)
        for name in ("absorbed", "read"):
            call, arg = calls[name]
            got = call(arg)
            assert torch.isfinite(got.float()).all()
        calls["append"][0](x)
    assert not torch.equal(cache, before)


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("wtype", [torch.float32, torch.float64, BF16, F16])
def test_append_norm_weight_types(kda_pkg, wtype, dtype, bits):
    """A norm weight of another type than x's is not rounded to x's: fp32 arithmetic, and the cache's rounding."""
    B, T, S, R, P = 2, 5, 9, 256, 32
    x = rand(B, T, R + P, seed=140, dtype=dtype, std=2.0)
    w = (1 + rand(R, seed=141, std=0.3)).to(wtype)
    cache = torch.zeros(B, S, R + P, dtype=dtype if bits == 16 else F8, device=DEV)
    sc = None if bits == 16 else torch.ones(B, S, 2, device=DEV)
    kda_pkg.mla_cache_append(x, cache, i32([0, 3]), R, cache_scale=sc, norm_weight=w, eps=1e-5)
    y = x.double()
    y[..., :R] = y[..., :R] * torch.rsqrt(y[..., :R].square().mean(-1, keepdim=True) + 1e-5) * w.double()
    held = cache.double() if bits == 16 else dequantised(cache, sc, R)
    for b, at in enumerate((0, 3)):
        got, want = held[b, at:at + T], y[b]
        if bits == 16:          # one rounding, and fp32 arithmetic (2^-21)
            close("row", got, want, (half_step(dtype) + 2.0 ** -21) * want.abs())
        else:                   # half a step of e4m3, and the scale's arithmetic
            step = sc[b, at:at + T].double() * 2.0 ** -10
            step = torch.cat([step[:, :1].expand(T, R), step[:, 1:].expand(T, P)], -1)
            close("row", got, want, (2.0 ** -4 + 2.0 ** -20) * want.abs() + step)
            assert ((sc[b, at:at + T, 0].double() - want[:, :R].abs().amax(-1) / 448).abs()
                    <= 2.0 ** -20 * sc[b, at:at + T, 0]).all()


def test_expanded_refusals_under_grad(kda_pkg):
    """What the library refuses is reported alike with and without inputs that require grad."""
    for N, P, kw in ((96, 32, {}), (64, 16, {}), (64, 32, dict(scale=0.0)), (64, 32, dict(scale=float("nan")))):
        xs = inputs(1, 6, 6, 2, N, P, BF16, seed=145)
        said = []
        for grad in (False, True):
            with pytest.raises(kda_pkg.KdaError) as e:
                kda_pkg.mla_expanded(*(x.detach().requires_grad_(grad) for x in xs), **kw)
            said.append(str(e.value))
        assert said[0] == said[1]


def test_expanded_tokens_far_apart(kda_pkg):
    """Inputs and an output gradient whose tokens are 2^23 elements apart (a time-major batch's) are copied."""
    T, H, N, P = 5, 2, 64, 32
    xs = inputs(1, T, T, H, N, P, BF16, seed=150)
    d_o = rand(1, T, H, N, seed=155, dtype=BF16)

    def apart(x):
        row = x[0, 0].numel()
        far = torch.empty(T * 2 ** 23, dtype=BF16, device=DEV).as_strided((T, row), (2 ** 23, 1))
        far.copy_(x.reshape(T, row))
        return far.view(x.shape)

    def call(xs, d_o):
        xs = [x.detach().requires_grad_() for x in xs]
        o = kda_pkg.mla_expanded(*xs)
        return [o.detach(), *torch.autograd.grad(o, xs, d_o)]

    want = call(xs, d_o)
    far = [apart(x) for x in xs]
    assert all(f.stride(1) == 2 ** 23 for f in far)
    assert all(torch.equal(a, b) for a, b in zip(call(far, apart(d_o)), want))
    assert all(torch.equal(a, b) for a, b in zip(call(xs, apart(d_o)), want))


@pytest.mark.parametrize("B,T,S,lengths,starts", [(1, 40, 16, [16], [-24]), (2, 300, 200, [200, 60], [-100, -299]),
                                                  (4, 700, 600, [600, 600, 1, 0], [-100, 0, -500, -3]),
                                                  (3, 130, 130, [130, 60, 5], [0, 0, -70])])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_expanded_rows_that_see_no_key_are_not_read(kda_pkg, B, T, S, lengths, starts, dtype):
    """q and the output's gradient may hold anything in rows at positions below 0 and past the sequence's end: the
    rows' own results are zeros and nobody else's change."""
    H, N, P = 2, 64, 32
    q, kn, pe, v = inputs(B, T, S, H, N, P, dtype, seed=160)
    d_o = rand(B, T, H, N, seed=165, dtype=dtype)
    n, st = i32(lengths), i32(starts)
    pos = st[:, None] + torch.arange(T, device=DEV)
    none = (pos < 0) | (pos >= n[:, None])

    def call(q, d_o):
        xs = [x.detach().clone().requires_grad_() for x in (q, kn, pe, v)]
        o = kda_pkg.mla_expanded(*xs, lengths=n, starts=st)
        return [o.detach(), *torch.autograd.grad(o, xs, d_o)]

    want = call(q, d_o)
    for bad in (float("nan"), float("inf")):
        q2, d2 = q.clone(), d_o.clone()
        q2[none], d2[none] = bad, bad
        got = call(q2, d2)
        assert (got[0][none] == 0).all() and (got[1][none] == 0).all()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("k", [-30, -3, 0, 5])
def test_append_8bit_scale_of_all_ones(kda_pkg, k):
    """A scale of 24 one bits, (2 - 2^-23) 2^k, at which 2^-9 2^k over it is just past the tie below e4m3's smallest
    value: the quotient is the exactly rounded one there too."""
    R, P = 128, 0
    w = torch.zeros(R, device=DEV)
    w[0], w[1], w[2] = 895.99994 * 2.0 ** k, 2.0 ** -9 * 2.0 ** k, -2.0 ** -9 * 2.0 ** k
    cache, sc = torch.zeros(1, 1, R, dtype=F8, device=DEV), torch.zeros(1, 1, 2, device=DEV)
    # rows of ones: their norm is one, and what is quantised is the weight
    kda_pkg.mla_cache_append(torch.ones(1, 1, R, dtype=BF16, device=DEV), cache, i32([0]), R, cache_scale=sc,
                             norm_weight=w, eps=0.0)
    assert sc[0, 0, 0].item() == (2 - 2.0 ** -23) * 2.0 ** k
    assert cache[0, 0, :4].float().tolist() == [448.0, 2.0 ** -9, -2.0 ** -9, 0.0]


# ---- an 8-bit cache's scales ------------------------------------------------

@pytest.mark.parametrize("top", [66, 70, 100, 115])
@pytest.mark.parametrize("B,T,H,S,R,P", [(1, 1, 16, 2, 512, 64), (2, 3, 5, 130, 128, 32), (3, 1, 16, 3000, 512, 64), (40, 1, 16, 700, 256, 64)])
def test_absorbed_8bit_scales_far_apart(kda_pkg, B, T, H, S, R, P, top):
    """Scales from 2^-60, which rows of zeros have, to 2^115: the softmax's denominator goes by the scores alone."""
    g = torch.Generator(device=DEV).manual_seed(110 + S)
    rows = rand(B, S, R + P, seed=111, dtype=torch.float32)
    size = torch.tensor([0.0, 0.0, 1.0, 2.0 ** (top + 7)], device=DEV)[torch.randint(0, 4, (B, S), generator=g, device=DEV)]
    size[:, 0], size[:, 1] = 0.0, 2.0 ** (top + 7)
    rows[..., :R] *= size[..., None]
    cache, scale = quantised(rows, R)
    q = rand(B, T, H, R + P, seed=112, dtype=BF16, std=0.5)
    q[..., :R] = 0
    lengths = [max(S - 7 * b, 0) for b in range(B)]
    got = kda_pkg.mla_absorbed(q, cache, i32(lengths), R, 0.1, cache_scale=scale)
    close("o", got, *absorbed_ref(q, dequantised(cache, scale, R), lengths, R, 0.1))


@pytest.mark.parametrize("late", [False, True])
@pytest.mark.parametrize("dtype,a,b", FAR, ids=lambda x: str(x)[6:] if isinstance(x, torch.dtype) else str(x))
@pytest.mark.parametrize("B,T,H,S", [(1, 1, 16, 100), (2, 3, 4, 1000), (70, 1, 16, 600)])
def test_absorbed_8bit_far_scores_and_scales(kda_pkg, B, T, H, S, dtype, a, b, late):
    """Scores of up to 2^126 in size over rows of different latent scales: the keys that share the largest share the
    weight, whatever their scales.  late: the far scores come behind keys whose scores are zero."""
    R, P = 128, 32
    q = torch.zeros(B, T, H, R + P, dtype=dtype, device=DEV)
    q[..., R] = float((1 if a > 0 else -1) * 2.0 ** abs(a))
    rows = rand(B, S, R + P, seed=113, dtype=torch.float32)
    span = 6 if dtype == F16 else 40
    rows[..., :R] *= torch.exp2(rand(B, S, 1, seed=114, dtype=torch.float32).clamp(-1, 1) * span)
    rows[..., R:] = 0
    rows[..., R] = (steps((B, S), 1) * 2.0 ** b).float()
    if late:
        rows[:, :S // 2, R] = 0
    cache, scale = quantised(rows, R)
    got = kda_pkg.mla_absorbed(q, cache, i32([S] * B), R, 1.0, cache_scale=scale)
    close("o", got, *absorbed_ref(q, dequantised(cache, scale, R), [S] * B, R, 1.0))
