"""4-bit weights against their definition in float64.

A product's bound per element: the result's own rounding (u = half a step of the
type, of the value) and K fp32 additions (K 2^-24 of the sum of magnitudes; the
weights are exact in the activation type, so the products are exact in fp32 but
for that), and fp16's smallest step.
"""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
VALUES = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def rand(*shape, seed, dtype=torch.float64, std=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(*shape, device=DEV, generator=g, dtype=torch.float64) * std).to(dtype)


def raw(t):
    return t if t.dtype == torch.uint8 else t.view(torch.uint8)


def values(data, scale):
    """The matrix [.., K] in float64; NaN where the scale is 255."""
    data, e = raw(data), raw(scale).double()
    v = torch.tensor(VALUES + [-x for x in VALUES], dtype=torch.float64, device=data.device)
    v = v[torch.stack([data % 16, data // 16], -1).flatten(-2).long()]
    p = torch.where(e == 255, torch.nan, torch.exp2(e - 127))
    return v * p.repeat_interleave(32, -1)


def definition(w, group=32, least=-126):
    """(codes [.., K], exponents + 127) of w in float64: by comparing with every power and every border."""
    g = w.double().unflatten(-1, (-1, group))
    top = g.abs().amax(-1, keepdim=True)
    powers = torch.exp2(torch.arange(least, 128, dtype=torch.float64, device=w.device))
    at = (top > 7 * powers).sum(-1)                        # the least power that leaves at most 7
    q = g / powers[at.clamp(max=powers.numel() - 1)][..., None]
    v = torch.tensor(VALUES, dtype=torch.float64, device=w.device)
    borders = (v[1:] + v[:-1]) / 2
    a = q.abs()[..., None]
    even = torch.arange(7, device=w.device) % 2 == 1       # a border below an even code belongs to that code
    code = ((a > borders) | ((a == borders) & even)).sum(-1)
    sign = torch.signbit(g)
    return (code + 8 * sign).flatten(-2), at + least + 127


def check(y, x, w, extra=None):
    x, w = x.double(), w.double()
    ref, mag = x @ w.t(), x.abs() @ w.abs().t()
    if extra is not None:
        ref, mag = ref + extra.double(), mag + extra.double().abs()
    bound = torch.finfo(y.dtype).eps / 2 * ref.abs() + (x.shape[-1] + 1) * 2.0 ** -24 * mag + 2.0 ** -24
    assert y.shape == ref.shape and bool(((y.double() - ref).abs() <= bound).all())


# ---- conversions ------------------------------------------------------------

@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("shape", [(1, 32), (7, 96), (3, 5, 64), (300, 2080), (64,)], ids=str)
def test_quantize(kda_pkg, shape, dtype):
    w = rand(*shape, seed=1) * torch.exp2(rand(*shape[:-1], 1, seed=2, std=4.0))
    if len(shape) > 1:
        w[0, ...] = 0
        w[-1, ..., :32] = torch.tensor(VALUES + [0.25, -0.25, 0.75, -0.75, 1.25, -1.25, 1.75, 2.5, 3.5, -3.5, 5, -5, 7, -6.5,
                                                 6.99, 0.26, 0.24, -2.51, -2.49, 0, 0, 0, 1, 1], device=DEV)
    w = w.to(dtype)
    data, scale = kda_pkg.mx4_quantize(w)
    assert data.dtype == torch.float4_e2m1fn_x2 and scale.dtype == torch.float8_e8m0fnu
    assert data.shape == (*shape[:-1], shape[-1] // 2) and scale.shape == (*shape[:-1], shape[-1] // 32)
    code, e = definition(w)
    got = torch.stack([raw(data) % 16, raw(data) // 16], -1).flatten(-2)
    assert torch.equal(raw(scale).long(), e)
    assert torch.equal(got.long() % 8, code % 8)
    assert torch.equal(got.long()[code % 8 > 0], code[code % 8 > 0])             # the sign of what is not zero
    back = kda_pkg.mx4_dequantize(data, scale, dtype=BF16 if dtype == F32 else dtype)
    assert torch.equal(back.double(), values(data, scale).to(back.dtype).double())
    again = kda_pkg.mx4_quantize(back)                                          # what it stands for stays what it is
    assert torch.equal(kda_pkg.mx4_dequantize(*again, dtype=back.dtype), back)


def test_quantize_borders(kda_pkg):
    """fp32 values next to each border, at powers over the whole range: the quotient is exact."""
    b = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    lo, hi = torch.nextafter(b, torch.zeros(7)), torch.nextafter(b, torch.full((7,), 9.0))
    row = torch.cat([lo, b, hi, torch.tensor([7.0]), torch.zeros(10)]).to(DEV)
    w = torch.stack([row * 2.0 ** n for n in (-120, -60, -9, 0, 3, 60, 124)])
    for x in (w, -w, w * (6.0 / 7)):
        data, scale = kda_pkg.mx4_quantize(x)
        code, e = definition(x)
        got = torch.stack([raw(data) % 16, raw(data) // 16], -1).flatten(-2).long()
        assert torch.equal(raw(scale).long(), e) and torch.equal(got % 8, code % 8)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_quantize_ends_of_the_range(kda_pkg, dtype):
    """The largest values, the smallest, and what is not finite, which its neighbours do not notice."""
    w = torch.zeros(6, 64, dtype=dtype, device=DEV)
    w[0] = torch.finfo(dtype).max
    w[1] = torch.finfo(dtype).tiny * torch.finfo(dtype).eps                      # the smallest subnormal number
    w[2] = torch.finfo(dtype).tiny
    w[3:, 32:] = 1.0
    w[3, 5], w[4, 31], w[5, 0] = float("inf"), float("nan"), -float("inf")
    data, scale = kda_pkg.mx4_quantize(w)
    code, e = definition(w[:3])
    got = torch.stack([raw(data) % 16, raw(data) // 16], -1).flatten(-2).long()
    assert torch.equal(raw(scale)[:3].long(), e) and torch.equal(got[:3] % 8, code % 8)
    assert (raw(scale)[3:, 0] == 255).all() and (raw(scale)[3:, 1] == 125).all()
    back = kda_pkg.mx4_dequantize(data, scale, dtype=BF16)
    assert back[3:, :32].isnan().all() and (back[3:, 32:] == 1).all()


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_dequantize_every_byte(kda_pkg, dtype):
    """Every pair of values times every scale, rounded once as the type rounds."""
    data = torch.arange(256, dtype=torch.uint8, device=DEV).view(1, 16, 16).repeat(256, 1, 1)
    scale = torch.arange(256, dtype=torch.uint8, device=DEV).view(256, 1, 1).repeat(1, 16, 1)
    got = kda_pkg.mx4_dequantize(data, scale, dtype=dtype)
    want = values(data, scale).to(dtype)
    assert got.shape == (256, 16, 32) and torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.nan_to_num(nan=0.0), want.nan_to_num(nan=0.0))


def test_layouts(kda_pkg):
    """Strided, transposed, unaligned and empty inputs; bytes or the format's own types."""
    big = rand(9, 6, 160, seed=3, dtype=F16)
    for w in (big[::2, :, 16:112], big[:, 1:3, :64], big.transpose(0, 1)[..., :32], big[..., 3:67], big[:1, :1, 32:64],
              big[:, 0, ::5][:, :32], big.expand(9, 6, 160)[:, :, :32], big[:0, :, :64]):
        data, scale = kda_pkg.mx4_quantize(w)
        want = kda_pkg.mx4_quantize(w.contiguous())
        assert torch.equal(raw(data), raw(want[0])) and torch.equal(raw(scale), raw(want[1]))
        got = kda_pkg.mx4_dequantize(raw(data).transpose(0, 1).contiguous().transpose(0, 1), raw(scale), dtype=F16)
        assert torch.equal(got, kda_pkg.mx4_dequantize(data, scale, dtype=F16))


# ---- the product ------------------------------------------------------------

def weight(kda_pkg, N, K, seed, std=1.0):
    data, scale = kda_pkg.mx4_quantize(rand(N, K, seed=seed, std=std * K ** -0.5, dtype=F32))
    return data, scale, values(data, scale)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("M", [1, 7, 16, 17, 33, 64, 65, 128, 200, 333])
@pytest.mark.parametrize("K,N", [(2048, 6416), (32, 16), (64, 1), (96, 47), (128, 2048), (544, 130), (1024, 17), (1152, 257),
                                 (4096, 576), (2080, 1003)])
def test_linear(kda_pkg, M, K, N, dtype):
    """Row and column tile edges, depths that end inside a chunk, rows of a longer buffer that hold NaN."""
    data, scale, w = weight(kda_pkg, N, K, seed=4)
    x = rand(M, K, seed=5, dtype=dtype)
    big = torch.full((M + 1, K + 24), float("nan"), dtype=dtype, device=DEV)
    big[:M, 8:K + 8] = x
    y = kda_pkg.mx4_linear(big[:M, 8:K + 8], data, scale)
    check(y, x, w)
    assert torch.equal(y, kda_pkg.mx4_linear(x, raw(data), raw(scale)))
    bias, res = rand(N, seed=6, dtype=dtype), rand(M, N, seed=7, dtype=dtype, std=3.0)
    z = kda_pkg.mx4_linear(x, data, scale, bias=bias)
    check(z, x, w, bias)
    assert torch.equal(kda_pkg.mx4_linear(x, data, scale, residual=res), res + y)
    assert torch.equal(kda_pkg.mx4_linear(x, data, scale, bias=bias, residual=res), res + z)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("M,N,K", [
    (1, 600, 9248), (16, 5000, 9248), (3, 11000, 4640), (2, 14000, 4640), (9, 14000, 4640), (4, 33000, 2080),      # up to 16 rows
    (20, 300, 9248), (20, 9000, 4640), (50, 300, 9248), (50, 5000, 9248), (50, 9000, 4640), (50, 30000, 1056)], ids=str)
def test_linear_deep_and_wide(kda_pkg, M, N, K, dtype):
    """Every tile of few rows at a depth at which each wave comes round again, and a last chunk of one group."""
    data, scale, w = weight(kda_pkg, N, K, seed=8)
    x = rand(M, K, seed=9, dtype=dtype)
    y = kda_pkg.mx4_linear(x, data, scale)
    check(y, x, w)
    for _ in range(2):
        assert torch.equal(y, kda_pkg.mx4_linear(x, data, scale))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("M,N,K", [(5000, 5003, 96), (4999, 5002, 64), (700, 2001, 160), (129, 6405, 288), (65, 8198, 32)], ids=str)
def test_linear_odd_widths(kda_pkg, M, N, K, dtype):
    """Rows of outputs that begin at any multiple of two bytes, in every tile of many rows."""
    data, scale, w = weight(kda_pkg, N, K, seed=50)
    x, bias = rand(M, K, seed=51, dtype=dtype), rand(N, seed=52, dtype=dtype)
    res = rand(M, N + 3, seed=53, dtype=dtype, std=3.0)[:, 1:N + 1]
    y = kda_pkg.mx4_linear(x, data, scale)
    check(y, x, w)
    z = kda_pkg.mx4_linear(x, data, scale, bias=bias)
    check(z, x, w, bias)
    assert torch.equal(kda_pkg.mx4_linear(x, data, scale, residual=res), res + y)
    assert torch.equal(kda_pkg.mx4_linear(x, data, scale, bias=bias, residual=res), res + z)


@pytest.mark.parametrize("M", [1, 20, 50, 130, 700])
@pytest.mark.parametrize("K", [64, 288, 4096])
def test_not_finite(kda_pkg, M, K):
    """What is not finite stays in its row of x or its row of the weight, and an infinity stays one."""
    N = 150
    data, scale, w = weight(kda_pkg, N, K, seed=8)
    x = rand(M, K, seed=9, dtype=BF16)
    want = kda_pkg.mx4_linear(x, data, scale)
    bad = x.clone()
    bad[M // 2, K - 1] = float("inf")                      # the last channel: chunks end behind it
    got = kda_pkg.mx4_linear(bad, data, scale)
    rest = torch.arange(M, device=DEV) != M // 2
    assert torch.equal(got[rest], want[rest])
    sign = torch.sign(w[:, K - 1])
    row = got[M // 2].float()
    assert (row[sign > 0] == float("inf")).all() and (row[sign < 0] == -float("inf")).all() and row[sign == 0].isnan().all()
    s = raw(scale).clone()
    s[N - 1, -1] = 255
    got = kda_pkg.mx4_linear(x, data, s)
    assert got[:, N - 1].isnan().all() and torch.equal(got[:, :N - 1], want[:, :N - 1])


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_scales_of_any_size(kda_pkg, dtype):
    """Powers from 2^-23 to 2^13 beside each other (exact in both types), and in bf16 over nearly all of the range."""
    K, N, M = 256, 37, 5
    g = torch.Generator(device=DEV).manual_seed(10)
    data = torch.randint(0, 256, (N, K // 2), generator=g, device=DEV, dtype=torch.uint8)
    lo, hi = (-23, 14) if dtype == F16 else (-100, 101)
    scale = (torch.randint(lo, hi, (N, 1), generator=g, device=DEV) + 127).to(torch.uint8).repeat(1, K // 32)
    scale[::2] = (torch.randint(lo, hi, (N, K // 32), generator=g, device=DEV) + 127).to(torch.uint8)[::2]
    x = rand(M, K, seed=11, dtype=dtype, std=2.0 ** -6)
    y = kda_pkg.mx4_linear(x, data, scale)
    ref, mag = x.double() @ values(data, scale).t(), x.double().abs() @ values(data, scale).abs().t()
    ok = mag < torch.finfo(dtype).max / 2
    bound = torch.finfo(dtype).eps / 2 * ref.abs() + K * 2.0 ** -24 * mag + (2.0 ** -25 if dtype == F16 else 0)
    assert ok.float().mean() > 0.5 and ((y.double() - ref).abs() <= bound)[ok].all()


def test_shapes_and_layouts(kda_pkg):
    K, N = 160, 40
    data, scale, w = weight(kda_pkg, N, K, seed=12)
    big = rand(4, 6, 192, seed=13, dtype=F16)
    for x in (big[..., :K], big[:, 2, 8:K + 8], big[1, 2, :K], big.transpose(0, 1)[..., :K], big[::2, ::3, 16:K + 16],
              big[..., 1:K + 1], big[:0, :, :K], big[:, :1, :K].expand(4, 5, K), big[:1, :1, :K]):
        y = kda_pkg.mx4_linear(x, data, scale)
        assert y.shape == (*x.shape[:-1], N)
        check(y.reshape(-1, N), x.reshape(-1, K), w)
        res = rand(*x.shape[:-1], 2 * N, seed=14, dtype=F16)[..., ::2]
        assert torch.equal(kda_pkg.mx4_linear(x, data, scale, residual=res), res + y)
    assert kda_pkg.mx4_linear(big[..., :K], raw(data)[:0], raw(scale)[:0]).shape == (4, 6, 0)
    odd = torch.empty(N * K // 2 + 3, dtype=torch.uint8, device=DEV)[3:].view(N, K // 2).copy_(raw(data))      # unaligned bytes
    assert torch.equal(kda_pkg.mx4_linear(big[..., :K], odd, scale), kda_pkg.mx4_linear(big[..., :K], data, scale))


@pytest.mark.parametrize("M", [3, 100])
def test_far_rows(kda_pkg, M):
    """Weights past 2^32 bytes, and rows of x far apart."""
    K, N = 2 ** 16, 2 ** 17 + 16
    data = torch.zeros(N, K // 2, dtype=torch.uint8, device=DEV)
    scale = torch.full((N, K // 32), 127, dtype=torch.uint8, device=DEV)
    x = rand(M, K, seed=15, dtype=BF16)
    at = [0, 1, 2 ** 16 + 5, 2 ** 17 - 1, N - 1]
    data[at] = torch.randint(0, 256, (5, K // 2), device=DEV, dtype=torch.uint8, generator=torch.Generator(device=DEV).manual_seed(16))
    y = kda_pkg.mx4_linear(x, data, scale)
    check(y[:, at], x, values(data[at], scale[at]))
    rest = torch.ones(N, dtype=torch.bool, device=DEV)
    rest[at] = False
    assert (y[:, rest] == 0).all()
    del data, scale
    far = torch.empty((M - 1) * 2 ** 23 + 64, dtype=BF16, device=DEV).as_strided((M, 64), (2 ** 23, 1))
    far.copy_(x[:, :64])
    data, scale, w = weight(kda_pkg, 24, 64, seed=17)
    check(kda_pkg.mx4_linear(far, data, scale), x[:, :64], w)


@pytest.mark.parametrize("M", [1, 33, 150])
def test_captured_and_on_another_stream(kda_pkg, M):
    K, N = 1024, 500
    data, scale, w = weight(kda_pkg, N, K, seed=18)
    x, res = rand(M, K, seed=19, dtype=BF16), rand(M, N, seed=20, dtype=BF16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = kda_pkg.mx4_linear(x, data, scale)
        q = kda_pkg.mx4_quantize(x)
    torch.cuda.current_stream().wait_stream(side)
    check(y, x, w)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        z = kda_pkg.mx4_linear(x, data, scale, residual=res)
        z2 = kda_pkg.mx4_dequantize(*kda_pkg.mx4_quantize(x), dtype=BF16)
    assert torch.equal(kda_pkg.mx4_dequantize(*q, dtype=BF16), kda_pkg.mx4_dequantize(*kda_pkg.mx4_quantize(x), dtype=BF16))
    for i in range(3):
        x.copy_(rand(M, K, seed=30 + i, dtype=BF16))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(z, res + kda_pkg.mx4_linear(x, data, scale))
        assert torch.equal(z2, kda_pkg.mx4_dequantize(*kda_pkg.mx4_quantize(x), dtype=BF16))


def test_refusals(kda_pkg):
    err, K, N = kda_pkg.KdaError, 64, 16
    data, scale, w = weight(kda_pkg, N, K, seed=21)
    x = rand(2, K, seed=22, dtype=F16)
    vec = torch.zeros(N, dtype=F16, device=DEV)
    bad = [
        lambda: kda_pkg.mx4_linear(x.float(), data, scale),
        lambda: kda_pkg.mx4_linear(x.cpu(), data, scale),
        lambda: kda_pkg.mx4_linear(x, raw(data).cpu(), scale),
        lambda: kda_pkg.mx4_linear(x, data, raw(scale).cpu()),
        lambda: kda_pkg.mx4_linear(x[:, :32], data, scale),
        lambda: kda_pkg.mx4_linear(x, raw(data).int(), scale),
        lambda: kda_pkg.mx4_linear(x, data, raw(scale).float()),
        lambda: kda_pkg.mx4_linear(x, data, raw(scale)[:, :1]),
        lambda: kda_pkg.mx4_linear(x, raw(data).view(1, N, -1), raw(scale).view(1, N, -1)),
        lambda: kda_pkg.mx4_linear(x, data, scale, bias=vec[:-1]),
        lambda: kda_pkg.mx4_linear(x, data, scale, residual=vec),
        lambda: kda_pkg.mx4_linear(x, data, scale, bias=vec.cpu()),
        lambda: kda_pkg.mx4_linear(x.clone().requires_grad_(), data, scale),
        lambda: kda_pkg.mx4_linear(x, data, scale, bias=vec.clone().requires_grad_()),
        lambda: kda_pkg.mx4_quantize(x[:, :48]),
        lambda: kda_pkg.mx4_quantize(x[:, :0]),
        lambda: kda_pkg.mx4_quantize(x.double()),
        lambda: kda_pkg.mx4_quantize(x.clone().requires_grad_()),
        lambda: kda_pkg.mx4_quantize(x[0, 0]),
        lambda: kda_pkg.mx4_dequantize(data, scale, dtype=F32),
        lambda: kda_pkg.mx4_dequantize(data, raw(scale)[:-1]),
        lambda: torch.vmap(lambda r: kda_pkg.mx4_linear(r, data, scale))(x),
        lambda: torch.vmap(kda_pkg.mx4_quantize)(x),
        lambda: torch.jit.trace(lambda r: kda_pkg.mx4_linear(r, data, scale), x),
        lambda: torch.func.jvp(lambda r: kda_pkg.mx4_linear(r, data, scale), (x,), (x,)),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(err):
            call()
            pytest.fail(f"call {i} was answered")
    with torch.no_grad():
        assert kda_pkg.mx4_linear(x.clone().requires_grad_(), data, scale).requires_grad is False


def test_autocast(kda_pkg):
    """As a projection in 16 bits: x is taken in autocast's type."""
    data, scale, w = weight(kda_pkg, 48, 128, seed=23)
    x = rand(5, 128, seed=24, dtype=F32)
    with torch.autocast("cuda", dtype=BF16):
        y = kda_pkg.mx4_linear(x, data, scale)
    assert y.dtype == BF16 and torch.equal(y, kda_pkg.mx4_linear(x.to(BF16), data, scale))


def test_outputs_are_ordinary_tensors(kda_pkg):
    """Of torch's own memory: counted, freed, resizable, usable by autograd unless made under inference mode."""
    data, scale, _ = weight(kda_pkg, 64, 256, seed=60)
    x = rand(3000, 256, seed=61, dtype=F16)
    held = torch.cuda.memory_allocated()
    made = [kda_pkg.mx4_linear(x, data, scale), kda_pkg.mx4_dequantize(data, scale, dtype=F16), *kda_pkg.mx4_quantize(x)]
    assert torch.cuda.memory_allocated() >= held + sum(t.numel() * t.element_size() for t in made)
    for t in made:
        assert t.device == x.device == t.untyped_storage().device and t.is_contiguous() and t._version == 0
        assert not t.requires_grad and not t.is_inference() and t.untyped_storage().resizable()
    w = made[0].detach().requires_grad_()
    w.float().sum().backward()
    assert torch.equal(w.grad, torch.ones_like(w))
    with torch.inference_mode():
        assert kda_pkg.mx4_linear(x, data, scale).is_inference()
    del made, t, w
    assert torch.cuda.memory_allocated() == held


@pytest.mark.parametrize("bias", [False, True])
def test_module(kda_pkg, bias):
    lin = torch.nn.Linear(256, 70, bias=bias).to(DEV, F16)
    mod = kda_pkg.Mx4Linear.from_linear(lin)
    data, scale = kda_pkg.mx4_quantize(lin.weight.detach())
    assert torch.equal(mod.weight, raw(data)) and torch.equal(mod.weight_scale, raw(scale))
    x = rand(2, 3, 256, seed=25, dtype=F16)
    check(mod(x).view(6, 70), x.view(6, 256), values(data, scale), lin.bias if bias else None)
    with torch.inference_mode():
        made = kda_pkg.Mx4Linear.from_linear(lin)
    assert torch.equal(made(x), mod(x)) and not made.weight.is_inference()


@pytest.mark.parametrize("K,N,dtype", [(32, 8, BF16), (64, 5, F16)])
def test_linear_most_rows(kda_pkg, K, N, dtype):
    """More rows than one launch's grid reaches in its second dimension, and the rows about that border."""
    data, scale, w = weight(kda_pkg, N, K, seed=70)
    border = 65535 * 64
    M = border + 200
    x = rand(1, K, seed=71, dtype=dtype).expand(M, K).contiguous()
    at = torch.tensor([0, 1, 5000, border - 1, border, border + 1, border + 130, M - 1], device=DEV)
    x[at] = rand(len(at), K, seed=72, dtype=dtype)
    res, bias = torch.ones(M, N + 3, dtype=dtype, device=DEV)[:, :N], rand(N, seed=73, dtype=dtype)
    y = kda_pkg.mx4_linear(x, data, scale, bias=bias, residual=res)
    z = kda_pkg.mx4_linear(x[at], data, scale, bias=bias)
    check(z, x[at], w, bias)
    assert torch.equal(y[at], res[at] + z)
    rest = torch.ones(M, dtype=torch.bool, device=DEV)
    rest[at] = False
    same = kda_pkg.mx4_linear(x[2:3], data, scale, bias=bias) + 1
    assert torch.equal(y[rest], same.expand(M - len(at), N))


@pytest.mark.parametrize("dtype,top", [(BF16, 125), (F16, 13)])
def test_exact_scales(kda_pkg, dtype, top):
    """Where a value times its scale is exact, and what is beyond: from the largest values whose group's power
    passes that, infinity."""
    least = -125 if dtype == BF16 else -23
    scale = (torch.arange(least, top + 1, device=DEV) + 127).to(torch.uint8)[:, None]
    data = torch.arange(16, dtype=torch.uint8, device=DEV).mul(17).expand(scale.shape[0], 16).contiguous()
    back = kda_pkg.mx4_dequantize(data, scale, dtype=dtype)
    assert torch.equal(back.double(), values(data, scale))
    w = torch.full((2, 32), torch.finfo(dtype).max, dtype=dtype, device=DEV)
    w[1] = 1.75 * 2.0 ** (top + 2)                           # 7 of the largest such power: taken as 6
    data, scale = kda_pkg.mx4_quantize(w)
    assert raw(scale).flatten().tolist() == [top + 1 + 127, top + 127]
    back = kda_pkg.mx4_dequantize(data, scale, dtype=dtype)
    assert (back[0] == float("inf")).all() and (back[1].double() == 6 * 2.0 ** top).all()
    x = torch.zeros(1, 32, dtype=dtype, device=DEV)
    x[0, 0] = 2.0 ** -10
    y = kda_pkg.mx4_linear(x, data, scale)[0]
    assert y[0].isnan() and y[1].item() == 6 * 2.0 ** (top - 10)         # (x's zeros times infinity; one product)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("M,N,K", [(1400, 5003, 1056), (1401, 5002, 1024), (1399, 5016, 1152), (1281, 5441, 1024), (2500, 5121, 1088),
                                   (2700, 6144, 1024), (1400, 5003, 992)], ids=str)
def test_linear_large_tiles(kda_pkg, M, N, K, dtype):
    """Products deep enough for the largest tiles, whose rounds are full (and one each that is not, and not deep enough),
    at widths of every alignment."""
    data, scale, w = weight(kda_pkg, N, K, seed=80)
    x, bias = rand(M, K, seed=81, dtype=dtype), rand(N, seed=82, dtype=dtype)
    res = rand(M, N + 3, seed=83, dtype=dtype, std=3.0)[:, 1:N + 1]
    y = kda_pkg.mx4_linear(x, data, scale)
    check(y, x, w)
    z = kda_pkg.mx4_linear(x, data, scale, bias=bias)
    check(z, x, w, bias)
    assert torch.equal(kda_pkg.mx4_linear(x, data, scale, residual=res), res + y)
    assert torch.equal(kda_pkg.mx4_linear(x, data, scale, bias=bias, residual=res), res + z)
    few = kda_pkg.mx4_linear(x[-70:], data, scale)
    check(few, x[-70:], w)
