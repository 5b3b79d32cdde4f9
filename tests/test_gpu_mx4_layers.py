"""The layers with projections and caches in 4 bits.

A layer whose projections are in 4 bits is the layer with the weights that they
stand for (exact in bf16 and, at these sizes, in fp16), summed in another order:
the tolerances are those of the 16-bit layers against their restatements, relative
L2 norms.  The two forms of latent attention over one 4-bit cache see the same rows.
"""

from __future__ import annotations

import copy

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF16, F16 = torch.bfloat16, torch.float16
FOUR = torch.float4_e2m1fn_x2
TOL = {BF16: 2e-2, F16: 5e-3}


def rel(a, b):
    a, b = a.detach().double(), b.detach().double()
    return ((a - b).norm() / b.norm()).item()


def kda_layer(kda_pkg, dtype, seed=0, **kw):
    torch.manual_seed(seed)
    cfg = kda_pkg.linear_attn_config(**{**dict(hidden_size=256, num_heads=2, gate_low_rank=32, output_gate_low_rank=32), **kw})
    return kda_pkg.KimiDeltaAttention(cfg).to(DEV, dtype).eval()


def latent_layer(kda_pkg, dtype, seed=0, **kw):
    torch.manual_seed(seed)
    cfg = kda_pkg.latent_attn_config(**{**dict(hidden_size=256, num_heads=4, head_dim=64, position_dim=32, rank=128,
                                               max_tokens=96), **kw})
    return kda_pkg.LatentAttention(cfg).to(DEV, dtype).eval()


def stands_for(kda_pkg, layer):
    """The layer in 16 bits with the weights of its 4-bit projections."""
    new = copy.deepcopy(layer)
    for name, m in layer.named_children():
        if isinstance(m, kda_pkg.Mx4Linear):
            lin = torch.nn.Linear(m.in_features, m.out_features, bias=m.bias is not None, device=DEV, dtype=layer.beta_proj.weight.dtype
                                  if hasattr(layer, "beta_proj") else layer.kv_up.weight.dtype)
            with torch.no_grad():
                lin.weight.copy_(kda_pkg.mx4_dequantize(m.weight, m.weight_scale, dtype=lin.weight.dtype))
                if m.bias is not None:
                    lin.bias.copy_(m.bias)
            setattr(new, name, lin)
    new._wcat = None
    return new


def cached(layer, x, pieces):
    out, state, at = [], None, 0
    for n in pieces:
        y, state = layer(x[:, at:at + n], state=state, use_cache=True)
        out.append(y)
        at += n
    return torch.cat(out, 1), state


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("kw", [{}, dict(proj_bias=True), dict(num_heads=4, head_dim=64, value_head_dim=128)], ids=str)
@torch.no_grad()
def test_kda_layer(kda_pkg, dtype, kw):
    layer = kda_layer(kda_pkg, dtype, **kw)
    before = layer(torch.ones(1, 3, 256, device=DEV, dtype=dtype))
    assert layer.quantize_mx4_() is layer and layer.quantize_mx4_() is layer
    same = stands_for(kda_pkg, layer)
    assert not torch.equal(layer(torch.ones(1, 3, 256, device=DEV, dtype=dtype)), before)
    x = torch.randn(3, 130, 256, device=DEV).to(dtype)
    assert rel(layer(x), same(x)) <= TOL[dtype]
    got, state = cached(layer, x, (70, 5, *[1] * 6))
    want, wstate = cached(same, x, (70, 5, *[1] * 6))
    assert rel(got, want) <= TOL[dtype] and rel(state["recurrent"], wstate["recurrent"]) <= TOL[dtype]
    y = layer.decode_step_(x[:, 81:82], state)
    assert rel(y, same.decode_step_(x[:, 81:82], wstate)) <= TOL[dtype]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("kw", [{}, dict(proj_bias=True), dict(rank=256, position_dim=0)], ids=str)
@pytest.mark.parametrize("cache_dtype", [None, FOUR])
@torch.no_grad()
def test_latent_layer(kda_pkg, dtype, kw, cache_dtype):
    layer = latent_layer(kda_pkg, dtype, cache_dtype=cache_dtype, **kw)
    layer.quantize_mx4_()
    same = stands_for(kda_pkg, layer)
    x = torch.randn(2, 80, 256, device=DEV).to(dtype)
    assert rel(layer(x), same(x)) <= TOL[dtype]
    if cache_dtype is None:          # (over a 4-bit cache a row of a sum next to a border moves by a whole step)
        assert rel(cached(layer, x, (50, 20, 1, 1, 1))[0], cached(same, x, (50, 20, 1, 1, 1))[0]) <= TOL[dtype]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("mx4", [False, True])
@torch.no_grad()
def test_latent_cache(kda_pkg, dtype, mx4):
    """Single tokens through the absorbed form give what the expanded form gives over the rows read back; a cache
    that is full is refused before anything is written."""
    layer = latent_layer(kda_pkg, dtype, cache_dtype=FOUR)
    if mx4:
        layer.quantize_mx4_()
    x = torch.randn(2, 96, 256, device=DEV).to(dtype)
    out, state = layer(x[:, :50], use_cache=True)
    assert state["latent"].dtype == FOUR and state["latent"].shape == (2, 96, 80)
    assert state["scale"].dtype == torch.float8_e8m0fnu and state["scale"].shape == (2, 96, 8)
    out, state = layer(x[:, 50:83], state=state, use_cache=True)
    rows = layer._held(state, 83, dtype)
    assert torch.equal(out, layer._expanded(x[:, 50:83], rows))
    for t in range(83, 96):
        out, state = layer(x[:, t:t + 1], state=state, use_cache=True)
        assert rel(out, layer._expanded(x[:, t:t + 1], layer._held(state, t + 1, dtype))) <= TOL[dtype]
    assert state["tokens"] == 96 and state["lengths"].tolist() == [96, 96]
    held = state["latent"].view(torch.uint8).clone()
    for call in (lambda: layer(x[:, :1], state=state, use_cache=True), lambda: layer.decode_step_(x[:, :1], state),
                 lambda: layer(x[:, :5], state=state, use_cache=True)):
        with pytest.raises(kda_pkg.KdaError, match="96"):
            call()
    assert torch.equal(state["latent"].view(torch.uint8), held)


def stack(kda_pkg, dtype):
    layers = [kda_layer(kda_pkg, dtype, seed=3), latent_layer(kda_pkg, dtype, seed=4, cache_dtype=FOUR),
              kda_layer(kda_pkg, dtype, seed=5, proj_bias=True)]
    return [m.quantize_mx4_() for m in layers]


@pytest.mark.parametrize("residual", [True, False])
@torch.no_grad()
def test_stack_captured(kda_pkg, residual):
    """Every replayed step is the eager layers', bit for bit, with prompts that reuse the capture."""
    from kimi_linear_amd.graph_decode import KdaGraphedDecoder
    layers = stack(kda_pkg, F16)
    x = torch.randn(2, 90, 256, device=DEV).half()
    dec = KdaGraphedDecoder(layers, residual=residual)
    graph = None
    for n, steps in ((40, 9), (61, 12), (5, 3)):
        h = dec.prefill(x[:, :n])
        assert graph is None or dec.graph is graph
        graph = dec.graph
        states, y = [None] * 3, x[:, :n]
        for i, layer in enumerate(layers):
            out, states[i] = layer(y, use_cache=True)
            y = y + out if residual else out
        assert torch.equal(h, y[:, -1])
        for t in range(n, n + steps):
            got = dec.step(x[:, t:t + 1]).clone()
            y = x[:, t:t + 1]
            for i, layer in enumerate(layers):
                out, states[i] = layer(y, state=states[i], use_cache=True)
                y = y + out if residual else out
            torch.cuda.synchronize()
            assert torch.equal(got, y[:, 0]), (n, t)


@torch.no_grad()
def test_weights_change(kda_pkg):
    """Other weights loaded in place, and layers turned to 4 bits after a capture, are what the next step runs."""
    from kimi_linear_amd.graph_decode import KdaGraphedDecoder
    x = torch.randn(1, 20, 256, device=DEV).half()

    def step(layers, dec=None):
        dec = dec or KdaGraphedDecoder(layers)
        dec.prefill(x[:, :19])
        return dec.step(x[:, 19:]).clone(), dec

    layers = stack(kda_pkg, F16)
    a, dec = step(layers)
    other = kda_layer(kda_pkg, F16, seed=9).quantize_mx4_()
    layers[0].load_state_dict(other.state_dict())
    b, _ = step(layers, dec)
    assert not torch.equal(a, b) and torch.equal(b, step(layers)[0])
    assert torch.equal(layers[0](x), other(x))
    plain = [kda_layer(kda_pkg, F16, seed=3), latent_layer(kda_pkg, F16, seed=4)]
    a, dec = step(plain)
    for m in plain:
        m.quantize_mx4_()
    b, _ = step(plain, dec)
    assert not torch.equal(a, b) and torch.equal(b, step(plain)[0])
    plain[0].in_proj_q.weight.data.random_(0, 255)                 # unseen by the version counter
    dec.refresh_weights()
    dec.prefill(x[:, :19])
    assert torch.equal(dec.step(x[:, 19:]), step(plain)[0])


def test_refusals(kda_pkg):
    err = kda_pkg.KdaError
    layer = kda_layer(kda_pkg, F16)
    x = torch.randn(1, 70, 256, device=DEV).half()
    mixed = copy.deepcopy(layer)
    mixed.in_proj_k = kda_pkg.Mx4Linear.from_linear(mixed.in_proj_k)
    small = copy.deepcopy(layer).quantize_mx4_()
    small.beta_proj = kda_pkg.Mx4Linear.from_linear(small.beta_proj)
    with torch.no_grad():
        for m in (mixed, small):
            with pytest.raises(err, match="Mx4Linear"):
                m(x)
    layer.quantize_mx4_()
    with pytest.raises(err, match="train"):
        layer(x)
    only_out = kda_layer(kda_pkg, F16)
    only_out.o_proj = kda_pkg.Mx4Linear.from_linear(only_out.o_proj)
    with pytest.raises(err, match="train"):
        only_out(x)
    with torch.no_grad():
        assert torch.isfinite(only_out(x)).all()
    with pytest.raises(err):
        latent_layer(kda_pkg, F16).quantize_mx4_()(x)              # under grad mode
    with pytest.raises(err):
        kda_layer(kda_pkg, F16).cpu().quantize_mx4_()
    with pytest.raises(err), torch.no_grad():
        layer(x.float())
    for bad in (torch.int8, torch.uint8, torch.float16, 4):
        with pytest.raises(err, match="cache_dtype"):
            latent_layer(kda_pkg, F16, cache_dtype=bad)
    assert latent_layer(kda_pkg, F16, cache_dtype=torch.float8_e4m3fn).cache_bits == 8


@torch.no_grad()
def test_inference_mode_and_autocast(kda_pkg):
    """Quantised and run under inference mode, then outside it; in fp32 modules under autocast."""
    x = torch.randn(2, 40, 256, device=DEV)
    layers = [kda_layer(kda_pkg, F16, seed=6), latent_layer(kda_pkg, F16, seed=7, cache_dtype=FOUR)]
    with torch.inference_mode():
        for m in layers:
            m.quantize_mx4_()
            _, state = m(x[:, :30].half(), use_cache=True)
            a, _ = m(x[:, 30:31].half(), state=state, use_cache=True)
    for m in layers:
        _, state = m(x[:, :30].half(), use_cache=True)
        assert torch.equal(m(x[:, 30:31].half(), state=state, use_cache=True)[0].isfinite().all(), torch.tensor(True, device=DEV))
    assert torch.equal(a, m(x[:, 30:31].half(), state=m(x[:, :30].half(), use_cache=True)[1], use_cache=True)[0])
    layer = latent_layer(kda_pkg, torch.float32, seed=8).quantize_mx4_()
    with torch.autocast("cuda", dtype=BF16):
        y = layer(x)
    assert y.dtype == BF16 and rel(y, latent_like(kda_pkg, layer)(x.to(BF16))) <= TOL[BF16]


def latent_like(kda_pkg, layer):
    """The fp32 layer's bf16 form."""
    return stands_for(kda_pkg, copy.deepcopy(layer).to(BF16))


def test_only_plain_projections_are_quantised(kda_pkg):
    """A projection that does more than its product is refused, and the layer stays as it was."""
    class Scaled(torch.nn.Linear):
        def forward(self, x):
            return 2 * super().forward(x)

    def wrap(kind, lin):
        if kind == "type":
            new = Scaled(lin.in_features, lin.out_features, bias=False, device=DEV, dtype=F16)
            return new
        if kind == "hook":
            lin.register_forward_hook(lambda m, a, out: 2 * out)
        else:
            lin.forward = lambda x: x
        return lin

    for kind in ("type", "hook", "forward"):
        for make, name in ((kda_layer, "o_proj"), (latent_layer, "q_proj")):
            layer = make(kda_pkg, F16)
            setattr(layer, name, wrap(kind, getattr(layer, name)))
            with pytest.raises(kda_pkg.KdaError, match="plain"):
                layer.quantize_mx4_()
            assert not any(isinstance(m, kda_pkg.Mx4Linear) for m in layer.modules())
    layer = kda_layer(kda_pkg, F16, proj_bias=True).quantize_mx4_()
    layer.in_proj_k.bias = None
    with pytest.raises(kda_pkg.KdaError, match="bias"), torch.no_grad():
        layer(torch.randn(1, 5, 256, device=DEV).half())


@torch.no_grad()
def test_hooks_on_quantised_projections(kda_pkg):
    """A hook on an output projection in 4 bits is called: it is a module like another."""
    layer = kda_layer(kda_pkg, F16).quantize_mx4_()
    x = torch.randn(2, 9, 256, device=DEV).half()
    want = layer(x)
    layer.o_proj.register_forward_hook(lambda m, a, out: 2 * out)
    assert torch.equal(layer(x), 2 * want)


@torch.no_grad()
def test_a_capture_keeps_its_weights(kda_pkg):
    """Layers turned to 4 bits, or given other parameters, after a capture: until the next one a step runs with what was
    captured, whose memory nothing else gets."""
    from kimi_linear_amd.graph_decode import KdaGraphedDecoder
    x = torch.randn(1, 20, 256, device=DEV).half()
    layers = [kda_layer(kda_pkg, F16, seed=3), latent_layer(kda_pkg, F16, seed=4), kda_layer(kda_pkg, F16, seed=5)]
    dec, same = KdaGraphedDecoder(layers), KdaGraphedDecoder([copy.deepcopy(m) for m in layers])
    for d in (dec, same):
        d.prefill(x[:, :10])
    assert torch.equal(dec.step(x[:, 10:11]), same.step(x[:, 10:11]))
    sizes = {t.untyped_storage().nbytes() for m in layers for t in m.parameters()}
    layers[0].quantize_mx4_()
    layers[1].quantize_mx4_()
    layers[1].kv_up.weight = torch.nn.Parameter(torch.randn_like(layers[1].kv_up.weight))
    layers[2].o_proj = torch.nn.Linear(256, 256, bias=False, device=DEV, dtype=F16)
    for m in layers[::2]:
        m.refresh_fused_weight()
    torch.cuda.synchronize()
    others = [torch.full((n // 2,), float("nan"), dtype=F16, device=DEV) for n in sizes for _ in range(40)]
    for t in range(11, 15):
        assert torch.equal(dec.step(x[:, t:t + 1]), same.step(x[:, t:t + 1]))
    fresh = KdaGraphedDecoder(layers)
    for d in (dec, fresh):
        d.prefill(x[:, :15])
    for t in range(15, 20):
        assert torch.equal(dec.step(x[:, t:t + 1]), fresh.step(x[:, t:t + 1]))
    assert len(others) > 0


@torch.no_grad()
def test_deterministic_mode(kda_pkg):
    """Where torch fills new memory: prompts, steps and captures are what they are without."""
    from kimi_linear_amd.graph_decode import KdaGraphedDecoder
    x = torch.randn(2, 24, 256, device=DEV).half()
    layers = stack(kda_pkg, F16)

    def run():
        dec = KdaGraphedDecoder(layers)
        out = [dec.prefill(x[:, :20]).clone()]
        out += [dec.step(x[:, t:t + 1]).clone() for t in range(20, 24)]
        data, scale = kda_pkg.mx4_quantize(x)
        return [*out, kda_pkg.mx4_dequantize(data, scale, dtype=F16), layers[1](x, use_cache=True)[0]]

    want = run()
    was = torch.are_deterministic_algorithms_enabled(), torch.is_deterministic_algorithms_warn_only_enabled()
    torch.use_deterministic_algorithms(True, warn_only=True)         # (a library's product may have no such form)
    try:
        got = run()
    finally:
        torch.use_deterministic_algorithms(was[0], warn_only=was[1])
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@torch.no_grad()
def test_hooks_on_quantised_inputs(kda_pkg):
    """A hook, another forward or a subclass in the place of a q, k or v projection in 4 bits is called too."""
    from kimi_linear_amd.graph_decode import KdaGraphedDecoder

    class Doubled(kda_pkg.Mx4Linear):
        def forward(self, x):
            return 2 * super().forward(x)

    def subclass(layer, name):
        old = getattr(layer, name)
        new = Doubled(old.in_features, old.out_features, old.bias is not None, device=DEV, dtype=F16)
        new.load_state_dict(old.state_dict())
        setattr(layer, name, new)

    def forward(layer, name):
        m = getattr(layer, name)
        m.forward = lambda x: 2 * type(m).forward(m, x)

    kinds = [lambda layer, name: getattr(layer, name).register_forward_hook(lambda m, a, out: 2 * out),
             lambda layer, name: getattr(layer, name).register_forward_pre_hook(lambda m, a: (2 * a[0],)), forward, subclass]
    x = torch.randn(2, 80, 256, device=DEV).half()
    for i, change in enumerate(kinds):
        layer = kda_layer(kda_pkg, F16, seed=20, proj_bias=i == 2, conv_bias=i != 1).quantize_mx4_()
        want = copy.deepcopy(layer)
        plain = layer(x)
        change(layer, "in_proj_v")
        want.in_proj_v.weight_scale.add_(1)                  # the same as a product twice as large
        if want.in_proj_v.bias is not None:
            want.in_proj_v.bias.mul_(2)
        assert torch.equal(layer(x), want(x)) and not torch.equal(layer(x), plain)
        got, ref = cached(layer, x, (70, 1, 1))[0], cached(want, x, (70, 1, 1))[0]
        assert torch.equal(got, ref)
        decs = [KdaGraphedDecoder([m]) for m in (layer, want)]
        for d in decs:
            d.prefill(x[:, :9])
        assert torch.equal(decs[0].step(x[:, 9:10]), decs[1].step(x[:, 9:10]))


@torch.no_grad()
def test_refreshed_joined_weights(kda_pkg):
    """Bytes, scales and biases written past the version counters are what a layer runs with after a refresh: the
    same as a layer that has joined nothing yet."""
    from kimi_linear_amd.graph_decode import KdaGraphedDecoder
    x = torch.randn(2, 12, 256, device=DEV).half()
    for i, name in enumerate(("weight", "weight_scale", "bias")):
        layer = kda_layer(kda_pkg, F16, seed=30 + i, proj_bias=True).quantize_mx4_()
        dec = KdaGraphedDecoder([layer])
        dec.prefill(x[:, :10])
        before, stepped = layer(x), dec.step_eager(x[:, 10:11]).clone()
        t = getattr(layer.in_proj_k, name).data
        t.copy_(torch.randint(0, 256, t.shape, device=DEV, dtype=torch.uint8) if name == "weight" else t + 1)
        new = copy.deepcopy(layer)
        new._w4cat = None
        dec.refresh_weights()
        assert torch.equal(layer(x), new(x)) and not torch.equal(layer(x), before), name
        assert layer._w4cat[1].data_ptr() in dec._wbufs[2]                          # refilled in place, as captured
        other = KdaGraphedDecoder([new])
        for d in (dec, other):
            d.prefill(x[:, :10])
        assert torch.equal(dec.step(x[:, 10:11]), other.step(x[:, 10:11])) and not torch.equal(dec.output_static, stepped)


@pytest.mark.parametrize("mx4", [False, True])
@torch.no_grad()
def test_a_step_looks_its_projections_up_once(kda_pkg, mx4):
    """Which projections are in 4 bits is asked of modules looked up once a call, which an eager step of 120 us notices."""
    layer = kda_layer(kda_pkg, F16)
    if mx4:
        layer.quantize_mx4_()
    x = torch.randn(1, 9, 256, device=DEV).half()
    _, state = layer(x, use_cache=True)
    looked, made = [], layer._input_mods

    def input_mods():
        looked.append(1)
        return made()

    layer._input_mods = input_mods
    layer.decode_step_(x[:, :1], state)
    layer(x[:, :1], state=state, use_cache=True)
    layer(x)
    assert len(looked) == 3
