"""GPU parity of the KDA layer (native core + torch projections) against the
layer oracle, and of its cache handling (chunked prefill, token-by-token decode).

The module's own parameters (after any cast) are handed to the oracle, so the
differences are compute precision only.  Tolerances on the layer output,
relative L2 error: fp32 2e-5, fp16 5e-3, bf16 2e-2.  An fp32 layer computes in
fp32 throughout (its core runs the fp32 token recurrence); fp16/bf16 layers
round every projection to 11/8 bits and feed the chunk pipeline's matrix
cores fp16 operands with fp32 accumulation.
"""

from __future__ import annotations

import pytest
import torch

from oracle.kda_layer_oracle import kda_layer_ref, make_layer_params

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
TOL = {torch.float32: 2e-5, torch.float16: 5e-3, torch.bfloat16: 2e-2}


def rel(a, b):
    a, b = a.detach().double().cpu(), b.detach().double().cpu()
    return ((a - b).norm() / b.norm()).item()


def make_layer(pkg, dtype, seed=0, **kw):
    cfg = pkg.linear_attn_config(**{"hidden_size": 256, "num_heads": 2, "gate_low_rank": 64,
                                    "output_gate_low_rank": 64, **kw})
    m = pkg.KimiDeltaAttention(cfg)
    m.load_state_dict(make_layer_params(cfg, seed=seed))
    m = m.to(device=DEV, dtype=dtype).eval()
    params = {n: t.detach().float().cpu() for n, t in m.state_dict().items()}
    return m, cfg, params


def make_x(B, T, d, dtype, seed):
    return torch.randn(B, T, d, generator=torch.Generator().manual_seed(seed)).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T", [150, 40, 64])
def test_layer_prefill_vs_oracle(kda_pkg, dtype, T):
    """T=150: chunkwise body of 128 + recurrent tail of 22; T=40: one chunk of
    40 (T < chunk_size); T=64: exactly one chunk."""
    m, cfg, p = make_layer(kda_pkg, dtype, seed=1)
    x = make_x(2, T, 256, dtype, seed=2)
    with torch.no_grad():
        out = m(x.to(DEV))
    ref = kda_layer_ref(p, cfg, x)
    e = rel(out, ref)
    print(f"[layer prefill {dtype} T={T}] rel {e:.3e}", flush=True)
    assert out.dtype == dtype and out.shape == (2, T, 256)
    assert e <= TOL[dtype]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_layer_prefill_then_decode_vs_oracle(kda_pkg, dtype):
    m, cfg, p = make_layer(kda_pkg, dtype, seed=3)
    x = make_x(3, 76, 256, dtype, seed=4)
    xd = x.to(DEV)
    with torch.no_grad():
        o, st = m(xd[:, :70], use_cache=True)
        outs = [o]
        for t in range(70, 76):
            o, st = m(xd[:, t:t + 1], state=st, use_cache=True)
            outs.append(o)
    out = torch.cat(outs, 1)
    ref, st_ref = kda_layer_ref(p, cfg, x, use_cache=True)
    e = rel(out, ref)
    es = rel(st["recurrent"], st_ref["recurrent"])
    print(f"[layer decode {dtype}] out rel {e:.3e} state rel {es:.3e}", flush=True)
    assert st["recurrent"].dtype == torch.float32            # fp32 state for fp16 activations
    assert e <= TOL[dtype] and es <= TOL[dtype]
    for n in ("q", "k", "v"):
        assert rel(st["conv"][n], st_ref["conv"][n]) <= TOL[dtype]


def test_layer_chunked_prefill_vs_one_pass(kda_pkg):
    m, cfg, p = make_layer(kda_pkg, torch.float16, seed=5)
    x = make_x(2, 228, 256, torch.float16, seed=6)
    xd = x.to(DEV)
    with torch.no_grad():
        o1, st = m(xd[:, :100], use_cache=True)      # body 64 + tail 36
        o2, st = m(xd[:, 100:], state=st, use_cache=True)
        one = m(xd)
    out = torch.cat([o1, o2], 1)
    ref = kda_layer_ref(p, cfg, x)
    e, e1 = rel(out, ref), rel(one, ref)
    print(f"[layer chunked prefill] rel {e:.3e} one-pass rel {e1:.3e}", flush=True)
    assert e <= TOL[torch.float16] and e1 <= TOL[torch.float16]


def test_layer_model_width(kda_pkg):
    """The Kimi-Linear attention width: hidden 2048, 16 heads of 128."""
    cfg = kda_pkg.linear_attn_config(hidden_size=2048, num_heads=16)
    m = kda_pkg.KimiDeltaAttention(cfg)
    m.load_state_dict(make_layer_params(cfg, seed=7))
    m = m.to(device=DEV, dtype=torch.float16).eval()
    p = {n: t.detach().float().cpu() for n, t in m.state_dict().items()}
    x = make_x(2, 192, 2048, torch.float16, seed=8)
    with torch.no_grad():
        out = m(x.to(DEV))
    e = rel(out, kda_layer_ref(p, cfg, x))
    print(f"[layer hidden 2048] rel {e:.3e}", flush=True)
    assert e <= TOL[torch.float16]


@pytest.mark.parametrize("proj_bias", [False, True])
def test_fused_projection_weight_follows_updates(kda_pkg, proj_bias):
    """The six projections of x run as one GEMM over a cached concatenation of
    their weights and biases: an in-place update or a replaced parameter must
    reach it; a write through ``.data`` reaches it after refresh_fused_weight()."""
    m, cfg, _ = make_layer(kda_pkg, torch.float16, seed=3, proj_bias=proj_bias)
    x = make_x(2, 48, cfg.hidden_size, torch.float16, seed=4).to(DEV)
    with torch.no_grad():
        m(x)                                                  # builds the cache
        w_buf = m._wcat[1].data_ptr()
        m.in_proj_k.weight.mul_(0.5)                          # in place
        if proj_bias:
            m.beta_proj.bias.add_(0.25)                       # a bias alone changes
        m.gk_proj[0].weight = torch.nn.Parameter(m.gk_proj[0].weight * 2.0)   # replaced
        m.load_state_dict({k: v for k, v in m.state_dict().items()})          # copy_ into params
        out = m(x)
        assert m._wcat[1].data_ptr() == w_buf                 # refilled in place
        fresh, _, _ = make_layer(kda_pkg, torch.float16, seed=3, proj_bias=proj_bias)
        fresh.load_state_dict(m.state_dict())
        assert torch.equal(out, fresh(x))
        m.in_proj_v.weight.data.mul_(0.5)                     # invisible to the version counter
        m.refresh_fused_weight()
        fresh.load_state_dict(m.state_dict())
        assert torch.equal(m(x), fresh(x))


def test_layer_config4_full_shape(kda_pkg):
    """The whole layer at its benchmark shape: B=4, T=2048, hidden 2048 (16 heads
    of 128), fp16 weights N(0, 0.02), fp32 recurrent state.  All four sequences
    run on the GPU in one call (the chunkwise kernel's instantiation for 64
    heads); sequences 0 and 3 are checked against the fp32 oracle."""
    cfg = kda_pkg.linear_attn_config(hidden_size=2048, num_heads=16)
    m = kda_pkg.KimiDeltaAttention(cfg)
    m.load_state_dict(make_layer_params(cfg, seed=11))
    m = m.to(device=DEV, dtype=torch.float16).eval()
    p = {n: t.detach().float().cpu() for n, t in m.state_dict().items()}
    x = make_x(4, 2048, 2048, torch.float16, seed=12)
    print("[layer config 4] B=4 T=2048 hidden 2048 fp16", flush=True)
    with torch.no_grad():
        out, st = m(x.to(DEV), use_cache=True)
    torch.cuda.synchronize()
    assert torch.isfinite(out).all()
    sel = [0, 3]
    ref, st_ref = kda_layer_ref(p, cfg, x[sel], use_cache=True)
    e = rel(out[sel], ref)
    es = rel(st["recurrent"][sel], st_ref["recurrent"])
    print(f"[layer config 4] out rel {e:.3e} state rel {es:.3e}", flush=True)
    # the final state at the core's bar for fp16 inputs (relative error <= 1e-3;
    # measured 4.2e-4), the output at the layer's fp16 bar
    assert e <= TOL[torch.float16] and es <= 1e-3


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hd,T", [(128, 128), (64, 192), (128, 40)])
def test_layer_fused_output_vs_oracle(kda_pkg, dtype, hd, T):
    """The output epilogue on the chunk kernel's tiles (fuse_output=True: one
    workgroup per head) against the oracle, and against the same layer run
    with the split kernels (fuse_output=False), state included."""
    m, cfg, p = make_layer(kda_pkg, dtype, seed=21, head_dim=hd, value_head_dim=hd, num_heads=2, hidden_size=256)
    x = make_x(2, T, 256, dtype, seed=22)
    with torch.no_grad():
        m.fuse_output = True
        out_f, st_f = m(x.to(DEV), use_cache=True)
        m.fuse_output = False
        out_s, st_s = m(x.to(DEV), use_cache=True)
    ref, st_ref = kda_layer_ref(p, cfg, x, use_cache=True)
    e, es = rel(out_f, ref), rel(st_f["recurrent"], st_ref["recurrent"])
    ed = rel(out_f, out_s)
    print(f"[layer fused output {dtype} d={hd} T={T}] out rel {e:.2e} state rel {es:.2e} vs split {ed:.2e}",
          flush=True)
    assert e <= TOL[dtype] and es <= TOL[dtype]
    assert torch.equal(st_f["recurrent"], st_s["recurrent"])
    assert ed <= TOL[dtype] / 4


def test_layer_long_prefill_takes_the_split_core(kda_pkg, monkeypatch):
    """One long sequence over few heads: the pre-processing kernel forms g and
    beta and the ungated core splits the body into parallel segments (the
    gated core has no split).  Output and recurrent state against the oracle
    and against the same layer run with the split turned off."""
    layer_mod = __import__("kimi_linear_amd.layer", fromlist=["long_segments"])
    dtype = torch.float16
    m, cfg, p = make_layer(kda_pkg, dtype, seed=5)
    la = cfg.linear_attn_config
    T = 4096 + 22                                   # body of 4096 + recurrent tail
    assert layer_mod.long_segments(1, 4096, la["num_heads"], la["head_dim"], la["value_head_dim"], dtype) >= 4
    x = make_x(1, T, 256, dtype, seed=6)
    print(f"[layer long prefill fp16 B=1 T={T} H={la['num_heads']}]", flush=True)
    with torch.no_grad():
        out, st = m(x.to(DEV), use_cache=True)
        monkeypatch.setattr(layer_mod, "long_segments", lambda *a: 1)
        out1, st1 = m(x.to(DEV), use_cache=True)
    ref, st_ref = kda_layer_ref(p, cfg, x, use_cache=True)
    e, es = rel(out, ref), rel(st["recurrent"], st_ref["recurrent"])
    e1, es1 = rel(out, out1), rel(st["recurrent"], st1["recurrent"])
    print(f"  vs oracle: out {e:.3e} state {es:.3e}; vs one pass: out {e1:.3e} state {es1:.3e}", flush=True)
    assert e <= TOL[dtype] and es <= TOL[dtype]
    assert e1 <= TOL[dtype] and es1 <= TOL[dtype]


# ----------------------------------------------------------------- methods of a subclass
@pytest.mark.parametrize("where", ["subclass", "instance", "class"])
def test_replaced_methods_are_called(kda_pkg, monkeypatch, where):
    """_projections, _output, init_state and decode_step_ replaced by a subclass,
    on the instance or on the class keep their arguments and results and take
    part in prefill, decode and the graph decoder."""
    import importlib
    import types
    decoder = importlib.import_module("kimi_linear_amd.graph_decode").KdaGraphedDecoder
    base = kda_pkg.KimiDeltaAttention
    old = {n: getattr(base, n) for n in ("_projections", "_output", "init_state", "decode_step_")}
    seen = []

    def _projections(self, x, conv_cache=None, use_cache=False, conv_out=None, gates=False):
        seen.append("_projections")
        *rest, og_low = old["_projections"](self, x, conv_cache=conv_cache, use_cache=use_cache, conv_out=conv_out,
                                            gates=gates)
        assert len(rest) == 6 and og_low.shape[:2] == x.shape[:2]
        return (*rest, og_low * 0)                  # an output gate of 1/2

    def _output(self, o_core, og_low):
        seen.append("_output")
        return old["_output"](self, o_core, og_low) + 1

    def init_state(self, batch, device=None, dtype=None):
        seen.append("init_state")
        state = old["init_state"](self, batch, device=device, dtype=dtype)
        state["conv"]["q"].fill_(0.5)
        return state

    def decode_step_(self, x, state):
        seen.append("decode_step_")
        return old["decode_step_"](self, x, state) * 2

    new = dict(_projections=_projections, _output=_output, init_state=init_state, decode_step_=decode_step_)
    mod, x = make_layer(kda_pkg, torch.float16)[0], make_x(2, 5, 256, torch.float16, 3).to(DEV)
    with torch.no_grad():
        start = old["init_state"](mod, 2, device=x.device, dtype=x.dtype)
        start["conv"]["q"].fill_(0.5)
        keep = mod.og_proj[1].weight.clone()        # the same layer by hand: a gate of 1/2 everywhere
        mod.og_proj[1].weight.zero_()
        y, st = mod(x[:, :4], state=start, use_cache=True)
        want = [y + 1, 2 * (mod.decode_step_(x[:, 4:], st) + 1)]
        mod.og_proj[1].weight.copy_(keep)
    if where == "subclass":
        mod.__class__ = type("Sub", (base,), new)
    for n, f in new.items():
        if where == "instance":
            setattr(mod, n, types.MethodType(f, mod))
        elif where == "class":
            monkeypatch.setattr(base, n, f)
    with torch.no_grad():
        y, st = mod(x[:, :4], use_cache=True)
        assert seen == ["init_state", "_projections", "_output"]
        step = mod.decode_step_(x[:, 4:], st)
        tol = TOL[torch.float16]        # the up-projections one by one: other sums, rounded the same
        assert rel(y, want[0]) <= tol and rel(step, want[1]) <= tol
        seen.clear()
        dec = decoder([mod])
        dec.prefill(x[:, :4])
        assert seen.count("decode_step_") == 4 and seen.count("_output") == 5      # 3 warm-up steps and the capture
        assert rel(dec.step(x[:, 4:]), (x[:, 4:] + want[1])[:, 0]) <= tol


def test_fused_weight_at_the_address_of_an_earlier_one(kda_pkg):
    """Parameters replaced by ones that the allocator puts where the old ones were: the caches are made again."""
    m, cfg, _ = make_layer(kda_pkg, torch.float16, seed=3)
    x = make_x(1, 48, cfg.hidden_size, torch.float16, seed=4).to(DEV)
    with torch.no_grad():
        for mod, name in ((m.in_proj_v, "weight"), (m, "A_log")):
            shape, dtype = getattr(mod, name).shape, getattr(mod, name).dtype
            setattr(mod, name, torch.nn.Parameter(torch.randn(shape, device=DEV, dtype=dtype)))
            m(x)                                                  # builds the caches
            at = getattr(mod, name).data_ptr()
            setattr(mod, name, None)
            tries = []
            while len(tries) < 64 and not (tries and tries[-1].data_ptr() == at):
                tries.append(torch.randn(shape, device=DEV, dtype=dtype))
            setattr(mod, name, torch.nn.Parameter(tries[-1]))
            out = m(x)
            fresh, _, _ = make_layer(kda_pkg, torch.float16, seed=3)
            fresh.load_state_dict(m.state_dict())
            assert torch.equal(out, fresh(x)), name


def test_fused_weights_made_under_inference_mode(kda_pkg):
    """Caches first made under inference mode are refilled outside it when a parameter changes."""
    m, cfg, _ = make_layer(kda_pkg, torch.float16, seed=3)
    x = make_x(1, 48, cfg.hidden_size, torch.float16, seed=4).to(DEV)
    with torch.inference_mode():
        m(x)
    with torch.no_grad():
        m.in_proj_k.weight.mul_(0.5)
        m.A_log.add_(0.25)
        out = m(x)
        m.refresh_fused_weight()
        fresh, _, _ = make_layer(kda_pkg, torch.float16, seed=3)
        fresh.load_state_dict(m.state_dict())
        assert torch.equal(out, fresh(x))
    with torch.inference_mode():
        assert torch.equal(m(x), out)
