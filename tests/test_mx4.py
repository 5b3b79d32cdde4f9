"""4-bit weights and caches: struct layouts, status codes and the wrappers' refusals (no kernel is launched)."""

from __future__ import annotations

import ctypes
import importlib
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

HEADER = Path(__file__).resolve().parent.parent / "include" / "kda_hip.h"
FAKE = 0x100000          # never dereferenced: every call here is answered before a launch
FOUR, E8M0 = torch.float4_e2m1fn_x2, torch.float8_e8m0fnu


@pytest.fixture(scope="module")
def native(kda_pkg):
    mod = importlib.import_module("kimi_linear_amd._native")
    mod.load()
    return mod


@pytest.mark.skipif(shutil.which("gcc") is None, reason="gcc not available")
@pytest.mark.parametrize("struct,cname", [("KdaMx4LinearArgs", "kda_mx4_linear_args"),
                                          ("KdaMx4ConvertArgs", "kda_mx4_convert_args"),
                                          ("KdaMlaReadArgs", "kda_mla_read_args")])
def test_struct_layout_matches_header(native, tmp_path, struct, cname):
    cls = getattr(native, struct)
    fields = [name for name, _ in cls._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(["#include <stdio.h>", "#include <stddef.h>", '#include "kda_hip.h"', "int main(void) {",
                              f'  printf("size %zu\\n", sizeof({cname}));']
                             + [f'  printf("{f} %zu\\n", offsetof({cname}, {f}));' for f in fields] + ["  return 0;", "}"]))
    subprocess.run(["gcc", f"-I{HEADER.parent}", str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout
    got = dict(line.split() for line in out.splitlines() if line)
    assert int(got["size"]) == ctypes.sizeof(cls)
    for f in fields:
        assert int(got[f]) == getattr(cls, f).offset, f


def filled(a, **kw):
    for name, val in kw.items():
        field = getattr(a, name)
        if isinstance(field, ctypes.Array):
            for i, x in enumerate(val):
                field[i] = x
        else:
            setattr(a, name, val)
    return ctypes.byref(a)


def test_linear_codes(native):
    call = native.load().kda_mx4_linear_fwd

    def rc(**kw):
        a = native.KdaMx4LinearArgs(M=3, N=5, K=64, x=FAKE, x_stride=64, w=FAKE, w_scale=FAKE, y=FAKE, dtype=native.DTYPE_F16)
        return call(filled(a, **kw), None)

    assert call(None, None) == 1
    assert rc(M=-1) == 2 and rc(N=-1) == 2 and rc(K=0) == 2 and rc(K=2 ** 23) == 2 and rc(M=2 ** 31) == 2 and rc(N=2 ** 31) == 2
    assert rc(dtype=native.DTYPE_F32) == 3 and rc(dtype=native.DTYPE_E2M1) == 3
    assert rc(K=48) == 4 and rc(x=FAKE + 2) == 4 and rc(x_stride=-64) == 4 and rc(x_stride=60) == 4 and rc(w=FAKE + 8) == 4
    assert rc(x_stride=2 ** 23) == 4 and rc(y=FAKE + 2) == 4 and rc(bias=FAKE + 1) == 4 and rc(residual=FAKE, residual_stride=-1) == 4
    for name in ("x", "w", "w_scale", "y"):
        assert rc(**{name: None}) == 1, name
    assert rc(M=0) == 0 and rc(N=0) == 0


def test_convert_codes(native):
    lib = native.load()

    def rc(call, **kw):
        a = native.KdaMx4ConvertArgs(N=3, K=64, values=FAKE, value_stride=64, data=FAKE, scale=FAKE, dtype=native.DTYPE_BF16)
        return call(filled(a, **kw), None)

    for call in (lib.kda_mx4_quantize, lib.kda_mx4_dequantize):
        assert call(None, None) == 1
        assert rc(call, N=-1) == 2 and rc(call, K=0) == 2 and rc(call, N=2 ** 30) == 2
        assert rc(call, dtype=native.DTYPE_E4M3) == 3 and rc(call, K=40) == 4
        assert rc(call, values=None) == 1 and rc(call, data=None) == 1 and rc(call, scale=None) == 1
        assert rc(call, values=FAKE + 8) == 4 and rc(call, data=FAKE + 4) == 4 and rc(call, value_stride=68) == 4
        assert rc(call, value_stride=-64) == 4 and rc(call, N=0) == 0
    assert rc(lib.kda_mx4_dequantize, dtype=native.DTYPE_F32) == 3
    assert rc(lib.kda_mx4_dequantize, value_stride=32) == 4                          # rows that overlap


def test_cache_codes(native):
    lib, four = native.load(), native.DTYPE_E2M1

    def absorbed(**kw):
        a = native.KdaMlaAbsorbedArgs(B=1, T=1, H=2, S=600, R=128, P=32, scale=0.1, dtype=native.DTYPE_F16, cache_dtype=four)
        for f in ("q", "cache", "cache_scale", "lengths", "o", "workspace"):
            setattr(a, f, FAKE)
        return lib.kda_mla_absorbed_fwd(filled(a, **kw), None)

    assert absorbed(cache_scale=None) == 1 and absorbed(cache=None) == 1 and absorbed(workspace=None) == 1
    assert absorbed(cache=FAKE + 8) == 4 and absorbed(cache_stride=(0, 8)) == 4 and absorbed(cache_stride=(0, -80)) == 4
    assert absorbed(cache_scale=FAKE + 4) == 4 and absorbed(scale_stride=(0, 4)) == 4 and absorbed(scale_stride=(0, -8)) == 4
    assert absorbed(scale_stride=(0, 2 ** 23)) == 4 and absorbed(cache_stride=(0, 2 ** 23)) == 4
    assert absorbed(R=192) == 4 and absorbed(P=16) == 4 and absorbed(B=0) == 0

    def append(**kw):
        a = native.KdaMlaAppendArgs(B=2, T=3, S=8, R=128, P=32, x_dtype=native.DTYPE_BF16, cache_dtype=four)
        for f in ("x", "cache", "cache_scale", "lengths"):
            setattr(a, f, FAKE)
        return lib.kda_mla_cache_append(filled(a, **{"x_stride": (480, 160), "cache_stride": (640, 80), "scale_stride": (64, 8), **kw}), None)

    assert append(cache_scale=None) == 1
    assert append(cache_stride=(640, 64)) == 4 and append(cache_stride=(80, 80)) == 4     # rows that overlap
    assert append(scale_stride=(64, 0)) == 4 and append(scale_stride=(8, 8)) == 4 and append(scale_stride=(64, 12)) == 4
    assert append(T=0) == 0

    def read(**kw):
        a = native.KdaMlaReadArgs(B=2, S=8, R=128, P=32, out_dtype=native.DTYPE_BF16, cache=FAKE, cache_scale=FAKE,
                                  out=FAKE * 16, cache_dtype=four)
        return lib.kda_mla_cache_read(filled(a, **{"cache_stride": (640, 80), "scale_stride": (64, 8), **kw}), None)

    assert read(cache_dtype=native.DTYPE_F16) == 3 and read(cache_dtype=9) == 3
    assert read(cache_scale=None) == 1 and read(scale_stride=(64, 2)) == 4 and read(cache_stride=(640, 72)) == 4
    assert read(out=FAKE + 1264) == 5 and read(B=0) == 0                        # the last row's last 16 bytes


def mx4(N=4, K=64):
    return torch.zeros(N, K // 2, dtype=torch.uint8), torch.zeros(N, K // 32, dtype=torch.uint8)


def test_refusals(kda_pkg):
    err = kda_pkg.KdaError
    x, (w, s) = torch.zeros(2, 64, dtype=torch.float16), mx4()
    bad = [
        lambda: kda_pkg.mx4_linear(x, w, s),                                     # no HIP tensors
        lambda: kda_pkg.mx4_linear("x", w, s),
        lambda: kda_pkg.mx4_linear(x, None, s),
        lambda: kda_pkg.mx4_quantize(x),
        lambda: kda_pkg.mx4_quantize(None),
        lambda: kda_pkg.mx4_dequantize(w, s),
        lambda: kda_pkg.mx4_dequantize(w, s[:, :1]),
        lambda: kda_pkg.mx4_dequantize(w.int(), s),
        lambda: kda_pkg.Mx4Linear(48, 3),
        lambda: kda_pkg.Mx4Linear(0, 3),
        lambda: kda_pkg.mla_cache_read(w.view(1, 4, 32).view(FOUR), s.view(1, 4, 2), 128),
    ]
    for call in bad:
        with pytest.raises(err):
            call()


def test_module(kda_pkg):
    mod = kda_pkg.Mx4Linear(64, 5, bias=True, dtype=torch.float16)
    assert {n: (tuple(b.shape), b.dtype) for n, b in mod.named_buffers()} == {
        "weight": ((5, 32), torch.uint8), "weight_scale": ((5, 2), torch.uint8), "bias": ((5,), torch.float16)}
    assert list(mod.parameters()) == []
    mod.weight.random_(0, 255)
    other = kda_pkg.Mx4Linear(64, 5, bias=True, dtype=torch.float16)
    other.load_state_dict(mod.state_dict())
    assert torch.equal(other.weight, mod.weight)
    half = other.to(torch.bfloat16)                       # the packed weight is no number to convert
    assert torch.equal(half.weight, mod.weight) and half.bias.dtype == torch.bfloat16
    assert "in_features=64" in repr(mod)


@pytest.mark.parametrize("cache_dtype", [None, torch.float8_e4m3fn, FOUR])
def test_new_state_in_deterministic_mode(kda_pkg, cache_dtype):
    """In torch's deterministic mode new memory is filled, which is not there for every type."""
    layer = kda_pkg.LatentAttention(kda_pkg.latent_attn_config(hidden_size=64, num_heads=1, head_dim=64, position_dim=32, rank=128,
                                                               max_tokens=6, cache_dtype=cache_dtype))
    was = torch.are_deterministic_algorithms_enabled()
    torch.use_deterministic_algorithms(True)
    try:
        state = layer.new_state(2, "cpu", torch.float16)
    finally:
        torch.use_deterministic_algorithms(was)
    other = layer.new_state(2, "cpu", torch.float16)
    for name in ("latent", "scale", "lengths"):
        a, b = state[name], other[name]
        assert (a is None and b is None) or (a.shape == b.shape and a.dtype == b.dtype and a.is_contiguous()), name
    assert state["latent"].dtype == (cache_dtype or torch.float16) and state["latent"].shape == (2, 6, 80 if cache_dtype == FOUR else 160)


def test_absorbed_workspace_by_cache_type(native):
    """A cache in 16 or 8 bits asks for 256 workgroups' parts at any length, one in 4 bits for 512 where it is cut into as many."""
    size, most = native.load().kda_mla_absorbed_cache_workspace_size, native.load().kda_mla_absorbed_workspace_size
    wide = (native.DTYPE_F16, native.DTYPE_BF16, native.DTYPE_E4M3)

    def parts(groups, tiles, R):                 # rows of sums, their maximum and denominator, and the tiles' spans
        return (groups + tiles) * 16 * (4 * R + 8) + 8 * tiles

    for B, T, H, S, R in ((64, 1, 16, 8192, 512), (200, 1, 16, 4096, 256), (1, 1, 16, 600, 128), (8, 5, 20, 1501, 256), (1, 1, 16, 400, 512),
                          (600, 1, 16, 8192, 512)):
        tiles = B * -(-T * H // 16)
        shared = tiles < 512 and S > 512
        long = tiles * -(-S // 64) >= 2048
        for t in wide:
            assert size(B, T, H, S, R, t) == (parts(256, tiles, R) if shared else 0)
        four = size(B, T, H, S, R, native.DTYPE_E2M1)
        assert four == (parts(512 if long else 256, tiles, R) if shared else 0) == most(B, T, H, S, R)
    assert size(1, 1, 16, 10000, 512, native.DTYPE_F32) == 0 and size(1, 1, 16, 10000, 512, 9) == 0
    assert size(1, 1, 16, 10000, 500, native.DTYPE_E2M1) == 0 and size(-1, 1, 16, 10000, 512, native.DTYPE_E2M1) == 0
