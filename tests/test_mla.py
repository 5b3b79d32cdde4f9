"""Latent attention: the C ABI's host-side checks and the wrapper's refusals (no kernel is launched)."""

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


@pytest.fixture(scope="module")
def native(kda_pkg):
    mod = importlib.import_module("kimi_linear_amd._native")
    mod.load()
    return mod


@pytest.mark.skipif(shutil.which("gcc") is None, reason="gcc not available")
@pytest.mark.parametrize("struct,cname", [("KdaMlaExpandedArgs", "kda_mla_expanded_args"),
                                          ("KdaMlaExpandedBwdArgs", "kda_mla_expanded_bwd_args"),
                                          ("KdaMlaAbsorbedArgs", "kda_mla_absorbed_args"),
                                          ("KdaMlaAppendArgs", "kda_mla_append_args"),
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


def fill(a, kw):
    for name, val in kw.items():
        field = getattr(a, name)
        if isinstance(field, ctypes.Array):
            for i, x in enumerate(val):
                field[i] = x
        else:
            setattr(a, name, val)
    return a


def expanded(native, **kw):
    a = native.KdaMlaExpandedArgs(B=1, T=8, S=8, H=2, N=64, P=32, V=64, scale=0.1, dtype=native.DTYPE_BF16)
    for f in ("q", "k", "k_pe", "v", "o"):
        setattr(a, f, FAKE)
    return fill(a, kw)


def test_expanded_codes(native):
    call = native.load().kda_mla_expanded_fwd

    def rc(**kw):
        return call(ctypes.byref(expanded(native, **kw)), None)

    assert call(None, None) == 1
    assert rc(B=-1) == 2 and rc(T=-1) == 2 and rc(S=2 ** 31) == 2 and rc(B=2 ** 30, T=2 ** 10) == 2
    assert rc(dtype=native.DTYPE_F32) == 3 and rc(dtype=7) == 3
    assert rc(N=48) == 4 and rc(N=128) == 4 and rc(P=16) == 4                   # V differs; no such kernels
    assert rc(scale=0.0) == 4 and rc(scale=-1.0) == 4 and rc(scale=float("nan")) == 4 and rc(scale=float("inf")) == 4
    assert rc(q=None) == 1 and rc(k=None) == 1 and rc(k_pe=None) == 1 and rc(v=None) == 1 and rc(o=None) == 1
    assert rc(q=FAKE + 2) == 4 and rc(k_stride=(0, 4, 0)) == 4 and rc(v_stride=(0, -8, 0)) == 4
    assert rc(B=0) == 0 and rc(H=0) == 0 and rc(T=0) == 0
    size = native.load().kda_mla_expanded_workspace_size
    assert size(1, 8, 8, 2, 64) == 0 and size(4, 2048, 2048, 16, 128) == 0 and size(1, 8, 4096, 2, 100) == 0
    assert size(1, 8, 4096, 2, 64) > 0 and rc(S=4096) == 1 and rc(S=4096, workspace=FAKE + 4) == 4


def test_expanded_bwd_codes(native):
    lib = native.load()

    def rc(fwd=None, **kw):
        g = native.KdaMlaExpandedBwdArgs()
        g.fwd = expanded(native, **{"lse": FAKE, "o_low": FAKE, **(fwd or {})})
        for f in ("d_o", "dq", "dk", "dk_pe", "dv", "workspace"):
            setattr(g, f, FAKE)
        return lib.kda_mla_expanded_bwd(ctypes.byref(fill(g, kw)), None)

    assert lib.kda_mla_expanded_bwd(None, None) == 1
    assert rc(fwd={"N": 96}) == 4 and rc(fwd={"lse": None}) == 1 and rc(fwd={"o_low": None}) == 1
    for name in ("d_o", "dq", "dk", "dk_pe", "dv", "workspace"):
        assert rc(**{name: None}) == 1, name
        assert rc(**{name: FAKE + 8}) == 4, name
    assert rc(fwd={"B": 0}) == 0
    size = lib.kda_mla_expanded_bwd_workspace_size
    assert size(2, 5, 7, 3, 32) == 128 + 2 * 7 * 3 * 32 * 4 and size(-1, 5, 7, 3, 32) == 0


def test_absorbed_codes(native):
    lib = native.load()

    def rc(**kw):
        a = native.KdaMlaAbsorbedArgs(B=1, T=1, H=2, S=600, R=128, P=32, scale=0.1, dtype=native.DTYPE_F16,
                                      cache_dtype=native.DTYPE_F16)
        for f in ("q", "cache", "lengths", "o", "workspace"):
            setattr(a, f, FAKE)
        return lib.kda_mla_absorbed_fwd(ctypes.byref(fill(a, kw)), None)

    assert lib.kda_mla_absorbed_fwd(None, None) == 1
    assert rc(T=-1) == 2 and rc(H=2 ** 31) == 2 and rc(T=2 ** 20, H=2 ** 10) == 2
    assert rc(dtype=native.DTYPE_F32) == 3 and rc(cache_dtype=native.DTYPE_BF16) == 3 and rc(cache_dtype=9) == 3
    assert rc(R=192) == 4 and rc(P=48) == 4 and rc(scale=0.0) == 4
    for name in ("q", "cache", "lengths", "o", "workspace"):
        assert rc(**{name: None}) == 1, name
    assert rc(cache_dtype=native.DTYPE_E4M3) == 1                               # no scales
    assert rc(cache=FAKE + 8) == 4 and rc(cache_stride=(0, 4)) == 4
    assert rc(cache_dtype=native.DTYPE_E4M3, cache_scale=FAKE, scale_stride=(0, 3)) == 4
    assert rc(B=0) == 0 and rc(T=0) == 0
    size = lib.kda_mla_absorbed_workspace_size
    assert size(1, 1, 16, 100, 512) == 0                                        # one workgroup has it all
    assert size(1, 1, 16, 10000, 512) > 0 and size(1, 1, 16, 10000, 500) == 0


def test_cache_codes(native):
    lib = native.load()

    def append(**kw):
        a = native.KdaMlaAppendArgs(B=2, T=3, S=8, R=128, P=32, x_dtype=native.DTYPE_BF16, cache_dtype=native.DTYPE_BF16)
        for f in ("x", "cache", "lengths"):
            setattr(a, f, FAKE)
        fill(a, {"x_stride": (480, 160), "cache_stride": (1280, 160), "scale_stride": (16, 2), **kw})
        return lib.kda_mla_cache_append(ctypes.byref(a), None)

    assert lib.kda_mla_cache_append(None, None) == 1
    assert append(B=-1) == 2 and append(S=2 ** 31) == 2
    assert append(x_dtype=native.DTYPE_F32) == 3 and append(cache_dtype=native.DTYPE_F16) == 3
    assert append(R=64) == 4 and append(P=8) == 4
    assert append(x=None) == 1 and append(cache=None) == 1 and append(lengths=None) == 1
    assert append(cache_dtype=native.DTYPE_E4M3) == 1
    assert append(x_stride=(480, 161)) == 4 and append(norm_weight=FAKE + 2) == 4
    assert append(cache_stride=(1280, 0)) == 4 and append(cache_stride=(0, 160)) == 4    # rows that overlap
    assert append(cache_dtype=native.DTYPE_E4M3, cache_scale=FAKE, scale_stride=(16, 0)) == 4
    assert append(T=0) == 0 and append(B=0) == 0 and append(S=0) == 0

    def read(**kw):
        a = native.KdaMlaReadArgs(B=2, S=8, R=128, P=32, out_dtype=native.DTYPE_BF16, cache=FAKE, cache_scale=FAKE,
                                  out=FAKE * 4)
        fill(a, {"cache_stride": (1280, 160), "scale_stride": (16, 2), **kw})
        return lib.kda_mla_cache_read(ctypes.byref(a), None)

    assert lib.kda_mla_cache_read(None, None) == 1
    assert read(S=-1) == 2 and read(out_dtype=native.DTYPE_E4M3) == 3 and read(R=96) == 4
    assert read(cache=None) == 1 and read(cache_scale=None) == 1 and read(out=None) == 1
    assert read(cache_stride=(1280, 8)) == 4 and read(out=FAKE + 16) == 5
    assert read(B=0) == 0 and read(S=0) == 0


def test_append_wants_distinct_rows(native):
    """Rows of different sequences may not share memory, in either order of the strides; sizes whose product
    passes 64 bits are refused."""
    lib = native.load()

    def append(cache, scales=None):
        a = native.KdaMlaAppendArgs(B=3, T=2, S=8, R=128, P=32, x_dtype=native.DTYPE_BF16,
                                    cache_dtype=native.DTYPE_BF16 if scales is None else native.DTYPE_E4M3)
        for f in ("x", "cache", "lengths") + (() if scales is None else ("cache_scale",)):
            setattr(a, f, FAKE)
        fill(a, {"x_stride": (320, 160), "cache_stride": cache, "scale_stride": scales or (0, 0)})
        return lib.kda_mla_cache_append(ctypes.byref(a), None)

    assert append((160, 160)) == 4 and append((1272, 160)) == 4 and append((160, 472)) == 4
    assert append((1280, 160), (2, 2)) == 4 and append((1280, 160), (14, 2)) == 4 and append((1280, 160), (2, 4)) == 4
    a = native.KdaMlaExpandedArgs(B=2 ** 31 - 1, T=2 ** 30, S=2 ** 30, H=2 ** 31 - 1, N=64, V=64, scale=1.0,
                                  dtype=native.DTYPE_F16)
    assert lib.kda_mla_expanded_fwd(ctypes.byref(a), None) == 2


def test_negative_scale_strides(native):
    """Strides of the scales may not be negative: the kernels form unsigned offsets from them."""
    lib = native.load()
    for stride in ((16, -2), (-16, 2)):
        a = native.KdaMlaAbsorbedArgs(B=2, T=1, H=2, S=8, R=128, P=32, scale=0.1, dtype=native.DTYPE_F16,
                                      cache_dtype=native.DTYPE_E4M3)
        for f in ("q", "cache", "cache_scale", "lengths", "o", "workspace"):
            setattr(a, f, FAKE)
        fill(a, {"q_stride": (320, 320, 160), "cache_stride": (1280, 160), "scale_stride": stride})
        assert lib.kda_mla_absorbed_fwd(ctypes.byref(a), None) == 4
        r = native.KdaMlaReadArgs(B=2, S=8, R=128, P=32, out_dtype=native.DTYPE_BF16, cache=FAKE, cache_scale=FAKE,
                                  out=FAKE * 4)
        fill(r, {"cache_stride": (1280, 160), "scale_stride": stride})
        assert lib.kda_mla_cache_read(ctypes.byref(r), None) == 4
        w = native.KdaMlaAppendArgs(B=2, T=1, S=8, R=128, P=32, x_dtype=native.DTYPE_BF16, cache_dtype=native.DTYPE_E4M3)
        for f in ("x", "cache", "cache_scale", "lengths"):
            setattr(w, f, FAKE)
        fill(w, {"x_stride": (160, 160), "cache_stride": (1280, 160), "scale_stride": stride})
        assert lib.kda_mla_cache_append(ctypes.byref(w), None) == 4


def test_append_norm_weight_code(native):
    a = native.KdaMlaAppendArgs(B=1, T=1, S=8, R=128, P=32, x_dtype=native.DTYPE_BF16, cache_dtype=native.DTYPE_BF16,
                                norm_f32=2)
    for f in ("x", "cache", "lengths", "norm_weight"):
        setattr(a, f, FAKE)
    fill(a, {"x_stride": (160, 160), "cache_stride": (1280, 160)})
    assert native.load().kda_mla_cache_append(ctypes.byref(a), None) == 3


def test_expanded_positions_stay_in_32_bits(native):
    """A query's position may be T below 0 or S past it: together they have to fit."""
    a = expanded(native, T=2 ** 30, S=2 ** 30, H=1)
    assert native.load().kda_mla_expanded_fwd(ctypes.byref(a), None) == 2


def test_wrapper_refuses_cpu_tensors(kda_pkg):
    q, k, pe = torch.zeros(1, 2, 2, 96, dtype=torch.bfloat16), torch.zeros(1, 2, 2, 64, dtype=torch.bfloat16), \
        torch.zeros(1, 2, 32, dtype=torch.bfloat16)
    n = torch.zeros(1, dtype=torch.int32)
    cache = torch.zeros(1, 2, 160, dtype=torch.bfloat16)
    for call in (lambda: kda_pkg.mla_expanded(q, k, pe, k), lambda: kda_pkg.mla_absorbed(cache[:, :, None], cache, n, 128, 1.0),
                 lambda: kda_pkg.mla_cache_append(cache, cache.clone(), n, 128),
                 lambda: kda_pkg.mla_cache_read(cache.to(torch.float8_e4m3fn), torch.ones(1, 2, 2), 128),
                 lambda: kda_pkg.mla_expanded(None, k, pe, k), lambda: kda_pkg.mla_absorbed(1, cache, n, 128, 1.0),
                 lambda: kda_pkg.mla_cache_append([1], cache, n, 128), lambda: kda_pkg.mla_cache_read(None, None, 128)):
        with pytest.raises(kda_pkg.KdaError):
            call()


@pytest.mark.gpu
def test_wrapper_refusals(kda_pkg):
    bf, dev = torch.bfloat16, "cuda:0"
    q, k, pe = (torch.zeros(*s, dtype=bf, device=dev) for s in ((1, 4, 2, 96), (1, 4, 2, 64), (1, 4, 32)))
    n = torch.zeros(1, dtype=torch.int32, device=dev)
    cache, x = torch.zeros(1, 4, 160, dtype=bf, device=dev), torch.zeros(1, 4, 160, dtype=bf, device=dev)
    f8, sc = cache.to(torch.float8_e4m3fn), torch.ones(1, 4, 2, device=dev)
    qa = torch.zeros(1, 1, 2, 160, dtype=bf, device=dev)
    E, A, W, R = kda_pkg.mla_expanded, kda_pkg.mla_absorbed, kda_pkg.mla_cache_append, kda_pkg.mla_cache_read
    E(q, k, pe, k), A(qa, cache, n, 128, 1.0), W(x, cache, n, 128), R(f8, sc, 128)
    need = qa.clone().requires_grad_()
    for bad in (lambda: E(q.float(), k, pe, k), lambda: E(q, k[..., :32], pe, k[..., :32]), lambda: E(q, k, None, k),
                lambda: E(q, k, pe, k[:, :3]), lambda: E(q, k.cpu(), pe, k), lambda: E(q, k, pe, k, scale=0.0),
                lambda: E(q, k, pe, k, lengths=[4]), lambda: E(q, k, pe, k, lengths=n.float()),
                lambda: E(q, k, pe, k, lengths=n.cpu()), lambda: E(q, k, pe, k, starts=torch.zeros(2, dtype=torch.int32, device=dev)),
                lambda: E(q[0], k, pe, k),
                lambda: A(qa.float(), cache, n, 128, 1.0), lambda: A(qa, cache, None, 128, 1.0),
                lambda: A(qa, cache, n, 96, 1.0), lambda: A(qa, cache, n, 128, -1.0), lambda: A(qa, cache.half(), n, 128, 1.0),
                lambda: A(qa, f8, n, 128, 1.0), lambda: A(qa, cache, n, 128, 1.0, cache_scale=sc),
                lambda: A(qa, f8, n, 128, 1.0, cache_scale=sc[:, :3]), lambda: A(need, cache, n, 128, 1.0),
                lambda: A(qa, cache[..., ::2], n, 128, 1.0), lambda: A(qa[0], cache, n, 128, 1.0),
                lambda: A(qa, torch.zeros(1, 4, 161, dtype=bf, device=dev)[..., 1:], n, 128, 1.0),
                lambda: W(x, cache.half(), n, 128), lambda: W(x, f8, n, 128), lambda: W(cache, cache, n, 128),
                lambda: W(x, cache, n, 128, norm_weight=torch.ones(64, device=dev)), lambda: W(x, cache, None, 128),
                lambda: W(x, cache[:, :1].expand(1, 4, 160), n, 128), lambda: W(x[0], cache, n, 128),
                lambda: W(x.clone().requires_grad_(), cache, n, 128),
                lambda: R(cache, sc, 128), lambda: R(f8, None, 128), lambda: R(f8, sc, 128, dtype=torch.float32),
                lambda: R(f8, sc, 128, tokens=5), lambda: R(f8, sc, 128, tokens=-1), lambda: R(f8, sc, 96)):
        with pytest.raises(kda_pkg.KdaError):
            bad()
