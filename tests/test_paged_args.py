"""Argument checks of the paged-cache operators, on the CPU: the refusals of hearth_amd/paged.py
with stand-ins for device tensors, those of the C entry points with addresses that a refused
call never touches, the ctypes mirrors' layouts, the rotary frequency tables, and the bounds
that the kernels put on lengths, tokens and pages, enumerated."""
from __future__ import annotations

import ctypes
import math
import re
import shutil
import subprocess
from ctypes import byref
from pathlib import Path

import numpy as np
import pytest

from hearth_amd import _native, paged

INC = Path(__file__).resolve().parents[1] / "include"


class _Dev:
    def __init__(self, type="cuda", index=0):
        self.type, self.index = type, index

    def __str__(self):
        return f"{self.type}:{self.index}"


class Fake:
    """shape, strides, dtype and device of a tensor whose memory nothing touches"""
    SIZES = {"float32": 4, "float64": 8, "bfloat16": 2, "float16": 2, "float8_e4m3fn": 1, "uint8": 1, "int32": 4, "int64": 8}

    def __init__(self, shape, dtype="bfloat16", strides=None, ptr=1 << 40, dev=None):
        self.shape, self.dtype, self._p, self.device = tuple(shape), "torch." + dtype, ptr, dev or _Dev()
        if strides is None:
            strides, n = [], 1
            for d in reversed(shape):
                strides.insert(0, n)
                n *= d
        self._s = tuple(strides)

    def stride(self):
        return self._s

    def get_device(self):
        return self.device.index if self.device.type == "cuda" else -1

    def data_ptr(self):
        return self._p

    def element_size(self):
        return self.SIZES[self.dtype.replace("torch.", "")]

    def numel(self):
        return int(np.prod(self.shape))

    def is_contiguous(self):
        return True


def cache(dtype="bfloat16", heads=2, width=64, page=16, pages=4, latent=False, **kw):
    k = Fake((pages, heads, page, width), dtype, **kw)
    sc = Fake((pages, heads, page, width // 32), "uint8") if dtype == "float8_e4m3fn" else None
    return paged.Cache(k, None if latent else k, sc, None if latent else sc)


def batch(S=2, per=4, max_q=3, max_kv=50, mask=None):
    return paged.Batch(Fake((S, per), "int32"), Fake((S,), "int32"), Fake((S + 1,), "int32"), max_q=max_q, max_kv=max_kv, mask=mask)


def test_cache_refusals():
    ok = Fake((4, 2, 16, 64))
    paged.Cache(ok, ok)
    for bad in (Fake((4, 2, 16, 64), "float32"), Fake((4, 2, 16)), Fake((4, 2, 24, 64)), Fake((4, 2, 8, 64)),
                Fake((4, 2, 16, 40)), Fake((4, 2, 16, 2048)), Fake((4, 2, 16, 64), strides=(4096, 64, 128, 1)),
                Fake((4, 2, 16, 64), strides=(2049, 1024, 64, 1)), Fake((4, 2, 16, 64), ptr=(1 << 40) + 2),
                Fake((4, 2, 16, 64), dev=_Dev("cpu")), Fake((4, 2, 16, 64), "int32")):
        with pytest.raises(ValueError):
            paged.Cache(bad, bad)
    with pytest.raises(ValueError):
        paged.Cache(ok, Fake((4, 2, 16, 128)))
    with pytest.raises(ValueError):
        paged.Cache(ok, Fake((4, 2, 16, 64), dev=_Dev(index=1)))
    codes, sc = Fake((4, 2, 16, 64), "float8_e4m3fn"), Fake((4, 2, 16, 2), "uint8")
    paged.Cache(codes, codes, sc, sc)
    for a, b in ((None, None), (sc, None), (sc, Fake((4, 2, 16, 4), "uint8")), (Fake((4, 2, 16, 2), "int32"), sc),
                 (Fake((4, 2, 16, 2), "uint8", strides=(64, 32, 1, 16)), sc)):
        with pytest.raises(ValueError):
            paged.Cache(codes, codes, a, b)
    with pytest.raises(ValueError):
        paged.Cache(ok, ok, sc, sc)


def test_batch_refusals():
    batch()
    i32 = lambda *s: Fake(s, "int32")
    for args in ((i32(2, 4), i32(3), i32(3)), (i32(2, 4), i32(2), i32(2)), (Fake((2, 4), "int64"), i32(2), i32(3)),
                 (i32(2, 4), Fake((2,), "float32"), i32(3)), (i32(8), i32(2), i32(3)),
                 (Fake((2, 4), "int32", strides=(1, 2)), i32(2), i32(3)), (Fake((2, 4), "int32", strides=(2, 1)), i32(2), i32(3))):
        with pytest.raises(ValueError):
            paged.Batch(*args, max_q=1, max_kv=16)
    for kw in (dict(max_q=-1), dict(max_kv=-1), dict(max_q=65, mask=Fake((9, 1), "int64")), dict(mask=Fake((9, 1), "int32")),
               dict(S=70000)):
        with pytest.raises(ValueError):
            batch(**kw)


@pytest.mark.parametrize("fn", [paged.append, paged.read])
def test_copy_refusals(fn):
    c, b = cache(), batch()
    rows = Fake((5, 2, 64))
    for args in ((rows, None), (Fake((5, 3, 64)), rows), (rows, Fake((4, 2, 64))), (rows, Fake((5, 2, 32))),
                 (rows, Fake((5, 2, 64), "float32")), (Fake((5, 128)), rows), (Fake((5, 2, 64), "float8_e4m3fn"), rows),
                 (Fake((5, 2, 64), strides=(128, 1, 2)), rows), (rows, Fake((5, 2, 64), dev=_Dev(index=1)))):
        with pytest.raises(ValueError):
            fn(c, b, *args)
    lat = cache(heads=1, width=576, latent=True)
    for args in ((Fake((5, 1, 512)), None), (Fake((5, 1, 512)), Fake((5, 1, 32))), (Fake((5, 2, 512)), Fake((5, 2, 64)))):
        with pytest.raises(ValueError):
            fn(lat, b, *args)
    with pytest.raises(ValueError):
        fn(c, batch(mask=Fake((4, 1), "int64")), rows, rows)     # fewer mask rows than tokens


def test_attend_refusals():
    c, b = cache(), batch()
    q = Fake((5, 4, 64))
    for args, kw in (((Fake((5, 3, 64)), Fake((5, 3, 64))), {}), ((q, Fake((5, 4, 32))), {}), ((q, Fake((4, 4, 64))), {}),
                     ((Fake((5, 4, 64), "float32"), Fake((5, 4, 64), "float32")), {}),
                     ((Fake((5, 4, 64), "float16"), Fake((5, 4, 64), "float16")), {}),
                     ((q, Fake((5, 4, 64), "float16")), {}), ((Fake((5, 4, 128)), Fake((5, 4, 128))), {}),
                     ((q, q), dict(lse=Fake((5, 4)))), ((q, q), dict(lse=Fake((4, 4), "float32"))),
                     ((q, q), dict(scale=math.nan)), ((q, q), dict(scale=math.inf)),
                     ((q, q), dict(workspace=Fake((64,), "uint8", dev=_Dev(index=2))))):
        with pytest.raises(ValueError):
            paged.attend(c, b, *args, **{"scale": 0.1, **kw})
    with pytest.raises(ValueError):
        paged.attend(cache(width=96), b, Fake((5, 4, 96)), Fake((5, 4, 96)), scale=0.1)
    with pytest.raises(ValueError):
        paged.attend(cache(heads=1, width=576, latent=True), b, Fake((5, 4, 576)), Fake((5, 4, 576)), scale=0.1)
    lat = cache(heads=1, width=576, latent=True)
    ql, qp = Fake((5, 4, 512)), Fake((5, 4, 64))
    for args in ((ql, None, ql), (ql, Fake((5, 4, 32)), ql), (ql, Fake((5, 3, 64)), ql), (ql, Fake((5, 4, 64), "float16"), ql)):
        with pytest.raises(ValueError):
            paged.attend_latent(lat, b, *args, scale=0.1)
    with pytest.raises(ValueError):
        paged.attend_latent(cache(), b, ql, qp, ql, scale=0.1)


def test_workspace():
    """None for short sequences; refused calls where one is needed and missing, small or askew."""
    short = batch(max_kv=64)
    assert paged.workspace_bytes(cache(), short, 4) == 0
    long = batch(S=1, per=4096, max_q=1, max_kv=65536)
    c = cache()
    need = paged.workspace_bytes(c, long, 4)
    assert need > 0 and need % 4 == 0
    assert paged.workspace_bytes(c, long, 4, tokens=2) == 2 * need
    q = Fake((1, 4, 64))
    for work in (None, Fake((need - 1,), "uint8"), Fake((need,), "uint8", ptr=(1 << 40) + 8)):
        with pytest.raises(ValueError):
            paged.attend(c, long, q, q, scale=0.1, workspace=work)
    with pytest.raises(ValueError):
        paged.workspace_bytes(c, long, 3)


def test_rope_refusals():
    x, pos, f = Fake((5, 4, 64)), Fake((5,), "int32"), Fake((32,), "float64")
    for args, kw in (((x, Fake((4,), "int32"), f), {}), ((x, Fake((5,), "float32"), f), {}), ((x, pos, Fake((32,), "float32")), {}),
                     ((x, pos, Fake((33,), "float64")), {}), ((x, pos, Fake((0,), "float64")), {}), ((x, pos, f), dict(offset=1)),
                     ((x, pos, f), dict(offset=-1)), ((x, pos, f), dict(layout="neox")), ((x, pos, f), dict(out=Fake((5, 4, 32)))),
                     ((x, pos, f), dict(k=Fake((5, 1, 32)))), ((x, pos, f), dict(k_out=x)), ((x, pos, f), dict(factor=math.nan)),
                     ((Fake((5, 64)), pos, f), {}), ((x, pos, f), dict(k=Fake((5, 1, 64), "float32"))),
                     ((x, pos, f), dict(out=Fake((5, 4, 64), strides=(512, 128, 1))))):
        with pytest.raises(ValueError):
            paged.rope(*args, **kw)


def test_sizes_past_the_index_types_are_refused():
    """Token counts that a 32-bit field would cut, and elements a token that a product would."""
    c, b = cache(), batch()
    many = Fake((1 << 31, 2, 64), strides=(0, 64, 1))
    with pytest.raises(ValueError):
        paged.append(c, b, many, many)
    x = Fake((1 << 31, 4, 64), strides=(0, 64, 1))
    with pytest.raises(ValueError):
        paged.rope(x, Fake((1 << 31,), "int32"), Fake((32,), "float64"))
    with pytest.raises(ValueError):
        paged.rope(Fake((1, 4097, 4096)), Fake((1,), "int32"), Fake((32,), "float64"))
    x = Fake((5, 4, 64))
    with pytest.raises(ValueError):      # rotated twice, by whichever thread comes first
        paged.rope(x, Fake((5,), "int32"), Fake((32,), "float64"), k=x)


def test_c_entries_refuse_sizes_and_addresses():
    """Rows past 2^30, grids past 2^32 threads, addresses off their type's size, a scale that
    overflows with log2 e: -1 before any device call; no tokens need no arrays."""
    L = _native.lib()
    for n, (res, args) in paged._PROTOS.items():
        getattr(L, n).restype, getattr(L, n).argtypes = res, args
    E = -1
    c, b = cache()._s, batch()._of(5)._obj
    q, r = paged._array(Fake((5, 4, 64)), "q", 0), paged._array(Fake((5, 2, 64)), "k", 0)
    lat = cache(heads=1, width=576, latent=True)._s

    def but(s, **kw):
        t = type(s)()
        ctypes.memmove(byref(t), byref(s), ctypes.sizeof(s))
        for name, value in kw.items():
            setattr(t, name, value)
        return t

    def attend(bb, lse=None, scale=0.1):
        return L.hearth_gpu_attend(byref(c), byref(bb), byref(q), byref(q), lse, scale, None, 0, 0, None)

    long = but(b, n_tokens=0x7fffffff, max_q=0x7fffffff)
    flat = but(r, token_stride=0)
    for fn in (L.hearth_gpu_kv_append, L.hearth_gpu_kv_read):
        assert fn(byref(c), byref(long), byref(flat), byref(flat), 0, None) == E
    far = but(b, max_kv=0x7fffffff, pages_per_seq=1 << 28, ld_pages=1 << 28)
    assert attend(far) == E and L.hearth_gpu_attend_workspace(byref(c), byref(far), 4) == E
    wide = but(b, n_seqs=65535, max_q=1 << 15, n_tokens=1 << 15)
    assert L.hearth_gpu_attend_workspace(byref(lat), byref(wide), 128) == E
    assert L.hearth_gpu_attend_workspace(byref(lat), byref(but(wide, max_q=1)), 128) >= 0
    for field, by in (("pages", 2), ("kv_len", 1), ("q_start", 3), ("mask", 4)):
        extra = {"mask_words": 1} if field == "mask" else {}
        bad = but(b, **{field: (1 << 40) + by}, **extra)
        assert attend(bad) == E, field
        assert L.hearth_gpu_kv_append(byref(c), byref(bad), byref(r), byref(r), 0, None) == E, field
    assert attend(b, lse=(1 << 40) + 2) == E
    assert attend(b, scale=3e38) == E
    none, no = but(b, n_tokens=0), lambda a: but(a, data=None)
    assert attend(none) == 0
    assert L.hearth_gpu_kv_append(byref(c), byref(none), byref(no(r)), byref(no(r)), 0, None) == 0
    assert L.hearth_gpu_attend(byref(c), byref(none), byref(no(q)), byref(no(q)), None, 0.1, None, 0, 0, None) == 0
    assert L.hearth_gpu_rope(byref(no(q)), byref(no(q)), byref(no(r)), byref(no(r)), 0, None, 0, 1 << 40, 32, 0, 0, 0, 1.0, 0, None) == 0


def test_c_entries_refuse():
    """NULL structs, shapes and strides that the kernels' indexing does not allow: -1, no device call."""
    L = _native.lib()
    for n, (res, args) in paged._PROTOS.items():
        getattr(L, n).restype, getattr(L, n).argtypes = res, args
    c, b = cache()._s, batch()._of(5)._obj
    q = paged._array(Fake((5, 4, 64)), "q", 0)
    r = paged._array(Fake((5, 2, 64)), "k", 0)
    E = -1
    assert L.hearth_gpu_kv_append(None, byref(b), byref(r), byref(r), 0, None) == E
    assert L.hearth_gpu_kv_append(byref(c), None, byref(r), byref(r), 0, None) == E
    assert L.hearth_gpu_kv_append(byref(c), byref(b), None, byref(r), 0, None) == E
    assert L.hearth_gpu_kv_append(byref(c), byref(b), byref(r), None, 0, None) == E
    assert L.hearth_gpu_kv_append(byref(c), byref(b), byref(r), byref(r), -1, None) == E
    assert L.hearth_gpu_attend(byref(c), byref(b), byref(q), None, None, 0.1, None, 0, 0, None) == E
    assert L.hearth_gpu_attend_latent(byref(c), byref(b), byref(q), None, byref(q), None, 0.1, None, 0, 0, None) == E

    def copy_of(s):
        t = type(s)()
        ctypes.memmove(byref(t), byref(s), ctypes.sizeof(s))
        return t

    for field, value in (("dtype", 0), ("dtype", 3), ("n_pages", 0), ("n_heads", 0), ("page", 24), ("page", 8192), ("width", 48),
                         ("width", 0)):
        bad = copy_of(c)
        setattr(bad, field, value)
        assert L.hearth_gpu_kv_read(byref(bad), byref(b), byref(r), byref(r), 0, None) == E, field
    for field, value in (("data", None), ("page_stride", 17), ("head_stride", 8), ("page_stride", -2048), ("data", (1 << 40) + 4),
                         ("page_stride", 1 << 50)):
        bad = copy_of(c)
        setattr(bad.k, field, value)
        assert L.hearth_gpu_kv_read(byref(bad), byref(b), byref(r), byref(r), 0, None) == E, field
    for field, value in (("n_seqs", -1), ("n_seqs", 70000), ("n_tokens", -1), ("max_q", -1), ("max_kv", -1), ("kv_len", None),
                         ("pages", None), ("ld_pages", 1), ("ld_pages", -4)):
        bad = copy_of(b)
        setattr(bad, field, value)
        assert L.hearth_gpu_kv_read(byref(c), byref(bad), byref(r), byref(r), 0, None) == E, field
    bad = copy_of(b)
    bad.mask, bad.mask_words = 1 << 40, 0
    assert L.hearth_gpu_attend(byref(c), byref(bad), byref(q), byref(q), None, 0.1, None, 0, 0, None) == E
    f = ctypes.c_void_p(1 << 40)
    for n, off in ((0, 0), (33, 0), (32, 1), (513, 0)):
        assert L.hearth_gpu_rope(byref(q), byref(q), None, None, 5, f, 0, f, n, off, 0, 0, 1.0, 0, None) == E
    assert L.hearth_gpu_rope(byref(q), byref(q), byref(r), None, 5, f, 0, f, 32, 0, 0, 0, 1.0, 0, None) == E
    # nothing to do is no error and no launch
    none = copy_of(b)
    none.n_tokens = 0
    assert L.hearth_gpu_attend(byref(c), byref(none), byref(q), byref(q), None, 0.1, None, 0, 0, None) == 0
    assert L.hearth_gpu_rope(byref(q), byref(q), None, None, 0, f, 0, f, 32, 0, 0, 0, 1.0, 0, None) == 0


def test_ctypes_mirrors_match_header(tmp_path):
    if not shutil.which("gcc"):
        pytest.skip("gcc not available")
    mirrors = {"hearth_gpu_rows": paged._Rows, "hearth_gpu_cache": paged._CacheS, "hearth_gpu_batch": paged._BatchS,
               "hearth_gpu_array": paged._Array}
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{INC / "hearth_gpu.h"}"', "int main(void) {"]
    for cname, m in mirrors.items():
        lines.append(f'    printf("{cname} size %zu\\n", sizeof({cname}));')
        lines += [f'    printf("{cname}.{f[0]} %zu\\n", offsetof({cname}, {f[0]}));' for f in m._fields_]
    lines += ['    printf("MX8 %d\\n", HEARTH_GPU_MX8);', "    return 0;", "}"]
    src, exe = tmp_path / "l.c", tmp_path / "l"
    src.write_text("\n".join(lines) + "\n")
    subprocess.run(["gcc", "-std=c11", "-I", str(INC), str(src), "-o", str(exe)], check=True)
    vals = dict(ln.rsplit(" ", 1) for ln in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines())
    assert int(vals["MX8"]) == paged.MX8
    for cname, m in mirrors.items():
        assert int(vals[f"{cname} size"]) == ctypes.sizeof(m)
        for f in m._fields_:
            assert int(vals[f"{cname}.{f[0]}"]) == getattr(m, f[0]).offset, (cname, f[0])


def test_rope_frequencies():
    f, a = paged.rope_frequencies(64, 10000.0)
    assert a == 1.0 and f[0] == 1.0 and np.allclose(f, [10000.0 ** (-2 * j / 64) for j in range(32)], rtol=1e-14)
    lin, _ = paged.rope_frequencies(64, 10000.0, "linear", factor=4.0)
    assert np.array_equal(lin, f / 4)
    ntk, _ = paged.rope_frequencies(64, 10000.0, "ntk", factor=4.0)
    assert ntk[0] == 1.0 and math.isclose(ntk[-1], f[-1] / 4, rel_tol=1e-12)
    yarn, a = paged.rope_frequencies(64, 10000.0, "yarn", factor=40.0, original=4096)
    turns = 4096 * f / (2 * math.pi)
    assert math.isclose(a, 0.1 * math.log(40) + 1)
    assert np.array_equal(yarn[turns > 40], f[turns > 40]) and np.allclose(yarn[turns < 0.7], f[turns < 0.7] / 40, rtol=1e-14)
    assert ((yarn <= f) & (yarn >= f / 40 * (1 - 1e-14))).all() and (np.diff(yarn) < 0).all()
    l3, _ = paged.rope_frequencies(128, 500000.0, "llama3", factor=8.0, original=8192)
    g, _ = paged.rope_frequencies(128, 500000.0)
    wave = 2 * math.pi / g
    assert np.array_equal(l3[wave < 8192 / 4], g[wave < 8192 / 4])
    assert np.allclose(l3[wave > 8192], g[wave > 8192] / 8, rtol=1e-14)
    for bad in (dict(rot=7), dict(rot=0), dict(rot=64, base=0), dict(rot=64, scaling="dynamic"), dict(rot=64, factor=0),
                dict(rot=2, scaling="ntk")):
        with pytest.raises(ValueError):
            paged.rope_frequencies(**bad)


def test_sequence_bounds():
    """seq_of of hx_paged.h, restated and enumerated over wild lengths and starts: tokens stay in
    [0, n_tokens), rows in [0, kv_cap), table entries in [0, pages_per_seq)."""
    text = (Path(paged.__file__).parent / "csrc" / "hx_paged.h").read_text()
    for line in ("const int lo = min(max(word_of(b.q_start, s), 0), b.n_tokens);", "const int hi = min(max(word_of(b.q_start, s + 1), lo), b.n_tokens);",
                 "const int len = max(word_of(b.kv_len, s), 0);", "r.kv = min(len, b.kv_cap);", "r.base = len - r.n;"):
        assert line in re.sub(r"[ ]+", " ", text), "the restatement below is of other code"
    wild = [-2 ** 31, -7, 0, 1, 5, 16, 40, 64, 100, 2 ** 31 - 1]
    n_tokens, per, page = 40, 4, 16
    for max_kv in (0, 20, 64, 2 ** 31 - 1):
        cap = min(max_kv, per * page)
        for a in wild:
            for b in wild:
                lo = min(max(a, 0), n_tokens)
                hi = min(max(b, lo), n_tokens)
                for L in wild:
                    n, length = hi - lo, max(L, 0)
                    kv, base = min(length, cap), length - n
                    assert 0 <= lo <= hi <= n_tokens and -2 ** 31 <= base < 2 ** 31 and base + n < 2 ** 31
                    for i in (0, n - 1):
                        p = base + i
                        if n and 0 <= p < kv:                       # append, read
                            assert p // page < per
                    if kv:
                        assert (kv - 1) // page < per               # attention reads rows below kv
