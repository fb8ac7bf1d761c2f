"""The bounds that include/hearth_gpu.h states, against what the C entry points take: on the CPU, with
a device that is not there, so that a call within them ends at the device (-4) and one past them
with -1."""
from __future__ import annotations

import ctypes
import re
from ctypes import byref
from pathlib import Path

from hearth_amd import paged
from test_paged_args import Fake, batch, cache

HEADER = re.sub(r"\s*\n \*\s*", " ", (Path(paged.__file__).resolve().parents[1] / "include" / "hearth_gpu.h").read_text())
NONE = 1000   # a device


def but(s, **kw):
    t = type(s)()
    ctypes.memmove(byref(t), byref(s), ctypes.sizeof(s))
    for name, value in kw.items():
        setattr(t, name, value)
    return t


def copy(fn, heads, width, tokens):
    """a write or read of so many tokens of one sequence (k and v: 2 heads width elements a token)"""
    c = cache(heads=heads, width=width)._s
    b = but(batch(S=1)._of(1)._obj, n_tokens=tokens, max_q=tokens)
    r = but(paged._array(Fake((1, heads, width)), "k", 0), token_stride=heads * width)
    return paged._fn(fn)(byref(c), byref(b), byref(r), byref(r), NONE, None)


def test_tokens_of_writes_and_reads():
    top, narrow = re.search(r"min\(max_q, n_tokens\) is at most 2\^26 - (\d+) \(more where a token's rows, k and v together, have at "
                            r"most (\d+) elements; reads alike\)", HEADER).groups()
    top, narrow = 2 ** 26 - int(top), int(narrow)
    for fn in ("hearth_gpu_kv_append", "hearth_gpu_kv_read"):
        for heads, width in ((4, 128 + 32), (4, 256), (16, 256)):           # 1280, 2048 and 8192 elements
            assert 2 * heads * width > narrow
            assert copy(fn, heads, width, top) == -4 and copy(fn, heads, width, top + 1) == -1, (fn, heads, width)
        assert copy(fn, narrow // 256, 128, top + 1) == -4
        assert copy(fn, 1, narrow // 2 + 32, top + 1) == -1                 # the next width


def test_columns_of_latent_attention():
    tiles = int(re.search(r"n_seqs times min\(max_q, n_tokens\) \* H / 64, rounded up, at most (\d+)", HEADER).group(1))
    lat, b = cache(heads=1, width=576, latent=True)._s, batch()._of(5)._obj
    need = lambda S, q, H: paged._fn("hearth_gpu_attend_workspace")(byref(lat), byref(but(b, n_seqs=S, max_q=q, n_tokens=q, ld_pages=4)), H)
    for S, H in ((4096, 128), (16, 5), (65535, 1)):
        q = tiles // S * 64 // H                                            # the most tokens
        assert need(S, q, H) >= 0 and need(S, q + 1 if H >= 64 else q + 64 // H + 1, H) == -1, (S, H)
