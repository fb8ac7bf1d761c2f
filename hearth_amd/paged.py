"""Operators over paged key-value caches on the GPU (the paged section of include/hearth_gpu.h).

For programs that keep many conversations' rows in pages next to (or without) an Engine:

    rope(x, pos, freqs)              rotary positions, in place or into `out`
    append(cache, batch, k, v)       new tokens' rows into the pages, 16-bit, 8-bit ("mx8") or 4-bit ("mx4")
    append_rotated(cache, batch, q, k, v, freqs)   rope of q and k and append in one launch
    read(cache, batch, k, v)         rows back out of the pages
    attend(cache, batch, q, out)     grouped-head attention: tokens, chains, draft trees, prompts
    attend_latent(...)               absorbed latent attention over one row a token

and, for long sequences of which each token looks at a few blocks of rows only:

    update_bounds(cache, batch, bounds)        bounds of the keys of each block, after append
    select(bounds, batch, q, chosen)           the blocks that each token is to look at
    attend_blocks(cache, batch, q, chosen, out)   attention over their rows

Arrays are device tensors: anything with data_ptr(), shape, stride(), dtype, get_device(),
element_size() and is_contiguous() as torch tensors have them (torch itself is not imported). Work is enqueued
on `stream` (a HIP stream handle such as torch.cuda.current_stream().cuda_stream; 0 is the
null stream) of the tensors' device and not waited for, so the tensors must live until it has
run; nothing is allocated, so a call may be captured into a graph. ValueError for arguments that do not fit together, HearthError for
a device error. The operators have no gradients: tensors that require one are refused where
gradients are recorded (call under torch.no_grad(), or detach them).

No counterpart in the reference, whose engine keeps one conversation in float32 on the host.
"""
from __future__ import annotations

import ctypes
import math
import sys
from ctypes import POINTER, Structure, byref, c_double, c_float, c_int, c_int32, c_int64, c_size_t, c_void_p

import numpy as np

from . import _native
from .engine import HearthError

__all__ = ["Cache", "Batch", "rope", "rope_frequencies", "append", "append_rotated", "read", "attend", "attend_latent",
           "workspace_bytes", "Bounds", "update_bounds", "select", "select_workspace_bytes", "attend_blocks",
           "attend_blocks_workspace_bytes"]

F32, F16, BF16, MX8, MX4 = 0, 1, 2, 16, 17
_DTYPES = {"float32": F32, "float16": F16, "bfloat16": BF16, "float8_e4m3fn": MX8, "float4_e2m1fn_x2": MX4}


class _Rows(Structure):
    _fields_ = [("data", c_void_p), ("scales", c_void_p), ("page_stride", c_int64), ("head_stride", c_int64),
                ("scale_page_stride", c_int64), ("scale_head_stride", c_int64)]


class _CacheS(Structure):
    _fields_ = [("k", _Rows), ("v", _Rows), ("dtype", c_int32), ("n_pages", c_int32), ("n_heads", c_int32),
                ("page", c_int32), ("width", c_int32)]


class _BatchS(Structure):
    _fields_ = [("pages", c_void_p), ("kv_len", c_void_p), ("q_start", c_void_p), ("mask", c_void_p),
                ("ld_pages", c_int64), ("n_seqs", c_int32), ("pages_per_seq", c_int32), ("n_tokens", c_int32),
                ("max_q", c_int32), ("max_kv", c_int32), ("mask_words", c_int32)]


class _Array(Structure):
    _fields_ = [("data", c_void_p), ("token_stride", c_int64), ("head_stride", c_int64), ("dtype", c_int32),
                ("n_heads", c_int32), ("width", c_int32)]


class _BoundsS(Structure):
    _fields_ = [("codes", c_void_p), ("scales", c_void_p), ("page_stride", c_int64), ("head_stride", c_int64),
                ("scale_page_stride", c_int64), ("scale_head_stride", c_int64), ("n_pages", c_int32), ("n_heads", c_int32),
                ("block", c_int32), ("blocks", c_int32), ("width", c_int32)]


class _BlocksS(Structure):
    _fields_ = [("chosen", c_void_p), ("token_stride", c_int64), ("head_stride", c_int64), ("top", c_int32), ("block", c_int32)]


_PROTOS = {
    "hearth_gpu_rope": (c_int, [POINTER(_Array), POINTER(_Array), POINTER(_Array), POINTER(_Array), c_int, c_void_p,
                                c_int, c_void_p, c_int, c_int, c_int, c_int, c_double, c_int, c_void_p]),
    "hearth_gpu_kv_append": (c_int, [POINTER(_CacheS), POINTER(_BatchS), POINTER(_Array), POINTER(_Array), c_int,
                                     c_void_p]),
    "hearth_gpu_kv_append_rotated": (c_int, [POINTER(_CacheS), POINTER(_BatchS), POINTER(_Array), POINTER(_Array), POINTER(_Array),
                                             POINTER(_Array), c_void_p, c_int, c_void_p, c_int, c_int, c_int, c_double, c_int,
                                             c_void_p]),
    "hearth_gpu_kv_read": (c_int, [POINTER(_CacheS), POINTER(_BatchS), POINTER(_Array), POINTER(_Array), c_int,
                                   c_void_p]),
    "hearth_gpu_attend": (c_int, [POINTER(_CacheS), POINTER(_BatchS), POINTER(_Array), POINTER(_Array), c_void_p,
                                  c_float, c_void_p, c_size_t, c_int, c_void_p]),
    "hearth_gpu_attend_latent": (c_int, [POINTER(_CacheS), POINTER(_BatchS), POINTER(_Array), POINTER(_Array),
                                         POINTER(_Array), c_void_p, c_float, c_void_p, c_size_t, c_int, c_void_p]),
    "hearth_gpu_key_bounds": (c_int, [POINTER(_CacheS), POINTER(_BatchS), POINTER(_BoundsS), c_int, c_void_p]),
    "hearth_gpu_select_blocks": (c_int, [POINTER(_BoundsS), POINTER(_BatchS), POINTER(_Array), POINTER(_BlocksS), c_int, c_int,
                                         c_void_p, c_size_t, c_int, c_void_p]),
    "hearth_gpu_attend_blocks": (c_int, [POINTER(_CacheS), POINTER(_BatchS), POINTER(_Array), POINTER(_BlocksS), POINTER(_Array),
                                         c_void_p, c_float, c_void_p, c_size_t, c_int, c_void_p]),
    "hearth_gpu_attend_blocks_workspace": (c_int64, [POINTER(_CacheS), POINTER(_BatchS), c_int, c_int, c_int]),
    "hearth_gpu_select_workspace": (c_int64, [POINTER(_BoundsS), POINTER(_BatchS)]),
    "hearth_gpu_attend_workspace": (c_int64, [POINTER(_CacheS), POINTER(_BatchS), c_int]),
}
_fns: dict = {}


def _one_runtime():
    """Streams and tensors of one copy of the HIP runtime mean nothing to another: a framework
    that brings its own copy must be imported before the library is loaded, which then takes
    that one."""
    try:
        with open("/proc/self/maps") as f:
            libs = {ln.split()[-1] for ln in f if "libamdhip64" in ln}
    except OSError:
        return
    if len(libs) > 1:
        raise HearthError("two copies of the HIP runtime are loaded (" + ", ".join(sorted(libs)) + "): import the "
                          "framework of the tensors before the first call of hearth_amd that loads its library")


def _fn(name):
    f = _fns.get(name)
    if f is None:
        f = getattr(_native.lib(), name)
        _one_runtime()
        f.restype, f.argtypes = _PROTOS[name]
        _fns[name] = f
    return f


_seen_dtypes: dict = {}


def _dtype(t) -> int:
    d = t.dtype
    c = _seen_dtypes.get(d)
    if c is None:
        c = _DTYPES.get(str(d).replace("torch.", ""))
        if c is None:
            raise ValueError(f"dtype {d} is none of float32, float16, bfloat16 (float8_e4m3fn, float4_e2m1fn_x2 in a cache)")
        _seen_dtypes[d] = c
    return c


def _device(t, what, want=None) -> int:
    i = t.get_device()
    if i < 0:
        raise ValueError(f"{what} is not on a GPU")
    if want is not None and i != want:
        raise ValueError(f"{what} is on device {i}, not on device {want}")
    return i


def _refuse_gradient(what):
    """For a tensor that requires a gradient: autograd would not see what the call reads or writes."""
    torch = sys.modules.get("torch")
    if torch is None or torch.is_grad_enabled():
        raise ValueError(f"{what} requires a gradient, and these operators have none: call under torch.no_grad() or detach it")


def _array(t, what, dev) -> _Array:
    """[tokens, heads, width] with a dense last dimension."""
    if getattr(t, "requires_grad", False):
        _refuse_gradient(what)
    shape = t.shape
    if len(shape) != 3:
        raise ValueError(f"{what}: shape {tuple(shape)} is not [tokens, heads, width]")
    _, heads, width = shape
    st, sh, sw = t.stride()
    if sw != 1 and width > 1:
        raise ValueError(f"{what}: the last dimension is not dense (stride {sw})")
    if t.get_device() != dev:
        _device(t, what, dev)
    dt = _seen_dtypes.get(t.dtype)
    if dt is None:
        dt = _dtype(t)
    if dt >= MX8:
        raise ValueError(f"{what}: {t.dtype} rows live in a cache only")
    return _Array(t.data_ptr(), st, sh, dt, heads, width)


_seen_ints: dict = {}


def _ints(t, what, dev, ndim, names=("torch.int32", "int32")):
    shape, name = t.shape, _seen_ints.get(t.dtype)
    if name is None:
        name = _seen_ints[t.dtype] = str(t.dtype)
    if name not in names or len(shape) != ndim:
        raise ValueError(f"{what}: {t.dtype}{tuple(shape)}, wanted {names[-1]} with {ndim} dimension(s)")
    if shape[-1] > 1 and t.stride()[-1] != 1:
        raise ValueError(f"{what}: the last dimension is not dense")
    if t.get_device() != dev:
        _device(t, what, dev)
    return t.data_ptr()


def _check(rc, what):
    if rc == 0:
        return
    if rc == -1:
        raise ValueError(f"{what}: arguments that do not fit together (see include/hearth_gpu.h)")
    if rc == -3:
        raise ValueError(f"{what}: the workspace is too small (workspace_bytes)")
    raise HearthError(f"{what} failed (code {rc}): device error")


class Cache:
    """Rows of all sequences: k and v [pages, heads, rows a page, width], float16, bfloat16,
    float8_e4m3fn or (two elements a byte, [.., width / 2]) float4_e2m1fn_x2, the latter two with
    scales (uint8 E8M0, [pages, heads, rows a page, width / 32]); v None:
    latent rows (latent vector, then its rotated part). The last two dimensions are dense; the
    tensors are the caller's and stay referenced."""

    def __init__(self, k, v=None, k_scale=None, v_scale=None):
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.device = _device(k, "k")
        dt = _dtype(k)
        if dt == F32:
            raise ValueError("cache rows are float16, bfloat16, float8_e4m3fn or float4_e2m1fn_x2")
        s = _CacheS()
        if len(k.shape) != 4:
            raise ValueError(f"k: shape {tuple(k.shape)} is not [pages, heads, rows a page, width]")
        s.dtype, (s.n_pages, s.n_heads, s.page, s.width) = dt, k.shape
        s.width *= 2 if dt == MX4 else 1
        s.k = self._rows(k, k_scale, "k", k, dt)
        if v is not None:
            s.v = self._rows(v, v_scale, "v", k, dt)
        elif v_scale is not None:
            raise ValueError("v_scale without v")
        if s.page < 16 or s.page > 4096 or s.page & (s.page - 1):
            raise ValueError(f"{s.page} rows a page: a power of two from 16 to 4096 is needed")
        if s.width % 32 or not 32 <= s.width <= 1024:
            raise ValueError(f"width {s.width}: a multiple of 32 up to 1024 is needed")
        self._s = s
        self._ref = byref(s)

    def _no_gradient(self):
        if getattr(self.k, "requires_grad", False) or getattr(self.v, "requires_grad", False):
            _refuse_gradient("the cache")

    def _rows(self, t, scale, what, like, dt) -> _Rows:
        if tuple(t.shape) != tuple(like.shape) or _dtype(t) != dt:
            raise ValueError(f"{what}: {t.dtype}{tuple(t.shape)} differs from k's {like.dtype}{tuple(like.shape)}")
        _device(t, what, self.device)
        st = t.stride()
        if st[3] != 1 or st[2] != t.shape[3]:
            raise ValueError(f"{what}: the last two dimensions are not dense (strides {st})")
        if any(b % 16 for b in (t.data_ptr(), st[0] * t.element_size(), st[1] * t.element_size())):
            raise ValueError(f"{what}: data and strides must be multiples of 16 bytes")
        r = _Rows(t.data_ptr(), None, st[0], st[1], 0, 0)
        if (scale is not None) != (dt >= MX8):
            raise ValueError(f"{what}: scales go with float8_e4m3fn and float4_e2m1fn_x2 rows, and only with them")
        if scale is not None:
            want = (*t.shape[:3], t.shape[3] // (16 if dt == MX4 else 32))
            if tuple(scale.shape) != want or str(scale.dtype) not in ("torch.uint8", "torch.float8_e8m0fnu"):
                raise ValueError(f"{what} scales: {scale.dtype}{tuple(scale.shape)}, wanted uint8{want}")
            _device(scale, f"{what} scales", self.device)
            ss = scale.stride()
            if (want[3] > 1 and ss[3] != 1) or ss[2] != want[3]:
                raise ValueError(f"{what} scales: the last two dimensions are not dense (strides {ss})")
            r.scales, r.scale_page_stride, r.scale_head_stride = scale.data_ptr(), ss[0], ss[1]
        return r


class Batch:
    """The sequences of a call, all in device memory: pages int32 [sequences, pages a sequence]
    (which page holds rows p * page .. of the sequence), kv_len int32 [sequences] (rows of each,
    the call's tokens included), q_start int32 [sequences + 1] (sequence s owns the call's
    tokens q_start[s] .. q_start[s + 1), its last ones). max_q and max_kv bound the token counts
    and lengths on the host: tokens and rows beyond them are not computed. mask int64
    [tokens, words]: token t attends its sequence's earlier rows and the call's token j of its
    sequence where bit j % 64 of word j / 64 is set; None: every row up to its own."""

    def __init__(self, pages, kv_len, q_start, *, max_q, max_kv, mask=None):
        self.pages, self.kv_len, self.q_start, self.mask = pages, kv_len, q_start, mask
        self.device = _device(pages, "pages")
        s = _BatchS()
        s.pages = _ints(pages, "pages", self.device, 2)
        s.kv_len = _ints(kv_len, "kv_len", self.device, 1)
        s.q_start = _ints(q_start, "q_start", self.device, 1)
        n = kv_len.shape[0]
        if pages.shape[0] != n or q_start.shape[0] != n + 1:
            raise ValueError(f"{pages.shape[0]} page rows, {n} lengths and {q_start.shape[0]} starts (one more wanted)")
        if n > 65535:
            raise ValueError(f"{n} sequences (at most 65535)")
        if max_q < 0 or max_kv < 0 or max_q > 0x7fffffff or max_kv > 0x7fffffff:
            raise ValueError(f"max_q {max_q}, max_kv {max_kv}")
        s.n_seqs, s.pages_per_seq = n, pages.shape[1]
        s.ld_pages = pages.stride()[0] if n > 1 else pages.shape[1]
        if s.ld_pages < s.pages_per_seq:
            raise ValueError("pages: rows overlap")
        s.max_q, s.max_kv = max_q, max_kv
        if mask is not None:
            s.mask = _ints(mask, "mask", self.device, 2, ("torch.int64", "torch.uint64", "int64"))
            s.mask_words = mask.shape[1]
            if 64 * mask.shape[1] < max_q:
                raise ValueError(f"mask: {mask.shape[1]} words hold fewer than max_q = {max_q} tokens")
            if mask.shape[0] > 1 and mask.stride()[0] != mask.shape[1]:
                raise ValueError("mask: rows are not dense")
        self._s = s

    def _of(self, n):
        """The struct of a call of n tokens: a copy, so that threads may share a Batch."""
        if n > 0x7fffffff:
            raise ValueError(f"{n} tokens (at most 2147483647)")
        if self.mask is not None and self.mask.shape[0] < n:
            raise ValueError(f"mask: {self.mask.shape[0]} rows for {n} tokens")
        s = _BatchS.from_buffer_copy(self._s)
        s.n_tokens = n
        return byref(s)


def _pair(cache, batch, k, v, what):
    if batch.device != cache.device:
        raise ValueError(f"{what}: the batch is on device {batch.device}, the cache on device {cache.device}")
    cache._no_gradient()
    a = _array(k, "k", cache.device)
    b = None
    if v is not None:
        b = _array(v, "v", cache.device)
        if v.shape[0] != k.shape[0] or b.dtype != a.dtype:
            raise ValueError(f"{what}: k is {k.dtype}{tuple(k.shape)}, v {v.dtype}{tuple(v.shape)}")
    c = cache._s
    heads, width, latent = c.n_heads, c.width, cache.v is None
    if not latent and v is None:
        raise ValueError(f"{what}: the cache holds keys and values, v is missing")
    total = a.width + b.width if latent and b is not None else a.width
    if a.n_heads != heads or (b is not None and b.n_heads != heads) or total != width or \
            (not latent and b.width != width) or a.width % 32 or (b is not None and b.width % 32):
        raise ValueError(f"{what}: rows {tuple(k.shape)}" + (f" and {tuple(v.shape)}" if v is not None else "") +
                         f" do not make cache rows of {heads} head(s) and width {width} in pieces of 32")
    return a, b, batch._of(k.shape[0])


def append(cache: Cache, batch: Batch, k, v=None, *, stream=0) -> None:
    """Writes the call's tokens' rows k, v [tokens, heads, width] (float32, float16 or bfloat16)
    into the cache; a latent cache takes the latents as k and their rotated parts as v."""
    a, b, bs = _pair(cache, batch, k, v, "append")
    rc = _fn("hearth_gpu_kv_append")(cache._ref, bs, byref(a), byref(b) if b is not None else None, cache.device, stream)
    if rc:
        _check(rc, "append")


def append_rotated(cache: Cache, batch: Batch, q, k, v, freqs, *, pos=None, factor=1.0, layout="half", offset=0, q_out=None,
                   stream=0) -> None:
    """rope of q and k and append of the rotated keys and of v in one launch, to the same bits: q
    [tokens, heads, width] in place or into q_out (None: keys alone), k on its way into the cache (the
    tensor stays as it is). A latent cache takes the latents as k and rotates v, their second part,
    whose width q has. pos [tokens] (int32 or int64), None: each token's row number in its sequence.
    Queries of tokens of no sequence (padding) and of those past max_q are left as they are, in q_out too.
    freqs, factor, layout, offset: as in rope; q_out is q or shares nothing with q, k and v."""
    if layout not in ("half", "interleaved"):
        raise ValueError(f"layout {layout!r} is neither 'half' nor 'interleaved'")
    a, b, bs = _pair(cache, batch, k, v, "append_rotated")
    dev, latent, tokens = cache.device, cache.v is None, k.shape[0]
    if latent and b is None:
        raise ValueError("append_rotated: v, the latent rows' rotated part, is missing")
    width = b.width if latent else a.width
    aq = ao = None
    if q is not None:
        ao = aq = _array(q, "q", dev)
        if q.shape[0] != tokens or aq.width != width or aq.dtype != a.dtype:
            raise ValueError(f"append_rotated: q is {q.dtype}{tuple(q.shape)}, the rotated rows {k.dtype} of width {width}")
        if q_out is not None and q_out is not q:
            ao = _array(q_out, "q_out", dev)
            if q_out.shape[0] != tokens or ao.n_heads != aq.n_heads or ao.width != width or ao.dtype != aq.dtype:
                raise ValueError(f"q_out is {q_out.dtype}{tuple(q_out.shape)}, q {q.dtype}{tuple(q.shape)}")
        if tokens and (ao.data == a.data or (b is not None and ao.data == b.data)):
            raise ValueError("q_out shares the elements of k or v")
    elif q_out is not None:
        raise ValueError("q_out without q")
    f = _ints(freqs, "freqs", dev, 1, ("torch.float64", "float64"))
    if getattr(freqs, "requires_grad", False):
        _refuse_gradient("freqs")
    n = freqs.shape[0]
    if not 1 <= n <= 512 or offset < 0 or offset + 2 * n > width:
        raise ValueError(f"{n} pairs at {offset} do not fit a width of {width}")
    p, p64 = None, False
    if pos is not None:
        p = _ints(pos, "pos", dev, 1, ("torch.int32", "torch.int64", "int32 or int64"))
        p64 = _seen_ints[pos.dtype] == "torch.int64"
        if pos.shape[0] != tokens:
            raise ValueError(f"{pos.shape[0]} positions for {tokens} tokens")
    rc = _fn("hearth_gpu_kv_append_rotated")(cache._ref, bs, byref(aq) if aq is not None else None, byref(ao) if ao is not None else None,
                                             byref(a), byref(b) if b is not None else None, p, p64, f, n, offset,
                                             layout == "interleaved", float(factor), dev, stream)
    if rc:
        _check(rc, "append_rotated")


def read(cache: Cache, batch: Batch, k, v=None, *, stream=0) -> None:
    """The inverse of append: fills k, v [tokens, heads, width] with the call's tokens' rows
    (zeros for rows that are not in the cache). q_start = running sum of kv_len reads whole
    sequences."""
    a, b, bs = _pair(cache, batch, k, v, "read")
    rc = _fn("hearth_gpu_kv_read")(cache._ref, bs, byref(a), byref(b) if b is not None else None, cache.device, stream)
    if rc:
        _check(rc, "read")


def _for_tokens(batch, tokens) -> _BatchS:
    """The struct of a call of `tokens` tokens (None: as many as sequences times max_q)."""
    s = _BatchS.from_buffer_copy(batch._s)
    s.n_tokens = n = min(s.n_seqs * s.max_q, 0x7fffffff) if tokens is None else tokens
    if s.n_tokens != n:
        raise ValueError(f"{n} tokens (at most 2147483647)")
    return s


def workspace_bytes(cache: Cache, batch: Batch, heads: int, tokens: int | None = None) -> int:
    """Bytes of device workspace that attend / attend_latent need for `tokens` query tokens
    (None: as many as sequences times max_q) of `heads` heads: 0 when none is."""
    s = _for_tokens(batch, tokens)
    n = _fn("hearth_gpu_attend_workspace")(cache._ref, byref(s), heads) if 1 <= heads <= 65536 else -1
    if n < 0:
        raise ValueError(f"no attention over this cache (heads {cache._s.n_heads}, width {cache._s.width}) "
                         f"with {heads} query heads")
    return n


def _attend(name, cache, batch, q, q_pe, out, lse, scale, workspace, stream, chosen=None, block=0):
    dev = cache.device
    if batch.device != dev:
        raise ValueError(f"{name}: the batch is on device {batch.device}, the cache on device {dev}")
    cache._no_gradient()
    a, o, tokens = _array(q, "q", dev), _array(out, "out", dev), q.shape[0]
    if out.shape[0] != tokens or o.n_heads != a.n_heads or o.width != a.width or a.dtype != o.dtype:
        raise ValueError(f"{name}: out is {out.dtype}{tuple(out.shape)}, q {q.dtype}{tuple(q.shape)}")
    if a.dtype == F32 or cache._s.dtype not in (MX8, MX4, a.dtype):
        raise ValueError(f"{name}: q is {q.dtype} over a cache of {cache.k.dtype}")
    lp = None
    if lse is not None:
        if tuple(lse.shape) != tuple(q.shape[:2]) or str(lse.dtype) != "torch.float32" or not lse.is_contiguous():
            raise ValueError(f"lse: {lse.dtype}{tuple(lse.shape)}, wanted dense float32{tuple(q.shape[:2])}")
        _device(lse, "lse", dev)
        if getattr(lse, "requires_grad", False):
            _refuse_gradient("lse")
        lp = lse.data_ptr()
    wp, wb = None, 0
    if workspace is not None:
        _device(workspace, "workspace", dev)
        if not workspace.is_contiguous():
            raise ValueError("workspace: not dense")
        wp, wb = workspace.data_ptr(), workspace.numel() * workspace.element_size()
    bs = batch._of(tokens)
    if chosen is not None:
        x = _blocks(chosen, "chosen", dev, tokens, cache._s.n_heads, block)
        rc = _fn("hearth_gpu_attend_blocks")(cache._ref, bs, byref(a), byref(x), byref(o), lp, float(scale), wp, wb, dev, stream)
    elif q_pe is None:
        rc = _fn("hearth_gpu_attend")(cache._ref, bs, byref(a), byref(o), lp, float(scale), wp, wb, dev, stream)
    else:
        pe = _array(q_pe, "q_pe", dev)
        if q_pe.shape[0] != tokens or pe.n_heads != a.n_heads or pe.dtype != a.dtype:
            raise ValueError(f"{name}: q_pe is {q_pe.dtype}{tuple(q_pe.shape)}, q {q.dtype}{tuple(q.shape)}")
        rc = _fn("hearth_gpu_attend_latent")(cache._ref, bs, byref(a), byref(pe), byref(o), lp, float(scale), wp, wb, dev, stream)
    if rc == -1 and (wp is None or wp % 16):
        if chosen is not None:
            need = attend_blocks_workspace_bytes(cache, batch, a.n_heads, x.top, block, tokens)
        else:
            need = workspace_bytes(cache, batch, a.n_heads, tokens)
        if need:
            raise ValueError(f"{name}: a workspace of {need} bytes on 16 is needed")
    if rc:
        _check(rc, name)


def attend(cache: Cache, batch: Batch, q, out, *, scale: float, lse=None, workspace=None, stream=0) -> None:
    """out = softmax(scale * q k) v of the call's tokens over the rows each attends; q, out
    [tokens, heads, width] of the cache's 16-bit dtype (either over mx8 and mx4 rows), heads a multiple of
    the cache's. lse: float32 [tokens, heads] or None. workspace: a device tensor of
    workspace_bytes; calls that may run at the same time must not share one. A token that
    attends nothing gets zeros, one all of whose scores are -inf gets NaN (lse -inf for both)."""
    _attend("attend", cache, batch, q, None, out, lse, scale, workspace, stream)


def attend_latent(cache: Cache, batch: Batch, q, q_pe, out, *, scale: float, lse=None, workspace=None,
                  stream=0) -> None:
    """Absorbed latent attention: q [tokens, heads, 512] and q_pe [tokens, heads, 64] over a
    latent cache of width 576 (not mx4), out [tokens, heads, 512]; the rest as attend."""
    if q_pe is None:
        raise ValueError("attend_latent: q_pe is missing")
    _attend("attend_latent", cache, batch, q, q_pe, out, lse, scale, workspace, stream)


class Bounds:
    """Bounds of the keys of each block of a cache's rows: low_high int8 [pages, heads, blocks a page, 2,
    width] (least and greatest value of each element in whole steps) and steps uint8 [pages, heads,
    blocks a page] (the step as exponent + 127). block: rows of a block, a power of two from 16 up to a
    page. Dense but for the first two dimensions; the tensors are the caller's, filled by update_bounds."""

    def __init__(self, low_high, steps, *, block: int):
        self.low_high, self.steps, self.block = low_high, steps, block
        self.device = _device(low_high, "low_high")
        shape = tuple(low_high.shape)
        if len(shape) != 5 or shape[3] != 2 or str(low_high.dtype) not in ("torch.int8", "int8"):
            raise ValueError(f"low_high: {low_high.dtype}{shape}, wanted int8 [pages, heads, blocks a page, 2, width]")
        if tuple(steps.shape) != shape[:3] or str(steps.dtype) not in ("torch.uint8", "uint8"):
            raise ValueError(f"steps: {steps.dtype}{tuple(steps.shape)}, wanted uint8{shape[:3]}")
        _device(steps, "steps", self.device)
        st, ss = low_high.stride(), steps.stride()
        if st[4] != 1 or st[3] != shape[4] or (shape[2] > 1 and st[2] != 2 * shape[4]) or (shape[2] > 1 and ss[2] != 1):
            raise ValueError(f"low_high, steps: strides {st} and {ss}, dense blocks are wanted")
        s = _BoundsS()
        s.codes, s.page_stride, s.head_stride = low_high.data_ptr(), st[0], st[1]
        s.scales, s.scale_page_stride, s.scale_head_stride = steps.data_ptr(), ss[0], ss[1]
        (s.n_pages, s.n_heads, s.blocks), s.width, s.block = shape[:3], shape[4], block
        if not 16 <= block <= 4096 or block & (block - 1) or s.blocks < 1 or s.blocks & (s.blocks - 1) or block * s.blocks > 4096:
            raise ValueError(f"{s.blocks} blocks of {block} rows do not make a page (powers of two, 16 to 4096 rows)")
        if s.width not in (64, 128, 256):
            raise ValueError(f"width {s.width} is none of 64, 128, 256")
        if s.codes % 16 or (s.n_pages > 1 and st[0] % 16) or (s.n_heads > 1 and st[1] % 16):
            raise ValueError("low_high: data and strides must be multiples of 16 bytes")
        self._s = s
        self._ref = byref(s)


def _blocks(chosen, what, dev, tokens, heads, block) -> _BlocksS:
    """int32 [tokens, heads, top]"""
    p = _ints(chosen, what, dev, 3)
    shape, st = chosen.shape, chosen.stride()
    if shape[0] != tokens or shape[1] != heads or not 1 <= shape[2] <= 1 << 20:
        raise ValueError(f"{what}: shape {tuple(shape)} is not [{tokens} tokens, {heads} heads, top]")
    if not 16 <= block <= 4096:
        raise ValueError(f"blocks of {block} rows (a power of two from 16 up to a page is needed)")
    return _BlocksS(p, st[0], st[1], shape[2], block)


def update_bounds(cache: Cache, batch: Batch, bounds: Bounds, *, stream=0) -> None:
    """Brings the bounds of the blocks that hold rows of the call's tokens (those of the batch: q_start,
    max_q) up to date, over all of their rows that exist. After append, before select."""
    dev = cache.device
    if batch.device != dev or bounds.device != dev:
        raise ValueError(f"update_bounds: cache, batch and bounds are on devices {dev}, {batch.device} and {bounds.device}")
    cache._no_gradient()
    c, s = cache._s, bounds._s
    if cache.v is None:
        raise ValueError("update_bounds: a latent cache has no keys of its own")
    if (s.n_pages, s.n_heads, s.block * s.blocks, s.width) != (c.n_pages, c.n_heads, c.page, c.width):
        raise ValueError(f"update_bounds: bounds of {s.n_pages} pages of {s.blocks} x {s.block} rows, {s.n_heads} heads of {s.width} over "
                         f"a cache of {c.n_pages} pages of {c.page} rows, {c.n_heads} heads of {c.width}")
    b = _BatchS.from_buffer_copy(batch._s)
    b.mask, b.mask_words, b.n_tokens = None, 0, 0x7fffffff     # the starts tell how many
    rc = _fn("hearth_gpu_key_bounds")(cache._ref, byref(b), bounds._ref, dev, stream)
    if rc:
        _check(rc, "update_bounds")


def select_workspace_bytes(bounds: Bounds, batch: Batch, tokens: int | None = None) -> int:
    """Bytes of device workspace that select needs for `tokens` query tokens (None: as many as sequences
    times max_q)."""
    s = _for_tokens(batch, tokens)
    n = _fn("hearth_gpu_select_workspace")(bounds._ref, byref(s))
    if n < 0:
        raise ValueError(f"select: {s.max_q} tokens of {s.max_kv} rows are beyond its limits (see include/hearth_gpu.h)")
    return n


def select(bounds: Bounds, batch: Batch, q, chosen, *, first: int = 1, last: int = 1, workspace=None, stream=0) -> None:
    """The best blocks of each token for each cache head: chosen int32 [tokens, heads of the bounds, top],
    ascending, -1 behind the last. q [tokens, heads, width], float16 or bfloat16, heads a multiple of the
    bounds'. Every token keeps its `first` first blocks and its `last` last ones (its own among them; in a
    tree all that hold the call's rows); the others come by an upper bound of their rows' scores (include/
    hearth_gpu.h), the lower block first where two are equal. workspace: a device tensor of
    select_workspace_bytes; calls that may run at the same time must not share one."""
    dev, s = bounds.device, bounds._s
    if batch.device != dev:
        raise ValueError(f"select: the batch is on device {batch.device}, the bounds on device {dev}")
    a, tokens = _array(q, "q", dev), q.shape[0]
    if a.dtype == F32 or a.width != s.width or a.n_heads % s.n_heads:
        raise ValueError(f"select: q is {q.dtype}{tuple(q.shape)} over bounds of {s.n_heads} heads of width {s.width}")
    o = _blocks(chosen, "chosen", dev, tokens, s.n_heads, s.block)
    if first < 0 or last < 1 or first + last > o.top:
        raise ValueError(f"select: the first {first} and last {last} (at least one) of {o.top} blocks")
    wp, wb = None, 0
    if workspace is not None:
        _device(workspace, "workspace", dev)
        if not workspace.is_contiguous():
            raise ValueError("workspace: not dense")
        wp, wb = workspace.data_ptr(), workspace.numel() * workspace.element_size()
    rc = _fn("hearth_gpu_select_blocks")(bounds._ref, batch._of(tokens), byref(a), byref(o), first, last, wp, wb, dev, stream)
    if rc == -1 and (wp is None or wp % 16) and (need := select_workspace_bytes(bounds, batch, tokens)):
        raise ValueError(f"select: arguments that do not fit together, or a workspace of {need} bytes on 16 is needed")
    if rc:
        _check(rc, "select")


def attend_blocks_workspace_bytes(cache: Cache, batch: Batch, heads: int, top: int, block: int, tokens: int | None = None) -> int:
    """Bytes of device workspace that attend_blocks needs for `tokens` query tokens (None: as many as
    sequences times max_q) of `heads` heads and `top` chosen blocks of `block` rows: 0 when none is."""
    s = _for_tokens(batch, tokens)
    n = -1
    if 1 <= heads <= 65536 and 1 <= top <= 1 << 20 and 16 <= block <= 4096:
        n = _fn("hearth_gpu_attend_blocks_workspace")(cache._ref, byref(s), heads, top, block)
    if n < 0:
        raise ValueError(f"no attention over {top} blocks of {block} rows of this cache (pages of {cache._s.page} rows, heads {cache._s.n_heads}, "
                         f"width {cache._s.width}) with {heads} query heads")
    return n


def attend_blocks(cache: Cache, batch: Batch, q, chosen, out, *, block: int, scale: float, lse=None, workspace=None, stream=0) -> None:
    """attend over the rows of chosen blocks alone: chosen int32 [tokens, cache heads, top], numbers of
    blocks of `block` rows (a power of two from 16 up to a page) of the token's sequence, negative ones for none,
    in any order, each once (one that stands twice counts twice). A token attends those of their rows that it would
    attend without a choice (its own row at most, its mask). The rest as attend; workspace:
    attend_blocks_workspace_bytes."""
    if cache.v is None:
        raise ValueError("attend_blocks: a latent cache has no keys of its own")
    if chosen is None:
        raise ValueError("attend_blocks: chosen is missing")
    _attend("attend_blocks", cache, batch, q, None, out, lse, scale, workspace, stream, chosen, block)


def rope(x, pos, freqs, *, factor=1.0, layout="half", offset=0, out=None, k=None, k_out=None, inverse=False,
         stream=0) -> None:
    """Rotates x [tokens, heads, width] (float32, float16 or bfloat16) by pos [tokens] (int32 or
    int64): pair j of the part [offset, offset + 2 n) turns by pos * freqs[j] radians and is
    multiplied by factor. freqs: float64 [n] on the device (rope_frequencies). layout "half":
    pairs (j, j + n); "interleaved": (2j, 2j + 1). In place, or into out, which then gets the
    other elements too (out is x or shares nothing with it). k, k_out: a second array of the
    same width that shares nothing with the first, rotated in the same launch. inverse: by the
    negative angle."""
    if layout not in ("half", "interleaved"):
        raise ValueError(f"layout {layout!r} is neither 'half' nor 'interleaved'")
    dev = _device(x, "x")
    ao = ax = _array(x, "x", dev)
    tokens = x.shape[0]
    if out is not None and out is not x:
        ao = _array(out, "out", dev)
        if out.shape[0] != tokens or ao.n_heads != ax.n_heads or ao.width != ax.width or ao.dtype != ax.dtype:
            raise ValueError(f"out is {out.dtype}{tuple(out.shape)}, x {x.dtype}{tuple(x.shape)}")
    ak = ako = None
    if k is not None:
        ako = ak = _array(k, "k", dev)
        if k.shape[0] != tokens or ak.width != ax.width or ak.dtype != ax.dtype:
            raise ValueError(f"k is {k.dtype}{tuple(k.shape)}, x {x.dtype}{tuple(x.shape)}")
        if k_out is not None and k_out is not k:
            ako = _array(k_out, "k_out", dev)
            if k_out.shape[0] != tokens or ako.n_heads != ak.n_heads or ako.width != ak.width or ako.dtype != ak.dtype:
                raise ValueError(f"k_out is {k_out.dtype}{tuple(k_out.shape)}, k {k.dtype}{tuple(k.shape)}")
    elif k_out is not None:
        raise ValueError("k_out without k")
    p = _ints(pos, "pos", dev, 1, ("torch.int32", "torch.int64", "int32 or int64"))
    f = _ints(freqs, "freqs", dev, 1, ("torch.float64", "float64"))
    if getattr(freqs, "requires_grad", False):
        _refuse_gradient("freqs")
    n = freqs.shape[0]
    if pos.shape[0] != tokens or tokens > 0x7fffffff:
        raise ValueError(f"{pos.shape[0]} positions for {tokens} tokens")
    if max(ax.n_heads, ak.n_heads if ak is not None else 0) * ax.width > 1 << 24:
        raise ValueError("more than 2^24 elements a token")
    if ak is not None and tokens and (ak.data == ax.data or ako.data == ao.data):
        raise ValueError("k shares x's elements")
    if not 1 <= n <= 512 or offset < 0 or offset + 2 * n > ax.width:
        raise ValueError(f"{n} pairs at {offset} do not fit a width of {ax.width}")
    rc = _fn("hearth_gpu_rope")(byref(ax), byref(ao), byref(ak) if ak is not None else None,
                                byref(ako) if ako is not None else None, tokens, p, _seen_ints[pos.dtype] == "torch.int64",
                                f, n, offset, layout == "interleaved", bool(inverse), float(factor), dev, stream)
    if rc:
        _check(rc, "rope")


def rope_frequencies(rot: int, base: float = 10000.0, scaling: str | None = None, *, factor: float = 1.0,
                     original: int = 4096, beta_fast: float = 32.0, beta_slow: float = 1.0, low: float = 1.0,
                     high: float = 4.0) -> tuple[np.ndarray, float]:
    """Radians a position of the rot / 2 pairs (float64) and the factor on sine and cosine.

    scaling None: base^(-2j / rot). "linear": positions divided by `factor` (position
    interpolation, Chen et al. 2023). "ntk": the base grows by factor^(rot / (rot - 2)), so that
    the slowest pair is stretched by `factor` and the fastest not at all. "yarn" (Peng et al.
    2023): pairs that turn fewer than beta_slow times over `original` positions are
    interpolated, those above beta_fast kept, a linear ramp over the pair index between; sine
    and cosine grow by 0.1 ln(factor) + 1. "llama3": by wavelength, kept below original / high,
    divided by factor above original / low, blended between."""
    if rot < 2 or rot % 2:
        raise ValueError(f"{rot} rotated elements: an even number is needed")
    if not (base > 0 and factor > 0 and original > 0):
        raise ValueError("base, factor and original must be positive")
    j = np.arange(0, rot, 2, dtype=np.float64)
    f = float(base) ** -(j / rot)
    if scaling is None:
        return f, 1.0
    if scaling == "linear":
        return f / factor, 1.0
    if scaling == "ntk":
        if rot < 4:
            raise ValueError("ntk scaling needs at least two pairs")
        return (base * factor ** (rot / (rot - 2))) ** -(j / rot), 1.0
    if scaling == "yarn":
        def index(turns):   # the pair that turns this often over the original length
            return rot * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))
        lo, hi = max(math.floor(index(beta_fast)), 0), min(math.ceil(index(beta_slow)), rot - 1)
        ramp = np.clip((np.arange(rot // 2) - lo) / max(hi - lo, 0.001), 0.0, 1.0)
        return f / factor * ramp + f * (1 - ramp), (0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0)
    if scaling == "llama3":
        smooth = np.clip((original * f / (2 * math.pi) - low) / (high - low), 0.0, 1.0)
        return (1 - smooth) * f / factor + smooth * f, 1.0
    raise ValueError(f"scaling {scaling!r} is none of linear, ntk, yarn, llama3")
