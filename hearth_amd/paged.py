"""Operators over paged key-value caches on the GPU (the paged section of include/hearth_gpu.h).

For programs that keep many conversations' rows in pages next to (or without) an Engine:

    rope(x, pos, freqs)              rotary positions, in place or into `out`
    append(cache, batch, k, v)       new tokens' rows into the pages, 16-bit or 8-bit ("mx8")
    read(cache, batch, k, v)         rows back out of the pages
    attend(cache, batch, q, out)     grouped-head attention: tokens, chains, draft trees, prompts
    attend_latent(...)               absorbed latent attention over one row a token

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

__all__ = ["Cache", "Batch", "rope", "rope_frequencies", "append", "read", "attend", "attend_latent",
           "workspace_bytes"]

F32, F16, BF16, MX8 = 0, 1, 2, 16
_DTYPES = {"float32": F32, "float16": F16, "bfloat16": BF16, "float8_e4m3fn": MX8}


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


_PROTOS = {
    "hearth_gpu_rope": (c_int, [POINTER(_Array), POINTER(_Array), POINTER(_Array), POINTER(_Array), c_int, c_void_p,
                                c_int, c_void_p, c_int, c_int, c_int, c_int, c_double, c_int, c_void_p]),
    "hearth_gpu_kv_append": (c_int, [POINTER(_CacheS), POINTER(_BatchS), POINTER(_Array), POINTER(_Array), c_int,
                                     c_void_p]),
    "hearth_gpu_kv_read": (c_int, [POINTER(_CacheS), POINTER(_BatchS), POINTER(_Array), POINTER(_Array), c_int,
                                   c_void_p]),
    "hearth_gpu_attend": (c_int, [POINTER(_CacheS), POINTER(_BatchS), POINTER(_Array), POINTER(_Array), c_void_p,
                                  c_float, c_void_p, c_size_t, c_int, c_void_p]),
    "hearth_gpu_attend_latent": (c_int, [POINTER(_CacheS), POINTER(_BatchS), POINTER(_Array), POINTER(_Array),
                                         POINTER(_Array), c_void_p, c_float, c_void_p, c_size_t, c_int, c_void_p]),
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
            raise ValueError(f"dtype {d} is none of float32, float16, bfloat16 (float8_e4m3fn in a cache)")
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
    if dt == MX8:
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
    """Rows of all sequences: k and v [pages, heads, rows a page, width], float16, bfloat16 or
    float8_e4m3fn with scales (uint8 E8M0, [pages, heads, rows a page, width / 32]); v None:
    latent rows (latent vector, then its rotated part). The last two dimensions are dense; the
    tensors are the caller's and stay referenced."""

    def __init__(self, k, v=None, k_scale=None, v_scale=None):
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.device = _device(k, "k")
        dt = _dtype(k)
        if dt == F32:
            raise ValueError("cache rows are float16, bfloat16 or float8_e4m3fn")
        s = _CacheS()
        if len(k.shape) != 4:
            raise ValueError(f"k: shape {tuple(k.shape)} is not [pages, heads, rows a page, width]")
        s.dtype, (s.n_pages, s.n_heads, s.page, s.width) = dt, k.shape
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
        if (scale is not None) != (dt == MX8):
            raise ValueError(f"{what}: scales go with float8_e4m3fn rows, and only with them")
        if scale is not None:
            want = (*t.shape[:3], t.shape[3] // 32)
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


def read(cache: Cache, batch: Batch, k, v=None, *, stream=0) -> None:
    """The inverse of append: fills k, v [tokens, heads, width] with the call's tokens' rows
    (zeros for rows that are not in the cache). q_start = running sum of kv_len reads whole
    sequences."""
    a, b, bs = _pair(cache, batch, k, v, "read")
    rc = _fn("hearth_gpu_kv_read")(cache._ref, bs, byref(a), byref(b) if b is not None else None, cache.device, stream)
    if rc:
        _check(rc, "read")


def workspace_bytes(cache: Cache, batch: Batch, heads: int, tokens: int | None = None) -> int:
    """Bytes of device workspace that attend / attend_latent need for `tokens` query tokens
    (None: as many as sequences times max_q) of `heads` heads: 0 when none is."""
    s = _BatchS.from_buffer_copy(batch._s)
    s.n_tokens = min(s.n_seqs * s.max_q, 0x7fffffff) if tokens is None else tokens
    n = _fn("hearth_gpu_attend_workspace")(cache._ref, byref(s), heads)
    if n < 0:
        raise ValueError(f"no attention over this cache (heads {cache._s.n_heads}, width {cache._s.width}) "
                         f"with {heads} query heads")
    return n


def _attend(name, cache, batch, q, q_pe, out, lse, scale, workspace, stream):
    dev = cache.device
    if batch.device != dev:
        raise ValueError(f"{name}: the batch is on device {batch.device}, the cache on device {dev}")
    cache._no_gradient()
    a, o, tokens = _array(q, "q", dev), _array(out, "out", dev), q.shape[0]
    if out.shape[0] != tokens or o.n_heads != a.n_heads or o.width != a.width or a.dtype != o.dtype:
        raise ValueError(f"{name}: out is {out.dtype}{tuple(out.shape)}, q {q.dtype}{tuple(q.shape)}")
    if a.dtype == F32 or cache._s.dtype not in (MX8, a.dtype):
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
    if q_pe is None:
        rc = _fn("hearth_gpu_attend")(cache._ref, bs, byref(a), byref(o), lp, float(scale), wp, wb, dev, stream)
    else:
        pe = _array(q_pe, "q_pe", dev)
        if q_pe.shape[0] != tokens or pe.n_heads != a.n_heads or pe.dtype != a.dtype:
            raise ValueError(f"{name}: q_pe is {q_pe.dtype}{tuple(q_pe.shape)}, q {q.dtype}{tuple(q.shape)}")
        rc = _fn("hearth_gpu_attend_latent")(cache._ref, bs, byref(a), byref(pe), byref(o), lp, float(scale), wp, wb, dev, stream)
    if rc == -1 and (wp is None or wp % 16) and (need := workspace_bytes(cache, batch, a.n_heads, tokens)):
        raise ValueError(f"{name}: a workspace of {need} bytes on 16 is needed")
    if rc:
        _check(rc, name)


def attend(cache: Cache, batch: Batch, q, out, *, scale: float, lse=None, workspace=None, stream=0) -> None:
    """out = softmax(scale * q k) v of the call's tokens over the rows each attends; q, out
    [tokens, heads, width] of the cache's 16-bit dtype (any over mx8 rows), heads a multiple of
    the cache's. lse: float32 [tokens, heads] or None. workspace: a device tensor of
    workspace_bytes; calls that may run at the same time must not share one. A token that
    attends nothing gets zeros, one all of whose scores are -inf gets NaN (lse -inf for both)."""
    _attend("attend", cache, batch, q, None, out, lse, scale, workspace, stream)


def attend_latent(cache: Cache, batch: Batch, q, q_pe, out, *, scale: float, lse=None, workspace=None,
                  stream=0) -> None:
    """Absorbed latent attention: q [tokens, heads, 512] and q_pe [tokens, heads, 64] over a
    latent cache of width 576, out [tokens, heads, 512]; the rest as attend."""
    if q_pe is None:
        raise ValueError("attend_latent: q_pe is missing")
    _attend("attend_latent", cache, batch, q, q_pe, out, lse, scale, workspace, stream)


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
