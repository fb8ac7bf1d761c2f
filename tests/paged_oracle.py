"""Plain float64 forms of the paged-cache operators, on the CPU, for their tests. A cache here
is the list of every sequence's rows, taken out of the pages by `rows_of`."""
from __future__ import annotations

import math

import numpy as np
import torch

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}   # half a step, relative
TOP = {torch.bfloat16: 127, torch.float16: 15, torch.float32: 127}                         # largest exponent


def mx8(x: torch.Tensor):
    """codes (float8_e4m3fn) and scale bytes of rows [..., width], block by block."""
    b = x.double().unflatten(-1, (-1, 32))
    amax = torch.where(b.isfinite(), b.abs(), 0.0).amax(-1)
    m, e = torch.frexp(amax)
    byte = torch.where(amax > 0, e - 1 + 127 - 8 + (m > 0.875), 1).clamp(min=1)
    s = torch.ldexp(b, (127 - byte).unsqueeze(-1))
    top = torch.where(byte == 127 + TOP[x.dtype] - 7, 240.0, 448.0).unsqueeze(-1)
    s = torch.minimum(torch.maximum(s, -top), top)
    codes = torch.where(b.isfinite(), s, math.nan).float().to(torch.float8_e4m3fn)
    codes = torch.where(b.isfinite(), codes.view(torch.uint8), 0x7f).to(torch.uint8)
    return codes.flatten(-2).view(torch.float8_e4m3fn), byte.to(torch.uint8)


def values(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    return torch.ldexp(codes.float().double().unflatten(-1, (-1, 32)), (scales.int() - 127).unsqueeze(-1)).flatten(-2)


def rows_of(data, scales, pages, length):
    """[heads, length, width] float64 of one sequence (rows of bad pages: zeros) and which rows exist."""
    P = data.shape[2]
    ids = pages[: -(-length // P)].long() if length else pages[:0].long()
    ok = (ids >= 0) & (ids < data.shape[0])
    safe = torch.where(ok, ids, 0)
    x = values(data.view(torch.uint8)[safe].view(torch.float8_e4m3fn), scales[safe]) if scales is not None else data[safe].double()
    x = torch.where(ok[:, None, None, None], x, 0.0)
    return x.transpose(0, 1).flatten(1, 2)[:, :length], ok.repeat_interleave(P)[:length]


def attention(q, K, V, exists, base, scale, kind, seen=None):
    """q [n, H, W] float64; K, V [Hkv, len, .]; token i attends rows < base + i + 1 that exist,
    or with `seen` [n, n] rows < base and the new rows seen[i]. Returns out [n, H, DV], lse, and
    the bound on a kernel's error: scores in float32, probabilities rounded to `kind`, sums in
    float32, one rounding of the result."""
    n, H, W = q.shape
    G, L = H // K.shape[0], K.shape[1]
    t = torch.arange(L)
    vis = torch.zeros(n, L, dtype=torch.bool)
    for i in range(n):
        vis[i] = t < (base + i + 1 if seen is None else base)
        if seen is not None:
            j = t - base
            inside = (j >= 0) & (j < n)
            vis[i] |= torch.where(inside, seen[i][j.clamp(0, n - 1)], False)
    vis &= exists[None]
    Kh, Vh = K.repeat_interleave(G, 0), V.repeat_interleave(G, 0)
    s = torch.einsum("nhw,hlw->hnl", q, Kh) * scale
    sabs = torch.einsum("nhw,hlw->hnl", q.abs(), Kh.abs()) * abs(scale)
    s = torch.where(vis[None], s, -math.inf)
    m = s.amax(-1, keepdim=True) if L else torch.full((H, n, 1), -math.inf, dtype=torch.float64)
    p = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
    p = torch.where(vis[None], p, 0.0)
    tot = p.sum(-1, keepdim=True)
    Vz = torch.where(vis[None, :, :, None], Vh[:, None], 0.0) if not torch.isfinite(Vh).all() else None
    mul = (lambda w, x: torch.einsum("hnl,hlv->hnv", w, x)) if Vz is None else (lambda w, x: torch.einsum("hnl,hnlv->hnv", w, x))
    vv = Vh if Vz is None else Vz
    o = mul(p, vv) / torch.where(tot == 0, 1.0, tot)
    h = HALF[kind]
    A = mul(p, vv.abs()) / torch.where(tot == 0, 1.0, tot)
    # a score of W products summed in float32 in any order, scaled: off by (W + 2) 2^-24 of the
    # sum of magnitudes; numerator and denominator both carry it. Sums of up to L terms over
    # 32-row steps and splits, powers of two to 2^-22: (L + 64) 2^-23 covers them.
    sb = torch.where(vis[None], sabs, 0.0).amax(-1, keepdim=True) if L else torch.zeros(H, n, 1, dtype=torch.float64)
    rel = 2 * (W + 8) * 2.0 ** -24 * sb + (L + 64) * 2.0 ** -23
    tol = h * o.abs() + A * (h + rel) * 1.02 + 1e-30
    if kind == torch.float16:      # probabilities and results below its normal range round to steps of 2^-24
        tol = tol + 2.0 ** -25 * (1 + mul(vis[None].double().expand(H, -1, -1), vv.abs()))
    lse = torch.where(tot == 0, -math.inf, m + torch.log(torch.where(tot == 0, 1.0, tot)))[..., 0]
    lse_tol = (W + 8) * 2.0 ** -24 * sb[..., 0] + (L + 64) * 2.0 ** -23 + 2.0 ** -21 * (1 + lse.abs())
    return o.transpose(0, 1), lse.T, tol.transpose(0, 1), lse_tol.T


def rope(x, pos, freqs, factor, layout, offset, inverse=False):
    """x float64 [T, H, W]"""
    n = len(freqs)
    a = pos.double()[:, None] * freqs.double() * (-1 if inverse else 1)
    c, s = (torch.cos(a) * factor)[:, None], (torch.sin(a) * factor)[:, None]
    y = x.clone()
    part = x[..., offset:offset + 2 * n]
    u, v = (part[..., :n], part[..., n:]) if layout == "half" else (part[..., 0::2], part[..., 1::2])
    a0, a1 = u * c - v * s, v * c + u * s
    y[..., offset:offset + 2 * n] = torch.cat([a0, a1], -1) if layout == "half" else torch.stack([a0, a1], -1).flatten(-2)
    mag = torch.zeros_like(x)
    w = u.abs() + v.abs()
    mag[..., offset:offset + 2 * n] = torch.cat([w, w], -1) if layout == "half" else torch.stack([w, w], -1).flatten(-2)
    return y, mag * abs(factor)


def tree(n, fan=4):
    par = [-1] + [(i - 1) // fan for i in range(1, n)]
    seen = torch.zeros(n, n, dtype=torch.bool)
    for i in range(n):
        if par[i] >= 0:
            seen[i] = seen[par[i]]
        seen[i, i] = True
    return seen


def words(seen_list, width):
    """int64 mask words [tokens, ceil(width / 64)]"""
    w = -(-max(width, 1) // 64)
    out = []
    for seen in seen_list:
        bits = np.zeros((seen.shape[0], w * 64), dtype=bool)
        bits[:, : seen.shape[1]] = seen.numpy()
        out.append(np.packbits(bits.reshape(seen.shape[0], w, 64), axis=-1, bitorder="little").view(np.int64).reshape(-1, w))
    return torch.from_numpy(np.concatenate(out).copy())
