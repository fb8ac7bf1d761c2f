"""Plain forms on the CPU of bounds of blocks, of the choice among them and of attention over the chosen
ones: whole numbers and float64."""
from __future__ import annotations

import math

import torch

import paged_oracle as O


def whole(x, dims):
    """float64 x -> whole numbers of up to 127 steps, exponent + 127 of the step (the least power of two, 2^-126 at
    least), one for all of `dims`"""
    x = torch.where(x.isfinite(), x, 0.0)
    top = x.abs().amax(dims, keepdim=True)
    m, e = torch.frexp(top)                          # top = m 2^e; top <= 127 * 2^(e - 7) where m <= 127 / 128
    byte = torch.where(top > 0, e + 127 - 7 + (m > 127 / 128), 1).clamp(min=1)
    return torch.round(torch.ldexp(x, 127 - byte)), byte


def bounds(K, exists, block):
    """K [heads, rows, width] float64, exists [rows]: codes [heads, blocks, 2, width], bytes [heads, blocks] (-1 where a
    block's rows do not exist)"""
    H, L, W = K.shape
    codes, byte, N = [], [], -(-L // block)
    for n in range(N):
        rows = torch.where(K[:, n * block:(n + 1) * block].isfinite(), K[:, n * block:(n + 1) * block], 0.0)
        c, b = whole(torch.stack([rows.amin(1), rows.amax(1)], 1), (1, 2))
        codes.append(c)
        byte.append(torch.where(exists[n * block], b[:, 0, 0], -1))
    if not N:
        return torch.zeros(H, 0, 2, W, dtype=torch.float64), torch.zeros(H, 0, dtype=torch.int64)
    return torch.stack(codes, 1), torch.stack(byte, 1)


def scores(codes, byte, q):
    """q [n, H, W] float64 against codes [Hkv, N, 2, W]: [n, Hkv, N]"""
    n, H, W = q.shape
    Hkv, N = byte.shape
    c, e = whole(q, (2,))
    c, e = c.view(n, Hkv, H // Hkv, W), e.view(n, Hkv, H // Hkv)
    s = torch.einsum("nhgw,hbw->nhgb", c.clamp(min=0), codes[:, :, 1]) + torch.einsum("nhgw,hbw->nhgb", c.clamp(max=0), codes[:, :, 0])
    return torch.ldexp(s, e.unsqueeze(-1) + byte[None, :, None] - 254).float().amax(2)


def choose(codes, byte, q, base, kv, block, top, first, last, tree=False):
    """[n, Hkv, top] int32 of tokens at rows base ..; kv: rows that exist for the call"""
    n, Hkv = q.shape[0], byte.shape[0]
    s = scores(codes, byte, q)
    out = torch.full((n, Hkv, top), -1, dtype=torch.int32)
    for t in range(n):
        own = min(base + t, kv - 1)
        if own < 0:
            continue
        N = own // block + 1
        tail = N - last
        if tree:
            tail = min(tail, max(base, 0) // block)
        for h in range(Hkv):
            can = [b for b in range(N) if byte[h, b] >= 0]
            rank = sorted(can, key=lambda b: (0 if b < first or b >= tail else 1, 0.0 if b < first or b >= tail else -s[t, h, b].item(), b))[:top]
            out[t, h, :len(rank)] = torch.tensor(sorted(rank), dtype=torch.int32)
    return out


def attention(q, K, V, exists, base, scale, kind, chosen, block, seen=None):
    """paged_oracle.attention over the rows of chosen [n, Hkv, top], token by token and head by head"""
    n, H, W = q.shape
    Hkv, L = K.shape[:2]
    G = H // Hkv
    outs = [torch.zeros(n, H, V.shape[2], dtype=torch.float64), torch.full((n, H), -math.inf, dtype=torch.float64),
            torch.zeros(n, H, V.shape[2], dtype=torch.float64), torch.zeros(n, H, dtype=torch.float64)]
    for t in range(n):
        for h in range(Hkv):
            rows = [r for b in chosen[t, h].tolist() if b >= 0 for r in range(b * block, min((b + 1) * block, L))]
            rows = torch.tensor(rows, dtype=torch.long)
            ok = exists[rows] & (rows <= base + t if seen is None else
                                 (rows < base) | torch.where((rows >= base) & (rows - base < n), seen[t][(rows - base).clamp(0, n - 1)], False))
            # every chosen row that it attends, as one token that attends all of them
            o = O.attention(q[t:t + 1, h * G:(h + 1) * G], K[h:h + 1, rows], V[h:h + 1, rows], ok, len(rows), scale, kind)
            for x, y in zip(outs, o):
                x[t, h * G:(h + 1) * G] = y[0]
    return outs
