"""Plain forms of 4-bit cache rows (mx4) on the CPU, for their tests: e2m1 codes, two a byte with the
even element in the low half, and a scale byte for each 32 elements."""
from __future__ import annotations

import torch

import paged_oracle as O

GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def mx4(x: torch.Tensor):
    """codes (uint8 [..., width / 2]) and scale bytes [..., width / 32] of rows of float16, bfloat16 or float32:
    the least power of two with amax <= 7 * it; a block with a NaN or an infinity has scale byte 255 and codes 0."""
    b = x.double().unflatten(-1, (-1, 32))
    fine = b.isfinite().all(-1)
    amax = torch.where(fine.unsqueeze(-1), b.abs(), 0.0).amax(-1)
    m, e = torch.frexp(amax)                        # amax = m 2^e, m in [0.5, 1): 7 = 0.875 * 2^3
    byte = torch.where(amax > 0, e + 127 - 3 + (m > 0.875), 1).clamp(min=1)
    s = torch.where(fine.unsqueeze(-1), torch.ldexp(b, (127 - byte).unsqueeze(-1)), 0.0)
    top = torch.where(byte == 127 + O.TOP[x.dtype] - 1, 3.0, 6.0).unsqueeze(-1)
    a = torch.minimum(s.abs(), top)
    # nearest, of two as near the one of even index: halfway points go up where the index above is even
    mid = (GRID[1:] + GRID[:-1]) / 2
    code = torch.zeros_like(a, dtype=torch.int64)
    for i, h in enumerate(mid):
        code += (a >= h) if i % 2 else (a > h)
    code = torch.where(fine.unsqueeze(-1), code + 8 * torch.signbit(s), 0).flatten(-2)
    return (code[..., 0::2] | code[..., 1::2] << 4).to(torch.uint8), torch.where(fine, byte, 255).to(torch.uint8)


def values(codes, scales):
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()
    x = torch.where(c >= 8, -1.0, 1.0) * GRID[c & 7]
    x = torch.ldexp(x.unflatten(-1, (-1, 32)), (scales.int() - 127).unsqueeze(-1))
    return torch.where((scales == 255).unsqueeze(-1), torch.nan, x).flatten(-2)


def rows_of(data, scales, pages, length):
    """paged_oracle.rows_of, of packed rows too"""
    if scales is None or data.element_size() != 1 or data.shape[-1] != 16 * scales.shape[-1]:
        return O.rows_of(data, scales, pages, length)
    P = data.shape[2]
    ids = pages[: -(-length // P)].long() if length else pages[:0].long()
    ok = (ids >= 0) & (ids < data.shape[0])
    safe = torch.where(ok, ids, 0)
    x = torch.where(ok[:, None, None, None], values(data.view(torch.uint8)[safe], scales[safe]), 0.0)
    return x.transpose(0, 1).flatten(1, 2)[:, :length], ok.repeat_interleave(P)[:length]


class Plain:
    """what test_gpu_paged takes from paged_oracle, with mx4 rows"""
    HALF, mx8, attention, words, tree, rope = O.HALF, staticmethod(O.mx8), staticmethod(O.attention), staticmethod(O.words), staticmethod(O.tree), staticmethod(O.rope)
    rows_of, values = staticmethod(rows_of), staticmethod(O.values)
