"""Long contexts over paged caches (hearth_amd/paged.py) as measurable cases.

Operators, in the order in which a serving program's layer calls them: `rotate` (rotary
positions applied to queries, and to keys on their way into the pages), `store4` (rows
into a cache held in 4 bits and back), `attend4` (grouped-head attention over such a cache),
`select` (bounds of the keys of each block of rows brought up to date, and the blocks that each
query is to look at) and `sparse` (attention over the chosen blocks alone).

4-bit rows ("mx4") hold e2m1 codes, two a byte (the even element in the low half), with one
power-of-two scale byte (exponent + 127) for each 32 elements; "mx8" rows e4m3 codes with scales
alike. Pages hold PAGE rows of one head side by side. Bounds hold, for each block of BLOCK rows
and head, the least and the greatest value of every key element as whole numbers of up to 127
steps, the step a power of two for the block: int8 [pages, heads, blocks a page, 2, width] and
scale bytes [pages, heads, blocks a page].

A sequence's new tokens are the last n of its rows; lengths follow from the case, pages are
dealt out in a shuffled order. Where `own` is false the operators run in elementary torch
operations.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

PAGE = BLOCK = 64
FIRST, LAST = 1, 2                                  # blocks that every query keeps: the first, its own and the one before
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
QWEN = dict(heads=32, kv_heads=4, dim=128)          # Qwen3-30B-A3B


def _case(name, op, seqs, ctx, n, type, store, heads=32, kv_heads=4, dim=128, **kw):
    c = dict(op=op, seqs=seqs, ctx=ctx, n=n, heads=heads, kv_heads=kv_heads, dim=dim, type=type, store=store, **kw)
    return dict(name=name, **c) if name else c


def listed():
    return [
        # one verify step of nine tokens in one chat: the shortest call there is
        _case("rotate_step", "rotate", 1, 4104, 9, "bf16", "bf16", **QWEN, layout="half", scaling="none", rot=128),
        # three prompts of odd lengths, positions stretched
        _case("rotate_prompt", "rotate", 3, 4093, 4093, "f16", "f16", **QWEN, layout="half", scaling="yarn", rot=128),
        # the new rows of 32 conversations' next tokens into 4-bit pages, and looked at again
        _case("store4_step", "store4", 32, 4096, 1, "bf16", "mx4"),
        # three prompts of odd lengths into 4-bit pages, and a snapshot of them
        _case("store4_prompt", "store4", 3, 4093, 4093, "bf16", "mx4"),
        # the next tokens of 32 conversations of uneven lengths
        _case("decode4_32", "attend4", 32, 8192, 1, "bf16", "mx4"),
        # one token at the end of a very long document
        _case("decode4_long", "attend4", 1, 131071, 1, "f16", "mx4"),
        # a piece of a prompt behind 4000 rows
        _case("prompt4_1000", "attend4", 1, 5000, 1000, "bf16", "mx4"),
        # which blocks of a very long document its next token looks at
        _case("select_1_long", "select", 1, 131071, 1, "bf16", "bf16", top=32),
        # the same for each token of a piece of a long prompt
        _case("select_prompt", "select", 1, 20000, 600, "f16", "f16", top=16),
        # 32 long conversations' next tokens, each over 2048 of its rows
        _case("sparse_decode_32", "sparse", 32, 32768, 1, "bf16", "bf16", top=32),
        # one token of a very long document in 4 bits, over 4096 rows
        _case("sparse4_1_long", "sparse", 1, 131071, 1, "f16", "mx4", top=64),
        # a piece of a long prompt in 8 bits, each token over 1024 rows
        _case("sparse_prompt", "sparse", 1, 20000, 600, "bf16", "mx8", top=16),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotate", "store4", "attend4", "attend4", "select", "sparse", "sparse"])
    type = rng.choice(["bf16", "bf16", "f16"])
    kv_heads = rng.choice([1, 2, 4, 8])
    dim = rng.choice([64, 128, 128, 256])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 7, 8, 16])
    if op == "rotate":
        seqs, ctx = _log(rng, 1, 64), _log(rng, 1, 4096)
        n = min(rng.choice([1, min(ctx, rng.randint(2, 16)), ctx]), max(1, 12279 * 40 * 128 // (seqs * (heads + 2 * kv_heads) * dim)))
        return _case(None, op, seqs, ctx, n, type, rng.choice([type, type, "mx8"]), heads, kv_heads, dim, layout=rng.choice(["half", "interleaved"]),
                     scaling=rng.choice(["none", "linear", "yarn"]), rot=rng.choice([d for d in (32, 64, 96, 128, 256) if d <= dim]))
    if op == "store4":
        seqs, ctx = _log(rng, 1, 64), _log(rng, 1, 4096)
        n = min(rng.choice([1, min(ctx, rng.randint(2, 16)), ctx]), max(1, 12279 * 4 * 128 // (seqs * kv_heads * dim)))
        return _case(None, op, seqs, ctx, n, type, "mx4", heads, kv_heads, dim)
    kind = rng.choice(["one", "few", "many"])
    n = 1 if kind == "one" else rng.randint(2, 16) if kind == "few" else _log(rng, 100, 600 * 128 // max(dim, 128))
    seqs = _log(rng, 1, 64) if n == 1 else _log(rng, 1, 8) if n <= 16 else 1
    if op == "attend4":
        top = 131071 if n == 1 else 16384 if n <= 16 else 4096
        top = min(top, 2 ** 26 // (seqs * kv_heads * dim))              # rows: at most the listed cases' bytes
        return _case(None, op, seqs, n + _log(rng, 1, max(2, top)), n, type, "mx4", heads if n <= 16 else min(heads, 32) // kv_heads * kv_heads or kv_heads,
                     kv_heads, dim)
    top = min(131071, 2 ** 28 // (seqs * kv_heads * dim)) if n <= 16 else 20000
    if n > 16:
        kv_heads, heads, dim = 4, rng.choice([4, 8, 12, 28, 32]), rng.choice([64, 128])
    return _case(None, op, seqs, n + _log(rng, 1, top), n, type, rng.choice([type, "mx8", "mx4"]), heads, kv_heads, dim,
                 top=rng.choice([8, 13, 16] if n > 16 else [8, 16, 29, 32]))


# ---------------------------------------------------------------- lengths and work

def _lens(case):
    """Rows of each sequence, its new tokens included: the first the longest."""
    c, n, S = case["ctx"], min(case["n"], case["ctx"]), case["seqs"]
    if n == c:
        n = 1                                       # whole prompts: lengths as uneven as contexts
    return [c - (s * 7919) % (max(1, (c - n) * 3 // 4 + 1)) for s in range(S)]


def _news(case):
    return [min(case["n"], L) for L in _lens(case)]


def _blocks(rows):
    return -(-rows // BLOCK)


def _pool(case):
    """Blocks among which the tokens of a sequence choose: neighbours look at much the same ones."""
    return 3 * case["top"]


def _row_bytes(store, width):
    return {"mx4": width // 2 + width // 32, "mx8": width + width // 32, "f32": 4 * width}.get(store, 2 * width)


def work(case):
    op, H, G, D = case["op"], case["kv_heads"], case["heads"], case["dim"]
    lens, news = _lens(case), _news(case)
    es = TYPES[case["type"]].itemsize
    row = _row_bytes(case["store"], D)
    if op == "rotate":
        return {"bytes": sum(news) * (2 * G * D * es + 2 * H * (D * es + row)), "flops": 3 * sum(news) * (G + H) * case["rot"]}
    if op == "store4":
        return {"bytes": 2 * sum(news) * H * (2 * D * es + row), "flops": 4 * sum(news) * H * D}
    if op == "attend4":
        pairs = sum((L - n) * n + n * (n + 1) // 2 for L, n in zip(lens, news)) * G
        return {"bytes": 2 * sum(lens) * H * row + 2 * sum(news) * G * D * es, "flops": 4 * D * pairs}
    if op == "select":
        new = sum(_blocks(L) - (L - n) // BLOCK for L, n in zip(lens, news))
        pairs = sum(sum(_blocks(L - n + i + 1) for i in range(n)) for L, n in zip(lens, news)) * G
        return {"bytes": sum(map(_blocks, lens)) * H * (2 * D + 1) + new * BLOCK * H * row + sum(news) * (G * D * es + 4 * H * case["top"]),
                "flops": 4 * D * pairs}
    rows = sum(min(_blocks(L), min(n * case["top"], _pool(case) + LAST + n // BLOCK)) for L, n in zip(lens, news)) * BLOCK
    seen = sum(sum(min(case["top"], _blocks(L - n + i + 1)) for i in range(n)) for L, n in zip(lens, news)) * BLOCK
    return {"bytes": 2 * rows * H * row + sum(news) * (2 * G * D * es + 4 * H * case["top"]), "flops": 4 * D * seen * G}


# ---------------------------------------------------------------- codes

def _halves(codes):
    """Two 4-bit codes a byte, in order."""
    return torch.stack([codes & 15, codes >> 4], -1).flatten(-2)


def _table(device="cuda"):
    t = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=device)
    return torch.cat([t, -t])


def _quantise(x, store):
    """Rows [..., width] -> codes (mx4: uint8, two a byte; mx8: float8_e4m3fn), scale bytes [..., width / 32].
    The scale is the least power of two that brings the block's largest magnitude within half a step
    of the largest code (mx4: 7 = 6 + 1; mx8: at most 448); codes round to nearest even."""
    b = x.float().unflatten(-1, (-1, 32))
    amax = b.abs().amax(-1)
    m, e = torch.frexp(amax)                        # amax = m 2^e, m in [0.5, 1); both largest magnitudes are 0.875 2^k
    e = torch.where(m > 0.875, e, e - 1) - (2 if store == "mx4" else 8)
    e = torch.where(amax > 0, e, -126).clamp(-126, 120).int()
    q = torch.ldexp(b, -e.unsqueeze(-1))
    scales = (e + 127).to(torch.uint8)
    if store == "mx8":
        return q.to(torch.float8_e4m3fn).flatten(-2), scales
    a = q.abs()
    code = (a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0) + 8 * (q < 0).to(torch.uint8)
    code = code.flatten(-2)
    return code[..., 0::2] | code[..., 1::2] << 4, scales


def _values(codes, scales, table):
    """codes and scale bytes -> float32 (16-bit rows, whose scales are None, as they are)"""
    if scales is None:
        return codes.float()
    x = table[_halves(codes).int()] if codes.dtype == torch.uint8 else codes.float()
    return torch.ldexp(x.unflatten(-1, (-1, 32)), scales.unsqueeze(-1).int() - 127).flatten(-2)


def _raw(codes):
    return codes.view(torch.uint8) if codes.dtype == torch.float8_e4m3fn else codes


# ---------------------------------------------------------------- inputs

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 1000003 + 29)
    return g


def _rows(g, type, *shape):
    """Normal rows with a few strong channels, as keys have."""
    x = torch.randn(*shape, generator=g, device="cuda")
    x[..., 3::37] *= 4.0
    return x.to(TYPES[type])


def _frequencies(case):
    """Radians a position for each pair, float64, and the factor on cos and sin."""
    R, base = case["rot"], 1e6
    f, factor = base ** -(np.arange(0, R, 2, dtype=np.float64) / R), 1.0
    if case["scaling"] == "linear":
        f = f / 8.0
    elif case["scaling"] == "yarn":
        turns = lambda r: R * math.log(4096 / (r * 2 * math.pi)) / (2 * math.log(base))
        lo, hi = max(math.floor(turns(32.0)), 0), min(math.ceil(turns(1.0)), R - 1)
        ramp = np.clip((np.arange(R // 2) - lo) / max(hi - lo, 0.001), 0, 1)
        f = f / 40.0 * ramp + f * (1 - ramp)
        factor = 0.1 * math.log(40.0) + 1
    return torch.tensor(f, device="cuda"), factor


def _key_bounds(x):
    """Rows [..., rows, width] float32 -> codes int8 [..., 2, width], scale bytes [...]: of the least and
    greatest value of each element, the step the least power of two with which 127 steps reach the
    largest magnitude."""
    lo, hi = x.amin(-2), x.amax(-2)
    amax = torch.maximum(lo.abs(), hi.abs()).amax(-1)
    m, e = torch.frexp(amax)                        # amax <= 127 * 2^(e - 7) where m <= 127 / 128
    e = torch.where(m > 127 / 128, e - 6, e - 7)
    e = torch.where(amax > 0, e, -126).clamp(-126, 127)
    codes = torch.round(torch.ldexp(torch.stack([lo, hi], -2), -e[..., None, None]))
    return codes.to(torch.int8), (e + 127).to(torch.uint8)


def _pages_of(lens, seed):
    """Pages dealt out in a shuffled order: table [S, most], pages in all"""
    used = [-(-L // PAGE) for L in lens]
    order = torch.randperm(sum(used) + 1, generator=torch.Generator().manual_seed(seed + 5)).int()
    pages = torch.zeros(len(lens), max(used), dtype=torch.int32)
    at = 0
    for s, u in enumerate(used):
        pages[s, :u] = order[at:at + u]
        at += u
    return pages, len(order)


def _choose(case, st, g):
    """[tokens, kv heads, top] ascending: the first block, a token's own and the one before, and the
    best of a pool of blocks that the sequence's tokens share."""
    H, top, N = case["kv_heads"], case["top"], st["pages"].shape[1]
    S = case["seqs"]
    pool = torch.rand(S, H, N, generator=g, device="cuda")
    pool = torch.where(pool >= pool.topk(min(_pool(case), N), -1).values[..., -1:], 4.0, 0.0) + torch.rand(S, H, N, generator=g, device="cuda")
    score = pool[st["seq"]] + torch.rand(len(st["seq"]), H, N, generator=g, device="cuda")
    b, own_block = torch.arange(N, device="cuda"), st["pos"][:, None, None] // BLOCK
    score = torch.where((b < FIRST) | (b > own_block - LAST), 9.0, score).masked_fill_(b > own_block, -1.0)
    best = score.topk(min(top, N), -1)
    chosen = torch.where(best.values < 0, N, best.indices).sort(-1).values
    chosen = torch.where(chosen == N, -1, chosen).int()
    return torch.nn.functional.pad(chosen, (0, top - chosen.shape[-1]), value=-1)


def prepare(case, seed):
    g, dt, op = _gen(seed), TYPES[case["type"]], case["op"]
    lens, news = _lens(case), _news(case)
    S, total, H, D = len(lens), sum(news), case["kv_heads"], case["dim"]
    pages, n_pages = _pages_of(lens, seed)
    starts = np.concatenate([[0], np.cumsum(news)])
    pos = np.concatenate([np.arange(L - n, L) for L, n in zip(lens, news)])
    seq = np.repeat(np.arange(S), news)
    dev = lambda x, t: torch.as_tensor(x, dtype=t).cuda()
    st = dict(case=case, table=_table(), pages=pages.cuda(), kv_len=dev(lens, torch.int32), q_start=dev(starts, torch.int32),
              pos=dev(pos, torch.int64), seq=dev(seq, torch.int64))
    # where every new token's row lies; its place among tokens laid out [sequences, most new tokens]
    st["page_of"], st["row_of"] = dev(pages.numpy()[seq, pos // PAGE], torch.int64), dev(pos % PAGE, torch.int64)
    st["most"] = max(news)
    st["flat"] = dev(seq * max(news) + np.arange(total) - starts[seq], torch.int64)
    filled, only_k = op in ("attend4", "select", "sparse"), op == "select"
    for name in ("k",) if only_k else ("k", "v"):
        if filled:
            rows = _rows(g, case["type"], n_pages, H, PAGE, D)
            st[name + "c"], st[name + "s"] = _quantise(rows, case["store"]) if case["store"] in ("mx4", "mx8") else (rows, None)
        else:
            mx = case["store"] in ("mx4", "mx8")
            c = torch.zeros(n_pages, H, PAGE, D // 2 if case["store"] == "mx4" else D, dtype=torch.uint8 if mx else dt, device="cuda")
            st[name + "c"] = c.view(torch.float8_e4m3fn) if case["store"] == "mx8" else c
            st[name + "s"] = torch.zeros(n_pages, H, PAGE, D // 32, dtype=torch.uint8, device="cuda") if mx else None
            st[name] = _rows(g, case["type"], total, H, D)
            st[name + "_back"] = torch.zeros_like(st[name])
    if op != "store4":
        st["q"] = _rows(g, case["type"], total, case["heads"], D)
    if op == "rotate":
        st["freqs"], st["factor"] = _frequencies(case)
        st["out"] = torch.zeros_like(st["q"])
    elif op == "select":
        st["low_high"], st["steps"] = _key_bounds(_values(st["kc"], st["ks"], st["table"]).unflatten(2, (-1, BLOCK)))
        st["chosen"] = torch.full((total, H, case["top"]), -2, dtype=torch.int32, device="cuda")
    elif op in ("attend4", "sparse"):
        st["out"] = torch.zeros_like(st["q"])
        if op == "sparse":
            st["chosen"] = _choose(case, st, g)
    if own:
        from hearth_amd import paged
        packed = lambda c: c.view(torch.float4_e2m1fn_x2) if case["store"] == "mx4" else c
        v, vs = (st["vc"], st["vs"]) if not only_k else (st["kc"], st["ks"])       # the keys alone are read
        st["cache"] = paged.Cache(packed(st["kc"]), packed(v), st["ks"], vs)
        st["batch"] = paged.Batch(st["pages"], st["kv_len"], st["q_start"], max_q=max(news), max_kv=max(lens))
        if op == "attend4":
            need = paged.workspace_bytes(st["cache"], st["batch"], case["heads"], total)
        elif op == "sparse":
            need = paged.attend_blocks_workspace_bytes(st["cache"], st["batch"], case["heads"], case["top"], BLOCK, total)
        elif op == "select":
            st["bounds"] = paged.Bounds(st["low_high"], st["steps"], block=BLOCK)
            need = paged.select_workspace_bytes(st["bounds"], st["batch"], total)
        else:
            need = 0
        st["work"] = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
    return st


# ---------------------------------------------------------------- the plain forms

def _put(st, name, x):
    """Rows x of the new tokens into the cache."""
    if st[name + "s"] is None:
        st[name + "c"][st["page_of"], :, st["row_of"]] = x
        return
    codes, scales = _quantise(x, st["case"]["store"])
    _raw(st[name + "c"])[st["page_of"], :, st["row_of"]] = _raw(codes)
    st[name + "s"][st["page_of"], :, st["row_of"]] = scales


def _back(st, name):
    """The new tokens' rows as they stand in the cache."""
    codes = _raw(st[name + "c"])[st["page_of"], :, st["row_of"]].view(st[name + "c"].dtype)
    scales = st[name + "s"]
    return _values(codes, None if scales is None else scales[st["page_of"], :, st["row_of"]], st["table"]).to(TYPES[st["case"]["type"]])


def _rotated(st, x):
    case = st["case"]
    a = st["pos"].double()[:, None] * st["freqs"][None]
    cos, sin = ((torch.cos(a) * st["factor"]).float()[:, None], (torch.sin(a) * st["factor"]).float()[:, None])
    y, R = x.float(), case["rot"]
    half = R // 2
    u, v = (y[..., :half], y[..., half:R]) if case["layout"] == "half" else (y[..., 0:R:2], y[..., 1:R:2])
    r = (u * cos - v * sin, v * cos + u * sin)
    r = torch.cat(r, -1) if case["layout"] == "half" else torch.stack(r, -1).flatten(-2)
    return torch.cat([r, y[..., R:]], -1).to(x.dtype)


def _plain_rotate(st):
    _put(st, "k", _rotated(st, st["k"]))
    _put(st, "v", st["v"])
    if st["ks"] is None:
        return {"q": _rotated(st, st["q"]), "k": st["kc"], "v": st["vc"]}
    return {"q": _rotated(st, st["q"]), "k": _back(st, "k"), "v": _back(st, "v")}


def _plain_store(st):
    _put(st, "k", st["k"])
    _put(st, "v", st["v"])
    return {"k": _back(st, "k"), "v": _back(st, "v")}


def _padded(st, x):
    """[tokens, ...] -> [sequences, most new tokens, ...]"""
    y = torch.zeros(st["case"]["seqs"] * st["most"], *x.shape[1:], dtype=x.dtype, device="cuda")
    y[st["flat"]] = x
    return y.unflatten(0, (-1, st["most"]))


def _softmax_times(s, seen, V):
    """softmax of scores [..., columns, rows] over the rows seen, times V [..., rows, width]"""
    s = s.masked_fill_(~seen, -math.inf)
    p = torch.exp_(s - s.amax(-1, keepdim=True))
    return (p.flatten(0, -3) @ V.flatten(0, -3)).view(*p.shape[:-1], -1) / p.sum(-1, keepdim=True)


def _plain_attend(st):
    case, G = st["case"], st["case"]["heads"] // st["case"]["kv_heads"]
    used = st["pages"].long()
    rows = lambda name: _values(_raw(st[name + "c"])[used], st[name + "s"][used], st["table"]).transpose(1, 2).flatten(2, 3).contiguous()   # [S, H, L, D]
    K, V = rows("k"), rows("v")
    pos = _padded(st, st["pos"] + 1) - 1                                  # -1: no token
    q = _padded(st, st["q"].float()).unflatten(2, (-1, G)).permute(0, 2, 3, 1, 4).flatten(2, 3).contiguous()        # [S, H, G n, D]
    s = (q.flatten(0, 1) @ K.flatten(0, 1).transpose(1, 2)).view(*q.shape[:3], -1) * case["dim"] ** -0.5
    seen = (torch.arange(K.shape[2], device="cuda") <= pos.clamp(min=0)[..., None]).repeat(1, G, 1)[:, None]
    o = _softmax_times(s, seen, V).unflatten(2, (G, -1)).permute(0, 3, 1, 2, 4)                                     # [S, n, H, G, D]
    return o.flatten(0, 1)[st["flat"]].flatten(1, 2).to(TYPES[case["type"]])


def _score_keys(low_high, steps, q):
    """q [S, H, C, W] and the bounds of each sequence's blocks [S, H, N, 2, W] -> [S, H, C, N]: the sum over the
    elements of the larger of q * low and q * high, q in whole numbers of up to 127 steps. The sums are whole
    numbers below 2^24: exact in any order."""
    q = torch.where(q.isfinite(), q.float(), 0.0)
    amax = q.abs().amax(-1)
    m, e = torch.frexp(amax)
    e = torch.where(m > 127 / 128, e - 6, e - 7)
    e = torch.where(amax > 0, e, -126).clamp(-126, 127)
    q = torch.round(torch.ldexp(q, -e[..., None]))
    flat = lambda x: x.flatten(0, 1)
    n = flat(q.clamp(min=0)) @ flat(low_high[..., 1, :].float()).transpose(1, 2) + flat(q.clamp(max=0)) @ flat(low_high[..., 0, :].float()).transpose(1, 2)
    return torch.ldexp(n.view(*q.shape[:3], -1), e[..., None] + steps[:, :, None].int() - 127)


def _plain_select(st):
    case, H, top = st["case"], st["case"]["kv_heads"], st["case"]["top"]
    S, G = case["seqs"], case["heads"] // H
    # the bounds of the blocks that hold new rows, from the rows that exist
    block = torch.arange(st["most"] // BLOCK + 2, device="cuda")[None] + ((st["kv_len"] - (st["q_start"][1:] - st["q_start"][:-1])) // BLOCK)[:, None]
    rows = block[..., None] * BLOCK + torch.arange(BLOCK, device="cuda")
    there = rows < st["kv_len"][:, None, None]
    at = there.any(-1).nonzero(as_tuple=True)
    page = st["pages"][at[0], block[at]].long()
    scales = st["ks"]
    x = _values(_raw(st["kc"])[page].view(st["kc"].dtype), None if scales is None else scales[page], st["table"])    # [B, H, PAGE, W]
    x = torch.where(x.isfinite(), x, 0.0)
    x = torch.where(there[at][:, None, :, None], x, x[:, :, :1])          # a block's first row exists
    st["low_high"][page, :, 0], st["steps"][page, :, 0] = _key_bounds(x)
    used = st["pages"].long()
    N = used.shape[1]
    q = _padded(st, st["q"]).unflatten(2, (H, G)).permute(0, 2, 1, 3, 4).flatten(2, 3)                               # [S, H, n G, W]
    s = _score_keys(st["low_high"][used][:, :, :, 0].transpose(1, 2), st["steps"][used][:, :, :, 0].transpose(1, 2), q)
    s = s.unflatten(2, (-1, G)).amax(3).transpose(1, 2).flatten(0, 1)[st["flat"]]                                    # [tokens, H, N]
    b, last = torch.arange(N, device="cuda"), st["pos"][:, None, None] // BLOCK
    s = torch.where((b < FIRST) | (b > last - LAST), math.inf, s).masked_fill_(b > last, -math.inf)
    order = torch.sort(s, dim=-1, descending=True, stable=True)               # ties: the lowest block first
    chosen = torch.where(order.values == -math.inf, N, order.indices)[..., :top].sort(-1).values
    chosen = torch.where(chosen == N, -1, chosen).int()
    st["chosen"].copy_(torch.nn.functional.pad(chosen, (0, top - chosen.shape[-1]), value=-1))
    return {"chosen": st["chosen"], "low_high": st["low_high"], "steps": st["steps"]}


def _chosen_rows(st):
    """K, V of every token's chosen blocks [tokens, H, top BLOCK, D] and which of these rows it attends"""
    chosen = st["chosen"].long()
    page = st["pages"][st["seq"][:, None, None], chosen.clamp(min=0)].long()
    head = torch.arange(chosen.shape[1], device="cuda")[:, None]
    take = lambda name: _values(_raw(st[name + "c"])[page, head].view(st[name + "c"].dtype), None if st[name + "s"] is None else st[name + "s"][page, head],
                                st["table"]).flatten(2, 3)
    rows = chosen[..., None] * BLOCK + torch.arange(BLOCK, device="cuda")
    seen = (rows <= st["pos"][:, None, None, None]) & (chosen >= 0)[..., None]
    return take("k"), take("v"), seen.flatten(2, 3)


def _plain_sparse(st):
    case, H = st["case"], st["case"]["kv_heads"]
    K, V, seen = _chosen_rows(st)
    q = st["q"].float().unflatten(1, (H, -1))
    s = (q.flatten(0, 1) @ K.flatten(0, 1).transpose(1, 2)).view(*q.shape[:3], -1) * case["dim"] ** -0.5
    return _softmax_times(s, seen[:, :, None], V).flatten(1, 2).to(TYPES[case["type"]])


def run(state):
    case = state["case"]
    op = case["op"]
    if not own:
        return {"rotate": _plain_rotate, "store4": _plain_store, "attend4": _plain_attend, "select": _plain_select, "sparse": _plain_sparse}[op](state)
    from hearth_amd import paged
    stream = torch.cuda.current_stream().cuda_stream
    cache, batch = state["cache"], state["batch"]
    if op == "rotate":
        paged.append_rotated(cache, batch, state["q"], state["k"], state["v"], state["freqs"], factor=state["factor"], layout=case["layout"],
                             q_out=state["out"], stream=stream)
        if state["ks"] is None:
            return {"q": state["out"], "k": state["kc"], "v": state["vc"]}
        paged.read(cache, batch, state["k_back"], state["v_back"], stream=stream)
        return {"q": state["out"], "k": state["k_back"], "v": state["v_back"]}
    if op == "store4":
        paged.append(cache, batch, state["k"], state["v"], stream=stream)
        paged.read(cache, batch, state["k_back"], state["v_back"], stream=stream)
        return {"k": state["k_back"], "v": state["v_back"]}
    if op == "select":
        paged.update_bounds(cache, batch, state["bounds"], stream=stream)
        paged.select(state["bounds"], batch, state["q"], state["chosen"], first=FIRST, last=LAST, workspace=state["work"], stream=stream)
        return {"chosen": state["chosen"], "low_high": state["low_high"], "steps": state["steps"]}
    if op == "attend4":
        paged.attend(cache, batch, state["q"], state["out"], scale=case["dim"] ** -0.5, workspace=state["work"], stream=stream)
    else:
        paged.attend_blocks(cache, batch, state["q"], state["chosen"], state["out"], block=BLOCK, scale=case["dim"] ** -0.5, workspace=state["work"],
                            stream=stream)
    return state["out"]


# ---------------------------------------------------------------- the definition in 64 bits

def _exact_rotated(st, x):
    case, R = st["case"], st["case"]["rot"]
    angle = st["pos"].double()[:, None] * st["freqs"]
    turn = torch.polar(torch.full_like(angle, st["factor"]), angle)[:, None]
    y = x.double()
    pairs = y[..., :R].unflatten(-1, (2, R // 2)).transpose(-1, -2) if case["layout"] == "half" else y[..., :R].unflatten(-1, (R // 2, 2))
    z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
    return torch.cat([(z.transpose(-1, -2) if case["layout"] == "half" else z).flatten(-2), y[..., R:]], -1)


def _nearest(x, grid, reach):
    """Rows rounded to the grid (nonnegative values, ascending) times a power of two for each 32 elements, the least with
    which reach * it is as large as any of them: the nearest value, of two as near the one of even index."""
    b = x.double().unflatten(-1, (-1, 32))
    top = b.abs().amax(-1).clamp(min=2.0 ** -118)
    e = torch.ceil(torch.log2(top / reach))
    e = torch.where(torch.exp2(e - 1) * reach >= top, e - 1, e).clamp(min=-126)[..., None]
    a = b.abs() / torch.exp2(e)
    up = torch.bucketize(a, grid).clamp(1, len(grid) - 1)           # grid[up - 1] < a <= grid[up]
    far, near = grid[up] - a, a - grid[up - 1]
    i = torch.where((far < near) | ((far == near) & (up % 2 == 0)), up, up - 1)
    return (torch.where(b < 0, -1.0, 1.0) * grid[i] * torch.exp2(e)).flatten(-2)


def _exact_rows(st, x):
    if st["case"]["store"] == "mx4":
        return _nearest(x, torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device="cuda"), 7.0)
    if st["case"]["store"] == "mx8":
        every = torch.arange(127, device="cuda", dtype=torch.uint8).view(torch.float8_e4m3fn).double()
        return _nearest(x, every, 448.0)
    return x.double()


def _exact_sequence(st, name, s):
    """Rows of a sequence [H, rows, D] in 64 bits"""
    used = st["pages"][s].long()
    x, sc = _raw(st[name + "c"])[used], st[name + "s"]
    if sc is None:
        x = x.double()
    else:
        if st["case"]["store"] == "mx4":
            mag, sign = _halves(x) % 8, 1.0 - 2.0 * (_halves(x) // 8).double()
            low, high = mag.double() / 2, (1 + (mag % 2).double() / 2) * torch.exp2((mag // 2).double() - 1)       # below and from 1 on
            x = sign * torch.where(mag < 2, low, high)
        else:
            x = x.view(torch.float8_e4m3fn).float().double()
        x = x * torch.exp2(sc[used].double() - 127.0).repeat_interleave(32, -1)
    return x.transpose(0, 1).flatten(1, 2)


def _exact_select(st):
    """Block by block from the rows themselves: whole numbers throughout."""
    case, H, W, top = st["case"], st["case"]["kv_heads"], st["case"]["dim"], st["case"]["top"]
    lens, news, G = _lens(case), _news(case), case["heads"] // st["case"]["kv_heads"]

    def whole(x, magnitude):
        """x in whole steps of a power of two for each magnitude [..., 1], the exponents"""
        e = torch.ceil(torch.log2(magnitude.clamp(min=2.0 ** -126) / 127.0))
        e = torch.where(torch.exp2(e - 1) * 127.0 >= magnitude, e - 1, e).clamp(min=-126)
        return torch.round(x / torch.exp2(e)), e

    low_high, steps = st["low_high"].clone(), st["steps"].clone()
    chosen = torch.full_like(st["chosen"], -1)
    at = 0
    for s, (L, n) in enumerate(zip(lens, news)):
        N = _blocks(L)
        K = _exact_sequence(st, "k", s)[:, :L]
        K = torch.cat([K, K[:, (N - 1) * BLOCK:(N - 1) * BLOCK + 1].expand(-1, N * BLOCK - L, -1)], 1).unflatten(1, (N, BLOCK))
        ends = torch.stack([K.amin(2), K.amax(2)], 2)                        # [H, N, 2, W]
        codes, e = whole(ends, ends.abs().amax((2, 3), keepdim=True))
        touched = slice((L - n) // BLOCK, N)
        page = st["pages"][s, touched].long()
        low_high[page, :, 0], steps[page, :, 0] = codes[:, touched].transpose(0, 1).to(torch.int8), (e[:, touched, 0, 0].T + 127).to(torch.uint8)
        for i in range(0, n, 32):
            q = st["q"][at + i:at + min(i + 32, n)].double()
            q, eq = whole(q, q.abs().amax(-1, keepdim=True))
            score = torch.full((len(q), H, N), -math.inf, dtype=torch.float64, device="cuda")
            for h in range(case["heads"]):
                z = q[:, h].clamp(min=0) @ codes[h // G, :, 1].T - (-q[:, h]).clamp(min=0) @ codes[h // G, :, 0].T
                score[:, h // G] = torch.maximum(score[:, h // G], z * torch.exp2(eq[:, h] + e[h // G, :, 0, 0]))
            b, last = torch.arange(N, device="cuda"), (torch.arange(L - n + i, L - n + i + len(q), device="cuda") // BLOCK)[:, None, None]
            score = torch.where((b < FIRST) | (b > last - LAST), math.inf, score).masked_fill_(b > last, -math.inf)
            rank = torch.argsort(torch.argsort(-score, dim=-1, stable=True), dim=-1)
            take = (rank < top) & (b <= last)
            place = take.cumsum(-1) - 1
            t, h, j = take.nonzero(as_tuple=True)
            chosen[at + i + t, h, place[t, h, j]] = j.int()
        at += n
    return {"chosen": chosen, "low_high": low_high, "steps": steps}


def _exact_attention(st):
    case, G = st["case"], st["case"]["heads"] // st["case"]["kv_heads"]
    lens, news, out, at = _lens(case), _news(case), [], 0
    for s, (L, n) in enumerate(zip(lens, news)):
        K, V = _exact_sequence(st, "k", s)[:, :L], _exact_sequence(st, "v", s)[:, :L]
        t = torch.arange(L, device="cuda")
        o = torch.empty(n, case["heads"], case["dim"], dtype=torch.float64, device="cuda")
        for h in range(case["heads"]):
            seen = t <= (L - n + torch.arange(n, device="cuda"))[:, None]
            if case["op"] == "sparse":
                c = st["chosen"][at:at + n, h // G].long()
                blocks = torch.zeros(n, _blocks(L) + 1, dtype=torch.bool, device="cuda")
                blocks.scatter_(1, torch.where(c < 0, _blocks(L), c), True)
                seen &= blocks[:, t // BLOCK]
            z = st["q"][at:at + n, h].double() @ K[h // G].T * case["dim"] ** -0.5
            o[:, h] = torch.softmax(torch.where(seen, z, -math.inf), -1) @ V[h // G]
        out.append(o)
        at += n
    return torch.cat(out)


def exact(case, seed):
    global own
    if case["op"] == "attend4" and work(case)["flops"] > 4e12:
        return None
    mine, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = mine
    if case["op"] == "rotate":
        if st["ks"] is None:
            out = {"q": _exact_rotated(st, st["q"])}
            for name, x in (("k", _exact_rotated(st, st["k"])), ("v", st["v"].double())):
                out[name] = torch.zeros(st[name + "c"].shape, dtype=torch.float64, device="cuda")
                out[name][st["page_of"], :, st["row_of"]] = x
            return out
        # a rotated key is rounded to its type and then to a code: neither alone is the definition's
        return {"q": _exact_rotated(st, st["q"]), "k": None, "v": _exact_rows(st, st["v"])}
    if case["op"] == "store4":
        return {"k": _exact_rows(st, st["k"]), "v": _exact_rows(st, st["v"])}
    if case["op"] == "select":
        return _exact_select(st)
    return _exact_attention(st)
