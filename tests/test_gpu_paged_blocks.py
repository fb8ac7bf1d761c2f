"""Attention over chosen blocks on the GPU: bounds, choice and attention against the plain forms
(block_oracle.py, paged_oracle.py): every cache type and width, block sizes from 16 rows to a page, groups of
query heads that do not fill a tile and that fill several, ties, trees, missing pages, rows that do
not exist, infinities and NaN, splits, strides, other streams, captured graphs, and all of it together."""
from __future__ import annotations

import math

import pytest
import torch

import block_oracle as B
import paged_oracle as O
import paged_oracle4 as P
import test_gpu_paged as base
import test_gpu_paged_mx4 as four
from hearth_amd import paged

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16
STORES = [(BF, "bf16"), (HF, "f16"), (BF, "mx8"), (HF, "mx4")]


def make(g, n_pages, heads, page, width, kind, store):
    """CPU copies of a cache, the device's, and the Cache"""
    if store == "mx4":
        c = four.make_cache(g, n_pages, heads, page, width, kind, store)
        return c, *four.on_gpu(c)
    c = base.make_cache(g, n_pages, heads, page, width, kind, store)
    return c, *base.on_gpu(c)


def new_bounds(n_pages, heads, page, block, width):
    lh = torch.full((n_pages, heads, page // block, 2, width), 77, dtype=torch.int8, device="cuda")
    st = torch.full((n_pages, heads, page // block), 201, dtype=torch.uint8, device="cuda")
    return paged.Bounds(lh, st, block=block)


def check_bounds(bd, c, pages, lens, news, block, touched=None):
    """the touched blocks of every sequence; everything else as it was (77, 201)"""
    lh, st = bd.low_high.cpu(), bd.steps.cpu()
    per = c["k"].shape[2] // block
    left = torch.ones(st.shape, dtype=torch.bool)
    for s, (L, n) in enumerate(zip(lens, news)):
        K, ok = P.rows_of(c["k"], c["ks"], pages[s], L)
        codes, byte = B.bounds(K, ok, block)
        for b in range(max(L - n, 0) // block, -(-L // block) if n else 0):
            pg = pages[s, b // per].item()
            if not 0 <= pg < st.shape[0]:
                continue
            assert torch.equal(lh[pg, :, b % per].double(), codes[:, b]), (s, b)
            assert torch.equal(st[pg, :, b % per].long(), byte[:, b]), (s, b)
            left[pg, :, b % per] = False
    assert (st[left] == 201).all() and (lh[left] == 77).all()


LENS, NEWS = [1, 16, 17, 70, 333, 0, 200, 4], [1, 16, 1, 33, 2, 0, 200, 9]


@pytest.mark.parametrize("kind,store", STORES)
@pytest.mark.parametrize("heads,width,page,block", [(2, 64, 64, 16), (4, 128, 64, 64), (1, 256, 32, 32), (3, 128, 256, 64)])
def test_bounds(kind, store, heads, width, page, block):
    g = base._gen(width + block)
    pages, n_pages = base.deal(g, LENS, page)
    c, d, cache = make(g, n_pages, heads, page, width, kind, store)
    if store != "mx4":                               # NaN and infinities count as 0; a block of zeros
        c["k"].view(torch.uint8 if store == "mx8" else torch.int16)[pages[4, 0].item(), 0, 5, 7] = {"bf16": 0x7fc0, "f16": 0x7c00, "mx8": 0x7f}[store]
    else:
        c["ks"][pages[4, 0].item(), 0, 5, 0] = 255
    c["k"].view(torch.uint8)[pages[2, 0].item()] = 0
    d["k"].view(torch.uint8).copy_(c["k"].view(torch.uint8))
    if c["ks"] is not None:
        d["ks"].copy_(c["ks"])
    bd = new_bounds(n_pages, heads, page, block, width)
    b, _ = base.batch_of(pages, LENS, NEWS)
    paged.update_bounds(cache, b, bd, stream=base._stream())
    check_bounds(bd, c, pages, LENS, NEWS, block)
    # the whole sequences
    b, _ = base.batch_of(pages, LENS, LENS)
    paged.update_bounds(cache, b, bd, stream=base._stream())
    check_bounds(bd, c, pages, LENS, LENS, block)


def test_bounds_of_limits_and_missing_pages():
    g = base._gen(2)
    pages = torch.tensor([[0, 99, 2, -5], [1, 3, 4, 5]], dtype=torch.int32)
    c, d, cache = make(g, 6, 2, 16, 64, BF, "bf16")
    bd = new_bounds(6, 2, 16, 16, 64)
    lens, news = [60, 50], [60, 30]
    b, _ = base.batch_of(pages, lens, news, max_q=20, max_kv=40)      # rows 0 .. 19 of one, 20 .. 39 of the other, whose rows past 40 do not exist
    paged.update_bounds(cache, b, bd, stream=base._stream())
    lh = bd.low_high.cpu()
    for s, blocks in ((0, [0]), (1, [1, 2])):
        K, ok = P.rows_of(c["k"], None, pages[s], 40)
        codes, _ = B.bounds(K, ok, 16)
        for n in blocks:
            assert torch.equal(lh[pages[s, n].item(), :, 0].double(), codes[:, n])
    assert (lh[[1, 2, 5]] == 77).all()


def choice(g, kind, store, heads, kv_heads, width, lens, news, page, block, top, first=1, last=1, trees=None, pages=None, n_pages=None, pad=2, edit=None, queries=None,
           max_kv=None, strided=False):
    if pages is None:
        pages, n_pages = base.deal(g, lens, page)
    c, d, cache = make(g, n_pages, kv_heads, page, width, kind, store)
    if edit:
        edit(c["k"], pages)
        d["k"].copy_(c["k"])
    bd = new_bounds(n_pages, kv_heads, page, block, width)
    whole, _ = base.batch_of(pages, lens, lens, max_kv=max_kv)
    paged.update_bounds(cache, whole, bd, stream=base._stream())
    T = sum(news)
    q = torch.randn(T + pad, heads, width, generator=g).to(kind)
    if queries:
        queries(q)
    mask = torch.cat([O.words(trees, max(news)), torch.zeros(pad, -(-max(news) // 64), dtype=torch.int64)]) if trees else None
    b, starts = base.batch_of(pages, lens, news, mask, max_kv=max_kv)
    buf = torch.full((T + pad, kv_heads, top + 3), -9, dtype=torch.int32, device="cuda") if strided else torch.full((T + pad, kv_heads, top), -9, dtype=torch.int32, device="cuda")
    chosen = buf[..., 1:top + 1] if strided else buf
    need = paged.select_workspace_bytes(bd, b, T + pad)
    work = torch.full((need + 64,), 255, dtype=torch.uint8, device="cuda")
    qd = q.cuda()
    paged.select(bd, b, qd, chosen, first=first, last=last, workspace=work[:need], stream=base._stream())
    got = chosen.cpu()
    assert (work[need:] == 255).all() and (got[T:] == -9).all()
    if strided:
        assert (buf[..., 0] == -9).all() and (buf[..., top + 1:] == -9).all()
    for s, (L, n) in enumerate(zip(lens, news)):
        kv = min(L, max_kv if max_kv is not None else L)
        K, ok = P.rows_of(c["k"], c["ks"], pages[s], kv)
        codes, byte = B.bounds(K, ok, block)
        want = B.choose(codes, byte, q[starts[s]:starts[s] + n].double(), L - n, kv, block, top, first, last, bool(trees))
        assert torch.equal(got[starts[s]:starts[s] + n], want), s
    return got


@pytest.mark.parametrize("kind,store", STORES)
@pytest.mark.parametrize("heads,kv_heads,width,page,block", [(8, 2, 128, 64, 64), (7, 1, 64, 64, 16), (4, 4, 256, 32, 32), (6, 2, 128, 128, 32), (40, 2, 64, 16, 16), (128, 1, 128, 64, 16)])
def test_choice(kind, store, heads, kv_heads, width, page, block):
    """Sequences with fewer blocks than are chosen, as many and more; no rows; more tokens than rows."""
    lens, news = [1, 70, 333, 0, 1200, 5, block * 8, block * 8 + 1], [1, 33, 2, 1, 4, 9, 1, 1]
    choice(base._gen(heads + width), kind, store, heads, kv_heads, width, lens, news, page, block, 8, 1, 2)


@pytest.mark.parametrize("top,first,last", [(1, 0, 1), (2, 1, 1), (5, 0, 1), (13, 3, 4), (64, 1, 1), (300, 0, 1), (7, 0, 7), (7, 6, 1)])
def test_choice_counts(top, first, last):
    choice(base._gen(top), BF, "bf16", 4, 2, 64, [2000, 130, 16 * top, 16 * top + 16], [3, 1, 2, 1], 64, 16, top, first, last, strided=True)


def test_choice_of_long_sequences():
    """Blocks shared out among workgroups; more than a workgroup's worth of keys."""
    choice(base._gen(8), HF, "f16", 4, 1, 64, [70001], [2], 64, 16, 32, 1, 2)
    choice(base._gen(9), BF, "mx4", 8, 2, 128, [20000, 9000], [1, 1], 64, 64, 16)


@pytest.mark.parametrize("heads,kv_heads,width", [(2, 2, 256), (4, 2, 64), (3, 1, 256), (7, 1, 256), (10, 1, 128), (16, 1, 256), (2, 2, 64), (4, 2, 128), (17, 1, 256)])
def test_choice_of_many_tokens(heads, kv_heads, width):
    """Tokens that fill several waves' rows, whole and in part, at every width and number of heads to a token."""
    choice(base._gen(heads * width), BF, "mx8", heads, kv_heads, width, [90, 400, 70, 1], [90, 71, 64, 1], 32, 16, 7, 1, 1)
    choice(base._gen(heads + width), HF, "f16", heads, kv_heads, width, [1300], [67], 64, 16, 9, 0, 3, trees=[O.tree(67)])


def test_choice_of_more_blocks_than_registers_hold():
    choice(base._gen(14), BF, "bf16", 1, 1, 64, [140001], [1], 64, 16, 25, 1, 2)


@pytest.mark.parametrize("rows", [600 * 16, 2500 * 16, 9000 * 16])
def test_ties_across_waves(rows):
    """Keys that repeat over long sequences: every second or seventh block scores the same; the lowest are taken, whichever wave
    they lie with."""
    for every in (2, 7):
        def edit(k, pages):
            for i in range(every, k.shape[0]):
                k[i] = k[i % every]

        n = rows // 16
        got = choice(base._gen(every), BF, "bf16", 2, 1, 64, [rows], [1], 16, 16, 11, 0, 1, pages=torch.arange(n, dtype=torch.int32)[None], n_pages=n, edit=edit)
        assert (got[0, 0, :10].diff() == every).all()


@pytest.mark.parametrize("tree", [True, False])
def test_choice_of_trees_and_max_kv(tree):
    news = [40, 7, 1]
    choice(base._gen(4), BF, "bf16", 8, 2, 64, [700, 7, 90], news, 32, 16, 12, 1, 2, trees=[O.tree(n) for n in news] if tree else None)
    choice(base._gen(5), BF, "bf16", 8, 2, 64, [700, 30, 90], news, 32, 16, 12, 1, 2, max_kv=300)


def test_choice_of_equal_scores():
    """Keys that repeat from block to block, and queries of zeros: the lowest blocks."""
    def edit(k, pages):
        for i in range(k.shape[0]):
            k[i] = k[i % 2]

    pages = torch.arange(40, dtype=torch.int32)[None]
    got = choice(base._gen(6), BF, "bf16", 4, 2, 64, [40 * 16], [2], 16, 16, 9, 0, 1, pages=pages, n_pages=40, edit=edit)
    assert (got[:2, :, :8].diff(dim=-1) == 2).all()                       # every second block scores the same
    got = choice(base._gen(7), BF, "bf16", 4, 2, 64, [40 * 16], [1], 16, 16, 9, 0, 1, pages=pages, n_pages=40, queries=lambda q: q.zero_())
    assert torch.equal(got[0, 0], torch.tensor([0, 1, 2, 3, 4, 5, 6, 7, 39], dtype=torch.int32))


def test_choice_skips_missing_pages_and_survives_infinities():
    pages = torch.tensor([[0, 77, 2, -3, 4, 5, 1, 6]], dtype=torch.int32)
    choice(base._gen(10), BF, "bf16", 4, 1, 64, [128], [3], 16, 16, 6, 2, 2, pages=pages, n_pages=7)
    choice(base._gen(11), BF, "bf16", 4, 1, 64, [128], [3], 16, 16, 8, 2, 2, pages=pages, n_pages=7)

    def edit(k, pages):
        k[2, :, 3, 5], k[4, :, :, 9], k[5, :, 1] = math.inf, -math.inf, math.nan

    def queries(q):
        q[0, 0, 5], q[1, 1, 9], q[2] = math.nan, math.inf, 3e38

    choice(base._gen(12), BF, "bf16", 4, 1, 64, [112], [3], 16, 16, 4, 0, 1, pages=torch.arange(7, dtype=torch.int32)[None], n_pages=7, edit=edit, queries=queries)


# ---------------------------------------------------------------- attention

def random_blocks(g, lens, news, heads, top, block, pad=2):
    """distinct blocks of each token in no order, some past its row, gaps of -1"""
    out = torch.full((sum(news) + pad, heads, top), -1, dtype=torch.int32)
    t = 0
    for L, n in zip(lens, news):
        N = max(-(-L // block), 1)
        for _ in range(n):
            for h in range(heads):
                x = torch.randperm(N, generator=g)[:top].int()
                x[torch.rand(len(x), generator=g) < 0.15] = -1
                out[t, h, :len(x)] = x
            t += 1
    return out


def sparse(g, kind, store, heads, kv_heads, width, lens, news, page, block, top, trees=None, pages=None, n_pages=None, edit=None, pad=2, chosen=None, scale=None):
    if pages is None:
        pages, n_pages = base.deal(g, lens, page)
    c, d, cache = make(g, n_pages, kv_heads, page, width, kind, store)
    if edit:
        edit(c, pages)
        for n, t in c.items():
            if t is not None:
                d[n].copy_(t)
    T = sum(news)
    q = torch.randn(T + pad, heads, width, generator=g).to(kind)
    chosen = random_blocks(g, lens, news, kv_heads, top, block, pad) if chosen is None else chosen
    scale = width ** -0.5 if scale is None else scale
    mask = torch.cat([O.words(trees, max(news)), torch.zeros(pad, -(-max(news) // 64), dtype=torch.int64)]) if trees else None
    b, starts = base.batch_of(pages, lens, news, mask)
    out = torch.full((T + pad, heads, width), 9.0, dtype=kind, device="cuda")
    lse = torch.full((T + pad, heads), 9.0, device="cuda")
    need = paged.attend_blocks_workspace_bytes(cache, b, heads, top, block, T + pad)
    work = torch.full((need + 64,), 255, dtype=torch.uint8, device="cuda")
    qd, cd = q.cuda(), chosen.cuda()
    paged.attend_blocks(cache, b, qd, cd, out, block=block, scale=scale, lse=lse, workspace=work[:need], stream=base._stream())
    got, glse = out.cpu(), lse.cpu()
    assert (work[need:] == 255).all() and (got[T:] == 9).all() and (glse[T:] == 9).all()
    for s, (L, n) in enumerate(zip(lens, news)):
        K, ok = P.rows_of(c["k"], c["ks"], pages[s], L)
        V, _ = P.rows_of(c["v"], c["vs"], pages[s], L)
        lo = starts[s]
        want, wl, tol, ltol = B.attention(q[lo:lo + n].double(), K, V, ok, L - n, scale, kind, chosen[lo:lo + n], block, trees[s] if trees else None)
        x, xl = got[lo:lo + n].double(), glse[lo:lo + n].double()
        fine = torch.isfinite(want)
        assert ((x - want).abs() <= tol)[fine].all(), (s, L, n)
        assert torch.equal(torch.isnan(x), torch.isnan(want)) and torch.equal(x.isinf(), want.isinf()), s
        empty = wl == -math.inf
        assert (xl[empty] == -math.inf).all() and (x[empty] == 0).all()
        live = torch.isfinite(wl)
        assert ((xl - wl).abs() <= ltol)[live].all(), s
    return got


@pytest.mark.parametrize("kind,store", STORES)
@pytest.mark.parametrize("heads,kv_heads,width,page,block", [(8, 2, 128, 64, 64), (7, 1, 64, 64, 16), (4, 4, 256, 32, 32), (40, 2, 64, 16, 16), (16, 1, 128, 128, 128)])
def test_sparse(kind, store, heads, kv_heads, width, page, block):
    lens, news = [1, 70, 333, 0, 700, 5, block * 8], [1, 5, 2, 1, 4, 9, 1]
    for top in (1, 5):
        sparse(base._gen(heads + width + top), kind, store, heads, kv_heads, width, lens, news, page, block, top)


@pytest.mark.parametrize("kind,store", STORES)
@pytest.mark.parametrize("width", [64, 128, 256])
def test_sparse_split(kind, store, width):
    """Rows that are split among workgroups and joined, by a group of threads and by several."""
    sparse(base._gen(width), kind, store, 8, 1, width, [4000, 100], [1, 1], 64, 64, 33)
    sparse(base._gen(width + 1), kind, store, 4, 1, width, [20000], [1], 64, 64, 200)


@pytest.mark.parametrize("kind,store", STORES)
@pytest.mark.parametrize("heads,kv_heads,width,page,block", [(8, 2, 128, 64, 64), (7, 1, 64, 64, 32), (4, 4, 256, 64, 64), (40, 2, 64, 256, 64), (16, 1, 128, 256, 128)])
def test_sparse_of_many_tokens(kind, store, heads, kv_heads, width, page, block):
    """Sequences of 15 tokens at most and of 16; lists with gaps of whole steps, without any block, and trees."""
    for n in (15, 16):
        g = base._gen(heads + width + n)
        lens, news = [1, 70, 700, n], [1, 3, n, n]
        chosen = random_blocks(g, lens, news, kv_heads, 5, block)
        chosen[4:8] = -1                                              # the third sequence's first four tokens: none,
        chosen[5, :, 0] = chosen[6, :, 4] = 0                         # the first entry, the last,
        chosen[7, :, 1] = chosen[7, :, 3] = torch.arange(kv_heads, dtype=torch.int32) % (700 // block)   # one twice between gaps
        chosen[7, :, 3] += 1
        sparse(g, kind, store, heads, kv_heads, width, lens, news, page, block, 5, chosen=chosen)
    news = [33, 16, 1]
    sparse(base._gen(width), kind, store, heads, kv_heads, width, [500, 16, 90], news, page, block, 9, trees=[O.tree(n) for n in news])


@pytest.mark.parametrize("kind,store", STORES)
def test_sparse_of_many_tokens_and_bad_rows(kind, store):
    """An infinity in a later row of the tokens' own block, a NaN there, pages that are not there."""
    def edit(c, pages):
        v = c["v"].view(torch.uint8 if store in ("mx8", "mx4") else torch.int16)
        if store == "mx4":
            c["vs"][pages[0, 3].item(), :, 15] = 255
        else:
            v[pages[0, 3].item(), 0, 14, 3] = {"bf16": 0x7f80, "f16": 0x7c00, "mx8": 0x7f}[store]
            v[pages[0, 3].item(), 1, 15, 5] = {"bf16": 0x7fc0, "f16": 0x7e00, "mx8": 0xff}[store]
        v[pages[0, 3].item(), :, 20:] = 0x7fff if v.dtype == torch.int16 else 0x7f
    g = base._gen(77)
    pages, n_pages = torch.tensor([[1, 99, 4, 2, 3], [0, 5, -8, 7, 6]], dtype=torch.int32), 8
    lens, news = [3 * 64 + 17, 300], [17, 20]
    chosen = torch.arange(5, dtype=torch.int32).expand(37 + 2, 2, 5).contiguous()
    got = sparse(g, kind, store, 8, 2, 128, lens, news, 64, 64, 5, pages=pages, n_pages=n_pages, edit=edit, chosen=chosen)
    assert got[:14].isfinite().all() and not got[15:17].isfinite().all()


def test_every_block_is_the_attention():
    """All blocks chosen: the bits of attend where the rows fall into the same steps, whatever the group."""
    g = base._gen(31)
    for heads, kv_heads in ((8, 1), (16, 2)):
        lens, news, page = [400, 130], [1, 1], 64
        pages, n_pages = base.deal(g, lens, page)
        _, _, cache = make(g, n_pages, kv_heads, page, 128, BF, "mx4")
        b, _ = base.batch_of(pages, lens, news)
        q = torch.randn(2, heads, 128, generator=g).to(BF).cuda()
        out = [torch.zeros_like(q) for _ in range(2)]
        lse = [torch.zeros(2, heads, device="cuda") for _ in range(2)]
        chosen = torch.arange(7, dtype=torch.int32, device="cuda").expand(2, kv_heads, 7)
        assert paged.workspace_bytes(cache, b, heads, 2) == 0 == paged.attend_blocks_workspace_bytes(cache, b, heads, 7, 64, 2)
        paged.attend(cache, b, q, out[0], scale=0.1, lse=lse[0], stream=base._stream())
        paged.attend_blocks(cache, b, q, chosen, out[1], block=64, scale=0.1, lse=lse[1], stream=base._stream())
        assert torch.equal(*out) and torch.equal(*lse)


def test_sparse_trees_scales_and_bad_input():
    g = base._gen(41)
    news = [40, 7, 1]
    sparse(g, BF, "bf16", 8, 2, 64, [300, 7, 90], news, 32, 16, 9, trees=[O.tree(n) for n in news])
    for scale in (-0.3, 0.0, 40.0):
        sparse(g, BF, "mx8", 8, 2, 128, [300, 90], [2, 1], 32, 32, 4, scale=scale)
    # missing pages; numbers that are no blocks; a block twice
    pages = torch.tensor([[0, 77, 2, 3, -1, 5, 1, 6]], dtype=torch.int32)
    sparse(g, BF, "bf16", 8, 2, 64, [120], [3], 16, 16, 6, pages=pages, n_pages=7)
    chosen = torch.full((4, 2, 5), -1, dtype=torch.int32)
    chosen[0, 0] = torch.tensor([0x7fffffff, -0x80000000, 3, 1 << 27, 9], dtype=torch.int32)
    chosen[1, 1] = torch.tensor([2, 2, -7, 2, 0], dtype=torch.int32)
    clean = chosen.clone()
    clean[0, 0] = torch.tensor([-1, -1, 3, -1, -1], dtype=torch.int32)
    out = [sparse(base._gen(42), BF, "bf16", 4, 2, 64, [60], [2], 16, 16, 5, chosen=x) for x in (clean,)]
    lens, page = [60], 16
    g = base._gen(42)
    pages, n_pages = base.deal(g, lens, page)
    _, _, cache = make(g, n_pages, 2, page, 64, BF, "bf16")
    q = torch.randn(4, 4, 64, generator=g).to(BF).cuda()
    b, _ = base.batch_of(pages, lens, [2])
    o = torch.full_like(q, 9.0)
    paged.attend_blocks(cache, b, q, chosen.cuda(), o, block=16, scale=0.125, stream=base._stream())
    assert torch.equal(o.cpu(), out[0])


@pytest.mark.parametrize("store", ["bf16", "mx8", "mx4"])
@pytest.mark.parametrize("split", [False, True])
def test_sparse_nan_and_infinity_in_rows_not_attended(store, split):
    """Behind a sequence's end, in a token's later rows and in blocks that are not chosen."""
    block, page, heads = 32, 64, 8
    L, n = (2000, 5) if split else (300, 5)
    N = -(-L // block)
    top = 40 if split else 6
    g = base._gen(51)
    chosen = torch.full((n + 2, 2, top), -1, dtype=torch.int32)
    for t in range(n):
        for h in range(2):
            x = torch.randperm(N - 2, generator=g)[:top - 1] + 1       # never block 0
            chosen[t, h, :len(x)] = x.int()
            chosen[t, h, top - 1] = N - 1

    def edit(c, pages):
        bad = lambda p, r: [c[x + "s"].__setitem__((p, slice(None), r), 255) if store == "mx4" else c[x].view(torch.uint8).__setitem__((p, slice(None), r, slice(3, None, 7)), 0x7f) if
                            store == "mx8" else c[x].__setitem__((p, slice(None), r, 3), math.inf if x == "v" else math.nan) for x in ("k", "v")]
        for r in range(L % page, page):
            bad(pages[0, (L - 1) // page].item(), r)
        bad(pages[0, (L - 2) // page].item(), (L - 2) % page)              # attended by the last two tokens
        bad(pages[0, 0].item(), 7)                                        # in block 0

    got = sparse(base._gen(52), BF, store, heads, 2, 64, [L], [n], page, block, top, edit=edit, chosen=chosen)
    assert got[:n - 2].isfinite().all() and not got[n - 2:n].isfinite().all(-1).any()


def test_sparse_strides():
    """q, out and the choice cut from wider arrays and heads first: the same bits as dense ones."""
    g = base._gen(61)
    lens, news, page = [300, 37], [5, 2], 16
    pages, n_pages = base.deal(g, lens, page)
    _, _, cache = make(g, n_pages, 2, page, 64, HF, "mx8")
    b, _ = base.batch_of(pages, lens, news)
    q, chosen = torch.randn(7, 8, 64, generator=g).to(HF).cuda(), random_blocks(g, lens, news, 2, 4, 16, 0).cuda()
    dense = torch.empty_like(q)
    paged.attend_blocks(cache, b, q, chosen, dense, block=16, scale=0.125, stream=base._stream())
    cuts = ((lambda: torch.zeros(7, 8, 131, dtype=HF, device="cuda")[..., 3:67], torch.zeros(7, 2, 9, dtype=torch.int32, device="cuda")[..., 2:6]),
            (lambda: torch.zeros(8, 7, 64, dtype=HF, device="cuda").transpose(0, 1), torch.zeros(2, 7, 4, dtype=torch.int32, device="cuda").transpose(0, 1)))
    for cut, c2 in cuts:
        q2, o2 = cut(), cut()
        q2.copy_(q), c2.copy_(chosen)
        paged.attend_blocks(cache, b, q2, c2, o2, block=16, scale=0.125, stream=base._stream())
        assert torch.equal(o2, dense)


def test_offsets_past_32_bits_on_a_side_stream():
    """Caches of more than 4 GiB a tensor, their last pages used by every operator."""
    page, heads, width, L = 64, 2, 128, 150
    n_pages = (9 << 29) // (heads * page * width * 2) + 2
    k = torch.empty(n_pages, heads, page, width, dtype=BF, device="cuda")
    v = torch.empty_like(k)
    lh = torch.empty(n_pages, heads, 4, 2, width, dtype=torch.int8, device="cuda")
    bd = paged.Bounds(lh, torch.empty(n_pages, heads, 4, dtype=torch.uint8, device="cuda"), block=16)
    g = base._gen(17)
    pages = torch.tensor([[n_pages - 1, 0, n_pages - 2]], dtype=torch.int32)
    b, _ = base.batch_of(pages, [L], [L])
    nk, nv, q = (torch.randn(L, heads * m, width, generator=g).to(BF) for m in (1, 1, 4))
    dk, dv, dq = nk.cuda(), nv.cuda(), q.cuda()
    cache = paged.Cache(k, v)
    out, chosen = torch.empty_like(dq), torch.empty(L, heads, 5, dtype=torch.int32, device="cuda")
    work = torch.empty(paged.select_workspace_bytes(bd, b, L), dtype=torch.uint8, device="cuda")
    more = torch.empty(max(paged.attend_blocks_workspace_bytes(cache, b, 8, 5, 16, L), 16), dtype=torch.uint8, device="cuda")
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        paged.append(cache, b, dk, dv, stream=side.cuda_stream)
        paged.update_bounds(cache, b, bd, stream=side.cuda_stream)
        paged.select(bd, b, dq, chosen, workspace=work, stream=side.cuda_stream)
        paged.attend_blocks(cache, b, dq, chosen, out, block=16, scale=width ** -0.5, workspace=more, stream=side.cuda_stream)
    side.synchronize()
    K, ok = nk.double().transpose(0, 1), torch.ones(L, dtype=torch.bool)
    want = B.choose(*B.bounds(K, ok, 16), q.double(), 0, L, 16, 5, 1, 1)
    assert torch.equal(chosen.cpu(), want)
    o, _, tol, _ = B.attention(q.double(), K, nv.double().transpose(0, 1), ok, 0, width ** -0.5, BF, want, 16)
    assert ((out.cpu().double() - o).abs() <= tol).all()


@pytest.mark.parametrize("store", ["bf16", "mx4"])
def test_together_eager_and_captured(store):
    """A layer's step over long sequences, token after token for two of them: append_rotated, update_bounds,
    select and attend_blocks; the same steps as one captured graph whose lengths live in device memory, replayed with
    eager work between; the last step against the plain forms; and a chain of the last tokens at once."""
    g = base._gen(33)
    page, block, H, Hkv, W, steps, top = 32, 16, 8, 2, 64, 20, 6
    pages = torch.randperm(64, generator=g).int().view(2, 32)
    n_pages = 64
    freqs = torch.from_numpy(paged.rope_frequencies(W, 1e4)[0]).cuda()
    q_start = torch.arange(3, dtype=torch.int32).cuda()
    qs, ks, vs = (torch.randn(steps, 2, h, W, generator=g).to(BF).cuda() for h in (H, Hkv, Hkv))
    lens0 = torch.tensor([5, 900], dtype=torch.int32)
    dp = pages.cuda()

    def fresh():
        c, d, cache = make(base._gen(34), n_pages, Hkv, page, W, BF, store)
        bd = new_bounds(n_pages, Hkv, page, block, W)
        b = paged.Batch(dp, lens0.cuda(), torch.tensor([0, 5, 905], dtype=torch.int32).cuda(), max_q=900, max_kv=900)
        paged.update_bounds(cache, b, bd, stream=base._stream())
        return d, cache, bd

    def layer(cache, bd, kv_len, q, k, v, bufs):
        b = paged.Batch(dp, kv_len, q_start, max_q=1, max_kv=1024)
        paged.append_rotated(cache, b, q, k, v, freqs, q_out=bufs["q"], stream=base._stream())
        paged.update_bounds(cache, b, bd, stream=base._stream())
        paged.select(bd, b, bufs["q"], bufs["chosen"], first=1, last=2, workspace=bufs["w1"], stream=base._stream())
        paged.attend_blocks(cache, b, bufs["q"], bufs["chosen"], bufs["out"], block=block, scale=W ** -0.5, workspace=bufs["w2"], stream=base._stream())

    def buffers(cache, bd, n=2):
        b = paged.Batch(dp, lens0.cuda(), q_start, max_q=n // 2, max_kv=1024)
        return dict(q=torch.empty(n, H, W, dtype=BF, device="cuda"), out=torch.empty(n, H, W, dtype=BF, device="cuda"),
                    chosen=torch.empty(n, Hkv, top, dtype=torch.int32, device="cuda"),
                    w1=torch.empty(paged.select_workspace_bytes(bd, b, n), dtype=torch.uint8, device="cuda"),
                    w2=torch.empty(max(paged.attend_blocks_workspace_bytes(cache, b, H, top, block, n), 16), dtype=torch.uint8, device="cuda"))

    d1, c1, b1 = fresh()
    bufs = buffers(c1, b1)
    eager = []
    for i in range(steps):
        layer(c1, b1, (lens0 + 1 + i).cuda(), qs[i], ks[i], vs[i], bufs)
        eager.append({n: bufs[n].clone() for n in ("q", "chosen", "out")})
    torch.cuda.synchronize()
    cpu = {n: None if t is None else t.cpu() for n, t in d1.items()}
    for s in range(2):
        L = int(lens0[s]) + steps
        K, ok = P.rows_of(cpu["k"], cpu["ks"], pages[s], L)
        V, _ = P.rows_of(cpu["v"], cpu["vs"], pages[s], L)
        q = eager[-1]["q"][s:s + 1].cpu().double()
        want = B.choose(*B.bounds(K, ok, block), q, L - 1, L, block, top, 1, 2)
        assert torch.equal(eager[-1]["chosen"][s:s + 1].cpu(), want)
        o, _, tol, _ = B.attention(q, K, V, ok, L - 1, W ** -0.5, BF, want, block)
        assert ((eager[-1]["out"][s:s + 1].cpu().double() - o).abs() <= tol).all()
    # captured
    d2, c2, b2 = fresh()
    st = {n: torch.empty_like(t[0]) for n, t in (("q", qs), ("k", ks), ("v", vs))}
    kv_len, bufs2 = lens0.cuda(), buffers(c2, b2)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kv_len += 1
        layer(c2, b2, kv_len, st["q"], st["k"], st["v"], bufs2)
    for i in range(steps):
        st["q"].copy_(qs[i]); st["k"].copy_(ks[i]); st["v"].copy_(vs[i])
        graph.replay()
        torch.cuda.synchronize()
        for n in ("q", "chosen", "out"):
            assert torch.equal(bufs2[n], eager[i][n]), (i, n)
        _ = (qs[i].float() @ qs[i].float().transpose(-1, -2)).sum().item()
    assert torch.equal(b1.low_high, b2.low_high) and torch.equal(b1.steps, b2.steps)
    # the last four tokens of either sequence as one chain: the same choices (last covers the blocks that the chain fills)
    b = paged.Batch(dp, (lens0 + steps).cuda(), torch.tensor([0, 4, 8], dtype=torch.int32).cuda(), max_q=4, max_kv=1024)
    chain = buffers(c1, b1, 8)
    q4 = torch.stack([eager[i]["q"][s] for s in range(2) for i in range(steps - 4, steps)])
    paged.select(b1, b, q4, chain["chosen"], first=1, last=2, workspace=chain["w1"], stream=base._stream())
    assert torch.equal(chain["chosen"], torch.stack([eager[i]["chosen"][s] for s in range(2) for i in range(steps - 4, steps)]))


def test_two_calls_at_once():
    """Two selections and attentions on two streams over one cache, each with its workspaces: the bits of
    the calls one after the other."""
    g = base._gen(47)
    lens, page, top = [9000, 5000], 64, 40
    pages, n_pages = base.deal(g, lens, page)
    _, _, cache = make(g, n_pages, 2, page, 128, BF, "mx8")
    bd = new_bounds(n_pages, 2, page, 64, 128)
    whole, _ = base.batch_of(pages, lens, lens)
    paged.update_bounds(cache, whole, bd, stream=base._stream())
    b, _ = base.batch_of(pages, lens, [1, 1])
    q = [torch.randn(2, 8, 128, generator=g).to(BF).cuda() for _ in range(2)]
    out, ref = ([torch.zeros(2, 8, 128, dtype=BF, device="cuda") for _ in range(2)] for _ in range(2))
    chosen = [torch.zeros(2, 2, top, dtype=torch.int32, device="cuda") for _ in range(2)]
    w1 = [torch.empty(paged.select_workspace_bytes(bd, b, 2), dtype=torch.uint8, device="cuda") for _ in range(2)]
    n2 = paged.attend_blocks_workspace_bytes(cache, b, 8, top, 64, 2)
    assert n2 > 0
    w2 = [torch.empty(n2, dtype=torch.uint8, device="cuda") for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]

    def call(i, o, s):
        paged.select(bd, b, q[i], chosen[i], workspace=w1[i], stream=s)
        paged.attend_blocks(cache, b, q[i], chosen[i], o, block=64, scale=0.09, workspace=w2[i], stream=s)

    for i in range(2):
        call(i, ref[i], base._stream())
    torch.cuda.synchronize()
    for _ in range(5):
        for i in range(2):
            call(i, out[i], streams[i].cuda_stream)
    torch.cuda.synchronize()
    for i in range(2):
        assert torch.equal(out[i], ref[i])


def test_no_tokens():
    _, _, cache = make(base._gen(1), 3, 2, 16, 64, BF, "bf16")
    bd = new_bounds(3, 2, 16, 16, 64)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
    e = lambda h: torch.empty(0, h, 64, dtype=BF, device="cuda")
    c = torch.empty(0, 2, 4, dtype=torch.int32, device="cuda")
    for b in (paged.Batch(torch.zeros(2, 1, dtype=torch.int32, device="cuda"), i32(5, 0), i32(0, 0, 0), max_q=4, max_kv=16),
              paged.Batch(torch.zeros(0, 1, dtype=torch.int32, device="cuda"), i32(), i32(0), max_q=0, max_kv=0)):
        paged.update_bounds(cache, b, bd, stream=base._stream())
        paged.select(bd, b, e(4), c, stream=base._stream())
        paged.attend_blocks(cache, b, e(4), c, e(4), block=16, scale=0.1, stream=base._stream())
    torch.cuda.synchronize()
    assert (bd.low_high == 77).all()
