"""The paged-cache operators (hearth_amd/paged.py) on the GPU against plain float64 forms
(paged_oracle.py): every type, head layout and page size, lengths around the kernels' steps,
masks that leave nothing, infinities and NaN in rows that are not attended, bad page ids,
padding, strides, and a run of the operators together, eager and as a replayed graph.

Tolerances count roundings (half a step of each type) and float32 sums; see
paged_oracle.attention and the comments at each test."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import paged_oracle as O
from hearth_amd import paged

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def _gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def _stream():
    return torch.cuda.current_stream().cuda_stream


def make_cache(g, n_pages, heads, page, width, kind, store, latent=False, fill=True):
    """CPU copies {k, ks, v, vs} of a cache, random rows of dtype `kind` stored as `store`"""
    out = {}
    for name in ("k",) if latent else ("k", "v"):
        x = torch.randn(n_pages, heads, page, width, generator=g)
        x[..., 3::37] *= 4
        x = (x if fill else torch.zeros_like(x)).to(kind)
        out[name], out[name + "s"] = O.mx8(x) if store == "mx8" else (x, None)
    return out


def on_gpu(c):
    d = {n: t if t is None else t.cuda() for n, t in c.items()}
    return d, paged.Cache(d["k"], d.get("v"), d["ks"], d.get("vs"))


def deal(g, lens, page, spare=2):
    """shuffled pages [S, per] and the number of pages"""
    used = [-(-L // page) for L in lens]
    n = sum(used) + spare
    order = torch.randperm(n, generator=g).int()
    pages = torch.full((len(lens), max(max(used), 1)), -1, dtype=torch.int32)
    at = 0
    for s, u in enumerate(used):
        pages[s, :u] = order[at:at + u]
        at += u
    return pages, n


def batch_of(pages, lens, news, mask=None, max_q=None, max_kv=None):
    starts = np.concatenate([[0], np.cumsum(news)]).astype(np.int32)
    return paged.Batch(pages.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), torch.from_numpy(starts).cuda(),
                       max_q=max(news) if max_q is None else max_q, max_kv=max(lens) if max_kv is None else max_kv,
                       mask=None if mask is None else mask.cuda()), starts


# ---------------------------------------------------------------- rotary positions

@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("T,H,W,rot,offset", [(1, 1, 64, 64, 0), (9, 32, 128, 128, 0), (5, 3, 192, 64, 128),
                                              (7, 2, 128, 96, 16), (3, 5, 130, 50, 7), (1100, 2, 64, 32, 8)])
def test_rope(dtype, layout, T, H, W, rot, offset):
    g = _gen(T * 31 + rot)
    x = torch.randn(T, H, W, generator=g).to(dtype)
    k = torch.randn(T, 2, W, generator=g).to(dtype)
    pos = torch.randint(0, 1000000, (T,), generator=g)
    freqs, factor = paged.rope_frequencies(rot, 1e6, "yarn", factor=16.0)
    f = torch.from_numpy(freqs)
    xd, kd = x.cuda(), k.cuda()
    out, kout = torch.full_like(xd, 7), torch.full_like(kd, 7)
    paged.rope(xd, pos.int().cuda(), f.cuda(), factor=factor, layout=layout, offset=offset, out=out, k=kd, k_out=kout,
               stream=_stream())
    paged.rope(xd, pos.cuda(), f.cuda(), factor=factor, layout=layout, offset=offset, stream=_stream())   # in place, int64
    assert torch.equal(out, xd)
    for got, src in ((out, x), (kout, k)):
        want, mag = O.rope(src.double(), pos, f, factor, layout, offset)
        # cosine and sine: the fraction of a turn rounded to float32 (pi 2^-24) and four steps of
        # the function; the factor and two products and a sum: 16 half steps of the magnitudes
        tol = O.HALF[dtype] * want.abs() + 16 * 2.0 ** -24 * mag + (2.0 ** -25 if dtype == HF else 0)
        assert ((got.cpu().double() - want).abs() <= tol).all()
        inside = torch.zeros(W, dtype=torch.bool)
        inside[offset:offset + rot] = True
        assert torch.equal(got.cpu()[..., ~inside], src[..., ~inside])


def test_rope_strided_and_inverse():
    """A slice of wider rows, heads before tokens, rows off 16 bytes; the inverse undoes it."""
    g = _gen(5)
    wide = torch.randn(6, 11, 200, generator=g)
    f = torch.from_numpy(paged.rope_frequencies(64)[0])
    pos = torch.arange(11) * 997
    for view in (lambda t: t[:, :, 101:165].transpose(0, 1), lambda t: t[:, :, 136:200].transpose(0, 1)):
        d = wide.cuda()
        paged.rope(view(d), pos.int().cuda(), f.cuda(), stream=_stream())
        want, mag = O.rope(view(wide).double(), pos, f, 1.0, "half", 0)
        assert ((view(d).cpu().double() - want).abs() <= 17 * 2.0 ** -24 * (mag + want.abs())).all()
        paged.rope(view(d), pos.int().cuda(), f.cuda(), inverse=True, stream=_stream())
        assert ((view(d).cpu() - view(wide)).abs() <= 64 * 2.0 ** -24 * (1 + mag)).all()
        keep = torch.ones_like(wide, dtype=torch.bool)
        view(keep).fill_(False)
        assert torch.equal(d.cpu()[keep], wide[keep])


# ---------------------------------------------------------------- writes and reads

@pytest.mark.parametrize("src", [BF, HF, F32])
@pytest.mark.parametrize("store", ["same", "mx8"])
@pytest.mark.parametrize("page,heads,width", [(16, 1, 32), (64, 4, 128), (32, 3, 96), (128, 2, 256)])
def test_append_and_read(src, store, page, heads, width):
    """Rows of ragged sequences: codes, scales and 16-bit rows equal to the plain form's, every
    other row of the cache untouched, and read back as the values they stand for."""
    kind = BF if src == F32 else src
    lens, news = [1, page, page + 1, 3 * page - 5, 40, 0, 7], [1, page, 3, 2 * page, 0, 0, 7]
    g = _gen(page + heads)
    pages, n_pages = deal(g, lens, page)
    c = make_cache(g, n_pages, heads, page, width, kind, store)
    d, cache = on_gpu(c)
    T = sum(news)
    new = {n: (torch.randn(T + 3, heads, width, generator=g) * torch.exp2(torch.randint(-20, 12, (T + 3, heads, 1), generator=g).float()))
           .to(src) for n in ("k", "v")}
    new["k"][0, 0, :32] = 0
    new["k"][1, 0, 5], new["v"][1, 0, 6], new["v"][2, 0, 7] = math.nan, math.inf, -math.inf
    big = {BF: 3.3895e38, HF: 65504.0, F32: 3.4028e38}[src]
    if T > 4:
        new["k"][4, 0, 3], new["k"][4, 0, 4] = big, -big
    b, starts = batch_of(pages, lens, news)
    paged.append(cache, b, new["k"].cuda(), new["v"].cuda(), stream=_stream())
    want = {n: (t.clone() if t is not None else None) for n, t in c.items()}
    for n in ("k", "v"):
        codes, sc = O.mx8(new[n]) if store == "mx8" else (new[n].to(kind), None)
        for s, (L, k) in enumerate(zip(lens, news)):
            for i in range(k):
                p, t = L - k + i, starts[s] + i
                if store == "mx8":
                    want[n].view(torch.uint8)[pages[s, p // page].item(), :, p % page] = codes.view(torch.uint8)[t]
                    want[n + "s"][pages[s, p // page].item(), :, p % page] = sc[t]
                else:
                    want[n][pages[s, p // page].item(), :, p % page] = codes[t]
    for n in ("k", "v"):
        if store == "mx8":
            assert torch.equal(d[n].cpu().view(torch.uint8), want[n].view(torch.uint8)), n
        else:                               # a converted NaN may have any payload
            nan = want[n].isnan()
            assert torch.equal(d[n].cpu().isnan(), nan), n
            assert torch.equal(d[n].cpu().view(torch.int16)[~nan], want[n].view(torch.int16)[~nan]), n
        if store == "mx8":
            assert torch.equal(d[n + "s"].cpu(), want[n + "s"]), n
    # whole sequences back
    whole, wstarts = batch_of(pages, lens, lens)
    back = {n: torch.full((sum(lens) + 2, heads, width), 5.0, dtype=src).cuda() for n in ("k", "v")}
    paged.read(cache, whole, back["k"], back["v"], stream=_stream())
    for n in ("k", "v"):
        for s, L in enumerate(lens):
            x, _ = O.rows_of(want[n], want.get(n + "s"), pages[s], L)
            exp = x.transpose(0, 1).to(src)
            got = back[n].cpu()[wstarts[s]:wstarts[s] + L]
            assert torch.equal(torch.nan_to_num(got, nan=12345.0), torch.nan_to_num(exp, nan=12345.0)), (n, s)
            assert torch.isfinite(got[torch.isfinite(x.transpose(0, 1))]).all()
        assert (back[n].cpu()[sum(lens):] == 5).all()


def test_append_bad_pages_negative_positions_and_limits():
    """Page ids outside the cache, more tokens than rows, tokens past max_q and rows past max_kv
    store nothing; reads of them give zeros."""
    g = _gen(3)
    page, heads, width = 16, 2, 64
    pages = torch.tensor([[0, 99, 2, -5], [1, 3, 4, 5]], dtype=torch.int32)
    c = make_cache(g, 6, heads, page, width, BF, "bf16")
    d, cache = on_gpu(c)
    lens, news = [60, 10], [60, 30]                 # sequence 1: twenty tokens before its first row
    k, v = (torch.randn(90, heads, width, generator=g).to(BF) for _ in range(2))
    b, starts = batch_of(pages, lens, news, max_q=45, max_kv=40)
    paged.append(cache, b, k.cuda(), v.cuda(), stream=_stream())
    want = c["k"].clone()
    for s, (L, n) in enumerate(zip(lens, news)):
        for i in range(min(n, 45)):
            p = L - n + i
            if 0 <= p < min(L, 40) and 0 <= pages[s, p // page] < 6:
                want[pages[s, p // page].item(), :, p % page] = k[starts[s] + i]
    assert torch.equal(d["k"].cpu().view(torch.int16), want.view(torch.int16))
    out = torch.full((90, heads, width), 3.0, dtype=BF).cuda()
    paged.read(cache, b, out, torch.empty_like(out), stream=_stream())
    exp = torch.full((90, heads, width), 3.0, dtype=BF)
    for s, (L, n) in enumerate(zip(lens, news)):
        for i in range(min(n, 45)):
            p = L - n + i
            ok = 0 <= p < min(L, 40) and 0 <= pages[s, p // page] < 6
            exp[starts[s] + i] = want[pages[s, p // page].item(), :, p % page] if ok else 0
    assert torch.equal(out.cpu(), exp)


@pytest.mark.parametrize("store", ["bf16", "mx8"])
def test_strided_cache_and_arrays(store):
    """Keys and values interleaved in one allocation, heads and pages of a larger one, and new
    rows cut out of a fused projection at odd elements."""
    g = _gen(9)
    page, heads, width, n_pages = 16, 2, 64, 5
    x = torch.randn(n_pages, 2, heads + 1, page, width, generator=g).to(BF)
    if store == "mx8":
        codes, sc = O.mx8(x)
        data, scd = codes.cuda(), sc.cuda()
        cache = paged.Cache(data[:, 0, :heads], data[:, 1, :heads], scd[:, 0, :heads], scd[:, 1, :heads])
    else:
        data = x.cuda()
        cache = paged.Cache(data[:, 0, :heads], data[:, 1, :heads])
    pages = torch.tensor([[4, 1], [0, 3]], dtype=torch.int32)
    b, starts = batch_of(pages, [20, 31], [20, 9])
    fused = torch.randn(29, heads * 3 * width + 3, generator=g).to(BF)
    part = lambda t, i: t[:, 1 + i * heads * width:1 + (i + 1) * heads * width].unflatten(1, (heads, width))
    fd = fused.cuda()
    paged.append(cache, b, part(fd, 1), part(fd, 2), stream=_stream())
    back = torch.zeros(29, heads * 3 * width + 3, dtype=BF, device="cuda")
    paged.read(cache, b, part(back, 1), part(back, 2), stream=_stream())
    for i in (1, 2):
        src = part(fused, i)
        exp = O.values(*O.mx8(src)).to(BF) if store == "mx8" else src
        assert torch.equal(part(back.cpu(), i), exp)
    rest = data.cpu()[:, :, heads]
    assert torch.equal(rest.view(torch.uint8), (O.mx8(x)[0] if store == "mx8" else x)[:, :, heads].contiguous().view(torch.uint8))


# ---------------------------------------------------------------- attention

def run_attend(g, kind, store, heads, kv_heads, width, lens, news, page, trees=None, latent=False, pages=None,
               n_pages=None, edit=None, pad=2, scale=None, max_kv=None, queries=None):
    """One call against the oracle; returns (out, lse) on the CPU"""
    if pages is None:
        pages, n_pages = deal(g, lens, page)
    W, DV = (576, 512) if latent else (width, width)
    c = make_cache(g, n_pages, kv_heads, page, W, kind, store, latent)
    if edit:
        edit(c, pages)
    d, cache = on_gpu(c)
    T = sum(news)
    q = torch.randn(T + pad, heads, W, generator=g).to(kind)
    if latent:
        q[..., :512] *= 0.35
    if queries:
        queries(q)
    scale = (192 ** -0.5 if latent else width ** -0.5) if scale is None else scale
    mask = O.words(trees, max(news)) if trees else None
    if mask is not None:
        mask = torch.cat([mask, torch.zeros(pad, mask.shape[1], dtype=torch.int64)])
    b, starts = batch_of(pages, lens, news, mask, max_kv=max_kv)
    out = torch.full((T + pad, heads, DV), 9.0, dtype=kind, device="cuda")
    lse = torch.full((T + pad, heads), 9.0, device="cuda")
    need = paged.workspace_bytes(cache, b, heads, T + pad)
    work = torch.full((need + 64,), 255, dtype=torch.uint8, device="cuda")    # NaN patterns
    qd = q.cuda()
    args = dict(scale=scale, lse=lse, workspace=work[:need], stream=_stream())
    if latent:
        paged.attend_latent(cache, b, qd[..., :512], qd[..., 512:], out, **args)
    else:
        paged.attend(cache, b, qd, out, **args)
    got, glse = out.cpu(), lse.cpu()
    assert (work[need:] == 255).all()
    assert (got[T:] == 9).all() and (glse[T:] == 9).all(), "padding rows were written"
    for s, (L, n) in enumerate(zip(lens, news)):
        K, ok = O.rows_of(c["k"], c["ks"], pages[s], L)
        V = K[..., :512] if latent else O.rows_of(c["v"], c["vs"], pages[s], L)[0]
        lo = starts[s]
        want, wl, tol, ltol = O.attention(q[lo:lo + n].double(), K, V, ok, L - n, scale, kind, trees[s] if trees else None)
        x, xl = got[lo:lo + n].double(), glse[lo:lo + n].double()
        fine = torch.isfinite(want)
        assert ((x - want).abs() <= tol)[fine].all(), (s, L, n, ((x - want).abs() / tol)[fine].max())
        assert torch.equal(torch.isnan(x), torch.isnan(want)) and torch.equal(x.isinf(), want.isinf()), s
        empty = wl == -math.inf
        assert (xl[empty] == -math.inf).all() and (x[empty] == 0).all()
        live = torch.isfinite(wl)
        assert ((xl - wl).abs() <= ltol)[live].all(), (s, (xl - wl).abs()[live].max())
    return got, glse


STORES = [(BF, "bf16"), (HF, "f16"), (BF, "mx8"), (HF, "mx8")]
LENS = [1, 2, 15, 16, 17, 31, 32, 33, 127, 128, 129, 300]


@pytest.mark.parametrize("kind,store", STORES)
@pytest.mark.parametrize("heads,kv_heads,width,page", [(8, 2, 64, 16), (32, 4, 128, 64), (4, 4, 256, 32), (7, 1, 128, 128)])
def test_attend_one_token(kind, store, heads, kv_heads, width, page):
    run_attend(_gen(heads + width), kind, store, heads, kv_heads, width, LENS, [1] * len(LENS), page)


@pytest.mark.parametrize("kind,store", STORES)
@pytest.mark.parametrize("heads,kv_heads,width", [(8, 2, 64), (16, 2, 128), (6, 2, 256), (128, 8, 64)])
def test_attend_several_tokens(kind, store, heads, kv_heads, width):
    lens = [9, 5, 40, 300, 131, 1, 700, 64]
    news = [9, 2, 17, 9, 40, 1, 33, 64]
    run_attend(_gen(heads * width), kind, store, heads, kv_heads, width, lens, news, 16)


@pytest.mark.parametrize("kind,store", STORES)
@pytest.mark.parametrize("width", [64, 128, 256])
def test_attend_prompts(kind, store, width):
    """Prompts from empty and behind a context, whole and odd numbers of steps."""
    run_attend(_gen(width), kind, store, 8, 2, width, [257, 130, 513], [257, 130, 100], 64)


@pytest.mark.parametrize("kind,store", [(BF, "bf16"), (HF, "mx8")])
def test_attend_long_split(kind, store):
    """Lengths that split: one long sequence, and a long one beside short ones."""
    run_attend(_gen(1), kind, store, 8, 1, 128, [20000], [1], 64)
    run_attend(_gen(2), kind, store, 8, 2, 64, [5000, 3, 0, 130], [3, 3, 0, 1], 256)


@pytest.mark.parametrize("kind,store", STORES)
@pytest.mark.parametrize("heads,kv_heads,width", [(8, 2, 64), (32, 4, 128)])
def test_attend_trees(kind, store, heads, kv_heads, width):
    trees = [O.tree(85), O.tree(7, 2), O.tree(1), O.tree(70, 1)]
    run_attend(_gen(width + 1), kind, store, heads, kv_heads, width, [85 + 50, 7, 33, 70 + 200], [85, 7, 1, 70], 32, trees)


@pytest.mark.parametrize("latent", [False, True])
def test_nothing_attended(latent):
    """Empty sequences, more tokens than rows, masks without a bit: zeros and -infinity."""
    g = _gen(11)
    dims = dict(heads=16, kv_heads=1, width=128, latent=latent)
    run_attend(g, BF, "bf16", lens=[0, 3, 40], news=[2, 10, 1], page=16, **dims)
    none = torch.zeros(4, 4, dtype=torch.bool)
    run_attend(g, HF, "mx8", lens=[4, 20], news=[4, 4], page=16, trees=[none, O.tree(4)], **dims)
    run_attend(g, BF, "mx8", lens=[0, 0], news=[1, 0], page=16, **dims)


@pytest.mark.parametrize("latent", [False, True])
@pytest.mark.parametrize("store", ["bf16", "mx8"])
@pytest.mark.parametrize("long", [0, 3000])
def test_nan_and_infinity_in_rows_not_attended(latent, store, long):
    """NaN and infinities in the rows behind a sequence's end, in a prompt's later rows and in
    tree siblings reach only the tokens that attend them."""
    page = 32
    lens, news = [long + 45, long + 20, 7], [40, 20, 1]
    trees = [O.tree(40), O.tree(20), O.tree(1)]

    def edit(c, pages):
        nan = 0x7f if store == "mx8" else None
        for n in ("k", "v"):
            if n not in c:
                continue
            for s, L in enumerate(lens):
                t, last = L % page, pages[s, (L - 1) // page].item()
                if t:
                    if nan:
                        c[n].view(torch.uint8)[last, :, t:] = nan
                    else:
                        c[n][last, :, t:] = math.nan
            p = long + 5 + 30                  # a token of sequence 0 that few others attend
            at = (pages[0, p // page].item(), slice(None), p % page)
            if n == "v" or latent:
                if nan:
                    c[n].view(torch.uint8)[at + (slice(0, 512, 5) if latent else slice(0, None, 5),)] = nan
                else:
                    c[n][at + (3,)] = math.inf
                    c[n][at + (4,)] = math.nan

    g = _gen(21 + long)
    dims = dict(heads=16, kv_heads=1 if latent else 4, width=64, latent=latent)
    run_attend(g, BF, store, lens=lens, news=news, page=page, trees=trees, edit=edit, **dims)
    run_attend(g, BF, store, lens=lens, news=news, page=page, edit=edit, **dims)


@pytest.mark.parametrize("latent", [False, True])
@pytest.mark.parametrize("heads", [4, 64])
def test_infinity_beside_a_missing_page(latent, heads):
    """A step that lacks a page and whose other rows everyone attends keeps their infinities."""
    pages = torch.tensor([[0, 77, 2, 3, 4, 5, 1, 6]], dtype=torch.int32)

    def edit(c, pages):
        c["k" if latent else "v"][2, :, 3, 7] = math.inf

    run_attend(_gen(14), BF, "bf16", heads, 1, 64, [128], [2], 16, pages=pages, n_pages=7, latent=latent, edit=edit)


@pytest.mark.parametrize("latent", [False, True])
def test_bad_pages_count_as_masked(latent):
    g = _gen(4)
    pages = torch.tensor([[0, 77, 2, 3], [1, 4, -1, 5], [88, 88, 88, 88]], dtype=torch.int32)
    run_attend(g, BF, "bf16", 16, 1, 64, [60, 64, 20], [3, 1, 2], 16, pages=pages, n_pages=6, latent=latent)
    run_attend(g, BF, "mx8", 16, 1, 64, [60, 64, 20], [3, 1, 2], 16, pages=pages, n_pages=6, latent=latent)


@pytest.mark.parametrize("kind,store", STORES)
@pytest.mark.parametrize("heads", [5, 16, 128])
def test_latent_tokens(kind, store, heads):
    run_attend(_gen(heads), kind, store, heads, 1, 0, [1, 16, 33, 65, 257, 130], [1, 1, 1, 1, 1, 1], 64, latent=True)
    run_attend(_gen(heads + 1), kind, store, heads, 1, 0, [9, 140, 70], [9, 9, 40], 16, latent=True)


@pytest.mark.parametrize("kind,store", STORES)
def test_latent_tree_and_split(kind, store):
    run_attend(_gen(6), kind, store, 16, 1, 0, [2000, 85], [5, 85], 64, [O.tree(5, 2), O.tree(85)], latent=True)


@pytest.mark.parametrize("latent", [False, True])
@pytest.mark.parametrize("heads", [8, 64])
@pytest.mark.parametrize("scale", [-0.3, 0.0, 40.0])
def test_attend_scales(scale, heads, latent):
    """A negative scale, none, and one that leaves a single row."""
    run_attend(_gen(8), BF, "bf16", heads, 1, 64, [50, 200], [3, 1], 16, scale=scale, latent=latent)


@pytest.mark.parametrize("kind,store", STORES)
@pytest.mark.parametrize("heads,latent", [(8, False), (64, False), (64, True)])
def test_scores_that_grow_along_the_rows(kind, store, heads, latent):
    """Each row's scores far above those of the rows before it, and far below: maxima that grow in
    every step, and a first maximum that stays."""
    def edit(c, pages):
        for s, up in ((0, True), (1, False)):
            for t in range(300):
                at = (pages[s, t // 16].item(), slice(None), t % 16)
                row = torch.zeros(c["k"].shape[1], c["k"].shape[-1])
                row[:, 64 if latent else 0] = (t if up else 300 - t) * 0.25
                row[:, 70 if latent else 5] = math.sin(t)
                row = row.to(kind)
                if store == "mx8":
                    codes, sc = O.mx8(row)
                    c["k"].view(torch.uint8)[at], c["ks"][at] = codes.view(torch.uint8), sc
                else:
                    c["k"][at] = row

    def queries(q):
        q.zero_()
        q[..., 64 if latent else 0] = 3.0
        q[..., 70 if latent else 5] = 1.0

    run_attend(_gen(61), kind, store, heads, 1, 64, [300, 300], [1, 2], 16, latent=latent, edit=edit, scale=1.0, queries=queries)


def test_attend_strided_unaligned():
    """q and out cut from wider rows, off 16 bytes and heads first: the same bits as dense ones."""
    g = _gen(13)
    lens, news, page = [100, 37], [5, 2], 16
    pages, n_pages = deal(g, lens, page)
    _, cache = on_gpu(make_cache(g, n_pages, 2, page, 64, BF, "mx8"))
    b, _ = batch_of(pages, lens, news)
    q = torch.randn(7, 8, 64, generator=g).to(BF).cuda()
    work = torch.empty(max(paged.workspace_bytes(cache, b, 8, 7), 16), dtype=torch.uint8, device="cuda")
    dense = torch.empty_like(q)
    paged.attend(cache, b, q, dense, scale=0.125, workspace=work, stream=_stream())
    for cut in (lambda: torch.zeros(7, 8, 131, dtype=BF, device="cuda")[..., 3:67],
                lambda: torch.zeros(8, 7, 64, dtype=BF, device="cuda").transpose(0, 1),
                lambda: torch.zeros(7, 16, 64, dtype=BF, device="cuda")[:, ::2]):
        q2, o2 = cut(), cut()
        q2.copy_(q)
        paged.attend(cache, b, q2, o2, scale=0.125, workspace=work, stream=_stream())
        assert torch.equal(o2, dense)


def test_other_stream_and_offsets_past_32_bits():
    """A cache of more than 4 GiB, its last pages used, on a side stream."""
    page, heads, width = 64, 2, 128
    n_pages = (9 << 29) // (heads * page * width * 2) + 2     # 4.5 GiB a tensor
    g = _gen(17)
    k = torch.empty(n_pages, heads, page, width, dtype=BF, device="cuda")
    v = torch.empty_like(k)
    side = torch.cuda.Stream()
    pages = torch.tensor([[n_pages - 1, 0, n_pages - 2]], dtype=torch.int32)
    L = 150
    b, _ = batch_of(pages, [L], [L])
    nk, nv, q = (torch.randn(L, heads * m, width, generator=g).to(BF) for m in (1, 1, 4))
    dk, dv, dq = nk.cuda(), nv.cuda(), q.cuda()
    cache = paged.Cache(k, v)
    out = torch.empty_like(dq)
    work = torch.empty(max(paged.workspace_bytes(cache, b, 8, L), 16), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        paged.append(cache, b, dk, dv, stream=side.cuda_stream)
        paged.attend(cache, b, dq, out, scale=width ** -0.5, workspace=work, stream=side.cuda_stream)
    side.synchronize()
    want, _, tol, _ = O.attention(q.double(), nk.double().transpose(0, 1), nv.double().transpose(0, 1),
                                  torch.ones(L, dtype=torch.bool), 0, width ** -0.5, BF)
    assert ((out.cpu().double() - want).abs() <= tol).all()


@pytest.mark.parametrize("store", ["bf16", "mx8"])
def test_decode_loop_together_eager_and_captured(store):
    """rope, append and attend as a program's layer calls them, token after token for two
    sequences; the same steps as one captured graph whose lengths live in device memory,
    replayed with eager work between the replays."""
    g = _gen(33)
    page, H, Hkv, W, steps = 16, 8, 2, 64, 20
    pages = torch.tensor([[3, 0, 6, 5], [1, 4, 2, 7]], dtype=torch.int32).cuda()
    freqs = torch.from_numpy(paged.rope_frequencies(W, 1e4)[0]).cuda()
    q_start = torch.arange(3, dtype=torch.int32).cuda()
    qs, ks, vs = (torch.randn(steps, 2, h, W, generator=g).to(BF).cuda() for h in (H, Hkv, Hkv))
    lens0 = torch.tensor([5, 30], dtype=torch.int32)

    def fresh():
        c = make_cache(_gen(34), 8, Hkv, page, W, BF, store)
        return on_gpu(c)

    def layer(cache, kv_len, q, k, v, q2, k2, out, work):
        b = paged.Batch(pages, kv_len, q_start, max_q=1, max_kv=64)
        paged.rope(q, kv_len, freqs, out=q2, k=k, k_out=k2, stream=_stream())
        paged.append(cache, b, k2, v, stream=_stream())
        paged.attend(cache, b, q2, out, scale=W ** -0.5, workspace=work, stream=_stream())

    d1, c1 = fresh()
    b = paged.Batch(pages, lens0.cuda(), q_start, max_q=1, max_kv=64)
    work = torch.empty(max(paged.workspace_bytes(c1, b, H), 16), dtype=torch.uint8, device="cuda")
    eager = []
    for i in range(steps):
        out, q2, k2 = torch.empty_like(qs[0]), torch.empty_like(qs[0]), torch.empty_like(ks[0])
        layer(c1, (lens0 + 1 + i).cuda(), qs[i], ks[i], vs[i], q2, k2, out, work)
        eager.append(out)
    # against the oracle: the last step over the cache as it stands
    i = steps - 1
    for s in range(2):
        L = int(lens0[s]) + steps
        K, ok = O.rows_of(d1["k"].cpu(), None if store != "mx8" else d1["ks"].cpu(), pages[s].cpu(), L)
        V, _ = O.rows_of(d1["v"].cpu(), None if store != "mx8" else d1["vs"].cpu(), pages[s].cpu(), L)
        rq, _ = O.rope(qs[i, s:s + 1].cpu().double(), torch.tensor([L]), freqs.cpu(), 1.0, "half", 0)
        want, _, tol, _ = O.attention(q2[s:s + 1].cpu().double(), K, V, ok, L - 1, W ** -0.5, BF)
        assert ((eager[-1][s:s + 1].cpu().double() - want).abs() <= tol).all()
        assert ((q2[s].cpu().double() - rq[0]).abs() <= 2.0 ** -8 * rq[0].abs() + 1e-4).all()
    d2, c2 = fresh()
    st = {n: torch.empty_like(t[0]) for n, t in (("q", qs), ("k", ks), ("v", vs))}
    kv_len = lens0.cuda()
    q2, k2, out = torch.empty_like(st["q"]), torch.empty_like(st["k"]), torch.empty_like(st["q"])
    work2 = torch.empty_like(work)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kv_len += 1
        layer(c2, kv_len, st["q"], st["k"], st["v"], q2, k2, out, work2)
    for i in range(steps):
        st["q"].copy_(qs[i]); st["k"].copy_(ks[i]); st["v"].copy_(vs[i])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager[i]), i
        _ = (qs[i].float() @ qs[i].float().transpose(-1, -2)).sum().item()
    assert torch.equal(d1["k"].cpu().view(torch.uint8), d2["k"].cpu().view(torch.uint8))


def test_calls_without_tokens():
    """Empty arrays (whose data may be no address at all) and batches without sequences."""
    g = _gen(41)
    d, cache = on_gpu(make_cache(g, 3, 2, 16, 64, BF, "bf16"))
    _, lat = on_gpu(make_cache(g, 3, 1, 16, 576, BF, "bf16", latent=True))
    before = d["k"].clone()
    e = lambda h, w: torch.empty(0, h, w, dtype=BF, device="cuda")
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
    freqs = torch.from_numpy(paged.rope_frequencies(64)[0]).cuda()
    for b in (paged.Batch(torch.zeros(2, 1, dtype=torch.int32, device="cuda"), i32(5, 0), i32(0, 0, 0), max_q=4, max_kv=16),
              paged.Batch(torch.zeros(0, 1, dtype=torch.int32, device="cuda"), i32(), i32(0), max_q=0, max_kv=0)):
        paged.rope(e(4, 64), i32(), freqs, k=e(2, 64), stream=_stream())
        paged.append(cache, b, e(2, 64), e(2, 64), stream=_stream())
        paged.read(cache, b, e(2, 64), e(2, 64), stream=_stream())
        paged.attend(cache, b, e(4, 64), e(4, 64), scale=0.1, stream=_stream())
        paged.append(lat, b, e(1, 512), e(1, 64), stream=_stream())
        paged.attend_latent(lat, b, e(4, 512), e(4, 64), e(4, 512), scale=0.1, stream=_stream())
    torch.cuda.synchronize()
    assert torch.equal(d["k"], before)


def test_rope_of_more_tokens_than_one_round():
    """2^22 + 5 tokens: the workgroups of one launch go round. One pair a token; bf16 results lie
    within half a step (2^-8) of the exact ones, plus 2^-21 of |u| + |v| for float32 sines, cosines and sums."""
    T = (1 << 22) + 5
    x = torch.randn(T, 1, 2, generator=_gen(43)).to(BF)
    pos = torch.arange(T, dtype=torch.int32)
    freqs = torch.tensor([0.37], dtype=torch.float64)
    got = x.cuda()
    paged.rope(got, pos.cuda(), freqs.cuda(), stream=_stream())
    want, size = O.rope(x.double(), pos, freqs, 1.0, "half", 0)
    assert ((got.cpu().double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -21 * size).all()


@pytest.mark.parametrize("store", ["bf16", "mx8"])
@pytest.mark.parametrize("heads,news,latent", [(8, 1, False), (64, 9, False), (16, 2, True)])
def test_split_calls_captured_and_replayed(store, heads, news, latent):
    """A split attention and its join (every kernel of rows), and a read of the cache, in one
    graph whose queries and lengths change between the replays; eager calls of the same
    workspace's size run between them. Each replay gives the eager call's bits."""
    g = _gen(heads + news)
    page, L = 64, 5000
    W, DV, kv_heads = (576, 512, 1) if latent else (128, 128, 4)
    pages, n_pages = deal(g, [L], page)
    _, cache = on_gpu(make_cache(g, n_pages, kv_heads, page, W, BF, store, latent))
    kv_len, q_start = torch.tensor([L], dtype=torch.int32).cuda(), torch.tensor([0, news], dtype=torch.int32).cuda()
    b = paged.Batch(pages.cuda(), kv_len, q_start, max_q=news, max_kv=L)
    need = paged.workspace_bytes(cache, b, heads, news)
    assert need > 0

    def call(q, out, lse, rows, work):
        kw = dict(scale=W ** -0.5, lse=lse, workspace=work, stream=_stream())
        if latent:
            paged.attend_latent(cache, b, q[..., :512], q[..., 512:], out, **kw)
            paged.read(cache, b, rows, stream=_stream())
        else:
            paged.attend(cache, b, q, out, **kw)
            paged.read(cache, b, rows, torch.empty_like(rows), stream=_stream())

    def buffers():
        return (torch.zeros(news, heads, DV, dtype=BF, device="cuda"), torch.zeros(news, heads, device="cuda"),
                torch.zeros(news, kv_heads, W, dtype=BF, device="cuda"), torch.zeros(need, dtype=torch.uint8, device="cuda"))

    q = torch.zeros(news, heads, W, dtype=BF, device="cuda")
    mine, other = buffers(), buffers()
    call(q, *other)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(q, *mine)
    for i in range(4):
        q.copy_(torch.randn(news, heads, W, generator=g).to(BF))
        kv_len.fill_(L - 700 * i)
        graph.replay()
        call(q, *other)
        torch.cuda.synchronize()
        for x, y in zip(mine[:3], other[:3]):
            assert torch.equal(x, y), i


@pytest.mark.parametrize("latent", [False, True])
def test_two_calls_at_once(latent):
    """Two split calls on two streams over one cache, each with its workspace, again and again:
    the bits of the calls one after the other."""
    g = _gen(47)
    lens, page = [3000, 1700], 32
    W, DV, heads, kv_heads = (576, 512, 16, 1) if latent else (128, 128, 16, 4)
    pages, n_pages = deal(g, lens, page)
    _, cache = on_gpu(make_cache(g, n_pages, kv_heads, page, W, BF, "mx8", latent))
    b, _ = batch_of(pages, lens, [1, 1])
    need = paged.workspace_bytes(cache, b, heads, 2)
    assert need > 0
    q = [torch.randn(2, heads, W, generator=g).to(BF).cuda() for _ in range(2)]
    out, ref = ([torch.zeros(2, heads, DV, dtype=BF, device="cuda") for _ in range(2)] for _ in range(2))
    work = [torch.empty(need, dtype=torch.uint8, device="cuda") for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]

    def call(i, o, s):
        kw = dict(scale=W ** -0.5, workspace=work[i], stream=s)
        if latent:
            paged.attend_latent(cache, b, q[i][..., :512], q[i][..., 512:], o, **kw)
        else:
            paged.attend(cache, b, q[i], o, **kw)

    for i in range(2):
        call(i, ref[i], _stream())
    torch.cuda.synchronize()
    for _ in range(5):
        for i in range(2):
            call(i, out[i], streams[i].cuda_stream)
    torch.cuda.synchronize()
    for i in range(2):
        assert torch.equal(out[i], ref[i])
