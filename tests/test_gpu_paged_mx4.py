"""4-bit cache rows (mx4) on the GPU against the plain float64 forms (paged_oracle4.py, and
paged_oracle.attention with its tolerances over the rows' values): writes and reads of every type,
attention of few and many query rows at every width, masks that leave nothing, NaN blocks in rows
that are not attended, bad pages, splits, odd addresses and a cache past 32-bit offsets."""
from __future__ import annotations

import math

import pytest
import torch

import paged_oracle as O
import paged_oracle4 as P
import test_gpu_paged as base
from hearth_amd import paged

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def make_cache(g, n_pages, heads, page, width, kind, store, latent=False, fill=True):
    out = {}
    for name in ("k",) if latent else ("k", "v"):
        x = torch.randn(n_pages, heads, page, width, generator=g)
        x[..., 3::37] *= 4
        x = (x if fill else torch.zeros_like(x)).to(kind)
        out[name], out[name + "s"] = P.mx4(x)
    return out


def on_gpu(c):
    d = {n: t.cuda() for n, t in c.items()}
    p = lambda n: d[n].view(torch.float4_e2m1fn_x2) if n in d else None
    return d, paged.Cache(p("k"), p("v"), d["ks"], d.get("vs"))


@pytest.fixture(autouse=True)
def packed(monkeypatch):
    monkeypatch.setattr(base, "make_cache", make_cache)
    monkeypatch.setattr(base, "on_gpu", on_gpu)
    monkeypatch.setattr(base, "O", P.Plain)


def attend(seed, kind, *args, **kw):
    return base.run_attend(base._gen(seed), kind, "mx4", *args, **kw)


# ---------------------------------------------------------------- writes and reads

@pytest.mark.parametrize("src", [BF, HF, F32])
@pytest.mark.parametrize("page,heads,width,latent", [(16, 1, 32, False), (64, 4, 128, False), (32, 3, 96, False), (128, 2, 256, False), (16, 1, 576, True)])
def test_append_and_read(src, page, heads, width, latent):
    """Codes and scales equal to the plain form's, every other row of the cache untouched; whole
    sequences read back as the values they stand for, blocks with a NaN or an infinity as NaN."""
    lens, news = [1, page, page + 1, 3 * page - 5, 40, 0, 7], [1, page, 3, 2 * page, 0, 0, 7]
    g = base._gen(page + heads)
    pages, n_pages = base.deal(g, lens, page)
    c = make_cache(g, n_pages, heads, page, width, BF, "mx4", latent)
    d, cache = on_gpu(c)
    T = sum(news)
    new = {n: (torch.randn(T + 3, heads, width, generator=g) * torch.exp2(torch.randint(-13, 11, (T + 3, heads, 1), generator=g).float())).to(src)
           for n in (("k",) if latent else ("k", "v"))}
    big = {BF: 3.3895e38, HF: 65504.0, F32: 3.4028e38}[src]
    for x in new.values():
        x[0, 0, :32] = 0
        x[1, 0, 5], x[2, 0, 6], x[3, 0, 7] = math.nan, math.inf, -math.inf
        x[4, 0, 3], x[4, 0, 4] = big, -big
        x[5, 0, :9] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0])
        x[6, 0, :32] = torch.finfo(src).smallest_normal * torch.linspace(-2, 2, 32)
    b, starts = base.batch_of(pages, lens, news)
    halves = (lambda x: (x[..., :512], x[..., 512:])) if latent else None
    args = [t.cuda() for t in (halves(new["k"]) if latent else new.values())]
    paged.append(cache, b, *args, stream=base._stream())
    want = {n: t.clone() for n, t in c.items()}
    for n, x in new.items():
        codes, sc = P.mx4(x)
        for s, (L, k) in enumerate(zip(lens, news)):
            for i in range(k):
                p, t = L - k + i, starts[s] + i
                want[n][pages[s, p // page].item(), :, p % page] = codes[t]
                want[n + "s"][pages[s, p // page].item(), :, p % page] = sc[t]
    for n in want:
        assert torch.equal(d[n].cpu(), want[n]), n
    whole, ws = base.batch_of(pages, lens, lens)
    back = {n: torch.full((sum(lens) + 2, heads, width), 5.0, dtype=src, device="cuda") for n in new}
    paged.read(cache, whole, *(halves(back["k"]) if latent else back.values()), stream=base._stream())
    for n in new:
        for s, L in enumerate(lens):
            exp = P.rows_of(want[n], want[n + "s"], pages[s], L)[0].transpose(0, 1).to(src)
            got = back[n].cpu()[ws[s]:ws[s] + L]
            assert torch.equal(torch.nan_to_num(got.double(), nan=12345.0), torch.nan_to_num(exp.double(), nan=12345.0)), (n, s)
        assert (back[n].cpu()[sum(lens):] == 5).all()


def test_rows_off_16_bytes_and_strided_pages():
    """Arrays whose rows start off 16 bytes, in a cache cut out of a wider one."""
    g = base._gen(7)
    lens, news, page, heads, width = [50, 17], [20, 9], 16, 2, 64
    pages, n_pages = base.deal(g, lens, page)
    data, sc = torch.zeros(n_pages, heads + 1, page, width // 2, dtype=torch.uint8, device="cuda"), torch.zeros(n_pages, heads + 1, page, width // 32, dtype=torch.uint8, device="cuda")
    part = data.view(torch.float4_e2m1fn_x2)[:, :heads], data.view(torch.float4_e2m1fn_x2)[:, :heads], sc[:, :heads], sc[:, :heads]
    cache = paged.Cache(*part)
    x = torch.randn(29, heads, width + 3, generator=g).to(BF)
    b, starts = base.batch_of(pages, lens, news)
    xd = x.cuda()[..., 1:width + 1]
    paged.append(cache, b, xd, xd, stream=base._stream())
    back = torch.zeros(29, heads, width + 3, dtype=BF, device="cuda")
    paged.read(cache, b, back[..., 2:width + 2], torch.empty(29, heads, width, dtype=BF, device="cuda"), stream=base._stream())
    assert torch.equal(back[..., 2:width + 2].cpu(), P.values(*P.mx4(x[..., 1:width + 1])).to(BF))
    assert (back[..., :2] == 0).all() and (back[..., width + 2:] == 0).all() and (data[:, heads] == 0).all() and (sc[:, heads] == 0).all()


# ---------------------------------------------------------------- attention

@pytest.mark.parametrize("kind", [BF, HF])
@pytest.mark.parametrize("heads,kv_heads,width,page", [(8, 2, 64, 16), (32, 4, 128, 64), (4, 4, 256, 32), (7, 1, 128, 128), (2, 1, 64, 4096)])
def test_one_token(kind, heads, kv_heads, width, page):
    attend(heads + width, kind, heads, kv_heads, width, base.LENS, [1] * len(base.LENS), page)


@pytest.mark.parametrize("kind", [BF, HF])
@pytest.mark.parametrize("heads,kv_heads,width", [(8, 2, 64), (16, 2, 128), (6, 2, 256), (128, 8, 64)])
def test_several_tokens(kind, heads, kv_heads, width):
    attend(heads * width, kind, heads, kv_heads, width, [9, 5, 40, 300, 131, 1, 700, 64], [9, 2, 17, 9, 40, 1, 33, 64], 16)


@pytest.mark.parametrize("kind", [BF, HF])
@pytest.mark.parametrize("width", [64, 128, 256])
def test_prompts(kind, width):
    attend(width, kind, 8, 2, width, [257, 130, 513], [257, 130, 100], 64)


@pytest.mark.parametrize("kind", [BF, HF])
def test_long_split(kind):
    attend(1, kind, 8, 1, 128, [20000], [1], 64)
    attend(2, kind, 8, 2, 64, [5000, 3, 0, 130], [3, 3, 0, 1], 256)
    attend(3, kind, 4, 1, 256, [2100], [1], 64)
    attend(4, kind, 32, 2, 128, [2500, 40], [30, 9], 32)


@pytest.mark.parametrize("kind", [BF, HF])
@pytest.mark.parametrize("heads,kv_heads,width", [(8, 2, 64), (32, 4, 128), (4, 2, 256)])
def test_trees(kind, heads, kv_heads, width):
    attend(width + 1, kind, heads, kv_heads, width, [85 + 50, 7, 33, 70 + 200], [85, 7, 1, 70], 32, [O.tree(85), O.tree(7, 2), O.tree(1), O.tree(70, 1)])
    attend(width + 2, kind, heads, kv_heads, width, [9, 4], [4, 4], 16, [O.tree(4, 2), torch.zeros(4, 4, dtype=torch.bool)])


@pytest.mark.parametrize("kind", [BF, HF])
@pytest.mark.parametrize("heads,kv_heads,width,n", [(4, 4, 64, 96), (4, 4, 64, 97), (6, 2, 128, 32), (6, 2, 128, 33), (2, 2, 256, 70), (32, 4, 128, 12), (32, 4, 128, 13)])
def test_columns_of_both_kernels(kind, heads, kv_heads, width, n):
    """Up to 96 query rows of a kv head and above: causal, trees of more than a word, splits."""
    lens, news = [n, 3000, n + 130, 5], [n, n, 40 if n > 40 else n, 2]
    for trees in (None, [O.tree(k) for k in news]):
        attend(heads + width + n, kind, heads, kv_heads, width, lens, news, 64, trees)


def test_nothing_attended():
    attend(11, BF, 16, 1, 128, [0, 3, 40], [2, 10, 1], 16)
    attend(12, HF, 16, 1, 128, [4, 20], [4, 4], 16, [torch.zeros(4, 4, dtype=torch.bool), O.tree(4)])
    attend(13, BF, 16, 1, 128, [0, 0], [1, 0], 16)


@pytest.mark.parametrize("width", [64, 128, 256])
@pytest.mark.parametrize("heads", [4, 32])
@pytest.mark.parametrize("long", [0, 3000])
def test_nan_blocks_in_rows_not_attended(width, heads, long):
    """Blocks of NaN behind a sequence's end, in a prompt's later rows and in tree siblings reach only
    the tokens that attend them."""
    page, n = 32, 7 if heads == 4 else 40
    lens, news = [long + n + 5, long + 20, 7], [n, min(n, 20), 1]

    def edit(c, pages):
        for x in ("ks", "vs"):
            for s, L in enumerate(lens):
                if L % page:
                    c[x][pages[s, (L - 1) // page].item(), :, L % page:] = 255
        p = long + 5 + n - 2                         # a token of sequence 0 that few others attend
        c["vs"][pages[0, p // page].item(), :, p % page, -1] = 255

    for trees in ([O.tree(k) for k in news], None):
        attend(21 + long, BF, heads, 4, width, lens, news, page, trees=trees, edit=edit)


def test_bad_pages_count_as_masked():
    pages = torch.tensor([[0, 77, 2, 3], [1, 4, -1, 5], [88, 88, 88, 88]], dtype=torch.int32)
    for heads in (16, 48):
        attend(4, BF, heads, 1, 64, [60, 64, 20], [3, 1, 2], 16, pages=pages, n_pages=6)


def test_scales_at_any_address():
    """Scale bytes that start at an odd address: the same bits as aligned ones."""
    for width in (64, 128, 256):
        g = base._gen(width)
        c = make_cache(g, 9, 2, 16, width, BF, "mx4")
        d, cache = on_gpu(c)
        off = {}
        for n in ("ks", "vs"):
            flat = torch.zeros(d[n].numel() + 1, dtype=torch.uint8, device="cuda")
            off[n] = flat[1:].view(d[n].shape)
            off[n].copy_(d[n])
        p = lambda n: d[n].view(torch.float4_e2m1fn_x2)
        other = paged.Cache(p("k"), p("v"), off["ks"], off["vs"])
        for heads, news in ((4, 1), (16, 9)):
            b, _ = base.batch_of(torch.arange(9, dtype=torch.int32)[None], [140], [news])
            q = torch.randn(news, heads, width, generator=g).to(BF).cuda()
            out = [torch.zeros_like(q) for _ in range(2)]
            for cc, o in zip((cache, other), out):
                paged.attend(cc, b, q, o, scale=0.1, stream=base._stream())
            assert torch.equal(*out) and out[0].isfinite().all()


def test_offsets_past_32_bits():
    """A cache of more than 4 GiB a tensor, its last pages used, on a side stream."""
    page, heads, width, L = 64, 2, 128, 150
    n_pages = (9 << 29) // (heads * page * width // 2) + 2
    k = torch.empty(n_pages, heads, page, width // 2, dtype=torch.uint8, device="cuda").view(torch.float4_e2m1fn_x2)
    sc = torch.empty(n_pages, heads, page, width // 32, dtype=torch.uint8, device="cuda")
    cache = paged.Cache(k, k, sc, sc)                # values are the keys
    g = base._gen(17)
    b, _ = base.batch_of(torch.tensor([[n_pages - 1, 0, n_pages - 2]], dtype=torch.int32), [L], [L])
    x, q = torch.randn(L, heads, width, generator=g).to(BF), torch.randn(L, heads * 4, width, generator=g).to(BF)
    xd, qd = x.cuda(), q.cuda()
    out, work = torch.empty_like(qd), torch.empty(max(paged.workspace_bytes(cache, b, 8, L), 16), dtype=torch.uint8, device="cuda")
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        paged.append(cache, b, xd, xd, stream=side.cuda_stream)
        paged.attend(cache, b, qd, out, scale=width ** -0.5, workspace=work, stream=side.cuda_stream)
    side.synchronize()
    rows = P.values(*P.mx4(x)).transpose(0, 1)
    want, _, tol, _ = O.attention(q.double(), rows, rows, torch.ones(L, dtype=torch.bool), 0, width ** -0.5, BF)
    assert ((out.cpu().double() - want).abs() <= tol).all()
