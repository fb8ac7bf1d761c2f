"""append_rotated on the GPU: the bits of rope and append one after the other, for every type, layout,
offset, stride and cache; keys against the float64 rotation; tokens that are not stored; positions
given and taken from the rows; a captured call."""
from __future__ import annotations

import pytest
import torch

import paged_oracle as O
import paged_oracle4 as P
import test_gpu_paged as base
from hearth_amd import paged

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def make_cache(n_pages, heads, page, width, store, latent=False):
    """zeroed device tensors {k, ks, v, vs} and the Cache"""
    d = {}
    kind = {"bf16": BF, "f16": HF}.get(store, torch.uint8)
    for n in ("k",) if latent else ("k", "v"):
        d[n] = torch.zeros(n_pages, heads, page, width // 2 if store == "mx4" else width, dtype=kind, device="cuda")
        d[n + "s"] = torch.zeros(n_pages, heads, page, width // 32, dtype=torch.uint8, device="cuda") if store.startswith("mx") else None
    view = lambda t: t.view({"mx4": torch.float4_e2m1fn_x2, "mx8": torch.float8_e4m3fn}.get(store, t.dtype))
    return d, paged.Cache(view(d["k"]), view(d["v"]) if not latent else None, d["ks"], d.get("vs"))


def same(a, b):
    return all((a[n] is None and b[n] is None) or torch.equal(a[n].view(torch.uint8), b[n].view(torch.uint8)) for n in a)


LENS, NEWS = [1, 40, 33, 3, 0, 70], [1, 9, 33, 5, 2, 0]      # one token, a chain, a prompt, more tokens than rows, no rows, no tokens


def both(store, src, layout, heads, kv_heads, width, rot, offset, pos, latent=False, cut=None, in_place=False, max_q=None, seed=0, q=True, lens=LENS, news=NEWS):
    """(arrays, q of the fused call, q of rope, caches of either)"""
    g = base._gen(seed + width + rot)
    page = 16
    pages, n_pages = base.deal(g, lens, page)
    T = sum(news) + 3
    rw = 64 if latent else width
    d1, c1 = make_cache(n_pages, kv_heads, page, 576 if latent else width, store, latent)
    d2, c2 = make_cache(n_pages, kv_heads, page, 576 if latent else width, store, latent)
    new = lambda *s: torch.randn(*s, generator=g).to(src).cuda()
    cut = cut or (lambda x: x.clone())
    qx, k, v = cut(new(T, heads, rw)), cut(new(T, kv_heads, 512 if latent else width)), cut(new(T, kv_heads, rw))
    b, starts = base.batch_of(pages, lens, news, max_q=max_q)
    freqs, factor = paged.rope_frequencies(rot, 1e6, "yarn", factor=16.0)
    f = torch.from_numpy(freqs).cuda()
    rows = torch.cat([torch.arange(L - n, L) for L, n in zip(lens, news)] + [torch.zeros(3, dtype=torch.int64)])
    at = {"rows": None, "int32": torch.randint(0, 1000000, (T,), generator=g).int().cuda(), "int64": torch.randint(0, 1 << 33, (T,), generator=g).cuda()}[pos]
    kw = dict(factor=factor, layout=layout, offset=offset, stream=base._stream())
    turned = v if latent else k
    before = [x.clone() for x in (k, v)]
    q1 = qx.clone() if in_place else torch.full_like(qx, 7)
    if q:
        paged.append_rotated(c1, b, q1 if in_place else qx, k, v, f, pos=at, q_out=None if in_place else q1, **kw)
    else:
        paged.append_rotated(c1, b, None, k, v, f, pos=at, **kw)
    assert torch.equal(k, before[0]) and torch.equal(v, before[1])
    q2, t2 = torch.empty(T, heads, rw, dtype=src, device="cuda"), torch.empty(turned.shape, dtype=src, device="cuda")
    paged.rope(qx, rows.cuda() if at is None else at, f, out=q2, k=turned, k_out=t2, **kw)
    paged.append(c2, b, *((k, t2) if latent else (t2, v)), stream=base._stream())
    assert same(d1, d2)
    done = torch.zeros(T, dtype=torch.bool)
    for s, n in enumerate(news):
        done[starts[s]:starts[s] + min(n, n if max_q is None else max_q)] = True
    if q:
        assert torch.equal(q1[done.cuda()], q2[done.cuda()])
        assert torch.equal(q1[~done.cuda()], qx[~done.cuda()]) if in_place else (q1[~done.cuda()] == 7).all()
    return d1, dict(k=k, v=v, f=f, factor=factor, pages=pages, lens=lens, news=news, starts=starts)


@pytest.mark.parametrize("src", [BF, HF, F32])
@pytest.mark.parametrize("store", ["bf16", "f16", "mx8", "mx4"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("heads,kv_heads,width,rot,offset", [(8, 2, 128, 128, 0), (7, 1, 64, 32, 0), (4, 4, 96, 96, 0), (3, 1, 256, 64, 192), (2, 2, 64, 16, 8), (4, 2, 32, 10, 3)])
def test_the_bits_of_both_calls(src, store, layout, heads, kv_heads, width, rot, offset):
    both(store, src, layout, heads, kv_heads, width, rot, offset, "rows")
    both(store, src, layout, heads, kv_heads, width, rot, offset, "int64", in_place=True)


@pytest.mark.parametrize("pos", ["rows", "int32", "int64"])
@pytest.mark.parametrize("store", ["bf16", "mx8", "mx4"])
def test_latent_rows(pos, store):
    both(store, BF, "interleaved", 16, 1, 576, 64, 0, pos, latent=True)


def test_strides_alignment_and_bounds():
    """Slices of wider rows, heads before tokens, rows off 16 bytes; tokens past max_q; keys alone; many short prompts."""
    for cut in (lambda t: torch.zeros(*t.shape[:2], t.shape[2] + 3, dtype=t.dtype, device="cuda")[..., 1:-2].copy_(t),
                lambda t: torch.zeros(t.shape[1], t.shape[0], t.shape[2], dtype=t.dtype, device="cuda").transpose(0, 1).copy_(t),
                lambda t: torch.zeros(t.shape[0], 2 * t.shape[1], t.shape[2], dtype=t.dtype, device="cuda")[:, ::2].copy_(t)):
        for src, store in ((BF, "bf16"), (HF, "mx4"), (F32, "mx8")):
            both(store, src, "half", 4, 2, 128, 64, 16, "int32", cut=cut)
    both("bf16", BF, "half", 8, 2, 128, 128, 0, "rows", max_q=7)
    both("mx8", BF, "half", 8, 2, 128, 128, 0, "rows", q=False)
    both("mx4", HF, "interleaved", 2, 1, 64, 64, 0, "rows", lens=[1100, 5], news=[1100, 2])       # several tokens a workgroup


@pytest.mark.parametrize("src", [BF, HF])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_keys_against_the_rotation(src, layout):
    """16-bit rows: half a step of the type, and 16 half steps of float32 for angle, sine, cosine, factor,
    products and sum (as in test_gpu_paged.test_rope)."""
    d, a = both("bf16" if src == BF else "f16", src, layout, 8, 2, 128, 96, 32, "rows")
    for s, (L, n) in enumerate(zip(a["lens"], a["news"])):
        lo = a["starts"][s]
        keep = [i for i in range(n) if L - n + i >= 0]
        if not keep:
            continue
        pos = torch.tensor([L - n + i for i in keep])
        want, mag = O.rope(a["k"].cpu()[lo:lo + n][keep].double(), pos, a["f"].cpu(), a["factor"], layout, 32)
        K = P.rows_of(d["k"].cpu(), None, a["pages"][s], L)[0].transpose(0, 1)
        tol = O.HALF[src] * want.abs() + 16 * 2.0 ** -24 * mag + (2.0 ** -25 if src == HF else 0)
        assert ((K[pos] - want).abs() <= tol).all()


def test_captured_and_replayed():
    """Lengths and positions change between the replays; each leaves the eager calls' bits."""
    g = base._gen(5)
    page, H, Hkv, W = 16, 8, 2, 64
    pages, n_pages = base.deal(g, [200, 90], page)
    pages = pages.cuda()
    f = torch.from_numpy(paged.rope_frequencies(W)[0]).cuda()
    kv_len, q_start = torch.tensor([5, 30], dtype=torch.int32).cuda(), torch.tensor([0, 2, 3], dtype=torch.int32).cuda()
    (d1, c1), (d2, c2) = make_cache(n_pages, Hkv, page, W, "mx4"), make_cache(n_pages, Hkv, page, W, "mx4")
    q, k, v = (torch.zeros(3, h, W, dtype=BF, device="cuda") for h in (H, Hkv, Hkv))
    o1, o2 = torch.zeros_like(q), torch.zeros_like(q)

    def call(c, o):
        b = paged.Batch(pages, kv_len, q_start, max_q=2, max_kv=200)
        paged.append_rotated(c, b, q, k, v, f, q_out=o, stream=base._stream())

    call(c2, o2)
    d2["k"].zero_(), d2["ks"].zero_(), d2["v"].zero_(), d2["vs"].zero_()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(c1, o1)
    for i in range(5):
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=g).to(BF))
        kv_len += 11
        graph.replay()
        call(c2, o2)
        torch.cuda.synchronize()
        assert torch.equal(o1, o2) and same(d1, d2), i
        _ = (q.float() @ q.float().transpose(-1, -2)).sum().item()


def test_no_tokens():
    d, c = make_cache(3, 2, 16, 64, "bf16")
    e = lambda h: torch.empty(0, h, 64, dtype=BF, device="cuda")
    f = torch.from_numpy(paged.rope_frequencies(64)[0]).cuda()
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
    for b in (paged.Batch(torch.zeros(2, 1, dtype=torch.int32, device="cuda"), i32(5, 0), i32(0, 0, 0), max_q=4, max_kv=16),
              paged.Batch(torch.zeros(0, 1, dtype=torch.int32, device="cuda"), i32(), i32(0), max_q=0, max_kv=0)):
        paged.append_rotated(c, b, e(4), e(2), e(2), f, pos=i32(), stream=base._stream())
    torch.cuda.synchronize()
    assert (d["k"] == 0).all()


@pytest.mark.parametrize("in_place", [False, True])
def test_queries_without_rows_and_of_no_sequence(in_place):
    """Queries of tokens whose rows have no page, lie past max_kv or before the first row are rotated; those of tokens past
    max_q and of no sequence (before and behind the sequences') are left alone."""
    g = base._gen(21)
    H, Hkv, W, T = 4, 2, 64, 40
    pages = torch.tensor([[0, 77, -1], [1, 2, 3], [4, 5, 6]], dtype=torch.int32).cuda()
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
    b = paged.Batch(pages, i32(48, 4, 40), i32(3, 15, 25, 36), max_q=10, max_kv=35)
    d, c = make_cache(7, Hkv, 16, W, "bf16")
    q, k, v = (torch.randn(T, h, W, generator=g).to(BF).cuda() for h in (H, Hkv, Hkv))
    f = torch.from_numpy(paged.rope_frequencies(W)[0]).cuda()
    rows = torch.zeros(T, dtype=torch.int64)
    done = torch.zeros(T, dtype=torch.bool)
    for lo, n, L in ((3, 12, 48), (15, 10, 4), (25, 11, 40)):
        rows[lo:lo + n] = torch.arange(L - n, L)
        done[lo:lo + min(n, 10)] = True
    want = torch.empty_like(q)
    paged.rope(q, rows.cuda(), f, out=want, stream=base._stream())
    old = q.clone() if in_place else torch.full_like(q, 5)
    out = q if in_place else old.clone()
    paged.append_rotated(c, b, q, k, v, f, q_out=None if in_place else out, stream=base._stream())
    torch.cuda.synchronize()
    assert torch.equal(out[done], want[done]) and torch.equal(out[~done], old[~done])
    # sequence 0 has no pages for rows 36 .. 45; of sequence 1 the last 4 of 10 tokens' rows exist; of sequence 2 rows 29 .. 34
    stored = torch.zeros(7, 16, dtype=torch.bool)
    stored[1, :4] = stored[5, 13:] = stored[6, :3] = True
    assert torch.equal(d["v"].cpu().ne(0).any(-1).any(1), stored) and torch.equal(d["k"].cpu().ne(0).any(-1).any(1), stored)
