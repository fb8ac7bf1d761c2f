"""The paged operators over caches that are not dense: scale bytes at odd addresses, strides of every
kind, offsets past 32 bits; against the plain float64 forms (paged_oracle.py) with the tolerances of
test_gpu_paged."""
from __future__ import annotations

import pytest
import torch

import test_gpu_paged as base
from hearth_amd import paged

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16
# heads, kv heads, width, lengths, new tokens, rows a page, latent: few query rows (up to 32 columns),
# many, latent rows
FEW, MANY, LATENT = ([300, 40, 17], [2, 1, 2]), ([300, 40, 130], [130, 40, 9]), ([130, 40, 17], [9, 1, 1])
CALLS = [(8, 2, 64, *FEW, 16), (8, 2, 128, *FEW, 32), (4, 2, 256, *FEW, 16), (8, 2, 64, *MANY, 32), (8, 2, 128, *MANY, 16),
         (4, 2, 256, *MANY, 16), (16, 1, 0, *LATENT, 16)]
IDS = ["few-64", "few-128", "few-256", "many-64", "many-128", "many-256", "latent"]


def put(t, page_stride, head_stride, first=0):
    """a copy of t [pages, heads, rows, width] on the GPU with these strides (elements), everything
    around it (of allocations that are not huge) ones: NaN as numbers and codes, 2^128 as scales"""
    P, H, R, W = t.shape
    n = first + (P - 1) * page_stride + (H - 1) * head_stride + R * W
    flat = torch.empty(n, dtype=t.dtype, device="cuda").view(torch.uint8)
    if flat.numel() < 1 << 26:
        flat.fill_(255)
    v = flat.view(t.dtype if t.element_size() > 1 else torch.uint8).as_strided(t.shape, (page_stride, head_stride, W, 1), first)
    v.copy_(t.view(v.dtype))
    return v.view(t.dtype)


def call(monkeypatch, place, kind, store, heads, kv_heads, width, lens, news, page):
    def on_gpu(c):
        d = {n: t if t is None else place(n, t) for n, t in c.items()}
        return d, paged.Cache(d["k"], d.get("v"), d["ks"], d.get("vs"))

    monkeypatch.setattr(base, "on_gpu", on_gpu)
    base.run_attend(base._gen(heads + width), kind, store, heads, kv_heads, width, lens, news, page, latent=not width)


@pytest.mark.parametrize("kind", [BF, HF])
@pytest.mark.parametrize("shape", CALLS, ids=IDS)
def test_scales_at_odd_addresses(monkeypatch, shape, kind):
    """Scale tensors cut one byte into a larger allocation, an odd number of bytes a page."""
    def place(name, t):
        block = t.shape[2] * t.shape[3]
        return put(t, t.shape[1] * block + 1, block, 1) if name.endswith("s") else t.cuda()

    call(monkeypatch, place, kind, "mx8", *shape)


@pytest.mark.parametrize("kind,store", [(BF, "bf16"), (HF, "f16"), (BF, "mx8"), (HF, "mx8")])
@pytest.mark.parametrize("layout", ["gaps", "heads first"])
@pytest.mark.parametrize("shape", CALLS, ids=IDS)
def test_strides(monkeypatch, shape, layout, kind, store):
    """Pages and heads cut out of a larger allocation, and heads before pages: rows and scale bytes
    each with strides of their own, what lies between NaN."""
    seen = []

    def place(name, t):
        P, H, R, W = t.shape
        block, gap = R * W, 16 * (1 + len(seen))                            # another stride for each tensor
        seen.append(name)
        if layout == "gaps":
            return put(t, H * (block + gap) + 3 * gap, block + gap, 2 * gap)
        return put(t, block + gap, P * (block + gap) + gap, gap)

    call(monkeypatch, place, kind, store, *shape)
    assert len(seen) == (1 if not shape[2] else 2) * (2 if store == "mx8" else 1)


@pytest.mark.parametrize("kind,store", [(BF, "bf16"), (BF, "mx8")])
@pytest.mark.parametrize("far,shape", [("pages", s) for s in CALLS] + [("heads", s) for s in CALLS if s[2]],   # latent rows: one head
                         ids=["pages-" + i for i in IDS] + ["heads-" + i for i in IDS[:-1]])
def test_offsets_past_32_bits(monkeypatch, shape, far, kind, store):
    """Pages, or heads, that lie more than 2^32 bytes apart: rows and scale bytes alike."""
    def place(name, t):
        P, H, R, W = t.shape
        block, es = R * W, t.element_size()
        if far == "heads":
            return put(t, block, (1 << 32) // es + 64)
        return put(t, -(-(1 << 33) // (es * (P - 1)) // 16) * 16, block)    # the last page 2^33 bytes behind the first

    try:
        call(monkeypatch, place, kind, store, *shape)
    finally:
        torch.cuda.empty_cache()


@pytest.mark.parametrize("heads,width", [(1, 64), (40, 64), (3, 0)], ids=["few", "many", "latent"])
def test_the_most_sequences(heads, width):
    """65535 sequences of one row, which is the token's own: its attention is that row's values, to the bit."""
    S, W, page = 65535, width or 576, 16
    g = torch.Generator(device="cuda")
    g.manual_seed(heads)
    k = torch.zeros(S, 1, page, W, dtype=BF, device="cuda")
    cache = paged.Cache(k, torch.zeros_like(k) if width else None)
    pages = torch.randperm(S, generator=g, device="cuda").int().view(S, 1)
    batch = paged.Batch(pages, torch.ones(S, dtype=torch.int32, device="cuda"), torch.arange(S + 1, dtype=torch.int32, device="cuda"),
                        max_q=1, max_kv=1)
    rows = torch.randn(S, 2, W, generator=g, device="cuda").to(BF)
    new = (rows[:, :1], rows[:, 1:]) if width else (rows[:, :1, :512], rows[:, :1, 512:])
    s = torch.cuda.current_stream().cuda_stream
    paged.append(cache, batch, *new, stream=s)
    back = torch.zeros_like(rows)
    paged.read(cache, batch, *((back[:, :1], back[:, 1:]) if width else (back[:, :1, :512], back[:, :1, 512:])), stream=s)
    q = torch.randn(S, heads, W, generator=g, device="cuda").to(BF)
    out = torch.zeros(S, heads, width or 512, dtype=BF, device="cuda")
    assert paged.workspace_bytes(cache, batch, heads) == 0
    if width:
        paged.attend(cache, batch, q, out, scale=0.1, stream=s)
    else:
        paged.attend_latent(cache, batch, q[..., :512], q[..., 512:], out, scale=0.1, stream=s)
    torch.cuda.synchronize()
    assert torch.equal(back[:, :1], rows[:, :1]) and (not width or torch.equal(back, rows))
    assert torch.equal(out, (new[1] if width else new[0]).expand_as(out))
