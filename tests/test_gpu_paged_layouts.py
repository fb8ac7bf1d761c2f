"""The paged operators over caches that are not dense: scale bytes at odd addresses, against the
plain float64 forms (paged_oracle.py) with the tolerances of test_gpu_paged."""
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
