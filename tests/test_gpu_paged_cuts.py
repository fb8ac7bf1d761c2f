"""Attention whose max_q and max_kv are below the counts and lengths in device memory: tokens past
max_q are left as they are, rows past max_kv are no part of any result; whole and split, against the
plain float64 form."""
from __future__ import annotations

import pytest
import torch

import paged_oracle as O
import test_gpu_paged as base

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


@pytest.mark.parametrize("kind,store", [(BF, "bf16"), (HF, "mx8")])
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("heads,kv_heads,width", [(8, 2, 64), (64, 2, 128), (16, 1, 0)], ids=["few", "many", "latent"])
@pytest.mark.parametrize("max_q,max_kv,lens", [(3, 90, [100, 95, 89, 300, 5]), (5, 2000, [2300, 2003, 2000, 40, 3]), (1, 4000, [4001, 4003, 17, 1, 9])])
def test_bounds_of_the_host(monkeypatch, kind, store, tree, heads, kv_heads, width, max_q, max_kv, lens):
    news = [6, 7, 2, 1, 5]
    trees = [O.tree(n, 2) for n in news] if tree else None
    make = base.batch_of
    monkeypatch.setattr(base, "batch_of", lambda pages, lens, news, mask=None, **kw: make(pages, lens, news, mask, max_q=max_q, max_kv=max_kv))

    def attention(q, K, V, exists, at, scale, kind, seen=None):
        want, lse, tol, ltol = O.attention(q, K, V, exists & (torch.arange(K.shape[1]) < max_kv), at, scale, kind, seen)
        want[max_q:], lse[max_q:], tol[max_q:], ltol[max_q:] = 9.0, 9.0, 0.0, 0.0      # what lay there
        return want, lse, tol, ltol

    class Plain:
        rows_of, words, mx8 = O.rows_of, O.words, O.mx8

    Plain.attention = staticmethod(attention)
    monkeypatch.setattr(base, "O", Plain)
    base.run_attend(base._gen(heads + max_kv), kind, store, heads, kv_heads, width, lens, news, 32, trees, latent=not width)
