"""Scores that are -infinity, against the plain float64 form: exp(-infinity) is 0, so such a row is no
part of a result that has other rows, and a token all of whose rows are such has 0 / 0, which is
NaN, where one that attends no row at all gets zeros; the logarithm of the sum is -infinity for both."""
from __future__ import annotations

import math

import pytest
import torch

import paged_oracle as O
import test_gpu_paged as base

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


@pytest.mark.parametrize("kind,store", [(BF, "bf16"), (HF, "f16")])
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("heads,kv_heads,width,news,long", [
    (8, 2, 64, 4, 200), (8, 2, 128, 4, 3000), (4, 1, 128, 4, 20000), (4, 2, 256, 3, 700),       # few query rows; in one piece, split
    (32, 2, 64, 5, 200), (32, 2, 128, 9, 2500), (16, 1, 256, 5, 700),                           # many
    (16, 1, 0, 3, 120), (16, 1, 0, 4, 700), (5, 1, 0, 2, 5000)])                                # latent rows
def test_scores_of_minus_infinity(monkeypatch, kind, store, heads, kv_heads, width, news, long, tree):
    page, e = 32, 520 if not width else 9
    # every row; all but the last ones; every second; none; no rows; more tokens than rows
    lens = [long, long, long // 2 + 3, 77, 0, 2]
    low = [lambda t: t >= 0, lambda t: t < long - news - 20, lambda t: t % 2 == 0, lambda t: t < 0, lambda t: t < 0, lambda t: t >= 0]

    def edit(c, pages):
        for s, L in enumerate(lens):
            t = torch.arange(L)
            t = t[low[s](t)]
            c["k"][pages[s].long()[t // page], :, t % page, e] = -math.inf

    def queries(q):
        q[..., e] = 1.0

    undefined = []

    def attention(q, K, V, exists, at, scale, kind, seen=None):
        gone = torch.isinf(K[..., e]).all(0)
        K = torch.where(torch.isinf(K), 0.0, K)
        want, lse, tol, ltol = O.attention(q, K, V, exists & ~gone, at, scale, kind, seen)
        some = O.attention(q, K, V, exists, at, scale, kind, seen)[1] > -math.inf
        nan = (lse == -math.inf) & some
        undefined.append(nan)
        return torch.where(nan[..., None], math.nan, want), torch.where(nan, math.nan, lse), tol, ltol

    class Plain:
        rows_of, words, mx8 = O.rows_of, O.words, O.mx8

    Plain.attention = staticmethod(attention)
    monkeypatch.setattr(base, "O", Plain)
    trees = [O.tree(news, 2) for _ in lens] if tree else None
    if tree:
        trees[3] = torch.zeros(news, news, dtype=torch.bool)
    got, lse = base.run_attend(base._gen(heads + long), kind, store, heads, kv_heads, width, lens, [news] * len(lens), page, trees,
                               latent=not width, edit=edit, queries=queries)
    nan = torch.cat(undefined)
    assert nan[:news].all() and not nan[news:4 * news].any() and nan[5 * news:].any()
    assert (lse[:len(nan)][nan] == -math.inf).all()
