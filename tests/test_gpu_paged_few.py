"""Paths of the paged attention that only few query rows, or only many splits, take, against the
plain float64 form (paged_oracle.py) with the tolerances of test_gpu_paged: the kernel of few
query rows under masks, and the join of more than 16 splits at every width."""
from __future__ import annotations

import math
import re
from pathlib import Path

import pytest
import torch

import paged_oracle as O
import test_gpu_paged as base
from hearth_amd import paged

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16
STORES = [(BF, "bf16"), (HF, "f16"), (BF, "mx8"), (HF, "mx8")]
SOURCE = (Path(paged.__file__).parent / "csrc" / "k_paged_attn.hip").read_text()
COLUMNS = int(re.search(r"takes_many\(int64_t cols\) \{ return cols > (\d+); \}", SOURCE).group(1))
MANY_SPLITS = int(re.search(r"JOIN_MANY = (\d+);", SOURCE).group(1))


def attend(g, kind, store, heads, kv_heads, width, lens, news, page, trees=None, splits=None, **kw):
    """base.run_attend, and a look at which kernels the call takes: splits is "one", "some" (joined by
    a group of threads) or "many" (by several), or None"""
    latent = not width
    assert latent or max(news) * (heads // kv_heads) <= COLUMNS, "another kernel than that of few query rows"
    need = []
    real = paged.workspace_bytes

    def count(cache, batch, h, tokens=None):
        need.append(real(cache, batch, h, tokens))
        return need[-1]

    with pytest.MonkeyPatch.context() as m:
        m.setattr(paged, "workspace_bytes", count)
        out = base.run_attend(g, kind, store, heads, kv_heads, width, lens, news, page, trees, latent=latent, **kw)
    n = max(1, need[0] // (4 * (sum(news) + 2) * heads * ((512 if latent else width) + 2)))
    assert splits is None or {"one": n == 1, "some": 1 < n <= MANY_SPLITS, "many": n > MANY_SPLITS}[splits], n
    return out


# heads, kv heads, nodes a tree: groups of 8, 1, 7 and 2 query heads
TREES = [(16, 2, 4), (8, 1, 3), (2, 2, 30), (7, 1, 4), (4, 2, 9)]


@pytest.mark.parametrize("kind,store", STORES)
@pytest.mark.parametrize("width", [64, 128, 256])
@pytest.mark.parametrize("heads,kv_heads,n", TREES)
@pytest.mark.parametrize("splits", ["one", "some"])
def test_trees_of_few_query_rows(kind, store, width, heads, kv_heads, n, splits):
    """Draft trees that begin at the start of a sequence, inside a step of 32 rows, at its end and
    across a split's; one token's mask empty; fewer tokens than the others; no rows before."""
    g = base._gen(heads * width + n)
    news = [n, n, n, 2, n, 1]
    lens = [n, n + 45, n + 32, 130, n + 127, 1]
    if splits == "some":
        lens[1], lens[4] = 2100 + n, 1536 - 2
    trees = [O.tree(k, 2) for k in news]
    trees[2] = torch.rand(n, n, generator=g) < 0.4
    trees[0][n - 1] = False                        # attends nothing: no row lies before the tree
    attend(g, kind, store, heads, kv_heads, width, lens, news, 16, trees, splits)


@pytest.mark.parametrize("kind,store", [(BF, "bf16"), (HF, "f16"), (BF, "mx8")])
@pytest.mark.parametrize("width", [64, 128, 256])
@pytest.mark.parametrize("heads,kv_heads,n", TREES)
@pytest.mark.parametrize("long", [13, 2000])
def test_infinity_and_nan_in_a_siblings_row(kind, store, width, heads, kv_heads, n, long):
    """They reach the tokens that attend the row and no others, in one piece and split."""
    page, lens, news = 32, [long + n, long // 2 + n], [n, n]
    trees = [O.tree(n, 2), O.tree(n, 3)]
    row = long + min(2, n - 1)                     # a leaf, or a node that its children alone attend

    def edit(c, pages):
        at = (pages[0, row // page].item(), slice(None), row % page)
        if store == "mx8":
            c["v"].view(torch.uint8)[at + (slice(5, None, 9),)] = 0x7f
        else:
            c["v"][at + (3,)], c["v"][at + (4,)], c["v"][at + (40,)] = math.inf, math.nan, -math.inf

    got, _ = attend(base._gen(n + long), kind, store, heads, kv_heads, width, lens, news, page, trees, "some" if long > 1000 else "one",
                    edit=edit)
    touched = ~torch.isfinite(got[:n]).all(-1).all(-1)
    assert torch.equal(touched, trees[0][:, row - long]) and touched.any() and not touched.all()


@pytest.mark.parametrize("kind,store", STORES)
@pytest.mark.parametrize("heads,kv_heads,width,lens,news", [
    (8, 1, 64, [9500, 700], [1, 1]), (4, 2, 64, [9300], [3]), (8, 1, 256, [9500, 40], [1, 1]), (4, 2, 256, [9200], [2]),
    (8, 2, 128, [9100, 8000], [2, 1]), (16, 1, 0, [3200, 60], [1, 1]), (16, 1, 0, [5000], [2])])
def test_many_splits_joined(kind, store, heads, kv_heads, width, lens, news):
    attend(base._gen(heads + lens[0]), kind, store, heads, kv_heads, width, lens, news, 64, None, "many")


@pytest.mark.parametrize("heads,kv_heads,width,L", [(8, 1, 64, 9500), (8, 1, 128, 9500), (8, 1, 256, 9500), (16, 1, 0, 3500)])
def test_many_splits_of_which_some_hold_nothing(heads, kv_heads, width, L):
    """Whole splits without a page, and a first row whose score lies far above all others."""
    page = 64
    g = base._gen(L + width)
    pages, n_pages = base.deal(g, [L], page)
    pages[0, 20:20 + L // page // 2] = -1

    def edit(c, pages):
        c["k"][pages[0, 0].item(), :, 0] *= 8

    attend(g, BF, "bf16", heads, kv_heads, width, [L], [1], page, None, "many", pages=pages, n_pages=n_pages, edit=edit)
