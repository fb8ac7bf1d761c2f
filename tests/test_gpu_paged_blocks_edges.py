"""The choice of blocks at the ends of what is allowed, on the GPU: calls without rows, scores
next to the ends of float32's range."""
from __future__ import annotations

import pytest
import torch

import block_oracle as B
import test_gpu_paged as base
from hearth_amd import paged
from test_gpu_paged_blocks import choice, new_bounds

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


def test_choice_without_rows():
    """max_kv of 0, and page tables of no columns: nothing can be taken, and nothing is attended."""
    bd = new_bounds(3, 2, 16, 16, 64)
    cache = paged.Cache(*(torch.ones(3, 2, 16, 64, dtype=BF, device="cuda") for _ in range(2)))
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
    for heads, news in ((4, [2, 1]), (4, [30, 40]), (64, [1, 1])):
        n = sum(news)
        starts, lens = i32(0, news[0], n), i32(50, 7)
        for pages, max_kv in ((torch.zeros(2, 1, dtype=torch.int32, device="cuda"), 0), (torch.zeros(2, 0, dtype=torch.int32, device="cuda"), 60)):
            b = paged.Batch(pages, lens, starts, max_q=max(news), max_kv=max_kv)
            q, out = torch.ones(n + 1, heads, 64, dtype=BF, device="cuda"), torch.full((n + 1, heads, 64), 3, dtype=BF, device="cuda")
            chosen = torch.full((n + 1, 2, 5), 9, dtype=torch.int32, device="cuda")
            paged.update_bounds(cache, b, bd, stream=base._stream())
            paged.select(bd, b, q, chosen, stream=base._stream())
            paged.attend_blocks(cache, b, q, chosen, out, block=16, scale=0.1, stream=base._stream())
            torch.cuda.synchronize()
            assert (chosen[:n] == -1).all() and (chosen[n:] == 9).all()
            assert (out[:n] == 0).all() and (out[n:] == 3).all()
    assert (bd.low_high == 77).all()


def scaled(sizes):
    """an edit of a cache's keys: block i (a page) keeps its random rows' directions times sizes[i % len(sizes)]"""
    def edit(k, pages):
        for i in range(k.shape[0]):
            k[i] = (k[i].double().sign() * sizes[i % len(sizes)]).to(k.dtype)
    return edit


@pytest.mark.parametrize("rows", [40 * 16, 600 * 16, 2500 * 16, 9000 * 16])
@pytest.mark.parametrize("sizes,size", [((1e20,), 1e20), ((1e20, -1e20, 1.0, 3e19), 1e20), ((2.0 ** 60,), 2.0 ** 64), ((2.0 ** 60, -1.5, 2.0 ** 59, 2.0 ** 56), 2.0 ** 64)])
def test_choice_of_scores_near_infinity(rows, sizes, size):
    """Scores of both signs up to the largest floats and past them (equal infinities: the lowest blocks). Each block's
    rows are alike, so that a score is its rows' own, of either sign; a choice of fewer than there are infinities, and of more."""
    def edit(k, pages):
        scaled(sizes)(k, pages)
        k[:] = k[:, :, :1]

    n = rows // 16
    order = torch.arange(n, dtype=torch.int32)[None]
    for top, heads in ((2, 1), (5, 1), (25, 3), (n // 3, 1)):
        choice(base._gen(top), BF, "bf16", heads, 1, 64, [rows], [1], 16, 16, top, 0, 1, pages=order, n_pages=n, edit=edit,
               queries=lambda q: q.copy_((q.double().sign() * size).to(BF)))


@pytest.mark.parametrize("rows", [40 * 16, 600 * 16, 9000 * 16])
@pytest.mark.parametrize("heads", [1, 3, 20])
def test_choice_of_scores_near_zero(rows, heads):
    """Products of steps below float32's least: scores of 0 from sums of either sign are equal, and the lowest blocks
    are taken; and least numbers of both signs, which are not."""
    def edit(k, pages):
        scaled((2.0 ** -120, -2.0 ** -122))(k, pages)
        k[:] = k[:, :, :1]

    n = rows // 16
    order = torch.arange(n, dtype=torch.int32)[None]
    for size, top in ((2.0 ** -110, 9), (2.0 ** -110, n // 2), (2.0 ** -30, 9), (2.0 ** -29, n // 2)):
        got = choice(base._gen(n), BF, "bf16", heads, 1, 64, [rows], [1], 16, 16, top, 0, 1, pages=order, n_pages=n, edit=edit,
                     queries=lambda q: q.copy_((q.double().sign() * size).to(BF)))
        if size == 2.0 ** -110:
            assert torch.equal(got[0, 0, :-1], torch.arange(top - 1, dtype=torch.int32))
