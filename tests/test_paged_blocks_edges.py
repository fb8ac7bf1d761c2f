"""Calls of the choice of blocks and of attention over them at the ends of what is allowed, on the CPU: with a
device that is not there (-4 where the arguments fit together, -1 where they are refused)."""
from __future__ import annotations

from ctypes import byref

import pytest

from hearth_amd import paged
from test_paged_args import Fake, batch, cache
from test_paged_blocks import bounds
from test_paged_bounds import NONE, but


@pytest.mark.parametrize("tokens,max_q,heads", [(1, 1, 4), (5, 3, 4), (40, 40, 4), (3, 3, 64)])
def test_choice_without_rows(tokens, max_q, heads):
    """max_kv of 0, and page tables of no columns: no scores, no workspace, and a call that reaches the device."""
    s, q, out = bounds(), Fake((tokens, heads, 64)), Fake((tokens, 2, 6), "int32")
    for b in (batch(max_q=max_q, max_kv=0), batch(per=0, max_q=max_q), batch(per=0, max_q=max_q, max_kv=0)):
        assert paged.select_workspace_bytes(s, b, tokens) == 0
        assert paged._fn("hearth_gpu_select_blocks")(s._ref, b._of(tokens), byref(paged._array(q, "q", 0)), byref(paged._blocks(out, "c", 0, tokens, 2, 16)), 1, 1,
                                                     None, 0, NONE, None) == -4


@pytest.mark.parametrize("heads,max_q,tokens,per,S", [(1, 1, 0x7fffffff, 1 << 26, 65535), (16, 16, 0x7fffffff, 1 << 26, 65535), (64, 3, 1 << 30, 1 << 26, 9), (4096, 2048, 0x7fffffff, 1 << 26, 65535),
                                                      (4096, 1, 1 << 27, 1 << 25, 1), (4096, 1, 1 << 26, 1 << 24, 1), (4, 1, 70, 4, 1)])
def test_workspace_of_the_choice_past_64_bits(heads, max_q, tokens, per, S):
    """Bytes that 64 bits do not hold are refused, not cut."""
    s = but(bounds(heads=2, blocks=1)._s, n_heads=heads)
    b = but(batch()._of(1)._obj, n_seqs=S, n_tokens=tokens, max_q=max_q, max_kv=0x3fff0000, pages_per_seq=per, ld_pages=per)
    want = tokens * heads * min(0x3fff0000 // 16, per) * 4
    assert paged._fn("hearth_gpu_select_workspace")(byref(s), byref(b)) == (want if want < 2 ** 63 else -1)


def test_attention_over_no_lists():
    """None in the place of the chosen blocks is no call of attend."""
    q = Fake((5, 4, 64))
    with pytest.raises(ValueError, match="chosen"):
        paged.attend_blocks(cache(), batch(), q, None, q, block=16, scale=0.1)


def test_workspaces_of_heads_that_no_array_has():
    """Bytes are told for the calls that the attentions take: up to 65536 heads an array."""
    one = batch(S=4, per=1 << 26, max_q=0x7fffffff, max_kv=0x3fff0000)
    for c in (cache(), cache(heads=1, width=576, latent=True)):
        for heads in (65536, 65538, 1 << 25, (1 << 32) + 4):
            if heads == 65536:
                assert paged.workspace_bytes(c, one, heads, 1) >= 0
            else:
                with pytest.raises(ValueError):
                    paged.workspace_bytes(c, one, heads, 1)
    assert paged.attend_blocks_workspace_bytes(cache(), one, 65536, 6, 16, 1) >= 0
    with pytest.raises(ValueError):
        paged.attend_blocks_workspace_bytes(cache(), one, 65538, 6, 16, 1)
    for tokens in (-1, 1 << 31, (1 << 32) + 5):          # no cut to 32 bits
        for call in (lambda: paged.workspace_bytes(cache(), one, 4, tokens), lambda: paged.select_workspace_bytes(bounds(), one, tokens),
                     lambda: paged.attend_blocks_workspace_bytes(cache(), one, 4, 6, 16, tokens)):
            with pytest.raises(ValueError):
                call()
