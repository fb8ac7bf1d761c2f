"""Choice of blocks and attention over them, on the CPU: the plain forms that the GPU tests hold the kernels
to against the definition, element by element; the refusals of hearth_amd/paged.py with stand-ins for device tensors
and of the C entry points with a device that is not there (-4 where the arguments fit together); the mirrors' layouts."""
from __future__ import annotations

import ctypes
import math
import re
import shutil
import subprocess
from ctypes import byref

import pytest
import torch

import block_oracle as B
from hearth_amd import paged
from test_paged_args import INC, Fake, _Dev, batch, cache
from test_paged_bounds import HEADER, NONE, but
from test_paged_gradients import leaf


# ---------------------------------------------------------------- the plain forms

def test_whole_numbers():
    """Up to 127 steps of the least power of two that reaches the largest magnitude, each value within half a step."""
    g = torch.Generator().manual_seed(1)
    x = (torch.randn(200, 64, generator=g) * torch.exp2(torch.randint(-20, 20, (200, 1), generator=g).float())).double()
    x[0], x[1, 0], x[2, 0], x[3, :2] = 0, 127.0, 127.5, torch.tensor([math.inf, math.nan])
    c, byte = B.whole(x, (1,))
    step = torch.exp2(byte.double() - 127)
    fine = torch.where(x.isfinite(), x, 0.0)
    assert (c.abs() <= 127).all() and ((c * step - fine).abs() <= step / 2).all() and (c == c.round()).all()
    top = fine.abs().amax(1, keepdim=True)
    assert ((top > 127 * step / 2) | (byte == 1))[1:].all() and (top <= 127 * step).all()


def test_scores_bound_the_rows():
    """A block's score is at least every row's, up to the rounding of both to whole numbers."""
    g = torch.Generator().manual_seed(2)
    K, q = torch.randn(2, 100, 64, generator=g).double(), torch.randn(3, 6, 64, generator=g).double()
    codes, byte = B.bounds(K, torch.ones(100, dtype=torch.bool), 16)
    s = B.scores(codes, byte, q)
    step = q.abs().amax(-1) / 63                     # at most a step of q, and of the keys
    for h in range(2):
        z = torch.einsum("nhw,lw->nhl", q[:, 3 * h:3 * h + 3], K[h]).amax(1)
        slack = 64 * (step.amax() * K.abs().amax() + q.abs().amax() * K.abs().amax() / 63) / 2
        for b in range(7):
            assert (s[:, h, b].double() >= z[:, b * 16:(b + 1) * 16].amax(1) - slack).all()
    # one score written out
    cq, e = B.whole(q[1, 4], (0,))
    want = sum(max(cq[d] * codes[1, 3, 0, d], cq[d] * codes[1, 3, 1, d]).item() for d in range(64)) * 2.0 ** (e.item() + byte[1, 3].item() - 254)
    others = [sum(max(a[d] * codes[1, 3, 0, d], a[d] * codes[1, 3, 1, d]).item() for d in range(64)) * 2.0 ** (x.item() + byte[1, 3].item() - 254)
              for a, x in (B.whole(q[1, j], (0,)) for j in (3, 5))]
    assert s[1, 1, 3].item() == max(want, *others)


def test_choice_by_hand():
    codes, byte = torch.zeros(1, 6, 2, 1, dtype=torch.float64), torch.full((1, 6), 127)
    codes[0, :, 1, 0] = torch.tensor([0.0, 5.0, 3.0, 5.0, 1.0, 4.0])
    q = torch.full((1, 1, 1), 127.0, dtype=torch.float64)
    pick = lambda top, first, last, base=95, tree=False: B.choose(codes, byte, q, base, 96, 16, top, first, last, tree)[0, 0].tolist()
    assert pick(3, 0, 1) == [1, 3, 5] and pick(2, 0, 1) == [1, 5] and pick(4, 1, 2) == [0, 1, 4, 5] and pick(8, 0, 1) == [0, 1, 2, 3, 4, 5, -1, -1]
    assert pick(2, 0, 1, base=60) == [1, 3] and pick(2, 0, 1, base=-1) == [-1, -1] and pick(3, 0, 1, base=40, tree=True) == [0, 1, 2]
    byte[0, 1] = -1
    assert pick(3, 0, 1) == [2, 3, 5] and pick(8, 0, 1) == [0, 2, 3, 4, 5, -1, -1, -1]


# ---------------------------------------------------------------- refusals

def bounds(pages=4, heads=2, blocks=2, width=64, block=16, ptr=1 << 40, dev=None, **kw):
    return paged.Bounds(Fake((pages, heads, blocks, 2, width), "int8", ptr=ptr, dev=dev, **kw), Fake((pages, heads, blocks), "uint8", dev=dev), block=block)


class I8(Fake):
    SIZES = {**Fake.SIZES, "int8": 1}


def test_bounds_refusals():
    bounds()
    lh, st = I8((4, 2, 2, 2, 64), "int8"), Fake((4, 2, 2), "uint8")
    for a, b, n in ((I8((4, 2, 2, 64), "int8"), st, 16), (I8((4, 2, 2, 3, 64), "int8"), st, 16), (Fake((4, 2, 2, 2, 64), "uint8"), st, 16), (lh, Fake((4, 2, 4), "uint8"), 16),
                    (lh, Fake((4, 2, 2), "int32"), 16), (lh, st, 8), (lh, st, 24), (lh, st, 4096), (I8((4, 2, 3, 2, 64), "int8"), Fake((4, 2, 3), "uint8"), 16),
                    (I8((4, 2, 2, 2, 96), "int8"), st, 16), (I8((4, 2, 2, 2, 64), "int8", ptr=(1 << 40) + 8), st, 16), (lh, Fake((4, 2, 2), "uint8", dev=_Dev(index=1)), 16),
                    (I8((4, 2, 2, 2, 64), "int8", strides=(520, 256, 128, 64, 1)), st, 16), (I8((4, 2, 2, 2, 64), "int8", strides=(512, 256, 128, 1, 2)), st, 16),
                    (lh, Fake((4, 2, 2), "uint8", strides=(4, 1, 2)), 16), (I8((4, 2, 2, 2, 64), "int8", dev=_Dev("cpu")), st, 16)):
        with pytest.raises(ValueError):
            paged.Bounds(a, b, block=n)


def test_update_refusals():
    c, b = cache(page=32), batch()
    for cc, bb in ((cache(page=16), bounds()), (cache(page=32, heads=4), bounds()), (cache(page=32, width=128), bounds()), (cache(page=32, pages=5), bounds()),
                   (cache(page=32), bounds(dev=_Dev(index=1))), (cache(page=32, heads=1, width=64, latent=True), bounds(heads=1))):
        with pytest.raises(ValueError):
            paged.update_bounds(cc, b, bb)
    c.k = leaf(4, 2, 32, 64)
    with pytest.raises(ValueError, match="requires a gradient"):
        paged.update_bounds(c, b, bounds())


def test_select_refusals():
    s, b = bounds(), batch()
    q, out, work = Fake((5, 4, 64)), Fake((5, 2, 6), "int32"), Fake((1 << 20,), "uint8")
    for args, kw in (((Fake((5, 3, 64)), out), {}), ((Fake((5, 4, 128)), out), {}), ((Fake((5, 4, 64), "float32"), out), {}), ((q, Fake((4, 2, 6), "int32")), {}),
                     ((q, Fake((5, 4, 6), "int32")), {}), ((q, Fake((5, 2, 6), "int64")), {}), ((q, Fake((5, 2, 6), "int32", strides=(12, 1, 2))), {}),
                     ((q, Fake((5, 2, 6), "int32", strides=(12, 4, 1))), {}), ((q, Fake((5, 2, 6), "int32", dev=_Dev(index=1))), {}),
                     ((q, out), dict(first=-1)), ((q, out), dict(last=0)), ((q, out), dict(first=4, last=3)), ((q, out), dict(first=7)),
                     ((q, out), dict(workspace=None)), ((q, out), dict(workspace=Fake((16,), "uint8"))), ((q, out), dict(workspace=Fake((1 << 20,), "uint8", ptr=(1 << 40) + 4))),
                     ((q, out), dict(workspace=Fake((1 << 20,), "uint8", dev=_Dev(index=1)))), ((Fake((5, 2 * 129, 64)), out), {}), ((leaf(5, 4, 64), out), {})):
        with pytest.raises(ValueError):
            paged.select(s, b, *args, **{"workspace": work, **kw})
    for kw in (dict(first=1 << 32), dict(last=(1 << 32) + 1)):       # no cut to 32 bits
        with pytest.raises(ValueError):
            paged.select(s, b, q, out, workspace=work, **kw)
    # a tree's own blocks, besides the first ones, have to fit: 33 rows touch at most 3 blocks of 16, wherever they begin
    assert max((at + 32) // 16 - at // 16 + 1 for at in range(16)) == 3
    m = paged.Batch(Fake((2, 4), "int32"), Fake((2,), "int32"), Fake((3,), "int32"), max_q=33, max_kv=100, mask=Fake((40, 1), "int64"))
    q33 = Fake((33, 4, 64))
    paged_call = lambda top: paged._fn("hearth_gpu_select_blocks")(s._ref, m._of(33), byref(paged._array(q33, "q", 0)),
                                                                 byref(paged._blocks(Fake((33, 2, top), "int32"), "c", 0, 33, 2, 16)), 1, 1, 1 << 40, 1 << 30, NONE, None)
    assert paged_call(3) == -1 and paged_call(4) == -4
    with pytest.raises(ValueError):
        paged.select_workspace_bytes(s, paged.Batch(Fake((1, 1 << 27), "int32"), Fake((1,), "int32"), Fake((2,), "int32"), max_q=1, max_kv=0x7fffffff))


def test_attend_blocks_refusals():
    c, b = cache(), batch()
    q, ch = Fake((5, 4, 64)), Fake((5, 2, 6), "int32")
    for args, kw in (((q, ch, Fake((5, 4, 32))), {}), ((q, Fake((4, 2, 6), "int32"), q), {}), ((q, Fake((5, 4, 6), "int32"), q), {}), ((q, Fake((5, 2, 6), "int64"), q), {}),
                     ((q, ch, q), dict(block=8)), ((q, ch, q), dict(block=32)), ((q, ch, q), dict(block=24)), ((q, ch, q), dict(scale=math.nan)), ((Fake((5, 3, 64)), ch, Fake((5, 3, 64))), {}),
                     ((q, Fake((5, 2, 0), "int32"), q), {}), ((q, Fake((5, 2, 6), "int32", dev=_Dev(index=1)), q), {}), ((leaf(5, 4, 64), ch, q), {}),
                     ((q, ch, q), dict(lse=Fake((5, 4))))):
        with pytest.raises(ValueError):
            paged.attend_blocks(c, b, *args, **{"block": 16, "scale": 0.1, **kw})
    with pytest.raises(ValueError):
        paged.attend_blocks(cache(heads=1, width=576, latent=True), b, Fake((5, 4, 576)), Fake((5, 1, 6), "int32"), Fake((5, 4, 576)), block=16, scale=0.1)
    with pytest.raises(ValueError):
        paged.attend_blocks_workspace_bytes(cache(width=96), b, 4, 6, 16)
    for kw in (dict(block=(1 << 32) + 16), dict(top=(1 << 32) + 6), dict(heads=(1 << 32) + 4), dict(top=0)):       # no cut to 32 bits
        with pytest.raises(ValueError):
            paged.attend_blocks_workspace_bytes(c, b, **{"heads": 4, "top": 6, "block": 16, **kw})
    with pytest.raises(ValueError):
        paged.attend_blocks(c, b, q, ch, q, block=(1 << 32) + 16, scale=0.1)
    # a workspace is asked for where rows are split
    one = batch(S=1, per=4096, max_q=1, max_kv=65536)
    q1, many = Fake((1, 4, 64)), Fake((1, 2, 200), "int32")
    need = paged.attend_blocks_workspace_bytes(c, one, 4, 200, 16, 1)
    assert need > 0 and paged.attend_blocks_workspace_bytes(c, one, 4, 200, 16, 2) == 2 * need and paged.attend_blocks_workspace_bytes(c, one, 4, 4, 16, 1) == 0
    for work in (None, Fake((need - 1,), "uint8"), Fake((need,), "uint8", ptr=(1 << 40) + 8)):
        with pytest.raises(ValueError):
            paged.attend_blocks(c, one, q1, many, q1, block=16, scale=0.1, workspace=work)


def test_c_entries():
    c, b, s = cache(page=32)._s, batch()._of(5)._obj, bounds()._s
    q, ch = paged._array(Fake((5, 4, 64)), "q", 0), paged._BlocksS(1 << 40, 12, 6, 6, 16)
    r = lambda x: byref(x) if x is not None else None
    bnd = lambda c=c, b=b, s=s, dev=NONE: paged._fn("hearth_gpu_key_bounds")(r(c), r(b), r(s), dev, None)
    sel = lambda s=s, b=b, q=q, o=ch, first=1, last=1, work=1 << 40, n=1 << 30, dev=NONE: paged._fn("hearth_gpu_select_blocks")(r(s), r(b), r(q), r(o), first, last, work, n, dev, None)
    att = lambda c=c, b=b, q=q, o=ch, out=q, lse=None, scale=0.1, work=1 << 40, n=1 << 30, dev=NONE: paged._fn("hearth_gpu_attend_blocks")(
        r(c), r(b), r(q), r(o), r(out), lse, scale, work, n, dev, None)
    assert bnd() == sel() == att() == -4
    for kw in (dict(c=None), dict(b=None), dict(s=None), dict(dev=-1), dict(s=but(s, n_pages=5)), dict(s=but(s, n_heads=1)), dict(s=but(s, block=32)), dict(s=but(s, width=128)),
               dict(s=but(s, codes=None)), dict(s=but(s, scales=None)), dict(s=but(s, codes=(1 << 40) + 8)), dict(s=but(s, page_stride=17)), dict(s=but(s, head_stride=128)),
               dict(s=but(s, scale_head_stride=1)), dict(s=but(s, page_stride=1 << 50)), dict(b=but(b, n_seqs=-1))):
        assert bnd(**kw) == -1, kw
    for kw in (dict(s=None), dict(b=None), dict(q=None), dict(o=None), dict(dev=-1), dict(first=-1), dict(last=0), dict(first=6), dict(first=0x7fffffff), dict(last=0x7fffffff),
               dict(q=but(q, dtype=0)), dict(q=but(q, width=128)), dict(q=but(q, n_heads=3)), dict(q=but(q, n_heads=258)), dict(o=but(ch, chosen=None)), dict(o=but(ch, chosen=(1 << 40) + 2)),
               dict(o=but(ch, top=0)), dict(o=but(ch, top=(1 << 20) + 1)), dict(o=but(ch, block=32)), dict(o=but(ch, token_stride=5)), dict(o=but(ch, head_stride=0)), dict(work=None),
               dict(work=(1 << 40) + 8)):
        assert sel(**kw) == -1, kw
    assert sel(n=16) == -3 and sel(q=but(q, n_heads=256)) == -4
    for kw in (dict(c=None), dict(b=None), dict(q=None), dict(o=None), dict(out=None), dict(dev=-1), dict(scale=math.inf), dict(lse=(1 << 40) + 2), dict(o=but(ch, chosen=None)),
               dict(o=but(ch, chosen=(1 << 40) + 1)), dict(o=but(ch, top=0)), dict(o=but(ch, block=8)), dict(o=but(ch, block=64)), dict(o=but(ch, block=48)), dict(q=but(q, dtype=1)),
               dict(o=but(ch, top=1 << 20, block=32, head_stride=0, token_stride=1 << 50))):
        assert att(**kw) == -1, kw
    assert att(o=but(ch, token_stride=0, head_stride=0)) == -4       # one list for all is read, not written
    none = but(b, n_tokens=0)
    assert bnd(b=none) == sel(b=none, work=None, n=0) == att(b=none, work=None, n=0) == 0
    assert bnd(b=but(b, max_q=0)) == sel(b=but(b, max_q=0), work=None, n=0) == 0


def test_stated_limits():
    c, b, s = cache(page=32)._s, batch()._of(5)._obj, bounds()._s
    need = lambda n, S=1: paged._fn("hearth_gpu_select_workspace")(byref(s), byref(but(b, n_seqs=S, n_tokens=n, max_q=n)))
    top = 2 ** int(re.search(r"n_heads \* min\(max_q, n_tokens\) up to 2\^(\d+); tokens of no sequence are left alone", HEADER).group(1)) // 2
    assert need(top) >= 0 and need(top + 1) == -1
    work = lambda n, heads, block=16, top=6: paged._fn("hearth_gpu_attend_blocks_workspace")(byref(c), byref(but(b, n_seqs=1, n_tokens=n, max_q=n)), heads, top, block)
    top = 2 ** int(re.search(r"\(query heads of a cache head / 16, rounded up\) up to 2\^(\d+) - 1;", HEADER).group(1)) - 1
    assert work(top // 2, 2) >= 0 and work(top // 2 + 1, 2) == -1 and work(1, 4, 32, 1 << 20) >= 0 and work(1, 4, 32, (1 << 20) + 1) == -1
    big = cache(page=4096)._s
    assert paged._fn("hearth_gpu_attend_blocks_workspace")(byref(big), byref(b), 4, 1 << 18, 4096) == -1     # 2^30 rows


def test_mirrors_match_the_header(tmp_path):
    if not shutil.which("gcc"):
        pytest.skip("gcc not available")
    mirrors = {"hearth_gpu_bounds": paged._BoundsS, "hearth_gpu_blocks": paged._BlocksS}
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{INC / "hearth_gpu.h"}"', "int main(void) {"]
    for cname, m in mirrors.items():
        lines.append(f'    printf("{cname} %zu\\n", sizeof({cname}));')
        lines += [f'    printf("{cname}.{f[0]} %zu\\n", offsetof({cname}, {f[0]}));' for f in m._fields_]
    src, exe = tmp_path / "l.c", tmp_path / "l"
    src.write_text("\n".join(lines + ["    return 0;", "}"]) + "\n")
    subprocess.run(["gcc", "-std=c11", "-I", str(INC), str(src), "-o", str(exe)], check=True)
    vals = dict(ln.rsplit(" ", 1) for ln in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines())
    for cname, m in mirrors.items():
        assert int(vals[cname]) == ctypes.sizeof(m)
        for f in m._fields_:
            assert int(vals[f"{cname}.{f[0]}"]) == getattr(m, f[0]).offset, (cname, f[0])
