"""4-bit cache rows on the CPU: the plain form that the GPU tests hold the kernels to, against the
definition of nearest; the refusals of packed caches."""
from __future__ import annotations

import ctypes
import shutil
import subprocess
from ctypes import byref

import pytest
import torch

import paged_oracle4 as P
from hearth_amd import _native, paged
from test_paged_args import INC, Fake as Base, _Dev, batch


class Fake(Base):
    SIZES = {**Base.SIZES, "float4_e2m1fn_x2": 1}


def cache4(heads=2, width=64, page=16, pages=4, latent=False, **kw):
    k = Fake((pages, heads, page, width // 2), "float4_e2m1fn_x2", **kw)
    sc = Fake((pages, heads, page, width // 32), "uint8")
    return paged.Cache(k, None if latent else k, sc, None if latent else sc)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_codes_are_the_nearest(dtype):
    """No code of the block's scale is nearer than the one taken, of two as near the even one is; no
    element is off by more than half a step; the scale is the least with that property."""
    g = torch.Generator().manual_seed(3)
    x = torch.randn(500, 64, generator=g) * torch.exp2(torch.randint(-12, 12, (500, 1), generator=g).float())
    x[0], x[1, :32] = 0, 7.0
    x[2, :32] = torch.linspace(-7, 7, 32)
    x[3, :9] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, -0.25])
    x = x.to(dtype)
    codes, sc = P.mx4(x)
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()
    step = torch.exp2(sc.double() - 127).repeat_interleave(32, -1)
    a = x.double().abs() / step
    off = (a.unsqueeze(-1) - P.GRID).abs()
    took = off.gather(-1, (c & 7).unsqueeze(-1)).squeeze(-1)
    assert (took <= off.amin(-1)).all() and ((off == took.unsqueeze(-1)).sum(-1) == 1)[(c & 1) == 1].all()
    assert torch.equal(c >= 8, torch.signbit(x.double())) and (took <= 1.0).all()
    amax = x.double().unflatten(-1, (-1, 32)).abs().amax(-1)
    least = amax <= 3.5 * torch.exp2(sc.double() - 127)           # half the scale would do
    assert not (least & (sc > 1)).any() and (amax <= 7 * torch.exp2(sc.double() - 127)).all()
    assert torch.equal(P.values(codes, sc), torch.where(c >= 8, -1.0, 1.0) * P.GRID[c & 7] * step)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_how_far_off_at_the_end_of_the_range(dtype):
    """Half a step of the codes up to 3.5 times the largest scale; above, where 4 would leave the type, up to the
    step from 3 to 4 and a quarter of the value."""
    big = torch.finfo(dtype).max
    top = 2.0 ** (15 if dtype == torch.float16 else 127)
    g = torch.Generator().manual_seed(4)
    x = (torch.rand(400, 32, generator=g, dtype=torch.float64) * 2 - 1) * big
    x[0, :6] = torch.tensor([big, -big, 1.75 * top, 1.5 * top, 1.25 * top, 1.75 * top * (1 + 2.0 ** -6)])
    x = x.to(dtype)
    codes, sc = P.mx4(x)
    v, a = P.values(codes, sc), x.double().abs()
    step = torch.exp2(sc.double() - 127).repeat_interleave(32, -1)
    gap = torch.where(a / step >= 4, 2.0, torch.where(a / step >= 2, 1.0, 0.5)) * step
    off, end = (v - x.double()).abs(), a > 1.75 * top
    assert (off[~end] <= gap[~end] / 2).all() and (off[end] <= gap[end]).all() and (off[end] <= a[end] / 4).all()
    assert end.sum() > 100 and (off[end] > gap[end] / 2).all() and torch.isfinite(v.to(dtype)).all()
    assert dtype != torch.float16 or (1.75 * top == 57344 and off[0, 0] == 65504 - 49152)


def test_ends_of_the_range():
    for dtype, big in ((torch.bfloat16, 3.3895e38), (torch.float16, 65504.0), (torch.float32, 3.4028e38)):
        x = torch.zeros(4, 32).to(dtype)
        x[0, 0], x[0, 1], x[1, 3], x[2, 4], x[3, 5] = big, -big, float("nan"), float("inf"), torch.finfo(dtype).smallest_normal
        codes, sc = P.mx4(x)
        v = P.values(codes, sc)
        assert torch.isfinite(v[0].to(dtype)).all() and (v[0, 0] - x[0, 0].double()).abs() <= 2.0 ** -2 * x[0, 0].double()
        assert sc[1] == sc[2] == 255 and v[1:3].isnan().all() and (codes[1:3] == 0).all()
        assert sc[3] >= 1


def test_cache_refusals():
    c = cache4()
    assert (c._s.width, c._s.dtype, c._s.page) == (64, paged.MX4, 16)
    k = Fake((4, 2, 16, 32), "float4_e2m1fn_x2")
    sc = Fake((4, 2, 16, 2), "uint8")
    for args in ((k, k), (k, k, sc), (k, k, None, sc), (k, k, Fake((4, 2, 16, 1), "uint8"), sc), (Fake((4, 2, 16, 24), "float4_e2m1fn_x2"), k, sc, sc),
                 (k, Fake((4, 2, 16, 32), "float8_e4m3fn"), sc, sc), (Fake((4, 2, 16, 32), "uint8"), Fake((4, 2, 16, 32), "uint8"), sc, sc),
                 (Fake((4, 2, 16, 1024), "float4_e2m1fn_x2"),) * 2 + (Fake((4, 2, 16, 64), "uint8"),) * 2,
                 (Fake((4, 2, 16, 32), "float4_e2m1fn_x2", ptr=(1 << 40) + 8), k, sc, sc),
                 (Fake((4, 2, 16, 32), "float4_e2m1fn_x2", dev=_Dev(index=1)), k, sc, sc)):
        with pytest.raises(ValueError):
            paged.Cache(*args)
    b, q = batch(), Fake((5, 4, 64))
    with pytest.raises(ValueError, match="live in a cache only"):
        paged.append(c, b, Fake((5, 2, 64), "float4_e2m1fn_x2"), Fake((5, 2, 64)))
    with pytest.raises(ValueError):
        paged.append(c, b, Fake((5, 2, 32)), Fake((5, 2, 32)))       # the packed width
    with pytest.raises(ValueError):
        paged.attend(c, b, Fake((5, 4, 64), "float32"), q, scale=0.1)
    lat = cache4(heads=1, width=576, latent=True)
    with pytest.raises(ValueError):
        paged.attend_latent(lat, b, Fake((5, 4, 512)), Fake((5, 4, 64)), Fake((5, 4, 512)), scale=0.1)
    with pytest.raises(ValueError):
        paged.workspace_bytes(lat, b, 4)


def test_c_entries_refuse():
    """Strides of packed rows are in bytes: half a row of elements is enough, less is not."""
    L = _native.lib()
    for n, (res, args) in paged._PROTOS.items():
        getattr(L, n).restype, getattr(L, n).argtypes = res, args
    c, b = cache4()._s, batch()._of(5)._obj
    r = paged._array(Fake((5, 2, 64)), "k", 0)
    call = lambda: L.hearth_gpu_kv_append(byref(c), byref(b), byref(r), byref(r), 1000, None)
    assert c.k.head_stride == 16 * 32 and call() == -4                # a device that is not there
    for field, bad in (("head_stride", 16 * 32 - 16), ("page_stride", 2 * 16 * 32 - 520), ("scale_head_stride", 31), ("scales", None), ("data", (1 << 40) + 8)):
        was = getattr(c.k, field)
        setattr(c.k, field, bad)
        assert call() == -1, field
        setattr(c.k, field, was)
    c.dtype = 18
    assert call() == -1


def test_the_header_names_the_type(tmp_path):
    if not shutil.which("gcc"):
        pytest.skip("gcc not available")
    src, exe = tmp_path / "l.c", tmp_path / "l"
    src.write_text(f'#include <stdio.h>\n#include "{INC / "hearth_gpu.h"}"\nint main(void) {{ printf("%d\\n", HEARTH_GPU_MX4); return 0; }}\n')
    subprocess.run(["gcc", "-std=c11", "-I", str(INC), str(src), "-o", str(exe)], check=True)
    assert int(subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout) == paged.MX4
