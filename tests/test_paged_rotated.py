"""The refusals of append_rotated, on the CPU: with stand-ins for device tensors, and of the C entry point
with a device that is not there (-4 where the arguments fit together)."""
from __future__ import annotations

import ctypes
import math
import re
from ctypes import byref

import pytest

from hearth_amd import paged
from test_paged_args import Fake, _Dev, batch, cache
from test_paged_bounds import HEADER, NONE, but
from test_paged_gradients import leaf

F = Fake((32,), "float64")


def test_refusals():
    c, b = cache(), batch()
    q, k = Fake((5, 4, 64)), Fake((5, 2, 64), ptr=1 << 41)
    for args, kw in (((q, k, None, F), {}), ((Fake((4, 4, 64)), k, k, F), {}), ((Fake((5, 4, 32)), k, k, F), {}), ((Fake((5, 4, 64), "float16"), k, k, F), {}),
                     ((q, k, k, Fake((33,), "float64")), {}), ((q, k, k, Fake((0,), "float64")), {}), ((q, k, k, Fake((32,), "float32")), {}),
                     ((q, k, k, F), dict(offset=1)), ((q, k, k, F), dict(offset=-1)), ((q, k, k, F), dict(layout="neox")),
                     ((q, k, k, F), dict(factor=math.nan)), ((q, k, k, F), dict(pos=Fake((4,), "int32"))), ((q, k, k, F), dict(pos=Fake((5,), "float32"))),
                     ((q, k, k, F), dict(q_out=Fake((5, 4, 32)))), ((q, k, k, F), dict(q_out=Fake((5, 3, 64)))), ((q, k, k, F), dict(q_out=Fake((5, 4, 64), "float32"))),
                     ((q, k, k, F), dict(q_out=Fake((5, 4, 64), strides=(256, 0, 1)))), ((q, k, k, F), dict(q_out=Fake((5, 4, 64), strides=(512, 64, 1)))),
                     ((None, k, k, F), dict(q_out=q)), ((q, Fake((5, 2, 64)), k, F), {}), ((q, k, Fake((5, 2, 64)), F), dict(q_out=q)),
                     ((q, Fake((5, 3, 64)), k, F), {}), ((q, Fake((5, 2, 64), "float8_e4m3fn"), k, F), {}), ((q, k, k, Fake((32,), "float64", dev=_Dev(index=1))), {}),
                     ((Fake((5, 4, 64), dev=_Dev(index=1)), k, k, F), {}), ((Fake((5, 4, 64), strides=(256, 1, 4)), k, k, F), {})):
        with pytest.raises(ValueError):
            paged.append_rotated(c, b, *args, **kw)
    lat = cache(heads=1, width=576, latent=True)
    l, pe, qp = Fake((5, 1, 512), ptr=1 << 41), Fake((5, 1, 64), ptr=1 << 42), Fake((5, 16, 64))
    for args in ((qp, Fake((5, 1, 576), ptr=1 << 41), None, F), (Fake((5, 16, 512)), l, pe, F), (qp, l, pe, Fake((33,), "float64"))):
        with pytest.raises(ValueError):
            paged.append_rotated(lat, b, *args)
    for args in ((leaf(5, 4, 64), k, k, F), (q, leaf(5, 2, 64), k, F), (q, k, leaf(5, 2, 64), F), (q, k, k, leaf(32, dtype="float64"))):
        with pytest.raises(ValueError, match="requires a gradient"):
            paged.append_rotated(c, b, *args)


def test_c_entry():
    fn = paged._fn("hearth_gpu_kv_append_rotated")
    c, b = cache()._s, batch()._of(5)._obj
    q, k, v = paged._array(Fake((5, 4, 64)), "q", 0), paged._array(Fake((5, 2, 64), ptr=1 << 41), "k", 0), paged._array(Fake((5, 2, 64), ptr=1 << 42), "v", 0)
    f = 1 << 40

    def call(c=c, b=b, q=q, q_out=q, k=k, v=v, pos=None, p64=0, freqs=f, n=32, offset=0, factor=1.0, dev=NONE):
        r = lambda s: byref(s) if s is not None else None
        return fn(r(c), r(b), r(q), r(q_out), r(k), r(v), pos, p64, freqs, n, offset, 0, factor, dev, None)

    assert call() == -4 and call(q=None, q_out=None) == -4 and call(pos=f) == -4
    for kw in (dict(c=None), dict(b=None), dict(k=None), dict(v=None), dict(q=None), dict(q_out=None), dict(freqs=None), dict(n=0), dict(n=33), dict(n=513), dict(offset=1),
               dict(offset=-1), dict(factor=math.inf), dict(dev=-1), dict(pos=f + 2), dict(pos=f + 4, p64=1), dict(freqs=f + 4), dict(q_out=but(q, width=32)),
               dict(q_out=but(q, n_heads=2)), dict(q_out=but(q, token_stride=512)), dict(q_out=but(q, data=1 << 43, head_stride=0)), dict(q_out=k, q=but(q, n_heads=2)),
               dict(q_out=but(q, data=k.data)), dict(q_out=but(q, data=v.data)), dict(q=but(q, dtype=1), q_out=but(q, dtype=1)), dict(k=but(k, dtype=0))):
        assert call(**kw) == -1, kw
    assert call(b=but(b, n_tokens=0)) == 0 and call(b=but(b, n_seqs=0)) == 0
    top = int(re.search(r"n_heads \* width of the cache up to 2\^23, min\(max_q, n_tokens\) up to 2\^(\d+) - 1\.", HEADER).group(1))
    flat = [but(x, token_stride=x.n_heads * x.width) for x in (q, k, v)]
    long = lambda n: call(b=but(b, n_tokens=n, max_q=n), q=flat[0], q_out=flat[0], k=flat[1], v=flat[2])
    assert long(2 ** top - 1) == -4 and long(2 ** top) == -1
