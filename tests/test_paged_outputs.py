"""Arrays that the paged operators write: one whose rows share elements (a broadcast dimension) is
refused, on the CPU, by the C entry points, before any device call; one that is read is not."""
from __future__ import annotations

from ctypes import byref

import pytest

from hearth_amd import paged
from test_paged_args import Fake, batch, cache

SHARED = [(0, 64, 1), (256, 0, 1), (256, 32, 1), (63, 1024, 1), (0, 0, 1)]


@pytest.mark.parametrize("strides", SHARED)
def test_rows_that_share_elements_are_refused(strides):
    c, b, lat = cache(heads=4), batch(), cache(heads=1, width=576, latent=True)
    bad, x = Fake((5, 4, 64), strides=strides), Fake((5, 4, 64), ptr=1 << 41)
    pos, f = Fake((5,), "int32"), Fake((32,), "float64")
    wide = Fake((5, 4, 512), strides=tuple(8 * s if s > 1 else s for s in strides))
    for call in (lambda: paged.rope(bad, pos, f), lambda: paged.rope(x, pos, f, out=bad), lambda: paged.rope(x, pos, f, k=bad),
                 lambda: paged.rope(x, pos, f, k=Fake((5, 4, 64)), k_out=bad),
                 lambda: paged.read(c, b, bad, x), lambda: paged.read(c, b, x, bad), lambda: paged.attend(c, b, x, bad, scale=0.1),
                 lambda: paged.attend_latent(lat, b, Fake((5, 4, 512)), x, wide, scale=0.1)):
        with pytest.raises(ValueError):
            call()


def test_one_row_has_no_neighbour():
    """The stride of a dimension of one element means nothing: such calls get as far as the device,
    which is none (-4), and not -1."""
    none = 1000
    heads = paged._array(Fake((5, 1, 64), strides=(64, 0, 1)), "x", 0)
    token = paged._array(Fake((1, 4, 64), strides=(0, 64, 1)), "x", 0)
    f = paged._fn("hearth_gpu_rope")
    for x, n in ((heads, 5), (token, 1)):
        assert f(byref(x), byref(x), None, None, n, 1 << 40, 0, 1 << 40, 32, 0, 0, 0, 1.0, none, None) == -4
