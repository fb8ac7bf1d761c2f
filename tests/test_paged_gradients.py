"""The paged operators have no gradients: tensors that require one are refused where autograd
records, on the CPU with stand-ins for device tensors and on the GPU with tensors."""
from __future__ import annotations

import pytest
import torch

from hearth_amd import paged
from test_paged_args import Fake, batch, cache

BF = torch.bfloat16


def leaf(*shape, dtype="bfloat16"):
    t = Fake(shape, dtype)
    t.requires_grad = True
    return t


def test_arrays_that_require_a_gradient_are_refused():
    c, b, lat = cache(), batch(), cache(heads=1, width=576, latent=True)
    x, q, pos, f = Fake((5, 2, 64)), Fake((5, 4, 64)), Fake((5,), "int32"), Fake((32,), "float64")
    ql, qp, out = Fake((5, 4, 512)), Fake((5, 4, 64)), Fake((5, 4, 512))
    for call in (lambda: paged.rope(leaf(5, 4, 64), pos, f), lambda: paged.rope(q, pos, leaf(32, dtype="float64")),
                 lambda: paged.rope(q, pos, f, out=leaf(5, 4, 64)), lambda: paged.rope(q, pos, f, k=leaf(5, 1, 64)),
                 lambda: paged.append(c, b, leaf(5, 2, 64), x), lambda: paged.append(c, b, x, leaf(5, 2, 64)),
                 lambda: paged.read(c, b, leaf(5, 2, 64), x),
                 lambda: paged.attend(c, b, leaf(5, 4, 64), q, scale=0.1), lambda: paged.attend(c, b, q, leaf(5, 4, 64), scale=0.1),
                 lambda: paged.attend(c, b, q, q, scale=0.1, lse=leaf(5, 4, dtype="float32")),
                 lambda: paged.attend_latent(lat, b, leaf(5, 4, 512), qp, out, scale=0.1),
                 lambda: paged.attend_latent(lat, b, ql, leaf(5, 4, 64), out, scale=0.1)):
        with pytest.raises(ValueError, match="requires a gradient"):
            call()


@pytest.mark.parametrize("which", ["k", "v"])
def test_caches_that_require_a_gradient_are_refused(which):
    c, b, x, q = cache(), batch(), Fake((5, 2, 64)), Fake((5, 4, 64))
    setattr(c, which, leaf(4, 2, 16, 64))
    for call in (lambda: paged.append(c, b, x, x), lambda: paged.read(c, b, x, x), lambda: paged.attend(c, b, q, q, scale=0.1)):
        with pytest.raises(ValueError, match="requires a gradient"):
            call()


def test_nothing_is_refused_where_nothing_is_recorded():
    x = leaf(5, 4, 64)
    for off in (torch.no_grad, torch.inference_mode):
        with off():
            assert paged._array(x, "x", 0).n_heads == 4


@pytest.mark.gpu
def test_on_tensors():
    """A leaf's rows rotated under no_grad; refused, and left as they were, where autograd records."""
    x = torch.randn(5, 2, 64, device="cuda").to(BF)
    pos, freqs = torch.arange(5, device="cuda"), torch.ones(32, dtype=torch.float64, device="cuda")
    p, s = torch.nn.Parameter(x.clone()), torch.cuda.current_stream().cuda_stream
    for t in (p, p * 1):
        with pytest.raises(ValueError, match="requires a gradient"):
            paged.rope(t, pos, freqs, stream=s)
    assert torch.equal(p.detach(), x)
    with torch.no_grad():
        paged.rope(p, pos, freqs, stream=s)
    paged.rope(x, pos, freqs, stream=s)
    assert torch.equal(p.detach(), x)
