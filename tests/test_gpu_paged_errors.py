"""What a refused call of the paged operators leaves behind, on the GPU."""
from __future__ import annotations

from ctypes import byref

import pytest
import torch

from hearth_amd import paged

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def test_a_call_for_a_device_that_is_not_there_ends_with_itself():
    """The refused call's device error does not reach the thread's next calls, and the current
    device stays what it was."""
    none = torch.cuda.device_count() + 3
    x = torch.randn(5, 2, 64, device="cuda").to(BF)
    pos, freqs = torch.arange(5, dtype=torch.int32, device="cuda"), torch.ones(32, dtype=torch.float64, device="cuda")
    k, v = (torch.zeros(4, 2, 16, 64, dtype=BF, device="cuda") for _ in range(2))
    cache = paged.Cache(k, v)
    batch = paged.Batch(torch.arange(1, dtype=torch.int32, device="cuda").view(1, 1), torch.full((1,), 5, dtype=torch.int32, device="cuda"),
                        torch.tensor([0, 5], dtype=torch.int32, device="cuda"), max_q=5, max_kv=16)
    a, out, s = paged._array(x, "x", 0), torch.zeros_like(x), torch.cuda.current_stream().cuda_stream
    o = paged._array(out, "out", 0)
    torch.cuda.synchronize()
    for dev in (none, none):
        assert paged._fn("hearth_gpu_rope")(byref(a), byref(a), None, None, 5, pos.data_ptr(), 0, freqs.data_ptr(), 32, 0, 0, 0, 1.0,
                                            dev, None) == -4
        paged.append(cache, batch, x, x, stream=s)
        assert paged._fn("hearth_gpu_kv_append")(cache._ref, batch._of(5), byref(a), byref(a), dev, None) == -4
        paged.read(cache, batch, out, torch.empty_like(x), stream=s)
        assert paged._fn("hearth_gpu_attend")(cache._ref, batch._of(5), byref(a), byref(o), None, 0.1, None, 0, dev, None) == -4
        paged.rope(x.clone(), pos, freqs, stream=s)
        assert torch.cuda.current_device() == 0
    torch.cuda.synchronize()
    assert torch.equal(out, x) and torch.equal(k[0, :, :5].transpose(0, 1), x)
