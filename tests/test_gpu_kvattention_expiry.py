"""Bounded waits of the attention kernels that run out, without a fault: with the bound
lowered to one SM cycle a block of the cache (or a tile's operands) has not come when it
is first waited for, the kernel records status 8, lets what it has in flight land,
frees its Tensor Memory and returns.  The context stays usable: the same call under the
default bound gives the result of before."""
import pytest
import torch

from cudalab_b200 import _native as nat
from cudalab_b200.build import build

pytestmark = pytest.mark.gpu


def _case(B, n, H, G, D, bits, page=64):
    g = torch.Generator(device="cuda").manual_seed(B + D)
    cache = build("kvcache")
    width = n // page
    pages = cache.empty(B * width, H, D, bits, page)
    k, v = torch.randn(2, B * n, H, D, device="cuda", generator=g).half()
    cache.write(k, v, pages, torch.arange(B * n, device="cuda"))
    table = torch.arange(B * width, device="cuda", dtype=torch.int32).view(B, width)
    q = torch.randn(B, H * G, D, device="cuda", generator=g).half()
    return q, pages, table, torch.full((B,), n, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("D,bits,G", [(128, 8, 8), (128, 4, 16), (64, 8, 1), (256, 8, 4)])
def test_wait_for_a_block_runs_out(D, bits, G):
    q, pages, table, lens = _case(64, 2048, 8, G, D, bits)
    far = torch.empty(1 << 28, dtype=torch.uint8, device="cuda").view(torch.float32)
    att = build("kvattention")
    ref = att.forward(q, pages, table, lens)
    torch.cuda.synchronize()
    assert nat.device_status(clear=True) == 0
    prev = nat.set_wait_budget(1)
    try:
        for _ in range(3):
            far.fill_(1.0)  # the cache's blocks come from memory, not from L2
            att.forward(q, pages, table, lens)
        torch.cuda.synchronize()  # returns: the waits are bounded
        assert nat.device_status(clear=True) == 8
    finally:
        nat.set_wait_budget(prev)
    again = att.forward(q, pages, table, lens)
    torch.cuda.synchronize()
    assert torch.equal(again, ref) and nat.device_status(clear=True) == 0


@pytest.mark.parametrize("D,bits", [(128, 8), (128, 4), (64, 8), (64, 4)])
def test_wait_for_a_prefix_tile_runs_out(D, bits):
    q, pages, table, lens = _case(16, 256, 4, 16, D, bits)
    _, far, prefix, _ = _case(1, 8192, 4, 1, D, bits)
    att = build("kvattention")
    args = (q, torch.cat((pages, far)), prefix[0] + len(pages), 8192, table, lens)
    ref = att.forward_shared(*args)
    torch.cuda.synchronize()
    assert nat.device_status(clear=True) == 0
    prev = nat.set_wait_budget(1)
    try:
        for _ in range(3):
            att.forward_shared(*args)
        torch.cuda.synchronize()
        assert nat.device_status(clear=True) == 8
    finally:
        nat.set_wait_budget(prev)
    again = att.forward_shared(*args)
    torch.cuda.synchronize()
    assert torch.equal(again, ref) and nat.device_status(clear=True) == 0
