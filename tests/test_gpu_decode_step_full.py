"""Steps past the end of a sequence's pages: the full sequence keeps its cache and is
recorded, the others go on as if alone."""
import pytest
import torch

from cudalab_b200 import _native as nat
from cudalab_b200.evaluator.decode_step import AttentionLayer

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("captured", [False, True])
def test_full_sequence(captured):
    a, b = (AttentionLayer(2, 512, 8, 2, 64, 30, 8, 16, 0, seed=5) for _ in range(2))
    assert a.capacity == 32 and a.table.shape[0] == 32
    g = torch.Generator().manual_seed(6)
    k, v = torch.randn(2, 31, 2, 64, generator=g).half().cuda()
    a.fill(k, v, 0)
    for layer in (a, b):
        layer.fill(k[:3], v[:3], 1)
    x = torch.randn(2, 512, generator=g).half().cuda()
    for layer in (a, b):
        layer.step(x)  # the last token that a's first sequence holds
    torch.cuda.synchronize()
    assert nat.device_status(clear=True) == 0
    full = a.pages[a.page_table[0].long()].clone()
    if captured:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ya = a.step(x)
    for _ in range(3):
        if captured:
            graph.replay()
        else:
            ya = a.step(x)
        yb = b.step(x)
        assert torch.equal(ya[1], yb[1]) and torch.isfinite(ya).all()
    torch.cuda.synchronize()
    assert nat.device_status(clear=True) == 7
    assert torch.equal(a.pages[a.page_table[0].long()], full)
