"""The bookkeeping of the decode step's layer at the end of its pages, on CPU tensors."""
import pytest
import torch

from cudalab_b200.evaluator.decode_step import AttentionLayer


class _Written:
    def __init__(self):
        self.slots = []

    def write(self, k, v, pages, slots):
        self.slots.append(slots.tolist())


def _layer(lengths, width=2, page=16, prefix=0):
    layer = object.__new__(AttentionLayer)
    B = len(lengths)
    layer.batch, layer.page_size, layer.prefix = B, page, prefix
    layer.capacity = width * page
    shared = -(-prefix // page)
    layer.page_table = torch.arange(B * width, dtype=torch.int32).flip(0).reshape(B, width)
    layer.prefix_pages = torch.arange(B * width, B * width + shared, dtype=torch.int32)
    layer.lengths = torch.tensor(lengths, dtype=torch.int32)
    layer.pages = torch.zeros(1, dtype=torch.uint8)
    layer.cache = _Written()
    layer._number_slots()
    return layer


def test_slots_of_full_sequences_are_skipped():
    layer = _layer([0, 15, 16, 31, 32, 33, 1000])
    table = layer.page_table.tolist()
    assert layer.slots().tolist() == [table[0][0] * 16, table[1][0] * 16 + 15, table[2][1] * 16,
                                      table[3][1] * 16 + 15, -1, -1, -1]


def test_fill_refuses_what_the_pages_do_not_hold():
    layer = _layer([0, 30], prefix=20)

    def rows(n):
        return torch.zeros(n, 1, 64, dtype=torch.float16)

    layer.fill(rows(2), rows(2), 1)
    assert layer.lengths.tolist() == [0, 32] and layer.cache.slots == [[14, 15]]
    for n, sequence in ((1, 1), (33, 0), (21, None)):
        with pytest.raises(RuntimeError, match="exceed"):
            layer.fill(rows(n), rows(n), sequence)
    layer.fill(rows(32), rows(32), 0)
    layer.fill(rows(20), rows(20), None)
    assert layer.lengths.tolist() == [32, 32] and len(layer.cache.slots) == 3


def test_a_refused_projection_leaves_the_lengths():
    layer = _layer([3, 4])

    class Refuses:
        def forward_rmsnorm(self, *args):
            raise RuntimeError("no")

    layer.gemv, layer.w_qkv, layer.norm = Refuses(), (None, None), None
    with pytest.raises(RuntimeError):
        layer.step(None)
    assert layer.lengths.tolist() == [3, 4]
