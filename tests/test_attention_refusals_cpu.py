"""What the attention operators refuse besides the cases of test_attention_cpu.py,
without a GPU."""
import ctypes

import pytest
import torch

from cudalab_b200 import _native as nat


def _rej(fn, text):
    with pytest.raises(RuntimeError) as e:
        fn()
    assert text in str(e.value), str(e.value)


def test_descriptor_refuses_what_its_fields_do_not_hold():
    """2^32 + 5 in a 32-bit field is an error, not 5."""
    for cls in (nat.QkNormRopeDesc, nat.KvCacheDesc, nat.KvAttentionDesc):
        for i, (name, ctype) in enumerate(cls._fields_):
            values = [1] * len(cls._fields_)
            for big in (1 << 31, (1 << 32) + 5):
                values[i] = big
                if ctype is ctypes.c_int32:
                    _rej(lambda: cls(*values), f"{name} must be below 2^31, got {big}")
                else:
                    assert getattr(cls(*values), name) == big or ctype is ctypes.c_float
            values[i] = (1 << 31) - 1
            assert int(getattr(cls(*values), name)) in ((1 << 31) - 1, 1 << 31)


def test_outputs_that_overlap_themselves():
    from cudalab_b200.attention_ext import _apart

    x = torch.zeros(4096)
    for size, stride in (((2, 2, 64), (200, 10, 1)), ((3, 2, 64), (64, 64, 1)),
                         ((2, 2, 64), (0, 64, 1)), ((2, 3, 64), (64, 63, 1)), ((2, 2), (1, 1))):
        shared = torch.as_strided(x, size, stride)
        _rej(lambda: _apart("out", shared), "out must not overlap itself")
    for size, stride in (((2, 2, 64), (200, 64, 1)), ((2, 3, 64), (64, 128, 1)), ((1, 2, 64), (0, 64, 1)),
                         ((2, 1, 64), (64, 5, 1)), ((0, 2, 64), (0, 0, 1)), ((3, 4, 60), (256, 61, 1))):
        _apart("out", torch.as_strided(x, size, stride))


def test_output_over_its_input():
    from cudalab_b200.attention_ext import _separate

    x = torch.zeros(3, 12, 64, dtype=torch.float16)
    for y in (x, x[1:], x[2, 7:], x[:, 4:8], x.flatten()[64 * 7:64 * 9]):
        _rej(lambda: _separate("out", y, "q", x[:, :8]), "out must not overlap q")
    _separate("out", x[2, 8:], "q", x[:, :8])
    _separate("out", x[2], "q", x[:2])
    _separate("out", x[:0], "q", x)
