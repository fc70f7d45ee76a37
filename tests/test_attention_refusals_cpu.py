"""What the attention operators refuse besides the cases of test_attention_cpu.py,
without a GPU."""
import ctypes

import pytest
import torch

from cudalab_b200 import _native as nat
from cudalab_b200.build import build_library


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


def test_more_row_tiles_than_the_plan_divides():
    """Tiles of 16 rows (8 at head_dim 256) of all heads of a sequence: 2^21 and more are
    refused before any device work."""
    build_library()
    lib = nat.load()
    fake = [1 << 20] * 9

    def call(**kw):
        d = nat.KvAttentionDesc(num_pages=4, batch=1, kv_heads=2, head_dim=64, bits=8, page_size=64,
                                max_pages=2, dtype=nat.CL_DTYPE_F16, scale=0.1, **kw)
        return lib.cl_kvattention(*fake, ctypes.byref(d), None)

    assert call(new_tokens=1 << 20, q_heads=32) == nat.CL_ERR_INVALID_ARGUMENT
    assert "too many query rows" in nat.last_error(lib)
    d = dict(num_pages=4, batch=1, kv_heads=1, head_dim=256, bits=8, page_size=64, max_pages=2,
             dtype=nat.CL_DTYPE_F16, scale=0.1, new_tokens=1 << 20, q_heads=16)
    assert lib.cl_kvattention(*fake, ctypes.byref(nat.KvAttentionDesc(**d)), None) == \
        nat.CL_ERR_INVALID_ARGUMENT
    assert "too many query rows" in nat.last_error(lib)
    # a prefix that the register-fed kernel would take (head_dim 256)
    d.update(batch=64, new_tokens=1 << 14, prefix_length=64, prefix_page_count=1, q_batch=1 << 14,
             q_new=1)
    assert lib.cl_kvattention(*fake, ctypes.byref(nat.KvAttentionDesc(**d)), None) == \
        nat.CL_ERR_INVALID_ARGUMENT
    assert "over the prefix" in nat.last_error(lib)
