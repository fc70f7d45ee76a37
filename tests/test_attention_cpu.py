"""The attention operators without a GPU: the C ABI refuses bad descriptors
before any device work, the extension objects refuse bad tensors in the order
of the arguments, and the cache's layout is a permutation that keeps the
kernel's shared-memory accesses free of bank conflicts."""
import ctypes
import itertools

import numpy as np
import pytest
import torch

from cudalab_b200 import _native as nat
from cudalab_b200.attention_ext import block_bytes
from cudalab_b200.build import build, build_library
from oracle import attention_oracle as oa

FAKE = 1 << 20  # a 16-byte aligned, never dereferenced address
BAD = nat.CL_ERR_INVALID_ARGUMENT


@pytest.fixture(scope="module")
def lib():
    build_library()
    return nat.load()


def _with(desc, **kw):
    d = type(desc).from_buffer_copy(desc)
    for name, value in kw.items():
        setattr(d, name, value)
    return ctypes.byref(d)


def test_rope_descriptor(lib):
    ok = nat.QkNormRopeDesc(tokens=1, table_rows=8, q_heads=4, kv_heads=2, head_dim=128,
                            rotary=128, dtype=nat.CL_DTYPE_F16, eps=1e-6)
    args = [FAKE] * 8

    def call(a=args, **kw):
        return lib.cl_qknorm_rope(*a, _with(ok, **kw), None)

    for kw, text in ((dict(tokens=-1), "tokens"), (dict(q_heads=0), "heads"),
                     (dict(head_dim=120), "head_dim"), (dict(head_dim=272), "head_dim"),
                     (dict(rotary=24), "rotary"), (dict(rotary=144), "rotary"),
                     (dict(rotary=0), "rotary"), (dict(dtype=nat.CL_DTYPE_F32), "dtype"),
                     (dict(eps=float("nan")), "eps"), (dict(eps=-1.0), "eps"),
                     (dict(table_rows=0), "table_rows"), (dict(tokens=1 << 60), "too many")):
        assert call(**kw) == BAD and text in nat.last_error(lib), kw
    assert call([None] + args[1:]) == BAD
    assert call(args[:2] + [None] + args[3:]) == BAD and "both" in nat.last_error(lib)
    assert call(args[:4] + [FAKE + 4] + args[5:]) == BAD and "aligned" in nat.last_error(lib)
    assert lib.cl_qknorm_rope(*args, None, None) == BAD
    assert call([None] * 8, tokens=0) == nat.CL_OK  # nothing to do, nothing touched


def test_cache_descriptor(lib):
    ok = nat.KvCacheDesc(tokens=1, num_pages=2, kv_heads=2, head_dim=128, bits=8, page_size=64,
                         dtype=nat.CL_DTYPE_BF16)
    for fn, pages_at in ((lib.cl_kvcache_write, 2), (lib.cl_kvcache_read, 0)):
        for kw, text in ((dict(tokens=-1), "tokens"), (dict(head_dim=96), "head_dim"),
                         (dict(bits=2), "bits"), (dict(page_size=24), "page_size"),
                         (dict(page_size=0), "page_size"), (dict(kv_heads=0), "kv_heads"),
                         (dict(num_pages=0), "num_pages"), (dict(dtype=1), "dtype"),
                         (dict(tokens=1 << 60), "too many")):
            assert fn(FAKE, FAKE, FAKE, FAKE, _with(ok, **kw), None) == BAD, kw
            assert text in nat.last_error(lib), kw
        args = [FAKE] * 4
        args[pages_at] = FAKE + 8
        assert fn(*args, _with(ok), None) == BAD and "aligned" in nat.last_error(lib)
        args[pages_at] = None
        assert fn(*args, _with(ok), None) == BAD


def test_attention_descriptor(lib):
    n = ctypes.c_size_t(0)
    assert lib.cl_kvattention_workspace(ctypes.byref(n)) == nat.CL_OK and n.value > 0
    assert lib.cl_kvattention_workspace(None) == BAD
    ok = nat.KvAttentionDesc(num_pages=4, batch=2, new_tokens=1, q_heads=8, kv_heads=2,
                             head_dim=128, bits=8, page_size=64, max_pages=2,
                             dtype=nat.CL_DTYPE_F16, scale=0.1)
    args = [FAKE] * 9

    def call(a=args, **kw):
        return lib.cl_kvattention(*a, _with(ok, **kw), None)

    for kw, text in ((dict(dtype=1), "dtype"), (dict(head_dim=80), "head_dim"),
                     (dict(bits=5), "bits"), (dict(page_size=40), "page_size"),
                     (dict(batch=4097), "batch"), (dict(new_tokens=0), "new_tokens"),
                     (dict(q_heads=7), "multiple"), (dict(window=-1), "window"),
                     (dict(scale=float("inf")), "scale"), (dict(max_pages=1 << 30), "max_pages"),
                     (dict(batch=4096, max_pages=1 << 24), "too many blocks"),
                     (dict(prefix_length=-1), "prefix"),
                     (dict(prefix_length=65, prefix_page_count=1), "prefix_pages"),
                     (dict(prefix_length=10, prefix_page_count=1, window=4), "window"),
                     (dict(prefix_length=10, prefix_page_count=1, new_tokens=2, q_batch=3, q_new=1),
                      "evenly")):
        assert call(**kw) == BAD and text in nat.last_error(lib), (kw, nat.last_error(lib))
    for i in (0, 1, 2, 3, 5, 8):
        assert call(args[:i] + [None] + args[i + 1:]) == BAD
    for i in (1, 5, 8):
        assert call(args[:i] + [FAKE + 2] + args[i + 1:]) == BAD and "aligned" in nat.last_error(lib)
    assert call([FAKE, FAKE] + [None] * 7, batch=0) == nat.CL_OK
    n = ctypes.c_size_t(0)
    assert lib.cl_kvattention_prefix_floats(_with(ok), ctypes.byref(n)) == nat.CL_OK and n.value == 0
    assert lib.cl_kvattention_prefix_floats(_with(ok, prefix_length=10, prefix_page_count=1),
                                            ctypes.byref(n)) == nat.CL_OK
    assert n.value >= 2 * 8 * 129 and n.value % (2 * 8 * 129) == 0
    assert call(prefix_length=10, prefix_page_count=1, a=args[:7] + [None] + args[8:]) == BAD
    assert call(prefix_length=10, prefix_page_count=1, a=args[:7] + [FAKE + 4] + args[8:]) == BAD


def _rej(fn, text):
    with pytest.raises(RuntimeError) as e:
        fn()
    assert text in str(e.value), str(e.value)


def test_ext_refusals():
    h = torch.float16
    rope, cache, att = build("qknorm_rope"), build("kvcache"), build("kvattention")
    q, k = torch.zeros(3, 4, 64, dtype=h), torch.zeros(3, 2, 64, dtype=h)
    w, table, pos = torch.ones(64, dtype=h), torch.zeros(8, 64), torch.zeros(3, dtype=torch.int64)
    _rej(lambda: rope.forward(q[0], k, w, w, table, pos), "q must be 3-D")
    _rej(lambda: rope.forward(q.float(), k, w, w, table, pos), "float16 or bfloat16")
    _rej(lambda: rope.forward(q.transpose(1, 2), k, w, w, table, pos), "contiguous")
    _rej(lambda: rope.forward(q, k, w, w, table, pos), "CUDA tensor")
    pages = cache.empty(2, 2, 64, 8, 16, device="cpu")
    assert pages.shape == (2, 2, 1, block_bytes(64, 8))
    slots = torch.zeros(3, dtype=torch.int64)
    _rej(lambda: cache.write(k.double(), k, pages, slots), "float16 or bfloat16")
    _rej(lambda: cache.write(k, k, pages, slots), "CUDA tensor")
    _rej(lambda: cache.read(pages, slots, 64, torch.float32), "float16 or bfloat16")
    _rej(lambda: cache.read(pages, slots, 96), "64, 128 or 256")
    _rej(lambda: cache.read(pages, slots, 256), "blocks of")
    _rej(lambda: cache.read(pages, slots, 64), "CUDA tensor")
    _rej(lambda: cache.empty(1, 1, 80), "head_dim")
    _rej(lambda: cache.empty(1, 1, 64, 6), "bits")
    _rej(lambda: cache.empty(1, 1, 64, 8, 24), "page_size")
    lens, pt = torch.zeros(3, dtype=torch.int32), torch.zeros(3, 1, dtype=torch.int32)
    _rej(lambda: att.forward(q[0], pages, pt, lens), "q must be [batch")
    _rej(lambda: att.forward(q, pages, pt, lens), "CUDA tensor")
    _rej(lambda: att.forward_shared(q, pages, pt[0], -1, pt, lens), "prefix_length")
    assert att.workspace_bytes > 0


@pytest.mark.parametrize("row", [32, 64, 128, 256])
def test_layout_is_a_permutation_without_bank_conflicts(row):
    j, b = np.arange(16)[:, None], np.arange(row)[None]
    at = oa.place(row, j, b)
    assert sorted(at.reshape(-1)) == list(range(16 * row))
    # what one instruction reads: K, lane (g, t): a quarter of token g's row in
    # accesses of up to 16 bytes; V, tokens 2t + {0, 1, 8, 9}: an eighth chosen by g
    lanes = list(itertools.product(range(8), range(4)))

    def conflict_free(first_bytes, size):
        phase = 128 // size  # lanes served together
        for p in range(0, 32, phase):
            banks = [(a // 4 + i) % 32 for a in first_bytes[p:p + phase] for i in range(size // 4)]
            assert len(set(banks)) == 32
    size = min(16, row // 4)
    for i in range(row // 4 // size):
        byte = {256: lambda t: (i >> 1) * 128 + 32 * t + 16 * (i & 1), 128: lambda t: 32 * t + 16 * i,
                64: lambda t: 16 * t, 32: lambda t: 8 * t}[row]
        for up in (0, 8):
            conflict_free([int(oa.place(row, g + up, byte(t))) for g, t in lanes], size)
    size = min(16, row // 8)
    for i in range(row // 8 // size):
        byte = (lambda g: 128 * i + 16 * g) if row == 256 else (lambda g: row // 8 * g)
        for x in (0, 1, 8, 9):
            conflict_free([int(oa.place(row, 2 * t + x, byte(g))) for g, t in lanes], size)


def test_oracle_write_round_trip():
    g = np.random.default_rng(0)
    for dim, bits in itertools.product((64, 128, 256), (8, 4)):
        k, v = g.standard_normal((2, 20, 2, dim)).astype(np.float32)
        pages = np.zeros((2, 2, 2, block_bytes(dim, bits)), np.uint8)
        slots = g.permutation(64)[:20]
        oa.write(pages, 32, slots, k, v, bits)
        row = oa.row_bytes(dim, bits)
        for t, slot in enumerate(slots):
            blk = pages[slot // 32, :, slot % 32 // 16]
            for part, x in enumerate((k, v)):
                q, s = oa.quantise(x[t], bits)
                raw = blk[:, part * 16 * row + oa.place(row, slot % 16, np.arange(row))]
                assert np.array_equal(raw, oa.pack_rows(q, bits))
                err = np.abs(oa.dequantise(q, s) - x[t]).max(-1)
                assert (err <= s.astype(np.float32) * 0.51).all()
