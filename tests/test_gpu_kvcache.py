"""The quantised paged cache (cl_kvcache_write / cl_kvcache_read): bytes equal
to the oracle's, which does the defining fp32 operations one by one, and
values read back equal to whole value times scale, rounded once."""
import numpy as np
import pytest
import torch

from cudalab_b200 import _native as nat
from cudalab_b200.build import build
from oracle import attention_oracle as oa

pytestmark = pytest.mark.gpu


def _kv(T, H, D, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(2, T, H, D, generator=g) * torch.exp(2 * torch.randn(2, T, H, 1, generator=g))
    return x.to(dtype).cuda().unbind(0)


def _slots(T, pages, page, seed):
    return torch.randperm(pages * page, generator=torch.Generator().manual_seed(seed))[:T]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("shape", [(1, 1, 128, 16), (37, 3, 64, 16), (50, 8, 128, 64),
                                   (21, 2, 256, 48), (200, 5, 64, 128)],
                         ids=lambda s: "x".join(map(str, s)))
def test_bytes_and_values(shape, bits, dtype):
    T, H, D, page = shape
    ext = build("kvcache")
    k, v = _kv(T, H, D, dtype, seed=T + D)
    n = -(-T // page) + 1
    pages = ext.empty(n, H, D, bits, page)
    pages.fill_(0xA5)  # what is not written must stay
    ref = pages.cpu().numpy().copy()
    slots = _slots(T, n, page, seed=T)
    slots[T // 2] = -1
    ext.write(k, v, pages, slots.cuda())
    oa.write(ref, page, slots.numpy(), k.float().cpu().numpy(), v.float().cpu().numpy(), bits)
    assert np.array_equal(pages.cpu().numpy(), ref)
    for back in (torch.float16, torch.bfloat16):
        rk, rv = ext.read(pages, slots.cuda(), D, back)
        for x, y in ((k, rk), (v, rv)):
            q, s = oa.quantise(x.float().cpu().numpy(), bits)
            val = torch.from_numpy(oa.dequantise(q, s)).to(back)
            val[T // 2] = 0
            assert torch.equal(y.cpu(), val)
    assert nat.device_status(clear=True) == 0


@pytest.mark.parametrize("bits", [8, 4])
def test_special_values(bits):
    """Zero rows, ties, infinities, NaN, scales below fp16 and above it."""
    D = 128
    x = torch.zeros(8, 1, D)
    x[1, 0, :8] = torch.tensor([7.0, 3.5, -3.5, 0.5, 1.5, -2.5, 6.5, -7.0])
    x[2, 0, 3] = float("inf")
    x[2, 0, 4] = -1000.0
    x[3, 0] = torch.linspace(-1, 1, D)
    x[3, 0, 5] = float("nan")
    x[4, 0] = 1e-7 * torch.linspace(-1, 1, D)
    x[5, 0] = 3e38 * torch.linspace(-1, 1, D)
    x[6, 0] = float("nan")
    x[7, 0, ::2], x[7, 0, 1::2] = float("-inf"), float("inf")
    k = x.bfloat16().cuda()
    ext = build("kvcache")
    pages = ext.empty(1, 1, D, bits, 16)
    ref = pages.cpu().numpy().copy()
    ext.write(k, k, pages, torch.arange(8, device="cuda"))
    f = k.float().cpu().numpy()
    oa.write(ref, 16, range(8), f, f, bits)
    assert np.array_equal(pages.cpu().numpy(), ref)
    rk, rv = ext.read(pages, torch.arange(8, device="cuda"), D, torch.bfloat16)
    assert torch.isfinite(rk).all() and torch.equal(rk, rv)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("bits", [8, 4])
def test_every_largest_value(bits, dtype):
    """Every magnitude that the type has as a row's largest: the scale and all
    fields, byte for byte."""
    D, T = 64, 1 << 15
    top = torch.arange(T, dtype=torch.int32).to(torch.int16).view(dtype).float()
    x = (top[:, None] * torch.linspace(1, -1, D)[None]).to(dtype).view(T, 1, D)
    k, v = x.cuda(), x.flip(-1).contiguous().cuda()
    ext = build("kvcache")
    pages = ext.empty(T // 16, 1, D, bits, 16)
    ref = pages.cpu().numpy().copy()
    ext.write(k, v, pages, torch.arange(T, device="cuda"))
    oa.write(ref, 16, range(T), k.float().cpu().numpy(), v.float().cpu().numpy(), bits)
    assert np.array_equal(pages.cpu().numpy(), ref)


def test_strided_inputs_and_outputs():
    """k and v as slices of a fused projection, rows with an odd stride, and a
    strided destination give the contiguous call's bytes."""
    T, H, D, page = 40, 4, 128, 32
    ext = build("kvcache")
    k, v = _kv(T, H, D, torch.float16, seed=1)
    slots = _slots(T, 2, page, seed=2).cuda()
    a, b, c = (ext.empty(2, H, D, 8, page) for _ in range(3))
    ext.write(k, v, a, slots)
    fused = torch.cat((k, v), 1)
    ext.write(fused[:, :H], fused[:, H:], b, slots)
    odd = torch.zeros(T, H, 2, D + 1, dtype=torch.float16, device="cuda")
    odd[:, :, 0, 1:], odd[:, :, 1, :D] = k, v
    ext.write(odd[:, :, 0, 1:], odd[:, :, 1, :D], c, slots)
    assert torch.equal(a, b) and torch.equal(a, c)
    rk, rv = ext.read(a, slots, D)
    out = torch.full((T, 2 * H + 1, D + 3), 5.0, dtype=torch.float16, device="cuda")
    ext.read_into(a, slots, out[:, :H, 1:D + 1], out[:, H:2 * H, 2:D + 2])
    assert torch.equal(out[:, :H, 1:D + 1], rk) and torch.equal(out[:, H:2 * H, 2:D + 2], rv)
    assert (out[:, 2 * H] == 5).all() and (out[:, :H, 0] == 5).all() and (out[:, :, D + 2] == 5).all()


def test_slots_outside_the_cache_are_recorded():
    ext = build("kvcache")
    k, v = _kv(3, 2, 64, torch.float16, seed=4)
    pages = ext.empty(2, 2, 64, 8, 16)
    slots = torch.tensor([5, 32, 1 << 40], device="cuda")
    ext.write(k, v, pages, slots)
    torch.cuda.synchronize()
    assert nat.device_status(clear=True) == 7
    rk, _ = ext.read(pages, slots, 64)
    assert torch.count_nonzero(rk[1:]) == 0 and torch.count_nonzero(rk[0]) > 0
    assert nat.device_status(clear=True) == 7
    assert torch.count_nonzero(pages[1]) == 0


def test_empty_call():
    ext = build("kvcache")
    pages = ext.empty(1, 2, 64)
    e = torch.empty(0, 2, 64, dtype=torch.float16, device="cuda")
    s = torch.empty(0, dtype=torch.int64, device="cuda")
    ext.write(e, e, pages, s)
    rk, rv = ext.read(pages, s, 64)
    assert rk.shape == (0, 2, 64) and torch.count_nonzero(pages) == 0
