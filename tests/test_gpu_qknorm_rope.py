"""Per-head RMSNorm and rotation (cl_qknorm_rope) against the formula in 64 bits.

Tolerance: the output rounds once (2^-11 or 2^-8 of it); before that the
element is a sum of two products of normalised values, each a chain of at most
12 fp32 roundings (mean of head_dim squares over lanes and shuffles, rsqrt,
two products, the rotation), 2^-24 each and rsqrt within 2 ulp: 16 * 2^-23 of
|a c| + |b s|, bounded by the row's largest value times sqrt(2)."""
import numpy as np
import pytest
import torch

from cudalab_b200 import _native as nat
from cudalab_b200.build import build
from oracle import attention_oracle as oa

pytestmark = pytest.mark.gpu
EPS = 1e-6


def _case(T, Hq, Hk, D, R, dtype, seed, rows=300):
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn(T, Hq + 2 * Hk, D, generator=g).to(dtype).cuda()
    w = [(1 + 0.3 * torch.randn(D, generator=g)).to(dtype).cuda() for _ in range(2)]
    a = torch.arange(rows)[:, None] * 10000.0 ** (-torch.arange(R // 2) / (R // 2))
    table = torch.cat((a.cos(), a.sin()), 1).contiguous().cuda()
    pos = torch.randint(0, rows, (T,), generator=g).cuda()
    return qkv[:, :Hq], qkv[:, Hq:Hq + Hk], w[0], w[1], table, pos


def _check(y, x, w, table, pos, interleaved):
    ref = oa.qknorm_rope(x.double().cpu().numpy(), None if w is None else w.double().cpu().numpy(),
                         table.cpu().numpy(), pos.cpu().numpy(), EPS, interleaved)
    bits = 11 if y.dtype == torch.float16 else 8
    top = np.abs(ref).max(-1, keepdims=True) * 2 ** 0.5
    tol = 2.0 ** -bits * np.abs(ref) + 16 * 2.0 ** -23 * top + 2.0 ** -25
    err = np.abs(y.double().cpu().numpy() - ref)
    assert (err <= tol).all(), float((err / tol).max())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("shape", [(1, 32, 8, 128, 128), (3, 8, 1, 64, 64), (17, 7, 7, 128, 32),
                                   (5, 5, 1, 80, 80), (9, 3, 2, 96, 48), (2, 4, 2, 256, 256),
                                   (33, 2, 1, 256, 64), (4, 1, 1, 16, 16), (1, 6, 3, 240, 16)],
                         ids=lambda s: "x".join(map(str, s)))
def test_formula(shape, interleaved, dtype):
    q, k, qw, kw, table, pos = _case(*shape, dtype, seed=sum(shape))
    ext = build("qknorm_rope")
    yq, yk = ext.forward(q, k, qw, kw, table, pos, eps=EPS, interleaved=interleaved)
    assert yq.is_contiguous() and yq.shape == q.shape and yk.shape == k.shape
    _check(yq, q, qw, table, pos, interleaved)
    _check(yk, k, kw, table, pos, interleaved)
    # without weights the rows turn and are not normalised
    yq, yk = ext.forward(q, k, None, None, table, pos.int(), eps=EPS, interleaved=interleaved)
    _check(yq, q, None, table, pos, interleaved)
    _check(yk, k, None, table, pos, interleaved)
    assert nat.device_status(clear=True) == 0


def test_into_in_place_and_odd_strides():
    """In place on a fused projection's slices, and rows that 16-byte accesses
    cannot take (an odd head stride) give the same bits as the contiguous call."""
    q, k, qw, kw, table, pos = _case(11, 6, 2, 128, 64, torch.float16, seed=3)
    ext = build("qknorm_rope")
    yq, yk = ext.forward(q, k, qw, kw, table, pos)
    odd = torch.zeros(11, 8, 131, dtype=torch.float16, device="cuda")
    oq, ok = odd[:, :6, 1:129], odd[:, 6:, 2:130]
    oq.copy_(q), ok.copy_(k)
    zq, zk = ext.forward(oq, ok, qw, kw, table, pos)
    assert torch.equal(zq, yq) and torch.equal(zk, yk)
    ext.forward_into(oq, ok, qw, kw, table, pos, oq, ok)
    assert torch.equal(oq, yq) and torch.equal(ok, yk)
    assert torch.count_nonzero(odd[:, :, 130]) == 0 and torch.count_nonzero(odd[:, :, 0]) == 0
    ext.forward_into(q, k, qw, kw, table, pos, q, k)
    assert torch.equal(q, yq) and torch.equal(k, yk)


def test_zero_rows_empty_and_extremes():
    ext = build("qknorm_rope")
    q, k, qw, kw, table, pos = _case(4, 2, 1, 64, 64, torch.float16, seed=5)
    q = torch.zeros_like(q)
    yq, _ = ext.forward(q, k, qw, kw, table, pos)
    assert torch.count_nonzero(yq) == 0
    yq, yk = ext.forward(q[:0], k[:0], qw, kw, table, pos[:0])
    assert yq.shape == (0, 2, 64) and yk.shape == (0, 1, 64)
    big = torch.full((1, 1, 64), 60000.0, dtype=torch.float16, device="cuda")
    yb, _ = ext.forward(big, big, qw, kw, table, torch.zeros(1, dtype=torch.int64, device="cuda"))
    _check(yb, big, qw, table, torch.zeros(1, dtype=torch.int64), False)
    # a NaN stays in its own head
    x = torch.ones(2, 3, 64, dtype=torch.float16, device="cuda")
    x[1, 1, 5] = float("nan")
    y, _ = ext.forward(x, x, qw, kw, table, torch.zeros(2, dtype=torch.int64, device="cuda"))
    bad = torch.isnan(y).any(-1)
    assert bad.sum() == 1 and bad[1, 1]


def test_infinity_past_the_rotation_stays_alone():
    q, k, _, _, table, pos = _case(3, 2, 1, 128, 32, torch.float16, seed=11)
    q = q.contiguous()
    q[1, 0, 70] = float("inf")
    for interleaved in (False, True):
        y, _ = build("qknorm_rope").forward(q, k, None, None, table, pos, interleaved=interleaved)
        assert torch.equal(y[..., 32:], q[..., 32:])
        assert torch.isfinite(y).sum() == y.numel() - 1


def test_position_outside_the_table_is_recorded():
    q, k, qw, kw, table, pos = _case(2, 2, 1, 64, 64, torch.float16, seed=7)
    pos[1] = table.shape[0]
    build("qknorm_rope").forward(q, k, qw, kw, table, pos)
    torch.cuda.synchronize()
    assert nat.device_status(clear=True) == 7
    assert nat.device_status() == 0


def test_other_stream():
    q, k, qw, kw, table, pos = _case(64, 8, 2, 128, 128, torch.bfloat16, seed=9)
    ext = build("qknorm_rope")
    ref = ext.forward(q, k, qw, kw, table, pos)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y = ext.forward(q, k, qw, kw, table, pos)
    s.synchronize()
    assert torch.equal(y[0], ref[0]) and torch.equal(y[1], ref[1])
