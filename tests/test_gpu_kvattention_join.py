"""Parts of a sequence, or of a prefix, that are computed apart and joined: every one
of them shows in the result (test_attention_join_cpu.py)."""
import numpy as np
import pytest
import torch

from cudalab_b200.build import build
from oracle import attention_oracle as oa
from test_attention_join_cpu import N, case, tolerance

pytestmark = pytest.mark.gpu


def _filled(k, v, bits, page):
    cache = build("kvcache")
    n, _, D = k.shape
    width = -(-n // page)
    pages = cache.empty(width, 1, D, bits, page)
    order = torch.randperm(width, generator=torch.Generator().manual_seed(n))
    j = torch.arange(n)
    cache.write(k.cuda(), v.cuda(), pages, (order[j // page] * page + j % page).cuda())
    return pages, order.int().cuda()


def _check(out, lse, q, k, v, n, D):
    ref, rl, pv, mag = (x[0] for x in oa.attention(q.double().numpy(), k, v, n, D ** -0.5))
    err = np.abs(out.double().cpu().numpy() - ref)
    tol = tolerance(ref, pv, mag, n, D)
    assert (err <= tol).all(), float((err / tol).max())
    assert (np.abs(lse.double().cpu().numpy() - rl) <= oa.lse_tolerance(rl, mag, n, D)).all()


@pytest.mark.parametrize("D,bits", [(64, 4), (128, 8), (256, 4)])
@pytest.mark.parametrize("copies", [1, 3, 60])
def test_parts_of_a_sequence(copies, D, bits):
    """One sequence over CTAs of its own, three, and 60 as one line whose segments the
    CTAs' ranges cut anywhere."""
    q, k, v, hk, hv = case(D, bits)
    pages, order = _filled(k, v, bits, 64)
    out, lse = build("kvattention").forward(
        q.cuda().expand(copies, -1, -1), pages, order.expand(copies, -1).contiguous(),
        torch.full((copies,), N, dtype=torch.int32, device="cuda"), return_lse=True)
    for b in range(copies):
        _check(out[b], lse[b], q, hk, hv, N, D)


@pytest.mark.parametrize("D,bits", [(64, 4), (128, 8), (256, 4)])
@pytest.mark.parametrize("copies", [1, 9])
def test_parts_of_a_prefix(copies, D, bits):
    """4 and 36 rows: the register-fed and the tensor-core kernel."""
    n = 5000
    q, k, v, hk, hv = case(D, bits, n=n)
    pages, order = _filled(k, v, bits, 64)
    out, lse = build("kvattention").forward_shared(
        q.cuda().expand(copies, -1, -1), pages, order, n,
        torch.zeros(copies, 1, dtype=torch.int32, device="cuda"),
        torch.zeros(copies, dtype=torch.int32, device="cuda"), return_lse=True)
    for b in range(copies):
        _check(out[b], lse[b], q, hk, hv, n, D)
