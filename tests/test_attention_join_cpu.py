"""A long sequence whose every part shows in the result: scores nearly alike, values
around 1.  The tolerance that the GPU test takes must see the loss of any one CTA's
part, of its sum over the values alone as of its softmax sum; here that is checked on
the oracle, part by part."""
import numpy as np
import pytest
import torch

from oracle import attention_oracle as oa

N = 20011


def case(D, bits, heads=4, n=N):
    """q [1, heads, D] fp16, k, v [n, 1, D] fp16 and the values that the cache holds."""
    g = torch.Generator().manual_seed(D + bits)
    q = (0.1 * torch.randn(1, heads, D, generator=g)).half()
    k = torch.randn(n, 1, D, generator=g).half()
    v = (1 + 0.3 * torch.randn(n, 1, D, generator=g)).half()
    held = []
    for x in (k, v):
        w, s = oa.quantise(x.float().numpy(), bits)
        held.append(w.astype(np.float64) * s.astype(np.float64)[..., None])
    return q, k, v, held[0], held[1]


def tolerance(out, pv, mag, tokens, dim):
    """attention_tolerance without its term for weights below fp16's normal range: here the
    smallest of a row is within 2^-8 of the largest, which is at least 2^7."""
    ds = (dim / 16 + 4) * 2.0 ** -22 * (mag[..., None] + 1)
    steps = (tokens / 16 + 64) * 2.0 ** -23
    return 2.0 ** -11 * np.abs(out) + 2.0 ** -11 * pv + 2 * (ds + steps) * pv


@pytest.mark.parametrize("D,bits", [(64, 4), (128, 8), (256, 4)])
def test_the_loss_of_any_part_exceeds_the_tolerance(D, bits):
    part = 128 if D == 256 else 256  # tokens of a CTA
    q, _, _, k, v = case(D, bits)
    q, k, v = q[0].double().numpy(), k[:, 0], v[:, 0]
    out, lse, pv, mag = (x[0] for x in oa.attention(q[None], k[:, None], v[:, None], N, D ** -0.5))
    s = q @ k.T * D ** -0.5
    w = np.exp(s - s.max(-1, keepdims=True))
    assert w.min() > 2.0 ** -8
    total = w.sum(-1, keepdims=True)
    tol, ltol = tolerance(out, pv, mag, N, D), oa.lse_tolerance(lse, mag, N, D)
    for a in range(0, N, part):
        lost = w[:, a:a + part]
        if lost.shape[1] < part // 2:
            continue  # the last CTA's few tokens
        without = out - lost @ v[a:a + part] / total
        assert (np.abs(without - out) > tol).mean() > 0.9, a
        assert (np.abs(np.log1p(-lost.sum(-1) / total[:, 0])) > ltol).all(), a
