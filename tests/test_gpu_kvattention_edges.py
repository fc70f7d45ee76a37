"""Attention over the quantised cache where it is easily wrong.  Oracle and
tolerances as in test_gpu_kvattention.py."""
import numpy as np
import pytest
import torch

from cudalab_b200 import _native as nat
from cudalab_b200.build import build
from oracle import attention_oracle as oa
from test_gpu_kvattention import BF16, F16, Cache, _check, _q

pytestmark = pytest.mark.gpu


def _set(c, k, v, bits):
    """Writes k, v [tokens, H, D] over a one-sequence cache's tokens."""
    j = torch.arange(len(k))
    slots = c.table[0].cpu().long()[j // c.page] * c.page + j % c.page
    k, v = k.half(), v.half()
    c.ext.write(k.cuda(), v.cuda(), c.pages, slots.cuda())
    for at, x in ((c.k, k), (c.v, v)):
        q, s = oa.quantise(x.float().numpy(), bits)
        at[0] = q.astype(np.float64) * s.astype(np.float64)[..., None]


def _over_prefix(p, q, scale, own=0, bits=8, prefix_pages=None, ref=None):
    """q [B, 1, Hq, D] over p's tokens as the shared prefix of B sequences of `own` tokens."""
    B, D = q.shape[0], q.shape[-1]
    c = Cache([own] * B, p.H, D, bits, p.page, seed=B)
    pages = torch.cat((c.pages, p.pages))
    table = p.table[0] if prefix_pages is None else prefix_pages
    table = torch.where(table < len(p.pages), table + len(c.pages), table).int()
    out, lse = build("kvattention").forward_shared(q, pages, table, p.lengths[0], c.table,
                                                   c.len_tensor(), scale=scale, return_lse=True)
    return out, lse, c


# An empty sequence in front of several new tokens, so that length - new tokens - window
# passes 32 bits where it is taken as it stands; few sequences have CTAs of their own,
# 300 are planned as one line.
@pytest.mark.parametrize("copies", [1, 60])
@pytest.mark.parametrize("D,bits,page", [(64, 8, 16), (128, 4, 64), (256, 8, 32)])
def test_window_without_an_end(D, bits, page, copies):
    lengths = [0, 1, 50, 3, 200] * copies
    c = Cache(lengths, 2, D, bits, page, seed=81)
    q = _q(len(lengths), 5, 6, D, F16, seed=82)
    att = build("kvattention")
    most = c.table.shape[1] * page
    args = (q, c.pages, c.table, c.len_tensor())
    out, lse = att.forward(*args, return_lse=True)
    _check(out, lse, q, c, D ** -0.5)
    for window in (most - 1, most, most + 4, most + 5, 2 ** 31 - 20, 2 ** 31 - 1):
        o, z = att.forward(*args, window=window, return_lse=True)
        if window >= 200:
            assert torch.equal(o, out) and torch.equal(z, lse), window
        _check(o, z, q, c, D ** -0.5, window)


def test_window_below_the_longest_page_table():
    """A page table of 2^31 - 16 tokens, in which a window of nearly as many counts."""
    D, page, new = 64, 16, 40
    c = Cache([50, 0, 7], 1, D, 8, page, seed=83)
    q = _q(3, new, 1, D, F16, seed=84)
    table = torch.zeros(3, (1 << 27) - 1, dtype=torch.int32, device="cuda")
    table[:, :c.table.shape[1]] = c.table
    att = build("kvattention")
    for window in (2 ** 31 - 17, 2 ** 31 - 1):
        out, lse = att.forward(q, c.pages, table, c.len_tensor(), window=window, return_lse=True)
        _check(out, lse, q, c, D ** -0.5, window)


@pytest.mark.parametrize("workspace", [True, False])
def test_window_past_32_bits_is_refused(workspace):
    """Not cut to its low bits (5 tokens here)."""
    att = build("kvattention")
    c = Cache([20, 5], 1, 64, 8, 16, seed=85)
    ws = att.workspace() if workspace else None
    with pytest.raises(RuntimeError, match="window must be below"):
        att.forward(_q(2, 1, 4, 64, F16, seed=86)[:, 0], c.pages, c.table, c.len_tensor(),
                    window=(1 << 32) + 5, workspace=ws)


# one row a head: the register-fed kernel; 132: the tensor-core prefix kernel
@pytest.mark.parametrize("batch", [1, 33])
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("above", [20.0, 100.0, 127.6, 200.0])
def test_token_without_values_outweighs_all(above, bits, batch):
    """Tokens of zero V whose base-2 logits lie far above all others', in the second or
    third tile of a part (40 tiles of 128 tokens make parts of three)."""
    n, D = 5000, 128
    g = torch.Generator().manual_seed(71)
    p = Cache([n], 1, D, bits, 64, seed=72)
    d = torch.sign(torch.randn(D, generator=g))
    k, v = 0.02 * torch.randn(n, 1, D, generator=g), torch.randn(n, 1, D, generator=g)
    for at in (700, 1408):
        k[at:at + 4, 0], v[at:at + 4] = d * (above * np.log(2) / D), 0
    _set(p, k, v, bits)
    q = d.expand(batch, 1, 4, D).half().cuda()
    out, lse, c = _over_prefix(p, q, 1.0, 1, bits)
    _check(out, lse, q, c, 1.0, prefix=p)


@pytest.mark.parametrize("workspace", [True, False])
def test_prefix_without_pages_is_refused(workspace):
    att = build("kvattention")
    c = Cache([20, 5], 1, 64, 8, 16, seed=77)
    ws = att.workspace() if workspace else None
    with pytest.raises(RuntimeError, match="prefix_pages"):
        att.forward_shared(_q(2, 1, 4, 64, F16, seed=78), c.pages, None, 16, c.table,
                           c.len_tensor(), workspace=ws)


@pytest.mark.parametrize("dtype", [F16, BF16], ids=str)
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("mean,strong", [(0.0, 30.0), (1.0, 30.0), (4.0, 1.0)])
def test_strong_channel_and_queries_with_a_mean(mean, strong, D, bits, dtype):
    """A K channel that sets its token's scale, and rows of q whose elements do not
    average to zero: a score keeps its bits whatever the fields' own sum is."""
    lengths = [1, 40, 300, 517]
    c = Cache(lengths, 2, D, bits, 32, seed=D + bits, spread=0.0)
    g = torch.Generator().manual_seed(73)
    for b, n in enumerate(lengths):
        k, v = torch.randn(2, n, 2, D, generator=g)
        k[..., 5] *= strong
        j = torch.arange(n)
        slots = c.table[b].cpu().long()[j // 32] * 32 + j % 32
        c.ext.write(k.half().cuda(), v.half().cuda(), c.pages, slots.cuda())
        for at, x in ((c.k, k), (c.v, v)):
            qx, s = oa.quantise(x.half().float().numpy(), bits)
            at[b] = qx.astype(np.float64) * s.astype(np.float64)[..., None]
    for heads in (2, 8, 24):  # 1, 4 and 12 rows a head
        q = (_q(4, 1, heads, D, F16, seed=heads).float() + mean)
        q[..., 5] *= 0.1
        q = q.to(dtype)
        out, lse = build("kvattention").forward(q, c.pages, c.table, c.len_tensor(),
                                                return_lse=True)
        _check(out, lse, q, c, D ** -0.5)


@pytest.mark.parametrize("batch", [1, 33])
@pytest.mark.parametrize("D,bits", [(64, 4), (128, 8)])
@pytest.mark.parametrize("shift", [0.0, -300.0])
@pytest.mark.parametrize("gone", [[3], [0, 1, 2, 3], list(range(8, 14)), [20], list(range(21))],
                         ids=lambda g: "-".join(map(str, g[:4])))
def test_prefix_pages_outside_the_cache_are_skipped(gone, shift, D, bits, batch):
    """Their tokens are left out, in both kernels, wherever they lie and however low the
    scores of what remains are; the error is recorded."""
    n, page = 1300, 64
    g = torch.Generator().manual_seed(79)
    p = Cache([n], 1, D, bits, page, seed=80)
    d = torch.sign(torch.randn(D, generator=g))
    k = 0.1 * torch.randn(n, 1, D, generator=g) + d * (shift / D)
    _set(p, k, torch.randn(n, 1, D, generator=g), bits)
    table = p.table[0].clone()
    table[gone] = 1 << 30
    q = (d + 0.1 * torch.randn(batch, 1, 4, D, generator=g)).half().cuda()
    out, lse, c = _over_prefix(p, q, 1.0, 0, bits, prefix_pages=table)
    torch.cuda.synchronize()
    assert nat.device_status(clear=True) == 7
    keep = [j for j in range(n) if j // page not in gone]
    p.k[0], p.v[0], p.lengths = p.k[0][keep], p.v[0][keep], [len(keep)]
    _check(out, lse, q, c, 1.0, prefix=p)


@pytest.mark.parametrize("batch", [1, 33])
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("first", [0, 9000])
def test_long_tail_of_small_weights(first, bits, batch):
    """One token outweighs each of the others 2^25.5 times and has no value where they
    have theirs, so those elements are the sum of the tail.  Tolerance: a weight is
    fp16, of which the row's largest takes at least 2^7, so one of the tail is right
    to half of fp16's smallest number, 2^-32 of the largest; the output rounds once
    and 2^-9 covers the rest."""
    n, D = 16384, 64
    p = Cache([n], 1, D, bits, 64, seed=74)
    k, v = torch.zeros(n, 1, D), torch.ones(n, 1, D)
    k[first, 0] = 25.5 * np.log(2) / D
    v[first, 0, 1:] = 0
    _set(p, k, v, bits)
    q = torch.ones(batch, 1, 4, D, dtype=F16, device="cuda")
    out, lse, c = _over_prefix(p, q, 1.0, 0, bits)
    ref, rl, _, _ = oa.attention(q[0].double().cpu().numpy(), p.k[0], p.v[0], n, 1.0)
    assert 2.0 ** -12 < ref[0, 0, 1] < 2.0 ** -11
    err = np.abs(out[:, 0].double().cpu().numpy() - ref)
    tol = 2.0 ** -9 * np.abs(ref) + n * 2.0 ** -32
    assert (err <= tol).all(), float((err / tol).max())
    assert np.abs(lse[:, 0].double().cpu().numpy() - rl).max() < 1e-5
    # 64 sequences of the same pages, so that a warp of the register-fed kernel meets the
    # large token and hundreds of the others
    table = p.table.expand(64, -1).contiguous()
    lens = torch.full((64,), n, dtype=torch.int32, device="cuda")
    out = build("kvattention").forward(q[:1, 0].expand(64, -1, -1), p.pages, table, lens, scale=1.0)
    err = np.abs(out.double().cpu().numpy() - ref)
    assert (err <= tol).all(), float((err / tol).max())


@pytest.mark.parametrize("batch", [1, 33])
@pytest.mark.parametrize("top", [1.5 * 2.0 ** -6, 1.0, 1e20])
def test_bf16_rows_of_mixed_magnitudes(top, batch):
    """The row's largest element meets a zero of K, the others are 2^-20 of it and make
    the scores alone: they keep bf16's bits."""
    n, D = 600, 128
    g = torch.Generator().manual_seed(75)
    p = Cache([n], 1, D, 8, 64, seed=76)
    k, v = torch.randn(2, n, 1, D, generator=g)
    k[..., 0] = 0
    _set(p, k, v, 8)
    q = torch.randn(batch, 1, 4, D, generator=g) * (top * 2.0 ** -20)
    q[..., 0] = top
    q = q.to(BF16).cuda()
    scale = float(0.3 / (top * 2.0 ** -20))
    out, lse, c = _over_prefix(p, q, scale)
    _check(out, lse, q, c, scale, prefix=p)


def test_output_over_q_is_refused():
    c = Cache([20, 5], 1, 64, 8, 16, seed=87)
    q = _q(2, 1, 4, 64, F16, seed=88)[:, 0]
    att = build("kvattention")
    ref = att.forward(q, c.pages, c.table, c.len_tensor())
    with pytest.raises(RuntimeError, match="out must not overlap q"):
        att.forward_into(q, c.pages, c.table, c.len_tensor(), q)
    out = torch.empty_like(q)
    att.forward_into(q, c.pages, c.table, c.len_tensor(), out)
    assert torch.equal(out, ref)


def test_line_of_more_than_2_to_31_tokens():
    """64 sequences of 65536 tokens (the same pages) times 8 heads times 72 row tiles: the
    line that the CTAs cut counts 2.4 * 10^9 tokens.  Every sequence gives the same."""
    n, D, page, new, H, G = 65536, 64, 64, 144, 8, 8
    g = torch.Generator(device="cuda").manual_seed(89)
    cache, att = build("kvcache"), build("kvattention")
    pages = cache.empty(n // page, H, D, 4, page)
    k, v = torch.randn(2, n, H, D, device="cuda", generator=g).half()
    cache.write(k, v, pages, torch.arange(n, device="cuda"))
    q = torch.randn(1, new, H * G, D, device="cuda", generator=g).half()
    table = torch.arange(n // page, device="cuda", dtype=torch.int32).expand(64, -1).contiguous()
    lens = torch.full((64,), n, dtype=torch.int32, device="cuda")
    one, z = att.forward(q, pages, table[:1], lens[:1], return_lse=True)
    out, lse = att.forward(q.expand(64, -1, -1, -1), pages, table, lens, return_lse=True)
    # other cuts of the same sums: the weights' sums differ by fp32 roundings, the outputs
    # (0.02 and less) by one of fp16
    assert (lse - z).abs().max() < 1e-5
    assert (out.float() - one.float()).abs().max() < 2.0 ** -14
    ref = att.forward(q[:, -1:], pages, table[:1], lens[:1])
    assert (one[:, -1:].float() - ref.float()).abs().max() < 2.0 ** -14


@pytest.mark.parametrize("dtype", [F16, BF16], ids=str)
@pytest.mark.parametrize("D,bits", [(64, 8), (64, 4), (128, 8), (128, 4)])
@pytest.mark.parametrize("rows", [8, 9, 17])
@pytest.mark.parametrize("prefix", [1, 15, 63, 64, 65, 127, 128, 129, 257, 511])
def test_short_prefixes_of_few_rows(prefix, rows, D, bits, dtype):
    """Around the rule's 9 rows a head, and tiles that end in either half."""
    p = Cache([prefix], 2, D, bits, 32, seed=prefix)
    q = _q(rows, 1, 2, D, dtype, seed=prefix + rows)
    out, lse, c = _over_prefix(p, q, D ** -0.5, 1, bits)
    _check(out, lse, q, c, D ** -0.5, prefix=p)
