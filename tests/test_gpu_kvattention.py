"""Attention over the quantised paged cache (cl_kvattention) against the
formula in 64 bits on the values the cache holds; tolerances from the kernel's
roundings (oracle.attention_oracle.attention_tolerance)."""
import numpy as np
import pytest
import torch

from cudalab_b200 import _native as nat
from cudalab_b200.build import build
from oracle import attention_oracle as oa

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


class Cache:
    """`tokens` random tokens per sequence in shuffled pages, and their values."""

    def __init__(self, lengths, H, D, bits, page, seed, spread=0.5, scales=0.5):
        self.ext = build("kvcache")
        g = torch.Generator().manual_seed(seed)
        self.page, self.D, self.H = page, D, H
        width = max(1, max(-(-n // page) for n in lengths))
        total = len(lengths) * width + 2
        order = torch.randperm(total, generator=g)
        self.table = order[:len(lengths) * width].view(len(lengths), width).int().cuda()
        self.pages = self.ext.empty(total, H, D, bits, page)
        # what no token was written to holds NaN scales and arbitrary bytes
        self.pages.fill_(0xFF)
        self.lengths = list(lengths)
        self.k, self.v = [], []
        for b, n in enumerate(lengths):
            k = torch.randn(n, H, D, generator=g) * torch.exp(spread * torch.randn(n, H, 1, generator=g))
            v = torch.randn(n, H, D, generator=g) * torch.exp(scales * torch.randn(n, H, 1, generator=g))
            j = torch.arange(n)
            slots = (self.table[b].cpu().long()[j // page] * page + j % page).cuda()
            k, v = k.half().cuda(), v.half().cuda()
            self.ext.write(k, v, self.pages, slots)
            vals = []
            for x in (k, v):
                q, s = oa.quantise(x.float().cpu().numpy(), bits)
                vals.append(q.astype(np.float64) * s.astype(np.float64)[..., None])
            self.k.append(vals[0])
            self.v.append(vals[1])

    def len_tensor(self):
        return torch.tensor(self.lengths, dtype=torch.int32, device="cuda")


def _q(B, n, Hq, D, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (scale * torch.randn(B, n, Hq, D, generator=g)).to(dtype).cuda()


def _check(out, lse, q, c, scale, window=0, prefix=None):
    """q, out [B, n, Hq, D], lse [B, n, Hq]."""
    out, lse = out.double().cpu().numpy(), lse.double().cpu().numpy()
    bits = 11 if q.dtype == F16 else 8
    for b, n in enumerate(c.lengths):
        k, v, pre = c.k[b], c.v[b], 0
        if prefix is not None:
            k, v, pre = (np.concatenate((prefix.k[0], k)), np.concatenate((prefix.v[0], v)),
                         prefix.lengths[0])
        ref, rl, pv, mag = oa.attention(q[b].double().cpu().numpy(), k, v, n, scale, window, pre)
        tokens, vmax = len(k), np.abs(v).max() if len(v) else 0.0
        tol = oa.attention_tolerance(ref, pv, mag, vmax, tokens, q.shape[-1], bits)
        err = np.abs(out[b] - ref)
        assert (err <= tol).all(), (b, n, float((err / tol).max()))
        assert np.array_equal(np.isinf(rl), np.isinf(lse[b])), (b, n)
        fin = np.isfinite(rl)
        ltol = oa.lse_tolerance(rl, mag, tokens, q.shape[-1])
        assert (np.abs(lse[b][fin] - rl[fin]) <= ltol[fin]).all(), (b, n)
    assert nat.device_status(clear=True) == 0


# every head_dim and format, lengths around the block, the page and the split
LENGTHS = [0, 1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 200, 517]


@pytest.mark.parametrize("dtype", [F16, BF16], ids=str)
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("group", [1, 5, 8, 12])
def test_lengths_and_formats(group, D, bits, dtype):
    c = Cache(LENGTHS, 2, D, bits, 32, seed=D + bits + group)
    q = _q(len(LENGTHS), 1, 2 * group, D, dtype, seed=group)
    att = build("kvattention")
    ws = att.workspace()
    for _ in range(2):  # the second call meets the workspace the first one left
        out, lse = att.forward(q[:, 0], c.pages, c.table, c.len_tensor(), workspace=ws,
                               return_lse=True)
        _check(out[:, None], lse[:, None], q, c, D ** -0.5)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("lengths", [[1] * 8, list(range(1, 10))], ids=["one", "few"])
def test_log_sum_exp_of_few_tokens(lengths, D, bits):
    """Few tokens, so nothing averages out: the log-sum-exp over all rows is
    within 1e-6 of itself.  Some ten roundings to 24 bits (the products' sum, the
    bias taken off, the scales' logarithm and its power, the sum, its logarithm)
    of numbers up to 8, each 8 2^-24 / sqrt(3) on average, are 0.9e-6 together,
    beside values of root mean square 1 and more."""
    c = Cache(lengths, 4, D, bits, 16, seed=D + bits, spread=0.0, scales=0.0)
    q = _q(len(lengths), 1, 32, D, F16, seed=D)
    out, lse = build("kvattention").forward(q, c.pages, c.table, c.len_tensor(), return_lse=True)
    _check(out, lse, q, c, D ** -0.5)
    ref = np.stack([oa.attention(q[b].double().cpu().numpy(), c.k[b], c.v[b], n, D ** -0.5, 0, 0)[1]
                    for b, n in enumerate(lengths)])
    off = lse.double().cpu().numpy() - ref
    assert np.linalg.norm(off) <= 1e-6 * np.linalg.norm(ref)


@pytest.mark.parametrize("n,window", [(2, 0), (5, 0), (1, 16), (1, 1), (4, 7), (8, 100), (3, 5000)])
@pytest.mark.parametrize("D,bits,page", [(64, 8, 16), (128, 4, 64), (256, 8, 48)])
def test_new_tokens_and_windows(D, bits, page, n, window):
    """Rows in front of a sequence's first token see nothing: zeros and -inf."""
    c = Cache([0, 1, 3, 8, 50, 300], 2, D, bits, page, seed=n + window + D)
    q = _q(6, n, 6, D, F16, seed=n)
    out, lse = build("kvattention").forward(q, c.pages, c.table, c.len_tensor(), window=window,
                                            return_lse=True)
    _check(out, lse, q, c, D ** -0.5, window)
    for b, length in enumerate(c.lengths):
        for i in range(n):
            if length - n + i < 0:
                assert torch.count_nonzero(out[b, i]) == 0 and (lse[b, i] == float("-inf")).all()


@pytest.mark.parametrize("D,bits", [(64, 4), (128, 8), (256, 4)])
def test_long_sequence_split_over_many_ctas(D, bits):
    """One head of one long sequence: every CTA holds a part of it, the parts
    are joined in two levels, and a second call gives the same bits."""
    c = Cache([20011], 1, D, bits, 64, seed=D)
    q = _q(1, 1, 4, D, F16, seed=5, scale=2.0)
    att = build("kvattention")
    ws = att.workspace()
    out, lse = att.forward(q, c.pages, c.table, c.len_tensor(), workspace=ws, return_lse=True)
    _check(out, lse, q, c, D ** -0.5)
    again = att.forward(q, c.pages, c.table, c.len_tensor(), workspace=ws)
    assert torch.equal(again, out)


def test_many_sequences():
    lengths = [(7 * i) % 90 for i in range(300)]
    c = Cache(lengths, 1, 64, 8, 16, seed=11)
    q = _q(300, 1, 3, 64, F16, seed=12)
    out, lse = build("kvattention").forward(q, c.pages, c.table, c.len_tensor(), return_lse=True)
    _check(out, lse, q, c, 64 ** -0.5)


def test_scales_of_every_size():
    """Values and keys whose scales span fp16: weights stay accurate because the
    softmax reference carries the scale."""
    c = Cache([700, 40], 2, 128, 8, 64, seed=13, spread=1.5, scales=3.0)
    q = _q(2, 1, 8, 128, F16, seed=14, scale=3.0)
    out, lse = build("kvattention").forward(q, c.pages, c.table, c.len_tensor(), return_lse=True)
    _check(out, lse, q, c, 128 ** -0.5)


def test_large_and_small_bf16_queries():
    c = Cache([300, 5], 1, 128, 8, 16, seed=15)
    for size in (1e-20, 1e30):
        q = _q(2, 1, 8, 128, BF16, seed=16, scale=size)
        scale = 0.1 / size
        out, lse = build("kvattention").forward(q, c.pages, c.table, c.len_tensor(), scale=scale,
                                                return_lse=True)
        _check(out, lse, q, c, scale)


def test_scale_argument_and_strided_q():
    c = Cache([90, 33, 1], 2, 128, 8, 32, seed=17)
    att = build("kvattention")
    qkv = _q(3, 2, 12, 131, F16, seed=18)
    q = qkv[:, :, 2:10, 1:129]  # odd strides: element accesses
    out, lse = att.forward(q, c.pages, c.table, c.len_tensor(), scale=0.3, return_lse=True)
    _check(out, lse, q, c, 0.3)
    same = torch.empty_like(out)
    att.forward_into(q.contiguous(), c.pages, c.table, c.len_tensor(), same, scale=0.3)
    assert torch.equal(same, out)


def test_nan_and_inf_stay_in_their_row():
    c = Cache([40, 40], 1, 128, 8, 16, seed=19)
    q = _q(2, 1, 8, 128, F16, seed=20)
    att = build("kvattention")
    clean = att.forward(q, c.pages, c.table, c.len_tensor())
    q[0, 0, 3, 7] = float("nan")
    q[1, 0, 5, 9] = float("inf")
    out, lse = att.forward(q, c.pages, c.table, c.len_tensor(), return_lse=True)
    bad = torch.isnan(out).any(-1)
    assert bad.sum() == 2 and bad[0, 0, 3] and bad[1, 0, 5]
    assert torch.isnan(lse[0, 0, 3])
    assert torch.equal(out[~bad], clean[~bad])


@pytest.mark.parametrize("dtype", [F16, BF16], ids=str)
@pytest.mark.parametrize("D,bits,group,n", [(64, 8, 1, 1), (128, 8, 8, 1), (128, 4, 4, 3),
                                            (256, 8, 2, 2), (64, 4, 16, 1)])
@pytest.mark.parametrize("prefix", [1, 16, 100, 1037])
def test_shared_prefix(prefix, D, bits, group, n, dtype):
    p = Cache([prefix], 2, D, bits, 32, seed=prefix)
    c = Cache([0, 1, 40, 7, 133], 2, D, bits, 32, seed=prefix + 1)
    # one cache: the prefix's pages behind the sequences'
    pages = torch.cat((c.pages, p.pages))
    prefix_pages = p.table[0] + c.pages.shape[0]
    q = _q(5, n, 2 * group, D, dtype, seed=prefix + 2)
    att = build("kvattention")
    out, lse = att.forward_shared(q, pages, prefix_pages, prefix, c.table, c.len_tensor(),
                                  workspace=att.workspace(), return_lse=True)
    _check(out, lse, q, c, D ** -0.5, prefix=p)
    none = att.forward_shared(q, pages, prefix_pages, 0, c.table, c.len_tensor())
    assert torch.equal(none, att.forward(q, pages, c.table, c.len_tensor()))


# The tensor-core prefix kernel (from 32 rows and 512 tokens): rows around its
# 128-row tiles, lengths around its 128-token tiles and the parts they are cut
# into, every format, one and several new tokens.
@pytest.mark.parametrize("dtype", [F16, BF16], ids=str)
@pytest.mark.parametrize("D,bits", [(64, 8), (64, 4), (128, 8), (128, 4)])
@pytest.mark.parametrize("batch,n,group,prefix", [(32, 1, 1, 512), (16, 1, 8, 513), (43, 1, 3, 640),
                                                  (9, 3, 5, 1000), (65, 1, 4, 2049)])
def test_shared_prefix_on_tensor_cores(batch, n, group, prefix, D, bits, dtype):
    p = Cache([prefix], 1, D, bits, 48, seed=prefix, spread=1.0, scales=1.0)
    c = Cache([i % 4 for i in range(batch)], 1, D, bits, 48, seed=prefix + 1)
    pages = torch.cat((c.pages, p.pages))
    q = _q(batch, n, group, D, dtype, seed=prefix + 2, scale=2.0)
    att = build("kvattention")
    out, lse = att.forward_shared(q, pages, p.table[0] + c.pages.shape[0], prefix, c.table,
                                  c.len_tensor(), workspace=att.workspace(), return_lse=True)
    _check(out, lse, q, c, D ** -0.5, prefix=p)


def test_shared_prefix_large_and_small_queries():
    """bf16 rows outside fp16's range, rows of zeros and a NaN, beside ordinary ones."""
    p = Cache([600], 1, 128, 8, 64, seed=31)
    c = Cache([2] * 40, 1, 128, 8, 64, seed=32)
    pages = torch.cat((c.pages, p.pages))
    q = _q(40, 1, 2, 128, BF16, seed=33)
    q[1], q[2], q[3] = q[1] * 1e30, q[2] * 1e-30, 0
    att = build("kvattention")
    args = (pages, p.table[0] + c.pages.shape[0], 600, c.table, c.len_tensor())
    scale = 1e-30  # the large rows then have ordinary scores, the others none to speak of
    out, lse = att.forward_shared(q, *args, scale=scale, return_lse=True)
    _check(out, lse, q, c, scale, prefix=p)
    q = _q(40, 1, 2, 128, BF16, seed=34)
    clean = att.forward_shared(q, *args)
    q[7, 0, 1, 5] = float("nan")
    out = att.forward_shared(q, *args)
    bad = torch.isnan(out).any(-1)
    assert bad.sum() == 1 and bad[7, 0, 1] and torch.equal(out[~bad], clean[~bad])


def test_shared_prefix_rising_scores():
    """Scores that grow along the prefix move the softmax reference at every tile, and one
    late token outweighs all before it."""
    n, D = 1300, 128
    p = Cache([n], 1, D, 8, 64, seed=41)
    c = Cache([1] * 33, 1, D, 8, 64, seed=42)
    g = torch.Generator().manual_seed(43)
    d = torch.randn(D, generator=g)
    k = torch.randn(n, 1, D, generator=g) * 0.1 + d * torch.linspace(-1, 1, n)[:, None, None]
    k[1200] = 6 * d
    j = torch.arange(n)
    slots = p.table[0].cpu().long()[j // 64] * 64 + j % 64
    p.ext.write(k.half().cuda(), torch.from_numpy(p.v[0]).half().cuda(), p.pages, slots.cuda())
    qk, s = oa.quantise(k.half().float().numpy(), 8)
    p.k[0] = qk.astype(np.float64) * s.astype(np.float64)[..., None]
    qv, s = oa.quantise(torch.from_numpy(p.v[0]).half().float().numpy(), 8)
    p.v[0] = qv.astype(np.float64) * s.astype(np.float64)[..., None]
    pages = torch.cat((c.pages, p.pages))
    q = (d + 0.3 * torch.randn(33, 1, 4, D, generator=g)).half().cuda()
    att = build("kvattention")
    out, lse = att.forward_shared(q, pages, p.table[0] + c.pages.shape[0], n, c.table,
                                  c.len_tensor(), scale=0.4, return_lse=True)
    _check(out, lse, q, c, 0.4, prefix=p)


def test_shared_prefix_in_a_graph_and_on_another_stream():
    p = Cache([700], 2, 128, 4, 32, seed=51)
    c = Cache([i % 50 for i in range(24)], 2, 128, 4, 32, seed=52)
    pages = torch.cat((c.pages, p.pages))
    q = _q(24, 1, 8, 128, F16, seed=53)
    att = build("kvattention")
    ws = att.workspace()
    args = (pages, p.table[0] + c.pages.shape[0], 700, c.table, c.len_tensor())
    ref = att.forward_shared(q, *args, workspace=ws)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            # q written by the kernel before: the launches must wait for it
            q2 = q * 1.0
            out = att.forward_shared(q2, *args, workspace=ws)
        for _ in range(5):
            q.neg_()
            graph.replay()
        q.neg_()
        graph.replay()
    s.synchronize()
    assert torch.equal(out, ref)


def test_index_errors_are_recorded():
    """A page outside the cache is skipped, a length beyond the table clamped."""
    c = Cache([64, 20], 1, 128, 8, 16, seed=21)
    q = _q(2, 1, 8, 128, F16, seed=22)
    att = build("kvattention")
    table = c.table.clone()
    table[0, 1] = c.pages.shape[0]
    table[0, 2] = -1
    out = att.forward(q, c.pages, table, c.len_tensor())
    torch.cuda.synchronize()
    assert nat.device_status(clear=True) == 7 and torch.isfinite(out).all()
    keep = np.r_[0:16, 48:64]
    ref, _, pv, mag = oa.attention(q[0].double().cpu().numpy(), c.k[0][keep], c.v[0][keep], 32,
                                   128 ** -0.5)
    tol = oa.attention_tolerance(ref, pv, mag, np.abs(c.v[0]).max(), 64, 128, 11)
    assert (np.abs(out[0].double().cpu().numpy() - ref) <= tol).all()
    lengths = torch.tensor([64, 10 ** 6], dtype=torch.int32, device="cuda")
    att.forward(q, c.pages, c.table, lengths)
    torch.cuda.synchronize()
    assert nat.device_status(clear=True) == 7


def test_other_stream_and_graph():
    c = Cache([500, 77, 0], 2, 128, 8, 64, seed=23)
    q = _q(3, 1, 16, 128, F16, seed=24)
    att = build("kvattention")
    ws, lens = att.workspace(), c.len_tensor()
    ref = att.forward(q, c.pages, c.table, lens, workspace=ws)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y = att.forward(q, c.pages, c.table, lens, workspace=ws)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            z = att.forward(q, c.pages, c.table, lens, workspace=ws)
        for _ in range(3):
            g.replay()
    s.synchronize()
    assert torch.equal(y, ref) and torch.equal(z, ref)


def test_empty_batch():
    c = Cache([3], 1, 64, 8, 16, seed=25)
    q = torch.empty(0, 2, 64, dtype=F16, device="cuda")
    out = build("kvattention").forward(q, c.pages, c.table[:0], c.len_tensor()[:0])
    assert out.shape == (0, 2, 64)


def test_cache_beyond_32_bits():
    """A cache of more than 4 GiB gives its far pages' tokens the bits that the
    same pages give in a small one: written, read, attended to, and shared."""
    H, D, page = 8, 128, 64
    c = Cache([700, 130], H, D, 8, page, seed=61)
    first = 40000 - c.pages.shape[0]
    far = c.ext.empty(40000, H, D, 8, page)
    assert first * far[0].numel() > 1 << 32
    slots = (c.table[0].long()[:, None] * page + torch.arange(page, device="cuda")).flatten()[:700]
    k, v = c.ext.read(c.pages, slots, D)
    c.ext.write(k, v, far, slots + first * page)
    for x, y in zip(c.ext.read(far, slots + first * page, D), c.ext.read(c.pages, slots, D)):
        assert torch.equal(x, y)
    far[first:] = c.pages
    q = _q(2, 1, 64, D, F16, seed=62)
    att = build("kvattention")
    args = (c.len_tensor(),)
    assert torch.equal(att.forward(q, far, c.table + first, *args),
                       att.forward(q, c.pages, c.table, *args))
    q = _q(8, 1, 64, D, F16, seed=63)  # 64 rows a head: the tensor-core prefix kernel
    lens = torch.tensor([0, 1, 17, 64, 100, 3, 5, 64], dtype=torch.int32, device="cuda")
    table = c.table[1:].expand(8, -1).contiguous()
    assert torch.equal(att.forward_shared(q, far, c.table[0] + first, 700, table + first, lens),
                       att.forward_shared(q, c.pages, c.table[0], 700, table, lens))
    assert nat.device_status(clear=True) == 0
