"""The attention half of a decoder layer, step by step through the public
operators (cudalab_b200.evaluator.decode_step), against the layer computed in
64 bits from the dequantised weights with an unquantised cache.

Bound: with int8 keys and values an element is off by at most half a step,
max|x| / 254, about 3 / 254 of its row's rms for rows of 128 normal values: 1.2 %
of the attention's output at most, which the output projection passes on; the
fp16 roundings in between are 2^-11 each.  2 % of the row's norm."""
import numpy as np
import pytest
import torch

from cudalab_b200 import _native as nat
from cudalab_b200.evaluator.decode_step import AttentionLayer
from cudalab_b200.int4gemv_quantize import dequantize_w
from oracle import attention_oracle as oa

pytestmark = pytest.mark.gpu
H, HQ, HK, D, EPS = 512, 8, 2, 64, 1e-5


def _w(pair):
    return dequantize_w(pair[0].cpu(), pair[1].cpu()).double().numpy()


class Plain:
    """The same layer in 64 bits; k and v of every token kept as they are."""

    def __init__(self, layer, prefix):
        self.layer, self.prefix = layer, prefix
        self.k = [[] for _ in range(layer.batch)]
        self.v = [[] for _ in range(layer.batch)]

    def step(self, x):
        L = self.layer
        x = x.double().cpu().numpy()
        n = x / np.sqrt((x * x).mean(-1, keepdims=True) + EPS) * L.norm.double().cpu().numpy()
        qkv = (n @ _w(L.w_qkv).T).reshape(len(x), -1, D)
        out = np.zeros((len(x), HQ * D))
        pre = 0 if self.prefix is None else len(self.prefix[0])
        for b in range(len(x)):
            pos = np.array([pre + len(self.k[b])])
            t = L.table.cpu().numpy()
            q = oa.qknorm_rope(qkv[b:b + 1, :HQ], L.q_norm.double().cpu().numpy(), t, pos, 1e-6, False)
            k = oa.qknorm_rope(qkv[b:b + 1, HQ:HQ + HK], L.k_norm.double().cpu().numpy(), t, pos,
                               1e-6, False)
            self.k[b].append(k[0])
            self.v[b].append(qkv[b, HQ + HK:])
            K, V = np.stack(self.k[b]), np.stack(self.v[b])
            if pre:
                K, V = np.concatenate((self.prefix[0], K)), np.concatenate((self.prefix[1], V))
            o = oa.attention(q, K, V, len(self.k[b]), D ** -0.5, prefix=pre)[0]
            out[b] = o[0].reshape(-1)
        return x + out @ _w(L.w_out).T


@pytest.mark.parametrize("prefix", [0, 37])
def test_steps(prefix):
    layer = AttentionLayer(3, H, HQ, HK, D, 64, 8, 16, prefix, seed=prefix)
    pre = None
    if prefix:
        k, v = torch.randn(2, prefix, HK, D, generator=torch.Generator().manual_seed(1)).half().cuda()
        layer.fill(k, v, None)
        pre = (k.double().cpu().numpy(), v.double().cpu().numpy())
    plain = Plain(layer, pre)
    g = torch.Generator().manual_seed(2)
    for _ in range(20):
        x = torch.randn(3, H, generator=g).half().cuda()
        y = layer.step(x).double().cpu().numpy()
        ref = plain.step(x)
        err = np.linalg.norm(y - ref, axis=-1) / np.linalg.norm(ref, axis=-1)
        assert (err < 0.02).all(), err
    assert layer.lengths.tolist() == [20, 20, 20]
    assert nat.device_status(clear=True) == 0


def test_step_in_a_graph_equals_eager():
    a = AttentionLayer(4, H, HQ, HK, D, 64, 4, 32, 0, seed=3)
    b = AttentionLayer(4, H, HQ, HK, D, 64, 4, 32, 0, seed=3)
    x = torch.randn(4, H, generator=torch.Generator().manual_seed(4)).half().cuda()
    first = a.step(x), b.step(x)
    assert torch.equal(*first)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = a.step(x)
    for _ in range(5):
        graph.replay()
        assert torch.equal(y, b.step(x))
