"""Paged steps of more sequences than the static batch, under tensor parallelism (no kernel runs)."""
from __future__ import annotations

from types import SimpleNamespace

import torch

from int4_b200 import decode
from int4_b200._lib import STATUS_SHAPE, Int4B200Error


def test_a_batch_beyond_the_exchange_buffers_leaves_the_fused_sums_on(monkeypatch):
    """The peers' exchange buffers hold max_batch rows.  A step of more rows is summed by NCCL; it must not make the
    library refuse, which would turn the fused sums off for every later step of the static batch too."""
    H, inter, max_batch = 16, 8, 2
    fused, summed = [], []

    def allreduce(peers, x, *q, prologue=0):
        if x.shape[0] * H > peers.capacity:
            raise Int4B200Error("w4a16_matmul_allreduce: refused", STATUS_SHAPE)
        fused.append(x.shape[0])
        return torch.zeros(x.shape[0], H)

    monkeypatch.setattr(decode, "w4a16_matmul_allreduce", allreduce)
    monkeypatch.setattr(decode, "w4a16_matmul_prologue", lambda kind, src, q, *a, **kw: torch.zeros(src.shape[0], q))
    monkeypatch.setattr(decode, "add_rmsnorm", lambda h, delta, weight, out, eps: out.copy_(h))

    class Layer:
        def __init__(self, n):
            self.q = (n, None, None)

        def __call__(self, x):
            return torch.zeros(x.shape[0], self.q[0])

    layer = {"ln1": None, "ln2": None, "qkv": Layer(24), "o": Layer(H), "gu": Layer(2 * inter), "down": Layer(H)}
    me = SimpleNamespace(embed=torch.zeros(5, H), nh_l=2, hd=8, device="cpu", inter_l=inter, w4=True, layers=[layer] * 2, eps=1e-5,
                         norm=None, hidden=H, max_batch=max_batch, peers=SimpleNamespace(capacity=max_batch * H), matmul_allreduce=True)
    me._matmul_allreduce_or_none = lambda *a: decode.LlamaTP._matmul_allreduce_or_none(me, *a)
    me._all_reduce = lambda x: summed.append(x.shape[0]) or x

    for B in (1, 3, 2, 32):
        fused.clear(), summed.clear()
        decode.LlamaTP._decode_layers_fused(me, torch.zeros(B, 1, dtype=torch.long), lambda i, qkv, att: None)
        assert me.matmul_allreduce, B
        assert (fused, summed) == (([B] * 4, []) if B <= max_batch else ([], [B] * 4))
