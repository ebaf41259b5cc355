"""The token operators where their definitions have corners: infinite scores, caps and limits of any size, calls that have to be refused."""
import math

import pytest
import torch

from tests.test_gpu_token_ops import TYPES, attention_inputs, ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("documents", [False, True])
@pytest.mark.parametrize("rows,keys", [(70, 70), (1, 3000), (900, 900)])
@pytest.mark.parametrize("value", [math.inf, -math.inf])
def test_attention_infinite_scores_are_not_numbers(dtype, documents, rows, keys, value):
    """A query whose seen scores are all infinite, or partly: its softmax is no number, in the result and in every gradient that it takes part
    in.  One that sees no key is zero, infinite or not.  (Rows by keys, split and not, and by rows.)"""
    token_attention = ops().token_attention
    H, Hk, D = 16 if rows == 900 else 2, 2, 32
    q, k, v, dout = attention_inputs(50, dtype, 1, rows, keys, H, Hk, D)
    k[0, :, 0, 5] = k[0, :, 0, 5].abs() + 0.25     # the first key head: every score has the sign of the query's channel 5
    r, G = rows // 2, H // Hk
    q[0, r, 0, 5] = value                          # all scores +inf, or all -inf
    q[0, r, G, 5] = value                          # the second key head: scores of both signs
    kw = {}
    if documents:
        ids_q = torch.full((1, rows), 3, device="cuda", dtype=torch.int32)
        ids_k = (torch.arange(keys, device="cuda", dtype=torch.int32) % 3 + 2)[None].contiguous()
        if rows > 1:
            q[0, 1] = value
            ids_q[0, 1], ids_q[0, 0] = 7, 7        # of a document without keys, one of the two infinite
        kw.update(q_docs=ids_q, k_docs=ids_k)
        seen = ids_k[0] == 3
    else:
        seen = torch.ones(keys, device="cuda", dtype=torch.bool)
    xs = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = token_attention(*xs, **kw)
    dq, dk, dv = torch.autograd.grad(out, xs, dout)
    none = torch.zeros(1, rows, H, dtype=torch.bool, device="cuda")
    none[0, r, 0] = none[0, r, G] = True
    for name, t in (("out", out), ("dq", dq), ("out without a graph", token_attention(q, k, v, **kw))):
        assert torch.equal(torch.isnan(t), none[..., None].expand_as(t)), name
        if documents and rows > 1:
            assert not t[0, :2].any(), name
    for name, t in (("dk", dk), ("dv", dv)):
        assert torch.isnan(t[0][seen]).all(), name
