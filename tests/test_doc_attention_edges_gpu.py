"""Attention over packed documents at the edges of its calls; references and bounds of test_doc_attention_gpu."""
import math

import pytest
import torch

from test_doc_attention_gpu import BF, offsets

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,kv_heads,keys", [(8, 8, 384), (8, 2, 5000), (32, 1, 384), (2, 2, 3)])
def test_no_queries_over_keys(heads, kv_heads, keys):
    from image_generator_amd import ops
    d = 96
    k, v = (torch.randn(keys, kv_heads * d, device="cuda").to(BF).requires_grad_(True) for _ in range(2))
    q = torch.empty(0, heads * d, device="cuda", dtype=BF, requires_grad=True)
    none, off = offsets([0, 0]).cuda(), offsets([keys // 2, keys - keys // 2]).cuda()
    out, lse = ops.doc_attention_fwd(q, k, v, heads=heads, kv_heads=kv_heads, q_offsets=none, k_offsets=off)
    assert out.shape == (0, heads * d) and lse.shape == (heads, 0)
    out = ops.doc_attention(q, k, v, heads=heads, kv_heads=kv_heads, q_offsets=none, k_offsets=off)
    out.sum().backward()
    assert q.grad.shape == q.shape and bool((k.grad == 0).all()) and bool((v.grad == 0).all())
