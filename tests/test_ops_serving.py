"""The torch operator registrations of the serving calls: shapes and dtypes without running anything,
and on the GPU the Python calls' results bit for bit."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import w4a16 as K  # registers the operators


def test_fake_shapes():
    ops = torch.ops.w4a16
    with FakeTensorMode():
        q = torch.empty(3, 8, 64, dtype=torch.bfloat16)
        pages = torch.empty(9, 2, 16, 64, dtype=torch.bfloat16)
        i = torch.empty(3, dtype=torch.int32)
        y = ops.paged_attention(q, pages, pages, torch.empty(3, 4, dtype=torch.int32), i)
        assert y.shape == (3, 8, 64) and y.dtype == torch.bfloat16
        x = ops.process_logits(torch.empty(2, 100, dtype=torch.float16), bias=torch.empty(100))
        assert x.shape == (2, 100) and x.dtype == torch.float16


@pytest.mark.gpu
def test_operators_match_python_calls():
    k = torch.randn(9, 2, 16, 64, device="cuda").half()
    v = torch.randn_like(k)
    q = torch.randn(2, 8, 64, device="cuda").half()
    tables = torch.randperm(9, device="cuda").int()[:8].view(2, 4).contiguous()
    n = torch.tensor([50, 7], dtype=torch.int32, device="cuda")
    seqs = torch.tensor([1, 0], dtype=torch.int32, device="cuda")
    assert torch.equal(torch.ops.w4a16.paged_attention(q, k, v, tables, n, seqs, 0.2), K.paged_attention(q, k, v, tables, n, seqs=seqs, scale=0.2))
    x = torch.randn(2, 1000, device="cuda")
    t = torch.randint(0, 1000, (2, 30), device="cuda")
    r = torch.tensor([1.3, 0.9], device="cuda")
    assert torch.equal(torch.ops.w4a16.process_logits(x, t, repetition=r), K.process_logits(x, tokens=t, repetition=r))
