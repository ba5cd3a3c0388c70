"""ColumnShardedLMHead.topk where the kernel does not stand in: no candidate, a matmul of its own with other types or
with a gradient."""

import pytest
import torch

from mlxturbo_b200 import distributed as D

pytestmark = pytest.mark.gpu


def head_of(dtype):
    g = torch.Generator().manual_seed(0)
    w = torch.randn((64, 32), generator=g).to(dtype).cuda()
    none = torch.zeros((64, 1), device="cuda")
    head = D.ColumnShardedLMHead.from_full(w, none, none, matmul=lambda x, w, s, b, group_size, bits: x @ w.T)
    return head, w, torch.randn((3, 2, 32), generator=g).to(dtype).cuda()


@pytest.mark.parametrize("dtype", [torch.float64, torch.float32, torch.float16])
@pytest.mark.parametrize("k", [0, 1, 2, 7, 64, 100])
def test_types_and_sizes(dtype, k):
    head, w, x = head_of(dtype)
    values, ids = head.topk(x, k)
    logits = (x.reshape(-1, 32) @ w.T).reshape(3, 2, 64)
    want = torch.topk(logits.float(), min(k, 64), dim=-1)
    assert values.shape == ids.shape == (3, 2, min(k, 64)) and values.dtype == torch.float32
    assert torch.equal(values, want.values) and torch.equal(ids, want.indices)


def test_gradient_of_a_matmul_of_its_own():
    head, w, x = head_of(torch.float32)
    x.requires_grad_()
    values, _ = head.topk(x, 5)
    values.sum().backward()
    y = x.detach().clone().requires_grad_()
    torch.topk(y.reshape(-1, 32) @ w.T, 5, dim=-1).values.sum().backward()
    assert torch.equal(x.grad, y.grad)
    with torch.no_grad():
        assert torch.equal(head.topk(x, 5)[0], values.detach())
