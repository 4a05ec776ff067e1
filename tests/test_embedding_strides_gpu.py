"""Gradients of embedding rows whose strides come from elsewhere: autograd's zero tensors are filled in with strides of 0, and an op is called with any."""

from __future__ import annotations

import pytest
import torch

from skyrl_amd import embedding as E

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_gradient_that_is_autograds_zero_tensor(cuda_device, dtype):
    weight = torch.randn(50, 24, device=cuda_device, dtype=dtype, requires_grad=True)
    ids = torch.randint(0, 50, (37,), device=cuda_device)
    zero = torch._efficientzerotensor((37, 24), device=cuda_device, dtype=dtype)
    for out in (E.embedding_lookup(weight, ids), E._Lookup.apply(weight, ids, 1.0, -1)):
        (grad,) = torch.autograd.grad(out, weight, zero)
        assert grad.shape == weight.shape and not grad.any()


def test_the_op_takes_rows_of_any_strides(cuda_device):
    ids = torch.randint(0, 50, (37,), device=cuda_device)
    d = torch.randn(37, 24, device=cuda_device)
    for rows in (d.t().contiguous().t(), d[:, :1].expand(37, 24), d[:1, :1].expand(37, 24), torch.cat([d, d], 1)[:, ::2], d.as_strided((37, 24), (3, 1))):
        assert torch.equal(E.lmhead_embedding_bwd(rows, ids, 50, 1.0, -1), E.lmhead_embedding_bwd(rows.contiguous(), ids, 50, 1.0, -1))
