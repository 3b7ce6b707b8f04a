"""Calls of the operators over feature rows that their documentation allows, beyond those of test_decoder_ops_gpu.py."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def ops():
    from neuralgaussiansplatting_amd import decoder_ops
    return decoder_ops


def test_dropout_of_a_long_flat_tensor(ops):
    """More than 2^31 elements in one dimension: the mask is a function of the element's number, so it is that of the same
    elements as rows (which test_far_offsets compares with the definition)."""
    x = torch.ones((1 << 31) + 24, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    y = ops.dropout(x, 0.5, 3)
    assert torch.equal(y.detach().view(-1, 8), ops.dropout(x.detach().view(-1, 8), 0.5, 3))
    (dx,) = torch.autograd.grad(y, [x], x.detach())
    assert torch.equal(dx, y.detach())
