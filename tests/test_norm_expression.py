"""The norm's defining expression on what the kernels take besides: no samples, no positions."""
import pytest
import torch


@pytest.mark.parametrize("shape", [(0, 8), (0, 5, 8), (3, 0, 8), (0, 0, 8)])
def test_empty_batches_under_a_transform(shape):
    from pde_amd import functional as K
    x = torch.empty(shape)
    y, g = torch.func.vjp(lambda t: K.group_norm_act(t, 2, torch.ones(8), torch.zeros(8), 1e-5, K.ACT_TANH), x)
    assert y.shape == x.shape and g(torch.ones_like(y))[0].shape == x.shape
