"""A recorded backward (create_graph=True) of a layer whose inputs depend on each other."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_weights_computed_from_one_another():
    """The recorded first derivatives are those of the kernels: the layer's own, to which the rest of the graph adds its part.

    Sums of 5 x 9 terms of about the same size either way, in another order: 64 steps of 2^-24 of the largest."""
    from pde_amd import KANLinear, functional as K
    torch.manual_seed(0)
    layer = KANLinear(5, 3, grid_size=6).cuda()
    grid, bw, sw, sc = layer._kernel_params()
    x = (torch.rand(40, 5, device="cuda") * 1.6 - 0.8).requires_grad_()
    root = torch.nn.Parameter(bw.detach().clone())
    parts = torch.randn(3, 5, sw.size(-1), device="cuda")

    def out():
        base = root * (1 + 0.1 * x.mean())
        return K.kan_layer(x, grid, base, parts * base.unsqueeze(-1), None, K.ACT_SILU, 6, 3)

    gy = torch.randn(40, 3, device="cuda")
    want = torch.autograd.grad(out(), (x, root), gy)
    got = torch.autograd.grad(out(), (x, root), gy, create_graph=True)
    for a, e in zip(got, want):
        assert float((a.detach() - e).abs().max()) <= 64 * 2.0 ** -24 * float(e.abs().max()) * 8      # (and 8 roundings a term)
