"""The norm with an activation where few bits, long sums, wide rows or dependent parameters could tell."""
import pytest
import torch

from test_gpu_norm import _definition, _kind, _repeats_match, _with_gradients

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _mean(t):
    """Over the first dimension, in stages of at most 1024 terms, each of many results: no reduction is split over blocks."""
    n = t.size(0)
    while t.size(0) > 1:
        step = min(1024, t.size(0))
        t = torch.cat([t, t.new_zeros(-t.size(0) % step, *t.shape[1:])]).view(-1, step, *t.shape[1:]).sum(1)
    return t[0] / n


def _statistics(x, groups, eps=1e-5):
    """The forward's own (mean, r) of each sample and group."""
    from pde_amd import functional as K
    _, stats = K._group_norm_forward(x, None, None, groups, eps, K.ACT_IDENTITY, True)
    return stats.view(x.size(0), groups, 2)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,s,c,groups,first,rest", [
    (64, 1 << 21, 8, 2, 0.0, 1e3), (64, 1 << 21, 8, 2, 0.0, 1e4), (512, 1 << 14, 8, 2, 0.0, 1e4), (512, 1 << 18, 4, 1, 0.0, 1e4),
    (512, 4096, 1024, 8, 30.0, 0.0), (512, 4096, 1024, 8, 1000.0, 0.0), (512, 4096, 257, 1, 1000.0, 0.0), (1, 1 << 20, 6, 3, 0.0, 1e4),
    (3, 5000, 90, 6, -1e4, 1e4), (600, 100, 24, 3, 1e4, 0.0)])
def test_a_first_position_far_from_the_rest(n, s, c, groups, first, rest, dtype):
    """Statistics of samples whose first position (a boundary value, say) stands apart, over chunks of any length.

    The sums are 64-bit: what is left are the roundings of the mean (2^-24) and of r (the variance's two and 2^-23 of the reciprocal
    root: 3 2^-24)."""
    gen = torch.Generator(device="cuda").manual_seed(n + s)
    x = torch.empty(n, s, c, device="cuda", dtype=dtype)
    for part in x.split(max(1, (1 << 26) // (s * c))):
        part.copy_(rest + torch.randn(part.shape, device="cuda", generator=gen))
    x[:, 0] = first
    got = _statistics(x, groups).double()
    for i in {0, n // 2, n - 1}:
        v = x[i].double().view(s, groups, c // groups)
        mean = _mean(v).mean(1)
        var = _mean((v - mean[:, None]).square()).mean(1)
        r = 1 / (var + 1e-5).sqrt()
        spread = _mean((v - mean[:, None]).abs()).mean(1)
        assert bool(((got[i, :, 0] - mean).abs() <= 1.1 * U * mean.abs() + 1e-9 * spread).all())
        rel = (got[i, :, 1] / r - 1).abs()
        assert bool((rel <= 3.2 * U).all()), (float(rel.max()), float(var.min()))
    del x
    torch.cuda.empty_cache()


@pytest.mark.parametrize("n,s,c,groups,dtype", [(512, 8192, 257, 1, torch.float32), (700, 4096, 64, 8, torch.float32),
                                                (513, 2048, 2048, 16, torch.bfloat16), (2, 1 << 21, 12, 2, torch.float16)])
def test_long_sums_of_the_backward(n, s, c, groups, dtype):
    """A constant cotangent, whose roundings all go one way in a long chain of additions: chains of 32 terms, the rest in 64 bits.

    gb is the sum of n s terms, 32 steps off at most in a chain, one more where a chunk's sum and the result are rounded.  gx is
    r (q - mean q - z mean(q z)) with q constant: nothing but the errors of the means, at most 34 steps of q and |z| times 34 steps
    of mean |z q|, and a rounding of each operand."""
    from pde_amd import functional as K
    gen = torch.Generator(device="cuda").manual_seed(s)
    x = torch.empty(n, s, c, device="cuda", dtype=dtype)
    for part in x.split(max(1, (1 << 26) // (s * c))):
        part.copy_(torch.randn(part.shape, device="cuda", generator=gen))
    x.requires_grad_()
    b = torch.zeros(c, device="cuda", requires_grad=True)
    y = K.group_norm_act(x, groups, None, b, 1e-5, K.ACT_IDENTITY)
    top = float(y.detach().abs().amax())
    gy = torch.full((), 0.1, device="cuda", dtype=dtype).expand(y.shape)
    del y
    gx, gb = torch.autograd.grad(K.group_norm_act(x, groups, None, b, 1e-5, K.ACT_IDENTITY), (x, b), gy)
    q = float(gy[0, 0, 0])
    want = q * n * s
    assert float((gb.double() - want).abs().max()) <= 36 * U * want
    # r of N(0, 1) data is 1 within a percent or so (samples of 2048 values at least); half a step of a 16-bit result besides
    bound = 1.1 * q * U * (40 + 40 * top) * (1 + top) * (1 + torch.finfo(dtype).eps)
    assert float(gx.abs().amax()) <= bound, (float(gx.abs().amax()), bound)
    del x, gx, gy
    torch.cuda.empty_cache()


@pytest.mark.parametrize("act", ["identity", "silu", "tanh"])
@pytest.mark.parametrize("shape", [(6, 32), (3, 20, 32), (3, 500, 32), (2, 20000, 32), (600, 70, 32)])
def test_all_of_a_non_finite_group_is_nan(shape, act):
    """Its mean is not finite, so nothing of the group has a value: no saturated activation stands in for one."""
    from pde_amd import functional as K
    gen = torch.Generator(device="cuda").manual_seed(4)
    x = torch.randn(*shape, device="cuda", generator=gen)
    for place in (0, -1):
        for bad in (float("nan"), float("inf"), -float("inf")):
            z = x.clone()
            z[(1, *[place] * (len(shape) - 2), 9)] = bad
            z.requires_grad_()
            y = K.group_norm_act(z, 4, None, None, 1e-5, _kind(act))
            gx, = torch.autograd.grad(y, z, torch.ones_like(y))
            for t in (y, gx):
                assert bool(t[1, ..., 8:16].isnan().all())
                assert bool(t[0].isfinite().all()) and bool(t[1, ..., :8].isfinite().all()) and bool(t[1, ..., 16:].isfinite().all())


@pytest.mark.parametrize("act", ["silu", "tanh"])
def test_activations_value_by_value(act):
    """With weights of zero the value is act(bias) and the bias' gradient its slope, each compared on its own.

    In steps of 2^-24.  tanh: below 0.625 a polynomial (its fit 0.1) with three roundings at the end; above, 1 - q, q =
    2 / (exp(2|u|) + 1): q is off by 2 of the exponential and 1 of its last rounding, 1 of the sum and of the quotient: 5 of q <=
    0.45, one of the result >= 0.55: 5 in all.  Its slope q (2 - q): 5 of q, 1 of 2 - q and of the product, 1 - t^2 below: 7.
    silu: u s, s = 1 / (1 + exp(-u)): exponential 3, sum 1, quotient 2, product 1: 7; the slope s + u s (1 - s) cancels near
    its zero at -1.28, so it is compared with the magnitudes of its terms: s 6, 1 - s 7 (itself below 0, where it is 1/2 at
    least, exp(-u) s above: 10), their product 17, the sum 18."""
    from pde_amd import functional as K
    b = torch.cat([torch.linspace(-1, 1, 4000), torch.linspace(-12, 12, 2000), torch.linspace(-80, 80, 2000),
                   torch.logspace(-30, 0, 192)]).cuda().requires_grad_()
    x = torch.randn(1, b.numel(), device="cuda")
    y = K.group_norm_act(x, b.numel() // 2, torch.zeros_like(b), b, 1e-5, _kind(act))
    slope, = torch.autograd.grad(y.sum(), b)
    u = b.detach().double()
    t, s = torch.tanh(u), torch.sigmoid(u)
    if act == "tanh":
        want, steep, scale, steps = t, 1 / torch.cosh(u) ** 2, 1 / torch.cosh(u) ** 2, (5, 7)
    else:
        want, steep, scale, steps = u * s, s + u * s * (1 - s), s + u.abs() * s * torch.sigmoid(-u), (7, 18)
    tiny = 2.0 ** -121                                            # the slope where exp(2|u|) nearly leaves fp32's range
    assert bool(((y[0].double() - want).abs() <= steps[0] * U * want.abs() + tiny).all()), \
        float(((y[0].double() - want).abs() / (U * want.abs() + tiny)).max())
    assert bool(((slope.double() - steep).abs() <= steps[1] * U * scale + tiny).all()), \
        float(((slope.double() - steep).abs() / (U * scale + tiny)).max())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("c,groups", [(8192, 1), (8192, 8192), (8191, 1), (7810, 2), (6000, 5)])
def test_the_widest_channels(c, groups, dtype):
    """Up to 8192 channels at every alignment: the statistics' 16 bytes a channel and the kernel's own LDS fit together."""
    from pde_amd import functional as K
    for shape in ((3, c), (2, 40, c)):
        x = torch.randn(*shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(c)).to(dtype).requires_grad_()
        y = K.group_norm_act(x, groups)
        gx, = torch.autograd.grad(y, x, torch.ones_like(y))
        ones, zeros = torch.ones(c, device="cuda").double(), torch.zeros(c, device="cuda").double()
        want = _definition(x.detach().double(), ones, zeros, groups, 1e-5, "identity")
        # half a step of the type, the roundings of the mean, the deviation, r and the product, of N(0, 1) data: 8 2^-24 of the scale
        assert float((y.detach().double() - want).abs().max()) <= (8 * U + torch.finfo(dtype).eps / 2) * max(1.0, float(want.abs().max()))
        # (a constant cotangent gives no gradient: r times the roundings of the means, 40 2^-24 each and |z| times that; r is near 1,
        # 316 where a group is a single value)
        assert float(gx.abs().max()) <= 2 * 80 * U * (1 + float(want.abs().max())) ** 2 * (1 if groups < c else 400)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape,groups", [((5000, 1536), 2), ((2049, 4100), 1), ((3000, 2, 384), 1), ((2500, 33, 40), 5), ((2048, 600), 1),
                                          ((20, 8192), 1), ((9000, 3, 257), 1)])
def test_wide_rows_and_many_samples(shape, groups, dtype):
    """More samples than the backward's blocks: each block adds up those it takes.  All gradients against the definition."""
    from pde_amd import functional as K
    gen = torch.Generator(device="cuda").manual_seed(3)
    c = shape[-1]
    x = torch.randn(*shape, device="cuda", generator=gen).to(dtype).requires_grad_()
    gy = torch.randn(*shape, device="cuda", generator=gen).to(dtype)
    w = (1 + 0.2 * torch.randn(c, device="cuda", generator=gen)).requires_grad_()
    b = (0.2 * torch.randn(c, device="cuda", generator=gen)).requires_grad_()
    y = K.group_norm_act(x, groups, w, b, 1e-5, K.ACT_TANH)
    gx, gw, gb = torch.autograd.grad(y, (x, w, b), gy)
    leaves = [t.detach().double().requires_grad_() for t in (x, w, b)]
    want = _definition(*leaves, groups, 1e-5, "tanh")
    ex, ew, eb = torch.autograd.grad(want, leaves, gy.double())
    half = torch.finfo(dtype).eps / 2
    # N(0, 1) data: each value and each term of a sum a few steps of magnitudes of at most a few; in the 2-norm 16 steps
    for got, e in ((y, want.detach()), (gx, ex)):
        assert float((got.double() - e).norm() / e.norm()) <= 16 * U + half
    for got, e in ((gw, ew), (gb, eb)):
        assert float((got.double() - e).norm() / e.norm()) <= 32 * U
    alone, = torch.autograd.grad(K.group_norm_act(x, groups, w.detach(), b.detach(), 1e-5, K.ACT_TANH), x, gy)
    assert torch.equal(alone, gx)                                 # without the parameters' gradients: the same
    only, = torch.autograd.grad(K.group_norm_act(x, groups, w.detach(), b, 1e-5, K.ACT_TANH), b, gy)
    assert torch.equal(only, gb)


def test_a_recorded_backward_of_parameters_that_depend_on_each_other():
    """weight and bias computed from x: a recorded backward hands on the norm's own derivatives, and the rest of the graph adds theirs."""
    from pde_amd import functional as K
    gen = torch.Generator(device="cuda").manual_seed(6)
    x0 = torch.randn(5, 12, device="cuda", generator=gen)

    def grads(x, norm):
        w = 1 + 0.3 * x.mean(0)
        y = norm(x, w, 0.5 * w * x.sum(0))
        g, = torch.autograd.grad(y.square().sum(), x, create_graph=True)
        h, = torch.autograd.grad(g.square().sum(), x)
        return g.detach().double(), h.double()

    got = grads(x0.clone().requires_grad_(), lambda x, w, b: K.group_norm_act(x, 3, w, b, 1e-5, K.ACT_TANH))
    want = grads(x0.double().requires_grad_(), lambda x, w, b: _definition(x, w, b, 3, 1e-5, "tanh"))
    for a, e in zip(got, want):
        assert float((a - e).norm() / e.norm()) < 1e-5            # groups of four of spread 1: a few r^3 of 2^-24 (second order: r^5)


def test_empty_batches_in_tensor_code():
    """The defining expression takes what the kernels take: no samples, no positions."""
    from pde_amd import functional as K
    for shape in ((0, 8), (0, 5, 8), (3, 0, 8)):
        x = torch.empty(shape, device="cuda", requires_grad=True)
        w = torch.ones(8, device="cuda", requires_grad=True)
        gx, gw = torch.autograd.grad(K.group_norm_act(x, 2, w).square().sum(), (x, w), create_graph=True)
        assert gx.shape == x.shape and not gw.any()


@pytest.mark.parametrize("shape,groups", [((3, 3000, 40), 5), ((600, 300, 24), 3), ((5000, 2, 384), 1)])
def test_captured_and_replayed(shape, groups):
    """Forward and backward of samples with several chunks, one, and many samples a block, captured without an eager call of the shape
    before and replayed on new values between eager work: the eager bits each time."""
    from pde_amd import functional as K
    gen = torch.Generator(device="cuda").manual_seed(11)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=gen)
    leaves = [rand(*shape), 1 + 0.2 * rand(shape[-1]), 0.2 * rand(shape[-1])]
    gy = rand(*shape)

    def both(leaves):
        leaves = [t.detach().requires_grad_() for t in leaves]
        y = K.group_norm_act(leaves[0], groups, leaves[1], leaves[2], 1e-5, K.ACT_SILU)
        return (y.detach(), *torch.autograd.grad(y, leaves, gy))

    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        held = both(leaves)
    for _ in range(4):
        for t in leaves:
            t.copy_(rand(*t.shape))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, both(leaves)))


def test_many_samples_beyond_32_bits():
    """2^22 samples of 33 positions, 2^32 values and more, 64 samples a block of the backward's sums: a block of samples over and over
    has the same bits everywhere, and its parameters' gradients as many times.

    Those are sums of one sign: chains of 32 rows and of 64 samples, two roundings besides, the base's own alike: 2 (32 + 64 + 2)."""
    from pde_amd import functional as K
    gen = torch.Generator(device="cuda").manual_seed(12)
    x = torch.randn(1 << 12, 33, 32, device="cuda", generator=gen).bfloat16()
    gy = torch.rand(1 << 12, 33, 32, device="cuda", generator=gen).bfloat16()
    w, b = torch.ones(32, device="cuda"), torch.zeros(32, device="cuda", requires_grad=True)
    copies = (1 << 10) + 1
    f = lambda t: K.group_norm_act(t, 2, w, b.detach(), 1e-5, K.ACT_TANH)
    want = [t.clone() for t in _with_gradients(f, x, gy)]
    got = _with_gradients(f, x.repeat(copies, 1, 1), gy.repeat(copies, 1, 1))
    assert got[0].numel() > 1 << 32
    assert all(_repeats_match(a, e) for a, e in zip(got, want))
    del got
    sums = [torch.autograd.grad(K.group_norm_act(x.repeat(c, 1, 1), 2, w, b), b, gy.repeat(c, 1, 1))[0].double() for c in (1, copies)]
    assert torch.allclose(sums[1], copies * sums[0], rtol=2 * 98 * U, atol=0)
    torch.cuda.empty_cache()
