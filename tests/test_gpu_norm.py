"""Group norm with an activation, channels last, on values and on jets, against the definition in 64 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu

ACTS = {"identity": lambda u: u, "silu": torch.nn.functional.silu, "tanh": torch.tanh}


def _kind(act):
    from pde_amd import functional as K
    return {"identity": K.ACT_IDENTITY, "silu": K.ACT_SILU, "tanh": K.ACT_TANH}[act]


def _definition(x, w, b, groups, eps, act):
    """In the type of x; the derivatives of this are what the gradients and jets are compared with."""
    n, c = x.size(0), x.size(-1)
    v = x.reshape(n, -1, groups, c // groups)
    d = v - v.mean((1, 3), keepdim=True)
    z = (d / (d.square().mean((1, 3), keepdim=True) + eps).sqrt()).reshape(x.shape)
    return ACTS[act](z * w + b)


def _bounds(x, w, b, groups, eps, act, gy):
    """Elementwise first-order error bounds of the kernels' value and input gradient, from the 64-bit quantities.

    A sum of M terms in any fixed order with partial sums a lane is off by at most D u sum|terms|, where D is the longest
    chain of additions (at most 2 + log2 M chained through lanes plus the terms a lane adds itself; 64 + M / 64 covers
    every kernel) and u = 2^-24.  The deviation e = x - mean is off by de = (D + 1) u (|x| + mean|x|); r is off by
    r (r de + (D + 3) u) relative to r <= ... since |dV| <= 2 mean|e| de + D u V and mean|e| <= sqrt(V); z = e r follows.
    The activations (1 ulp exp2 and reciprocal) are off by at most 8 u of max(1, |u|), their slopes are at most 1.1 and
    1.1.  The gradient is r (q - mean q - z mean(q z)) with q = w gy f'(u).  A factor 2 covers the second order."""
    u = 2.0 ** -24
    n, c = x.size(0), x.size(-1)
    grp = lambda t: t.reshape(n, -1, groups, c // groups)
    mean = lambda t: t.mean((1, 3), keepdim=True)
    per = lambda t: t.view(groups, c // groups)
    X = grp(x)
    M = X.size(1) * X.size(3)
    D = 64 + M / 64
    e = X - mean(X)
    r = 1 / (mean(e * e) + eps).sqrt()
    de = (D + 1) * u * (X.abs() + mean(X.abs()))
    rel_r = r * mean(de) + (D + 3) * u
    z = e * r
    dz = r * de + z.abs() * (rel_r + u)
    pre = z * per(w) + per(b)
    dpre = per(w).abs() * dz + 2 * u * ((z * per(w)).abs() + per(b).abs())
    y = 1.1 * dpre + 8 * u * pre.abs().clamp(min=1)
    bound_y = 2 * y.reshape(x.shape)
    if gy is None:
        return bound_y, None
    pre_ = pre.detach().requires_grad_()
    slope = torch.autograd.grad(ACTS[act](pre_).sum(), pre_)[0]
    g = grp(gy)
    q = per(w) * g * slope
    dq = (per(w) * g).abs() * (1.1 * dpre + 10 * u)
    s2 = mean(q * z)
    ds = D * u * (mean(q.abs()) + z.abs() * mean((q * z).abs()))
    gx = q - mean(q) - z * s2
    dgx = dq + mean(dq) + z.abs() * (mean(dq * z.abs()) + mean(q.abs() * dz)) + dz * s2.abs() + ds \
        + 4 * u * (q.abs() + mean(q.abs()) + (z * s2).abs()) + gx.abs() * (rel_r + 2 * u)
    return bound_y, 2 * (r * dgx).reshape(x.shape)


def _make(shape, dtype, seed, offset=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    c = shape[-1]
    rand = lambda *s: torch.randn(*s, device="cuda", generator=gen)
    x = (0.7 * rand(*shape) + offset * rand(c)).to(dtype)
    gy = rand(*shape).to(dtype)
    return x, 1 + 0.2 * rand(c), 0.2 * rand(c), gy


def _check(got, want, bound, dtype):
    half = torch.finfo(dtype).eps / 2
    smallest = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps       # half a step of a subnormal
    off = (got.double() - want).abs()
    tol = bound * (1 + half) + half * want.abs() + smallest
    assert bool((off <= tol).all()), (float((off - tol).max()), float((off / tol).max()))


SHAPES = [((1, 1), 1), ((3, 1), 1), ((7, 2), 1), ((5, 6), 6), ((1, 8), 2), ((33, 64), 8), ((1001, 64), 8), ((257, 90), 6),
          ((64, 96), 1), ((19, 320), 32), ((9, 512), 1), ((5, 1024), 2), ((3, 513), 1), ((2, 4097), 1), ((70, 384), 384),
          ((2, 1, 8), 2), ((1, 2, 4), 4), ((3, 5, 6), 3), ((2, 4096, 64), 8), ((3, 1999, 90), 6), ((1, 777, 1), 1),
          ((130, 9, 24), 3), ((2, 16, 16, 40), 4), ((1, 20000, 10), 5), ((2, 33, 2050), 1), ((4, 300, 257), 257),
          ((300, 32, 16), 1), ((70, 31, 5), 1), ((5000, 3, 7), 7), ((1, 70000, 6), 2), ((2000, 5, 64), 64), ((9, 33, 15), 3)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape,groups", SHAPES)
def test_value_and_gradients(shape, groups, dtype):
    from pde_amd import functional as K
    for k, act in enumerate(ACTS):
        x, w, b, gy = _make(shape, dtype, 7 + k)
        x.requires_grad_()
        w.requires_grad_()
        b.requires_grad_()
        y = K.group_norm_act(x, groups, w, b, 1e-5, _kind(act))
        gx, gw, gb = torch.autograd.grad(y, (x, w, b), gy)
        assert y.dtype == gx.dtype == dtype and gw.dtype == gb.dtype == torch.float32
        xd, wd, bd, gd = (t.detach().double() for t in (x, w, b, gy))
        leaves = [t.clone().requires_grad_() for t in (xd, wd, bd)]
        want = _definition(*leaves, groups, 1e-5, act)
        ex, ew, eb = torch.autograd.grad(want, leaves, gd)
        by, bx = _bounds(xd, wd, bd, groups, 1e-5, act, gd)
        _check(y, want.detach(), by, dtype)
        _check(gx, ex, bx, dtype)
        # the sums over the rows: each term is off by its own bound, the sum by D u of the terms' magnitudes
        n, c = x.size(0), x.size(-1)
        z = _definition(xd, torch.ones_like(wd), torch.zeros_like(bd), groups, 1e-5, "identity")
        bz, _ = _bounds(xd, torch.ones_like(wd), torch.zeros_like(bd), groups, 1e-5, "identity", None)
        rows = xd.numel() // c
        D = 64 + rows / 64
        flat = lambda t: t.reshape(rows, c)
        mag = 1.1 * flat(gd.abs())
        dp = flat(gd.abs() * by)
        _check(gb, eb, 2 * (dp.sum(0) + (D + 8) * 2.0 ** -24 * mag.sum(0)), torch.float32)
        _check(gw, ew, 2 * ((dp * flat(z.abs()) + mag * flat(bz)).sum(0) + (D + 8) * 2.0 ** -24 * (mag * flat(z.abs())).sum(0)),
               torch.float32)


def test_one_value_groups_are_the_bias():
    """A group of one value has no deviation: y = act(b) to the last bit of the activation, and no gradient reaches x."""
    from pde_amd import functional as K
    x, w, b, gy = _make((50, 24), torch.float32, 1)
    x.requires_grad_()
    y = K.group_norm_act(x, 24, w, b)
    assert torch.equal(y, b.expand_as(y))
    assert torch.equal(torch.autograd.grad(y, x, gy)[0], torch.zeros_like(x))
    jet = torch.randn(50, 24, 4, device="cuda").requires_grad_()
    y = K.group_norm_act_jet(jet, 24, w, b)
    assert torch.equal(y[..., 0], b.expand(50, 24)) and not y[..., 1:].any()
    assert not torch.autograd.grad(y, jet, torch.ones_like(y))[0].any()


@pytest.mark.parametrize("shape", [(40, 64), (3, 700, 64)])
def test_constant_and_far_groups(shape):
    """A constant group normalises to 0 whatever its value, and a large common offset costs accuracy only in proportion."""
    from pde_amd import functional as K
    x = torch.full(shape, 12345.678, device="cuda")
    assert not K.group_norm_act(x, 8).any()
    x, w, b, gy = _make(shape, torch.float32, 3)
    x = x + 1000.0
    y = K.group_norm_act(x, 8, w, b, 1e-5)
    by, _ = _bounds(x.double(), w.double(), b.double(), 8, 1e-5, "identity", None)
    _check(y, _definition(x.double(), w.double(), b.double(), 8, 1e-5, "identity"), by, torch.float32)


@pytest.mark.parametrize("shape", [(6, 32), (3, 500, 32)])
def test_non_finite_values_stay_in_their_group(shape):
    from pde_amd import functional as K
    x, w, b, gy = _make(shape, torch.float32, 4)
    clean = K.group_norm_act(x, 4, w, b, 1e-5, K.ACT_SILU)
    for bad in (float("nan"), float("inf"), -float("inf")):
        z = x.clone()
        z[1, ..., 9] = bad                                   # group 1 of sample 1
        y = K.group_norm_act(z, 4, w, b, 1e-5, K.ACT_SILU)
        touched = torch.zeros_like(y, dtype=torch.bool)
        touched[1, ..., 8:16] = True
        assert torch.equal(y[~touched], clean[~touched]) and bool(y[touched].isnan().any())


def test_strides_offsets_and_types():
    from pde_amd import functional as K
    x, w, b, gy = _make((64, 48), torch.float32, 5)
    want = K.group_norm_act(x, 6, w, b, 1e-5, K.ACT_TANH)
    wide = torch.zeros(64, 49, device="cuda")
    wide[:, 1:] = x
    assert torch.equal(K.group_norm_act(wide[:, 1:], 6, w, b, 1e-5, K.ACT_TANH), want)          # a strided view
    flat = torch.zeros(64 * 48 + 1, device="cuda")
    flat[1:] = x.reshape(-1)
    assert torch.allclose(K.group_norm_act(flat[1:].view(64, 48), 6, w, b, 1e-5, K.ACT_TANH), want, atol=2e-6)   # 4-byte aligned
    assert torch.equal(K.group_norm_act(x.t().contiguous().t(), 6, w, b, 1e-5, K.ACT_TANH), want)
    wh, bh = w.bfloat16().requires_grad_(), b.bfloat16().requires_grad_()
    y = K.group_norm_act(x, 6, wh, bh)
    gw, gb = torch.autograd.grad(y, (wh, bh), gy)
    assert gw.dtype == gb.dtype == torch.bfloat16
    assert torch.equal(y, K.group_norm_act(x, 6, wh.float(), bh.float()))
    assert torch.equal(K.group_norm_act(x, 6), K.group_norm_act(x, 6, torch.ones_like(w), torch.zeros_like(b)))
    jet = torch.randn(64 * 48 * 4 + 1, device="cuda")
    view = jet[1:].view(64, 48, 4)
    assert torch.equal(K.group_norm_act_jet(view, 6, w, b), K.group_norm_act_jet(view.clone(), 6, w, b))
    with pytest.raises(TypeError):
        K.group_norm_act(x.double(), 6)
    with pytest.raises(TypeError):
        K.group_norm_act_jet(view.half(), 6)
    with pytest.raises(RuntimeError):
        K.group_norm_act(x, 6, w.cpu(), b)


def test_empty_batches():
    from pde_amd import functional as K
    for shape in ((0, 8), (0, 5, 8), (3, 0, 8)):
        x = torch.empty(shape, device="cuda", requires_grad=True)
        w = torch.ones(8, device="cuda", requires_grad=True)
        y = K.group_norm_act(x, 2, w)
        gx, gw = torch.autograd.grad(y, (x, w), torch.empty_like(y))
        assert y.shape == gx.shape == x.shape and not gw.any()
    jet = torch.empty(0, 8, 4, device="cuda", requires_grad=True)
    y = K.group_norm_act_jet(jet, 2)
    assert torch.autograd.grad(y, jet, torch.empty_like(y))[0].shape == jet.shape


def test_second_order_and_transforms():
    from torch.func import jacrev, vmap
    from pde_amd import functional as K
    x, w, b, gy = _make((3, 12), torch.float32, 6)
    x.requires_grad_()
    y = K.group_norm_act(x, 3, w, b, 1e-5, K.ACT_TANH)
    g, = torch.autograd.grad(y, x, gy, create_graph=True)
    h, = torch.autograd.grad(g.square().sum(), x)
    xd = x.detach().double().requires_grad_()
    g2, = torch.autograd.grad(_definition(xd, w.double(), b.double(), 3, 1e-5, "tanh"), xd, gy.double(), create_graph=True)
    h2, = torch.autograd.grad(g2.square().sum(), xd)
    # second derivatives of groups of four of spread 0.7: amplification r^3 and sums of 12 terms of 2^-24
    assert float((h.double() - h2).norm() / h2.norm()) < 1e-5
    j = jacrev(lambda t: K.group_norm_act(t, 3, w, b, 1e-5, K.ACT_TANH).sum(0))(x.detach())
    assert j.shape == (12, 3, 12)
    v = vmap(lambda t: K.group_norm_act(t.unsqueeze(0), 3, w, b)[0])(x.detach())
    assert torch.allclose(v, K.group_norm_act(x.detach(), 3, w, b), atol=1e-5)


def _with_gradients(f, x, gy):
    """(f(x), its gradient in x along gy)"""
    x = x.detach().requires_grad_()
    y = f(x)
    return y.detach(), torch.autograd.grad(y, x, gy)[0]


def _jet_definition(jet, w, b, groups, eps, act, n_dir, n_second):
    """Derivatives along x + t x'_d + t^2 x''_d / 2 of the values' definition, by nested forward differentiation."""
    from torch.func import jvp
    f = lambda t: _definition(t, w, b, groups, eps, act)
    x0 = jet[..., 0].clone()
    slots, seconds = [f(x0)], []
    for d in range(n_dir):
        first = lambda t, t1: jvp(f, (t,), (t1,))[1]
        x1 = jet[..., 1 + d]
        if d < n_second:
            y1, y2 = jvp(first, (x0, x1), (x1, jet[..., 1 + n_dir + d]))
            seconds.append(y2)
        else:
            y1 = first(x0, x1)
        slots.append(y1)
    return torch.stack(slots + seconds, -1)


@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("n_dir,n_second", [(2, 1), (6, 5)])
@pytest.mark.parametrize("n,c,groups", [(1, 4, 1), (1, 5, 1), (7, 16, 2), (301, 64, 8), (40, 64, 1), (33, 130, 10), (9, 256, 8),
                                        (5, 300, 2), (3, 512, 1), (17, 1024, 32), (1000, 10, 2)])
def test_jets(n, c, groups, n_dir, n_second, act):
    """Every slot and gradient within 1e-5 of the derivatives of the definition in 64 bits, in the 2-norm.

    Groups of at least four channels about 1.2 apart: r is near 1 and the largest power r^7 A^2 multiplies errors by a few
    tens at most, each a few 2^-24."""
    from pde_amd import functional as K
    gen = torch.Generator(device="cuda").manual_seed(n + c)
    J = 1 + n_dir + n_second
    rand = lambda *s: torch.randn(*s, device="cuda", generator=gen)
    # the channels of a group at distinct offsets: no group is close to constant, so r stays near 1
    offset = torch.linspace(-2, 2, c // groups, device="cuda").repeat(groups)
    x = 0.4 * rand(n, c, J)
    x[..., 0] += offset
    w, b, gy = 1 + 0.2 * rand(c), 0.2 * rand(c), rand(n, c, J)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    y = K.group_norm_act_jet(x, groups, w, b, 1e-5, _kind(act), n_dir, n_second)
    got = torch.autograd.grad(y, leaves, gy)
    ref = [t.detach().double() for t in leaves]
    f = lambda x, w, b: _jet_definition(x, w, b, groups, 1e-5, act, n_dir, n_second)
    want, pull = torch.func.vjp(f, *ref)
    exact = pull(gy.double())
    rel = lambda a, e: float((a.double() - e).norm() / e.norm())
    for j in range(J):
        assert rel(y[..., j], want[..., j]) < 1e-5, j
        assert rel(got[0][..., j], exact[0][..., j]) < 1e-5, j
    assert rel(got[1], exact[1]) < 1e-5 and rel(got[2], exact[2]) < 1e-5


def test_jets_against_differences():
    """The first and second derivative slots against central differences of the 64-bit values along one curve."""
    from pde_amd import functional as K
    x = torch.randn(20, 16, 4, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2))
    y = K.group_norm_act_jet(x, 2, act=K.ACT_TANH).double()
    X = x.double()
    one = torch.ones(16, device="cuda", dtype=torch.float64)
    at = lambda t, d: _definition(X[..., 0] + t * X[..., 1 + d] + (0.5 * t * t * X[..., 3] if d == 0 else 0), one, 0 * one, 2,
                                  1e-5, "tanh")
    h = 1e-4                                                  # differences: h^2 = 1e-8 and 1e-16 / h^2 = 1e-8 off
    scale = y.abs().max()
    assert float((y[..., 1] - (at(h, 0) - at(-h, 0)) / (2 * h)).abs().max()) < 1e-5 * scale
    assert float((y[..., 2] - (at(h, 1) - at(-h, 1)) / (2 * h)).abs().max()) < 1e-5 * scale
    assert float((y[..., 3] - (at(h, 0) - 2 * at(0, 0) + at(-h, 0)) / h ** 2).abs().max()) < 2e-5 * scale


def test_results_repeat_on_streams_and_in_graphs():
    """Fixed summation order: the same bits on another stream, twice, and from a replayed graph between eager work."""
    from pde_amd import functional as K
    cases = [_make((5000, 64), torch.float32, 8), _make((4, 1500, 40), torch.bfloat16, 9)]
    for x, w, b, gy in cases:
        def step():
            leaves = [t.detach().requires_grad_() for t in (x, w, b)]
            y = K.group_norm_act(leaves[0], 8, leaves[1], leaves[2], 1e-5, K.ACT_SILU)
            return [y.detach()] + list(torch.autograd.grad(y, leaves, gy))
        want = [t.clone() for t in step()]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            again = step()
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(a, e) for a, e in zip(again, want))
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = step()
        source = x.clone()
        for k in range(3):
            x.copy_(source * (1 + k))
            graph.replay()
            eager = step()
            torch.cuda.synchronize()
            assert all(torch.equal(a, e) for a, e in zip(held, eager))
        x.copy_(source)


def _repeats_match(y, want, tol=None):
    """Every copy of a block [rows, ...] along y's leading axis: the same bits, or off by at most ``tol`` elementwise."""
    copies = y.view(-1, *want.shape)
    for part in copies.split(max(1, (1 << 28) // want.numel())):
        ok = part == want if tol is None else (part.double() - want).abs() <= tol
        if not bool(ok.all()):
            return False
    return True


def test_offsets_beyond_32_bits():
    """2^32 values and more: one block of points over and over has to give the same bits everywhere."""
    from pde_amd import functional as K
    x, w, b, gy = _make((1 << 15, 128), torch.bfloat16, 8)
    gy = gy.abs()
    copies = (1 << 10) + 1
    want = [t.clone() for t in _with_gradients(lambda t: K.group_norm_act(t, 8, w, b, 1e-5, K.ACT_TANH), x, gy)]
    got = _with_gradients(lambda t: K.group_norm_act(t, 8, w, b, 1e-5, K.ACT_TANH), x.repeat(copies, 1), gy.repeat(copies, 1))
    assert got[0].numel() > 1 << 32
    assert all(_repeats_match(a, e) for a, e in zip(got, want))
    del got
    torch.cuda.empty_cache()
    # gradients of the parameters: 2^25 points over 2048 blocks of 8 points at a time are chains of 2^11 additions of
    # one sign: at most 2^11 (and the 64-bit finish) times 2^-24
    bias = b.clone().requires_grad_()
    K.group_norm_act(x.repeat(copies, 1), 8, w, bias).backward(gy.repeat(copies, 1))
    assert torch.allclose(bias.grad.double(), copies * gy.double().sum(0), rtol=2.0 ** -12, atol=0)
    torch.cuda.empty_cache()
    jets, copies = torch.randn(1 << 14, 64, 4, device="cuda", generator=torch.Generator(device="cuda").manual_seed(9)), (1 << 10) + 1
    w, b = w[:64].contiguous(), b[:64].contiguous()
    cot = torch.randn_like(jets)
    f = lambda t: K.group_norm_act_jet(t, 8, w, b, 1e-5, K.ACT_TANH)
    want = [t.clone() for t in _with_gradients(f, jets, cot)]
    got = _with_gradients(f, jets.repeat(copies, 1, 1), cot.repeat(copies, 1, 1))
    assert got[0].numel() > 1 << 32
    assert all(_repeats_match(a, e) for a, e in zip(got, want))
    del got
    torch.cuda.empty_cache()


def test_long_samples_beyond_32_bits():
    """Three samples of 2^31 values: positions over and over have the statistics of one round of them."""
    from pde_amd import functional as K
    s, c, groups, copies = 1 << 14, 128, 8, 1 << 10
    x, w, b, gy = _make((3, s, c), torch.bfloat16, 10)
    gy = gy.abs()
    long = lambda t: t.unsqueeze(1).expand(3, copies, s, c).reshape(3, copies * s, c)
    got = _with_gradients(lambda t: K.group_norm_act(t, groups, w, b, 1e-5, K.ACT_SILU), long(x), long(gy))
    assert got[0].numel() > 1 << 32
    xd = x.double().requires_grad_()
    y = _definition(xd, w.double(), b.double(), groups, 1e-5, "silu")
    gx, = torch.autograd.grad(y, xd, gy.double())
    # a thread adds 2^24 / 128 chunks / 16 rows = 2^13 values of a channel, so the sums are off by D = 2^13 + 2^8 steps of
    # 2^-24 relative to the sums of the magnitudes; values and gradients take that times slopes and normalised values: of
    # data of spread 1 and |z| < 6, (1 + |z|) |w| 1.1 D u for the value and twice r (|w| max|gy|) (1 + |z|)^2 D u for the gradient
    d = (2 ** 13 + 2 ** 8) * 2.0 ** -24
    half = 2.0 ** -8
    z = _definition(x.double(), torch.ones(c, device="cuda").double(), torch.zeros(c, device="cuda").double(), groups, 1e-5, "identity")
    spread = x.double().reshape(3, s, groups, -1).std((1, 3), keepdim=True)
    r = (1 / spread).expand(3, s, groups, c // groups).reshape(3, s, c)
    shift = 1 + x.double().abs() * r                              # sums of magnitudes against the spread
    tol_y = 2.2 * d * (1 + z.abs()) * w.double().abs() * shift + half * y.detach().abs() + 1e-30
    tol_g = 4 * d * r * (1 + z.abs()) ** 2 * (w.double().abs() * gy.double().abs()).amax() * shift + half * gx.abs() + 1e-30
    for i in range(3):
        assert _repeats_match(got[0][i], y.detach()[i], tol_y[i])
        assert _repeats_match(got[1][i], gx[i], tol_g[i])
    del got
    torch.cuda.empty_cache()


def test_under_transforms_of_something_else():
    """Inside a transform a call whose own tensors are constants takes the tensor code; a norm on jets refuses."""
    from pde_amd import functional as K
    x, w, b, _ = _make((5, 12), torch.float32, 12)
    g = torch.func.grad(lambda t: (K.group_norm_act(x, 3, w, b) * t).sum())(torch.ones(5, 12, device="cuda"))
    assert torch.allclose(g, K.group_norm_act(x, 3, w, b), atol=1e-5)
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda t: K.group_norm_act_jet(t, 2))(torch.ones(3, 2, 4, 4, device="cuda"))


def test_outside_of_a_recording():
    """Calls that leave no trace give the same bits; forward derivatives are refused, not dropped."""
    import torch.autograd.forward_ad as fwad
    from pde_amd import functional as K
    x, w, b, _ = _make((9, 12), torch.float32, 13)
    jet = torch.randn(9, 12, 4, device="cuda")
    for f, t in ((lambda t: K.group_norm_act(t, 3, w, b), x), (lambda t: K.group_norm_act_jet(t, 3, w, b), jet)):
        want = f(t.clone().requires_grad_())
        assert want.requires_grad
        with torch.no_grad():
            got = f(t.clone().requires_grad_())
        assert not got.requires_grad and torch.equal(got, want)
        with torch.inference_mode():
            assert torch.equal(f(t), want)
        with fwad.dual_level(), pytest.raises(Exception, match="jvp|forward"):
            f(fwad.make_dual(t, torch.ones_like(t)))
