"""KAN stacks with norms between their layers: values, derivatives, training steps, and Muon on top of them."""
import copy
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu


def _model(widths, groups=4, grid=5, act=torch.nn.Tanh, base=torch.nn.SiLU, seed=0):
    from pde_amd import KAN
    torch.manual_seed(seed)
    m = KAN(widths, grid_size=grid, base_activation=base, norm_groups=groups, norm_activation=act)
    with torch.no_grad():
        for p in m.parameters():
            p.add_(0.2 * torch.randn_like(p))
    return m


def _reference(model):
    """The model in 64 bits on the CPU, as a function of (parameters, points): tensor code, differentiable at will."""
    from torch.func import functional_call
    m = copy.deepcopy(model).cpu().double()
    params = {k: v.detach() for k, v in m.named_parameters()}
    return params, lambda p, x: functional_call(m, p, (x,))


def _jets(f, x):
    """(value, first derivatives, second derivatives of all but the last column) by forward differentiation."""
    from torch.func import jvp
    d = x.size(1)
    cols, seconds = [], []
    value = None
    for j in range(d):
        v = torch.zeros_like(x)
        v[:, j] = 1
        first = lambda t: jvp(f, (t,), (v,))[1]
        if j < d - 1:
            y1, y2 = jvp(first, (x,), (v,))
            seconds.append(y2)
        else:
            value, y1 = jvp(f, (x,), (v,))
        cols.append(y1)
    return value, cols, seconds


def _tolerances(compute, params, x):
    """Relative tolerances of ``compute(params, x)`` (a dict of tensors) in 32 bits, from its condition in 64 bits.

    A calculation in 32 bits is the exact one for data off by a few u = 2^-24 at each operation.  So every parameter and
    every point is moved by u relative, with random signs, and 64 times what that moves a result by (the largest of four
    draws, in the 2-norm) is allowed: on the longest way through two norms, three layers and the backward of each, each
    value passes about 200 roundings of either sign, and errors of random sign add like sqrt(200) = 14, four deviations.
    This counts the condition of the norms themselves: small variances, and groups of two channels, whose normalised
    values are nearly signs and whose derivatives are differences of almost equal terms."""
    gen = torch.Generator().manual_seed(99)
    move = lambda t: t * (1 + 2.0 ** -24 * (2.0 * torch.randint(0, 2, t.shape, generator=gen).double() - 1))
    base = compute(params, x)
    worst = {k: 0.0 for k in base}
    for _ in range(4):
        other = compute({k: move(v) for k, v in params.items()}, move(x))
        for k in base:
            worst[k] = max(worst[k], float((other[k] - base[k]).detach().norm() / base[k].detach().norm()))
    return base, {k: 1e-6 + 64 * v for k, v in worst.items()}


def _rel(a, e):
    return float((a.detach().double().cpu() - e.detach().cpu()).norm() / e.detach().cpu().norm())


@pytest.mark.parametrize("groups", [4, 2])
@pytest.mark.parametrize("widths,act,base", [([2, 8, 8, 1], torch.nn.Tanh, torch.nn.SiLU), ([2, 64, 64, 3], torch.nn.SiLU, torch.nn.Identity),
                                             ([6, 32, 16, 1], torch.nn.Identity, torch.nn.SiLU)])
def test_values_and_jets(widths, act, base, groups):
    model = _model(widths, groups, act=act, base=base).cuda()
    x = torch.rand(77, widths[0], generator=torch.Generator().manual_seed(1)) * 1.6 - 0.8
    params, f = _reference(model)

    def compute(p, t):
        value, first, second = _jets(lambda v: f(p, v), t)
        return {str(j): v for j, v in enumerate([value] + first + second)}

    want, tol = _tolerances(compute, params, x.double())
    jet = model.forward_jet(x.cuda())
    assert _rel(model(x.cuda()), want["0"]) < tol["0"]
    for j in range(jet.size(2)):
        assert _rel(jet[..., j], want[str(j)]) < tol[str(j)], j
    # any leading dimensions: the norm works point by point
    assert torch.equal(model(x.cuda().view(7, 11, -1)), model(x.cuda()).view(7, 11, -1))


def _loss(f, params, x, target, n_global):
    from pde_amd.pinn import BS_RATE, BS_SIGMA
    value, first, second = _jets(lambda t: f(params, t), x)
    res = first[-1] + BS_RATE * value
    for j, s in enumerate(second):
        xj = x[:, j:j + 1]
        res = res - 0.5 * BS_SIGMA ** 2 * xj ** 2 * s - BS_RATE * xj * first[j]
    return ((res[:, 0] - target) ** 2).sum() / n_global, res[:, 0]


@pytest.mark.parametrize("widths,groups,grid", [([2, 8, 8, 1], 4, 5), ([2, 8, 8, 1], 2, 5), ([2, 64, 64, 1], 4, 5), ([2, 64, 64, 1], 2, 5),
                                                ([6, 32, 16, 1], 4, 5), ([6, 32, 16, 1], 2, 5), ([2, 64, 64, 1], 8, 10),
                                                ([6, 64, 64, 1], 8, 10), ([2, 64, 1], 1, 20)])
def test_step_matches_the_definition(widths, groups, grid):
    """Loss, residual and every gradient of the layer-by-layer step against 64-bit differentiation of the tensor code, in
    one pass, in micro-batches and within a workspace budget."""
    from pde_amd.pinn import BlackScholesStep
    model = _model(widths, groups, grid).cuda()
    n = 97
    x = torch.rand(n, widths[0], generator=torch.Generator().manual_seed(2)) * 1.6 - 0.8
    target = torch.randn(n, generator=torch.Generator().manual_seed(3))
    params, f = _reference(model)

    def compute(p, t):
        grads, (loss, res) = torch.func.grad(
            lambda q: (lambda l, r: (l, (l, r)))(*_loss(f, q, t, target.double(), 150)), has_aux=True)(p)
        return {**grads, "loss": loss, "res": res}

    want, tol = _tolerances(compute, params, x.double())
    for kw in ({}, {"micro_batch": 40}, {"workspace_budget": 1 << 30}):
        step = BlackScholesStep(model, **kw)
        out = torch.empty(n, device="cuda")
        got = step(x.cuda(), target=target.cuda(), n_global=150, residual_out=out)
        assert _rel(got, want["loss"]) < tol["loss"] and _rel(out, want["res"]) < tol["res"]
        for k, p in model.named_parameters():
            assert _rel(p.grad, want[k]) < tol[k], (k, kw)
    # the autograd route through forward_jet agrees
    from pde_amd.pinn import bs_residual_from_jet
    jet = model.forward_jet(x.cuda())
    r = bs_residual_from_jet(x.cuda(), jet)
    got = torch.autograd.grad(((r - target.cuda()) ** 2).sum() / 150, list(model.parameters()))
    for (k, p), g in zip(model.named_parameters(), got):
        assert _rel(g, p.grad.double()) < 2 * tol[k], k


def test_shared_norms():
    """One norm between several layers gets the sum of its gradients."""
    from pde_amd.pinn import BlackScholesStep, bs_residual_from_jet
    model = _model([2, 8, 8, 8, 1], 2)
    model.norms[2] = model.norms[0]
    model = model.cuda()
    x = torch.rand(97, 2, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2))
    r = bs_residual_from_jet(x, model.forward_jet(x))
    want = torch.autograd.grad((r ** 2).sum() / 97, list(model.parameters()))
    for kw in ({}, {"micro_batch": 40}):
        BlackScholesStep(model, **kw)(x)
        for (k, p), g in zip(model.named_parameters(), want):
            # the same kernels and other orders of the sums: 1e-4 is over a hundred roundings of sums of 97 points times
            # the conditions (below 10) that the tolerances of the other tests of this model come out at
            assert _rel(p.grad, g.double()) < 1e-4, (k, kw)


def test_gradient_against_differences():
    """The step's gradient along a direction against central differences of the 64-bit loss."""
    from pde_amd.pinn import BlackScholesStep
    model = _model([2, 16, 16, 1]).cuda()
    x = torch.rand(50, 2, generator=torch.Generator().manual_seed(4))
    BlackScholesStep(model)(x.cuda())
    params, f = _reference(model)
    gen = torch.Generator().manual_seed(5)
    way = {k: torch.randn(v.shape, generator=gen, dtype=torch.float64) for k, v in params.items()}
    zero = torch.zeros(50, dtype=torch.float64)
    at = lambda h: _loss(f, {k: v + h * way[k] for k, v in params.items()}, x.double(), zero, 50)[0]
    want = (at(1e-6) - at(-1e-6)) / 2e-6                # 1e-12 of curvature and 1e-16 / 1e-6 of rounding, relative
    got = sum(float((p.grad.double().cpu() * way[k]).sum()) for k, p in model.named_parameters())
    size = sum(float((p.grad.double().cpu() * way[k]).abs().sum()) for k, p in model.named_parameters())
    _, tol = _tolerances(lambda p, t: torch.func.grad(lambda q: _loss(f, q, t, zero, 50)[0])(p), params, x.double())
    assert abs(got - float(want)) < max(tol.values()) * size + 1e-6 * abs(float(want))


def test_norm_and_muon_train_together_in_a_graph():
    """The step of a normalised stack and the Muon update, captured together and replayed between eager work while an eager
    graph of the same parameters is alive: the bits of the eager loop."""
    from pde_amd import Muon
    from pde_amd.pinn import BlackScholesStep, GraphedStep
    a, b = _model([2, 64, 64, 1], groups=8, grid=10).cuda(), _model([2, 64, 64, 1], groups=8, grid=10).cuda()
    b.load_state_dict(a.state_dict())                    # (the spline fit of a seeded construction is not bit-reproducible)
    x = torch.rand(3000, 2, device="cuda")
    sa, sb = BlackScholesStep(a), BlackScholesStep(b)
    oa, ob = Muon(a.parameters(), lr=0.01), Muon(b.parameters(), lr=0.01)
    for s, o in ((sa, oa), (sb, ob)):
        s(x)
        o.step()
    alive = b(x[:10].clone()).sum()                              # an eager graph over the same leaves
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        sb(x)
        ob.step()
    for k in range(4):
        x.copy_(torch.rand(3000, 2, device="cuda"))
        la = sa(x).clone()
        oa.step()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(la, sb.loss) and torch.isfinite(la)
        assert all(torch.equal(p, q) for p, q in zip(a.parameters(), b.parameters())), k
    with pytest.raises(RuntimeError):                    # its parameters have changed since, and autograd knows
        alive.backward()
    g = GraphedStep(sb, x)
    want = sa(x).clone()
    for _ in range(3):
        assert torch.equal(g(), want)
        torch.cuda.synchronize()


def test_deeponet_with_norms_and_muon():
    """A normalised trunk takes the layer-by-layer training step; a plain one keeps the one-call step, with either
    optimiser."""
    from pde_amd import KAN
    from pde_amd.deeponet import PI_DeepONet
    ident = torch.nn.Identity
    gen = torch.Generator().manual_seed(6)
    m = 30
    u1, u2 = torch.rand(2, m, 3, generator=gen).cuda()
    bc, pde = [[torch.rand(25, generator=gen).cuda() for _ in range(3)] for _ in range(2)]

    def net(groups):
        torch.manual_seed(0)
        plain = [KAN([3, 2, 1], base_activation=ident), KAN([3, 2, 1], base_activation=ident), KAN([m, 2, 4], base_activation=ident)]
        return PI_DeepONet(*plain, KAN([2, 6, 4], base_activation=ident, norm_groups=groups)).cuda()

    a = net(2)
    loss, pde_loss, bc_loss = a.train_step(torch.optim.SGD(a.parameters(), lr=0.0), u1, u2, None, None, bc, pde)
    assert a._step.calls == 0
    want_bc = a.loss_bcs(u1, u2, None, None, *bc)
    want_pde = a.loss_res(u1, u2, None, None, *pde)
    assert torch.allclose(loss, want_pde + 8 * want_bc, rtol=1e-5)
    grads = torch.autograd.grad(want_pde + 8 * want_bc, list(a.parameters()))
    for p, g in zip(a.parameters(), grads):
        assert torch.allclose(p.grad, g, rtol=1e-4, atol=1e-5 * float(g.abs().max()))
    loader = [tuple(bc)], [tuple(pde)]
    for groups in (None, 2):
        b = net(groups)
        before = [p.detach().clone() for p in b.parameters()]
        b.fit(u1, u2, None, None, *loader, epochs=3, optimizer="muon")
        assert (b._step.calls == 3) == (groups is None)
        assert all(bool(torch.isfinite(p).all()) for p in b.parameters())
        assert all(not torch.equal(p, q) for p, q in zip(b.parameters(), before))
    with pytest.raises(ValueError):
        net(None).fit(u1, u2, None, None, *loader, epochs=1, optimizer="sgd")


def test_refusals():
    from pde_amd import KAN
    from pde_amd.pinn import BlackScholesStep
    with pytest.raises(ValueError):
        KAN([2, 6, 1], norm_groups=4)
    model = KAN([2, 8, 1], norm_groups=2, norm_activation=torch.nn.GELU).cuda()
    with pytest.raises(NotImplementedError):
        BlackScholesStep(model)
    assert torch.isfinite(model(torch.rand(5, 2, device="cuda"))).all()
    with pytest.raises(NotImplementedError):
        model.forward_jet(torch.rand(5, 2, device="cuda"))
    plain = KAN([2, 8, 1])
    assert plain.norms is None and not any("norm" in k for k in plain.state_dict())


def test_update_grid_runs_through_norms():
    model = _model([2, 8, 1]).cuda()
    x = torch.rand(200, 2, device="cuda")
    with torch.no_grad():
        y = model(x, update_grid=True)
    assert y.shape == (200, 1) and torch.isfinite(y).all()


def test_example_runs_with_muon():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "run1_pi_deeponet.py")
    spec = importlib.util.spec_from_file_location("run1_pi_deeponet", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    for more in ([], ["--graph"]):
        out = mod.main(["--P", "300", "--Q", "200", "--batch", "100", "--epochs", "2", "--seed", "0", "--optimizer", "muon"] + more)
        assert all(a == a and b == b for a, b in out["history"])
