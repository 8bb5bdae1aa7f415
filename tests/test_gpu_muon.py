"""Newton-Schulz orthogonalisation and the Muon step against their definitions in 64 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu

A, B, C = 3.4445, -4.7750, 2.0315
U = 2.0 ** -24


def _definition(g, steps=5, eps=1e-7, coefficients=(A, B, C)):
    """In 64 bits, and how far (Frobenius norm) the products may be off.

    A product of two-piece operands rounds each term by at most 3 u (two representations and the left-out lo lo) and the
    sum over K inner values in about 3 K / 32 matrix instructions; rounding errors of either sign add like the square root
    of their number, four standard deviations are allowed: e = 4 u sqrt(3 K / 32 + 9) of the operands' norms.  In step k the
    errors of S and R move X by |b| e |S| + 2 |c| e |S|^2 + e |R| and of the sum by u (a + |R|), relative to |X_k|_F; the
    later steps multiply what a singular direction is off by at most their slope at 0, |a| each."""
    a, b, c = coefficients
    x = g.double()
    if x.size(-2) > x.size(-1):
        out, off = _definition(g.transpose(-2, -1), steps, eps, coefficients)
        return out.transpose(-2, -1), off
    x = x / (x.square().sum((-2, -1), keepdim=True).sqrt() + eps)
    m, n = x.shape[-2:]
    fro = lambda t: t.square().sum((-2, -1)).sqrt()
    off = 2 * U * fro(x)
    em, en = (4 * U * (3 * k / 32 + 9) ** 0.5 for k in (m, n))
    for _ in range(steps):
        s = x @ x.transpose(-2, -1).contiguous()
        r = b * s + c * (s @ s)
        e = torch.linalg.eigvalsh(s)
        top, rn = e[..., -1], (b * e + c * e * e).abs().amax(-1)
        step = abs(b) * en * top + abs(c) * (2 * en + em) * top ** 2 + em * rn + U * (abs(a) + rn)
        off = max(abs(a), 1.0) * off + step * fro(x)
        x = a * x + r @ x
    return x, off


def _check(got, want, off):
    half = torch.finfo(got.dtype).eps / 2
    fro = lambda t: t.square().sum((-2, -1)).sqrt()
    d, tol = fro(got.double() - want), off * (1 + half) + half * fro(want)
    assert bool((d <= tol).all()), (d.flatten()[:4].tolist(), tol.flatten()[:4].tolist())


def _matrix(shape, seed, kind="noise", dtype=torch.float32):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    *lead, m, n = shape
    g = torch.randn(*shape, device="cuda", generator=gen)
    if kind == "low rank":
        r = max(1, min(m, n) // 8)
        g = torch.randn(*lead, m, r, device="cuda", generator=gen) @ torch.randn(*lead, r, n, device="cuda", generator=gen) + 0.1 * g
    return (1e-3 * g).to(dtype)


SHAPES = [(1, 1), (1, 7), (5, 1), (1, 5000), (2, 2), (2, 64), (3, 40), (16, 16), (33, 65), (64, 2), (64, 64), (64, 832), (100, 31),
          (128, 128), (257, 129), (300, 1000), (1000, 300), (65, 4097), (129, 2000), (512, 512), (2, 70000), (70000, 3),
          (640, 1500), (20, 500), (20, 600), (96, 96), (96, 128), (90, 161), (128, 64), (128, 1664), (40, 4000), (100, 70), (4100, 64)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", SHAPES)
def test_orthogonalize(shape, dtype):
    from pde_amd import functional as K
    for kind in ("noise", "low rank"):
        g = _matrix(shape, sum(shape), kind, dtype)
        keep = g.clone()
        out = K.orthogonalize(g)
        assert out.dtype == dtype and out.shape == g.shape and torch.equal(g, keep)
        _check(out, *_definition(g))
        assert torch.equal(out, K.orthogonalize(g))              # one summation order


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_blocks_of_128(dtype):
    """Large enough for the larger blocks: along the long axis (one matrix), among squares too (a stack of four)."""
    from pde_amd import functional as K
    g = _matrix((4, 2090, 2049), 5, "low rank", dtype)
    for out, m in ((K.orthogonalize(g[1]), g[1]), (K.orthogonalize(g)[3], g[3])):
        _check(out, *_definition(m))


def test_singular_values_end_near_one():
    """The quintic carries every singular value above |g|_F / 100 into 0.65 .. 1.25 in five steps (0.01 a^4 > 1 before the
    curve bends; the composed polynomial stays within these bounds beyond)."""
    from pde_amd import functional as K
    g = _matrix((200, 700), 1)
    s = torch.linalg.svdvals(K.orthogonalize(g).double())
    assert float(s.min()) > 0.65 and float(s.max()) < 1.25


@pytest.mark.parametrize("shape", [(3, 64, 64), (2, 3, 40, 100), (5, 90, 33), (7, 1, 50), (4, 200, 300), (1000, 4, 6)])
def test_stacks_are_matrix_by_matrix(shape):
    from pde_amd import functional as K
    g = _matrix(shape, 2)
    out = K.orthogonalize(g)
    _check(out, *_definition(g))
    flat, each = out.reshape(-1, *shape[-2:]), g.reshape(-1, *shape[-2:])
    for i in (0, len(flat) - 1):
        # (a stack may split its long axis differently from a single matrix: equal to rounding)
        assert float((K.orthogonalize(each[i]) - flat[i]).abs().max()) < 2e-4


def test_lists_of_matrices():
    from pde_amd import functional as K
    shapes = [(64, 2), (64, 26), (1, 64), (64, 832), (300, 200), (2, 5, 7), (0, 4), (40, 40)] * 3        # 24: two launches
    mats = [_matrix(s, i) if 0 not in s else torch.empty(s, device="cuda") for i, s in enumerate(shapes)]
    mats[3] = mats[3].t().contiguous().t()                        # a strided one
    mats[7] = mats[15]                                            # the same one twice
    out = K.orthogonalize(mats)
    assert isinstance(out, list) and len(out) == len(mats)
    for g, o in zip(mats, out):
        assert o.shape == g.shape
        if g.numel():
            _check(o, *_definition(g))
    assert torch.equal(out[7], out[15])


@pytest.mark.parametrize("scale", [1e-30, 1e-20, 1e-9, 1.0, 1e15, 1e30])
@pytest.mark.parametrize("shape", [(20, 30), (1, 30), (150, 90)])
def test_scales(shape, scale):
    """The norm is summed in 64 bits: gradients of any size fp32 holds; far below eps the result is a^5 g / eps."""
    from pde_amd import functional as K
    g = _matrix(shape, 3) * scale
    want, off = _definition(g)
    # the rounding errors are relative to X, which is far smaller than 1 where eps dominates: off is already in |X|_F
    _check(K.orthogonalize(g), want, off + 1e-37)


def test_strips_of_zeros_and_tiny_values():
    """Columns of zeros and of far smaller values than the rest: a block that holds only those takes part as the others do."""
    from pde_amd import functional as K
    for shape in ((50, 900), (900, 50), (120, 700), (30, 60)):
        for scale in (1.0, 1e-25):
            g = _matrix(shape, 12) * scale
            long = g if shape[1] > shape[0] else g.t()
            long[:, :len(long[0]) // 3] = 0
            long[:, -len(long[0]) // 3:] *= 1e-9
            want, off = _definition(g)
            _check(K.orthogonalize(g), want, off + 1e-37)


def test_zero_and_non_finite_matrices():
    from pde_amd import functional as K
    for shape in ((3, 40, 70), (3, 1, 50), (3, 200, 140), (3, 60, 1000)):
        g = _matrix(shape, 4)
        clean = K.orthogonalize(g)
        g[0] = 0
        for bad in (float("nan"), float("inf")):
            g[2, 0, 3] = bad
            out = K.orthogonalize(g)
            assert not out[0].any() and torch.equal(out[1], clean[1]) and bool(out[2].isnan().any())


@pytest.mark.parametrize("steps,coefficients", [(1, (A, B, C)), (2, (A, B, C)), (3, (1.5, -0.5, 0.0)), (8, (15 / 8, -10 / 8, 3 / 8)),
                                                (12, (2.0, -1.5, 0.5))])
def test_other_steps_and_coefficients(steps, coefficients):
    from pde_amd import functional as K
    for shape in ((40, 60), (1, 33), (180, 150)):
        g = _matrix(shape, 5)
        _check(K.orthogonalize(g, steps=steps, coefficients=coefficients, eps=1e-5),
               *_definition(g, steps, 1e-5, coefficients))
    with pytest.raises(RuntimeError):
        K.orthogonalize(g, coefficients=(3.4445, 4.7750, 2.0315))


def test_refusals_on_the_gpu():
    from pde_amd import functional as K
    g = _matrix((4, 8), 6)
    with pytest.raises(TypeError):
        K.orthogonalize(g.double())
    with pytest.raises(TypeError):
        K.orthogonalize([g, g.half()])
    with pytest.raises(RuntimeError):
        K.orthogonalize([g, g.cpu()])
    x = g.clone().requires_grad_()
    assert not K.orthogonalize(x).requires_grad


def _reference_step(p, g, m, rows, cols, lr, mu, nesterov, decay, gain):
    m = mu * m + (1 - mu) * g
    u = (1 - mu) * g + mu * m if nesterov else m
    o, off = _definition(u.reshape(rows, cols).float())          # the direction as the kernel's 32-bit U has it
    return p * (1 - lr * decay) - lr * gain * o.reshape(p.shape), m, off


@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("adjust", ["original", "match_rms_adamw", "none"])
def test_muon_step(nesterov, adjust):
    """Three steps over parameters of every shape a KAN has; each step starts the reference from the optimiser's state."""
    from pde_amd.optim import Muon, _matrix_shape
    gen = torch.Generator(device="cuda").manual_seed(7)
    shapes = [(64, 2), (64, 2, 13), (64, 64), (64, 64, 13), (1, 64), (64,), (), (300, 40, 3), (5,), (2, 6, 8), (150, 130)]
    params = [torch.nn.Parameter(0.1 * torch.randn(s, device="cuda", generator=gen)) for s in shapes]
    frozen = torch.nn.Parameter(torch.ones(3, device="cuda"))
    opt = Muon([{"params": params[:4]}, {"params": params[4:] + [frozen], "lr": 0.5, "weight_decay": 0.0}], lr=0.02,
               momentum=0.9, nesterov=nesterov, weight_decay=0.1, adjust_lr=adjust)
    for _ in range(3):
        before = [p.detach().double() for p in params]
        moments = [opt.state[p]["momentum_buffer"].double() if p in opt.state else torch.zeros_like(b)
                   for p, b in zip(params, before)]
        for p in params:
            p.grad = 1e-3 * torch.randn(p.shape, device="cuda", generator=gen)
        opt.step()
        for i, (p, b, m) in enumerate(zip(params, before, moments)):
            lr, decay = (0.02, 0.1) if i < 4 else (0.5, 0.0)
            rows, cols = _matrix_shape(p)
            gain = Muon._gain(rows, cols, adjust)
            want, wm, off = _reference_step(b, p.grad.double(), m, rows, cols, lr, 0.9, nesterov, decay, gain)
            got = opt.state[p]["momentum_buffer"].double()
            assert bool(((got - wm).abs() <= 3 * U * (wm.abs() + m.abs() + p.grad.double().abs())).all())
            # U in 32 bits from the rounded momentum is 4 u |U| off, which five steps multiply by at most a^5
            tol = lr * gain * (float(off) + 4 * U * A ** 5) + 3 * U * float(want.norm() + b.norm())
            assert float((p.detach().double() - want).norm()) <= tol, i
    assert torch.equal(frozen, torch.ones(3, device="cuda")) and frozen not in opt.state


def test_muon_state_dict_schedule_and_strided_gradients():
    from pde_amd.optim import Muon
    gen = torch.Generator(device="cuda").manual_seed(8)
    make = lambda: [torch.nn.Parameter(t.clone()) for t in (torch.ones(30, 20, device="cuda"), torch.ones(9, device="cuda"))]
    grads = [[torch.randn(30, 20, device="cuda", generator=gen), torch.randn(9, device="cuda", generator=gen)] for _ in range(4)]
    a, b = make(), make()
    lr = torch.tensor(0.1, device="cuda")
    oa, ob = Muon(a, lr=0.1), Muon(b, lr=lr)
    for k in range(4):
        for p, q, g in zip(a, b, grads[k]):
            p.grad = g
            q.grad = g.t().contiguous().t()                      # same values, other strides
        for group in oa.param_groups:
            group["lr"] = 0.1 / (1 + k)
        lr.copy_(torch.tensor(0.1 / (1 + k)))
        oa.step()
        ob.step()
        assert all(torch.equal(p, q) for p, q in zip(a, b))
        if k == 1:                                               # carry on from a saved state
            c = [torch.nn.Parameter(p.detach().clone()) for p in b]
            oc = Muon(c, lr=lr)
            oc.load_state_dict(ob.state_dict())
            oc.param_groups[0]["lr"] = lr
            b, ob = c, oc


def test_muon_in_a_graph():
    """Captured after one eager step and replayed with new gradients and learning rates between eager work: the bits of the
    eager optimiser."""
    from pde_amd.optim import Muon
    gen = torch.Generator(device="cuda").manual_seed(9)
    shapes = [(64, 64), (64, 832), (1, 64), (200, 300), (10,)]
    start = [torch.randn(s, device="cuda", generator=gen) for s in shapes]
    a, b = ([torch.nn.Parameter(t.clone()) for t in start] for _ in range(2))
    lr = torch.tensor(0.1, device="cuda")
    oa, ob = Muon(a, lr=lr, weight_decay=0.1), Muon(b, lr=lr, weight_decay=0.1)
    fresh = Muon([torch.nn.Parameter(torch.ones(4, 4, device="cuda"))])
    fresh.param_groups[0]["params"][0].grad = torch.ones(4, 4, device="cuda")
    held = [torch.randn(s, device="cuda", generator=gen) for s in shapes]
    for p, q, g in zip(a, b, held):
        p.grad, q.grad = g, g
    oa.step()
    ob.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ob.step()
        with pytest.raises(RuntimeError):
            fresh.step()                                         # its buffers would be made inside the capture
    for k in range(4):
        for g in held:
            g.copy_(torch.randn(g.shape, device="cuda", generator=gen))
        lr.fill_(0.1 / (1 + k))
        oa.step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(a, b)), k


def test_muon_refusals_on_the_gpu():
    from pde_amd.optim import Muon
    base = torch.ones(6, 4, device="cuda")
    p, q = torch.nn.Parameter(base), torch.nn.Parameter(base.view(4, 6))
    p.grad, q.grad = torch.ones_like(p), torch.ones_like(q)
    with pytest.raises(RuntimeError):
        Muon([p, q]).step()                                      # one memory, two updates
    h = torch.nn.Parameter(base.half())
    h.grad = torch.ones_like(h)
    with pytest.raises(TypeError):
        Muon([h]).step()
    t = torch.nn.Parameter(torch.ones(4, 6, device="cuda").t())
    t.grad = torch.ones_like(t)
    with pytest.raises(RuntimeError):
        Muon([t]).step()
    s = torch.nn.Parameter(torch.ones(4, 6, device="cuda"))
    s.grad = torch.ones(4, 6, device="cuda").to_sparse()
    with pytest.raises(RuntimeError):
        Muon([s]).step()
    ok = torch.nn.Parameter(torch.ones(4, 6, device="cuda"))
    ok.grad = torch.ones_like(ok)
    for lr in (torch.tensor([0.1, 0.2], device="cuda"), torch.tensor(0.1, device="cuda", dtype=torch.float64)):
        with pytest.raises(RuntimeError):
            Muon([ok], lr=lr).step()
    assert torch.equal(ok, torch.ones(4, 6, device="cuda"))
    opt = Muon([ok], lr=torch.tensor(0.1))                       # a number on the host
    opt.step()
    assert opt.step(lambda: torch.tensor(3.0)) == 3.0


def test_streams():
    from pde_amd import functional as K
    g = [_matrix((300, 400), 10), _matrix((64, 64), 11)]
    want = K.orthogonalize(g)
    side = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    out = []
    for _ in range(4):                                           # two calls at once, each with its own workspace
        for s in side:
            with torch.cuda.stream(s):
                out.append(K.orthogonalize(g))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for o in out for a, b in zip(o, want))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_largest_matrix(dtype):
    """2^30 values, workspaces beyond 2^32 bytes: [B B ... B] of 2^10 copies has the factor [O O ... O] / 2^5 of B's O."""
    from pde_amd import functional as K
    base = _matrix((1024, 1024), 14, "noise", dtype)
    copies = 1 << 10
    out = K.orthogonalize(base.repeat(1, copies))
    assert out.numel() == 1 << 30
    want, off = _definition(base, eps=0.0)
    # the rounding errors of the sums over the long axis add like the root of its length
    off, want, half = off * copies ** 0.5, want / 32, torch.finfo(dtype).eps / 2
    for k in range(0, copies, 32):
        d = (out[:, k * 1024:(k + 32) * 1024].reshape(1024, 32, 1024).double() - want.unsqueeze(1)).square().sum((0, 2)).sqrt()
        assert bool((d <= off / 32 * (1 + half) + half * want.square().sum().sqrt()).all()), k
    with pytest.raises(RuntimeError):
        K.orthogonalize(torch.empty(1025, 1 << 20, device="cuda", dtype=dtype))
    del out
    torch.cuda.empty_cache()


def test_a_vector_of_two_to_the_30():
    from pde_amd.optim import Muon
    p = torch.nn.Parameter(torch.zeros(1 << 30, device="cuda"))
    p.grad = torch.randn(1 << 30, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3))
    Muon([p], lr=1.0, momentum=0.0, ns_steps=1, ns_coefficients=(1.0, 0.0, 0.0), adjust_lr="none").step()
    norm = sum(float(t.double().square().sum()) for t in p.grad.split(1 << 27)) ** 0.5
    for a, g in zip(p.detach().split(1 << 27), p.grad.split(1 << 27)):
        assert torch.allclose(a, -g / norm, rtol=2e-6, atol=0)
    del p
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("shape", [(64, 40), (256, 300), (300, 256), (3, 160, 200), (1, 4096)])
def test_any_alignment(shape, dtype):
    """A matrix may start anywhere: wide reads where they fit, single ones where not."""
    from pde_amd import functional as K
    flat = torch.empty(_matrix(shape, 0).numel() + 8, device="cuda", dtype=dtype)
    for start in (0, 1, 2, 4, 5):
        g = flat[start:start + flat.numel() - 8].view(shape)
        g.copy_(_matrix(shape, 21, dtype=dtype))
        _check(K.orthogonalize(g), *_definition(g))
