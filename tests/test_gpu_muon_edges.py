"""Newton-Schulz orthogonalisation and the Muon step where few bits, large values, long lists or shared memory could tell."""
import ctypes

import pytest
import torch

from test_gpu_muon import A, B, C, U, _check, _definition, _matrix

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(160, 1000), (1000, 160), (2, 200, 300), (2090, 2300)])
def test_sixteen_bit_results_are_rounded_once(shape, dtype):
    """Whatever is held between the steps, a 16-bit result is the 64-bit one rounded, but where fp32's error carries a value over
    the border between two roundings.

    An error d of a value whose neighbours lie `ulp` apart changes its rounding with probability |d| / ulp, by ulp: the squares
    of the changes add up to sum |d| ulp + d^2 <= |d| |ulp| + |d|^2 in the mean, and twice that is more than four standard
    deviations away (dozens of changes at least).  The slopes of (1.5, -0.5, 0) leave `off` at a few 2^-24.  Where steps are
    composed, their products carry the multiple of one through the sums: five products of at most 3 m / 32 additions each, of
    which each may be 2 u of the result off: m u."""
    from pde_amd import functional as K
    for steps in (4, 5):
        g = _matrix(shape, steps, "noise", dtype)
        want, off = _definition(g, steps, 1e-7, (1.5, -0.5, 0.0))
        out = K.orthogonalize(g, steps=steps, coefficients=(1.5, -0.5, 0.0))
        fro = lambda t: t.square().sum((-2, -1)).sqrt()
        off = off + min(shape[-2:]) * U * fro(want)
        d = fro(out.double() - want.to(dtype).double())
        tol = (2 * (off * torch.finfo(dtype).eps * fro(want) + off ** 2)).sqrt()
        assert bool((d <= tol).all()), (steps, float((d / fro(want)).max()), float((tol / fro(want)).max()))


@pytest.mark.parametrize("shape,dtype", [((2048, 8192), torch.bfloat16), ((4, 1000, 771), torch.float16), ((256, 5888), torch.float32),
                                         ((2048, 2048), torch.float32)])
def test_the_same_bits_every_time(shape, dtype):
    from pde_amd import functional as K
    g = _matrix(shape, 31, "low rank", dtype)
    first = K.orthogonalize(g)
    for _ in range(4):
        assert torch.equal(K.orthogonalize(g), first)


@pytest.mark.parametrize("mu", [0.5, 0.95, 0.99, 0.999])
@pytest.mark.parametrize("shape", [(1, 60), (1, 70000), (40, 60), (60, 1000), (200, 140)])
def test_the_gradient_s_coefficient(shape, mu):
    """1 - mu comes from 64 bits: the first momentum is (1 - mu) g, two roundings off (the coefficient's and the product's)."""
    from pde_amd.optim import Muon
    p = torch.nn.Parameter(torch.zeros(shape, device="cuda"))
    p.grad = _matrix(shape, 7)
    opt = Muon([p], lr=0.0, momentum=mu)
    opt.step()
    want = (1 - mu) * p.grad.double()
    assert bool(((opt.state[p]["momentum_buffer"].double() - want).abs() <= 2.1 * U * want.abs()).all())


def _error(out, g):
    want = _definition(g)[0]
    return float((out.double() - want).norm() / want.norm())


def test_small_matrices_beside_larger_ones():
    """A matrix of few rows is as accurate in a list that takes more launches as alone: the mean errors of 60 matrices (each varies by
    about a third, their means by 6 percent) within a fifth."""
    from pde_amd import functional as K
    mats = [_matrix((5, 64), 100 + i) for i in range(60)]
    alone = sum(_error(K.orthogonalize(g), g) for g in mats) / 60
    for other in ((300, 300), (60, 1000)):
        beside = 0.0
        for i in range(0, 60, 15):
            out = K.orthogonalize(mats[i:i + 15] + [_matrix(other, 5)])
            beside += sum(_error(o, g) for o, g in zip(out, mats[i:i + 15])) / 60
        assert beside <= 1.2 * alone, (other, beside, alone)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_long_stacks_beside_a_larger_matrix(dtype):
    """Large stacks of small matrices and of vectors in one list with larger ones: no workspace beyond their kind, the same results."""
    from pde_amd import functional as K
    mats = [_matrix(s, i, dtype=dtype) for i, s in enumerate([(20000, 4, 6), (300, 300), (30000, 1, 50), (600, 40, 900), (7, 5, 9)])]
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    out = K.orthogonalize(mats)
    kept = sum(o.numel() * o.element_size() for o in out)
    assert torch.cuda.max_memory_allocated() - before - kept < 1 << 30
    for g, o in zip(mats, out):
        _check(o, *_definition(g))


@pytest.mark.parametrize("kind", ["1e38", "largest", "one largest"])
@pytest.mark.parametrize("shape", [(1, 300), (20, 30), (100, 90), (60, 1000), (200, 140), (140, 200)])
def test_the_largest_values(shape, kind):
    """Entries up to the largest fp32 number, whose norm fp32 does not hold: as accurate as any others."""
    from pde_amd import functional as K
    g = _matrix(shape, 9) * 1e3
    big = torch.finfo(torch.float32).max
    if kind == "one largest":
        g[0, 3] = -big                                           # the rest vanishes beside it
    else:
        g = (g / g.abs().max()).clamp(-1, 1).double() * (1e38 if kind == "1e38" else big)
        g = g.float()
    assert bool(g.isfinite().all())
    _check(K.orthogonalize(g), *_definition(g))


def test_the_largest_values_in_a_step():
    from pde_amd.optim import Muon
    big = torch.finfo(torch.float32).max
    for shape in ((1, 300), (20, 30), (60, 1000), (200, 140)):
        p = torch.nn.Parameter(torch.zeros(shape, device="cuda"))
        g = _matrix(shape, 9)
        p.grad = (g / g.abs().max()).clamp(-1, 1) * big
        Muon([p], lr=1.0, momentum=0.0, adjust_lr="none").step()
        _check(-p.detach(), *_definition(p.grad))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(3, 40, 70), (3, 70, 40), (3, 1, 50), (3, 1, 70000), (3, 200, 140), (3, 60, 1000), (3, 1100, 50)])
def test_all_of_a_non_finite_matrix_is_nan(shape, dtype):
    from pde_amd import functional as K
    g = _matrix(shape, 4, dtype=dtype)
    clean = K.orthogonalize(g)
    for bad in (float("nan"), float("inf"), -float("inf")):
        g[2, 0, 3] = bad
        out = K.orthogonalize(g)
        assert torch.equal(out[:2], clean[:2]) and bool(out[2].isnan().all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_a_result_in_its_matrix_s_place(dtype):
    """`out` may be `g`, on every path and in a list of all of them: the bits of a result in a place of its own."""
    from pde_amd import _lib, functional as K
    lib = _lib.load()
    coefficients = (ctypes.c_float * 3)(A, B, C)

    def run(mats, outs):
        desc = (_lib.PdekanMatrix * len(mats))()
        for d, g, o in zip(desc, mats, outs):
            rows, cols = g.shape[-2:]
            d.g, d.out, d.rows, d.cols, d.batch = g.data_ptr(), o.data_ptr(), rows, cols, g.numel() // (rows * cols)
        need = lib.pdekan_orthogonalize_workspace_bytes(desc, len(mats))
        ws = K._workspace(need, "cuda")
        _lib.check(lib.pdekan_orthogonalize(desc, len(mats), K.DTYPES[dtype], 5, coefficients, 1e-7, ws.data_ptr(), need,
                                            K._raw_stream(mats[0].device)))

    shapes = [(1, 500), (1, 70000), (40, 60), (60, 40), (60, 1000), (1000, 60), (200, 140), (140, 200), (3, 50, 70), (2, 2100, 2050)]
    for group in [[s] for s in shapes] + [shapes[:6], shapes[:9]]:
        mats = [_matrix(s, 40 + i, dtype=dtype) for i, s in enumerate(group)]
        apart = [torch.empty_like(g) for g in mats]
        run(mats, apart)
        run(mats, mats)
        assert all(torch.equal(g, o) for g, o in zip(mats, apart)), group
