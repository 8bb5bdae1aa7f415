"""Refusals of the orthogonalised update and of the Muon optimiser, before any kernel runs."""
import ctypes

import pytest
import torch

FAKE = 0x1000        # never dereferenced: every call below is refused before a launch
C = (ctypes.c_float * 3)(3.4445, -4.7750, 2.0315)


def _lib():
    from pde_amd import _lib
    return _lib.load()


def _mats(*shapes, g=FAKE, out=FAKE):
    from pde_amd._lib import PdekanMatrix
    return (PdekanMatrix * len(shapes))(*[PdekanMatrix(g, out, r, c, b) for r, c, b in shapes])


@pytest.mark.parametrize("shape", [(0, 4, 1), (4, 0, 1), (4, 4, 0), (40000, 40000, 1), (2, 1 << 25, 1), (1 << 31, 1, 1),
                                   (64, 64, 1 << 20), (64, 64, (1 << 17) + 1), (1, 4, (1 << 17) + 1), (32768, 32768, 2)])
def test_bad_matrices_are_refused(shape):
    lib = _lib()
    mats = _mats((8, 8, 1), shape)
    assert lib.pdekan_orthogonalize_workspace_bytes(mats, 2) == 0
    assert b"matrix 1" in lib.pdekan_last_error()
    assert lib.pdekan_orthogonalize(mats, 2, 0, 5, C, 1e-7, FAKE, 1 << 40, None) == -1


def test_bad_arguments_are_refused():
    lib = _lib()
    mats = _mats((8, 8, 1))
    need = lib.pdekan_orthogonalize_workspace_bytes(mats, 1)
    assert need > 0
    run = lambda **k: lib.pdekan_orthogonalize(k.get("mats", mats), k.get("n", 1), k.get("dtype", 0), k.get("steps", 5),
                                               k.get("c", C), k.get("eps", 1e-7), k.get("ws", FAKE), k.get("bytes", need), None)
    big = (ctypes.c_float * 3)(3.4445, 4.7750, 2.0315)
    nan = (ctypes.c_float * 3)(3.4445, float("nan"), 2.0315)
    assert run(mats=None) == -1 and run(n=0) == -1 and run(dtype=3) == -1 and run(steps=0) == -1 and run(steps=101) == -1
    assert run(c=None) == -1 and run(c=big) == -1 and run(c=nan) == -1
    assert run(eps=0.0) == -1 and run(eps=-1.0) == -1 and run(eps=float("nan")) == -1 and run(eps=float("inf")) == -1
    assert run(ws=None) == -2 and run(bytes=need - 1) == -2 and run(ws=FAKE + 8) == -2
    assert run(mats=_mats((8, 8, 1), g=None)) == -1 and run(mats=_mats((8, 8, 1), out=None)) == -1
    # a list of more than one launch: the last entry is refused before the first launch
    many = _mats(*[(8, 8, 1)] * 40)
    many[39].g = None
    assert run(mats=many, n=40, bytes=1 << 40) == -1 and b"matrix 39" in lib.pdekan_last_error()


def test_workspace_is_that_of_the_largest_launch():
    lib = _lib()
    one = lib.pdekan_orthogonalize_workspace_bytes(_mats((100, 200, 1)), 1)
    assert lib.pdekan_orthogonalize_workspace_bytes(_mats(*[(100, 200, 1)] * 16), 16) == 16 * one
    assert lib.pdekan_orthogonalize_workspace_bytes(_mats(*[(100, 200, 1)] * 40), 40) == 16 * one


def test_bad_optimiser_steps_are_refused():
    from pde_amd._lib import PdekanMuonParam
    lib = _lib()

    def run(p=FAKE, g=FAKE, m=FAKE, gain=1.0, lr=0.1, mu=0.9, decay=0.0, steps=5, ws=FAKE, nbytes=1 << 40, shape=(8, 8)):
        par = (PdekanMuonParam * 1)(PdekanMuonParam(p, g, m, *shape, gain, 0))
        return lib.pdekan_muon_step(par, 1, lr, None, mu, 1, decay, steps, C, 1e-7, ws, nbytes, None)

    assert run(p=None) == -1 and run(g=None) == -1 and run(m=None) == -1 and run(gain=-1.0) == -1
    assert run(gain=float("nan")) == -1 and run(lr=-0.1) == -1 and run(lr=float("nan")) == -1 and run(mu=1.0) == -1
    assert run(mu=-0.1) == -1 and run(decay=-1.0) == -1 and run(steps=0) == -1 and run(shape=(0, 8)) == -1
    assert run(ws=None) == -2 and run(nbytes=128) == -2


def test_python_entry_points_refuse():
    from pde_amd import functional as K
    from pde_amd.optim import Muon
    x = torch.randn(4, 8)
    with pytest.raises(RuntimeError):
        K.orthogonalize(x)                                       # no CPU implementation
    assert K.orthogonalize([]) == []
    for bad in (lambda: K.orthogonalize(x[0]), lambda: K.orthogonalize(x, steps=0), lambda: K.orthogonalize(x, eps=0.0),
                lambda: K.orthogonalize(x, coefficients=(1.0, 2.0)), lambda: Muon([x.requires_grad_()], lr=-1.0),
                lambda: Muon([x], momentum=1.0), lambda: Muon([x], weight_decay=-0.1), lambda: Muon([x], ns_steps=0),
                lambda: Muon([x], eps=0.0), lambda: Muon([x], adjust_lr="rms"), lambda: Muon([x], ns_coefficients=(1.0,)),
                lambda: Muon([{"params": [x], "momentum": 1.5}])):
        with pytest.raises(ValueError):
            bad()
    p = torch.nn.Parameter(torch.randn(4, 8))
    p.grad = torch.ones_like(p)
    with pytest.raises(RuntimeError):
        Muon([p]).step()
    opt = Muon([p], lr=0.5)
    assert opt.step.__self__ is opt and opt.param_groups[0]["lr"] == 0.5
    p.grad = None
    opt.step()                                                   # nothing to do


def test_gains():
    from pde_amd.optim import Muon, _matrix_shape
    assert _matrix_shape(torch.empty(4, 3, 5)) == (4, 15) and _matrix_shape(torch.empty(7)) == (1, 7)
    assert _matrix_shape(torch.empty(())) == (1, 1)
    assert Muon._gain(8, 2, "original") == 2.0 and Muon._gain(2, 8, "original") == 1.0
    assert Muon._gain(4, 100, "match_rms_adamw") == 2.0 and Muon._gain(4, 100, "none") == 1.0
