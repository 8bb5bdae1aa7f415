"""Refusals of the group norm (they come before any kernel) and its defining expression, on the CPU."""
import ctypes

import pytest
import torch


def _lib():
    from pde_amd import _lib
    return _lib.load()


FAKE = 0x1000        # never dereferenced: every call below is refused before a launch


@pytest.mark.parametrize("n,s,c,g,word", [(4, 1, 6, 4, b"divide"), (0, 1, 8, 2, b"empty"), (4, 0, 8, 2, b"empty"),
                                          (4, 1, 8, 0, b"empty"), (4, 1, 8200, 1, b"8192"), (4, 1 << 25, 8, 1, b"many"),
                                          (1 << 24, 40, 8, 1, b"samples")])
def test_bad_shapes_are_refused(n, s, c, g, word):
    lib = _lib()
    assert lib.pdekan_group_norm_workspace_bytes(n, s, c, g, 1) == 0
    assert word in lib.pdekan_last_error()
    assert lib.pdekan_group_norm_stats_floats(n, s, c, g) == -1
    assert lib.pdekan_group_norm_forward(FAKE, 0, n, s, c, g, None, None, 1e-5, 0, FAKE, None, None, 0, None) == -1
    assert lib.pdekan_group_norm_backward(FAKE, FAKE, 0, n, s, c, g, None, None, 1e-5, 0, None, FAKE, None, None, None, 0,
                                          None) == -1


def test_bad_arguments_are_refused():
    lib = _lib()
    fwd = lambda **k: lib.pdekan_group_norm_forward(
        k.get("x", FAKE), k.get("dtype", 0), 4, k.get("s", 1), 8, 2, None, None, k.get("eps", 1e-5), k.get("act", 0),
        k.get("y", FAKE), None, k.get("ws"), k.get("ws_bytes", 0), None)
    assert fwd(x=None) == -1 and fwd(y=None) == -1 and fwd(dtype=3) == -1 and fwd(dtype=-1) == -1
    assert fwd(act=3) == -1 and fwd(act=-1) == -1
    assert fwd(eps=-1.0) == -1 and fwd(eps=float("nan")) == -1 and fwd(eps=float("inf")) == -1
    need = lib.pdekan_group_norm_workspace_bytes(4, 4096, 8, 2, 0)
    assert need > 0
    assert fwd(s=4096) == -2                                               # none given
    assert fwd(s=4096, ws=FAKE, ws_bytes=need - 1) == -2                   # too small
    assert fwd(s=4096, ws=FAKE + 16, ws_bytes=need) == -2                  # misaligned
    need = lib.pdekan_group_norm_workspace_bytes(4, 4096, 8, 2, 1)
    assert lib.pdekan_group_norm_backward(FAKE, FAKE, 0, 4, 4096, 8, 2, None, None, 1e-5, 0, None, FAKE, None, None, FAKE,
                                          need, None) == -1                # the statistics of the forward are missing
    assert b"statistics" in lib.pdekan_last_error()


def test_bad_jets_are_refused():
    lib = _lib()
    fwd = lambda **k: lib.pdekan_group_norm_jet_forward(
        k.get("x", FAKE), k.get("n", 4), k.get("c", 8), k.get("g", 2), k.get("nd", 2), k.get("ns", 1), None, None, 1e-5,
        k.get("act", 0), k.get("y", FAKE), None)
    assert fwd(nd=0, ns=0) == -1 and fwd(nd=2, ns=2) == -1 and fwd(nd=6, ns=1) == -1 and fwd(nd=0, ns=1) == -1
    assert fwd(x=None) == -1 and fwd(y=None) == -1 and fwd(n=0) == -1 and fwd(c=7) == -1 and fwd(act=9) == -1
    assert fwd(x=FAKE + 4) == -1 and b"aligned" in lib.pdekan_last_error()
    assert fwd(c=1026, g=2) == -1 and b"512" in lib.pdekan_last_error()
    bwd = lambda gy, gx, ws, n=1 << 20: lib.pdekan_group_norm_jet_backward(
        FAKE, gy, n, 8, 2, 2, 1, None, None, 1e-5, 0, gx, None, None, ws, 64, None)
    assert bwd(None, FAKE, FAKE) == -1 and bwd(FAKE, None, FAKE) == -1 and bwd(FAKE, FAKE, FAKE) == -2
    assert bwd(FAKE + 8, FAKE, FAKE, n=1) == -1 and b"aligned" in lib.pdekan_last_error()


def test_python_entry_points_refuse():
    from pde_amd import functional as K
    from pde_amd.norm import GroupNormAct
    x = torch.randn(4, 8)
    with pytest.raises(RuntimeError):
        K.group_norm_act(x, 2)                                            # no CPU implementation
    with pytest.raises(RuntimeError):
        K.group_norm_act_jet(torch.randn(4, 8, 4), 2)
    for bad in (lambda: K.group_norm_act(x, 3), lambda: K.group_norm_act(x, 0), lambda: K.group_norm_act(x[0], 2),
                lambda: K.group_norm_act(x, 2, torch.ones(7)), lambda: K.group_norm_act(x, 2, None, torch.ones(1, 8)),
                lambda: K.group_norm_act(x, 2, eps=-1.0), lambda: K.group_norm_act(x, 2, eps=float("nan")),
                lambda: K.group_norm_act(x, 2, act=7), lambda: GroupNormAct(3, 8), lambda: GroupNormAct(0, 8),
                lambda: K.group_norm_act_jet(torch.randn(4, 8, 4), 2, n_dir=2, n_second=2),
                lambda: K.group_norm_act_jet(torch.randn(4, 8, 5), 2), lambda: K.group_norm_act_jet(x, 2)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(NotImplementedError):
        GroupNormAct(2, 8, activation=torch.nn.GELU).forward_jet(torch.randn(4, 8, 4), 2, 1)


@pytest.mark.parametrize("shape,groups", [((5, 12), 3), ((3, 7, 12), 4), ((2, 3, 5, 6), 1), ((4, 6), 6)])
def test_expression_is_the_group_norm(shape, groups):
    """The tensor-code route (torch.func transforms, recorded backwards) against torch's own norm, in 64 bits."""
    from torch.func import jvp
    from pde_amd import functional as K
    gen = torch.Generator().manual_seed(0)
    x = torch.randn(shape, dtype=torch.float64, generator=gen)
    w, b = torch.randn(2, shape[-1], dtype=torch.float64, generator=gen)
    for act, f in ((K.ACT_IDENTITY, lambda t: t), (K.ACT_SILU, torch.nn.functional.silu), (K.ACT_TANH, torch.tanh)):
        want = lambda t: f(torch.nn.functional.group_norm(t.movedim(-1, 1), groups, w, b, 1e-5).movedim(1, -1))
        v = torch.randn(shape, dtype=torch.float64, generator=gen)
        y, dy = jvp(lambda t: K.group_norm_act(t, groups, w, b, 1e-5, act), (x,), (v,))
        assert torch.allclose(y, want(x), rtol=1e-11, atol=1e-11)
        h = 1e-5                                                            # central difference: error h^2 + 1e-16 / h
        assert torch.allclose(dy, (want(x + h * v) - want(x - h * v)) / (2 * h), rtol=1e-6, atol=1e-6)
