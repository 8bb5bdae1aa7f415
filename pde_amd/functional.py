"""``torch.autograd.Function`` wrappers around the C ABI of libpdekan.so.

PyTorch is used here for device memory, streams and the autograd tape only;
every number comes out of the HIP kernels.  Tensors handed to the library must
live on a ROCm device - a CPU tensor raises instead of taking another path.
"""
from __future__ import annotations

import contextlib
import ctypes
import functools
import math
from typing import Optional, Sequence, Tuple, Union

import torch

from . import _lib
from ._lib import PdekanLayer, PdekanLayerGrad, PdekanMatrix

ACT_IDENTITY = 0
ACT_SILU = 1
ACT_TANH = 2                      # group norm only

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}   # element types of the group norm and orthogonalize


def _require_gpu(t: torch.Tensor, what: str) -> None:
    if not t.is_cuda:
        raise RuntimeError(
            f"pde_amd: {what} is on {t.device}; the KAN hot path runs only on a ROCm GPU "
            "(there is no CPU implementation in this package)")
    if t.dtype != torch.float32:
        raise TypeError(f"pde_amd: {what} must be float32, got {t.dtype}")


def _require_gpu_float(t: torch.Tensor, what: str) -> None:
    if not t.is_cuda:
        raise RuntimeError(f"pde_amd: {what} is on {t.device}; this operator runs only on a ROCm GPU "
                           "(there is no CPU implementation in this package)")
    if t.dtype not in DTYPES:
        raise TypeError(f"pde_amd: {what} must be float32, bfloat16 or float16, got {t.dtype}")


def under_func_transform() -> bool:
    """True inside a torch.func transform (grad / vmap / jvp level), also where a call's own tensors are not wrapped."""
    return torch._C._are_functorch_transforms_active()


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def _stream(device) -> ctypes.c_void_p:
    return ctypes.c_void_p(torch.cuda.current_stream(device).cuda_stream)


_NO_SWITCH = contextlib.nullcontext()


def _on(device):
    """The tensors' device as the current one; switching costs host time, so only where it is not already."""
    return _NO_SWITCH if torch.cuda.current_device() == device.index else torch.cuda.device(device)


def _raw_stream(device) -> int:
    return torch._C._cuda_getCurrentRawStream(device.index)


def layer_struct(grid, base_weight, spline_weight, spline_scaler, act_kind, grid_size, spline_order) -> PdekanLayer:
    out_f, in_f = base_weight.shape
    return PdekanLayer(in_f, out_f, grid_size, spline_order, act_kind, 0,
                       grid.data_ptr(), base_weight.data_ptr(), spline_weight.data_ptr(),
                       0 if spline_scaler is None else spline_scaler.data_ptr())


def _workspace(nbytes: int, device) -> torch.Tensor:
    # torch's caching allocator returns 512-byte aligned blocks
    return torch.empty(max(int(nbytes), 256), dtype=torch.uint8, device=device)


def _prep(t: Optional[torch.Tensor], what: str) -> Optional[torch.Tensor]:
    if t is None:
        return None
    t = t.detach()
    _require_gpu(t, what)
    return t.contiguous()


def seed_jets(x: torch.Tensor, n_dir: int, n_second: int) -> torch.Tensor:
    """Input jets ``[N, d, J]`` of points ``x [N, d]`` (strided views welcome)."""
    _require_gpu(x, "x")
    assert x.dim() == 2
    lib = _lib.load()
    n, d = x.shape
    jet = torch.empty(n, d, 1 + n_dir + n_second, dtype=torch.float32, device=x.device)
    xd = x.detach()
    with torch.cuda.device(x.device):
        _lib.check(lib.pdekan_seed_jets(_ptr(xd), xd.stride(0), xd.stride(1), n, d, n_dir, n_second,
                                        _ptr(jet), _stream(x.device)))
    return jet


def _dense_layer(x, grid, base_weight, spline_weight, spline_scaler, act_kind, grid_size, spline_order):
    """``KANLinear.forward`` (kan.py:153-166) of ``x [N, in]`` as its defining expression around the dense-basis
    kernel: every op in it is differentiable to any order (``_BasisDense`` carries its own derivative rule)."""
    bases = _BasisDense.apply(x, grid, 0, grid_size, spline_order)
    act = torch.nn.functional.silu(x) if act_kind == ACT_SILU else x
    w = spline_weight if spline_scaler is None else spline_weight * spline_scaler.unsqueeze(-1)
    return torch.nn.functional.linear(act, base_weight) + \
        torch.nn.functional.linear(bases.reshape(x.size(0), -1), w.reshape(w.size(0), -1))


class _KanLayerJet(torch.autograd.Function):
    """y_jet = layer(x_jet); backward gives gx_jet and the parameter gradients.

    First-order backward (``loss.backward()``, run1.py:225) is the library's backward kernels.  A backward that is
    itself being recorded (``torch.autograd.grad(..., create_graph=True)``, the nested-gradient way of forming
    the s_x / s_xx of run1.py:122-123) cannot come from an opaque kernel call: for plain values (J = 1) it is then
    formed by differentiating the layer's defining expression around the dense-basis kernel, which is closed under
    differentiation of any order; for jets (J > 1) it raises - ``forward_jet`` already carries those derivatives."""

    @staticmethod
    def forward(ctx, x_jet, grid, base_weight, spline_weight, spline_scaler, act_kind, grid_size,
                spline_order, n_dir, n_second):
        lib = _lib.load()
        xj = _prep(x_jet, "input")
        g, bw, sw = _prep(grid, "grid"), _prep(base_weight, "base_weight"), _prep(spline_weight, "spline_weight")
        sc = _prep(spline_scaler, "spline_scaler")
        n, in_f, j = xj.shape
        assert j == 1 + n_dir + n_second and in_f == bw.shape[1]
        layer = layer_struct(g, bw, sw, sc, act_kind, grid_size, spline_order)
        y = torch.empty(n, bw.shape[0], j, dtype=torch.float32, device=xj.device)
        with torch.cuda.device(xj.device):
            ws = _workspace(lib.pdekan_layer_workspace_bytes(ctypes.byref(layer), n, n_dir, n_second), xj.device)
            _lib.check(lib.pdekan_layer_forward(ctypes.byref(layer), _ptr(xj), _ptr(y), n, n_dir, n_second,
                                                _ptr(ws), ws.numel(), _stream(xj.device)))
        # the inputs themselves (not detached copies): a recorded backward differentiates through them
        ctx.save_for_backward(x_jet, grid, base_weight, spline_weight,
                              spline_scaler if spline_scaler is not None else torch.empty(0))
        ctx.meta = (act_kind, grid_size, spline_order, n_dir, n_second, spline_scaler is not None)
        return y

    @staticmethod
    def backward(ctx, gy):
        x_jet, grid, base_weight, spline_weight, spline_scaler = ctx.saved_tensors
        act_kind, grid_size, spline_order, n_dir, n_second, has_sc = ctx.meta
        spline_scaler = spline_scaler if has_sc else None
        if torch.is_grad_enabled():                    # this backward is being recorded (create_graph=True)
            return _KanLayerJet._recorded_backward(ctx, gy, x_jet, grid, base_weight, spline_weight, spline_scaler)
        lib = _lib.load()
        xj = _prep(x_jet, "input")
        g, bw, sw = _prep(grid, "grid"), _prep(base_weight, "base_weight"), _prep(spline_weight, "spline_weight")
        sc = _prep(spline_scaler, "spline_scaler")
        gy = _prep(gy, "grad_output")
        n = xj.shape[0]
        layer = layer_struct(g, bw, sw, sc, act_kind, grid_size, spline_order)
        need_x = ctx.needs_input_grad[0]
        need_w = any(ctx.needs_input_grad[2:5])
        gx = torch.empty_like(xj) if need_x else None
        gbw = torch.empty_like(bw) if need_w else None
        gsw = torch.empty_like(sw) if need_w else None
        gsc = torch.empty_like(sc) if (need_w and has_sc) else None
        grads = PdekanLayerGrad(0 if gbw is None else gbw.data_ptr(), 0 if gsw is None else gsw.data_ptr(),
                                0 if gsc is None else gsc.data_ptr())
        with torch.cuda.device(xj.device):
            ws = _workspace(lib.pdekan_layer_workspace_bytes(ctypes.byref(layer), n, n_dir, n_second), xj.device)
            _lib.check(lib.pdekan_layer_backward(ctypes.byref(layer), _ptr(xj), _ptr(gy), n, n_dir, n_second,
                                                 _ptr(gx), ctypes.byref(grads) if need_w else None, 0,
                                                 _ptr(ws), ws.numel(), _stream(xj.device)))
        return gx, None, gbw, gsw, gsc, None, None, None, None, None

    @staticmethod
    def _recorded_backward(ctx, gy, x_jet, grid, base_weight, spline_weight, spline_scaler):
        act_kind, grid_size, spline_order, n_dir, n_second, _ = ctx.meta
        if n_dir or n_second:
            raise RuntimeError(
                "pde_amd: a differentiable backward (create_graph=True) through a layer on jets is not provided; "
                "KAN.forward_jet already returns the input derivatives that nested gradients would form, and its "
                "first-order backward gives their parameter gradients")
        with torch.enable_grad():
            # of views: where one input was computed from another, each derivative is that of the layer alone
            x_jet, base_weight, spline_weight, spline_scaler = (
                t if t is None else t.view_as(t) for t in (x_jet, base_weight, spline_weight, spline_scaler))
            y = _dense_layer(x_jet.squeeze(-1), grid, base_weight, spline_weight, spline_scaler, act_kind, grid_size,
                             spline_order).unsqueeze(-1)
            wanted = [(i, t) for i, t in ((0, x_jet), (2, base_weight), (3, spline_weight), (4, spline_scaler))
                      if t is not None and ctx.needs_input_grad[i]]
            got = torch.autograd.grad(y, [t for _, t in wanted], gy, create_graph=True, allow_unused=True)
        out = [None] * 10
        for (i, _), g in zip(wanted, got):
            out[i] = g
        return tuple(out)


def kan_layer_jet(x_jet, grid, base_weight, spline_weight, spline_scaler, act_kind, grid_size, spline_order,
                  n_dir, n_second):
    return _KanLayerJet.apply(x_jet, grid, base_weight, spline_weight, spline_scaler, act_kind, grid_size,
                              spline_order, n_dir, n_second)


def kan_layer(x, grid, base_weight, spline_weight, spline_scaler, act_kind, grid_size, spline_order):
    """``KANLinear.forward`` on a 2-D batch ``[N, in] -> [N, out]`` with
    first-order autograd (values are jets with J = 1)."""
    _require_gpu(x, "x")
    y = _KanLayerJet.apply(x.contiguous().unsqueeze(-1), grid, base_weight, spline_weight, spline_scaler,
                           act_kind, grid_size, spline_order, 0, 0)
    return y.squeeze(-1)


class _BasisDense(torch.autograd.Function):
    """Dense B-spline bases ``[N, in, coeff]`` of ``x [N, in]`` or their ``order``-th derivative with respect to
    ``x``, as ONE elementwise kernel that knows its own derivative: the backward (and the forward-mode rule) of
    order k is order k+1 times the incoming tangent / cotangent, order 4 of a cubic is zero, and a batched call
    folds the batch into the rows.  That closes the op under ``torch.func`` transforms of any depth (``jacrev``,
    ``hessian``, ``vmap``, ``grad``), which is what lets ``KANLinear.forward`` stay on the GPU kernels under them."""

    generate_vmap_rule = False

    @staticmethod
    def forward(x, grid, order, grid_size, spline_order):
        _require_gpu(x, "x")
        lib = _lib.load()
        xd = x.detach().contiguous()
        gd = grid.detach().contiguous()
        n, in_f = xd.shape
        out = torch.empty(n, in_f, grid_size + spline_order, dtype=torch.float32, device=x.device)
        if n > 0:
            with torch.cuda.device(x.device):
                _lib.check(lib.pdekan_basis_dense(_ptr(gd), _ptr(xd), n, in_f, grid_size, spline_order, order,
                                                  _ptr(out), _stream(x.device)))
        return out

    @staticmethod
    def setup_context(ctx, inputs, output):
        x, grid, order, grid_size, spline_order = inputs
        ctx.save_for_backward(x, grid)
        ctx.save_for_forward(x, grid)
        ctx.meta = (order, grid_size, spline_order)

    @staticmethod
    def backward(ctx, gout):
        x, grid = ctx.saved_tensors
        order, grid_size, spline_order = ctx.meta
        if order >= spline_order:                      # derivative of a piecewise constant
            return torch.zeros_like(x), None, None, None, None
        nxt = _BasisDense.apply(x, grid, order + 1, grid_size, spline_order)
        return (gout * nxt).sum(-1), None, None, None, None

    @staticmethod
    def jvp(ctx, x_t, grid_t, *_):
        x, grid = ctx.saved_tensors
        order, grid_size, spline_order = ctx.meta
        if x_t is None or order >= spline_order:
            return torch.zeros(x.shape + (grid_size + spline_order,), dtype=x.dtype, device=x.device)
        return _BasisDense.apply(x, grid, order + 1, grid_size, spline_order) * x_t.unsqueeze(-1)

    @staticmethod
    def vmap(info, in_dims, x, grid, order, grid_size, spline_order):
        x_bdim, grid_bdim = in_dims[0], in_dims[1]
        if grid_bdim is not None:
            raise NotImplementedError("pde_amd: a batched knot grid under vmap is not supported")
        if x_bdim is None:
            return _BasisDense.apply(x, grid, order, grid_size, spline_order), None
        xb = x.movedim(x_bdim, 0)                      # [B, N, in]: the op is row-wise, so the batch folds into N
        b, n, in_f = xb.shape
        out = _BasisDense.apply(xb.reshape(b * n, in_f), grid, order, grid_size, spline_order)
        return out.view(b, n, in_f, -1), 0


def basis_dense(x: torch.Tensor, grid: torch.Tensor, grid_size: int, spline_order: int, order: int = 0) -> torch.Tensor:
    """``b_splines`` (kan.py:78-111) of ``x [N, in]`` on the GPU kernel, ``[N, in, grid_size + spline_order]``;
    differentiable in ``x`` to any order and usable under ``torch.func`` transforms."""
    return _BasisDense.apply(x, grid, order, grid_size, spline_order)


def fit_coefficients(x: torch.Tensor, grid: torch.Tensor, grid_size: int, spline_order: int,
                     y: Optional[torch.Tensor] = None, old_grid: Optional[torch.Tensor] = None,
                     old_spline_weight: Optional[torch.Tensor] = None,
                     old_spline_scaler: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``curve2coeff`` (kan.py:113-143) on the GPU: ``[out, in, grid_size + spline_order]`` least-squares spline
    coefficients through ``x [N, in]`` and ``y [N, in, out]`` (any strides), solved per feature in fp64 inside one
    kernel.  With ``y=None`` the samples are the edge functions of the layer given by ``old_grid`` /
    ``old_spline_weight`` / ``old_spline_scaler`` - the refit of ``update_grid`` (kan.py:173-180, :215) without
    the ``[N, in, out]`` tensor."""
    _require_gpu(x, "x")
    lib = _lib.load()
    n, in_f = x.shape
    gd = grid.detach().contiguous()
    xd = x.detach()
    if y is not None:
        yd = y.detach()
        out_f = yd.shape[2]
        ys = yd.stride()
        og = ow = osc = None
    else:
        yd, ys = None, (0, 0, 0)
        og = old_grid.detach().contiguous()
        ow = old_spline_weight.detach().contiguous()
        osc = None if old_spline_scaler is None else old_spline_scaler.detach().contiguous()
        out_f = ow.shape[0]
    coeff = torch.empty(out_f, in_f, grid_size + spline_order, dtype=torch.float32, device=x.device)
    with torch.cuda.device(x.device):
        _lib.check(lib.pdekan_fit_coefficients(_ptr(gd), _ptr(xd), xd.stride(0), xd.stride(1), n, in_f, out_f, grid_size,
                                               spline_order, _ptr(yd), ys[0], ys[1], ys[2], _ptr(og), _ptr(ow),
                                               _ptr(osc), _ptr(coeff), _stream(x.device)))
    return coeff


def fit_on_device(x: torch.Tensor, grid_size: int, spline_order: int) -> bool:
    """Whether ``fit_coefficients`` takes these samples (float32 on a GPU, cubic splines, at most 20 intervals)."""
    return x.is_cuda and x.dtype == torch.float32 and spline_order == 3 and 1 <= grid_size <= 20 and x.size(0) > 0


# ---- group norm with an activation, channels last ---------------------------------------------------------------------

def _norm_check(channels: int, groups: int, weight, bias, eps: float, act: int) -> None:
    if groups < 1 or channels < 1 or channels % groups:
        raise ValueError(f"pde_amd: {channels} channels do not divide into {groups} groups")
    for t, what in ((weight, "weight"), (bias, "bias")):
        if t is not None and tuple(t.shape) != (channels,):
            raise ValueError(f"pde_amd: the norm's {what} must have shape ({channels},), got {tuple(t.shape)}")
    if not 0.0 <= eps < float("inf"):
        raise ValueError(f"pde_amd: eps must be finite and not negative, got {eps}")
    if act not in (ACT_IDENTITY, ACT_SILU, ACT_TANH):
        raise ValueError(f"pde_amd: activation kind {act} unknown")


def _group_norm_expression(x, groups, weight, bias, eps, act):
    """``group_norm_act`` as its defining expression, differentiable to any order and under ``torch.func``."""
    v = x.reshape(x.size(0), math.prod(x.shape[1:-1]), groups, x.size(-1) // groups)        # (0 samples leave no -1 to infer)
    if v.dtype in (torch.bfloat16, torch.float16):
        v = v.float()
    v = v - v.mean((1, 3), keepdim=True)
    z = (v * torch.rsqrt((v * v).mean((1, 3), keepdim=True) + eps)).reshape(x.shape)
    z = z if weight is None else z * weight
    z = z if bias is None else z + bias
    z = torch.nn.functional.silu(z) if act == ACT_SILU else torch.tanh(z) if act == ACT_TANH else z
    return z.to(x.dtype)


@functools.lru_cache(maxsize=1024)
def _norm_sizes(n: int, s: int, c: int, groups: int):
    """(floats of statistics, workspace bytes of the forward, of the backward) of a shape the library takes."""
    lib = _lib.load()
    floats = lib.pdekan_group_norm_stats_floats(n, s, c, groups)
    if floats < 0:
        _lib.check(int(floats))
    return (floats, lib.pdekan_group_norm_workspace_bytes(n, s, c, groups, 0),
            lib.pdekan_group_norm_workspace_bytes(n, s, c, groups, 1))


def _address(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _contiguous(t: Optional[torch.Tensor]):
    return t if t is None or t.is_contiguous() else t.contiguous()


def _group_norm_forward(x, weight, bias, groups, eps, act, keep_stats):
    """The value and, where the backward wants it, the statistics."""
    xd, w, b = _contiguous(x), _contiguous(weight), _contiguous(bias)
    y = torch.empty_like(xd)
    stats = None
    n, c = xd.shape[0], xd.shape[-1]
    if y.numel():
        s = y.numel() // (n * c)
        floats, need, _ = _norm_sizes(n, s, c, groups)
        device = x.device
        if floats and keep_stats:
            stats = torch.empty(floats, dtype=torch.float32, device=device)
        ws = _workspace(need, device) if need else None
        with _on(device):
            rc = _lib.load().pdekan_group_norm_forward(xd.data_ptr(), DTYPES[xd.dtype], n, s, c, groups, _address(w),
                                                       _address(b), eps, act, y.data_ptr(), _address(stats),
                                                       _address(ws), need, _raw_stream(device))
        _lib.check(rc)
    return y, stats


def _recorded(*tensors) -> bool:
    """Whether a call on these leaves a trace: a backward, or a forward derivative."""
    if torch.autograd.forward_ad._current_level >= 0:
        return True
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


class _GroupNormAct(torch.autograd.Function):
    """First-order backward on the kernels; a recorded backward (``create_graph=True``) differentiates the expression."""

    @staticmethod
    def forward(ctx, x, weight, bias, groups, eps, act):
        y, stats = _group_norm_forward(x, weight, bias, groups, eps, act, any(ctx.needs_input_grad))
        ctx.save_for_backward(x, weight, bias, stats)
        ctx.meta = (groups, eps, act)
        return y

    @staticmethod
    def backward(ctx, gy):
        x, weight, bias, stats = ctx.saved_tensors
        groups, eps, act = ctx.meta
        if torch.is_grad_enabled():                    # this backward is being recorded (create_graph=True)
            # of views: where one input was computed from another, each derivative is that of the norm alone
            own = [t if t is None else t.view_as(t) for t in (x, weight, bias)]
            y = _group_norm_expression(own[0], groups, own[1], own[2], eps, act)
            wanted = [i for i in range(3) if ctx.needs_input_grad[i]]
            got = torch.autograd.grad(y, [own[i] for i in wanted], gy, create_graph=True, allow_unused=True)
            out = [None] * 6
            for i, g in zip(wanted, got):
                out[i] = g
            return tuple(out)
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        xd = _contiguous(x)
        gd = _contiguous(gy)
        w = _contiguous(weight)
        b = _contiguous(bias)
        n, c = xd.shape[0], xd.shape[-1]
        gx = torch.empty_like(xd)
        gw = torch.empty_like(w) if need_w else None
        gb = torch.empty_like(b) if need_b else None
        if gx.numel():
            s = gx.numel() // (n * c)
            need = _norm_sizes(n, s, c, groups)[2]
            device = x.device
            ws = _workspace(need, device) if need else None
            with _on(device):
                rc = _lib.load().pdekan_group_norm_backward(xd.data_ptr(), gd.data_ptr(), DTYPES[xd.dtype], n, s, c, groups,
                                                            _address(w), _address(b), eps, act, _address(stats),
                                                            gx.data_ptr(), _address(gw), _address(gb), _address(ws), need,
                                                            _raw_stream(device))
            _lib.check(rc)
        else:
            for g in (gw, gb):
                if g is not None:
                    g.zero_()
        return gx if need_x else None, gw, gb, None, None, None


def group_norm_act(x: torch.Tensor, groups: int, weight: Optional[torch.Tensor] = None,
                   bias: Optional[torch.Tensor] = None, eps: float = 1e-5, act: int = ACT_IDENTITY) -> torch.Tensor:
    """``act(group_norm(x) * weight + bias)`` with the channels last.

    ``x`` is ``[N, C]`` or ``[N, ..., C]`` in float32, bfloat16 or float16; the statistics of a group run over the
    positions of a sample and the ``C / groups`` channels of the group (biased variance), in float32 or more whatever the type.
    ``weight`` and ``bias`` are ``[C]`` or None; other types than float32 are converted.  ``act`` is one of
    ``ACT_IDENTITY``, ``ACT_SILU``, ``ACT_TANH``.  Differentiable in ``x``, ``weight`` and ``bias`` (to any order; beyond the
    first on tensor code) and usable under ``torch.func`` transforms (tensor code).  At most 8192 channels."""
    if x.dim() < 2:
        raise ValueError(f"pde_amd: the norm takes [N, ..., channels], got {tuple(x.shape)}")
    _norm_check(x.size(-1), groups, weight, bias, eps, act)
    if under_func_transform():
        return _group_norm_expression(x, groups, weight, bias, eps, act)
    _require_gpu_float(x, "x")
    weight = weight if weight is None or weight.dtype == torch.float32 else weight.to(torch.float32)
    bias = bias if bias is None or bias.dtype == torch.float32 else bias.to(torch.float32)
    _same_device(x, weight, bias)
    if not _recorded(x, weight, bias):
        return _group_norm_forward(x, weight, bias, int(groups), float(eps), int(act), False)[0]
    return _GroupNormAct.apply(x, weight, bias, int(groups), float(eps), int(act))


def _same_device(x, *others) -> None:
    for t in others:
        if t is not None and t.device != x.device:
            raise RuntimeError(f"pde_amd: tensors on {x.device} and {t.device} in one call")


def _group_norm_jet_forward(x_jet, weight, bias, groups, eps, act, n_dir, n_second):
    xd, w, b = _aligned(_contiguous(x_jet)), _contiguous(weight), _contiguous(bias)
    n, c, _ = xd.shape
    y = torch.empty_like(xd)
    if n:
        device = x_jet.device
        with _on(device):
            rc = _lib.load().pdekan_group_norm_jet_forward(xd.data_ptr(), n, c, groups, n_dir, n_second, _address(w),
                                                           _address(b), eps, act, y.data_ptr(), _raw_stream(device))
        _lib.check(rc)
    return y


class _GroupNormActJet(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x_jet, weight, bias, groups, eps, act, n_dir, n_second):
        y = _group_norm_jet_forward(x_jet, weight, bias, groups, eps, act, n_dir, n_second)
        ctx.save_for_backward(x_jet, weight, bias)
        ctx.meta = (groups, eps, act, n_dir, n_second)
        return y

    @staticmethod
    def backward(ctx, gy):
        if torch.is_grad_enabled():
            raise RuntimeError("pde_amd: a differentiable backward (create_graph=True) through a norm on jets is not "
                               "provided; KAN.forward_jet already returns the input derivatives")
        x_jet, weight, bias = ctx.saved_tensors
        groups, eps, act, n_dir, n_second = ctx.meta
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        xd = _aligned(_contiguous(x_jet))
        gd = _aligned(_contiguous(gy))
        w = _contiguous(weight)
        b = _contiguous(bias)
        n, c, _ = xd.shape
        gx = torch.empty_like(xd)
        gw = torch.empty_like(w) if need_w else None
        gb = torch.empty_like(b) if need_b else None
        if n:
            device = x_jet.device
            need = _norm_sizes(n, 1, c, groups)[2]
            ws = _workspace(need, device) if need else None
            with _on(device):
                rc = _lib.load().pdekan_group_norm_jet_backward(xd.data_ptr(), gd.data_ptr(), n, c, groups, n_dir, n_second,
                                                                _address(w), _address(b), eps, act, gx.data_ptr(),
                                                                _address(gw), _address(gb), _address(ws), need,
                                                                _raw_stream(device))
            _lib.check(rc)
        else:
            for g in (gw, gb):
                if g is not None:
                    g.zero_()
        return (gx if need_x else None, gw, gb) + (None,) * 5


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """A view at an odd offset as a tensor of its own: the jet kernels read 16 bytes at a time."""
    return t if t.data_ptr() % 16 == 0 else t.clone()


def group_norm_act_jet(x_jet: torch.Tensor, groups: int, weight: Optional[torch.Tensor] = None,
                       bias: Optional[torch.Tensor] = None, eps: float = 1e-5, act: int = ACT_IDENTITY, n_dir: int = 2,
                       n_second: int = 1) -> torch.Tensor:
    """:func:`group_norm_act` of points ``[N, C]`` on their jets ``[N, C, 1 + n_dir + n_second]`` (float32): the value and,
    by the chain rule through the statistics, its derivatives, as ``KAN.forward_jet`` carries them.
    (``n_dir``, ``n_second``) is (0, 0), (2, 1) or (6, 5); at most 512 channels a group for the latter two."""
    if x_jet.dim() != 3 or x_jet.size(2) != 1 + n_dir + n_second or (n_dir, n_second) not in ((0, 0), (2, 1), (6, 5)):
        raise ValueError(f"pde_amd: jets [N, C, 1 + n_dir + n_second] of (0, 0), (2, 1) or (6, 5) derivatives wanted, got "
                         f"{tuple(x_jet.shape)} with ({n_dir}, {n_second})")
    if n_dir == 0:
        return group_norm_act(x_jet.squeeze(-1), groups, weight, bias, eps, act).unsqueeze(-1)
    _norm_check(x_jet.size(1), groups, weight, bias, eps, act)
    if under_func_transform():
        raise RuntimeError("pde_amd: a norm on jets does not run inside torch.func transforms")
    _require_gpu(x_jet, "x_jet")
    weight = weight if weight is None or weight.dtype == torch.float32 else weight.to(torch.float32)
    bias = bias if bias is None or bias.dtype == torch.float32 else bias.to(torch.float32)
    _same_device(x_jet, weight, bias)
    if not _recorded(x_jet, weight, bias):
        return _group_norm_jet_forward(x_jet, weight, bias, int(groups), float(eps), int(act), int(n_dir), int(n_second))
    return _GroupNormActJet.apply(x_jet, weight, bias, int(groups), float(eps), int(act), int(n_dir), int(n_second))


# ---- orthogonalised updates ----------------------------------------------------------------------------------------------

# the usual quintic: slope 3.4445 at zero, singular values end up within 0.7 .. 1.2 after five steps
NS_COEFFICIENTS = (3.4445, -4.7750, 2.0315)


def ns_settings(steps: int, eps: float, coefficients: Sequence[float]):
    """(steps, eps, coefficients as a C array), checked."""
    coefficients = tuple(float(c) for c in coefficients)
    if len(coefficients) != 3:
        raise ValueError(f"pde_amd: three Newton-Schulz coefficients wanted, got {len(coefficients)}")
    if not 1 <= int(steps) <= 100:
        raise ValueError(f"pde_amd: 1 to 100 Newton-Schulz steps, got {steps}")
    if not 1e-30 <= eps < float("inf"):
        raise ValueError(f"pde_amd: eps must be at least 1e-30 and finite, got {eps}")
    return int(steps), float(eps), (ctypes.c_float * 3)(*coefficients)


@torch.no_grad()
def orthogonalize(g: Union[torch.Tensor, Sequence[torch.Tensor]], steps: int = 5, eps: float = 1e-7,
                  coefficients: Tuple[float, float, float] = NS_COEFFICIENTS):
    """The nearly orthogonal factor of a matrix ``[rows, cols]``, of each matrix of a stack ``[..., rows, cols]``, or of
    each tensor of a sequence (one list back), by ``steps`` Newton-Schulz products (the update of the Muon optimiser).

    ``X = g / (|g|_F + eps)`` with its short side first, then ``steps`` times ``X <- a X + (b S + c S S) X``, ``S = X X^T``.
    float32, bfloat16 or float16 (one type and device a call); the products have float32 accuracy; the steps of a
    large 16-bit matrix are composed, which leaves about 5e-6 before its one rounding.  Not differentiable.  A matrix holding
    a NaN or an infinity becomes NaN and leaves the others alone."""
    one = isinstance(g, torch.Tensor)
    mats = [g] if one else list(g)
    steps, eps, c = ns_settings(steps, eps, coefficients)
    if not mats:
        return []
    for t in mats:
        if t.dim() < 2:
            raise ValueError(f"pde_amd: orthogonalize takes matrices [..., rows, cols], got {tuple(t.shape)}")
        _require_gpu_float(t, "g")
        if t.dtype != mats[0].dtype:
            raise TypeError(f"pde_amd: matrices of types {mats[0].dtype} and {t.dtype} in one call")
    _same_device(*mats)
    device = mats[0].device
    src = [t if t.is_contiguous() else t.contiguous() for t in mats]
    out = [torch.empty_like(t) for t in src]
    todo = [(s, o) for s, o in zip(src, out) if s.numel()]
    if todo:
        lib = _lib.load()
        desc = (PdekanMatrix * len(todo))()
        for d, (s, o) in zip(desc, todo):
            rows, cols = s.shape[-2:]
            d.g, d.out, d.rows, d.cols, d.batch = s.data_ptr(), o.data_ptr(), rows, cols, s.numel() // (rows * cols)
        need = lib.pdekan_orthogonalize_workspace_bytes(desc, len(todo))
        if need == 0:
            _lib.check(-1)
        ws = _workspace(need, device)
        with _on(device):
            rc = lib.pdekan_orthogonalize(desc, len(todo), DTYPES[src[0].dtype], steps, c, eps, ws.data_ptr(), need,
                                          _raw_stream(device))
        _lib.check(rc)
    return out[0] if one else out
