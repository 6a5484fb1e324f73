"""Newton-Schulz orthogonalisation and the fused Muon step on the sm_100a tensor cores.

``orthogonalize`` replaces every singular value of a matrix by a value near 1
with products alone; ``cuda_muon_step_`` is the optimizer step built on it
(momentum stored by a rounding rule, orthogonalised update, parameter).
"""

from __future__ import annotations

import ctypes
import math
import struct

import torch

from ..formats import StateFormat, resolve_formats
from ..rounding import native_codes
from . import _native
from ._fused import rng_words
from ._launch import device_guard, stream_handle
from ._tables import Update, _row_flags
from ._validate import check_disjoint, check_layout, check_nonnegative, spans_of

# a, b, c of X <- (a I + b G + c G^2) X, G = X X^T: the quintic steps that bring
# singular values from (0, 1] to about [0.7, 1.2] in five steps.
NEWTON_SCHULZ = (3.4445, -4.7750, 2.0315)
SCALE_RULES = ("spectral", "rms")

_FORMATS = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
# Matrices of one shape are updated together, as many as this much workspace holds.
_WORKSPACE_BYTES = 2 << 30


def newton_settings(steps, coefficients, eps) -> _native.SrsNewton:
    if isinstance(steps, bool) or not isinstance(steps, int) or not (
            1 <= steps <= _native.NEWTON_MAX_STEPS):
        raise ValueError(f"steps must be an integer in [1, {_native.NEWTON_MAX_STEPS}]")
    coefficients = tuple(float(c) for c in coefficients)
    if len(coefficients) != 3 or not all(math.isfinite(c) for c in coefficients):
        raise ValueError("coefficients must be three finite numbers")
    check_nonnegative("eps", eps)
    newton = _native.SrsNewton()
    newton.steps, newton.eps = steps, eps
    newton.coefficients[:] = coefficients
    return newton


def update_scale(rule: str, m: int, n: int) -> float:
    """Factor of the learning rate for an m x n matrix: ``"spectral"``
    sqrt(max(1, m / n)), ``"rms"`` 0.2 * sqrt(max(m, n)) (the update's root mean
    square is then about 0.2, as AdamW's is)."""
    if rule == "spectral":
        return max(1.0, m / n) ** 0.5
    if rule == "rms":
        return 0.2 * max(m, n) ** 0.5
    raise ValueError(f"scale must be one of {SCALE_RULES}")


def orthogonalize(x, *, steps=5, coefficients=NEWTON_SCHULZ, eps=1e-7, dtype=None):
    """Newton-Schulz orthogonalisation of the matrices in the last two dimensions of ``x``.

    X_0 = x / (|x|_F + eps), then ``steps`` times X <- (a I + b G + c G^2) X with
    G = X X^T (for tall matrices X (a I + b G + c G^2), G = X^T X).  ``dtype``
    (default: that of ``x``) is the result's and sets the products' precision: BF16
    results come from FP16 operands (relative errors of the whole matrix of 1e-3 to 3e-3,
    about those of rounding it to BF16; up to 6e-3 for a few orthogonal rows and for ranks
    of a few at sides of ten thousand), FP16 and FP32 results from pairs of FP16 operands
    (1e-5 for sides of some hundreds, 1e-4 for ten thousand; 3e-4 and 3e-3 with ranks of a
    few; three times the products); sums are FP32.
    Singular values must stay below 15 through the steps (the default coefficients keep
    them below 1.3).  ``x``: FP32, BF16 or FP16, any strides; leading dimensions are a
    batch (at most 65535 matrices, of 2^32 elements and 2^24 rows or columns).
    A matrix with a NaN or infinity gives NaN.  Returns a new contiguous tensor without a
    gradient.
    """
    newton = newton_settings(steps, coefficients, eps)
    _native.launcher().check_device(x.device, "orthogonalize")
    out_dtype = x.dtype if dtype is None else dtype
    for t in (x.dtype, out_dtype):
        if t not in _FORMATS:
            raise TypeError(f"orthogonalize takes FP32, BF16 or FP16 matrices, got {t}")
    if x.dim() < 2:
        raise ValueError(f"orthogonalize needs matrices, got shape {tuple(x.shape)}")
    y = torch.empty(x.shape, dtype=out_dtype, device=x.device)
    if x.numel() == 0:
        return y
    m, n = x.shape[-2:]
    src = x.detach()
    if src.dim() != 3:
        src = src.reshape(-1, m, n)
    if (src.stride(2) != 1 and n > 1) or src.stride(1) < 0 or src.stride(0) < 0:
        src = src.contiguous()
    launcher = _native.launcher()
    with device_guard(x.device):
        need = launcher.newton_workspace(src.shape[0], m, n, _FORMATS[out_dtype])
        space = torch.empty(need, dtype=torch.uint8, device=x.device)
        launcher.orthogonalize(src.data_ptr(), _FORMATS[src.dtype], src.stride(1), src.stride(0),
                               y.data_ptr(), _FORMATS[out_dtype], src.shape[0], m, n, newton,
                               space, stream_handle(x.device))
    return y


def _shape_classes(updates):
    """[(m, n, [index, ...])] of the updates, by shape, those with the longest sums first
    (they set the length of a phase, so the others fill in behind them)."""
    classes = {}
    for i, u in enumerate(updates):
        m = u.tensors[0].shape[0]
        classes.setdefault((m, u.numel // m), []).append(i)
    return sorted(((m, n, members) for (m, n), members in classes.items()),
                  key=lambda c: -max(c[0], c[1]))


def _calls(classes, launcher):
    """The classes as calls of at most MUON_MAX_CLASSES shapes and MUON_MAX_MATRICES matrices
    whose workspace stays within _WORKSPACE_BYTES (one matrix is always taken):
    [[(m, n, members), ...], ...]."""
    calls, current, room, places = [], [], _WORKSPACE_BYTES, _native.MUON_MAX_MATRICES
    for m, n, members in classes:
        size, done = launcher.newton_workspace(1, m, n, _FORMATS[torch.bfloat16]), 0
        while done < len(members):
            fits = min(len(members) - done, room // size, places)
            if (fits < 1 and current) or len(current) == _native.MUON_MAX_CLASSES:
                calls.append(current)
                current, room, places = [], _WORKSPACE_BYTES, _native.MUON_MAX_MATRICES
                continue
            fits = max(1, fits)
            current.append((m, n, members[done:done + fits]))
            room, places, done = room - fits * size, places - fits, done + fits
    return calls + [current] if current else calls


_ROW = struct.Struct("<QQQQqqIIII")  # srs_row


def _plan(updates, *, lr, scale):
    """The calls of a step of ``updates`` (matrices of one device): [(rows, classes, workspace
    bytes), ...].  Sizes that the kernels do not take are refused here, before any launch."""
    launcher = _native.launcher()
    calls = []
    for call in _calls(_shape_classes(updates), launcher):
        table = (_native.SrsMuonClass * len(call))()
        members = [updates[i] for _, _, chosen in call for i in chosen]
        rows = ctypes.create_string_buffer(_ROW.size * len(members))
        for i, u in enumerate(members):
            p, g, state = u.tensors
            _ROW.pack_into(rows, _ROW.size * i, p.data_ptr(), g.data_ptr(), state.data_ptr(), 0,
                           u.numel, 0, u.param_index & 0xFFFFFFFF, u.offset, _row_flags(u, 0), 0)
        for entry, (m, n, chosen) in zip(table, call):
            entry.count, entry.m, entry.n = len(chosen), m, n
            entry.neg_step = -(lr * update_scale(scale, m, n))
        calls.append((rows, table, launcher.muon_workspace(table)))
    return calls


def muon_launch(updates, codes, *, lr, momentum, weight_decay, nesterov, scale, newton, rng,
                calls=None):
    """Enqueue the step of ``updates`` (matrices of one device) on its current stream;
    ``calls``: their plan, if it has been made."""
    device = updates[0].tensors[0].device
    launcher = _native.launcher()
    fmt, rule = codes
    hp = _native.SrsMuonHparams()
    hp.momentum, hp.decay = momentum, 1.0 - lr * weight_decay
    hp.nesterov = int(nesterov)
    if calls is None:
        calls = _plan(updates, lr=lr, scale=scale)
    with device_guard(device):
        stream = stream_handle(device)
        space = torch.empty(max(size for _, _, size in calls), dtype=torch.uint8, device=device)
        for rows, table, _ in calls:
            launcher.muon_multi(rows, table, fmt, rule, hp, newton, rng, space, stream)


def check_products(device) -> None:
    """RuntimeError when a wait inside a product kernel (Newton-Schulz, FP8 blocks) has run out
    on ``device`` since the last check: the results since then are not valid.  Waits for the
    device; the product calls themselves ask, without waiting, about the calls before."""
    with device_guard(device):
        where = _native.launcher().product_status()
    if where:
        raise RuntimeError(f"a wait inside a product kernel on {device} ran out ({where:#x}): the "
                           "results of product calls since the last check are not valid")


def check_muon(lr, momentum, weight_decay, scale) -> None:
    check_nonnegative("learning rate", lr)
    check_nonnegative("weight_decay", weight_decay)
    if not 0 <= momentum < 1:
        raise ValueError(f"invalid momentum value: {momentum}")
    if scale not in SCALE_RULES:
        raise ValueError(f"scale must be one of {SCALE_RULES}")


def check_matrix(parameter) -> None:
    if parameter.dim() < 2:
        raise ValueError("Muon updates matrices (parameters of two or more dimensions, rows "
                         f"first); got shape {tuple(parameter.shape)}")


def check_updates(updates) -> None:
    """Same device, no overlap between anything written and anything else."""
    if len({u.tensors[0].device for u in updates}) > 1:
        raise ValueError("all tensors must be on the same CUDA device")
    check_disjoint([s for u in updates for s in spans_of(u.tensors, u.numel)])


@torch.no_grad()
def cuda_muon_step_(parameters, gradients, momenta, *, lr, momentum_factor=0.95,
                    weight_decay=0.0, nesterov=True, scale="spectral", seeds, offsets=None,
                    rounding=None, formats=None, steps=5, coefficients=NEWTON_SCHULZ, eps=1e-7):
    """One Muon update of a list of matrices, in place, on the current CUDA stream.

    Per matrix, in FP32: u' = u*momentum_factor + g; v = u'*momentum_factor + g
    (``nesterov``) or u'; p' = p*(1 - lr*weight_decay) - lr*s*O, where O is the
    orthogonalised v and s the shape's factor (``update_scale``).  u' is stored
    with the momenta's format (one for all) under counter base
    state_key(seeds[i], 0).  Parameters and gradients FP32 or BF16; dimensions
    after the first are flattened.  Matrices of a shape are updated together.

    In a CUDA graph (after one such call outside it) a step replays with the learning rate
    and the seeds of its capture: the same rounding draws every time.
    """
    parameters, gradients, momenta = list(parameters), list(gradients), list(momenta)
    seeds = list(seeds)
    offsets = [0] * len(parameters) if offsets is None else list(offsets)
    if len({len(parameters), len(gradients), len(momenta), len(seeds), len(offsets)}) != 1:
        raise ValueError("parameters, gradients, momenta, seeds and offsets must have one length")
    check_muon(lr, momentum_factor, weight_decay, scale)
    newton = newton_settings(steps, coefficients, eps)
    if not parameters:
        return
    if formats is None:
        formats = (StateFormat(momenta[0].dtype, "stochastic" if rounding is None else rounding),)
        rounding = None
    (fmt,) = resolve_formats(("momentum_buffer",), formats, rounding=rounding, backend="cuda")
    updates = []
    for p, g, u, seed, offset in zip(parameters, gradients, momenta, seeds, offsets):
        if u.dtype != fmt.dtype:
            raise ValueError("state dtype does not match its state format")
        check_matrix(p)
        _native.launcher().check_device(p.device)
        check_layout((p, g, u))
        if p.numel():
            updates.append(Update((p, g, u), int(seed), p.numel(), int(offset) & 0xFFFFFFFF,
                                  None))
    if not updates:
        return
    check_updates(updates)
    muon_launch(updates, native_codes(fmt.dtype, fmt.rounding), lr=lr, momentum=momentum_factor,
                weight_decay=weight_decay, nesterov=nesterov, scale=scale, newton=newton,
                rng=rng_words(0, 0, _native.KEY_GIVEN))


def muon_group_step(optimizer, group, formats, items, rng_step) -> None:
    """The ``_step_group`` hook of the Muon optimizers: validate the whole group,
    then launch device by device."""
    optimizer._validate_group(group)
    newton = newton_settings(group["ns_steps"], group["ns_coefficients"], group["eps"])
    (fmt,) = formats
    codes = native_codes(fmt.dtype, fmt.rounding)
    by_device = {}
    for parameter, state, param_index, _, offset in items:
        check_matrix(parameter)
        tensors = (parameter, parameter.grad, state["momentum_buffer"])
        check_layout(tensors)
        _native.launcher().check_device(parameter.device)
        if parameter.numel():
            by_device.setdefault(parameter.device, []).append(
                Update(tensors, int(param_index), parameter.numel(), int(offset) & 0xFFFFFFFF,
                       None))
    plans = []
    for updates in by_device.values():
        check_updates(updates)
        plans.append((updates, _plan(updates, lr=group["lr"], scale=group["scale"])))
    rng = rng_words(group["sr_seed"], rng_step)
    for updates, calls in plans:
        muon_launch(updates, codes, lr=group["lr"], momentum=group["momentum"],
                    weight_decay=group["weight_decay"], nesterov=group["nesterov"],
                    scale=group["scale"], newton=newton, rng=rng, calls=calls)
