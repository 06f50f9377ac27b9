"""Optimizer steps over many tensors at once, as functions of the tensors and their state.

* :func:`adamw_`: one (R)Adam(-atan2)W step with both moments in 8 bits, or in fp32 with fp32
  master weights (or, without masters, in any 16- or 32-bit type: the step of ``THORN``'s
  non-orthogonalized group).
* :func:`momentum_`: the orthogonalized group's Nesterov momentum held in 8 bits, returning the
  normalised Newton-Schulz inputs.
* :func:`apply_update_`: an orthogonalized update applied to fp32 master weights.
* :func:`state8_zeros`, :func:`state8_read`, :func:`state8_write`: making, reading and converting
  8-bit state.

8-bit state is a tensor of ``torch.float8_e4m3fn`` codes of the parameter's shape and a tensor of
``torch.float8_e8m0fnu`` scales, one for each block of 128 consecutive elements; a value is its
code times its block's scale.  The blocks run over the flat tensor (scales ``[blocks]``), or, for
:func:`momentum_`, restart at each matrix of a stack (scales ``[matrices, blocks]``).  Codes are
rounded stochastically, so that changes smaller than half a step survive on average; ``seeds``
gives one integer per tensor and should be new for every step (the same seeds give the same bits).

``THORN`` makes the same calls for groups with ``state_dtype=torch.float8_e4m3fn`` or
``master_weights=True``.  All functions run on the current stream of the tensors' device and
change their tensors in place, which autograd sees as it does torch's in-place operations (not for
8-bit state, which no operation saves).  They take host scalars, which a captured CUDA graph would
repeat at every replay, so they refuse to be captured.  The reference has no counterpart: it keeps
state in the parameter's dtype (thorn.py:1591-1599) and updates 16-bit parameters in place.
"""
from __future__ import annotations

import struct
from contextlib import nullcontext
from functools import lru_cache
from math import prod
from typing import Optional, Sequence, Union

import torch

from . import _native as N

__all__ = ["adamw_", "momentum_", "apply_update_", "state8_zeros", "state8_read", "state8_write"]

CODES = torch.float8_e4m3fn
SCALES = torch.float8_e8m0fnu
BLOCK = 128
_U64 = (1 << 64) - 1
HALF = (torch.bfloat16, torch.float16)

# layouts of thorn_adamw_state_tensor, thorn_momentum8_tensor and thorn_apply_master_tensor
_ADAM = struct.Struct("<7QqQ3fi")
_MOMENTUM = struct.Struct("<4Q4qQQ")
_APPLY = struct.Struct("<5Q3qf4x")
_NO_POINTERS = (0,) * 7


def _records(struct_type, parts):
    """A C array of records: from a list of packed ones, or over a buffer that holds them."""
    if isinstance(parts, bytearray):
        return (struct_type * (len(parts) // N.ctypes.sizeof(struct_type))).from_buffer(parts)
    return (struct_type * max(1, len(parts))).from_buffer_copy(b"".join(parts) or bytes(N.ctypes.sizeof(struct_type)))


def _count(struct_, parts) -> int:
    return len(parts) // struct_.size if isinstance(parts, bytearray) else len(parts)


def _per_tensor(x, n: int, what: str) -> list:
    if isinstance(x, (int, float)):
        return [x] * n
    x = x if type(x) is list else list(x)
    if len(x) != n:
        raise ValueError(f"{what}: {len(x)} values for {n} tensors")
    return x


def _lists(**named):
    """The given tensor lists as lists of one length."""
    out = [v if v is None or type(v) is list else list(v) for v in named.values()]
    n = len(out[0])
    for k, v in zip(named, out):
        if v is not None and len(v) != n:
            raise ValueError(f"{k}: {len(v)} tensors, expected {n}")
    return out


# what a list's tensors have to be like (host_records.cpp)
_ANY, _SAME_SHAPE, _FLAT_BLOCKS, _MATRIX_BLOCKS = 0, 1, 2, 3


def _expected_shape(like, mode):
    if mode == _SAME_SHAPE:
        return tuple(like.shape)
    runs, n = _runs(like.shape, mode == _MATRIX_BLOCKS)
    return (runs, _blocks(n)) if mode == _MATRIX_BLOCKS else (_blocks(n),)


def _pointers(rec, offset, stride, ts, dtype, dev, what, like=None, mode=_ANY, distinct=True) -> None:
    """Checks the tensors and writes their pointers into the records at ``offset``."""
    index = dev.index if dev.index is not None else -1  # -1: the CPU
    if N.host().pointers(rec, offset, stride, ts, dtype, index, like, mode, distinct):
        return
    for i, t in enumerate(ts):
        if t.dtype is not dtype:
            raise TypeError(f"{what}[{i}] must be {dtype}, got {t.dtype}")
        if t.device != dev:
            raise RuntimeError(f"{what}[{i}] is on {t.device}, expected {dev}")
        if t.layout is not torch.strided or not t.is_contiguous():
            raise ValueError(f"{what}[{i}] must be contiguous")
        if mode != _ANY and tuple(t.shape) != _expected_shape(like[i], mode):
            raise ValueError(f"{what}[{i}] must have shape {_expected_shape(like[i], mode)}, got {tuple(t.shape)}")
    raise ValueError(f"{what}: the same tensor is given twice, or two share memory")


_here = nullcontext()


def _on(dev):
    """Makes ``dev`` the current device, which it mostly is already."""
    return _here if torch._C._cuda_getDevice() == dev.index else torch.cuda.device(dev)


def refuse_capture(dev) -> None:
    """Raises where the current stream of ``dev`` is being captured."""
    if dev.type != "cuda":
        return
    if torch._C._cuda_getDevice() == dev.index:  # the usual case, without a context
        capturing = torch.cuda.is_current_stream_capturing()
    else:
        with torch.cuda.device(dev):
            capturing = torch.cuda.is_current_stream_capturing()
    if capturing:
        raise RuntimeError("this call takes host scalars (step, learning rate, seeds) that a captured CUDA graph would "
                           "repeat at every replay: call it outside of graph capture")


def _stream(dev) -> int:
    """The current stream of ``dev``."""
    return torch._C._cuda_getCurrentRawStream(dev.index)


def _device(t) -> torch.device:
    dev = t.device
    if dev.type != "cuda":
        raise RuntimeError(f"thorn_b200 runs its step on CUDA devices only; got a tensor on {dev}")
    refuse_capture(dev)
    return dev


@lru_cache(maxsize=4096)
def _momentum_scratch(B: int, R: int, C: int) -> int:
    return int(N.load().thorn_momentum8_scratch_bytes(B, R, C))


@lru_cache(maxsize=None)
def _scratch_fn() -> int:
    """Address of thorn_momentum8_scratch_bytes."""
    return N.ctypes.cast(N.load().thorn_momentum8_scratch_bytes, N.ctypes.c_void_p).value


def _blocks(numel: int) -> int:
    return -(-numel // BLOCK)


def radam_rect(beta2: float, step: int, rectify: bool) -> float:
    """RAdam rectification (thorn.py:782-798)."""
    if beta2 > 0.0:
        rho_inf = 2 / (1 - beta2) - 1
        rho = rho_inf - 2 * step * (beta2 ** step) / (1 - beta2 ** step)
        r = ((rho - 4) * (rho - 2) * rho_inf / ((rho_inf - 4) * (rho_inf - 2) * rho)) ** 0.5 if rho > 4.0 else 0.0
        return r ** float(rectify)
    return 1.0


def _adam_scalars(steps, lrs, b1: float, b2: float, rectify: bool, n: int):
    """lr * rect, the bias corrections and the degenerate flag: four numbers where step and rate
    are one for all tensors, else four lists."""
    def of(t):
        rect = radam_rect(b2, t, rectify)
        return rect, 1 / (1 - b1 ** t), 1 / (1 - b2 ** t), 1 if rect == 0.0 else 0

    if isinstance(steps, int) and isinstance(lrs, (int, float)):
        rect, c1, c2, first = of(steps)
        return lrs * rect, c1, c2, first
    steps = [steps] * n if isinstance(steps, int) else steps
    lrs = [lrs] * n if isinstance(lrs, (int, float)) else lrs
    known = {t: of(t) for t in set(steps)}
    rects, c1, c2, first = zip(*[known[t] for t in steps])
    return [x * r for x, r in zip(lrs, rects)], list(c1), list(c2), list(first)


# ------------------------------------------------------------------ launches (checked arguments)
def adam_record(p, g, w, m, v, ms, vs, numel, seed, lr, bc1, bc2, degenerate) -> bytes:
    """One thorn_adamw_state_tensor; pointers as integers, 0 for NULL."""
    return _ADAM.pack(p, g, w, m, v, ms, vs, numel, seed & _U64, lr, bc1, bc2, degenerate)


def launch_adam(records, p_dtype, eight: bool, betas, weight_decay: float, eps: float, stream) -> None:
    lib = N.load()
    fn = lib.thorn_adamw8_multi if eight else lib.thorn_adamw_master_multi
    eps = max(eps, 2.0 ** -126) if eps > 0 else eps  # fp32 would round it to zero, which means the arc tangent
    N.check(fn(_records(N.AdamStateTensor, records), _count(_ADAM, records), N.dtype_code(p_dtype), float(betas[0]),
               float(betas[1]), float(weight_decay), float(eps), stream),
            "adamw8_multi" if eight else "adamw_master_multi")


def launch_momentum8(items, p_dtype, x_dtype, beta: float, dev, stream) -> None:
    """``items``: (g, m, m_scale, x pointer or 0, batch, rows, cols, ldx, seed)."""
    need = [_momentum_scratch(B, R, C) if x else 0 for _, _, _, x, B, R, C, _, _ in items]
    scratch = torch.empty(max(16, sum(need)), dtype=torch.uint8, device=dev)
    recs, at = [], scratch.data_ptr()
    for (g, m, ms, x, B, R, C, ldx, seed), nb in zip(items, need):
        recs.append(_MOMENTUM.pack(g, m, ms, x, B, R, C, ldx, seed & _U64, at if nb else 0))
        at += nb
    _momentum_call(recs, p_dtype, x_dtype, beta, stream)


def _momentum_call(recs, p_dtype, x_dtype, beta: float, stream) -> None:
    N.check(N.load().thorn_momentum8_multi(_records(N.Momentum8Tensor, recs), _count(_MOMENTUM, recs),
                                           N.dtype_code(p_dtype), N.dtype_code(x_dtype), beta, stream),
            "momentum8_multi")


def launch_apply(items, u_dtype, p_dtype, weight_decay: float, stream) -> None:
    """``items``: (U, p, w, row_scale, mat_stats pointers, batch, rows, cols, lr), or their records."""
    recs = items if isinstance(items, bytearray) else [_APPLY.pack(*it) for it in items]
    N.check(N.load().thorn_apply_master_multi(_records(N.ApplyMasterTensor, recs), _count(_APPLY, recs),
                                              N.dtype_code(u_dtype), N.dtype_code(p_dtype),
                                              float(weight_decay), stream), "apply_master_multi")


# ------------------------------------------------------------------------------------- operators
def adamw_(params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor], moments: Sequence[torch.Tensor],
           variances: Sequence[torch.Tensor], *, step: Union[int, Sequence[int]],
           lr: Union[float, Sequence[float]], betas=(0.9, 0.95), eps: float = 0.0, weight_decay: float = 0.1,
           rectify: bool = False, moment_scales: Optional[Sequence[torch.Tensor]] = None,
           variance_scales: Optional[Sequence[torch.Tensor]] = None,
           masters: Optional[Sequence[torch.Tensor]] = None, seeds: Optional[Sequence[int]] = None) -> None:
    """One (R)Adam(-atan2)W step of all ``params`` (one dtype), in place::

        m <- m + (g - m)(1 - beta1);  v <- beta2 v + (1 - beta2) g^2
        u  = atan2(m bc1, sqrt(v bc2))  (eps == 0)   or   m bc1 / (sqrt(v bc2) + eps),   bc = 1 / (1 - beta^step)
        u <- u + weight_decay p  where u p >= 0;   p <- p - lr u

    The dtype of ``moments`` chooses the state: ``torch.float8_e4m3fn`` with ``moment_scales``,
    ``variance_scales`` and ``seeds`` (8 bits; the update uses the moments before they are
    rounded); ``torch.float32`` with ``masters``; or, without masters, fp32, bf16 or fp16.
    ``masters``: fp32 copies of 16-bit ``params`` that take the update; ``params`` receive their
    rounding.  ``step`` counts from 1; it and ``lr`` may differ per tensor.  ``rectify``: RAdam.
    """
    params, grads, moments, variances, ms, vs, masters = _lists(
        params=params, grads=grads, moments=moments, variances=variances, moment_scales=moment_scales,
        variance_scales=variance_scales, masters=masters)
    n = len(params)
    if n == 0:
        return
    dev, pdt, sdt = _device(params[0]), params[0].dtype, moments[0].dtype
    N.dtype_code(pdt)
    eight = sdt is CODES
    steps = step if isinstance(step, int) else _per_tensor(step, n, "step")
    lrs = lr if isinstance(lr, (int, float)) else _per_tensor(lr, n, "lr")
    if (steps if isinstance(steps, int) else min(steps)) < 1:
        raise ValueError("step counts from 1")
    b1, b2 = betas
    if not (0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0):
        raise ValueError(f"betas must be in [0, 1), got {tuple(betas)}")
    if not eps >= 0.0:
        raise ValueError(f"eps must be >= 0, got {eps}")
    size = _ADAM.size
    scalars = _adam_scalars(steps, lrs, b1, b2, rectify, n)
    one = not isinstance(scalars[0], list)  # the same four for all tensors
    rec = bytearray(_ADAM.pack(*_NO_POINTERS, 0, 0, *scalars) * n if one else size * n)
    _pointers(rec, 0, size, params, pdt, dev, "params")
    _pointers(rec, 8, size, grads, pdt, dev, "grads", params, _SAME_SHAPE, distinct=False)
    if masters is not None:
        if pdt not in HALF:
            raise TypeError(f"masters are fp32 copies of 16-bit parameters, got {pdt} parameters")
        _pointers(rec, 16, size, masters, torch.float32, dev, "masters", params, _SAME_SHAPE)
    _pointers(rec, 24, size, moments, sdt, dev, "moments", params, _SAME_SHAPE)
    _pointers(rec, 32, size, variances, sdt, dev, "variances", params, _SAME_SHAPE)
    host = N.host()
    if eight:
        if ms is None or vs is None or seeds is None:
            raise ValueError("8-bit moments need moment_scales, variance_scales and seeds")
        _pointers(rec, 40, size, ms, SCALES, dev, "moment_scales", params, _FLAT_BLOCKS)
        _pointers(rec, 48, size, vs, SCALES, dev, "variance_scales", params, _FLAT_BLOCKS)
        host.values(rec, 64, size, n, "Q", _per_tensor(seeds, n, "seeds"))
    else:
        if ms is not None or vs is not None:
            raise ValueError(f"scales are given with {sdt} moments")
        N.dtype_code(sdt)
        if masters is not None and sdt is not torch.float32:
            raise TypeError(f"masters need fp32 or 8-bit moments, got {sdt}")
    host.numels(rec, 56, size, params)
    if not one:
        for at, kind, column in zip((72, 76, 80, 84), "fffi", scalars):
            host.values(rec, at, size, n, kind, column)
    with _on(dev):
        stream = _stream(dev)
        if eight or masters is not None:
            launch_adam(rec, pdt, eight, (b1, b2), weight_decay, eps, stream)
        else:
            recs = [N.AdamTensor(p, g, m, v, k, rate, c1, c2, deg) for p, g, _, m, v, _, _, k, _, rate, c1, c2, deg
                    in _ADAM.iter_unpack(rec)]
            N.check(N.load().thorn_adamw_multi(N.array(N.AdamTensor, recs), n, N.dtype_code(pdt), N.dtype_code(sdt),
                                               float(b1), float(b2), float(weight_decay), float(eps), stream),
                    "adamw_multi")
    if eight:  # no operation saves codes or scales for a backward pass
        host.written(params, masters)
    else:
        host.written(params, moments, variances, masters)


def momentum_(grads: Sequence[torch.Tensor], moments: Sequence[torch.Tensor], scales: Sequence[torch.Tensor], *,
              beta: float, seeds: Sequence[int], dtype: torch.dtype = torch.float16,
              out: Optional[Sequence[torch.Tensor]] = None) -> list:
    """Momentum in 8 bits of ``grads`` (matrices or stacks of them, one dtype) and the normalised
    Newton-Schulz input of every matrix, in ``dtype`` (fp16 or bf16)::

        m <- beta m + g  (rounded to 8 bits);   u = g + beta m;   x = u / (||u||_F + 1e-8)

    ``moments`` and ``scales`` as :func:`state8_zeros` with ``per_matrix=True`` makes them.
    Returns the list of x (``out`` when given, else views of one new allocation), which
    ``torch.ops.thorn_b200.polar_decomp`` takes.
    """
    grads, moments, scales, out = _lists(grads=grads, moments=moments, scales=scales, out=out)
    n = len(grads)
    if n == 0:
        return []
    dev, pdt = _device(grads[0]), grads[0].dtype
    N.dtype_code(pdt)
    if dtype not in HALF:
        raise TypeError(f"the Newton-Schulz input is float16 or bfloat16, got {dtype}")
    if not 0.0 <= beta < 1.0:
        raise ValueError(f"beta must be in [0, 1), got {beta}")
    seeds = _per_tensor(seeds, n, "seeds")
    size = _MOMENTUM.size
    rec = bytearray(size * n)
    host = N.host()
    _pointers(rec, 0, size, grads, pdt, dev, "grads", distinct=False)
    elems, need = host.matrices(rec, 32, size, grads, _scratch_fn())
    _pointers(rec, 8, size, moments, CODES, dev, "moments", grads, _SAME_SHAPE)
    _pointers(rec, 16, size, scales, SCALES, dev, "scales", grads, _MATRIX_BLOCKS)
    host.values(rec, 64, size, n, "Q", seeds)
    given = out
    if out is None:  # views of one allocation, each starting on 16 bytes
        out = host.views(torch.empty(elems, dtype=dtype, device=dev), grads, rec, 24, size)
    else:
        _pointers(rec, 24, size, out, dtype, dev, "out", grads, _SAME_SHAPE)
    scratch = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    host.scratch(rec, 32, 72, size, n, _scratch_fn(), 0 if scratch is None else scratch.data_ptr())
    with _on(dev):
        _momentum_call(rec, pdt, dtype, float(beta), _stream(dev))
    if given is not None:
        host.written(given)
    return out


def apply_update_(params: Sequence[torch.Tensor], updates: Sequence[torch.Tensor], *,
                  masters: Sequence[torch.Tensor], lr: Union[float, Sequence[float]],
                  weight_decay: float = 0.1) -> None:
    """Applies 16-bit ``updates`` (Newton-Schulz results) to fp32 ``masters`` and rounds them into
    the 16-bit ``params``::

        u <- u + weight_decay w  where u w >= 0;   w <- w - lr u;   p = round(w)
    """
    params, updates, masters = _lists(params=params, updates=updates, masters=masters)
    n = len(params)
    if n == 0:
        return
    dev, pdt, udt = _device(params[0]), params[0].dtype, updates[0].dtype
    if pdt not in HALF or udt not in HALF:
        raise TypeError(f"params and updates must be float16 or bfloat16, got {pdt} and {udt}")
    one = isinstance(lr, (int, float))
    lrs = lr if one else _per_tensor(lr, n, "lr")
    size = _APPLY.size
    rec = bytearray(_APPLY.pack(*_NO_POINTERS[:5], 1, 1, 0, lrs if one else 0.0) * n)  # one row of all elements
    host = N.host()
    _pointers(rec, 8, size, params, pdt, dev, "params")
    _pointers(rec, 0, size, updates, udt, dev, "updates", params, _SAME_SHAPE, distinct=False)
    _pointers(rec, 16, size, masters, torch.float32, dev, "masters", params, _SAME_SHAPE)
    host.numels(rec, 56, size, params)
    if not one:
        host.values(rec, 64, size, n, "f", lrs)
    with _on(dev):
        launch_apply(rec, udt, pdt, weight_decay, _stream(dev))
    host.written(params, masters)


# ------------------------------------------------------------------------------------ 8-bit state
def _runs(shape, per_matrix: bool) -> tuple:
    """(number of block runs, elements of a run)."""
    if not per_matrix:
        return 1, prod(shape)
    if len(shape) < 2:
        raise ValueError("per_matrix state needs a matrix or a stack of matrices")
    return prod(shape[:-2]), shape[-2] * shape[-1]


def state8_zeros(like: torch.Tensor, per_matrix: bool = False) -> tuple:
    """``(codes, scales)`` of an all-zero 8-bit state of ``like``'s shape, on its device."""
    runs, n = _runs(like.shape, per_matrix)
    codes = torch.zeros(like.shape, dtype=torch.uint8, device=like.device).view(CODES)
    scales = torch.zeros((runs, _blocks(n)) if per_matrix else (_blocks(n),), dtype=torch.uint8, device=like.device)
    return codes, scales.view(SCALES)


def state8_read(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """The fp32 values of an 8-bit state."""
    runs, n = _runs(codes.shape, scales.ndim == 2)
    s = scales.reshape(runs, _blocks(n)).float().repeat_interleave(BLOCK, 1)[:, :n]
    return (codes.reshape(runs, n).float() * s).reshape(codes.shape)


def state8_write(x: torch.Tensor, per_matrix: bool = False, positive: bool = False) -> tuple:
    """``(codes, scales)`` of ``x`` rounded to the nearest 8-bit values, for converting state that
    was kept in 16 or 32 bits.  ``positive`` (second moments): values of a block that is not all
    zero are held at no less than the smallest code, as :func:`adamw_` holds them."""
    runs, n = _runs(x.shape, per_matrix)
    codes, scales = state8_zeros(x, per_matrix)
    if not x.numel():
        return codes, scales
    nb = _blocks(n)
    v = torch.zeros((runs, nb * BLOCK), dtype=torch.float32, device=x.device)
    v[:, :n] = x.reshape(runs, n)
    v = v.view(runs, nb, BLOCK)
    top = v.abs().amax(-1)
    f, e = torch.frexp(top)  # top = f 2^e with f in [1/2, 1); 448 = 0.875 * 2^9
    byte = (e - 9 + (f > 0.875).int() + 127).clamp(0, 254)
    byte = torch.where(top > 0, byte, torch.zeros_like(byte))
    byte = torch.where(torch.isfinite(top), byte, torch.full_like(byte, 255))
    scales.view(torch.uint8).copy_(byte.to(torch.uint8).reshape(scales.shape))
    y = torch.ldexp(v, (127 - byte.clamp_max(254))[..., None])
    y = torch.where((byte < 255)[..., None], y, torch.full_like(y, float("nan")))
    if positive:
        y = torch.where((top > 0)[..., None], y.clamp_min(2.0 ** -9), y)
    y = y.reshape(runs, nb * BLOCK)[:, :n].clamp(-448, 448).to(CODES)
    codes.view(torch.uint8).copy_(y.view(torch.uint8).reshape(x.shape))
    return codes, scales
