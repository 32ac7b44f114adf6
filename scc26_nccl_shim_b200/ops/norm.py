"""Root-mean-square norm of a sum: what follows an AllReduce of activations.

The partial sums of a row-parallel product (1 to 8 tensors of one GPU; after a
collective its one sum) and the residual are added and normalised in one pass, with
the result in the input's type or in e4m3 with scales; and the gradient of that.

The kernels run on the current stream of the tensors' device, whichever device
is current, and can be captured into a CUDA graph. Gradients are computed by
an explicit call; nothing here is recorded by autograd.
"""
from __future__ import annotations

import ctypes as C
import functools
import math
import operator
import struct
from typing import NamedTuple, Sequence

import torch

from . import emu

# ncclDataType_t
DTYPE = {torch.float16: 6, torch.float32: 7, torch.bfloat16: 9}
E4M3 = torch.float8_e4m3fn
NCCL_E4M3 = 10
GROUPS = (0, 32, 64, 128)

# nb_norm_t, by the number of partial sums (the arrays' other places are zero)
_FWD = [struct.Struct(f"{n}Q{8 * (8 - n)}x{n}q{8 * (8 - n)}x{n}q{8 * (8 - n)}xQ2q5Q2q7if") for n in range(9)]
_BWD = struct.Struct("Q2qQ2qQ2qQQQQQQ2q4i")    # nb_norm_grad_t
_CONTIGUOUS = torch.contiguous_format
_ERR = emu.ERR.size


class NormOut(NamedTuple):
    """What add_rms_norm returns. `y` is the normalised sum; `scale` holds the
    scales of an e4m3 `y` (else None): y's value is y * scale of its group;
    `h` is the sum (the next residual); `rstd` is 1 / rms of each row, which the
    gradient needs."""
    y: torch.Tensor
    scale: torch.Tensor | None
    h: torch.Tensor
    rstd: torch.Tensor


@functools.lru_cache(maxsize=1)
def lib() -> C.CDLL:
    L = emu.lib()
    for f in (L.nb_add_rms_norm, L.nb_add_rms_norm_backward):
        f.argtypes = [C.c_char_p, C.c_void_p, C.c_char_p, C.c_size_t]
    L.nb_add_rms_norm_backward_workspace.argtypes = [C.c_int, C.c_int64, C.c_int, C.c_int]
    L.nb_add_rms_norm_backward_workspace.restype = C.c_uint64
    return L


def _strides(t: torch.Tensor) -> tuple[int, int, int]:
    """(inner, outer stride, inner stride): row r of `t` starts at
    (r // inner) * outer stride + (r % inner) * inner stride elements."""
    hidden = t.shape[-1]
    if t.is_contiguous():
        return 1, hidden, 0
    if t.stride(-1) != 1 and hidden > 1:
        raise ValueError("the last dimension must be contiguous")
    dims: list[list[int]] = []  # [size, stride], neighbours merged
    for n, s in zip(t.shape[:-1], t.stride()[:-1]):
        if n == 1:
            continue
        if dims and dims[-1][1] == n * s:
            dims[-1] = [dims[-1][0] * n, s]
        else:
            dims.append([n, s])
    if not dims:
        return 1, hidden, 0
    if len(dims) == 1:
        return 1, dims[0][1], 0
    if len(dims) == 2:
        return dims[1][0], dims[0][1], dims[1][1]
    raise ValueError("rows at more than two different strides (call .contiguous())")


def _rows(ts: Sequence[torch.Tensor]) -> tuple[int, list[int], list[int]]:
    """The split of the row number that all of these share (its inner size),
    and each one's outer and inner strides."""
    for t in ts:
        if not t.is_contiguous():
            break
    else:
        return 1, [ts[0].shape[-1]] * len(ts), [0] * len(ts)
    got = [_strides(t) for t in ts]
    inner = 1
    for n, _, _ in got:
        if n != 1:
            if inner != 1 and inner != n:
                raise ValueError("the tensors' rows are split at different places (call .contiguous())")
            inner = n
    if inner == 1:
        return 1, [o for _, o, _ in got], [i for _, _, i in got]
    return inner, [o if n != 1 else inner * o for n, o, _ in got], [i if n != 1 else o for n, o, i in got]


def _span(t: torch.Tensor) -> tuple[int, int]:
    last = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
    return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()


def _disjoint(a: torch.Tensor, b: torch.Tensor) -> bool:
    if not a.numel() or not b.numel():
        return True
    (s, e), (p, q) = _span(a), _span(b)
    return e <= p or q <= s


def _check_weight(weight: torch.Tensor, hidden: int, dtype: torch.dtype, device: torch.device) -> int:
    if weight.dim() != 1 or weight.shape[0] != hidden:
        raise ValueError(f"weight: expected shape ({hidden},), got {tuple(weight.shape)}")
    if weight.dtype != dtype and weight.dtype != torch.float32:
        raise TypeError(f"weight: expected {dtype} or torch.float32, got {weight.dtype}")
    if not weight.is_contiguous():
        raise ValueError("weight: must be contiguous")
    if weight.device != device:
        raise ValueError(f"weight: on {weight.device}, the input on {device}")
    return DTYPE[weight.dtype]


def _integer(n, name: str) -> int:
    try:
        return operator.index(n)
    except TypeError:
        raise TypeError(f"{name}: expected an integer, got {n!r}") from None


def _like(t: torch.Tensor, ref: torch.Tensor, name: str) -> None:
    if t.dtype != ref.dtype:
        raise TypeError(f"{name}: expected {ref.dtype}, got {t.dtype}")
    if t.shape != ref.shape:
        raise ValueError(f"{name}: expected shape {tuple(ref.shape)}, got {tuple(t.shape)}")
    if t.device != ref.device:
        raise ValueError(f"{name}: on {t.device}, expected {ref.device}")


def _raise(err, rc: int) -> None:
    raise (ValueError if rc == -1 else RuntimeError)(f"{err.value.decode()} ({rc})")


def _empty(shape: tuple, dtype: torch.dtype, device: torch.device) -> torch.Tensor:
    # torch.empty takes more than twice as long to read its arguments.
    if len(shape) == 1:
        return torch.empty_strided(shape, (1,), dtype=dtype, device=device)
    if len(shape) == 2:
        return torch.empty_strided(shape, (shape[1] or 1, 1), dtype=dtype, device=device)
    return torch.empty(shape, dtype=dtype, device=device)


class _Plan(NamedTuple):
    """What a call needs to know of its tensors' types, shapes, strides and
    devices: made, with all checks of them, once for each combination."""
    pack: object
    strides: tuple  # of the inputs, as the struct has them
    extra: tuple    # of the residual (or dh)
    tail: tuple     # the struct's numbers
    device: int
    ydtype: torch.dtype | None = None
    scale_shape: tuple | None = None
    lead: tuple = ()
    nbytes: int = 0


def _describe(t: torch.Tensor) -> tuple:
    return t.dtype, t.shape, t.stride(), t.device


_plans: dict[tuple, _Plan] = {}


def _keep(key: tuple, plan: _Plan) -> _Plan:
    if len(_plans) >= 1024:
        _plans.clear()
    _plans[key] = plan
    return plan


def _plan_forward(xs: list, weight: torch.Tensor, residual: torch.Tensor | None, eps: float,
                  out_dtype: torch.dtype | None, group: int) -> _Plan:
    n = len(xs)
    if not 1 <= n <= 8:
        raise ValueError(f"1 to 8 partial sums, got {n}")
    x0 = xs[0]
    dtype, shape, dev = x0.dtype, x0.shape, x0.device
    if dtype not in DTYPE:
        raise TypeError(f"x: expected fp16, bf16 or fp32, got {dtype}")
    if not shape or shape[-1] < 1:
        raise ValueError(f"x: expected shape [..., hidden] with hidden >= 1, got {tuple(shape)}")
    hidden, lead = shape[-1], tuple(shape[:-1])
    for i in range(1, n):
        _like(xs[i], x0, f"x[{i}]")
    if residual is not None:
        _like(residual, x0, "residual")
    wcode = _check_weight(weight, hidden, dtype, dev)
    f8 = out_dtype == E4M3
    if not f8 and out_dtype is not None and out_dtype != dtype:
        raise TypeError(f"out_dtype: expected {dtype} or {E4M3}, got {out_dtype}")
    if group not in GROUPS or (group and not f8):
        raise ValueError(f"group: one of {GROUPS} with e4m3 output, else 0, got {group}")
    if not 1.2e-38 <= eps <= 3.4e38:
        raise ValueError(f"eps: must be a positive normal fp32 number, got {eps}")
    inner, outers, inners = _rows(xs if residual is None else xs + [residual])
    device = dev.index if dev.type == "cuda" else -1
    return _Plan(_FWD[n].pack, (*outers[:n], *inners[:n]), (outers[n], inners[n]) if residual is not None else (0, 0),
                 (math.prod(lead), inner, device, hidden, n, DTYPE[dtype], wcode, NCCL_E4M3 if f8 else DTYPE[dtype],
                  group, eps), device, E4M3 if f8 else dtype,
                 lead + (-(-hidden // group) if group else 1,) if f8 else None, lead)


def add_rms_norm(x, weight: torch.Tensor, residual: torch.Tensor | None = None, *, eps: float = 1e-6,
                 out_dtype: torch.dtype | None = None, group: int = 0, out: NormOut | None = None) -> NormOut:
    """h = x_0 + ... + x_{n-1} + residual; y = h / sqrt(mean(h^2) + eps) * weight.

    `x` is a tensor [..., hidden] or a sequence of 1 to 8 of them (the partial
    sums, added in order in fp32); fp16, bf16 or fp32, rows at up to two
    strides. `weight` [hidden] has x's type or fp32. y is computed from the fp32
    sum and rounded once; `h` is the sum rounded to x's type. A single x without
    a residual comes back as `h` itself. Nothing is recorded by autograd, whether inputs
    require gradients or not: call add_rms_norm_backward.

    `out_dtype=torch.float8_e4m3fn`: y in e4m3, round to nearest even, with fp32
    scales [..., ceil(hidden / group)] (`group` 32, 64 or 128 columns) or
    [..., 1] (`group` 0: one per row); scale = max(largest magnitude / 448,
    2^-126). A NaN makes its group's scale NaN.

    Squares are summed in fp32: rows beyond about 1e19 overflow to y = 0.

    `out` gives the outputs' memory (contiguous; `out.h` may be the residual or
    x_0 itself, nothing else may overlap). Autograd sees that they were changed: a
    graph that holds the residual for its backward pass then raises there.
    """
    xs = [x] if isinstance(x, torch.Tensor) else list(x)
    if type(group) is not int:  # 32.0 would be the same key as 32
        group = _integer(group, "group")
    key = (eps, out_dtype, group, _describe(weight), None if residual is None else _describe(residual),
           *[_describe(t) for t in xs])
    plan = _plans.get(key) or _keep(key, _plan_forward(xs, weight, residual, eps, out_dtype, group))
    x0 = xs[0]
    alone = residual is None and len(xs) == 1
    if out is not None:
        _check_out(out, xs, weight, residual, plan)
    if plan.device < 0:
        raise ValueError(f"the tensors must be on a CUDA device, got {x0.device}")
    if out is None:
        y = torch.empty_like(x0, dtype=plan.ydtype, memory_format=_CONTIGUOUS)
        scale = _empty(plan.scale_shape, torch.float32, x0.device) if plan.scale_shape else None
        h = x0 if alone else torch.empty_like(x0, memory_format=_CONTIGUOUS)
        rstd = _empty(plan.lead, torch.float32, x0.device)
    else:
        y, scale, h, rstd = out
        if alone and h.data_ptr() == x0.data_ptr():
            h = x0
    err = emu.ERR.buf
    rc = lib().nb_add_rms_norm(
        plan.pack(*[t.data_ptr() for t in xs], *plan.strides, 0 if residual is None else residual.data_ptr(),
                  *plan.extra, weight.data_ptr(), y.data_ptr(), 0 if scale is None else scale.data_ptr(),
                  0 if alone and h is x0 else h.data_ptr(), rstd.data_ptr(), *plan.tail),
        emu.raw_stream(plan.device), err, _ERR)
    if rc:
        _raise(err, rc)
    if out is not None:  # autograd has to see that the caller's tensors were changed
        written = [t for t in (y, scale, None if alone and h is x0 else h, rstd) if t is not None and not t.is_inference()]
        if written:
            torch.autograd.graph.increment_version(written)
    return NormOut(y, scale, h, rstd)


def _check_out(out: NormOut, xs: list, weight: torch.Tensor, residual: torch.Tensor | None, plan: _Plan) -> None:
    x0 = xs[0]
    inputs = xs + [weight] + ([residual] if residual is not None else [])
    want = [("y", out.y, x0.shape, plan.ydtype), ("h", out.h, x0.shape, x0.dtype),
            ("rstd", out.rstd, x0.shape[:-1], torch.float32)]
    if plan.scale_shape is not None:
        want.append(("scale", out.scale, plan.scale_shape, torch.float32))
    elif out.scale is not None:
        raise ValueError("out.scale: only an e4m3 output has scales")
    for name, t, shape, dtype in want:
        if t is None or t.shape != shape or t.dtype != dtype or t.device != x0.device:
            raise ValueError(f"out.{name}: expected {tuple(shape)} of {dtype} on {x0.device}")
    for i, (name, t, _, _) in enumerate(want):
        same = [s for s in (xs[0], residual) if name == "h" and s is not None and
                s.data_ptr() == t.data_ptr() and s.stride() == t.stride()]
        if not t.is_contiguous():
            raise ValueError(f"out.{name}: must be contiguous")
        for other in inputs + [w[1] for w in want[i + 1:]]:
            if not any(other is s for s in same) and not _disjoint(t, other):
                raise ValueError(f"out.{name}: overlaps another tensor of the call")


def _plan_backward(dy: torch.Tensor, h: torch.Tensor, weight: torch.Tensor, rstd: torch.Tensor,
                   dh: torch.Tensor | None) -> _Plan:
    dtype, shape, dev = h.dtype, h.shape, h.device
    if dtype not in DTYPE:
        raise TypeError(f"h: expected fp16, bf16 or fp32, got {dtype}")
    if not shape or shape[-1] < 1:
        raise ValueError(f"h: expected shape [..., hidden] with hidden >= 1, got {tuple(shape)}")
    hidden = shape[-1]
    _like(dy, h, "dy")
    if dh is not None:
        _like(dh, h, "dh")
    wcode = _check_weight(weight, hidden, dtype, dev)
    if rstd.dtype != torch.float32 or rstd.shape != shape[:-1] or not rstd.is_contiguous():
        raise ValueError(f"rstd: expected {tuple(shape[:-1])} of torch.float32, contiguous")
    if rstd.device != dev:
        raise ValueError(f"rstd: on {rstd.device}, expected {dev}")
    inner, outers, inners = _rows([dy, h] if dh is None else [dy, h, dh])
    if dev.type != "cuda":
        raise ValueError(f"the tensors must be on a CUDA device, got {dev}")
    rows, code = rstd.numel(), DTYPE[dtype]
    nbytes = int(lib().nb_add_rms_norm_backward_workspace(dev.index, rows, hidden, code))
    return _Plan(_BWD.pack, ((outers[0], inners[0]), (outers[1], inners[1])),
                 (0, 0) if dh is None else (outers[2], inners[2]), (rows, inner, dev.index, hidden, code, wcode),
                 dev.index, nbytes=nbytes)


def add_rms_norm_backward(dy: torch.Tensor, h: torch.Tensor, weight: torch.Tensor, rstd: torch.Tensor,
                          dh: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """The gradient of add_rms_norm: (dx, dweight).

    dx = rstd * (dy * w - n * mean(dy * w * n)) + dh with n = h * rstd is the
    gradient of every partial sum and of the residual; `dh` is the gradient that
    reaches the sum on its other way (the residual stream). dweight = sum over
    rows of dy * n, in the weight's type, added without atomics: the same values give the
    same bits as long as the sizes, types, strides and alignment of the tensors and the
    number of the GPU's SMs are the same (another of them may take another kernel, or other
    blocks). `h` and `rstd` are add_rms_norm's; dy, h and dh have one type.
    """
    key = (_describe(dy), _describe(h), _describe(weight), _describe(rstd), None if dh is None else _describe(dh))
    plan = _plans.get(key) or _keep(key, _plan_backward(dy, h, weight, rstd, dh))
    dx = torch.empty_like(h, memory_format=_CONTIGUOUS)
    dw = torch.empty_like(weight)
    ws = _empty((plan.nbytes // 4,), torch.float32, h.device)
    err = emu.ERR.buf
    (ydo, ydi), (ho, hi) = plan.strides
    rc = lib().nb_add_rms_norm_backward(
        plan.pack(dy.data_ptr(), ydo, ydi, h.data_ptr(), ho, hi, 0 if dh is None else dh.data_ptr(), *plan.extra,
                  weight.data_ptr(), rstd.data_ptr(), dx.data_ptr(), dw.data_ptr(), ws.data_ptr(), plan.nbytes,
                  *plan.tail),
        emu.raw_stream(plan.device), err, _ERR)
    if rc:
        _raise(err, rc)
    return dx, dw
