"""AdamW and the gradients' norm over many tensors at once: what follows a
ReduceScatter or AllReduce of gradients.

Both are bound to their tensors once (an optimizer's parameters, gradient
buckets and states stay where they are), then run with a launch or two per
call on the current stream of their device, whichever device is current; calls
can be captured into a CUDA graph. A gradient may be given as 1 to 8 partial
ones of that device (of micro-batches, or of ranks that share it), added in order in fp32.
"""
from __future__ import annotations

import ctypes as C
import functools
import itertools
import math
import weakref
from typing import Sequence

import torch

from . import emu

# ncclDataType_t
DTYPE = {torch.float16: 6, torch.float32: 7, torch.bfloat16: 9}
E4M3 = torch.float8_e4m3fn
NCCL_E4M3 = 10
BLOCK = 256  # elements that share a scale in the 8-bit states
_ERR = emu.ERR.size
_data_ptr, _storage_ptr = torch.Tensor.data_ptr, torch.UntypedStorage.data_ptr


class _Desc(C.Structure):  # nb_adamw_t
    _fields_ = [("device", C.c_int32), ("count", C.c_int32), ("parts", C.c_int32), ("param_dtype", C.c_int32),
                ("grad_dtype", C.c_int32), ("copy_dtype", C.c_int32), ("state_dtype", C.c_int32),
                ("seed", C.c_uint32)] + [
        (n, C.c_void_p) for n in ("size", "param", "copy", "grad", "m", "v", "m_scale", "v_scale", "weight_decay")] + [
        ("beta1", C.c_double), ("beta2", C.c_double), ("eps", C.c_double)]


@functools.lru_cache(maxsize=1)
def lib() -> C.CDLL:
    L = emu.lib()
    L.nb_adamw_create.argtypes = [C.POINTER(_Desc), C.c_char_p, C.c_size_t]
    L.nb_adamw_create.restype = C.c_void_p
    L.nb_adamw_step.argtypes = [C.c_void_p, C.c_int64, C.c_void_p, C.c_double, C.c_void_p, C.c_double, C.c_void_p,
                                C.c_void_p, C.c_char_p, C.c_size_t]
    L.nb_adamw_destroy.argtypes = [C.c_void_p]
    L.nb_adamw_destroy.restype = None
    L.nb_grad_norm_create.argtypes = [C.c_int, C.c_int, C.c_int, C.c_int, C.c_void_p, C.c_void_p, C.c_char_p,
                                      C.c_size_t]
    L.nb_grad_norm_create.restype = C.c_void_p
    L.nb_grad_norm_partials.argtypes = [C.c_void_p]
    L.nb_grad_norm.argtypes = [C.c_void_p, C.c_double, C.c_double, C.c_void_p, C.c_void_p, C.c_void_p, C.c_char_p,
                               C.c_size_t]
    L.nb_grad_norm_destroy.argtypes = [C.c_void_p]
    L.nb_grad_norm_destroy.restype = None
    return L


def _addresses(ts) -> C.Array:
    return (C.c_uint64 * len(ts))(*[t.data_ptr() for t in ts])


def _partials(grads) -> list[list[torch.Tensor]]:
    out = [[g] if isinstance(g, torch.Tensor) else list(g) for g in grads]
    if not out:
        raise ValueError("no tensors")
    if not 1 <= len(out[0]) <= 8 or any(len(g) != len(out[0]) for g in out):
        raise ValueError("each gradient must have the same number of partial ones, 1 to 8")
    return out


def _check(t: torch.Tensor, name: str, numel: int, dtype: torch.dtype, device: torch.device) -> None:
    if t.dtype != dtype:
        raise TypeError(f"{name}: expected {dtype}, got {t.dtype}")
    if t.numel() != numel:
        raise ValueError(f"{name}: expected {numel} elements, got {t.numel()}")
    if not t.is_contiguous():
        raise ValueError(f"{name}: must be contiguous")
    if t.device != device:
        raise ValueError(f"{name}: on {t.device}, expected {device}")


def _check_overlap(written: Sequence[torch.Tensor], read: Sequence[torch.Tensor]) -> None:
    """No tensor that a step writes may share memory with another of its tensors."""
    spans = [(t.data_ptr(), t.data_ptr() + t.numel() * t.element_size(), w)
             for ts, w in ((written, True), (read, False)) for t in ts if t.numel()]
    end_written = end_read = 0
    for start, end, w in sorted(spans):
        if start < end_written or (w and start < end_read):
            raise ValueError("two tensors overlap, one of which is written (the same tensor twice?)")
        if w:
            end_written = max(end_written, end)
        else:
            end_read = max(end_read, end)


class _Bound:
    """The tensors that a handle points to: their memory is held alive, and
    refused if a storage was resized or moved since."""

    def __init__(self, device: torch.device, tensors: Sequence[torch.Tensor]):
        if device.type != "cuda":
            raise ValueError(f"the tensors must be on a CUDA device, got {device}")
        self.device = device
        self._index = device.index
        self._held = [t.detach() for t in tensors]
        storages = {}
        for t in self._held:
            s = t.untyped_storage()
            storages[s.data_ptr()] = s
        self._storages = list(storages.values())
        self._where = list(storages)

    def __reduce_ex__(self, protocol):  # a copy would share the handle, and its tensors would not be the handle's
        raise TypeError(f"{type(self).__name__} is bound to its tensors: make a new one instead of copying it")

    def _check_storages(self) -> None:
        if [*map(_storage_ptr, self._storages)] != self._where:
            raise RuntimeError("a tensor's storage was resized or moved since this was made")


class GradNorm(_Bound):
    """The L2 norm of many gradients, as if they were one vector.

    `grads`: tensors (fp16, bf16 or fp32, one type, contiguous, any shapes), or
    for each gradient a sequence of 1 to 8 partial ones that are added first. They are
    bound by their memory: a gradient that is replaced (by a backward pass after
    `zero_grad(set_to_none=True)`, torch's default) is not seen, the old one is read.
    """

    def __init__(self, grads):
        parts = _partials(grads)
        first = parts[0][0]
        if first.dtype not in DTYPE:
            raise TypeError(f"grads: expected fp16, bf16 or fp32, got {first.dtype}")
        for i, g in enumerate(parts):
            for k, t in enumerate(g):
                _check(t, f"grads[{i}][{k}]", g[0].numel(), first.dtype, first.device)
        flat = [t for g in parts for t in g]
        super().__init__(first.device, flat)
        sizes = (C.c_uint64 * len(parts))(*[g[0].numel() for g in parts])
        err = emu.ERR.buf
        self._handle = lib().nb_grad_norm_create(self._index, len(parts), len(parts[0]), DTYPE[first.dtype], sizes,
                                                 _addresses(flat), err, _ERR)
        if not self._handle:
            raise RuntimeError(err.value.decode())
        weakref.finalize(self, lib().nb_grad_norm_destroy, self._handle)
        self._partials = lib().nb_grad_norm_partials(self._handle)

    def __call__(self, max_norm: float = math.inf, scale: float = 1.0) -> torch.Tensor:
        """fp32 [norm, coefficient] on the device: norm = scale * the gradients'
        norm, coefficient = scale * min(1, max_norm / (norm + 1e-6)), what the
        gradients are to be multiplied with (AdamW.step takes it as its scale).
        Where the norm is not finite the coefficient is NaN; a norm above 2^126
        (before the scale) counts as infinite, since fp32 has no normal number for its
        reciprocal. The same inputs give the same bits."""
        self._check_storages()
        out = torch.empty_strided((2,), (1,), dtype=torch.float32, device=self.device)
        ws = torch.empty_strided((self._partials,), (1,), dtype=torch.float64, device=self.device)
        err = emu.ERR.buf
        rc = lib().nb_grad_norm(self._handle, max_norm, scale, out.data_ptr(), ws.data_ptr(), emu.raw_stream(self._index),
                                err, _ERR)
        if rc:
            raise (ValueError if rc == -1 else RuntimeError)(f"{err.value.decode()} ({rc})")
        return out


class AdamW(_Bound):
    """AdamW with decoupled weight decay over many tensors in one launch.

    g = scale * sum of the partial gradients; m = b1 m + (1 - b1) g;
    v = b2 v + (1 - b2) g^2; p = p (1 - lr wd) - lr mhat / (sqrt(vhat) + eps).

    `params`: fp32, bf16 or fp16 tensors (one type, contiguous), updated in
    place, in fp32, rounded once. `grads`: one per parameter, or a sequence of
    1 to 8 partial ones each; one type. `copies`: bf16 or fp16 tensors that
    receive fp32 parameters rounded. `weight_decay`: a number, or one per tensor.

    `state="float32"`: `exp_avg`, `exp_avg_sq` are fp32 tensors. `state="8bit"`:
    they are pairs (e4m3 codes, fp32 scale per block of 256 elements), of m and
    of sqrt(v), rounded at random with bits that are a hash of (`seed`, t, tensor,
    element); `moments(i)` gives their values. The mean of m and of sqrt(v) is kept; v
    itself is 5 % high on average at beta2 = 0.999, and a single one between 0.6 and
    1.7 times the exact v (5th to 95th percentile, simulated with gradients of one distribution;
    2.5 %, 0.7 and 1.5 at 0.95). `states=(exp_avg, exp_avg_sq)` takes given ones instead of
    zeros (to resume).

    A gradient (times `scale`) that is not finite, or beyond 1.8e19, whose square fp32 does not
    hold, spoils the states of its block in 8 bits, of its element in fp32: clip with
    GradNorm's coefficient, which brings large ones down and skips a step with one that is
    not finite.

    The tensors are bound by their memory: give new ones to a new AdamW. A step
    refuses a storage that was resized; and it looks at one parameter and its copy, the
    next step at the next ones, and refuses if they were given other memory (`.data =`,
    Module.to). It cannot see that a gradient was replaced: after
    `zero_grad(set_to_none=True)`, torch's default, a backward pass makes new ones and
    the step would read the old; zero the bound ones in place (set_to_none=False).
    No two tensors may overlap where one is written.
    """

    def __init__(self, params, grads, *, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay=0.01,
                 state: str = "float32", states=None, copies=None, seed: int = 0):
        params = list(params)
        if not params:
            raise ValueError("no tensors")
        first = params[0]
        device = first.device
        if first.dtype not in DTYPE:
            raise TypeError(f"params: expected fp16, bf16 or fp32, got {first.dtype}")
        sizes = [p.numel() for p in params]
        for i, p in enumerate(params):
            _check(p, f"params[{i}]", sizes[i], first.dtype, device)
        parts = _partials(grads)
        if len(parts) != len(params):
            raise ValueError(f"grads: {len(parts)} for {len(params)} parameters")
        gtype = parts[0][0].dtype
        if gtype not in DTYPE:
            raise TypeError(f"grads: expected fp16, bf16 or fp32, got {gtype}")
        for i, g in enumerate(parts):
            for k, t in enumerate(g):
                _check(t, f"grads[{i}][{k}]", sizes[i], gtype, device)
        ctype = None
        if copies is not None:
            copies = list(copies)
            if first.dtype != torch.float32 or len(copies) != len(params):
                raise ValueError("copies: one per parameter, of fp32 parameters")
            ctype = copies[0].dtype
            if ctype not in (torch.float16, torch.bfloat16):
                raise TypeError(f"copies: expected fp16 or bf16, got {ctype}")
            for i, c in enumerate(copies):
                _check(c, f"copies[{i}]", sizes[i], ctype, device)
        decay = [float(weight_decay)] * len(params) if isinstance(weight_decay, (int, float)) else \
            [float(w) for w in weight_decay]
        if len(decay) != len(params) or not all(math.isfinite(w) for w in decay):
            raise ValueError("weight_decay: a finite number, or one per parameter")
        b1, b2 = betas
        if not (0 <= b1 < 1 and 0 <= b2 < 1) or not 1.2e-38 <= eps <= 3.4e38:
            raise ValueError("betas must be in [0, 1) and eps a positive normal fp32 number")
        if state not in ("float32", "8bit"):
            raise ValueError(f'state: "float32" or "8bit", got {state!r}')
        self._eight = state == "8bit"
        if states is None:
            if device.type != "cuda":
                raise ValueError(f"the tensors must be on a CUDA device, got {device}")
            self.exp_avg, self.exp_avg_sq = [[self._zeros(n, device) for n in sizes] for _ in range(2)]
        else:
            self.exp_avg, self.exp_avg_sq = list(states[0]), list(states[1])
            for name, s in (("exp_avg", self.exp_avg), ("exp_avg_sq", self.exp_avg_sq)):
                if len(s) != len(params):
                    raise ValueError(f"states: {len(s)} of {name} for {len(params)} parameters")
                for i, x in enumerate(s):
                    if self._eight:
                        codes, scale = x
                        _check(codes, f"{name}[{i}] codes", sizes[i], E4M3, device)
                        _check(scale, f"{name}[{i}] scales", -(-sizes[i] // BLOCK), torch.float32, device)
                    else:
                        _check(x, f"{name}[{i}]", sizes[i], torch.float32, device)
        m, v = self.exp_avg, self.exp_avg_sq
        written = params + (copies or []) + ([t for pair in m + v for t in pair] if self._eight else m + v)
        flat = [t for g in parts for t in g]
        _check_overlap(written, flat)
        super().__init__(device, written + flat)
        # Whether a tensor still has its memory: a look at 64 would take 4 of a step's 13 us, so a
        # step looks at one parameter (and its copy), the next step at the next.
        owned = zip(params, copies) if copies else zip(params)
        self._looks = itertools.cycle([(ts, [t.data_ptr() for t in ts]) for ts in owned])
        # Autograd has to see that parameters were changed.
        self._versions = [t for t in params + (copies or []) if not t.is_inference()]
        tables = [(C.c_uint64 * len(params))(*sizes), _addresses(params), _addresses(copies) if copies else None,
                  _addresses(flat), *[_addresses([x[0] for x in s] if self._eight else s) for s in (m, v)],
                  *[_addresses([x[1] for x in s]) if self._eight else None for s in (m, v)],
                  (C.c_float * len(params))(*decay)]
        desc = _Desc(self._index, len(params), len(parts[0]), DTYPE[first.dtype], DTYPE[gtype],
                     DTYPE[ctype] if ctype else 0, NCCL_E4M3 if self._eight else DTYPE[torch.float32],
                     seed & 0xFFFFFFFF, *[C.cast(t, C.c_void_p) if t is not None else None for t in tables], b1, b2, eps)
        err = emu.ERR.buf
        self._step = lib().nb_adamw_step
        self._handle = lib().nb_adamw_create(C.byref(desc), err, _ERR)
        if not self._handle:
            raise RuntimeError(err.value.decode())
        weakref.finalize(self, lib().nb_adamw_destroy, self._handle)

    def _zeros(self, n: int, device: torch.device):
        if not self._eight:
            return torch.zeros(n, dtype=torch.float32, device=device)
        return (torch.zeros(n, dtype=torch.uint8, device=device).view(E4M3),
                torch.zeros(-(-n // BLOCK), dtype=torch.float32, device=device))

    def _scalar(self, x, name: str, dtype: torch.dtype):
        """(host value, device address) of a number or a one-element tensor."""
        if not isinstance(x, torch.Tensor):
            return x, None
        if x.dtype != dtype or x.numel() != 1 or x.device != self.device:
            raise ValueError(f"{name}: a number, or one element of {dtype} on {self.device}")
        return 1, x.data_ptr()

    def step(self, t, lr, scale=1.0) -> None:
        """Step number `t` (from 1) at learning rate `lr`, the gradients multiplied
        with `scale`. Each may be a one-element tensor on the device (t int64, the
        others fp32), read when the kernel runs, so that a captured step can be
        replayed with new ones. A device scale that is not finite (GradNorm's
        coefficient after an overflow), or a device lr that is not, leaves parameters and
        states as they were; a device t below 1 counts as 1."""
        self._check_storages()
        tensors, addresses = next(self._looks)
        if [*map(_data_ptr, tensors)] != addresses:
            raise RuntimeError("a parameter or its copy was moved to other memory since this was made")
        t, t_dev = self._scalar(t, "t", torch.int64)
        lr, lr_dev = self._scalar(lr, "lr", torch.float32)
        scale, scale_dev = self._scalar(scale, "scale", torch.float32)
        err = emu.ERR.buf
        rc = self._step(self._handle, t, t_dev, lr, lr_dev, scale, scale_dev, emu.raw_stream(self._index), err, _ERR)
        if rc:
            raise (ValueError if rc == -1 else RuntimeError)(f"{err.value.decode()} ({rc})")
        if self._versions:
            torch.autograd.graph.increment_version(self._versions)

    def moments(self, i: int) -> tuple[torch.Tensor, torch.Tensor]:
        """m and v of tensor `i` as fp32 values (copies for 8-bit states)."""
        if not self._eight:
            return self.exp_avg[i], self.exp_avg_sq[i]
        m, r = [codes.float().view(-1) * scale.repeat_interleave(BLOCK)[:codes.numel()]
                for codes, scale in (self.exp_avg[i], self.exp_avg_sq[i])]
        return m, r * r
