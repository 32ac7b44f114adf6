"""What the norm and optimizer operators refuse (CPU): every check of types,
shapes, strides and overlaps is made before the device is looked at."""
import copy
import ctypes as C
import pickle

import pytest
import torch

from scc26_nccl_shim_b200.ops import norm, optim

E4M3 = torch.float8_e4m3fn


def x(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype)


W = x(64)


@pytest.mark.parametrize("kind, call", [
    (TypeError, lambda: norm.add_rms_norm(x(4, 64, dtype=torch.float64), W)),
    (TypeError, lambda: norm.add_rms_norm(x(4, 64), x(64, dtype=torch.float16))),
    (TypeError, lambda: norm.add_rms_norm([x(4, 64), x(4, 64, dtype=torch.float16)], W)),
    (TypeError, lambda: norm.add_rms_norm(x(4, 64), W, x(4, 64, dtype=torch.float32))),
    (TypeError, lambda: norm.add_rms_norm(x(4, 64), W, out_dtype=torch.float16)),
    (ValueError, lambda: norm.add_rms_norm([], W)),
    (ValueError, lambda: norm.add_rms_norm([x(4, 64)] * 9, W)),
    (ValueError, lambda: norm.add_rms_norm([x(4, 64), x(5, 64)], W)),
    (ValueError, lambda: norm.add_rms_norm(x(4, 64), W, x(1, 64))),
    (ValueError, lambda: norm.add_rms_norm(x(4, 64), x(63))),
    (ValueError, lambda: norm.add_rms_norm(x(4, 64), x(128)[::2])),
    (ValueError, lambda: norm.add_rms_norm(x(4, 0), x(0))),
    (ValueError, lambda: norm.add_rms_norm(x(4, 64), W, group=64)),
    (ValueError, lambda: norm.add_rms_norm(x(4, 64), W, out_dtype=E4M3, group=48)),
    (ValueError, lambda: norm.add_rms_norm(x(4, 64), W, eps=0.0)),
    (ValueError, lambda: norm.add_rms_norm(x(4, 64), W, eps=float("nan"))),
    (ValueError, lambda: norm.add_rms_norm(x(4, 128)[:, ::2], W)),
    (ValueError, lambda: norm.add_rms_norm(x(2, 8, 8, 8, 64)[:, :3, :3, :3], W)),
    (ValueError, lambda: norm.add_rms_norm(x(4, 3, 4, 64)[:, :, :2], W, x(4, 4, 2, 64)[:, :3])),
    (TypeError, lambda: norm.add_rms_norm_backward(x(4, 64, dtype=torch.float32), x(4, 64), W, torch.zeros(4))),
    (ValueError, lambda: norm.add_rms_norm_backward(x(5, 64), x(4, 64), W, torch.zeros(4))),
    (ValueError, lambda: norm.add_rms_norm_backward(x(4, 64), x(4, 64), W, torch.zeros(5))),
    (ValueError, lambda: norm.add_rms_norm_backward(x(4, 64), x(4, 64), W, torch.zeros(8)[::2])),
    (ValueError, lambda: norm.add_rms_norm_backward(x(4, 64), x(4, 64), W, torch.zeros(4), dh=x(4, 32))),
])
def test_norm_refuses(kind, call):
    with pytest.raises(kind) as e:
        call()
    assert "CUDA" not in str(e.value)  # not merely the CPU tensors


def test_norm_refuses_overlapping_outputs():
    h = x(4, 64)
    buf = x(8, 64)
    rstd = torch.zeros(4)
    for out in (norm.NormOut(h, None, x(4, 64), rstd),             # y is the input
                norm.NormOut(buf[:4], None, buf[2:6], rstd),       # y and h overlap
                norm.NormOut(x(4, 64), None, buf[1:5], rstd),      # h overlaps the residual, shifted
                norm.NormOut(x(4, 64), rstd, x(4, 64), rstd),      # scales without e4m3
                norm.NormOut(x(4, 128)[:, ::2], None, x(4, 64), rstd),
                norm.NormOut(x(4, 64), None, x(5, 64), rstd)):
        with pytest.raises(ValueError, match="out"):
            norm.add_rms_norm(h, W, buf[:4], out=out)


def test_row_strides():
    a = torch.empty(6, 5, 64)
    assert norm._rows([a]) == (1, [64], [0])
    assert norm._rows([a[:, :3]]) == (3, [320], [64])
    assert norm._rows([a[:, 1]]) == (1, [320], [0])
    assert norm._rows([a[:, :3], torch.empty(6, 3, 64)]) == (3, [320, 192], [64, 64])
    assert norm._rows([torch.empty(6, 3, 64), a[:, :3]]) == (3, [192, 320], [64, 64])
    assert norm._rows([a[:, :, :32]]) == (1, [64], [0])
    assert norm._rows([a[:1, :1]]) == (1, [64], [0])
    assert norm._rows([torch.empty(64).expand(6, 5, 64)]) == (1, [0], [0])


f = torch.zeros


@pytest.mark.parametrize("kind, call", [
    (ValueError, lambda: optim.AdamW([], [])),
    (TypeError, lambda: optim.AdamW([f(4, dtype=torch.float64)], [f(4)])),
    (TypeError, lambda: optim.AdamW([f(4)], [f(4, dtype=torch.float64)])),
    (TypeError, lambda: optim.AdamW([f(4), f(4).half()], [f(4), f(4)])),
    (ValueError, lambda: optim.AdamW([f(4)], [f(4), f(4)])),
    (ValueError, lambda: optim.AdamW([f(4)], [f(5)])),
    (ValueError, lambda: optim.AdamW([f(4)], [[]])),
    (ValueError, lambda: optim.AdamW([f(4)], [[f(4)] * 9])),
    (ValueError, lambda: optim.AdamW([f(4), f(4)], [[f(4)], [f(4), f(4)]])),
    (ValueError, lambda: optim.AdamW([f(8)[::2]], [f(4)])),
    (ValueError, lambda: optim.AdamW([f(4).half()], [f(4)], copies=[f(4).half()])),
    (TypeError, lambda: optim.AdamW([f(4)], [f(4)], copies=[f(4)])),
    (ValueError, lambda: optim.AdamW([f(4)], [f(4)], weight_decay=[0.1, 0.1])),
    (ValueError, lambda: optim.AdamW([f(4)], [f(4)], weight_decay=float("inf"))),
    (ValueError, lambda: optim.AdamW([f(4)], [f(4)], betas=(1.0, 0.9))),
    (ValueError, lambda: optim.AdamW([f(4)], [f(4)], eps=0.0)),
    (ValueError, lambda: optim.AdamW([f(4)], [f(4)], state="4bit")),
    (ValueError, lambda: optim.AdamW([f(4)], [f(4)], states=([f(4)], []))),
    (TypeError, lambda: optim.AdamW([f(4)], [f(4)], states=([f(4).half()], [f(4)]))),
    (ValueError, lambda: optim.AdamW([f(300)], [f(300)], state="8bit",
                                     states=tuple([(f(300).to(E4M3), f(1))] for _ in "mv"))),
    (ValueError, lambda: optim.GradNorm([])),
    (TypeError, lambda: optim.GradNorm([f(4, dtype=torch.int32)])),
    (TypeError, lambda: optim.GradNorm([f(4), f(4).half()])),
    (ValueError, lambda: optim.GradNorm([f(8)[::2]])),
])
def test_optim_refuses(kind, call):
    with pytest.raises(kind) as e:
        call()
    assert "CUDA" not in str(e.value)


def test_adamw_refuses_overlaps():
    buf, m, v = f(100), f(40), f(40)
    for params, grads in (([buf[:40], buf[39:79]], [f(40), f(40)]),  # two parameters
                          ([buf[:40], buf[:40]], [f(40), f(40)]),    # the same twice
                          ([buf[:40]], [buf[20:60]])):               # a parameter and a gradient
        n = len(params)
        with pytest.raises(ValueError, match="overlap"):
            optim.AdamW(params, grads, states=([f(40) for _ in range(n)], [f(40) for _ in range(n)]))
    with pytest.raises(ValueError, match="overlap"):
        optim.AdamW([f(40)], [f(40)], states=([m], [m]))
    g = f(40)  # the same gradient twice is only read
    with pytest.raises(ValueError, match="CUDA"):
        optim.AdamW([f(40), f(40)], [g, g], states=([m, f(40)], [v, f(40)]))


def test_cpu_tensors_are_refused():
    for call in (lambda: norm.add_rms_norm(x(4, 64), W), lambda: optim.GradNorm([f(4)]),
                 lambda: optim.AdamW([f(4)], [f(4)]),
                 lambda: norm.add_rms_norm_backward(x(4, 64), x(4, 64), W, torch.zeros(4))):
        with pytest.raises(ValueError, match="CUDA"):
            call()


@pytest.mark.parametrize("group", [32.0, 64.0, "32"])
def test_norm_refuses_a_group_that_is_not_an_integer(group):
    """And what it refuses is not kept: 32 == 32.0, so that both would be one combination of types and shapes."""
    for g in (group, group):
        with pytest.raises((TypeError, ValueError), match="group"):
            norm.add_rms_norm(x(4, 64), W, out_dtype=E4M3, group=g)
    with pytest.raises(ValueError, match="CUDA"):
        norm.add_rms_norm(x(4, 64), W, out_dtype=E4M3, group=int(float(group)))


@pytest.mark.parametrize("eps", [1e-50, 1e-42, 1e39, -1e-6, float("inf")])
def test_norm_refuses_an_eps_beyond_fp32(eps):
    with pytest.raises(ValueError, match="eps"):
        norm.add_rms_norm(x(4, 64), W, eps=eps)


@pytest.mark.parametrize("cls", [optim.AdamW, optim.GradNorm])
@pytest.mark.parametrize("how", [copy.copy, copy.deepcopy, pickle.dumps])
def test_bound_tensors_are_not_copied(cls, how):
    bound = cls.__new__(cls)  # what is refused does not depend on the tensors
    bound._handle = 1
    with pytest.raises(TypeError, match="make a new one"):
        how(bound)


def test_c_entry_points_refuse_with_a_message():
    """The C ABI's own checks, without a device."""
    L, err = norm.lib(), C.create_string_buffer(256)
    a = 1 << 20  # an aligned address that no refused call touches

    def fwd(x0=a, parts=1, y=a, rows=4, inner=1, hidden=64, dtype=9, wdtype=9, odtype=9, group=0, eps=1e-6, w=a):
        p = norm._FWD[8].pack(x0, *[a] * 7, *[hidden] * 8, *[0] * 8, 0, 0, 0, w, y, a, a, a, rows, inner, 0, hidden,
                           parts, dtype, wdtype, odtype, group, eps)
        return L.nb_add_rms_norm(p, None, err, 256), err.value

    assert fwd(rows=0) == (0, b"")
    for kw in (dict(x0=0), dict(x0=a + 1), dict(y=0), dict(y=a + 1), dict(parts=0), dict(parts=9), dict(rows=-1),
               dict(inner=0), dict(rows=5, inner=2), dict(hidden=0), dict(hidden=(1 << 24) + 1), dict(rows=1 << 31),
               dict(dtype=8), dict(wdtype=6), dict(odtype=7), dict(group=32), dict(odtype=10, group=16),
               dict(eps=0.0), dict(eps=float("inf")), dict(eps=float("nan")), dict(w=0), dict(w=a + 1)):
        rc, msg = fwd(**kw)
        assert rc == -1 and msg.startswith(b"bad arguments"), (kw, rc, msg)
    assert L.nb_add_rms_norm(None, None, err, 256) == -1

    def bwd(dy=a, ws=a, nbytes=1 << 40, dw=a, rows=4, dtype=9):
        p = norm._BWD.pack(dy, 64, 0, a, 64, 0, 0, 0, 0, a, a, a, dw, ws, nbytes, rows, 1, 0, 64, dtype, 9)
        return L.nb_add_rms_norm_backward(p, None, err, 256), err.value

    for kw in (dict(dy=0), dict(dy=a + 1), dict(dw=0), dict(rows=-1), dict(dtype=0)):
        rc, msg = bwd(**kw)
        assert rc == -1 and msg.startswith(b"bad arguments"), (kw, rc, msg)

    O = optim.lib()
    assert O.nb_adamw_create(None, err, 256) is None and err.value
    one = (C.c_uint64 * 1)(4)
    bad = (C.c_uint64 * 1)(a + 1)
    good = (C.c_uint64 * 1)(a)
    for args in ((0, 1, 7, one, good), (1, 0, 7, one, good), (1, 9, 7, one, good), (1, 1, 8, one, good),
                 (1, 1, 7, one, bad), (1, 1, 7, None, good), (1, 1, 7, one, None)):
        assert O.nb_grad_norm_create(0, *args, err, 256) is None
        assert err.value.startswith(b"bad arguments")
    assert O.nb_adamw_step(None, 1, None, 0.1, None, 1.0, None, None, err, 256) == -1
    assert O.nb_grad_norm(None, 1.0, 1.0, None, None, None, err, 256) == -1
    assert O.nb_grad_norm_partials(None) == -1
    O.nb_adamw_destroy(None)
    O.nb_grad_norm_destroy(None)
