"""The norm of a sum and its gradient (ops/norm.py) against their formulas in
64 bits.

Tolerances, per element, with u = 2^-24 (half a step of fp32) and half a step
of each stored type:
* the sum of n terms in fp32 is off by at most n u (sum of magnitudes);
* a row's sum of squares is added over at most 64 terms in a thread and 10
  levels of a tree (rows up to 16384 here; the long rows: 128), so
  it is off by less than 2^-17 of itself; rstd by half that plus what the
  sum's own error moves it; the products after it add a few u: 2^-16 covers all.
"""
import ctypes as C

import pytest
import torch

from conftest import need_gpus

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
E4M3 = torch.float8_e4m3fn
U = 2.0 ** -24
CHAIN = 2.0 ** -16
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}


def norm():
    need_gpus(1)
    from scc26_nccl_shim_b200.ops import norm as m
    return m


def half_step(ref, dtype):
    return ref.abs() * (torch.finfo(dtype).eps / 2) + TINY[dtype] / 2


def data(shape, dtype, seed, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, device=DEV, generator=g) * scale).to(dtype)


def reference(xs, w, residual, eps):
    terms = [x.double() for x in xs] + ([residual.double()] if residual is not None else [])
    h = sum(terms)
    slack = (len(terms) - 1) * U * sum(t.abs() for t in terms) if len(terms) > 1 else torch.zeros_like(h)
    ms = h.square().mean(-1, keepdim=True) + eps
    rstd = ms.rsqrt()
    # d rstd / rstd = - mean(h dh) / ms
    rel = CHAIN + (h.abs() * slack).mean(-1, keepdim=True) / ms
    y = h * rstd * w.double()
    y_tol = y.abs() * rel + slack * rstd * w.double().abs()
    return h, slack, rstd, rel, y, y_tol


def check(out, xs, w, residual, eps, group=0):
    h, slack, rstd, rel, y, y_tol = reference(xs, w, residual, eps)
    dtype = xs[0].dtype
    assert ((out.rstd.double() - rstd[..., 0]).abs() <= rstd[..., 0] * rel[..., 0]).all()
    assert ((out.h.double() - h).abs() <= half_step(h, dtype) * 1.001 + slack).all()
    if out.y.dtype != E4M3:
        assert out.scale is None
        assert ((out.y.double() - y).abs() <= half_step(y, dtype) * 1.001 + y_tol).all()
        return
    hidden = y.shape[-1]
    wide = group or hidden
    top = torch.stack([c.abs().amax(-1) for c in y.split(wide, -1)], -1)
    top_tol = torch.stack([c.amax(-1) for c in y_tol.split(wide, -1)], -1)
    scale = (top / 448).clamp(min=2.0 ** -126)
    assert out.scale.shape == scale.shape
    assert ((out.scale.double() - scale).abs() <= scale * 4 * U + top_tol / 448).all()
    # Half a step of e4m3: 2^-4 of a normal value, 2^-10 scales of a subnormal one.
    s = out.scale.double().repeat_interleave(wide, -1)[..., :hidden]
    value = out.y.double() * s
    assert ((value - y).abs() <= y.abs() * 2.0 ** -4 * 1.001 + s * 2.0 ** -10 + y_tol * 1.1).all()


SHAPES = [(1, 1), (3, 2), (5, 7), (2, 8), (9, 31), (33, 64), (70, 100), (17, 128), (4, 200), (5, 256), (7, 257),
          (300, 264), (3, 1000), (2, 1001), (40, 2048), (5, 4096), (3, 5001), (200, 8192), (2, 8192), (2, 12345),
          (3, 16384), (2, 16392), (2, 20001), (1, 32768)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows, hidden", SHAPES)
def test_norm(rows, hidden, dtype):
    m = norm()
    x, res = data((rows, hidden), dtype, 1), data((rows, hidden), dtype, 2, 3.0)
    for w in (data((hidden,), dtype, 3), data((hidden,), torch.float32, 4)):
        check(m.add_rms_norm(x, w, res), [x], w, res, 1e-6)
        for group in (0, 32, 64, 128):
            check(m.add_rms_norm(x, w, res, out_dtype=E4M3, group=group), [x], w, res, 1e-6, group)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("parts", range(1, 9))
@pytest.mark.parametrize("residual", [False, True])
def test_partials(parts, residual, dtype):
    m = norm()
    for rows, hidden in ((5, 96), (6, 1024), (3, 1003), (2, 17000)):
        xs = [data((rows, hidden), dtype, 10 + k) for k in range(parts)]
        res = data((rows, hidden), dtype, 9, 2.0) if residual else None
        w = data((hidden,), dtype, 3)
        out = m.add_rms_norm(xs, w, res, eps=1e-5)
        check(out, xs, w, res, 1e-5)
        if parts == 1 and not residual:
            assert out.h is xs[0]
        check(m.add_rms_norm(xs, w, res, eps=1e-5, out_dtype=E4M3, group=128), xs, w, res, 1e-5, 128)


# Many rows: blocks that walk over them, at each row width's number of threads.
MANY = [(40000, 8), (30001, 24), (20001, 128), (9000, 256), (5003, 264), (3001, 1024), (2500, 2048), (1300, 4096),
        (700, 5120), (1000, 8192), (400, 8200), (333, 12288), (650, 16384), (150, 16392)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows, hidden", MANY)
def test_many_rows(rows, hidden, dtype):
    m = norm()
    xs = [data((rows, hidden), dtype, k) for k in range(2)]
    res, w = data((rows, hidden), dtype, 5, 2.0), data((hidden,), torch.float32, 3)
    check(m.add_rms_norm(xs[0], w, res), xs[:1], w, res, 1e-6)
    check(m.add_rms_norm(xs, w.to(dtype)), xs, w.to(dtype), None, 1e-6)
    for group in (0, 128):
        check(m.add_rms_norm(xs, w, res, out_dtype=E4M3, group=group), xs, w, res, 1e-6, group)
    # in place, where rows are fetched ahead of the row that is written
    want = m.add_rms_norm(xs, w, res)
    got = m.add_rms_norm(xs, w, res, out=m.NormOut(torch.empty_like(res), None, res, torch.empty_like(want.rstd)))
    assert torch.equal(got.y, want.y) and torch.equal(res, want.h)


# Rows of one block, of two that share a row, and of 1, 2 and 4 sums at a time: on
# both sides of the widths where that changes.
WIDE = [(5, 8200), (300, 4608), (300, 7168), (200, 8960), (180, 9216), (200, 9224), (160, 10240), (170, 12296),
        (150, 14336), (149, 16392), (150, 20480), (3, 24584), (149, 28672), (2, 32768), (149, 32776)]


@pytest.mark.parametrize("parts", [1, 2, 3, 5])
@pytest.mark.parametrize("rows, hidden", WIDE)
def test_wide_rows(rows, hidden, parts):
    m = norm()
    for dtype, wtype in ((torch.bfloat16,) * 2, (torch.float16, torch.float32), (torch.float32,) * 2):
        xs = [data((rows, hidden), dtype, k) for k in range(parts)]
        res, w = data((rows, hidden), dtype, 9, 2.0), data((hidden,), wtype, 3)
        want = m.add_rms_norm(xs, w, res)
        check(want, xs, w, res, 1e-6)
        for group in (0, 32, 128):
            check(m.add_rms_norm(xs, w, out_dtype=E4M3, group=group), xs, w, None, 1e-6, group)
        got = m.add_rms_norm(xs, w, res, out=m.NormOut(torch.empty_like(res), None, res, torch.empty_like(want.rstd)))
        assert torch.equal(got.y, want.y) and torch.equal(res, want.h) and torch.equal(got.rstd, want.rstd)


def test_sum_has_the_bits_of_the_collectives_fold():
    m = norm()
    from scc26_nccl_shim_b200.ops import emu
    xs = [data((37, 1024), torch.bfloat16, k) for k in range(5)]
    want = torch.empty_like(xs[0])
    emu.reduce([x.view(-1) for x in xs], [want.view(-1)])
    assert torch.equal(m.add_rms_norm(xs, data((1024,), torch.bfloat16, 9)).h, want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strides_and_alignment(dtype):
    m = norm()
    packed = data((6, 12, 128), dtype, 1)
    w = data((128,), dtype, 2)
    q = packed[:, 4:9]                                     # heads out of a packed projection
    check(m.add_rms_norm(q, w), [q], w, None, 1e-6)
    check(m.add_rms_norm(q, w, packed[:, 1:6]), [q], w, packed[:, 1:6], 1e-6)
    r = data((6, 5, 128), dtype, 3)                        # with a contiguous partner
    check(m.add_rms_norm([q, r], w, r), [q, r], w, r, 1e-6)
    cols = data((9, 300), dtype, 4)[:, 3:103]              # rows off every vector's boundary
    check(m.add_rms_norm(cols, w[:100]), [cols], w[:100], None, 1e-6)
    check(m.add_rms_norm(cols, w[1:101], cols, out_dtype=E4M3, group=64), [cols], w[1:101], cols, 1e-6, 64)
    same = data((256,), dtype, 5).expand(7, 256)           # one row for all
    w2 = data((256,), dtype, 6)
    check(m.add_rms_norm(same, w2), [same], w2, None, 1e-6)
    swapped = data((5, 4, 256), dtype, 7).transpose(0, 1)
    out = m.add_rms_norm(swapped, w2, swapped)
    assert out.y.is_contiguous() and out.rstd.shape == (4, 5)
    check(out, [swapped], w2, swapped, 1e-6)
    one = data((256,), dtype, 8)                           # a single row without a row dimension
    out = m.add_rms_norm(one, w2)
    assert out.rstd.shape == ()
    check(out, [one], w2, None, 1e-6)
    flat = data((4096 + 8,), dtype, 9)
    for off in (0, 1, 2, 4):                               # the base off the boundary
        v = flat[off:off + 4096].view(16, 256)
        check(m.add_rms_norm(v, w2), [v], w2, None, 1e-6)


def test_no_rows():
    m = norm()
    w = data((64,), torch.bfloat16, 1)
    e = torch.empty(0, 64, dtype=torch.bfloat16, device=DEV)
    out = m.add_rms_norm(e, w, e, out_dtype=E4M3, group=32)
    assert out.y.shape == (0, 64) and out.scale.shape == (0, 2) and out.rstd.shape == (0,)
    dx, dw = m.add_rms_norm_backward(e, e, w, out.rstd)
    assert dx.shape == (0, 64) and torch.equal(dw, torch.zeros_like(w))


@pytest.mark.parametrize("hidden", [64, 100, 1024, 20000])
def test_zero_nan_and_infinity_stay_in_their_rows(hidden):
    m = norm()
    x = data((6, hidden), torch.float32, 1)
    w = data((hidden,), torch.float32, 2)
    x[1] = 0
    x[2, hidden // 2] = float("nan")
    x[3, 0] = float("inf")
    x[4] = 1e-30
    good = m.add_rms_norm(data((6, hidden), torch.float32, 1), w)
    out = m.add_rms_norm(x, w)
    for r in (0, 5):
        assert torch.equal(out.y[r], good.y[r])
    assert (out.y[1] == 0).all() and out.y[2].isnan().all()
    assert out.y[3, 0].isnan() and (out.y[3, 1:] == 0).all()
    assert out.y[4].isfinite().all()
    q = m.add_rms_norm(x, w, out_dtype=E4M3, group=64)
    gq = m.add_rms_norm(data((6, hidden), torch.float32, 1), w, out_dtype=E4M3, group=64)
    for r in (0, 5):
        assert torch.equal(q.y[r].float(), gq.y[r].float()) and torch.equal(q.scale[r], gq.scale[r])
    assert (q.y[1].float() == 0).all() and (q.scale[1] == 2.0 ** -126).all()
    assert q.scale[2].isnan().all() and q.y[2].float().isnan().all()
    assert q.scale[3, 0].isnan() and (q.scale[3, 1:] == 2.0 ** -126).all()


def test_large_values_in_16_bits():
    m = norm()
    x = data((3, 512), torch.float16, 1, 1e4).clamp(-65504, 65504)
    w = torch.ones(512, device=DEV)
    out = m.add_rms_norm([x, x], w)  # the sum overflows fp16, the norm does not
    h = 2 * x.double()
    y = h * (h.square().mean(-1, keepdim=True) + 1e-6).rsqrt()
    assert ((out.y.double() - y).abs() <= half_step(y, torch.float16) * 1.001 + y.abs() * CHAIN).all()
    assert out.h[h.abs() > 65520].isinf().all()


@pytest.mark.parametrize("hidden", [96, 1000, 4096, 20000])
def test_in_place_and_guards(hidden):
    m = norm()
    rows = 5
    x, res, w = data((rows, hidden), torch.bfloat16, 1), data((rows, hidden), torch.bfloat16, 2), \
        data((hidden,), torch.bfloat16, 3)
    groups = -(-hidden // 128)
    want = m.add_rms_norm(x, w, res)
    wantq = m.add_rms_norm(x, w, res, out_dtype=E4M3, group=128)

    def guarded(n, dtype):
        buf = torch.full((n + 128,), 0x5A, dtype=torch.uint8, device=DEV).repeat(dtype.itemsize).view(dtype) \
            if dtype != E4M3 else torch.full((n + 128,), 0x5A, dtype=torch.uint8, device=DEV).view(E4M3)
        return buf, buf[64:64 + n]

    for inplace in ("residual", "x", None):
        for q in (False, True):
            x2, r2 = x.clone(), res.clone()
            ybuf, y = guarded(rows * hidden, E4M3 if q else torch.bfloat16)
            rbuf, rstd = guarded(rows, torch.float32)
            sbuf, scale = guarded(rows * groups, torch.float32)
            hbuf, h = guarded(rows * hidden, torch.bfloat16)
            hv = {"residual": r2, "x": x2, None: h.view(rows, hidden)}[inplace]
            out = m.NormOut(y.view(rows, hidden), scale.view(rows, groups) if q else None, hv, rstd)
            got = m.add_rms_norm(x2, w, r2, out_dtype=E4M3 if q else None, group=128 if q else 0, out=out)
            ref = wantq if q else want
            assert got.y.data_ptr() == y.data_ptr() and got.h.data_ptr() == hv.data_ptr()
            assert torch.equal(got.y.view(torch.uint8), ref.y.view(torch.uint8))
            assert torch.equal(got.h, ref.h) and torch.equal(got.rstd, ref.rstd)
            if q:
                assert torch.equal(got.scale, ref.scale)
            for buf, n in ((ybuf, rows * hidden), (rbuf, rows), (sbuf, rows * groups), (hbuf, rows * hidden)):
                edge = torch.cat([buf.view(torch.uint8)[:64 * buf.element_size()],
                                  buf.view(torch.uint8)[(64 + n) * buf.element_size():]])
                assert (edge == 0x5A).all()
            if inplace != "x":
                assert torch.equal(x2, x)
            if inplace != "residual":
                assert torch.equal(r2, res)


@pytest.mark.parametrize("hidden", [96, 301, 1001, 4096, 5001, 20000])
def test_one_source_with_a_copy_of_it(hidden):
    """A single x without a residual, and `h` asked for apart from it."""
    m = norm()
    x, w = data((70, hidden), torch.bfloat16, 1), data((hidden,), torch.bfloat16, 2)
    want = m.add_rms_norm(x, w)
    out = m.NormOut(torch.empty_like(x), None, torch.full_like(x, 7), torch.empty(70, device=DEV))
    got = m.add_rms_norm(x, w, out=out)
    assert torch.equal(got.h, x) and torch.equal(got.y, want.y) and torch.equal(got.rstd, want.rstd)
    same = m.add_rms_norm(x, w, out=m.NormOut(torch.empty_like(x), None, x, torch.empty(70, device=DEV)))
    assert same.h is x and torch.equal(same.y, want.y)


def test_what_out_overwrites_is_seen_by_autograd():
    m = norm()
    res = data((3, 64), torch.float32, 1)
    x, w = data((3, 64), torch.float32, 2), data((64,), torch.float32, 3)
    leaf = data((3, 64), torch.float32, 4).requires_grad_()
    loss = (leaf * res).sum()  # holds res for its gradient
    out = m.NormOut(torch.empty_like(x), None, res, torch.empty(3, device=DEV))
    before = [t._version for t in (out.y, res, out.rstd, x)]
    m.add_rms_norm(x, w, res, out=out)
    assert [t._version > v for t, v in zip((out.y, res, out.rstd, x), before)] == [True, True, True, False]
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        loss.backward()
    # e4m3 with scales; a single x that comes back as h itself is not written
    out = m.NormOut(torch.empty(3, 64, dtype=E4M3, device=DEV), torch.empty(3, 1, device=DEV), x,
                    torch.empty(3, device=DEV))
    written = (out.y, out.scale, out.rstd)
    before = [t._version for t in (*written, x)]
    m.add_rms_norm(x, w, out_dtype=E4M3, out=out)
    assert [t._version > v for t, v in zip((*written, x), before)] == [True, True, True, False]
    with torch.inference_mode():  # tensors of that mode have no version
        free = m.NormOut(torch.empty_like(x), None, torch.empty_like(x), torch.empty(3, device=DEV))
        m.add_rms_norm(x, w, res, out=free)
        before = res._version
        m.add_rms_norm(x, w, res, out=m.NormOut(free.y, None, res, free.rstd))
        assert res._version > before


@pytest.mark.parametrize("hidden", [301, 511])
def test_short_rows_of_many_sources(hidden):
    """More of them than shared memory holds for a block of rows: fp32 rows off the boundary, read again in each pass."""
    m = norm()
    xs = [data((37, hidden), torch.float32, k) for k in range(8)]
    res, w = data((37, hidden), torch.float32, 8), data((hidden,), torch.float32, 9)
    for out_dtype, group in ((None, 0), (E4M3, 0), (E4M3, 64)):
        check(m.add_rms_norm(xs, w, res, out_dtype=out_dtype, group=group), xs, w, res, 1e-6, group)


# ------------------------------------------------------------------ gradient

def grad_reference(dy, h, w, rstd, dh):
    d, n, w, r = dy.double(), h.double() * rstd.double()[..., None], w.double(), rstd.double()[..., None]
    hidden = h.shape[-1]
    g = d * w
    c = (g * n).mean(-1, keepdim=True)
    dx = r * (g - n * c)
    c_tol = CHAIN * (g * n).abs().mean(-1, keepdim=True)
    tol = r * (8 * U * (g.abs() + (n * c).abs()) + n.abs() * c_tol)
    if dh is not None:
        dx = dx + dh.double()
        tol = tol + 4 * U * dh.double().abs()
    flat = (d * n).reshape(-1, hidden)
    dw = flat.sum(0)
    # A column's products are added over at most all rows in one chain.
    dw_tol = (flat.shape[0] + 64) * U * flat.abs().sum(0)
    return dx, tol, dw, dw_tol


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows, hidden", SHAPES + MANY + [(1, 4096), (9, 17000)])
def test_gradient(rows, hidden, dtype):
    m = norm()
    h, dy = data((rows, hidden), dtype, 1, 2.0), data((rows, hidden), dtype, 2)
    rstd = (h.double().square().mean(-1) + 1e-6).rsqrt().float()
    for w in (data((hidden,), dtype, 3), data((hidden,), torch.float32, 4)):
        for dh in (None, data((rows, hidden), dtype, 5)):
            dx, dw = m.add_rms_norm_backward(dy, h, w, rstd, dh)
            rx, tx, rw, tw = grad_reference(dy, h, w, rstd, dh)
            assert dx.dtype == dtype and dw.dtype == w.dtype
            assert ((dx.double() - rx).abs() <= half_step(rx, dtype) * 1.001 + tx).all()
            assert ((dw.double() - rw).abs() <= half_step(rw, w.dtype) * 1.001 + tw).all()
            again = m.add_rms_norm_backward(dy, h, w, rstd, dh)
            assert torch.equal(again[0], dx) and torch.equal(again[1], dw)


def test_gradient_strides():
    m = norm()
    packed = data((40, 9, 128), torch.bfloat16, 1)
    for h, dy, dh in ((packed[:, 3:6], data((40, 3, 128), torch.bfloat16, 2), packed[:, 6:9]),
                      (packed[:, 0], packed[:, 1], None),
                      (data((4, 10, 99), torch.bfloat16, 3)[:, :, 3:], packed.view(-1)[5:5 + 3840].view(4, 10, 96),
                       None),
                      (packed, data((128,), torch.bfloat16, 5).expand(40, 9, 128), None)):
        w = data((h.shape[-1],), torch.float32, 4)
        rstd = (h.double().square().mean(-1) + 1e-6).rsqrt().float()
        dx, dw = m.add_rms_norm_backward(dy, h, w, rstd, dh)
        rx, tx, rw, tw = grad_reference(dy, h, w, rstd, dh)
        assert dx.is_contiguous()
        assert ((dx.double() - rx).abs() <= half_step(rx, torch.bfloat16) * 1.001 + tx).all()
        assert ((dw.double() - rw).abs() <= half_step(rw, torch.float32) * 1.001 + tw).all()


@pytest.mark.parametrize("hidden", [60, 1000])
def test_gradient_against_differences(hidden):
    """dx and dweight along random directions against differences of the
    formula in 64 bits: L = sum(y * dy) + sum(h * dh), step 1e-5, whose own error
    (its third derivative times 1e-10, and 1e-16 / 1e-5 of rounding) is far
    below the kernel's."""
    m = norm()
    rows = 6
    h, dy, dh = [data((rows, hidden), torch.float32, k) for k in range(3)]
    w = data((hidden,), torch.float32, 3)
    out = m.add_rms_norm(h, w)
    dx, dw = m.add_rms_norm_backward(dy, h, w, out.rstd, dh)
    _, tx, _, tw = grad_reference(dy, h, w, out.rstd, dh)

    def loss(x, w):
        y = x * (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w
        return (y * dy.double()).sum() + (x * dh.double()).sum()

    for k in range(8):
        ex, ew = data((rows, hidden), torch.float64, 20 + k), data((hidden,), torch.float64, 30 + k)
        step = 1e-5
        got = (loss(h.double() + step * ex, w.double()) - loss(h.double() - step * ex, w.double())) / (2 * step)
        # rstd itself came rounded from the forward: CHAIN of every term that holds it
        slack = ((tx + (dx.double() - dh.double()).abs() * 4 * CHAIN) * ex.abs()).sum() + 1e-6
        assert abs(got - (dx.double() * ex).sum()) <= slack + U * (dx.double() * ex).abs().sum()
        got = (loss(h.double(), w.double() + step * ew) - loss(h.double(), w.double() - step * ew)) / (2 * step)
        slack = ((tw + (dy.double() * h.double() * out.rstd.double()[:, None]).abs().sum(0) * CHAIN) * ew.abs()).sum()
        assert abs(got - (dw.double() * ew).sum()) <= slack + 1e-6 + U * (dw.double() * ew).abs().sum()


def test_streams_and_graphs():
    m = norm()
    x, res, w = data((64, 1024), torch.bfloat16, 1), data((64, 1024), torch.bfloat16, 2), \
        data((1024,), torch.bfloat16, 3)
    dy = data((64, 1024), torch.bfloat16, 4)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        a = m.add_rms_norm(x, w, res, out_dtype=E4M3, group=128)
    side.synchronize()
    b = m.add_rms_norm(x, w, res, out_dtype=E4M3, group=128)
    assert torch.equal(a.y.view(torch.uint8), b.y.view(torch.uint8))
    graphs = []
    for _ in range(2):  # two graphs alive at once, each with a workspace of its own
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = m.add_rms_norm(x, w, res)
            dx, dw = m.add_rms_norm_backward(dy, out.h, w, out.rstd, dy)
        graphs.append((g, out, dx, dw))
    for seed in (5, 6):
        x.copy_(data((64, 1024), torch.bfloat16, seed))
        for g, *_ in graphs:
            g.replay()
        out = m.add_rms_norm(x, w, res)
        dx, dw = m.add_rms_norm_backward(dy, out.h, w, out.rstd, dy)
        for _, o, gx, gw in graphs:
            assert torch.equal(o.y, out.y) and torch.equal(o.h, out.h)
            assert torch.equal(gx, dx) and torch.equal(gw, dw)


def test_offsets_beyond_32_bits():
    """Rows behind 2^32 bytes and 2^31 elements of one tensor."""
    m = norm()
    rows, hidden = (1 << 31) // 1024 + 3, 1024
    x = torch.zeros(rows, hidden, dtype=torch.bfloat16, device=DEV)
    tail = data((4, hidden), torch.bfloat16, 1)
    x[-4:] = tail
    w = data((hidden,), torch.bfloat16, 2)
    out = m.add_rms_norm(x, w)
    want = m.add_rms_norm(tail, w)
    assert torch.equal(out.y[-4:], want.y) and not out.y[:-4].any()
    del out
    dy = x  # any gradient
    rstd = torch.ones(rows, dtype=torch.float32, device=DEV)
    dx, dw = m.add_rms_norm_backward(dy, x, w, rstd)
    tx, tw = m.add_rms_norm_backward(tail, tail, w, rstd[:4])
    assert torch.equal(dx[-4:], tx) and not dx[:-4].any()
    # four rows that are not zero, in another grouping: fp32 sums of four terms
    assert ((dw.double() - tw.double()).abs() <= tw.double().abs() * 2.0 ** -7 + 1e-6).all()


def test_a_device_that_is_not_there_leaves_no_error_behind():
    """The refused call returns its code; torch, which looks at CUDA's last error after its own launches, finds none."""
    m = norm()
    from scc26_nccl_shim_b200.ops import optim
    x, w = data((4, 64), torch.bfloat16, 1), data((64,), torch.bfloat16, 2)
    y, rstd, err = torch.empty_like(x), torch.empty(4, device=DEV), C.create_string_buffer(256)
    p, missing = x.data_ptr(), 60
    call = m._FWD[1].pack(p, 64, 0, 0, 0, 0, w.data_ptr(), y.data_ptr(), 0, 0, rstd.data_ptr(), 4, 1, missing, 64, 1, 9, 9,
                          9, 0, 1e-6)
    assert m.lib().nb_add_rms_norm(call, None, err, 256) > 0 and b"device" in err.value
    torch.zeros(8, device=DEV)
    assert m.lib().nb_add_rms_norm_backward_workspace(missing, 4, 64, 9) == 0
    torch.zeros(8, device=DEV)
    one, at = (C.c_uint64 * 1)(4), (C.c_uint64 * 1)(p)
    assert optim.lib().nb_grad_norm_create(missing, 1, 1, 9, one, at, err, 256) is None and b"device" in err.value
    torch.zeros(8, device=DEV)
    assert torch.cuda.current_device() == 0


@pytest.mark.parametrize("rows, hidden", [(3, 64), (300, 1000), (70, 4096), (5, 9000)])
def test_gradient_at_two_alignments(rows, hidden):
    """The same values at another offset take another kernel: dweight is added in another order, within the same bound."""
    m = norm()
    w = data((hidden,), torch.float32, 3)
    h, dy = data((rows, hidden), torch.bfloat16, 1, 2.0), data((rows, hidden), torch.bfloat16, 2)
    rstd = (h.double().square().mean(-1) + 1e-6).rsqrt().float()
    rx, tx, rw, tw = grad_reference(dy, h, w, rstd, None)
    flat = torch.empty(2, rows * hidden + 1, dtype=torch.bfloat16, device=DEV)
    for t, v in zip(flat, (dy, h)):
        t[1:].copy_(v.view(-1))
    for d, hh in ((dy, h), [t[1:].view(rows, hidden) for t in flat]):
        dx, dw = m.add_rms_norm_backward(d, hh, w, rstd)
        assert ((dx.double() - rx).abs() <= half_step(rx, torch.bfloat16) * 1.001 + tx).all()
        assert ((dw.double() - rw).abs() <= half_step(rw, torch.float32) * 1.001 + tw).all()
        again = m.add_rms_norm_backward(d, hh, w, rstd)
        assert torch.equal(again[0], dx) and torch.equal(again[1], dw)
