"""AdamW and the gradients' norm over many tensors (ops/optim.py) against their
formulas in 64 bits.

Tolerances with u = 2^-24: m and v are sums of two products (3 u of the terms'
magnitudes) of a gradient that is a sum of n terms (n u of theirs); the update
is a quotient of them with a square root, a constant and eps (16 u covers its
roundings and the constants' own); p a difference of a product and the update.
"""
import math

import pytest
import torch

from conftest import need_gpus

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
E4M3 = torch.float8_e4m3fn
U = 2.0 ** -24
SIZES = [1, 7, 8, 255, 256, 257, 2047, 2048, 2049, 5000, 0, 70000]
BETAS, EPS, LR = (0.9, 0.999), 1e-8, 1e-2
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}


def optim():
    need_gpus(1)
    from scc26_nccl_shim_b200.ops import optim as m
    return m


def data(n, dtype, seed, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(n, device=DEV, generator=g) * scale).to(dtype)


def half_step(ref, dtype):
    return ref.abs() * (torch.finfo(dtype).eps / 2) + TINY[dtype] / 2


def gradient(parts, scale):
    terms = [g.double() for g in parts]
    return sum(terms) * scale, (len(terms) + 1) * U * abs(scale) * sum(t.abs() for t in terms)


def expected(p, parts, m, v, t, lr, wd, scale, betas=BETAS):
    """p, m, v after the step and how far fp32 may be off each."""
    b1, b2 = betas
    g, g_tol = gradient(parts, scale)
    m1, v1 = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    m_tol = 4 * U * (abs(b1 * m) + (1 - b1) * g.abs()) + (1 - b1) * g_tol
    v_tol = 5 * U * (b2 * v + (1 - b2) * g * g) + (1 - b2) * 2 * g.abs() * g_tol + 2.0 ** -148
    size = lr / (1 - b1 ** t) if b1 else lr
    den = (v1 / (1 - b2 ** t if b2 else 1)).sqrt() + EPS
    update = size * m1 / den
    # relative error of the root is half that of v; where v is zero the bound is that of its tiny values
    root_rel = torch.where(v1 > 0, v_tol / v1.clamp(min=1e-300), torch.zeros_like(v1)).clamp(max=1.0)
    p1 = p * (1 - lr * wd) - update
    p_tol = 4 * U * p.abs() + update.abs() * (16 * U + root_rel) + size * m_tol / den
    return (p1, p_tol), (m1, m_tol), (v1, v_tol)


def near(got, want, dtype=torch.float32):
    ref, tol = want
    return ((got.double() - ref).abs() <= half_step(ref, dtype) * 1.001 + tol * 1.001).all()


def tensors(sizes, dtype, seed, scale, packed):
    """Separate tensors, or views one after another in one buffer (odd offsets)."""
    flat = data(sum(sizes) + 1, dtype, seed, scale)
    if packed:
        out, at = [], 1
        for n in sizes:
            out.append(flat[at:at + n])
            at += n
        return out
    return [t.clone() for t in flat[:-1].split(sizes)]


@pytest.mark.parametrize("ptype, ctype", [(torch.float32, None), (torch.float32, torch.bfloat16),
                                          (torch.float32, torch.float16), (torch.bfloat16, None),
                                          (torch.float16, None)])
@pytest.mark.parametrize("gtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("packed", [False, True])
def test_adamw(ptype, ctype, gtype, packed):
    m = optim()
    for parts in (1, 3):
        params = tensors(SIZES, ptype, 1, 1.0, packed)
        grads = [list(g) for g in zip(*[tensors(SIZES, gtype, 2 + k, 0.1, packed) for k in range(parts)])]
        ms, vs = tensors(SIZES, torch.float32, 20, 0.1, packed), \
            [x.square() for x in tensors(SIZES, torch.float32, 21, 0.1, packed)]
        copies = tensors(SIZES, ctype, 22, 1.0, packed) if ctype else None
        decay = [0.1 * (i % 3) for i in range(len(SIZES))]
        before = [[x.double() for x in ts] for ts in (params, ms, vs)]
        held = [[g.clone() for g in gs] for gs in grads]
        opt = m.AdamW(params, grads, betas=BETAS, eps=EPS, weight_decay=decay, states=(ms, vs), copies=copies)
        opt.step(3, LR, scale=0.5)
        for i in range(len(SIZES)):
            p, mm, v = expected(before[0][i], grads[i], before[1][i], before[2][i], 3, LR, decay[i], 0.5)
            assert near(params[i], p, ptype) and near(ms[i], mm) and near(vs[i], v)
            if ctype:
                assert torch.equal(copies[i], params[i].to(ctype))
            assert all(torch.equal(a, b) for a, b in zip(grads[i], held[i]))


def test_adamw_first_steps_and_betas():
    m = optim()
    for betas in ((0.9, 0.999), (0.0, 0.95), (0.9, 0.0), (0.0, 0.0)):
        p, g = data(3000, torch.float32, 1), data(3000, torch.float32, 2)
        opt = m.AdamW([p], [g], betas=betas, eps=EPS, weight_decay=0.0)
        mm, v = torch.zeros(3000, device=DEV).double(), torch.zeros(3000, device=DEV).double()
        for t in (1, 2, 3):
            want = expected(p.double(), [g], opt.exp_avg[0].double(), opt.exp_avg_sq[0].double(), t, LR, 0.0, 1.0,
                            betas)
            opt.step(t, LR)
            assert near(p, want[0]) and near(opt.exp_avg[0], want[1]) and near(opt.exp_avg_sq[0], want[2])


def test_many_tensors_take_several_launches():
    m = optim()
    sizes = [1 + (i * 37) % 300 for i in range(1500)]
    params, grads = tensors(sizes, torch.float32, 1, 1.0, True), tensors(sizes, torch.bfloat16, 2, 1.0, True)
    before = [p.double() for p in params]
    opt = m.AdamW(params, grads, weight_decay=0.1)
    opt.step(1, LR)
    zero = torch.zeros(1, device=DEV).double()
    for i in range(0, 1500, 31):
        assert near(params[i], expected(before[i], [grads[i]], zero, zero, 1, LR, 0.1, 1.0)[0])
    got = m.GradNorm(grads)()
    ref = torch.cat(grads).double().norm()
    assert abs(got[0].double() - ref) <= 32 * U * ref


# ------------------------------------------------------------------ 8-bit states

def hash_bits(n, tensor, seed, t):
    low = 0xFFFFFFFF
    x = torch.arange(n, dtype=torch.int64, device=DEV)
    x = (x * 0x9E3779B9 + tensor * 0x3C6EF35F + seed * 0x27D4EB2F + t * 0x165667B1) & low
    x = ((x ^ (x >> 16)) * 0xA5CB9243) & low
    x = ((x ^ (x >> 15)) * 0x5D8A37E5) & low
    return x ^ (x >> 16)


def blocks(x):
    n = x.numel()
    return torch.nn.functional.pad(x.view(-1), (0, -n % 256)).view(-1, 256)


def check_codes(codes, scale, want, bits16, positive):
    """`want` (value, tolerance) against e4m3 codes that were rounded with
    bits16 / 65536 of a step."""
    ref, tol = want
    n = ref.numel()
    b, bt = blocks(ref), blocks(tol)
    top = b.abs().amax(1)
    s = (top / 448).clamp(min=2.0 ** -126)
    s_tol = bt.amax(1) / 448 + 4 * U * s
    assert ((scale.double() - s).abs() <= s_tol).all()
    z = (b.abs() / s[:, None]).clamp(max=448.0)
    z_tol = (bt + b.abs() * (s_tol / s)[:, None]) / s[:, None] + 4 * U * z
    step = torch.exp2((torch.floor(torch.log2(z.clamp(min=2.0 ** -9)))).clamp(min=-6) - 3)
    u = blocks(bits16.double() / 65536)
    q = torch.floor(z / step + u) * step
    if positive:
        q = torch.where(b > 0, q.clamp(min=2.0 ** -9), q)
    got = blocks(codes.double())
    assert (got * b >= 0).all()
    edge = (z / step + u) - torch.round(z / step + u)
    sure = edge.abs() > z_tol / step + 16 * 4 * U
    binade = torch.log2(z.clamp(min=2.0 ** -9))
    sure &= (binade - torch.round(binade)).abs() > 1e-5           # a step's own size is in doubt there
    off = (got.abs() != q) & sure
    assert not off.view(-1)[:n].any(), (int(off.sum()), n)
    assert ((got.abs() - q).abs() <= 1.01 * 2 * step).all()
    if n >= 1000:  # the comparison is not empty (padding behind a tensor is always at an edge)
        assert sure.view(-1)[:n].double().mean() > 0.95
    assert not got.view(-1)[n:].any()


@pytest.mark.parametrize("gtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("packed", [False, True])
def test_adamw_8bit(gtype, packed):
    m = optim()
    sizes = [1, 7, 255, 256, 257, 2049, 5000, 0, 70000]
    params, grads = tensors(sizes, torch.float32, 1, 1.0, packed), tensors(sizes, gtype, 2, 0.1, packed)
    for g in grads:
        g[::7] = 0
    byte = lambda n: tensors(sizes, torch.float32, n, 3.0, False)  # noqa: E731
    codes = []
    for k in (0, 1):
        flat = torch.zeros(sum(sizes) + 1, dtype=torch.uint8, device=DEV).view(E4M3)
        at, views = (1 if packed else 0), []
        for n, x in zip(sizes, byte(30 + k)):
            views.append(flat[at:at + n] if packed else torch.zeros(n, dtype=torch.uint8, device=DEV).view(E4M3))
            views[-1].copy_((x.abs() if k else x).clamp(-448, 448).to(E4M3))
            at += n
        codes.append(views)
    scales = [[data(-(-n // 256), torch.float32, 40 + k, 0.01).abs() for n in sizes] for k in (0, 1)]
    states = [list(zip(c, s)) for c, s in zip(codes, scales)]
    opt = m.AdamW(params, grads, betas=BETAS, eps=EPS, weight_decay=0.1, state="8bit", states=states, seed=77)
    before = [[x.double() for x in opt.moments(i)] + [params[i].double()] for i in range(len(sizes))]
    opt.step(9, LR, scale=2.0)
    for i, n in enumerate(sizes):
        if not n:
            continue
        mm, v, p = before[i]
        wp, wm, wv = expected(p, [grads[i]], mm, v, 9, LR, 0.1, 2.0)
        # the dequantised states are products of two and three fp32 numbers
        wm = (wm[0], wm[1] + 2 * U * mm.abs())
        wv = (wv[0], wv[1] + 4 * U * v.abs())
        wp = (wp[0], wp[1] + 8 * U * LR * 20 * torch.ones_like(p))
        assert near(params[i], wp)
        bits = hash_bits(n, i, 77, 9)
        check_codes(opt.exp_avg[i][0], opt.exp_avg[i][1], wm, bits >> 16, False)
        root = wv[0].sqrt()
        check_codes(opt.exp_avg_sq[i][0], opt.exp_avg_sq[i][1],
                    (root, wv[1] / root.clamp(min=1e-18) + 2 * U * root), bits & 0xFFFF, True)
        mq, vq = opt.moments(i)
        assert ((vq > 0) | (wv[0] == 0)).all()  # a positive v stays positive


def test_8bit_rounding_keeps_the_mean():
    """Over many elements the rounded state's mean error is zero within six
    standard deviations (at most half a step each)."""
    m = optim()
    n = 1 << 20
    p, g = torch.zeros(n, device=DEV), data(n, torch.float32, 2)
    opt = m.AdamW([p], [g], betas=BETAS, state="8bit", weight_decay=0.0)
    opt.step(1, 0.0)
    for got, want in zip(opt.moments(0), (g.double() * 0.1, None)):
        if want is None:
            got, want = got.double().sqrt(), (g.double() * math.sqrt(0.001)).abs()
        scale = blocks(want).abs().amax(1) / 448
        z = blocks(want).abs() / scale[:, None]
        step = torch.exp2(torch.floor(torch.log2(z.clamp(min=2.0 ** -9))).clamp(min=-6) - 3) * scale[:, None]
        keep = (z > 2.0 ** -8).view(-1)  # where the least code of sqrt(v) plays no part
        err = ((got.double().abs() - want.abs()) / step.view(-1))[keep]
        assert abs(err.mean()) <= 6 * 0.5 / math.sqrt(err.numel())
        assert err.abs().max() <= 1.001


def test_8bit_states_follow_the_32bit_ones():
    """The same noise for 300 steps: states that were rounded to nearest would
    stand still after some 16 steps (a step moves sqrt(v) by less than half a
    code), here the mean of sqrt(v) stays with the 32-bit one's. Each of 65536
    roundings a step is unbiased; what remains is the least code (2^-9 of 448)
    and the curvature of the root under noise, a variance of at most 1/16 of a
    step's square per step: under 10 % of the mean."""
    m = optim()
    n = 65536
    g = torch.empty(n, device=DEV)
    p8, p32 = torch.zeros(n, device=DEV), torch.zeros(n, device=DEV)
    a = m.AdamW([p8], [g], state="8bit", weight_decay=0.0)
    b = m.AdamW([p32], [g], weight_decay=0.0)
    for t in range(1, 301):
        g.copy_(data(n, torch.float32, 1000 + t))
        a.step(t, 1e-3)
        b.step(t, 1e-3)
    r8, r32 = a.moments(0)[1].sqrt().double(), b.moments(0)[1].sqrt().double()
    assert abs(r8.mean() / r32.mean() - 1) < 0.1


def test_8bit_roots_are_the_rounded_ones():
    """The kernel's own square root against torch's rounded one, on a million
    values over the range that it is used for: with one element a block, the new
    scale is sqrt(v) times 1/448. It may miss by one unit in the last place
    where the root lies next to the middle of two numbers: Newton's step leaves
    an error below 2^-42 of it, so in less than one of 2^17 cases."""
    m = optim()
    n = 1 << 20
    g = torch.Generator(device=DEV).manual_seed(3)
    scale = torch.exp(torch.rand(n, device=DEV, generator=g) * 60 - 40)  # 4e-18 to 5e8
    codes = torch.zeros(n * 256, dtype=torch.uint8, device=DEV)
    codes[::256] = 0x7E  # 448
    zero = (torch.zeros(n * 256, dtype=torch.uint8, device=DEV).view(E4M3), torch.zeros(n, device=DEV))
    p, grad = torch.zeros(n * 256, dtype=torch.bfloat16, device=DEV), \
        torch.zeros(n * 256, dtype=torch.bfloat16, device=DEV)
    before = scale.clone()
    opt = m.AdamW([p], [grad], betas=(0.9, 0.7), state="8bit", states=([zero], [(codes.view(E4M3), scale)]))
    opt.step(5, 0.0)
    r = before * 448
    want = torch.sqrt(r * r * 0.7) * torch.tensor(1 / 448, device=DEV)
    assert ((scale.view(torch.int32) - want.view(torch.int32)).abs() <= 1).all()
    assert (scale != want).sum() <= n >> 17


@pytest.mark.parametrize("size", [1e-30, 1e-20, 1e8, 1e14, 1e18])
def test_8bit_extreme_gradients(size):
    """v between the smallest subnormal numbers and the largest ones."""
    m = optim()
    p, g = torch.zeros(3000, device=DEV), data(3000, torch.float32, 2, size)
    opt = m.AdamW([p], [g], betas=BETAS, eps=1e-37, weight_decay=0.0, state="8bit")
    opt.step(1, LR)
    v = 0.001 * g.double().square()
    # In fp32, v below 2^-126 loses bits: off by up to 2^-149 (three roundings).
    v_tol = 8 * U * v + 3 * 2.0 ** -149
    low, high = (v - v_tol).clamp(min=0), v + v_tol
    mhat = g.double()
    got = -p.double() / LR
    big = mhat.abs() > 0
    lo = mhat.abs() / ((high * 1000).sqrt() + 1e-37) * (1 - 64 * U)
    hi = mhat.abs() / ((low * 1000).sqrt() + 1e-37) * (1 + 64 * U)
    assert (got.sign() == mhat.sign())[big].all()
    # (the squares below 2^-149 vanish: the update is then m / eps)
    assert ((got.abs() >= lo) & (got.abs() <= hi))[big].all()
    mq, vq = opt.moments(0)
    assert ((mq.double() - 0.1 * g.double()).abs() <= 0.1 * g.double().abs() / 8 * 1.001 + opt.exp_avg[0][1].double()
            .repeat_interleave(256)[:3000] * 2.0 ** -9).all()
    assert vq.isfinite().all()


def test_nan_gradient_stays_in_its_block():
    m = optim()
    p, g = data(1024, torch.float32, 1), data(1024, torch.float32, 2)
    g[300] = float("nan")
    opt = m.AdamW([p], [g], state="8bit")
    opt.step(1, LR)
    assert p.isnan().nonzero().view(-1).tolist() == [300]
    scale = opt.exp_avg[0][1]
    assert scale[1].isnan() and scale[[0, 2, 3]].isfinite().all()


# ------------------------------------------------------------------ the gradients' norm

@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("parts", [1, 2, 8])
@pytest.mark.parametrize("packed", [False, True])
def test_grad_norm(dtype, parts, packed):
    m = optim()
    grads = [list(g) for g in zip(*[tensors(SIZES, dtype, k, 0.3, packed) for k in range(parts)])]
    f = m.GradNorm(grads)
    total = sum(gradient(g, 1.0)[0].square().sum() for g in grads)
    slack = sum((2 * gradient(g, 1.0)[0].abs() * gradient(g, 1.0)[1]).sum() for g in grads)
    ref = total.sqrt()
    # eight squares in fp32 (9 u), the rest in fp64, the result rounded
    tol = ref * 16 * U + slack / (2 * ref)
    for max_norm, scale in ((1.0, 1.0), (float(ref) * 10, 1.0), (3.0, 0.25), (math.inf, 1.0)):
        out = f(max_norm, scale).double()
        assert abs(out[0] - scale * ref) <= scale * tol
        coef = scale * min(1.0, max_norm / (scale * float(ref) + 1e-6))
        assert abs(out[1] - coef) <= coef * (4 * U + float(tol / ref))
    assert torch.equal(f(), f())


def test_grad_norm_not_finite_and_empty():
    m = optim()
    for bad in (float("nan"), float("inf"), 3e38):
        g = [data(1000, torch.float32, 1), data(3000, torch.float32, 2)]
        g[1][2999] = bad
        out = m.GradNorm(g)(1.0)
        assert not out[0].isfinite() and out[1].isnan()
    out = m.GradNorm([torch.empty(0, device=DEV)])(1.0)
    assert out.tolist() == [0.0, 1.0]
    with pytest.raises(ValueError, match="max_norm"):
        m.GradNorm([data(8, torch.float32, 1)])(0.0)
    with pytest.raises(ValueError, match="scale"):
        m.GradNorm([data(8, torch.float32, 1)])(1.0, scale=float("nan"))


def test_a_step_is_skipped_after_an_overflow():
    m = optim()
    for state in ("float32", "8bit"):
        p, g = data(5000, torch.float32, 1), data(5000, torch.float32, 2)
        copy = p.bfloat16()
        opt = m.AdamW([p], [g], state=state, copies=[copy])
        norm = m.GradNorm([g])
        opt.step(1, LR, scale=norm(1.0)[1])
        kept = [p.clone(), copy.clone(), *[x.clone() for x in opt.moments(0)]]
        g[17] = float("inf")
        opt.step(2, LR, scale=norm(1.0)[1])
        for a, b in zip(kept, [p, copy, *opt.moments(0)]):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("parts", [1, 3])
@pytest.mark.parametrize("size", [1e-39, 1e-30, 1e-22, 1e-19, 6e18, 1e20, 1e30, 1e35])
def test_grad_norm_where_squares_leave_fp32(dtype, parts, size):
    m = optim()
    for at in (0, 1):
        grads = [[data(n + 1, dtype, 10 * k + n, size)[at:at + n] for k in range(parts)] for n in (5, 2048, 5003)]
        f = m.GradNorm(grads)
        total = sum(gradient(g, 1.0)[0].square().sum() for g in grads)
        slack = sum((2 * gradient(g, 1.0)[0].abs() * gradient(g, 1.0)[1]).sum() for g in grads)
        ref = total.sqrt()
        # eight squares (9 u), the result rounded (u, or half of 2^-149)
        tol = ref * 16 * U + slack / (2 * ref) + 2.0 ** -149
        for max_norm, scale in ((1.0, 1.0), (float(ref) / 2, 1.0), (1.0, 0.25)):
            out = f(max_norm, scale).double()
            assert abs(out[0] - scale * ref) <= scale * tol + 2.0 ** -149
            coef = scale * min(1.0, max_norm / (scale * float(ref) + 1e-6))
            assert abs(out[1] - coef) <= coef * (4 * U + float(tol / ref)) + 2.0 ** -149


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_grad_norm_of_one_large_or_small_element(dtype):
    m = optim()
    for big in (3e18, 2e19, 1e25, 8e37):  # beside 5000 of about 1, and 5000 of nothing
        g = data(5000, dtype, 1)
        g[4321] = big
        out = m.GradNorm([g, torch.zeros(5000, dtype=dtype, device=DEV)])(1.0).double()
        ref = float(g[4321].double())
        assert abs(out[0] - ref) <= ref * 16 * U and abs(out[1] - 1 / ref) <= 16 * U / ref
    g = torch.zeros(5000, dtype=dtype, device=DEV)
    assert m.GradNorm([g])(1.0).tolist() == [0.0, 1.0]
    g[4321] = 2.0 ** -120
    assert m.GradNorm([g])(1.0).tolist() == [2.0 ** -120, 1.0]
    # From 2^126 on, 1 / norm is no normal number: an overflow.
    g[4321] = 2.0 ** 126
    out = m.GradNorm([g])(1.0)
    assert float(out[0]) == 2.0 ** 126 and float(out[1]) == 2.0 ** -126
    g[1] = 2.0 ** 126
    out = m.GradNorm([g])(1.0)
    assert out[0].isinf() and out[1].isnan()


def test_a_step_is_clipped_not_skipped_after_a_large_gradient():
    m = optim()
    for state in ("float32", "8bit"):
        p, g = data(5000, torch.float32, 1), data(5000, torch.float32, 2)
        g[17] = 1e20
        opt, before = m.AdamW([p], [g], state=state, weight_decay=0.0), p.clone()
        opt.step(1, LR, scale=m.GradNorm([g])(1.0)[1])
        # g[17] is scaled to 1 - 1e-13: the first step's update is lr g / (|g| + eps)
        assert abs(float(before[17] - p[17]) - LR) <= 32 * U * LR + 4 * U * abs(float(before[17]))
        assert p.isfinite().all() and all(x.isfinite().all() for x in opt.moments(0))


@pytest.mark.parametrize("state", ["float32", "8bit"])
def test_a_device_lr_that_is_not_finite_changes_nothing(state):
    m = optim()
    p, g = data(5000, torch.float32, 1), data(5000, torch.float32, 2)
    copy = p.bfloat16()
    opt = m.AdamW([p], [g], state=state, copies=[copy])
    lr, t = torch.full((1,), LR, device=DEV), torch.ones(1, dtype=torch.int64, device=DEV)
    opt.step(1, lr)
    kept = [p.clone(), copy.clone(), *[x.clone() for x in opt.moments(0)]]
    for bad in (math.nan, math.inf, -math.inf, 2e38):  # 2e38 / (1 - 0.9) is not finite
        lr.fill_(bad)
        opt.step(1, lr)
        opt.step(t, lr)
    opt.step(t, 2e38)
    for a, b in zip(kept, [p, copy, *opt.moments(0)]):
        assert torch.equal(a, b)
    lr.fill_(LR)
    opt.step(2, lr)
    assert not torch.equal(kept[0], p) and p.isfinite().all()


# ------------------------------------------------------------------ use

def test_device_scalars_and_graphs():
    m = optim()

    def make(state):
        ps, gs = tensors([3000, 5], torch.float32, 1, 1.0, False), tensors([3000, 5], torch.bfloat16, 2, 1.0, False)
        return ps, gs, m.AdamW(ps, gs, state=state), m.GradNorm(gs)

    for state in ("float32", "8bit"):
        ps, gs, opt, norm = make(state)
        qs, hs, ref, rnorm = make(state)
        t = torch.ones(1, dtype=torch.int64, device=DEV)
        lr = torch.full((1,), LR, device=DEV)
        side = torch.cuda.Stream()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            opt.step(t, lr, scale=norm(1.0)[1])
            t += 1
        for k in (1, 2, 3, 4):
            for a, b in zip(gs, hs):
                a.copy_(data(a.numel(), torch.bfloat16, 50 + k))
                b.copy_(a)
            lr.fill_(LR / k)
            graph.replay()
            ref.step(k, LR / k, scale=rnorm(1.0)[1])
        torch.cuda.synchronize()
        for a, b in zip(ps, qs):
            # the bias corrections and 1 - lr wd in fp32 on the device, in fp64 on the host: a few u of
            # each update, of at most lr times 10 a step (|mhat| / sqrt(vhat) < 10 with these betas)
            tol = 4 * (8 * U * 10 * LR + 4 * U * b.double().abs())
            if state == "8bit":  # a code may then round to its neighbour: an eighth of an update
                assert ((a.double() - b.double()).abs() > tol).double().mean() < 1e-3
                tol = tol + 4 * 10 * LR / 8
            assert ((a.double() - b.double()).abs() <= tol).all()


def test_moved_storage_is_refused_and_versions_are_bumped():
    m = optim()
    p, g = data(100, torch.float32, 1).requires_grad_(), data(100, torch.float32, 2)
    opt = m.AdamW([p], [g])
    before = p._version
    opt.step(1, LR)
    assert p._version > before
    y = (p * p).sum()
    opt.step(2, LR)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.backward()
    g.untyped_storage().resize_(4000)
    with pytest.raises(RuntimeError, match="moved"):
        opt.step(3, LR)


def test_refused_steps_change_nothing():
    m = optim()
    p, g = data(100, torch.float32, 1), data(100, torch.float32, 2)
    opt = m.AdamW([p], [g])
    held = p.clone()
    for kw in (dict(t=0, lr=LR), dict(t=1, lr=math.nan), dict(t=1, lr=LR, scale=math.inf),
               dict(t=torch.ones(1, device=DEV), lr=LR), dict(t=1, lr=torch.ones(1)),
               dict(t=1, lr=torch.ones(2, device=DEV)), dict(t=1, lr=LR, scale=torch.ones(1, device=DEV).double())):
        with pytest.raises(ValueError):
            opt.step(**kw)
    assert torch.equal(p, held)


def test_numbers_beyond_fp32_are_refused():
    m = optim()
    p, g = data(100, torch.float32, 1), data(100, torch.float32, 2)
    opt = m.AdamW([p], [g], betas=(0.999, 0.999))
    held = p.clone()
    # 1e37 is one, 1e37 / (1 - 0.999) is not.
    for kw in (dict(t=1, lr=1e39), dict(t=1, lr=1e37), dict(t=1, lr=LR, scale=1e39),
               dict(t=torch.ones(1, dtype=torch.int64, device=DEV), lr=1e39)):
        with pytest.raises(ValueError, match="fp32"):
            opt.step(**kw)
    assert torch.equal(p, held)
    for norm_of in (dict(scale=math.inf), dict(scale=1e39), dict(max_norm=0.0), dict(max_norm=math.nan)):
        with pytest.raises(ValueError):
            m.GradNorm([g])(**norm_of)


def test_guards_around_every_tensor():
    m = optim()
    sizes = [5, 300, 2049]
    for state in ("float32", "8bit"):
        flats = {k: torch.full((sum(sizes) + 64 * 4,), 0x5A, dtype=torch.uint8, device=DEV).repeat(w)
                 for k, w in (("p", 4), ("c", 2), ("m", 4 if state == "float32" else 1),
                              ("v", 4 if state == "float32" else 1))}
        dt = {"p": torch.float32, "c": torch.bfloat16, "m": torch.float32 if state == "float32" else E4M3,
              "v": torch.float32 if state == "float32" else E4M3}
        views = {k: [] for k in flats}
        inside = {k: torch.zeros_like(f, dtype=torch.bool) for k, f in flats.items()}
        for k, f in flats.items():
            at, w = 64, dt[k].itemsize
            for n in sizes:
                v = f.view(dt[k])[at:at + n]
                v.view(torch.uint8).zero_()
                views[k].append(v)
                inside[k][at * w:(at + n) * w] = True
                at += n + 64
        scales = [[torch.zeros(-(-n // 256), device=DEV) for n in sizes] for _ in "mv"]
        states = (views["m"], views["v"]) if state == "float32" else \
            [list(zip(views[k], s)) for k, s in zip("mv", scales)]
        grads = [data(n, torch.bfloat16, n) for n in sizes]
        opt = m.AdamW(views["p"], grads, states=states, copies=views["c"], state=state)
        opt.step(1, LR)
        for k, f in flats.items():
            assert (f[~inside[k]] == 0x5A).all()


def test_offsets_beyond_32_bits():
    m = optim()
    n = (1 << 31) + 5000
    p = torch.zeros(n, dtype=torch.bfloat16, device=DEV)
    g = torch.zeros(n, dtype=torch.bfloat16, device=DEV)
    tail = data(6000, torch.bfloat16, 1)
    g[-6000:] = tail
    out = m.GradNorm([g])()
    ref = tail.double().norm()
    assert abs(out[0].double() - ref) <= 32 * U * ref
    zeros = torch.zeros(n, dtype=torch.uint8, device=DEV)
    states = tuple([(z.view(E4M3), torch.zeros(-(-n // 256), device=DEV))] for z in (zeros, zeros.clone()))
    opt = m.AdamW([p], [g], state="8bit", states=states, weight_decay=0.0)
    opt.step(1, LR)
    want = -LR * tail.double() / (tail.double().abs() + EPS)
    got = p[-6000:].double()
    assert ((got - want).abs() <= half_step(want, torch.bfloat16) * 1.001 + want.abs() * 32 * U).all()
    assert not p[:-6000].any()


def test_parameters_and_copies_given_other_memory_are_refused():
    m = optim()
    for which in (0, 1):
        p, g = data(100, torch.float32, 1).requires_grad_(), data(100, torch.float32, 2)
        copy = p.detach().bfloat16()
        opt = m.AdamW([p], [g], copies=[copy])
        opt.step(1, LR)
        t = (p, copy)[which]
        home, held = t.data, [x.clone() for x in (p, opt.exp_avg[0])]
        t.data = t.data.clone()
        with pytest.raises(RuntimeError, match="moved"):
            opt.step(2, LR)
        assert all(torch.equal(a, b) for a, b in zip((p, opt.exp_avg[0]), held))
        t.data = home
        opt.step(2, LR)


def test_one_of_many_parameters_given_other_memory_is_refused():
    """Each step looks at the next one."""
    m = optim()
    p = [data(100, torch.float32, k) for k in range(41)]
    opt = m.AdamW(p, [data(100, torch.float32, 50)] * 41)
    for t in range(1, 24):
        opt.step(t, LR)
    p[33].data = p[33].clone()
    with pytest.raises(RuntimeError, match="moved"):
        for t in range(24, 24 + 41):
            opt.step(t, LR)
