"""The operators behind a reduction run together as a training program runs
them: with the collectives of virtual ranks on one GPU (ops/emu.py) before and
after, and as one captured step."""
import pytest
import torch

from conftest import need_gpus

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def mods():
    need_gpus(1)
    from scc26_nccl_shim_b200.ops import emu, norm, optim
    return emu, norm, optim


def data(shape, dtype, seed, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, device=DEV, generator=g) * scale).to(dtype)


@pytest.mark.parametrize("ranks", [2, 4, 8])
def test_partial_sums_of_tensor_parallel_ranks(ranks):
    """A row-parallel product's partial sums into the norm, against the
    AllReduce of the same partial sums, the addition and the norm one by one. The
    AllReduce rounds its sum to bf16, the fused form does not."""
    emu, norm, _ = mods()
    rows, inner, hidden = 33, 256, 1024
    parts = [data((rows, inner), torch.bfloat16, r) @ data((inner, hidden), torch.bfloat16, 100 + r, 0.05)
             for r in range(ranks)]
    res, w = data((rows, hidden), torch.bfloat16, 50), 1 + data((hidden,), torch.float32, 51, 0.1)
    got = norm.add_rms_norm(parts, w, res)
    flat = [p.reshape(-1).clone() for p in parts]
    summed = [torch.empty_like(f) for f in flat]
    emu.plan("ar_twoshot", "allreduce", flat, summed)
    two = norm.add_rms_norm(summed[0].view(rows, hidden), w, res)
    exact = sum(p.double() for p in parts)
    # Half a step of bf16 is 2^-8 of a value (finfo(bfloat16).eps / 2): the
    # AllReduce's sum is rounded so once, each h once; fp32 adds ranks terms.
    half = torch.finfo(torch.bfloat16).eps / 2
    h = exact + res.double()
    fold = ranks * 2.0 ** -24 * (sum(p.double().abs() for p in parts) + res.double().abs())
    assert ((got.h.double() - h).abs() <= h.abs() * half * 1.001 + fold).all()
    assert ((got.h.double() - two.h.double()).abs() <=
            exact.abs() * half + 2 * (h.abs() + exact.abs() * half) * half * 1.001 + 2 * fold).all()


@pytest.mark.parametrize("ranks", [2, 4])
@pytest.mark.parametrize("state", ["float32", "8bit"])
def test_sharded_step(ranks, state):
    """ReduceScatter of fp32 gradients, the norm over all shards, AdamW on each
    rank's shard, AllGather of the bf16 copies; against one AdamW that takes the
    ranks' gradients as partial ones. Both fold in rank order in fp32, so the
    32-bit states and parameters agree to the bit."""
    emu, _, optim = mods()
    per = 256 * 40
    n = per * ranks
    grads = [data(n, torch.float32, r) for r in range(ranks)]
    start = data(n, torch.float32, 99)

    # one process that holds everything
    p1, c1 = start.clone(), torch.empty(n, dtype=torch.bfloat16, device=DEV)
    whole = optim.AdamW([p1], [grads], copies=[c1], weight_decay=0.1, state=state)
    whole_norm = optim.GradNorm([grads])

    # a shard per rank
    p2 = [start[r * per:(r + 1) * per].clone() for r in range(ranks)]
    shard = [torch.empty(per, device=DEV) for _ in range(ranks)]
    c2 = [torch.empty(per, dtype=torch.bfloat16, device=DEV) for _ in range(ranks)]
    opts = [optim.AdamW([p2[r]], [shard[r]], copies=[c2[r]], weight_decay=0.1, state=state) for r in range(ranks)]
    norms = [optim.GradNorm([s]) for s in shard]
    full = [torch.empty(n, dtype=torch.bfloat16, device=DEV) for _ in range(ranks)]

    for t in (1, 2):
        out = whole_norm(1.0, scale=1.0 / ranks)
        whole.step(t, 1e-2, scale=out[1])
        emu.plan("rs_pull", "reducescatter", grads, shard)
        parts = torch.stack([f(scale=1.0 / ranks)[0] for f in norms])
        total = parts.square().sum().sqrt()
        # each shard's squares are rounded to fp32 once more
        assert abs(total - out[0]) <= out[0] * ranks * 2.0 ** -23
        for r in range(ranks):
            opts[r].step(t, 1e-2, scale=out[1])  # the same coefficient, so that bits can agree
        emu.plan("ag_push", "allgather", c2, full)
        if state == "float32":
            for f in full:
                assert torch.equal(f, c1)
            assert torch.equal(torch.cat(p2), p1)
            assert torch.equal(torch.cat([o.exp_avg[0] for o in opts]), whole.exp_avg[0])
        elif t == 1:  # the random rounding goes by the element's place, which a shard changes
            assert torch.equal(torch.cat(p2), p1)


def test_captured_training_step():
    """Norm, a linear loss, the norm's gradient, clipping and AdamW in one graph:
    replays give what the same calls give one by one."""
    _, norm, optim = mods()
    rows, hidden = 64, 512
    dy = data((rows, hidden), torch.bfloat16, 7)

    def build():
        x, res = data((rows, hidden), torch.bfloat16, 1), data((rows, hidden), torch.bfloat16, 2)
        w = torch.ones(hidden, device=DEV)
        gw, gx = torch.zeros(hidden, device=DEV), torch.zeros(rows, hidden, dtype=torch.float32, device=DEV)
        opt = optim.AdamW([w, emb := torch.zeros(rows, hidden, device=DEV)], [gw, gx], weight_decay=[0.0, 0.1])
        clip = optim.GradNorm([gw, gx])
        t = torch.ones(1, dtype=torch.int64, device=DEV)
        lr = torch.full((1,), 1e-2, device=DEV)

        def step():
            out = norm.add_rms_norm([x, emb.bfloat16()], w, res)
            dx, dw = norm.add_rms_norm_backward(dy, out.h, w, out.rstd, dy)
            gw.copy_(dw)
            gx.copy_(dx)
            opt.step(t, lr, scale=clip(1.0)[1])
            t.add_(1)
        return step, w, emb

    eager, w1, e1 = build()
    for _ in range(4):
        eager()
    captured, w2, e2 = build()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        captured()
    for _ in range(4):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(w1, w2) and torch.equal(e1, e2)
    assert not torch.equal(w1, torch.ones_like(w1))


def test_two_threads_share_a_handle():
    import threading
    _, _, optim = mods()
    p, g = data(100000, torch.float32, 1), data(100000, torch.float32, 2)
    norm = optim.GradNorm([g])
    want = norm(1.0)
    got = []

    def work():
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(50):
                out = norm(1.0)
            torch.cuda.current_stream().synchronize()
            got.append(out)

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work) for _ in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert all(torch.equal(o, want) for o in got) and len(got) == 2
