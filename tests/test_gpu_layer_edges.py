"""GPU: what the transformer-layer operators must refuse, must keep and must not round away, at the edges of their types, strides and weights.  Tolerances as in
test_gpu_layer_ops: half a step of a type for each rounding, 2^-24 for each fp32 operation of the longest chain."""
import pytest
import torch

from mo_yolo_amd import _lib as L
from mo_yolo_amd import modules as M
from mo_yolo_amd import ops

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
U32 = 2.0 ** -24


def half_step(t):
    return torch.finfo(t).eps / 2


def tiny(t):
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2


def rand(gen, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, device="cuda", generator=gen) * scale).to(dtype)


def gen_of(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


# ---------------------------------------------------------------------------------------------------------------- prepared weights
def layer_case(gen, dtype=torch.float32):
    shapes = [(9, 13), (5, 7), (3, 4)]
    S = sum(h * w for h, w in shapes)
    embed, pos, feats = rand(gen, 2, 30, 256, dtype=dtype), rand(gen, 2, 30, 256, dtype=dtype), rand(gen, 2, S, 256, dtype=dtype)
    return shapes, embed, pos, feats, torch.rand(2, 30, 4, device="cuda", generator=gen) * 0.6 + 0.2


def agree(layer, shapes, embed, pos, feats, box):
    """forward against forward_train: two orders of the same fp32 sums, outputs of unit size."""
    with torch.no_grad():
        a = layer(embed, box, feats, [tuple(s) for s in shapes], track_query_pos=pos)
        b = layer.forward_train(embed, box, feats, shapes, track_query_pos=pos)
    return float((a - b).abs().max()) < 1e-4


def test_forward_sees_what_a_replayed_training_step_changed():
    """A replay changes the weights behind the back of their version counters."""
    layer = M.MOTRDecoderLayer(256, 8, 512, 0.0, None, 3, 4).cuda()
    case = layer_case(gen_of(5))
    shapes, embed, pos, feats, box = case
    sizes = torch.tensor(shapes, dtype=torch.int64, device="cuda")
    dy = rand(gen_of(6), 2, 30, 256)
    params = list(layer.parameters())
    assert agree(layer, *case)                                                 # (prepared weights are there)

    def step():
        grads = torch.autograd.grad(layer.forward_train(embed, box, feats, sizes, track_query_pos=pos), params, dy)
        with torch.no_grad():
            for p, g in zip(params, grads):
                p.sub_(g, alpha=1e-3)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step()
    torch.cuda.synchronize()
    for _ in range(3):
        before = [p.detach().clone() for p in params]
        graph.replay()
        torch.cuda.synchronize()
        assert any(not torch.equal(a, p) for a, p in zip(before, params))
        assert agree(layer, *case)
    layer.requires_grad_(False)                                                # trained: kept again
    assert agree(layer, *case) and agree(layer, *case)


def test_a_captured_forward_follows_the_weights():
    """The inference form of a layer that is being trained, in a graph: each replay uses the weights as they are then, also after eager forwards in between."""
    layer = M.MOTRDecoderLayer(256, 8, 512, 0.0, None, 3, 4).cuda()
    shapes, embed, pos, feats, box = layer_case(gen_of(7))
    run = lambda: layer(embed, box, feats, shapes, track_query_pos=pos)  # noqa: E731
    opt = torch.optim.SGD(layer.parameters(), lr=1e-3)

    def train():
        opt.zero_grad()
        layer.forward_train(embed, box, feats, shapes, track_query_pos=pos).sum().backward()
        opt.step()
    train()
    opt.zero_grad(set_to_none=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.no_grad():
        with torch.cuda.stream(side):
            run()
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                out = run()
    torch.cuda.synchronize()
    for _ in range(3):
        train()
        with torch.no_grad():
            want = run()
            graph.replay()
            torch.cuda.synchronize()
        assert torch.equal(out, want)


# ------------------------------------------------------------------------------------------------------------- what 16 bits cannot hold
@pytest.mark.parametrize("rows", [2, 40, 700])
@pytest.mark.parametrize("n", [64, 37])
def test_linear_keeps_a_finite_argument_with_its_sign(rows, n):
    """fp16: arguments of the activation past 65504 and below half of 2^-24.  The gradients are those of the activation's flat and straight ends and of ReLU's open side."""
    K = 64
    x, dy = torch.zeros(rows, K, device="cuda", dtype=torch.float16), torch.full((rows, n), 0.125, device="cuda", dtype=torch.float16)
    w = torch.zeros(n, K, device="cuda", dtype=torch.float16)
    x[:, 0], x[:, 1:3], w[:, 0], w[:, 1:3] = 60000.0, 100.0, 1.0, 100.0        # z = 60000 + 2e4 = 8e4, or -8e4
    for sign, slope in ((1.0, 1.0), (-1.0, 0.0)):
        leaves = [(x * sign).requires_grad_(True), w.clone().requires_grad_(True)]
        for act, one in (("SILU", slope), ("RELU", slope), ("SIGMOID", 0.0)):
            dx, dw = torch.autograd.grad(M.linear(*leaves, None, getattr(L, "ACT_" + act)), leaves, dy)
            assert torch.isfinite(dx).all() and torch.isfinite(dw[:, 1:]).all(), (act, sign)            # (dw's first column: rows * 60000 / 8, past fp16's range from 9 rows on)
            assert torch.equal(dx[:, 0], torch.full_like(dx[:, 0], one * n / 8)) and torch.equal(dw[:, 1], torch.full_like(dw[:, 1], one * sign * rows * 12.5)), (act, sign)
    x = torch.full((rows, K), 2.0 ** -14, device="cuda", dtype=torch.float16)
    w = torch.zeros(n, K, device="cuda", dtype=torch.float16)
    w[:, 0] = 2.0 ** -12                                                       # z = 2^-26, which fp16 rounds to 0
    for sign in (1.0, -1.0):
        leaves = [(x * sign).requires_grad_(True), w.clone().requires_grad_(True)]
        y, z = ops.linear_forward(leaves[0].detach(), w, None, L.ACT_RELU, None, True)
        dx, _ = torch.autograd.grad(M.linear(*leaves, None, L.ACT_RELU), leaves, dy)
        assert not y.any() and bool((z * sign > 0).all())
        assert torch.equal(dx[:, 0], torch.full_like(dx[:, 0], n * 2.0 ** -15 if sign > 0 else 0.0))
    x = x.clone()
    x[0, 0], x[1, 0] = float("nan"), float("inf")                              # what is not finite stays so
    z = ops.linear_forward(x, w, None, L.ACT_RELU, None, True)[1]
    assert torch.isnan(z[0]).all() and torch.isposinf(z[1]).all()


def test_attention_gradient_of_values_under_small_weights():
    """fp16, 40000 keys: weights of some 2^-15 and less keep all their bits on the way into dV (incoming gradients carry the usual loss scale)."""
    gen = gen_of(8)
    B, Lq, Lk, H, D = 1, 3, 40000, 2, 64
    q, k, v, do = rand(gen, B, Lq, H, D, dtype=torch.float16), rand(gen, B, Lk, H, D, dtype=torch.float16), rand(gen, B, Lk, H, D, dtype=torch.float16), rand(
        gen, B, Lq, H, D, dtype=torch.float16, scale=1024.0)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    dv = torch.autograd.grad(M.biased_attention(*leaves, q_start=0), v, do)[0]
    u = half_step(torch.float16)                                               # (a row's sum: 64 splits of four waves, 40 additions in a lane: chains below 128)
    for h in range(H):
        qd, kd, g = q[0, :, h].detach().double(), k[0, :, h].detach().double(), do[0, :, h].double()
        s = qd @ kd.t() * D ** -0.5
        p = torch.softmax(s, -1)
        rel = U32 * (2 * (D + 8) * (qd.abs() @ kd.abs().t() * D ** -0.5).amax(-1, keepdim=True) + 2 * s.abs().amax(-1, keepdim=True) + 128)
        want = p.t() @ g
        tol = (p * (u + rel + Lq * U32)).t() @ g.abs() * (1 + u) + u * want.abs() + tiny(torch.float16)
        bad = (dv[0, :, h].double() - want).abs() / tol
        assert float(bad.max()) <= 1.0, float(bad.max())


# ------------------------------------------------------------------------------------------------------ other ways to differentiate and to record
def calls(gen, dtype=torch.float32):
    """The three operators as functions of their leaves, and the leaves."""
    x, w, b, W, B = (rand(gen, *s, dtype=dtype) for s in ((6, 64), (64,), (64,), (48, 64), (48,)))
    q, k, v, t, lut = *(rand(gen, 2, 5, 2, 32, dtype=dtype) for _ in range(3)), rand(gen, 8, 2, dtype=dtype), ops.relative_buckets(8, 8)
    return [(lambda x, w, b, r: M.layer_norm(x, w, b, residual=r), (x, w, b, x * 0.5)), (lambda x, w, b, r: M.linear(x, w, b, L.ACT_SILU, r), (x, W, B, x[:, :48] * 0.5)),
            (lambda q, k, v, t: M.biased_attention(q, k, v, t, lut, q_start=0), (q, k, v, t))]


def test_forward_mode_is_refused():
    """A tangent on any argument, whether its primal wants a gradient or not, is an error and never dropped; so is one on the gradient that comes in."""
    from torch.autograd import forward_ad as fw
    for f, args in calls(gen_of(1)):
        for n in range(len(args)):
            for wants in (False, True):
                with fw.dual_level():
                    some = [fw.make_dual(a.clone().requires_grad_(wants), torch.ones_like(a)) if i == n else a for i, a in enumerate(args)]
                    with pytest.raises(RuntimeError, match="forward-mode|jvp"):
                        f(*some)
                    with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode|jvp"):
                        f(*some)
        every = [a.clone().requires_grad_(True) for a in args]
        y = f(*every)
        with fw.dual_level(), pytest.raises(RuntimeError, match="forward-mode|jvp"):
            torch.autograd.grad(y, every, fw.make_dual(torch.ones_like(y), torch.ones_like(y)))


@pytest.mark.filterwarnings("ignore")
def test_recording_a_trace_is_refused():
    """A recorder that keeps torch's operations and not the launches would keep an output that nothing writes."""
    from torch.fx.experimental.proxy_tensor import make_fx
    for f, args in calls(gen_of(2)):
        with pytest.raises(RuntimeError, match="recorded"):
            torch.jit.trace(f, args, check_trace=False)
        with pytest.raises(RuntimeError, match="recorded"):
            make_fx(f)(*args)
        y = f(*args)
        assert torch.isfinite(y).all()


# ------------------------------------------------------------------------------------------------------------------------ strides
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_linear_takes_rows_that_lie_far_apart(dtype):
    """The last token of each sequence (rows over 4 MiB apart) as x, residual, incoming gradient and weight: as from dense copies, bit for bit."""
    dt, gen = DT[dtype], gen_of(3)
    K, N = 256, 192
    step = (1 << 22) // (K * torch.finfo(dt).bits // 8) + 3                    # rows to a sequence
    for rows in (1, 2, 40):
        h = torch.empty(rows, step, K, device="cuda", dtype=dt)
        h[:, -1] = rand(gen, rows, K, dtype=dt)
        x, w, b = h[:, -1], rand(gen, N, K, dtype=dt, scale=K ** -0.5), rand(gen, N, dtype=dt)
        rr, gg = (torch.empty(rows, step + 99, N + 64, device="cuda", dtype=dt) for _ in range(2))
        rr[:, -1], gg[:, -1] = rand(gen, rows, N + 64, dtype=dt), rand(gen, rows, N + 64, dtype=dt)
        r, dy = rr[:, -1, 64:], gg[:, -1, 64:]
        assert rows == 1 or min(x.stride(0), r.stride(0), dy.stride(0)) * x.element_size() > 1 << 22
        runs = []
        for xs, rs, ds in ((x, r, dy), (x.clone(), r.clone(), dy.clone())):
            leaves = [t.detach().requires_grad_(True) for t in (xs, w, b, rs)]
            y = M.linear(leaves[0], *leaves[1:3], L.ACT_SILU, leaves[3])
            runs.append((y, ops.linear_forward(xs, w, b, L.ACT_SILU, rs), *torch.autograd.grad(y, leaves, ds)))
        for a, c in zip(*runs):
            assert torch.isfinite(a).all() and torch.equal(a, c)
        assert torch.equal(ops.linear_forward(w, x), ops.linear_forward(w, x.clone()))                # ... as the weight
        g = rand(gen, N, rows, dtype=dt)
        for a, c in zip(ops.linear_backward(g, w, x, need=(True, True, False)), ops.linear_backward(g, w, x.clone(), need=(True, True, False))):
            assert a is c is None or torch.equal(a, c)
        assert torch.equal(ops.layer_norm_forward(x), ops.layer_norm_forward(x.clone()))


# ------------------------------------------------------------------------------------------------------------------------ keys ahead
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("Lq,Lk,D,start", [(20, 200, 64, 10), (1, 3000, 32, 40), (130, 700, 128, 0), (4, 900, 40, 505), (300, 330, 64, 7), (64, 64, 32, -20)])
def test_keys_ahead_of_every_query_are_not_looked_at(Lq, Lk, D, start, dtype):
    """Causal attention over a cache that is allocated ahead: what stands behind the last query's position (NaN, infinities) changes nothing and gets zeros."""
    gen, dt = gen_of(Lq * 7 + Lk), DT[dtype]
    q, k, v, do = (rand(gen, 2, n, h, D, dtype=dt) for n, h in ((Lq, 4), (Lk, 2), (Lk, 2), (Lq, 4)))
    table, lut = rand(gen, 16, 4, dtype=dt), ops.relative_buckets(16, 30)
    how = dict(causal=True, q_start=start)
    runs = []
    for fill in (0.0, float("nan"), float("inf")):
        k2, v2 = k.clone(), v.clone()
        k2[:, max(0, start + Lq):], v2[:, max(0, start + Lq):] = fill, -fill
        leaves = [t.clone().requires_grad_(True) for t in (q, k2, v2, table)]
        y = M.biased_attention(*leaves, lut, **how)
        with torch.no_grad():
            assert torch.equal(y, M.biased_attention(*leaves, lut, **how))
        runs.append((y, *torch.autograd.grad(y, leaves, do)))
        assert not runs[-1][2][:, max(0, start + Lq):].any() and not runs[-1][3][:, max(0, start + Lq):].any()
    for got in runs[1:]:
        for a, b in zip(got, runs[0]):
            assert torch.isfinite(a).all() and torch.equal(a, b)
