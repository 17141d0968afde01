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


def test_weights_laid_out_in_a_capture_stay_in_its_graph():
    """A layer whose first inference call is captured: an eager call before any replay lays out its own, and a replay after an update uses the new weights."""
    warm, layer = (M.MOTRDecoderLayer(256, 8, 512, 0.0, None, 3, 4).cuda() for _ in range(2))
    shapes, embed, pos, feats, box = layer_case(gen_of(12))
    run = lambda layer: layer(embed, box, feats, shapes, track_query_pos=pos)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.no_grad():
        with torch.cuda.stream(side):
            run(warm)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                out = run(layer)
        torch.cuda.synchronize()
        want = run(layer)
        warm.load_state_dict(layer.state_dict())
        assert torch.equal(want, run(warm))
        for _ in range(2):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want) and torch.equal(run(layer), want)
            for p in layer.parameters():
                p.mul_(0.9)
            want = run(layer)


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


def test_linear_and_norm_offsets_past_32_bits():
    """Operands and results whose last rows lie past 2^31 elements."""
    n, pitch, gen = 70000, 40000, gen_of(4)
    big = torch.empty(n, pitch, device="cuda", dtype=torch.bfloat16)
    big[:, :192] = rand(gen, n, 192, dtype=torch.bfloat16)
    x, dy, w = big[:, :64], big[:, 64:192], rand(gen, 128, 64, dtype=torch.bfloat16)
    y, z = ops.linear_forward(x, w, act=L.ACT_SILU, residual=dy, keep_pre=True)
    yc, zc = ops.linear_forward(x.clone(), w, act=L.ACT_SILU, residual=dy.clone(), keep_pre=True)
    assert torch.equal(y, yc) and torch.equal(z, zc)
    for a, b in zip(ops.linear_backward(dy, x, w, z, L.ACT_SILU), ops.linear_backward(dy.clone(), x.clone(), w, z, L.ACT_SILU)):
        assert torch.equal(a, b)
    assert torch.equal(ops.linear_forward(x[-20:], w), ops.linear_forward(x[-20:].clone(), w))
    y, stat = ops.layer_norm_forward(x, residual=dy[:, :64], stats=True)
    yc, sc = ops.layer_norm_forward(x.clone(), residual=dy[:, :64].clone(), stats=True)
    assert torch.equal(y, yc) and torch.equal(stat, sc)
    for a, b in zip(ops.layer_norm_backward(dy[:, :64], x, None, stat), ops.layer_norm_backward(dy[:, :64].clone(), x.clone(), None, stat)):
        assert torch.equal(a, b)
    del big, x, dy, y, z, yc, zc
    rows = (1 << 21) + 1000                                                    # dense ones of 2^31 elements and more: x, y, z, dy and dx
    x, w, b = rand(gen, rows, 8, dtype=torch.bfloat16), rand(gen, 1024, 8, dtype=torch.bfloat16), rand(gen, 1024, dtype=torch.bfloat16)
    y, z = ops.linear_forward(x, w, b, L.ACT_SILU, keep_pre=True)
    part = torch.cat((torch.arange(500), torch.arange(rows - 1500, rows))).cuda()
    yc, zc = ops.linear_forward(x[part], w, b, L.ACT_SILU, keep_pre=True)
    assert y.numel() > 1 << 31 and torch.equal(y[part], yc) and torch.equal(z[part], zc)
    dx = ops.linear_backward(y, x, w, z, L.ACT_SILU, need=(True, False, False))[0]
    a, b = dx[part].float(), ops.linear_backward(yc, x[part], w, zc, L.ACT_SILU, need=(True, False, False))[0].float()
    # (few rows split their sums: a bf16 step, and 1024 fp32 additions of terms that add up to less than 1100 in size)
    assert bool(((a - b).abs() <= 2.0 ** -7 * b.abs() + 1024 * U32 * 1100).all())
    s, stat = ops.layer_norm_forward(y, stats=True)
    sc, tc = ops.layer_norm_forward(yc, stats=True)
    assert torch.equal(s[part], sc)
    assert torch.equal(ops.layer_norm_backward(z, y, None, stat, need=(True, False, False))[0][part], ops.layer_norm_backward(zc, yc, None, tc, need=(True, False, False))[0])


# ---------------------------------------------------------------------------------------------------- what is not rounded on the way
def forward_tolerance(y, p, v, rel, n, dt):
    """Of o and of o + rest where P enters its product as two operands: P errs by its fp32 statistics (rel, n additions) and by the square of a half step (the
    remainder's own rounding; fp16: no less than half of 2^-24, the reference of the exponentials at most 2^8 below the largest weight); o is rounded once, o + rest by the square of a half step."""
    u, ya = half_step(dt), p @ v.abs()
    wide = dt == torch.float32
    inner = ((0 if wide else u * u) + rel + n * U32) * ya + (tiny(dt) * (p > 0).double() @ v.abs() if dt == torch.float16 else 0)
    return inner + u * y.abs() + tiny(dt), inner + (u if wide else u * u) * y.abs() + tiny(dt)


def tight_reference(q, k, v, do, table, lut, start):
    """One head in 64 bits: y, dtable, and the tolerances of y and of dtable where nothing but a result is rounded to 16 bits."""
    dt, (Lq, D), Lk, far = q.dtype, q.shape, k.shape[0], lut.shape[0] // 2
    qd, kd, vd, g, td = (t.double() for t in (q, k, v, do, table))
    at = lut.to(q.device).long()[(torch.arange(Lk, device=q.device)[None] - torch.arange(Lq, device=q.device)[:, None] - start).clamp(-far, far) + far]
    s = qd @ kd.t() * D ** -0.5 + td[at]
    size = qd.abs() @ kd.abs().t() * D ** -0.5 + td[at].abs()
    p = torch.softmax(s, -1)
    rel = U32 * (2 * (D + 8) * size.amax(-1, keepdim=True) + 2 * s.abs().amax(-1, keepdim=True) + Lk + 16)
    y = p @ vd
    ty, to = forward_tolerance(y, p, vd, rel, Lk, dt)
    dp, dpa = g @ vd.t(), g.abs() @ vd.abs().t()
    delta = (g * y).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    off = (g.abs() * to).sum(-1, keepdim=True) + 2 * U32 * (D + 8) * (g.abs() * y.abs()).sum(-1, keepdim=True)
    te = p * (rel * (dp - delta).abs() + U32 * (D + 8) * dpa + off + 2 * U32 * (dp.abs() + delta.abs())) + (Lk + 64 + Lq) * U32 * ds.abs()
    add = lambda t: torch.zeros(td.shape[0], dtype=torch.float64, device=q.device).index_add_(0, at.reshape(-1), t.reshape(-1))  # noqa: E731
    dtable = add(ds)
    return dict(y=y, dtable=dtable), dict(y=ty, dtable=add(te) * (1 + half_step(dt)) + half_step(dt) * dtable.abs() + tiny(dt))


TIGHT = [(300, 300, 32, 3, 2), (70, 400, 64, 3, 2), (33, 200, 128, 3, 2), (5, 2000, 64, 3, 2), (1, 9, 8, 100, 64)]   # (the last: one bucket, so dtable is 0)


def tight_inputs(gen, Lq, Lk, D, H, dt):
    r = lambda *s: torch.randn(*s, device=gen.device, generator=gen).to(dt)  # noqa: E731
    return r(Lq, H, D), r(Lk, H, D), r(Lk, H, D), r(Lq, H, D), r(16, H)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("Lq,Lk,D,start,H", TIGHT)
def test_attention_rounds_its_results_alone(Lq, Lk, D, start, H, dtype):
    """o and dtable within one rounding of their own: the forward's weights are not rounded to 16 bits, nor is what delta is taken from."""
    dt, lut = DT[dtype], ops.relative_buckets(16, 30)
    ins = tight_inputs(gen_of(Lq + Lk), Lq, Lk, D, H, dt)
    leaves = [t[None].requires_grad_(True) for t in ins[:3]] + [ins[4].requires_grad_(True)]
    y = M.biased_attention(*leaves, lut, q_start=start)
    dtable = torch.autograd.grad(y, leaves[3], ins[3][None])[0]
    for h in range(H):
        want, tol = tight_reference(*(t.detach()[:, h] for t in ins), lut, start)
        for name, got in (("y", y[0, :, h]), ("dtable", dtable[:, h])):
            far = (got.detach().double() - want[name]).abs() / tol[name]
            assert float(far.max()) <= 1.0, (name, h, float(far.max()))


# -------------------------------------------------------------------------------------------------------------- whole layers, closer
@pytest.mark.parametrize("held,dtype,gtol", [(torch.float32, torch.bfloat16, 8.5e-2), (torch.float32, torch.float16, 3e-2), (torch.bfloat16, torch.bfloat16, 8.5e-2),
                                             (torch.float16, torch.float16, 3e-2), (torch.bfloat16, torch.float32, 3e-5), (torch.bfloat16, torch.float16, 3e-2)])
def test_decoder_layer_gradients(held, dtype, gtol, monkeypatch):
    """Every gradient of the layer, parameters held in any type, against 64 bits (relative 2-norms).  The bounds are those that test_gpu_layer_train derives for the
    ReLU's sqrt(2 p), twice that for a parameter, and half a step of its type.  The gradient of a place that is sampled jumps at a cell's edge, and a few of 26880 places lie
    over one for a rounding of their arguments (one that did carried 84 % of the error of embed's gradient here); so the formulas take the places that the layer took,
    which leaves no such step, and the sampling's parameters are held to the same bounds (fp32 activations: ten times those, the offsets' terms over their sums)."""
    from oracle import track_oracle as O
    from test_gpu_layer_train import decoder_case, double_of, fill, off, oracle_layer
    layer = fill(M.MOTRDecoderLayer(256, 8, 512, 0.0, None, 3, 4), 23).to("cuda", held)
    shapes, embed, pos, feats, box, dy = decoder_case(24)
    rnd = lambda t: t.to(dtype).double()  # noqa: E731
    dev = [t.to("cuda", dtype).requires_grad_(True) for t in (embed, pos, feats)]
    places, sample, core = [], M.MSDeformAttnFunction.apply, O.msda_core
    monkeypatch.setattr(M.MSDeformAttnFunction, "apply", lambda v, sizes, first, loc, aw, step: (places.append(loc.detach().cpu().double()), sample(v, sizes, first, loc, aw, step))[1])
    out = layer.forward_train(dev[0], box.cuda(), dev[2], shapes, track_query_pos=dev[1])
    out.backward(dy.to("cuda", dtype))
    monkeypatch.setattr(O, "msda_core", lambda v, sizes, loc, aw: core(v, sizes, loc + (places[0] - loc).detach(), aw))
    sd, by = double_of(layer, "l")
    ref = [rnd(t).requires_grad_(True) for t in (embed, pos, feats)]
    want = oracle_layer(shapes, ref[0], box.double(), ref[2], ref[1], sd)
    want.backward(rnd(dy))
    assert len(places) == 1 and off(out, want) < {torch.float32: 3e-5, torch.float16: 6e-3, torch.bfloat16: 4e-2}[dtype]
    for name, a, b in zip(("embed", "pos", "feats"), dev, ref):
        assert off(a.grad, b.grad) < gtol + half_step(dtype), (name, off(a.grad, b.grad))
    for n, p in layer.named_parameters():
        bound = gtol * (10 if dtype == torch.float32 and ("sampling_offsets" in n or "attention_weights" in n) else 2)
        assert p.grad.dtype == held and off(p.grad, by[n].grad) < bound + half_step(held), (n, off(p.grad, by[n].grad))


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("M", [1, 16, 17, 32, 33])
@pytest.mark.parametrize("K", [2048, 2049, 4096])
def test_linear_either_side_of_the_kernel_for_few_rows(M, K, dtype):
    from test_gpu_layer_ops import check_linear
    dt, gen = DT[dtype], gen_of(M + K)
    N = 200
    check_linear(rand(gen, M, K, dtype=dt), rand(gen, N, K, dtype=dt, scale=K ** -0.5), rand(gen, N, dtype=dt), rand(gen, M, N, dtype=dt), "silu", rand(gen, M, N, dtype=dt))


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="wants two devices")
def test_a_second_device():
    """Each device is asked for its kernels' LDS; the current one stays as it is."""
    for f, args in calls(gen_of(9)):
        runs = []
        for dev in ("cuda:0", "cuda:1"):
            leaves = [a.detach().to(dev).requires_grad_(True) for a in args]
            y = f(*leaves) if leaves[0].dim() == 2 else M.biased_attention(*leaves, ops.relative_buckets(8, 8, device=dev), q_start=0)
            runs.append([t.cpu() for t in (y, *torch.autograd.grad(y, leaves, torch.ones_like(y)))])
            assert torch.cuda.current_device() == 0
        assert all(torch.equal(a, b) for a, b in zip(*runs))


# ------------------------------------------------------------------------------------------------------------------- saved tensors
def test_saved_tensors_that_went_through_hooks():
    """Kept on the host and brought back: the same gradients.  Brought back in another type or size: an error."""
    for f, args in calls(gen_of(10), torch.bfloat16):
        every = [a.clone().requires_grad_(True) for a in args]
        y = f(*every)
        want = torch.autograd.grad(y, every, torch.ones_like(y))
        with torch.autograd.graph.save_on_cpu():
            y = f(*every)
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, every, torch.ones_like(y)), want))
        for change in (lambda t: t.float() if t.dtype == torch.bfloat16 else t, lambda t: t[:1] if t.dtype == torch.bfloat16 else t):
            with torch.autograd.graph.saved_tensors_hooks(lambda t: t, change):
                y = f(*every)
            with pytest.raises(RuntimeError, match="forward's size"):
                torch.autograd.grad(y, every, torch.ones_like(y))


# -------------------------------------------------------------------------------------------------------------------- largest sizes
def test_linear_of_more_rows_than_a_launch_of_small_tiles_counts():
    """2^30 rows and some: 64-row tiles would be 2^32 threads and some, of which a launch runs the rest."""
    n = (1 << 30) + 64
    x, w = torch.full((n, 8), 0.5, device="cuda", dtype=torch.bfloat16), torch.ones(8, 8, device="cuda", dtype=torch.bfloat16)
    x[n // 2], x[-1] = 1.0, 2.0
    y = ops.linear_forward(x, w)
    for i, want in ((0, 4.0), (n // 2, 8.0), (n - 1, 16.0), (64, 4.0), (n - 65, 4.0)):
        assert bool((y[i] == want).all()), i
    assert float(y.view(-1).narrow(0, 0, 1 << 30).amin()) == 4.0
    dx = ops.linear_backward(y, x, w, need=(True, False, False))[0]
    assert bool((dx[-1] == 128.0).all()) and bool((dx[5] == 32.0).all()) and bool((dx[n // 2] == 64.0).all())


def test_attention_of_more_heads_than_a_launch_counts_is_refused():
    q = torch.zeros(1, 1, 8, 8, device="cuda", dtype=torch.bfloat16).expand(1 << 21, 1, 8, 8)
    with pytest.raises(RuntimeError, match="not implemented"):
        ops.attention_forward(q, q, q)
