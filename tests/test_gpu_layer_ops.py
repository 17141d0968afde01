"""GPU: the transformer-layer operators (layer norm, linear with its epilogue, attention with a bucketed position bias), forward and backward, against
plain implementations in 64 bits.  Tolerances: half a step of the output's type relative to the value, plus the fp32 rounding of the sums behind it (2^-24 for
each operation of the longest chain, relative to the sum of the terms' magnitudes), plus, where a kernel rounds an intermediate to 16 bits for the
matrix cores, half a step of that relative to the magnitudes it enters with."""
import math

import pytest
import torch

from mo_yolo_amd import _lib as L
from mo_yolo_amd import modules, ops

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
U32 = 2.0 ** -24


def half_step(t):
    return torch.finfo(t).eps / 2


def tiny(t):
    """Half the spacing of the type's subnormal numbers (fp16's show at these magnitudes)."""
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2


def close(got, want, tol, what):
    got, want = got.detach().double(), want.detach()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    bad = ~((got - want).abs() <= tol)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {((got - want).abs() / tol).nan_to_num(9e9).max().item():.2f} of the tolerance"


def rand(gen, *shape, dtype=torch.float32, scale=1.0, shift=0.0):
    return (torch.randn(*shape, device="cuda", generator=gen) * scale + shift).to(dtype)


def gen_of(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def captured(step, warm=2):
    """A graph of step() with its static outputs; warmed up on a side stream first."""
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(warm):
            step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    return g, out


# ------------------------------------------------------------------------------------------------------------------ layer norm
def norm_reference(x, w, b, r, dy, eps):
    """(y, dx, dw, db) in 64 bits and the magnitudes that their fp32 errors scale with."""
    s = x.double() + (0 if r is None else r.double())
    n, c = s.shape
    wd = torch.ones(c, dtype=torch.float64, device=s.device) if w is None else w.double()
    bd = torch.zeros(c, dtype=torch.float64, device=s.device) if b is None else b.double()
    mu = s.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt((s - mu).square().mean(-1, keepdim=True) + eps)
    xh = (s - mu) * rstd
    size = (s.abs() + s.abs().mean(-1, keepdim=True)) * rstd        # what xh's fp32 error is relative to
    y = xh * wd + bd
    g = dy.double() * wd
    dx = rstd * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
    out = dict(y=y, dx=dx, dw=(dy.double() * xh).sum(0), db=dy.double().sum(0))
    ga = g.abs()
    mag = dict(y=size * wd.abs() + bd.abs(), dx=rstd * (ga + ga.mean(-1, keepdim=True) + size * (ga * size).mean(-1, keepdim=True)),
               dw=(dy.double().abs() * size).sum(0), db=dy.double().abs().sum(0))
    return out, mag


def norm_tolerance(out, mag, name, rows, dtype):
    # chains: 16 values in a lane, 6 steps over the wave, 16 waves, then a handful for the formula; dw / db: the rows of a group, the groups, 32 + 32 partials
    chain = 64 + (rows if name in ("dw", "db") else 0)
    return half_step(dtype) * out[name].abs() + tiny(dtype) + 4 * chain * U32 * mag[name]


@pytest.mark.parametrize("wt", ["own", "f32"])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("rows,c", [(1, 1), (1, 8), (3, 7), (300, 256), (5, 257), (70, 100), (17, 1283), (9, 600), (33, 2048), (6, 3000), (3, 5001), (2, 8192)])
def test_layer_norm(rows, c, dtype, residual, wt):
    dt, gen = DT[dtype], gen_of(rows * 7 + c)
    w_t = dt if wt == "own" else torch.float32
    x, r, dy = rand(gen, rows, c, dtype=dt, scale=2.0, shift=0.5), rand(gen, rows, c, dtype=dt) if residual else None, rand(gen, rows, c, dtype=dt)
    w, b = rand(gen, c, dtype=w_t, scale=0.3, shift=1.0), rand(gen, c, dtype=w_t)
    leaves = [t.requires_grad_(True) for t in (x, w, b, r) if t is not None]
    y = modules.layer_norm(x, w, b, 1e-5, residual=r)
    grads = torch.autograd.grad(y, leaves, dy)
    out, mag = norm_reference(x.detach(), w.detach(), b.detach(), None if r is None else r.detach(), dy, 1e-5)
    close(y, out["y"], norm_tolerance(out, mag, "y", rows, dt), "y")
    close(grads[0], out["dx"], norm_tolerance(out, mag, "dx", rows, dt), "dx")
    close(grads[1], out["dw"], norm_tolerance(out, mag, "dw", rows, w_t), "dw")
    close(grads[2], out["db"], norm_tolerance(out, mag, "db", rows, w_t), "db")
    if residual:
        assert torch.equal(grads[3], grads[0])
    with torch.no_grad():
        assert torch.equal(modules.layer_norm(x, w, b, 1e-5, residual=r), y)


def test_layer_norm_widest_rows_and_far_mean():
    gen = gen_of(3)
    for dt, c in ((torch.bfloat16, 16384), (torch.float16, 16383), (torch.float32, 8191)):
        x, dy = rand(gen, 3, c, dtype=dt), rand(gen, 3, c, dtype=dt)
        y, stat = ops.layer_norm_forward(x, stats=True)
        dx, dw, db = ops.layer_norm_backward(dy, x, None, stat)
        out, mag = norm_reference(x, None, None, None, dy, 1e-5)
        for name, got in (("y", y), ("dx", dx), ("dw", dw), ("db", db)):
            close(got, out[name], norm_tolerance(out, mag, name, 3, got.dtype), f"{name} {c}")
    # a mean 4096 times the spread: the variance is taken around the mean, so nothing of it cancels
    x = rand(gen, 40, 256, shift=4096.0)
    out, mag = norm_reference(x, None, None, None, x, 1e-5)
    close(ops.layer_norm_forward(x), out["y"], norm_tolerance(out, mag, "y", 40, torch.float32), "far mean")
    # constant rows: variance 0
    assert torch.equal(ops.layer_norm_forward(torch.full((3, 65), 7.0, device="cuda")), torch.zeros(3, 65, device="cuda"))


def test_layer_norm_strides_alignment_and_shapes():
    gen = gen_of(4)
    wide, other = rand(gen, 50, 700, dtype=torch.bfloat16), rand(gen, 50, 611, dtype=torch.bfloat16)
    x, r = wide[:, 3:260], other[1::2, 7:264].repeat_interleave(2, 0)[:50]
    assert torch.equal(ops.layer_norm_forward(x, residual=r), ops.layer_norm_forward(x.contiguous(), residual=r.contiguous()))
    t = rand(gen, 6, 5, 4, 33)
    assert torch.equal(ops.layer_norm_forward(t), ops.layer_norm_forward(t.reshape(-1, 33)).view(6, 5, 4, 33))
    p = rand(gen, 33, 20).t()                                      # unit stride on the other axis
    assert torch.equal(ops.layer_norm_forward(p), ops.layer_norm_forward(p.contiguous()))
    e = rand(gen, 1, 40).expand(7, 40)
    assert torch.equal(ops.layer_norm_forward(e), ops.layer_norm_forward(e.contiguous()))
    x = rand(gen, 7, 40).requires_grad_(True)
    modules.layer_norm(x).sum().backward()                         # an expanded scalar as dy
    assert float(x.grad.abs().max()) < 1e-5
    w = torch.ones(40, device="cuda", requires_grad=True)
    y = modules.layer_norm(torch.empty(0, 40, device="cuda", requires_grad=True), w)
    assert y.shape == (0, 40) and torch.equal(torch.autograd.grad(y, w, torch.empty_like(y))[0], torch.zeros(40, device="cuda"))


def test_layer_norm_leaves_neighbours_alone_and_repeats():
    gen = gen_of(5)
    x, dy, w = rand(gen, 3001, 97, dtype=torch.float16), rand(gen, 3001, 97, dtype=torch.float16), rand(gen, 97)
    runs = []
    for _ in range(3):
        y, stat = ops.layer_norm_forward(x, w, stats=True)
        runs.append((y, *ops.layer_norm_backward(dy, x, w, stat)))
    for a in runs[1:]:
        assert all(torch.equal(u, v) for u, v in zip(a, runs[0]))
    pad = torch.full((10, 128), 5.0, device="cuda", dtype=torch.float16)      # C ABI: rows of a wider buffer
    L.check(L.lib().moy_layer_norm(x.data_ptr(), 97, None, 0, None, None, 0, 10, 97, 1e-5, pad.data_ptr(), 128, None, None, L.F16, ops._st()))
    assert torch.equal(pad[:, :97], ops.layer_norm_forward(x[:10])) and bool((pad[:, 97:] == 5.0).all())


def test_layer_norm_gradient_against_differences():
    gen = gen_of(6)
    x, w, b, r, dy = (rand(gen, *s) for s in ((4, 50), (50,), (50,), (4, 50), (4, 50)))
    leaves = [t.requires_grad_(True) for t in (x, w, b, r)]
    grads = torch.autograd.grad(modules.layer_norm(x, w, b, residual=r), leaves, dy)
    with torch.no_grad():
        for i, (t, g) in enumerate(zip(leaves, grads)):
            d = rand(gen, *t.shape)
            h = 2.0 ** -6
            f = [float((modules.layer_norm(*[u + s * h * d if u is t else u for u in (x, w, b)], residual=r + s * h * d if t is r else r).double() * dy.double()).sum())
                 for s in (1, -1)]
            want = float((g.double() * d.double()).sum())
            # the difference quotient: h^2 / 6 of a third derivative (order of the values' sizes cubed) and 2^-24 of the sum over h
            assert abs((f[0] - f[1]) / (2 * h) - want) < 5e-2 * max(1.0, abs(want)), i


def test_layer_norm_other_stream_and_graph():
    gen = gen_of(7)
    x, dy = rand(gen, 301, 256, dtype=torch.bfloat16).requires_grad_(True), rand(gen, 301, 256, dtype=torch.bfloat16)
    w, b = (rand(gen, 256).requires_grad_(True) for _ in range(2))
    step = lambda: (lambda y: (y.detach(), *torch.autograd.grad(y, (x, w, b), dy)))(modules.layer_norm(x, w, b))  # noqa: E731
    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert all(torch.equal(u, v) for u, v in zip(got, want))
    g, out = captured(step)
    for k in range(4):
        with torch.no_grad():
            x.copy_(rand(gen, 301, 256, dtype=torch.bfloat16))
            dy.copy_(rand(gen, 301, 256, dtype=torch.bfloat16))
        want = step()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(u, v) for u, v in zip(out, want)), k


def test_gradients_that_are_not_asked_for_and_asked_for_twice():
    gen = gen_of(40)
    x, w, b, r, dy = rand(gen, 60, 64), rand(gen, 64), rand(gen, 64), rand(gen, 60, 64), rand(gen, 60, 64)
    W, B, R = rand(gen, 48, 64), rand(gen, 48), rand(gen, 60, 48)
    q, t, lut = rand(gen, 2, 30, 2, 32), rand(gen, 8, 2), ops.relative_buckets(8, 8)
    calls = [(lambda *a: modules.layer_norm(a[0], a[1], a[2], residual=a[3]), (x, w, b, r)), (lambda *a: modules.linear(a[0], a[1], a[2], L.ACT_SILU, a[3]), (x, W, B, R)),
             (lambda *a: modules.biased_attention(a[0], a[1], a[2], a[3], lut, q_start=0), (q, q.clone(), q.clone(), t)),
             (lambda *a: modules.linear(a[0], a[1], None, L.ACT_NONE, a[2]), (x, W, R)), (lambda *a: modules.layer_norm(a[0], None, a[1]), (x, b))]
    for f, args in calls:
        every = [a.clone().requires_grad_(True) for a in args]
        y = f(*every)
        g = rand(gen, *y.shape)
        want = torch.autograd.grad(y, every, g)
        for only in range(len(args)):                                          # each leaf alone: the same gradient, nothing else computed
            some = [a.clone().requires_grad_(i == only) for i, a in enumerate(args)]
            assert torch.equal(torch.autograd.grad(f(*some), some[only], g)[0], want[only])
        y = f(*every)
        first = torch.autograd.grad(y, every[0], g.clone().requires_grad_(True), create_graph=True)[0]
        assert torch.equal(first.detach(), want[0])
        with pytest.raises(RuntimeError, match="cannot be differentiated again"):
            torch.autograd.grad((first * first).sum() + f(*every).sum(), every[0])
        y = f(*every)
        with torch.no_grad():
            every[0].add_(1.0)                                                 # a saved input that changed: autograd notices
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(y, every[0], g)


# ------------------------------------------------------------------------------------------------------------------- attention
def attention_reference(q, k, v, table=None, lut=None, causal=False, q_start=None, k_len=None, attn_mask=None, scale=None, dout=None):
    """({y, dq, dk, dv, dtable} in 64 bits, their tolerances)."""
    dt = q.dtype
    B, Lq, H, D = q.shape
    Lk, Hk = k.shape[1:3]
    share, sc = H // Hk, D ** -0.5 if scale is None else scale
    hs16 = half_step(dt) if dt != torch.float32 else 0.0                       # P and dS as matrix operands
    under = tiny(dt) if dt == torch.float16 else 0.0
    z = lambda *s: torch.zeros(*s, dtype=torch.float64, device=q.device)  # noqa: E731
    out = dict(y=z(B, Lq, H, D), dq=z(B, Lq, H, D), dk=z(B, Lk, Hk, D), dv=z(B, Lk, Hk, D))
    tol = {n: torch.zeros_like(t) for n, t in out.items()}
    mag = {n: torch.zeros_like(t) for n, t in out.items()}
    if table is not None:
        out["dtable"], tol["dtable"], mag["dtable"] = (z(*table.shape) for _ in range(3))
    for b in range(B):
        n = Lk if k_len is None else min(max(int(k_len[b]), 0), Lk)
        start = (n - Lq) if q_start is None else q_start
        if n == 0:
            continue
        i, j = torch.arange(Lq, device=q.device)[:, None] + start, torch.arange(n, device=q.device)[None]
        for h in range(H):
            hk = h // share
            qd, kd, vd = q[b, :, h].double(), k[b, :n, hk].double(), v[b, :n, hk].double()
            hidden = (j > i) if causal else torch.zeros(Lq, n, dtype=torch.bool, device=q.device)
            if attn_mask is not None:
                m = attn_mask if attn_mask.dim() == 2 else attn_mask.expand(B, H, Lq, Lk)[b, h]
                hidden = hidden | (m != 0)[:, :n]
                if m.shape[0] == 1 or (m.dim() == 2 and m.stride(0) == 0):
                    kd, vd = kd.masked_fill((m[:1, :n] != 0).t(), 0), vd.masked_fill((m[:1, :n] != 0).t(), 0)
            s, sm = qd @ kd.t() * sc, qd.abs() @ kd.abs().t() * abs(sc)
            if table is not None:
                far = lut.shape[0] // 2
                at = lut.long()[(j - i).clamp(-far, far) + far].clamp(max=table.shape[0] - 1)
                s, sm = s + table.double()[at, h], sm + table.double()[at, h].abs()
            s = s.masked_fill(hidden, float("-inf"))
            none = hidden.all(-1, keepdim=True)
            p = torch.softmax(s.masked_fill(none, 0.0), -1).masked_fill(hidden | none, 0.0)
            # relative error of a probability: its score's (D products, scale, bias in 32 bits), the largest one's of the row through maximum and sum, the exponentials
            rel = U32 * (2 * (D + 8) * sm.masked_fill(hidden, 0).amax(-1, keepdim=True) + 2 * s.masked_fill(hidden, 0).abs().amax(-1, keepdim=True) + n + 16)
            y, ya, va = p @ vd, p @ vd.abs(), (~hidden).double() @ vd.abs()
            out["y"][b, :, h] = y
            ty = half_step(dt) * y.abs() + tiny(dt) + (hs16 + rel + n * U32) * ya + under * va
            tol["y"][b, :, h] = ty
            if dout is None:
                continue
            do = dout[b, :, h].double()
            dp, dpa = do @ vd.t(), do.abs() @ vd.abs().t()
            delta = (do * y).sum(-1, keepdim=True)
            ds = p * (dp - delta)
            off = (do.abs() * ty).sum(-1, keepdim=True) + U32 * (D + 8) * (do.abs() * y.abs()).sum(-1, keepdim=True)
            te = p * (rel * (dp - delta).abs() + U32 * (D + 8) * dpa + off + 2 * U32 * (dp.abs() + delta.abs()))     # of dS in 32 bits
            th = te + hs16 * ds.abs() + under                                                                          # ... rounded for the products
            out["dq"][b, :, h] = sc * ds @ kd
            tol["dq"][b, :, h] = abs(sc) * ((th + n * U32 * ds.abs()) @ kd.abs())
            out["dk"][b, :n, hk] += sc * ds.t() @ qd
            tol["dk"][b, :n, hk] += abs(sc) * ((th + Lq * share * U32 * ds.abs()).t() @ qd.abs())
            out["dv"][b, :n, hk] += p.t() @ do
            tol["dv"][b, :n, hk] += (p * (rel + hs16 + Lq * share * U32) + under).t() @ do.abs()
            if table is not None:
                out["dtable"][:, h].index_add_(0, at.reshape(-1), ds.reshape(-1))
                tol["dtable"][:, h].index_add_(0, at.reshape(-1), te.reshape(-1) + (Lk + 64 + B * Lq) * U32 * ds.abs().reshape(-1))
    for n in out:
        if n != "y":
            tol[n] = tol[n] * (1 + half_step(dt)) + half_step(dt) * out[n].abs() + tiny(dt)
    return out, tol


def attention_inputs(seed, B, Lq, Lk, H, Hk, D, dtype, buckets=None, far=None, both=True, grad=True):
    dt, gen = DT[dtype], gen_of(seed)
    q, k, v, dout = rand(gen, B, Lq, H, D, dtype=dt), rand(gen, B, Lk, Hk, D, dtype=dt), rand(gen, B, Lk, Hk, D, dtype=dt), rand(gen, B, Lq, H, D, dtype=dt)
    table = lut = None
    if buckets:
        table, lut = rand(gen, buckets, H, dtype=dt), ops.relative_buckets(buckets, far, both)
    for t in (q, k, v, table):
        if t is not None and grad:
            t.requires_grad_(True)
    return q, k, v, table, lut, dout


def check_attention(q, k, v, table, lut, dout, **how):
    """Forward (alone and with gradients) and backward against the reference."""
    leaves = [t for t in (q, k, v, table) if t is not None]
    y = modules.biased_attention(q, k, v, table, lut, **how)
    grads = torch.autograd.grad(y, leaves, dout)
    with torch.no_grad():
        assert torch.equal(modules.biased_attention(q, k, v, table, lut, **how).nan_to_num(7.0), y.nan_to_num(7.0))
    d = lambda t: None if t is None else t.detach()  # noqa: E731
    out, tol = attention_reference(d(q), d(k), d(v), d(table), lut, dout=dout, **how)
    for name, got in zip(("y", "dq", "dk", "dv", "dtable"), (y, *grads)):
        close(got, out[name], tol[name], name)


KLEN = {"none": None, "ragged": [0, 3, 1 << 20, -4]}
ATTENTION = [
    # B, Lq, Lk, H, Hk, D, buckets, far, both, causal, q_start, k_len, mask
    (1, 1, 1, 1, 1, 8, 8, 8, True, False, None, None, None),
    (2, 5, 7, 2, 1, 40, 8, 6, True, False, 0, None, None),
    (1, 64, 64, 2, 2, 32, 32, 128, True, False, 0, None, None),
    (2, 77, 130, 4, 2, 64, 16, 40, True, False, 0, [130, 41], None),
    (1, 300, 300, 2, 2, 32, 32, 128, True, False, 0, None, "square"),
    (1, 129, 257, 3, 3, 128, 64, 200, False, True, None, None, None),
    (4, 33, 65, 1, 1, 72, 4, 2, True, True, 0, [0, 3, 1 << 20, -4], None),
    (3, 2, 300, 8, 2, 64, 32, 20, False, True, None, [300, 1, 0], None),
    (2, 1, 5000, 4, 1, 128, 32, 128, False, False, None, [5000, 4097], None),
    (1, 3, 2111, 6, 6, 16, None, None, True, True, None, None, None),
    (1, 40, 2050, 3, 1, 32, 32, 900, True, False, 100, None, "rows"),
    (2, 70, 90, 2, 2, 24, 16, 1024, True, True, -20, None, "full"),
    (2, 130, 200, 4, 4, 64, None, None, True, False, 0, None, "keys"),
    (2, 9, 90, 4, 2, 96, 16, 30, True, False, 50, [80, 90], "keys"),
    (1, 500, 190, 2, 1, 64, 32, 64, True, True, -150, None, None),
]


def attention_mask(kind, seed, B, H, Lq, Lk):
    if kind is None:
        return None
    gen = gen_of(seed + 1)
    shape = {"square": (Lq, Lk), "rows": (1, H, Lq, Lk), "full": (B, H, Lq, Lk), "keys": (B, 1, 1, Lk)}[kind]
    m = torch.rand(*shape, device="cuda", generator=gen) < 0.4
    if kind != "keys":
        m[..., Lq // 2, :] = True                                             # a query that sees nothing
        m[..., 0, :] = False
    return m


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("shape", ATTENTION, ids=lambda s: "-".join(map(str, s)))
def test_attention(shape, dtype):
    B, Lq, Lk, H, Hk, D, buckets, far, both, causal, q_start, k_len, mask = shape
    seed = Lq * 1000 + Lk
    q, k, v, table, lut, dout = attention_inputs(seed, B, Lq, Lk, H, Hk, D, dtype, buckets, far, both)
    kl = None if k_len is None else torch.tensor(k_len, dtype=torch.int32, device="cuda")
    check_attention(q, k, v, table, lut, dout, causal=causal, q_start=q_start, k_len=kl, attn_mask=attention_mask(mask, seed, B, H, Lq, Lk))


@pytest.mark.parametrize("dtype", list(DT))
def test_attention_of_one_key_has_no_gradient_in_q_k_table(dtype):
    """All the weight on one key: dS is exactly zero, so are dq, dk and dtable; y is the value and dv the sum of dout."""
    q, k, v, table, lut, dout = attention_inputs(1, 3, 37, 9, 4, 2, 64, dtype, 8, 8)
    how = dict(q_start=0, k_len=torch.ones(3, dtype=torch.int32, device="cuda"))
    y = modules.biased_attention(q, k, v, table, lut, **how)
    dq, dk, dv, dt = torch.autograd.grad(y, (q, k, v, table), dout)
    assert not dq.any() and not dk.any() and not dt.any()
    assert torch.equal(y, v[:, :1].repeat_interleave(2, 2).expand(-1, 37, -1, -1))
    out, tol = attention_reference(q.detach(), k.detach(), v.detach(), table.detach(), lut, dout=dout, **how)
    close(dv, out["dv"], tol["dv"], "dv")


def test_attention_ignores_what_stands_behind_the_keys():
    """NaN and infinities in rows past k_len, and in rows that a key mask hides, change nothing; their gradients are zeros."""
    for lq, lk, d, dtype in ((70, 200, 64, "bf16"), (2, 2000, 32, "f32"), (1, 2500, 128, "f16")):
        q, k, v, table, lut, dout = attention_inputs(5, 2, lq, lk, 4, 2, d, dtype, 32, 100)
        n = [lk - 77, lk - 130]
        mask = torch.zeros(2, 1, 1, lk, dtype=torch.bool, device="cuda")
        mask[0, ..., 5:40] = True
        how = dict(q_start=0, k_len=torch.tensor(n, dtype=torch.int32, device="cuda"), attn_mask=mask)
        want = modules.biased_attention(q, k, v, table, lut, **how)
        gw = torch.autograd.grad(want, (q, k, v, table), dout)
        with torch.no_grad():
            for t in (k, v):
                t[0, n[0]:], t[1, n[1]:], t[0, 5:20], t[0, 20:40] = float("nan"), float("inf"), float("nan"), float("-inf")
        got = modules.biased_attention(q, k, v, table, lut, **how)
        gg = torch.autograd.grad(got, (q, k, v, table), dout)
        assert torch.isfinite(want).all() and torch.equal(got, want)
        for a, b in zip(gg, gw):
            assert torch.isfinite(a).all() and torch.equal(a, b)
        assert not gg[1][0, n[0]:].any() and not gg[2][1, n[1]:].any() and not gg[2][0, 5:40].any()


def test_attention_lowest_scores_and_nan():
    """Scores at the type's ends: a table entry of the lowest value leaves its keys out; NaN in a key that counts shows in every query."""
    q, k, v, table, lut, dout = attention_inputs(6, 1, 50, 50, 2, 2, 32, "bf16", 8, 8, False, grad=False)
    table[7] = torch.finfo(torch.bfloat16).min                                # the bucket of every distance of 7 and more
    how = dict(causal=True, q_start=0)
    far = torch.arange(50, device="cuda")[None] - torch.arange(50, device="cuda")[:, None] <= -8
    got, want = ops.attention_forward(q, k, v, table, lut, **how), ops.attention_forward(q, k, v, table, lut, attn_mask=far, **how)
    assert torch.equal(got, want)
    k[0, 3, 0, 0] = float("nan")
    y = ops.attention_forward(q, k, v, q_start=0)
    assert torch.isnan(y[0, :, 0]).all() and torch.isfinite(y[0, :, 1]).all()


def test_attention_strides_and_layouts():
    gen = gen_of(8)
    B, L, H, D = 2, 150, 4, 64
    qkv = rand(gen, B, L, 3, H, D, dtype=torch.bfloat16)
    q, k, v = qkv.unbind(2)                                                   # one packed buffer
    want = ops.attention_forward(q.contiguous(), k.contiguous(), v.contiguous(), causal=True)
    assert torch.equal(ops.attention_forward(q, k, v, causal=True), want)
    heads_first = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
    assert torch.equal(ops.attention_forward(*heads_first, causal=True), want)
    odd = torch.empty(B, L, H, D + 3, device="cuda", dtype=torch.bfloat16)    # rows off the 16-byte steps: copied
    odd[..., 3:] = q
    assert torch.equal(ops.attention_forward(odd[..., 3:], k, v, causal=True), want)
    one = k[:, :, :1].expand(B, L, H, D)                                      # one key head, expanded (stride 0)
    assert torch.equal(ops.attention_forward(q, one, v), ops.attention_forward(q, one.contiguous(), v))
    m = torch.rand(L, L, device="cuda", generator=gen) < 0.3
    assert torch.equal(ops.attention_forward(q, k, v, attn_mask=m.t()), ops.attention_forward(q, k, v, attn_mask=m.t().contiguous()))
    assert torch.equal(ops.attention_forward(q, k, v, attn_mask=m), ops.attention_forward(q, k, v, attn_mask=m[None, None].expand(B, H, L, L).contiguous()))
    x = q.contiguous().requires_grad_(True)
    y = modules.biased_attention(x, k, v)
    a = torch.autograd.grad(y, x, torch.ones(1, 1, 1, 1, device="cuda", dtype=torch.bfloat16).expand_as(y), retain_graph=True)[0]
    assert torch.equal(a, torch.autograd.grad(y, x, torch.ones_like(y))[0])
    e = ops.attention_forward(q[:, :0], k, v)
    assert e.shape == (B, 0, H, D)
    assert not ops.attention_forward(q, k[:, :0], v[:, :0]).any()
    x, kk = q.contiguous().requires_grad_(True), k[:, :0].contiguous().requires_grad_(True)
    gx, gk = torch.autograd.grad(modules.biased_attention(x, kk, v[:, :0]), (x, kk), torch.ones_like(x))
    assert not gx.any() and gk.shape == kk.shape


def test_attention_offsets_past_32_bits():
    """A cache whose rows stand 40000 elements apart: the last ones lie past 2^31 elements."""
    n, pitch = 70000, 40000
    big = torch.empty(n, pitch, device="cuda", dtype=torch.bfloat16)
    gen = gen_of(9)
    big[:, :128] = rand(gen, n, 128, dtype=torch.bfloat16)
    k, v = big[None, :, None, :64], big[None, :, None, 64:128]
    q = rand(gen, 1, 1, 1, 64, dtype=torch.bfloat16)
    assert torch.equal(ops.attention_forward(q, k, v), ops.attention_forward(q, k.contiguous(), v.contiguous()))
    q = rand(gen, 1, 128 * 64, 1, 64, dtype=torch.bfloat16)                   # ... and through the kernel for many queries
    assert torch.equal(ops.attention_forward(q, k, v), ops.attention_forward(q, k.contiguous(), v.contiguous()))


def test_attention_gradient_against_differences():
    q, k, v, table, lut, dout = attention_inputs(10, 2, 20, 33, 4, 2, 16, "f32", 16, 20)
    how = dict(q_start=4, attn_mask=attention_mask("square", 3, 2, 4, 20, 33))
    leaves = (q, k, v, table)
    grads = torch.autograd.grad(modules.biased_attention(*leaves, lut, **how), leaves, dout)
    gen, h = gen_of(11), 2.0 ** -6
    with torch.no_grad():
        for n, (t, g) in enumerate(zip(leaves, grads)):
            d = rand(gen, *t.shape)
            f = [float((modules.biased_attention(*[u + s * h * d if u is t else u for u in leaves], lut, **how).double() * dout.double()).sum()) for s in (1, -1)]
            want = float((g.double() * d.double()).sum())
            size = float((g.double().abs() * d.double().abs()).sum())
            assert abs((f[0] - f[1]) / (2 * h) - want) < 1e-2 * size, n       # h^2 / 6 = 4e-5 of the third derivative along d


def test_attention_repeats_on_any_stream_and_in_graphs():
    q, k, v, table, lut, dout = attention_inputs(12, 2, 200, 333, 4, 2, 64, "bf16", 32, 64)
    k_len = torch.tensor([333, 100], dtype=torch.int32, device="cuda")
    step = lambda: (lambda y: (y.detach(), *torch.autograd.grad(y, (q, k, v, table), dout)))(modules.biased_attention(q, k, v, table, lut, q_start=0, k_len=k_len))  # noqa: E731
    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    with torch.no_grad():
        one = lambda: ops.attention_forward(q[:, :1], k, v, table, lut, k_len=k_len)  # noqa: E731
        g1, o1 = captured(one)
    g2, o2 = captured(step)
    gen = gen_of(13)
    for n in ((333, 100), (5, 0), (1, 333), (200, 201)):                      # the graphs read the lengths anew
        with torch.no_grad():
            k_len.copy_(torch.tensor(n, dtype=torch.int32))
            q.copy_(rand(gen, *q.shape, dtype=torch.bfloat16))
        want, w1 = step(), one().detach()
        g2.replay()
        g1.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(o2, want)) and torch.equal(o1, w1), n


# ---------------------------------------------------------------------------------------------------------------------- linear
ACT = {"none": L.ACT_NONE, "silu": L.ACT_SILU, "relu": L.ACT_RELU, "sigmoid": L.ACT_SIGMOID}


def linear_reference(x, w, b, r, act, dy):
    """({y, dx, dw, db} in 64 bits, tolerances)."""
    dt, K = x.dtype, x.shape[1]
    M, N = x.shape[0], w.shape[0]
    xd, wd, g = x.double(), w.double(), dy.double()
    z, zm = xd @ wd.t(), xd.abs() @ wd.abs().t()
    if b is not None:
        z, zm = z + b.double(), zm + b.double().abs()
    ez = (K + 8) * U32 * zm                                                   # of z in 32 bits
    s = torch.sigmoid(z)
    f, d1, d2 = {"none": (z, torch.ones_like(z), 0 * z), "relu": (z.clamp(min=0), (z > 0).double(), 0 * z), "sigmoid": (s, s * (1 - s), s * (1 - s)),
                 "silu": (z * s, s * (1 + z * (1 - s)), torch.full_like(z, 0.5))}[act]
    slope = 1.1                                                               # bounds every |act'|
    y = f + (0 if r is None else r.double())
    ty = half_step(dt) * y.abs() + tiny(dt) + slope * ez + 16 * U32 * (f.abs() + y.abs() + (s * (1 + z.abs()) if act in ("silu", "sigmoid") else 0))
    rz = half_step(dt) * z.abs() + tiny(dt) if dt != torch.float32 else 0     # the z that is kept
    dz = g * d1
    flip = ((z.abs() <= ez).double() * g.abs()) if act == "relu" else 0       # the sign of a z near 0 may come out either way
    tz = g.abs() * d2.abs().clamp(max=0.5) * (ez + rz) + 32 * U32 * g.abs() + flip
    tzr = tz + (half_step(dt) * dz.abs() + tiny(dt) if dt != torch.float32 and act != "none" else 0)
    dx, dw, db = dz @ wd, dz.t() @ xd, dz.sum(0)
    e = 1 + half_step(dt)
    tol = dict(y=ty, dx=e * (tzr @ wd.abs() + (N + 32) * U32 * (dz.abs() @ wd.abs())) + half_step(dt) * dx.abs() + tiny(dt),
               dw=e * (tzr.t() @ xd.abs() + (M + 32) * U32 * (dz.abs().t() @ xd.abs())) + half_step(dt) * dw.abs() + tiny(dt),
               db=tz.sum(0) + (M + 600) * U32 * dz.abs().sum(0))
    return dict(y=y, dx=dx, dw=dw, db=db), tol


def check_linear(x, w, b, r, act, dy):
    leaves = [t for t in (x, w, b, r) if t is not None]
    for t in leaves:
        t.requires_grad_(True)
    y = modules.linear(x, w, b, ACT[act], r)
    grads = dict(zip([n for n, t in zip(("dx", "dw", "db", "dr"), (x, w, b, r)) if t is not None], torch.autograd.grad(y, leaves, dy)))
    with torch.no_grad():
        assert torch.equal(modules.linear(x, w, b, ACT[act], r), y)
    d = lambda t: None if t is None else t.detach()  # noqa: E731
    out, tol = linear_reference(d(x), d(w), d(b), d(r), act, dy)
    if b is not None:
        tol["db"] = tol["db"] * (1 + half_step(b.dtype)) + half_step(b.dtype) * out["db"].abs() + tiny(b.dtype)
    close(y, out["y"], tol["y"], "y")
    for n in ("dx", "dw", "db"):
        if n in grads:
            close(grads[n], out[n], tol[n], n)
    if r is not None:
        assert torch.equal(grads["dr"], dy)


LINEAR = [
    # M, N, K, act, bias, residual
    (1, 1, 1, "none", None, False), (1, 4096, 1024, "silu", "own", False), (3, 70, 33, "relu", "f32", True), (16, 256, 256, "sigmoid", "own", True),
    (17, 130, 520, "none", "own", True), (32, 48, 2050, "silu", "f32", False), (33, 64, 64, "relu", "own", False), (300, 1024, 256, "relu", "f32", True),
    (300, 256, 1024, "none", "own", True), (127, 129, 131, "silu", "own", True), (1000, 8, 8, "sigmoid", None, False), (4096, 24, 40, "silu", "own", False),
    (64, 1000, 5000, "none", None, False), (1803, 770, 514, "sigmoid", "own", True), (2500, 640, 128, "silu", "own", False), (70, 3, 4100, "none", "f32", True),
]


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("shape", LINEAR, ids=lambda s: "-".join(map(str, s)))
def test_linear(shape, dtype):
    M, N, K, act, bias, residual = shape
    dt, gen = DT[dtype], gen_of(M * 31 + N)
    x, w, dy = rand(gen, M, K, dtype=dt), rand(gen, N, K, dtype=dt, scale=K ** -0.5), rand(gen, M, N, dtype=dt)
    b = None if bias is None else rand(gen, N, dtype=dt if bias == "own" else torch.float32)
    check_linear(x, w, b, rand(gen, M, N, dtype=dt) if residual else None, act, dy)


@pytest.mark.parametrize("dtype", list(DT))
def test_linear_large_tiles(dtype):
    """Enough tiles for the 256-row blocks in every product, with edges that are no multiple of a tile."""
    dt, gen = DT[dtype], gen_of(77)
    M, N, K = 4000, 3600, 3500 if dtype == "f32" else 3496
    x, w, dy = rand(gen, M, K, dtype=dt), rand(gen, N, K, dtype=dt, scale=K ** -0.5), rand(gen, M, N, dtype=dt)
    check_linear(x, w, rand(gen, N, dtype=dt), rand(gen, M, N, dtype=dt), "silu", dy)


def test_linear_exact_on_small_whole_numbers():
    """Products of small integers are exact in every type and order: a wrong element, a tile too much or too little shows."""
    for dtype, dt in DT.items():
        for M, N, K in ((5, 37, 72), (200, 200, 200), (513, 257, 96), (1100, 700, 64), (3000, 2000, 40), (2048, 4096, 72)):
            gen = gen_of(M)
            ints = lambda *s: torch.randint(-1, 2, s, device="cuda", generator=gen).to(dt)  # noqa: E731
            x, w, dy = ints(M, K).requires_grad_(True), ints(N, K).requires_grad_(True), ints(M, N) * (torch.rand(M, N, device="cuda", generator=gen) < 0.04)
            y = modules.linear(x, w)
            dx, dw = torch.autograd.grad(y, (x, w), dy)
            with torch.no_grad():
                for got, want in ((y, x.float() @ w.float().t()), (dx, dy.float() @ w.float()), (dw, dy.float().t() @ x.float())):
                    assert float(want.abs().max()) <= 256 and torch.equal(got.float(), want), (dtype, M, N, K)


def test_linear_strides_alignment_and_shapes():
    gen = gen_of(21)
    for dt in (torch.bfloat16, torch.float32):
        wide = rand(gen, 90, 600, dtype=dt)
        w, b = rand(gen, 64, 256, dtype=dt), rand(gen, 64, dtype=dt)
        for x in (wide[:, 8:264], wide[:, 3:259], wide[::2, 16:272], wide.t()[:256].t()):     # 16-byte steps, odd ones, every other row, the other axis
            r = wide[:x.shape[0], 5:69]
            assert torch.equal(ops.linear_forward(x, w, b, L.ACT_SILU, r), ops.linear_forward(x.contiguous(), w, b, L.ACT_SILU, r.contiguous()))
        wt = rand(gen, 256, 64, dtype=dt).t()
        assert torch.equal(ops.linear_forward(wide[:, :256], wt), ops.linear_forward(wide[:, :256], wt.contiguous()))
        x = rand(gen, 2, 5, 9, 256, dtype=dt)
        assert torch.equal(ops.linear_forward(x, w, b), ops.linear_forward(x.view(90, 256), w, b).view(2, 5, 9, 64))
        x = rand(gen, 90, 256, dtype=dt).requires_grad_(True)
        y = modules.linear(x, w, b, L.ACT_RELU)
        e = torch.autograd.grad(y, x, torch.ones(1, 1, device="cuda", dtype=dt).expand_as(y), retain_graph=True)[0]
        assert torch.equal(e, torch.autograd.grad(y, x, torch.ones_like(y))[0])
    w = rand(gen, 4, 8).requires_grad_(True)
    y = modules.linear(torch.empty(0, 8, device="cuda"), w)
    assert y.shape == (0, 4) and not torch.autograd.grad(y, w, torch.empty_like(y))[0].any()
    # C ABI: y in a wider buffer, its other columns left alone
    x, w = rand(gen, 70, 64, dtype=torch.bfloat16), rand(gen, 30, 64, dtype=torch.bfloat16)
    buf = torch.full((70, 48), 3.0, device="cuda", dtype=torch.bfloat16)
    a = L.LinearArgs()
    a.x, a.ldx, a.w, a.ldw, a.M, a.N, a.K, a.dtype, a.y, a.ldy = x.data_ptr(), 64, w.data_ptr(), 64, 70, 30, 64, L.BF16, buf.data_ptr(), 48
    assert L.lib().moy_linear_ws(a) == 0
    L.check(L.lib().moy_linear(a, ops._st()))
    assert torch.equal(buf[:, :30], ops.linear_forward(x, w)) and bool((buf[:, 30:] == 3.0).all())


def test_linear_gradient_against_differences():
    gen = gen_of(22)
    x, w, b, r, dy = rand(gen, 40, 50), rand(gen, 30, 50, scale=0.14), rand(gen, 30), rand(gen, 40, 30), rand(gen, 40, 30)
    for act in ("none", "silu", "sigmoid"):
        leaves = [t.requires_grad_(True) for t in (x, w, b, r)]
        grads = torch.autograd.grad(modules.linear(x, w, b, ACT[act], r), leaves, dy)
        with torch.no_grad():
            for t, g in zip(leaves, grads):
                d, h = rand(gen, *t.shape), 2.0 ** -6
                f = [float((modules.linear(*[u + s * h * d if u is t else u for u in (x, w, b)], ACT[act], r + s * h * d if t is r else r).double() * dy.double()).sum())
                     for s in (1, -1)]
                want, size = float((g.double() * d.double()).sum()), float((g.double().abs() * d.double().abs()).sum())
                assert abs((f[0] - f[1]) / (2 * h) - want) < 1e-2 * size, act


def test_linear_repeats_on_any_stream_and_in_graphs():
    gen = gen_of(23)
    x, w, b, r = (rand(gen, *s, dtype=torch.float16).requires_grad_(True) for s in ((700, 256), (1024, 256), (1024,), (700, 1024)))
    dy = rand(gen, 700, 1024, dtype=torch.float16)
    step = lambda: (lambda y: (y.detach(), *torch.autograd.grad(y, (x, w, b, r), dy)))(modules.linear(x, w, b, L.ACT_SILU, r))  # noqa: E731
    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(got, want))
    g, out = captured(step)
    for _ in range(4):
        with torch.no_grad():
            x.copy_(rand(gen, 700, 256, dtype=torch.float16))
            dy.copy_(rand(gen, 700, 1024, dtype=torch.float16))
        want = step()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(out, want))


@pytest.mark.parametrize("Lq,Lk,dtype", [(3, 1, "f32"), (70, 5, "bf16"), (33, 15, "f16"), (130, 16, "bf16"), (65, 17, "f32"), (64, 63, "f16"), (200, 130, "bf16"), (5, 600, "f16"),
                                         (129, 331, "f32")])
@pytest.mark.parametrize("D", [32, 64, 128])
def test_attention_masks_of_any_bytes_and_strides(Lq, Lk, dtype, D):
    """A mask by batch, head and query as bytes of any value but 0, at odd addresses and row strides, hides what the dense boolean one does: bit for bit."""
    B, H, Hk = 2, 4, 2
    q, k, v, table, lut, dout = attention_inputs(Lq * 7 + Lk, B, Lq, Lk, H, Hk, D, dtype, 8, 20)
    g = torch.Generator().manual_seed(Lq + Lk)
    hidden = torch.rand(B, H, Lq, Lk, generator=g) < 0.4
    hidden[0, 1, Lq // 2] = True                                               # a row without a key
    wide = torch.zeros(B, H, Lq, Lk + 9, dtype=torch.uint8)
    wide[..., 3:3 + Lk] = torch.where(hidden, torch.randint(1, 256, hidden.shape, generator=g), torch.zeros(1, dtype=torch.int64)).to(torch.uint8)
    wide[..., :3] = wide[..., 3 + Lk:] = 255                                   # what stands beside the rows is not looked at
    odd = wide.cuda()[..., 3:3 + Lk]
    assert odd.stride(2) == Lk + 9 and odd.storage_offset() == 3
    leaves = (q, k, v, table)
    runs = []
    for m in (hidden.cuda(), odd):
        y = modules.biased_attention(q, k, v, table, lut, q_start=0, attn_mask=m)
        runs.append((y, *torch.autograd.grad(y, leaves, dout)))
    for a, b in zip(*runs):
        assert torch.isfinite(a).all() and torch.equal(a, b)
    assert not runs[0][0][0, Lq // 2, 1].any() and not runs[0][1][0, Lq // 2, 1].any()
    out, tol = attention_reference(q.detach(), k.detach(), v.detach(), table.detach(), lut, dout=dout, q_start=0, attn_mask=hidden.cuda())
    for name, got in zip(("y", "dq", "dk", "dv", "dtable"), runs[1]):
        close(got, out[name], tol[name], name)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("Lk", [255, 256, 511, 512, 513, 5000])
def test_attention_one_query_either_side_of_the_split(Lk, dtype):
    """One query for each of three caches, one of them empty and one of a single key, where the keys are taken whole and where they are split."""
    q, k, v, table, lut, _ = attention_inputs(Lk, 3, 1, Lk, 8, 2, 64, dtype, 32, 100, grad=False)
    how = dict(causal=True, k_len=torch.tensor([0, 1, Lk - 1], dtype=torch.int32, device="cuda"))
    y = modules.biased_attention(q, k, v, table, lut, **how)
    out, tol = attention_reference(q, k, v, table, lut, **how)
    close(y, out["y"], tol["y"], "y")
    assert not y[0].any() and torch.equal(y[1, 0], v[1, 0].repeat_interleave(4, 0))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_attention_masked_with_two_tiles_to_a_wave(dtype):
    """Heads enough that a wave takes 32 queries (keys): the mask's rows and words of both halves, with a ragged end."""
    B, H, Lq, Lk = 64, 8, 75, 141
    q, k, v, table, lut, dout = attention_inputs(3, B, Lq, Lk, H, H, 64, dtype, 16, 30)
    hidden = torch.rand(B, 1, Lq, Lk, generator=torch.Generator().manual_seed(4)) < 0.3
    kl = torch.full((B,), Lk, dtype=torch.int32)
    kl[::3] = 100
    check_attention(q, k, v, table, lut, dout, q_start=20, causal=True, k_len=kl.cuda(), attn_mask=hidden.cuda())
