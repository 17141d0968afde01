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
        y, mean, rstd = ops.layer_norm_forward(x, stats=True)
        dx, dw, db = ops.layer_norm_backward(dy, x, None, mean, rstd)
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
        y, mean, rstd = ops.layer_norm_forward(x, w, stats=True)
        runs.append((y, *ops.layer_norm_backward(dy, x, w, mean, rstd)))
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
