"""CPU: host-side rules of the transformer-layer operators and modules at their edges (no launch)."""
import copy
import ctypes as C

import pytest
import torch

from mo_yolo_amd import _lib, modules, ops


# ---------------------------------------------------------------------------------------------------------------- prepared weights
def _weights(layer):
    return layer._prepared(torch.device("cpu"), torch.float32, layer._build)["w"][:, :layer.cin]      # (the padded copy: "wf" is the parameter itself here)


def test_prepared_weights_follow_the_parameters():
    lin = modules._Linear(8, 12)
    first = _weights(lin)
    assert torch.equal(first, lin.weight) and lin._prepared(torch.device("cpu"), torch.float32, lin._build) is lin._prep.data
    with torch.no_grad():
        lin.weight.add_(1.0)                                                   # in place: the version
    assert torch.equal(_weights(lin), lin.weight)
    old = lin.weight.data
    for _ in range(4):                                                         # other memory, twice between two calls: never the address of what was prepared
        lin.weight.data = lin.weight.data.clone() + 1.0
        lin.weight.data = lin.weight.data.clone() + 1.0
        assert torch.equal(_weights(lin), lin.weight)
    lin.weight.data = old
    assert torch.equal(_weights(lin), old)
    lin.weight.data.mul_(2.0)                                                  # through .data nothing counts it
    modules.forget_prepared(torch.nn.Sequential(lin))
    assert torch.equal(_weights(lin), lin.weight)


def test_a_module_in_training_prepares_its_weights_in_every_call():
    lin = modules._Linear(8, 12)
    with torch.no_grad():
        lin._trains()                                                          # (the differentiable form without a gradient: not training)
    keeps = lambda: lin._prepared(torch.device("cpu"), torch.float32, lin._build) is lin._prepared(torch.device("cpu"), torch.float32, lin._build)  # noqa: E731
    assert keeps()
    lin._trains()
    for _ in range(3):
        lin.weight.data.add_(1.0)                                              # as a replayed graph does: no version
        lin.bias.data.add_(1.0)
        got = lin._prepared(torch.device("cpu"), torch.float32, lin._build)
        assert torch.equal(got["w"][:, :8], lin.weight) and torch.equal(got["b"], lin.bias) and not keeps()
    lin.weight.requires_grad_(False)
    assert not keeps()                                                         # (its bias still trains)
    lin.requires_grad_(False)
    assert keeps() and torch.equal(_weights(lin), lin.weight)
    lin.load_state_dict({"weight": torch.ones(12, 8), "bias": torch.zeros(12)})
    assert torch.equal(_weights(lin), torch.ones(12, 8))


def test_copies_of_a_module_prepare_their_own_weights():
    lin = modules._Linear(8, 12)
    _weights(lin)
    lin._trains()
    twin = copy.deepcopy(lin)
    assert twin._prep is not lin._prep and twin._prep.data is None and not twin._prep.trained
    with torch.no_grad():
        twin.weight.add_(1.0)
    assert torch.equal(_weights(twin), twin.weight) and torch.equal(_weights(lin), lin.weight)


def test_the_differentiable_forms_say_that_they_train():
    """Every holder of parameters that the differentiable forms of the layer and of QIM use."""
    import inspect
    for cls in (modules._Linear, modules._MHA):
        assert "self._trains()" in inspect.getsource(cls.forward_train)
    held = [m for top in (modules.MOTRDecoderLayer(), modules.QueryInteractionModule(None, 256, 256)) for m in top.modules() if isinstance(m, modules._ParamModule)]
    assert held and all(isinstance(m, (modules._Linear, modules._MHA)) for m in held)


# ------------------------------------------------------------------------------------------------------ other ways to differentiate and to record
def _host_calls():
    """The differentiable entry points of the host side, past the checks that want a GPU: they refuse before they look at a device."""
    h, x, w = _lib.host(), torch.ones(6, 8), torch.ones(8)
    q, t, lut = torch.ones(2, 5, 2, 8), torch.ones(8, 2), ops.relative_buckets(8, 8, device="cpu")
    return [(lambda x, w, b, r: h.layer_norm(x, w, b, 1e-5, r), (x, w, w.clone(), x.clone())), (lambda x, w, b, r: h.linear(x, w, b, _lib.ACT_SILU, r), (x, x.clone(), torch.ones(6), torch.ones(6, 6))),
            (lambda q, k, v, t: h.attention(q, k, v, t, lut, None, None, False, False, 0, 1.0), (q, q.clone(), q.clone(), t))]


def test_forward_mode_is_refused():
    """A tangent is never dropped, on whichever argument it is and whether or not gradients are computed."""
    from torch.autograd import forward_ad as fw
    for f, args in _host_calls():
        for n in range(len(args)):
            for grad in (True, False):
                with fw.dual_level(), torch.set_grad_enabled(grad), pytest.raises(NotImplementedError, match="forward-mode"):
                    f(*[fw.make_dual(a, torch.ones_like(a)) if i == n else a for i, a in enumerate(args)])


@pytest.mark.filterwarnings("ignore")
def test_recording_a_trace_is_refused():
    from torch.fx.experimental.proxy_tensor import make_fx
    for f, args in _host_calls():
        with pytest.raises(RuntimeError, match="recorded"):
            torch.jit.trace(f, args, check_trace=False)
        for before_dispatch in (False, True):
            with pytest.raises(RuntimeError, match="recorded"):
                make_fx(f, pre_dispatch=before_dispatch)(*args)


# ------------------------------------------------------------------------------------------------------------------------ strides
def test_linear_strides_that_the_entry_points_take():
    """Rows over 4 MiB apart: where there is one, or few going forward; the workspace queries answer as the calls do."""
    def query(bwd=False, **kw):
        a = _lib.LinearArgs()
        a.x = a.w = a.y = 0x10000
        a.M, a.N, a.K, a.ldx, a.ldw, a.ldy, a.dtype = 1, 64, 4096, 4096, 4096, 64, _lib.BF16
        if bwd:
            a.dy = a.dx = a.dw = 0x10000
            a.ldd = 64
        for n, x in kw.items():
            setattr(a, n, x)
        return (_lib.lib().moy_linear_bwd_ws if bwd else _lib.lib().moy_linear_ws)(C.byref(a))
    far = 513 * 4096                                                           # elements of 16 bits: 4 KiB over the limit
    for kw in (dict(ldx=far), dict(ldx=1 << 40, ldy=1 << 40, r=0x10000, ldr=1 << 40), dict(M=16, ldx=far, dtype=_lib.F32), dict(M=32, K=2048, ldx=1 << 33, ldw=1 << 33), dict(M=40, N=1, ldw=1 << 40)):
        assert query(**kw) >= 0, kw
    assert query(True, ldx=1 << 40, ldd=1 << 40) >= 0 and query(True, M=40, N=1, ldw=1 << 40) >= 0
    for kw in (dict(M=2, ldx=far), dict(M=17, ldx=far, dtype=_lib.F32)):
        assert query(**kw) == _lib.ENOSYS, kw
    for kw in (dict(ldx=far), dict(ldw=far), dict(ldy=far), dict(r=0x10000, ldr=far)):
        assert query(M=33, **kw) == _lib.ENOSYS, kw
    for kw in (dict(ldx=far), dict(ldw=far), dict(ldd=far)):
        assert query(True, M=2, **kw) == _lib.ENOSYS, kw
    assert query(M=33, ldr=far) >= 0                                           # (no residual)
    assert query(M=33, ldx=512 * 4096) >= 0 and query(K=1 << 22, ldx=1 << 22, ldw=1 << 22) == _lib.ENOSYS



def test_the_tight_bounds_see_a_rounded_weight_and_a_rounded_output():
    """The bounds of test_gpu_layer_edges.test_attention_rounds_its_results_alone, on the CPU with the roundings planted: weights rounded to 16 bits miss them for y, and
    a delta from the rounded output misses them for dtable; weights as two operands and a delta with what the rounding left out do not."""
    import test_gpu_layer_edges as E
    lut = ops.relative_buckets(16, 30, device="cpu")
    for dt in (torch.bfloat16, torch.float16):
        seen = dict(y=False, dtable=False)
        for Lq, Lk, D, start, H in E.TIGHT:
            ins = E.tight_inputs(torch.Generator().manual_seed(Lq + Lk), Lq, Lk, D, H, dt)
            at = lut.long()[(torch.arange(Lk)[None] - torch.arange(Lq)[:, None] - start).clamp(-30, 30) + 30]
            for h in range(H):
                q, k, v, do, table = (t[:, h] for t in ins)
                want, tol = E.tight_reference(q, k, v, do, table, lut, start)
                qd, kd, vd, g = (t.double() for t in (q, k, v, do))
                p = torch.softmax(qd @ kd.t() * D ** -0.5 + table.double()[at], -1)
                r = lambda t: t.to(dt).double()  # noqa: E731
                top = p.amax(-1, keepdim=True)
                w = p / top                                                        # as the kernel holds them: the largest 1
                two = (r(w) + r(w - r(w))) @ vd * top
                by = lambda delta: torch.zeros(16, dtype=torch.float64).index_add_(0, at.reshape(-1), (p * (g @ vd.t() - delta)).reshape(-1))  # noqa: E731
                o, one = r(two), r(r(w) @ vd * top)
                good = dict(y=o, dtable=r(by((g * (o + r(two - o))).sum(-1, keepdim=True))))
                bad = dict(y=one, dtable=r(by((g * o).sum(-1, keepdim=True))))
                for name in want:
                    assert bool(((good[name] - want[name]).abs() <= tol[name]).all()), (name, dt, Lq)
                    seen[name] |= bool(((bad[name] - want[name]).abs() > tol[name]).any())
        assert all(seen.values()), (dt, seen)


# ------------------------------------------------------------------------------------------------------------------- saved tensors
def test_backward_refuses_what_the_forward_did_not_save():
    """Another type or size of any tensor that a backward pass is given is an error before a kernel could read past its end."""
    h, code = _lib.host(), torch.float32
    x, w = torch.ones(6, 8, dtype=torch.bfloat16), torch.ones(8)
    W, z = torch.ones(5, 8, dtype=torch.bfloat16), torch.ones(6, 5, dtype=torch.bfloat16)
    q, k, t = (torch.ones(*s, dtype=torch.bfloat16) for s in ((2, 5, 4, 8), (2, 7, 2, 8), (8, 4)))
    lut, n, m, lse = ops.relative_buckets(8, 8, device="cpu"), torch.ones(2, dtype=torch.int32), torch.zeros(5, 7, dtype=torch.bool), torch.ones(2, 4, 5)
    norm = (lambda dy, x, w, stat, r: h.layer_norm_backward(dy, x, w, stat, r, True, True, True, code), (x, x, w, torch.ones(2, 6), x))
    linear = (lambda dy, x, w, z: h.linear_backward(dy, x, w, z, _lib.ACT_SILU, True, True, True, code), (z, x, W, z))
    attention = (lambda *a: h.attention_backward(*a, False, False, 0, 1.0, True, True, True, True), (q, q, k, k, q, lse, q, t, lut, n, m))
    for f, args in (norm, linear, attention):
        with pytest.raises(RuntimeError) as e:                                 # as they were: only the missing GPU stops them
            f(*args)
        assert "forward's size" not in str(e.value)
        for i, a in enumerate(args):
            other = torch.float64 if a.dtype == torch.float32 else torch.float32
            # (of the statistics and of z the count is what matters; a table of any length goes with a map that is clamped to it)
            counted, table = a is lse or f is norm[0] and i == 3 or f is linear[0] and i == 3, a is t
            for bad in (a.to(other), a[..., :-1], *([] if table else [torch.cat((a, a))]), *([] if counted else [a[None]])):
                with pytest.raises(RuntimeError, match="forward's size"):
                    f(*[bad if j == i else b for j, b in enumerate(args)])


# -------------------------------------------------------------------------------------------------------------------- largest sizes
def test_sizes_whose_launches_would_count_past_32_bits_are_refused():
    """The workspace queries answer as the calls do."""
    a = _lib.AttentionArgs()
    for n in ("q", "k", "v", "o", "dout", "lse", "dq"):
        setattr(a, n, 0x10000)
    a.H, a.Hk, a.Lq, a.Lk, a.D, a.scale, a.dtype = 8, 8, 1, 1, 8, 0.125, _lib.BF16
    forward, backward = (lambda f=f, **kw: [setattr(a, n, x) for n, x in kw.items()] and f(C.byref(a)) for f in (_lib.lib().moy_attention_ws, _lib.lib().moy_attention_bwd_ws))
    assert forward(B=(1 << 21) - 1) == 0 and backward(B=(1 << 21) - 1) > 0
    assert forward(B=1 << 21) == backward(B=1 << 21) == _lib.ENOSYS
    assert forward(B=1 << 20, Lq=65) == _lib.ENOSYS and forward(B=1 << 20, Lq=64) == 0
    assert forward(B=1 << 20, Lq=1, Lk=65) == 0 and backward(B=1 << 20, Lq=1, Lk=130) == _lib.ENOSYS       # (the gradients of keys walk the keys)
    assert forward(B=1 << 15, Lq=1, Lk=16384) == 0 and forward(B=1 << 21, Lq=1, Lk=600) == _lib.ENOSYS    # (the kernel for few queries)

    def linear(bwd=False, **kw):
        b = _lib.LinearArgs()
        b.x = b.w = b.y = b.dy = b.dx = 0x10000
        b.N, b.K, b.ldx, b.ldw, b.ldy, b.ldd, b.dtype = 8, 8, 8, 8, 8, 8, _lib.BF16
        for n, x in kw.items():
            setattr(b, n, x)
        return (_lib.lib().moy_linear_bwd_ws if bwd else _lib.lib().moy_linear_ws)(C.byref(b))
    for bwd in (False, True):
        assert linear(bwd, M=(1 << 30) + 64) >= 0 and linear(bwd, M=0x7fffffff - 512) >= 0
        assert linear(bwd, M=0x7fffffff - 511) == _lib.ENOSYS
    wide = dict(M=1 << 30, N=1 << 20, K=1 << 20, ldw=1 << 20, ldx=1 << 20, ldy=1 << 20, ldd=1 << 20)
    assert linear(**wide) == linear(True, **wide) == _lib.ENOSYS
