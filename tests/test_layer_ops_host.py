"""CPU: refusals and host-side rules of the transformer-layer operators (no launch, no device access)."""
import ctypes as C

import pytest
import torch

from mo_yolo_amd import _lib, modules, ops

FAKE = 0x10000          # aligned, never dereferenced: every refusal comes before a launch


# ------------------------------------------------------------------------------------------------------------------ layer norm
def _ln(**kw):
    a = dict(x=FAKE, ldx=256, r=None, ldr=0, w=FAKE, b=FAKE, w_dtype=_lib.F32, rows=4, C=256, eps=1e-5, y=FAKE, ldy=256, mean=None, rstd=None,
             dtype=_lib.BF16)
    a.update(kw)
    return _lib.lib().moy_layer_norm(*a.values(), None)


def _ln_bwd(**kw):
    a = dict(dy=FAKE, ldd=256, x=FAKE, ldx=256, r=None, ldr=0, w=FAKE, w_dtype=_lib.F32, mean=FAKE, rstd=FAKE, rows=4, C=256, dx=FAKE, ldo=256,
             dw=FAKE, db=FAKE, ws=FAKE, ws_len=1 << 20, dtype=_lib.BF16)
    a.update(kw)
    return _lib.lib().moy_layer_norm_bwd(*a.values(), None)


@pytest.mark.parametrize("kw", [dict(x=None), dict(y=None), dict(rows=0), dict(rows=-1), dict(C=0), dict(dtype=7), dict(w_dtype=_lib.F16), dict(mean=FAKE),
                                dict(eps=-1.0), dict(eps=float("nan")), dict(ldy=255), dict(ldx=-1), dict(x=FAKE + 1), dict(w=FAKE + 2), dict(r=FAKE, ldr=-4)])
def test_layer_norm_refuses(kw):
    assert _ln(**kw) == _lib.EINVAL


@pytest.mark.parametrize("kw", [dict(dy=None), dict(mean=None), dict(dx=None, dw=None, db=None), dict(ws=None), dict(ws_len=10), dict(ldo=100), dict(rows=0),
                                dict(w_dtype=_lib.F16), dict(dw=FAKE + 2)])
def test_layer_norm_backward_refuses(kw):
    assert _ln_bwd(**kw) == _lib.EINVAL


def test_layer_norm_widths():
    assert _ln(C=16385, ldy=16385) == _lib.ENOSYS and _ln(C=8193, ldy=8193, dtype=_lib.F32) == _lib.ENOSYS
    ws = _lib.lib().moy_layer_norm_bwd_ws
    assert ws(1 << 40, 16384, _lib.BF16) == 512 * 2 * 16384 and ws(1, 256, _lib.F32) == 512 and ws(4, 16385, _lib.F16) == _lib.ENOSYS
    assert ws(0, 256, _lib.F32) == _lib.EINVAL


def test_layer_ops_refuse_cpu_tensors():
    x = torch.zeros(2, 8)
    with pytest.raises(RuntimeError, match="Not implemented on the CPU"):
        ops.layer_norm_forward(x)
    with pytest.raises(RuntimeError, match="Not implemented on the CPU"):
        modules.layer_norm(x.requires_grad_(True), torch.ones(8), torch.zeros(8))


# ------------------------------------------------------------------------------------------------------------------- attention
def _attn(bwd=False, **kw):
    a = _lib.AttentionArgs()
    for n in ("q", "k", "v", "o"):
        setattr(a, n, FAKE)
    a.B, a.H, a.Hk, a.Lq, a.Lk, a.D, a.scale, a.dtype = 2, 4, 2, 5, 7, 64, 0.125, _lib.BF16
    a.q_sb, a.q_sl, a.q_sh, a.k_sb, a.k_sl, a.k_sh, a.v_sb, a.v_sl, a.v_sh = 5 * 256, 256, 64, 7 * 128, 128, 64, 7 * 128, 128, 64
    if bwd:
        a.dout = a.lse = a.dq = a.ws = FAKE
        a.g_sb, a.g_sl, a.g_sh, a.ws_len = 5 * 256, 256, 64, 1 << 20
    for n, x in kw.items():
        setattr(a, n, x)
    f = _lib.lib().moy_attention_bwd if bwd else _lib.lib().moy_attention
    return f(C.byref(a), None), (_lib.lib().moy_attention_bwd_ws if bwd else _lib.lib().moy_attention_ws)(C.byref(a))


BAD_ATTENTION = [dict(q=None), dict(k=None), dict(v=None), dict(o=None), dict(B=0), dict(Lq=0), dict(Lk=-1), dict(H=3), dict(Hk=0), dict(D=12), dict(D=0),
                 dict(dtype=9), dict(q=FAKE + 8), dict(q_sl=257), dict(k_sb=-128), dict(table=FAKE), dict(lut=FAKE),
                 dict(table=FAKE, lut=FAKE, num_buckets=65, max_distance=128), dict(table=FAKE, lut=FAKE, num_buckets=32, max_distance=0),
                 dict(table=FAKE, lut=FAKE, num_buckets=32, max_distance=1025), dict(scale=float("inf")), dict(scale=-0.5), dict(o_rest=FAKE + 8), dict(scale=float("nan")), dict(q_start=(1 << 30) + 1),
                 dict(mask=FAKE, m_sq=-1), dict(k_len=FAKE + 2), dict(B=1 << 20, H=1 << 10, Hk=1)]


@pytest.mark.parametrize("kw", BAD_ATTENTION)
def test_attention_refuses(kw):
    assert _attn(**kw) == (_lib.EINVAL, _lib.EINVAL)
    assert _attn(True, **kw) == (_lib.EINVAL, _lib.EINVAL)


def test_attention_refuses_on_the_way_back():
    for kw in (dict(dout=None), dict(lse=None), dict(dq=None), dict(dtable=FAKE), dict(dk=FAKE + 4), dict(g_sl=3)):
        assert _attn(True, **kw)[0] == _lib.EINVAL, kw
    assert _attn(True, ws=None)[0] == _lib.EINVAL and _attn(True, ws_len=39)[0] == _lib.EINVAL
    assert _attn(D=136) == (_lib.ENOSYS, _lib.ENOSYS)
    assert _lib.lib().moy_attention(None, None) == _lib.EINVAL and _lib.lib().moy_attention_bwd_ws(None) == _lib.EINVAL
    # a long cache is split: partial results need a workspace
    assert _attn(Lq=1, Lk=8192, ws_len=10, ws=FAKE)[0] == _lib.EINVAL
    assert _attn(Lq=1, Lk=8192)[1] == 32 * 2 * 4 * 1 * (2 + 64)


def test_attention_args_layout_matches_header():
    import os
    import re
    txt = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "moyolo.h")).read()
    body = txt[txt.index("typedef struct moy_attention_args {"):txt.index("} moy_attention_args;")].split("{", 1)[1]
    assert [re.split(r"[ *]+", d.strip())[-1] for d in body.split(";") if d.strip()] == [f[0] for f in _lib.AttentionArgs._fields_]


def test_relative_buckets():
    b = ops.relative_buckets(32, 128, True, "cpu")
    at = lambda d: int(b[d + 128])  # noqa: E731
    assert b.dtype == torch.uint8 and b.shape == (257,)
    assert [at(-d) for d in (0, 1, 7, 8, 11, 12, 15, 16, 127, 128)] == [0, 1, 7, 8, 8, 9, 9, 10, 15, 15]      # 8 * (128 / 8)^(t / 8): 8, 11.3, 16, 22.6, ...
    assert [at(d) for d in (1, 8, 128)] == [17, 24, 31]
    one = ops.relative_buckets(8, 16, False, "cpu").tolist()                  # exact borders: 4 * 4^(t / 4) = 4, 5.66, 8, 11.3
    assert one == [7] * 5 + [6] * 4 + [5] * 2 + [4] * 2 + [3, 2, 1, 0] + [0] * 16
    for bad in ((3, 8, True), (65, 128, False), (1, 8, False), (32, 8, True), (32, 1025, True)):
        with pytest.raises(ValueError):
            ops.relative_buckets(*bad, device="cpu")


def test_attention_refuses_cpu_tensors():
    q = torch.zeros(1, 2, 1, 8)
    with pytest.raises(RuntimeError, match="Not implemented on the CPU"):
        ops.attention_forward(q, q, q)
    with pytest.raises(RuntimeError, match="Not implemented on the CPU"):
        modules.biased_attention(q.requires_grad_(True), q, q)


# ---------------------------------------------------------------------------------------------------------------------- linear
def _lin(bwd=False, **kw):
    a = _lib.LinearArgs()
    a.x = a.w = a.ws = FAKE
    a.M, a.N, a.K, a.ldx, a.ldw, a.dtype, a.act, a.ws_len = 100, 64, 128, 128, 128, _lib.BF16, _lib.ACT_SILU, 1 << 40
    if bwd:
        a.dy = a.z = a.dx = a.dw = a.db = FAKE
        a.ldd = 64
    else:
        a.y, a.ldy = FAKE, 64
    for n, x in kw.items():
        setattr(a, n, x)
    f = _lib.lib().moy_linear_bwd if bwd else _lib.lib().moy_linear
    return f(C.byref(a), None), (_lib.lib().moy_linear_bwd_ws if bwd else _lib.lib().moy_linear_ws)(C.byref(a))


@pytest.mark.parametrize("kw", [dict(x=None), dict(w=None), dict(M=0), dict(N=0), dict(K=-1), dict(dtype=3), dict(act=4), dict(act=-1), dict(b_dtype=_lib.F16),
                                dict(x=FAKE + 1), dict(ldx=-128)])
def test_linear_refuses(kw):
    assert _lin(**kw) == (_lib.EINVAL, _lib.EINVAL) and _lin(True, **kw) == (_lib.EINVAL, _lib.EINVAL)


def test_linear_refuses_by_direction_and_size():
    for kw in (dict(y=None), dict(ldy=63), dict(r=FAKE, ldr=-1), dict(z=FAKE + 1)):
        assert _lin(**kw)[0] == _lib.EINVAL, kw
    for kw in (dict(dy=None), dict(z=None), dict(dx=None, dw=None, db=None), dict(dw=FAKE + 1), dict(ws=None), dict(ws_len=1), dict(ws=FAKE + 8)):
        assert _lin(True, **kw)[0] == _lib.EINVAL, kw
    assert _lin(K=1 << 22, ldx=1 << 22, ldw=1 << 22)[0] == _lib.ENOSYS and _lin(ldx=1 << 22)[0] == _lib.ENOSYS
    # workspaces: none where the rows are whole dwords and the product fills the chip, padded copies of odd 16-bit rows
    assert _lin(M=16, N=256, ldy=256)[1] == 0 and _lin(M=16, K=101, ldx=101, ldw=101)[1] == 0
    assert _lin(M=40, K=102, ldx=102, ldw=102)[1] == 0 and _lin(M=40, K=101, ldx=101, ldw=101, dtype=_lib.F32)[1] == 0
    assert _lin(M=40, K=101, ldx=101, ldw=101, N=256, ldy=256)[1] == -(-40 * 104 * 2 // 256) * 256 + 256 * 104 * 2


def test_linear_args_layout_matches_header():
    import os
    import re
    txt = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "moyolo.h")).read()
    body = txt[txt.index("typedef struct moy_linear_args {"):txt.index("} moy_linear_args;")].split("{", 1)[1]
    assert [re.split(r"[ *]+", d.strip())[-1] for d in body.split(";") if d.strip()] == [f[0] for f in _lib.LinearArgs._fields_]


def test_linear_refuses_cpu_tensors():
    x, w = torch.zeros(2, 8), torch.zeros(4, 8)
    with pytest.raises(RuntimeError, match="Not implemented on the CPU"):
        ops.linear_forward(x, w)
    with pytest.raises(RuntimeError, match="Not implemented on the CPU"):
        modules.linear(x, w.requires_grad_(True))


def test_host_module_is_built_and_missing_fails_loudly(monkeypatch):
    import builtins
    import sys

    from mo_yolo_amd import build
    build.build(verbose=False)
    h = _lib.host()
    assert h is _lib.host() and callable(h.layer_norm) and callable(h.linear) and callable(h.attention)
    monkeypatch.setattr(_lib, "_host_module", None)
    monkeypatch.delitem(sys.modules, "mo_yolo_amd._host", raising=False)
    monkeypatch.delattr(sys.modules["mo_yolo_amd"], "_host", raising=False)
    real = builtins.__import__

    def no_host(name, globals=None, locals=None, fromlist=(), level=0):
        if fromlist and "_host" in fromlist:
            raise ImportError("not there")
        return real(name, globals, locals, fromlist, level)
    monkeypatch.setattr(builtins, "__import__", no_host)
    with pytest.raises(_lib.MoyoloError, match="_host.so"):
        _lib.host()


def test_sizes_that_do_not_fit_the_entry_points_are_refused(monkeypatch):
    """Sizes are 32-bit behind the checks: a broadcast axis beyond that is an error, not a smaller size."""
    monkeypatch.setattr(ops, "_one_device", lambda *t: None)
    long = torch.zeros(1).expand(1, (1 << 32) + 8)
    with pytest.raises(ValueError, match="layer_norm"):
        ops._norm_check(long, None, None, 1e-5, None)
    with pytest.raises(ValueError, match="linear"):
        ops._linear_check(torch.zeros(2, 8), torch.zeros(1, 8).expand((1 << 32) + 8, 8), None, _lib.ACT_NONE, None)
    q, k = torch.zeros(1, 4, 2, 8), torch.zeros(1, 1, 2, 8).expand(1, (1 << 32) + 8, 2, 8)
    with pytest.raises(ValueError, match="attention"):
        ops._attention_check(q, k, k, None, None, None, None, None, None)
