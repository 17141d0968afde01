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
