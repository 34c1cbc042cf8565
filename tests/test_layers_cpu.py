"""The host side of psgd_pro_b200.layers and its C entries, without a GPU: constants, refusals, sizes of workspaces."""
import ctypes
import os
import re

import pytest
import torch

from psgd_pro_b200 import _capi, layers

HDR = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "psgd_b200.h")
EINVAL, ESPACE = -1, -4


def test_header_constants_match_binding():
    defs = dict(re.findall(r"#define (PSGD_\w+) (\d+)", open(HDR).read()))
    for name in ("PSGD_F32", "PSGD_BF16", "PSGD_F16", "PSGD_NORM_RMS", "PSGD_NORM_LAYER", "PSGD_REDUCE_NONE",
                 "PSGD_REDUCE_MEAN", "PSGD_REDUCE_SUM"):
        assert int(defs[name]) == getattr(_capi, name)
    assert int(defs["PSGD_JOINT_MAX_D"]) == _capi.JOINT_MAX_D
    assert int(defs["PSGD_ERR_BAD_TARGET"]) in _capi.ERR_BITS


def test_layers_refuse_host_tensors():
    x, t = torch.ones(4, 8), torch.zeros(4, dtype=torch.int64)
    for bad in (lambda: layers.dropout(x, 0.5, 1), lambda: layers.residual_norm(x, x), lambda: layers.linear_cross_entropy(x, x, t)):
        with pytest.raises(RuntimeError):
            bad()


def test_entries_reject_bad_specs_before_any_launch():
    L = _capi.lib()
    d = _capi.Dropout(n=8, dtype=_capi.PSGD_F32, threshold=65537)
    assert L.psgd_dropout(ctypes.byref(d), None) == EINVAL
    assert L.psgd_dropout(None, None) == EINVAL
    assert L.psgd_dropout(ctypes.byref(_capi.Dropout(n=0)), None) == 0
    j = _capi.Joint(rows=4, d=16, ld_x=16, ld_y=16)
    assert L.psgd_joint_forward(ctypes.byref(j), None) == EINVAL  # null pointers
    for bad in (dict(d=0), dict(d=_capi.JOINT_MAX_D + 1), dict(dtype=3), dict(kind=2), dict(param_dtype=1),
                dict(gate=16, gates=3), dict(rows=-1), dict(threshold=70000)):
        k = _capi.Joint(rows=4, d=16, ld_x=16, ld_y=16)
        for name, v in bad.items():
            setattr(k, name, v)
        assert L.psgd_joint_forward(ctypes.byref(k), None) == EINVAL, bad
        assert L.psgd_joint_workspace(ctypes.byref(k)) == EINVAL, bad
    assert L.psgd_joint_forward(ctypes.byref(_capi.Joint(rows=0, d=16)), None) == 0
    a = _capi.Lce(n=4, d=8, v=10, ld_h=8, ld_w=8)
    assert L.psgd_lce(ctypes.byref(a), None, None) == EINVAL
    for bad in (dict(d=0), dict(v=0), dict(dtype=3), dict(ld_h=7), dict(reduction=3), dict(piece_bytes=-1)):
        k = _capi.Lce(n=4, d=8, v=10, ld_h=8, ld_w=8)
        for name, v in bad.items():
            setattr(k, name, v)
        assert L.psgd_lce_workspace(ctypes.byref(k)) == EINVAL, bad
    assert L.psgd_lce_scale(None, 0, 4, None, None) == EINVAL


def test_a_workspace_that_is_too_small_is_refused():
    L = _capi.lib()
    a = _capi.Lce(n=4, d=8, v=10, ld_h=8, ld_w=8, piece_bytes=1 << 20)
    word = (ctypes.c_int * 4)()
    at = (ctypes.addressof(word) + 15) // 16 * 16
    for name in ("h", "w", "target", "loss", "workspace"):
        setattr(a, name, at)
    a.workspace_bytes = L.psgd_lce_workspace(ctypes.byref(a)) - 1
    assert L.psgd_lce(ctypes.byref(a), ctypes.addressof(word), None) == ESPACE


@pytest.mark.parametrize("dtype,kept", [(_capi.PSGD_BF16, 2), (_capi.PSGD_F32, 10)])
def test_workspace_of_the_loss_is_bounded_by_its_pieces(dtype, kept):
    """What grows with tokens x vocabulary is kept for a piece of the tokens only."""
    L = _capi.lib()
    n, d, v, cap = 1 << 16, 64, 32000, 64 << 20
    size = lambda **k: L.psgd_lce_workspace(ctypes.byref(_capi.Lce(n=n, d=d, v=v, ld_h=d, ld_w=d, dtype=dtype, **k)))  # noqa: E731
    whole = size(grads=1, piece_bytes=1 << 50)
    assert whole > n * v * kept
    states = 6 * d * (n + v) + 64 * n  # operands, indices
    sums = 16 * 4 * max(n, v) * d      # split and accumulated gradients
    assert size(grads=1, piece_bytes=cap) < cap + states + sums
    assert size(grads=0, piece_bytes=cap) < cap + states


def test_gate_shapes_on_the_host():
    ok = lambda *s: layers._gates(torch.empty(s), (4, 6, 24), 24)  # noqa: E731
    assert [ok(24), ok(8, 24), ok(24, 24), ok(4, 1, 24), ok(4, 6, 24), ok(1, 1, 24)] == [1, 8, 24, 4, 24, 1]
    for bad in ((23,), (5, 24), (1, 6, 24), (4, 6, 1), (2, 1, 24)):
        with pytest.raises(RuntimeError):
            ok(*bad)
