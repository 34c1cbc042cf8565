"""Host side of psgd_pro_b200.layers and its C entries at their edges, without a GPU."""
import ctypes
import os
import re
import threading
import time

import pytest
import torch
from torch.autograd import forward_ad

from psgd_pro_b200 import _capi, layers

HDR = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "psgd_b200.h")
CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "psgd_pro_b200", "csrc")


def test_every_bounded_launch_takes_the_settable_wait_limit():
    """A kernel's limit comes from wait_limit(), which psgd_set_wait_limit_ns sets: the constant itself is only its default and
    the limit of what an aborting CTA has in flight."""
    given = []
    for name in sorted(os.listdir(CSRC)):
        text = re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, name)).read())
        assert not re.search(r"wait_ns\s*=\s*WAIT_LIMIT_NS", text), name
        given += re.findall(r"wait_limit\(\)\)|wait_ns = wait_limit\(\)", text)
    assert len(given) >= 4


@pytest.fixture
def launches(monkeypatch):
    """The launches replaced by plain ones, so that calls on host tensors run through autograd's side of the module."""
    monkeypatch.setattr(layers, "_dropout", lambda x, p, seed, offset, residual: x * 2 if residual is None else residual + x * 2)
    monkeypatch.setattr(layers, "residual_norm_forward", lambda x, y, **_: (x + y, x + y, torch.ones(1)))
    monkeypatch.setattr(layers, "residual_norm_grad", lambda d_out, d_normed, out, y, *_, **__: layers.ResidualNormGrads(
        torch.ones_like(out), torch.ones_like(y), *[None] * 5))
    monkeypatch.setattr(layers, "_lce", lambda h, w, t, need, *_, **__: ((h @ w.T).sum(), torch.ones_like(h), torch.ones_like(w)))


CALLS = {
    "dropout": lambda a, b: layers.dropout(a, 0.5, 1),
    "dropout residual": lambda a, b: layers.dropout(b, 0.5, 1, residual=a),
    "joint": lambda a, b: layers.residual_norm(a, b),
    "joint weight": lambda a, b: layers.residual_norm(b, b, weight=a),
    "loss": lambda a, b: layers.linear_cross_entropy(a, b, torch.zeros(4, dtype=torch.int64)),
    "loss weight": lambda a, b: layers.linear_cross_entropy(b, a, torch.zeros(4, dtype=torch.int64)),
}


@pytest.mark.parametrize("call", list(CALLS))
@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_is_refused(launches, call, grad):
    """A tangent is not lost without a word, whether or not gradients are recorded; the same call without one runs."""
    a, b = torch.ones(4, 4), torch.ones(4, 4)
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        CALLS[call](a, b)
        with pytest.raises(RuntimeError, match="forward mode"):
            CALLS[call](forward_ad.make_dual(a, torch.ones(4, 4)), b)


@pytest.mark.parametrize("call", ["dropout", "dropout residual", "joint"])
def test_a_seed_tensor_changed_before_the_backward_pass_is_noticed(launches, call):
    x = torch.ones(4, 4, requires_grad=True)
    rng = torch.tensor([3, 0])
    f = {"dropout": lambda: layers.dropout(x, 0.5, rng), "dropout residual": lambda: layers.dropout(x, 0.5, rng, residual=x),
         "joint": lambda: sum(layers.residual_norm(x, x, dropout_p=0.5, seed=rng))}[call]
    torch.autograd.grad(f().sum(), x)
    y = f().sum()
    rng[1] += 1
    with pytest.raises(RuntimeError, match="inplace"):
        torch.autograd.grad(y, x)


def test_first_calls_of_several_threads_share_one_error_word(monkeypatch):
    """A second word would leave the one that a kernel was given to the allocator."""
    made = []

    def pin(t):
        made.append(t)
        time.sleep(0.05)  # (the other threads arrive meanwhile)
        return t

    monkeypatch.setattr(torch.Tensor, "pin_memory", pin)
    words, got = layers._ErrorWords(), []
    threads = [threading.Thread(target=lambda: got.append(words.get(0))) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(made) == 1 and len(got) == 4 and len(set(got)) == 1


def test_sizes_of_the_loss_beyond_its_index_arithmetic_are_refused():
    defs = dict(re.findall(r"#define (PSGD_\w+) (\d+)", open(HDR).read()))
    assert int(defs["PSGD_LCE_MAX"]) == _capi.LCE_MAX
    L = _capi.lib()
    for name in ("n", "d", "v"):
        k = _capi.Lce(n=1, d=1, v=1, ld_h=1 << 40, ld_w=1 << 40)
        setattr(k, name, _capi.LCE_MAX)
        assert L.psgd_lce_workspace(ctypes.byref(k)) > 0
        setattr(k, name, _capi.LCE_MAX + 1)
        assert L.psgd_lce_workspace(ctypes.byref(k)) == -1, name


def test_joint_row_strides_below_a_row_are_refused():
    """Also negative ones: rows would be read from before the tensor."""
    L = _capi.lib()
    at = dict(x="ld_x", y="ld_y", d_out="ld_d_out", d_normed="ld_d_normed")
    base = dict({p: 16 for p in at}, **{ld: 16 for ld in at.values()}, rows=4, d=16, eps=1.0)
    assert L.psgd_joint_workspace(ctypes.byref(_capi.Joint(**base))) > 0
    for p, ld in at.items():
        for bad in (15, 0, -16, 1 << 31):
            j = _capi.Joint(**dict(base, **{ld: bad}))
            assert L.psgd_joint_workspace(ctypes.byref(j)) == -1, (ld, bad)
            assert L.psgd_joint_forward(ctypes.byref(j), None) == -1 and L.psgd_joint_backward(ctypes.byref(j), 16, 1 << 30, None) == -1
    for p, ld in at.items():
        if p != "x":  # a matrix that is not there needs no stride
            assert L.psgd_joint_workspace(ctypes.byref(_capi.Joint(**dict(base, **{p: None, ld: 0})))) > 0
