"""psgd_pro_b200.layers where its kernels change their ways: sizes at which another kernel, tile or launch is taken, and inputs
at the ends of their types. References are formed in 64 bits on the GPU; tolerances as in test_layers_gpu.py."""
import math

import pytest
import torch

from psgd_pro_b200 import _capi, layers

pytestmark = pytest.mark.gpu
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
PRODUCT = {"fp32": 1e-5, "bf16": 2.0 ** -8, "fp16": 2.0 ** -10}


def rel(a, b):
    a, b = a.detach().double(), b.detach().double()
    assert a.shape == b.shape and torch.isfinite(a).all()
    return ((a - b).norm() / b.norm().clamp_min(1e-300)).item()


def lce_case(n, d, v, dtype, ignored, cuda, spread=1.5):
    g = torch.Generator(device="cuda").manual_seed(n * 7 + d * 3 + v)
    w = torch.randn(v, d, generator=g, device=cuda) * spread / math.sqrt(d)
    t = torch.randint(0, v, (n,), generator=g, device=cuda)
    h = torch.randn(n, d, generator=g, device=cuda) + torch.rand(n, 1, generator=g, device=cuda) * 6 * w[t]
    t[torch.randperm(n, generator=g, device=cuda)[:int(n * ignored)]] = -100
    return h.to(TYPES[dtype]), w.to(TYPES[dtype]), t


def lce_ref(h, w, t, smoothing=0.0, z=0.0, reduction="mean", grad=None):
    """(loss, dh, dw) in 64 bits from the formulas."""
    h, w = h.double(), w.double()
    rows = (t != -100).nonzero()[:, 0]
    logits = h[rows] @ w.T
    lse = logits.logsumexp(1)
    at = t[rows][:, None]
    one = (1 - smoothing) * (lse - logits.gather(1, at)[:, 0]) + smoothing * (lse - logits.mean(1)) + z * lse * lse
    loss = torch.zeros(t.shape, dtype=torch.float64, device=h.device).index_copy(0, rows, one)
    share = 1.0 / max(len(rows), 1) if reduction == "mean" else 1.0
    up = torch.ones(len(rows), dtype=torch.float64, device=h.device) if grad is None else \
        (grad.double()[rows] if reduction == "none" else grad.double().expand(len(rows)))
    g = (logits - lse[:, None]).exp() * (1 + 2 * z * lse)[:, None] - smoothing / w.shape[0]
    g.scatter_add_(1, at, torch.full_like(lse, smoothing - 1)[:, None])
    g *= (up * share)[:, None]
    dh = torch.zeros_like(h).index_copy(0, rows, g @ w)
    return (loss if reduction == "none" else loss.sum() * share), dh, g.T @ h[rows]


# ---- waits -----------------------------------------------------------------------------------------------------------
def test_loss_stays_inside_a_shorter_wait_limit(cuda):
    lib = _capi.lib()
    h, w, t = lce_case(700, 136, 3001, "bf16", 0.2, cuda)
    want = layers.linear_cross_entropy_grad(h, w, t)
    assert lib.psgd_set_wait_limit_ns(200_000_000) == 2_000_000_000  # 200 ms: far above any legitimate wait
    try:
        got = layers.linear_cross_entropy_grad(h, w, t)
        layers.check_errors()
    finally:
        assert lib.psgd_set_wait_limit_ns(0) == 200_000_000
    assert all(torch.equal(a, b) for a, b in zip(got, want))


# ---- autograd --------------------------------------------------------------------------------------------------------
def test_seed_tensors_under_autograd(cuda):
    """The masks of a seed tensor are those of the same numbers, forward and backward, and a change of it in between raises."""
    x, y, up = (torch.randn(20, 48, device=cuda, requires_grad=k < 2) for k in range(3))
    rng = torch.tensor([11, 5], device=cuda)

    def both(**k):
        a = layers.dropout(x, 0.3, residual=y, **k)
        b, c = layers.residual_norm(x, y, dropout_p=0.3, **k)
        return a, b, c

    got, want = both(seed=rng), both(seed=11, offset=5)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    for pair in zip(got, want):
        a, b = (torch.autograd.grad(v, (x, y), up, retain_graph=True) for v in pair)  # (out and normed are of one node)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    late = both(seed=rng)
    rng[1] += 1
    for a in late:
        with pytest.raises(RuntimeError, match="inplace"):
            torch.autograd.grad(a, (x, y), up)
