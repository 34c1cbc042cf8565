"""psgd_pro_b200.layers against their formulas in 64 bits (torch autograd on the CPU) on the same inputs.

Tolerances (relative, 2-norm): one rounding to the output's type moves a value by at most 2^-8 (bf16) or 2^-11 (fp16) of
itself, and many values of all magnitudes by less than half of that in the 2-norm; dropout is compared value by value.
bf16 and fp16 gradients of the cross entropy also carry the rounding of g, once to the same type (fp16: and of the kept
exponentials, 2^-12), so twice the bound; fp32 ones the rounding of sums of up to a few thousand fp32 products, 2^-24 each
and random in sign, with a factor of ten to spare, and the truncation of the tensor cores' sums. The joint and dropout in
fp32: a few roundings of 2^-24 each, sums over rows as above."""
import math

import numpy as np
import pytest
import torch

from psgd_pro_b200 import layers
from noise_ref import philox4x32_10

pytestmark = pytest.mark.gpu
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
ONE = {"fp32": 2e-6, "bf16": 2.0 ** -9, "fp16": 2.0 ** -12}       # one rounding (fp32: a few)
PRODUCT = {"fp32": 1e-5, "bf16": 2.0 ** -8, "fp16": 2.0 ** -10}   # gradients through the tensor cores


def rel(a, b):
    a, b = a.detach().double().cpu(), b.detach().double().cpu()
    assert a.shape == b.shape and torch.isfinite(a).all()
    return ((a - b).norm() / b.norm().clamp_min(1e-30)).item()


def rand(g, *shape, std=1.0, mean=0.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=g) * std + mean).to(dtype)


def mask(shape, p, seed, offset):
    """0 or the scale of each element, from the generator's definition in numpy."""
    n = math.prod(shape)
    blocks = np.arange(-(-n // 8), dtype=np.uint64)
    c = np.stack([blocks & 0xFFFFFFFF, blocks >> np.uint64(32), np.full_like(blocks, offset & 0xFFFFFFFF),
                  np.full_like(blocks, offset >> 32)], axis=1)
    words = philox4x32_10(c, (seed & 0xFFFFFFFF, seed >> 32)).astype(np.uint32)
    fields = words.view(np.uint16).reshape(-1)[:n].reshape(shape).astype(np.int64)
    t = int(round(p * 65536))
    return torch.from_numpy(fields >= t).double() * (65536.0 / (65536 - t) if t < 65536 else 0.0)


def rounded(got, want, parts=0.0):
    """Each value is `want` after one rounding to its type and two fp32 roundings of operands up to `parts`."""
    unit = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[got.dtype]
    tiny = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}[got.dtype]
    off = (got.double().cpu() - want).abs()
    return bool((off <= unit * want.abs() * (1 + 2.0 ** -10) + 2.0 ** -22 * (want.abs() + parts) + tiny).all())


# ---- dropout --------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n", [1, 7, 8, 9, 4095, 100003])
def test_dropout(cuda, dtype, n):
    g = torch.Generator().manual_seed(n)
    x, r = rand(g, n, dtype=TYPES[dtype]), rand(g, n, dtype=TYPES[dtype])
    seed, offset, p = 0x9ABCDEF012345678, 0xF00000001, 0.3
    m = mask((n,), p, seed, offset)
    y = layers.dropout(x.to(cuda), p, seed, offset)
    assert torch.equal(y.cpu() != 0, (m * x.double()) != 0)
    assert rounded(y, x.double() * m)
    both = layers.dropout(x.to(cuda), p, seed, offset, residual=r.to(cuda))
    assert rounded(both, r.double() + x.double() * m, r.double().abs() + (x.double() * m).abs())
    assert torch.equal(layers.dropout_grad(x.to(cuda), p, seed, offset), y)


def test_dropout_strides_alignment_and_seed_tensor(cuda):
    g = torch.Generator().manual_seed(0)
    base = rand(g, 40, 33, dtype=torch.bfloat16).to(cuda)
    m = mask((33, 40), 0.5, 3, 0)
    assert rel(layers.dropout(base.t(), 0.5, 3), base.t().double().cpu() * m) <= ONE["bf16"]
    odd = rand(g, 1001, dtype=torch.bfloat16).to(cuda)[1:]  # two bytes past an aligned address
    want = odd.double().cpu() * mask((1000,), 0.5, 3, 9)
    assert rel(layers.dropout(odd, 0.5, 3, 9), want) <= ONE["bf16"]
    assert rel(layers.dropout(odd, 0.5, torch.tensor([3, 9], device=cuda)), want) <= ONE["bf16"]


def test_dropout_ends(cuda):
    x = torch.tensor([float("inf"), float("nan"), 1.0, -2.0] * 5, device=cuda)
    assert torch.equal(layers.dropout(x, 0.0, 1)[2:4], x[2:4])
    assert torch.equal(layers.dropout(x, 1.0, 1), torch.zeros_like(x))  # what is dropped is zero, whatever it was
    assert layers.dropout(x[:0], 0.5, 1).numel() == 0
    kept = layers.dropout(torch.ones(1 << 20, device=cuda), 0.1, 5) != 0
    assert abs(kept.float().mean().item() - 0.9) < 6 * math.sqrt(0.09 / 2 ** 20)  # six deviations of the count


def test_dropout_autograd(cuda):
    x = torch.randn(33, 5, device=cuda, requires_grad=True)
    r = torch.randn(33, 5, device=cuda, requires_grad=True)
    dy = torch.randn(33, 5, device=cuda)
    gx, gr = torch.autograd.grad(layers.dropout(x, 0.25, 11, 2, residual=r), (x, r), dy)
    assert torch.equal(gx, layers.dropout_grad(dy, 0.25, 11, 2)) and torch.equal(gr, dy)


def test_dropout_refusals(cuda):
    x = torch.ones(8, device=cuda)
    for bad in (lambda: layers.dropout(x, -0.1, 0), lambda: layers.dropout(x, 1.5, 0), lambda: layers.dropout(x.cpu(), 0.5, 0),
                lambda: layers.dropout(x.int(), 0.5, 0), lambda: layers.dropout(x, 0.5, 0, residual=x[:4]),
                lambda: layers.dropout(x, 0.5, 0, residual=x.half()), lambda: layers.dropout(x, 0.5, torch.ones(2, device=cuda)),
                lambda: layers.dropout(x, 0.5, torch.ones(3, dtype=torch.int64, device=cuda))):
        with pytest.raises(RuntimeError):
            bad()


# ---- the joint -------------------------------------------------------------------------------------------------------
def joint_ref(x, y, norm, post_norm, w, b, pw, pb, gate, scale, eps, drop):
    def n(a, weight, bias):
        if norm == "layer":
            a = a - a.mean(-1, keepdim=True)
        a = a / (a.pow(2).mean(-1, keepdim=True) + eps).sqrt()
        a = a if weight is None else a * weight
        return a if bias is None else a + bias

    u = n(y, pw, pb) if post_norm else y
    if drop is not None:
        u = u * drop
    if gate is not None:
        u = (u.reshape(gate.numel() // gate.shape[-1], -1, x.shape[-1]) * gate.reshape(-1, 1, x.shape[-1])).view_as(u)
    out = x + scale * u
    return out, n(out, w, b)


JOINTS = [
    # rows, d, type, norm, post norm, gate rows, p, parameters' type
    (1, 1, "fp32", "rms", False, 0, 0.0, "fp32"),
    (1, 8, "bf16", "layer", True, 1, 0.0, "fp32"),
    (65, 192, "fp32", "layer", False, 0, 0.0, "fp32"),
    (65, 192, "bf16", "layer", True, 5, 0.1, "bf16"),
    (640, 64, "bf16", "rms", True, 640, 0.0, "fp32"),
    (640, 64, "fp16", "rms", False, 320, 0.0, "fp16"),
    (33, 67, "fp32", "layer", True, 3, 0.2, "fp32"),
    (33, 515, "bf16", "rms", True, 1, 0.2, "bf16"),
    (1200, 256, "fp32", "layer", True, 2, 0.0, "fp32"),
    (777, 1024, "bf16", "layer", False, 0, 0.1, "bf16"),
    (500, 2048, "bf16", "rms", True, 1, 0.0, "fp32"),
    (40, 4096, "fp16", "layer", True, 4, 0.0, "fp32"),
    (37, 4104, "bf16", "rms", True, 37, 0.1, "bf16"),
    (9, 8192, "fp32", "layer", True, 1, 0.1, "fp32"),
    (5, 8191, "bf16", "layer", True, 5, 0.1, "fp32"),
    (3000, 24, "bf16", "layer", True, 1, 0.0, "fp32"),
    (12000, 32, "bf16", "layer", True, 300, 0.0, "fp32"),
    (3000, 40, "fp16", "rms", False, 30, 0.1, "fp32"),
]


def joint_case(rows, d, dtype, norm, post, gates, p, params, cuda, seed=1):
    g = torch.Generator().manual_seed(rows * 10000 + d)
    dt, pd = TYPES[dtype], TYPES[params]
    layer = norm == "layer"
    t = dict(x=rand(g, rows, d, std=2.0, dtype=dt), y=rand(g, rows, d, std=1.5, mean=0.5, dtype=dt),
             weight=rand(g, d, std=0.2, mean=1.0, dtype=pd), bias=rand(g, d, dtype=pd) if layer else None,
             post_weight=rand(g, d, std=0.2, mean=1.0, dtype=pd) if post else None,
             post_bias=rand(g, d, dtype=pd) if post and layer else None,
             gate=rand(g, gates, d, dtype=dt) if gates else None)
    options = dict(norm=norm, post_norm=post, scale=0.75, eps=1e-5, dropout_p=p, seed=seed, offset=3)
    drop = mask((rows, d), p, seed, 3) if p else None
    on = {k: None if v is None else v.to(cuda) for k, v in t.items()}
    wide = {k: None if v is None else v.double().requires_grad_() for k, v in t.items()}
    return t, on, wide, options, drop, g


@pytest.mark.parametrize("case", JOINTS, ids=lambda c: "-".join(str(v) for v in c))
def test_joint_forward_and_backward(cuda, case):
    rows, d, dtype, norm, post, gates, p, params = case
    t, on, wide, options, drop, g = joint_case(*case, cuda)
    out, normed, stats = layers.residual_norm_forward(**on, **options)
    args = (norm, post, wide["weight"], wide["bias"], wide["post_weight"], wide["post_bias"], wide["gate"], 0.75, 1e-5, drop)
    ref_out, ref_normed = joint_ref(wide["x"], wide["y"], *args)
    assert rel(out, ref_out) <= ONE[dtype]
    # a row of one or two elements under a layer norm is all cancellation: eps and the mean decide it
    assert rel(normed, ref_normed) <= ONE[dtype] * (10 if d < 4 else 1)
    # backward: the formulas from the rounded output that the pass is given
    d_out, d_normed = rand(g, rows, d, dtype=TYPES[dtype]), rand(g, rows, d, dtype=TYPES[dtype])
    o = out.double().cpu().requires_grad_()
    names = ["weight"] + (["bias"] if norm == "layer" else [])

    def pre(a):
        if norm == "layer":
            a = a - a.mean(-1, keepdim=True)
        a = a / (a.pow(2).mean(-1, keepdim=True) + 1e-5).sqrt() * wide["weight"]
        return a if wide["bias"] is None else a + wide["bias"]

    got = layers.residual_norm_grad(d_out.to(cuda), d_normed.to(cuda), out, on["y"], stats, weight=on["weight"],
                                    bias=on["bias"], post_weight=on["post_weight"], post_bias=on["post_bias"],
                                    gate=on["gate"], **options)
    first = torch.autograd.grad(pre(o), [o] + [wide[k] for k in names], d_normed.double())
    dx = first[0] + d_out.double()
    want = dict(zip(["dx"] + ["d" + k for k in names], (dx, *first[1:])))
    rest = ["y"] + [k for k in ("post_weight", "post_bias", "gate") if wide[k] is not None]
    zero = wide["x"].detach() * 0
    added = joint_ref(zero, wide["y"], *args)[0]
    want.update(zip(["d" + k for k in rest], torch.autograd.grad(added, [wide[k] for k in rest], dx)))
    # the statistics are those of the unrounded output: a 16-bit `out` differs from it by one rounding
    slack = 1.0 if dtype == "fp32" else 2.0
    for k, w in want.items():
        v = getattr(got, k)
        kind = dtype if k in ("dx", "dy", "dgate") else (params if params != "fp32" else dtype)
        if norm == "layer" and d < 4:
            continue
        assert rel(v, w) <= max(ONE[kind], 1e-5) * slack, k
    for k in ("dbias", "dpost_weight", "dpost_bias", "dgate"):
        if k not in want:
            assert getattr(got, k) is None


def test_joint_gradients_against_differences(cuda):
    """Central differences of the kernels' own outputs along random directions; step 1e-2: truncation and the fp32
    rounding of the two sums are each below 1e-3 of the slope."""
    case = (24, 72, "fp32", "layer", True, 3, 0.1, "fp32")
    t, on, _, options, _, g = joint_case(*case, cuda)
    a, b = rand(g, 24, 72).to(cuda), rand(g, 24, 72).to(cuda)
    leaves = {k: v.clone().requires_grad_() for k, v in on.items()}
    out, normed = layers.residual_norm(**leaves, **options)
    grads = torch.autograd.grad((out * a).sum() + (normed * b).sum(), list(leaves.values()))

    def value(moved):
        o, n = layers.residual_norm(**moved, **options)
        return ((o.double() * a).sum() + (n.double() * b).sum()).item()

    for (k, v), dv in zip(on.items(), grads):
        u = rand(g, *v.shape).to(cuda)
        slope = (value({**on, k: v + 0.01 * u}) - value({**on, k: v - 0.01 * u})) / 0.02
        want = (dv.double() * u).sum().item()
        size = (dv.double().norm() * u.double().norm()).item()
        assert abs(slope - want) <= 3e-3 * size, k


def test_joint_strides_views_and_missing_gradients(cuda):
    g = torch.Generator().manual_seed(5)
    big = rand(g, 6, 10, 80).to(cuda)
    x, y = big[..., :40], big[:, :, 40:]  # rows 80 apart, read in place
    for dtype, tol in ((torch.float32, 2e-6), (torch.bfloat16, 2.0 ** -9)):
        xs, ys = big.to(dtype)[..., :40], big.to(dtype)[..., 40:]
        out, normed, stats = layers.residual_norm_forward(xs, ys, post_norm=True)
        ref = joint_ref(xs.double().cpu(), ys.double().cpu(), "rms", True, None, None, None, None, None, 1.0, 1e-6, None)
        assert out.shape == (6, 10, 40) and rel(out, ref[0]) <= tol and rel(normed, ref[1]) <= tol
    out, normed, stats = layers.residual_norm_forward(x.transpose(0, 1), y.transpose(0, 1))
    ref = joint_ref(x.double().cpu().transpose(0, 1), y.double().cpu().transpose(0, 1), "rms", False, None, None, None, None,
                    None, 1.0, 1e-6, None)
    assert rel(normed, ref[1]) <= 2e-6
    x, y = x.contiguous(), y.contiguous()
    out, normed, stats = layers.residual_norm_forward(x, y)
    d = rand(g, 6, 10, 40).to(cuda)
    alone = layers.residual_norm_grad(d, None, out, y, stats)
    assert torch.equal(alone.dx, d) and torch.equal(alone.dy, d) and alone.dweight is None
    zero = torch.zeros_like(d)
    assert rel(layers.residual_norm_grad(None, d, out, y, stats).dx,
               layers.residual_norm_grad(zero, d, out, y, stats).dx) == 0.0


@pytest.mark.parametrize("d", [6, 40, 200, 333, 938, 2057, 4104])
@pytest.mark.parametrize("norm", ["rms", "layer"])
def test_joint_without_some_parameters(cuda, d, norm):
    """Missing weights count as ones and missing biases as zeros, wherever a row ends inside a warp."""
    g = torch.Generator().manual_seed(d)
    x, y, up = (rand(g, 9, d, mean=0.3) for _ in range(3))
    names = ["weight", "post_weight"] + (["bias", "post_bias"] if norm == "layer" else [])
    for there in range(1 << len(names)):
        on = {k: rand(g, d, std=0.2, mean=1.0) for i, k in enumerate(names) if there >> i & 1}
        leaves = {k: v.to(cuda).requires_grad_() for k, v in dict(on, x=x, y=y).items()}
        out, normed = layers.residual_norm(norm=norm, post_norm=True, scale=0.5, eps=1e-5, **leaves)
        wide = {k: v.double().requires_grad_() for k, v in dict(on, x=x, y=y).items()}
        ref = joint_ref(wide["x"], wide["y"], norm, True, *(wide.get(k) for k in ("weight", "bias", "post_weight", "post_bias")),
                        None, 0.5, 1e-5, None)
        assert rel(out, ref[0]) <= 2e-6 and rel(normed, ref[1]) <= 2e-6, on.keys()
        got = torch.autograd.grad(normed, list(leaves.values()), up.to(cuda))
        want = torch.autograd.grad(ref[1], list(wide.values()), up.double())
        for k, a, b in zip(leaves, got, want):
            assert rel(a, b) <= 2e-5, (k, on.keys())


@pytest.mark.parametrize("d", [2056, 2057, 3001, 4095, 4100])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_joint_backward_of_long_rows_without_norm_or_gate(cuda, d, dtype):
    """Rows of over 2048 elements, aligned or not, where neither y nor a gate is read."""
    g = torch.Generator().manual_seed(d)
    x, y, up, un = (rand(g, 7, d, dtype=TYPES[dtype]) for _ in range(4))
    w = rand(g, d, std=0.2, mean=1.0)
    out, _, stats = layers.residual_norm_forward(x.to(cuda), y.to(cuda), weight=w.to(cuda))
    got = layers.residual_norm_grad(up.to(cuda), un.to(cuda), out, y.to(cuda), stats, weight=w.to(cuda))
    o, w64 = out.double().cpu().requires_grad_(), w.double().requires_grad_()
    n = o / (o.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * w64
    do, dw = torch.autograd.grad(n, (o, w64), un.double())
    slack = 1.0 if dtype == "fp32" else 2.0
    assert rel(got.dx, do + up.double()) <= ONE[dtype] * slack and rel(got.dy, do + up.double()) <= ONE[dtype] * slack
    assert rel(got.dweight, dw) <= max(ONE[dtype], 1e-5) * slack


@pytest.mark.parametrize("shape", [(4, 1, 24), (4, 6, 24), (1, 1, 24)])
def test_joint_gate_shapes(cuda, shape):
    g = torch.Generator().manual_seed(1)
    x, y, gate, up = (rand(g, *s).to(cuda) for s in ((4, 6, 24), (4, 6, 24), shape, (4, 6, 24)))
    leaves = [v.requires_grad_() for v in (x, y, gate)]
    out, _ = layers.residual_norm(x, y, gate=gate)
    got = torch.autograd.grad(out, leaves, up)
    wide = [v.detach().double().requires_grad_() for v in leaves]
    want = torch.autograd.grad(wide[0] + wide[1] * wide[2], wide, up.double())
    assert all(rel(a, b) <= 2e-6 for a, b in zip(got, want))


def test_joint_empty_and_nonfinite_rows(cuda):
    w = torch.ones(16, device=cuda)
    out, normed, stats = layers.residual_norm_forward(torch.empty(0, 16, device=cuda), torch.empty(0, 16, device=cuda), weight=w)
    got = layers.residual_norm_grad(out, normed, out, out, stats, weight=w)
    assert out.shape == (0, 16) and torch.equal(got.dweight, torch.zeros_like(w))
    x, y = torch.randn(3, 16, device=cuda), torch.randn(3, 16, device=cuda)
    y[1, 4] = float("nan")
    out, normed, _ = layers.residual_norm_forward(x, y, post_norm=True)
    assert torch.isfinite(normed[[0, 2]]).all() and torch.isnan(normed[1]).all()
    z = torch.zeros(2, 16, device=cuda)
    assert torch.equal(layers.residual_norm_forward(z, z, post_norm=True, norm="layer")[1], z)  # eps alone


def test_joint_dropped_infinities_stay_out(cuda):
    """y infinite or NaN exactly where dropout drops it: output, gradients and the gate's gradient are those of zeros there."""
    g = torch.Generator().manual_seed(8)
    keep = mask((40, 72), 0.3, 6, 2) != 0
    x, y, gate, up = (rand(g, 40, 72).to(cuda), rand(g, 40, 72), rand(g, 4, 72).to(cuda), rand(g, 40, 72).to(cuda))
    clean, dirty = (torch.where(keep, y, torch.tensor(v)).to(cuda) for v in (0.0, float("inf")))
    dirty.view(-1)[(~keep).view(-1).nonzero()[::2, 0].to(cuda)] = float("nan")
    got = []
    for v in (clean, dirty):
        options = dict(gate=gate, dropout_p=0.3, seed=6, offset=2)
        out, normed, stats = layers.residual_norm_forward(x, v, **options)
        b = layers.residual_norm_grad(up, up, out, v, stats, **options)
        got.append((out, normed, b.dx, b.dy, b.dgate))
    assert all(torch.equal(a, b) for a, b in zip(*got)) and all(torch.isfinite(t).all() for t in got[1])


def test_second_derivatives_are_refused(cuda):
    x = torch.randn(4, 8, device=cuda, requires_grad=True)
    w = torch.randn(5, 8, device=cuda, requires_grad=True)
    t = torch.zeros(4, dtype=torch.int64, device=cuda)
    for loss in (layers.residual_norm(x, x)[1].sum(), layers.dropout(x, 0.5, 1).sum(), layers.linear_cross_entropy(x, w, t)):
        g, = torch.autograd.grad(loss, x, create_graph=True)
        with pytest.raises(RuntimeError):
            g.sum().backward()


def test_joint_refusals(cuda):
    x, w = torch.ones(4, 16, device=cuda), torch.ones(16, device=cuda)
    f = layers.residual_norm
    for bad in (lambda: f(x, x[:2]), lambda: f(x, x.half()), lambda: f(x.cpu(), x.cpu()), lambda: f(x, x, norm="batch"),
                lambda: f(x, x, weight=w[:8]), lambda: f(x, x, weight=w.half()), lambda: f(x, x, bias=w),
                lambda: f(x, x, post_weight=w), lambda: f(x, x, gate=torch.ones(3, 16, device=cuda)),
                lambda: f(x, x, gate=w.half()), lambda: f(x, x, eps=0.0), lambda: f(x, x, dropout_p=2.0),
                lambda: f(torch.ones(1, 8193, device=cuda), torch.ones(1, 8193, device=cuda)),
                lambda: f(x, x, norm="layer", weight=w, bias=w.bfloat16()),
                lambda: layers.residual_norm_grad(x, x, x, x, torch.ones(4, 3, device=cuda))):
        with pytest.raises(RuntimeError):
            bad()


# ---- the loss --------------------------------------------------------------------------------------------------------
def lce_case(n, d, v, dtype, ignored, cuda, spread=1.5):
    g = torch.Generator().manual_seed(n * 7 + d * 3 + v)
    w = torch.randn(v, d, generator=g) * spread / math.sqrt(d)
    t = torch.randint(0, v, (n,), generator=g)
    h = torch.randn(n, d, generator=g) + torch.rand(n, 1, generator=g) * 6 * w[t]
    t[torch.randperm(n, generator=g)[:int(n * ignored)]] = -100
    h, w = h.to(TYPES[dtype]), w.to(TYPES[dtype])
    return h, w, t


def lce_ref(h, w, t, smoothing=0.0, z=0.0, reduction="mean", grad=None):
    h, w = h.double().cpu().requires_grad_(), w.double().cpu().requires_grad_()
    rows = (t != -100).nonzero()[:, 0]
    logits = h[rows] @ w.T
    lse = logits.logsumexp(1)
    one = (1 - smoothing) * (lse - logits.gather(1, t[rows][:, None])[:, 0])
    one = one + smoothing * (lse - logits.mean(1)) + z * lse * lse
    loss = torch.zeros(t.shape, dtype=torch.float64).index_copy(0, rows, one)
    if reduction != "none":
        loss = loss.sum() / (max(len(rows), 1) if reduction == "mean" else 1)
    up = torch.ones_like(loss) if grad is None else grad.double().cpu()
    return loss.detach(), *torch.autograd.grad(loss, (h, w), up)


LOSSES = [
    # n, d, v, type, ignored, smoothing, z
    (1, 8, 2, "fp32", 0.0, 0.0, 0.0),
    (1, 1, 1, "bf16", 0.0, 0.0, 0.0),
    (5, 16, 10, "bf16", 0.0, 0.1, 0.0),
    (128, 192, 10, "fp32", 0.0, 0.1, 0.0),
    (64, 64, 256, "fp16", 0.0, 0.0, 0.0),
    (65, 72, 257, "bf16", 0.3, 0.0, 1e-3),
    (127, 200, 1000, "fp16", 0.5, 0.1, 1e-3),
    (129, 77, 513, "fp32", 0.5, 0.0, 1e-3),
    (300, 515, 2003, "bf16", 0.1, 0.1, 0.0),
    (513, 264, 5003, "bf16", 0.0, 0.0, 0.0),
    (1025, 520, 4100, "bf16", 0.2, 0.0, 1e-4),
    # few classes and many tokens (dw is split over the tokens), rows that 32-byte stores do not fit, few tokens
    (4100, 136, 10, "bf16", 0.3, 0.0, 0.0),
    (3000, 100, 33, "fp16", 0.9, 0.1, 0.0),
    (2500, 67, 5, "fp32", 0.2, 0.0, 0.0),
    (700, 301, 3001, "bf16", 0.0, 0.0, 0.0),
    (700, 301, 1501, "fp32", 0.0, 0.0, 0.0),
    (3, 1000, 9001, "fp16", 0.0, 0.0, 0.0),
]


@pytest.mark.parametrize("case", LOSSES, ids=lambda c: "-".join(str(v) for v in c))
def test_loss_and_gradients(cuda, case):
    n, d, v, dtype, ignored, smoothing, z = case
    h, w, t = lce_case(n, d, v, dtype, ignored, cuda)
    loss, dh, dw = layers.linear_cross_entropy_grad(h.to(cuda), w.to(cuda), t.to(cuda), label_smoothing=smoothing, z_loss=z)
    want = lce_ref(h, w, t, smoothing, z)
    assert abs(loss.item() - want[0].item()) <= 1e-5 * max(1.0, abs(want[0].item()))
    for got, ref in ((dh, want[1]), (dw, want[2])):
        if ref.norm() > 0:
            assert rel(got, ref) <= PRODUCT[dtype]
        else:
            assert not got.any()
    assert not dh[(t == -100).to(cuda)].any()
    rows = layers.linear_cross_entropy(h.to(cuda), w.to(cuda), t.to(cuda), label_smoothing=smoothing, z_loss=z, reduction="none")
    ref = lce_ref(h, w, t, smoothing, z, "none")[0]
    assert (rows.double().cpu() - ref).abs().max().item() <= 1e-5 * max(1.0, ref.abs().max().item())
    layers.check_errors()


@pytest.mark.parametrize("dtype", list(TYPES))
def test_loss_in_pieces_matches_the_whole(cuda, dtype):
    h, w, t = lce_case(700, 136, 1111, dtype, 0.25, cuda)
    on = [x.to(cuda) for x in (h, w, t)]
    whole = layers.linear_cross_entropy_grad(*on)
    pieces = layers.linear_cross_entropy_grad(*on, piece_bytes=1)  # 256 tokens each; the last one holds no counted row
    want = lce_ref(h, w, t)
    assert abs(whole[0].item() - pieces[0].item()) <= 1e-6 * abs(whole[0].item())
    assert torch.equal(whole[1], pieces[1]) or rel(pieces[1], want[1]) <= PRODUCT[dtype]
    assert rel(pieces[2], want[2]) <= PRODUCT[dtype]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
def test_loss_autograd_with_upstream_gradients(cuda, dtype, reduction):
    h, w, t = lce_case(90, 48, 300, dtype, 0.3, cuda)
    g = torch.Generator().manual_seed(0)
    up = rand(g, 90) * 100 if reduction == "none" else torch.tensor(-3.5)
    a, b = h.to(cuda).requires_grad_(), w.to(cuda).requires_grad_()
    loss = layers.linear_cross_entropy(a, b, t.to(cuda), reduction=reduction, label_smoothing=0.05)
    got = torch.autograd.grad(loss, (a, b), up.to(cuda), retain_graph=True)
    again = torch.autograd.grad(loss, (a, b), up.to(cuda))
    want = lce_ref(h, w, t, 0.05, 0.0, reduction, up)
    assert rel(loss, want[0]) <= 1e-5
    for x, y, ref in zip(got, again, want[1:]):
        assert rel(x, ref) <= PRODUCT[dtype] and torch.equal(x, y)


@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_loss_gradients_of_one_input(cuda, reduction):
    h, w, t = (x.to(cuda) for x in lce_case(300, 72, 500, "bf16", 0.2, cuda))
    up = torch.ones((), device=cuda) if reduction == "mean" else torch.ones(300, device=cuda)
    a, b = h.clone().requires_grad_(), w.clone().requires_grad_()
    both = torch.autograd.grad(layers.linear_cross_entropy(a, b, t, reduction=reduction), (a, b), up)
    dh, = torch.autograd.grad(layers.linear_cross_entropy(a, w, t, reduction=reduction), a, up)
    dw, = torch.autograd.grad(layers.linear_cross_entropy(h, b, t, reduction=reduction), b, up)
    assert torch.equal(dh, both[0]) and torch.equal(dw, both[1])


def test_loss_against_differences(cuda):
    """Central differences of the kernel's fp32 loss along random directions, step 0.02: the loss (about 5) is right to
    1e-6 of itself, so the slope to 2.5e-4; truncation is of that order too."""
    h, w, t = lce_case(40, 24, 130, "fp32", 0.2, cuda)
    h, w, t = h.to(cuda), w.to(cuda), t.to(cuda)
    g = torch.Generator().manual_seed(2)
    _, dh, dw = layers.linear_cross_entropy_grad(h, w, t, z_loss=1e-2, reduction="sum")
    f = lambda a, b: layers.linear_cross_entropy(a, b, t, z_loss=1e-2, reduction="sum").double().item()  # noqa: E731
    for base, grad, at in ((h, dh, 0), (w, dw, 1)):
        u = rand(g, *base.shape).to(cuda)
        u /= u.norm()
        lo, hi = [h, w], [h, w]
        lo[at], hi[at] = base - 0.02 * u, base + 0.02 * u
        slope = (f(*hi) - f(*lo)) / 0.04
        assert abs(slope - (grad.double() * u).sum().item()) <= 0.02 * grad.double().norm().item()


def test_loss_of_nothing(cuda):
    h, w = torch.randn(70, 24, device=cuda), torch.randn(33, 24, device=cuda)
    t = torch.full((70,), -100, device=cuda)
    for h_ in (h, torch.full_like(h, float("nan"))):  # ignored rows are not read
        loss, dh, dw = layers.linear_cross_entropy_grad(h_, w, t)
        assert loss.item() == 0.0 and not dh.any() and not dw.any()
    loss, dh, dw = layers.linear_cross_entropy_grad(h[:0], w, t[:0])
    assert loss.item() == 0.0 and dh.shape == (0, 24) and not dw.any()
    assert layers.linear_cross_entropy(h[:0], w, t[:0], reduction="none").shape == (0,)


def test_loss_ignored_rows_with_nan_and_counted_ones(cuda):
    h, w, t = lce_case(200, 40, 77, "bf16", 0.4, cuda)
    want = layers.linear_cross_entropy_grad(h.to(cuda), w.to(cuda), t.to(cuda))
    dirty = h.clone()
    dirty[t == -100] = float("nan")
    got = layers.linear_cross_entropy_grad(dirty.to(cuda), w.to(cuda), t.to(cuda))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    row = int((t != -100).nonzero()[0, 0])
    h[row, 3] = float("nan")
    rows = layers.linear_cross_entropy(h.to(cuda), w.to(cuda), t.to(cuda), reduction="none")
    assert torch.isnan(rows[row]) and torch.isfinite(rows).sum().item() == 199


def test_loss_extreme_logits(cuda):
    """Logits of +-1e4: one class takes all, or none of 300 that are equal is ahead."""
    h = torch.zeros(4, 16, device=cuda)
    h[:, 0] = torch.tensor([100.0, -100.0, 0.0, 1.0], device=cuda)
    w = torch.zeros(300, 16, device=cuda)
    w[7, 0] = 100.0
    t = torch.tensor([7, 8, 0, 7], device=cuda)
    rows = layers.linear_cross_entropy(h, w, t, reduction="none").double().cpu()
    want = lce_ref(h, w, t.cpu(), reduction="none")[0]
    assert (rows - want).abs().max().item() <= 1e-5 * max(1.0, want.abs().max().item())
    _, dh, dw = layers.linear_cross_entropy_grad(h, w, t)
    ref = lce_ref(h, w, t.cpu())
    assert rel(dh, ref[1]) <= 1e-5 and rel(dw, ref[2]) <= 1e-5


def test_loss_penalty_alone(cuda):
    """One class: p is one and only the log-normaliser's penalty is left, 2 z lse, with z lse from 1e-5 on (in 1 + 2 z lse that
    would be right to 1e-7 / 2e-5 only)."""
    g = torch.Generator().manual_seed(4)
    h, w, t = rand(g, 40, 64, std=0.1), rand(g, 1, 64), torch.zeros(40, dtype=torch.int64)
    _, dh, dw = layers.linear_cross_entropy_grad(h.to(cuda), w.to(cuda), t.to(cuda), z_loss=1e-5)
    want = lce_ref(h, w, t, 0.0, 1e-5)
    assert rel(dh, want[1]) <= 1e-5 and rel(dw, want[2]) <= 1e-5


def test_loss_of_certain_rows(cuda):
    """Targets ahead by 7 to 12: losses of 3e-2 down to 2e-4 at logits of about 34, whose fp32 rounding (of their
    log-normaliser) is 2e-6, a hundredth of the smallest loss. Differences with the maximum are exact here (the logits
    are multiples of 2^-10), so loss and 1 - p are right to the rounding of sums of 1 and small numbers, 6e-8 an addition and 16
    additions at most: 5e-3 of the smallest."""
    v = 50
    h = torch.eye(6, 16, device=cuda)
    ahead = torch.tensor([7.0, 8.0, 9.0, 10.0, 11.0, 12.0])
    w = torch.zeros(v, 16)
    w[:, :6] = 21.5 + (torch.randint(0, 1024, (v, 6), generator=torch.Generator().manual_seed(0)) / 1024)
    for k in range(6):
        w[k, k] = w[:, k].max() + ahead[k]
    t = torch.arange(6)
    rows = layers.linear_cross_entropy(h, w.to(cuda), t.to(cuda), reduction="none").double().cpu()
    want = lce_ref(h, w, t, reduction="none")
    assert ((rows - want[0]).abs() / want[0]).max().item() <= 5e-3
    _, dh, _ = layers.linear_cross_entropy_grad(h, w.to(cuda), t.to(cuda), reduction="none")
    assert ((dh.double().cpu() - want[1]).norm(dim=1) / want[1].norm(dim=1)).max().item() <= 5e-3


def test_loss_strides_shapes_and_alignment(cuda):
    h, w, t = lce_case(96, 40, 150, "bf16", 0.0, cuda)
    want = layers.linear_cross_entropy_grad(h.to(cuda), w.to(cuda), t.to(cuda))
    wide = torch.zeros(96, 51, dtype=torch.bfloat16, device=cuda)
    wide[:, 3:43] = h.to(cuda)
    tall = torch.zeros(150, 43, dtype=torch.bfloat16, device=cuda)
    tall[:, 1:41] = w.to(cuda)
    got = layers.linear_cross_entropy_grad(wide[:, 3:43].view(8, 12, 40), tall[:, 1:41], t.view(8, 12).to(cuda))
    assert got[1].shape == (8, 12, 40)
    assert got[0] == want[0] and torch.equal(got[1].view(96, 40), want[1]) and torch.equal(got[2], want[2])


def test_loss_bad_target_is_reported(cuda):
    h, w = torch.randn(10, 16, device=cuda), torch.randn(20, 16, device=cuda)
    t = torch.arange(10, device=cuda)
    want = layers.linear_cross_entropy(h[1:], w, t[1:])
    for bad in (20, -1):
        t[0] = bad
        try:
            loss = layers.linear_cross_entropy(h, w, t)
            with pytest.raises(RuntimeError):
                layers.check_errors()
            assert loss.item() == pytest.approx(want.item(), rel=1e-6)
        finally:
            layers.reset_errors()


def test_loss_refusals(cuda):
    h, w, t = torch.ones(4, 16, device=cuda), torch.ones(8, 16, device=cuda), torch.zeros(4, dtype=torch.int64, device=cuda)
    f = layers.linear_cross_entropy
    for bad in (lambda: f(h, w[:, :8], t), lambda: f(h, w.half(), t), lambda: f(h.cpu(), w.cpu(), t.cpu()), lambda: f(h, w, t[:3]),
                lambda: f(h, w, t.int()), lambda: f(h, w, t, reduction="median"), lambda: f(h, w, t, label_smoothing=1.5),
                lambda: f(h.int(), w.int(), t), lambda: f(h, w[:0], t),
                lambda: layers.linear_cross_entropy_grad(h, w, t, grad=torch.ones(4, device=cuda)),
                lambda: layers.linear_cross_entropy_grad(h, w, t, reduction="none", grad=torch.ones((), device=cuda))):
        with pytest.raises(RuntimeError):
            bad()


def test_repeated_calls_give_the_same_bits(cuda):
    """No sum depends on the order in which blocks run."""
    h, w, t = (x.to(cuda) for x in lce_case(400, 96, 9000, "bf16", 0.1, cuda))
    first = layers.linear_cross_entropy_grad(h, w, t)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, layers.linear_cross_entropy_grad(h, w, t)))


def test_own_stream_and_graph_capture(cuda):
    h, w, t = (x.to(cuda) for x in lce_case(64, 64, 500, "bf16", 0.1, cuda))
    x, y = torch.randn(32, 64, device=cuda), torch.randn(32, 64, device=cuda)
    rng = torch.tensor([4, 0], device=cuda)
    want = layers.linear_cross_entropy_grad(h, w, t), layers.residual_norm(x, y, dropout_p=0.5, seed=4, offset=1)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = layers.linear_cross_entropy_grad(h, w, t)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want[0]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, dh, dw = layers.linear_cross_entropy_grad(h, w, t)
        out, normed = layers.residual_norm(x, y, dropout_p=0.5, seed=rng)
    rng[1] = 1
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(dh, want[0][1]) and torch.equal(dw, want[0][2])
    assert torch.equal(out, want[1][0]) and torch.equal(normed, want[1][1])
