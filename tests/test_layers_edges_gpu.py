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


def test_sizes_beyond_the_index_arithmetic_are_refused(cuda):
    """Not taken modulo 2^32, which four billion rows (expanded ones here: no memory) would be on their way to the kernels."""
    one = torch.zeros(1, 1, device=cuda)
    many, targets = one.expand((1 << 32) + 3, 1), torch.zeros(1, dtype=torch.int64, device=cuda).expand((1 << 32) + 3)
    for h, w, t in ((many, one, targets), (one, many, targets[:1])):
        with pytest.raises(RuntimeError, match="rows"):
            layers.linear_cross_entropy(h, w, t)


# ---- upstream gradients by row ---------------------------------------------------------------------------------------
def by_rows_bounds(h, w, t, up, smoothing, z):
    """What may be lost of dh's rows and of dw's, in 64 bits: the kept exponentials rounded once to fp16 (2^-11 of p's part of
    g), g once more (2^-11 of a value, or the 2^-25 of what is below the type's range, at 2^8 times g), a hundredth of that
    for the fp32 arithmetic in between, and each value of the result rounded once to fp16."""
    rows = (t != -100).nonzero()[:, 0]
    h, w, up = h.double()[rows], w.double(), up.double()[rows]
    logits = h @ w.T
    lse = logits.logsumexp(1)
    part = (logits - lse[:, None]).exp() * (1 + 2 * z * lse)[:, None]
    g = (part - smoothing / w.shape[0]).scatter_add_(1, t[rows][:, None], torch.full_like(lse, smoothing - 1)[:, None])
    dg = (1.01 * 2.0 ** -11 * (g.abs() + part.abs()) + 2.0 ** -32) * up.abs()[:, None]
    dh, dw = (g * up[:, None]) @ w, (g * up[:, None]).T @ h
    off_h = dg @ w.abs() + dh.abs() * 2.0 ** -11 + 2.0 ** -24
    off_w = dg.T @ h.abs() + dw.abs() * 2.0 ** -11 + 2.0 ** -24
    return rows, dh, dw, off_h, off_w


@pytest.mark.parametrize("n,d,v,pieces", [(300, 264, 2003, False), (300, 264, 2003, True), (2500, 72, 300, False), (700, 301, 1003, True)])
def test_fp16_losses_by_row_with_upstream_gradients_of_all_sizes(cuda, n, d, v, pieces):
    """Rows do not affect each other: upstream gradients over 24 binary orders, zeros among them, and every value of dh and dw
    within what the roundings to fp16 take."""
    h, w, t = lce_case(n, d, v, "fp16", 0.2, cuda)
    g = torch.Generator(device="cuda").manual_seed(n)
    up = torch.randn(n, generator=g, device=cuda) * 2.0 ** (torch.rand(n, generator=g, device=cuda) * 24 - 16)
    up[::17] = 0.0
    _, dh, dw = layers.linear_cross_entropy_grad(h, w, t, grad=up, reduction="none", label_smoothing=0.05, z_loss=1e-3,
                                                 **({"piece_bytes": 1} if pieces else {}))
    rows, want_h, want_w, off_h, off_w = by_rows_bounds(h, w, t, up, 0.05, 1e-3)
    assert ((dh.double()[rows] - want_h).abs() <= off_h).all()
    assert ((dw.double() - want_w).abs() <= off_w).all()
    assert not dh[t == -100].any() and not dh[::17].any()
    a, b = h.clone().requires_grad_(), w.clone().requires_grad_()
    loss = layers.linear_cross_entropy(a, b, t, reduction="none", label_smoothing=0.05, z_loss=1e-3)
    again = torch.autograd.grad(loss, (a, b), up)
    if not pieces:
        assert torch.equal(again[0], dh) and torch.equal(again[1], dw)
    layers.check_errors()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_an_infinite_upstream_gradient_stays_in_its_row(cuda, dtype, bad):
    h, w, t = lce_case(300, 264, 2003, dtype, 0.2, cuda)
    up = torch.linspace(0.5, 2.0, 300, device=cuda)
    row = int((t != -100).nonzero()[7, 0])
    want = layers.linear_cross_entropy_grad(h, w, t, grad=up, reduction="none")
    up[row] = bad
    _, dh, dw = layers.linear_cross_entropy_grad(h, w, t, grad=up, reduction="none")
    others = torch.arange(300, device=cuda) != row
    assert torch.equal(dh[others], want[1][others]) and not torch.isfinite(dh[row]).any() and not torch.isfinite(dw).any()


def test_fp16_losses_by_row_of_nothing(cuda):
    """All upstream gradients zero, or none of the rows counted."""
    h, w, t = lce_case(300, 264, 2003, "fp16", 0.2, cuda)
    for up, target in ((torch.zeros(300, device=cuda), t), (torch.ones(300, device=cuda), torch.full_like(t, -100))):
        _, dh, dw = layers.linear_cross_entropy_grad(h, w, target, grad=up, reduction="none")
        assert not dh.any() and not dw.any()


# ---- where other kernels, tiles and launches of the loss begin ---------------------------------------------------------
UNIT = {"fp32": 5e-6, "bf16": 2.0 ** -8, "fp16": 2.0 ** -11}  # one rounding of a value (fp32: limbs and truncated sums)


def check_rows(dtype, h, w, t, got, smoothing, z, reduction="mean", grad=None):
    """dh and dw row by row: the roundings of g, at most a unit of a value each and independent of one another, and of the
    result. fp16 rounds twice on the way to g (kept exponentials) and has 2^-25 where values are below its range (2^-33 in g)."""
    loss, dh, dw = lce_ref(h, w, t, smoothing, z, reduction, grad)
    rows = (t != -100).nonzero()[:, 0]
    H, W = h.double()[rows], w.double()
    logits = H @ W.T
    lse = logits.logsumexp(1)
    g = (logits - lse[:, None]).exp() * (1 + 2 * z * lse)[:, None]
    part = g.abs().clone()
    g = (g - smoothing / W.shape[0]).scatter_add_(1, t[rows][:, None], torch.full_like(lse, smoothing - 1)[:, None]).abs() + part
    up = torch.ones(len(rows), dtype=torch.float64, device=h.device) if grad is None else \
        (grad.double()[rows] if reduction == "none" else grad.double().expand(len(rows)))
    g *= (up.abs() / (max(len(rows), 1) if reduction == "mean" else 1))[:, None]
    u, low = UNIT[dtype] * (2 if dtype == "fp16" else 1), 2.0 ** -25 if dtype == "fp16" else 0.0

    def within(a, ref, spread):
        off = (a.double() - ref).norm(dim=1)
        few = low * (math.sqrt(ref.shape[1]) + spread.max())
        return bool((off <= u * (spread + ref.norm(dim=1)) + few).all())

    assert within(got[1][rows], dh[rows], (g.square() @ W.square().sum(1)).sqrt())
    assert within(got[2], dw, (g.T.square() @ H.square().sum(1)).sqrt())
    assert rel(got[1], dh) <= PRODUCT[dtype] and rel(got[2], dw) <= PRODUCT[dtype]
    assert not got[1][t == -100].any()
    assert ((got[0].double() - loss).abs() <= 1e-5 * loss.abs().clamp_min(1.0)).all()


@pytest.mark.parametrize("case", [
    # n, d, v, type, ignored, smoothing, z: logits in tiles of 256 columns from 148 of them on, and sums over several
    # accumulators (16-bit types: depths over 1024; limbs: over 512), with remainders everywhere
    (2100, 1100, 4500, "bf16", 0.2, 0.0, 1e-3),
    (1300, 1090, 8200, "fp16", 0.1, 0.1, 0.0),
    (300, 700, 2003, "fp32", 0.1, 0.1, 1e-3),
    # the gradients' tiles of 256 columns too; without splits; of aligned rows
    (2100, 1100, 8200, "bf16", 0.0, 0.1, 0.0),
    (2309, 1301, 9001, "fp16", 0.3, 0.0, 1e-4),
    (2304, 2048, 8192, "bf16", 0.0, 0.0, 0.0),
    # a plan of its own launch (over 2048 tokens) with few classes, and its second turn (over 65536)
    (2049, 24, 1003, "bf16", 0.5, 0.0, 0.0),
    (65537, 16, 20, "fp32", 0.3, 0.0, 1e-3),
    (140003, 8, 40, "bf16", 0.5, 0.1, 0.0),
    # one token, and a token more than a tile
    (1, 520, 9001, "bf16", 0.0, 0.0, 0.0),
    (257, 96, 300, "fp16", 0.0, 0.0, 1e-3),
], ids=lambda c: "-".join(str(x) for x in c))
def test_loss_where_its_kernels_change(cuda, case):
    n, d, v, dtype, ignored, smoothing, z = case
    h, w, t = lce_case(n, d, v, dtype, ignored, cuda)
    options = dict(label_smoothing=smoothing, z_loss=z)
    got = layers.linear_cross_entropy_grad(h, w, t, **options)
    check_rows(dtype, h, w, t, got, smoothing, z)
    rows = layers.linear_cross_entropy(h, w, t, reduction="none", **options)
    ref = lce_ref(h, w, t, smoothing, z, "none")[0]
    assert ((rows.double() - ref).abs() <= 1e-5 * ref.abs().clamp_min(1.0)).all()
    assert abs(layers.linear_cross_entropy(h, w, t, **options).item() - got[0].item()) <= 1e-6 * abs(got[0].item())
    layers.check_errors()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("ignored", [0.25, 0.5, 0.9])
def test_loss_in_pieces_of_which_some_are_empty(cuda, dtype, ignored):
    """Pieces of 256 tokens of 700: 525, 350 and 70 counted rows, so one, one and two pieces short of rows, of which the second
    and third case leave the last one and the last two without any."""
    h, w, t = lce_case(700, 136, 1111, dtype, ignored, cuda)
    options = dict(label_smoothing=0.1, z_loss=1e-3, piece_bytes=1)
    up = torch.randn(700, generator=torch.Generator(device="cuda").manual_seed(1), device=cuda)
    for reduction, grad in (("mean", None), ("sum", torch.tensor(-0.25, device=cuda)), ("none", up)):
        got = layers.linear_cross_entropy_grad(h, w, t, reduction=reduction, grad=grad, **options)
        check_rows(dtype, h, w, t, got, 0.1, 1e-3, reduction, grad)
        alone = layers.linear_cross_entropy(h, w, t, reduction=reduction, **options)
        assert ((alone - got[0]).abs() <= 1e-6 * got[0].abs().clamp_min(1.0)).all()
    layers.check_errors()


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_only_the_kept_exponentials_and_g_are_rounded_on_the_way(cuda, dtype):
    """What a 16-bit gradient differs by from its formula is the rounding of exp(l - max) of 64 columns to fp16, of g to the
    inputs' type, and its own. With the first two formed in 64 bits, what is left is fp32 arithmetic: sums off by up to 1e-4 of
    themselves, which rounds one value in 40 the other way (2e-4 of the 2^-7 between neighbours in bf16). So 95 of 100 values are
    the right rounding (98 to 99.8 measured; of the formula itself six to eight of ten are)."""
    h, w, t = lce_case(600, 264, 2003, dtype, 0.0, cuda)
    _, dh, dw = layers.linear_cross_entropy_grad(h, w, t)
    H, W = h.double(), w.double()
    logits = H @ W.T
    lse = logits.logsumexp(1, keepdim=True)
    top = torch.cat([c.amax(1, keepdim=True).expand_as(c) for c in logits.split(64, 1)], 1)
    p = ((logits - top).exp() * 2.0 ** 15).half().double() * 2.0 ** -15 * (top - lse).exp()
    g = p.scatter(1, t[:, None], torch.expm1(logits.gather(1, t[:, None]) - lse))
    scale = 256.0 if dtype == "fp16" else 1.0
    g = (g * scale).to(TYPES[dtype]).double() / (scale * 600)
    for got, want in ((dh, g @ W), (dw, g.T @ H)):
        assert (got == want.to(TYPES[dtype])).double().mean().item() >= 0.95


def test_saved_tensor_hooks_and_checkpointing(cuda):
    """What the backward passes need goes through autograd's hooks, and a recomputed forward pass gives the same gradients."""
    from torch.autograd.graph import save_on_cpu
    from torch.utils.checkpoint import checkpoint
    h, w, t = lce_case(60, 48, 500, "bf16", 0.2, cuda)
    rng = torch.tensor([4, 9], device=cuda)
    leaves = [v.clone().requires_grad_() for v in (h, torch.randn_like(h), torch.ones(48, device=cuda, dtype=h.dtype), w)]

    def model(x, y, weight, head):
        x = layers.dropout(x, 0.2, rng)
        x, normed = layers.residual_norm(x, y, post_norm=True, weight=weight, dropout_p=0.2, seed=rng)
        return layers.linear_cross_entropy(normed, head, t) + layers.linear_cross_entropy(normed, head, t, reduction="none").sum()

    want = torch.autograd.grad(model(*leaves), leaves)
    with save_on_cpu():
        loss = model(*leaves)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(loss, leaves), want))
    for reentrant in (True, False):
        again = [v.detach().clone().requires_grad_() for v in leaves]
        checkpoint(model, *again, use_reentrant=reentrant).backward()
        assert all(torch.equal(a.grad, b) for a, b in zip(again, want))
    seen = []
    x = leaves[0].detach().clone().requires_grad_()
    y = layers.dropout(x, 0.2, rng)
    y.register_hook(lambda g: seen.append(1) or 2 * g)
    got, = torch.autograd.grad(model(y, *leaves[1:]), x)
    assert seen == [1] and torch.isfinite(got).all()


def test_fp16_losses_by_row_of_one_input_and_in_a_graph(cuda):
    """Either gradient alone has the bits of both together, and a captured call those of a launched one, for other upstream
    gradients too."""
    h, w, t = lce_case(600, 136, 1003, "fp16", 0.2, cuda)
    up = torch.randn(600, device=cuda) * torch.logspace(-3, 3, 600, device=cuda)
    want = layers.linear_cross_entropy_grad(h, w, t, grad=up, reduction="none")
    a, b = h.clone().requires_grad_(), w.clone().requires_grad_()
    dh, = torch.autograd.grad(layers.linear_cross_entropy(a, w, t, reduction="none"), a, up)
    dw, = torch.autograd.grad(layers.linear_cross_entropy(h, b, t, reduction="none"), b, up)
    assert torch.equal(dh, want[1]) and torch.equal(dw, want[2])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = layers.linear_cross_entropy_grad(h, w, t, grad=up, reduction="none")
    for turn in range(2):
        graph.replay()
        want = layers.linear_cross_entropy_grad(h, w, t, grad=up, reduction="none")
        assert all(torch.equal(x, y) for x, y in zip(got, want))
        up.copy_(up.flip(0) * 3)
