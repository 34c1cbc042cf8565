"""Cases that time and check the model-side training operators of psgd_pro_b200.layers: the joint between two blocks of
a network (residual_norm), counter-based dropout (dropout) and the vocabulary loss with its gradients
(linear_cross_entropy).

`own` False computes them in a plain form (elementary torch operations in fp32, rounded once at the end); `own` True
calls the package. A case is a dict of plain values; prepare() makes what a training program holds before the call,
run() is one pass through one operator, work() the bytes and operations that the pass cannot do without and exact()
the same outputs in fp64.

Formulas
  linear_cross_entropy: l = h w^T; per token n with target t (rows whose target is IGNORE count nothing)
      lse = log sum_v exp l_v;  loss_n = lse - (1 - s) l_t - s mean_v l_v + z lse^2
      d loss_n / d l_v = (1 + 2 z lse) exp(l_v - lse) - (1 - s) [v = t] - s / V
      mean: the sum over counted tokens divided by their number (at least 1); dh = g w, dw = g^T h
  residual_norm: u = post(y) (a norm, or y itself), k = dropout(u), out = x + scale gate k, normed = pre(out);
      rms: a / sqrt(mean a^2 + eps) weight;  layer: (a - mean a) / sqrt(var a + eps) weight + bias
  dropout: element i keeps its value / (1 - T / 65536), T = round(65536 p), when 16-bit field i % 8 of the
      Philox4x32-10 block (i / 8, offset) under key seed is at least T; else it is zero
"""
import math

import numpy as np
import torch

own = False

IGNORE = -100
EPS = 1e-6
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


# ---- the cases -------------------------------------------------------------------------------------------------------
def _lce(name, n, d, v, dtype, direction, ignored=0.0, smoothing=0.0, z=0.0):
    return {"name": name, "op": "lce", "n": n, "d": d, "v": v, "dtype": dtype, "direction": direction,
            "ignored": ignored, "smoothing": smoothing, "z": z}


def _joint(name, rows, d, dtype, direction, kind, post, gate, p, params):
    return {"name": name, "op": "joint", "rows": rows, "d": d, "dtype": dtype, "direction": direction, "kind": kind,
            "post": post, "gate": gate, "p": p, "params": params}


def _drop(name, n, dtype, direction, p, residual):
    return {"name": name, "op": "dropout", "n": n, "dtype": dtype, "direction": direction, "p": p,
            "residual": residual}


def listed():
    return [
        # the classifier head of the ViT-Tiny set on one batch of images: ten classes, fp32, with label smoothing; all
        # latency
        _lce("lce_classes_fp32", 128, 192, 10, "fp32", "train", smoothing=0.1),
        # one packed context of the GPT-2-medium set: odd vocabulary (50257), tied head in bf16
        _lce("lce_gpt2_bf16", 1024, 1024, 50257, "bf16", "train"),
        # a training micro-batch of the Llama-style set (4 sequences of 2048), a quarter of the tokens prompt or
        # padding, with the log-normaliser's penalty: the largest case
        _lce("lce_llama_bf16", 8192, 2048, 32000, "bf16", "train", ignored=0.25, z=1e-4),
        # evaluation of the Llama-style set: per-token losses, no gradients
        _lce("lce_llama_eval_bf16", 4096, 2048, 32000, "bf16", "eval"),
        # fp32 training of a small head, odd sizes everywhere
        _lce("lce_odd_fp32", 1001, 515, 5003, "fp32", "train", ignored=0.1),
        # a block joint of the ViT-Tiny set: 65 positions of one image, fp32 layer norm, pre-norm form
        _joint("joint_vit_fp32", 65, 192, "fp32", "forward", "layer", False, 0, 0.0, "fp32"),
        # a block joint of the Llama-style set with norms on both sides and a gate per channel, bf16 with fp32 weights
        _joint("joint_llama_bf16", 8192, 2048, "bf16", "forward", "rms", True, 1, 0.0, "fp32"),
        # and its backward pass
        _joint("joint_llama_bf16_bwd", 8192, 2048, "bf16", "backward", "rms", True, 1, 0.0, "fp32"),
        # the GPT-2-medium set's joint in training: residual dropout, layer norm with bias; backward pass, 16 contexts
        _joint("joint_gpt2_bf16_bwd", 16384, 1024, "bf16", "backward", "layer", False, 0, 0.1, "bf16"),
        # embedding dropout of one short fp32 sequence: all latency
        _drop("dropout_small_fp32", 65 * 192, "fp32", "forward", 0.1, False),
        # hidden activations of the Llama-style set's feed-forward layer: 8192 tokens of 5632, dropout and residual add
        _drop("dropout_ffn_bf16", 8192 * 5632, "bf16", "forward", 0.1, True),
        # backward pass over an odd number of fp16 values
        _drop("dropout_odd_fp16_bwd", 16384 * 1024 + 3, "fp16", "backward", 0.25, False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["lce", "joint", "dropout"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "lce":
        while True:
            n, v, d = _log(rng, 1, 8192), _log(rng, 2, 50257), _log(rng, 16, 4096)
            if n * v * d <= 6144 * 32000 * 2048 and n * v <= 8192 * 32000:
                break
        if rng.random() < 0.7:
            d = max(16, d // 16 * 16)
        c = _lce("", n, d, v, dtype, rng.choice(["train", "train", "eval"]), ignored=rng.choice([0.0, 0.1, 0.5]),
                 smoothing=rng.choice([0.0, 0.0, 0.1]), z=rng.choice([0.0, 1e-4]))
    elif op == "joint":
        d = _log(rng, 8, 8192)
        if rng.random() < 0.8:
            d = max(8, d // 8 * 8)
        rows = _log(rng, 1, max(1, 16384 * 1024 // d))
        gates = [0, 1, rows] + [g for g in (2, 4, 8) if rows % g == 0]
        c = _joint("", rows, d, dtype, rng.choice(["forward", "backward"]), rng.choice(["rms", "layer"]),
                   rng.random() < 0.5, rng.choice(gates), rng.choice([0.0, 0.0, 0.1]), rng.choice([dtype, "fp32"]))
    else:
        direction = rng.choice(["forward", "backward"])
        c = _drop("", _log(rng, 1, 8192 * 5632), dtype, direction, rng.choice([0.05, 0.1, 0.25, 0.5]),
                  direction == "forward" and rng.random() < 0.5)
    del c["name"]
    return c


def work(case):
    e = SIZE[case["dtype"]]
    if case["op"] == "lce":
        n, d, v = case["n"], case["d"], case["v"]
        counted = n - int(n * case["ignored"])
        train = case["direction"] == "train"
        matrices = counted * d * e + v * d * e  # the counted rows of h, and w
        bytes_ = matrices + 8 * n + ((n * d + v * d) * e + 4 if train else 4 * n)
        return {"bytes": bytes_, "flops": (6 if train else 2) * counted * v * d}
    if case["op"] == "joint":
        rows, d, g = case["rows"], case["d"], case["gate"]
        wb = SIZE[case["params"]] * d * ((2 if case["kind"] == "layer" else 1) * (2 if case["post"] else 1))
        if case["direction"] == "forward":  # x, y in; out, normed and the statistics out
            return {"bytes": 4 * rows * d * e + wb + g * d * e + 16 * rows, "flops": 12 * rows * d}
        # d_out, d_normed, out in and d_x, d_y out; y only where a norm or a gate needs it; the parameters' gradients out
        reads_y = 1 if case["post"] or g else 0
        return {"bytes": (5 + reads_y) * rows * d * e + 2 * wb + 2 * g * d * e + 16 * rows, "flops": 24 * rows * d}
    moved = 3 if case["residual"] else 2
    return {"bytes": moved * case["n"] * e, "flops": 2 * case["n"]}


# ---- what a program holds before the call ----------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def randn(*shape, std=1.0, mean=0.0, dtype=dt):
        t = torch.randn(*shape, generator=g, device="cuda")
        return t.mul_(std).add_(mean).to(dtype)

    s = {"case": case}
    if case["op"] == "lce":
        n, d, v = case["n"], case["d"], case["v"]
        # logits of spread 1.5, and a share of each token's state along its target's row, so that the target's
        # probability runs from chance to almost one as in a partly trained model
        w = torch.randn(v, d, generator=g, device="cuda").mul_(1.5 / math.sqrt(d))
        t = torch.randint(0, v, (n,), generator=g, device="cuda")
        a = torch.rand(n, 1, generator=g, device="cuda").mul_(6.0)
        h = torch.randn(n, d, generator=g, device="cuda").addcmul_(a, w[t])
        t[torch.randperm(n, generator=g, device="cuda")[:int(n * case["ignored"])]] = IGNORE
        s.update(h=h.to(dt), w=w.to(dt), t=t)
    elif case["op"] == "joint":
        rows, d, pd = case["rows"], case["d"], DTYPES[case["params"]]
        s.update(x=randn(rows, d, std=2.0), y=randn(rows, d), w=randn(d, std=0.1, mean=1.0, dtype=pd), b=None,
                 pw=None, pb=None, gate=None, scale=0.5, seed=seed, offset=seed % 7)
        if case["kind"] == "layer":
            s["b"] = randn(d, std=0.1, dtype=pd)
        if case["post"]:
            s["pw"] = randn(d, std=0.1, mean=1.0, dtype=pd)
            s["pb"] = randn(d, std=0.1, dtype=pd) if case["kind"] == "layer" else None
        if case["gate"]:
            s["gate"] = randn(case["gate"], d, std=0.3, mean=0.5)
        if case["direction"] == "backward":  # x is the joint's output here; its statistics are kept by the forward pass
            s["d_out"], s["d_normed"] = randn(rows, d), randn(rows, d)
            s["stats"] = torch.cat([*_stats(s["y"].float(), case["kind"]), *_stats(s["x"].float(), case["kind"])], 1)
    else:
        s.update(x=randn(case["n"]), r=randn(case["n"]) if case["residual"] else None, seed=seed, offset=seed % 5)
    return s


# ---- one pass --------------------------------------------------------------------------------------------------------
def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    from psgd_pro_b200 import layers
    c = s["case"]
    if c["op"] == "lce":
        options = dict(ignore_index=IGNORE, label_smoothing=c["smoothing"], z_loss=c["z"])
        if c["direction"] == "eval":
            return layers.linear_cross_entropy(s["h"], s["w"], s["t"], reduction="none", **options)
        loss, dh, dw = layers.linear_cross_entropy_grad(s["h"], s["w"], s["t"], **options)
        return {"loss": loss, "dh": dh, "dw": dw}
    if c["op"] == "joint":
        options = dict(norm=c["kind"], post_norm=c["post"], weight=s["w"], bias=s["b"], post_weight=s["pw"],
                       post_bias=s["pb"], gate=s["gate"], scale=s["scale"], eps=EPS, dropout_p=c["p"], seed=s["seed"],
                       offset=s["offset"])
        if c["direction"] == "forward":
            out, normed, stats = layers.residual_norm_forward(s["x"], s["y"], **options)
            return {"out": out, "normed": normed}
        return layers.residual_norm_grad(s["d_out"], s["d_normed"], s["x"], s["y"], s["stats"], **options)._asdict()
    if c["direction"] == "forward":
        return layers.dropout(s["x"], c["p"], s["seed"], s["offset"], residual=s["r"])
    return layers.dropout_grad(s["x"], c["p"], s["seed"], s["offset"])


def _run_plain(s):
    c = s["case"]
    dt = DTYPES[c["dtype"]]
    if c["op"] == "lce":
        return _plain_lce(s, c, dt)
    if c["op"] == "joint":
        return _plain_joint(s, c, dt) if c["direction"] == "forward" else _plain_joint_backward(s, c, dt)
    keep, scale = _keep(c["n"], c["p"], s["seed"], s["offset"])
    out = torch.where(keep, s["x"].float() * scale, 0.0)
    return (out if s["r"] is None else s["r"].float() + out).to(dt)


def _plain_lce(s, c, dt):
    h, w, t = s["h"].float(), s["w"].float(), s["t"]
    smooth, z = c["smoothing"], c["z"]
    counted = t != IGNORE
    at = torch.where(counted, t, 0)[:, None]
    logits = h @ w.T
    top = logits.max(dim=1, keepdim=True).values
    e = torch.exp(logits - top)
    total = e.sum(dim=1, keepdim=True)
    lse = top + torch.log(total)
    loss = lse - (1.0 - smooth) * logits.gather(1, at) + z * lse * lse
    if smooth:
        loss = loss - smooth * logits.mean(dim=1, keepdim=True)
    loss = torch.where(counted, loss[:, 0], 0.0)
    if c["direction"] == "eval":
        return loss
    share = 1.0 / counted.sum().clamp(min=1).float()
    g = e.mul_((1.0 + 2.0 * z * lse) / total)
    if smooth:
        g -= smooth / c["v"]
    g.scatter_add_(1, at, torch.full_like(lse, smooth - 1.0))
    g *= (counted.float() * share)[:, None]
    return {"loss": loss.sum() * share, "dh": (g @ w).to(dt), "dw": (g.T @ h).to(dt)}


def _stats(a, kind):
    """(mean, 1 / deviation) of each row, as columns; the mean of an rms norm is zero."""
    mean = a.mean(dim=1, keepdim=True) if kind == "layer" else torch.zeros_like(a[:, :1])
    return mean, torch.rsqrt(((a - mean) ** 2).mean(dim=1, keepdim=True) + EPS)


def _affine(a, weight, bias):
    a = a * weight.float()
    return a if bias is None else a + bias.float()


def _groups(s, a):
    """The gate in fp32 with a row for each row of a (each of its rows serves as many rows in a row)."""
    gate = s["gate"].float()
    return gate.repeat_interleave(a.shape[0] // gate.shape[0], dim=0)


def _plain_joint(s, c, dt):
    x, u = s["x"].float(), s["y"].float()
    if c["post"]:
        mean, r = _stats(u, c["kind"])
        u = _affine((u - mean) * r, s["pw"], s["pb"])
    if c["p"]:
        keep, k = _keep(u.numel(), c["p"], s["seed"], s["offset"])
        u = torch.where(keep.view_as(u), u * k, 0.0)
    if s["gate"] is not None:
        u = u * _groups(s, u)
    out = x + s["scale"] * u
    mean, r = _stats(out, c["kind"])
    return {"out": out.to(dt), "normed": _affine((out - mean) * r, s["w"], s["b"]).to(dt)}


def _norm_backward(dy, a, mean, r, weight, kind):
    """Gradients of a norm's input, weight and bias: a its input, r = 1 / deviation."""
    hat = (a - mean) * r
    dhat = dy * weight.float()
    inner = dhat - hat * (dhat * hat).mean(dim=1, keepdim=True)
    if kind == "layer":
        inner = inner - dhat.mean(dim=1, keepdim=True)
    return r * inner, (dy * hat).sum(dim=0), dy.sum(dim=0)


def _plain_joint_backward(s, c, dt):
    kind, pd = c["kind"], DTYPES[c["params"]]
    mean_y, r_y, mean_o, r_o = s["stats"].split(1, dim=1)
    y, layer = s["y"].float(), kind == "layer"
    da, dw, db = _norm_backward(s["d_normed"].float(), s["x"].float(), mean_o, r_o, s["w"], kind)
    dx = s["d_out"].float() + da
    got = {"dx": dx.to(dt), "dy": None, "dweight": dw.to(pd), "dbias": db.to(pd) if layer else None,
           "dpost_weight": None, "dpost_bias": None, "dgate": None}
    du = s["scale"] * dx
    keep, k = _keep(y.numel(), c["p"], s["seed"], s["offset"]) if c["p"] else (None, 1.0)
    if s["gate"] is not None:
        u = _affine((y - mean_y) * r_y, s["pw"], s["pb"]) if c["post"] else y
        u = torch.where(keep.view_as(u), u * k, 0.0) if c["p"] else u
        got["dgate"] = (du * u).view(c["gate"], -1, c["d"]).sum(dim=1).to(dt)
        du = du * _groups(s, du)
    if c["p"]:
        du = torch.where(keep.view_as(du), du * k, 0.0)
    if c["post"]:
        du, dpw, dpb = _norm_backward(du, y, mean_y, r_y, s["pw"], kind)
        got["dpost_weight"], got["dpost_bias"] = dpw.to(pd), dpb.to(pd) if layer else None
    got["dy"] = du.to(dt)
    return got


# ---- the counter-based generator -------------------------------------------------------------------------------------
def _mul(a, b):
    """High and low 32 bits of a constant times 32-bit values held in 64 bits."""
    low = a * (b & 0xFFFF)
    high = a * (b >> 16) + (low >> 16)
    return high >> 16, ((high & 0xFFFF) << 16) | (low & 0xFFFF)


def _philox(c0, c1, c2, c3, k0, k1):
    for _ in range(10):
        h0, l0 = _mul(0xD2511F53, c0)
        h1, l1 = _mul(0xCD9E8D57, c2)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return c0, c1, c2, c3


def _keep(n, p, seed, offset):
    """Which of n elements stay, and the scale of those that do."""
    threshold = int(round(p * 65536))
    block = torch.arange(-(-n // 8), device="cuda")
    zero = torch.zeros_like(block)
    words = torch.stack(_philox(block & 0xFFFFFFFF, block >> 32, zero + (offset & 0xFFFFFFFF), zero + (offset >> 32),
                                seed & 0xFFFFFFFF, seed >> 32), dim=1)
    fields = torch.stack([words & 0xFFFF, words >> 16], dim=2).view(-1)[:n]
    return fields >= threshold, 65536.0 / (65536 - threshold)


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "lce":
        h, w = s["h"].double(), s["w"].double()
        train = case["direction"] == "train"
        h.requires_grad_(train), w.requires_grad_(train)
        rows = (s["t"] != IGNORE).nonzero()[:, 0]
        logits = torch.nn.functional.linear(h[rows], w)
        lse = logits.logsumexp(1)
        one = (lse - logits[torch.arange(len(rows), device="cuda"), s["t"][rows]]) * (1 - case["smoothing"])
        one = one + case["smoothing"] * (lse - logits.sum(1) / case["v"]) + case["z"] * lse.square()
        if not train:
            return torch.zeros(case["n"], dtype=torch.float64, device="cuda").index_copy(0, rows, one)
        loss = one.sum() / max(len(rows), 1)
        dh, dw = torch.autograd.grad(loss, (h, w))
        return {"loss": loss.detach(), "dh": dh, "dw": dw}
    if case["op"] == "joint":
        return _exact_joint(s, case)
    keep = _exact_keep(case["n"], case["p"], s["seed"], s["offset"])
    out = s["x"].double() * keep
    return out if s["r"] is None else out + s["r"].double()


def _exact_keep(n, p, seed, offset):
    """0 or the scale for each element, in 64 bits; the generator in unsigned whole numbers on the host."""
    low = np.uint64(0xFFFFFFFF)
    at = np.arange(-(-n // 8), dtype=np.uint64)
    c = [at & low, at >> np.uint64(32), np.full_like(at, offset & 0xFFFFFFFF), np.full_like(at, offset >> 32)]
    k = [seed & 0xFFFFFFFF, seed >> 32]
    for _ in range(10):
        p0, p1 = np.uint64(0xD2511F53) * c[0], np.uint64(0xCD9E8D57) * c[2]
        c = [(p1 >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), p1 & low,
             (p0 >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), p0 & low]
        k = [(k[0] + 0x9E3779B9) % 2 ** 32, (k[1] + 0xBB67AE85) % 2 ** 32]
    fields = np.stack(c, axis=1).astype("<u4").view("<u2").reshape(-1)[:n]
    threshold = int(round(p * 65536))
    return torch.from_numpy(fields >= threshold).cuda().double() / (1.0 - threshold / 65536.0)


def _exact_joint(s, case):
    names = ("x", "y", "w", "b", "pw", "pb", "gate")
    v = {k: s[k].double().requires_grad_() for k in names if s[k] is not None}

    def norm(a, weight, bias):
        if case["kind"] == "layer":
            a = a - a.mean(-1, keepdim=True)
        a = a / (a.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * weight
        return a if bias is None else a + bias

    u = norm(v["y"], v["pw"], v.get("pb")) if case["post"] else v["y"]
    if case["p"]:
        u = u * _exact_keep(u.numel(), case["p"], s["seed"], s["offset"]).view_as(u)
    if "gate" in v:
        u = (u.view(case["gate"], -1, case["d"]) * v["gate"][:, None]).view_as(u)
    add = s["scale"] * u
    if case["direction"] == "forward":
        out = v["x"] + add
        return {"out": out.detach(), "normed": norm(out, v["w"], v.get("b")).detach()}
    # the backward pass starts from the joint's output (x): its gradient, then the gradients through what was added
    normed = norm(v["x"], v["w"], v.get("b"))
    first = [k for k in ("x", "w", "b") if k in v]
    got = dict(zip(first, torch.autograd.grad(normed, [v[k] for k in first], s["d_normed"].double())))
    dx = got["x"] + s["d_out"].double()
    second = [k for k in ("y", "pw", "pb", "gate") if k in v]
    got.update(zip(second, torch.autograd.grad(add, [v[k] for k in second], dx)))
    return {"dx": dx, "dy": got["y"], "dweight": got["w"], "dbias": got.get("b"), "dpost_weight": got.get("pw"),
            "dpost_bias": got.get("pb"), "dgate": got.get("gate")}
