"""The model-side operators together, under autograd and with the optimizer, as examples/train_layers.py runs them."""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu
PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "train_layers.py")


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("train_layers", PATH)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def plain_loss(model, p, tokens, target):
    """The example's loss without dropout in fp64 torch, from parameters p by name."""
    norm = lambda a, w: a / (a.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * w  # noqa: E731
    x = p["embed"][tokens]
    normed = norm(x, p["first"])
    for k in range(len(model.blocks)):
        q = {n.rsplit(".", 1)[1]: v for n, v in p.items() if n.startswith(f"blocks.{k}.")}
        before = torch.nn.functional.pad(normed[:, :-1], (0, 0, 1, 0))
        y = torch.relu(torch.cat([normed, before], -1) @ q["up"].t()) @ q["down"].t()
        x = x + q["gate"] * norm(y, q["post"])
        normed = norm(x, q["pre"])
    return torch.nn.functional.cross_entropy((normed @ p["head"].t()).flatten(0, 1), target.flatten())


def test_gradients_of_the_whole_model(cuda, example):
    """Every parameter's fp32 gradient against fp64 autograd of the same model: the products of the blocks are torch's own
    in fp32 (1e-6 each, a dozen in a row), so 1e-4 bounds them all."""
    model = example.Model(vocabulary=101, d=40, hidden=64, blocks=2, dropout=0.0, dtype=torch.float32)
    tokens, target = example.batch(101, 4, 17, torch.Generator().manual_seed(3))
    loss = model(tokens, target, 0)
    grads = torch.autograd.grad(loss, list(model.parameters()))
    p = {n: v.detach().double().requires_grad_() for n, v in model.named_parameters()}
    ref = plain_loss(model, p, tokens, target)
    want = torch.autograd.grad(ref, list(p.values()))
    assert abs(loss.item() - ref.item()) <= 1e-5 * ref.item()
    for (name, _), a, b in zip(model.named_parameters(), grads, want):
        assert (a.double() - b).norm() <= 1e-4 * b.norm(), name


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_the_example_learns(cuda, example, dtype):
    first, last = example.train(steps=60, dtype=dtype, say=lambda _: None)
    assert last < 0.8 * first


def test_scalar_loss_upstream_gradients(cuda):
    """The gradients held from the forward pass: scaled by the upstream gradient, formed anew by a second pass."""
    from psgd_pro_b200 import layers
    g = torch.Generator().manual_seed(0)
    h, w = (torch.randn(*s, generator=g).to(cuda).requires_grad_() for s in ((50, 24), (90, 24)))
    t = torch.randint(0, 90, (50,), generator=g).to(cuda)
    loss = layers.linear_cross_entropy(h, w, t)
    one = torch.autograd.grad(loss, (h, w), retain_graph=True)
    kept = [x.clone() for x in one]
    three = torch.autograd.grad(3.0 * loss, (h, w), retain_graph=True)
    again = torch.autograd.grad(loss, (h, w))
    assert all(torch.equal(a, b) for a, b in zip(one, kept))
    assert all((a - 3 * b).norm() <= 1e-6 * a.norm() for a, b in zip(three, kept))
    assert all(torch.equal(a, b) for a, b in zip(again, kept))
    eighth = torch.autograd.grad(0.125 * layers.linear_cross_entropy(h, w, t), (h, w))
    assert all(torch.equal(a, 0.125 * b) for a, b in zip(eighth, kept))
