"""The feed-forward block of examples/feed_forward.py, whose calls run the norm,
linear and grouped layers together, against float64 autograd.

Each stored activation and gradient is rounded to bfloat16 (2^-8); a gradient
passes through at most six such roundings, so its norm is within 6 2^-8.
"""
import os
import sys

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
TOL = 6 * 2.0 ** -8


def example():
    sys.path.insert(0, os.path.join(ROOT, "examples"))
    import feed_forward
    return feed_forward


def reference(block, x, expert):
    """The block in float64 on autograd leaves."""
    p = {k: v.double().requires_grad_() for k, v in block.params.items()}
    x = x.double().requires_grad_()
    F = torch.nn.functional
    h = F.layer_norm(x, x.shape[1:], p["gamma"], p["beta"], 1e-5)
    if expert is None:
        u = F.gelu(h @ p["w1"] + p["b1"], approximate="tanh")
        return x + u @ p["w2"] + p["b2"], x, p
    z = torch.einsum("td,tdh->th", h, p["w1"][expert]) + p["b1"][expert]
    u = F.gelu(z, approximate="tanh")
    return x + torch.einsum("th,thd->td", u, p["w2"][expert]) + p["b2"][expert], x, p


@pytest.mark.parametrize("experts", [0, 5])
def test_block_against_autograd(experts):
    E = example()
    g = torch.Generator(device="cuda").manual_seed(4)
    block = E.Block(96, 264, experts)
    x = torch.randn(333, 96, generator=g, device="cuda").bfloat16()
    grad = torch.randn(333, 96, generator=g, device="cuda").bfloat16()
    expert = None
    if experts:
        expert = torch.randint(experts - 1, (333,), generator=g, device="cuda")  # one gets none
    y, kept = block.forward(x, expert, train=True)
    dx, grads = block.backward(grad, kept)
    want, leaf, p = reference(block, x, expert)
    want.backward(grad.double())
    assert (y.double() - want).norm() <= TOL * want.norm()
    assert (dx.double() - leaf.grad).norm() <= TOL * leaf.grad.norm()
    for k in grads:
        assert (grads[k].double() - p[k].grad).norm() <= TOL * p[k].grad.norm(), k
        if experts and k[0] in "wb" and k[-1] in "12":
            assert not grads[k][experts - 1].any()


def test_example_learns():
    losses = example().main(tokens=512, width=128, hidden=512, experts=4, steps=8)
    for v in losses.values():      # a rate below 2 over the curvature, 0.16 hidden / width
        assert v[-1] < v[0]
