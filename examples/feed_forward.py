"""A pre-norm feed-forward block, dense or with experts, trained and then used
for single tokens.

    y = x + act(norm(x) W1 + b1) W2 + b2

Every product, norm and gradient is a call of phptensors; torch holds the
memory, sorts the tokens by expert and applies the updates.

    python examples/feed_forward.py            # on a B200
"""
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                "php-gpu-tensors_b200"))
import phptensors as P  # noqa: E402

arr = P.CudaArray.from_torch


class Block:
    """experts = 0 is the dense layer; otherwise W1, b1, W2, b2 have a leading
    axis of experts, and each token uses the one its router names."""

    def __init__(self, width, hidden, experts=0, dtype=torch.bfloat16, activation="gelu_tanh",
                 seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        lead = [experts] if experts else []

        def weight(a, b):
            return (torch.randn(*lead, a, b, generator=g, device="cuda") * a ** -0.5).to(dtype)
        self.experts, self.activation = experts, activation
        self.params = {"gamma": torch.ones(width, device="cuda", dtype=dtype),
                       "beta": torch.zeros(width, device="cuda", dtype=dtype),
                       "w1": weight(width, hidden), "w2": weight(hidden, width),
                       "b1": torch.zeros(*lead, hidden, device="cuda", dtype=dtype),
                       "b2": torch.zeros(*lead, width, device="cuda", dtype=dtype)}

    def _sorted(self, x, expert):
        """Rows in the order of their experts, the order, and the groups' ends."""
        if not self.experts:
            return x, None, None
        order = torch.argsort(expert, stable=True)
        ends = torch.bincount(expert, minlength=self.experts).cumsum(0).to(torch.int32)
        return x[order], order, ends

    def forward(self, x, expert=None, train=False):
        """y for rows x; with `train` also what backward needs."""
        p = {k: arr(v) for k, v in self.params.items()}
        x, order, ends = self._sorted(x, expert)
        xa = arr(x)
        h, mean, rstd = xa.layer_norm(p["gamma"], p["beta"], save_stats=True)
        first = dict(bias=p["b1"], activation=self.activation, save_pre=train)
        if ends is None:
            u = h.linear(p["w1"], **first)
        else:
            u = h.grouped_linear(p["w1"], ends, **first)
        u, pre = u if train else (u, None)
        if ends is None:
            y = u.linear(p["w2"], p["b2"], residual=xa)
        else:
            y = u.grouped_linear(p["w2"], ends, p["b2"], residual=xa)
        y = y.to_torch()
        if order is not None:
            y = torch.empty_like(y).index_copy_(0, order, y)
        return (y, (xa, h, mean, rstd, u, pre, order, ends)) if train else y

    def backward(self, grad, kept):
        """Gradients of the parameters and of x."""
        xa, h, mean, rstd, u, pre, order, ends = kept
        p = {k: arr(v) for k, v in self.params.items()}
        g = arr(grad if order is None else grad[order])
        if ends is None:
            du, dw2, db2 = P.linear_backward(g, u, p["w2"])
            dh, dw1, db1 = P.linear_backward(du, h, p["w1"], pre, self.activation)
        else:
            du, dw2, db2 = P.grouped_linear_backward(g, u, p["w2"], ends)
            dh, dw1, db1 = P.grouped_linear_backward(du, h, p["w1"], ends, pre, self.activation)
        dx, dgamma, dbeta = P.layer_norm_backward(dh, xa, p["gamma"], mean, rstd)
        dx = dx.to_torch() + g.to_torch()                 # the residual's gradient is g
        if order is not None:
            dx = torch.empty_like(dx).index_copy_(0, order, dx)
        grads = {"gamma": dgamma, "beta": dbeta, "w1": dw1, "b1": db1, "w2": dw2, "b2": db2}
        return dx, {k: v.to_torch() for k, v in grads.items()}

    def step(self, x, target, rate, expert=None):
        """One step of gradient descent on the mean square error; the loss."""
        y, kept = self.forward(x, expert, train=True)
        diff = y.float() - target.float()
        grad = (diff * (2.0 / diff.numel())).to(y.dtype)
        _, grads = self.backward(grad, kept)
        for k, v in self.params.items():
            v.sub_((grads[k].float() * rate).to(v.dtype))
        return diff.square().mean()


def main(tokens=4096, width=1024, hidden=4096, experts=8, steps=20):
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(tokens, width, generator=g, device="cuda").bfloat16()
    target = torch.randn(tokens, width, generator=g, device="cuda").bfloat16()
    expert = torch.randint(experts, (tokens,), generator=g, device="cuda")
    losses = {}
    for name, block, route in (("dense", Block(width, hidden), None),
                               ("experts", Block(width, hidden, experts), expert)):
        losses[name] = [block.step(x, target, 1.0, route).item() for _ in range(steps)]
        print("%-8s loss %.4f -> %.4f" % (name, losses[name][0], losses[name][-1]))
        # serving: eight single tokens give what the whole batch gave them
        few = block.forward(x[:8], None if route is None else route[:8])
        whole = block.forward(x, route)[:8]
        print("%-8s eight tokens alone: largest difference %.3g"
              % (name, (few.float() - whole.float()).abs().max().item()))
    return losses


if __name__ == "__main__":
    main()
