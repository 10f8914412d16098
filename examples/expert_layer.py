"""A layer of experts, trained and then served, on the products for linear layers.

    python examples/expert_layer.py [--steps 30] [--tokens 512] [--experts 8]

Training: every token goes through a shared expert, two dense products with the
activation and the residual in them, and through its own: a router chooses it and
sorts the tokens by expert for two grouped products with a ReLU between, whose result
is weighted with the router's probability.  A head gives the outputs.  The loss has
the router's balance loss in it; the gradients are clipped to a common norm, and the
experts' and the head's weights move along their orthogonalised momentum.  Serving:
the head and each expert's matrices are brought to 4 bits, and single tokens go
through them; the example prints how far the outputs are from the unquantised
layer's.

Everything stays on the GPU: the groups' offsets are made there and the host never
reads them.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import ozaki_triton_amd as ozk  # noqa: E402


class ExpertLayer:
    def __init__(self, width, hidden, outputs, experts, dtype=torch.bfloat16, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)

        def weight(*size):
            w = torch.randn(*size, generator=g, device="cuda") * size[-2] ** -0.5
            return w.to(dtype).requires_grad_()

        self.router = torch.randn(width, experts, generator=g, device="cuda").requires_grad_()
        self.up = weight(experts, width, hidden)
        self.down = weight(experts, hidden, width)
        # of the shared expert and the head: [out, in], as fused_linear reads them
        self.shared_up = weight(width, hidden).detach().mT.contiguous().requires_grad_()
        self.shared_down = weight(hidden, width).detach().mT.contiguous().requires_grad_()
        self.head = weight(width, outputs).detach().mT.contiguous().requires_grad_()
        self.bias = torch.zeros(outputs, device="cuda", dtype=dtype, requires_grad=True)
        self.momentum = [torch.zeros_like(w) for w in self.weights()]

    def weights(self):
        """Those that move along their orthogonalised momentum."""
        return [self.up, self.down, self.shared_up, self.shared_down, self.head]

    def shared(self, x):
        h = ozk.fused_linear(x, self.shared_up, activation="gelu")
        return ozk.fused_linear(h, self.shared_down, residual=x)

    def __call__(self, x):
        """The outputs and the router's balance loss."""
        r = ozk.route_tokens(x.float() @ self.router, 1, normalize=False)
        h = ozk.grouped_matmul(x[r.order], self.up, r.offsets).relu()
        y = ozk.grouped_matmul(h, self.down, r.offsets)[r.place[:, 0]] * r.weights.to(x.dtype)
        return ozk.fused_linear(self.shared(x) + y, self.head, self.bias), r.balance_loss

    def step(self, x, target, rate):
        y, balance = self(x)
        loss = (y.float() - target).square().mean()
        (loss + 0.01 * balance).backward()
        others = [self.router, self.bias]
        with torch.no_grad():
            ozk.clip_gradients([w.grad for w in self.weights() + others], 1.0)
            for w, m in zip(self.weights(), self.momentum):
                m.mul_(0.9).add_(w.grad)
                w.sub_(ozk.orthogonalize(m), alpha=rate)
            for w in others:
                w.sub_(w.grad, alpha=5 * rate)
            for w in self.weights() + others:
                w.grad = None
        return loss.detach()


class ServedLayer:
    """The same layer with 4-bit weights, for a few tokens at a time."""

    def __init__(self, layer, group_size=64):
        self.layer, self.group_size = layer, group_size
        pack = lambda w: ozk.quantize_w4(w.detach().T, group_size, zeros=True)  # noqa: E731
        self.up = [pack(w) for w in layer.up]
        self.down = [pack(w) for w in layer.down]
        self.head = pack(layer.head.mT)

    def _times(self, x, weights):
        return ozk.matmul_w4(x, *weights, group_size=self.group_size)

    @torch.no_grad()
    def token(self, x, expert):
        """x [1, width], its expert known to the caller (a serving loop batches by it)."""
        y = self._times(self._times(x, self.up[expert]).relu(), self.down[expert])
        p = (x.float() @ self.layer.router).softmax(-1)[:, expert:expert + 1]
        return self._times(self.layer.shared(x) + y * p.to(x.dtype), self.head) + self.layer.bias


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=30)
    ap.add_argument("--tokens", type=int, default=512)
    ap.add_argument("--experts", type=int, default=8)
    a = ap.parse_args(argv)
    layer = ExpertLayer(256, 512, 128, a.experts)
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(a.tokens, 256, generator=g, device="cuda").to(torch.bfloat16)
    target = torch.randn(256, 128, generator=g, device="cuda") / 16
    target = (x.float() @ target).tanh()
    losses = [layer.step(x, target, 0.02) for _ in range(a.steps)]
    losses = [float(v) for v in losses]
    print(f"loss {losses[0]:.4f} -> {losses[-1]:.4f} in {a.steps} steps")

    served = ServedLayer(layer)
    with torch.no_grad():
        whole, _ = layer(x)
    experts = (x.float() @ layer.router).argmax(-1)[:8].tolist()
    got = torch.cat([served.token(x[i:i + 1], e) for i, e in enumerate(experts)])
    off = float((got.float() - whole[:8].float()).norm() / whole[:8].float().norm())
    print(f"8 tokens on 4-bit weights: {off:.3f} of the outputs' norm from the trained layer's")
    return losses, off


if __name__ == "__main__":
    main()
