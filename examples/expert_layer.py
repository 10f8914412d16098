"""A layer of experts, trained and then served, on the products for linear layers.

    python examples/expert_layer.py [--steps 30] [--tokens 512] [--experts 8]

Training: a router sends every token to its best expert; the tokens are sorted by
expert and go through two grouped products with a ReLU between, a head gives the
outputs.  The experts' and the head's weights move along their orthogonalised
momentum.  Serving: the head and each expert's matrices are brought to 4 bits, and
single tokens go through them; the example prints how far the outputs are from the
unquantised layer's.

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

        self.router = torch.randn(width, experts, generator=g, device="cuda")   # fixed
        self.up = weight(experts, width, hidden)
        self.down = weight(experts, hidden, width)
        self.head = weight(1, width, outputs)
        self.momentum = [torch.zeros_like(w) for w in self.weights()]

    def weights(self):
        return [self.up, self.down, self.head]

    def __call__(self, x):
        expert = (x.float() @ self.router).argmax(-1)
        order = expert.argsort(stable=True)
        ends = torch.bincount(expert, minlength=self.router.shape[1]).cumsum(0)
        offsets = torch.nn.functional.pad(ends, (1, 0))
        h = ozk.grouped_matmul(x[order], self.up, offsets).relu()
        y = torch.empty_like(x).index_copy(0, order, ozk.grouped_matmul(h, self.down, offsets))
        whole = torch.tensor([0, x.shape[0]], device=x.device)
        return ozk.grouped_matmul(x + y, self.head, whole)

    def step(self, x, target, rate):
        loss = (self(x).float() - target).square().mean()
        loss.backward()
        with torch.no_grad():
            for w, m in zip(self.weights(), self.momentum):
                m.mul_(0.9).add_(w.grad)
                w.sub_(ozk.orthogonalize(m), alpha=rate)
                w.grad = None
        return loss.detach()


class ServedLayer:
    """The same layer with 4-bit weights, for a few tokens at a time."""

    def __init__(self, layer, group_size=64):
        self.router, self.group_size = layer.router, group_size
        pack = lambda w: ozk.quantize_w4(w.detach().T, group_size, zeros=True)  # noqa: E731
        self.up = [pack(w) for w in layer.up]
        self.down = [pack(w) for w in layer.down]
        self.head = pack(layer.head[0])

    def _times(self, x, weights):
        return ozk.matmul_w4(x, *weights, group_size=self.group_size)

    @torch.no_grad()
    def token(self, x, expert):
        """x [1, width], its expert known to the caller (a serving loop batches by it)."""
        y = self._times(self._times(x, self.up[expert]).relu(), self.down[expert])
        return self._times(x + y, self.head)


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
        whole = layer(x)
    experts = (x.float() @ layer.router).argmax(-1)[:8].tolist()
    got = torch.cat([served.token(x[i:i + 1], e) for i, e in enumerate(experts)])
    off = float((got.float() - whole[:8].float()).norm() / whole[:8].float().norm())
    print(f"8 tokens on 4-bit weights: {off:.3f} of the outputs' norm from the trained layer's")
    return losses, off


if __name__ == "__main__":
    main()
