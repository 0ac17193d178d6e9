"""A conditioned image block, served and fine-tuned.

    python examples/conditioned_block.py [--size 64] [--steps 30]

The block refines a batch of feature maps [N, H, W, 64] (a noisy render's, say)
under an encoder's states [N, L, 64] of another length, some samples' shorter
than others and one sample's dropped altogether:

    h = conv(group norm + silu(x));  h = x + dropout(conv(group norm + silu(h)))
    y = h + project(cross attention(queries of group norm(h), keys and values of the states))

serve() runs it in float16 with the framework's convolutions, norms and
attention. train() keeps the convolutions frozen (they have no gradient) and
fits the conditioning branch -- the norm's affine parameters and the four
projections -- to a target by gradient descent, in bfloat16 with float32
parameters; the norm, the attention and the dropout record themselves for
torch's autograd."""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import rdv_project_b200 as rdv  # noqa: E402

CHANNELS, HEADS, GROUPS = 64, 4, 8


class Block:
    def __init__(self, seed=0, device="cuda"):
        g = torch.Generator().manual_seed(seed)

        def rand(*shape, scale=1.0):
            return (torch.randn(*shape, generator=g) * scale).to(device)

        c = CHANNELS
        self.norms = [(1 + 0.1 * rand(c), 0.1 * rand(c)) for _ in range(3)]
        self.convs = [rdv.Conv3x3Winograd(rand(3, 3, c, c, scale=(1 / (9 * c)) ** 0.5), 0.1 * rand(c)) for _ in range(2)]
        self.query, self.key, self.value, self.out = (rand(c, c, scale=c ** -0.5) for _ in range(4))

    def features(self, x, p=0.0, seed=0):
        """The residual branch: x [N, H, W, 64] float16."""
        h = self.convs[0](rdv.group_norm(x, GROUPS, *self.norms[0], activation="silu"), out_dtype=torch.float16)
        h = self.convs[1](rdv.group_norm(h, GROUPS, *self.norms[1], activation="silu"), out_dtype=torch.float16)
        return rdv.dropout(h, p, seed, residual=x)

    def condition(self, h, states, lengths):
        """The conditioning branch, in h's type."""
        n, height, width, c = h.shape
        heads = (HEADS, c // HEADS)
        w = [t.to(h.dtype) for t in (self.query, self.key, self.value, self.out)]
        z = rdv.group_norm(h, GROUPS, *self.norms[2]).reshape(n, -1, c)
        q = (z @ w[0]).unflatten(2, heads)
        k, v = (states.to(h.dtype) @ t for t in w[1:3])
        a = rdv.cross_attention(q, k.unflatten(2, heads), v.unflatten(2, heads), lengths=lengths)
        return h + (a.flatten(2) @ w[3]).reshape(h.shape)


def inputs(size, seed=1, device="cuda"):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(4, size, size, CHANNELS, generator=g).to(device, torch.float16)
    states = torch.randn(4, 77, CHANNELS, generator=g).to(device)
    return x, states, torch.tensor([77, 40, 1, 0], dtype=torch.int32, device=device)


def serve(size=64):
    block = Block()
    x, states, lengths = inputs(size)
    with torch.no_grad():
        return block.condition(block.features(x), states, lengths)


def train(size=32, steps=30):
    """Losses of `steps` steps toward another block's conditioning."""
    block, target_block = Block(), Block(seed=5)
    x, states, lengths = inputs(size)
    with torch.no_grad():
        h = block.features(x).bfloat16()
        target = target_block.condition(h, states, lengths)
    block.norms[2] = tuple(t.requires_grad_() for t in block.norms[2])
    params = [block.query, block.key, block.value, block.out]
    for t in params:
        t.requires_grad_()
    opt = torch.optim.Adam([*params, *block.norms[2]], lr=3e-3)
    losses = []
    counters = (h.numel() + 3) // 4
    for step in range(steps):
        opt.zero_grad()
        noisy = rdv.dropout(h, 0.05, seed=11, offset=step * counters)  # the next mask of one stream
        loss = (block.condition(noisy, states, lengths) - target).float().square().mean()
        loss.backward()
        opt.step()
        losses.append(loss.item())
    return losses


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--size", type=int, default=64)
    ap.add_argument("--steps", type=int, default=30)
    a = ap.parse_args()
    y = serve(a.size)
    print(f"served {tuple(y.shape)}, mean {y.float().mean().item():.4f}, deviation {y.float().std().item():.4f}")
    losses = train(min(a.size, 32), a.steps)
    print(f"trained {a.steps} steps: loss {losses[0]:.4f} -> {losses[-1]:.4f}")


if __name__ == "__main__":
    main()
