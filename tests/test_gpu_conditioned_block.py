"""The example block end to end: served, against the same block from plain
operations in 64 bits, and fine-tuned, whose loss falls."""
import os
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


def plain(block, x, states, lengths):
    import conditioned_block as cb

    def norm(t, w, b):
        s = t.reshape(t.shape[0], -1, cb.GROUPS, t.shape[-1] // cb.GROUPS)
        mean, var = s.mean((1, 3), keepdim=True), s.var((1, 3), keepdim=True, unbiased=False)
        return ((s - mean) / (var + 1e-5).sqrt()).reshape(t.shape) * w.double() + b.double()

    silu = torch.nn.functional.silu
    h = x.double()
    for k, conv in enumerate(block.plain_convs):
        z = silu(norm(h, *block.norms[k])).permute(0, 3, 1, 2)
        h = torch.nn.functional.conv2d(z, conv[0].double(), conv[1].double(), padding=1).permute(0, 2, 3, 1)
    h = h + x.double()
    n, c = h.shape[0], h.shape[-1]
    q = (norm(h, *block.norms[2]).reshape(n, -1, c) @ block.query.double()).unflatten(2, (cb.HEADS, -1))
    k, v = ((states.double() @ t.double()).unflatten(2, (cb.HEADS, -1)) for t in (block.key, block.value))
    out = torch.zeros(n, q.shape[1], c, dtype=torch.float64, device=x.device)
    for i, length in enumerate(lengths.tolist()):
        if length:
            s = torch.einsum("qhd,khd->hqk", q[i], k[i, :length]) * q.shape[-1] ** -0.5
            out[i] = torch.einsum("hqk,khd->qhd", torch.softmax(s, -1), v[i, :length]).flatten(1)
    return h + (out @ block.out.double()).reshape(h.shape)


def test_served_block_matches_plain_operations(cuda_device):
    import conditioned_block as cb

    x, states, lengths = cb.inputs(24)
    block = cb.Block()
    g = torch.Generator().manual_seed(0)  # the block's own weights, drawn in its order
    draw = lambda *s: torch.randn(*s, generator=g).to(cuda_device)  # noqa: E731
    for _ in range(6):
        draw(cb.CHANNELS)
    block.plain_convs = []
    for _ in range(2):
        w = draw(3, 3, cb.CHANNELS, cb.CHANNELS) * (1 / (9 * cb.CHANNELS)) ** 0.5
        block.plain_convs.append((w.permute(3, 2, 0, 1), 0.1 * draw(cb.CHANNELS)))
    with torch.no_grad():
        got = block.condition(block.features(x), states, lengths)
    exact = plain(block, x, states, lengths)
    # float16 operands at every stage: the convolutions' tolerance, 1e-2, over the whole map
    assert ((got.double() - exact).norm() / exact.norm()).item() <= 1e-2
    assert torch.equal(got, cb.serve(24))


def test_fine_tuning_lowers_the_loss(cuda_device):
    import conditioned_block as cb
    import rdv_project_b200 as rdv

    losses = cb.train(size=16, steps=25)
    assert losses[-1] < 0.7 * losses[0] and all(b == b for b in losses)
    assert losses == cb.train(size=16, steps=25)  # the same bits every time
    assert rdv.device_status() == 0
