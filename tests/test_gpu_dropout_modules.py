"""Modules that drop values, several of them in one network."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_modules_at_their_defaults_drop_different_values():
    """Four modules over 20000 values each, p = 0.5.  Two masks that are independent agree in half of the values; 6 standard deviations of that are 6 sqrt(20000 / 4) = 425."""
    from fgms_b200 import nn
    x, w = torch.ones((100, 200), device="cuda"), torch.ones(200, device="cuda")
    drops = [nn.Dropout(0.5), nn.Dropout(0.5)]
    norms = [nn.RMSNorm(200, dropout=0.5), nn.RMSNorm(200, dropout=0.5)]
    masks = []
    for _ in range(2):  # two steps
        masks += [d(x) != 0 for d in drops] + [n(x, torch.zeros_like(x))[1].detach() != 0 for n in norms]
    for i in range(8):
        for j in range(i):
            assert abs((masks[i] == masks[j]).sum().item() - 10000) < 425, (i, j)
    torch.manual_seed(7)
    a = nn.Dropout(0.5)
    torch.manual_seed(7)
    b = nn.Dropout(0.5)
    assert torch.equal(a(x), b(x))


@pytest.mark.parametrize("states", ["module", "tensors"])
def test_a_segment_that_is_computed_again_drops_the_same_values(states):
    """Gradients with and without checkpoints are the same bits: two segments of a network, one state shared by both."""
    from torch.utils.checkpoint import checkpoint

    from fgms_b200 import nn
    gen = torch.Generator(device="cuda").manual_seed(5)
    normal = lambda *s: torch.randn(s, generator=gen, device="cuda").bfloat16()
    x, res, dy, dh = (normal(60, 136) for _ in range(4))
    shared = nn.rng_state(11)

    class Block(torch.nn.Module):
        def __init__(self, seed):
            super().__init__()
            self.norm, self.drop = nn.RMSNorm(136, dropout=0.3, seed=seed), nn.Dropout(0.5, seed=seed + 1)

        def forward(self, x, res):
            y, h = self.norm(x, res)
            return nn.dropout(self.drop(y), 0.25, shared, residual=h), h

    blocks = [Block(20), Block(30)]
    rngs = [shared] + [m.rng for b in blocks for m in (b.norm, b.drop)]
    leaves = [x.requires_grad_(), res.requires_grad_()] + [b.norm.weight for b in blocks]
    start = [r.clone() for r in rngs]

    def step(through):
        a, b = x, res
        for block in blocks:
            a, b = through(block, a, b)
        return a.detach(), b.detach(), torch.autograd.grad((a, b), leaves, (dy, dh))

    def again(block, a, b):
        of = (block, shared) if states == "module" else (shared, block.norm.rng, block.drop.rng)
        return checkpoint(block, a, b, use_reentrant=False, preserve_rng_state=False, context_fn=lambda: nn.recomputed(*of))

    for _ in range(2):  # the second step goes on from the calls of the first
        want = step(lambda block, a, b: block(a, b))
        after = [r.clone() for r in rngs]
        for r, s in zip(rngs, start):
            r.copy_(s)
        got = step(again)
        assert all(torch.equal(g, w) for g, w in zip((got[0], got[1], *got[2]), (want[0], want[1], *want[2])))
        assert all(torch.equal(r, s) for r, s in zip(rngs, after))
        start = after
    for r, s in zip(rngs, start):
        r.copy_(s)
    eager = step(again)
    for r, s in zip(rngs, start):
        r.copy_(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(again)
    graph.replay()
    assert all(torch.equal(g, w) for g, w in zip((got[0], got[1], *got[2]), (eager[0], eager[1], *eager[2])))


def test_a_graph_gone_through_twice():
    """What is computed again is computed again as often as it is asked for."""
    from torch.utils.checkpoint import checkpoint

    from fgms_b200 import nn
    x, drop = torch.ones((40, 80), device="cuda", requires_grad=True), nn.Dropout(0.5, seed=3)
    y = checkpoint(lambda v: drop(v).square(), x, use_reentrant=False, context_fn=lambda: nn.recomputed(drop))
    drop(x)  # another call in between
    grads = [torch.autograd.grad(y.sum(), x, retain_graph=True)[0] for _ in range(2)]
    assert torch.equal(grads[0], grads[1]) and torch.equal(grads[0], torch.where(y > 0, 8.0, 0.0)) and drop.rng.tolist() == [3, 2, 0]
