"""The dense operators together, as a token or map trunk uses them: layer norm, expansion with GELU, projection joined to
the residual, backward, gradients clipped, an optimizer step.  Every operator is checked on the values that reached it,
with its own test's bounds."""
import pytest
import torch

import test_gradclip as clip
import test_layernorm as norm
import test_linear as linear

F32, BF16 = torch.float32, torch.bfloat16


class Block(torch.nn.Module):
    def __init__(self, width, hidden):
        super().__init__()
        self.norm = torch.nn.LayerNorm(width)
        self.up, self.down = torch.nn.Linear(width, hidden), torch.nn.Linear(hidden, width)

    def forward(self, x, seen=None):
        from vfdepth_amd import layers
        h = layers.layer_norm(self.norm, x)
        u = layers.linear_act(self.up, h, 'gelu')
        y = layers.linear_act(self.down, u, 'none', x)
        if seen is not None:
            seen.update(h=h, u=u, y=y)
            for t in (h, u, y):
                t.retain_grad()
        return y


@pytest.mark.gpu
@pytest.mark.parametrize('amp', [False, True])
def test_block_step(amp):
    from vfdepth_amd import kernels as KN
    torch.manual_seed(0)
    blk = Block(96, 200).cuda()
    opt = torch.optim.SGD(blk.parameters(), lr=0.1)
    dt = BF16 if amp else F32
    x = torch.randn(2, 6, 25, 96, device='cuda').to(dt).requires_grad_(True)
    g = torch.randn(2, 6, 25, 96, device='cuda').to(dt)
    seen = {}
    with torch.autocast('cuda', dtype=BF16, enabled=amp):
        y = blk(x, seen)
    y.backward(g)
    flat = lambda t: t.detach().reshape(-1, t.shape[-1])  # noqa: E731
    cast = lambda t: t.detach().to(dt)  # noqa: E731
    h, u = seen['h'], seen['u']
    vals, tol = linear._oracle(flat(u), cast(blk.down.weight), cast(blk.down.bias), flat(x), flat(g), 'none')
    linear._check([flat(y), flat(u.grad), cast(blk.down.weight.grad), cast(blk.down.bias.grad)], vals, tol)
    vals, tol = linear._oracle(flat(h), cast(blk.up.weight), cast(blk.up.bias), None, flat(u.grad), 'gelu')
    linear._check([flat(u), flat(h.grad), cast(blk.up.weight.grad), cast(blk.up.bias.grad)], vals, tol)
    vals, tol = norm._oracle(flat(x), blk.norm.weight, blk.norm.bias, flat(h.grad))
    norm._check([flat(h), None, blk.norm.weight.grad, blk.norm.bias.grad], vals, tol)
    # x's gradient: the norm's and the residual's, added by autograd in x's type
    want, lim = vals[1] + flat(g).cpu().double(), tol[1] + 2 * norm.HALF[dt] * (vals[1].abs() + flat(g).cpu().double().abs())
    assert bool(((flat(x.grad).cpu().double() - want).abs() <= lim).all())
    # clip and step
    before = {k: p.detach().clone() for k, p in blk.named_parameters()}
    n, clipped = clip._oracle([p.grad for p in blk.parameters()], 0.05)
    got = KN.clip_grad_norm_(blk.parameters(), 0.05)
    assert n > 0.05 and abs(float(got) - n) <= 2.0 ** -24 * n * (1 + 1e-6)
    for p, c in zip(blk.parameters(), clipped):
        clip._near(p.grad, c, 2 * 2.0 ** -24 * (1 + 1e-6))
    opt.step()
    for (k, p), c in zip(blk.named_parameters(), clipped):
        ref = before[k].cpu().double() - 0.1 * c
        assert bool(((p.detach().cpu().double() - ref).abs() <= 2.0 ** -22 * (before[k].cpu().double().abs() + 0.1 * c.abs())).all())


@pytest.mark.gpu
def test_block_step_captured():
    """The whole step in a graph: the same values as the eager step on every replay, with eager steps between."""
    from vfdepth_amd import kernels as KN
    torch.manual_seed(1)
    blk = Block(64, 160).cuda()
    ps = list(blk.parameters())
    x, g = torch.randn(300, 64, device='cuda'), torch.randn(300, 64, device='cuda')

    def step():
        grads = torch.autograd.grad(blk(x), ps, g)
        return KN.clip_grads(grads, 0.5), grads
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm_, grads = step()
    for k in range(4):
        x.copy_(torch.randn(300, 64, generator=torch.Generator().manual_seed(k)))
        graph.replay()
        torch.cuda.synchronize()
        want_n, want = step()
        assert torch.equal(norm_, want_n) and all(torch.equal(a, b) for a, b in zip(grads, want))
