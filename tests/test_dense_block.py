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


class Map(torch.nn.Module):
    """The map forms: channel norm, 1x1 convolution with activation and residual."""

    def __init__(self, width):
        super().__init__()
        self.norm, self.conv = torch.nn.LayerNorm(width), torch.nn.Conv2d(width, width, 1)

    def forward(self, x):
        from vfdepth_amd import layers
        return layers.linear_act(self.conv, layers.channel_norm(self.norm, x), 'silu', x)


def _plain_block(m, x):
    f = torch.nn.functional
    if isinstance(m, Block):
        return m.down(f.gelu(m.up(m.norm(x)))) + x
    return f.silu(m.conv(m.norm(x.permute(0, 2, 3, 1)).permute(0, 3, 1, 2))) + x


def _recorded_cases():
    return [(Block(24, 40).cuda(), (5, 24)), (Map(16).cuda(), (2, 16, 3, 4))]


@pytest.mark.gpu
@pytest.mark.parametrize('grad', [False, True])
def test_traced_block(grad):
    """A trace, with a graph or without, computes its outputs from its inputs as the block does."""
    import warnings
    for m, shape in _recorded_cases():
        with torch.set_grad_enabled(grad), warnings.catch_warnings():
            warnings.simplefilter('ignore', torch.jit.TracerWarning)
            traced = torch.jit.trace(m, torch.randn(shape, device='cuda'), check_trace=False)
            for _ in range(3):
                x = torch.randn(shape, device='cuda')
                junk = [torch.full(shape, float('nan'), device='cuda') for _ in range(8)]      # (for memory not written)
                del junk
                assert torch.allclose(traced(x), _plain_block(m, x), rtol=1e-5, atol=1e-5)


@pytest.mark.gpu
def test_recorded_by_dispatch_modes():
    """make_fx and torch.export record torch's operators; a mode that counts them counts the block's products."""
    from torch.fx.experimental.proxy_tensor import make_fx
    from torch.utils.flop_counter import FlopCounterMode
    for m, shape in _recorded_cases():
        x, z = torch.randn(shape, device='cuda'), torch.randn(shape, device='cuda')
        with torch.no_grad():
            want = _plain_block(m, z)
            for fn in (make_fx(m)(x), torch.export.export(m, (x,)).module()):
                assert torch.allclose(fn(z), want, rtol=1e-5, atol=1e-5)
        with FlopCounterMode(display=False) as count:
            m(x)
        products = 2 * 2 * 5 * 24 * 40 if isinstance(m, Block) else 2 * 2 * 12 * 16 * 16
        assert count.get_total_flops() == products


@pytest.mark.gpu
@pytest.mark.parametrize('grad', [False, True])
def test_forward_mode_and_functional_transforms(grad):
    """The tangent of a dual input is carried through, with a graph or without, and a transform sees the operators."""
    import torch.autograd.forward_ad as fw
    for m, shape in _recorded_cases():
        x, v = torch.randn(shape, device='cuda'), torch.randn(shape, device='cuda')
        with torch.set_grad_enabled(grad):
            with fw.dual_level():
                got = fw.unpack_dual(m(fw.make_dual(x, v)))
                want = fw.unpack_dual(_plain_block(m, fw.make_dual(x, v)))
                assert got.tangent is not None
                assert all(torch.allclose(a, b, rtol=1e-5, atol=1e-5) for a, b in zip(got, want))
            y, t = torch.func.jvp(m, (x,), (v,))
            assert torch.allclose(y, want.primal, rtol=1e-5, atol=1e-5) and torch.allclose(t, want.tangent, rtol=1e-5, atol=1e-5)
            xs = torch.stack([x, v])
            assert torch.allclose(torch.func.vmap(m)(xs), torch.stack([_plain_block(m, a) for a in xs]), rtol=1e-5, atol=1e-5)


@pytest.mark.gpu
def test_kernel_calls_refuse_forward_mode():
    """The calls below the layers have no tangents to give: refused, with a graph or without."""
    import torch.autograd.forward_ad as fw
    from vfdepth_amd import kernels as KN
    x, w = torch.randn(4, 8, device='cuda'), torch.randn(6, 8, device='cuda')
    with torch.no_grad(), fw.dual_level():
        dual = fw.make_dual(x, x)
        for call in (lambda: KN.LayerNorm.infer(dual, None, None, 1e-5), lambda: KN.LayerNorm.apply(dual, None, None, 1e-5),
                     lambda: KN.LinearAct.infer(dual, w, None, None, 'gelu'), lambda: KN.LinearAct.apply(dual, w, None, None, 'gelu')):
            with pytest.raises(NotImplementedError, match='jvp'):
                call()
    traced = torch.jit.trace(lambda t: KN.LayerNorm.infer(t, None, None, 1e-5), x, check_trace=False)
    z = torch.randn(4, 8, device='cuda')
    assert torch.equal(traced(z), KN.LayerNorm.infer(z, None, None, 1e-5))


class _Doubled(torch.nn.Linear):
    def forward(self, x):
        return 2 * super().forward(x)


class _Shifted(torch.nn.LayerNorm):
    def forward(self, x):
        return super().forward(x) + 1


def _hooked(kind):
    """(module, whether it is a linear layer) with something hanging on its call."""
    if kind == 'subclass':
        return _Doubled(24, 16), True
    if kind == 'norm_subclass':
        return _Shifted(24), False
    m = torch.nn.LayerNorm(24) if kind.startswith('norm') else torch.nn.Linear(24, 16)
    if kind in ('pre', 'norm_pre'):
        m.register_forward_pre_hook(lambda mod, args: (args[0] * 3,))
    elif kind in ('post', 'norm_post'):
        m.register_forward_hook(lambda mod, args, out: out - 2)
    elif kind == 'backward':
        m.register_full_backward_hook(lambda mod, gi, go: (gi[0] * 5,))
    elif kind == 'instance':
        m.forward = lambda x: torch.nn.functional.linear(x, m.weight)
    elif kind == 'weight_norm':
        m = torch.nn.utils.weight_norm(m)                     # the weight is computed by a hook before each call
    elif kind == 'parametrized':
        m = torch.nn.utils.parametrizations.weight_norm(m)
    return m, not kind.startswith('norm')


HOOKED = ['pre', 'post', 'backward', 'instance', 'subclass', 'weight_norm', 'parametrized', 'norm_pre', 'norm_post', 'norm_subclass']


@pytest.mark.parametrize('device', ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)])
@pytest.mark.parametrize('grad', [True, False])
@pytest.mark.parametrize('kind', HOOKED)
def test_what_hangs_on_a_module(kind, grad, device):
    """Hooks, forwards of subclasses and of objects, and weights computed before a call count on either device."""
    from vfdepth_amd import layers
    torch.manual_seed(3)
    m, linear_ = _hooked(kind)
    m = m.to(device)
    with torch.no_grad():
        for p in m.parameters():                              # a weight that was computed at construction is out of date now
            p.mul_(1.5)
    x = torch.randn(7, 24, device=device, requires_grad=grad)
    run = (lambda: layers.linear_act(m, x, 'silu')) if linear_ else (lambda: layers.layer_norm(m, x))
    plain = (lambda: torch.nn.functional.silu(m(x))) if linear_ else (lambda: m(x))
    with torch.set_grad_enabled(grad):
        y, want = run(), plain()
        assert torch.allclose(y, want, rtol=1e-5, atol=1e-5)
        if grad:
            ps = [x] + list(m.parameters())
            for a, b in zip(*(torch.autograd.grad(t.square().sum(), ps, allow_unused=True) for t in (y, want))):
                assert (a is None) == (b is None) and (a is None or torch.allclose(a, b, rtol=1e-4, atol=1e-4))


@pytest.mark.parametrize('device', ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)])
def test_global_hooks_see_the_modules(device):
    from vfdepth_amd import layers
    ln, lin = torch.nn.LayerNorm(8).to(device), torch.nn.Linear(8, 8).to(device)
    seen = []
    handle = torch.nn.modules.module.register_module_forward_hook(lambda mod, args, out: seen.append(mod))
    try:
        layers.linear_act(lin, layers.layer_norm(ln, torch.randn(3, 8, device=device)), 'relu')
    finally:
        handle.remove()
    assert seen == [ln, lin]


@pytest.mark.parametrize('device', ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)])
def test_scripted_modules_and_other_callables(device):
    """What is no ordinary module is called, on either device."""
    import warnings
    from vfdepth_amd import layers
    lin, ln = torch.nn.Linear(6, 4).to(device), torch.nn.LayerNorm(6).to(device)
    x = torch.randn(3, 6, device=device)
    with warnings.catch_warnings():
        warnings.simplefilter('ignore')
        scripted = torch.jit.script(lin), torch.jit.script(ln)
    for a, b in (scripted, (lambda t: lin(t), lambda t: ln(t))):
        assert torch.allclose(layers.linear_act(a, x, 'relu'), torch.relu(lin(x)), rtol=1e-5, atol=1e-5)
        assert torch.allclose(layers.layer_norm(b, x), ln(x), rtol=1e-5, atol=1e-5)


@pytest.mark.gpu
def test_plain_modules_take_the_kernels():
    """Ordinary modules, a subclass without a forward and a parametrized weight are not sent to the module."""
    from vfdepth_amd import layers

    class Named(torch.nn.Linear):
        pass
    para = torch.nn.utils.parametrizations.weight_norm(torch.nn.Linear(24, 16))
    for m in (torch.nn.Linear(24, 16), Named(24, 16), para, torch.nn.Conv2d(24, 16, 1), layers.conv2d_block(24, 16, 1)[0]):
        m = m.cuda()
        x = torch.randn(2, 24, 3, 5, device='cuda') if isinstance(m, torch.nn.Conv2d) else torch.randn(7, 24, device='cuda')
        fn = layers.linear_act(m, x, 'silu').grad_fn
        while 'Permute' in type(fn).__name__:
            fn = fn.next_functions[0][0]
        assert type(fn).__name__ == 'LinearActBackward'
    y = layers.layer_norm(torch.nn.LayerNorm(8).cuda(), torch.randn(3, 8, device='cuda'))
    assert type(y.grad_fn).__name__ == 'LayerNormBackward'


def _relaid(t):
    """The same values, stored the other way round: last dimension apart, rows beside each other."""
    return t if t.dim() < 2 else t.transpose(-1, -2).contiguous().transpose(-1, -2)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('how', ['cpu', 'relaid', 'spread'])
def test_saved_tensors_come_back_in_another_layout(how, dtype):
    """Saved-tensor hooks (save_on_cpu packs densely) may change how far apart the saved rows lie: the gradients are those
    of a backward without hooks, bit for bit."""
    from vfdepth_amd import kernels as KN
    graph = torch.autograd.graph
    spread = lambda t: t if t.dim() < 2 else torch.nn.functional.pad(t, (3, 6))[..., 3:-6]  # noqa: E731
    hooks = {'cpu': lambda: graph.save_on_cpu(), 'relaid': lambda: graph.saved_tensors_hooks(_relaid, lambda t: t),
             'spread': lambda: graph.saved_tensors_hooks(spread, lambda t: t)}[how]
    wide = torch.randn(150, 107, device='cuda').to(dtype)
    w, b = torch.randn(40, 96, device='cuda').to(dtype), torch.randn(40, device='cuda').to(dtype)
    ln_w = torch.randn(96, device='cuda')
    for x in (wide[:, 5:101], wide[::3, 2:98], wide[:, :96].contiguous(), wide[:1, :96], wide[:96, :96].t()):
        runs = []
        for hooked in (False, True):
            leaves = [t.detach().requires_grad_(True) for t in (x, w, b, ln_w)]
            xl, wl, bl, nl = leaves
            with hooks() if hooked else torch.enable_grad():
                y, z = KN.LinearAct.apply(xl, wl, bl, None, 'gelu'), KN.LayerNorm.apply(xl, nl, None, 1e-5)
            gen = torch.Generator(device='cuda').manual_seed(7)
            gy, gz = (torch.randn(t.shape, generator=gen, device='cuda').to(dtype) for t in (y, z))
            runs.append(torch.autograd.grad(y, leaves[:3], gy) + torch.autograd.grad(z, (xl, nl), gz))
        assert all(torch.equal(a, c) for a, c in zip(*runs))


@pytest.mark.gpu
@pytest.mark.parametrize('change', [lambda t: t.cpu(), lambda t: t.double(), lambda t: t.flatten()[:-1], lambda t: t.half()])
def test_saved_tensors_that_come_back_as_others_are_refused(change):
    from vfdepth_amd import kernels as KN
    x, w = torch.randn(12, 8, device='cuda', requires_grad=True), torch.randn(6, 8, device='cuda', requires_grad=True)
    lw = torch.randn(8, device='cuda', requires_grad=True)
    for call, leaves in ((lambda: KN.LinearAct.apply(x, w, None, None, 'silu'), (x, w)), (lambda: KN.LayerNorm.apply(x, lw, None, 1e-5), (x, lw))):
        with torch.autograd.graph.saved_tensors_hooks(change, lambda t: t):
            y = call()
        with pytest.raises(RuntimeError, match='saved-tensor hook'):
            torch.autograd.grad(y, leaves, torch.ones_like(y))


@pytest.mark.gpu
@pytest.mark.parametrize('reentrant', [False, True])
def test_checkpointed_block(reentrant):
    from torch.utils.checkpoint import checkpoint
    torch.manual_seed(4)
    blk = Block(48, 100).cuda()
    x = torch.randn(70, 48, device='cuda', requires_grad=True)
    g = torch.randn(70, 48, device='cuda')
    runs = []
    for y in (lambda: blk(x), lambda: checkpoint(blk, x, use_reentrant=reentrant)):
        for t in (x, *blk.parameters()):
            t.grad = None
        y().backward(g)
        runs.append([t.grad for t in (x, *blk.parameters())])
    assert all(torch.equal(a, b) for a, b in zip(*runs))
