"""Global gradient norm and clipping (gradclip.hip, kernels.grad_norm / clip_grads / clip_grad_norm_).

Tolerances: the kernels sum squares in fp64 (relative error under n 2^-53, nothing beside an fp32 half step) and round
the norm once to fp32: 2^-24.  A clipped gradient carries the factor's rounding (2^-24) and its own (the output type's
half step); both are counted."""
import array
import ctypes
import math

import pytest
import torch

F32, BF16 = torch.float32, torch.bfloat16
HALF = {F32: 2.0 ** -24, BF16: 2.0 ** -8}


def _sizes(kind):
    return {'one': [1], 'tail': [16383, 16384, 16385, 4096, 1, 3], 'empty': [0, 7, 0, 16384, 0],
            'many': [(i * 37) % 511 + 1 for i in range(400)], 'large': [3_000_001, 5, 1_048_576]}[kind]


def _make(sizes, dtype, seed=0, scale=1.0, device='cuda'):
    gen = torch.Generator().manual_seed(seed)
    return [(torch.randn(n, generator=gen) * scale).to(dtype).to(device) for n in sizes]


def _oracle(grads, max_norm=None, norm_type=2.0):
    wide = [g.detach().cpu().double() for g in grads]
    if norm_type == math.inf:
        n = max([float(w.abs().max()) for w in wide if w.numel()] or [0.0])
    else:
        n = math.sqrt(math.fsum(float((w * w).sum()) for w in wide))
    if max_norm is None:
        return n
    c = min(1.0, max_norm / (n + 1e-6))
    return n, [w * c for w in wide]


def _near(got, want, rel, what=''):
    err = (got.detach().cpu().double() - want).abs()
    assert bool((err <= rel * want.abs()).all()), (what, float((err / want.abs().clamp_min(1e-300)).max()))


# ------------------------------------------------------------------------------------------------ CPU
def _c_call(ptrs, numel, outs=None, dtypes=None, odt=None, max_norm=1.0, ws=1 << 20):
    from vfdepth_amd import _lib
    lib = _lib.load()
    n = len(ptrs)
    p, q = array.array('Q', ptrs), array.array('q', numel)
    o = array.array('Q', outs) if outs is not None else None
    rc = lib.vfd_clip_grads(n, p.buffer_info()[0], q.buffer_info()[0], dtypes or bytes(n), 0, max_norm,
                            o.buffer_info()[0] if o else None, (odt or bytes(n)) if o else None, 1 << 40, 1 << 41, ws,
                            None)
    return rc, lib.vfd_last_error().decode()


# made-up addresses: every one of these is refused on the host before anything is launched
@pytest.mark.parametrize('ptrs,numel,outs,kw,word', [
    ([4096, 4096], [10, 10], None, {}, 'share memory'),
    ([4096, 4100], [10, 10], None, {}, 'share memory'),
    ([8192, 4096], [1, 1025], None, {}, 'share memory'),
    ([4096, 8192], [10, 10], [65536, 65540], {}, 'share memory'),
    ([4096, 65536], [4096, 10], [1 << 20, 4096 + 4 * 4095], {}, 'with a gradient'),
    ([4096], [10], [4096], {}, 'with a gradient'),
    ([4096, 8192], [2000, 1], [1 << 20, 9000], {'odt': bytes([0, 1])}, 'with a gradient'),
    ([0], [1], None, {}, 'bad tensor'),
    ([4096], [-1], None, {}, 'bad tensor'),
    ([4096], [1], None, {'dtypes': bytes([2])}, 'bad tensor'),
    ([4096], [1], [0], {}, 'bad output'),
    ([4096], [1], [8192], {'odt': bytes([7])}, 'bad output'),
    ([4096], [1], None, {'max_norm': -1.0}, 'max_norm'),
    ([4096], [1], None, {'max_norm': math.nan}, 'max_norm'),
    ([4096], [1], None, {'ws': 8}, 'workspace'),
    ([4096], [1 << 43], None, {}, 'bad tensor'),
])
def test_c_refusals(ptrs, numel, outs, kw, word):
    rc, msg = _c_call(ptrs, numel, outs, **kw)
    assert rc == -1 and word in msg, (rc, msg)


def test_workspace_counts_partials():
    from vfdepth_amd import _lib
    lib = _lib.load()

    def ws(numel):
        a = array.array('q', numel)
        return lib.vfd_grad_norm_workspace(len(numel), a.buffer_info()[0])
    assert ws([]) == 8 and ws([0, 0]) == 8
    assert ws([1]) == 16 and ws([16384]) == 16 and ws([16385]) == 24
    assert ws([1] * 177) == 8 * (177 + 1)
    assert ws([16384 * 2049]) == 8 * (1025 + 1)            # two rounds of 1025 blocks, not 2048 and 1


def test_refuses_cpu_tensors_and_types():
    from vfdepth_amd import kernels as KN
    for fn in (KN.grad_norm, lambda g: KN.clip_grads(g, 1.0)):
        with pytest.raises(RuntimeError, match='HIP device'):
            fn([torch.zeros(3)])
    p = torch.nn.Parameter(torch.zeros(2))
    p.grad = torch.ones(2)
    with pytest.raises(RuntimeError, match='HIP device'):
        KN.clip_grad_norm_([p], 1.0)


def test_dense_layouts():
    from vfdepth_amd.kernels import _dense
    x = torch.zeros(2, 3, 4, 5)
    assert _dense(x) and _dense(x.to(memory_format=torch.channels_last)) and _dense(x.permute(3, 1, 0, 2))
    assert _dense(x[:1]) and _dense(torch.zeros(())) and _dense(torch.zeros(0, 3))
    assert not _dense(x[:, :2]) and not _dense(torch.zeros(3, 1).expand(3, 4)) and not _dense(torch.zeros(8)[::2])


def test_config_refuses_a_negative_limit():
    from vfdepth_amd.config import mono_cfg
    from vfdepth_amd.vfdepth import VFDepthAlgo
    for bad in (-1.0, math.nan):
        with pytest.raises(ValueError, match='max_grad_norm'):
            VFDepthAlgo(mono_cfg(max_grad_norm=bad), 'cpu')


def test_clip_gradients_on_the_cpu_rehearsal():
    """The optimizer's parameters are clipped with torch where there is no HIP device, and left alone by default."""
    from vfdepth_amd.config import mono_cfg
    from vfdepth_amd.vfdepth import VFDepthAlgo
    algo = VFDepthAlgo(mono_cfg(max_grad_norm=0.5, height=32, width=64), 'cpu')
    ps = [p for g in algo.optimizer.param_groups for p in g['params']]
    for p in ps[1:]:
        p.grad = torch.ones_like(p)
    n = math.sqrt(sum(p.numel() for p in ps[1:]))
    algo.clip_gradients()
    assert abs(float(algo.grad_norm) - n) <= 1e-5 * n
    total = math.sqrt(sum(float((p.grad.double() ** 2).sum()) for p in ps[1:]))
    assert abs(total - 0.5) <= 1e-5
    off = VFDepthAlgo(mono_cfg(height=32, width=64), 'cpu')
    off.clip_gradients()
    assert off.grad_norm is None


# ------------------------------------------------------------------------------------------------ GPU
gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize('norm_type', [2.0, math.inf])
@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('kind', ['one', 'tail', 'empty', 'many', 'large'])
def test_norm(kind, dtype, norm_type):
    from vfdepth_amd import kernels as KN
    grads = _make(_sizes(kind), dtype)
    n = KN.grad_norm(grads, norm_type)
    assert n.dtype == F32 and n.dim() == 0 and n.is_cuda
    want = _oracle(grads, norm_type=norm_type)
    assert abs(float(n) - want) <= HALF[F32] * want * (1 + 1e-6)
    assert float(KN.grad_norm(grads, norm_type)) == float(n)


@gpu
@pytest.mark.parametrize('over', [True, False])
@pytest.mark.parametrize('dtype,odtype', [(F32, None), (BF16, None), (F32, F32), (F32, BF16), (BF16, F32), (BF16, BF16)])
@pytest.mark.parametrize('kind', ['one', 'tail', 'empty', 'many', 'large'])
def test_clip(kind, dtype, odtype, over):
    from vfdepth_amd import kernels as KN
    grads = _make(_sizes(kind), dtype, seed=3)
    n0 = _oracle(grads)
    limit = n0 * (0.3 if over else 1.5) + 1e-3
    n, want = _oracle(grads, limit)
    before = [g.clone() for g in grads]
    outs = None
    if odtype is not None:           # outputs are odd slices of one buffer, with a guard on each side
        total = sum(g.numel() for g in grads)
        flat = torch.full((total + 2,), 7.0, dtype=odtype, device='cuda')
        outs = list(flat[1:-1].split([g.numel() for g in grads]))
    got_n = KN.clip_grads(grads, limit, out=outs)
    assert abs(float(got_n) - n) <= HALF[F32] * n * (1 + 1e-6)
    got = grads if outs is None else outs
    for g, w in zip(got, want):
        if g.numel():
            _near(g, w, (HALF[F32] + HALF[g.dtype]) * (1 + 1e-6))
    if outs is not None:
        assert float(flat[0]) == 7.0 and float(flat[-1]) == 7.0
        assert all(torch.equal(a, b) for a, b in zip(grads, before))
    elif not over:
        assert all(torch.equal(a, b) for a, b in zip(grads, before))


@gpu
def test_mixed_types_views_and_layouts():
    from vfdepth_amd import kernels as KN
    flat = torch.randn(5000, device='cuda')
    grads = [flat[1:4000], torch.randn(33, 7, device='cuda').to(BF16).t(), flat[4001:],
             torch.randn(4, 6, 5, 3, device='cuda').to(memory_format=torch.channels_last)]
    guard = float(flat[0]), float(flat[4000])
    n, want = _oracle(grads, 0.5)
    v = [g._version for g in grads]
    got = KN.clip_grads(grads, 0.5)
    assert abs(float(got) - n) <= HALF[F32] * n * (1 + 1e-6)
    for g, w in zip(grads, want):
        _near(g, w, (HALF[F32] + HALF[g.dtype]) * (1 + 1e-6))
    assert (float(flat[0]), float(flat[4000])) == guard
    assert all(g._version > x for g, x in zip(grads, v))


@gpu
def test_extreme_magnitudes():
    """Squares of these overflow (or vanish) in 32 bits; the norm does not."""
    from vfdepth_amd import kernels as KN
    for scale in (1e30, 1e-30):
        grads = _make([1000, 77], F32, scale=scale)
        n = _oracle(grads)
        assert abs(float(KN.grad_norm(grads)) - n) <= HALF[F32] * n * (1 + 1e-6)
    grads = _make([5000], F32, scale=1e30)
    n, want = _oracle(grads, 1.0)
    KN.clip_grads(grads, 1.0)
    _near(grads[0], want[0], 2 * HALF[F32] * (1 + 1e-6))


@gpu
@pytest.mark.parametrize('norm_type', [2.0, math.inf])
def test_non_finite(norm_type):
    """As torch.nn.utils.clip_grad_norm_: an infinite norm zeroes what is finite, a NaN one spoils everything."""
    from vfdepth_amd import kernels as KN
    for bad in (math.inf, -math.inf, math.nan):
        mine = _make([300, 9000], F32)
        mine[1][8999] = bad
        ps = [torch.nn.Parameter(torch.zeros_like(g)) for g in mine]
        for p, g in zip(ps, mine):
            p.grad = g.clone()
        ref = torch.nn.utils.clip_grad_norm_(ps, 1.0, norm_type)
        got = KN.clip_grads(mine, 1.0, norm_type)
        assert torch.equal(torch.isnan(got), torch.isnan(ref)) and (math.isnan(float(got)) or float(got) == float(ref))
        for g, p in zip(mine, ps):
            assert torch.equal(torch.isnan(g), torch.isnan(p.grad))
            assert torch.equal(torch.nan_to_num(g), torch.nan_to_num(p.grad))


@gpu
def test_zero_limit_empty_list_and_zero_gradients():
    from vfdepth_amd import kernels as KN
    assert float(KN.grad_norm([])) == 0.0 and float(KN.clip_grads([], 1.0)) == 0.0
    assert float(KN.clip_grad_norm_([], 1.0)) == 0.0
    assert float(KN.grad_norm([torch.zeros(0, device='cuda')])) == 0.0
    g = torch.randn(100, device='cuda')
    KN.clip_grads([g], 0.0)
    assert not g.any()
    assert float(KN.clip_grads([g], 1.0)) == 0.0 and not g.any()


@gpu
def test_python_refusals():
    from vfdepth_amd import kernels as KN
    g = torch.randn(4, 6, device='cuda')
    for call, err in [
            (lambda: KN.clip_grads([g[:, :3]], 1.0), 'densely'),
            (lambda: KN.clip_grads([g, g], 1.0), 'share memory'),
            (lambda: KN.clip_grads([g], 1.0, out=[g]), 'with a gradient'),
            (lambda: KN.clip_grads([g], 1.0, out=[]), 'outputs'),
            (lambda: KN.clip_grads([g], 1.0, out=[torch.zeros(6, 4, device='cuda')]), 'into output'),
            (lambda: KN.clip_grads([g], 1.0, out=[torch.zeros(6, 4, device='cuda').t()]), 'contiguous or laid out'),
            (lambda: KN.clip_grads([g], -1.0), 'max_norm'),
            (lambda: KN.clip_grads([g], math.nan), 'max_norm'),
            (lambda: KN.grad_norm([g], 1.0), 'norm_type'),
            (lambda: KN.grad_norm([g.half()]), 'fp32 or bf16'),
            (lambda: KN.grad_norm([g.to_sparse()]), 'strided'),
            (lambda: KN.grad_norm([g, g.cpu()]), 'HIP device')]:
        with pytest.raises((RuntimeError, ValueError), match=err):
            call()
    # what in-place refuses is clipped into an output
    n, want = _oracle([g[:, :3]], 0.1)
    out = torch.empty(4, 3, device='cuda')
    KN.clip_grads([g[:, :3]], 0.1, out=[out])
    _near(out, want[0], 2 * HALF[F32] * (1 + 1e-6))
    assert float(KN.grad_norm([g, g])) > 0                        # reading one twice is fine


@gpu
def test_parameters_and_a_parameter_listed_twice():
    from vfdepth_amd import kernels as KN
    torch.manual_seed(0)
    ps = [torch.nn.Parameter(torch.randn(n, device='cuda')) for n in (10, 4097, 3)]
    ps[0].grad, ps[1].grad = torch.randn(10, device='cuda'), torch.randn(4097, device='cuda')
    n, want = _oracle([ps[0].grad, ps[1].grad], 0.7)
    got = KN.clip_grad_norm_(iter([ps[0], ps[1], ps[2], ps[1]]), 0.7)
    assert abs(float(got) - n) <= HALF[F32] * n * (1 + 1e-6) and ps[2].grad is None
    for p, w in zip(ps, want):
        _near(p.grad, w, 2 * HALF[F32] * (1 + 1e-6))


@gpu
def test_offsets_beyond_32_bits():
    """One tensor of 2.2 billion values, all zero but for a few at its ends."""
    from vfdepth_amd import kernels as KN
    g = torch.zeros((1 << 31) + 70001, dtype=BF16, device='cuda')
    g[:3], g[-5:] = 3.0, 4.0
    n = math.sqrt(3 * 9 + 5 * 16)
    out = torch.full(g.shape, 7.0, dtype=BF16, device='cuda')
    got = KN.clip_grads([g], 1.0, out=[out])
    assert abs(float(got) - n) <= HALF[F32] * n * (1 + 1e-6)
    _near(out[:3], g[:3].cpu().double() / (n + 1e-6), (HALF[F32] + HALF[BF16]) * (1 + 1e-6))
    _near(out[-5:], g[-5:].cpu().double() / (n + 1e-6), (HALF[F32] + HALF[BF16]) * (1 + 1e-6))
    assert int(out.count_nonzero()) == 8


@gpu
def test_another_stream_and_a_captured_graph():
    from vfdepth_amd import kernels as KN
    src = _make([5000, 17, 123], F32)
    n, want = _oracle(src, 0.4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        grads = [g.clone() for g in src]
        got = KN.clip_grads(grads, 0.4)
    torch.cuda.current_stream().wait_stream(side)
    assert abs(float(got) - n) <= HALF[F32] * n * (1 + 1e-6)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = KN.clip_grads(grads, 0.4)
    other = torch.cuda.CUDAGraph()
    with torch.cuda.graph(other):
        norm2 = KN.grad_norm(grads)
    for k in range(4):
        for g, s in zip(grads, src):
            g.copy_(s * (k + 1))
        n, want = _oracle(grads, 0.4)
        graph.replay()
        other.replay()
        torch.cuda.synchronize()
        assert abs(float(norm) - n) <= HALF[F32] * n * (1 + 1e-6)
        assert abs(float(norm2) - 0.4) <= 1e-5
        for g, w in zip(grads, want):
            _near(g, w, 2 * HALF[F32] * (1 + 1e-6))
        KN.clip_grads([g.clone() for g in grads], 0.1)             # eager work between replays


@gpu
def test_training_step_clips():
    """VFDepthAlgo.train_step with training.max_grad_norm: the gradients left by the step have the limit's norm."""
    from vfdepth_amd import kernels as KN
    from vfdepth_amd import synth
    from vfdepth_amd.config import mono_cfg
    from vfdepth_amd.vfdepth import VFDepthAlgo
    cfg = mono_cfg(max_grad_norm=1e-3, height=64, width=96)
    algo = VFDepthAlgo(cfg, 0)
    algo.set_train()
    algo.train_step(dict(synth.make_batch(cfg, seed=1)))
    before = float(algo.grad_norm)
    grads = [p.grad for g in algo.optimizer.param_groups for p in g['params'] if p.grad is not None]
    after = float(KN.grad_norm(grads))
    assert before > 1e-3 and abs(after - 1e-3 * before / (before + 1e-6)) <= 1e-3 * 1e-5


@gpu
@pytest.mark.parametrize('norm_type', [2.0, math.inf])
@pytest.mark.parametrize('into', [False, True])
def test_thousands_of_tensors(into, norm_type):
    """More partial norms than every scaling block joins for itself (8192): they are joined first."""
    from vfdepth_amd import kernels as KN
    sizes = [i % 3 + 1 for i in range(8500)]
    flat = torch.randn(sum(sizes), generator=torch.Generator().manual_seed(2)).cuda()
    flat[-1] = 4.0                                           # the largest, in the last tensor
    grads, before = list(flat.split(sizes)), flat.clone()
    n = float(flat.double().norm(norm_type))
    assert abs(float(KN.grad_norm(grads, norm_type)) - n) <= HALF[F32] * n * (1 + 1e-6)
    outs = torch.full_like(flat, 7.0) if into else None
    got = KN.clip_grads(grads, 0.25 * n, norm_type, out=None if outs is None else list(outs.split(sizes)))
    assert abs(float(got) - n) <= HALF[F32] * n * (1 + 1e-6)
    _near(flat if outs is None else outs, before.cpu().double() * (0.25 * n / (n + 1e-6)), 2 * HALF[F32] * (1 + 1e-6))
    assert outs is None or torch.equal(flat, before)


@gpu
@pytest.mark.parametrize('over', [True, False])
def test_captured_training_step_clips(over):
    """A captured step with training.max_grad_norm: at every replay `step.grad_norm` is that batch's norm before clipping,
    and the gradients that the optimizer takes have the limit's norm, or their own where it is under the limit."""
    from vfdepth_amd import kernels as KN
    from vfdepth_amd import synth
    from vfdepth_amd.config import mono_cfg
    from vfdepth_amd.vfdepth import VFDepthAlgo
    limit = 1e-3 if over else 1e6
    cfg = mono_cfg(max_grad_norm=limit, height=64, width=96)
    algo = VFDepthAlgo(cfg, 0)
    algo.set_train()
    algo.set_optimizer(capturable=True)
    batches = [synth.make_batch(cfg, seed=s, device='cuda') for s in (1, 2, 3)]
    step = algo.graphed_train_step(batches[0], warmup=2)
    params = [p for g in algo.optimizer.param_groups for p in g['params']]
    norms = []
    for k in (0, 1, 2, 0):
        step(batches[k])
        torch.cuda.synchronize()
        before = float(step.grad_norm)
        after = float(KN.grad_norm([p.grad for p in params if p.grad is not None]))       # eager work between replays
        want = limit * before / (before + 1e-6) if over else before
        assert before > 1e-3 and math.isfinite(before) and abs(after - want) <= want * (1e-5 if over else 2 * HALF[F32])
        norms.append(before)
    assert len(set(norms)) == len(norms)                     # other batches and weights: other norms


def test_no_limit_leaves_no_norm():
    from vfdepth_amd.config import mono_cfg
    from vfdepth_amd.vfdepth import VFDepthAlgo
    for cfg in (mono_cfg(height=32, width=64), mono_cfg(max_grad_norm=None, height=32, width=64)):
        algo = VFDepthAlgo(cfg, 'cpu')
        assert algo.max_grad_norm == 0.0
        algo.clip_gradients()
        assert algo.grad_norm is None
