"""Layer norm forward / backward (layernorm.hip, kernels.LayerNorm, layers.layer_norm / channel_norm).

Tolerances (u = 2^-24, half an fp32 step): a sum over C values passes at most D = max(26, C / 256 + 10) additions per
value (16 or C / 256 in a lane, then a tree), so the mean is off by D u mean|x| and the variance relatively by
(D + 2) u plus what the mean adds in second order; h = (x - m) r is then off by
    dh = u ((D + 4) r mean|x| + (D / 2 + 5) |h|)
and each output by what dh and its own sums and roundings add, written out in `_bounds`; the output type's half step is
added last.  A column sum over R rows passes at most R / 256 + 40 additions a value (rows of a lane, wave, block, blocks)."""
import ctypes
import math

import pytest
import torch

F32, BF16 = torch.float32, torch.bfloat16
U = 2.0 ** -24
HALF = {F32: 2.0 ** -24, BF16: 2.0 ** -8}
TINY = 2.0 ** -126                       # what is below the types' normal range may round away
EPS = 1e-5


def _case(rows, C, dtype, seed=0, mean=0.3):
    gen = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, C, generator=gen) * (0.5 + torch.rand(C, generator=gen)) + mean).to(dtype)
    w = torch.randn(C, generator=gen) * 0.2 + 1
    b = torch.randn(C, generator=gen) * 0.1
    g = torch.randn(rows, C, generator=gen).to(dtype)
    return x, w, b, g


def _oracle(x, w, b, g, eps=EPS):
    """Values in 64 bits and how far a 32-bit evaluation may be off, for y, dx, dw, db."""
    x, g = x.detach().cpu().double(), g.detach().cpu().double()
    R, C = x.shape
    w = torch.ones(C, dtype=torch.float64) if w is None else w.detach().cpu().double()
    b = torch.zeros(C, dtype=torch.float64) if b is None else b.detach().cpu().double()
    m = x.mean(1, keepdim=True)
    r = 1 / ((x - m).square().mean(1, keepdim=True) + eps).sqrt()
    h = (x - m) * r
    gw = g * w
    c1, c2 = gw.mean(1, keepdim=True), (gw * h).mean(1, keepdim=True)
    dx = r * (gw - c1 - h * c2)
    vals = [h * w + b, dx, (g * h).sum(0), g.sum(0)]
    D, Dr = max(26, C / 256 + 10), R / 256 + 40
    dh = U * ((D + 4) * r * x.abs().mean(1, keepdim=True) + (D / 2 + 5) * h.abs())
    ab = lambda t: t.abs().mean(1, keepdim=True)  # noqa: E731
    dc1 = (D + 2) * U * ab(gw)
    dc2 = (gw.abs() * dh).mean(1, keepdim=True) + (D + 2) * U * ab(gw * h)
    ddx = r * (dc1 + dh * c2.abs() + h.abs() * dc2 + 4 * U * (gw.abs() + c1.abs() + (h * c2).abs()))
    tol = [w.abs() * dh + 2 * U * ((h * w).abs() + b.abs()), ddx + (D / 2 + 5) * U * dx.abs(),
           (g.abs() * dh).sum(0) + Dr * U * (g * h).abs().sum(0), Dr * U * g.abs().sum(0)]
    return vals, tol


def _check(got, vals, tol, names=('y', 'dx', 'dw', 'db')):
    for t, v, e, name in zip(got, vals, tol, names):
        if t is None:
            continue
        err = (t.detach().cpu().double() - v).abs()
        lim = e + HALF[t.dtype] * (v.abs() + e) + TINY
        assert t.shape == v.shape and bool((err <= lim).all()), (name, float((err / lim).max()))


def _run(x, w, b, g, eps=EPS):
    from vfdepth_amd import kernels as KN
    leaves = [t.requires_grad_(True) for t in (x, w, b) if t is not None]
    y = KN.LayerNorm.apply(x, w, b, eps)
    return y, torch.autograd.grad(y, leaves, g)


# ------------------------------------------------------------------------------------------------ CPU
@pytest.mark.parametrize('rows,cols,ldx,dtype', [(1, 0, 0, 0), (-1, 4, 4, 0), (1, 4, 3, 0), (1, 4, 4, 2), (1, 1 << 29, 1 << 29, 0)])
def test_c_refuses_bad_descriptors(rows, cols, ldx, dtype):
    from vfdepth_amd import _lib
    lib = _lib.load()
    d = _lib.NormDesc(rows, cols, ldx, 1e-5, dtype)
    assert lib.vfd_layer_norm_fwd(ctypes.byref(d), *[None] * 7) == -1 and b'descriptor' in lib.vfd_last_error()
    assert lib.vfd_layer_norm_bwd(ctypes.byref(d), *[None] * 9, 0, None) == -1
    assert lib.vfd_layer_norm_bwd_workspace(ctypes.byref(d)) == 0


def test_c_refuses_null_tensors_and_small_workspaces():
    from vfdepth_amd import _lib
    lib = _lib.load()
    d = _lib.NormDesc(10, 64, 64, 1e-5, 0)
    p = 1 << 40
    assert lib.vfd_layer_norm_fwd(ctypes.byref(d), None, p, p, p, p, p, None) == -1
    assert lib.vfd_layer_norm_fwd(ctypes.byref(d), p, p, p, p, p, None, None) == -1
    need = lib.vfd_layer_norm_bwd_workspace(ctypes.byref(d))
    assert need > 0
    assert lib.vfd_layer_norm_bwd(ctypes.byref(d), p, p, p, p, p, p, p, p, p, need - 1, None) == -1
    assert b'workspace' in lib.vfd_last_error()
    assert lib.vfd_layer_norm_fwd(ctypes.byref(_lib.NormDesc(0, 64, 64, 1e-5, 0)), *[None] * 7) == 0       # no rows


@pytest.mark.parametrize('cols,dtype', [(1, 0), (16, 0), (16, 1), (4096, 1), (9001, 0)])
def test_workspace_of_the_most_rows(cols, dtype):
    from vfdepth_amd import _lib
    lib = _lib.load()
    ws = [lib.vfd_layer_norm_bwd_workspace(ctypes.byref(_lib.NormDesc(rows, cols, cols, 1e-5, dtype)))
          for rows in ((1 << 31) - 1, (1 << 31) - 65)]
    assert ws[0] == ws[1] > 0


def test_descriptor_layout(tmp_path):
    import os
    import subprocess
    from vfdepth_amd import _lib
    src = tmp_path / 'sz.c'
    src.write_text('#include "vfd_capi.h"\n#include <stdio.h>\n#include <stddef.h>\nint main(){printf("%zu %zu %zu %zu", '
                   'sizeof(vfd_norm_desc), offsetof(vfd_norm_desc, ldx), offsetof(vfd_norm_desc, eps), '
                   'offsetof(vfd_norm_desc, dtype)); return 0;}\n')
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    subprocess.check_call(['gcc', '-I', os.path.join(root, 'include'), str(src), '-o', str(tmp_path / 'sz')])
    got = [int(v) for v in subprocess.check_output([str(tmp_path / 'sz')]).split()]
    N = _lib.NormDesc
    assert got == [ctypes.sizeof(N), N.ldx.offset, N.eps.offset, N.dtype.offset]


def test_cpu_takes_the_module():
    from vfdepth_amd import kernels as KN
    from vfdepth_amd import layers
    ln = torch.nn.LayerNorm(6)
    x = torch.randn(2, 6, 3, 4)
    y = layers.channel_norm(ln, x)
    want = torch.nn.functional.layer_norm(x.permute(0, 2, 3, 1), (6,), ln.weight, ln.bias).permute(0, 3, 1, 2)
    assert y.shape == x.shape and torch.equal(y, want)
    with pytest.raises(RuntimeError, match='HIP device'):
        KN.LayerNorm.apply(x, None, None, 1e-5)


# ------------------------------------------------------------------------------------------------ GPU
gpu = pytest.mark.gpu
WIDTHS = [1, 2, 3, 4, 5, 7, 8, 16, 31, 32, 33, 64, 65, 127, 128, 255, 256, 257, 512, 513, 1000, 1021, 1024, 1025, 2048,
          2049, 4096, 4097, 8191, 8192, 8193, 20001]


@gpu
@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('C', WIDTHS)
def test_widths(C, dtype):
    for rows in (1, 37):
        x, w, b, g = (t.cuda() for t in _case(rows, C, dtype, seed=C))
        y, (dx, dw, db) = _run(x, w, b, g)
        assert y.dtype == dx.dtype == dtype and dw.dtype == db.dtype == F32
        _check((y, dx, dw, db), *_oracle(x, w, b, g))


@gpu
@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('rows,C', [(2, 64), (4097, 24), (30001, 64), (9000, 256), (5761, 1021), (1500, 4096), (700, 9001), (150, 40001)])
def test_many_rows(rows, C, dtype):
    x, w, b, g = (t.cuda() for t in _case(rows, C, dtype, seed=rows))
    y, grads = _run(x, w, b, g)
    _check((y, *grads), *_oracle(x, w, b, g))
    y2, grads2 = _run(x, w, b, g)                            # fixed order of every sum
    assert torch.equal(y, y2) and all(torch.equal(a, c) for a, c in zip(grads, grads2))


@gpu
def test_inference_keeps_nothing():
    from vfdepth_amd import layers
    ln, x = torch.nn.LayerNorm(8).cuda(), torch.randn(1 << 20, 8, device='cuda')
    want = layers.layer_norm(ln, x).detach()
    with torch.no_grad():
        base = torch.cuda.memory_allocated()
        torch.cuda.reset_peak_memory_stats()
        y = layers.layer_norm(ln, x)
        assert torch.cuda.max_memory_allocated() - base <= 1.1 * y.numel() * 4
    assert not y.requires_grad and torch.equal(y, want)


@gpu
def test_no_rows_and_no_values():
    from vfdepth_amd import kernels as KN
    w = torch.ones(5, device='cuda', requires_grad=True)
    b = torch.ones(5, device='cuda', requires_grad=True)
    x = torch.empty(0, 3, 5, device='cuda', requires_grad=True)
    y = KN.LayerNorm.apply(x, w, b, EPS)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.empty_like(y))
    assert y.shape == dx.shape == (0, 3, 5) and not dw.any() and not db.any()
    with pytest.raises(RuntimeError, match='last dimension'):
        KN.LayerNorm.apply(torch.empty(3, 0, device='cuda'), None, None, EPS)
    with pytest.raises(RuntimeError, match='last dimension'):
        KN.LayerNorm.apply(torch.tensor(1.0, device='cuda'), None, None, EPS)


@gpu
@pytest.mark.parametrize('dtype', [F32, BF16])
def test_strides_and_offsets(dtype):
    """Slices of wider rows, odd starts, transposed, expanded and channels-last inputs."""
    wide = torch.randn(50, 137, device='cuda').to(dtype)
    w, b = torch.randn(100, device='cuda'), torch.randn(100, device='cuda')
    for x in (wide[:, 3:103], wide[::2, 1:101], wide[:, 37:], torch.randn(100, 60, device='cuda').to(dtype).t(),
              torch.randn(100, device='cuda').to(dtype).expand(9, 100), wide.as_strided((20, 100), (7, 1))):
        x = x.detach()
        g = torch.randn(x.shape, device='cuda').to(dtype)
        y, grads = _run(x, w, b, g)
        _check((y, *grads), *_oracle(x, w, b, g))
    x = torch.randn(2, 3, 5, 100, device='cuda').to(dtype)[:, :, 1:4]            # rows not evenly spaced: copied
    y, grads = _run(x, w, b, torch.ones(x.shape, device='cuda', dtype=dtype))
    vals, tol = _oracle(x.reshape(-1, 100), w, b, torch.ones(18, 100))
    _check((y.reshape(-1, 100), grads[0].reshape(-1, 100), *grads[1:]), vals, tol)


@gpu
@pytest.mark.parametrize('fmt', [torch.channels_last, torch.contiguous_format])
def test_channel_norm(fmt):
    from vfdepth_amd import layers
    ln = torch.nn.LayerNorm(64).cuda()
    torch.nn.init.normal_(ln.weight)
    torch.nn.init.normal_(ln.bias)
    x = torch.randn(2, 64, 6, 10, device='cuda').contiguous(memory_format=fmt).requires_grad_(True)
    g = torch.randn(2, 64, 6, 10, device='cuda')
    y = layers.channel_norm(ln, x)
    y.backward(g)
    flat = lambda t: t.detach().permute(0, 2, 3, 1).reshape(-1, 64)  # noqa: E731
    vals, tol = _oracle(flat(x), ln.weight, ln.bias, flat(g))
    assert y.is_contiguous(memory_format=torch.channels_last)
    _check((flat(y), flat(x.grad), ln.weight.grad, ln.bias.grad), vals, tol)


@gpu
def test_parts_of_the_gradient_and_missing_parameters():
    from vfdepth_amd import kernels as KN
    x, w, b, g = (t.cuda() for t in _case(300, 96, F32))
    vals, tol = _oracle(x, w, b, g)
    for need in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (0, 1, 1), (1, 0, 1)):
        leaves = [t.clone().requires_grad_(bool(n)) for t, n in zip((x, w, b), need)]
        y = KN.LayerNorm.apply(*leaves, EPS)
        grads = iter(torch.autograd.grad(y, [t for t in leaves if t.requires_grad], g))
        _check([y] + [next(grads) if n else None for n in need], vals, tol)
    for ww, bb in ((None, None), (w, None), (None, b)):
        y, grads = _run(x.clone(), ww, bb, g)
        vals2, tol2 = _oracle(x, ww, bb, g)
        grads = iter(grads)
        _check([y, next(grads), None if ww is None else next(grads), None if bb is None else next(grads)], vals2, tol2)


@gpu
def test_gradient_against_differences():
    """<d loss / d leaf, v> against central differences of the loss in 64 bits; the step's own error is h^2 / 6 f'''."""
    x, w, b, g = (t.cuda() for t in _case(40, 33, F32, seed=5))
    _, grads = _run(x, w, b, g)
    xs = [t.detach().cpu().double() for t in (x, w, b)]
    gd = g.cpu().double()

    def loss(x, w, b):
        m = x.mean(1, keepdim=True)
        return float(((x - m) / ((x - m).square().mean(1, keepdim=True) + EPS).sqrt() * w + b).mul(gd).sum())
    for k in range(3):
        v = torch.randn(xs[k].shape, dtype=torch.float64, generator=torch.Generator().manual_seed(k))
        step = 1e-4
        up, dn = ([t + s * step * v if i == k else t for i, t in enumerate(xs)] for s in (1, -1))
        diff = (loss(*up) - loss(*dn)) / (2 * step)
        got = float((grads[k].cpu().double() * v).sum())
        assert abs(got - diff) <= 1e-5 * float((grads[k].cpu().double() * v).abs().sum())


@gpu
def test_constant_rows_large_means_and_non_finite_rows():
    from vfdepth_amd import kernels as KN
    w, b = torch.randn(64, device='cuda'), torch.randn(64, device='cuda')
    x = torch.full((3, 64), 5.0, device='cuda')
    assert torch.equal(KN.LayerNorm.apply(x, w, b, EPS), b.expand(3, 64))
    x, w, b, g = (t.cuda() for t in _case(50, 64, F32, mean=300.0))
    y, grads = _run(x, w, b, g)
    _check((y, *grads), *_oracle(x, w, b, g))
    x = torch.randn(5, 300, device='cuda')
    good = KN.LayerNorm.apply(x.clone(), None, None, EPS)
    x[1, 7], x[3, 299] = math.inf, math.nan
    y = KN.LayerNorm.apply(x, None, None, EPS)
    assert torch.isnan(y[1]).all() and torch.isnan(y[3]).all() and torch.equal(y[[0, 2, 4]], good[[0, 2, 4]])


@gpu
def test_refusals():
    from vfdepth_amd import kernels as KN
    x = torch.randn(4, 8, device='cuda')
    w = torch.ones(8, device='cuda')
    for args, word in (((x.half(), w, None), 'fp32 or bf16'), ((x, w[:7], None), r'float32 \[8\]'),
                       ((x, w.to(BF16), None), r'float32 \[8\]'), ((x, w, w.view(2, 4)), r'float32 \[8\]'),
                       ((x, w.cpu(), None), 'HIP device'), ((x.cpu(), w, None), 'HIP device')):
        with pytest.raises(RuntimeError, match=word):
            KN.LayerNorm.apply(*args, EPS)
    xg = x.clone().requires_grad_(True)
    y = KN.LayerNorm.apply(xg, w, None, EPS)
    dx, = torch.autograd.grad(y.square().sum(), xg, create_graph=True)
    with pytest.raises(RuntimeError, match='once_differentiable|twice'):
        dx.sum().backward()


@gpu
def test_refuses_sizes_that_32_bits_do_not_hold():
    from vfdepth_amd import kernels as KN
    x = torch.randn(1, 1, device='cuda')
    for C in ((1 << 28) + 1, (1 << 32) + 8):                 # (the second is 8 in 32 bits)
        with pytest.raises(RuntimeError, match='2\\^28 at most'):
            KN.LayerNorm.apply(x.expand(1, C), None, None, EPS)
    with pytest.raises(RuntimeError, match='rows'):
        KN.LayerNorm.apply(x.expand((1 << 31) + 3, 1), None, None, EPS)


@gpu
def test_module_parameters_in_bf16_and_autocast():
    from vfdepth_amd import layers
    ln = torch.nn.LayerNorm(96).cuda()
    torch.nn.init.normal_(ln.weight)
    x, _, _, g = (t.cuda() for t in _case(64, 96, BF16))
    vals, tol = _oracle(x, ln.weight, ln.bias, g)
    with torch.autocast('cuda', dtype=BF16):
        y = layers.layer_norm(ln, x.requires_grad_(True))
    _check((y, *torch.autograd.grad(y, (x, ln.weight, ln.bias), g)), vals, tol)
    ln.to(BF16)                                              # parameters kept in bf16: their gradients are rounded to it
    vals, tol = _oracle(x, ln.weight, ln.bias, g)
    y = layers.layer_norm(ln, x)
    grads = torch.autograd.grad(y, (x, ln.weight, ln.bias), g)
    assert all(t.dtype == BF16 for t in (y, *grads))
    _check((y, *grads), vals, tol)


@gpu
def test_offsets_beyond_32_bits():
    """2.2 billion values: the last rows are the same as on their own, and nothing wraps onto the first ones."""
    from vfdepth_amd import kernels as KN
    rows, C = (1 << 21) + 5, 1024
    x = torch.empty(rows, C, dtype=BF16, device='cuda').normal_()
    g = torch.empty(rows, C, dtype=BF16, device='cuda').normal_()
    w, b = torch.randn(C, device='cuda'), torch.randn(C, device='cuda')
    y = KN.LayerNorm.apply(x.requires_grad_(True), w, b, EPS)
    dx, = torch.autograd.grad(y, x, g)
    for part in (slice(0, 7), slice(rows - 9, rows)):
        xs = x.detach()[part].clone().requires_grad_(True)
        ys = KN.LayerNorm.apply(xs, w, b, EPS)
        ds, = torch.autograd.grad(ys, xs, g[part].clone())
        assert torch.equal(y[part], ys) and torch.equal(dx[part], ds)


@gpu
def test_most_rows():
    """2^31 - 1 rows of two values: the first and the last ones are the same as on their own."""
    from vfdepth_amd import kernels as KN
    rows = (1 << 31) - 1
    x = torch.empty(rows, 2, dtype=BF16, device='cuda').normal_()
    g = torch.empty(rows, 2, dtype=BF16, device='cuda').normal_()
    w, b = torch.randn(2, device='cuda'), torch.randn(2, device='cuda', requires_grad=True)
    y = KN.LayerNorm.apply(x.requires_grad_(True), w, b, EPS)
    dx, db = torch.autograd.grad(y, (x, b), g)
    for part in (slice(0, 7), slice(rows - 131, rows)):
        xs = x.detach()[part].clone().requires_grad_(True)
        ys = KN.LayerNorm.apply(xs, w, b, EPS)
        ds, = torch.autograd.grad(ys, xs, g[part].clone())
        assert torch.equal(y[part], ys) and torch.equal(dx[part], ds)
    assert db.shape == (2,) and bool(torch.isfinite(db).all())


@gpu
def test_widest_rows_backward():
    """2^25 columns and some: the weight's and bias's sums are over more columns than one launch has blocks of them for."""
    x, w, b, g = (t.cuda() for t in _case(2, (1 << 25) + 19, F32, seed=4))
    y, grads = _run(x, w, b, g)
    _check((y, *grads), *_oracle(x, w, b, g))


@gpu
def test_streams_and_captured_graph():
    from vfdepth_amd import kernels as KN
    x, w, b, g = (t.cuda() for t in _case(500, 200, F32, seed=9))
    for t in (x, w, b):
        t.requires_grad_(True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = KN.LayerNorm.apply(x, w, b, EPS)
        grads = torch.autograd.grad(y, (x, w, b), g)
    torch.cuda.current_stream().wait_stream(side)
    _check((y, *grads), *_oracle(x, w, b, g))
    del y, grads
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = KN.LayerNorm.apply(x, w, b, EPS)
        grads = torch.autograd.grad(y, (x, w, b), g)
    y = y.detach()
    for k in range(4):
        with torch.no_grad():
            for t, s in zip((x, w, b, g), _case(500, 200, F32, seed=20 + k)):
                t.copy_(s)
        graph.replay()
        torch.cuda.synchronize()
        _check((y, *grads), *_oracle(x, w, b, g))
        with torch.no_grad():
            assert torch.equal(KN.LayerNorm.apply(x, w, b, EPS), y)             # eager work between replays
