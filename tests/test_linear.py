"""Linear layer with bias, activation and residual in the product's epilogue (linear.hip, kernels.LinearAct,
layers.linear_act), forward and backward.

Tolerances (u = 2^-24, h = the type's half step): a product over K values is off by at most (K + 8) u sum|a b| in any
order of summation (products of bf16 values are exact in 32 bits); an activation adds its slope's bound times that and
8 u (|z| + 1) of its own; the backward reads the pre-activation rounded to the type (h |z|), which moves a slope by its
Lipschitz constant times that, and the products take the gradient behind the activation rounded to the type (h |gz|).
Where a pre-activation lies within its own error of the kink of relu or lrelu, either slope is right.  Each output is
rounded once."""
import ctypes
import math

import pytest
import torch

F32, BF16 = torch.float32, torch.bfloat16
U = 2.0 ** -24
HALF = {F32: 2.0 ** -24, BF16: 2.0 ** -8}
TINY = 2.0 ** -126
ACTS = ['none', 'relu', 'lrelu', 'elu', 'gelu', 'silu']


def _slope(z, act):
    """(value, slope, bound of the slope's own slope) in 64 bits."""
    one = torch.ones_like(z)
    if act == 'none':
        return z, one, 0.0
    if act == 'relu':
        return z.clamp_min(0), (z > 0).double(), 0.0
    if act == 'lrelu':
        s = torch.where(z > 0, one, 0.1 * one)
        return z * s, s, 0.0
    if act == 'elu':
        n = z.clamp_max(0)
        return torch.where(z > 0, z, torch.expm1(n)), torch.exp(n), 1.0
    if act == 'gelu':
        c = 0.5 * torch.erfc(-z / math.sqrt(2))
        return z * c, c + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi), 0.8
    s = torch.sigmoid(z)
    return z * s, s * (1 + z * (1 - s)), 0.5


def _case(M, K, N, dtype, bias=True, residual=True, seed=0, device='cuda'):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    x, w, b, res, g = r(M, K), r(N, K) * K ** -0.5, r(N) * 0.3, r(M, N), r(M, N)
    return [t.to(dtype).to(device) if t is not None else None
            for t in (x, w, b if bias else None, res if residual else None, g)]


def _oracle(x, w, b, res, g, act):
    """Values and allowed errors (before the output's rounding) of y, dx, dw, db, dr."""
    hT = HALF[x.dtype]
    x, w, b, res, g = (None if t is None else t.detach().cpu().double() for t in (x, w, b, res, g))
    M, K = x.shape
    N = w.shape[0]
    z = x @ w.t()
    dz = (K + 8) * U * (x.abs() @ w.abs().t())
    if b is not None:
        z = z + b
        dz = dz + U * z.abs()
    a, s, lip = _slope(z, act)
    y = a if res is None else a + res
    ey = 1.13 * dz + (8 * U * (z.abs() + 1) if act != 'none' else 0) + U * y.abs()
    gz = g * s
    es = lip * (dz + hT * z.abs()) + 8 * U
    if act in ('relu', 'lrelu'):
        es = es + (z.abs() <= dz).double()
    eg = g.abs() * es + U * gz.abs() if act != 'none' else torch.zeros_like(gz)
    er = eg + (hT * (gz.abs() + eg) if act != 'none' else 0)
    vals = [y, gz @ w, gz.t() @ x, gz.sum(0), g]
    tol = [ey, er @ w.abs() + (N + 8) * U * (gz.abs() @ w.abs()), er.t() @ x.abs() + (M + 8) * U * (gz.abs().t() @ x.abs()),
           eg.sum(0) + (M / 64 + 60) * U * gz.abs().sum(0), torch.zeros_like(g)]
    return vals, tol


def _check(got, vals, tol):
    for t, v, e, name in zip(got, vals, tol, ('y', 'dx', 'dw', 'db', 'dr')):
        if t is None:
            continue
        err = (t.detach().cpu().double() - v).abs()
        lim = e + HALF[t.dtype] * (v.abs() + e) + TINY
        assert t.shape == v.shape and bool((err <= lim).all()), (name, float((err / lim).max()))


def _run(x, w, b, res, g, act):
    from vfdepth_amd import kernels as KN
    leaves = [t.requires_grad_(True) for t in (x, w, b, res) if t is not None]
    y = KN.LinearAct.apply(x, w, b, res, act)
    grads = iter(torch.autograd.grad(y, leaves, g))
    return [y] + [next(grads) if t is not None else None for t in (x, w, b, res)]


def _near_product(got, a, b, what, extra=0.0):
    """got against a @ b in 64 bits, for operands with random signs, tightly enough that a few missing terms show.  Of n
    terms every partial sum is rounded, by at most u of itself: together at most u sum_k |S_k|.  The partial sums of terms
    of random signs walk: |S_k| is some sqrt(sum of the terms' squares), 0.53 of it on average over k, over 3 of it on
    average in no entry here; n + 8 counts the roundings of any order, splits and products among them."""
    a, b = a.double(), b.double()
    v = a @ b
    e = 3 * (a.shape[1] + 8) * U * (a.square() @ b.square()).sqrt() + extra
    err = (got.double() - v).abs()
    lim = e + HALF[got.dtype] * (v.abs() + e) + TINY
    assert got.shape == v.shape and bool((err <= lim).all()), (what, float((err / lim).max()))


# ------------------------------------------------------------------------------------------------ CPU
def _desc(rows=4, k=8, n=8, act=0, ldx=8, dtype=0):
    from vfdepth_amd import _lib
    return _lib.LinearDesc(rows, k, n, act, ldx, dtype)


@pytest.mark.parametrize('bad', [dict(rows=-1), dict(k=0, ldx=0), dict(n=0), dict(n=-2), dict(act=6), dict(act=-1), dict(ldx=7), dict(dtype=2),
                                 dict(rows=(1 << 30) + 1), dict(rows=1 << 30, n=1 << 30)])
def test_c_refuses_bad_descriptors(bad):
    from vfdepth_amd import _lib
    lib = _lib.load()
    d = _desc(**bad)
    p = 1 << 40
    for rc in (lib.vfd_linear_fwd(ctypes.byref(d), p, p, p, p, p, p, p, 1 << 40, None),
               lib.vfd_linear_bwd(ctypes.byref(d), p, p, p, p, p, p, p, p, 1 << 40, None)):
        assert rc == -1 and (b'descriptor' in lib.vfd_last_error() or b'tiles' in lib.vfd_last_error())
    assert lib.vfd_linear_fwd_workspace(ctypes.byref(d)) == lib.vfd_linear_bwd_workspace(ctypes.byref(d), p, p, p, 1, 1) == 0


def test_c_refuses_null_tensors_and_small_workspaces():
    from vfdepth_amd import _lib
    lib = _lib.load()
    p, no = 1 << 40, None
    d = _desc()

    def bwd(g=p, z=no, w=p, x=p, dx=p, dw=p, db=p, ws=p, n=1 << 40):
        return lib.vfd_linear_bwd(ctypes.byref(d), g, z, w, x, dx, dw, db, ws, n, no)
    assert lib.vfd_linear_fwd(ctypes.byref(d), no, p, no, no, p, no, p, 1 << 40, no) == -1
    assert lib.vfd_linear_fwd(ctypes.byref(d), p, p, no, no, no, no, p, 1 << 40, no) == -1
    assert bwd(g=no) == bwd(w=no) == bwd(x=no) == bwd(ws=no) == -1
    assert bwd(dx=no, dw=no, db=no) == 0                                         # nothing asked for: nothing is launched
    d = _desc(act=4)
    assert bwd() == -1 and b'null' in lib.vfd_last_error()
    d = _desc(rows=100000, k=128, n=128, ldx=128)
    need = lib.vfd_linear_bwd_workspace(ctypes.byref(d), p, p, p, 1, 1)
    assert need > 0 and bwd(n=need - 1) == -1 and b'workspace' in lib.vfd_last_error()
    assert lib.vfd_linear_bwd_workspace(ctypes.byref(d), p, p, p, 0, 0) < need
    odd = _desc(rows=50000, k=333, n=97, ldx=333, dtype=1)                       # rows of an odd length are laid out anew
    even = _desc(rows=50000, k=334, n=98, ldx=334, dtype=1)
    copies = 2 * (50000 * 104 + 97 * 336 + 50000 * 336)
    ws = [lib.vfd_linear_bwd_workspace(ctypes.byref(t), p, p, p, 1, 1) for t in (odd, even)]
    assert ws[0] >= copies and ws[1] < copies
    assert lib.vfd_linear_bwd_workspace(ctypes.byref(even), p, p, p + 2, 1, 1) >= ws[1] + 2 * 50000 * 336     # an odd start
    d = _desc(rows=300, k=8192, n=128, ldx=8192)                                 # few tiles: the contraction is split
    need = lib.vfd_linear_fwd_workspace(ctypes.byref(d))
    assert need > 0 and lib.vfd_linear_fwd(ctypes.byref(d), p, p, no, no, p, no, p, need - 1, no) == -1
    assert lib.vfd_linear_fwd(ctypes.byref(_desc(rows=0)), *[no] * 7, 0, no) == 0


@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('M,K,N', [(18686, 584, 66), (16825, 143, 8), (17993, 8, 65), (9000, 72, 136), (300, 517, 771)])
def test_product_bound_sees_missing_terms(M, K, N, dtype):
    """The bound of the products' tests, on mistakes planted here: rows left out, added twice or taken from elsewhere, in one
    32 x 32 block of the product alone."""
    x, _, _, _, gz = _case(M, K, N, dtype, residual=False, seed=M, device='cpu')
    good = gz.double().t() @ x.double()
    _near_product(good.to(dtype), gz.t(), x, 'dw')
    c = min(N, 32), min(K, 32)
    a, b = gz[:, :c[0]].double(), x[:, :c[1]].double()
    for wrong in (-a[-32:].t() @ b[-32:], a[:16].t() @ b[:16], a[64:96].t() @ (b[96:128] - b[64:96])):
        bad = good.clone()
        bad[:c[0], :c[1]] += wrong
        with pytest.raises(AssertionError, match='dw'):
            _near_product(bad.to(dtype), gz.t(), x, 'dw')


@pytest.mark.parametrize('dtype', [0, 1])
def test_bias_gradient_alone_needs_no_activation_gradient(dtype):
    """Only column sums: one fp32 row for each of at most 1024 row blocks."""
    from vfdepth_amd import _lib
    lib = _lib.load()
    for act in (0, 3, 4):
        d = _desc(rows=92160, k=256, n=1024, act=act, ldx=256, dtype=dtype)
        need = lib.vfd_linear_bwd_workspace(ctypes.byref(d), 1 << 40, 1 << 40, 1 << 40, 0, 0)
        assert 0 < need <= 1024 * 1024 * 4, need


@pytest.mark.parametrize('rows,k,n,ldx,dx,dw,most', [
    (10_000_000, 255, 1, 255, 0, 1, 160e6), (10_000_000, 255, 1, 255, 1, 1, 160e6),       # one output: 160 MB of g, 5 GB of x
    (10_000_000, 1, 255, 1, 1, 1, 160e6), (50_000, 7, 9001, 7, 1, 1, 100e6),               # rows of x below a chunk: 5 GB, 0.9 GB of g
    (9, 20_001, 20_001, 20_001, 0, 1, 3e5), (1_000_003, 333, 31, 333, 1, 0, 32e6),         # contractions inside their first tile
    (100_003, 1001, 1003, (1 << 20) + 2, 0, 1, 100e6)])                                    # rows of x too far apart
def test_no_copies_for_products_that_cannot_stream(rows, k, n, ldx, dx, dw, most):
    """Odd bf16 rows are laid out anew only for a product that can then stream both operands."""
    from vfdepth_amd import _lib
    lib = _lib.load()
    p = 1 << 40
    got = lib.vfd_linear_bwd_workspace(ctypes.byref(_desc(rows=rows, k=k, n=n, ldx=ldx, dtype=1)), p, p, p, dx, dw)
    assert got < most, got
    even = 100_004, 1002, 1004, 1002                                             # and where it can: g, w and x
    odd = 100_003, 1001, 1003, 1001
    ws = [lib.vfd_linear_bwd_workspace(ctypes.byref(_desc(rows=r, k=k, n=n, ldx=l, dtype=1)), p, p, p, 1, 1)
          for r, k, n, l in (even, odd)]
    assert ws[1] >= 2 * (100_003 * 1008 + 1003 * 1008 + 100_003 * 1008) > ws[0]


def test_descriptor_layout(tmp_path):
    import os
    import subprocess
    from vfdepth_amd import _lib
    src = tmp_path / 'sz.c'
    src.write_text('#include "vfd_capi.h"\n#include <stdio.h>\n#include <stddef.h>\nint main(){printf("%zu %zu %zu %zu", '
                   'sizeof(vfd_linear_desc), offsetof(vfd_linear_desc, act), offsetof(vfd_linear_desc, ldx), '
                   'offsetof(vfd_linear_desc, dtype)); return 0;}\n')
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    subprocess.check_call(['gcc', '-I', os.path.join(root, 'include'), str(src), '-o', str(tmp_path / 'sz')])
    got = [int(v) for v in subprocess.check_output([str(tmp_path / 'sz')]).split()]
    D = _lib.LinearDesc
    assert got == [ctypes.sizeof(D), D.act.offset, D.ldx.offset, D.dtype.offset]


@pytest.mark.parametrize('act', ACTS)
def test_cpu_takes_the_module(act):
    from vfdepth_amd import layers
    torch.manual_seed(0)
    lin, conv = torch.nn.Linear(5, 7).double(), torch.nn.Conv2d(5, 7, 1).double()
    x, r = torch.randn(2, 3, 5).double(), torch.randn(2, 3, 7).double()
    want = _slope(x @ lin.weight.t() + lin.bias, act)[0] + r
    assert torch.allclose(layers.linear_act(lin, x, act, r), want, rtol=1e-12, atol=1e-12)
    m = torch.randn(2, 5, 3, 4).double()
    want = _slope(torch.einsum('nkhw,ok->nohw', m, conv.weight[:, :, 0, 0]) + conv.bias[:, None, None], act)[0]
    assert torch.allclose(layers.linear_act(conv, m, act), want, rtol=1e-12, atol=1e-12)


def test_layer_refusals():
    from vfdepth_amd import kernels as KN
    from vfdepth_amd import layers
    with pytest.raises(ValueError, match='act is one of'):
        layers.linear_act(torch.nn.Linear(2, 2), torch.zeros(1, 2), 'tanh')
    for conv in (torch.nn.Conv2d(4, 4, 3), torch.nn.Conv2d(4, 4, 1, stride=2), torch.nn.Conv2d(4, 4, 1, groups=2),
                 torch.nn.Conv2d(4, 4, 1, padding=1)):
        with pytest.raises(ValueError, match='1x1'):
            layers.linear_act(conv, torch.zeros(1, 4, 5, 5))
    with pytest.raises(ValueError, match='1x1'):
        layers.linear_act(torch.nn.Conv2d(4, 4, 1), torch.zeros(4, 5, 5))
    with pytest.raises(RuntimeError, match='HIP device'):
        KN.LinearAct.apply(torch.zeros(2, 3), torch.zeros(4, 3), None, None, 'none')


# ------------------------------------------------------------------------------------------------ GPU
gpu = pytest.mark.gpu
SHAPES = [(1, 1, 1), (1, 8, 8), (2, 3, 5), (5, 3, 7), (17, 64, 64), (6, 2048, 256), (33, 100, 31), (64, 96, 300), (65, 40, 513),
          (128, 128, 128), (129, 127, 130), (256, 64, 256), (257, 1024, 96), (300, 517, 771), (1000, 8, 2000), (3000, 40, 24),
          (520, 260, 260), (16, 4096, 512), (9000, 72, 136),
          (3001, 127, 131), (2100, 259, 130), (700, 1001, 515), (1024, 126, 250), (1500, 131, 258)]


@gpu
@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('M,K,N', SHAPES)
def test_shapes(M, K, N, dtype):
    args = _case(M, K, N, dtype, seed=M + K)
    _check(_run(*args, 'gelu'), *_oracle(*args, 'gelu'))


@gpu
@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('bias,residual', [(True, True), (True, False), (False, True), (False, False)])
@pytest.mark.parametrize('act', ACTS)
def test_activations(act, bias, residual, dtype):
    args = _case(200, 96, 136, dtype, bias, residual, seed=len(act))
    out = _run(*args, act)
    _check(out, *_oracle(*args, act))
    again = _run(*args, act)
    assert all(torch.equal(a, b) for a, b in zip(out, again) if a is not None)
    from vfdepth_amd import kernels as KN
    with torch.no_grad():                                        # without a pre-activation to keep: the same bits
        assert torch.equal(KN.LinearAct.apply(*args[:4], act), out[0])
        assert torch.equal(KN.LinearAct.infer(*args[:4], act), out[0])


@gpu
@pytest.mark.parametrize('dtype', [F32, BF16])
def test_large_product(dtype):
    """Enough tiles for the largest tile form, ragged in each direction; odd pitches, whose rows the backward lays out anew."""
    for M, K, N in ((4200, 1160, 4104), (4100, 333, 771), (4099, 1001, 515)):
        args = _case(M, K, N, dtype, seed=7)
        _check(_run(*args, 'silu'), *_oracle(*args, 'silu'))
        x, w, b, _, g = args
        args = [x[:, 1:], w[:, 1:].detach(), b, None, g]                # an odd start and a pitch of its own
        args = [t if t is None else t.detach() for t in args]
        _check(_run(*args, 'none'), *_oracle(*args, 'none'))


# Ragged sizes at which each tile form and split is taken, in either type (forward, data gradient or weight gradient)
FORMS = [(12687, 9, 193), (17993, 8, 65), (16825, 143, 8), (12431, 216, 528), (18686, 584, 66), (12887, 523, 208), (66, 4786, 1610),
         (4491, 66, 1637), (1175, 3280, 8), (818, 8, 2255), (4679, 823, 10), (71, 1291, 4321), (2645, 65, 1800), (16759, 662, 1041),
         (19948, 1040, 560), (1092, 3354, 3601)]


@gpu
@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('M,K,N', FORMS)
def test_tile_forms(M, K, N, dtype):
    args = _case(M, K, N, dtype, seed=M)
    _check(_run(*args, 'elu'), *_oracle(*args, 'elu'))


@gpu
@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('act', ['none', 'elu', 'gelu'])
@pytest.mark.parametrize('M,K,N', SHAPES + FORMS + [(4200, 1160, 4104)])
def test_products(M, K, N, act, dtype):
    """Every product against 64 bits on the operands that it really took.  The pre-activation is what the layer without an
    activation returns; its gradient is what a layer of unit weights gives back (times one and plus zeros: exact)."""
    from vfdepth_amd import kernels as KN
    x, w, b, _, g = _case(M, K, N, dtype, residual=False, seed=M + N)
    y, dx, dw, db, _ = _run(x, w, b, None, g, act)
    with torch.no_grad():
        z = KN.LinearAct.infer(x, w, b, None, 'none')
        zd, bd = x.double() @ w.double().t(), b.double()
        _near_product(z, torch.cat([x, b.new_ones(M, 1)], 1), torch.cat([w, b[:, None]], 1).t(), 'z', U * (zd.abs() + bd.abs()))
    gz = g
    if act != 'none':
        one = torch.eye(N, device='cuda', dtype=dtype)
        gz, = torch.autograd.grad(KN.LinearAct.apply(z.requires_grad_(True), one, None, None, act), z, g)
    with torch.no_grad():
        gd = g.double()
        _, slope, _ = _slope(z.double(), act)
        exact = gd * slope
        if act == 'none':
            assert torch.equal(y, z)
        else:
            e = 8 * U * gd.abs() + U * exact.abs()
            assert bool(((gz.double() - exact).abs() <= e + HALF[dtype] * (exact.abs() + e) + TINY).all())
        _near_product(dx, gz, w, 'dx')
        _near_product(dw, gz.t(), x, 'dw')
        _near_product(db[None], torch.ones(1, M, device='cuda'), exact, 'db', 8 * U * gd.abs().sum(0) if act != 'none' else 0)


@gpu
@pytest.mark.parametrize('dtype', [F32, BF16])
def test_strides_offsets_and_leading_dimensions(dtype):
    wide = torch.randn(60, 211, device='cuda').to(dtype)
    w = (torch.randn(50, 100, device='cuda') * 0.1).to(dtype)
    b = torch.randn(50, device='cuda').to(dtype)
    for x in (wide[:, 8:108], wide[:, 3:103], wide[::2, 1:101], torch.randn(100, 60, device='cuda').to(dtype).t(),
              torch.randn(100, device='cuda').to(dtype).expand(9, 100), wide.as_strided((20, 100), (7, 1))):
        M = x.shape[0]
        g = torch.randn(M, 50, device='cuda').to(dtype)
        res = torch.randn(50, M, device='cuda').to(dtype).t()
        args = [x.detach(), w, b, res.detach(), g]
        _check(_run(*args, 'elu'), *_oracle(*args, 'elu'))
    wt = (torch.randn(100, 50, device='cuda') * 0.1).to(dtype).t()              # a weight stored transposed
    x = torch.randn(2, 3, 7, 100, device='cuda').to(dtype)
    res = torch.randn(7, 50, device='cuda').to(dtype).expand(2, 3, 7, 50)
    g = torch.randn(2, 3, 7, 50, device='cuda').to(dtype)
    out = _run(x, wt, b, res.detach(), g, 'lrelu')
    assert out[0].shape == g.shape and out[1].shape == x.shape
    flat = lambda t: t.detach().reshape(-1, t.shape[-1])  # noqa: E731
    vals, tol = _oracle(flat(x), wt, b, flat(res), flat(g), 'lrelu')
    _check([flat(out[0]), flat(out[1]), out[2], out[3], flat(out[4])], vals, tol)
    shared = torch.randn(1, 1, 1, 50, device='cuda').to(dtype).requires_grad_(True)          # a broadcast residual's gradient
    from vfdepth_amd import kernels as KN
    y = KN.LinearAct.apply(x, wt, b, shared.expand(2, 3, 7, 50), 'none')
    ds, = torch.autograd.grad(y, shared, g)
    want = g.cpu().double().sum((0, 1, 2))
    lim = (HALF[dtype] + 50 * U) * g.cpu().double().abs().sum((0, 1, 2))
    assert bool(((ds.flatten().cpu().double() - want).abs() <= lim).all())
    s = KN.LinearAct.apply(x, wt, b, None, 'none').sum()                          # an expanded incoming gradient
    s.backward()


@gpu
def test_no_rows():
    from vfdepth_amd import kernels as KN
    x = torch.empty(2, 0, 12, device='cuda', requires_grad=True)
    w = torch.randn(5, 12, device='cuda', requires_grad=True)
    b = torch.randn(5, device='cuda', requires_grad=True)
    y = KN.LinearAct.apply(x, w, b, None, 'gelu')
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.empty_like(y))
    assert y.shape == (2, 0, 5) and dx.shape == x.shape and not dw.any() and not db.any()


@gpu
@pytest.mark.parametrize('act', ['none', 'gelu'])
def test_parts_of_the_gradient(act):
    from vfdepth_amd import kernels as KN
    x, w, b, res, g = _case(70, 48, 56, F32, seed=2)
    vals, tol = _oracle(x, w, b, res, g, act)
    for need in ((1, 0, 0, 0), (0, 1, 0, 0), (0, 0, 1, 0), (0, 0, 0, 1), (0, 1, 1, 0), (1, 0, 0, 1)):
        leaves = [t.clone().requires_grad_(bool(n)) for t, n in zip((x, w, b, res), need)]
        y = KN.LinearAct.apply(*leaves, act)
        grads = iter(torch.autograd.grad(y, [t for t in leaves if t.requires_grad], g))
        _check([y] + [next(grads) if n else None for n in need], vals, tol)


@gpu
@pytest.mark.parametrize('act', ['none', 'silu'])
@pytest.mark.parametrize('M,K,N', [(2_000_000, 255, 3), (2_000_000, 3, 255), (30_001, 7, 9001), (9, 13_001, 13_003), (200_003, 333, 31),
                                   (40_001, 255, 257)])
def test_odd_rows_of_short_products(M, K, N, act):
    """Odd bf16 rows with one size below a chunk or a tile (no copies), and above (copies), enough terms for either: the last
    rows and columns against the oracle, the weight's gradient of rows that are zero but for those."""
    from vfdepth_amd import kernels as KN
    x, w, b, _, g = _case(M, K, N, BF16, residual=False, seed=K)
    g[:-300] = 0
    y, dx, dw, db, _ = _run(x, w, b, None, g, act)
    vals, tol = _oracle(x[-300:], w, b, None, g[-300:], act)
    _check([y[-300:], dx[-300:], dw, db], vals, tol)
    assert not dx[:-300].any()
    dw2, = torch.autograd.grad(KN.LinearAct.apply(x.detach(), w, b.detach(), None, act), w, g)       # its copies alone
    dx2, = torch.autograd.grad(KN.LinearAct.apply(x, w.detach(), b.detach(), None, act), x, g)
    _check([None, dx2[-300:], dw2], vals, tol)


@gpu
@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('act', ACTS)
def test_bias_gradient_alone(act, dtype):
    """No product reads the activation's gradient here: the sums are the same bits as beside the other gradients."""
    from vfdepth_amd import kernels as KN
    x, w, b, _, g = _case(2100, 96, 300, dtype, seed=21)
    want = _run(x, w, b, None, g, act)[3]
    b = b.detach().requires_grad_(True)
    db, = torch.autograd.grad(KN.LinearAct.apply(x.detach(), w.detach(), b, None, act), b, g)
    assert torch.equal(db, want)


@gpu
def test_gradient_against_differences():
    args = _case(20, 24, 28, F32, seed=5)
    grads = _run(*args, 'gelu')[1:]
    xs = [t.detach().cpu().double() for t in args[:4]]
    gd = args[4].cpu().double()

    def loss(x, w, b, res):
        return float(((_slope(x @ w.t() + b, 'gelu')[0] + res) * gd).sum())
    for k in range(4):
        v = torch.randn(xs[k].shape, dtype=torch.float64, generator=torch.Generator().manual_seed(k))
        up, dn = ([t + s * 1e-4 * v if i == k else t for i, t in enumerate(xs)] for s in (1, -1))
        diff = (loss(*up) - loss(*dn)) / 2e-4
        prod = grads[k].cpu().double() * v
        assert abs(float(prod.sum()) - diff) <= 1e-5 * float(prod.abs().sum())


@gpu
@pytest.mark.parametrize('dtype', [F32, BF16])
def test_non_finite_rows_stay_in_their_rows(dtype):
    """Garbage in one row (or beyond the last) does not reach another: tiles are ragged in every direction here."""
    from vfdepth_amd import kernels as KN
    x, w, b, _, g = _case(150, 77, 90, dtype, seed=3)
    with torch.no_grad():
        good = KN.LinearAct.apply(x, w, b, None, 'relu')
        wide = torch.full((152, 80), math.nan, device='cuda').to(dtype)
        wide[1:151, 2:79] = x
        wide[40, 5] = math.inf
        y = KN.LinearAct.apply(wide[1:151, 2:79], w, b, None, 'relu')
    keep = [i for i in range(150) if i != 39]
    assert torch.equal(y[keep], good[keep]) and not torch.isfinite(y[39]).all()
    xn = x.clone()
    xn[3, 4] = math.nan
    assert torch.isnan(KN.LinearAct.apply(xn, w, b, None, 'relu')[3]).all()


@gpu
@pytest.mark.parametrize('dtype', [F32, BF16])
def test_relu_stops_non_finite_gradients(dtype):
    x, w, b, _, g = _case(70, 24, 40, dtype, seed=9)
    with torch.no_grad():
        off = (x.float() @ w.float().t() + b.float() < -0.05)
    clean, bad = g.masked_fill(off, 0), g.masked_fill(off, math.inf)
    bad[1::2] = g[1::2].masked_fill(off[1::2], math.nan)
    outs = [_run(x.detach(), w.detach(), b.detach(), None, t, 'relu') for t in (clean, bad)]
    for a, c in zip(*outs):
        assert a is None or torch.equal(a, c)


@gpu
def test_inference_keeps_nothing():
    """Without a graph neither a pre-activation is written nor its memory taken, though the weights want gradients."""
    from vfdepth_amd import layers
    lin = torch.nn.Linear(64, 4096).cuda()
    x = torch.randn(4096, 64, device='cuda')
    want = layers.linear_act(lin, x, 'gelu').detach()
    with torch.no_grad():
        base = torch.cuda.memory_allocated()
        torch.cuda.reset_peak_memory_stats()
        y = layers.linear_act(lin, x, 'gelu')
        assert torch.cuda.max_memory_allocated() - base <= 1.25 * y.numel() * 4
    assert not y.requires_grad and torch.equal(y, want)


@gpu
def test_very_wide_output():
    """A row of x against more weights than one launch of the few-rows form has blocks for: K = 1, so a product is exact to
    its rounding."""
    from vfdepth_amd import kernels as KN
    w = torch.randn((1 << 26) + 133, 1, device='cuda').bfloat16()
    x = torch.tensor([[1.5], [-3.0]], device='cuda').bfloat16()
    y = KN.LinearAct.infer(x, w, None, None, 'none')
    assert torch.equal(y, (x.float() * w.float().t()).bfloat16())


@gpu
def test_very_wide_output_backward():
    """As many bias gradients as one launch has no blocks for.  A sum of two bf16 values is rounded once to 32 bits and once
    to its type, and their products are exact in 32 bits: K = 1 leaves one addition a weight."""
    x, w, b, _, g = _case(2, 1, (1 << 26) + 133, BF16, residual=False, seed=6)
    y, dx, dw, db, _ = _run(x, w, b, None, g, 'none')
    x, w, b = x.detach().double(), w.detach().double(), b.detach().double()
    near = lambda t, v, e: bool(((t.double() - v).abs() <= e + HALF[BF16] * (v.abs() + e) + TINY).all())  # noqa: E731
    with torch.no_grad():
        assert torch.equal(db, (g[0].float() + g[1].float()).bfloat16())
        z = x @ w.t()
        assert near(y, z + b, 10 * U * (z.abs() + b.abs()))
        gd = g.double()
        assert near(dw, gd.t() @ x, 10 * U * (gd.abs().t() @ x.abs()))
        assert near(dx, gd @ w, (w.shape[0] + 8) * U * (gd.abs() @ w.abs()))


@gpu
def test_most_rows():
    from vfdepth_amd import kernels as KN
    x = torch.empty(1 << 30, 1, device='cuda', dtype=BF16).uniform_(-2, 2)
    w = torch.full((1, 1), 1.75, device='cuda', dtype=BF16)
    y = KN.LinearAct.infer(x, w, None, None, 'none')
    assert torch.equal(y, (x.float() * 1.75).bfloat16())


@gpu
def test_refusals():
    from vfdepth_amd import kernels as KN
    x, w, b, r, _ = _case(4, 8, 6, F32)
    for args, word in (((x, w.to(BF16), None, None), 'weight'), ((x, w[:, :7], None, None), 'weight'),
                       ((x, w, b[:5], None), 'bias'), ((x, w, b, r[:3]), 'residual'), ((x, w, b, r.to(BF16)), 'residual'),
                       ((x.half(), w.half(), None, None), 'fp32 or bf16'), ((x, w.cpu(), None, None), 'HIP device'),
                       ((x, w, b.cpu(), None), 'HIP device'), ((x, w.view(-1), None, None), 'weight'),
                       ((x[:, :0], w[:, :0], None, None), 'at least 1'), ((x, w[:0], None, None), 'at least 1')):
        with pytest.raises(RuntimeError, match=word):
            KN.LinearAct.apply(*args, 'none')
    with pytest.raises(ValueError, match='act is one of'):
        KN.LinearAct.apply(x, w, b, r, 'softmax')
    y = KN.LinearAct.apply(x.requires_grad_(True), w, b, r, 'gelu')
    dx, = torch.autograd.grad(y.square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match='once_differentiable|twice'):
        dx.sum().backward()


@gpu
def test_refuses_sizes_that_32_bits_do_not_hold():
    from vfdepth_amd import kernels as KN
    one = torch.randn(1, 1, device='cuda')
    for n in ((1 << 30) + 1, (1 << 32) + 8):                         # (the second is 8 in 32 bits)
        with pytest.raises(RuntimeError, match='at most 2\\^30'):
            KN.LinearAct.apply(one, one.expand(n, 1), None, None, 'none')
        with pytest.raises(RuntimeError, match='at most 2\\^30'):
            KN.LinearAct.apply(one.expand(1, n), one.expand(1, n), None, None, 'none')
    with pytest.raises(RuntimeError, match='descriptor|rows'):
        KN.LinearAct.apply(one.expand((1 << 31) + 3, 1), one, None, None, 'none')


@gpu
@pytest.mark.parametrize('fmt', [torch.channels_last, torch.contiguous_format])
def test_conv_1x1(fmt):
    from vfdepth_amd import layers
    conv = torch.nn.Conv2d(40, 24, 1).cuda().to(memory_format=fmt)
    x = torch.randn(2, 40, 5, 9, device='cuda').contiguous(memory_format=fmt).requires_grad_(True)
    r = torch.randn(2, 24, 5, 9, device='cuda').contiguous(memory_format=fmt).requires_grad_(True)
    g = torch.randn(2, 24, 5, 9, device='cuda')
    y = layers.linear_act(conv, x, 'elu', r)
    y.backward(g)
    assert y.is_contiguous(memory_format=torch.channels_last) and conv.weight.grad.shape == (24, 40, 1, 1)
    flat = lambda t: t.detach().permute(0, 2, 3, 1).reshape(-1, t.shape[1])  # noqa: E731
    vals, tol = _oracle(flat(x), conv.weight.flatten(1), conv.bias, flat(r), flat(g), 'elu')
    _check([flat(y), flat(x.grad), conv.weight.grad.flatten(1), conv.bias.grad, flat(r.grad)], vals, tol)


@gpu
def test_autocast():
    """Under bf16 autocast the operands are cast once, and the fp32 parameters get fp32 gradients of the cast's."""
    from vfdepth_amd import layers
    lin = torch.nn.Linear(64, 72).cuda()
    x, _, _, r, g = _case(90, 64, 72, BF16, seed=4)
    x.requires_grad_(True)
    with torch.autocast('cuda', dtype=BF16):
        y = layers.linear_act(lin, x, 'gelu', r)
    dx, dw, db = torch.autograd.grad(y, (x, lin.weight, lin.bias), g)
    assert y.dtype == dx.dtype == BF16 and dw.dtype == db.dtype == F32
    vals, tol = _oracle(x, lin.weight.to(BF16), lin.bias.to(BF16), r, g, 'gelu')
    _check([y, dx, dw.to(BF16), db.to(BF16)], vals, tol)


@gpu
def test_autocast_leaves_64_bits():
    """As torch's autocast: fp64 operands are not cast, and mixed ones do not pass."""
    from vfdepth_amd import layers
    lin = torch.nn.Linear(24, 16).cuda().double()
    x = torch.randn(7, 24, device='cuda', dtype=torch.float64, requires_grad=True)
    with torch.autocast('cuda', dtype=BF16):
        y, want = layers.linear_act(lin, x, 'elu', x[:, :16]), torch.nn.functional.elu(lin(x)) + x[:, :16]
        assert y.dtype == torch.float64 and torch.allclose(y, want, rtol=1e-12, atol=1e-12)
        assert torch.autograd.grad(y.sum(), x)[0].dtype == torch.float64
        narrow = torch.nn.Linear(24, 16).cuda()
        for m, t in ((lin, x.detach().float()), (narrow, torch.ones(7, 24, dtype=torch.int64, device='cuda'))):
            for call in (lambda: m(t), lambda: layers.linear_act(m, t, 'elu')):
                with pytest.raises(RuntimeError):
                    call()


@gpu
@pytest.mark.parametrize('conv', [False, True])
def test_autocast_adds_a_wider_residual_in_its_type(conv):
    """Under bf16 autocast an fp32 residual stays fp32 and makes the output fp32, as in torch: only the product and its
    activation are rounded to bf16, and the residual's gradient is the incoming one."""
    from vfdepth_amd import layers
    lin = (torch.nn.Conv2d(64, 72, 1) if conv else torch.nn.Linear(64, 72)).cuda()
    x, _, _, _, _ = _case(90, 64, 72, BF16, seed=14)
    gen = torch.Generator().manual_seed(15)
    r, g = (torch.randn(90, 72, generator=gen).cuda() for _ in range(2))
    shaped = (lambda t: t.view(2, 5, 9, -1).permute(0, 3, 1, 2)) if conv else (lambda t: t)
    flat = (lambda t: t.permute(0, 2, 3, 1).reshape(90, -1)) if conv else (lambda t: t)
    x.requires_grad_(True), r.requires_grad_(True)
    for grad in (True, False):
        with torch.autocast('cuda', dtype=BF16), torch.set_grad_enabled(grad):
            y = layers.linear_act(lin, shaped(x), 'gelu', shaped(r))
            assert y.dtype == (_slope(lin(shaped(x)).detach(), 'none')[0] + shaped(r)).dtype == F32
        w, b = lin.weight.detach().view(72, 64).to(BF16), lin.bias.detach().to(BF16)
        vals, tol = _oracle(x, w, b, None, g.to(BF16), 'gelu')
        yd, rd = flat(y).detach().cpu().double(), r.detach().cpu().double()
        lim = tol[0] + HALF[BF16] * (vals[0].abs() + tol[0]) + U * (yd.abs() + rd.abs())
        assert bool(((yd - rd - vals[0]).abs() <= lim).all())
        if grad:
            dx, dw, db, dr = torch.autograd.grad(y, (x, lin.weight, lin.bias, r), shaped(g))
            assert torch.equal(dr, g)
            _check([None, dx, dw.view(72, 64).to(BF16), db.to(BF16)], vals, tol)


@gpu
def test_offsets_beyond_32_bits():
    """Input, output and weight-gradient reads of 2.2 billion values each: rows at both ends against the oracle."""
    from vfdepth_amd import kernels as KN
    M, K, N = (1 << 21) + 37, 1032, 1032
    x = torch.empty(M, K, dtype=BF16, device='cuda').normal_()
    w = (torch.randn(N, K, device='cuda') * K ** -0.5).to(BF16)
    b = torch.randn(N, device='cuda').to(BF16)
    with torch.no_grad():
        y = KN.LinearAct.apply(x, w, b, None, 'gelu')
    for part in (slice(0, 40), slice(M - 300, M)):
        vals, tol = _oracle(x[part], w, b, None, torch.zeros(1, N), 'gelu')
        _check([y[part]], vals, tol)
    # the weight's gradient of rows that are zero but for the last ones: theirs alone
    g = torch.zeros(M, N, dtype=BF16, device='cuda')
    g[-20:] = torch.randn(20, N, device='cuda').to(BF16)
    wg = w.clone().requires_grad_(True)
    xg = x.requires_grad_(True)
    dx, dw = torch.autograd.grad(KN.LinearAct.apply(xg, wg, b, None, 'none'), (xg, wg), g)
    vals, tol = _oracle(x[-20:], w, b, None, g[-20:], 'none')
    _check([None, dx[-20:], dw], vals, tol)
    assert not dx[:1000].any()


@gpu
@pytest.mark.parametrize('dtype', [F32, BF16])
def test_streams_and_captured_graph(dtype):
    from vfdepth_amd import kernels as KN
    args = _case(3000, 40, 24, dtype, seed=9)                        # the weight's gradient is split and joined
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = _run(*args, 'silu')
    torch.cuda.current_stream().wait_stream(side)
    _check(out, *_oracle(*args, 'silu'))
    del out
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _run(*args, 'silu')
    out = [t.detach() for t in out]
    for k in range(4):
        with torch.no_grad():
            for t, s in zip(args, _case(3000, 40, 24, dtype, seed=30 + k)):
                t.copy_(s)
        graph.replay()
        torch.cuda.synchronize()
        _check(out, *_oracle(*args, 'silu'))
        with torch.no_grad():
            assert torch.equal(KN.LinearAct.apply(*args[:4], 'silu'), out[0])         # eager work between replays
