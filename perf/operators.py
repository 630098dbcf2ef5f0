"""The transformer-style dense operators of the framework as measured cases: layer norm, the matrix product with bias,
activation and residual in its epilogue, and the global gradient norm with clipping.

`run` computes a case in its plain form (elementary torch operations in 32 bits, rounded once at the end) or, with `own` set,
by the calls that a user makes of `vfdepth_amd.layers` and `vfdepth_amd.kernels`.
"""
import math

import torch

own = False

DTYPES = {'fp32': torch.float32, 'bf16': torch.bfloat16}
LN_EPS = 1e-5

# Row counts are tokens or map positions: 23 040 = 6 cameras x 48 x 80 (the 1/8 maps of a 384 x 640 step), 92 160 = the 1/4
# maps, 368 640 = the half-resolution maps; 64, 256, 512, 1024 and 2048 are the widths of the encoders and of reduce_dim.


def listed():
    return [
        # layer norm: one frame's camera tokens at inference, where the launch is all there is
        dict(name='norm_tokens_fwd_bf16', op='norm', dtype='bf16', train=False, rows=6, cols=256, wide=0),
        # the fused 1/8 maps of a training step in the framework's default precision
        dict(name='norm_map_train_fp32', op='norm', dtype='fp32', train=True, rows=23040, cols=256, wide=0),
        # narrow rows, very many of them: the half-resolution maps
        dict(name='norm_narrow_train_bf16', op='norm', dtype='bf16', train=True, rows=368640, cols=64, wide=0),
        # wide hidden rows, the largest activations
        dict(name='norm_wide_train_bf16', op='norm', dtype='bf16', train=True, rows=23040, cols=4096, wide=0),
        # odd width, taken out of a wider buffer (a slice of concatenated features)
        dict(name='norm_odd_train_fp32', op='norm', dtype='fp32', train=True, rows=5761, cols=1021, wide=7),
        # product: a head on one frame's six cameras (squeeze of the widest encoder), the weight's bytes count
        dict(name='linear_tokens_fwd_bf16', op='linear', dtype='bf16', train=False, rows=6, k=2048, n=256, act='relu',
             bias=True, residual=False),
        # ragged everything at inference, joined to a residual
        dict(name='linear_odd_fwd_bf16', op='linear', dtype='bf16', train=False, rows=1471, k=517, n=771, act='lrelu',
             bias=True, residual=True),
        # expansion of the 1/8 maps in a training step, default precision
        dict(name='linear_map_train_fp32', op='linear', dtype='fp32', train=True, rows=23040, k=256, n=1024, act='elu',
             bias=True, residual=False),
        # projection back with the residual joined, mixed precision: memory and matrix cores in balance
        dict(name='linear_join_train_bf16', op='linear', dtype='bf16', train=True, rows=92160, k=1024, n=256, act='none',
             bias=True, residual=True),
        # a wide hidden layer: bound by the matrix cores
        dict(name='linear_wide_train_bf16', op='linear', dtype='bf16', train=True, rows=16384, k=2048, n=8192, act='gelu',
             bias=True, residual=False),
        # gradients of both networks below the limit, clipped in place: only the norm is computed
        dict(name='clip_nets_under_fp32', op='clip', dtype='fp32', out='', tensors=162, elements=28_000_000, over=False),
        # bf16 gradients of a large model over the limit, clipped into an optimizer's fp32 buffer
        dict(name='clip_large_over_bf16', op='clip', dtype='bf16', out='fp32', tensors=291, elements=200_000_000, over=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(['norm', 'linear', 'linear', 'clip'])
    dtype = rng.choice(['fp32', 'bf16'])
    even = rng.random() < 0.5                       # half of the drawn widths are multiples of 8, the others as they fall
    width = (lambda lo, hi: max(8, _log(rng, lo, hi) // 8 * 8)) if even else (lambda lo, hi: _log(rng, lo, hi))
    if op == 'norm':
        # a row of under 8 values has most of its gradient cancelled by the two means: no type holds what is left
        cols = width(8, 8192)
        rows = _log(rng, 1, min(368640, (1 << 26) // cols))
        return dict(op=op, dtype=dtype, train=rng.random() < 0.7, rows=rows, cols=cols, wide=rng.choice([0, 0, 0, 8, 3]))
    if op == 'linear':
        train = rng.random() < 0.6
        # the slope of relu / lrelu at a pre-activation next to zero is decided by its last bit: in 32 bits their training
        # outputs cannot be compared between two orders of summation, so those draws take the smooth activations
        kinds = ['none', 'elu', 'gelu', 'silu'] + ([] if train and dtype == 'fp32' else ['relu', 'lrelu'])
        k, n = width(8, 4096), width(8, 4096)
        rows = _log(rng, 1, min(92160, (1 << 26) // max(k, n), 10 ** 11 // (k * n)))
        return dict(op=op, dtype=dtype, train=train, rows=rows, k=k, n=n, act=rng.choice(kinds), bias=rng.random() < 0.8,
                    residual=rng.random() < 0.5)
    tensors = _log(rng, 1, 400)
    over = rng.random() < 0.6
    return dict(op=op, dtype=dtype, out=rng.choice(['fp32', 'bf16']) if over else '', tensors=tensors,
                elements=_log(rng, 40 * tensors, 60_000_000), over=over)


def _randn(shape, gen, scale=1.0, shift=0.0, dtype=torch.float32):
    return (torch.randn(shape, generator=gen, device='cuda') * scale + shift).to(dtype)


def _sizes(tensors, elements):
    """Sizes of a model's gradients: a few large weights, many small vectors, lengths as they fall."""
    share = [(1.0, 0.02, 4.0, 0.005, 16.0, 0.01)[i % 6] for i in range(tensors)]
    each = [max(1, int(elements * s / sum(share))) for s in share]
    each[0] += max(0, elements - sum(each))
    return each


def prepare(case, seed):
    gen = torch.Generator(device='cuda').manual_seed(int(seed))
    dt = DTYPES[case['dtype']]
    st = dict(case)
    if case['op'] == 'norm':
        R, C = case['rows'], case['cols']
        # activations have means and spreads of their own in each channel
        base = _randn((R, C + case['wide']), gen)
        base = base * (0.5 + torch.rand(C + case['wide'], generator=gen, device='cuda')) + 0.3
        x = base.to(dt)[:, :C]
        ln = torch.nn.LayerNorm(C, eps=LN_EPS, device='cuda')       # parameters stay fp32 (mixed precision's master copy)
        with torch.no_grad():
            ln.weight.copy_(_randn((C,), gen, 0.2, 1.0))
            ln.bias.copy_(_randn((C,), gen, 0.1))
        st.update(ln=ln, x=x)
        if case['train']:
            x.requires_grad_(True)
            st['g'] = _randn((R, C), gen, 1.0, 0.0, dt)
    elif case['op'] == 'linear':
        M, K, N = case['rows'], case['k'], case['n']
        lin = torch.nn.Linear(K, N, bias=case['bias'], device='cuda', dtype=dt)
        with torch.no_grad():
            lin.weight.copy_(_randn((N, K), gen, K ** -0.5))
            if case['bias']:
                lin.bias.copy_(_randn((N,), gen, 0.1))
        st.update(lin=lin, x=_randn((M, K), gen, 1.0, 0.0, dt),
                  r=_randn((M, N), gen, 1.0, 0.0, dt) if case['residual'] else None)
        if case['train']:
            st['x'].requires_grad_(True)
            if st['r'] is not None:
                st['r'].requires_grad_(True)
            st['g'] = _randn((M, N), gen, 1.0, 0.0, dt)
    else:
        sizes = _sizes(case['tensors'], case['elements'])
        sigma = 1e-3
        flat = _randn((sum(sizes),), gen, sigma, 0.0, dt)
        views = list(flat.split(sizes))
        expect = sigma * math.sqrt(sum(sizes))
        st['max_norm'] = expect * (0.25 if case['over'] else 4.0)
        if case['out']:
            # gradients as autograd leaves them, each of its own, and one flat buffer that takes the clipped ones
            st['grads'] = [v.clone() for v in views]
            st['flat'] = torch.empty(flat.shape, dtype=DTYPES[case['out']], device='cuda')
            st['outs'] = list(st['flat'].split(sizes))
        else:
            st.update(grads=views, flat=flat, outs=None)            # views of one all-reduce bucket
    return st


# ------------------------------------------------------------------------------------------ the framework's calls
def _own(st):
    from vfdepth_amd import kernels, layers
    if st['op'] == 'clip':
        norm = kernels.clip_grads(st['grads'], st['max_norm'], out=st['outs'])
        return [norm, st['flat']]
    if st['op'] == 'norm':
        call, leaves = (lambda: layers.layer_norm(st['ln'], st['x'])), [st['x'], st['ln'].weight, st['ln'].bias]
    else:
        lin = st['lin']
        call = lambda: layers.linear_act(lin, st['x'], st['act'], st['r'])  # noqa: E731
        leaves = [t for t in (st['x'], lin.weight, lin.bias, st['r']) if t is not None]
    if not st['train']:
        with torch.no_grad():
            return [call()]
    y = call()
    return [y.detach()] + list(torch.autograd.grad(y, leaves, st['g']))


# ------------------------------------------------------------------------------------------ plain forms
def _norm_plain(st):
    x, w, b = st['x'].detach().float(), st['ln'].weight.detach(), st['ln'].bias.detach()
    mean = x.mean(1, keepdim=True)
    xc = x - mean
    rstd = 1 / ((xc * xc).mean(1, keepdim=True) + LN_EPS).sqrt()
    xh = xc * rstd
    y = (xh * w + b).to(st['x'].dtype)
    if not st['train']:
        return [y]
    g = st['g'].float()
    gw = g * w
    dx = rstd * (gw - gw.mean(1, keepdim=True) - xh * (gw * xh).mean(1, keepdim=True))
    return [y, dx.to(y.dtype), (g * xh).sum(0), g.sum(0)]


def _act(z, kind):
    """(value, slope) of an activation."""
    if kind == 'none':
        return z, torch.ones_like(z)
    if kind == 'relu':
        return z * (z > 0), (z > 0).to(z.dtype)
    if kind == 'lrelu':
        s = torch.where(z > 0, torch.ones_like(z), torch.full_like(z, 0.1))
        return z * s, s
    if kind == 'elu':
        e = torch.exp(torch.clamp(z, max=0))
        return torch.where(z > 0, z, torch.expm1(torch.clamp(z, max=0))), e
    if kind == 'gelu':
        cdf = 0.5 * (1 + torch.erf(z * 0.5 ** 0.5))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) * (2 * math.pi) ** -0.5
    s = 1 / (1 + torch.exp(-z))
    return z * s, s * (1 + z * (1 - s))


def _linear_plain(st, wide=torch.float32):
    """In `wide` bits throughout; the outputs are rounded by the caller."""
    lin = st['lin']
    x, w = st['x'].detach().to(wide), lin.weight.detach().to(wide)
    z = x @ w.t()
    if lin.bias is not None:
        z = z + lin.bias.detach().to(wide)
    a, slope = _act(z, st['act'])
    y = a if st['r'] is None else a + st['r'].detach().to(wide)
    if not st['train']:
        return [y]
    g = st['g'].to(wide)
    gz = g * slope
    out = [y, gz @ w, gz.t() @ x]
    if lin.bias is not None:
        out.append(gz.sum(0))
    return out if st['r'] is None else out + [g]


def _clip_plain(st):
    flat = torch.cat([g.reshape(-1) for g in st['grads']]) if st['out'] else st['flat']
    wide = flat.float()
    norm = (wide * wide).sum(dtype=torch.float64).sqrt().float()
    coef = torch.clamp(st['max_norm'] / (norm + 1e-6), max=1.0)
    st['flat'].copy_(wide * coef)
    return [norm, st['flat']]


def run(state):
    if own:
        return _own(state)
    if state['op'] == 'norm':
        return _norm_plain(state)
    if state['op'] == 'linear':
        return [t.to(state['x'].dtype) for t in _linear_plain(state)]
    return _clip_plain(state)


# ------------------------------------------------------------------------------------------ definitions in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    if case['op'] == 'norm':
        x, w, b = st['x'].detach().double(), st['ln'].weight.detach().double(), st['ln'].bias.detach().double()
        var, mean = torch.var_mean(x, dim=1, unbiased=False, keepdim=True)
        inv = torch.rsqrt(var + LN_EPS)
        xh = (x - mean) * inv
        y = w * xh + b
        if not case['train']:
            return [y]
        g = st['g'].double()
        C = x.shape[1]
        # d y_j / d x_i = w_j inv (delta_ij - 1/C - xh_i xh_j / C)
        s1, s2 = (g @ w)[:, None] / C, ((g * xh) @ w)[:, None] / C
        return [y, inv * (w * g - s1 - xh * s2), torch.einsum('rc,rc->c', g, xh), g.sum(0)]
    if case['op'] == 'linear':
        x, w = st['x'].detach().double(), st['lin'].weight.detach().double()
        z = torch.nn.functional.linear(x, w, None if st['lin'].bias is None else st['lin'].bias.detach().double())
        z.requires_grad_(True)
        f = torch.nn.functional
        a = {'none': lambda t: t * 1, 'relu': f.relu, 'lrelu': lambda t: f.leaky_relu(t, 0.1), 'elu': f.elu, 'gelu': f.gelu,
             'silu': f.silu}[case['act']](z)
        y = a.detach() if st['r'] is None else a.detach() + st['r'].detach().double()
        if not case['train']:
            return [y]
        gz, = torch.autograd.grad(a, z, st['g'].double())
        out = [y, gz.mm(w), gz.t().mm(x)] + ([gz.sum(0)] if case['bias'] else [])
        return out + ([st['g'].double()] if case['residual'] else [])
    flat = torch.cat([g.reshape(-1) for g in st['grads']]).double()
    norm = float(torch.linalg.vector_norm(flat))
    return [torch.tensor(norm, dtype=torch.float64), flat * min(1.0, st['max_norm'] / (norm + 1e-6))]


# ------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    size = 4 if case['dtype'] == 'fp32' else 2
    if case['op'] == 'norm':
        R, C = case['rows'], case['cols']
        if not case['train']:
            return {'bytes': 2 * R * C * size + 8 * C, 'flops': 8 * R * C}
        return {'bytes': 4 * R * C * size + 16 * C, 'flops': 24 * R * C}
    if case['op'] == 'linear':
        M, K, N = case['rows'], case['k'], case['n']
        res, bias = int(case['residual']), int(case['bias'])
        fwd = M * K + N * K + bias * N + (1 + res) * M * N
        if not case['train']:
            return {'bytes': size * fwd, 'flops': 2 * M * N * K}
        return {'bytes': size * (fwd + M * N + M * K + N * K + bias * N), 'flops': 6 * M * N * K}
    n = sum(_sizes(case['tensors'], case['elements']))
    out = {'': 0, 'fp32': 4, 'bf16': 2}[case['out']]
    return {'bytes': n * (size + out), 'flops': (3 if case['over'] else 2) * n}
