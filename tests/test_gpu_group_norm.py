"""group_norm_act against its definition in float64, elementwise, at tolerances that follow from the roundings it makes.

u = 2^-24, r the half step of the data's type.  The statistics are fp64 sums, so the mean (two fp32 parts) is off by 2^-48 of
itself and rstd by 2 u of itself.  xhat = (x - mean) rstd takes three roundings: 5 u |xhat|.  z = xhat w + b one more:
ez = 6 u |xhat w| + 2 u |b|.  The activations' slopes are at most 1.1, their exponentials are good to (|z| + 4) u (one rounded
product in the exponent, 1 ulp, expm1's polynomial 4 u).  dz = dy act'(z); act' moves by at most 1 per unit of z (elu, silu).
Sums over a thread's pixels are fp32: at most P u of the sum of sizes; threads and samples meet in fp64.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}
# N, pixels, C, groups: which of the kernels' ways they take in fp32 (a sample in one workgroup, or in pieces)
CASES = {
    'tiny': (1, (), 4, 1),
    'one_value': (3, (), 7, 7),
    'odd_channels': (3, (5,), 33, 11),
    'even_channels': (2, (9, 9), 36, 6),
    'wave': (70, (2, 2), 64, 8),
    'small': (5, (4, 4), 64, 8),
    'middle': (4, (14, 14), 64, 8),
    'large_resident': (2, (28, 28), 64, 4),
    'split_groups': (2, (40, 40), 320, 32),
    'wide_resident': (2, (3, 3), 2400, 5),
    'wide_pieces': (1, (70,), 2400, 3),
    'many_samples': (1100, (1,), 16, 4),
    'long': (1, (150, 150), 8, 2),
    'one_group': (2, (33, 31), 96, 1),
}


def make(device, N, pix, C, dtype, seed=0, offset=0.0, wdtype=None):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(N, *pix, C, generator=g) * (0.5 + torch.rand(C, generator=g)) + torch.randn(C, generator=g) + offset
    dy = torch.randn(N, *pix, C, generator=g)
    w, b = 1 + 0.3 * torch.randn(C, generator=g), 0.3 * torch.randn(C, generator=g)
    wt = wdtype or torch.float32
    return x.to(device, TYPES[dtype]), w.to(device, wt), b.to(device, wt), dy.to(device, TYPES[dtype])


def reference(x, w, b, dy, G, eps, act):
    """(y, dx, dw, db), their tolerances, and the smallest |z| / its tolerance (relu is only comparable away from 0)."""
    u, r = 2.0 ** -24, torch.finfo(x.dtype).eps / 2
    N, C = x.shape[0], x.shape[-1]
    X, D = x.double().reshape(N, -1, G, C // G), dy.double().reshape(N, -1, G, C // G)
    P = X.shape[1]
    W = (torch.ones(C) if w is None else w).double().to(x.device).view(G, C // G)
    B = (torch.zeros(C) if b is None else b).double().to(x.device).view(G, C // G)
    mean = X.mean((1, 3), keepdim=True)
    rs = 1 / (((X - mean) ** 2).mean((1, 3), keepdim=True) + eps).sqrt()
    xh = (X - mean) * rs
    exh = 5 * u * xh.abs() + 2.0 ** -46 * mean.abs() * rs
    z = xh * W + B
    ez = exh * W.abs() + 2 * u * z.abs() + 2 * u * B.abs()
    s = torch.sigmoid(z)
    y, sl = {None: (z, torch.ones_like(z)), 'relu': (z.clamp_min(0), (z > 0).double()),
             'elu': (torch.where(z > 0, z, torch.expm1(z)), torch.where(z > 0, 1.0, torch.exp(z))),
             'silu': (z * s, s * (1 + z * (1 - s)))}[act]
    ty = 1.1 * ez + (2 * z.abs() + 12) * u * y.abs() + r * (y.abs() + 1.1 * ez) + u * 1e-6
    esl = 0 if act in (None, 'relu') else ez + (2 * z.abs() + 16) * u * 1.1
    dz = D * sl
    edz = D.abs() * esl + u * dz.abs()
    S1, S2 = dz.sum(1, keepdim=True), (dz * xh).sum(1, keepdim=True)
    e1 = edz.sum(1, keepdim=True) + (P + 2) * u * dz.abs().sum(1, keepdim=True)
    e2 = (edz * xh.abs() + dz.abs() * exh).sum(1, keepdim=True) + (P + 3) * u * (dz * xh).abs().sum(1, keepdim=True)
    M = P * (C // G)
    m1, m2 = ((W * t).sum(3, keepdim=True) / M for t in (S1, S2))
    f1, f2 = ((W.abs() * t).sum(3, keepdim=True) / M for t in (e1, e2))
    f1, f2 = f1 + 2 * u * m1.abs(), f2 + 2 * u * m2.abs()
    dx = rs * (dz * W - m1 - xh * m2)
    tx = rs * (edz * W.abs() + f1 + xh.abs() * f2 + exh * m2.abs() + 6 * u * ((dz * W).abs() + m1.abs() + (xh * m2).abs()))
    tx = tx * (1 + r) + r * dx.abs()
    ref = w if w is not None else b                          # the parameters' gradients are rounded to their type
    wr = torch.finfo(ref.dtype).eps / 2 if ref is not None else u
    dw, db = S2.sum(0).view(C), S1.sum(0).view(C)
    tw, tb = e2.sum(0).view(C) + wr * dw.abs() + 1e-30, e1.sum(0).view(C) + wr * db.abs() + 1e-30
    tiny = 2.0 ** -24 if x.dtype == torch.float16 else 1e-37
    shape = x.shape
    return [y.reshape(shape), dx.reshape(shape), dw, db], [ty.reshape(shape) + tiny, tx.reshape(shape) + tiny, tw + tiny, tb + tiny], \
        float((z.abs() / ez.clamp_min(1e-300)).min())


def run(x, w, b, dy, G, **kw):
    from cmvae_amd.norm import group_norm_act
    leaves = [t.detach().requires_grad_() for t in (x, w, b) if t is not None]
    it = iter(leaves)
    x, w, b = (None if t is None else next(it) for t in (x, w, b))
    y = group_norm_act(x, G, w, b, **kw)
    return [y.detach(), *torch.autograd.grad(y, leaves, dy)]


def compare(got, want, tol):
    for name, a, b, t in zip(('y', 'dx', 'dw', 'db'), got, want, tol):
        assert a.shape == b.shape and torch.isfinite(a).all(), name
        off = (a.double() - b).abs() - t
        assert float(off.max()) <= 0, '%s: %.3g over its tolerance' % (name, float(off.max()))


@pytest.mark.parametrize('act', [None, 'elu', 'silu', 'relu'])
@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('case', CASES)
def test_against_float64(device, case, dtype, act):
    N, pix, C, G = CASES[case]
    x, w, b, dy = make(device, N, pix, C, dtype)
    if act == 'relu':
        # relu's slope steps at 0, where a rounding decides: its inputs are kept a tolerance away by their bias
        b = b.sign() * (b.abs() + 0.01) if case == 'one_value' else b
        z0 = reference(x, w, b, dy, G, 1e-5, act)[2]
        if z0 <= 1:
            b = b + 1e-3
            z0 = reference(x, w, b, dy, G, 1e-5, act)[2]
        assert z0 > 1
    want, tol, _ = reference(x, w, b, dy, G, 1e-5, act)
    compare(run(x, w, b, dy, G, act=act), want, tol)


@pytest.mark.parametrize('case', ['middle', 'long'])
def test_mean_far_from_zero(device, case):
    """A mean 10^4 deviations from zero: the sums of squares keep the variance, the two-part mean the differences."""
    N, pix, C, G = CASES[case]
    x, w, b, dy = make(device, N, pix, C, 'f32', offset=1e4)
    want, tol, _ = reference(x, w, b, dy, G, 1e-5, 'silu')
    compare(run(x, w, b, dy, G, act='silu'), want, tol)


@pytest.mark.parametrize('case', ['middle', 'split_groups'])
def test_parameters_of_the_datas_type_and_none(device, case):
    N, pix, C, G = CASES[case]
    x, w, b, dy = make(device, N, pix, C, 'bf16', wdtype=torch.bfloat16)
    want, tol, _ = reference(x, w, b, dy, G, 1e-5, 'elu')
    got = run(x, w, b, dy, G, act='elu')
    assert got[2].dtype == got[3].dtype == torch.bfloat16
    compare(got, want, tol)
    want, tol, _ = reference(x, None, None, dy, G, 1e-3, None)
    compare(run(x, None, None, dy, G, eps=1e-3), want[:2], tol[:2])
    want, tol, _ = reference(x, None, b, dy, G, 1e-5, None)
    got = run(x, None, b, dy, G)
    compare(got[:2] + [want[2]] + got[2:], want, tol)


@pytest.mark.parametrize('case', ['wave', 'middle', 'large_resident', 'split_groups'])
def test_every_run_gives_the_same_bits_and_the_forward_alone(device, case):
    from cmvae_amd.norm import group_norm_act
    N, pix, C, G = CASES[case]
    x, w, b, dy = make(device, N, pix, C, 'f32')
    a, c = run(x, w, b, dy, G, act='elu'), run(x, w, b, dy, G, act='elu')
    assert all(torch.equal(s, t) for s, t in zip(a, c))
    with torch.no_grad():
        assert torch.equal(group_norm_act(x, G, w, b, act='elu'), a[0])


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
def test_strided_views(device, dtype):
    """A column slice of wider rows, one pixel per sample out of several, a misaligned tensor, a transposed one, an expanded
    gradient."""
    wide = make(device, 6, (30,), 128, dtype)[0]
    x, (_, w, b, _) = wide[:, :, 64:], make(device, 6, (30,), 64, dtype, seed=1)
    dy = torch.ones(64, device=device, dtype=x.dtype).mul_(torch.arange(64, device=device)).expand(6, 30, 64)
    want = run(x.contiguous(), w, b, dy.contiguous(), 8, act='silu')
    assert all(torch.equal(s, t) for s, t in zip(want, run(x, w, b, dy, 8, act='silu')))
    odd = wide[:, :, 3:67]                                       # rows that no vector load fits
    a, c = run(odd.contiguous(), w, b, dy, 8), run(odd, w, b, dy, 8)
    ref, tol, _ = reference(odd, w, b, dy, 8, 1e-5, None)
    compare(a, ref, tol)
    compare(c, ref, tol)
    nchw = x.transpose(1, 2).contiguous().transpose(1, 2)        # channels not adjacent: copied
    assert all(torch.equal(s, t) for s, t in zip(want, run(nchw, w, b, dy, 8, act='silu')))


def test_a_sample_that_is_not_finite_stays_alone(device):
    for case in ('middle', 'split_groups'):
        N, pix, C, G = CASES[case]
        x, w, b, dy = make(device, N, pix, C, 'f32')
        clean = run(x, w, b, dy, G, act='elu')
        x[1].view(-1)[5] = float('nan')
        got = run(x, w, b, dy, G, act='elu')
        assert torch.equal(got[0][0], clean[0][0]) and torch.equal(got[1][0], clean[1][0])
        assert torch.isnan(got[0][1]).any()


def test_empty(device):
    from cmvae_amd.norm import group_norm_act
    for shape in ((0, 4, 8), (3, 0, 8)):
        x = torch.zeros(shape, device=device, requires_grad=True)
        w = torch.ones(8, device=device, requires_grad=True)
        y = group_norm_act(x, 2, w, w)
        gx, gw = torch.autograd.grad(y.sum(), (x, w))
        assert y.shape == shape and gx.shape == shape and not gw.any()


def test_gradients_against_differences(device):
    """(f(x + t d) - f(x - t d)) / 2t for f = <y, dy>: t = 2^-6 leaves a third derivative's t^2 / 6 and y's roundings over 2t,
    both under 1 % of the gradient's norm."""
    from cmvae_amd.norm import group_norm_act
    x, w, b, dy = make(device, 3, (6, 6), 32, 'f32')
    grads = run(x, w, b, dy, 4, act='silu')[1:]
    g = torch.Generator().manual_seed(4)
    t = 2.0 ** -6
    for i in range(3):
        d = torch.randn(grads[i].shape, generator=g).to(device)
        f = []
        for s in (t, -t):
            a = [x, w, b]
            a[i] = a[i] + s * d
            f.append(float((group_norm_act(a[0], 4, a[1], a[2], act='silu').double() * dy.double()).sum()))
        want = float((grads[i].double() * d.double()).sum())
        assert abs((f[0] - f[1]) / (2 * t) - want) <= 0.01 * float(grads[i].double().norm())


@pytest.mark.parametrize('case', ['middle', 'split_groups'])
def test_graph_replays_and_other_stream(device, case):
    N, pix, C, G = CASES[case]
    x, w, b, dy = make(device, N, pix, C, 'bf16')
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(x, w, b, dy, G, act='elu')
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(s, t) for s, t in zip(got, run(x, w, b, dy, G, act='elu')))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(x, w, b, dy, G, act='elu')
    for seed in (3, 4, 5):
        for t, n in zip((x, w, b, dy), make(device, N, pix, C, 'bf16', seed=seed)):
            t.copy_(n)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(s, t) for s, t in zip(out, run(x, w, b, dy, G, act='elu')))


def test_refusals(device):
    from cmvae_amd.norm import group_norm_act
    x, w, b, _ = make(device, 2, (3,), 8, 'bf16')
    for args, kw in [((x, 3), {}), ((x, 0), {}), ((x, 2.0), {}), ((x.double(), 2), {}), ((x[0, 0], 2), {}), ((x, 2, w[:4]), {}),
                     ((x, 2, w.half(), b.half()), {}), ((x, 2, w.cpu()), {}), ((x, 2, w, b.bfloat16()), {}),
                     ((x, 2), dict(act='gelu')), ((x, 2), dict(eps=-1.0)), ((x, 2), dict(eps=float('nan'))), ((x.cpu(), 2), {}),
                     ((x[:, :, :0], 1), {})]:
        with pytest.raises(RuntimeError, match='group_norm_act'):
            group_norm_act(*args, **kw)


@pytest.mark.parametrize('P', [40, 300])
def test_offsets_beyond_32_bits(device, P):
    """Pixels 2^23 elements apart: the 257th lies past 2^31 elements.  With 40 of them it is the second sample that does."""
    apart, sample = 2 ** 23, 2 ** 31 if P == 40 else 64
    x, w, b, dy = make(device, 2, (P,), 64, 'bf16')
    buf = torch.empty(sample + P * apart, dtype=torch.bfloat16, device=device)
    far = buf.as_strided((2, P, 64), (sample, apart, 1))
    far.copy_(x)
    want = run(x, w, b, dy, 8, act='silu')
    assert all(torch.equal(s, t) for s, t in zip(want, run(far, w, b, dy, 8, act='silu')))


def test_two_calls_at_once(device):
    """Calls in flight on two streams use workspaces of their own."""
    sets = [make(device, 2, (40, 40), 320, 'f32', seed=s) for s in (1, 2)]
    want = [run(*s, 32, act='elu') for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        got = []
        for st, s in zip(streams, sets):
            with torch.cuda.stream(st):
                got.append(run(*s, 32, act='elu'))
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for a, b in zip(want, got) for x, y in zip(a, b))


# rows of which only pairs are aligned, channel pieces of unequal width, groups across thread and piece borders
MORE = {
    'pairs': (3, (5, 5), 34, 17),
    'pairs_in_pieces': (1, (60, 60), 66, 3),
    'uneven_pieces': (1, (40, 41), 1284, 12),
    'narrow_pieces': (2, (90, 90), 6, 1),
    'many_groups': (2, (3, 5), 1152, 576),
    'more_groups_than_threads': (1, (2, 1), 1536, 1536),
}


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('case', MORE)
def test_more_shapes_against_float64(device, case, dtype):
    N, pix, C, G = MORE[case]
    x, w, b, dy = make(device, N, pix, C, dtype, seed=6)
    want, tol, _ = reference(x, w, b, dy, G, 1e-5, 'silu')
    compare(run(x, w, b, dy, G, act='silu'), want, tol)


@pytest.mark.parametrize('value', [1000.1, 100000.1, 1234567.1])
@pytest.mark.parametrize('case', ['wave', 'middle', 'large_resident', 'odd_channels', 'split_groups', 'long'])
def test_groups_of_one_value_far_from_zero(device, case, value):
    """A group that holds one value has no variance, however large the value: rstd is that of eps.  So it is beside a
    sample whose values lie one apart around it."""
    N, pix, C, G = CASES[case]
    x, w, b, dy = make(device, N, pix, C, 'f32', seed=2)
    x = x.round() + value
    x[0] = value
    want, tol, _ = reference(x, w, b, dy, G, 1e-5, 'silu')
    compare(run(x, w, b, dy, G, act='silu'), want, tol)


@pytest.mark.parametrize('dtype', ['bf16', 'f16'])
def test_groups_of_one_value_in_16_bits(device, dtype):
    for case in ('middle', 'split_groups'):
        N, pix, C, G = CASES[case]
        x, w, b, dy = make(device, N, pix, C, dtype)
        x[0] = 50000.0
        want, tol, _ = reference(x, w, b, dy, G, 1e-5, None)
        compare(run(x, w, b, dy, G), want, tol)
