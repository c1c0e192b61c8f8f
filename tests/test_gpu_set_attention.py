"""set_attention against its definition in float64, elementwise, at tolerances that follow from the roundings it makes.

With u = 2^-24, r the half step of the element type, A_ij = scale sum_c |q_ic k_jc| >= |s_ij|:
  * a score is a D-term fp32 sum, scaled by a rounded constant, subtracted from a maximum / log-sum-exp of at most
    A + log(Sk) and put through a 1-ulp exponential: relative error of p_ij at most e = u ((D + 6) max A + log(Sk) + 8);
    normalisation doubles it and adds the Sk-term sum of the row;
  * 16-bit types round p (and dS) once more as factors, and o when it is saved for delta;
  * the exponential gives 0 under 2^-126, and what is under a type's smallest normal may be rounded as that: an error of
    up to z = 2^-126 (dS in fp16: 2^-25, half its smallest step; p in fp16 is held times 2^15: 2^-40) per factor, absolute,
    which a sum takes times the other factor;
  * every product sum over n terms adds n u of the sum of absolute terms; results are rounded once.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}


def make(device, B, Sq, Sk, H, Hkv, D, dtype, seed=0, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    mk = lambda *s: (torch.randn(*s, generator=g) * spread).to(device=device, dtype=TYPES[dtype])  # noqa: E731
    return mk(B, Sq, H, D), mk(B, Sk, Hkv, D), mk(B, Sk, Hkv, D), mk(B, Sq, H, D)


def reference(q, k, v, do, scale, causal, ql, kl, residual):
    """(o, dq, dk, dv) and their elementwise tolerances, all float64."""
    B, Sq, H, D = q.shape
    Sk, Hkv = k.shape[1:3]
    u, r = 2.0 ** -24, torch.finfo(q.dtype).eps / 2
    f = r if q.dtype != torch.float32 else 0.0              # rounding of p and dS to factors
    zp, zd = (2.0 ** -40, 2.0 ** -25) if q.dtype == torch.float16 else (2.0 ** -126, 2.0 ** -126)
    z = lambda *s: torch.zeros(*s, dtype=torch.float64, device=q.device)  # noqa: E731
    out = [z(B, Sq, H, D), z(B, Sq, H, D), z(B, Sk, Hkv, D), z(B, Sk, Hkv, D)]
    tol = [t.clone() for t in out]
    for b in range(B):
        nq, nk = (Sq if ql is None else ql[b]), (Sk if kl is None else kl[b])
        if nq == 0:
            continue
        for h in range(H):
            g = h // (H // Hkv)
            Q, G = q[b, :nq, h].double(), do[b, :nq, h].double()
            K, V = k[b, :nk, g].double(), v[b, :nk, g].double()
            s = scale * Q @ K.T
            ok = torch.ones_like(s, dtype=torch.bool)
            if causal:
                i, j = torch.arange(nq, device=q.device)[:, None], torch.arange(nk, device=q.device)[None]
                ok = j <= i + nk - nq
            s = s.masked_fill(~ok, -math.inf)
            if nk:
                p = torch.exp(s - s.amax(1, keepdim=True).clamp_min(-1e300))
                p = p / p.sum(1, keepdim=True).clamp_min(1e-300)
                A = float((scale * Q.abs() @ K.abs().T).max())
            else:
                p, A = s, 0.0
            e = u * ((D + 6) * A + math.log(max(nk, 1)) + 8)
            ep = 2 * e + (nk + 4) * u                        # relative, of a normalised probability
            o = p @ V
            ov = p @ V.abs()
            to = (ep + f + (nk + 4) * u) * ov + zp * V.abs().sum(0)
            out[0][b, :nq, h] = o + (Q if residual else 0)
            tol[0][b, :nq, h] = to + (r + 2 * u) * (o + (Q if residual else 0)).abs() + r * to
            dp, adp = G @ V.T, G.abs() @ V.abs().T
            delta = (G * o).sum(1, keepdim=True)
            e_dl = (G.abs() * (to + (r + D * u) * o.abs())).sum(1, keepdim=True)
            ds = p * (dp - delta)
            e_ds = (p * ((D + 2) * u * adp + e_dl) + (ep + f + 4 * u) * ds.abs() + p * ep * (D * u * adp + e_dl)) * ok \
                + zd + 2.0 ** -126 * (adp + delta.abs())
            ds = ds * ok
            p = p * ok
            dq = scale * ds @ K
            tq = scale * (e_ds + (nk + 4) * u * ds.abs()) @ K.abs()
            out[1][b, :nq, h] = dq + (G if residual else 0)
            tol[1][b, :nq, h] = tq + (r + 3 * u) * (dq + (G if residual else 0)).abs() + r * tq + u * dq.abs()
            n = nq * (H // Hkv)
            out[2][b, :nk, g] += scale * ds.T @ Q
            tol[2][b, :nk, g] += scale * (e_ds + (n + 6) * u * ds.abs()).T @ Q.abs()
            out[3][b, :nk, g] += p.T @ G
            tol[3][b, :nk, g] += ((ep + f + (n + 6) * u) * p + zp).T @ G.abs()
    for i in (2, 3):
        tol[i] = tol[i] * (1 + r) + (r + 3 * u) * out[i].abs()
    tiny = float(torch.finfo(q.dtype).smallest_normal) * (1 if q.dtype != torch.float16 else 2.0 ** -10)
    return out, [t + tiny for t in tol]


def run(q, k, v, do, **kw):
    from cmvae_amd.attention import set_attention
    q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
    o = set_attention(q, k, v, **kw)
    return [o.detach(), *torch.autograd.grad(o, (q, k, v), do)]


def lens(x, device):
    return None if x is None else torch.tensor(x, dtype=torch.int32, device=device)


def compare(got, want, tol):
    for name, a, b, t in zip(('o', 'dq', 'dk', 'dv'), got, want, tol):
        assert torch.isfinite(a).all(), name
        off = (a.double() - b).abs() - t
        assert float(off.max()) <= 0, '%s: %.3g over its tolerance' % (name, float(off.max()))


# B, Sq, Sk, H, Hkv, D, causal, q_len, k_len, residual
CASES = {
    'one_one': (1, 1, 1, 1, 1, 64, False, None, None, False),
    'one_one_128': (1, 1, 1, 2, 1, 128, True, None, None, True),
    'one_query': (2, 1, 700, 4, 2, 64, False, None, [700, 333], False),
    'one_query_causal': (3, 1, 1300, 8, 2, 128, True, None, [1300, 1, 0], False),
    'one_key': (2, 70, 1, 2, 2, 64, False, None, None, True),
    'odd': (1, 33, 65, 2, 1, 128, True, None, None, False),
    'block': (2, 200, 200, 4, 4, 64, False, None, None, True),
    'padded': (4, 77, 301, 6, 2, 64, False, [77, 0, 5, 64], [301, 100, 0, 33], True),
    'padded_causal': (3, 150, 150, 4, 1, 64, True, [150, 1, 97], [150, 1, 97], False),
    'more_rows_than_keys': (2, 130, 97, 2, 2, 64, True, None, [97, 31], True),
    'causal_lens': (2, 260, 520, 4, 2, 128, True, [260, 130], [520, 131], False),
    'wide_grid': (16, 40, 70, 16, 16, 64, False, None, None, False),
    'wide_grid_128': (16, 40, 70, 16, 16, 128, True, None, [70, 64, 63, 65] * 4, True),
    'four_waves_shared': (4, 300, 500, 32, 16, 64, True, [300, 299, 128, 17], [500, 499, 128, 64], False),
    'few_keys': (1, 2000, 40, 2, 1, 64, False, None, None, False),
    'long': (1, 1100, 2100, 2, 1, 64, True, None, None, False),
}


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('case', CASES)
def test_against_float64(device, case, dtype):
    B, Sq, Sk, H, Hkv, D, causal, ql, kl, residual = CASES[case]
    q, k, v, do = make(device, B, Sq, Sk, H, Hkv, D, dtype)
    got = run(q, k, v, do, causal=causal, q_len=lens(ql, device), k_len=lens(kl, device), residual=residual)
    want, tol = reference(q, k, v, do, 1 / math.sqrt(D), causal, ql, kl, residual)
    compare(got, want, tol)
    for b in range(B):
        if ql is not None:
            assert not got[0][b, ql[b]:].any() and not got[1][b, ql[b]:].any()
        if kl is not None:
            assert not got[2][b, kl[b]:].any() and not got[3][b, kl[b]:].any()


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
def test_peaked_rows(device, dtype):
    """Scores in the hundreds: one key takes almost all of each row, the running maximum moves from tile to tile."""
    q, k, v, do = make(device, 2, 90, 400, 2, 1, 64, dtype, seed=3, spread=3.0)
    got = run(q, k, v, do, scale=1.0, causal=True)
    want, tol = reference(q, k, v, do, 1.0, True, None, None, False)
    compare(got, want, tol)


def test_forward_without_gradients_is_the_same(device):
    from cmvae_amd.attention import set_attention
    q, k, v, do = make(device, 2, 77, 300, 4, 2, 64, 'bf16')
    with torch.no_grad():
        o = set_attention(q, k, v, residual=True)
    assert torch.equal(o, run(q, k, v, do, residual=True)[0])


@pytest.mark.parametrize('case', ['one_query', 'padded', 'causal_lens', 'four_waves_shared', 'few_keys'])
def test_every_run_gives_the_same_bits(device, case):
    B, Sq, Sk, H, Hkv, D, causal, ql, kl, residual = CASES[case]
    q, k, v, do = make(device, B, Sq, Sk, H, Hkv, D, 'f32')
    kw = dict(causal=causal, q_len=lens(ql, device), k_len=lens(kl, device), residual=residual)
    a, b = run(q, k, v, do, **kw), run(q, k, v, do, **kw)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
def test_rows_behind_a_length_are_not_read(device, dtype):
    B, Sq, Sk, H, Hkv, D, causal, ql, kl, residual = CASES['padded']
    q, k, v, do = make(device, B, Sq, Sk, H, Hkv, D, dtype)
    kw = dict(causal=True, q_len=lens(ql, device), k_len=lens(kl, device), residual=residual)
    clean = run(q, k, v, do, **kw)
    for b in range(B):
        q[b, ql[b]:], do[b, ql[b]:] = math.nan, math.inf
        k[b, kl[b]:], v[b, kl[b]:] = math.inf, math.nan
    assert all(torch.equal(x, y) for x, y in zip(clean, run(q, k, v, do, **kw)))


def test_lengths_outside_the_tensor_are_clamped(device):
    q, k, v, do = make(device, 2, 20, 50, 2, 2, 64, 'f32')
    a = run(q, k, v, do, q_len=lens([20, 0], device), k_len=lens([50, 0], device))
    b = run(q, k, v, do, q_len=lens([10 ** 6, -3], device), k_len=lens([2 ** 31 - 1, -1], device))
    assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
def test_strided_views(device, dtype):
    """q, k, v as slices of one packed projection, as head-major views, as a misaligned and as an expanded tensor; dO
    expanded."""
    B, S, H, D = 2, 70, 4, 64
    g = torch.Generator().manual_seed(1)
    packed = torch.randn(B, S, 3, H, D, generator=g).to(device=device, dtype=TYPES[dtype])
    q, k, v = packed.unbind(2)
    do = torch.randn(D, generator=g).to(device=device, dtype=TYPES[dtype]).expand(B, S, H, D)
    want = run(q.contiguous(), k.contiguous(), v.contiguous(), do.contiguous(), causal=True)
    assert all(torch.equal(x, y) for x, y in zip(want, run(q, k, v, do, causal=True)))
    hm = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
    assert all(torch.equal(x, y) for x, y in zip(want, run(*hm, do, causal=True)))
    buf = torch.empty(q.numel() + 1, device=device, dtype=q.dtype)
    off = buf[1:].view(q.shape).copy_(q)
    assert all(torch.equal(x, y) for x, y in zip(want, run(off, k, v, do, causal=True)))
    from cmvae_amd.attention import set_attention
    one = k[:1].detach().clone().requires_grad_()
    o = set_attention(q, one.expand(B, S, H, D), v)
    (gk,) = torch.autograd.grad(o, one, do)
    full = run(q, one.detach().expand(B, S, H, D).contiguous(), v, do)[2]
    assert torch.equal(gk, full.sum(0, keepdim=True))


def test_empty_batches_and_sets(device):
    from cmvae_amd.attention import set_attention
    for B, Sq, Sk in ((0, 3, 3), (2, 0, 3), (2, 3, 0)):
        q, k, v, do = make(device, B, Sq, Sk, 2, 2, 64, 'f32')
        o, dq, dk, dv = run(q, k, v, do, residual=True)
        assert o.shape == q.shape and torch.equal(o, q) and torch.equal(dq, do)
        assert dk.shape == k.shape and not dk.any() and not dv.any()
        assert not set_attention(q, k, v).any()


def test_gradients_against_differences(device):
    """f(x) = <o(x), do>: (f(x + t d) - f(x - t d)) / 2t along random directions.  t = 2^-6 leaves t^2 / 6 of a third
    derivative of the gradient's own size, and sqrt(n) roundings of o (2^-22 of a row's |v|) over 2t: 1 % covers both."""
    from cmvae_amd.attention import set_attention
    q, k, v, do = make(device, 2, 40, 72, 4, 2, 64, 'f32', seed=9)
    kw = dict(causal=True, q_len=lens([40, 21], device), k_len=lens([72, 50], device), residual=True)
    grads = run(q, k, v, do, **kw)[1:]
    g = torch.Generator().manual_seed(2)
    t = 2.0 ** -6
    for i in range(3):
        d = torch.randn(grads[i].shape, generator=g).to(device)
        f = []
        for s in (t, -t):
            x = [q, k, v]
            x[i] = x[i] + s * d
            f.append(float((set_attention(*x, **kw).double() * do.double()).sum()))
        want = float((grads[i].double() * d.double()).sum())
        assert abs((f[0] - f[1]) / (2 * t) - want) <= 0.01 * float(grads[i].double().norm())


def test_on_another_stream_and_in_a_graph(device):
    """The call runs on the current stream; captured with its backward pass it replays on new inputs."""
    q, k, v, do = make(device, 2, 65, 900, 4, 2, 64, 'bf16')
    kl = lens([900, 451], device)
    want = run(q, k, v, do, k_len=kl)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(q, k, v, do, k_len=kl)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for x, y in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(q, k, v, do, k_len=kl)
    for seed in (5, 6, 7):
        for t, n in zip((q, k, v, do), make(device, 2, 65, 900, 4, 2, 64, 'bf16', seed=seed)):
            t.copy_(n)
        kl.copy_(lens([900 - seed, 451 + seed], device))
        graph.replay()
        torch.cuda.synchronize()
        want = run(q, k, v, do, k_len=kl)
        assert all(torch.equal(x, y) for x, y in zip(want, out))


def test_refusals(device):
    from cmvae_amd.attention import set_attention
    q, k, v, _ = make(device, 2, 8, 9, 4, 2, 64, 'f32')
    one = torch.ones(2, dtype=torch.int32, device=device)
    bad = [((q, k, v[:, :8]), {}), ((q, k[:1], v[:1]), {}), ((q[..., :32], k[..., :32], v[..., :32]), {}),
           ((q, k.bfloat16(), v.bfloat16()), {}), ((q.double(), k.double(), v.double()), {}), ((q[:, :, :3], k, v), {}),
           ((q[0], k[0], v[0]), {}), ((q, k.cpu(), v), {}), ((q, k, v), dict(scale=0.0)), ((q, k, v), dict(scale=-1.0)),
           ((q, k, v), dict(scale=math.nan)), ((q, k, v), dict(q_len=one.long())), ((q, k, v), dict(k_len=one[:1])),
           ((q, k, v), dict(k_len=one.cpu())), ((q, k, v), dict(q_len=[8, 8])), ((q[:, :, :0], k, v), {}),
           ((q, k[:, :, :0], v[:, :, :0]), {})]
    for args, kw in bad:
        with pytest.raises(RuntimeError, match='set_attention'):
            set_attention(*args, **kw)


# more entries than one lane each, lists of 3, 6, 8 and 16 rows, tiles that span several short heads, pieces of long walks
MORE = {
    'seventy_entries': (70, 37, 90, 2, 1, 64, True, [37 - b % 38 for b in range(70)], [90 - (7 * b) % 91 for b in range(70)], True),
    'seventy_entries_wide': (70, 140, 66, 8, 8, 64, False, None, [66 - b % 67 for b in range(70)], False),
    'three_rows': (2, 1, 2500, 6, 2, 64, False, None, [2500, 7], True),
    'six_rows': (3, 3, 777, 4, 2, 128, True, [3, 2, 0], [777, 1, 500], False),
    'eight_rows': (2, 4, 1500, 4, 2, 64, True, None, [1500, 3], True),
    'sixteen_rows': (2, 1, 5000, 32, 2, 128, True, None, [5000, 1234], False),
    'short_heads': (2, 5, 300, 16, 2, 64, True, [5, 3], [300, 4], False),
    'odd_group': (2, 75, 210, 9, 3, 128, True, [75, 31], [210, 31], True),
    'all_masked': (2, 30, 40, 2, 2, 64, True, [0, 30], [40, 0], False),
}


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('case', MORE)
def test_more_shapes_against_float64(device, case, dtype):
    B, Sq, Sk, H, Hkv, D, causal, ql, kl, residual = MORE[case]
    q, k, v, do = make(device, B, Sq, Sk, H, Hkv, D, dtype, seed=4)
    got = run(q, k, v, do, causal=causal, q_len=lens(ql, device), k_len=lens(kl, device), residual=residual)
    want, tol = reference(q, k, v, do, 1 / math.sqrt(D), causal, ql, kl, residual)
    compare(got, want, tol)


@pytest.mark.parametrize('Sq', [1, 530])
def test_offsets_beyond_32_bits(device, Sq):
    """Rows just under 2^22 elements apart: 2^31 elements are passed by the 513th, 2^32 bytes too."""
    H, Hkv, D, Sk, apart = 2, 1, 64, 530, 2 ** 22 - 8
    q, k, v, do = make(device, 1, Sq, Sk, H, Hkv, D, 'bf16')
    buf = torch.empty(Sk * apart, dtype=torch.bfloat16, device=device)
    far, at = [], 0
    for t in (q, k, v, do):
        S, h = t.shape[1:3]
        far.append(buf.as_strided((1, S, h, D), (8, apart, D, 1), at).copy_(t))
        at += h * D
    want = run(q, k, v, do, causal=True)
    assert all(torch.equal(x, y) for x, y in zip(want, run(*far, causal=True)))


def test_two_calls_at_once(device):
    """Calls in flight on two streams use workspaces of their own."""
    sets = [make(device, 4, 96, 3000, 4, 2, 64, 'f32', seed=s) for s in (1, 2)]
    want = [run(*s) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        got = []
        for st, s in zip(streams, sets):
            with torch.cuda.stream(st):
                got.append(run(*s))
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for a, b in zip(want, got) for x, y in zip(a, b))


# walks in pieces under both kinds of workgroup, whole walks where four tiles of rows fill the card
PIECES = {
    'four_tiles_in_pieces': (1, 300, 2600, 4, 2, 64, False, None, None, True),
    'four_tiles_in_pieces_causal': (1, 1500, 1500, 2, 1, 128, True, None, None, False),
    'one_tile_in_pieces': (1, 30, 4100, 4, 4, 64, False, None, [4001], False),
    'whole': (9, 500, 330, 8, 8, 64, False, None, None, False),
    'whole_128': (6, 290, 700, 15, 15, 128, True, None, None, True),
}


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('case', PIECES)
def test_pieces_against_float64(device, case, dtype):
    B, Sq, Sk, H, Hkv, D, causal, ql, kl, residual = PIECES[case]
    q, k, v, do = make(device, B, Sq, Sk, H, Hkv, D, dtype, seed=8)
    kw = dict(causal=causal, q_len=lens(ql, device), k_len=lens(kl, device), residual=residual)
    got = run(q, k, v, do, **kw)
    want, tol = reference(q, k, v, do, 1 / math.sqrt(D), causal, ql, kl, residual)
    compare(got, want, tol)
    assert all(torch.equal(x, y) for x, y in zip(got, run(q, k, v, do, **kw)))


# walks shared out by waves, of four tiles, in pieces; short and long, so that p and dS are small
SMALL_DS = {
    'few_rows': (1, 33, 8000, 2, 1, 64, False, None, None),
    'one_query': (2, 1, 5000, 4, 2, 128, True, None, [5000, 777]),
    'long_causal': (1, 1500, 1500, 4, 2, 128, True, None, None),
    'padded': (4, 500, 2049, 8, 2, 64, False, [500, 129, 1, 0], [2049, 513, 2000, 64]),
    'whole': (9, 500, 330, 8, 8, 64, False, None, None),
    'few_keys': (1, 3000, 40, 2, 1, 64, False, None, None),
}


def eighths(do, seed):
    """Multiples of 1/8 in [-4, 4], none of them 0: exact in fp16 down to 2^-21 times themselves."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randint(1, 33, do.shape, generator=g) * (1 - 2 * torch.randint(0, 2, do.shape, generator=g))
    return (x / 8).to(do)


@pytest.mark.parametrize('power', [-14, -8, 8])
@pytest.mark.parametrize('case', SMALL_DS)
def test_fp16_gradients_are_as_exact_for_small_and_large_do(device, case, power):
    """The gradients are linear in dO and every step but the results' rounding is the same for dO and 2^power dO, so they are
    2^power times each other to those roundings: half a step of each result, 2^-11 of it or 2^-25."""
    B, Sq, Sk, H, Hkv, D, causal, ql, kl = SMALL_DS[case]
    q, k, v, do = make(device, B, Sq, Sk, H, Hkv, D, 'f16', seed=11)
    do = eighths(do, 12)
    kw = dict(causal=causal, q_len=lens(ql, device), k_len=lens(kl, device))
    f = 2.0 ** power
    want, got = run(q, k, v, do, **kw), run(q, k, v, (do.float() * f).half(), **kw)
    assert torch.equal(want[0], got[0])
    for name, a, b in zip(('dq', 'dk', 'dv'), got[1:], want[1:]):
        b = b.double() * f
        assert torch.isfinite(a).all() and torch.isfinite(b).all(), name
        off = (a.double() - b).abs() - 2.0 ** -10 * (1 + 2.0 ** -10) * b.abs() - 2.0 ** -25 * (1 + f)
        assert float(off.max()) <= 0, '%s: %.3g over its tolerance' % (name, float(off.max()))


def test_fp16_gradients_of_rows_of_unequal_size(device):
    """Every row of dO times a power of two of its own: dq's rows are its multiples, a small row loses nothing beside a large
    one."""
    q, k, v, do = make(device, 1, 200, 3000, 2, 2, 64, 'f16', seed=13)
    do = eighths(do, 14)
    f = 2.0 ** torch.randint(-14, 9, (1, 200, 2, 1), generator=torch.Generator().manual_seed(15)).to(device).double()
    want, got = run(q, k, v, do)[1].double() * f, run(q, k, v, (do.double() * f).half())[1]
    off = (got.double() - want).abs() - 2.0 ** -10 * (1 + 2.0 ** -10) * want.abs() - 2.0 ** -25 * (1 + f)
    assert float(off.max()) <= 0


@pytest.mark.parametrize('case', [(1, 64, 8, 2, 1, 64), (1, 64, 8, 2, 1, 128), (16, 130, 8, 16, 16, 64)])
def test_fp16_ds_beyond_its_range(device, case):
    """dS over 65504 (large values, gradients as a loss scale leaves them) under results that fit."""
    B, Sq, Sk, H, Hkv, D = case
    q, k, v, do = make(device, B, Sq, Sk, H, Hkv, D, 'f16', seed=16)
    q, k, v, do = q * 0.25, k * 0.05, v * 16 + 4 * v.sign(), (do * 1500).clamp(-6900, 6900)
    heads = lambda t: t.double().repeat_interleave(H // t.shape[2], 2).transpose(1, 2).contiguous()  # noqa: E731
    p = torch.softmax(heads(q) @ heads(k).transpose(2, 3).contiguous() / math.sqrt(D), -1)
    dp = heads(do) @ heads(v).transpose(2, 3).contiguous()
    assert float((p * (dp - (p * dp).sum(-1, keepdim=True))).abs().max()) > 65504
    want, tol = reference(q, k, v, do, 1 / math.sqrt(D), False, None, None, False)
    assert all(float(w.abs().max()) < 65504 for w in want)
    compare(run(q, k, v, do), want, tol)


def bounds(q, k, v, do, scale, causal):
    """(o, dq, dk, dv) in float64 and what each may be off by BEFORE its own rounding: reference()'s terms without lengths, with
    factors held to f = r^2 (two parts of the element type), o's low part kept for delta (r^2, or half fp16's smallest step) and fp16's
    dS held until its column's largest is over 2^12."""
    B, Sq, H, D = q.shape
    Sk, Hkv = k.shape[1:3]
    u, r = 2.0 ** -24, torch.finfo(q.dtype).eps / 2
    f, half = r * r, q.dtype == torch.float16
    zp, zd, zo = (2.0 ** -40, 2.0 ** -37, 2.0 ** -25) if half else (2.0 ** -126, 0.0, 0.0)
    heads = lambda t: t.double().repeat_interleave(H // t.shape[2], 2).transpose(1, 2).contiguous()  # noqa: E731
    Q, K, V, G = (heads(t) for t in (q, k, v, do))
    T = lambda t: t.transpose(2, 3).contiguous()  # noqa: E731
    s = scale * Q @ T(K)
    if causal:
        s = s.masked_fill(torch.ones_like(s, dtype=torch.bool).triu(1 + Sk - Sq), -math.inf)
    p = torch.softmax(s, -1)
    e = u * ((D + 6) * float((scale * Q.abs() @ T(K.abs())).max()) + math.log(Sk) + 8)
    ep = 2 * e + (Sk + 4) * u
    o = p @ V
    to = (ep + f + (Sk + 4) * u) * (p @ V.abs()) + zp * V.abs().sum(2, keepdim=True)
    dp, adp = G @ T(V), G.abs() @ T(V.abs())
    ds = p * (dp - (G * o).sum(-1, keepdim=True))
    edl = (G.abs() * (to + (r * r + D * u) * o.abs() + zo)).sum(-1, keepdim=True)
    eds = p * (1 + ep) * ((D + 2) * u * adp + edl) + (ep + f + 4 * u) * ds.abs() + 2.0 ** -126 * adp
    row, col = (eds + zd * ds.abs().amax(i, keepdim=True) for i in (3, 2))
    n = Sq * H // Hkv
    tq = scale * (row + (Sk + 5) * u * ds.abs()) @ K.abs()
    tk = scale * T(col + (n + 6) * u * ds.abs()) @ Q.abs()
    tv = T((ep + f + (n + 6) * u) * p + zp) @ G.abs()
    back = lambda t: t.transpose(1, 2)  # noqa: E731
    sums = lambda t: back(t).unflatten(2, (Hkv, H // Hkv)).sum(3)  # noqa: E731
    return [back(o), back(scale * ds @ K), sums(scale * T(ds) @ Q), sums(T(p) @ G)], [back(to), back(tq), sums(tk), sums(tv)]


@pytest.mark.parametrize('dtype', ['bf16', 'f16'])
@pytest.mark.parametrize('case', [(2, 1, 700, 2, 2, 64, False), (2, 1, 600, 4, 2, 128, True), (1, 1, 500, 8, 2, 64, False),
                                  (2, 150, 150, 4, 2, 64, True), (2, 90, 210, 2, 1, 128, False), (16, 130, 140, 16, 16, 64, True),
                                  (16, 130, 100, 16, 8, 128, False)])
def test_16_bit_results_are_off_by_their_own_rounding(device, case, dtype):
    """p and dS as factors, and the o that delta is of, hold twice the type's bits: a result is within half a step of float64's and
    the little that is left of fp32's sums and of those factors."""
    B, Sq, Sk, H, Hkv, D, causal = case
    q, k, v, do = make(device, B, Sq, Sk, H, Hkv, D, dtype, seed=21)
    r, tiny = torch.finfo(q.dtype).eps / 2, float(torch.finfo(q.dtype).smallest_normal)
    want, tol = bounds(q, k, v, do, 1 / math.sqrt(D), causal)
    for name, a, b, t in zip(('o', 'dq', 'dk', 'dv'), run(q, k, v, do, causal=causal), want, tol):
        step = r * torch.exp2(torch.log2((b.abs() + t).clamp_min(tiny)).floor())
        off = (a.double() - b).abs() - step - t
        assert float(off.max()) <= 0, '%s: %.3g of a half step over its tolerance' % (name, float((off / step).max()))
