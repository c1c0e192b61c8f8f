"""adamw_step against the definition in float64.

32-bit states, u = 2^-24: each moment is two products and a sum with rounded coefficients, 4 u of the sum of their sizes; the
update m / (sqrt(v) rc + eps) adds 12 u of itself to what m is off by, the parameter three roundings and its own type's.
8-bit states: the codes are the nearest of the exact moments, so they have to be equal (the float64 test decides as the
kernel does unless a moment lies within 2^-50 of a border; the scales are one division rounded to fp32).
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}
SHAPES = [(1,), (3,), (4,), (255,), (256,), (257,), (5, 7), (64, 3, 3, 3), (4096,), (4097,), (33, 129), (0,), (20000,)]
HYPER = dict(lr=1e-2, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.05)


def v_table(device):
    c = torch.arange(255, device=device)
    val = torch.exp2(((c >> 3) - 31).double()) * (1 + (c & 7).double() / 8)
    return torch.where(c == 0, 0.0, val)


def nearest(table, y):
    """Index of the table value nearest to y, the even index where two are as near."""
    hi = torch.searchsorted(table, y.contiguous()).clamp(1, table.numel() - 1)
    up, down = table[hi] - y, y - table[hi - 1]
    return torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, hi - 1)


def make(device, shapes, dtype, bits, seed=0, off=0):
    """Parameters, gradients and states of a run under way; `off` shifts every tensor's first byte by that many values."""
    from cmvae_amd.optim import state_size
    g = torch.Generator().manual_seed(seed)

    def place(x):
        buf = torch.empty(x.numel() + off, device=device, dtype=dtype)
        return buf[off:].view(x.shape).copy_(x)

    p = [place(torch.randn(s, generator=g) * 0.1) for s in shapes]
    gr = [place(torch.randn(s, generator=g) * 10.0 ** float(torch.randint(-4, 1, (1,), generator=g))) for s in shapes]
    sizes = [state_size(x.numel()) for x in p]
    n = sum(sizes)
    inside = torch.cat([torch.arange(k) < x.numel() for k, x in zip(sizes, p)] + [torch.zeros(0, dtype=torch.bool)])
    if bits == 32:
        m, v, sc = torch.randn(n, generator=g) * 1e-2 * inside, torch.rand(n, generator=g) ** 8 * 1e-3 * inside, None
    else:
        m = (torch.randn(n, generator=g).clamp(-4, 4) * 112 * inside).to(torch.float8_e4m3fn)
        v = (torch.randint(0, 255, (n,), generator=g) * inside).to(torch.uint8)
        sm = torch.rand(n // 256, generator=g) * 1e-4 + 1e-7
        sc = torch.stack([sm, sm * sm * 1e4]).to(device)
    return p, gr, m.to(device), v.to(device), sc


def reference(p, g, m, v, sc, t, lr, betas, eps, weight_decay):
    """Float64: per tensor (p, tolerance) and the states (m, v with tolerances; 8 bits: codes and scales)."""
    u = 2.0 ** -24
    b1, b2 = betas
    out, at = [], 0
    st = [torch.zeros(m.numel(), dtype=torch.float64, device=m.device) for _ in range(4)]
    codes = [torch.zeros(m.numel(), dtype=torch.int64, device=m.device) for _ in range(2)]
    scales = None if sc is None else sc.clone()
    if sc is not None:
        tab = (torch.arange(127, device=m.device).to(torch.uint8).view(torch.float8_e4m3fn).float().double(), v_table(m.device))
    for x, gr in zip(p, g):
        n = x.numel()
        k = (n + 255) // 256 * 256
        sl, at = slice(at, at + k), at + k
        if n == 0:
            out.append((x.double(), x.double()))
            continue
        gd = torch.zeros(k, dtype=torch.float64, device=m.device)
        gd[:n] = gr.reshape(-1).double()
        if sc is None:
            mo, vo = m[sl].double(), v[sl].double()
        else:
            bs = slice(sl.start // 256, sl.stop // 256)
            mo = m[sl].float().double() * sc[0, bs].double().repeat_interleave(256)
            vo = tab[1][v[sl].long()] * sc[1, bs].double().repeat_interleave(256)
        mn, vn = b1 * mo + (1 - b1) * gd, b2 * vo + (1 - b2) * gd * gd
        em = 4 * u * (b1 * mo.abs() + (1 - b1) * gd.abs())
        st[0][sl], st[1][sl], st[2][sl], st[3][sl] = mn, vn, em + 2e-38, 5 * u * vn + 2e-38
        if sc is not None:
            for i, (tb, top, val) in enumerate(((tab[0], 448.0, mn), (tab[1], 1.75, vn))):
                w = val.view(-1, 256)
                s = (w.abs().amax(1) / top).clamp_min(2.0 ** -126).float()
                scales[i, bs] = s
                c = nearest(tb, (w.abs() / s.double()[:, None]).clamp_max(top))
                if i:
                    c = torch.where((c == 0) & (w > 0), 1, c)
                codes[i][sl] = (c * (torch.sign(w).long() if i == 0 else 1)).flatten()
        den = (vn[:n] / (1 - b2 ** t)).sqrt() + eps
        step = lr / (1 - b1 ** t)
        q = mn[:n] / den
        pd = x.reshape(-1).double()
        pn = pd * (1 - lr * weight_decay) - step * q
        r = torch.finfo(x.dtype).eps / 2
        # a root under 2^-149's own root is lost in eps; fp16 below its normal range is off by half its smallest step
        tol = 3 * u * pd.abs() + step * (em[:n] / den + 14 * u * q.abs()) + r * pn.abs() * (1 + 4 * u) + 2.0 ** -25 * (x.dtype == torch.float16) + 2e-38
        out.append((pn.view(x.shape), tol.view(x.shape)))
    return out, st, codes, scales


def within(a, b, t, what):
    off = (a.double() - b).abs() - t
    assert a.numel() == 0 or float(off.max()) <= 0, '%s: %.3g over its tolerance' % (what, float(off.max()))


def check_step(p, g, m, v, sc, t, **hyper):
    from cmvae_amd.optim import adamw_step
    want, st, codes, scales = reference(p, g, m, v, sc, t, **hyper)
    adamw_step(p, g, m, v, sc, step=t, **hyper)
    for i, (x, (w, tol)) in enumerate(zip(p, want)):
        within(x, w, tol, 'p[%d]' % i)
    if sc is None:
        within(m, st[0], st[2], 'm')
        within(v, st[1], st[3], 'v')
        return
    assert torch.equal(sc, scales)
    table = torch.arange(127, device=m.device).to(torch.uint8).view(torch.float8_e4m3fn).float()
    assert torch.equal(m.float(), table[codes[0].abs()] * codes[0].sign())
    assert torch.equal(v.long(), codes[1])


@pytest.mark.parametrize('bits', [32, 8])
@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('off', [0, 1])
def test_against_float64(device, dtype, bits, off):
    """Three steps on; `off` = 1: no tensor starts at a multiple of 4 values."""
    p, g, m, v, sc = make(device, SHAPES, TYPES[dtype], bits, off=off)
    for t in (100, 101, 102):
        check_step(p, g, m, v, sc, t, **HYPER)


@pytest.mark.parametrize('bits', [32, 8])
def test_first_steps_from_zero(device, bits):
    from cmvae_amd.optim import AdamW
    p, g, _, _, _ = make(device, SHAPES, torch.float32, bits, seed=3)
    opt = AdamW(p, state_bits=bits, **HYPER)
    for t in (1, 2):
        check_step(p, g, opt.exp_avg, opt.exp_avg_sq, opt.scales, t, **HYPER)


@pytest.mark.parametrize('bits', [32, 8])
def test_many_tensors_of_mixed_types(device, bits):
    """More tensors than one launch holds."""
    from cmvae_amd.optim import adamw_step, state_size
    parts = [make(device, [(n,) for n in range(1 + k, 2000, 23)], dt, bits, seed=k) for k, dt in enumerate(TYPES.values())]
    ps, gs = [p for x in parts for p in x[0]], [g for x in parts for g in x[1]]
    m, v = torch.cat([x[2].view(torch.uint8) for x in parts]).view(parts[0][2].dtype), torch.cat([x[3] for x in parts])
    sc = None if bits == 32 else torch.cat([x[4] for x in parts], 1)
    assert len(ps) > 200 and sum(state_size(p.numel()) for p in ps) == m.numel()
    check_step(ps, gs, m, v, sc, 7, **HYPER)


def test_values_and_extremes_of_8_bit_states(device):
    """Blocks of zeros, of one value, of tiny and of huge gradients; what the states stand for."""
    from cmvae_amd.optim import adamw_state_values
    n = 256 * 6
    g = torch.zeros(n, device=device)
    g[256:512] = 0.25
    g[512:768] = 1e-18 * torch.randn(256, generator=torch.Generator().manual_seed(0)).to(device)
    g[768:1024] = 1e18
    g[1024] = 1e3
    g[1025:1280] = 1e-12
    g[1280:] = torch.logspace(-30, 3, 256, device=device)
    p, m = torch.ones(n, device=device), torch.zeros(n, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)
    v, sc = torch.zeros(n, dtype=torch.uint8, device=device), torch.zeros(2, n // 256, device=device)
    for t in (1, 2, 3):
        check_step([p], [g], m, v, sc, t, **HYPER)
        mv, vv = adamw_state_values(m, v, sc)
        assert torch.equal(mv, m.float() * sc[0].repeat_interleave(256))
        assert torch.equal(vv, (v_table(device)[v.long()] * sc[1].double().repeat_interleave(256)).float())
    assert torch.equal(p[:256], torch.full_like(p[:256], (1 - 5e-4) ** 3)) or (p[:256] - (1 - 5e-4) ** 3).abs().max() < 4e-7
    assert torch.isfinite(p).all()


@pytest.mark.parametrize('bits', [32, 8])
def test_a_gradient_that_is_not_finite_stays_alone(device, bits):
    from cmvae_amd.optim import adamw_step
    p, g, m, v, sc = make(device, [(700,)], torch.float32, bits)
    ref = [t.clone() for t in (p[0], m.view(torch.uint8), v)]
    sr = None if sc is None else sc.clone()
    g[0][[5, 300]] = 0.0
    clean = [g[0].clone()]
    adamw_step([ref[0]], clean, ref[1].view(m.dtype), ref[2], sr, step=9, **HYPER)
    g[0][5], g[0][300] = float('nan'), float('inf')
    adamw_step(p, g, m, v, sc, step=9, **HYPER)
    keep = torch.ones(700, dtype=torch.bool, device=device)
    keep[[5, 300]] = False
    assert not torch.isfinite(p[0][~keep]).any() and torch.isfinite(p[0][keep]).all()
    if bits == 32:
        assert torch.equal(p[0][keep], ref[0][keep])
        return
    # the two values' blocks lose their part in the scales only: compare where the clean run's maximum is another value's
    assert torch.isnan(m.float()[[5, 300]]).all() and (v[[5, 300]] == 255).all()
    assert torch.equal(p[0][keep], ref[0][keep])
    assert torch.isfinite(sc).all() and torch.equal(sc[:, 2], sr[:, 2])
    adamw_step(p, [torch.zeros_like(p[0])], m, v, sc, step=10, **HYPER)
    assert not torch.isfinite(p[0][~keep]).any() and torch.isfinite(p[0][keep]).all()


def test_missing_gradients_and_other_strides(device):
    from cmvae_amd.optim import adamw_step
    p, g, m, v, _ = make(device, [(40,), (6, 8, 5, 5), (300,)], torch.float32, 32)
    want, st, _, _ = reference(p, g, m, v, None, 4, **HYPER)
    old = [p[0].clone(), m[:256].clone(), v[:256].clone()]
    g[1] = g[1].to(memory_format=torch.channels_last)           # same values, other order than the parameter's
    adamw_step(p, [None, g[1], g[2]], m, v, step=4, **HYPER)
    assert torch.equal(p[0], old[0]) and torch.equal(m[:256], old[1]) and torch.equal(v[:256], old[2])
    for i in (1, 2):
        within(p[i], *want[i], 'p[%d]' % i)
    within(m[256:], st[0][256:], st[2][256:], 'm')
    cl = torch.randn(6, 8, 5, 5, generator=torch.Generator().manual_seed(1)).to(device).to(memory_format=torch.channels_last)
    a, b = cl.clone(memory_format=torch.preserve_format), cl.contiguous().clone()
    ms = [torch.zeros(1280, device=device) for _ in range(4)]
    adamw_step([a], [cl], ms[0], ms[1], step=1)
    adamw_step([b], [cl.contiguous()], ms[2], ms[3], step=1)
    assert torch.equal(a, b)


@pytest.mark.parametrize('bits', [32, 8])
def test_class_state_dict_and_flat_grads(device, bits):
    """AdamW over leaves' .grad and over a FlatGrads, saved and resumed; the same bits as adamw_step."""
    from cmvae_amd.dist import FlatGrads
    from cmvae_amd.optim import AdamW, adamw_step
    p, g, _, _, _ = make(device, [(9, 9), (300,), (2, 2)], torch.float32, bits)
    sets = [[torch.nn.Parameter(x.clone()) for x in p] for _ in range(3)]
    plain = [x.clone() for x in p]
    flat = FlatGrads(sets[1])
    opts = [AdamW(sets[0], state_bits=bits, **HYPER), AdamW(flat, state_bits=bits, **HYPER),
            AdamW(sets[2], state_bits=bits, **HYPER).device_step()]
    ref = AdamW(plain, state_bits=bits, **HYPER)
    for t in range(1, 4):
        flat.zero()
        for s in sets:
            for x, y in zip(s, g):
                x.grad = y.clone()
        flat.allreduce()
        for o in opts:
            o.step()
        adamw_step(plain, g, ref.exp_avg, ref.exp_avg_sq, ref.scales, step=t, **HYPER)
        if t == 2:
            sd = {k: (v.clone() if torch.is_tensor(v) else v) for k, v in opts[0].state_dict().items()}
            opts[0] = AdamW(sets[0], state_bits=bits, **HYPER)
            opts[0].load_state_dict(sd)
    for s in sets:
        assert all(torch.equal(a.detach(), b) for a, b in zip(s, plain))
    assert int(opts[2].state_dict()['step']) == opts[0].state_dict()['step'] == 3
    with pytest.raises(RuntimeError, match='saved states'):
        AdamW(sets[0], state_bits=40 - bits).load_state_dict(sd)


@pytest.mark.parametrize('bits', [32, 8])
def test_graph_replays_and_other_stream(device, bits):
    from cmvae_amd.optim import AdamW
    p, g, _, _, _ = make(device, [(500,), (64, 64), (7,)], torch.bfloat16, bits)
    a, b = [x.clone() for x in p], [x.clone() for x in p]
    oa, ob = AdamW(a, state_bits=bits, **HYPER).device_step(), AdamW(b, state_bits=bits, **HYPER)
    for x, y in zip(a, g):
        x.grad = y
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        oa.step()
    side = torch.cuda.Stream()
    for t in range(4):
        for y in g:
            y.mul_(0.5)
        graph.replay()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for x, y in zip(b, g):
                x.grad = y
            ob.step()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        # the device computes 1 - b^t with its own pow: one fp32 rounding of a coefficient may differ
        for x, y in zip(a, b):
            assert (x.float() - y.float()).abs().max() <= 2.0 ** -8 * y.float().abs().max() * 2.0 ** -1 + 1e-6
        assert torch.equal(oa.exp_avg.view(torch.uint8), ob.exp_avg.view(torch.uint8))
        assert torch.equal(oa.exp_avg_sq, ob.exp_avg_sq)


def test_refusals(device):
    from cmvae_amd.optim import AdamW, adamw_state_values, adamw_step
    z = lambda n, dt=torch.float32: torch.zeros(n, device=device, dtype=dt)  # noqa: E731
    p, g, m, v = z(100), z(100), z(256), z(256)
    m8, v8, sc = z(256, torch.uint8).view(torch.float8_e4m3fn), z(256, torch.uint8), z(2).view(2, 1)
    for args, kw in [(([p], [g, g], m, v), {}), (([p, p], [g, g], z(512), z(512)), {}), (([p], [g.bfloat16()], m, v), {}),
                     (([p.double()], [g.double()], m, v), {}), (([p], [z(99)], m, v), {}), (([p], [g], z(512), z(512)), {}),
                     (([p], [g], m, z(512)), {}), (([p], [g], z(100), z(100)), {}), (([p], [g], m8, v8), {}),
                     (([p], [g], m, v, sc), {}), (([p], [g], m8, v8, sc.double()), {}), (([p], [g], m8, v8, z(4).view(2, 2)), {}),
                     (([p], [g], m, v), dict(step=0)), (([p], [g], m, v), dict(step=torch.ones(1, device=device))),
                     (([p], [g], m, v), dict(betas=(1.0, 0.9))), (([p], [g], m, v), dict(lr=float('nan'))),
                     (([z(200)[::2]], [g], m, v), {}), (([p.cpu()], [g.cpu()], m, v), {}), (([p], [g], m.view(2, 128), v), {})]:
        with pytest.raises(RuntimeError, match='adamw'):
            adamw_step(*args, **kw)
    with pytest.raises(RuntimeError, match='adamw'):
        adamw_state_values(m, v, None)
    with pytest.raises(RuntimeError, match='AdamW'):
        AdamW([p], state_bits=16)


@pytest.mark.parametrize('bits', [32, 8])
def test_more_values_than_32_bits_count(device, bits):
    """A tensor of 2^31 + 300 values, with something in its last 1024 only, behind a small one: they become what a tensor of
    those 1024 becomes, the others stay."""
    from cmvae_amd.optim import adamw_step, state_size
    n, tail = 2 ** 31 + 300, 300 + 256 * 3
    small, gs, m, v, sc = make(device, [(tail,)], torch.bfloat16, bits, seed=5)
    k = state_size(n) + 256
    p, g = (torch.zeros(n, dtype=torch.bfloat16, device=device) for _ in range(2))
    p[-tail:], g[-tail:] = small[0], gs[0]
    M, V = (torch.zeros(k * x.element_size(), dtype=torch.uint8, device=device).view(x.dtype) for x in (m, v))
    at = k - m.numel()
    M[at:], V[at:] = m, v
    S = None
    if bits == 8:
        S = torch.zeros(2, k // 256, device=device)
        S[:, at // 256:] = sc
    one = [torch.ones(2, dtype=torch.bfloat16, device=device) for _ in range(2)]
    adamw_step([one[0], p], [one[1], g], M, V, S, step=7, **HYPER)
    adamw_step(small, gs, m, v, sc, step=7, **HYPER)
    assert torch.equal(p[-tail:], small[0]) and not p[:-tail].any()
    assert torch.equal(M[at:].view(torch.uint8), m.view(torch.uint8)) and torch.equal(V[at:], v)
    assert sc is None or torch.equal(S[:, at // 256:], sc)
    assert not V[256:at].any()


def test_tensors_that_overlap_are_refused(device):
    from cmvae_amd.optim import adamw_step
    z = lambda n: torch.zeros(n, device=device)  # noqa: E731
    buf, g = z(300), z(100)
    m, v = z(512), z(512)
    for params, exp_avg, exp_avg_sq in (([buf[:100], buf[99:199]], m, v), ([buf[100:200], buf[:100], buf[150:250]], z(768), z(768)),
                                        ([buf[:100], z(100)], m, m), ([m[:100], z(100)], m, v), ([z(100), v[412:]], m, v)):
        with pytest.raises(RuntimeError, match='overlap'):
            adamw_step(params, [g] * len(params), exp_avg, exp_avg_sq)
    adamw_step([buf[:100], buf[100:200]], [g, g], m, v)


def test_what_is_read_overlaps_nothing_that_is_written(device):
    """A gradient inside of another stepped parameter, of a state, or shifted against its own parameter, and a step count inside
    of a state would be read before or after they are written, as it happens: refused.  Nothing is launched."""
    from cmvae_amd.optim import adamw_step
    z = lambda n, dt=torch.float32: torch.zeros(n, device=device, dtype=dt)  # noqa: E731
    m, v, p, g, buf = z(10240), z(10240), z(5000), z(5000), z(5001)
    for params, grads, step in (([p, g], [g, z(5000)], 1), ([p, g], [z(5000), p], 1), ([buf[:5000], p], [buf[1:], g], 1),
                                ([buf[1:], p], [buf[:5000], g], 1), ([p, z(5000)], [g, m[5120:10120]], 1),
                                ([p, z(5000)], [v[:5000], g], 1), ([p, z(5000)], [g, z(5000)], m.view(torch.int64)[7:8])):
        with pytest.raises(RuntimeError, match='overlap'):
            adamw_step(params, grads, m, v, step=step)
    m8, v8, scales = z(10496, torch.uint8).view(torch.float8_e4m3fn), z(10496, torch.uint8), z(82).view(2, 41)
    with pytest.raises(RuntimeError, match='overlap'):
        adamw_step([z(10160), z(80)], [z(10160), scales.view(-1)[1:81]], m8, v8, scales)
    assert not any(t.any() for t in (m, v, p, g, buf, scales))


def test_gradients_that_may_share_memory(device):
    """One gradient of several parameters, a parameter that is left out, neighbours in one buffer, a parameter as its own gradient."""
    from cmvae_amd.optim import adamw_step
    g = torch.Generator().manual_seed(8)
    flat = torch.randn(4 * 5000, generator=g).to(device)
    p0, g0, p1, g1 = flat.view(4, 5000).unbind(0)
    for ps, gs in (([p0, p1], [g0, g1]), ([p0, p1], [g0, g0]), ([p0, g1], [p1, None]), ([p0, p1], [p0, g1])):
        m, v = torch.zeros(10240, device=device), torch.zeros(10240, device=device)
        want, _, _, _ = reference(ps, [torch.zeros_like(p) if x is None else x for p, x in zip(ps, gs)], m, v, None, 1, **HYPER)
        old = g1.clone()
        adamw_step(ps, gs, m, v, step=1, **HYPER)
        for p, x, (w, tol) in zip(ps, gs, want):
            if x is None:
                assert torch.equal(p, old)
            else:
                within(p, w, tol, 'p')
