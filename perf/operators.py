"""Measured cases of three training operators: set attention with its recomputing backward pass
(`cmvae_amd.attention.set_attention`), the AdamW step over many tensors (`cmvae_amd.optim.adamw_step`) and group norm with
an activation on channels-last data (`cmvae_amd.norm.group_norm_act`).

`run` computes an operator in its plain form, in elementary torch operations, or (`own`) by the framework's call; `exact`
restates the definition in float64.
"""
import math
import random

import torch
import torch.nn.functional as F

own = False

DEV = 'cuda'
TYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}
BLOCK = 256                 # values per scale of the 8-bit optimizer states


# ----------------------------------------------------------------------------- cases
def listed():
    return [
        # pooling a whole set by one learned query: 200 samples x 32 Monte-Carlo draws, the latents of one Omniglot episode
        dict(name='pool_f32', op='attn', B=4, Sq=1, Sk=6400, H=4, Hkv=4, D=64, dtype='f32', causal=False, ragged=False,
             residual=True, train=False),
        # single-token step against a long cache, grouped heads: what an answering model runs per token
        dict(name='token_bf16', op='attn', B=16, Sq=1, Sk=8191, H=32, Hkv=8, D=128, dtype='bf16', causal=True, ragged=True,
             residual=False, train=False),
        # the set-attention block of one Omniglot meta-batch (4 episodes of 200 samples): latency
        dict(name='block_f32', op='attn', B=4, Sq=200, Sk=200, H=4, Hkv=4, D=64, dtype='f32', causal=False, ragged=False,
             residual=True, train=True),
        # a padded meta-batch of episodes with unequal numbers of samples
        dict(name='sets_f32', op='attn', B=16, Sq=1531, Sk=1531, H=4, Hkv=4, D=64, dtype='f32', causal=False, ragged=True,
             residual=True, train=True),
        # queries of one set against the padded support of another, shared key heads
        dict(name='cross_f16', op='attn', B=8, Sq=777, Sk=2049, H=8, Hkv=2, D=64, dtype='f16', causal=False, ragged=True,
             residual=False, train=True),
        # training on long sequences
        dict(name='long_bf16', op='attn', B=2, Sq=4096, Sk=4096, H=16, Hkv=4, D=128, dtype='bf16', causal=True, ragged=False,
             residual=False, train=True),
        # every parameter of the Omniglot model (58 tensors, 1.14 M values), one step: latency
        dict(name='adamw32_model', op='adamw', layers=0, width=64, dtype='f32', bits=32),
        # a stack of wide layers, states in 32 bits beside 16-bit parameters
        dict(name='adamw32_bf16', op='adamw', layers=4, width=1600, dtype='bf16', bits=32),
        # the same kind of stack with states in 8 bits: what decides whether the optimizer fits
        dict(name='adamw8_f32', op='adamw', layers=5, width=1283, dtype='f32', bits=8),
        # last encoder layer of an episode: few pixels per sample
        dict(name='norm_small_f32', op='norm', N=800, P=16, C=64, G=8, dtype='f32', act='elu', train=True),
        # second encoder layer of an Omniglot meta-batch: 14 x 14 pixels, 64 channels
        dict(name='norm_enc_f32', op='norm', N=800, P=196, C=64, G=8, dtype='f32', act='elu', train=True),
        # a wide convolutional stage on large images
        dict(name='norm_wide_bf16', op='norm', N=16, P=9216, C=320, G=32, dtype='bf16', act='silu', train=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(['attn', 'attn', 'adamw', 'norm'])
    if op == 'attn':
        while True:
            Hkv, G = rng.choice([1, 2, 4, 8]), rng.choice([1, 1, 2, 4])
            c = dict(op='attn', B=_log_int(rng, 1, 16), Sq=rng.choice([1, _log_int(rng, 2, 4096), _log_int(rng, 64, 4096)]),
                     Sk=_log_int(rng, 64, 8192), H=Hkv * G, Hkv=Hkv, D=rng.choice([64, 128]),
                     dtype=rng.choice(['f32', 'bf16', 'f16']), causal=rng.random() < 0.4, ragged=rng.random() < 0.5,
                     residual=rng.random() < 0.4, train=rng.random() < 0.7)
            if c['causal'] and c['Sq'] > c['Sk']:
                c['Sq'] = c['Sk']
            if c['B'] * c['H'] * c['Sq'] * c['Sk'] * c['D'] <= 1.2e10:
                return c
    if op == 'adamw':
        bits = rng.choice([8, 32])
        if rng.random() < 0.25:
            return dict(op='adamw', layers=0, width=rng.choice([64, 128, 192]), dtype=rng.choice(['f32', 'bf16', 'f16']),
                        bits=bits)
        return dict(op='adamw', layers=rng.randint(1, 4), width=_log_int(rng, 61, 1280),
                    dtype=rng.choice(['f32', 'bf16', 'f16']), bits=bits)
    while True:
        G = rng.choice([1, 2, 4, 8, 16, 32])
        c = dict(op='norm', N=_log_int(rng, 1, 1024), P=_log_int(rng, 1, 16384), C=G * _log_int(rng, 2, 40), G=G,
                 dtype=rng.choice(['f32', 'bf16', 'f16']), act=rng.choice(['none', 'elu', 'silu']), train=rng.random() < 0.7)
        if 65536 <= c['N'] * c['P'] * c['C'] <= 40_000_000 and c['P'] * c['C'] // G >= 16:
            return c


# ----------------------------------------------------------------------------- shapes that follow from a case
def _lens(S, B, salt):
    """Lengths of a padded batch: one full, the others spread over (S / 4, S]."""
    r = random.Random(S * 1009 + B * 31 + salt)
    return [S] + [r.randint(max(1, S // 4), S) for _ in range(B - 1)]


def _qk_lens(c):
    if not c['ragged']:
        return None, None
    kl = _lens(c['Sk'], c['B'], 1)
    if c['Sq'] == 1:
        return None, kl
    if c['Sq'] == c['Sk']:
        return kl, kl
    ql = _lens(c['Sq'], c['B'], 2)
    return ([min(a, b) for a, b in zip(ql, kl)] if c['causal'] else ql), kl


def _pairs(c):
    """Valid (query, key) pairs per head, over the batch."""
    ql, kl = _qk_lens(c)
    ql, kl = ql or [c['Sq']] * c['B'], kl or [c['Sk']] * c['B']
    if not c['causal']:
        return sum(a * b for a, b in zip(ql, kl))
    return sum(a * b - a * (a - 1) // 2 for a, b in zip(ql, kl))


def _shapes(c):
    w = c['width']
    if c['layers'] == 0:                                   # the Omniglot model's parameters at hidden size w
        enc = [[w, 1, 3, 3], [w], [w], [w]] + 3 * [[w, w, 3, 3], [w], [w], [w]]
        f = 4 * w
        heads = 2 * (4 * [[f, f], [f]]) + [[2 * 64, f], [2 * 64]]
        causal = [[2048, 64], [2048], [64, 32, 1], [64, 1]]
        proj = [[f, 64], [f], [f, f], [f], [f, f], [f]]
        dec = [[w, w, 4, 4], [w], [w], [w], [w, w, 3, 3], [w], [w], [w], [w, w, 4, 4], [w], [w], [w], [w, 1, 4, 4], [1]]
        return enc + heads + causal + proj + dec
    return c['layers'] * [[w, w], [w, w], [w, w], [w, w], [w], [w], [4 * w, w], [4 * w], [w, 4 * w], [w], [w]]


def _numel(shape):
    return math.prod(shape)


def _padded(n):
    return (n + BLOCK - 1) // BLOCK * BLOCK


def work(c):
    if c['op'] == 'attn':
        e = 4 if c['dtype'] == 'f32' else 2
        ql, kl = _qk_lens(c)
        nq = sum(ql or [c['Sq']] * c['B']) * c['H'] * c['D'] * e
        nk = sum(kl or [c['Sk']] * c['B']) * c['Hkv'] * c['D'] * e
        fl = _pairs(c) * c['H'] * c['D']
        if c['train']:                                     # q, k, v, do read; o, dq, dk, dv written
            return {'bytes': 4 * nq + 4 * nk, 'flops': 14 * fl}
        return {'bytes': 2 * nq + 2 * nk, 'flops': 4 * fl}
    if c['op'] == 'adamw':
        n = sum(_numel(s) for s in _shapes(c))
        e = 4 if c['dtype'] == 'f32' else 2
        # parameter read and written, gradient read, states read and written; 8-bit states come back as 32-bit values too
        return {'bytes': n * (3 * e + (16 if c['bits'] == 32 else 4 + 8)), 'flops': 16 * n}
    e = 4 if c['dtype'] == 'f32' else 2
    n = c['N'] * c['P'] * c['C']
    return {'bytes': n * e * (4 if c['train'] else 2), 'flops': n * (30 if c['train'] else 10)}


# ----------------------------------------------------------------------------- inputs
def _decode_v(code):
    """The 8-bit form of the second moment: 5 exponent bits, 3 mantissa bits, no sign; 0 is zero."""
    c = code.to(torch.int64)
    val = torch.exp2(((c >> 3) - 31).double()) * (1 + (c & 7).double() / 8)
    return torch.where(c == 0, torch.zeros_like(val), val)


def prepare(c, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = TYPES[c['dtype']]

    def randn(*shape):
        return torch.randn(*shape, device=DEV, generator=g)

    if c['op'] == 'attn':
        s = dict(c)
        B, Sq, Sk, H, Hkv, D = (c[k] for k in ('B', 'Sq', 'Sk', 'H', 'Hkv', 'D'))
        # keys of one set share a direction (their episode's mean), queries lean towards it: peaked but not one-hot rows
        mean = randn(B, 1, 1, D)
        s['q'] = (randn(B, Sq, H, D) + 0.3 * mean).to(dt)
        s['k'] = (randn(B, Sk, Hkv, D) + 0.3 * mean).to(dt)
        s['v'] = randn(B, Sk, Hkv, D).to(dt)
        s['do'] = randn(B, Sq, H, D).to(dt) if c['train'] else None
        ql, kl = _qk_lens(c)
        s['q_len'] = None if ql is None else torch.tensor(ql, dtype=torch.int32, device=DEV)
        s['k_len'] = None if kl is None else torch.tensor(kl, dtype=torch.int32, device=DEV)
        s['scale'] = 1 / math.sqrt(D)
        if c['train']:
            for n in 'qkv':
                s[n].requires_grad_()
        return s
    if c['op'] == 'adamw':
        s = dict(c)
        shapes = _shapes(c)
        s['p'] = [(randn(*sh) * 0.05).to(dt) for sh in shapes]
        # gradients of one tensor differ by orders of magnitude between its rows
        s['g'] = [(randn(*sh) * 1e-2 * torch.exp(1.5 * randn(*([sh[0]] + [1] * (len(sh) - 1))))).to(dt) for sh in shapes]
        total = sum(_padded(_numel(sh)) for sh in shapes)
        inside = torch.cat([torch.arange(_padded(_numel(sh)), device=DEV) < _numel(sh) for sh in shapes])
        s['t'], s['lr'], s['b1'], s['b2'], s['eps'], s['wd'] = 100, 1e-3, 0.9, 0.999, 1e-8, 1e-2
        if c['bits'] == 32:
            s['m'] = randn(total) * 3e-3 * inside
            s['v'] = torch.exp(randn(total) - 9.2) * inside
            s['scales'] = None
        else:
            s['m'] = (randn(total).clamp_(-4, 4) * 112 * inside).to(torch.float8_e4m3fn)
            s['v'] = (torch.randint(120, 255, (total,), device=DEV, generator=g) * inside).to(torch.uint8)
            sm = torch.rand(total // BLOCK, device=DEV, generator=g) * 1e-4 + 1e-6
            s['scales'] = torch.stack([sm, (sm * 100).square()])
        return s
    s = dict(c)
    # activations with an offset and a spread that differ by channel, as a convolution with bias leaves them
    x = randn(c['N'], c['P'], c['C'])
    s['x'] = x.mul_(0.5 + torch.rand(c['C'], device=DEV, generator=g)).add_(randn(c['C'])).to(dt)
    s['w'] = 1 + 0.2 * randn(c['C'])
    s['b'] = 0.2 * randn(c['C'])
    s['dy'] = randn(c['N'], c['P'], c['C']).to(dt) if c['train'] else None
    s['eps'] = 1e-5
    if c['train']:
        for n in 'xwb':
            s[n].requires_grad_()
    return s


# ----------------------------------------------------------------------------- plain forms
def _valid(s):
    """[B, 1, Sq, Sk] truth values: pairs that count."""
    B, Sq, Sk = s['B'], s['Sq'], s['Sk']
    ql = s['q_len'] if s['q_len'] is not None else torch.full((B,), Sq, device=DEV, dtype=torch.int32)
    kl = s['k_len'] if s['k_len'] is not None else torch.full((B,), Sk, device=DEV, dtype=torch.int32)
    i = torch.arange(Sq, device=DEV).view(1, Sq, 1)
    j = torch.arange(Sk, device=DEV).view(1, 1, Sk)
    ql, kl = ql.view(B, 1, 1), kl.view(B, 1, 1)
    ok = (i < ql) & (j < kl)
    if s['causal']:
        ok = ok & (j <= i + kl - ql)
    return ok.unsqueeze(1), (i < ql).view(B, 1, Sq, 1)


def _heads(x, G):
    """[B, S, h, D] -> float [B, h * G, S, D]."""
    x = x.detach().float().transpose(1, 2)
    return (x.repeat_interleave(G, 1) if G > 1 else x).contiguous()


def _attn_plain(s):
    G, dt = s['H'] // s['Hkv'], s['q'].dtype
    q, k, v = _heads(s['q'], 1), _heads(s['k'], G), _heads(s['v'], G)
    ok, row = _valid(s)
    sc = torch.matmul(q, k.transpose(2, 3).contiguous()) * s['scale']
    sc = sc.masked_fill_(~ok, -math.inf)
    p = torch.exp(sc - sc.amax(-1, keepdim=True).clamp_min(-3e38))
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-38)
    o = torch.matmul(p, v)
    if s['residual']:
        o = o + q * row
    out = o.transpose(1, 2).to(dt).contiguous()
    if not s['train']:
        return out
    do = _heads(s['do'], 1) * row
    dv = torch.matmul(p.transpose(2, 3).contiguous(), do)
    ds = torch.matmul(do, v.transpose(2, 3).contiguous())
    ds = p * (ds - (p * ds).sum(-1, keepdim=True)) * s['scale']
    dq = torch.matmul(ds, k)
    dk = torch.matmul(ds.transpose(2, 3).contiguous(), q)
    if s['residual']:
        dq = dq + do
    if G > 1:
        dk, dv = (t.unflatten(1, (s['Hkv'], G)).sum(2) for t in (dk, dv))
    return [out] + [t.transpose(1, 2).to(dt).contiguous() for t in (dq, dk, dv)]


def _blocks(x, n):
    return F.pad(x, (0, _padded(n) - n)).view(-1, BLOCK)


def _nearest(x, bits, least):
    """x rounded to `bits` mantissa bits, ties to even, with no quantum below 2^(least - bits)."""
    e = (torch.frexp(x)[1] - 1).clamp_min(least) - bits
    return torch.ldexp(torch.round(torch.ldexp(x, -e)), e)


def _adamw_tensor(s, p, g, m, v, sc):
    """One tensor's update in place; returns what its states now stand for."""
    n = p.numel()
    c1, c2 = 1 - s['b1'] ** s['t'], 1 - s['b2'] ** s['t']
    if s['bits'] == 32:
        gf = g.float().reshape(-1)
        m[:n] = s['b1'] * m[:n] + (1 - s['b1']) * gf
        v[:n] = s['b2'] * v[:n] + (1 - s['b2']) * gf * gf
        m1, v1, pf = m[:n], v[:n], p.float().reshape(-1)
    else:                                  # 64 bits: which of two neighbouring 8-bit values a number becomes is a border
        gf = _blocks(g.double().reshape(-1), n)
        m1 = s['b1'] * (m.float().double().view(-1, BLOCK) * sc[0].double()[:, None]) + (1 - s['b1']) * gf
        v1 = s['b2'] * (_decode_v(v).view(-1, BLOCK) * sc[1].double()[:, None]) + (1 - s['b2']) * gf * gf
        sc[0] = (m1.abs().amax(1) / 448).clamp_min(2.0 ** -126).float()
        sc[1] = (v1.amax(1) / 1.75).clamp_min(2.0 ** -126).float()
        mq = _nearest(m1 / sc[0].double()[:, None], 3, -6).clamp(-448, 448)
        vn = v1 / sc[1].double()[:, None]
        vq = torch.where(v1 > 0, _nearest(vn, 3, -1000).clamp(1.125 * 2.0 ** -31, 1.75), 0.0)
        e = torch.frexp(vq)[1] - 1
        code = torch.where(vq > 0, (e + 31) * 8 + torch.round(torch.ldexp(vq, -e) * 8 - 8).int(), 0)
        m.copy_(mq.float().reshape(-1).to(torch.float8_e4m3fn))
        v.copy_(code.reshape(-1).to(torch.uint8))
        m1, v1, pf = m1.reshape(-1)[:n], v1.reshape(-1)[:n], p.double().reshape(-1)
    step = (m1 / c1) / (torch.sqrt(v1 / c2) + s['eps'])
    p.copy_((pf * (1 - s['lr'] * s['wd']) - s['lr'] * step).view(p.shape))
    if s['bits'] == 32:
        return m, v
    return (mq * sc[0].double()[:, None]).float().reshape(-1), (vq * sc[1].double()[:, None]).float().reshape(-1)


def _adamw_plain(s):
    sizes = [_padded(p.numel()) for p in s['p']]
    ms, vs = s['m'].split(sizes), s['v'].split(sizes)
    scs = s['scales'].split([n // BLOCK for n in sizes], 1) if s['scales'] is not None else [None] * len(sizes)
    got = [_adamw_tensor(s, *a) for a in zip(s['p'], s['g'], ms, vs, scs)]
    if s['bits'] == 32:
        return s['p'] + [s['m'], s['v']]
    return s['p'] + [torch.cat([a for a, _ in got]), torch.cat([b for _, b in got])]


def _act(z, act):
    if act == 'elu':
        return torch.where(z > 0, z, torch.expm1(z.clamp_max(0))), torch.where(z > 0, 1.0, torch.exp(z.clamp_max(0)))
    if act == 'silu':
        sg = 1 / (1 + torch.exp(-z))
        return z * sg, sg * (1 + z * (1 - sg))
    return z, torch.ones_like(z)


def _norm_plain(s):
    N, P, C, G = s['N'], s['P'], s['C'], s['G']
    x = s['x'].detach().float().view(N, P, G, C // G)
    w, b = s['w'].detach().view(G, C // G), s['b'].detach().view(G, C // G)
    mean = x.mean((1, 3), keepdim=True)
    xc = x - mean
    rstd = 1 / torch.sqrt((xc * xc).mean((1, 3), keepdim=True) + s['eps'])
    xh = xc * rstd
    y, slope = _act(xh * w + b, s['act'])
    y = y.view(N, P, C).to(s['x'].dtype)
    if not s['train']:
        return y
    dz = s['dy'].float().view(N, P, G, C // G) * slope
    dw, db = (dz * xh).sum((0, 1)).view(C), dz.sum((0, 1)).view(C)
    dxh = dz * w
    dx = rstd * (dxh - dxh.mean((1, 3), keepdim=True) - xh * (dxh * xh).mean((1, 3), keepdim=True))
    return [y, dx.view(N, P, C).to(s['x'].dtype), dw, db]


# ----------------------------------------------------------------------------- one pass
def _run_own(s):
    if s['op'] == 'attn':
        from cmvae_amd.attention import set_attention
        o = set_attention(s['q'], s['k'], s['v'], scale=s['scale'], causal=s['causal'], q_len=s['q_len'], k_len=s['k_len'],
                          residual=s['residual'])
        return [o.detach(), *torch.autograd.grad(o, (s['q'], s['k'], s['v']), s['do'])] if s['train'] else o
    if s['op'] == 'adamw':
        from cmvae_amd.optim import adamw_step, adamw_state_values
        adamw_step(s['p'], s['g'], s['m'], s['v'], s['scales'], step=s['t'], lr=s['lr'], betas=(s['b1'], s['b2']),
                   eps=s['eps'], weight_decay=s['wd'])
        if s['bits'] == 32:
            return s['p'] + [s['m'], s['v']]
        return s['p'] + list(adamw_state_values(s['m'], s['v'], s['scales']))
    from cmvae_amd.norm import group_norm_act
    y = group_norm_act(s['x'], s['G'], s['w'], s['b'], eps=s['eps'], act=None if s['act'] == 'none' else s['act'])
    return [y.detach(), *torch.autograd.grad(y, (s['x'], s['w'], s['b']), s['dy'])] if s['train'] else y


def run(s):
    if own:
        return _run_own(s)
    return {'attn': _attn_plain, 'adamw': _adamw_plain, 'norm': _norm_plain}[s['op']](s)


# ----------------------------------------------------------------------------- the definitions in 64 bits
def _exact_attn(c, s):
    B, Sq, H, D = s['q'].shape
    Sk, Hkv = s['k'].shape[1:3]
    ql, kl = _qk_lens(c)
    out = [torch.zeros(B, Sq, H, D, dtype=torch.float64, device=DEV) for _ in range(2)]
    kv = [torch.zeros(B, Sk, Hkv, D, dtype=torch.float64, device=DEV) for _ in range(2)]
    for b in range(B):
        nq, nk = (Sq if ql is None else ql[b]), (Sk if kl is None else kl[b])
        for h in range(H):
            q = s['q'].detach()[b, :nq, h].double()
            k = s['k'].detach()[b, :nk, h * Hkv // H].double()
            v = s['v'].detach()[b, :nk, h * Hkv // H].double()
            z = s['scale'] * q @ k.T
            if c['causal']:
                z = z + torch.full_like(z, -math.inf).triu(nk - nq + 1)
            p = torch.softmax(z, 1)
            out[0][b, :nq, h] = p @ v + (q if c['residual'] else 0)
            if not c['train']:
                continue
            g = s['do'][b, :nq, h].double()
            dp = g @ v.T
            dz = s['scale'] * p * (dp - (g * (p @ v)).sum(1, keepdim=True))
            out[1][b, :nq, h] = dz @ k + (g if c['residual'] else 0)
            kv[0][b, :nk, h * Hkv // H] += dz.T @ q
            kv[1][b, :nk, h * Hkv // H] += p.T @ g
    return out + kv if c['train'] else out[0]


def _exact_adamw(c, s):
    ps, ms, vs, at = [], [], [], 0
    for p, g in zip(s['p'], s['g']):
        n = p.numel()
        end = at + _padded(n)
        gf = torch.zeros(end - at, dtype=torch.float64, device=DEV)
        gf[:n] = g.double().flatten()
        if c['bits'] == 32:
            m, v = s['m'][at:end].double(), s['v'][at:end].double()
        else:
            a, b = (t[at // BLOCK:end // BLOCK].double().repeat_interleave(BLOCK) for t in s['scales'])
            m, v = s['m'][at:end].float().double() * a, _decode_v(s['v'][at:end]) * b
        m.mul_(s['b1']).add_(gf, alpha=1 - s['b1'])
        v.mul_(s['b2']).add_(gf * gf, alpha=1 - s['b2'])
        denom = (v[:n] / (1 - s['b2'] ** s['t'])).sqrt() + s['eps']
        pd = p.double().flatten()
        ps.append((pd - s['lr'] * s['wd'] * pd - s['lr'] / (1 - s['b1'] ** s['t']) * m[:n] / denom).view(p.shape))
        if c['bits'] == 8:
            # every value 8 bits can hold, in order; a number becomes the nearest, the even code where two are as near
            tiny = torch.tensor(2.0 ** -126, dtype=torch.float64, device=DEV)
            mt = torch.arange(127, device=DEV).to(torch.uint8).view(torch.float8_e4m3fn).float().double()
            vt = _decode_v(torch.arange(255, device=DEV))
            rows = []
            for t, table, x in ((448, mt, m), (1.75, vt, v)):
                x = x.view(-1, BLOCK)
                sc = torch.maximum(x.abs().amax(1, keepdim=True) / t, tiny).float().double()
                y = (x / sc).abs().clamp_max(t)
                hi = torch.searchsorted(table, y.contiguous()).clamp(1, table.numel() - 1)
                lo = hi - 1
                up, down = table[hi] - y, y - table[lo]
                take = torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
                if t == 1.75:
                    take = torch.where((take == 0) & (y > 0), 1, take)
                rows.append((table[take] * sc * x.sign()).flatten())
            m, v = rows
        ms.append(m)
        vs.append(v)
        at = end
    return ps + [torch.cat(ms), torch.cat(vs)]


def _exact_norm(c, s):
    ins = [s[n].detach().double() for n in 'xwb']
    N, P, C, G = c['N'], c['P'], c['C'], c['G']
    step = max(1, 8_000_000 // (P * C))
    ys, dxs, dw, db = [], [], 0, 0
    for n0 in range(0, N, step):
        x, w, b = (t.requires_grad_() for t in (ins[0][n0:n0 + step].clone(), ins[1].clone(), ins[2].clone()))
        xg = x.view(-1, P, G, C // G).transpose(1, 2).flatten(2)
        var, mean = torch.var_mean(xg, 2, correction=0, keepdim=True)
        z = ((xg - mean) / (var + s['eps']).sqrt()).view(-1, G, P, C // G).transpose(1, 2).reshape(-1, P, C) * w + b
        y = {'none': lambda t: t, 'elu': F.elu, 'silu': F.silu}[c['act']](z)
        ys.append(y.detach())
        if c['train']:
            gx, gw, gb = torch.autograd.grad(y, (x, w, b), s['dy'][n0:n0 + step].double())
            dxs.append(gx)
            dw, db = dw + gw, db + gb
    return [torch.cat(ys), torch.cat(dxs), dw, db] if c['train'] else torch.cat(ys)


def exact(c, seed):
    s = prepare(c, seed)
    return {'attn': _exact_attn, 'adamw': _exact_adamw, 'norm': _exact_norm}[c['op']](c, s)
