"""Set attention, group norm and AdamW as the framework's blocks and training loop use them: MAB / SAB on large, unequal and
padded sets, a training step of all three (eager, and replayed from a HIP graph), the Trainer's --optimizer."""
import os
import subprocess
import sys

import numpy as np
import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def rel(a, b):
    a, b = a.detach().double().cpu(), b.detach().double().cpu()
    return float((a - b).norm() / b.norm().clamp_min(1e-30))


def mab64(m, Q, K, ql=None, kl=None):
    """MAB.forward (omniglot/module.py:88-112, ln=False) in float64, one episode and head at a time."""
    def lin(x, l):
        return x @ l.weight.double().T + l.bias.double()
    q, k, v = lin(Q, m.fc_q), lin(K, m.fc_k), lin(K, m.fc_v)
    rows = []
    for b in range(Q.shape[0]):
        nq, nk = (Q.shape[1] if ql is None else ql[b]), (K.shape[1] if kl is None else kl[b])
        heads = [qh[:nq] + torch.softmax(qh[:nq] @ kh[:nk].T / np.sqrt(m.dim_V), 1) @ vh[:nk]
                 for qh, kh, vh in zip(*(t[b].split(64, 1) for t in (q, k, v)))]
        rows.append(F.pad(torch.cat(heads, 1), (0, 0, 0, Q.shape[1] - nq)))
    o = torch.stack(rows)
    return o + torch.relu(lin(o, m.fc_o))


@pytest.mark.parametrize('B,Sq,Sk,heads,ql,kl', [(2, 1100, 1100, 4, None, None), (3, 40, 300, 2, None, None),
                                                   (3, 1, 70, 1, None, [70, 3, 33]), (4, 90, 90, 4, [90, 5, 64, 1], [90, 5, 64, 1])])
def test_mab_on_large_unequal_and_padded_sets(device, B, Sq, Sk, heads, ql, kl):
    """Against float64 in value and in every gradient.  fp32 contractions of up to 64 heads + Sk terms: 1e-5 of the norm is 80
    roundings, as for the equal-shaped block's test (tests/test_gpu_linear.py); gradients go through four of them."""
    from cmvae_amd.module import MAB
    torch.manual_seed(0)
    C = 64 * heads
    m = MAB(128, 128, C, heads).to(device)
    Q = torch.randn(B, Sq, 128, device=device, requires_grad=True)
    K = Q if (Sq, ql) == (Sk, kl) else torch.randn(B, Sk, 128, device=device, requires_grad=True)
    lens = [None if x is None else torch.tensor(x, dtype=torch.int32, device=device) for x in (ql, kl)]
    keep = torch.ones(B, Sq, 1, device=device)
    for b in range(B if ql else 0):
        keep[b, ql[b]:] = 0
    go = torch.randn(B, Sq, C, device=device) * keep
    y = m(Q, K, *lens)
    leaves = [Q] + ([] if K is Q else [K]) + list(m.parameters())
    got = torch.autograd.grad(y, leaves, go)
    Q64 = Q.detach().double().requires_grad_()
    K64 = Q64 if K is Q else K.detach().double().requires_grad_()
    y64 = mab64(m, Q64, K64, ql, kl)
    want = torch.autograd.grad(y64, [Q64] + ([] if K is Q else [K64]) + list(m.parameters()), go.double())
    assert rel(y * keep, y64 * keep) < 1e-5
    names = ['Q'] + ([] if K is Q else ['K']) + [n for n, _ in m.named_parameters()]
    for n, a, b in zip(names, got, want):
        if n == 'fc_k.bias':                       # shifts every score of a row alike: zero up to rounding
            assert float(a.abs().max()) < 1e-5 * float(want[-2].abs().max())
        else:
            assert rel(a, b) < 5e-5, n


def test_padded_sets_give_what_each_set_gives_alone(device):
    from cmvae_amd.module import SAB
    torch.manual_seed(1)
    sab = SAB(64, 128, 2).to(device)
    lens = [50, 13, 1, 37]
    X = torch.randn(4, 50, 64, device=device)
    y = sab(X, torch.tensor(lens, dtype=torch.int32, device=device))
    for b, n in enumerate(lens):
        assert rel(y[b, :n], sab(X[b:b + 1, :n])[0]) < 1e-5


def test_sets_as_before_run_as_before(device):
    """Equal sets of up to 1024 rows without lengths keep their kernels: bit for bit what `linear.attention` gives."""
    from cmvae_amd import linear
    from cmvae_amd.module import MAB
    torch.manual_seed(2)
    m = MAB(64, 64, 128, 2).to(device)
    Q, K = torch.randn(2, 33, 64, device=device), torch.randn(2, 33, 64, device=device)
    o = linear.attention(m.fc_q(Q).detach() * 0 + linear.linear(Q, m.fc_q.weight, m.fc_q.bias),
                         linear.linear(K, m.fc_k.weight, m.fc_k.bias), linear.linear(K, m.fc_v.weight, m.fc_v.bias), 2,
                         1.0 / np.sqrt(128))
    assert torch.equal(m(Q, K), o + linear.linear(o, m.fc_o.weight, m.fc_o.bias, 'relu'))


class Step:
    """Channels-last features -> group norm + ELU -> one token per sample -> a set block over the episode -> a loss; AdamW."""

    def __init__(self, device, bits):
        from cmvae_amd.module import SAB
        from cmvae_amd.optim import AdamW
        torch.manual_seed(3)
        self.gamma = torch.nn.Parameter(1 + 0.1 * torch.randn(64, device=device))
        self.beta = torch.nn.Parameter(0.1 * torch.randn(64, device=device))
        self.sab = SAB(64, 128, 2).to(device)
        self.params = [self.gamma, self.beta] + list(self.sab.parameters())
        self.opt = AdamW(self.params, lr=1e-3, weight_decay=0.01, state_bits=bits).device_step()

    def loss(self, x, lens, keep):
        from cmvae_amd.norm import group_norm_act
        B, S = x.shape[:2]
        tokens = group_norm_act(x.flatten(0, 1), 8, self.gamma, self.beta, act='elu').mean(1).view(B, S, 64)
        return (self.sab(tokens, lens) * keep).square().mean()

    def __call__(self, x, lens, keep):
        self.opt.zero_grad()
        loss = self.loss(x, lens, keep)
        loss.backward()
        self.opt.step()
        return loss.detach()


def batch(device, seed=0):
    g = torch.Generator().manual_seed(seed)
    lens = torch.tensor([12, 5, 9], dtype=torch.int32)
    keep = (torch.arange(12)[None] < lens[:, None]).float()[:, :, None]
    return torch.randn(3, 12, 49, 64, generator=g).to(device), lens.to(device), keep.to(device)


@pytest.mark.parametrize('bits', [32, 8])
def test_training_step_of_all_three(device, bits):
    """Every gradient against float64, and the step against the definition on those gradients."""
    step = Step(device, bits)
    x, lens, keep = batch(device)
    g64 = [p.detach().double().requires_grad_() for p in step.params[:2]]
    z = F.group_norm(x.double().flatten(0, 1).transpose(1, 2), 8, g64[0], g64[1]).transpose(1, 2)
    tokens = F.elu(z).mean(1).view(3, 12, 64)
    loss64 = (mab64(step.sab.mab, tokens, tokens, [12, 5, 9], [12, 5, 9]) * keep.double()).square().mean()
    want = torch.autograd.grad(loss64, g64 + list(step.sab.parameters()))
    old = [p.detach().double().clone() for p in step.params]
    loss = step(x, lens, keep)
    assert abs(float(loss) - float(loss64)) < 1e-5 * float(loss64)
    for p, w, o, (n, _) in zip(step.params, want, old, [('gamma', 0), ('beta', 0)] + list(step.sab.named_parameters())):
        if n != 'mab.fc_k.bias':
            assert rel(p.grad, w) < 5e-5, n
        g = p.grad.double()                                       # the first step: m = (1 - b1) g, v = (1 - b2) g^2
        new = o * (1 - 1e-5) - 1e-3 * g / (g.abs() + 1e-8)
        assert float((p.detach().double() - new).abs().max()) < 2e-6, n


@pytest.mark.parametrize('bits', [32, 8])
def test_training_step_replayed_from_a_graph(device, bits):
    """Forward, backward and optimizer in one HIP graph against the same steps run eagerly: the same bits."""
    eager, graphed = Step(device, bits), Step(device, bits)
    x, lens, keep = batch(device)
    sx, sl, sk = x.clone(), lens.clone(), keep.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = graphed(sx, sl, sk)
    for seed in range(4):
        x, lens, keep = batch(device, seed)
        sx.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        want = eager(x, lens, keep)
        assert torch.equal(out, want)
        assert all(torch.equal(a, b) for a, b in zip(eager.params, graphed.params))
        assert torch.equal(eager.opt.exp_avg_sq, graphed.opt.exp_avg_sq)


def test_two_graphs_of_one_operator_replay_beside_each_other(device):
    """Two captured calls with workspaces (one query cut into pieces, pieces of group-norm sums), replayed at once on two
    streams: each graph owns its scratch."""
    from cmvae_amd.attention import set_attention
    from cmvae_amd.norm import group_norm_act
    g = torch.Generator().manual_seed(0)
    ins = [[torch.randn(2, n, 4, 64, generator=g).to(device) for n in (1, 5000, 5000)] + [torch.randn(2, 20000, 32, generator=g).to(device)]
           for _ in range(2)]
    f = lambda q, k, v, x: (set_attention(q, k, v), group_norm_act(x, 4, act='silu'))  # noqa: E731
    want = [f(*i) for i in ins]
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in range(2)]
    for i in ins:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(f(*i))
    torch.cuda.synchronize()
    for _ in range(20):
        for gr, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                gr.replay()
    torch.cuda.synchronize()
    for a, b in zip(outs, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_second_derivatives_say_so(device):
    """create_graph works as long as the gradient is not differentiated again; that is refused, not silently zero."""
    from cmvae_amd.attention import set_attention
    from cmvae_amd.norm import group_norm_act
    q = torch.randn(1, 4, 1, 64, device=device, requires_grad=True)
    x = torch.randn(2, 3, 8, device=device, requires_grad=True)
    for leaf, y in ((q, set_attention(q, q, q)), (x, group_norm_act(x, 2))):
        (g,) = torch.autograd.grad(y.square().sum(), leaf, create_graph=True)
        with pytest.raises(RuntimeError, match='differentiable once'):
            torch.autograd.grad(g.square().sum(), leaf)


@pytest.mark.parametrize('optimizer', ['adamw', 'adamw8'])
@pytest.mark.parametrize('variant', ['omniglot', 'mimgnet'])
def test_trainer_with_adamw(tmp_path, variant, optimizer):
    """--optimizer: the loop runs (mimgnet: its step replayed from a graph), checkpoints carry the states, a resumed trainer
    has them."""
    from cmvae_amd.optim import AdamW
    from cmvae_amd.trainer import Trainer
    from tests.test_gpu_trainer import _args, _make
    extra = () if variant == 'omniglot' else ('--per-class', '60', '--dim', '256')
    d = _make(tmp_path, variant, *extra)
    np.random.seed(10086)
    torch.manual_seed(10086)
    kw = {} if variant == 'omniglot' else dict(sample_size=5, batch_size=4, instances_per_class=60, train_iters=6, freq_iters=6)
    tr = Trainer(_args(d, str(tmp_path / 'run'), optimizer=optimizer, **kw), variant)
    w0 = [p.detach().clone() for p in tr.model.parameters()]
    first = tr.optimizer
    tr.train()
    assert isinstance(first, AdamW) and first.state_bits == (8 if optimizer == 'adamw8' else 32)
    assert any(not torch.equal(a, b) for a, b in zip(w0, first.params)) and all(torch.isfinite(p).all() for p in first.params)
    path = next(iter(tr.best_files.values()))
    tr2 = Trainer(_args(d, str(tmp_path / 'run2'), optimizer=optimizer, **kw), variant)
    state = tr2.load_checkpoint(path, resume_optimizer=True)
    assert tr2.optimizer.state_dict()['step'] == state['optimizer']['step'] > 0
    assert torch.equal(tr2.optimizer.exp_avg_sq, state['optimizer']['exp_avg_sq'])


def test_command_line_flag(tmp_path):
    from cmvae_amd.main import build_parser
    p = build_parser('omniglot')
    base = ['--data-dir', 'd', '--save-dir', 's']
    assert p.parse_args(base).optimizer == 'adam' and p.parse_args(base + ['--optimizer', 'adamw8']).optimizer == 'adamw8'
    assert subprocess.run([sys.executable, '-m', 'cmvae_amd.main', 'omniglot', *base, '--optimizer', 'sgd'], cwd=ROOT,
                          capture_output=True).returncode != 0


def second_derivative_cases(device):
    """name -> (leaf, call, what the gradient is asked from): inputs that are copied or viewed on the way in, with a gradient of y
    that is a constant and nothing else that wants one."""
    from cmvae_amd.attention import set_attention
    from cmvae_amd.norm import group_norm_act
    leaf = lambda *s: torch.randn(*s, device=device, requires_grad=True)  # noqa: E731
    nchw, image, pixel, flat = leaf(2, 8, 3, 3), leaf(2, 3, 3, 8), leaf(5, 8), leaf(2 * 4 * 2 * 64 + 1)
    tall, thin = leaf(2, 6, 3, 8), leaf(2, 3, 3, 8)
    wide, frozen, scale = leaf(2, 4, 2, 128), torch.ones(8, device=device), leaf(16)
    q, k, v = torch.randn(3, 2, 4, 2, 64, device=device)
    row = flat[1:].view(2, 4, 2, 64)                            # rows that do not start at multiples of 16 bytes
    col = wide[..., ::2]                                        # channels that are not adjacent
    x = torch.randn(2, 3, 3, 8, device=device)
    return {
        'channels first': (nchw, lambda: group_norm_act(nchw.permute(0, 2, 3, 1), 2)),
        'channels first, frozen parameters': (nchw, lambda: group_norm_act(nchw.permute(0, 2, 3, 1), 2, frozen, frozen, act='silu')),
        'an image': (image, lambda: group_norm_act(image, 2, act='elu')),
        'one pixel': (pixel, lambda: group_norm_act(pixel, 2)),
        'every other image row': (tall, lambda: group_norm_act(tall[:, ::2], 2)),
        'one channel': (thin, lambda: group_norm_act(thin[..., :1], 1, act='silu')),
        'strided parameters': (scale, lambda: group_norm_act(x, 2, scale[::2], act='silu')),
        'misaligned q': (flat, lambda: set_attention(row, k, v)),
        'misaligned k': (flat, lambda: set_attention(q, row, v)),
        'strided v': (wide, lambda: set_attention(q, k, col)),
        'all copied': (wide, lambda: set_attention(col, col, col)),
    }


@pytest.mark.parametrize('name', ['channels first', 'channels first, frozen parameters', 'an image', 'one pixel',
                                  'every other image row', 'one channel', 'strided parameters', 'misaligned q', 'misaligned k', 'strided v', 'all copied'])
def test_second_derivatives_of_copied_inputs_say_so(device, name):
    """The same where the kernels read a copy or a view of the input and dO is a constant: without its refusal a penalty on the gradient
    would be dropped.  A gradient under create_graph that is not differentiated is the plain one."""
    leaf, call = second_derivative_cases(device)[name]
    d = torch.randn_like(call())
    (plain,) = torch.autograd.grad(call(), leaf, d)
    (g,) = torch.autograd.grad(call(), leaf, d, create_graph=True)
    assert g.requires_grad and torch.equal(g, plain)
    with pytest.raises(RuntimeError, match='differentiable once'):
        g.square().sum().backward(retain_graph=True)
    with pytest.raises(RuntimeError, match='differentiable once'):
        torch.autograd.grad(g.square().sum(), leaf, allow_unused=True)
