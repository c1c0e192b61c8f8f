"""AdamW over many tensors at once, on the HIP library (cmvae_amd/csrc/optim.hip).

`linear.FlatAdam` is the reference's optimizer (L2 added to the gradient, one flat fp32 buffer; omniglot/trainer.py:48-52);
`AdamW` decouples the weight decay, takes the parameters where they are (float32, bfloat16, float16) and holds its two
moments in 32 bits or in 8 (1.03 bytes per value and moment, scales included).
"""
import ctypes

import torch

from . import ops
from ._lib import lib
from .attention import DTYPES

BLOCK = 256                    # values that share a scale; every tensor's states start at a multiple of it
_p = ops._p


def state_size(n):
    """State values a tensor of n values takes."""
    return (n + BLOCK - 1) // BLOCK * BLOCK


def _states(exp_avg, exp_avg_sq, scales):
    """Checked states; returns (bits, length, device)."""
    for t, n in ((exp_avg, 'exp_avg'), (exp_avg_sq, 'exp_avg_sq')):
        if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dim() != 1 or not t.is_contiguous():
            raise RuntimeError('cmvae_amd adamw: %s must be a flat GPU tensor (there is no CPU path)' % n)
    n, dev = exp_avg.numel(), exp_avg.device
    if exp_avg_sq.numel() != n or exp_avg_sq.device != dev or n % BLOCK:
        raise RuntimeError('cmvae_amd adamw: exp_avg and exp_avg_sq must have one length, a multiple of %d, and one device'
                           % BLOCK)
    if scales is None:
        if exp_avg.dtype != torch.float32 or exp_avg_sq.dtype != torch.float32:
            raise RuntimeError('cmvae_amd adamw: states without scales must be float32')
        return 32, n, dev
    if exp_avg.dtype != torch.float8_e4m3fn or exp_avg_sq.dtype != torch.uint8:
        raise RuntimeError('cmvae_amd adamw: 8-bit states are float8_e4m3fn (exp_avg) and uint8 (exp_avg_sq)')
    if not isinstance(scales, torch.Tensor) or scales.device != dev or scales.dtype != torch.float32 or \
            tuple(scales.shape) != (2, n // BLOCK) or not scales.is_contiguous():
        raise RuntimeError('cmvae_amd adamw: scales must be a float32 tensor [2, %d] beside the states' % (n // BLOCK))
    return 8, n, dev


def adamw_step(params, grads, exp_avg, exp_avg_sq, scales=None, step=1, lr=1e-3, betas=(0.9, 0.999), eps=1e-8,
               weight_decay=1e-2):
    """One AdamW step, in place, over the tensors `params` with gradients `grads` (None: the tensor and its states are left
    as they are).

    params: dense float32 / bfloat16 / float16 tensors (types may be mixed; a gradient has its parameter's).
    exp_avg, exp_avg_sq: the flat states of all tensors in order, each padded to a multiple of 256 values in the order of
    its parameter's memory (`state_size`); float32, or float8_e4m3fn and uint8 with `scales` [2, length / 256].
    step: 1, 2, ...; or an int64 tensor of one value on the device (for a step replayed from a HIP graph).

    Of 8-bit states: 256 values share a scale per moment; exp_avg is e4m3 of m / scale, exp_avg_sq holds 5 exponent and 3
    mantissa bits of v / scale (0 is zero, 255 not finite, read as infinity), both to nearest even, a positive v never as 0.  The update uses
    the moments before that rounding."""
    bits, length, dev = _states(exp_avg, exp_avg_sq, scales)
    params, grads = list(params), list(grads)
    if len(params) != len(grads):
        raise RuntimeError('cmvae_amd adamw: %d parameters and %d gradients' % (len(params), len(grads)))
    flat, at, done, keep = [], 0, [], []
    for p, g in zip(params, grads):
        n = p.numel()
        here, at = at, at + (n + BLOCK - 1) // BLOCK * BLOCK
        if g is None:
            continue
        dt, st = p.dtype, p.stride()
        if dt not in DTYPES or g.dtype is not dt or p.device != dev or g.device != dev or g.shape != p.shape:
            raise RuntimeError('cmvae_amd adamw: a parameter %s %s on %s with a gradient %s %s on %s (float32, bfloat16 or '
                               'float16, alike, on the states\' device)' % (p.dtype, tuple(p.shape), p.device, g.dtype,
                                                                            tuple(g.shape), g.device))
        if not p.is_contiguous() and not (p.dim() == 4 and p.is_contiguous(memory_format=torch.channels_last)):
            raise RuntimeError('cmvae_amd adamw: a parameter of shape %s has strides %s: it must be dense'
                               % (tuple(p.shape), st))
        if g.stride() != st:
            g = torch.empty_like(p).copy_(g)
            keep.append(g)
        if n:
            done.append(p)
            flat += (p.data_ptr(), g.data_ptr(), n, here, DTYPES[dt])
    if len(set(flat[::5])) != len(done):
        raise RuntimeError('cmvae_amd adamw: a parameter appears twice')
    if at != length:
        raise RuntimeError('cmvae_amd adamw: the parameters take %d state values, the states hold %d' % (at, length))
    step_dev = None
    if isinstance(step, torch.Tensor):
        if step.device != dev or step.dtype != torch.int64 or step.numel() != 1:
            raise RuntimeError('cmvae_amd adamw: step must be a number or an int64 tensor of one value beside the states')
        step, step_dev = 0, step
    if not done:
        return
    ops._call('cmvae_adamw_step', lib.cmvae_adamw_step, dev, (ctypes.c_int64 * len(flat))(*flat), len(done), bits,
              exp_avg.data_ptr(), exp_avg_sq.data_ptr(), _p(scales), length, int(step), _p(step_dev), lr, betas[0], betas[1],
              eps, weight_decay)
    torch.autograd.graph.increment_version(done)


def adamw_state_values(exp_avg, exp_avg_sq, scales):
    """(m, v): the float32 values that 8-bit states stand for."""
    bits, n, dev = _states(exp_avg, exp_avg_sq, scales)
    if bits == 32:
        raise RuntimeError('cmvae_amd adamw: states in 32 bits are their values')
    m, v = (torch.empty(n, device=dev, dtype=torch.float32) for _ in range(2))
    ops._call('cmvae_adamw_state_values', lib.cmvae_adamw_state_values, dev, _p(exp_avg), _p(exp_avg_sq), _p(scales), n, _p(m),
              _p(v))
    return m, v


class AdamW:
    """AdamW over `params` (tensors, whose `.grad` is read; or a `dist.FlatGrads`, whose exchanged gradients are), with
    the interface of `linear.FlatAdam`; state_bits 32 or 8."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits=32):
        self.flat_grads = params if hasattr(params, 'views') else None
        self.params = list(params.params if self.flat_grads is not None else params)
        if not self.params or any(not p.is_cuda for p in self.params):
            raise RuntimeError('cmvae_amd AdamW: parameters must live on the GPU (there is no CPU path)')
        if state_bits not in (8, 32):
            raise RuntimeError('cmvae_amd AdamW: states of 8 or 32 bits, not %r' % (state_bits,))
        self.lr, self.betas, self.eps, self.weight_decay, self.state_bits = lr, betas, eps, weight_decay, state_bits
        n = sum(state_size(p.numel()) for p in self.params)
        dev = self.params[0].device
        if state_bits == 32:
            self.exp_avg, self.exp_avg_sq = (torch.zeros(n, device=dev) for _ in range(2))
            self.scales = None
        else:
            self.exp_avg = torch.zeros(n, device=dev, dtype=torch.uint8).view(torch.float8_e4m3fn)
            self.exp_avg_sq = torch.zeros(n, device=dev, dtype=torch.uint8)
            self.scales = torch.zeros(2, n // BLOCK, device=dev)
        self.t = 0
        self.step_dev = None

    def device_step(self):
        """Keep the step count on the device from now on (see `FlatAdam.device_step`); idempotent."""
        if self.step_dev is None:
            self.step_dev = torch.full((1,), self.t, dtype=torch.int64, device=self.exp_avg.device)
        return self

    @torch.no_grad()
    def step(self):
        if self.step_dev is not None:
            self.step_dev += 1
        else:
            self.t += 1
        grads = self.flat_grads.views if self.flat_grads is not None else [p.grad for p in self.params]
        adamw_step([p.detach() for p in self.params], grads, self.exp_avg, self.exp_avg_sq, self.scales,
                   step=self.t if self.step_dev is None else self.step_dev, lr=self.lr, betas=self.betas, eps=self.eps,
                   weight_decay=self.weight_decay)

    def zero_grad(self):
        if self.flat_grads is not None:
            self.flat_grads.zero()
        else:
            for p in self.params:
                p.grad = None

    def state_dict(self):
        t = self.t if self.step_dev is None else int(self.step_dev)
        sd = {'step': t, 'exp_avg': self.exp_avg, 'exp_avg_sq': self.exp_avg_sq}
        if self.scales is not None:
            sd['scales'] = self.scales
        return sd

    def load_state_dict(self, sd):
        if sd['exp_avg'].dtype != self.exp_avg.dtype or sd['exp_avg'].shape != self.exp_avg.shape or \
                ('scales' in sd) != (self.scales is not None):
            raise RuntimeError('cmvae_amd AdamW: the saved states are %s %s, this optimizer\'s %s %s' % (
                sd['exp_avg'].dtype, tuple(sd['exp_avg'].shape), self.exp_avg.dtype, tuple(self.exp_avg.shape)))
        self.t = int(sd['step'])
        if self.step_dev is not None:
            self.step_dev.fill_(self.t)
        self.exp_avg.copy_(sd['exp_avg'])
        self.exp_avg_sq.copy_(sd['exp_avg_sq'])
        if self.scales is not None:
            self.scales.copy_(sd['scales'])
