"""AdamW over many tensors at once, on the HIP library (cmvae_amd/csrc/optim.hip).

`linear.FlatAdam` is the reference's optimizer (L2 added to the gradient, one flat fp32 buffer; omniglot/trainer.py:48-52);
`AdamW` decouples the weight decay, takes the parameters where they are (float32, bfloat16, float16) and holds its two
moments in 32 bits or in 8 (1.02 bytes per value and moment, scales included).
"""
import torch

from . import _lib  # noqa: F401  (loads the operators)

BLOCK = 256                    # values that share a scale; every tensor's states start at a multiple of it
_adamw_step = torch.ops.cmvae_amd.adamw_step.default
_adamw_state_values = torch.ops.cmvae_amd.adamw_state_values.default


def state_size(n):
    """State values a tensor of n values takes."""
    return (n + BLOCK - 1) // BLOCK * BLOCK


def adamw_step(params, grads, exp_avg, exp_avg_sq, scales=None, step=1, lr=1e-3, betas=(0.9, 0.999), eps=1e-8,
               weight_decay=1e-2):
    """One AdamW step, in place, over the tensors `params` with gradients `grads` (None: the tensor and its states are left
    as they are).

    params: dense float32 / bfloat16 / float16 tensors that overlap neither each other nor the states nor what is read: other
    tensors' gradients, `step` (types may be mixed; a gradient has its parameter's).
    exp_avg, exp_avg_sq: the flat states of all tensors in order, each padded to a multiple of 256 values in the order of
    its parameter's memory (`state_size`); float32, or float8_e4m3fn and uint8 with `scales` [2, length / 256].
    step: 1, 2, ...; or an int64 tensor of one value on the device (for a step replayed from a HIP graph).

    Of 8-bit states: 256 values share a scale per moment; exp_avg is e4m3 of m / scale, exp_avg_sq holds 5 exponent and 3
    mantissa bits of v / scale (0 is zero, 255 not finite, read as infinity), both to nearest even, a positive v never as 0.  The update uses
    the moments before that rounding."""
    step_dev = None
    if isinstance(step, torch.Tensor):
        step, step_dev = 0, step
    _adamw_step(params, grads, exp_avg, exp_avg_sq, scales, step, step_dev, lr, betas[0], betas[1], eps, weight_decay)


def adamw_state_values(exp_avg, exp_avg_sq, scales):
    """(m, v): the float32 values that 8-bit states stand for."""
    return _adamw_state_values(exp_avg, exp_avg_sq, scales)


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
        adamw_step(self.params, grads, self.exp_avg, self.exp_avg_sq, self.scales,
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
