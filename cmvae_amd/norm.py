"""Group norm with an activation on channels-last data, on the HIP library (cmvae_amd/csrc/group_norm.hip).

The BatchNorm of the encoder and decoder (omniglot/module.py:15-31, 51-59) takes its statistics over the whole meta-batch,
an exchange between ranks per layer and step; group norm's belong to one sample and need none.
"""
import ctypes
import math

import torch

from . import ops
from ._lib import lib, GroupNormDesc
from .attention import DTYPES

ACT = {None: 0, 'none': 0, 'relu': 1, 'elu': 2, 'silu': 3}
_p = ops._p


def _rows(x):
    """[N, ..., C] -> [N, P, C] with adjacent channels (a copy where strides do not allow it)."""
    if x.dim() != 3:
        x = x.reshape(x.shape[0], math.prod(x.shape[1:-1]), x.shape[-1])
    return x if x.stride(2) == 1 else x.contiguous()


def _check(x, groups, weight, bias, eps, act):
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise RuntimeError('cmvae_amd group_norm_act: x must be a GPU tensor (there is no CPU path)')
    if x.dtype not in DTYPES or x.dim() < 2:
        raise RuntimeError('cmvae_amd group_norm_act: x must be a float32, bfloat16 or float16 tensor [N, ..., C], got %s %s'
                           % (x.dtype, tuple(x.shape)))
    C = x.shape[-1]
    if not isinstance(groups, int) or groups < 1 or C < 1 or C % groups:
        raise RuntimeError('cmvae_amd group_norm_act: %r groups of %d channels' % (groups, C))
    if act not in ACT:
        raise RuntimeError('cmvae_amd group_norm_act: act must be one of %s, got %r' % (sorted(k for k in ACT if k), act))
    if not 0 <= eps < math.inf:
        raise RuntimeError('cmvae_amd group_norm_act: eps must be finite and not negative, got %r' % eps)
    for t, n in ((weight, 'weight'), (bias, 'bias')):
        if t is None:
            continue
        if not isinstance(t, torch.Tensor) or t.device != x.device or tuple(t.shape) != (C,) or \
                t.dtype not in (torch.float32, x.dtype):
            raise RuntimeError('cmvae_amd group_norm_act: %s must be a [%d] tensor beside x, of float32 or its type' % (n, C))
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise RuntimeError('cmvae_amd group_norm_act: weight is %s, bias %s' % (weight.dtype, bias.dtype))


def _strides(x3):
    n, p, _ = x3.stride()
    return n if x3.shape[0] > 1 else 0, p if x3.shape[1] > 1 else 0


def _desc(x3, groups, weight, bias, eps, act, dy3=None):
    ref = weight if weight is not None else bias
    return GroupNormDesc(DTYPES[x3.dtype], DTYPES[ref.dtype] if ref is not None else 0, act, *x3.shape, groups, eps,
                         x3.data_ptr(), _p(weight), _p(bias), _p(dy3), _strides(x3),
                         _strides(dy3) if dy3 is not None else (0, 0))


def _run(name, fn, d, backward, device):
    n = lib.cmvae_group_norm_workspace_bytes(ctypes.byref(d), backward)
    ws = torch.empty(n, dtype=torch.uint8, device=device) if n else None
    ops._call(name, fn, device, ctypes.byref(d), _p(ws), n)


def group_norm_fwd(x3, groups, weight, bias, eps, act, save):
    """(y [N, P, C], stats [N, groups, 4] or None); stats: mean in two parts, 1 / deviation."""
    dev = x3.device
    y = torch.empty(x3.shape, device=dev, dtype=x3.dtype)
    stats = torch.empty((x3.shape[0], groups, 4), device=dev, dtype=torch.float32) if save else None
    if y.numel():
        d = _desc(x3, groups, weight, bias, eps, act)
        d.y, d.stats = y.data_ptr(), _p(stats)
        _run('cmvae_group_norm_fwd', lib.cmvae_group_norm_fwd, d, 0, dev)
    return y, stats


def group_norm_bwd(x3, dy3, groups, weight, bias, stats, eps, act, need_params):
    """(dx, dweight, dbias) of one `group_norm_fwd` that saved its stats."""
    dev = x3.device
    dx = torch.empty(x3.shape, device=dev, dtype=x3.dtype)
    dw = torch.empty_like(weight) if weight is not None and need_params else None
    db = torch.empty_like(bias) if bias is not None and need_params else None
    if dx.numel() == 0:
        return dx, (None if dw is None else dw.zero_()), (None if db is None else db.zero_())
    d = _desc(x3, groups, weight, bias, eps, act, dy3)
    d.stats, d.dx, d.dweight, d.dbias = stats.data_ptr(), dx.data_ptr(), _p(dw), _p(db)
    _run('cmvae_group_norm_bwd', lib.cmvae_group_norm_bwd, d, 1, dev)
    return dx, dw, db


class _GroupNormAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, groups, weight, bias, eps, act):
        x3 = _rows(x)
        weight = None if weight is None else weight.contiguous()
        bias = None if bias is None else bias.contiguous()
        save = any(ctx.needs_input_grad)
        y, stats = group_norm_fwd(x3, groups, weight, bias, eps, act, save)
        if save:
            ctx.args = (groups, eps, act, x.shape)
            ctx.save_for_backward(x3, weight, bias, stats)
        return y if x.dim() == 3 else y.view(x.shape)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x3, weight, bias, stats = ctx.saved_tensors
        groups, eps, act, shape = ctx.args
        dx, dw, db = group_norm_bwd(x3, _rows(dy), groups, weight, bias, stats, eps, act,
                                    ctx.needs_input_grad[2] or ctx.needs_input_grad[3])
        return dx if len(shape) == 3 else dx.view(shape), None, dw, db, None, None


def group_norm_act(x, groups, weight=None, bias=None, eps=1e-5, act=None):
    """act(group_norm(x) * weight + bias) for channels-last x [N, ..., C] (float32, bfloat16, float16).

    Each sample's C channels form `groups` groups of neighbours; mean and biased variance are those of a group's channels
    over all of the sample's pixels.  weight, bias: [C] of float32 or x's type, or None.  act: None, 'relu', 'elu' or
    'silu'.  x may be a view with other sample and pixel strides; the result is dense.  Differentiable once in x, weight
    and bias (relu's slope at 0 is 0); every result is the same bits on every run."""
    _check(x, groups, weight, bias, eps, act)
    return _GroupNormAct.apply(x, groups, weight, bias, float(eps), ACT[act])
