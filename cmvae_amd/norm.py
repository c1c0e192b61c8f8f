"""Group norm with an activation on channels-last data, on the HIP library (cmvae_amd/csrc/group_norm.hip).

The BatchNorm of the encoder and decoder (omniglot/module.py:15-31, 51-59) takes its statistics over the whole meta-batch,
an exchange between ranks per layer and step; group norm's belong to one sample and need none.
"""
import torch

from . import _lib  # noqa: F401  (loads the operators)

ACT = {None: 0, 'none': 0, 'relu': 1, 'elu': 2, 'silu': 3}
_group_norm_act = torch.ops.cmvae_amd.group_norm_act.default


def group_norm_act(x, groups, weight=None, bias=None, eps=1e-5, act=None):
    """act(group_norm(x) * weight + bias) for channels-last x [N, ..., C] (float32, bfloat16, float16).

    Each sample's C channels form `groups` groups of neighbours; mean and biased variance are those of a group's channels
    over all of the sample's pixels.  weight, bias: [C] of float32 or x's type, or None.  act: None, 'relu', 'elu' or
    'silu'.  x may be a view with other sample and pixel strides; the result is dense.  Differentiable once in x, weight
    and bias (relu's slope at 0 is 0); every result is the same bits on every run."""
    if act not in ACT:
        raise RuntimeError('cmvae_amd group_norm_act: act must be one of %s, got %r' % (sorted(k for k in ACT if k), act))
    return _group_norm_act(x, groups, weight, bias, eps, ACT[act])
