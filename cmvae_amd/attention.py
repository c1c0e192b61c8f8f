"""Set attention for any set sizes, on the HIP library (cmvae_amd/csrc/set_attention.hip).

`set_attention(q, k, v)` is the softmax core of MAB (omniglot/module.py:92-99) beyond the shapes of `linear.attention`:
unequal and large sets, padded batches, shared key heads, causal order, 16-bit types.  Its backward pass recomputes the
probabilities from the saved log-sum-exp, so nothing of size queries x keys is ever stored.
"""
import ctypes
import math

import torch

from . import ops
from ._lib import lib, SetAttnDesc

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_p = ops._p


def _rows16(t):
    """t with adjacent channels and rows that start at multiples of 16 bytes (a copy if it has not)."""
    b, r, h, c = t.stride()
    if c != 1 or t.data_ptr() % 16 or (b | r | h) % (16 // t.element_size()):
        return t.clone(memory_format=torch.contiguous_format)
    return t


def _check(q, k, v, scale, q_len, k_len):
    for t, n in ((q, 'q'), (k, 'k'), (v, 'v')):
        if not isinstance(t, torch.Tensor) or not t.is_cuda:
            raise RuntimeError('cmvae_amd set_attention: %s must be a GPU tensor (there is no CPU path)' % n)
        if t.dtype not in DTYPES or t.dtype != q.dtype or t.device != q.device:
            raise RuntimeError('cmvae_amd set_attention: q, k, v must share one device and one of float32, bfloat16, '
                               'float16; %s is %s on %s' % (n, t.dtype, t.device))
        if t.dim() != 4:
            raise RuntimeError('cmvae_amd set_attention: %s must be [batch, rows, heads, channels], got %s'
                               % (n, tuple(t.shape)))
    B, Sq, H, D = q.shape
    if k.shape != v.shape or k.shape[0] != B or k.shape[3] != D or k.shape[2] < 1 or H < 1 or H % k.shape[2]:
        raise RuntimeError('cmvae_amd set_attention: q %s, k %s and v %s do not fit (equal batch and channels, k and v '
                           'alike, query heads a multiple of key heads)' % (tuple(q.shape), tuple(k.shape), tuple(v.shape)))
    if D not in (64, 128):
        raise RuntimeError('cmvae_amd set_attention: heads of 64 or 128 channels are supported, got %d' % D)
    if not 1e-30 <= scale <= 1e30:
        raise RuntimeError('cmvae_amd set_attention: scale must be a positive finite number, got %r' % scale)
    for t, n, S in ((q_len, 'q_len', Sq), (k_len, 'k_len', k.shape[1])):
        if t is None:
            continue
        if not isinstance(t, torch.Tensor) or t.device != q.device or t.dtype != torch.int32 or tuple(t.shape) != (B,):
            raise RuntimeError('cmvae_amd set_attention: %s must be an int32 tensor of shape [%d] beside q' % (n, B))
        if ops.CHECK_INDICES:
            ops.check_index_range(t, S + 1, n)


def _desc(q, k, v, scale, causal, q_len, k_len, residual, do=None):
    B, Sq, H, D = q.shape
    return SetAttnDesc(DTYPES[q.dtype], B, Sq, k.shape[1], H, k.shape[2], D, causal, residual, scale, q.data_ptr(),
                       k.data_ptr(), v.data_ptr(), _p(do), q.stride()[:3], k.stride()[:3], v.stride()[:3],
                       do.stride()[:3] if do is not None else (0, 0, 0), _p(q_len), _p(k_len))


def _workspace(d, backward, device):
    # from the caching allocator, per call: a captured graph owns its own
    n = lib.cmvae_set_attention_workspace_bytes(ctypes.byref(d), backward)
    ws = torch.empty(n, dtype=torch.uint8, device=device) if n else None
    return ws, n


def set_attention_fwd(q, k, v, scale, causal, q_len, k_len, residual, save):
    """(o, attn, lse) of one call; attn and lse are None unless `save` (attn: o without the residual)."""
    B, Sq, H, D = q.shape
    dev = q.device
    o = torch.empty((B, Sq, H, D), device=dev, dtype=q.dtype)
    attn = (torch.empty_like(o) if residual else o) if save else None
    lse = torch.empty((B, H, Sq), device=dev, dtype=torch.float32) if save else None
    if o.numel() == 0:
        return o, attn, lse
    d = _desc(q, k, v, scale, causal, q_len, k_len, residual)
    d.o, d.attn, d.lse = o.data_ptr(), (_p(attn) if residual else None), _p(lse)
    ws, n = _workspace(d, 0, dev)
    ops._call('cmvae_set_attention_fwd', lib.cmvae_set_attention_fwd, dev, ctypes.byref(d), _p(ws), n)
    return o, attn, lse


def set_attention_bwd(q, k, v, attn, lse, do, scale, causal, q_len, k_len, residual):
    """(dq, dk, dv) from the tensors `set_attention_fwd` was given and saved."""
    dev = q.device
    dq = torch.empty(q.shape, device=dev, dtype=q.dtype)
    dk = torch.empty(k.shape, device=dev, dtype=q.dtype)
    dv = torch.empty(k.shape, device=dev, dtype=q.dtype)
    if dq.numel() == 0:
        return dq, dk.zero_(), dv.zero_()
    delta = torch.empty_like(lse)
    do = _rows16(do)
    d = _desc(q, k, v, scale, causal, q_len, k_len, residual, do)
    d.o = d.attn = attn.data_ptr()
    d.lse, d.delta, d.dq, d.dk, d.dv = lse.data_ptr(), delta.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr()
    ws, n = _workspace(d, 1, dev)
    ops._call('cmvae_set_attention_bwd', lib.cmvae_set_attention_bwd, dev, ctypes.byref(d), _p(ws), n)
    return dq, dk, dv


class _SetAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, scale, causal, q_len, k_len, residual):
        q, k, v = _rows16(q), _rows16(k), _rows16(v)
        save = any(ctx.needs_input_grad[:3])
        o, attn, lse = set_attention_fwd(q, k, v, scale, causal, q_len, k_len, residual, save)
        ctx.args = (scale, causal, residual)
        if save:
            ctx.save_for_backward(q, k, v, attn, lse, q_len, k_len)
        return o

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, do):
        q, k, v, attn, lse, q_len, k_len = ctx.saved_tensors
        scale, causal, residual = ctx.args
        dq, dk, dv = set_attention_bwd(q, k, v, attn, lse, do, scale, causal, q_len, k_len, residual)
        return dq, dk, dv, None, None, None, None, None


def set_attention(q, k, v, scale=None, causal=False, q_len=None, k_len=None, residual=False):
    """softmax(scale * q k^T) v (+ q if `residual`) per (batch, head).

    q [B, Sq, H, D], k and v [B, Sk, Hkv, D]: float32, bfloat16 or float16, D 64 or 128, any strides (copied where
    channels are not adjacent or rows not 16-byte aligned); H a multiple of Hkv, query head h reads key head
    h // (H // Hkv).  scale: 1 / sqrt(D) by default.  q_len, k_len: int32 [B], the rows of each batch entry that count
    (padded batches; values are clamped to [0, S]); output rows behind q_len and all gradients of rows behind a length
    are zeros, and what such rows hold is never read.  causal: query i sees keys j <= i + k_len - q_len.  A query that
    sees no key gets zeros (plus its own row if `residual`).  Differentiable once in q, k, v; every result is the same
    bits on every run."""
    scale = 1.0 / math.sqrt(q.shape[-1]) if scale is None else float(scale)
    _check(q, k, v, scale, q_len, k_len)
    return _SetAttention.apply(q, k, v, scale, bool(causal), q_len, k_len, bool(residual))
