"""Set attention for any set sizes, on the HIP library (cmvae_amd/csrc/set_attention.hip).

`set_attention(q, k, v)` is the softmax core of MAB (omniglot/module.py:92-99) beyond the shapes of `linear.attention`:
unequal and large sets, padded batches, shared key heads, causal order, 16-bit types.  Its backward pass recomputes the
probabilities from the saved log-sum-exp, so nothing of size queries x keys is ever stored.
"""
import ctypes
import math

import torch

from . import ops
from ._lib import lib, check, SetAttnDesc

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_p = ops._p


def _rows16(t):
    """t with adjacent channels and rows that start at multiples of 16 bytes (a copy if it has not)."""
    per = 16 // t.element_size()
    if t.stride(3) != 1 or t.data_ptr() % 16 or any(s % per for s in t.stride()[:3]):
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


def _desc(q, k, v, scale, causal, q_len, k_len, residual):
    d = SetAttnDesc()
    d.dtype = DTYPES[q.dtype]
    d.B, d.Sq, d.H, d.D = q.shape
    d.Sk, d.Hkv = k.shape[1:3]
    d.causal, d.residual, d.scale = int(causal), int(residual), scale
    d.q, d.k, d.v, d.q_len, d.k_len = _p(q), _p(k), _p(v), _p(q_len), _p(k_len)
    d.q_stride[:], d.k_stride[:], d.v_stride[:] = q.stride()[:3], k.stride()[:3], v.stride()[:3]
    return d


def _workspace(d, backward, device):
    # from the caching allocator, per call: a captured graph owns its own
    n = lib.cmvae_set_attention_workspace_bytes(ctypes.byref(d), backward)
    return (torch.empty(n, dtype=torch.uint8, device=device) if n else None), n


def set_attention_fwd(q, k, v, scale, causal, q_len, k_len, residual, save):
    """(o, attn, lse) of one call; attn and lse are None unless `save` (attn: o without the residual)."""
    B, Sq, H, D = q.shape
    o = torch.empty(B, Sq, H, D, device=q.device, dtype=q.dtype)
    attn = (torch.empty_like(o) if residual else o) if save else None
    lse = torch.empty(B, H, Sq, device=q.device, dtype=torch.float32) if save else None
    if o.numel() == 0:
        return o, attn, lse
    d = _desc(q, k, v, scale, causal, q_len, k_len, residual)
    d.o, d.attn, d.lse = _p(o), (_p(attn) if residual else None), _p(lse)
    with torch.cuda.device(q.device):
        ws, n = _workspace(d, 0, q.device)
        check(lib.cmvae_set_attention_fwd(ctypes.byref(d), _p(ws), n, ops._stream()), 'cmvae_set_attention_fwd')
    return o, attn, lse


def set_attention_bwd(q, k, v, attn, lse, do, scale, causal, q_len, k_len, residual):
    """(dq, dk, dv) from the tensors `set_attention_fwd` was given and saved."""
    B, Sq, H, D = q.shape
    dq = torch.empty(B, Sq, H, D, device=q.device, dtype=q.dtype)
    dk, dv = (torch.empty(k.shape, device=q.device, dtype=q.dtype) for _ in range(2))
    if dq.numel() == 0:
        return dq, dk.zero_(), dv.zero_()
    delta = torch.empty_like(lse)
    d = _desc(q, k, v, scale, causal, q_len, k_len, residual)
    do = _rows16(do)
    d.dO, d.dO_stride[:] = _p(do), do.stride()[:3]
    d.o = d.attn = _p(attn)
    d.lse, d.delta, d.dq, d.dk, d.dv = _p(lse), _p(delta), _p(dq), _p(dk), _p(dv)
    with torch.cuda.device(q.device):
        ws, n = _workspace(d, 1, q.device)
        check(lib.cmvae_set_attention_bwd(ctypes.byref(d), _p(ws), n, ops._stream()), 'cmvae_set_attention_bwd')
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
