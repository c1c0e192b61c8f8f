"""Set attention for any set sizes, on the HIP library (cmvae_amd/csrc/set_attention.hip).

`set_attention(q, k, v)` is the softmax core of MAB (omniglot/module.py:92-99) beyond the shapes of `linear.attention`:
unequal and large sets, padded batches, shared key heads, causal order, 16-bit types.  Its backward pass recomputes the
probabilities from the saved log-sum-exp, so nothing of size queries x keys is ever stored.
"""
import math

import torch

from . import ops

_set_attention = torch.ops.cmvae_amd.set_attention.default


def set_attention(q, k, v, scale=None, causal=False, q_len=None, k_len=None, residual=False):
    """softmax(scale * q k^T) v (+ q if `residual`) per (batch, head).

    q [B, Sq, H, D], k and v [B, Sk, Hkv, D]: float32, bfloat16 or float16, D 64 or 128, any strides (copied where
    channels are not adjacent or rows not 16-byte aligned); H a multiple of Hkv, query head h reads key head
    h // (H // Hkv).  scale: 1 / sqrt(D) by default.  q_len, k_len: int32 [B], the rows of each batch entry that count
    (padded batches; values are clamped to [0, S]); output rows behind q_len and all gradients of rows behind a length
    are zeros, and what such rows hold is never read.  causal: query i sees keys j <= i + k_len - q_len.  A query that
    sees no key gets zeros (plus its own row if `residual`).  Differentiable once in q, k, v; every result is the same
    bits on every run.

    Probabilities are fp32 and carry a relative error of 2^-24 of their row's largest score; in 16-bit types they, and the scores'
    gradients, are factors of twice the type's bits, so that results are off by their own rounding.  A key that is NaN or infinite
    may reach any row of its batch entry, also those that the causal order hides it from; an infinite value makes NaN.  Scores
    beyond 2^22 are out of range in float16, beyond 2^30 in the other types."""
    scale = 1.0 / math.sqrt(q.shape[-1]) if scale is None and q.shape[-1] else scale
    if ops.CHECK_INDICES:
        for t, n, x in ((q_len, 'q_len', q), (k_len, 'k_len', k)):
            if t is not None:
                ops.check_index_range(t, x.shape[1] + 1, n)
    return _set_attention(q, k, v, scale, causal, q_len, k_len, residual)
