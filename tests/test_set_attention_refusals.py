"""CPU: what set attention refuses, in Python and at the C entry points (nothing is launched)."""
import ctypes

import pytest
import torch


def test_python_refusals_name_the_argument():
    from cmvae_amd.attention import set_attention
    x = torch.zeros(1, 4, 2, 64)
    with pytest.raises(RuntimeError, match='GPU tensor'):
        set_attention(x, x, x)


def _desc(**kw):
    from cmvae_amd._lib import SetAttnDesc
    d = SetAttnDesc()
    vals = dict(dtype=0, B=1, Sq=4, Sk=4, H=2, Hkv=2, D=64, causal=0, residual=0, scale=0.125, q=4096, k=4096, v=4096,
                dO=4096, o=4096, attn=None, lse=4096, delta=4096, dq=4096, dk=4096, dv=4096)
    strides = dict(q_stride=(512, 128, 64), k_stride=(512, 128, 64), v_stride=(512, 128, 64), dO_stride=(512, 128, 64))
    for n in strides:
        if n in kw:
            strides[n] = kw.pop(n)
    vals.update(kw)
    for n, v in vals.items():
        setattr(d, n, v)
    for n, v in strides.items():
        getattr(d, n)[:] = v
    return d


BAD = [dict(dtype=3), dict(dtype=-1), dict(B=0), dict(Sq=0), dict(Sk=-1), dict(H=3), dict(Hkv=0), dict(D=32), dict(D=96),
       dict(scale=0.0), dict(scale=-1.0), dict(scale=float('nan')), dict(scale=float('inf')), dict(q=None), dict(o=None),
       dict(k=None), dict(v=None), dict(q=4100), dict(o=4104), dict(q_stride=(512, 130, 64)), dict(k_stride=(512, 128, 2)),
       dict(v_stride=(-512, 128, 64)), dict(Sq=1 << 30), dict(Sk=1 << 30), dict(dtype=1, k_stride=(512, 132, 64))]


@pytest.mark.parametrize('kw', BAD, ids=lambda k: ','.join('%s=%s' % i for i in k.items()))
def test_c_entry_refuses(kw):
    """A bad descriptor is refused on the host, before any launch, with a message."""
    from cmvae_amd._lib import lib
    d = _desc(**kw)
    assert lib.cmvae_set_attention_fwd(ctypes.byref(d), None, 0, None) < 0
    assert b'cmvae_set_attention_fwd' in lib.cmvae_last_error()


@pytest.mark.parametrize('kw', [dict(dO=None), dict(lse=None), dict(delta=None), dict(dq=None), dict(dk=None),
                                dict(residual=1, attn=None), dict(dO=4100), dict(dO_stride=(512, 2, 64)), dict(dk=4104)],
                         ids=lambda k: ','.join('%s=%s' % i for i in k.items()))
def test_c_backward_refuses(kw):
    from cmvae_amd._lib import lib
    d = _desc(**kw)
    assert lib.cmvae_set_attention_bwd(ctypes.byref(d), None, 0, None) < 0
    assert b'cmvae_set_attention_bwd' in lib.cmvae_last_error()


def test_c_entry_needs_its_workspace():
    """One query against many keys is cut into pieces that are joined: the call without room for them is refused."""
    from cmvae_amd._lib import lib
    d = _desc(Sq=1, Sk=4096)
    need = lib.cmvae_set_attention_workspace_bytes(ctypes.byref(d), 0)
    assert need > 0
    assert lib.cmvae_set_attention_fwd(ctypes.byref(d), None, 0, None) < 0
    assert lib.cmvae_set_attention_fwd(ctypes.byref(d), 4096, need - 1, None) < 0
    assert lib.cmvae_set_attention_fwd(ctypes.byref(d), 4100, need, None) < 0
    need = lib.cmvae_set_attention_workspace_bytes(ctypes.byref(d), 1)
    assert need > 0 and lib.cmvae_set_attention_bwd(ctypes.byref(d), 4096, need - 1, None) < 0
    assert lib.cmvae_set_attention_fwd(None, None, 0, None) < 0
    assert lib.cmvae_set_attention_workspace_bytes(None, 0) == 0
