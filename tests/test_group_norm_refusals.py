"""CPU: what group norm refuses, in Python and at its C entry points (nothing is launched)."""
import ctypes

import pytest
import torch


def test_python_refuses_cpu_tensors():
    from cmvae_amd.norm import group_norm_act
    with pytest.raises(RuntimeError, match='GPU tensor'):
        group_norm_act(torch.zeros(2, 3, 8), 2)


def _desc(**kw):
    from cmvae_amd._lib import GroupNormDesc
    d = GroupNormDesc()
    vals = dict(dtype=0, wdtype=0, act=0, N=2, P=100, C=64, G=8, eps=1e-5, x=4096, weight=4096, bias=4096, dy=4096, y=4096,
                stats=4096, dx=4096, dweight=4096, dbias=4096)
    strides = dict(x_stride=(6400, 64), dy_stride=(6400, 64))
    for n in strides:
        strides[n] = kw.pop(n, strides[n])
    for n, v in {**vals, **kw}.items():
        setattr(d, n, v)
    for n, v in strides.items():
        getattr(d, n)[:] = v
    return d


@pytest.mark.parametrize('kw', [dict(dtype=3), dict(dtype=1, wdtype=2), dict(N=0), dict(P=0), dict(C=0), dict(G=0), dict(G=7),
                                dict(act=4), dict(act=-1), dict(eps=-1.0), dict(eps=float('nan')), dict(eps=float('inf')),
                                dict(x=None), dict(y=None), dict(x=4097), dict(weight=4098), dict(stats=4104),
                                dict(x_stride=(-1, 64)), dict(x_stride=(6400, -64)), dict(N=1 << 30)],
                         ids=lambda k: ','.join('%s=%s' % i for i in k.items()))
def test_c_forward_refuses(kw):
    from cmvae_amd._lib import lib
    assert lib.cmvae_group_norm_fwd(ctypes.byref(_desc(**kw)), None, 0, None) < 0
    assert b'cmvae_group_norm_fwd' in lib.cmvae_last_error()


@pytest.mark.parametrize('kw', [dict(dy=None), dict(dx=None), dict(stats=None), dict(dx=4098), dict(dy_stride=(-1, 1)), {}],
                         ids=lambda k: ','.join('%s=%s' % i for i in k.items()) or 'no workspace')
def test_c_backward_refuses(kw):
    from cmvae_amd._lib import lib
    assert lib.cmvae_group_norm_bwd(ctypes.byref(_desc(**kw)), None, 0, None) < 0
    assert b'cmvae_group_norm_bwd' in lib.cmvae_last_error()


def test_c_entry_needs_its_workspace():
    """A sample that no workgroup can hold is summed in pieces: the call without room for them is refused."""
    from cmvae_amd._lib import lib
    d = _desc(P=100000, x_stride=(6400000, 64))
    need = lib.cmvae_group_norm_workspace_bytes(ctypes.byref(d), 0)
    assert need > 0 and lib.cmvae_group_norm_workspace_bytes(ctypes.byref(_desc()), 0) == 0
    assert lib.cmvae_group_norm_fwd(ctypes.byref(d), None, 0, None) < 0
    assert lib.cmvae_group_norm_fwd(ctypes.byref(d), 4096, need - 1, None) < 0
    assert lib.cmvae_group_norm_fwd(ctypes.byref(d), 4104, need, None) < 0
    assert lib.cmvae_group_norm_fwd(None, None, 0, None) < 0
    assert lib.cmvae_group_norm_workspace_bytes(None, 1) == 0
