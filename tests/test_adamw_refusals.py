"""CPU: what the AdamW step refuses, in Python and at its C entry points (nothing is launched)."""
import ctypes

import pytest
import torch


def test_python_refuses_cpu_tensors():
    from cmvae_amd.optim import AdamW, adamw_state_values, adamw_step
    p = torch.zeros(4)
    with pytest.raises(RuntimeError, match='GPU'):
        adamw_step([p], [p], torch.zeros(256), torch.zeros(256))
    with pytest.raises(RuntimeError, match='GPU'):
        adamw_state_values(torch.zeros(256), torch.zeros(256), torch.zeros(2, 1))
    with pytest.raises(RuntimeError, match='GPU'):
        AdamW([p])


GOOD = dict(tensors=[(4096, 8192, 100, 0, 0)], bits=32, m=4096, v=8192, scales=None, length=256, step=1, step_dev=None, lr=1e-3,
            b1=0.9, b2=0.999, eps=1e-8, wd=0.01)


@pytest.mark.parametrize('kw', [
    dict(tensors=[(0, 8192, 100, 0, 0)]), dict(tensors=[(4096, 0, 100, 0, 0)]), dict(tensors=[(4096, 8192, -1, 0, 0)]),
    dict(tensors=[(4096, 8192, 257, 0, 0)]), dict(tensors=[(4096, 8192, 100, 256, 0)]), dict(tensors=[(4096, 8192, 1, 4, 0)]),
    dict(tensors=[(4096, 8192, 1, -256, 0)]), dict(tensors=[(4096, 8192, 100, 0, 3)]), dict(tensors=[(4098, 8192, 100, 0, 0)]),
    dict(tensors=[(4096, 8193, 100, 0, 1)]), dict(bits=16), dict(bits=8), dict(m=None), dict(v=None), dict(m=4100),
    dict(length=100), dict(length=-256), dict(step=0), dict(lr=float('nan')), dict(b1=1.0), dict(b2=-0.1), dict(eps=-1.0),
    dict(wd=float('inf')), dict(tensors=None)], ids=str)
def test_c_entry_refuses(kw):
    from cmvae_amd._lib import lib
    a = {**GOOD, **kw}
    t = None if a['tensors'] is None else (ctypes.c_int64 * 5)(*a['tensors'][0])
    assert lib.cmvae_adamw_step(t, 1, a['bits'], a['m'], a['v'], a['scales'], a['length'], a['step'], a['step_dev'], a['lr'],
                                a['b1'], a['b2'], a['eps'], a['wd'], None) < 0
    assert b'cmvae_adamw_step' in lib.cmvae_last_error()


def test_c_values_refuse():
    from cmvae_amd._lib import lib
    assert lib.cmvae_adamw_state_values(4096, 4096, 4096, 100, 4096, 4096, None) < 0
    assert lib.cmvae_adamw_state_values(None, 4096, 4096, 256, 4096, 4096, None) < 0
    assert lib.cmvae_adamw_state_values(4096, 4096, 4096, 256, 4100, 4096, None) < 0
    assert lib.cmvae_adamw_state_values(None, None, None, 0, None, None, None) == 0
