"""The sequence operators over packs have no forward-mode derivatives: both routes refuse a tensor that carries one, whichever
argument it is, also where no gradient is recorded."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

from test_sequence import DEV, spc  # noqa: F401


@pytest.mark.gpu
@pytest.mark.parametrize('which', ['q', 'k', 'v', 'norm q', 'norm k', 'q_weight', 'k_weight', 'freqs', 'positions', 'gates',
                                   'feats', 'initial'])
@pytest.mark.parametrize('recorded', [False, True])
def test_forward_mode_is_refused(spc, which, recorded):
    b = torch.ones(4, dtype=torch.bool, device=DEV)
    x, y = torch.rand(4, 2, 8, device=DEV), torch.rand(4, 8, device=DEV)
    f, w = torch.rand(4, dtype=torch.float64, device=DEV), torch.rand(8, device=DEV)
    call, args = {
        'q': (lambda *a: spc.pack_attention(*a, b), [x, x, x]),
        'norm q': (lambda *a: spc.norm_rotary(*a[:5], positions=a[5]), [x, x, w, w, f, y[:, 0].contiguous()]),
        'gates': (lambda *a: spc.linear_recurrence(*a[:2], b, initial=a[2]), [y, y, y]),
    }['q' if which in 'qkv' else 'gates' if which in ('gates', 'feats', 'initial') else 'norm q']
    at = {'q': 0, 'k': 1, 'v': 2, 'norm q': 0, 'norm k': 1, 'q_weight': 2, 'k_weight': 3, 'freqs': 4, 'positions': 5,
          'gates': 0, 'feats': 1, 'initial': 2}[which]
    with fwAD.dual_level(), torch.set_grad_enabled(recorded):
        args[at] = fwAD.make_dual(args[at], torch.ones_like(args[at]))
        with pytest.raises(NotImplementedError, match='jvp'):
            call(*args)
