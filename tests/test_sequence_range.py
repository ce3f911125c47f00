"""The sequence operators over packs with numbers far from 1: values, gradients and gates that are large, small or of very
different sizes, within their types' range."""
import math

import pytest
import torch

from seq_util import attention, check, marks
from seq_wide_util import attention_heads
from test_sequence import DEV, TYPES, _leaf, _normal, spc  # noqa: F401


def test_wide_form_is_the_definition():
    """The batched plain form against the one head by head, and its bounds no wider where nothing is small."""
    b, qb = marks([5, 9, 3], lead=1), marks([2, 12, 3])
    q, g = (_normal(i, 17, 4, 16, dtype=torch.float16) for i in range(2))
    k, v = (_normal(2 + i, 18, 2, 16, dtype=torch.float16) for i in range(2))
    for causal in (False, True):
        want, tols = attention(q, k, v, b, qb, causal, grad=g, dtype=torch.float16)
        outs, tight = attention_heads(q, k, v, b, qb, causal, grad=g)
        for x, y, t, w in zip(outs, want, tight, tols):
            assert torch.allclose(x, y, rtol=1e-12, atol=1e-14)
            assert (t <= 1.01 * w).all()  # 1 %: dk's and dv's own rounding counts once for its result here, there in its sum


def _gradients(spc, inputs, grad, b, **kw):
    leaves = [_leaf(x) for x in inputs]
    if 'q_boundaries' in kw:
        kw['q_boundaries'] = kw['q_boundaries'].to(DEV)
    o = spc.pack_attention(*leaves, b.to(DEV), **kw)
    return [o, *torch.autograd.grad(o, leaves, grad.to(DEV))]


def _compare(spc, inputs, grad, b, names=('o', 'dq', 'dk', 'dv'), **kw):
    outs, tols = attention_heads(*inputs, b, grad=grad, **kw)
    for name, x, want, tol in zip(('o', 'dq', 'dk', 'dv'), _gradients(spc, inputs, grad, b, **kw), outs, tols):
        if name in names:
            check(name, x, want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('lens,heads,kv,dim,causal,big', [
    ([256], 1, 1, 128, True, 3000.0), ([90, 300, 1], 4, 2, 64, False, 3000.0), ([65, 130], 3, 1, 32, True, 15000.0),
    ([700], 8, 8, 64, True, 8000.0),
])
def test_attention_gradients_with_large_values(spc, dtype, lens, heads, kv, dim, causal, big):
    """Values of thousands, and gradients so small that q's and k's stay within float16."""
    b = marks(lens)
    n = len(b)
    q, k = _normal(0, n, heads, dim, dtype=dtype, scale=0.3), _normal(1, n, kv, dim, dtype=dtype, scale=0.3)
    v, g = _normal(2, n, kv, dim, dtype=dtype, scale=big).clamp(-6e4, 6e4), _normal(3, n, heads, dim, dtype=dtype,
                                                                                  scale=0.01)
    _compare(spc, (q, k, v), g, b, causal=causal)


@pytest.mark.gpu
def test_attention_gradients_of_two_opposite_values(spc):
    """Two keys of equal weight and values of 200 and -200: ds is 6400 each way, and their products with k are small."""
    dim = 64
    q, k = torch.zeros(1, 1, dim), torch.full((2, 1, dim), 0.05)
    k[1] = -0.05
    q, k = q.half(), k.half()
    v = torch.full((2, 1, dim), 200.0).half()
    v[1] = -200.0
    g = torch.ones(1, 1, dim).half()
    _compare(spc, (q, k, v), g, marks([2]), q_boundaries=marks([1]))


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('causal', [False, True])
def test_attention_gradients_of_very_different_packs(spc, dtype, causal):
    """Gradients of 1e3 in one pack, 1e-3 and 1e-5 in others, an infinity in one more: each pack is as exact as alone."""
    lens, sizes = [40, 200, 70, 30], [1e3, 1e-3, 1e-5, 1.0]
    b = marks(lens)
    n = len(b)
    q, k, v = (_normal(i, n, h, 32, dtype=dtype) for i, h in enumerate((4, 2, 2)))
    size = torch.cat([torch.full((m, 1, 1), x) for m, x in zip(lens, sizes)])
    g = (_normal(3, n, 4, 32) * size).to(dtype)
    outs, tols = attention_heads(q, k, v, b, grad=g, causal=causal)
    dirty = g.clone()
    dirty[325, 1, 5] = math.inf
    got = _gradients(spc, (q, k, v), dirty, b, causal=causal)
    for name, x, want, tol in zip(('o', 'dq', 'dk', 'dv'), got, outs, tols):
        x, clean = x.cpu(), torch.ones(want.shape[:2], dtype=torch.bool)
        if name == 'dq':
            clean[325, 1] = False
        elif name != 'o':  # the keys that row 325 sees, of its key head
            clean[310:, 0] = False
        check(name, x[clean], want[clean], tol[clean])
        if name != 'o':
            assert not torch.isfinite(x[~clean]).all()
