"""The sequence operators over packs at sizes where a workgroup walks many tiles, takes several rounds of rows or looks back
over many segments, against 64-bit plain forms."""
import math

import pytest
import torch

from seq_util import check, marks, norm_rotary, recurrence
from seq_wide_util import attention_heads, recurrence_scan
from test_sequence import DEV, TYPES, _leaf, _normal, spc  # noqa: F401


def test_scanned_form_is_the_definition():
    """The recurrence in doubling steps against the one row by row."""
    b = marks([40, 1, 70], lead=3)
    n = len(b)
    a, x, g, h0 = (_normal(i, m, 3).double() for i, m in enumerate((n, n, n, 3)))
    for reverse in (False, True):
        for first in (None, h0):
            want, _ = recurrence(a, x, b, first, reverse, grad=g, dtype=torch.float64)
            for (_, y, _), z in zip(recurrence_scan(a, x, b, first, reverse, g), want):
                assert torch.allclose(y, z, rtol=1e-10, atol=1e-12)


# Enough workgroups that neither the keys of a tile of rows nor the rows of a tile of keys are split (more than 1024 and
# 2048 waves): 700 rows are 6 tiles of 128 (22 of 32 for float heads of 32) and as many steps of 64 as 11.
@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('lens,heads,kv,dim,causal', [
    ([700, 45], 96, 96, 32, True), ([700, 45], 96, 96, 64, False), ([700, 45], 96, 96, 64, True),
    ([700, 45], 96, 96, 128, True), ([1, 699], 96, 96, 80, False), ([700], 192, 96, 64, True),
])
def test_attention_many_tiles(spc, dtype, lens, heads, kv, dim, causal):
    b = marks(lens)
    q, k, v, g = (_normal(i, len(b), h, dim, dtype=dtype) for i, h in enumerate((heads, kv, kv, heads)))
    outs, tols = attention_heads(q.to(DEV), k.to(DEV), v.to(DEV), b, causal=causal, grad=g.to(DEV))
    leaves = [_leaf(x) for x in (q, k, v)]
    o = spc.pack_attention(*leaves, b.to(DEV), causal=causal)
    for name, x, want, tol in zip(('o', 'dq', 'dk', 'dv'), [o, *torch.autograd.grad(o, leaves, g.to(DEV))], outs, tols):
        check(name, x, want, tol)


# Splits of more than two tiles each: few heads, long packs
@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('lens,heads,kv,dim', [([5000], 2, 1, 32), ([3, 6000, 40], 4, 4, 64), ([4001], 4, 2, 128)])
def test_attention_long_splits(spc, dtype, lens, heads, kv, dim):
    b = marks(lens)
    q, k, v, g = (_normal(i, len(b), h, dim, dtype=dtype) for i, h in enumerate((heads, kv, kv, heads)))
    outs, tols = attention_heads(q.to(DEV), k.to(DEV), v.to(DEV), b, causal=True, grad=g.to(DEV))
    leaves = [_leaf(x) for x in (q, k, v)]
    o = spc.pack_attention(*leaves, b.to(DEV), causal=True)
    for name, x, want, tol in zip(('o', 'dq', 'dk', 'dv'), [o, *torch.autograd.grad(o, leaves, g.to(DEV))], outs, tols):
        check(name, x, want, tol)


# Infinities and NaN in a row's masked places, over many tiles without splits
@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('dim', [32, 64, 128])
def test_attention_many_tiles_beside_nan(spc, dtype, dim):
    b = marks([300, 400])
    q, k, v, g = (_normal(i, 700, 96, dim, dtype=dtype) for i in range(4))
    outs, tols = attention_heads(q.to(DEV), k.to(DEV), v.to(DEV), b, causal=True, grad=g.to(DEV))
    bad = [x.clone() for x in (q, k, v)]
    bad[0][7, :, 3], bad[1][100, ::2, 1], bad[2][299, :, 0] = math.nan, math.inf, -math.inf
    leaves = [_leaf(x) for x in bad]
    o = spc.pack_attention(*leaves, b.to(DEV), causal=True)
    for name, x, want, tol in zip(('o', 'dq', 'dk', 'dv'), [o, *torch.autograd.grad(o, leaves, g.to(DEV))], outs, tols):
        check(name, x[300:], want[300:], tol[300:])
        if name == 'o':  # rows before the first bad key, but for the bad query
            check(name, x[:7], want[:7], tol[:7])
            check(name, x[8:100], want[8:100], tol[8:100])


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('rows,heads,kv,dim,turn,interleaved', [(20011, 1, 1, 16, 16, False), (17000, 2, 1, 64, 20, False),
                                                                (16500, 3, 2, 32, 8, True), (40000, 1, 0, 8, 4, False)])
def test_norm_rotary_many_rounds(spc, dtype, rows, heads, kv, dim, turn, interleaved):
    """More rows than the backward's 1024 workgroups take in one round."""
    x = {'q': _normal(0, rows, heads, dim, dtype=dtype, scale=2.0), 'k': _normal(1, rows, kv, dim, dtype=dtype)}
    w = {n: (1 + _normal(2 + i, dim, scale=0.3)).to(dtype) for i, n in enumerate('qk')}
    g = {n: _normal(4 + i, *x[n].shape, dtype=dtype) for i, n in enumerate('qk')}
    f = 100.0 ** (-torch.arange(turn // 2).double() * 2 / turn)
    b = marks([rows // 3, 1, rows - rows // 3 - 1])
    at = torch.arange(rows)
    place = torch.where(at < rows // 3, at, torch.where(at == rows // 3, 0, at - rows // 3 - 1))
    leaves = [_leaf(y) for y in (x['q'], x['k'], w['q'], w['k'])]
    y = spc.norm_rotary(*leaves, f.to(DEV), boundaries=b.to(DEV), interleaved=interleaved)
    grads = torch.autograd.grad(y, leaves, [g[n].to(DEV) for n in 'qk'])
    for i, n in enumerate('qk'):
        outs, tols = norm_rotary(x[n], w[n], f, place, 1e-6, interleaved, grad=g[n], dtype=dtype)
        for name, got, want, tol in zip(('y', 'dx', 'dw'), (y[i], grads[i], grads[2 + i]), outs, tols):
            check(f'{name} of {n}', got, want, tol)


# 9000 x 260: chunks, a scan, the walk, with few segments; 200,000 x 4 and 140,001 x 3: more than a wave's lanes hold
@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES + [torch.float64])
@pytest.mark.parametrize('lens,dim', [([9000], 260), ([2999, 1, 6000], 260), ([70000, 1, 129999], 4), ([140001], 3),
                                      ([30, 70, 139900], 3)])
@pytest.mark.parametrize('reverse', [False, True])
@pytest.mark.parametrize('first', [False, True])
def test_recurrence_many_segments(spc, dtype, lens, dim, reverse, first):
    b, n = marks(lens), sum(lens)
    a = torch.sigmoid(_normal(0, n, dim, scale=3.0) + 2)
    a[::3] = torch.where(a[::3] > 0.5, a[::3], -a[::3])
    a[n // 2:n // 2 + 40000] = 1 - 1e-3 * a[n // 2:n // 2 + 40000].abs()  # states that last over many chunks
    a = a.to(dtype)
    x, g = _normal(1, n, dim, dtype=dtype), _normal(2, n, dim, dtype=dtype)
    h0 = _normal(3, len(lens), dim, dtype=dtype) if first else None
    leaves = [_leaf(y) for y in (a, x, h0)]
    h = spc.linear_recurrence(leaves[0], leaves[1], b.to(DEV), initial=leaves[2], reverse=reverse)
    got = [h, *torch.autograd.grad(h, [y for y in leaves if y is not None], g.to(DEV))]
    for y, (name, want, tol) in zip(got, recurrence_scan(a, x, b, h0, reverse, g)):
        check(name, y, want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize('lens,dim', [([3000, 2000, 4000], 260), ([60000, 20000, 60001], 3)])
@pytest.mark.parametrize('reverse', [False, True])
def test_recurrence_segments_beside_nan(spc, lens, dim, reverse):
    """Infinities and NaN of the middle pack stay in it where packs span many segments."""
    b, n = marks(lens), sum(lens)
    a, x, g = torch.sigmoid(_normal(0, n, dim) + 2), _normal(1, n, dim), _normal(2, n, dim)
    want = recurrence_scan(a, x, b, None, reverse, g)
    at = torch.arange(n)
    middle = (at >= lens[0]) & (at < lens[0] + lens[1])
    a, x = a.clone(), x.clone()
    a[middle & (at % 3 == 0)] = math.nan
    x[middle & (at % 3 == 1)] = math.inf
    leaves = [_leaf(y) for y in (a, x)]
    h = spc.linear_recurrence(*leaves, b.to(DEV), reverse=reverse)
    for y, (name, w, tol) in zip([h, *torch.autograd.grad(h, leaves, g.to(DEV))], want):
        check(name, y.cpu()[~middle], w[~middle], tol[~middle])
