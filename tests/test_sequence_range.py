"""The sequence operators over packs with numbers far from 1: values, gradients and gates that are large, small or of very
different sizes, within their types' range."""
import math

import pytest
import torch

from seq_util import attention, check, marks, norm_rotary, recurrence
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


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('rows,sharp', [(131072, 3.0), (4096, 0.0)])
def test_attention_gradients_of_small_weights(spc, dtype, rows, sharp):
    """The values' gradients of one query over many keys, of weights down to 2^-24 and less: a long pack, and one whose first
    key has nearly all the weight."""
    dim = 64
    q, k, v, g = (_normal(i, m, 1, dim, dtype=dtype) for i, m in enumerate((1, rows, rows, 1)))
    if sharp:
        k = (k.float() * sharp).to(dtype)
    else:  # scores of 0 and some -14.6: weights of 1 and 2^-21
        k = torch.where(torch.arange(rows)[:, None, None] == 0, 0.0, -117 / dim + 0.01 * k.float()).to(dtype)
        q = torch.ones_like(q)
    g = (1000 * g.float()).to(dtype)
    _compare(spc, (q, k, v), g, marks([rows]), q_boundaries=marks([1]))


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
def test_attention_many_small_weights(spc, dtype):
    """131,071 keys of weights 2^-25.5 of the first one's, whose sum counts: enough rows that their keys are not split."""
    n, rows, heads, dim = 131072, 4096, 16, 8
    k, v = torch.full((n, heads, dim), -6.25), torch.ones(n, heads, dim)
    k[0], v[0] = 0, 0
    q, k, v = torch.ones(rows, heads, dim).to(dtype), k.to(dtype), v.to(dtype)
    b = marks([n])
    (want,), (tol,) = attention_heads(q[:1], k, v, b, marks([1]))
    assert (want > 2e-3).all() and (tol < 0.05 * want).all()
    o = spc.pack_attention(q.to(DEV), k.to(DEV), v.to(DEV), b.to(DEV), q_boundaries=marks([rows]).to(DEV))
    check('o', o, want.expand(rows, heads, dim), tol.expand(rows, heads, dim))


def _recurrence(spc, a, x, b, first=None, reverse=False, grad=None):
    outs, tols = recurrence(a, x, b, first, reverse, grad=grad, dtype=a.dtype)
    leaves = [_leaf(y) for y in (a, x, first)]
    h = spc.linear_recurrence(leaves[0], leaves[1], b.to(DEV), initial=leaves[2], reverse=reverse)
    got = [h, *torch.autograd.grad(h, [y for y in leaves if y is not None], grad.to(DEV))]
    for name, y, want, tol in zip(('h', 'da', 'db', 'dinitial'), got, outs, tols):
        assert torch.isfinite(want).all() and torch.isfinite(y).all(), name
        check(name, y, want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float64])
@pytest.mark.parametrize('n,dim', [(200, 3), (700, 8), (3000, 40), (9000, 260)])  # one launch, segments, three launches
@pytest.mark.parametrize('reverse', [False, True])
def test_recurrence_gates_above_one_over_zeros(spc, dtype, n, dim, reverse):
    """States that are exactly 0 stay so however long gates of 2 run over them, and so do the gradients that are 0."""
    lens = [n // 2, n - n // 2]
    b = marks(lens)
    a, x, g = torch.full((n, dim), 2.0), torch.zeros(n, dim), torch.zeros(n, dim)
    for at, m in zip((0, n // 2), lens):
        rows = list(range(at, at + m))[::-1 if reverse else 1]
        for i in range(6):  # features in the last rows that the states walk, gradients in the last that theirs do (the
            x[rows[-6 + i]] = 0.5 + i  # first): 2^6 each, where from the other end they would grow to 2^m
            g[rows[i]] = 1.0 - 0.25 * i
    _recurrence(spc, a.to(dtype), x.to(dtype), b, None, reverse, g.to(dtype))


@pytest.mark.gpu
@pytest.mark.parametrize('dtype,step,low', [(torch.float32, 2.0 ** 12, 2.0 ** -100), (torch.bfloat16, 2.0 ** 12, 2.0 ** -100),
                                            (torch.float64, 2.0 ** 100, 2.0 ** -800)])
@pytest.mark.parametrize('n,dim', [(100, 3), (256, 8), (1500, 40), (9000, 260)])
@pytest.mark.parametrize('reverse', [False, True])
def test_recurrence_gates_that_take_turns(spc, dtype, step, low, n, dim, reverse):
    """16 rows whose gates are large, then 16 that undo them: their products pass the type's range, the states, between
    `low` and low * step ** 16, do not."""
    walked = torch.arange(n).flip(0) if reverse else torch.arange(n)
    up, few = walked // 16 % 2 == 0, walked % 32 == 0  # few: where states are smallest
    a = torch.where(up[:, None], step, 1 / step).to(torch.float64).expand(n, dim)
    x = torch.where(few[:, None], _normal(0, n, dim).double() * low * 2.0 ** -10, 0.0)
    g, first = _normal(1, n, dim).double() * low, _normal(2, 1, dim).double() * low
    _recurrence(spc, a.to(dtype), x.to(dtype), marks([n]), first.to(dtype), reverse, g.to(dtype))


@pytest.mark.gpu
@pytest.mark.parametrize('n,dim', [(200, 3), (700, 8), (9000, 260)])
def test_recurrence_infinite_gates_and_features(spc, n, dim):
    """A pack with an infinite gate is not finite from that row on, one with an infinite feature infinite up to the
    next gate of 0; rows before it and other packs are as without them."""
    lens = [n // 2, n - n // 2]
    b = marks(lens)
    a, x = torch.sigmoid(_normal(0, n, dim) + 2), _normal(1, n, dim)
    (want, *_), (tol, *_) = recurrence(a, x, b, dtype=torch.float32)
    for where in (a, x):
        keep = where[20].clone()
        where[20] = math.inf
        h = spc.linear_recurrence(a.to(DEV), x.to(DEV), b.to(DEV)).cpu()
        check('h', h[:20], want[:20], tol[:20])
        check('h', h[n // 2:], want[n // 2:], tol[n // 2:])
        assert not torch.isfinite(h[20:n // 2]).any()
        if where is x:
            assert (h[20:n // 2] == math.inf).all()
        where[20] = keep


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('size,eps', [(1e25, 1e-6), (1e37, 0.0), (1e-25, 0.0), (1e-25, 1e-6), (1e-30, 1e-38), (1.0, 1e38),
                                      (1e-20, 1e-35)])
@pytest.mark.parametrize('heads,kv,dim,turn,interleaved', [(3, 1, 128, 128, False), (2, 2, 40, 8, True), (1, 5, 256, 64, False)])
def test_norm_of_heads_far_from_one(spc, dtype, size, eps, heads, kv, dim, turn, interleaved):
    """Heads whose squares, or eps, leave a float's range, beside ones of order 1 and one of zeros in the same rows."""
    n = 37
    x = {'q': _normal(0, n, heads, dim), 'k': _normal(1, n, kv, dim)}
    for y in x.values():
        y[::2] *= size
        y[5:7, :1] = 0
    if eps == 0:  # a head of zeros has no norm then
        for y in x.values():
            y[5:7, :1] = 1
    x = {m: y.to(dtype) for m, y in x.items()}
    w = {m: (1 + _normal(2 + i, dim, scale=0.3)).to(dtype) for i, m in enumerate('qk')}
    g = {m: _normal(4 + i, *x[m].shape, dtype=dtype) for i, m in enumerate('qk')}
    f = 100.0 ** (-torch.arange(turn // 2).double() * 2 / turn)
    leaves = [_leaf(y) for y in (x['q'], x['k'], w['q'], w['k'])]
    y = spc.norm_rotary(*leaves, f.to(DEV), positions=torch.arange(n, device=DEV), eps=eps, interleaved=interleaved)
    grads = torch.autograd.grad(y, leaves, [g[m].to(DEV) for m in 'qk'])
    eps = float(torch.tensor(eps, dtype=torch.float32))
    for i, m in enumerate('qk'):
        outs, tols = norm_rotary(x[m], w[m], f, torch.arange(n), eps, interleaved, grad=g[m], dtype=dtype)
        for name, got, want, tol in zip(('y', 'dx', 'dw'), (y[i], grads[i], grads[2 + i]), outs, tols):
            check(f'{name} of {m}', got, want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize('rows,at', [(26200, 2000), (26200, 8000), (3000, 2000)])  # chunks of 20 rows and a scan, of 8
@pytest.mark.parametrize('reverse', [False, True])
def test_recurrence_states_that_left_the_range(spc, rows, at, reverse):
    """20 gates of 2^-1000 take a state to 0, and 16 of 2^1000 do not bring it back; 20 of 2^1000 take it to infinity, and
    16 of 2^-1000 do not bring it back either; a state of 0 stays 0."""
    h0 = torch.tensor([2.0 ** 500, -2.0 ** 500, 0.0], dtype=torch.float64)[None].repeat(1, 67)[:, :200]
    for first, then, left in ((-1000, 1000, 0.0), (1000, -1000, math.inf)):
        a = torch.ones(rows, 200, dtype=torch.float64)
        a[at:at + 20], a[at + 20:at + 36] = 2.0 ** first, 2.0 ** then
        x = torch.zeros_like(a)
        if reverse:
            a = a.flip(0).contiguous()
        h = spc.linear_recurrence(a.to(DEV), x.to(DEV), marks([rows]).to(DEV), initial=h0.to(DEV), reverse=reverse).cpu()
        h = h.flip(0) if reverse else h
        assert torch.equal(h[:at], h0.expand(at, 200))
        want = torch.where(h0 == 0, 0.0, torch.where(h0 < 0, -left, left))
        assert torch.equal(h[at + 19:], want.expand(rows - at - 19, 200))
