"""The sequence operators over packs (kaolin.render.spc.pack_attention, norm_rotary, linear_recurrence): against
64-bit plain forms with derived bounds (seq_util.py), their masks and sizes at the edges, refusals, captured and
repeated calls, and a run of them together with the packed ray ops."""
import math

import pytest
import torch

from seq_util import attention, check, marks, norm_rotary, recurrence, spans

DEV = 'cuda'
TYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.fixture(params=['compiled', 'python'])
def spc(request, monkeypatch):
    """The operators through their compiled nodes and through the Python ones."""
    import kaolin
    from kaolin import _ext
    if request.param == 'python':
        monkeypatch.setattr(_ext, '_mod', None)
    elif torch.cuda.is_available():
        assert _ext.get() is not None, 'the compiled nodes are not built'
    return kaolin.render.spc


def _normal(seed, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


def _leaf(x):
    return None if x is None else x.to(DEV).requires_grad_()


# ------------------------------------------------------------------------------- the plain forms themselves
def test_plain_attention_gradients_are_differences():
    b = marks([3, 4], lead=1)
    q, k, v, g = (_normal(i, 8, h, 8).double() for i, h in enumerate((2, 1, 1, 2)))
    outs, _ = attention(q, k, v, b, causal=True, grad=g, dtype=torch.float32)
    for i, x in enumerate((q, k, v)):
        d = _normal(9 + i, *x.shape).double()
        args = [q, k, v]
        sides = []
        for s in (1e-5, -1e-5):
            args[i] = x + s * d
            sides.append((attention(*args, b, causal=True, dtype=torch.float32)[0][0] * g).sum())
        # a central difference over 2e-5 is off by some 1e-10, and by 1e-11 from rounding
        assert abs((sides[0] - sides[1]) / 2e-5 - (outs[1 + i] * d).sum()) < 1e-7


def test_plain_norm_gradients_are_differences():
    f = torch.tensor([1.0, 0.1, 0.01], dtype=torch.float64)
    pos = torch.tensor([0.0, 3.0, 700.0])
    x, w, g = _normal(0, 3, 2, 16).double(), _normal(1, 16).double(), _normal(2, 3, 2, 16).double()
    for inter in (False, True):
        outs, _ = norm_rotary(x, w, f, pos, 1e-3, inter, grad=g, dtype=torch.float32)
        for i, y in enumerate((x, w)):
            d = _normal(5 + i, *y.shape).double()
            sides = []
            for s in (1e-5, -1e-5):
                args = [x, w]
                args[i] = y + s * d
                sides.append((norm_rotary(*args, f, pos, 1e-3, inter, dtype=torch.float32)[0][0] * g).sum())
            assert abs((sides[0] - sides[1]) / 2e-5 - (outs[1 + i] * d).sum()) < 1e-7


def test_plain_recurrence_gradients_are_differences():
    b = marks([3, 1, 4], lead=2)
    a, x, h0, g = (_normal(i, n, 3).double() for i, n in enumerate((10, 10, 2, 10)))  # the last pack has no initial
    for rev in (False, True):
        outs, _ = recurrence(a, x, b, h0, rev, grad=g, dtype=torch.float64)
        for i, y in enumerate((a, x, h0)):
            d = _normal(5 + i, *y.shape).double()
            sides = []
            for s in (1e-5, -1e-5):
                args = [a, x, h0]
                args[i] = y + s * d
                sides.append((recurrence(args[0], args[1], b, args[2], rev, dtype=torch.float64)[0][0] * g).sum())
            assert abs((sides[0] - sides[1]) / 2e-5 - (outs[1 + i] * d).sum()) < 1e-7


def test_rotary_frequencies(spc):
    f = spc.rotary_frequencies(8, base=100.0, device='cpu')
    assert f.dtype == torch.float64
    assert torch.allclose(f, 100.0 ** (-torch.arange(4).double() / 4), rtol=1e-15, atol=0)
    assert torch.allclose(spc.rotary_frequencies(8, 100.0, factor=4.0, device='cpu'), f / 4, rtol=1e-15, atol=0)
    # in 2 pi * 64 units the four pairs turn 64, 20.2, 6.4 and 2.02 times: the first stays, the others lose the share
    # (32 - turns) / 31 of their frequency's difference to a quarter of it
    g = spc.rotary_frequencies(8, 100.0, factor=4.0, original_length=2 * math.pi * 64, device='cpu')
    keep = ((64 * f - 1) / 31).clamp(0, 1)
    assert keep[0] == 1 and 0 < keep[3] < keep[2] < keep[1] < 1
    assert torch.allclose(g, f * keep + f / 4 * (1 - keep), rtol=1e-14, atol=0)
    assert spc.rotary_frequencies(0, device='cpu').shape == (0,)
    for args in (dict(turn=7), dict(turn=8, base=0.0), dict(turn=8, factor=0.0), dict(turn=8, original_length=0),
                 dict(turn=8, slow=2.0, fast=2.0)):
        with pytest.raises(RuntimeError, match='rotary_frequencies'):
            spc.rotary_frequencies(device='cpu', **args)


# ------------------------------------------------------------------------------- refusals, on the CPU
def test_refusals_before_any_gpu(spc):
    from kaolin.render.spc import sequence
    b = torch.tensor([True, False, True])
    q = torch.rand(3, 2, 8)
    with pytest.raises(RuntimeError, match='on CPU'):
        spc.pack_attention(q, q, q, b)
    with pytest.raises(RuntimeError, match='boundaries must hold one value for each'):
        spc.pack_attention(q, q, q, b[:2])
    with pytest.raises(RuntimeError, match='q_boundaries must hold one value for each'):
        sequence._check_boundaries('pack_attention', 'q_boundaries', b, q[:1])
    with pytest.raises(RuntimeError, match='boundaries must be Bool'):
        spc.linear_recurrence(q[:, 0], q[:, 0], b.float())
    with pytest.raises(RuntimeError, match='on CPU'):
        spc.linear_recurrence(q[:, 0], q[:, 0], b)
    f = torch.ones(4, dtype=torch.float64)
    with pytest.raises(RuntimeError, match='either boundaries or positions'):
        spc.norm_rotary(q, q, None, None, f)
    with pytest.raises(RuntimeError, match='either boundaries or positions'):
        spc.norm_rotary(q, q, None, None, f, boundaries=b, positions=torch.zeros(3))
    with pytest.raises(RuntimeError, match='positions cannot take a gradient'):
        spc.norm_rotary(q, q, None, None, f, positions=torch.zeros(3, requires_grad=True))
    with pytest.raises(RuntimeError, match='freqs cannot take a gradient'):
        spc.norm_rotary(q, q, None, None, f.requires_grad_(), positions=torch.zeros(3))
    with pytest.raises(RuntimeError, match='on CPU'):
        spc.norm_rotary(q, q, None, None, f.detach(), positions=torch.zeros(3))


def test_library_refusals_without_gpu():
    """Sizes that the library itself refuses, before it launches anything."""
    import ctypes

    from kaolin import _native as N
    lib = N.lib()
    st = (ctypes.c_int64 * 6)()

    def attend(dtype=0, nq=1, nk=1, heads=1, kv=1, dim=8, scale=1.0, ws=1 << 30):
        return lib.kl_pack_attention_forward(dtype, nq, nk, heads, kv, dim, None, None, None, st, None, None, None, None,
                                             scale, 0, None, None, None, None, ws, None), lib.kl_last_error()
    for kw, what in ((dict(dim=12), b'multiple of 8'), (dict(dim=136), b'multiple of 8'), (dict(heads=3, kv=2), b'heads'),
                     (dict(scale=0.0), b'scale'), (dict(scale=float('nan')), b'scale'), (dict(nq=-1), b'rows'),
                     (dict(nq=1 << 31), b'rows'), (dict(nk=(1 << 31) - 1), b'rows'), (dict(ws=0), b'workspace'),
                     (dict(nq=1 << 30, heads=4, kv=1), b'too many'), (dict(dtype=1), b'Half, BFloat16 or Float')):
        rc, msg = attend(**kw)
        assert rc == -1 and what in msg, (kw, msg)
    rc = lib.kl_pack_attention_backward(0, 1, 1, 1, 1, 8, None, None, None, None, st, None, None, None, None, None, None,
                                        None, 1.0, 0, None, 16, None, None, 1 << 30, None)
    assert rc == -1 and b'go together' in lib.kl_last_error()
    assert lib.kl_pack_layout(1 << 31, None, None, None, None, 1 << 30, None) == -1
    assert lib.kl_pack_layout(70000, None, None, None, None, 0, None) == -1
    assert b'workspace' in lib.kl_last_error()
    for n, m, ws in ((1 << 31, 1, 1 << 30), (1, -1, 1 << 30), (-1, 1, 1 << 30), (1, 1, 256), (70000, 70000, 300)):
        assert lib.kl_pack_layout_pair(n, None, None, None, m, None, None, None, None, ws, None) == -1, (n, m)
    for i in range(6):  # a tile's rows have to lie within 2^32 bytes, and forward
        st[i] = -8
        assert attend()[0] == -1 and b'negative stride' in lib.kl_last_error()
        st[i] = 1 << 25
        assert i % 2 or attend()[0] == -1 and b'too far apart' in lib.kl_last_error()
        st[i] = 0
    p16 = ctypes.c_void_p(16)
    for i, at in ((0, 24), (1, 16), (2, 24)):  # an address, a row's stride, a head's stride
        st[0], st[1] = (60, 16) if i == 1 else (64, 12 if i == 2 else 16)
        rc = lib.kl_pack_attention_forward(2, 2, 2, 2, 2, 16, ctypes.c_void_p(at), p16, p16, st, None, None, None, None,
                                           1.0, 0, None, None, None, None, 1 << 30, None)
        assert rc == -1 and b'multiples of 16 bytes' in lib.kl_last_error(), (i, lib.kl_last_error())
        rc = lib.kl_norm_rotary_forward(2, 2, 2, 2, 16, 8, 0, ctypes.c_void_p(at), p16, st, None, None, 0, None, 3, None,
                                        None, None, 1e-6, None, None, None)
        assert rc == -1 and b'multiples of 16 bytes' in lib.kl_last_error(), (i, lib.kl_last_error())
    st[0] = st[1] = 0

    def norm(dim=8, turn=8, eps=1e-6, kind=3, n=1):
        return lib.kl_norm_rotary_forward(0, n, 1, 1, dim, turn, 0, None, None, st, None, None, 0, None, kind, None, None,
                                          None, eps, None, None, None)
    for kw in (dict(dim=10), dict(dim=264, turn=8), dict(turn=10), dict(turn=3), dict(eps=-1.0), dict(kind=4),
               dict(n=1 << 31)):
        assert norm(**kw) == -1, kw
    assert lib.kl_linear_recurrence_forward(0, 1 << 31, 1, None, None, None, 0, None, None, 0, None, None, 1 << 40,
                                            None) == -1
    assert lib.kl_linear_recurrence_forward(0, 1000, 64, None, None, None, 0, None, None, 0, None, None, 0, None) == -1
    assert b'workspace' in lib.kl_last_error()
    assert lib.kl_linear_recurrence_forward(3, 1, 1, None, None, None, 0, None, None, 0, None, None, 1 << 20, None) == -1


@pytest.mark.gpu
def test_refusals_on_gpu(spc):
    b = torch.tensor([True, False, True], device=DEV)
    q = torch.rand(3, 2, 8, device=DEV)

    def refuses(match, fn, *args, **kw):
        with pytest.raises(RuntimeError, match=match):
            fn(*args, **kw)
    refuses('multiple of 8 up to 128', spc.pack_attention, q[..., :4], q[..., :4], q[..., :4], b)
    refuses('multiple of 8 up to 128', spc.pack_attention, q, torch.rand(3, 2, 16, device=DEV),
            torch.rand(3, 2, 16, device=DEV), b)
    refuses('multiple of the heads', spc.pack_attention, q[:, :1], q, q, b)
    refuses('same type', spc.pack_attention, q, q.half(), q, b)
    refuses('same size', spc.pack_attention, q, q, q[:, :1], b)
    refuses('Half, BFloat16, Float', spc.pack_attention, q.double(), q.double(), q.double(), b)
    refuses('scale must be positive', spc.pack_attention, q, q, q, b, scale=0.0)
    refuses('one value for each', spc.pack_attention, q[:2], q, q, b)
    refuses('boundaries is on cpu', spc.pack_attention, q, q, q, b.cpu())
    refuses('3-dimensional', spc.pack_attention, q[0], q, q, b, q_boundaries=b[:2])
    f = torch.ones(4, dtype=torch.float64, device=DEV)
    p = torch.zeros(3, device=DEV)
    refuses('scalar type', spc.norm_rotary, q, q, None, None, f.float(), positions=p)
    refuses('do not fit', spc.norm_rotary, q, q, None, None, torch.ones(5, dtype=torch.float64, device=DEV), positions=p)
    refuses('scalar type', spc.norm_rotary, q, q, None, None, f, positions=p.double())
    refuses('size', spc.norm_rotary, q, q, None, None, f, positions=p[:2])
    refuses('same rows and head size', spc.norm_rotary, q, q[:2], None, None, f, positions=p)
    refuses('one type', spc.norm_rotary, q.half(), q.half(), torch.ones(8, device=DEV),
            torch.ones(8, device=DEV).half(), f, positions=p)
    refuses('eps', spc.norm_rotary, q, q, None, None, f, positions=p, eps=-1.0)
    x = torch.rand(3, 2, device=DEV)
    refuses('same size', spc.linear_recurrence, x, x[:, :1], b)
    refuses('same type', spc.linear_recurrence, x, x.half(), b)
    refuses('size 2 at dimension 1', spc.linear_recurrence, x, x, b, initial=torch.rand(2, 3, device=DEV))
    refuses('scalar type', spc.linear_recurrence, x.int(), x.int(), b)


@pytest.mark.gpu
def test_second_derivatives_are_refused(spc):
    b = torch.ones(3, dtype=torch.bool, device=DEV)
    x = torch.rand(3, 2, 8, device=DEV, requires_grad=True)
    f = torch.rand(4, dtype=torch.float64, device=DEV)
    for y in (spc.linear_recurrence(x[:, 0].contiguous(), x[:, 1].contiguous(), b), spc.pack_attention(x, x, x, b),
              spc.norm_rotary(x, x, None, None, f, boundaries=b)[0]):
        with pytest.raises(RuntimeError, match='once_differentiable|create_graph=True is not supported'):
            g, = torch.autograd.grad(y.square().sum(), x, create_graph=True)
            g.sum().backward()


# ------------------------------------------------------------------------------- the pack arrays
@pytest.mark.gpu
@pytest.mark.parametrize('n', [0, 1, 5, 1023, 1024, 1025, 40000, 65536, 65537, 200001])
@pytest.mark.parametrize('kind', ['some', 'none', 'all', 'bytes'])
def test_pack_layout(n, kind):
    import kaolin
    gen = torch.Generator().manual_seed(n)
    b = torch.rand(n, generator=gen) < 0.1
    if kind in ('none', 'all'):
        b[:] = kind == 'all'
    mask = b
    if kind == 'bytes':  # any byte that is not 0 marks a row; an odd address
        mask = torch.where(b, torch.randint(1, 256, (n,), generator=gen), 0).to(torch.uint8)
    held = torch.zeros(n + 3, dtype=mask.dtype, device=DEV)
    held[3:] = mask.to(DEV)
    ids, starts = kaolin._C.render.spc.pack_layout_cuda(held[3:])
    rows = torch.nonzero(b)[:, 0].int()
    assert torch.equal(ids.cpu(), b.long().cumsum(0).int() - 1)
    want = torch.full((n + 1,), n, dtype=torch.int32)
    want[:len(rows)] = rows
    assert torch.equal(starts.cpu(), want)


@pytest.mark.gpu
@pytest.mark.parametrize('n, m', [(1, 1), (0, 5), (1025, 3), (70001, 40), (40, 70001), (65537, 66000), (513, 0)])
def test_pack_layout_pair(n, m):
    import kaolin
    from kaolin import _native as N
    gen = torch.Generator().manual_seed(n + m)
    masks = [(torch.rand(k, generator=gen) < 0.1).to(DEV) for k in (n, m)]
    out = [(torch.full((k,), -7, dtype=torch.int32, device=DEV), torch.full((k + 1,), -7, dtype=torch.int32, device=DEV))
           for k in (n, m)]
    size = sum(N.size('kl_pack_layout_workspace_bytes', k) for k in (n, m))
    ws = N.workspace(size, masks[0].device)
    args = [x for k, mask, o in zip((n, m), masks, out) for x in (k, N.ptr(mask), N.ptr(o[0]), N.ptr(o[1]))]
    N.check(N.lib().kl_pack_layout_pair(*args, N.ptr(ws), size, N.stream_of(masks[0].device)), 'pack_layout_pair')
    for mask, o in zip(masks, out):
        want = kaolin._C.render.spc.pack_layout_cuda(mask)
        assert torch.equal(o[0], want[0]) and torch.equal(o[1], want[1])


# ------------------------------------------------------------------------------- attention
CASES = [  # dim, heads, kv_heads, lengths, rows of no pack first, causal
    (32, 4, 4, [24, 1, 95, 3, 2, 7, 31, 32, 33], 0, False),
    (64, 4, 2, [70, 130, 3], 2, True),
    (128, 6, 2, [300, 1, 17], 0, True),
    (80, 3, 1, [65, 64, 1, 63], 5, False),
    (8, 1, 1, [1], 0, False),
    (16, 8, 1, [200], 0, True),
    (24, 5, 5, [1] * 70, 1, True),
    (96, 12, 3, [129, 2], 130, True),
    (104, 7, 1, [257], 0, False),
]


def _attention_inputs(dtype, case, seed=0):
    dim, heads, kv, lens, lead, causal = case
    b = marks(lens, lead)
    q, k, v, g = (_normal(seed + i, len(b), h, dim, dtype=dtype) for i, h in enumerate((heads, kv, kv, heads)))
    return b, q, k, v, g, causal


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('case', CASES)
def test_attention_against_64_bits(spc, dtype, case):
    b, q, k, v, g, causal = _attention_inputs(dtype, case)
    outs, tols = attention(q, k, v, b, causal=causal, grad=g, dtype=dtype)
    leaves = [_leaf(x) for x in (q, k, v)]
    o = spc.pack_attention(*leaves, b.to(DEV), causal=causal)
    assert o.dtype == dtype and o.is_contiguous()
    got = [o, *torch.autograd.grad(o, leaves, g.to(DEV))]
    for name, x, want, tol in zip(('o', 'dq', 'dk', 'dv'), got, outs, tols):
        check(name, x, want, tol)
    with torch.no_grad():  # without a backward to come: the same output
        assert torch.equal(spc.pack_attention(*leaves, b.to(DEV), causal=causal), o)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('lens,q_lens,heads,kv,dim,causal', [
    ([24, 1, 95, 3], [1, 1, 1, 1], 4, 2, 32, False),
    ([1500, 1, 700], [1, 1, 1], 8, 1, 64, True),
    ([5, 9, 300], [2, 9, 33], 2, 2, 16, True),       # the last rows of each sequence
    ([5, 9, 3], [2, 12, 3], 2, 1, 48, True),         # more queries than keys: the first of them see none
    ([5, 9], [2, 3, 4], 2, 1, 8, False),             # the last pack of queries has no keys
    ([5, 9, 4], [2, 3], 2, 1, 128, False),           # nobody asks for the last pack of keys
    ([3000], [1], 16, 2, 128, True),
    ([130, 140], [260, 3], 3, 3, 40, False),
])
def test_attention_across(spc, dtype, lens, q_lens, heads, kv, dim, causal):
    b, qb = marks(lens), marks(q_lens)
    q, g = (_normal(i, len(qb), heads, dim, dtype=dtype) for i in range(2))
    k, v = (_normal(2 + i, len(b), kv, dim, dtype=dtype) for i in range(2))
    outs, tols = attention(q, k, v, b, qb, causal, grad=g, dtype=dtype)
    leaves = [_leaf(x) for x in (q, k, v)]
    o = spc.pack_attention(*leaves, b.to(DEV), q_boundaries=qb.to(DEV), causal=causal)
    got = [o, *torch.autograd.grad(o, leaves, g.to(DEV))]
    for name, x, want, tol in zip(('o', 'dq', 'dk', 'dv'), got, outs, tols):
        check(name, x, want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
def test_attention_rows_that_see_nothing(spc, dtype):
    q, k, v = (_leaf(_normal(i, 6, 2, 16, dtype=dtype)) for i in range(3))
    none = torch.zeros(6, dtype=torch.bool, device=DEV)
    o = spc.pack_attention(q, k, v, none)
    assert not o.any()
    for x in torch.autograd.grad(o, (q, k, v), torch.ones_like(o)):
        assert not x.any()
    e = torch.zeros(0, 2, 16, dtype=dtype, device=DEV, requires_grad=True)
    o = spc.pack_attention(e, e, e, none[:0])
    assert o.shape == (0, 2, 16) and torch.autograd.grad(o.sum(), e)[0].shape == (0, 2, 16)
    o = spc.pack_attention(q, e, e, none[:0], q_boundaries=~none)  # queries without any keys
    dq, dk = torch.autograd.grad(o, (q, e), torch.ones_like(o))
    assert not o.any() and not dq.any() and dk.shape == (0, 2, 16)
    o = spc.pack_attention(e, k, v, ~none, q_boundaries=none[:0])  # keys without any queries
    assert o.shape == (0, 2, 16)
    dk, dv = torch.autograd.grad(o, (k, v), torch.ones_like(o))
    assert not dk.any() and not dv.any()


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('bad', [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize('causal', [False, True])
def test_attention_masked_places_do_not_leak(spc, dtype, bad, causal):
    """Infinities and NaN in one pack (and, causal, in a pack's last rows) leave every row that does not see
    them as it is without them, in the output and in all gradients."""
    b = marks([40, 30, 90], lead=3)
    q, k, v, g = (_normal(i, len(b), h, 32, dtype=dtype) for i, h in enumerate((4, 2, 2, 4)))
    if causal:  # rows 150.. of the last pack: the rows before them do not see them
        dirty_rows = torch.cat((torch.arange(43, 73), torch.arange(150, len(b)), torch.arange(3)))
    else:
        dirty_rows = torch.cat((torch.arange(43, 73), torch.arange(3)))
    clean = torch.ones(len(b), dtype=torch.bool)
    clean[dirty_rows] = False
    outs, tols = attention(q, k, v, b, causal=causal, grad=torch.where(clean[:, None, None], g, 0).to(dtype), dtype=dtype)
    xs = []
    for i, x in enumerate((q, k, v)):
        x = x.clone()
        x[dirty_rows[i::3]] = bad
        xs.append(_leaf(x))
    o = spc.pack_attention(*xs, b.to(DEV), causal=causal)
    gg = torch.where(clean[:, None, None], g, 0).to(dtype)
    got = [o, *torch.autograd.grad(o, xs, gg.to(DEV))]
    for name, x, want, tol in zip(('o', 'dq', 'dk', 'dv'), got, outs, tols):
        rows = clean
        if name in ('dk', 'dv') and causal:
            continue  # rows before 150 are seen by the dirty ones: their gradients are those rows' own
        check(name, x.cpu()[rows], want[rows], tol[rows])
    if math.isnan(bad):  # and rows that do see them show it
        seen = o.cpu()[43:73]
        assert torch.isnan(seen).all()


@pytest.mark.gpu
def test_attention_seen_infinities(spc):
    """A value of infinity that a row sees is in its output; a key that scores -inf has no weight."""
    b = marks([3]).to(DEV)
    q = torch.ones(3, 1, 8, device=DEV)
    k, v = torch.zeros(3, 1, 8, device=DEV), torch.ones(3, 1, 8, device=DEV)
    k[2] = -math.inf
    v[1, 0, 3] = math.inf
    o = spc.pack_attention(q, k, v, b)
    want = torch.ones(3, 1, 8)
    want[:, 0, 3] = math.inf
    assert torch.equal(o.cpu(), want)
    k[2] = math.inf
    assert torch.isnan(spc.pack_attention(q, k, v, b)).all()


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('lens,heads', [([5, 300], 1), ([5, 4096], 32)])  # with the keys split and not
def test_attention_scores_all_minus_infinity(spc, dtype, lens, heads):
    """A row whose keys all score -inf has no softmax (0 / 0), unlike one that sees no key, which is 0; the other
    pack's rows have theirs."""
    b = marks(lens, lead=2)
    n = len(b)
    q, k, v = (torch.ones(n, heads, 8, dtype=dtype) for _ in range(3))
    k[2:7] = -math.inf
    leaves = [_leaf(x) for x in (q, k, v)]
    o = spc.pack_attention(*leaves, b.to(DEV))
    dq, _, dv = torch.autograd.grad(o, leaves, torch.ones_like(o))
    for x in (o, dq, dv):
        assert not x[:2].any() and torch.isnan(x[2:7]).all()
    assert torch.equal(o[7:], torch.ones_like(o[7:])) and torch.isfinite(dq[7:]).all()
    one = spc.pack_attention(leaves[0][6:8].detach(), leaves[1].detach(), leaves[2].detach(), b.to(DEV),
                             q_boundaries=torch.ones(2, dtype=torch.bool, device=DEV))
    assert torch.isnan(one[0]).all() and torch.equal(one[1], torch.ones_like(one[1]))


@pytest.mark.gpu
def test_single_rows_of_any_stride(spc):
    """The stride of a dimension of size one is whatever a view made it."""
    x = _normal(0, 16).to(DEV)
    far, b = x.as_strided((1, 2, 8), (1 << 40, 8, 1)), torch.ones(1, dtype=torch.bool, device=DEV)
    near, f = x.view(1, 2, 8), torch.ones(4, dtype=torch.float64, device=DEV)
    assert torch.equal(spc.pack_attention(far, far, far, b), spc.pack_attention(near, near, near, b))
    for y, want in zip(spc.norm_rotary(far, far, None, None, f, boundaries=b),
                       spc.norm_rotary(near, near, None, None, f, boundaries=b)):
        assert torch.equal(y, want)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
def test_attention_strides(spc, dtype):
    """Slices of one projection, heads in another order, expanded keys, a view that has to be copied: as the
    contiguous call."""
    b = marks([50, 20, 41]).to(DEV)
    n = len(b)
    x = _normal(0, n, 10 * 16, dtype=dtype).to(DEV)
    heads = x.view(n, 10, 16)
    q, k, v = heads[:, :6], heads[:, 6:8], heads[:, 8:]
    want = spc.pack_attention(q.contiguous(), k.contiguous(), v.contiguous(), b, causal=True)
    assert torch.equal(spc.pack_attention(q, k, v, b, causal=True), want)
    swapped = q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(spc.pack_attention(swapped, k, v, b, causal=True), want)
    columns = q.transpose(1, 2).contiguous().transpose(1, 2)
    assert columns.stride(2) != 1 and torch.equal(spc.pack_attention(columns, k, v, b, causal=True), want)
    odd = torch.empty(n * 96 + 1, dtype=dtype, device=DEV)[1:].view(n, 6, 16)
    odd.copy_(q)
    assert torch.equal(spc.pack_attention(odd, k, v, b, causal=True), want)
    one = k[:, :1].expand(n, 2, 16)
    assert torch.equal(spc.pack_attention(q, one, one, b), spc.pack_attention(q, one.contiguous(), one.contiguous(), b))
    mask = torch.zeros(2 * n, dtype=torch.bool, device=DEV)
    mask[::2] = b
    assert torch.equal(spc.pack_attention(q, k, v, mask[::2], causal=True), want)
    # the gradient of an expanded result and of an expanded input
    leaf = _leaf(k[:, :1].detach())
    o = spc.pack_attention(q, leaf.expand(n, 2, 16), v, b)
    dk, = torch.autograd.grad(o.sum(), leaf)
    two = _leaf(k[:, :1].expand(n, 2, 16).detach().contiguous())
    dk2, = torch.autograd.grad(spc.pack_attention(q, two, v, b).sum(), two)
    assert torch.equal(dk, dk2.sum(1, keepdim=True))


@pytest.mark.gpu
def test_attention_which_gradients(spc):
    b = marks([50, 20]).to(DEV)
    q, k, v = (_leaf(_normal(i, 70, 2, 16)) for i in range(3))
    full = torch.autograd.grad(spc.pack_attention(q, k, v, b).sum(), (q, k, v))
    for want, x, args in ((full[0], q, (q, k.detach(), v.detach())), (full[1], k, (q.detach(), k, v.detach())),
                          (full[2], v, (q.detach(), k.detach(), v))):
        got, = torch.autograd.grad(spc.pack_attention(*args, b).sum(), x)
        assert torch.equal(got, want)
    same = _leaf(q.detach())
    got, = torch.autograd.grad(spc.pack_attention(same, same, same, b).sum(), same)
    three = [_leaf(q.detach()) for _ in range(3)]
    parts = torch.autograd.grad(spc.pack_attention(*three, b).sum(), three)
    # two additions of the same three values, in an order of torch's choice: within two roundings of it
    assert ((got - sum(parts)).abs() <= 2 ** -22 * sum(p.abs() for p in parts)).all()


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
def test_attention_extreme_scores(spc, dtype):
    """Scores of thousands: the softmax is one key's, and small float16 gradients keep their bits."""
    b = marks([30, 200])
    q, k, v, g = (_normal(i, 230, 2, 64, dtype=dtype, scale=s) for i, s in enumerate((30.0, 30.0, 1.0, 1e-4)))
    outs, tols = attention(q, k, v, b, causal=True, grad=g, dtype=dtype)
    leaves = [_leaf(x) for x in (q, k, v)]
    o = spc.pack_attention(*leaves, b.to(DEV), causal=True)
    got = [o, *torch.autograd.grad(o, leaves, g.to(DEV))]
    for name, x, want, tol in zip(('o', 'dq', 'dk', 'dv'), got, outs, tols):
        check(name, x, want, tol)


@pytest.mark.gpu
def test_attention_small_float16_gradients(spc):
    """Gradients near float16's smallest numbers come out as the formula's, rounded to it."""
    b = marks([64])
    q, k, v, g = (_normal(i, 64, 1, 32, dtype=torch.float16, scale=s) for i, s in enumerate((1.0, 1.0, 1.0, 1e-5)))
    outs, tols = attention(q, k, v, b, grad=g, dtype=torch.float16)
    leaves = [_leaf(x) for x in (q, k, v)]
    o = spc.pack_attention(*leaves, b.to(DEV))
    for name, x, want, tol in zip(('dq', 'dk', 'dv'), torch.autograd.grad(o, leaves, g.to(DEV)), outs[1:], tols[1:]):
        check(name, x, want, tol)
        assert float(x.float().norm()) > 0.9 * float(want.norm())


@pytest.mark.gpu
def test_attention_offsets_past_32_bits(spc):
    """Rows that lie more than 2^31 elements apart."""
    n, stride = 300, 8_000_000
    held = torch.zeros((n - 1) * stride + 64, dtype=torch.float16, device=DEV)
    k = held.as_strided((n, 1, 16), (stride, 16, 1))
    v = held.as_strided((n, 1, 16), (stride, 16, 1), 16)
    q = held.as_strided((n, 2, 16), (stride, 16, 1), 32)
    for i, x in enumerate((k, v, q)):
        x.copy_(_normal(i, *x.shape, dtype=torch.float16))
    b = marks([7, 290, 3]).to(DEV)
    assert held.numel() > 1 << 31
    o = spc.pack_attention(q, k, v, b)
    assert torch.equal(o, spc.pack_attention(q.contiguous(), k.contiguous(), v.contiguous(), b))
    f = torch.rand(8, dtype=torch.float64, device=DEV)
    pos = torch.arange(n, device=DEV)
    for x, y in zip(spc.norm_rotary(q, k, None, None, f, positions=pos),
                    spc.norm_rotary(q.contiguous(), k.contiguous(), None, None, f, positions=pos)):
        assert torch.equal(x, y)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype,n,dim', [(torch.float16, 130, 64), (torch.float32, 70, 64), (torch.float32, 70, 32)])
def test_attention_rows_as_far_apart_as_allowed(spc, dtype, n, dim):
    """A tile's rows span all but 2^32 bytes; rows further apart than that are copied first."""
    stride = (1 << 25) - 8
    held = torch.empty((n - 1) * stride + 3 * dim, dtype=dtype, device=DEV)
    far = [held.as_strided((n, 1, dim), (stride, dim, 1), i * dim) for i in range(3)]
    near = [_normal(i, n, 1, dim, dtype=dtype).to(DEV) for i in range(3)]
    for x, y in zip(far, near):
        x.copy_(y)
    b, g = marks([3, n - 7, 4]).to(DEV), _normal(5, n, 1, dim, dtype=dtype).to(DEV)
    got = []
    for xs in (far, near):
        leaves = [x.detach().requires_grad_() for x in xs]
        o = spc.pack_attention(*leaves, b, causal=True)
        got.append([o, *torch.autograd.grad(o, leaves, g)])
    for x, y in zip(*got):
        assert torch.equal(x, y)
    further = held.as_strided((9, 1, dim), (6 * stride, dim, 1))
    assert torch.equal(spc.pack_attention(further, further, further, b[:9]),
                       spc.pack_attention(further.contiguous(), further.contiguous(), further.contiguous(), b[:9]))


# ------------------------------------------------------------------------------- norm and rotation
@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('rows,heads,kv,dim,turn', [
    (7, 4, 2, 64, 64), (1, 32, 8, 128, 128), (130, 3, 1, 80, 40), (33, 1, 1, 8, 4), (5, 2, 2, 16, 0), (19, 2, 1, 256, 250),
    (300, 5, 3, 24, 6), (65, 0, 2, 32, 32), (65, 2, 0, 32, 2), (2051, 1, 1, 40, 20),
])
@pytest.mark.parametrize('interleaved', [False, True])
def test_norm_rotary_against_64_bits(spc, dtype, rows, heads, kv, dim, turn, interleaved):
    x = {'q': _normal(0, rows, heads, dim, dtype=dtype, scale=3.0), 'k': _normal(1, rows, kv, dim, dtype=dtype)}
    w = {n: (1 + _normal(2 + i, dim, scale=0.3)).to(dtype) for i, n in enumerate('qk')}
    g = {n: _normal(4 + i, *x[n].shape, dtype=dtype) for i, n in enumerate('qk')}
    f = 10000.0 ** (-torch.arange(turn // 2).double() * 2 / max(turn, 1))
    pos = torch.randint(0, 1 << 20, (rows,), generator=torch.Generator().manual_seed(3))
    xs, ws = {n: _leaf(x[n]) for n in 'qk'}, {n: _leaf(w[n]) for n in 'qk'}
    y = dict(zip('qk', spc.norm_rotary(xs['q'], xs['k'], ws['q'], ws['k'], f.to(DEV), positions=pos.to(DEV), eps=1e-5,
                                       interleaved=interleaved)))
    grads = torch.autograd.grad([y[n] for n in 'qk'], [xs['q'], xs['k'], ws['q'], ws['k']], [g[n].to(DEV) for n in 'qk'])
    for i, n in enumerate('qk'):
        outs, tols = norm_rotary(x[n], w[n], f, pos, 1e-5, interleaved, grad=g[n], dtype=dtype)
        for name, got, want, tol in zip(('y', 'dx', 'dw'), (y[n], grads[i], grads[2 + i]), outs, tols):
            assert got.dtype == dtype
            check(f'{name} of {n}', got, want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
def test_norm_rotary_positions(spc, dtype):
    """Places in packs, int32 and int64 positions, and depths; f32 weights, one weight, no weights."""
    b = marks([5, 1, 40], lead=3)
    n = len(b)
    q, k = _normal(0, n, 2, 32, dtype=dtype), _normal(1, n, 1, 32, dtype=dtype)
    f = 100.0 ** (-torch.arange(8).double() / 8)
    place = torch.cat([torch.zeros(3, dtype=torch.long)] + [torch.arange(e - s) for s, e in spans(b)])
    wide = _leaf(1 + _normal(2, 32, scale=0.2))
    yq, yk = spc.norm_rotary(q.to(DEV), k.to(DEV), wide, None, f.to(DEV), boundaries=b.to(DEV))
    for got, x, w in ((yq, q, wide.detach().cpu()), (yk, k, None)):
        (want,), (tol,) = norm_rotary(x, w, f, place, 1e-6, False, dtype=dtype)
        check('y', got, want, tol)
    for t in (torch.int32, torch.int64, torch.float32):
        again = spc.norm_rotary(q.to(DEV), k.to(DEV), wide, None, f.to(DEV), positions=place.to(DEV).to(t))
        assert torch.equal(again[0], yq) and torch.equal(again[1], yk)
    dw, = torch.autograd.grad(yq, wide, torch.ones_like(yq))
    assert dw.dtype == torch.float32
    outs, tols = norm_rotary(q, wide.detach().cpu(), f, place, 1e-6, False, grad=torch.ones(n, 2, 32), dtype=dtype,
                             w_dtype=torch.float32)
    check('dw', dw, outs[2], tols[2])
    far = (torch.rand(n, generator=torch.Generator().manual_seed(5)) * 1e6 - 5e5).float()
    yq, yk = spc.norm_rotary(q.to(DEV), k.to(DEV), None, None, f.to(DEV), positions=far.to(DEV), interleaved=True)
    for got, x in ((yq, q), (yk, k)):
        (want,), (tol,) = norm_rotary(x, None, f, far, 1e-6, True, dtype=dtype)
        check('y', got, want, tol)


@pytest.mark.gpu
def test_norm_rotary_strides_and_empty(spc):
    n = 37
    x = _normal(0, n, 8 * 24, dtype=torch.bfloat16).to(DEV).view(n, 8, 24)
    f = torch.rand(12, dtype=torch.float64, device=DEV)
    pos = torch.arange(n, device=DEV)
    want = spc.norm_rotary(x[:, :5].contiguous(), x[:, 5:7].contiguous(), None, None, f, positions=pos)
    got = spc.norm_rotary(x[:, :5], x[:, 5:7], None, None, f, positions=pos)
    odd = torch.empty(n * 120 + 1, dtype=torch.bfloat16, device=DEV)[1:].view(n, 5, 24)
    odd.copy_(x[:, :5])
    again = spc.norm_rotary(odd, x[:, 5:7], None, None, f, positions=torch.stack((pos, pos), 1)[:, 0])
    for a, b, c in zip(got, want, again):
        assert torch.equal(a, b) and torch.equal(a, c)
    e = _leaf(torch.zeros(0, 2, 8))
    w = _leaf(torch.ones(8))
    yq, yk = spc.norm_rotary(e, e, w, w, f[:4], positions=pos[:0])
    assert yq.shape == (0, 2, 8)
    dw, = torch.autograd.grad(yq.sum() + yk.sum(), w)
    assert not dw.any()


# ------------------------------------------------------------------------------- recurrence
@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES + [torch.float64])
@pytest.mark.parametrize('lens,lead,dim', [
    ([1], 0, 1), ([24, 1, 95, 3, 2], 0, 64), ([5, 1, 1, 7], 3, 5), ([400], 0, 12), ([1] * 50, 0, 4), ([90, 700, 40], 17, 3),
    ([], 9, 2),
])
@pytest.mark.parametrize('reverse', [False, True])
@pytest.mark.parametrize('first', ['none', 'all', 'some'])
def test_recurrence_against_64_bits(spc, dtype, lens, lead, dim, reverse, first):
    b = marks(lens, lead)
    n = len(b)
    a = torch.sigmoid(_normal(0, n, dim, scale=3.0) + 2).to(dtype) * torch.where(_normal(5, n, dim) > -1, 1, -1).to(dtype)
    x, g = _normal(1, n, dim, dtype=dtype), _normal(2, n, dim, dtype=dtype)
    count = {'none': None, 'all': len(lens), 'some': len(lens) // 2}[first]
    h0 = None if count is None else _normal(3, count, dim, dtype=dtype)
    outs, tols = recurrence(a, x, b, h0, reverse, grad=g, dtype=dtype)
    leaves = [_leaf(y) for y in (a, x, h0)]
    h = spc.linear_recurrence(leaves[0], leaves[1], b.to(DEV), initial=leaves[2], reverse=reverse)
    assert h.dtype == dtype
    got = [h, *torch.autograd.grad(h, [y for y in leaves if y is not None], g.to(DEV))]
    for name, y, want, tol in zip(('h', 'da', 'db', 'dinitial'), got, outs, tols):
        check(name, y, want, tol)


@pytest.mark.gpu
def test_recurrence_more_initial_rows_than_packs(spc):
    """Rows of `initial` that no pack has: no effect, gradient 0."""
    b = marks([4, 3], lead=1).to(DEV)
    a, x = (_leaf(_normal(i, 8, 6)) for i in range(2))
    h0 = _leaf(_normal(2, 12, 6))
    h = spc.linear_recurrence(a, x, b, initial=h0)
    d, = torch.autograd.grad(h.sum(), h0)
    assert torch.equal(h, spc.linear_recurrence(a, x, b, initial=h0[:2])) and not d[2:].any() and d[:2].all()
    e = torch.zeros(0, 6, device=DEV, requires_grad=True)
    h = spc.linear_recurrence(e, e, b[:0], initial=h0)
    assert h.shape == (0, 6)
    d, = torch.autograd.grad(h.sum(), h0)
    assert not d.any()


@pytest.mark.gpu
@pytest.mark.parametrize('reverse', [False, True])
def test_recurrence_packs_do_not_touch(spc, reverse):
    """Infinities and NaN of one pack stay in it, over many chunks of rows."""
    lens = [500, 300, 700]
    b = marks(lens, lead=20)
    n = len(b)
    a, x, g = (_normal(i, n, 8, scale=s) for i, s in enumerate((0.5, 1.0, 1.0)))
    outs, tols = recurrence(a, x, b, None, reverse, grad=g, dtype=torch.float32)
    a2, x2 = a.clone(), x.clone()
    dirty = torch.cat((torch.arange(20), torch.arange(520, 820)))
    a2[dirty[::3]] = math.nan
    x2[dirty[1::3]] = math.inf
    leaves = [_leaf(y) for y in (a2, x2)]
    h = spc.linear_recurrence(*leaves, b.to(DEV), reverse=reverse)
    got = [h, *torch.autograd.grad(h, leaves, g.to(DEV))]
    clean = torch.ones(n, dtype=torch.bool)
    clean[dirty] = False
    for name, y, want, tol in zip(('h', 'da', 'db'), got, outs, tols):
        check(name, y.cpu()[clean], want[clean], tol[clean])
        assert not y[:20].any()
    assert not torch.isfinite(h[520:820]).all()


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES + [torch.float64])
@pytest.mark.parametrize('lens,lead', [([2], 0), ([63, 1], 0), ([64, 1], 0), ([1, 64], 5), ([100, 156], 0), ([256], 0),
                                       ([250], 6), ([257], 0), ([1] * 200 + [56], 0), ([3, 190, 60], 3)])
@pytest.mark.parametrize('reverse', [False, True])
def test_recurrence_few_rows(spc, dtype, lens, lead, reverse):
    """Rows that fit one workgroup, with an infinity and a NaN in the packs next to the one that is compared."""
    b = marks(lens, lead)
    n, dim = len(b), 16
    a, x, g = (_normal(i, n, dim, scale=s, dtype=dtype) for i, s in enumerate((0.5, 1.0, 1.0)))
    h0 = _normal(3, len(lens), dim, dtype=dtype)
    outs, tols = recurrence(a, x, b, h0, reverse, grad=g, dtype=dtype)
    which = lens.index(max(lens))
    begin = lead + sum(lens[:which])
    others = torch.ones(n, dtype=torch.bool)
    others[begin:begin + lens[which]] = False
    a, x = a.clone(), x.clone()
    a[others & (torch.arange(n) % 2 == 0)] = math.nan
    x[others] = math.inf
    leaves = [_leaf(y) for y in (a, x, h0)]
    h = spc.linear_recurrence(leaves[0], leaves[1], b.to(DEV), initial=leaves[2], reverse=reverse)
    got = [h, *torch.autograd.grad(h, leaves, g.to(DEV))]
    for name, y, want, tol in zip(('h', 'da', 'db', 'dinitial'), got, outs, tols):
        rows = slice(which, which + 1) if name == 'dinitial' else ~others
        check(name, y.cpu()[rows], want[rows], tol[rows])


@pytest.mark.gpu
@pytest.mark.parametrize('dtype,dim', [(torch.float32, 131), (torch.float16, 269), (torch.bfloat16, 268),
                                       (torch.float64, 67)])
@pytest.mark.parametrize('reverse', [False, True])
def test_recurrence_rows_of_odd_length(spc, dtype, dim, reverse):
    """Enough rows for pieces of 16 bytes where a row is not a whole number of them."""
    b = marks([1500, 1, 2400, 99], lead=30)
    n = len(b)
    a = torch.sigmoid(_normal(0, n, dim, scale=3.0) + 2).to(dtype)
    x, g, h0 = _normal(1, n, dim, dtype=dtype), _normal(2, n, dim, dtype=dtype), _normal(3, 4, dim, dtype=dtype)
    outs, tols = recurrence(a, x, b, h0, reverse, grad=g, dtype=dtype)
    leaves = [_leaf(y) for y in (a, x, h0)]
    h = spc.linear_recurrence(leaves[0], leaves[1], b.to(DEV), initial=leaves[2], reverse=reverse)
    got = [h, *torch.autograd.grad(h, leaves, g.to(DEV))]
    for name, y, want, tol in zip(('h', 'da', 'db', 'dinitial'), got, outs, tols):
        check(name, y, want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('n,dim', [(40, 16), (300, 24), (5000, 269)])
def test_recurrence_at_any_address(spc, dtype, n, dim):
    b = marks([n // 3, n - n // 3]).to(DEV)
    near = [_normal(i, n, dim, dtype=dtype).to(DEV) for i in range(3)]
    odd = []
    for x in near:
        odd.append(torch.empty(n * dim + 1, dtype=dtype, device=DEV)[1:].view(n, dim))
        odd[-1].copy_(x)
    got = []
    for a, x, g in (near, odd):
        leaves = [a.detach().requires_grad_(), x.detach().requires_grad_()]
        h = spc.linear_recurrence(*leaves, b)
        got.append([h, *torch.autograd.grad(h, leaves, g)])
    for y, z in zip(*got):
        assert torch.equal(y, z)


@pytest.mark.gpu
def test_recurrence_is_cumsum_with_gates_of_one(spc):
    b = marks([30, 1, 300], lead=2).to(DEV)
    x = torch.randint(-8, 8, (333, 7), generator=torch.Generator().manual_seed(0)).float().to(DEV)
    for rev in (False, True):  # whole numbers: exact in any order
        assert torch.equal(spc.linear_recurrence(torch.ones_like(x), x, b, reverse=rev), spc.cumsum(x, b, reverse=rev))


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('n,dim', [(70001, 8), (33000, 72), (9000, 260), (900, 64), (4001, 72), (6000, 260), (30000, 8),
                                   (2500, 5)])
def test_recurrence_long(spc, dtype, n, dim):
    """Sizes at which chunks are many and long, against the same rows as many short calls would give them."""
    b = torch.zeros(n, dtype=torch.bool)
    b[[0, 11, n // 3]] = True
    a = (0.9 + 0.1 * torch.rand(n, dim, generator=torch.Generator().manual_seed(1))).to(dtype)
    x = _normal(2, n, dim, dtype=dtype)
    h = spc.linear_recurrence(a.to(DEV), x.to(DEV), b.to(DEV)).double().cpu()
    state, size = torch.zeros(dim, dtype=torch.float64), torch.zeros(dim, dtype=torch.float64)
    ad, xd = a.double(), x.double()
    want, bound = torch.empty_like(xd), torch.empty_like(xd)
    for t in range(n):
        if b[t]:
            state, size = torch.zeros_like(state), torch.zeros_like(size)
        state, size = ad[t] * state + xd[t], ad[t] * size + xd[t].abs()
        want[t], bound[t] = state, size
    # gates under 1: an error made s rows ago has shrunk by their product, which `size` has too; over 300 rows of
    # gates near 0.95 nothing is left of it, so 300 roundings of the size bound it
    u = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}[dtype]
    check('h', h, want, u * want.abs() + 300 * 2.0 ** -24 * bound)


# ------------------------------------------------------------------------------- repeated, captured, elsewhere
def _model(spc, p, x, boundaries, depth):
    """One layer along rays: projection, norm and rotation by depth, attention, recurrence, integration."""
    n = x.shape[0]
    z = (x @ p['in']).view(n, 8, 16)
    q, k = spc.norm_rotary(z[:, :4], z[:, 4:6], p['qw'], p['kw'], p['freqs'], positions=depth)
    o = spc.pack_attention(q, k, z[:, 6:], boundaries, causal=True).reshape(n, 64)
    gates = torch.sigmoid(x @ p['gate'])
    h = spc.linear_recurrence(gates, o @ p['out'], boundaries)
    return h


def _model_inputs(dtype=torch.float32, lens=(24, 1, 60, 7, 33)):
    b = marks(list(lens))
    n = len(b)
    p = {'in': _normal(0, 24, 128, scale=0.2, dtype=dtype), 'gate': _normal(1, 24, 12, dtype=dtype),
         'out': _normal(2, 64, 12, scale=0.1, dtype=dtype), 'qw': (1 + _normal(3, 16, scale=0.1)).to(dtype),
         'kw': (1 + _normal(4, 16, scale=0.1)).to(dtype), 'freqs': 10.0 ** -torch.arange(4).double()}
    return b, p, _normal(5, n, 24, dtype=dtype), torch.rand(n, generator=torch.Generator().manual_seed(6)) * 10


@pytest.mark.gpu
def test_together_against_64_bits(spc):
    """The three operators in a row, then the packed ray ops, forward and backward, against torch in 64 bits."""
    b, p, x, depth = _model_inputs()
    names = [n for n in p if n != 'freqs']

    def plain(p, x):
        n = len(x)
        z = (x @ p['in']).view(n, 8, 16)

        def turn(y, w):
            y = y * (y.pow(2).mean(-1, keepdim=True) + 1e-6).rsqrt() * w
            angle = depth.double()[:, None, None] * p['freqs']
            a, c = y[..., :4], y[..., 4:8]
            return torch.cat((a * angle.cos() - c * angle.sin(), a * angle.sin() + c * angle.cos(), y[..., 8:]), -1)
        q, k, v = turn(z[:, :4], p['qw']), turn(z[:, 4:6], p['kw']), z[:, 6:]
        same = (b.long().cumsum(0)[:, None] == b.long().cumsum(0)).tril()
        s = torch.einsum('ihd,jhd->hij', q, k.repeat_interleave(2, 1)) / 4
        w = s.masked_fill(~same, -math.inf).softmax(-1)
        o = torch.einsum('hij,jhd->ihd', w, v.repeat_interleave(2, 1)).reshape(n, 64) @ p['out']
        gates, rows = torch.sigmoid(x @ p['gate']), []
        for t in range(n):
            rows.append(o[t] if b[t] else gates[t] * rows[-1] + o[t])
        h = torch.stack(rows)
        return torch.stack([h[s:e].sum(0) for s, e in spans(b)]), h
    p64 = {n: y.double().requires_grad_(n != 'freqs') for n, y in p.items()}
    want, h64 = plain(p64, x.double())
    weight = _normal(8, *want.shape).double()
    grads64 = torch.autograd.grad((want * weight).sum(), [p64[n] for n in names])
    pd = {n: _leaf(y) if n != 'freqs' else y.to(DEV) for n, y in p.items()}
    h = _model(spc, pd, x.to(DEV), b.to(DEV), depth.to(DEV))
    got = spc.sum_reduce(h, b.to(DEV))
    grads = torch.autograd.grad((got * weight.float().to(DEV)).sum(), [pd[n] for n in names])
    # some 2^10 roundings in 32 bits lie between the inputs and any of these sums, of terms that are no more than 2^4
    # times the largest result
    for name, y, y64 in (('h', h, h64), ('sums', got, want), *zip(names, grads, grads64)):
        check(name, y, y64, y64.detach().abs().max() * 2.0 ** (10 + 4 - 24))


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
def test_same_result_every_time(spc, dtype):
    b, p, x, depth = _model_inputs(dtype, lens=(300, 1, 500, 90))
    pd = {n: _leaf(y) if n != 'freqs' else y.to(DEV) for n, y in p.items()}
    runs = []
    for _ in range(3):
        h = _model(spc, pd, x.to(DEV), b.to(DEV), depth.to(DEV))
        runs.append([h, *torch.autograd.grad(h.float().square().sum(), [pd[n] for n in p if n != 'freqs'])])
    for other in runs[1:]:
        for y, z in zip(runs[0], other):
            assert torch.equal(y, z)


@pytest.mark.gpu
def test_captured_forward_and_backward(spc):
    """One graph of a forward and a backward replayed on new inputs, with eager work of the same operators between
    the replays; two graphs share no scratch."""
    b, p, x, depth = _model_inputs(lens=(300, 1, 500, 90))
    b, depth = b.to(DEV), depth.to(DEV)
    names = [n for n in p if n != 'freqs']

    def step(pd, x):
        h = _model(spc, pd, x, b, depth)
        return [h, *torch.autograd.grad(h, [pd[n] for n in names], h.detach())]
    graphs = []
    for _ in range(2):
        static = {n: _leaf(y) if n != 'freqs' else y.to(DEV) for n, y in p.items()}
        sx = x.to(DEV)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(static, sx)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(static, sx)
        graphs.append((g, sx, out, static))  # a graph reads its parameters where they were
    eager = {n: _leaf(y) if n != 'freqs' else y.to(DEV) for n, y in p.items()}
    for i in range(3):
        new = [_normal(20 + 2 * i + j, *x.shape).to(DEV) for j in range(2)]
        want = [step(eager, y) for y in new]
        for (_, sx, _, _), y in zip(graphs, new):
            sx.copy_(y)
        for g, _, _, _ in graphs:
            g.replay()
        step(eager, new[0])
        torch.cuda.synchronize()
        for (_, _, out, _), w in zip(graphs, want):
            for y, z in zip(out, w):
                assert torch.equal(y, z)


@pytest.mark.gpu
def test_captured_boundaries_change(spc):
    """The packs of a captured call are read when it is replayed."""
    q, k, v = (_normal(i, 90, 2, 16).to(DEV) for i in range(3))
    a, x = (_normal(3 + i, 90, 5).to(DEV) for i in range(2))
    b = marks([90]).to(DEV)
    f = torch.rand(4, dtype=torch.float64, device=DEV)

    def step():
        y = spc.norm_rotary(q, k, None, None, f, boundaries=b)
        return [*y, spc.pack_attention(*y, v, b, causal=True), spc.linear_recurrence(a, x, b)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for lens in ([40, 50], [1] * 90, [3, 87], [90]):
        b.copy_(marks(lens))
        g.replay()
        torch.cuda.synchronize()
        for y, z in zip(out, step()):
            assert torch.equal(y, z)


@pytest.mark.gpu
def test_other_streams(spc):
    """The same calls on two streams at once: each has scratch of its own."""
    b, p, x, depth = _model_inputs(lens=(300, 1, 500, 90))
    pd = {n: y.to(DEV) for n, y in p.items()}
    b, x, depth = b.to(DEV), x.to(DEV), depth.to(DEV)
    one = marks([1] * 90 + [1]).to(DEV)[:4]
    want = _model(spc, pd, x, b, depth)
    k = _normal(9, 891, 1, 16).to(DEV)
    q = _normal(10, 4, 1, 16).to(DEV)
    want2 = spc.pack_attention(q, k, k, b, q_boundaries=one)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append((_model(spc, pd, x, b, depth), spc.pack_attention(q, k, k, b, q_boundaries=one)))
    torch.cuda.synchronize()
    for y, z in got[0] + got[1]:
        assert torch.equal(y, want) and torch.equal(z, want2)
