"""The sequence operators over packs: attention, norm with rotation, and the gated linear recurrence.

A pack is a run of consecutive rows: the samples along one ray, or one sequence of a longer kind.
`boundaries` marks the first row of each.  Every case says what it stands for in real use; `run`
computes it with elementary torch operations, or, where `own` is true, with the framework's kernels.
"""
import math
import os
import random
import sys

import torch

own = False

TYPES = {'f32': torch.float32, 'f16': torch.float16, 'bf16': torch.bfloat16}
EPS = 1e-6


# ------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one learned query per ray reads that ray's samples out (a batch of rays in a viewer)
        dict(name='attend_readout', op='attend', kind='rays', dtype='f32', packs=512, longest=64, heads=4, kv_heads=4,
             dim=32, one=True, causal=False, train=False, cut=1),
        # samples of a ray attend to each other, one training step of a radiance model on a batch of rays
        dict(name='attend_rays_train', op='attend', kind='rays', dtype='f32', packs=8192, longest=95, heads=4,
             kv_heads=4, dim=32, one=False, causal=False, train=True, cut=2),
        # whole packed sequences of very different lengths, causal, shared key heads: the forward pass
        dict(name='attend_long', op='attend', kind='long', dtype='bf16', packs=6, rows=16385, heads=32, kv_heads=8,
             dim=128, one=False, causal=True, train=False, cut=3),
        # the same kind in training
        dict(name='attend_long_train', op='attend', kind='long', dtype='bf16', packs=4, rows=8191, heads=16,
             kv_heads=4, dim=64, one=False, causal=True, train=True, cut=4),
        # one new row for each of a batch of sequences, over all rows before it
        dict(name='attend_step', op='attend', kind='mixed', dtype='f16', packs=96, longest=16384, heads=32, kv_heads=8,
             dim=128, one=True, causal=True, train=False, cut=5),
        # one new row of one very long sequence
        dict(name='attend_step_one', op='attend', kind='long', dtype='bf16', packs=1, rows=65537, heads=16, kv_heads=2,
             dim=64, one=True, causal=True, train=False, cut=6),
        # one new row of each sequence, at far positions
        dict(name='norm_rotary_step', op='norm_rotary', dtype='f16', rows=96, heads=32, kv_heads=8, dim=128,
             turn=128, interleaved=False, train=False, far=1 << 20, packed=False, cut=7),
        # queries and keys out of one fused projection of packed sequences, turned by their places in them
        dict(name='norm_rotary_long', op='norm_rotary', kind='long', dtype='bf16', packs=6, rows=16385, heads=32,
             kv_heads=8, dim=128, turn=128, interleaved=False, train=False, far=0, packed=True, cut=8),
        # samples turned by their depth along the ray, part of each head, one training step
        dict(name='norm_rotary_rays_train', op='norm_rotary', dtype='f32', rows=262147, heads=4, kv_heads=4, dim=32,
             turn=16, interleaved=True, train=True, far=0, packed=False, cut=9),
        # all rays march one sample on, from the state of the sample before
        dict(name='recur_step', op='recur', kind='rays', dtype='f32', packs=4096, longest=1, dim=64, first=True,
             reverse=False, train=False, cut=10),
        # states carried along the samples of each ray, one training step
        dict(name='recur_rays_train', op='recur', kind='rays', dtype='f32', packs=8192, longest=95, dim=64,
             first=False, reverse=False, train=True, cut=11),
        # a layer of a long-sequence model, one training step
        dict(name='recur_long_train', op='recur', kind='long', dtype='bf16', packs=2, rows=65537, dim=1024, first=True,
             reverse=False, train=True, cut=12),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(['attend', 'attend', 'attend', 'norm_rotary', 'recur', 'recur'])
    dtype = rng.choice(['f32', 'f16', 'bf16'])
    cut = rng.randrange(1 << 30)
    train = rng.random() < 0.5
    if op == 'attend':
        kind = rng.choice(['rays', 'long', 'mixed'])
        kv = rng.choice([1, 2, 3, 4, 8])
        case = dict(op=op, kind=kind, dtype=dtype, kv_heads=kv, heads=kv * rng.choice([1, 2, 3, 4]),
                    causal=rng.random() < 0.5, cut=cut)
        if kind == 'rays':
            case.update(packs=_spread(rng, 64, 6000), longest=_spread(rng, 4, 90), dim=rng.choice([8, 16, 24, 32, 64]),
                        one=rng.random() < 0.3)
            case['heads'], case['kv_heads'] = min(case['heads'], 8), min(kv, 2)
            case['heads'] -= case['heads'] % case['kv_heads']
        elif kind == 'long':
            case.update(packs=rng.randint(1, 6), rows=_spread(rng, 128, 2500 if dtype == 'f32' else 6000),
                        dim=rng.choice([32, 64, 80, 128]), one=False)
        else:
            case.update(packs=_spread(rng, 1, 100), longest=_spread(rng, 64, 16000), dim=rng.choice([32, 64, 96, 128]),
                        one=True)
        case['train'] = train and not case['one']
        return case
    if op == 'norm_rotary':
        dim = rng.choice([16, 32, 64, 80, 128])
        kv = rng.choice([1, 2, 4, 8])
        packs = rng.randint(1, 60)
        return dict(op=op, kind='long', dtype=dtype, packs=packs, rows=_spread(rng, 1, 16000) + packs, kv_heads=kv,
                    heads=kv * rng.choice([1, 2, 4]), dim=dim, turn=rng.choice([dim, dim // 2, dim // 4]), interleaved=rng.random() < 0.5, train=train,
                    far=rng.choice([0, 1 << 20]), packed=False if train else rng.random() < 0.5, cut=cut)
    kind = rng.choice(['rays', 'long'])
    case = dict(op=op, kind=kind, dtype=dtype, first=rng.random() < 0.5, reverse=rng.random() < 0.3, train=train,
                cut=cut)
    if kind == 'rays':
        case.update(packs=_spread(rng, 16, 8000), longest=_spread(rng, 1, 95), dim=_spread(rng, 1, 130))
    else:
        case.update(packs=rng.randint(1, 8), rows=_spread(rng, 1000, 60000), dim=_spread(rng, 16, 1000))
    return case


def lengths(case):
    """The rows of each pack, from the case alone."""
    rng = random.Random(case['cut'])
    n = case['packs']
    if case['kind'] == 'rays':  # many short packs, most of them well under the longest
        return [1 + int((case['longest'] - 1) * rng.random() ** 1.5) for _ in range(n)]
    if case['kind'] == 'mixed':  # sequences at every stage between the first row and the longest
        return [_spread(rng, 1, case['longest']) for _ in range(n)]
    cuts = sorted(rng.sample(range(1, case['rows']), n - 1))  # a row range cut at random places
    return [b - a for a, b in zip([0] + cuts, cuts + [case['rows']])]


def _normal(gen, *shape, scale=1.0, dtype=torch.float32):
    return (torch.randn(shape, generator=gen, device='cuda') * scale).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device='cuda').manual_seed(int(seed))
    t = TYPES[case['dtype']]
    s = dict(case)
    if case['op'] != 'norm_rotary' or case['packed']:
        lens = lengths(case)
        starts = torch.tensor([0] + lens[:-1]).cumsum(0)
        rows = sum(lens)
        boundaries = torch.zeros(rows, dtype=torch.bool)
        boundaries[starts] = True
        s.update(lens=lens, starts=starts.cuda(), boundaries=boundaries.cuda())
    train = case['train']
    if case['op'] == 'attend':
        n = case['packs'] if case['one'] else rows
        h, kv, d = case['heads'], case['kv_heads'], case['dim']
        s.update(q=_normal(gen, n, h, d, dtype=t).requires_grad_(train),
                 k=_normal(gen, rows, kv, d, dtype=t).requires_grad_(train),
                 v=_normal(gen, rows, kv, d, dtype=t).requires_grad_(train),
                 q_boundaries=torch.ones(n, dtype=torch.bool, device='cuda') if case['one'] else None)
        if train:
            s['grad'] = _normal(gen, n, h, d, scale=0.1, dtype=t)
    elif case['op'] == 'norm_rotary':
        n, h, kv, d = case['rows'], case['heads'], case['kv_heads'], case['dim']
        if case['packed']:  # one projection's output: queries, keys and values side by side
            s['qkv'] = _normal(gen, n, (h + 2 * kv) * d, scale=2.0, dtype=t)
        else:
            s.update(q=_normal(gen, n, h, d, scale=2.0, dtype=t).requires_grad_(train),
                     k=_normal(gen, n, kv, d, scale=2.0, dtype=t).requires_grad_(train))
        s.update(q_weight=(1 + _normal(gen, d, scale=0.1)).to(t).requires_grad_(train),
                 k_weight=(1 + _normal(gen, d, scale=0.1)).to(t).requires_grad_(train),
                 freqs=10000.0 ** (-torch.arange(case['turn'] // 2, device='cuda', dtype=torch.float64) * 2
                                   / case['turn']))
        if case['packed']:
            s['positions'] = None
        elif case['far']:
            s['positions'] = torch.randint(0, case['far'], (n,), generator=gen, device='cuda')
        else:  # depths along a ray, as the ray tracer gives them
            s['positions'] = torch.rand(n, generator=gen, device='cuda') * 1000
        if train:
            s.update(grad_q=_normal(gen, n, h, d, scale=0.1, dtype=t),
                     grad_k=_normal(gen, n, kv, d, scale=0.1, dtype=t))
    else:
        c = case['dim']
        s.update(gates=torch.sigmoid(_normal(gen, rows, c, scale=2.0) + 2).to(t).requires_grad_(train),
                 feats=_normal(gen, rows, c, dtype=t).requires_grad_(train),
                 initial=_normal(gen, case['packs'], c, dtype=t).requires_grad_(train) if case['first'] else None)
        if train:
            s['grad'] = _normal(gen, rows, c, scale=0.1, dtype=t)
    return s


def _pairs(case):
    if case['one']:
        return sum(lengths(case))
    return sum(n * (n + 1) // 2 if case['causal'] else n * n for n in lengths(case))


def work(case):
    size = 4 if case['dtype'] == 'f32' else 2
    if case['op'] == 'attend':
        rows = sum(lengths(case))
        n = case['packs'] if case['one'] else rows
        q, k = n * case['heads'] * case['dim'] * size, rows * case['kv_heads'] * case['dim'] * size
        # forward: two products of a pair; backward: five more.  Training reads q, k, v and the gradient, and writes
        # the output and three gradients
        return dict(bytes=(4 * q + 4 * k if case['train'] else 2 * q + 2 * k) + rows,
                    flops=(14 if case['train'] else 4) * _pairs(case) * case['heads'] * case['dim'])
    if case['op'] == 'norm_rotary':
        x = case['rows'] * (case['heads'] + case['kv_heads']) * case['dim']
        return dict(bytes=x * size * (4 if case['train'] else 2) + case['rows'] * (1 if case['packed'] else 4), flops=x * (20 if case['train'] else 7))
    x = sum(lengths(case)) * case['dim']
    f = case['packs'] * case['dim'] * size if case['first'] else 0
    return dict(bytes=(6 * x * size + 2 * f if case['train'] else 3 * x * size + f) + sum(lengths(case)),
                flops=x * (5 if case['train'] else 2))


# ------------------------------------------------------------------------------------- plain forms
def _attend_block(q, k, v, keep, scale, grad=None):
    """q (B, M, G, L, D) against k, v (B, M, K, D), keep (B, L, K): the output, and the three gradients."""
    b, m, g, n, d = q.shape
    qs = q.reshape(b, m, g * n, d)
    mask = keep[:, None, None]
    s = torch.matmul(qs, k.transpose(2, 3)).view(b, m, g, n, -1) * scale
    s = torch.where(mask, s, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-30)
    del s
    pf = p.view(b, m, g * n, -1)
    o = torch.matmul(pf, v)
    if grad is None:
        return o.view(q.shape), None, None, None
    go = grad.reshape(b, m, g * n, d)
    dv = torch.matmul(pf.transpose(2, 3), go)
    dp = torch.matmul(go, v.transpose(2, 3))
    ds = pf * (dp - (go * o).sum(-1, keepdim=True)) * scale
    del dp
    return o.view(q.shape), torch.matmul(ds, k).view(q.shape), torch.matmul(ds.transpose(2, 3), qs), dv


def _attend_plain(s):
    t, h, kv, d = TYPES[s['dtype']], s['heads'], s['kv_heads'], s['dim']
    scale = d ** -0.5
    q, k, v = (s[x].detach().float() for x in 'qkv')
    grad = s['grad'].float() if s['train'] else None
    lens, one = s['lens'], s['one']
    if s['kind'] != 'rays':  # a few long sequences, each by itself
        parts, at = [], 0
        for i, n in enumerate(lens):
            rows = slice(at, at + n)
            mine = slice(i, i + 1) if one else rows
            at += n
            lq = 1 if one else n
            keep = torch.ones((1, lq, n), dtype=torch.bool, device=q.device)
            if s['causal']:
                keep = keep.tril(n - lq)

            def heads(x, pick):
                return x[pick].view(1, lq, kv, h // kv, d).permute(0, 2, 3, 1, 4)
            o, dq, dk, dv = _attend_block(heads(q, mine), k[rows].transpose(0, 1)[None], v[rows].transpose(0, 1)[None],
                                          keep, scale, None if grad is None else heads(grad, mine))
            back = [x[0].permute(2, 0, 1, 3).reshape(lq, h, d) for x in (o, dq) if x is not None]
            parts.append(back + [x[0].transpose(0, 1) for x in (dk, dv) if x is not None])
        out = [torch.cat(x).to(t) for x in zip(*parts)]
    else:  # many short packs, padded to the longest
        longest, packs = max(lens), len(lens)
        lq = 1 if one else longest
        pack = s['boundaries'].long().cumsum(0) - 1
        place = torch.arange(len(pack), device=q.device) - s['starts'][pack]
        size = torch.zeros(packs, dtype=torch.long, device=q.device).index_add_(0, pack, torch.ones_like(pack))
        step = torch.arange(longest, device=q.device)
        inside = step[None] < size[:, None]
        rows = (s['starts'][:, None] + step).clamp_max(len(pack) - 1)
        keep = inside[:, None, :].expand(packs, lq, longest)
        if not one:
            keep = keep & inside[:, :, None]
            if s['causal']:
                keep = keep.tril()

        def spread(x):
            return (x[:, None] if one else x[rows]).view(packs, lq, kv, h // kv, d).permute(0, 2, 3, 1, 4)
        o, dq, dk, dv = _attend_block(spread(q), k[rows].transpose(1, 2), v[rows].transpose(1, 2), keep, scale,
                                      None if grad is None else spread(grad))

        def gather(x, n):
            x = x.permute(0, 3, 1, 2, 4).reshape(packs * n, -1, d) if x.dim() == 5 \
                else x.transpose(1, 2).reshape(packs * n, -1, d)
            return (x if one else x[pack * n + place]).to(t)
        out = [gather(x, lq if x.dim() == 5 else longest) for x in (o, dq, dk, dv) if x is not None]
    return dict(zip(('o', 'dq', 'dk', 'dv'), out))


def _turn(x, c, s, turn, interleaved):
    """The first `turn` of each head rotated by the angles whose cosine and sine are c, s (N, 1, turn / 2)."""
    head, rest = x[..., :turn], x[..., turn:]
    if interleaved:
        a, b = head[..., 0::2], head[..., 1::2]
        head = torch.stack((a * c - b * s, a * s + b * c), -1).flatten(-2)
    else:
        a, b = head[..., :turn // 2], head[..., turn // 2:]
        head = torch.cat((a * c - b * s, a * s + b * c), -1)
    return torch.cat((head, rest), -1)


def _norm_rotary_plain(s):
    t = TYPES[s['dtype']]
    q, k = _queries_keys(s)
    angle = _positions(s).double()[:, None, None] * s['freqs']
    c, sn = angle.cos().float(), angle.sin().float()
    out = {}
    for name, x in (('q', q), ('k', k)):
        x, w = x.detach().float(), s[name + '_weight'].detach().float()
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
        y = x * r
        out[name] = _turn(y * w, c, sn, s['turn'], s['interleaved']).to(t)
        if s['train']:
            g = _turn(s['grad_' + name].float(), c, -sn, s['turn'], s['interleaved'])
            out['d' + name + '_weight'] = (g * y).sum((0, 1)).to(t)
            g = g * w
            out['d' + name] = (r * (g - y * (g * y).mean(-1, keepdim=True))).to(t)
    return out


def _positions(s):
    if not s['packed']:
        return s['positions']
    row = torch.arange(s['rows'], device='cuda')
    return row - s['starts'][s['boundaries'].long().cumsum(0) - 1]


def _queries_keys(s):
    if not s['packed']:
        return s['q'], s['k']
    h, kv, d = s['heads'], s['kv_heads'], s['dim']
    x = s['qkv'].view(s['rows'], h + 2 * kv, d)
    return x[:, :h], x[:, h:h + kv]


def _scan(a, b, longest):
    """h[t] = a[t] h[t-1] + b[t] along dimension 0, in doubling steps up to the longest pack."""
    a, b = a.clone(), b.clone()
    step = 1
    while step < longest:
        b[step:] += a[step:] * b[:-step]
        a[step:] = a[step:] * a[:-step]
        step *= 2
    return b


def _recur_plain(s):
    t = TYPES[s['dtype']]
    a, b = s['gates'].detach().float(), s['feats'].detach().float()
    first, starts = s['initial'], s['starts']
    ends = torch.cat((starts[1:], starts.new_tensor([len(a)]))) - 1
    if s['reverse']:
        a, b = a.flip(0), b.flip(0)
        starts, ends = (len(a) - 1 - ends).flip(0), (len(a) - 1 - starts).flip(0)
        first = first.flip(0) if first is not None else None
    gate, add = a.clone(), b.clone()
    gate[starts] = 0
    if first is not None:
        add[starts] += a[starts] * first.detach().float()
    h = _scan(gate, add, max(s['lens']))
    out = {'h': h}
    if s['train']:
        g = s['grad'].float()
        g = g.flip(0) if s['reverse'] else g
        after = torch.cat((a[1:], torch.zeros_like(a[:1])))
        after[ends] = 0
        db = _scan(after.flip(0), g.flip(0), max(s['lens'])).flip(0)
        before = torch.cat((torch.zeros_like(h[:1]), h[:-1]))
        before[starts] = 0 if first is None else first.detach().float()
        out.update(dgates=db * before, dfeats=db)
        if first is not None:
            out['dinitial'] = a[starts] * db[starts]
    return {n: (x.flip(0) if s['reverse'] else x).to(t) for n, x in out.items()}


# ------------------------------------------------------------------------------------- the framework's operators
def _spc():
    package = os.path.join(os.getcwd(), 'kaolin-windows_amd')
    if package not in sys.path:
        sys.path.insert(0, package)
    import kaolin
    return kaolin.render.spc


def _attend_own(s):
    o = _spc().pack_attention(s['q'], s['k'], s['v'], s['boundaries'], q_boundaries=s['q_boundaries'],
                              causal=s['causal'])
    if not s['train']:
        return dict(o=o)
    dq, dk, dv = torch.autograd.grad(o, (s['q'], s['k'], s['v']), s['grad'])
    return dict(o=o, dq=dq, dk=dk, dv=dv)


def _norm_rotary_own(s):
    q, k = _queries_keys(s)
    yq, yk = _spc().norm_rotary(q, k, s['q_weight'], s['k_weight'], s['freqs'],
                                boundaries=s['boundaries'] if s['packed'] else None, positions=s['positions'], eps=EPS,
                                interleaved=s['interleaved'])
    if not s['train']:
        return dict(q=yq, k=yk)
    dq, dk, dqw, dkw = torch.autograd.grad((yq, yk), (q, k, s['q_weight'], s['k_weight']), (s['grad_q'], s['grad_k']))
    return dict(q=yq, dq=dq, dq_weight=dqw, k=yk, dk=dk, dk_weight=dkw)


def _recur_own(s):
    h = _spc().linear_recurrence(s['gates'], s['feats'], s['boundaries'], initial=s['initial'], reverse=s['reverse'])
    if not s['train']:
        return dict(h=h)
    of = [s['gates'], s['feats']] + ([s['initial']] if s['initial'] is not None else [])
    return dict(zip(('h', 'dgates', 'dfeats', 'dinitial'), (h,) + torch.autograd.grad(h, of, s['grad'])))


def run(state):
    op = state['op']
    if own:
        return {'attend': _attend_own, 'norm_rotary': _norm_rotary_own, 'recur': _recur_own}[op](state)
    return {'attend': _attend_plain, 'norm_rotary': _norm_rotary_plain, 'recur': _recur_plain}[op](state)


# ------------------------------------------------------------------------------------- 64 bits
def _attend_exact(case, s):
    """Packs of one length at a time, one key head at a time; gradients by differentiation of the definition."""
    lens, one, train = s['lens'], case['one'], case['train']
    g, d = case['heads'] // case['kv_heads'], case['dim']
    starts = s['starts'].cpu()
    q, k, v = (s[x].detach() for x in 'qkv')
    outs = {'o': torch.zeros(q.shape, dtype=torch.float64, device='cuda')}
    if train:
        outs.update({'d' + n: torch.zeros(x.shape, dtype=torch.float64, device='cuda') for n, x in zip('qkv', (q, k, v))})
    by_size = {}
    for i, n in enumerate(lens):
        by_size.setdefault(n, []).append(i)
    for n, packs in by_size.items():
        packs = torch.tensor(packs)
        krows = (starts[packs][:, None] + torch.arange(n)).cuda()
        qrows = packs[:, None].cuda() if one else krows
        for m in range(case['kv_heads']):
            kk, vv = k[krows, m].double(), v[krows, m].double()
            for j in range(m * g, (m + 1) * g):
                qq = q[qrows, j].double()
                if train:
                    qq, kk, vv = (x.detach().requires_grad_(True) for x in (qq, kk, vv))
                s2 = torch.bmm(qq, kk.transpose(1, 2).contiguous()) / math.sqrt(d)
                if case['causal'] and not one:
                    later = torch.arange(n, device='cuda')[None, :] > torch.arange(n, device='cuda')[:, None]
                    s2 = s2.masked_fill(later, -math.inf)
                o = torch.bmm(torch.softmax(s2, -1), vv)
                outs['o'][qrows, j] = o.detach()
                if train:
                    dq, dk, dv = torch.autograd.grad(o, (qq, kk, vv), s['grad'][qrows, j].double())
                    outs['dq'][qrows, j] = dq
                    outs['dk'][krows, m] += dk
                    outs['dv'][krows, m] += dv
                del s2, o
    return outs


def _norm_rotary_exact(case, s):
    """Each pair as a complex number, times the unit number of its angle; gradients by differentiation."""
    q, k = _queries_keys(s)
    half = case['turn'] // 2
    at = s['positions'] if not case['packed'] else torch.cat([torch.arange(n, device='cuda') for n in s['lens']])
    angle = at.double()[:, None, None] * s['freqs']
    unit = torch.polar(torch.ones_like(angle), angle)
    outs = {}
    for name, x in (('q', q), ('k', k)):
        x = x.detach().double().requires_grad_(case['train'])
        w = s[name + '_weight'].detach().double().requires_grad_(case['train'])
        y = x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / case['dim'] + EPS) * w
        first = y[..., :case['turn']]
        pair = first.unflatten(-1, (half, 2)) if case['interleaved'] else first.unflatten(-1, (2, half)).transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * unit)
        z = z.flatten(-2) if case['interleaved'] else z.transpose(-1, -2).flatten(-2)
        z = torch.cat((z, y[..., case['turn']:]), -1)
        outs[name] = z.detach()
        if case['train']:
            outs['d' + name], outs['d' + name + '_weight'] = torch.autograd.grad(z, (x, w),
                                                                               s['grad_' + name].double())
    return outs


def _recur_exact(case, s):
    """Step by step, all packs at once: step i of every pack that is that long (the longest packs come first)."""
    lens = torch.tensor(s['lens'])
    order = lens.argsort(descending=True)
    starts, lens = s['starts'].cpu()[order], lens[order]
    longest = int(lens[0])
    live = (lens[None] > torch.arange(longest)[:, None]).sum(1).tolist()
    base = (starts + lens - 1 if case['reverse'] else starts).cuda()
    way = -1 if case['reverse'] else 1
    a, b = s['gates'].detach().double(), s['feats'].detach().double()
    order = order.cuda()
    h0 = torch.zeros((len(lens), a.shape[1]), dtype=torch.float64, device='cuda')
    if s['initial'] is not None:
        h0 = s['initial'].detach().double()[order]
    h, out = h0, torch.zeros_like(b)
    for i in range(longest):
        at = base[:live[i]] + way * i
        h = a[at] * h[:live[i]] + b[at]
        out[at] = h
    outs = {'h': out}
    if case['train']:
        g, da, db = s['grad'].double(), torch.zeros_like(a), torch.zeros_like(a)
        carry = torch.zeros_like(h0)
        for i in reversed(range(longest)):
            n = live[i]
            at = base[:n] + way * i
            t = g[at] + carry[:n]
            db[at] = t
            da[at] = t * (out[at - way] if i else h0)
            carry[:n] = a[at] * t
        outs.update(dgates=da, dfeats=db)
        if s['initial'] is not None:
            first = torch.zeros_like(carry)
            first[order] = carry
            outs['dinitial'] = first
    return outs


def exact(case, seed):
    s = prepare(case, seed)
    return {'attend': _attend_exact, 'norm_rotary': _norm_rotary_exact, 'recur': _recur_exact}[case['op']](case, s)
