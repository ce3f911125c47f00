"""64-bit plain forms, and bounds on the kernels' rounding, shared by the tests of the sequence operators
over packs.

Bounds: u = half a step of the outputs' type relative to the value (2^-24, 2^-11, 2^-8), E = 2^-24 one
rounding in 32 bits.  A sum of n products in any order is off by at most about n E times the sum of their
magnitudes.  Products of such small numbers are left out, and the bounds are doubled for them.
"""
import math

import torch

HALF_STEP = {torch.float64: 2.0 ** -53, torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
# half the distance of the smallest numbers of a type: what rounding to it loses at least
FLOOR = {torch.float64: 0.0, torch.float32: 2.0 ** -126, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -126}
E = 2.0 ** -24


def marks(lens, lead=0):
    """The boundary mask of packs of these lengths (at least one row each) after `lead` rows of no pack."""
    b = torch.zeros(lead + sum(lens), dtype=torch.bool)
    at = lead
    for n in lens:
        b[at] = True
        at += n
    return b


def spans(boundaries):
    """(start, end) of each pack."""
    starts = torch.nonzero(boundaries)[:, 0].tolist()
    return list(zip(starts, starts[1:] + [len(boundaries)]))


def check(name, got, want, bound):
    got, want = got.detach().double().cpu(), want.detach().double()
    assert got.shape == want.shape, name
    off = (got - want).abs()
    bad = ~(off <= bound.expand(off.shape))
    assert not bad.any(), (f'{name}: {int(bad.sum())} of {bad.numel()} values are off, the first at '
                           f'{torch.nonzero(bad)[0].tolist()}: {got[bad][0]} for {want[bad][0]}, off {off[bad][0]} '
                           f'where {bound.expand(off.shape)[bad][0]} is allowed')


def attention(q, k, v, boundaries, q_boundaries=None, causal=False, scale=None, grad=None, dtype=None):
    """The definition, pack by pack and head by head, in 64 bits; the output, the three gradients where
    `grad` is given, and a bound on the kernels' rounding of each for inputs of `dtype`."""
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    qb = boundaries if q_boundaries is None else q_boundaries
    group, d = q.shape[1] // k.shape[1], q.shape[2]
    u, floor = HALF_STEP[dtype], FLOOR[dtype]
    q, k, v = (x.detach().double() for x in (q, k, v))
    outs = [torch.zeros_like(q)] + ([torch.zeros_like(x) for x in (q, k, v)] if grad is not None else [])
    tols = [torch.zeros_like(x) for x in outs]
    biggest = float(grad.abs().max()) if grad is not None and grad.numel() else 0.0
    for (q0, q1), (k0, k1) in zip(spans(qb), spans(boundaries)):
        nq, nk = q1 - q0, k1 - k0
        for h in range(q.shape[1]):
            qq, kk, vv = q[q0:q1, h], k[k0:k1, h // group], v[k0:k1, h // group]
            s = qq @ kk.t() * scale
            size = qq.abs() @ kk.abs().t() * scale
            seen = torch.ones(nq, nk, dtype=torch.bool)
            if causal:
                seen = torch.arange(nk)[None] <= torch.arange(nq)[:, None] + nk - nq
            s = torch.where(seen, s, -math.inf)
            top = s.max(-1, keepdim=True).values
            p = torch.where(seen, torch.exp(s - torch.where(top == -math.inf, 0.0, top)), 0.0)
            total = p.sum(-1, keepdim=True)
            p = p / torch.where(total == 0, 1.0, total)
            # a weight's relative error: twice a score's error (its own and the maximum's), the exponential's and
            # the sum's; then its rounding to the type, or to nothing below the type's smallest number
            far = torch.where(seen, size, 0.0).max(-1, keepdim=True).values
            e = E * (2 * (d + 3) * far + nk + 16)
            o, ov = p @ vv, p @ vv.abs()
            to = u * (o.abs() + ov) + e * ov + floor * (1 + seen.double() @ vv.abs())
            outs[0][q0:q1, h] = o
            tols[0][q0:q1, h] = 2 * to
            if grad is None:
                continue
            g = grad[q0:q1, h].double()
            dp, delta = g @ vv.t(), (g * o).sum(-1, keepdim=True)
            ds = p * (dp - delta)
            tp = e * p
            tds = e * ds.abs() + p * (E * (d + 3) * (g.abs() @ vv.abs().t()) + (g.abs() * to).sum(-1, keepdim=True)
                                      + E * (d + 3) * (g.abs() * o.abs()).sum(-1, keepdim=True))
            # ds is rounded to the type after a power of two put the largest gradient at 16 or more
            tds = tds + u * ds.abs() + seen * floor * (biggest / 16 if dtype == torch.float16 else 1)
            tp = tp + u * p + seen * floor
            n = E * (nk + 2)
            outs[1][q0:q1, h] = scale * (ds @ kk)
            tols[1][q0:q1, h] = 2 * (u * (scale * (ds @ kk)).abs() + scale * ((tds + n * ds.abs()) @ kk.abs()) + floor)
            n = E * (nq * group + 2)
            outs[2][k0:k1, h // group] += scale * (ds.t() @ qq)
            tols[2][k0:k1, h // group] += 2 * (scale * ((tds + (n + u) * ds.abs()).t() @ qq.abs()) + floor)
            outs[3][k0:k1, h // group] += p.t() @ g
            tols[3][k0:k1, h // group] += 2 * ((tp + (n + u) * p).t() @ g.abs() + floor)
    return outs, tols


def _rotate(x, c, s, interleaved):
    half = c.shape[-1]
    y = x.clone()
    if interleaved:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        y[..., 0:2 * half:2], y[..., 1:2 * half:2] = a * c - b * s, a * s + b * c
    else:
        a, b = x[..., :half], x[..., half:2 * half]
        y[..., :half], y[..., half:2 * half] = a * c - b * s, a * s + b * c
    return y


def norm_rotary(x, w, freqs, positions, eps, interleaved, grad=None, dtype=None, w_dtype=None):
    """One tensor (rows, heads, dim) in 64 bits: the output, its gradients (x, w) where `grad` is given, bounds."""
    x = x.detach().double()
    w = torch.ones(x.shape[-1], dtype=torch.float64) if w is None else w.detach().double()
    d, u, floor = x.shape[-1], HALF_STEP[dtype], FLOOR[dtype]
    angle = positions.double()[:, None, None] * freqs
    c, s = angle.cos(), angle.sin()
    r = ((x * x).mean(-1, keepdim=True) + eps) ** -0.5
    n = x * r
    y = _rotate(n * w, c, s, interleaved)
    # half the relative error of the mean square, the root's, the products', the unit's and the rotation's
    e = E * (d / 2 + 24)
    size = _rotate((n * w).abs(), torch.ones_like(c), -torch.ones_like(s), interleaved)
    size = torch.maximum(size, _rotate((n * w).abs(), torch.ones_like(c), torch.ones_like(s), interleaved)).abs()
    outs, tols = [y], [2 * (u * y.abs() + e * size + floor)]
    if grad is not None:
        g = _rotate(grad.double(), c, -s, interleaved)
        ga = _rotate(grad.double().abs(), torch.ones_like(c), -torch.ones_like(s), interleaved)
        ga = torch.maximum(ga, _rotate(grad.double().abs(), torch.ones_like(c), torch.ones_like(s), interleaved)).abs()
        mean = (g * w * n).mean(-1, keepdim=True)
        dx = r * (g * w - n * mean)
        dxa = r * (ga * w.abs() + n.abs() * (ga * w.abs() * n.abs()).mean(-1, keepdim=True))
        outs.append(dx)
        tols.append(2 * (u * dx.abs() + (2 * e + E * d) * dxa + floor))
        dw = (g * n).sum((0, 1))
        outs.append(dw)
        tols.append(2 * (HALF_STEP[w_dtype or dtype] * dw.abs() + (e + E * x.shape[0] * x.shape[1])
                         * (ga * n.abs()).sum((0, 1)) + FLOOR[w_dtype or dtype]))
    return outs, tols


def recurrence(a, b, boundaries, initial=None, reverse=False, grad=None, dtype=None):
    """The definition row by row in 64 bits: h, the gradients of a, b (and initial) where `grad` is given, bounds."""
    u, floor = HALF_STEP[dtype], FLOOR[dtype]
    e32 = 2.0 ** -53 if dtype == torch.float64 else E
    a, b = a.detach().double(), b.detach().double()
    first = initial.detach().double() if initial is not None else None
    h, ha = torch.zeros_like(b), torch.zeros_like(b)
    da, db, ga = torch.zeros_like(a), torch.zeros_like(b), torch.zeros_like(b)
    tda = torch.zeros_like(a)
    di = torch.zeros_like(first) if first is not None else None
    tdi = torch.zeros_like(first) if first is not None else None
    steps = torch.zeros(len(b), 1, dtype=torch.float64)
    for p, (r0, r1) in enumerate(spans(boundaries)):
        rows = list(range(r0, r1))[::-1] if reverse else list(range(r0, r1))
        start = first[p] if first is not None and p < len(first) else torch.zeros_like(b[0])
        state, size = start, start.abs()
        steps[r0:r1] = len(rows) + 8
        for t in rows:
            state, size = a[t] * state + b[t], a[t].abs() * size + b[t].abs()
            h[t], ha[t] = state, size
        if grad is None:
            continue
        carry = carry_a = torch.zeros_like(b[0])
        for i in reversed(range(len(rows))):
            t = rows[i]
            g, gs = grad[t].double() + carry, grad[t].double().abs() + carry_a
            before, before_a = (h[rows[i - 1]], ha[rows[i - 1]]) if i else (start, start.abs())
            db[t], ga[t], da[t] = g, gs, g * before
            n = e32 * (2 * len(rows) + 16)
            tda[t] = gs * (n * before_a + u * before.abs() + n * before.abs())
            carry, carry_a = a[t] * g, a[t].abs() * gs
        if first is not None and p < len(first):
            di[p], tdi[p] = carry, e32 * (2 * len(rows) + 16) * carry_a
    n = e32 * 2 * steps
    outs, tols = [h], [2 * (u * h.abs() + n * ha + floor)]
    if grad is not None:
        outs += [da, db]
        tols += [2 * (u * da.abs() + tda + floor), 2 * (u * db.abs() + n * ga + floor)]
        if first is not None:
            outs.append(di)
            tols.append(2 * (u * di.abs() + tdi + floor))
    return outs, tols
