"""Attention over packs in 64 bits for all heads of a pack at once (on the inputs' device), with bounds that take no part of
a type's smallest numbers from other rows: what tests of long packs and of numbers far from 1 compare with.

Bounds: as seq_util.py (u half a step of the type, E one rounding in 32 bits, n products in any order off by n E times
their magnitudes, all doubled for what is left out), but for float16's smallest numbers.  Half their distance is F = 2^-25,
and what is rounded to float16 for a second product is first multiplied by a power of two:
- the forward's weights so that a row's largest is at least 2^7: each is off by F / 2^7 of that one, which is no more than
  the weights' sum: 2^-32 in a normalised weight;
- ds for dq so that a row's largest is at least 2^11, ds and p for dk and dv so that a key's are (or, with numbers under
  2^-45, by 2^60): each is off by F / 2^11 = 2^-36 of the largest, and by 2^-85.
"""
import math

import torch

from seq_util import E, FLOOR, HALF_STEP, spans


def attention_heads(q, k, v, boundaries, q_boundaries=None, causal=False, scale=None, grad=None):
    """The output, the three gradients where `grad` is given, and their bounds, on the CPU."""
    dtype, (_, heads, d), group = q.dtype, q.shape, q.shape[1] // k.shape[1]
    scale = d ** -0.5 if scale is None else scale
    u, floor, small = HALF_STEP[dtype], FLOOR[dtype], dtype == torch.float16
    q, k, v = (x.detach().double() for x in (q, k, v))
    grad = grad.double() if grad is not None else None
    outs = [torch.zeros_like(q)] + ([torch.zeros_like(x) for x in (q, k, v)] if grad is not None else [])
    tols = [torch.zeros_like(x) for x in outs]

    def shared(x):  # the sum over the heads that share a key head
        return x.unflatten(0, (-1, group)).sum(1).transpose(0, 1)

    def times(a, b):
        return torch.bmm(a, b.contiguous())
    for (q0, q1), (k0, k1) in zip(spans(boundaries if q_boundaries is None else q_boundaries), spans(boundaries)):
        nq, nk = q1 - q0, k1 - k0
        qq = q[q0:q1].transpose(0, 1).contiguous()
        kk, vv = (x[k0:k1].transpose(0, 1).repeat_interleave(group, 0) for x in (k, v))
        kt, vt = kk.transpose(1, 2).contiguous(), vv.transpose(1, 2).contiguous()
        seen = torch.ones(nq, nk, dtype=torch.bool, device=q.device)
        if causal:
            seen = seen.tril(nk - nq)
        s = torch.where(seen, times(qq, kt) * scale, -math.inf)
        far = torch.where(seen, times(qq.abs(), kt.abs()) * scale, 0.0).amax(-1, keepdim=True)
        top = s.amax(-1, keepdim=True)
        p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
        total = p.sum(-1, keepdim=True)
        p = p / torch.where(total == 0, 1.0, total)
        e = E * (2 * (d + 3) * far + nk + 16)
        all_seen = seen.double().expand(heads, nq, nk)
        o, ov = times(p, vv), times(p, vv.abs())
        to = u * (o.abs() + ov) + e * ov + floor + (2.0 ** -32 if small else floor) * times(all_seen, vv.abs())
        outs[0][q0:q1], tols[0][q0:q1] = o.transpose(0, 1), 2 * to.transpose(0, 1)
        if grad is None:
            continue
        g = grad[q0:q1].transpose(0, 1).contiguous()
        delta = (g * o).sum(-1, keepdim=True)
        ds = p * (times(g, vt) - delta)
        tds = e * ds.abs() + p * (E * (d + 3) * times(g.abs(), vt.abs()) + (g.abs() * to).sum(-1, keepdim=True)
                                  + E * (d + 3) * (g.abs() * o.abs()).sum(-1, keepdim=True)) + u * ds.abs()
        tp = (e + u) * p

        def rounded(x, dim):  # what the smallest numbers cost
            if not small:
                return all_seen * floor
            most = x.abs().amax(dim, keepdim=True)
            if dim == 1:  # a key's largest, over the heads that share it
                most = most.unflatten(0, (-1, group)).amax(1).repeat_interleave(group, 0)
            return all_seen * (2.0 ** -36 * most + 2.0 ** -85)
        dq, n = scale * times(ds, kk), E * (nk + 2)
        outs[1][q0:q1] = dq.transpose(0, 1)
        tols[1][q0:q1] = 2 * (u * dq.abs() + floor + scale * times(tds + rounded(ds, 2) + n * ds.abs(),
                                                                  kk.abs())).transpose(0, 1)
        n = E * (nq * group + 2)
        dk, dv = shared(scale * times(ds.transpose(1, 2), qq)), shared(times(p.transpose(1, 2), g))
        outs[2][k0:k1], outs[3][k0:k1] = dk, dv
        tk = tds + rounded(ds, 1) + n * ds.abs()
        tv = tp + rounded(p, 1) + n * p
        tols[2][k0:k1] = 2 * (u * dk.abs() + floor + shared(scale * times(tk.transpose(1, 2), qq.abs())))
        tols[3][k0:k1] = 2 * (u * dv.abs() + floor + shared(times(tv.transpose(1, 2), g.abs())))
    return [x.cpu() for x in outs], [x.cpu() for x in tols]


def _scan(a, b, starts, longest):
    """h[t] = a[t] h[t - 1] + b[t] down dimension 0, a[starts] taken as 0, in doubling steps."""
    a, b = a.clone(), b.clone()
    a[starts] = 0
    step = 1
    while step < longest:
        b[step:] += a[step:] * b[:-step]
        a[step:] = a[step:] * torch.cat((torch.zeros_like(a[:step]), a[:-step]))[step:]
        step *= 2
    return b


def recurrence_scan(a, b, boundaries, initial=None, reverse=False, grad=None):
    """As seq_util.recurrence for many rows: h, the gradients of a, b (and initial, with a row for every pack) where `grad`
    is given, bounds.

    Bounds: whatever the order of products and sums, what enters at row r is off by one rounding for each row that it is
    carried over and each sum, so h[t] by E (scan(|a|, size) + 16 size) for the recurrence of magnitudes `size`."""
    dtype = b.dtype
    u, floor, e = HALF_STEP[dtype], FLOOR[dtype], 2.0 ** -53 if dtype == torch.float64 else E
    a, b = a.detach().double(), b.detach().double()
    n = len(b)
    starts = torch.nonzero(boundaries)[:, 0]
    lead = int(starts[0]) if len(starts) else n
    first = initial.detach().double() if initial is not None else torch.zeros(len(starts), b.shape[1], dtype=torch.float64)
    ends = torch.cat((starts[1:], starts.new_tensor([n]))) - 1
    longest = int((ends - starts).max()) + 1
    out_rows = torch.ones(n, 1, dtype=torch.float64)
    out_rows[:lead] = 0
    if reverse:
        a, b, out_rows = a.flip(0), b.flip(0), out_rows.flip(0)
        starts, ends, first = (n - 1 - ends).flip(0), (n - 1 - starts).flip(0), first.flip(0)
    a, b = a * out_rows, b * out_rows

    def walk(a, x, s0, starts):
        x = x.clone()
        x[starts] += a[starts] * s0
        return _scan(a, x, starts, longest)
    h, size = walk(a, b, first, starts), walk(a.abs(), b.abs(), first.abs(), starts)
    zero = torch.zeros_like(first)
    eh = e * (walk(a.abs(), size, zero, starts) + 16 * size)
    res = [('h', h, u * h.abs() + eh)]
    if grad is not None:
        g = grad.double().flip(0) if reverse else grad.double()
        g = g * out_rows
        after = torch.cat((a[1:], torch.zeros_like(a[:1]))) * out_rows
        ends_up = (n - 1 - ends).flip(0)

        def back(gates, x):
            return _scan(gates.flip(0), x.flip(0), ends_up, longest).flip(0)
        db, ga = back(after, g), back(after.abs(), g.abs())
        eg = e * (back(after.abs(), ga) + 16 * ga)

        def before(x, s0):
            y = torch.cat((torch.zeros_like(x[:1]), x[:-1]))
            y[starts] = s0
            return y * out_rows
        hb, ehb = before(h, first), before(eh, zero)
        da = db * hb
        res += [('da', da, u * da.abs() + (eg + 2 * e * ga) * hb.abs() + ga * (u * hb.abs() + ehb)),
                ('db', db, u * db.abs() + eg)]
        if initial is not None:
            di = a[starts] * db[starts]
            res.append(('dinitial', di, u * di.abs() + a[starts].abs() * (eg + 2 * e * ga)[starts]))
    return [(name, x.flip(0) if reverse else x, 2 * ((t.flip(0) if reverse else t) + floor)) for name, x, t in res]
