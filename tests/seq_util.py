"""64-bit plain forms and inputs shared by the tests of the sequence operators over packs."""
import math

import torch

HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


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


def attention(q, k, v, boundaries, q_boundaries=None, causal=False, scale=None):
    """The definition, pack by pack and head by head, in the inputs' precision (float64 in the tests)."""
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    qb = boundaries if q_boundaries is None else q_boundaries
    group = q.shape[1] // k.shape[1]
    out = torch.zeros_like(q)
    pieces = []
    for (q0, q1), (k0, k1) in zip(spans(qb), spans(boundaries)):
        nq, nk = q1 - q0, k1 - k0
        heads = []
        for h in range(q.shape[1]):
            s = q[q0:q1, h] @ k[k0:k1, h // group].t() * scale
            if causal:
                last = torch.arange(nq)[:, None] + nk - nq
                s = s.masked_fill(torch.arange(nk)[None] > last, -math.inf)
            top = s.max(-1, keepdim=True).values
            p = torch.where(s == -math.inf, 0.0, torch.exp(s - torch.where(top == -math.inf, 0.0, top)))
            total = p.sum(-1, keepdim=True)
            p = p / torch.where(total == 0, 1.0, total)
            heads.append(p @ v[k0:k1, h // group])
        pieces.append((q0, q1, torch.stack(heads, 1)))
    for q0, q1, x in pieces:
        mask = torch.zeros(len(q), 1, 1, dtype=torch.bool)
        mask[q0:q1] = True
        full = torch.cat((torch.zeros_like(q[:q0]), x, torch.zeros_like(q[q1:])))
        out = torch.where(mask, full, out)
    return out
