"""``_C.render.spc`` entries of the sequence operators over packs (csrc/packs.hip, attend.hip,
attendgrad.hip, normrotary.hip, recurrence.hip): argument checks, outputs and one library call each.  The reference has
none of these; they follow its packed ray ops' conventions (rows grouped by a boundary mask)."""
import ctypes
import math

import torch

from . import _native as N
from ._checks import (Arg, check_all_same_gpu, check_contiguous, check_dim, check_same_size, check_same_type,
                      check_size, check_size_dim)

_NAMES = {torch.float16: 'Half', torch.bfloat16: 'BFloat16', torch.float32: 'Float', torch.float64: 'Double',
          torch.bool: 'Bool', torch.uint8: 'Byte', torch.int32: 'Int', torch.int64: 'Long'}
_FLOATS = (torch.float16, torch.bfloat16, torch.float32)
# BFloat16 is a type of these entries alone
_CODES = {torch.float16: N.KL_F16, torch.bfloat16: N.KL_BF16, torch.float32: N.KL_F32, torch.float64: N.KL_F64}


def check_type(func, a, allowed):
    if a.t.dtype not in allowed:
        what = ', '.join(_NAMES[d] for d in allowed)
        what = f'one of {what}' if len(allowed) > 1 else what
        raise RuntimeError(f"Expected scalar type of {a} to be {what}; but got "
                           f"{_NAMES.get(a.t.dtype, a.t.dtype)} (while checking arguments for {func})")


def check_rows(func, n):
    if n >= (1 << 31) - 256:
        raise RuntimeError(f'{func}: {n} rows are more than its 31-bit row numbers hold')


def pack_layout_cuda(boundaries):
    """Each row's pack (N,) and each pack's first row (N + 1,), int32, from the marks of the packs'
    first rows (Bool or Byte): row i is of pack ids[i] (-1 before the first), pack p is the rows
    [starts[p], starts[p + 1]), and starts is N past the last pack.  Nothing is read back."""
    func = 'pack_layout_cuda'
    a = Arg(boundaries, 'boundaries', 1)
    check_dim(func, a, 1)
    check_all_same_gpu(func, [a])
    check_contiguous(func, [a])
    check_type(func, a, (torch.bool, torch.uint8))
    n, dev = boundaries.shape[0], boundaries.device
    check_rows(func, n)
    ids = torch.empty((n,), dtype=torch.int32, device=dev)
    starts = torch.empty((n + 1,), dtype=torch.int32, device=dev)
    with N.on_device(dev):
        ws_bytes = N.size('kl_pack_layout_workspace_bytes', n)
        ws = N.scratch(ws_bytes, dev)
        N.check(N.lib().kl_pack_layout(n, N.ptr(boundaries), N.ptr(ids), N.ptr(starts), N.ptr(ws), ws_bytes,
                                       N.stream_of(dev)), func)
    return ids, starts


def usable_heads(t):
    """(rows, heads, dim) as the kernels read it: rows of a head contiguous, 16-byte aligned, and less than 2^25
    elements apart."""
    e = 16 // t.element_size()
    if t.is_contiguous() and t.data_ptr() % 16 == 0 or (
            t.stride(2) == 1 and t.stride(0) % e == 0 and t.stride(1) % e == 0 and t.stride(0) < 1 << 25
            and t.data_ptr() % 16 == 0):
        return t
    return t.contiguous() if not t.is_contiguous() else t.clone()


def _attention_args(func, q, k, v, q_layout, k_layout, scale):
    aq, ak, av = Arg(q, 'q', 1), Arg(k, 'k', 2), Arg(v, 'v', 3)
    for a in (aq, ak, av):
        check_dim(func, a, 3)
    check_all_same_gpu(func, [aq, ak, av])
    check_type(func, aq, _FLOATS)
    check_same_type(func, ak, aq)
    check_same_type(func, av, aq)
    check_same_size(func, av, ak)
    if q.shape[2] != k.shape[2] or q.shape[2] % 8 or not 0 < q.shape[2] <= 128:
        raise RuntimeError(f'{func}: the head size must be the same multiple of 8 up to 128 for q, k and v; got '
                           f'{q.shape[2]} and {k.shape[2]}')
    if k.shape[1] == 0 or q.shape[1] == 0 or q.shape[1] % k.shape[1] or q.shape[1] > 4096:
        raise RuntimeError(f'{func}: the heads of q (at most 4096) must be a multiple of the heads of k and v; got '
                           f'{q.shape[1]} and {k.shape[1]}')
    if not (scale > 0 and math.isfinite(scale)):
        raise RuntimeError(f'{func}: the scale must be positive and finite; got {scale}')
    for t, (ids, starts), name in ((q, q_layout, 'q'), (k, k_layout, 'k')):
        check_rows(func, t.shape[0])
        check_size(func, Arg(ids, f'{name}_ids', 0), (t.shape[0],))
        check_size(func, Arg(starts, f'{name}_starts', 0), (t.shape[0] + 1,))
        check_all_same_gpu(func, [aq, Arg(ids, f'{name}_ids', 0), Arg(starts, f'{name}_starts', 0)])
        check_type(func, Arg(ids, f'{name}_ids', 0), (torch.int32,))
        check_type(func, Arg(starts, f'{name}_starts', 0), (torch.int32,))
        check_contiguous(func, [Arg(ids, f'{name}_ids', 0), Arg(starts, f'{name}_starts', 0)])
    return usable_heads(q), usable_heads(k), usable_heads(v)


def _strides(*tensors):
    """Row and head strides; a single row's stride may be anything and is not used."""
    s = [x for t in tensors for x in (t.stride(0) if t.shape[0] > 1 else 0, t.stride(1))]
    return (ctypes.c_int64 * len(s))(*s)


def pack_attention_forward_cuda(q, k, v, q_layout, k_layout, scale, causal, for_backward):
    """Attention of the rows of q over the rows of k, v of the pack with the same number.  Returns the
    output (num_q, heads, dim) and, for_backward, the base-2 logarithms of the softmax sums (num_q, heads) and
    (f16, bf16) what the output's rounding left out, as the output; else None."""
    func = 'pack_attention_forward_cuda'
    q, k, v = _attention_args(func, q, k, v, q_layout, k_layout, scale)
    dev = q.device
    out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device=dev) if for_backward else None
    low = torch.empty_like(out) if for_backward and q.dtype != torch.float32 else None
    code = _CODES[q.dtype]
    with N.on_device(dev):
        ws_bytes = N.size('kl_pack_attention_workspace_bytes', code, q.shape[0], k.shape[0], q.shape[1], k.shape[1],
                          q.shape[2])
        ws = N.scratch(ws_bytes, dev)
        N.check(N.lib().kl_pack_attention_forward(
            code, q.shape[0], k.shape[0], q.shape[1], k.shape[1], q.shape[2], N.ptr(q), N.ptr(k), N.ptr(v),
            _strides(q, k, v), N.ptr(q_layout[0]), N.ptr(q_layout[1]), N.ptr(k_layout[0]), N.ptr(k_layout[1]),
            scale, int(causal), N.ptr(out), N.ptr(low), N.ptr(lse), N.ptr(ws), ws_bytes, N.stream_of(dev)), func)
    return out, lse, low


def pack_attention_backward_cuda(grad_out, q, k, v, q_layout, k_layout, out, lse, low, scale, causal, need_q, need_kv):
    """The gradients of q and of (k, v), None where not needed."""
    func = 'pack_attention_backward_cuda'
    q, k, v = _attention_args(func, q, k, v, q_layout, k_layout, scale)
    grad_out = usable_heads(grad_out.contiguous())
    ag, ao = Arg(grad_out, 'grad_out', 0), Arg(out, 'out', 0)
    check_same_size(func, ag, Arg(q, 'q', 1))
    check_same_type(func, ag, Arg(q, 'q', 1))
    check_same_size(func, ao, Arg(q, 'q', 1))
    check_same_type(func, ao, Arg(q, 'q', 1))
    check_size(func, Arg(lse, 'lse', 0), q.shape[:2])
    check_type(func, Arg(lse, 'lse', 0), (torch.float32,))
    check_contiguous(func, [ao, Arg(lse, 'lse', 0)])
    if low is not None:
        check_same_size(func, Arg(low, 'low', 0), ao)
        check_same_type(func, Arg(low, 'low', 0), ao)
        check_contiguous(func, [Arg(low, 'low', 0)])
        check_all_same_gpu(func, [ao, Arg(low, 'low', 0)])
    check_all_same_gpu(func, [Arg(q, 'q', 1), ag, ao, Arg(lse, 'lse', 0)])
    dev = q.device
    dq = torch.empty(q.shape, dtype=q.dtype, device=dev) if need_q else None
    dk = torch.empty(k.shape, dtype=k.dtype, device=dev) if need_kv else None
    dv = torch.empty(k.shape, dtype=k.dtype, device=dev) if need_kv else None
    with N.on_device(dev):
        ws_bytes = N.size('kl_pack_attention_bwd_workspace_bytes', _CODES[q.dtype], q.shape[0], k.shape[0], q.shape[1],
                          k.shape[1], q.shape[2])
        ws = N.scratch(ws_bytes, dev)
        N.check(N.lib().kl_pack_attention_backward(
            _CODES[q.dtype], q.shape[0], k.shape[0], q.shape[1], k.shape[1], q.shape[2], N.ptr(grad_out),
            N.ptr(q), N.ptr(k), N.ptr(v), _strides(q, k, v), N.ptr(q_layout[0]), N.ptr(q_layout[1]),
            N.ptr(k_layout[0]), N.ptr(k_layout[1]), N.ptr(out), N.ptr(low), N.ptr(lse), scale, int(causal), N.ptr(dq), N.ptr(dk),
            N.ptr(dv), N.ptr(ws), ws_bytes, N.stream_of(dev)), func)
    return dq, dk, dv


_POSITIONS = {torch.int32: 1, torch.int64: 2, torch.float32: 3}


def _norm_args(func, q, k, q_weight, k_weight, freqs, layout, positions, eps):
    """Checks; returns q, k as the kernels read them and the arguments from the strides to eps."""
    aq, ak, af = Arg(q, 'q', 1), Arg(k, 'k', 2), Arg(freqs, 'freqs', 5)
    check_dim(func, aq, 3)
    check_dim(func, ak, 3)
    check_all_same_gpu(func, [aq, ak, af])
    check_type(func, aq, _FLOATS)
    check_same_type(func, ak, aq)
    n, dim = q.shape[0], q.shape[2]
    check_rows(func, n)
    if k.shape[0] != n or k.shape[2] != dim:
        raise RuntimeError(f'{func}: q and k must have the same rows and head size; got {tuple(q.shape)} and '
                           f'{tuple(k.shape)}')
    if dim % 8 or not 0 < dim <= 256:
        raise RuntimeError(f'{func}: the head size must be a multiple of 8 up to 256; got {dim}')
    if q.shape[1] + k.shape[1] > 1 << 16:
        raise RuntimeError(f'{func}: at most 65536 heads; got {q.shape[1]} and {k.shape[1]}')
    check_dim(func, af, 1)
    check_type(func, af, (torch.float64,))
    check_contiguous(func, [af])
    if 2 * freqs.shape[0] > dim:
        raise RuntimeError(f'{func}: {freqs.shape[0]} pairs do not fit a head of {dim}')
    if not (eps >= 0 and math.isfinite(eps)):
        raise RuntimeError(f'{func}: eps must not be negative; got {eps}')
    kinds = set()
    for i, (w, name) in enumerate(((q_weight, 'q_weight'), (k_weight, 'k_weight'))):
        if w is not None:
            a = Arg(w, name, 3 + i)
            check_size(func, a, (dim,))
            check_all_same_gpu(func, [aq, a])
            check_type(func, a, (q.dtype,) if q.dtype == torch.float32 else (q.dtype, torch.float32))
            check_contiguous(func, [a])
            kinds.add(w.dtype)
    if len(kinds) > 1:
        raise RuntimeError(f'{func}: the weights must have one type')
    kind, ids, starts = 0, None, None
    if positions is not None:
        ap = Arg(positions, 'positions', 7)
        check_size(func, ap, (n,))
        check_all_same_gpu(func, [aq, ap])
        check_type(func, ap, tuple(_POSITIONS))
        check_contiguous(func, [ap])
        kind = _POSITIONS[positions.dtype]
    else:
        ids, starts = layout
        for t, name, size in ((ids, 'ids', n), (starts, 'starts', n + 1)):
            a = Arg(t, name, 6)
            check_size(func, a, (size,))
            check_type(func, a, (torch.int32,))
            check_all_same_gpu(func, [aq, a])
            check_contiguous(func, [a])
    q, k = usable_heads(q), usable_heads(k)
    return q, k, (_strides(q, k), N.ptr(q_weight), N.ptr(k_weight), int(kinds == {torch.float32}), N.ptr(freqs), kind,
                  N.ptr(positions), N.ptr(ids), N.ptr(starts), eps)


def norm_rotary_forward_cuda(q, k, q_weight, k_weight, freqs, layout, positions, eps, interleaved):
    """The normed and rotated q and k, contiguous."""
    func = 'norm_rotary_forward_cuda'
    q, k, rest = _norm_args(func, q, k, q_weight, k_weight, freqs, layout, positions, eps)
    dev = q.device
    yq, yk = (torch.empty(x.shape, dtype=x.dtype, device=dev) for x in (q, k))
    with N.on_device(dev):
        N.check(N.lib().kl_norm_rotary_forward(
            _CODES[q.dtype], q.shape[0], q.shape[1], k.shape[1], q.shape[2], 2 * freqs.shape[0], int(interleaved),
            N.ptr(q), N.ptr(k), *rest, N.ptr(yq), N.ptr(yk), N.stream_of(dev)), func)
    return yq, yk


def norm_rotary_backward_cuda(grad_q_out, grad_k_out, q, k, q_weight, k_weight, freqs, layout, positions, eps,
                              interleaved, need_weights):
    """The gradients of q, k and of the weights (None where a weight is None or, without need_weights)."""
    func = 'norm_rotary_backward_cuda'
    q, k, rest = _norm_args(func, q, k, q_weight, k_weight, freqs, layout, positions, eps)
    gq, gk = usable_heads(grad_q_out.contiguous()), usable_heads(grad_k_out.contiguous())
    for g, x, name in ((gq, q, 'grad_q_out'), (gk, k, 'grad_k_out')):
        check_same_size(func, Arg(g, name, 0), Arg(x, name[5], 0))
        check_same_type(func, Arg(g, name, 0), Arg(x, name[5], 0))
        check_all_same_gpu(func, [Arg(q, 'q', 1), Arg(g, name, 0)])
    dev = q.device
    dq, dk = (torch.empty(x.shape, dtype=x.dtype, device=dev) for x in (q, k))
    dqw, dkw = (torch.empty_like(w) if w is not None and need_weights else None for w in (q_weight, k_weight))
    with N.on_device(dev):
        ws_bytes = N.size('kl_norm_rotary_bwd_workspace_bytes', q.shape[2])
        ws = N.scratch(ws_bytes, dev)
        N.check(N.lib().kl_norm_rotary_backward(
            _CODES[q.dtype], q.shape[0], q.shape[1], k.shape[1], q.shape[2], 2 * freqs.shape[0], int(interleaved),
            N.ptr(gq), N.ptr(gk), N.ptr(q), N.ptr(k), *rest, N.ptr(dq), N.ptr(dk), N.ptr(dqw), N.ptr(dkw), N.ptr(ws),
            ws_bytes, N.stream_of(dev)), func)
    return dq, dk, dqw, dkw


def _recurrence_args(func, gates, other, name, initial, layout):
    ag, ao = Arg(gates, 'gates', 1), Arg(other, name, 2)
    check_dim(func, ag, 2)
    check_same_size(func, ao, ag)
    args = [ag, ao]
    if initial is not None:
        ai = Arg(initial, 'initial', 4)
        check_dim(func, ai, 2)
        check_size_dim(func, ai, 1, gates.shape[1])
        args.append(ai)
    check_all_same_gpu(func, args)
    check_contiguous(func, args)
    check_type(func, ag, (torch.float16, torch.bfloat16, torch.float32, torch.float64))
    for a in args[1:]:
        check_same_type(func, a, ag)
    n, dim = gates.shape
    check_rows(func, n)
    if dim >= 1 << 24 or (initial is not None and initial.shape[0] >= 1 << 31):
        raise RuntimeError(f'{func}: sizes out of range: {tuple(gates.shape)}')
    for t, what, size in zip(layout, ('ids', 'starts'), (n, n + 1)):
        a = Arg(t, what, 3)
        check_size(func, a, (size,))
        check_type(func, a, (torch.int32,))
        check_all_same_gpu(func, [ag, a])
        check_contiguous(func, [a])


def linear_recurrence_forward_cuda(gates, feats, layout, initial, reverse):
    """h[t] = gates[t] h[t - 1] + feats[t] along each pack."""
    func = 'linear_recurrence_forward_cuda'
    _recurrence_args(func, gates, feats, 'feats', initial, layout)
    dev, (n, dim), code = gates.device, gates.shape, _CODES[gates.dtype]
    out = torch.empty_like(gates)
    with N.on_device(dev):
        ws_bytes = N.size('kl_linear_recurrence_workspace_bytes', code, n, dim)
        ws = N.scratch(ws_bytes, dev)
        N.check(N.lib().kl_linear_recurrence_forward(
            code, n, dim, N.ptr(gates), N.ptr(feats), N.ptr(initial), 0 if initial is None else initial.shape[0],
            N.ptr(layout[0]), N.ptr(layout[1]), int(reverse), N.ptr(out), N.ptr(ws), ws_bytes, N.stream_of(dev)), func)
    return out


def linear_recurrence_backward_cuda(grad_out, gates, out, layout, initial, reverse):
    """The gradients of gates, feats and initial (None without it)."""
    func = 'linear_recurrence_backward_cuda'
    _recurrence_args(func, gates, grad_out, 'grad_out', initial, layout)
    _recurrence_args(func, gates, out, 'out', initial, layout)
    dev, (n, dim), code = gates.device, gates.shape, _CODES[gates.dtype]
    da, db = torch.empty_like(gates), torch.empty_like(gates)
    di = torch.empty_like(initial) if initial is not None else None
    with N.on_device(dev):
        ws_bytes = N.size('kl_linear_recurrence_workspace_bytes', code, n, dim)
        ws = N.scratch(ws_bytes, dev)
        N.check(N.lib().kl_linear_recurrence_backward(
            code, n, dim, N.ptr(grad_out), N.ptr(gates), N.ptr(out), N.ptr(initial),
            0 if initial is None else initial.shape[0], N.ptr(layout[0]), N.ptr(layout[1]), int(reverse), N.ptr(da),
            N.ptr(db), N.ptr(di), N.ptr(ws), ws_bytes, N.stream_of(dev)), func)
    return da, db, di
