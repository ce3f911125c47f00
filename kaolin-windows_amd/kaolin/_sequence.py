"""``_C.render.spc`` entries of the sequence operators over packs (csrc/packs.hip, attend.hip,
attendgrad.hip): argument checks, outputs and one library call each.  The reference has none of
these; they follow its packed ray ops' conventions (rows grouped by a boundary mask)."""
import ctypes
import math

import torch

from . import _native as N
from ._checks import Arg, check_all_same_gpu, check_contiguous, check_dim, check_same_size, check_same_type, check_size

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
        ws = N.workspace(ws_bytes, dev)
        N.check(N.lib().kl_pack_layout(n, N.ptr(boundaries), N.ptr(ids), N.ptr(starts), N.ptr(ws), ws_bytes,
                                       N.stream_of(dev)), func)
    return ids, starts


def usable_heads(t):
    """(rows, heads, dim) as the kernels read it: rows of a head contiguous and 16-byte aligned."""
    e = 16 // t.element_size()
    if t.numel() == 0 or (t.stride(2) == 1 and t.stride(0) % e == 0 and t.stride(1) % e == 0 and t.stride(0) >= 0
                          and t.stride(1) >= 0 and t.data_ptr() % 16 == 0):
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


def _strides(q, k, v):
    return (ctypes.c_int64 * 6)(q.stride(0), q.stride(1), k.stride(0), k.stride(1), v.stride(0), v.stride(1))


def pack_attention_forward_cuda(q, k, v, q_layout, k_layout, scale, causal, with_lse):
    """Attention of the rows of q over the rows of k, v of the pack with the same number.  Returns the
    output (num_q, heads, dim) and, with_lse, the base-2 logarithms of the softmax sums (num_q, heads)."""
    func = 'pack_attention_forward_cuda'
    q, k, v = _attention_args(func, q, k, v, q_layout, k_layout, scale)
    dev = q.device
    out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device=dev) if with_lse else None
    code = _CODES[q.dtype]
    with N.on_device(dev):
        ws_bytes = N.size('kl_pack_attention_workspace_bytes', code, q.shape[0], k.shape[0], q.shape[1], k.shape[1],
                          q.shape[2])
        ws = N.workspace(ws_bytes, dev)
        N.check(N.lib().kl_pack_attention_forward(
            code, q.shape[0], k.shape[0], q.shape[1], k.shape[1], q.shape[2], N.ptr(q), N.ptr(k), N.ptr(v),
            _strides(q, k, v), N.ptr(q_layout[0]), N.ptr(q_layout[1]), N.ptr(k_layout[0]), N.ptr(k_layout[1]),
            scale, int(causal), N.ptr(out), N.ptr(lse), N.ptr(ws), ws_bytes, N.stream_of(dev)), func)
    return out, lse


def pack_attention_backward_cuda(grad_out, q, k, v, q_layout, k_layout, out, lse, scale, causal, need_q, need_kv):
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
    check_all_same_gpu(func, [Arg(q, 'q', 1), ag, ao, Arg(lse, 'lse', 0)])
    dev = q.device
    dq = torch.empty(q.shape, dtype=q.dtype, device=dev) if need_q else None
    dk = torch.empty(k.shape, dtype=k.dtype, device=dev) if need_kv else None
    dv = torch.empty(k.shape, dtype=k.dtype, device=dev) if need_kv else None
    with N.on_device(dev):
        ws_bytes = N.size('kl_pack_attention_bwd_workspace_bytes', q.shape[0], q.shape[1])
        ws = N.workspace(ws_bytes, dev)
        N.check(N.lib().kl_pack_attention_backward(
            _CODES[q.dtype], q.shape[0], k.shape[0], q.shape[1], k.shape[1], q.shape[2], N.ptr(grad_out),
            N.ptr(q), N.ptr(k), N.ptr(v), _strides(q, k, v), N.ptr(q_layout[0]), N.ptr(q_layout[1]),
            N.ptr(k_layout[0]), N.ptr(k_layout[1]), N.ptr(out), N.ptr(lse), scale, int(causal), N.ptr(dq), N.ptr(dk),
            N.ptr(dv), N.ptr(ws), ws_bytes, N.stream_of(dev)), func)
    return dq, dk, dv
