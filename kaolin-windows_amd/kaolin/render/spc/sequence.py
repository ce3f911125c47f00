"""Learned operators along packs: attention, norm with rotation, and the gated linear recurrence.  They take packs as
the packed ray ops do (raytrace.py): rows grouped by a boundary mask, and read nothing back to the host.

A plain call (types, sizes and strides that the kernels read as they are) runs as a compiled autograd node
(csrc/torch_ops.cpp); the nodes here take every other one, copy what has to be copied, and refuse what is
wrong.  Both call the same library entries."""
import math

import torch
from torch.autograd.function import once_differentiable

from ... import _C, _ext
from ..._native import stream_of

__all__ = ['pack_attention', 'norm_rotary', 'rotary_frequencies', 'linear_recurrence']


class PackAttention(torch.autograd.Function):

    @staticmethod
    def forward(ctx, q, k, v, q_layout, k_layout, scale, causal):
        needs = any(ctx.needs_input_grad[:3])
        out, lse, low = _C.render.spc.pack_attention_forward_cuda(q, k, v, q_layout, k_layout, scale, causal, needs)
        if needs:
            ctx.save_for_backward(q, k, v, out, lse, low, *q_layout, *k_layout)
            ctx.scale, ctx.causal = scale, causal
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out):
        q, k, v, out, lse, low, qi, qs, ki, ks = ctx.saved_tensors
        dq, dk, dv = _C.render.spc.pack_attention_backward_cuda(
            grad_out, q, k, v, (qi, qs), (ki, ks), out, lse, low, ctx.scale, ctx.causal, ctx.needs_input_grad[0],
            ctx.needs_input_grad[1] or ctx.needs_input_grad[2])
        return (dq, dk if ctx.needs_input_grad[1] else None, dv if ctx.needs_input_grad[2] else None, None, None, None,
                None)


def pack_attention(q, k, v, boundaries, q_boundaries=None, causal=False, scale=None):
    r"""Attention along packs: each row of ``q`` attends to the rows of ``k`` and ``v`` of its own pack,
    ``out[i] = sum_j softmax_j(scale * q[i] . k[j]) v[j]``.

    Args:
        q (Tensor): (num_q, heads, dim), f16, bf16 or f32; ``dim`` a multiple of 8 up to 128.
        k, v (Tensor): (num_k, kv_heads, dim) of the same type.  ``heads`` is a multiple of ``kv_heads``:
            query head ``h`` reads key head ``h // (heads // kv_heads)``.
        boundaries (Tensor): (num_k,) bool, True at the first row of each pack of ``k`` and ``v``
            (:func:`mark_pack_boundaries`).  Packs lie one behind the other: of a cache with spare rows, gather those
            that count first.
        q_boundaries (Tensor): (num_q,) bool, the packs of ``q``; pack p of ``q`` attends to pack p of ``k``.
            Default: ``boundaries`` (rows attend to rows of their own pack).  With one row per pack, all
            True: one query reads out each pack, or the newest row of each attends to those before it.
        causal (bool): the last row of a pack of ``q`` sees all keys of the pack, each row before it one
            key fewer (with the same packs on both sides, row i sees the rows up to i).
        scale (float): positive; default ``dim ** -0.5``.

    Returns:
        (Tensor): (num_q, heads, dim).  Rows that see no key (before the first pack, of a pack that has no
        keys, or masked altogether) are 0, and their gradients are 0.  A row whose scores are all -inf has no
        softmax and is NaN.

    Rows of q, k and v may be strided, such as the slices of one projection's output; a last dimension
    that is not contiguous, or rows that do not start at multiples of 16 bytes, are copied first.  Keys that
    a row does not see have no effect on it whatever they hold (infinities and NaN too).  Scores and sums are
    in 32 bits; f16 and bf16 weights are rounded to the type for the product with ``v``.  Results are the same
    on every run.  Differentiable once, backwards, with respect to q, k and v.
    """
    scale = (max(q.shape[-1], 1) if q.dim() else 1) ** -0.5 if scale is None else float(scale)
    ext = _ext.get() if q.is_cuda else None
    if ext is not None:
        out = ext.pack_attention(q, k, v, boundaries, q_boundaries, bool(causal), scale, stream_of(q.device))
        if out is not None:
            return out
    _check_boundaries('pack_attention', 'boundaries', boundaries, k)
    k_layout = _C.render.spc.pack_layout_cuda(boundaries.contiguous())
    if q_boundaries is None:
        _check_boundaries('pack_attention', 'boundaries', boundaries, q)
        q_layout = k_layout
    else:
        _check_boundaries('pack_attention', 'q_boundaries', q_boundaries, q)
        q_layout = _C.render.spc.pack_layout_cuda(q_boundaries.contiguous())
    return PackAttention.apply(q, k, v, q_layout, k_layout, scale, bool(causal))


class NormRotary(torch.autograd.Function):

    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, freqs, layout, positions, eps, interleaved):
        ctx.save_for_backward(q, k, q_weight, k_weight, freqs, *(layout or (None, None)), positions)
        ctx.rest = eps, interleaved
        return _C.render.spc.norm_rotary_forward_cuda(q, k, q_weight, k_weight, freqs, layout, positions, eps,
                                                      interleaved)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_q, grad_k):
        q, k, q_weight, k_weight, freqs, ids, starts, positions = ctx.saved_tensors
        eps, interleaved = ctx.rest
        grads = _C.render.spc.norm_rotary_backward_cuda(grad_q, grad_k, q, k, q_weight, k_weight, freqs, (ids, starts),
                                                        positions, eps, interleaved, any(ctx.needs_input_grad[2:4]))
        return tuple(g if need else None for g, need in zip(grads, ctx.needs_input_grad)) + (None,) * 5


def norm_rotary(q, k, q_weight, k_weight, freqs, boundaries=None, positions=None, eps=1e-6, interleaved=False):
    r"""RMS norm of each head of queries and keys, and the rotation of its first elements by the row's
    position, in one pass: ``y = x * rsqrt(mean(x^2) + eps) * weight``, then each pair ``(a, b)`` of the first
    ``2 * len(freqs)`` elements becomes ``(a cos t - b sin t, a sin t + b cos t)``, ``t = position * freqs[pair]``.

    Args:
        q, k (Tensor): (num_rows, heads, dim) and (num_rows, kv_heads, dim), f16, bf16 or f32; ``dim`` a multiple
            of 8 up to 256.  Either may have no heads.
        q_weight, k_weight (Tensor): (dim,) of their type or f32 (both the same), or None for ones.
        freqs (Tensor): (pairs,) f64, radians per unit of position (:func:`rotary_frequencies`); at most
            ``dim / 2``, the elements past ``2 * pairs`` are normed only.
        boundaries (Tensor): (num_rows,) bool; a row's position is its place in its pack, from 0 (rows before
            the first pack: 0).  Either this or ``positions``.
        positions (Tensor): (num_rows,) int32, int64 or f32 (such as the sample's depth along its ray).
        eps (float): added to the mean square.
        interleaved (bool): pairs are elements ``(2 i, 2 i + 1)``; default ``(i, i + pairs)``.

    Returns:
        (Tensor, Tensor): the new q and k, contiguous.

    Angles are formed in 64 bits, the rest in 32 (heads whose squares would leave a float's range are scaled first), and the
    outputs are rounded once.  Differentiable once, backwards, with respect to q, k and the weights; the sums for the
    weights have a fixed order.  Strides: as :func:`pack_attention`.
    """
    ext = _ext.get() if q.is_cuda else None
    if ext is not None:
        out = ext.norm_rotary(q, k, q_weight, k_weight, freqs, boundaries, positions, float(eps), bool(interleaved),
                              stream_of(q.device))
        if out is not None:
            return out
    for name, t in (('freqs', freqs), ('positions', positions)):
        if t is not None and t.requires_grad:
            raise RuntimeError(f'norm_rotary: {name} cannot take a gradient; detach it')
    if (boundaries is None) == (positions is None):
        raise RuntimeError('norm_rotary: give either boundaries or positions')
    layout = None
    if boundaries is not None:
        _check_boundaries('norm_rotary', 'boundaries', boundaries, q)
        layout = _C.render.spc.pack_layout_cuda(boundaries.contiguous())
    return NormRotary.apply(q, k, q_weight.contiguous() if q_weight is not None else None,
                            k_weight.contiguous() if k_weight is not None else None, freqs.contiguous(), layout,
                            positions.contiguous() if positions is not None else None, float(eps), bool(interleaved))


def rotary_frequencies(turn, base=10000.0, factor=1.0, original_length=None, slow=1.0, fast=32.0, device='cuda'):
    r"""The frequencies ``base ** (-2 i / turn)``, i < turn / 2, for :func:`norm_rotary` as (turn / 2,) f64.

    ``factor`` stretches them to positions that many times further than trained.  Without
    ``original_length`` all are divided by it.  With it (the trained length), pairs that turn more than ``fast``
    times in that length stay, those that turn less than ``slow`` times are divided, and in between the share that
    is divided falls linearly with the number of turns.
    """
    if turn < 0 or turn % 2:
        raise RuntimeError(f'rotary_frequencies: turn must be even; got {turn}')
    if not (base > 0 and factor > 0 and (original_length is None or original_length > 0) and fast > slow):
        raise RuntimeError('rotary_frequencies: base, factor and original_length must be positive and fast > slow')
    f = float(base) ** (torch.arange(turn // 2, dtype=torch.float64) * (-2.0 / max(turn, 1)))
    if original_length is None:
        f = f / factor
    else:
        turns = f * (float(original_length) / (2 * math.pi))
        keep = ((turns - slow) / (fast - slow)).clamp(0, 1)
        f = f * (keep + (1 - keep) / factor)
    return f.to(device)


class LinearRecurrence(torch.autograd.Function):

    @staticmethod
    def forward(ctx, gates, feats, initial, layout, reverse):
        out = _C.render.spc.linear_recurrence_forward_cuda(gates, feats, layout, initial, reverse)
        ctx.save_for_backward(gates, out, initial, *layout)
        ctx.reverse = reverse
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out):
        gates, out, initial, ids, starts = ctx.saved_tensors
        grads = _C.render.spc.linear_recurrence_backward_cuda(grad_out.contiguous(), gates, out, (ids, starts), initial,
                                                              ctx.reverse)
        return tuple(g if need else None for g, need in zip(grads, ctx.needs_input_grad)) + (None, None)


def linear_recurrence(gates, feats, boundaries, initial=None, reverse=False):
    r"""Gated linear recurrence along packs, in every column by itself: ``h[t] = gates[t] * h[t-1] + feats[t]``.
    With gates of 1 it is :func:`cumsum`.

    Args:
        gates, feats (Tensor): (num_rows, dim), f16, bf16, f32 or f64.
        boundaries (Tensor): (num_rows,) bool, True at the first row of each pack.
        initial (Tensor): (num_packs, dim), the state before each pack's first row; default 0, also for packs
            past its last row.  With packs of one row each this is one step of every sequence.
        reverse (bool): from each pack's last row to its first, ``h[t] = gates[t] * h[t+1] + feats[t]``.

    Returns:
        (Tensor): the states h (num_rows, dim).  Rows before the first pack are 0, and so are their gradients.

    States are carried in 32 bits (64 for f64) and rounded once each; a pack is never touched by another's
    values.  Gates may be any numbers: a state is off by some roundings of the recurrence of the magnitudes,
    ``s[t] = |gates[t]| * s[t-1] + |feats[t]|``, and finite where that is.  From a row with an infinite gate on, a pack's
    states are infinite or NaN.  Differentiable once, backwards, with respect to gates, feats and initial; the
    gradient of the gates takes the states as they were rounded.
    """
    ext = _ext.get() if gates.is_cuda else None
    if ext is not None:
        out = ext.linear_recurrence(gates, feats, boundaries, initial, bool(reverse), stream_of(gates.device))
        if out is not None:
            return out
    _check_boundaries('linear_recurrence', 'boundaries', boundaries, gates)
    layout = _C.render.spc.pack_layout_cuda(boundaries.contiguous())
    return LinearRecurrence.apply(gates.contiguous(), feats.contiguous(),
                                  initial.contiguous() if initial is not None else None, layout, bool(reverse))


def _check_boundaries(func, name, boundaries, rows):
    if boundaries.dim() != 1 or rows.dim() == 0 or boundaries.shape[0] != rows.shape[0]:
        raise RuntimeError(f'{func}: {name} must hold one value for each of the {tuple(rows.shape)[:1]} rows; got '
                           f'{tuple(boundaries.shape)}')
    if boundaries.dtype not in (torch.bool, torch.uint8):
        raise RuntimeError(f'{func}: {name} must be Bool (or Byte); got {boundaries.dtype}')
    if boundaries.device != rows.device:
        raise RuntimeError(f'{func}: {name} is on {boundaries.device}, the rows are on {rows.device}')
