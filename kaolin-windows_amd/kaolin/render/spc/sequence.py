"""Learned operators along packs: attention.  They take packs as the packed ray ops do (raytrace.py):
rows grouped by a boundary mask, and read nothing back to the host."""
import torch
from torch.autograd.function import once_differentiable

from ... import _C

__all__ = ['pack_attention']


class PackAttention(torch.autograd.Function):

    @staticmethod
    def forward(ctx, q, k, v, q_layout, k_layout, scale, causal):
        needs = any(ctx.needs_input_grad[:3])
        out, lse = _C.render.spc.pack_attention_forward_cuda(q, k, v, q_layout, k_layout, scale, causal, needs)
        if needs:
            ctx.save_for_backward(q, k, v, out, lse, *q_layout, *k_layout)
            ctx.scale, ctx.causal = scale, causal
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out):
        q, k, v, out, lse, qi, qs, ki, ks = ctx.saved_tensors
        dq, dk, dv = _C.render.spc.pack_attention_backward_cuda(
            grad_out, q, k, v, (qi, qs), (ki, ks), out, lse, ctx.scale, ctx.causal, ctx.needs_input_grad[0],
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
            (:func:`mark_pack_boundaries`).
        q_boundaries (Tensor): (num_q,) bool, the packs of ``q``; pack p of ``q`` attends to pack p of ``k``.
            Default: ``boundaries`` (rows attend to rows of their own pack).  With one row per pack, all
            True: one query reads out each pack, or the newest row of each attends to those before it.
        causal (bool): the last row of a pack of ``q`` sees all keys of the pack, each row before it one
            key fewer (with the same packs on both sides, row i sees the rows up to i).
        scale (float): positive; default ``dim ** -0.5``.

    Returns:
        (Tensor): (num_q, heads, dim).  Rows that see no key (before the first pack, of a pack that has no
        keys, or masked altogether) are 0, and their gradients are 0.

    Rows of q, k and v may be strided, such as the slices of one projection's output; a last dimension
    that is not contiguous, or rows that do not start at multiples of 16 bytes, are copied first.  Keys that
    a row does not see have no effect on it whatever they hold (infinities and NaN too).  Scores and sums are
    in 32 bits; f16 and bf16 weights are rounded to the type for the product with ``v``.  Results are the same
    on every run.  Differentiable once, with respect to q, k and v.
    """
    scale = (max(q.shape[-1], 1) if q.dim() else 1) ** -0.5 if scale is None else float(scale)
    _check_boundaries('pack_attention', 'boundaries', boundaries, k)
    k_layout = _C.render.spc.pack_layout_cuda(boundaries.contiguous())
    if q_boundaries is None:
        _check_boundaries('pack_attention', 'boundaries', boundaries, q)
        q_layout = k_layout
    else:
        _check_boundaries('pack_attention', 'q_boundaries', q_boundaries, q)
        q_layout = _C.render.spc.pack_layout_cuda(q_boundaries.contiguous())
    return PackAttention.apply(q, k, v, q_layout, k_layout, scale, bool(causal))


def _check_boundaries(func, name, boundaries, rows):
    if boundaries.dim() != 1 or rows.dim() == 0 or boundaries.shape[0] != rows.shape[0]:
        raise RuntimeError(f'{func}: {name} must hold one value for each of the {tuple(rows.shape)[:1]} rows; got '
                           f'{tuple(boundaries.shape)}')
    if boundaries.dtype not in (torch.bool, torch.uint8):
        raise RuntimeError(f'{func}: {name} must be Bool (or Byte); got {boundaries.dtype}')
    if boundaries.device != rows.device:
        raise RuntimeError(f'{func}: {name} is on {boundaries.device}, the rows are on {rows.device}')
