"""Token rows into expert order and back, for code that brings its own experts and for training:
both directions have gradients. The sort itself is `kernels`' (`sort_by_expert`), the kernels are in
csrc/rows.cu. Beyond the reference, which infers only.

    plan = rows.plan(idx, n_experts)              # idx [N, k]: every token's experts
    x = rows.permute_rows(h, plan)                # [N*k, H], expert e owns plan.offsets[e]:plan.offsets[e+1]
    y = my_experts(x, plan.offsets)
    out = rows.unpermute_rows(y, w, plan)         # [N, H]: every token's rows, weighted and summed

Rows are fp16, bf16 or fp32 with a row of a multiple of 16 bytes, top_k is at most 8. Everything is
enqueued on the current stream; nothing synchronises. There are no workspaces: what a captured graph
keeps are the addresses of its tensors. Make the first call on a device outside a capture (it loads
the library there). RuntimeError on any other argument, and for an input with a forward-mode
tangent (the operators have gradients, no forward-mode derivatives)."""

from typing import NamedTuple

import torch
from torch.autograd import forward_ad


class SortPlan(NamedTuple):
    """Where every choice's row goes. pos_of[t, j] is the sorted row of token t's j-th choice, -1
    where its expert id is outside [0, experts): such a choice has no row, and as many rows at
    the end belong to none (permute_rows sets them to zero)."""
    counts: torch.Tensor   # int32 [experts] rows per expert
    offsets: torch.Tensor  # int32 [experts + 1] exclusive prefix of counts
    token: torch.Tensor    # int32 [N*k] token of each sorted row (undefined from offsets[experts] on)
    pos_of: torch.Tensor   # int32 [N, k]


_kernels = None


def _ext():
    """The kernel library's calls (kernels imports this module: looked up at the first call)."""
    global _kernels
    if _kernels is None:
        from . import kernels
        _kernels = kernels
    return _kernels.ext()


def plan(idx, n_experts):
    """The plan of idx [N, k] (int32 or int64): a stable sort of the choices by expert. Ids outside
    [0, n_experts) are skipped and leave status 6 (kernels.Ext.device_status)."""
    if idx.dim() != 2 or idx.dtype not in (torch.int32, torch.int64):
        raise RuntimeError(f"plan: idx must be int32 or int64 [tokens, top_k], got {idx.dtype} {list(idx.shape)}")
    if idx.dtype is torch.int64:
        idx = idx.clamp(-1, n_experts).to(torch.int32)  # (an id past 32 bits must not come back as another)
    counts, offsets, token, _, pos_of = _ext().sort_by_expert(idx.contiguous(), None, n_experts)
    return SortPlan(counts, offsets, token, pos_of.view(idx.shape))


def refuse_tangents(name, *tensors):
    """Raises for dual tensors: they do not ask for a gradient, so their tangents would get lost in silence."""
    if any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError(f"{name} has no forward-mode derivative: unpack its dual inputs first")


def _incoming(d):
    """A gradient as the kernels take it. Autograd may hand over any view of its producer's: expanded, strided, or
    a slice of a flat buffer that starts between 16-byte boundaries."""
    d = d.contiguous()
    return d if d.data_ptr() % 16 == 0 else d.clone()


class _NoSecond(torch.autograd.Function):
    """Hands its first tensors on, in a graph with all of them, and has no gradient."""

    @staticmethod
    def forward(ctx, count, *tensors):
        return tensors[:count]

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError("permute_rows and unpermute_rows have no second derivatives")


def _last(grads, *inputs):
    """The gradients, made from `inputs`. Where a graph of them is being recorded they are tied to those inputs: a
    derivative of theirs is then refused, wherever it is asked for, and not left out of a sum (which is what
    happens with torch's once_differentiable, whose error hangs on no input)."""
    if not (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in inputs)):
        return grads
    tied = iter(_NoSecond.apply(sum(g is not None for g in grads), *(g for g in grads if g is not None), *inputs))
    return tuple(next(tied) if g is not None else None for g in grads)


class _Permute(torch.autograd.Function):
    @staticmethod
    def forward(ctx, h, offsets, pos_of):
        ctx.save_for_backward(pos_of)
        return _ext().permute_rows(h, pos_of, offsets)

    @staticmethod
    def backward(ctx, dx):
        pos_of, = ctx.saved_tensors
        return _last((_ext().unpermute_rows(_incoming(dx), None, pos_of), None, None), dx)


class _Unpermute(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, w, offsets, pos_of):
        ctx.save_for_backward(y if w is not None and ctx.needs_input_grad[1] else None, w, offsets, pos_of)
        return _ext().unpermute_rows(y, w, pos_of)

    @staticmethod
    def backward(ctx, dout):
        y, w, offsets, pos_of = ctx.saved_tensors
        need_dy, need_dw = ctx.needs_input_grad[:2]
        dy, dw = _ext().unpermute_rows_grad(_incoming(dout), y, w, pos_of, offsets, need_dy, need_dw)
        return _last((dy, dw, None, None), dout, y, w)


def permute_rows(h, plan):
    """x [N*k, H]: row plan.pos_of[t, j] is h[t]. Gradient: every token's rows of dx summed in float32
    in ascending row, rounded once."""
    refuse_tangents("permute_rows", h)
    h = h.contiguous()
    if torch.is_grad_enabled() and h.requires_grad:
        return _Permute.apply(h, plan.offsets, plan.pos_of)
    return _ext().permute_rows(h, plan.pos_of, plan.offsets)


def unpermute_rows(y, w, plan):
    """out [N, H]: sum over j of w[t, j] * y[plan.pos_of[t, j]], in float32 in ascending row (the order of
    `combine`), rounded once. w [N, k] in y's dtype or float32, or None for a plain sum. Gradients:
    dy (rows of no choice: zero) and dw, the dot products in float32."""
    refuse_tangents("unpermute_rows", y, w)
    y = y.contiguous()
    w = w.contiguous() if w is not None else None
    if torch.is_grad_enabled() and (y.requires_grad or (w is not None and w.requires_grad)):
        return _Unpermute.apply(y, w, plan.offsets, plan.pos_of)
    return _ext().unpermute_rows(y, w, plan.pos_of)
