"""Token rows into expert order and back, for code that brings its own experts and for training:
both directions have gradients. The sort itself is `kernels`' (`sort_by_expert`), the kernels are in
csrc/rows.cu, the autograd nodes in csrc/rows_torch.cpp. Beyond the reference, which infers only.

    plan = rows.plan(idx, n_experts)              # idx [N, k]: every token's experts
    x = rows.permute_rows(h, plan)                # [N*k, H], expert e owns plan.offsets[e]:plan.offsets[e+1]
    y = my_experts(x, plan.offsets)
    out = rows.unpermute_rows(y, w, plan)         # [N, H]: every token's rows, weighted and summed

Rows are fp16, bf16 or fp32 with a row of a multiple of 16 bytes, top_k is at most 8. A tensor that is
not contiguous is copied first, one that is has to start on a 16-byte boundary; gradients may come in any
form. Everything is enqueued on the current stream; nothing synchronises. There are no workspaces: what a captured graph
keeps are the addresses of its tensors. Make the first call on a device outside a capture (it loads
the library there), and capture a backward pass with no eager graph of the same leaves alive (torch
ties a leaf's gradient to the stream of the first). RuntimeError on any other argument, and for an input with a forward-mode
tangent (the operators have gradients, no forward-mode and no second derivatives)."""

from typing import NamedTuple

import torch


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


def permute_rows(h, plan):
    """x [N*k, H]: row plan.pos_of[t, j] is h[t]. Gradient: every token's rows of dx summed in float32
    in ascending row, rounded once."""
    return _ext().rows.permute_autograd(h, plan.pos_of, plan.offsets)


def unpermute_rows(y, w, plan):
    """out [N, H]: sum over j of w[t, j] * y[plan.pos_of[t, j]], in float32 in ascending row (the order of
    `combine`), rounded once. w [N, k] in y's dtype or float32, or None for a plain sum. Gradients:
    dy (rows of no choice: zero) and dw, the dot products in float32."""
    return _ext().rows.unpermute_autograd(y, w, plan.pos_of, plan.offsets)
