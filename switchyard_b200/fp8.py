"""Experts in 8-bit floats: e4m3 values with a float32 scale for each block of 128 (1 x 128 for rows,
128 x 128 for weights), quantised by csrc/quant8.cu and multiplied by csrc/gemm_fp8.cu. Half the bytes
of the 16-bit experts where decode reads weights, twice the tensor-core rate where prefill
multiplies. Beyond the reference, which has 16-bit experts only.

    gate_up8 = fp8.quantize_weight(gate_up, halves=2)     # [E, 2*I, H], once at load
    down8 = fp8.quantize_weight(down)                      # [E, H, I]
    out = kernels.moe_layer(h, router, gate_up8, down8, top_k, norm)

For inference: no call here has a gradient, and an input that requires one is refused while
gradients are recorded, one with a forward-mode tangent always. Everything is enqueued on the current stream; nothing synchronises, there are
no workspaces. Make the first call on a device outside a capture (it loads the library there)."""

from typing import NamedTuple

import torch

from . import rows as _rows


class Rows8(NamedTuple):
    """q float8_e4m3fn [rows, K], scale float32 [ceil(K/128), rows]: row r, column c stands for
    q[r, c] * scale[c // 128, r]."""
    q: torch.Tensor
    scale: torch.Tensor

    def dequantize(self, dtype=torch.float32):
        K = self.q.shape[1]
        return (self.q.float() * self.scale.t().repeat_interleave(128, 1)[:, :K]).to(dtype)


class _Weight8(NamedTuple):
    q: torch.Tensor
    scale: torch.Tensor


class Weight8(_Weight8):
    """q float8_e4m3fn [E, N, K], scale float32 [E, halves * ceil(N/halves/128), ceil(K/128)] for blocks
    of 128 x 128; a gate_up stack counts its blocks in each half on its own (halves 2), which
    is the plain layout when the halves are multiples of 128. Where they are not, the two layouts can have
    the same shape (N = 400: four blocks of rows either way), so a weight says which it has: `halves`, None
    in one put together from its two tensors alone, which is taken for what it is used as."""

    halves = None

    def __new__(cls, q, scale, halves=None):
        self = super().__new__(cls, q, scale)
        if halves is not None:
            self.halves = halves
        return self

    def _replace(self, **changed):
        return type(self)(**{**self._asdict(), "halves": self.halves, **changed})

    @property
    def shape(self):
        return self.q.shape

    @property
    def device(self):
        return self.q.device

    def check_halves(self, name, halves):
        """Raises where the blocks of rows are known to be counted otherwise than in `halves`."""
        if self.halves not in (None, halves) and self.q.shape[1] % 256:
            raise RuntimeError(f"{name}: a weight of {self.q.shape[1]} rows quantised with halves={self.halves} has other "
                               f"blocks than halves={halves}")

    def dequantize(self, dtype=torch.float32, halves=None):
        """The values, [E, N, K]. halves: needed where the weight does not know its own."""
        E, N, K = self.q.shape
        halves = halves or self.halves or 1
        self.check_halves("dequantize", halves)
        if self.scale.shape[1] != halves * ((N // halves + 127) // 128):
            raise RuntimeError(f"dequantize: {self.scale.shape[1]} blocks of rows are not those of {N} rows with halves={halves}")
        s = self.scale.reshape(E * halves, -1, self.scale.shape[-1])
        s = s.repeat_interleave(128, 1)[:, :N // halves].repeat_interleave(128, 2)[:, :, :K]
        return (self.q.float() * s.reshape(E, N, K)).to(dtype)


def refuse(name, *weights):
    """Raises where a path that has 16-bit experts only is given 8-bit ones."""
    if any(isinstance(w, Weight8) for w in weights):
        raise RuntimeError(f"{name}: 8-bit experts (fp8.Weight8) are for one GPU; pass the 16-bit stacks")


def _no_grad(name, *tensors):
    asks = _rows._ext().rows.asks(*tensors)
    if asks == 2:
        raise RuntimeError(f"{name} has no forward-mode derivative: unpack its dual inputs first")
    if asks:
        raise RuntimeError(f"{name} has no gradient: detach its inputs or call it under torch.no_grad()")


def quantize_rows(x, plan=None):
    """Rows8 of x [N, H] (fp16, bf16 or fp32, H a multiple of 16). With a rows.SortPlan the rows come in
    expert order (as rows.permute_rows brings them), each token quantised once. With m the largest
    magnitude of a block, at least 2^-96: scale = m / 448, q = e4m3(448 x / m), the nearest value,
    ties to even; of fp32 x, 448 x and the quotient are rounded to float32 first, so that one within 2^-23 of a
    midpoint can go either way.
    A NaN or infinity in a block makes its scale NaN or infinite."""
    _no_grad("quantize_rows", x)
    x = x.contiguous()
    if plan is None:
        return Rows8(*_rows._ext().quantize_rows(x))
    return Rows8(*_rows._ext().quantize_rows(x, plan.pos_of, plan.offsets))


def quantize_weight(w, halves=1):
    """Weight8 of w [E, N, K] (fp16, bf16 or fp32, K a multiple of 16). halves=2 for a gate_up stack."""
    _no_grad("quantize_weight", w)
    return Weight8(*_rows._ext().quantize_weight(w.contiguous(), halves), halves)


def grouped_gemm(x, w, offsets, swiglu=False, scale=None, dtype=torch.bfloat16):
    """Every expert's rows times its weights: x Rows8 in expert order, w Weight8, offsets int32 [E+1].
    C [rows, N] = x w^T; with scale [rows] (dtype) every row times its own; with swiglu (w quantised
    in two halves) C [rows, N/2] = silu(x gate^T) * (x up^T). Float32 up to the one rounding to `dtype`
    (bf16 or fp16). dtype float8_e4m3fn, with swiglu: the result as Rows8 for the next product, quantised
    where it is computed (scale = m / 448 and q = e4m3(v * (448 / m)) of the float32 values). Rows of no
    expert are zero. A row's bits depend on nothing but the row and its expert's weights."""
    _no_grad("grouped_gemm", x.q, x.scale, w.q, w.scale, scale)
    w.check_halves("grouped_gemm", 2 if swiglu else 1)
    out = _rows._ext().grouped_gemm_fp8(x.q, x.scale, w.q, w.scale, offsets, swiglu, scale, dtype)
    return Rows8(*out) if dtype is torch.float8_e4m3fn else out


def sorted_experts(h, plan, wsorted, gate_up, down, mode="auto"):
    """The expert FFN on 8-bit weights for a sorted batch: rows quantised into expert order, gate/up
    product with SwiGLU, its float32 result quantised where it is computed, down product times the router
    weights wsorted. There is one path for every batch (a result in h's dtype quantised by a launch of its own is
    within 3 % up to 256 tokens, and 5-9 % slower beyond): `mode` is checked and chooses nothing,
    and a row's bits do not depend on the batch. Returns y [N*k, H] in h's dtype, for combine."""
    if mode not in ("auto", "gemv", "gemm", "cublas"):
        raise RuntimeError(f"sorted_experts: unknown mode {mode!r}")
    if not (isinstance(gate_up, Weight8) and isinstance(down, Weight8)):
        raise RuntimeError("sorted_experts: gate_up and down must both be 8-bit (fp8.Weight8) or both 16-bit")
    act = grouped_gemm(quantize_rows(h, plan), gate_up, plan.offsets, swiglu=True, dtype=torch.float8_e4m3fn)
    return grouped_gemm(act, down, plan.offsets, scale=wsorted, dtype=h.dtype)
