"""Plain 64-bit forms of the row operators, the e4m3 quantisers and the 8-bit product, and the
rounding bounds the tests hold the kernels to. Everything runs on the CPU."""

import torch

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}  # eps / 2
SMALLEST = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}  # half the least subnormal
TINY = 2.0 ** -96


def rounding(ref, dtype):
    """Most that rounding `ref` once to dtype can change it."""
    return HALF_STEP[dtype] * ref.abs() + SMALLEST[dtype]


def choices(N, k, E, seed, bad=0):
    """idx int32 [N, k]: distinct experts per token; `bad` choices get an id outside [0, E)."""
    g = torch.Generator().manual_seed(seed)
    idx = torch.rand(N, E, generator=g).topk(k, 1).indices.int() if N else torch.zeros(0, k, dtype=torch.int32)
    if bad:
        at = torch.randperm(N * k, generator=g)[:bad]
        idx.view(-1)[at] = torch.where(torch.arange(bad) % 2 == 0, -1, E).int()
    return idx


def places(idx, E):
    """(offsets, pos_of) of the stable sort; choices outside [0, E) have no place (-1)."""
    flat = idx.flatten().long()
    ok = (flat >= 0) & (flat < E)
    order = torch.argsort(torch.where(ok, flat, E), stable=True)
    pos = torch.full_like(flat, -1)
    used = int(ok.sum())
    pos[order[:used]] = torch.arange(used)
    offsets = torch.zeros(E + 1, dtype=torch.int64)
    offsets[1:] = torch.bincount(flat[ok], minlength=E).cumsum(0)
    return offsets, pos.view(idx.shape)


def permute64(h, pos, M):
    x = torch.zeros(M, h.shape[1], dtype=torch.float64)
    for j in range(pos.shape[1]):
        ok = pos[:, j] >= 0
        x[pos[ok, j]] = h.double()[ok]
    return x


def unpermute64(y, w, pos):
    """(sum, sum of magnitudes) in 64 bits."""
    N, k = pos.shape
    out = torch.zeros(N, y.shape[1], dtype=torch.float64)
    mag = torch.zeros_like(out)
    for j in range(k):
        ok = pos[:, j] >= 0
        term = y.double()[pos[:, j].clamp(min=0)] * (w.double()[:, j:j + 1] if w is not None else 1.0)
        out[ok] += term[ok]
        mag[ok] += term[ok].abs()
    return out, mag


def sum_bound(ref, mag, terms, dtype):
    """A float32 sum of `terms` float32 products (2^-24 each for product and addition), then one
    rounding to dtype of a value that far off."""
    off = 2 * terms * 2.0 ** -24 * mag
    return off + rounding(ref.abs() + off, dtype)


def nearest8(v):
    """The nearest e4m3 value, ties to even, saturating at 448; steps 2^(exponent-3), 2^-9 below 2^-6."""
    v = v.double()
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6, max=1e300))) - 3)
    r = torch.round(v / step) * step
    return torch.where(v.isnan(), v, r.clamp(-448, 448))


def quantize64(x, block_rows):
    """(values as float64, scales as float32) of x [R, K] in blocks block_rows x 128."""
    R, K = x.shape
    q, scale = torch.empty(R, K, dtype=torch.float64), torch.empty(-(-R // block_rows), -(-K // 128))
    for r in range(0, R, block_rows):
        for c in range(0, K, 128):
            b = x[r:r + block_rows, c:c + 128]
            m = b.float().abs().amax()
            m = m if m.isnan() else m.clamp(min=TINY)
            scale[r // block_rows, c // 128] = m / torch.tensor(448.0)  # float32 division of tensors
            # both sides of the float32 division carry 2^-16, as in the kernel: no overflow
            quotient = (b.float() * (448.0 * 2.0 ** -16)) / (m * 2.0 ** -16)
            q[r:r + block_rows, c:c + 128] = nearest8(quotient)
    return q, scale


def product64(xq, xs, wq, ws, offsets, swiglu, scale):
    """(result, sum of magnitudes behind gate and up or the plain sum) in 64 bits from e4m3 values
    (as float64) and float32 scales."""
    E, Nf, K = wq.shape
    parts = 2 if swiglu else 1
    N = Nf // parts
    x = xq.double() * xs.double().t().repeat_interleave(128, 1)[:, :K]
    s = ws.double().view(E * parts, -1, ws.shape[-1]).repeat_interleave(128, 1)[:, :N].repeat_interleave(128, 2)[:, :, :K]
    w = wq.double() * s.reshape(E, Nf, K)
    acc = torch.zeros(x.shape[0], Nf, dtype=torch.float64)
    mag = torch.zeros_like(acc)
    for e in range(E):
        a, b = int(offsets[e]), int(offsets[e + 1])
        acc[a:b] = x[a:b] @ w[e].t()
        mag[a:b] = x[a:b].abs() @ w[e].abs().t()
    if scale is not None:
        return acc * scale.double()[:, None], mag * scale.double().abs()[:, None]
    return acc, mag


def product_bound(acc, mag, K, dtype):
    """Float32 sums of K exact products: each of the K additions and of the ceil(K/128) promotions
    (scale product, multiply-add) is off by at most 2^-23 of the magnitudes summed so far."""
    off = (K + 3 * -(-K // 128) + 1) * 2.0 ** -23 * mag
    return off, off + rounding(acc.abs() + off, dtype)


def swiglu_bound(acc, mag, K, N, dtype):
    """silu(g) * u with g and u off as above: |silu'| <= 1.1, exp and division within 2^-20."""
    off, _ = product_bound(acc, mag, K, dtype)
    g, u = acc[:, :N], acc[:, N:]
    silu = g * torch.sigmoid(g)
    ref = silu * u
    far = 1.1 * off[:, :N] * (u.abs() + off[:, N:]) + silu.abs() * off[:, N:] + 2.0 ** -20 * ref.abs()
    return ref, far + rounding(ref.abs() + far, dtype)
