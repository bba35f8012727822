"""The e4m3 quantisers and the experts' 8-bit product (switchyard_b200.fp8) against plain 64-bit
forms. The quantisers are exact: the same e4m3 values, the same float32 scales. The product's
bounds are derived in rows_fp8_cases (product_bound, swiglu_bound)."""

import pytest
import torch

import rows_fp8_cases as rc
from rows_fp8_cases import places, product64, product_bound, quantize64, rounding, swiglu_bound

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module")
def Q():
    from switchyard_b200 import fp8, kernels
    kernels.ext()
    yield fp8
    assert kernels.ext().device_status(DEV) == 0


def same(a, b):
    """Equal, NaN where NaN."""
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(a[~a.isnan()], b[~b.isnan()])


def same_bits(a, b):
    return a.dtype == b.dtype and torch.equal(a.view(torch.int16), b.view(torch.int16))


def hard_rows(N, H, dtype, seed):
    """Rows with the values that a quantiser can get wrong: zeros, the type's ends, subnormals, one
    large value among small ones, values midway between two e4m3 values, infinities, NaN."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(N, H, generator=g) * torch.exp(3 * torch.randn(N, 1, generator=g))
    x = x.to(dtype)
    info = torch.finfo(dtype)
    x[0] = 0
    if N > 1:
        x[1, : min(H, 64)] = info.max
        x[1, min(H, 64):] = -info.max
    if N > 2:
        x[2] = info.smallest_normal / 2
    if N > 3:
        x[3] *= 1e-3
        x[3, 0] = info.max / 2
    if N > 4:
        x[4] = torch.arange(H).to(dtype) % 17 / 16
        x[4, 0] = 1.75  # 448 / 256: quotients of sixteenths lie midway between e4m3 values
    if N > 5:
        x[5, 1] = float("inf")
    if N > 6:
        x[6, H - 1] = float("nan")
    return x


@pytest.mark.parametrize("N,H", [(1, 16), (1, 2048), (7, 128), (9, 144), (40, 1040), (300, 256), (8, 4112)])
@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_quantize_rows_is_exact(Q, N, H, dtype):
    x = hard_rows(N, H, dtype, N + H)
    got = Q.quantize_rows(x.to(DEV))
    q, s = quantize64(x, 1)
    assert got.q.dtype == torch.float8_e4m3fn and got.q.shape == (N, H) and got.scale.shape == (-(-H // 128), N)
    assert same(got.scale.cpu().t(), s) and same(got.q.cpu().double(), q)


@pytest.mark.parametrize("N,k,E,H,bad", [(1, 8, 64, 2048, 0), (5, 3, 8, 48, 0), (130, 8, 64, 256, 0), (33, 4, 60, 1040, 9)])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_quantize_rows_into_expert_order(Q, N, k, E, H, bad, dtype):
    from switchyard_b200 import kernels, rows
    idx = rc.choices(N, k, E, N, bad)
    offsets, pos = places(idx, E)
    plan = rows.plan(idx.to(DEV), E)
    assert kernels.ext().device_status(DEV) == (6 if bad else 0)
    x = hard_rows(N, H, dtype, 3)
    got = Q.quantize_rows(x.to(DEV), plan)
    q, s = quantize64(x, 1)
    want_q, want_s = torch.zeros(N * k, H, dtype=torch.float64), torch.zeros(N * k, s.shape[1])
    for j in range(k):
        ok = pos[:, j] >= 0
        want_q[pos[ok, j]], want_s[pos[ok, j]] = q[ok], s[ok]
    assert same(got.q.cpu().double(), want_q) and same(got.scale.cpu().t(), want_s)


@pytest.mark.parametrize("E,N,K,halves", [(1, 8, 16, 1), (2, 128, 128, 1), (3, 200, 144, 2), (5, 136, 1040, 1), (2, 2048, 256, 2)])
@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_quantize_weight_is_exact(Q, E, N, K, halves, dtype):
    w = torch.stack([hard_rows(N, K, dtype, 7 + e) for e in range(E)])
    got = Q.quantize_weight(w.to(DEV), halves=halves)
    parts = w.view(E * halves, N // halves, K)
    each = [quantize64(p, 128) for p in parts]
    assert same(got.q.cpu().double(), torch.stack([q for q, _ in each]).view(E, N, K))
    assert same(got.scale.cpu(), torch.stack([s for _, s in each]).view(E, -1, got.scale.shape[2]))
    fine = torch.randn(E, N, K, generator=torch.Generator().manual_seed(1))
    back = Q.quantize_weight(fine.to(DEV), halves).dequantize(halves=halves).cpu()
    # half a step of e4m3 relative to the value, or half its least subnormal (2^-10) times a scale below
    # 6 / 448 (no value reaches 6), and the roundings of the division and of the product back
    assert ((back - fine).abs() <= fine.abs() * (2.0 ** -4 + 2.0 ** -22) + 2.0 ** -10 * 6 / 448).all()


@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_quotients_next_to_a_midpoint(Q, dtype):
    """448 x / m within the type's rounding of the middle between two e4m3 values. Of 16-bit values the result is the
    e4m3 value nearest to the exact quotient (the oracle's division is in 64 bits, and no quotient of two 16-bit
    numbers is nearer than 2^-20 to a midpoint that it is not). Of float32 values 448 x and the quotient are rounded
    to float32 on the way, which may move a value across a midpoint: the result is within those two
    roundings of half a step, not always the nearest."""
    g = torch.Generator().manual_seed(5)
    N = 256
    m = (torch.rand(N, 1, generator=g) * 3 + 1).to(dtype)
    if dtype is F32:
        m[0] = 1.220261812210083
    low = torch.randint(0, 0x7e, (N, 127), generator=g).to(torch.uint8)
    mid = (low.view(torch.float8_e4m3fn).double() + (low + 1).view(torch.float8_e4m3fn).double()) / 2
    x = (mid * m.double() / 448).to(dtype) * (1 - 2 * torch.randint(0, 2, (N, 127), generator=g)).to(dtype)
    if dtype is F32:
        x[0, 0] = 0.18521831929683685
    x = torch.cat([m, x], 1)
    for scale in (1.0, 2.0 ** -12, 2.0 ** 12) + ((2.0 ** -95, 2.0 ** 126 if dtype is F32 else 2.0 ** 100) if dtype is not HF else ()):
        xs = x * scale
        top = xs.abs().amax(1, keepdim=True)
        exact = 448 * xs.double() / top.double()
        want = rc.nearest8(exact)
        if dtype is F32:
            want, nearest = rc.nearest8((xs * (448 * 2.0 ** -16)) / (top * 2.0 ** -16)), want
            assert (want != nearest).any()
            assert ((want - exact).abs() <= (nearest - exact).abs() + 2.0 ** -22 * exact.abs()).all()
        assert same(Q.quantize_rows(xs.to(DEV)).q.cpu().double(), want), scale
        w = torch.cat([xs[:1], xs[1:2] * 0, xs[2:3] * 0], 0)[None]  # a block of one row's maximum
        assert same(Q.quantize_weight(w.to(DEV)).q.cpu().double()[0, 0], want[0])


def operands(counts, K, N, swiglu, seed):
    """Rows in expert order and weights, e4m3 values and scales on the CPU."""
    g = torch.Generator().manual_seed(seed)
    M, E, parts = sum(counts), len(counts), 2 if swiglu else 1
    offsets = torch.tensor([0] + counts).cumsum(0).int()
    xq = (torch.randn(M, K, generator=g) * 100).to(torch.float8_e4m3fn)
    wq = (torch.randn(E, parts * N, K, generator=g) * 100).to(torch.float8_e4m3fn)
    xs = torch.rand(-(-K // 128), M, generator=g) * 0.01 + 1e-4
    ws = torch.rand(E, parts * -(-N // 128), -(-K // 128), generator=g) * 3e-4 + 1e-5
    return offsets, xq, xs, wq, ws


SHAPES = [([1], 16, 8), ([3, 0, 1, 70], 128, 128), ([0, 0, 5], 144, 136), ([130, 1, 257], 272, 392), ([64] * 8, 256, 256),
          ([0, 300, 0, 33, 1, 0], 1040, 1000), ([1] * 40, 2048, 64), ([600, 200], 512, 264),
          ([33, 5, 64, 1] * 8, 656, 1040)]  # the last: several rounds of every tile


@pytest.mark.parametrize("counts,K,N", SHAPES)
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("kind", ["plain", "scale", "swiglu"])
def test_grouped_gemm(Q, counts, K, N, dtype, kind):
    from switchyard_b200 import kernels
    swiglu = kind == "swiglu"
    offsets, xq, xs, wq, ws = operands(counts, K, N, swiglu, K + N)
    M = xq.shape[0]
    scale = (torch.rand(M, generator=torch.Generator().manual_seed(1)) * 2 - 1).to(dtype) if kind == "scale" else None
    acc, mag = product64(xq, xs, wq, ws, offsets, swiglu, scale)
    if swiglu:
        ref, bound = swiglu_bound(acc, mag, K, N, dtype)
    else:
        ref, (_, bound) = acc, product_bound(acc, mag, K, dtype)
    dev = [t.to(DEV) for t in (xq, xs, wq, ws, offsets)]
    sd = scale.to(DEV) if scale is not None else None
    got = Q.grouped_gemm(Q.Rows8(*dev[:2]), Q.Weight8(*dev[2:4]), dev[4], swiglu=swiglu, scale=sd, dtype=dtype)
    assert got.shape == (M, N) and got.dtype == dtype
    # (some operands drawn above 464 are NaN in e4m3: their rows and columns have to be NaN, and no others)
    nan = ref.isnan()
    assert torch.equal(got.cpu().isnan(), nan)
    over = ((got.cpu().double() - ref).abs() - bound)[~nan]
    assert (over <= 0).all(), over.max()
    for tile in (1, 2, 3):  # every tile gives the same bits
        again = kernels.ext().grouped_gemm_fp8(*dev, swiglu, sd, dtype, tile)
        assert torch.equal(again.isnan(), got.isnan()) and torch.equal(again[~nan], got[~nan]), tile


@pytest.mark.parametrize("counts,K,N", [(c, k, n) for c, k, n in SHAPES if n % 16 == 0] + [([5, 0, 140], 128, 400), ([300], 256, 1040)])
def test_swiglu_straight_to_8_bits(Q, counts, K, N):
    """The SwiGLU result as Rows8. With v the exact value, d the bound of its float32 one and M the block's
    exact largest magnitude: the scale is within d's maximum (and three roundings) of M / 448, and
    q * scale is v up to d, half a step of e4m3 (2^-4 of the value, or half its least subnormal, 2^-10
    scales) and the roundings of 448 / m, of the product and of the scale."""
    from switchyard_b200 import kernels
    offsets, xq, xs, wq, ws = operands(counts, K, N, True, 2 * K + N)
    acc, mag = product64(xq, xs, wq, ws, offsets, True, None)
    ref, bound = swiglu_bound(acc, mag, K, N, F32)
    dev = [t.to(DEV) for t in (xq, xs, wq, ws, offsets)]
    got = Q.grouped_gemm(Q.Rows8(*dev[:2]), Q.Weight8(*dev[2:4]), dev[4], swiglu=True, dtype=torch.float8_e4m3fn)
    M, blocks = xq.shape[0], -(-N // 128)
    assert got.q.dtype == torch.float8_e4m3fn and got.q.shape == (M, N) and got.scale.shape == (blocks, M)
    q, scale = got.q.cpu().double(), got.scale.cpu().double()
    for b in range(blocks):
        cols = slice(b * 128, min(N, b * 128 + 128))
        v, d, s = ref[:, cols], bound[:, cols], scale[b]
        bad = v.isnan().any(1)  # a NaN makes its row's block NaN
        assert torch.equal(s.isnan(), bad) and q[:, cols][bad].isnan().all()
        v, d, s, c = v[~bad], d[~bad], s[~bad], q[:, cols][~bad]
        m = v.abs().amax(1)
        assert ((s * 448 - m.clamp(min=2.0 ** -96)).abs() <= d.amax(1) + 2.0 ** -22 * m).all()
        far = d + (v.abs() + d) * (2.0 ** -4 + 2.0 ** -21) + 2.0 ** -10 * s[:, None]
        assert ((c * s[:, None] - v).abs() <= far).all()
    for tile in (1, 2, 3):
        again = kernels.ext().grouped_gemm_fp8(*dev, True, None, torch.float8_e4m3fn, tile)
        assert torch.equal(again[0].view(torch.uint8), got.q.view(torch.uint8))
        assert torch.equal(again[1].view(torch.int32), got.scale.view(torch.int32))
    # rows of no expert: zero values and scales
    short = dev[4].clone()
    short[-1] = max(int(short[-2]), int(short[-1]) - 1)
    less = Q.grouped_gemm(Q.Rows8(*dev[:2]), Q.Weight8(*dev[2:4]), short, swiglu=True, dtype=torch.float8_e4m3fn)
    assert (less.q[int(short[-1]):].float() == 0).all() and (less.scale[:, int(short[-1]):] == 0).all()
    assert torch.equal(less.q[:int(short[-1])].view(torch.uint8), got.q[:int(short[-1])].view(torch.uint8))


@pytest.mark.parametrize("dtype", [BF, HF, torch.float8_e4m3fn])
def test_swiglu_of_very_negative_gates(Q, dtype):
    """silu far below zero, where sigmoid is e^g: one k block and one term per sum, so gate g and value u are
    exact and only the epilogue rounds. Its relative error is that of exp2's argument, two roundings of
    126 at most (2^-17 each, times ln 2), exp2 itself and four products: below 2^-16. Below
    -87 exp is zero in float32, which leaves |g u| 2^-126. In 8 bits then half a step (2^-4, or 2^-10 scales) and
    the roundings of test_swiglu_straight_to_8_bits."""
    gates = torch.tensor([-30.0, -40, -44, -48, -60, -80, -112, -448, -1, 0, 2, 44, 208, 448, -52, -72])
    N, K, rows = 128, 16, 5
    xq, wq = torch.zeros(rows, K), torch.zeros(1, 2 * N, K)
    xq[:, 0] = torch.tensor([1.0, 1, 1, 0.5, 1])
    wq[0, :N, 0] = gates.repeat(8)
    wq[0, N:, 0] = torch.tensor([1.0, -448, 0.5, 3]).repeat(32)
    wq[0, :N, 0][64:] = wq[0, :N, 0][64:].clamp(max=-44)
    xs = torch.tensor([[1.0, 1, 0.25, 1, 2]])
    ws = torch.tensor([[[1.0], [2.0 ** 40]]])
    dev = [t.to(DEV) for t in (xq.to(torch.float8_e4m3fn), xs, wq.to(torch.float8_e4m3fn), ws)]
    offsets = torch.tensor([0, rows], dtype=torch.int32, device=DEV)
    if dtype is HF:
        dev[3] = torch.tensor([[[1.0], [2.0 ** -4]]], device=DEV)
    x = xq.double()[:, :1] * xs.double()[0][:, None]
    g, u = x * wq[0, :N, 0].double(), x * wq[0, N:, 0].double() * float(dev[3][0, 1, 0])
    ref = g * torch.exp(g) / (1 + torch.exp(g))
    ref = torch.where(g > 0, g / (1 + torch.exp(-g)), ref) * u
    d = 2.0 ** -16 * ref.abs() + (g * u).abs() * 2.0 ** -126
    for rows_ in (slice(0, rows), slice(0, 2), slice(2, 3)):
        for cols in (slice(0, N), slice(64, N)):  # the second: no gate above -44 * 0.25 in the whole block
            n = cols.stop - cols.start
            w = torch.cat([dev[2][:, :N].view(torch.uint8)[:, cols], dev[2][:, N:].view(torch.uint8)[:, cols]], 1).view(torch.float8_e4m3fn)
            M = rows_.stop - rows_.start
            got = Q.grouped_gemm(Q.Rows8(dev[0].view(torch.uint8)[rows_].view(torch.float8_e4m3fn), dev[1][:, rows_].contiguous()),
                                 Q.Weight8(w.contiguous(), dev[3]), (offsets * 0 + torch.tensor([0, M], device=DEV)).int(),
                                 swiglu=True, dtype=dtype)
            v, e = ref[rows_, cols], d[rows_, cols]
            if dtype is torch.float8_e4m3fn:
                s = got.scale.cpu().double()[0][:, None]
                e = e + (v.abs() + e) * (2.0 ** -4 + 2.0 ** -21) + 2.0 ** -10 * s
                assert ((s[:, 0] * 448 - v.abs().amax(1).clamp(min=2.0 ** -96)).abs() <= d[rows_, cols].amax(1) + 2.0 ** -22 * v.abs().amax(1)).all()
                got = got.q.cpu().double() * s
            else:
                e, got = e + rounding(v.abs() + e, dtype), got.cpu().double()
            assert got.shape == (M, n) and ((got - v).abs() <= e).all(), ((got - v).abs() / e).max()


@pytest.mark.parametrize("dtype", [BF, HF, torch.float8_e4m3fn])
def test_swiglu_of_very_negative_gates_in_every_tile(Q, dtype):
    """As above, through each tile, with more rows than one CTA of a pair has, two column blocks and an expert
    whose gates are all below -43. One term per sum, its operands of 4, 4 and 8 significant bits and powers of
    two: gate and value are exact, the bound is the one above, and the bits are the same in every tile."""
    from switchyard_b200 import kernels
    counts, N, K = [300, 70], 144, 16
    M, E = sum(counts), len(counts)
    g = torch.Generator().manual_seed(31)
    xq, wq = torch.zeros(M, K), torch.zeros(E, 2 * N, K)
    xq[:, 0] = 0.8 + 0.2 * torch.rand(M, generator=g)
    wq[0, :N, 0] = -(56 + 34 * torch.rand(N, generator=g))
    wq[1, :N, 0] = 150 * torch.rand(N, generator=g) - 130
    wq[:, N:, 0] = torch.randn(E, N, generator=g) * 3
    xq, wq = xq.to(torch.float8_e4m3fn), wq.to(torch.float8_e4m3fn)
    xs = (torch.randint(256, 320, (1, M), generator=g) / 256.0)
    up = torch.tensor([2.0 ** 60, 2.0 ** -4] if dtype is HF else [2.0 ** 40, 2.0 ** 40])
    ws = torch.ones(E, 4, 1)
    ws[:, 2:, 0] = up[:, None]
    offsets = torch.tensor([0] + counts).cumsum(0).int()
    e = torch.repeat_interleave(torch.arange(E), torch.tensor(counts))
    x = xq.double()[:, :1] * xs.double().t()
    gate, value = x * wq.double()[e, :N, 0], x * wq.double()[e, N:, 0] * up.double()[e, None]
    assert (gate[:300] < -43).all() and (gate[300:] > -43).any() and (gate[300:] < -43).any()
    ref = torch.where(gate > 0, gate / (1 + torch.exp(-gate)), gate * torch.exp(gate) / (1 + torch.exp(gate))) * value
    d = 2.0 ** -16 * ref.abs() + (gate * value).abs() * 2.0 ** -126
    dev = [t.to(DEV) for t in (xq, xs, wq, ws, offsets)]
    first = None
    for tile in (1, 2, 3):
        got = kernels.ext().grouped_gemm_fp8(*dev, True, None, dtype, tile)
        if dtype is torch.float8_e4m3fn:
            bits = (got[0].view(torch.uint8), got[1].view(torch.int32))
            for b, cols in enumerate((slice(0, 128), slice(128, N))):
                v, off, s = ref[:, cols], d[:, cols], got[1].cpu().double()[b]
                m = v.abs().amax(1)
                assert ((s * 448 - m.clamp(min=2.0 ** -96)).abs() <= off.amax(1) + 2.0 ** -22 * m).all(), tile
                far = off + (v.abs() + off) * (2.0 ** -4 + 2.0 ** -21) + 2.0 ** -10 * s[:, None]
                assert ((got[0].cpu().double()[:, cols] * s[:, None] - v).abs() <= far).all(), tile
        else:
            bits = (got.view(torch.int16),)
            assert ((got.cpu().double() - ref).abs() <= d + rounding(ref.abs() + d, dtype)).all(), tile
        first = first or bits
        assert all(torch.equal(a, b) for a, b in zip(bits, first)), tile


def test_a_rows_bits_do_not_depend_on_its_expert_s_other_rows(Q):
    from switchyard_b200 import kernels
    offsets, xq, xs, wq, ws = (t.to(DEV) for t in operands([200], 384, 160, False, 3))
    full = kernels.ext().grouped_gemm_fp8(xq, xs, wq, ws, offsets, False, None, BF)
    for at in ([7], [199, 0, 64], list(range(30, 160))):
        sub = torch.tensor([0, len(at)], dtype=torch.int32, device=DEV)
        got = kernels.ext().grouped_gemm_fp8(xq.view(torch.uint8)[at].view(xq.dtype), xs[:, at].contiguous(), wq, ws, sub, False,
                                             None, BF)
        assert same_bits(got, full[at])


def test_rows_of_no_expert_are_zero_and_offsets_are_kept_inside(Q):
    _, xq, xs, wq, ws = (t.to(DEV) for t in operands([10, 20, 10], 256, 72, False, 5))
    x, w = Q.Rows8(xq, xs), Q.Weight8(wq, ws)
    run = lambda offs: Q.grouped_gemm(x, w, torch.tensor(offs, dtype=torch.int32, device=DEV))
    whole = run([0, 10, 30, 40])
    part = run([0, 10, 30, 33])
    assert same_bits(part[:33], whole[:33]) and (part[33:] == 0).all()
    late = run([4, 10, 30, 40])
    assert same_bits(late[4:], whole[4:]) and (late[:4] == 0).all()
    assert (run([0, 0, 0, 0]) == 0).all()
    # not what a sort gives, but nothing outside the rows is read or written
    wild = run([-5, 10, 30, 4000])
    assert same_bits(wild, whole)
    falling = run([0, 30, 10, 40])
    assert torch.isfinite(falling).all()
    none = Q.grouped_gemm(Q.Rows8(xq[:0], xs[:, :0].contiguous()), w, torch.zeros(4, dtype=torch.int32, device=DEV))
    assert none.shape == (0, 72)


def test_a_row_that_is_not_finite_stays_alone(Q):
    offsets, xq, xs, wq, ws = (t.to(DEV) for t in operands([40, 8], 256, 72, False, 6))
    x = torch.randn(48, 256, device=DEV)
    x[3, 200] = float("nan")
    x[41, 0] = float("inf")
    got = Q.grouped_gemm(Q.quantize_rows(x), Q.Weight8(wq, ws), offsets)
    assert got[3].isnan().all() and got[41].isnan().all()
    assert torch.isfinite(got[[r for r in range(48) if r not in (3, 41)]]).all()


def test_more_than_2_31_elements(Q):
    """Rows, and rows of results, whose place passes 32 bits: the last rows are those of a small batch."""
    M, K, N = 1_060_000, 2048, 2056
    assert M * K > 1 << 31
    x = torch.randn(64, K, device=DEV, dtype=BF).repeat(M // 64 + 1, 1)[:M].contiguous()
    w = Q.quantize_weight(torch.randn(2, N, K, device=DEV) * K ** -0.5)
    x8 = Q.quantize_rows(x)
    offsets = torch.tensor([0, 1000, M], dtype=torch.int32, device=DEV)
    del x
    out = Q.grouped_gemm(x8, w, offsets)
    last = 1000
    few8 = Q.Rows8(x8.q[-last:].contiguous(), x8.scale[:, -last:].contiguous())
    few = Q.grouped_gemm(few8, w, torch.tensor([0, 0, last], dtype=torch.int32, device=DEV))
    assert same_bits(out[-last:], few)
    assert same_bits(out[64_000:64_064], out[M - M % 64 - 64:M - M % 64])


def layer(N, E, k, H, I, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    h = torch.randn(N, H, generator=g).to(dtype).to(DEV)
    router = (torch.randn(E, H, generator=g) * 0.2).to(dtype).to(DEV)
    gate_up = (torch.randn(E, 2 * I, H, generator=g) * H ** -0.5).to(dtype).to(DEV)
    down = (torch.randn(E, H, I, generator=g) * I ** -0.5).to(dtype).to(DEV)
    return h, router, gate_up, down


@pytest.mark.parametrize("N,E,k,H,I,dtype", [(1, 64, 8, 256, 128, BF), (7, 8, 2, 128, 48, HF), (64, 64, 8, 256, 128, HF),
                                             (333, 64, 8, 256, 144, BF), (2100, 8, 4, 256, 128, BF), (0, 8, 2, 128, 64, BF)])
def test_the_layer_on_8_bit_experts(Q, N, E, k, H, I, dtype):
    """moe_layer with Weight8 experts: route, sort, quantise into expert order, product with SwiGLU and
    its result to 8 bits where it is computed, product with router weights, combine: the bits of the
    operators called one by one in every mode, with a residual and through GraphedLayer too; and
    near the 16-bit layer."""
    from switchyard_b200 import kernels, rows
    h, router, gate_up, down = layer(N, E, k, H, I, dtype)
    gu8, dn8 = Q.quantize_weight(gate_up, halves=2), Q.quantize_weight(down)
    out = kernels.moe_layer(h, router, gu8, dn8, k, False)
    assert out.shape == h.shape and out.dtype == dtype
    if N == 0:
        return
    idx, w, counts, offsets, token, wsorted, pos_of = kernels.route_and_sort(h, router, k, False)
    plan = rows.SortPlan(counts, offsets, token, pos_of.view(N, k))
    x8 = Q.quantize_rows(h, plan)
    act = Q.grouped_gemm(x8, gu8, offsets, swiglu=True, dtype=torch.float8_e4m3fn)
    y = Q.grouped_gemm(act, dn8, offsets, scale=wsorted, dtype=dtype)
    assert torch.equal(out, kernels.ext().combine(y, pos_of, idx, N))
    for mode in ("gemv", "gemm", "cublas"):
        assert torch.equal(kernels.moe_layer(h, router, gu8, dn8, k, False, mode), out)
    some = torch.arange(0, N, 3, device=DEV)  # a row's bits do not depend on the batch
    assert torch.equal(kernels.experts(h[some], idx[some], w[some], gu8, dn8), out[some])
    assert torch.equal(kernels.experts(h, idx, w, gu8, dn8), out)
    x = torch.randn_like(h)
    assert torch.equal(kernels.moe_layer(h, router, gu8, dn8, k, False, residual=x), x + out)
    graphed = kernels.GraphedLayer(router, gu8, dn8, k, False)
    for s in (1, 2):
        hs = layer(N, E, k, H, I, dtype, seed=s)[0]
        assert torch.equal(graphed(hs), kernels.moe_layer(hs, router, gu8, dn8, k, False))
    graphed.check()
    # four operands are rounded to e4m3, each by at most 2^-4 of its values: to first order the result
    # moves by at most 4 * 2^-4 of what a sum of magnitudes would be; in the 2-norm, by less
    ref = kernels.moe_layer(h, router, gate_up, down, k, False).double()
    assert (out.double() - ref).norm() <= 0.25 * ref.norm()


def test_the_decoder_on_8_bit_experts(Q):
    """olmoe.quantize_experts: the model's own hook on 8-bit experts. A replayed decode step gives the eager
    one's bits, tokens are generated, and the logits stay near the 16-bit model's: per layer the MoE
    output moves by at most 4 * 2^-4 of itself (four operands rounded to e4m3), and what a layer adds
    is a part of the residual stream, so three layers move the normalised stream by less than 0.75."""
    from switchyard_b200 import kernels, olmoe
    c = olmoe.Config(vocab=211, hidden=256, intermediate=128, layers=3, heads=4, kv_heads=2, head_dim=64, experts=16, top_k=4,
                     max_positions=128)
    w = olmoe.random_weights(c, DEV, HF, seed=3, std=0.06)
    def decoder(w):
        hook = lambda i, h: kernels.moe_layer(h, w["layers"][i]["router"], w["layers"][i]["gate_up"], w["layers"][i]["down"],
                                              c.top_k, c.norm_topk_prob, "gemv")
        return olmoe.Decoder(c, w, hook)
    d16, d8 = decoder(w), decoder(olmoe.quantize_experts(w))
    toks = torch.randint(3, c.vocab, (3, 11), generator=torch.Generator().manual_seed(8)).to(DEV)
    a, b = d16.forward(toks).double(), d8.forward(toks).double()
    assert (a - b).norm() <= 0.75 * a.norm()
    prompts = [toks[0].tolist(), toks[1, :6].tolist()]
    assert d8.generate(prompts, 8, graph=True) == d8.generate(prompts, 8, graph=False)


def test_the_decoder_s_8_bit_experts_are_its_own(Q):
    """The 8-bit decoder against the same decoder on 16-bit experts: the dequantised ones, from which only the
    rounding of two activations to e4m3 differs, and the originals. With Z what the logits move by when the
    experts return nothing: an operand moves by at most 2^-4 of itself, so to first order an MoE output by at
    most a 2^-4 part per rounded operand, and the logits by as much of Z: Z/8 for two, Z/4 for four, and
    twice that for what lies beyond first order. Experts that return nothing or the
    opposite, of another layer, or in another order move the logits by more than that."""
    from switchyard_b200 import kernels, olmoe
    c = olmoe.Config(vocab=211, hidden=256, intermediate=128, layers=3, heads=4, kv_heads=2, head_dim=64, experts=16, top_k=4,
                     max_positions=128)
    w = olmoe.random_weights(c, DEV, HF, seed=3, std=0.06)
    toks = torch.randint(3, c.vocab, (3, 11), generator=torch.Generator().manual_seed(8)).to(DEV)
    def logits(stacks, factor=1):
        hook = lambda i, h: factor * kernels.moe_layer(h, w["layers"][i]["router"], *stacks[i], c.top_k, c.norm_topk_prob)
        return olmoe.Decoder(c, w, hook).forward(toks).double()
    plain = [(L["gate_up"], L["down"]) for L in w["layers"]]
    rounded = [(Q.quantize_weight(gu, halves=2).dequantize(HF), Q.quantize_weight(dn).dequantize(HF)) for gu, dn in plain]
    eight = [(L["gate_up"], L["down"]) for L in olmoe.quantize_experts(w)["layers"]]
    got, ref, original = logits(eight), logits(rounded), logits(plain)
    zero = (logits(rounded, 0) - ref).norm()
    assert (got - ref).norm() <= zero / 4
    assert (got - original).norm() <= zero / 2
    shifted = [tuple(Q.Weight8(t.q.view(torch.uint8).roll(1, 0).view(t.q.dtype), t.scale.roll(1, 0), t.halves) for t in pair)
               for pair in eight]
    for wrong in (logits(eight, 0), logits(eight, -1), logits(eight[1:] + eight[:1]), logits(shifted)):
        assert (wrong - ref).norm() > zero / 2


def test_a_stack_quantised_as_one_is_not_taken_for_gate_and_up(Q):
    """Experts of width 200: the two layouts' scales have the same shape (four blocks of rows)."""
    from switchyard_b200 import kernels
    h, router, gate_up, _ = layer(4, 8, 2, 128, 200, BF)
    plain, halved = Q.quantize_weight(gate_up), Q.quantize_weight(gate_up, halves=2)
    assert plain.scale.shape == halved.scale.shape and not torch.equal(plain.scale, halved.scale)
    x8, offsets = Q.quantize_rows(h), torch.tensor([0] + [4] * 8, dtype=torch.int32, device=DEV)
    for w, swiglu in ((plain, True), (halved, False)):
        with pytest.raises(RuntimeError, match="halves"):
            Q.grouped_gemm(x8, w, offsets, swiglu=swiglu)
    down = Q.quantize_weight(torch.zeros(8, 128, 208, device=DEV))
    with pytest.raises(RuntimeError, match="halves"):
        kernels.moe_layer(h, router, plain, down, 2, False)
    x, wide = x8.dequantize().cpu().double(), plain.dequantize()[0].cpu().double()
    want, mag = x @ wide.t(), x.abs() @ wide.abs().t()
    got = Q.grouped_gemm(x8, plain, offsets).cpu().double()
    # (dequantize rounds value times scale to float32 on either side)
    assert ((got - want).abs() <= product_bound(want, mag, 128, BF)[1] + 2.0 ** -22 * mag).all()


def test_sizes_past_32_bits_are_refused(Q):
    """Not taken for what their lower 32 bits say: 2^32 + 16 columns for 16."""
    x = torch.empty(1, (1 << 32) + 16, dtype=BF, device=DEV)
    with pytest.raises(RuntimeError, match="at most"):
        Q.quantize_rows(x)
    with pytest.raises(RuntimeError, match="at most"):
        Q.quantize_weight(x[None])
    del x
    from switchyard_b200 import rows
    p = rows.plan(torch.zeros(1, 1, dtype=torch.int32, device=DEV), 1)
    h = torch.empty(1, (1 << 32) + 16, dtype=BF, device=DEV)
    for call in (lambda: rows.permute_rows(h, p), lambda: rows.unpermute_rows(h, None, p)):
        with pytest.raises(RuntimeError, match="at most"):
            call()


def test_functional_transforms_are_refused(Q):
    x, w = torch.randn(4, 128, device=DEV), torch.randn(2, 8, 128, device=DEV)
    w8, offsets = Q.quantize_weight(w), torch.tensor([0, 2, 4], dtype=torch.int32, device=DEV)
    x8 = Q.quantize_rows(x)
    total = lambda r: (r.scale if isinstance(r, tuple) else r).sum()
    calls = (lambda a: Q.quantize_rows(a), lambda a: Q.quantize_weight(a[None]),
             lambda a: Q.grouped_gemm(x8, w8, offsets, scale=a[:, 0].bfloat16()))
    for call in calls:
        for transformed in (lambda: torch.func.grad(lambda a: total(call(a)))(x), lambda: torch.func.jvp(lambda a: total(call(a)), (x,), (x,)),
                            lambda: torch.func.vmap(lambda a: total(call(a)))(torch.stack([x, x]))):
            with pytest.raises(RuntimeError):
                transformed()


def test_streams_and_graphs(Q):
    """The same call on two streams at once and replayed from a graph, on new inputs."""
    offsets, xq, xs, wq, ws = (t.to(DEV) for t in operands([20, 0, 300], 256, 256, True, 9))
    w = Q.Weight8(wq, ws)
    x = torch.randn(320, 256, device=DEV).to(BF)
    run = lambda: Q.grouped_gemm(Q.quantize_rows(x), w, offsets, swiglu=True)
    want = run()
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for s in streams * 3:
        with torch.cuda.stream(s):
            outs.append(run())
    torch.cuda.synchronize()
    assert all(same_bits(o, want) for o in outs)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    x.copy_(torch.randn(320, 256, device=DEV).to(BF))
    graph.replay()
    torch.cuda.synchronize()
    assert same_bits(out, run())


def test_refusals(Q):
    from switchyard_b200 import kernels
    from switchyard_b200.rows import plan
    offsets, xq, xs, wq, ws = (t.to(DEV) for t in operands([4, 4], 128, 64, False, 1))
    x, w = Q.Rows8(xq, xs), Q.Weight8(wq, ws)
    bad = [dict(x=x._replace(scale=xs.t())), dict(x=x._replace(q=xq.float())), dict(w=w._replace(scale=ws[:1])),
           dict(w=w._replace(q=wq.cpu())), dict(offsets=offsets[:2]), dict(offsets=offsets.long()), dict(dtype=F32),
           dict(scale=torch.ones(8, device=DEV)), dict(scale=torch.ones(7, device=DEV, dtype=BF)),
           dict(swiglu=True, scale=torch.ones(8, device=DEV, dtype=BF)), dict(dtype=torch.float8_e4m3fn)]
    for change in bad:
        with pytest.raises(RuntimeError):
            Q.grouped_gemm(**{**dict(x=x, w=w, offsets=offsets), **change})
    odd = operands([4, 4], 120, 64, False, 1)
    with pytest.raises(RuntimeError, match="multiple of 16"):
        Q.grouped_gemm(Q.Rows8(odd[1].to(DEV), odd[2].to(DEV)), Q.Weight8(odd[3].to(DEV), odd[4].to(DEV)), offsets)
    for t in (torch.zeros(4, 24, device=DEV), torch.zeros(4, 32), torch.zeros(4, 32, device=DEV).double(), torch.zeros(32, device=DEV)):
        with pytest.raises(RuntimeError):
            Q.quantize_rows(t)
    for t, halves in ((torch.zeros(2, 3, 32, device=DEV), 2), (torch.zeros(3, 32, device=DEV), 1), (torch.zeros(1, 8, 40, device=DEV), 1),
                      (torch.zeros(1, 9, 32, device=DEV), 3)):
        with pytest.raises(RuntimeError):
            Q.quantize_weight(t, halves)
    with pytest.raises(RuntimeError, match="multiple of 16"):  # experts of width 136: 16-bit only
        Q.quantize_weight(layer(1, 8, 2, 256, 136, BF)[3])
    p = plan(torch.zeros(4, 2, dtype=torch.int32, device=DEV), 8)
    for places_ in ((p.pos_of, None), (None, p.offsets), (p.pos_of[:3], p.offsets), (p.pos_of.long(), p.offsets)):
        with pytest.raises(RuntimeError, match="quantize_rows"):
            kernels.ext().quantize_rows(torch.zeros(4, 32, device=DEV), *places_)
    leaf = torch.zeros(4, 32, device=DEV, requires_grad=True)
    with pytest.raises(RuntimeError, match="no gradient"):
        Q.quantize_rows(leaf)
    with torch.no_grad():
        Q.quantize_rows(leaf)
    h, router, gate_up, down = layer(4, 8, 2, 128, 64, BF)
    gu8 = Q.quantize_weight(gate_up, halves=2)
    with pytest.raises(RuntimeError, match="both"):
        kernels.moe_layer(h, router, gu8, down, 2, False)
    with pytest.raises(RuntimeError, match="mode"):
        kernels.moe_layer(h, router, gu8, Q.quantize_weight(down), 2, False, "other")
    with pytest.raises(RuntimeError, match="8-bit"):
        kernels.ffn(h, None, offsets, None, None, gu8, down, 4, "gemv")
