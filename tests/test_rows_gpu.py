"""Token rows into expert order and back (switchyard_b200.rows) and their gradients against plain
64-bit forms. Bounds (rows_fp8_cases): copies are exact; a sum of n products in float32 is off by
at most 2 n 2^-24 of the magnitudes summed, then half a step of the result's type."""

import pytest
import torch

import rows_fp8_cases as rc
from rows_fp8_cases import permute64, places, rounding, sum_bound, unpermute64

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32

#        N    k  E    H     seed, choices without a valid expert
SIZES = [(1, 8, 64, 2048, 0), (1, 1, 1, 8, 0), (5, 2, 8, 24, 0), (33, 3, 60, 264, 0), (64, 8, 64, 256, 0),
         (257, 4, 60, 1000, 0), (40, 8, 128, 4104, 0), (1031, 8, 64, 64, 0), (19, 4, 16, 136, 7), (6, 2, 8, 512, 12)]


@pytest.fixture(scope="module")
def R():
    from switchyard_b200 import kernels, rows
    kernels.ext()
    yield rows
    assert kernels.ext().device_status(DEV) == 0


def clear_status():
    """The sort reports choices it skipped (status 6); the tests that plant them take the report."""
    from switchyard_b200 import kernels
    return kernels.ext().device_status(DEV)


def setup(R, N, k, E, bad, seed=0):
    idx = rc.choices(N, k, E, seed + N + k, bad)
    offsets, pos = places(idx, E)
    p = R.plan(idx.to(DEV), E)
    assert torch.equal(p.offsets.cpu().long(), offsets) and torch.equal(p.pos_of.cpu().long(), pos)
    assert torch.equal(p.counts.cpu().long(), offsets[1:] - offsets[:-1])
    if bad:
        assert clear_status() == 6
    return idx, pos, p


@pytest.mark.parametrize("N,k,E,H,bad", SIZES)
@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_permute_and_its_gradient(R, N, k, E, H, bad, dtype):
    idx, pos, p = setup(R, N, k, E, bad)
    g = torch.Generator().manual_seed(N * k + H)
    h, dx = torch.randn(N, H, generator=g).to(dtype), torch.randn(N * k, H, generator=g).to(dtype)
    hd = h.to(DEV).requires_grad_()
    x = R.permute_rows(hd, p)
    assert x.shape == (N * k, H) and x.dtype == dtype
    assert torch.equal(x.detach().cpu().double(), permute64(h, pos, N * k))
    with torch.no_grad():
        assert torch.equal(R.permute_rows(hd, p), x)
    dh, = torch.autograd.grad(x, hd, dx.to(DEV))
    ref, mag = unpermute64(dx, None, pos)
    assert ((dh.cpu().double() - ref).abs() <= sum_bound(ref, mag, k, dtype)).all()
    for t in torch.nonzero((pos < 0).all(1)).flatten():
        assert (dh[t] == 0).all()


@pytest.mark.parametrize("N,k,E,H,bad", SIZES)
@pytest.mark.parametrize("dtype,wdtype", [(BF, BF), (BF, F32), (HF, HF), (HF, F32), (F32, F32)])
def test_unpermute_and_its_gradients(R, N, k, E, H, bad, dtype, wdtype):
    idx, pos, p = setup(R, N, k, E, bad)
    g = torch.Generator().manual_seed(N * k + H + 1)
    y, dout = torch.randn(N * k, H, generator=g).to(dtype), torch.randn(N, H, generator=g).to(dtype)
    w = torch.randn(N, k, generator=g).to(wdtype)
    yd, wd = y.to(DEV).requires_grad_(), w.to(DEV).requires_grad_()
    out = R.unpermute_rows(yd, wd, p)
    ref, mag = unpermute64(y, w, pos)
    assert out.dtype == dtype and ((out.detach().cpu().double() - ref).abs() <= sum_bound(ref, mag, k, dtype)).all()
    dy, dw = torch.autograd.grad(out, (yd, wd), dout.to(DEV))
    want = torch.zeros(N * k, H, dtype=torch.float64)
    dots, magw = torch.zeros(N, k, dtype=torch.float64), torch.zeros(N, k, dtype=torch.float64)
    for j in range(k):
        ok = pos[:, j] >= 0
        want[pos[ok, j]] = (dout.double() * w.double()[:, j:j + 1])[ok]
        term = dout.double() * y.double()[pos[:, j].clamp(min=0)] * ok[:, None]
        dots[:, j], magw[:, j] = term.sum(1), term.abs().sum(1)
    # one product in float32 (exact for 16-bit operands), one rounding
    assert dy.dtype == dtype and ((dy.cpu().double() - want).abs() <= rounding(want, dtype) + 2.0 ** -24 * want.abs()).all()
    assert dw.dtype == wdtype and dw.shape == (N, k)
    assert ((dw.cpu().double() - dots).abs() <= sum_bound(dots, magw, H, wdtype)).all()
    # each gradient alone has the same bits
    for leaf, full in ((yd, dy), (wd, dw)):
        other = [t.detach() if t is not leaf else t for t in (yd, wd)]
        assert torch.equal(torch.autograd.grad(R.unpermute_rows(*other, p), leaf, dout.to(DEV))[0], full)
    # a plain sum
    plain = R.unpermute_rows(yd.detach(), None, p)
    ref, mag = unpermute64(y, None, pos)
    assert ((plain.cpu().double() - ref).abs() <= sum_bound(ref, mag, k, dtype)).all()
    dplain, = torch.autograd.grad(R.unpermute_rows(yd, None, p), yd, dout.to(DEV))
    assert torch.equal(dplain.cpu().double(), permute64(dout, pos, N * k))


def test_no_tokens(R):
    p = R.plan(torch.zeros(0, 8, dtype=torch.int32, device=DEV), 64)
    assert p.offsets.tolist() == [0] * 65
    h = torch.zeros(0, 256, dtype=BF, device=DEV, requires_grad=True)
    x = R.permute_rows(h, p)
    w = torch.zeros(0, 8, device=DEV, requires_grad=True)
    out = R.unpermute_rows(x, w, p)
    assert x.shape == (0, 256) and out.shape == (0, 256)
    dh, dw = torch.autograd.grad(out.sum(), (h, w))
    assert dh.shape == (0, 256) and dw.shape == (0, 8)


def test_gradients_against_differences(R):
    """Both operators are linear in the rows and in the weights, so a central difference of any
    width is the directional derivative; float32 rows of H=64. With |dout|, |w| and the direction's
    entries below 6, y below 6: each of the N*k*H products is below 6^4, summed in 64 bits from
    float32 values that are k 2^-24 off."""
    N, k, E, H = 23, 4, 16, 64
    idx, pos, p = setup(R, N, k, E, 0, seed=5)
    g = torch.Generator().manual_seed(9)
    rnd = lambda *s: torch.randn(*s, generator=g).clamp(-5.9, 5.9).to(DEV)
    y, w, dout, vy, vw, h, vh, dx = (rnd(N * k, H), rnd(N, k), rnd(N, H), rnd(N * k, H), rnd(N, k), rnd(N, H), rnd(N, H),
                                     rnd(N * k, H))
    ya, wa, ha = y.clone().requires_grad_(), w.clone().requires_grad_(), h.clone().requires_grad_()
    dy, dw = torch.autograd.grad(R.unpermute_rows(ya, wa, p), (ya, wa), dout)
    dh, = torch.autograd.grad(R.permute_rows(ha, p), ha, dx)
    dot = lambda a, b: (a.double() * b.double()).sum().item()
    off = N * H * 6.0 * (2 * (k + 2) * 2.0 ** -24) * k * 6.0 * 12.0  # dout * (float32 error of either side)
    assert abs(dot(dout, R.unpermute_rows(y + vy, w, p)) - dot(dout, R.unpermute_rows(y - vy, w, p)) - 2 * dot(dy, vy)) <= off
    assert abs(dot(dout, R.unpermute_rows(y, w + vw, p)) - dot(dout, R.unpermute_rows(y, w - vw, p)) - 2 * dot(dw, vw)) <= \
        off + N * k * 6 * 2 * H * 2.0 ** -24 * H * 36
    assert abs(dot(dx, R.permute_rows(h + vh, p)) - dot(dx, R.permute_rows(h - vh, p)) - 2 * dot(dh, vh)) <= off


def test_second_derivatives_are_refused_not_lost(R):
    """dy depends on w and dw on y, whether or not the gradient that came in asks for one of its own: a gradient
    of them has to end in an error, and not in the rest of a sum."""
    idx, pos, p = setup(R, 6, 2, 4, 0, seed=14)
    y, w = torch.randn(12, 64, device=DEV, requires_grad=True), torch.rand(6, 2, device=DEV, requires_grad=True)
    dout = torch.ones(6, 64, device=DEV)
    first, second = torch.autograd.grad(R.unpermute_rows(y, w, p), (y, w), dout, create_graph=True)
    for loss, leaf in ((first.sum(), w), (second.sum(), y), ((first ** 2).sum() + w.sum(), w), (second.sum() + y.sum(), y)):
        with pytest.raises(RuntimeError, match="second"):
            torch.autograd.grad(loss, leaf, retain_graph=True)
    d = dout.clone().requires_grad_()
    h = torch.randn(6, 64, device=DEV, requires_grad=True)
    dh, = torch.autograd.grad(R.permute_rows(h, p), h, torch.cat([d, d]), create_graph=True)
    with pytest.raises(RuntimeError, match="second"):
        torch.autograd.grad(dh.sum() + d.sum(), d)
    assert torch.equal(first.detach(), torch.autograd.grad(R.unpermute_rows(y, w, p), y, dout)[0])
    one, = torch.autograd.grad(R.unpermute_rows(y, w.detach(), p), y, d, create_graph=True)  # w alone is a constant
    assert torch.equal(one, first)
    with pytest.raises(RuntimeError, match="second"):
        torch.autograd.grad(one.sum() + d.sum(), d)


def test_within_autograd(R):
    """What autograd lets a user do with the nodes: ask for one of two gradients, run backward twice on a kept
    graph and not on a freed one, recompute under checkpoint, keep saved tensors on the host, change a saved
    plan (an error), and run from two threads."""
    import threading

    from torch.utils.checkpoint import checkpoint
    idx, pos, p = setup(R, 21, 4, 16, 0, seed=15)
    g = torch.Generator().manual_seed(4)
    rnd = lambda *s: torch.randn(*s, generator=g).to(BF).to(DEV)
    h, w, d = rnd(21, 128).requires_grad_(), torch.rand(21, 4, generator=g).to(DEV).requires_grad_(), rnd(21, 128)
    layer = lambda h, w: R.unpermute_rows(R.permute_rows(h, p) * 2, w, p)
    out = layer(h, w)
    dh, dw = torch.autograd.grad(out, (h, w), d, retain_graph=True)
    for leaf, want in ((h, dh), (w, dw)):
        assert torch.equal(torch.autograd.grad(out, leaf, d, retain_graph=True)[0], want)
    out.backward(d)
    assert torch.equal(h.grad, dh) and torch.equal(w.grad, dw)
    with pytest.raises(RuntimeError, match="second time"):
        out.backward(d)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(checkpoint(layer, h, w, use_reentrant=False), (h, w), d), (dh, dw)))
    h.grad = w.grad = None
    checkpoint(layer, h, w, use_reentrant=True).backward(d)
    assert torch.equal(h.grad, dh) and torch.equal(w.grad, dw)
    with torch.autograd.graph.save_on_cpu():
        out = layer(h, w)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, (h, w), d), (dh, dw)))
    with torch.no_grad():
        assert not layer(h, w).requires_grad
    got = [None, None]
    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got[i] = torch.autograd.grad(layer(h, w), (h, w), d)
            torch.cuda.current_stream().synchronize()
    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [t.start() for t in threads], [t.join() for t in threads]
    assert all(torch.equal(a, b) for pair in got for a, b in zip(pair, (dh, dw)))
    mine = R.SortPlan(*(t.clone() for t in p))
    x = R.permute_rows(h, mine)
    mine.pos_of.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        x.sum().backward()


def test_functional_transforms_are_refused(R):
    """Their wrappers have no memory of their own: an error, not a result without the transform."""
    idx, pos, p = setup(R, 5, 2, 4, 0, seed=16)
    h, y, w = torch.randn(5, 64, device=DEV), torch.randn(10, 64, device=DEV), torch.rand(5, 2, device=DEV)
    calls = (lambda: torch.func.grad(lambda a: R.permute_rows(a, p).sum())(h), lambda: torch.func.grad(lambda a: R.unpermute_rows(y, a, p).sum())(w),
             lambda: torch.func.jvp(lambda a: R.permute_rows(a, p), (h,), (h,)), lambda: torch.func.jvp(lambda a: R.unpermute_rows(a, w, p), (y,), (y,)),
             lambda: torch.func.vmap(lambda a: R.permute_rows(a, p))(torch.stack([h, h])),
             lambda: torch.func.vmap(lambda a: R.unpermute_rows(y, a, p))(torch.stack([w, w])))
    for call in calls:
        with pytest.raises(RuntimeError):
            call()


def test_the_order_of_the_sum_is_combines(R):
    """Without weights unpermute_rows gives combine's bits; with the weights applied to the rows
    first (float32 rows and products exact) the weighted sum's bits."""
    from switchyard_b200 import kernels
    for dtype in (BF, HF):
        idx, pos, p = setup(R, 130, 8, 64, 0, seed=3)
        y = torch.randn(130 * 8, 512, generator=torch.Generator().manual_seed(1)).to(dtype).to(DEV)
        want = kernels.ext().combine(y, p.pos_of.view(-1), idx.to(DEV), 130)
        assert torch.equal(R.unpermute_rows(y, None, p), want)
        assert torch.equal(R.unpermute_rows(y, torch.ones(130, 8, device=DEV), p), want)


def test_the_same_expert_twice(R):
    idx = torch.tensor([[3, 3, 1], [1, 1, 1]], dtype=torch.int64, device=DEV)
    p = R.plan(idx, 4)
    assert p.pos_of.tolist() == [[4, 5, 0], [1, 2, 3]] and p.offsets.tolist() == [0, 0, 4, 4, 6]
    h = torch.randn(2, 64, device=DEV, requires_grad=True)
    x = R.permute_rows(h, p)
    out = R.unpermute_rows(x, torch.full((2, 3), 0.5, device=DEV), p)
    assert torch.equal(out, 1.5 * h)
    dh, = torch.autograd.grad(out, h, torch.ones_like(out))
    assert (dh == 1.5).all()


def test_strided_inputs_and_expanded_gradients(R):
    idx, pos, p = setup(R, 31, 4, 16, 0, seed=11)
    g = torch.Generator().manual_seed(2)
    wide = torch.randn(31, 2 * 72, generator=g).to(DEV)
    h = wide[:, ::2].requires_grad_()  # every other column
    x = R.permute_rows(h, p)
    assert torch.equal(x.cpu().double(), permute64(h.detach().cpu(), pos, 31 * 4))
    assert (torch.autograd.grad(x.sum(), h)[0] == 4).all()  # the incoming gradient is one expanded number
    w = torch.randn(4, 31, generator=g).to(DEV).t().requires_grad_()
    y = x.detach().requires_grad_()
    out = R.unpermute_rows(y, w, p)
    dy, dw = torch.autograd.grad(out.sum(), (y, w))
    assert torch.equal(dy.cpu().double(), permute64(torch.ones(31, 72), pos, 124) *
                       w.detach().cpu().double().flatten()[torch.argsort(pos.flatten())][:, None])
    rows_sum = y.detach().cpu().double().sum(1)[pos]
    mag = y.detach().cpu().double().abs().sum(1)[pos]
    assert ((dw.cpu().double() - rows_sum).abs() <= sum_bound(rows_sum, mag, 72, F32)).all()


def test_gradients_that_start_between_16_byte_boundaries(R):
    """A flat torch.cat hands its inputs slices of one gradient, which may start anywhere."""
    from switchyard_b200 import kernels
    idx, pos, p = setup(R, 9, 2, 4, 0, seed=12)
    g = torch.Generator().manual_seed(3)
    h, one = torch.randn(9, 64, generator=g).to(DEV).requires_grad_(), torch.zeros(1, device=DEV, requires_grad=True)
    w = torch.rand(9, 2, generator=g).to(DEV).requires_grad_()
    x = R.permute_rows(h, p)
    d = torch.randn(1 + x.numel(), generator=g).to(DEV)
    dh, = torch.autograd.grad(torch.cat([one, x.flatten()]), h, d)
    assert torch.equal(dh, kernels.ext().unpermute_rows(d[1:].clone().view(x.shape), None, p.pos_of))
    y = x.detach().requires_grad_()
    out = R.unpermute_rows(y, w, p)
    d = d[:1 + out.numel()].clone()
    dy, dw = torch.autograd.grad(torch.cat([one, out.flatten()]), (y, w), d)
    want = kernels.ext().unpermute_rows_grad(d[1:].clone().view(out.shape), y.detach(), w.detach(), p.pos_of, p.offsets)
    assert torch.equal(dy, want[0]) and torch.equal(dw, want[1])


def test_values_that_are_not_finite_stay_in_their_token(R):
    idx, pos, p = setup(R, 9, 2, 8, 0, seed=4)
    y = torch.ones(18, 16, dtype=BF)
    y[pos[2, 0]], y[pos[5, 1], 3] = float("nan"), float("inf")
    w = torch.ones(9, 2)
    w[2, 0] = 0.0  # 0 * NaN is NaN, as in the plain form
    out = R.unpermute_rows(y.to(DEV), w.to(DEV), p).cpu()
    assert out[2].isnan().all() and out[5, 3] == float("inf") and torch.isfinite(out[[0, 1, 3, 4, 6, 7, 8]]).all()
    assert torch.isfinite(out[5, :3]).all()


def test_rows_of_skipped_choices_get_zero_gradients(R):
    """A choice without a row: nothing is read through it, its weight's gradient is zero, the rows
    behind the last one are zero in x and in dy."""
    N, k, E, H = 12, 4, 8, 40
    idx, pos, p = setup(R, N, k, E, 9, seed=8)
    used = int(p.offsets[-1])
    assert used == N * k - 9
    h = torch.randn(N, H, device=DEV, requires_grad=True)
    w = torch.rand(N, k, device=DEV, requires_grad=True)
    x = R.permute_rows(h, p)
    assert (x[used:] == 0).all()
    y = torch.full_like(x, float("nan"))  # what an expert would leave in rows it does not own
    y[:used] = 1.0
    y.requires_grad_()
    out = R.unpermute_rows(y, w, p)
    assert torch.isfinite(out).all()
    dy, dw = torch.autograd.grad(out, (y, w), torch.ones_like(out))
    assert (dy[used:] == 0).all() and (dw.cpu()[pos < 0] == 0).all() and (dw.cpu()[pos >= 0] == H).all()


def test_on_another_stream_and_in_a_graph(R):
    N, k, E, H = 77, 8, 64, 320
    idx, pos, p = setup(R, N, k, E, 0, seed=6)
    h, w = torch.randn(N, H, device=DEV).to(BF), torch.rand(N, k, device=DEV)
    want = R.unpermute_rows(R.permute_rows(h, p), w, p)
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    outs = []
    for s in (side, other, side):  # two streams at once, on the same plan
        with torch.cuda.stream(s):
            outs.append(R.unpermute_rows(R.permute_rows(h, p), w, p))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = R.unpermute_rows(R.permute_rows(h, p), w, p)
            ext_dy, ext_dw = R._ext().unpermute_rows_grad(h, R.permute_rows(h, p), w, p.pos_of, p.offsets)
    h.copy_(torch.randn(N, H, device=DEV).to(BF))
    graph.replay()
    torch.cuda.synchronize()
    x = R.permute_rows(h, p)
    assert torch.equal(out, R.unpermute_rows(x, w, p))
    dy, dw = R._ext().unpermute_rows_grad(h, x, w, p.pos_of, p.offsets)
    assert torch.equal(dy, ext_dy) and torch.equal(dw, ext_dw)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_a_trained_layer(R, dtype):
    """Router softmax, both operators and one matrix per expert, forward and backward, against the
    same layer in 64 bits by autograd. The 64-bit layer gets the operators' own 16-bit x and y
    where they enter a product, so that what is compared is these operators' arithmetic."""
    N, k, E, H = 37, 3, 8, 64
    g = torch.Generator().manual_seed(21)
    h, router = torch.randn(N, H, generator=g).to(dtype), torch.randn(E, H, generator=g) * 0.3
    mats, dout = torch.randn(E, H, H, generator=g) * H ** -0.5, torch.randn(N, H, generator=g).to(dtype)
    hd, rd, md = h.to(DEV).requires_grad_(), router.to(DEV).requires_grad_(), mats.to(DEV).requires_grad_()
    probs = torch.softmax(hd.float() @ rd.t(), -1)
    w, idx = probs.topk(k, -1)
    p = R.plan(idx, E)
    x = R.permute_rows(hd, p)
    off = p.offsets.tolist()
    y = torch.cat([x[off[e]:off[e + 1]].double() @ md[e].double() for e in range(E)]).to(dtype)
    out = R.unpermute_rows(y, w, p)
    grads = torch.autograd.grad(out, (hd, rd, md), dout.to(DEV))
    h64, r64, m64 = (t.detach().double().requires_grad_() for t in (hd, rd, md))
    p64 = torch.softmax(h64 @ r64.t(), -1)
    each = torch.stack([h64 @ m64[e] for e in range(E)], 1)  # [N, E, H]
    picked = each.gather(1, idx[..., None].expand(-1, -1, H))
    out64 = (picked * p64.gather(1, idx)[..., None]).sum(1)
    grads64 = torch.autograd.grad(out64, (h64, r64, m64), dout.to(DEV).double())
    # every result passes at most four roundings to dtype (x is exact; y, dy, dx, dh or out) and float32
    # arithmetic of fewer than H * E terms; norms add up by the triangle inequality, and none of the
    # linear maps between a rounding and a result amplifies it by more than its own norm over the result's:
    # below 8 for these unit-variance inputs
    tol = 8 * (4 * rc.HALF_STEP[dtype] + H * E * 2.0 ** -24)
    for got, ref in zip((out,) + grads, (out64,) + grads64):
        assert (got.double() - ref).norm() <= tol * ref.norm()


def test_ids_past_32_bits_are_skipped(R):
    idx = torch.tensor([[1, 1 << 32], [(1 << 32) + 2, 2], [-(1 << 40), 0]], device=DEV)
    p = R.plan(idx, 4)
    assert p.pos_of.tolist() == [[1, -1], [-1, 2], [-1, 0]] and p.counts.tolist() == [1, 1, 1, 0]
    assert clear_status() == 6


def test_more_than_2_31_elements(R):
    """Rows whose place times their length passes 32 bits."""
    N, k, H = 140_000, 8, 2048
    assert N * k * H > 1 << 31
    idx = (torch.arange(N, device=DEV)[:, None] + torch.arange(k, device=DEV) * 7) % 64
    p = R.plan(idx.int(), 64)
    h = torch.randn(N, H, device=DEV, dtype=BF)
    x = R.permute_rows(h, p)
    t = torch.tensor([0, 1, 12_345, N - 2, N - 1], device=DEV)
    assert torch.equal(x[p.pos_of[t].long()], h[t][:, None].expand(-1, k, -1))
    last = p.token[-3:].long()
    assert torch.equal(x[-3:], h[last])
    out = R.unpermute_rows(x, None, p)
    assert torch.equal(out, 8 * h)  # eight equal rows: exact
    dy, dw = R._ext().unpermute_rows_grad(h, x, torch.full((N, k), 0.5, device=DEV), p.pos_of, p.offsets)
    assert torch.equal(dy[p.pos_of[t].long()], (0.5 * h[t])[:, None].expand(-1, k, -1)) and torch.equal(dy[-3:], 0.5 * h[last])
    sq = (h[t].double() ** 2).sum(1)
    assert ((dw[t].double() - sq[:, None]).abs() <= 2 * H * 2.0 ** -24 * sq[:, None]).all()


def test_a_captured_training_step(R):
    """Forward and both gradients in one graph, replayed on new values, give the eager step's bits."""
    N, k, E, H = 50, 4, 16, 128
    idx, pos, p = setup(R, N, k, E, 0, seed=13)
    h, w, dout = torch.randn(N, H, device=DEV).to(BF), torch.rand(N, k, device=DEV), torch.randn(N, H, device=DEV).to(BF)
    def step():
        a, b = h.detach().requires_grad_(), w.detach().requires_grad_()
        out = R.unpermute_rows(R.permute_rows(a, p) * 2, b, p)
        return [out.detach()] + list(torch.autograd.grad(out, (a, b), dout))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for s in range(2):
        for t in (h, w, dout):
            t.copy_(torch.randn(t.shape, device=DEV).to(t.dtype))
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals(R):
    p = R.plan(torch.zeros(4, 2, dtype=torch.int32, device=DEV), 8)
    h = torch.zeros(4, 64, device=DEV)
    y = torch.zeros(8, 64, device=DEV)
    w = torch.zeros(4, 2, device=DEV)
    for bad in (torch.zeros(4, 2, device=DEV), torch.zeros(4, 2, dtype=torch.bool, device=DEV), torch.zeros(4, 2, dtype=torch.uint8, device=DEV)):
        with pytest.raises(RuntimeError, match="int32 or int64"):
            R.plan(bad, 8)
    for bad in (h.cpu(), h[:3], h.double(), h.int(), h[0], torch.zeros(4, 6, device=DEV)):
        with pytest.raises(RuntimeError):
            R.permute_rows(bad, p)
    for by, bw in ((y.cpu(), w), (y[:7], w), (y, w[:3]), (y, w.half()), (y.half(), w.bfloat16()), (y, w.cpu()), (y.double(), w)):
        with pytest.raises(RuntimeError):
            R.unpermute_rows(by, bw, p)
    with pytest.raises(RuntimeError):
        R.plan(torch.zeros(4, device=DEV, dtype=torch.int32), 8)
    with pytest.raises(RuntimeError, match="256|experts"):
        R.plan(torch.zeros(4, 2, device=DEV, dtype=torch.int32), 257)
    with pytest.raises(RuntimeError, match="top_k"):
        R.permute_rows(h, p._replace(pos_of=torch.zeros(4, 9, dtype=torch.int32, device=DEV)))
    with pytest.raises(RuntimeError, match="aligned"):
        R.permute_rows(torch.zeros(4 * 64 + 1, device=DEV)[1:].view(4, 64), p)
    hr = h.clone().requires_grad_()
    dh, = torch.autograd.grad(R.permute_rows(hr, p).sum(), hr, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(dh.sum(), hr)  # no second derivative
