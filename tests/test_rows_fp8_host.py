"""What the row operators, the quantisers and the 8-bit product refuse before anything touches a
device (C ABI and Python), and the plain forms the GPU tests compare with."""

import ctypes

import pytest
import torch

import rows_fp8_cases as rc


@pytest.fixture(scope="module")
def lib():
    from switchyard_b200 import _lib, build
    build.build()
    return _lib.load()


P = ctypes.c_void_p(1 << 20)  # an aligned address that a refused call must not look at


def refused(lib, rc_, text):
    assert rc_ == -1 and text in lib.sy_last_error(), (rc_, lib.sy_last_error())


def test_row_operators_refuse(lib):
    refused(lib, lib.sy_permute_rows(P, P, P, 4, 9, 8, 64, 1, P, None), b"top_k")
    refused(lib, lib.sy_permute_rows(P, P, P, 4, 0, 8, 64, 1, P, None), b"top_k")
    refused(lib, lib.sy_permute_rows(P, P, P, 4, 2, 8, 60, 1, P, None), b"multiple of 8")
    refused(lib, lib.sy_permute_rows(P, P, P, 4, 2, 8, 6, 2, P, None), b"multiple of 4")
    refused(lib, lib.sy_permute_rows(P, P, P, 4, 2, 8, 64, 3, P, None), b"dtype")
    refused(lib, lib.sy_permute_rows(P, P, P, -1, 2, 8, 64, 1, P, None), b"top_k")
    refused(lib, lib.sy_permute_rows(P, P, P, 1 << 30, 8, 8, 64, 1, P, None), b"2^31")
    refused(lib, lib.sy_permute_rows(P, P, P, 4, 2, 0, 64, 1, P, None), b"expert")
    refused(lib, lib.sy_permute_rows(None, P, P, 4, 2, 8, 64, 1, P, None), b"null")
    refused(lib, lib.sy_permute_rows(ctypes.c_void_p(8), P, P, 4, 2, 8, 64, 1, P, None), b"aligned")
    refused(lib, lib.sy_unpermute_rows(P, P, 0, P, 4, 2, 64, 1, P, None), b"weights")
    refused(lib, lib.sy_unpermute_rows(P, P, 1, P, 4, 2, 64, 2, P, None), b"weights")
    refused(lib, lib.sy_unpermute_rows(P, None, 0, None, 4, 2, 64, 1, P, None), b"null")
    refused(lib, lib.sy_unpermute_rows_grad(P, P, P, 0, P, P, 4, 2, 8, 64, 1, P, P, None), b"weights")
    refused(lib, lib.sy_unpermute_rows_grad(P, None, P, 1, P, P, 4, 2, 8, 64, 1, P, P, None), b"null")
    # the largest sizes: a block's last token and a row's last column are 32-bit numbers
    most = 0x7fffffff
    refused(lib, lib.sy_permute_rows(P, P, P, most, 1, 8, 64, 1, P, None), b"2^31")
    refused(lib, lib.sy_unpermute_rows(P, None, 1, P, most - 100, 1, 64, 1, P, None), b"2^31")
    refused(lib, lib.sy_unpermute_rows_grad(P, P, P, 1, P, P, 1, 1, 8, most - 7, 1, P, P, None), b"at most")
    # nothing to do: no pointer is needed
    assert lib.sy_permute_rows(None, None, None, 0, 2, 8, 64, 1, None, None) == 0
    assert lib.sy_unpermute_rows(None, None, 0, None, 0, 2, 64, 1, None, None) == 0
    assert lib.sy_unpermute_rows_grad(None, None, None, 0, None, None, 4, 2, 8, 64, 1, None, None, None) == 0


def test_quantisers_and_the_product_refuse(lib):
    refused(lib, lib.sy_quantize_rows(P, None, None, 4, 2, 0, 64, 1, P, P, None), b"one place")
    refused(lib, lib.sy_quantize_rows(P, P, P, 4, 2, 8, 40, 1, P, P, None), b"multiple of 16")
    refused(lib, lib.sy_quantize_rows(P, P, P, 4, 9, 8, 64, 1, P, P, None), b"top_k")
    refused(lib, lib.sy_quantize_rows(P, P, None, 4, 2, 8, 64, 1, P, P, None), b"null")
    refused(lib, lib.sy_quantize_rows(P, P, P, 4, 2, 8, 64, 7, P, P, None), b"dtype")
    refused(lib, lib.sy_quantize_weight(P, 1, 0, 64, 1, P, P, None), b"rows")
    refused(lib, lib.sy_quantize_weight(P, 1 << 20, 8, 64, 1, P, P, None), b"matrices")
    refused(lib, lib.sy_quantize_weight(P, 1, 8, 40, 1, P, P, None), b"multiple of 16")
    args = lambda E=8, rows=4, n=64, k=128, sw=0, scale=None, dt=1, tile=0, x=P, cs=None: (x, P, P, P, P, E, rows, n, k, sw, scale, P,
                                                                                        cs, dt, tile, None)
    refused(lib, lib.sy_grouped_gemm_fp8(*args(E=257)), b"experts")
    refused(lib, lib.sy_grouped_gemm_fp8(*args(k=120)), b"multiple of 16")
    refused(lib, lib.sy_grouped_gemm_fp8(*args(n=60)), b"multiple of 8")
    refused(lib, lib.sy_grouped_gemm_fp8(*args(sw=1, scale=P)), b"separate")
    refused(lib, lib.sy_grouped_gemm_fp8(*args(dt=2)), b"dtype")
    refused(lib, lib.sy_grouped_gemm_fp8(*args(tile=4)), b"tile")
    refused(lib, lib.sy_grouped_gemm_fp8(*args(cs=P)), b"SwiGLU")
    refused(lib, lib.sy_grouped_gemm_fp8(*args(cs=P, sw=1, n=72)), b"multiple of 16")
    refused(lib, lib.sy_grouped_gemm_fp8(*args(x=None)), b"null")
    refused(lib, lib.sy_grouped_gemm_fp8(*args(x=ctypes.c_void_p(8))), b"aligned")
    most = 0x7ffffff0  # the largest multiple of 16
    refused(lib, lib.sy_quantize_rows(P, None, None, most, 1, 0, 64, 1, P, P, None), b"2^31")
    refused(lib, lib.sy_quantize_rows(P, None, None, 1, 1, 0, most, 1, P, P, None), b"at most")
    refused(lib, lib.sy_quantize_weight(P, 1, 8, most, 1, P, P, None), b"at most")
    refused(lib, lib.sy_grouped_gemm_fp8(*args(rows=most)), b"rows")
    refused(lib, lib.sy_grouped_gemm_fp8(*args(k=most)), b"at most")
    assert lib.sy_grouped_gemm_fp8(*args(rows=0, x=None)) == 0
    refused(lib, lib.sy_sort_by_expert(P, P, 8, 2, 8, 0, P, P, P, None, P, None, 0, None), b"null")


def test_sizes_past_32_bits_reach_the_library_as_the_largest(lib):
    from switchyard_b200 import kernels
    assert [kernels._size(v) for v in (0, 7, 0x7fffffff, 1 << 31, (1 << 32) + 16)] == [0, 7] + [0x7fffffff] * 3
    most = kernels._size(1 << 32)
    refused(lib, lib.sy_quantize_rows(P, None, None, most, 1, 0, 64, 1, P, P, None), b"2^31")
    refused(lib, lib.sy_quantize_rows(P, None, None, 1, 1, 0, most, 1, P, P, None), b"at most")
    refused(lib, lib.sy_quantize_weight(P, most, 8, 64, 1, P, P, None), b"matrices")
    refused(lib, lib.sy_quantize_weight(P, 1, most, 64, 1, P, P, None), b"rows")
    refused(lib, lib.sy_quantize_weight(P, 1, 8, most, 1, P, P, None), b"at most")
    for sizes in ((most, 4, 64, 128), (8, most, 64, 128), (8, 4, most, 128), (8, 4, 64, most)):
        assert lib.sy_grouped_gemm_fp8(P, P, P, P, P, *sizes, 0, None, P, None, 1, 0, None) == -1


def test_the_sort_refuses_more_choices_than_it_can_count(lib):
    """Just below 2^31 a block's end would pass 32 bits and an index come out negative."""
    for m in (0x7fffffff, 0x7fff0000, 0x7ffe0001):
        refused(lib, lib.sy_sort_by_expert(P, None, m, 1, 64, 0, P, P, P, None, P, P, 1 << 30, None), b"2^31")
        assert lib.sy_sort_scratch_bytes(m, 64) == 0
    assert lib.sy_sort_scratch_bytes(0x7ffe0000, 64) == 128 * 64 * 4


def test_tensors_on_the_host_are_refused(lib):
    """There is no CPU path: every public call says so instead of computing something else."""
    from switchyard_b200 import fp8, rows
    idx = torch.zeros(4, 2, dtype=torch.int32)
    plan = rows.SortPlan(torch.zeros(8, dtype=torch.int32), torch.zeros(9, dtype=torch.int32), torch.zeros(8, dtype=torch.int32), idx)
    x, w = torch.zeros(4, 64), torch.zeros(4, 2)
    w8 = fp8.Weight8(torch.zeros(2, 64, 64).to(torch.float8_e4m3fn), torch.zeros(2, 1, 1))
    x8 = fp8.Rows8(torch.zeros(4, 64).to(torch.float8_e4m3fn), torch.zeros(1, 4))
    for call in (lambda: rows.plan(idx, 8), lambda: rows.permute_rows(x, plan), lambda: rows.unpermute_rows(torch.zeros(8, 64), w, plan),
                 lambda: fp8.quantize_rows(x), lambda: fp8.quantize_rows(x, plan), lambda: fp8.quantize_weight(torch.zeros(2, 64, 64)),
                 lambda: fp8.grouped_gemm(x8, w8, torch.zeros(3, dtype=torch.int32)),
                 lambda: rows.permute_rows(x.requires_grad_(), plan)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_8_bit_calls_refuse_inputs_that_require_a_gradient(lib):
    from switchyard_b200 import fp8
    t = lambda *shape, grad=False: torch.zeros(*shape, requires_grad=grad)
    x, w = fp8.Rows8(t(4, 128), t(1, 4)), fp8.Weight8(t(1, 8, 128), t(1, 1, 1))
    offsets = torch.zeros(2, dtype=torch.int32)
    for changed in (dict(x=x._replace(scale=t(1, 4, grad=True))), dict(w=w._replace(scale=t(1, 1, 1, grad=True))),
                    dict(scale=t(4, grad=True))):
        args = {**dict(x=x, w=w, offsets=offsets), **changed}
        with pytest.raises(RuntimeError, match="no gradient"):
            fp8.grouped_gemm(**args)
        with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA"):  # without recording: the next check
            fp8.grouped_gemm(**args)
    for call in (fp8.quantize_rows, fp8.quantize_weight):
        with pytest.raises(RuntimeError, match="no gradient"):
            call(t(4, 32, grad=True))


def test_forward_mode_tangents_are_refused(lib):
    """A dual tensor asks for no gradient: a call that looked at that alone would drop its tangent."""
    from torch.autograd import forward_ad as fwd

    from switchyard_b200 import fp8, rows
    pos = torch.zeros(4, 2, dtype=torch.int32)
    plan = rows.SortPlan(torch.zeros(8, dtype=torch.int32), torch.zeros(9, dtype=torch.int32), torch.zeros(8, dtype=torch.int32), pos)
    h, y, w = torch.zeros(4, 128), torch.zeros(8, 128), torch.zeros(4, 2)
    x8, w8 = fp8.Rows8(h.to(torch.float8_e4m3fn), torch.zeros(1, 4)), fp8.Weight8(torch.zeros(1, 8, 128).to(torch.float8_e4m3fn), torch.zeros(1, 1, 1))
    offsets = torch.zeros(2, dtype=torch.int32)
    with fwd.dual_level():
        dual = lambda t: fwd.make_dual(t, torch.ones_like(t))
        calls = (lambda: rows.permute_rows(dual(h), plan), lambda: rows.permute_rows(dual(h)[:, ::2], plan),
                 lambda: rows.unpermute_rows(dual(y), w, plan), lambda: rows.unpermute_rows(y, dual(w), plan),
                 lambda: rows.unpermute_rows(dual(y), None, plan), lambda: fp8.quantize_rows(dual(h)),
                 lambda: fp8.quantize_weight(dual(torch.zeros(1, 8, 128))),
                 lambda: fp8.grouped_gemm(x8._replace(scale=dual(x8.scale)), w8, offsets),
                 lambda: fp8.grouped_gemm(x8, w8, offsets, scale=dual(torch.zeros(4))))
        for call in calls:
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                call()
        with pytest.raises(RuntimeError, match="CUDA"):  # no tangent: the next check
            rows.permute_rows(h, plan)


def test_the_plain_quantiser_is_torchs_e4m3(lib):
    """nearest8 against torch's own conversion on every 16-bit value it can take, ties included."""
    v = torch.arange(-(1 << 15), 1 << 15, dtype=torch.int32).to(torch.int16).view(torch.float16).float()
    v = v[v.abs() <= 448]
    assert torch.equal(rc.nearest8(v), v.to(torch.float8_e4m3fn).double())
    q, s = rc.quantize64(torch.zeros(3, 130), 1)
    assert (q == 0).all() and torch.equal(s, torch.full((3, 2), rc.TINY) / torch.tensor(448.0))


def test_the_plain_plan_is_the_sort(lib):
    from oracle import moe_oracle as mo
    idx = rc.choices(50, 4, 16, 1)
    offsets, pos = rc.places(idx, 16)
    want = mo.sort_by_expert(idx, torch.zeros(50, 4).half(), 16)
    assert torch.equal(offsets.int(), want[1]) and torch.equal(pos.flatten().int(), want[4])


def test_dequantize_is_the_layout(lib):
    from switchyard_b200 import fp8
    g = torch.Generator().manual_seed(0)
    x = torch.randn(5, 144, generator=g)
    q, s = rc.quantize64(x, 1)
    r8 = fp8.Rows8(q.float().to(torch.float8_e4m3fn), s.t().contiguous())
    assert ((r8.dequantize() - x).abs() <= x.abs() * (2.0 ** -4 + 2.0 ** -22) + 2.0 ** -10 * 6 / 448).all()
    w = torch.randn(2, 272, 144, generator=g)
    parts = [rc.quantize64(p, 128) for p in w.view(4, 136, 144)]
    w8 = fp8.Weight8(torch.stack([a for a, _ in parts]).view(2, 272, 144).float().to(torch.float8_e4m3fn),
                     torch.stack([b for _, b in parts]).view(2, 4, 2))
    assert ((w8.dequantize(halves=2) - w).abs() <= w.abs() * (2.0 ** -4 + 2.0 ** -22) + 2.0 ** -10 * 6 / 448).all()


def test_a_weight_knows_how_its_blocks_are_counted(lib):
    """400 rows are four blocks of rows either way: 128, 128, 128, 16, or 128, 72 in each half. The layout that
    was not asked for has to be refused, not read with the wrong scales."""
    import copy

    from switchyard_b200 import fp8
    g = torch.Generator().manual_seed(2)
    w = torch.randn(1, 400, 128, generator=g)
    q, s = zip(*[rc.quantize64(p, 128) for p in w.view(2, 200, 128)])
    w8 = fp8.Weight8(torch.cat(q).view(1, 400, 128).float().to(torch.float8_e4m3fn), torch.cat(s).view(1, 4, 1), halves=2)
    q, scale = w8
    assert len(w8) == 2 and q is w8.q and scale is w8.scale
    near = lambda v: ((v - w).abs() <= w.abs() * (2.0 ** -4 + 2.0 ** -22) + 2.0 ** -10 * 6 / 448).all()
    for kept in (w8, copy.deepcopy(w8), w8._replace(q=w8.q.clone())):
        assert kept.halves == 2 and near(kept.dequantize()) and near(kept.dequantize(halves=2))
        with pytest.raises(RuntimeError, match="halves"):
            kept.dequantize(halves=1)
    bare = fp8.Weight8(w8.q, w8.scale)
    assert bare.halves is None and near(bare.dequantize(halves=2))
    x8, offsets = fp8.Rows8(torch.zeros(4, 128).to(torch.float8_e4m3fn), torch.zeros(1, 4)), torch.zeros(2, dtype=torch.int32)
    plain = fp8.Weight8(w8.q, w8.scale, halves=1)
    with pytest.raises(RuntimeError, match="halves"):
        fp8.grouped_gemm(x8, plain, offsets, swiglu=True)
    with pytest.raises(RuntimeError, match="halves"):
        fp8.grouped_gemm(x8, w8, offsets)
    for weight, swiglu in ((w8, True), (plain, False), (bare, True), (bare, False)):
        with pytest.raises(RuntimeError, match="CUDA"):  # the next check
            fp8.grouped_gemm(x8, weight, offsets, swiglu=swiglu)
    # halves that are multiples of 128: one layout
    even = fp8.Weight8(torch.zeros(1, 256, 128).to(torch.float8_e4m3fn), torch.zeros(1, 2, 1), halves=1)
    even.dequantize(halves=2)
    with pytest.raises(RuntimeError, match="CUDA"):
        fp8.grouped_gemm(x8, even, offsets, swiglu=True)
    with pytest.raises(RuntimeError, match="blocks of rows"):  # three blocks where two halves of 136 have four
        fp8.Weight8(torch.zeros(1, 272, 128).to(torch.float8_e4m3fn), torch.zeros(1, 3, 1)).dequantize(halves=2)


def test_expert_parallelism_refuses_8_bit_experts(lib):
    from switchyard_b200 import fp8
    from switchyard_b200.ep import ExpertParallel
    w8 = fp8.Weight8(torch.zeros(2, 64, 64).to(torch.float8_e4m3fn), torch.zeros(2, 1, 1))
    ep = ExpertParallel(["cpu", "cpu"], 4, 2, False, ops=object())
    with pytest.raises(RuntimeError, match="one GPU"):
        ep.layer([torch.zeros(1, 64)] * 2, [torch.zeros(4, 64)] * 2, [w8, w8], [w8, w8])
    with pytest.raises(RuntimeError, match="one GPU"):
        ep.layer_rank(None, 0, torch.zeros(1, 64), torch.zeros(4, 64), w8, torch.zeros(2, 64, 32))
