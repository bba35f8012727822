// The experts' product in 8-bit floats: every expert's slice of the sorted rows times its weights,
// both e4m3 with float32 scales for blocks of 128 along k (1 x 128 for rows, 128 x 128 for weights):
//
//   acc[r, n] = sum_b sx[b, r] * sw[e, n / 128, b] * sum_{k in block b} x[r, k] * w[e, n, k]
//   C[r, n]   = round(acc[r, n] * scale[r])   or, with SwiGLU, round(silu(acc[r, gate n]) * acc[r, up n])
//
// or that SwiGLU result as e4m3 with scales for 128 columns, which is what the down projection reads.
//
// Float32 scales cannot ride in the tensor core, so the inner sums of each block of 128 (four
// tcgen05.mma of k = 32) go to tensor memory on their own, and eight warps multiply them by the two
// scales and add them up in float32 registers (the promotion) while the next block is being
// multiplied: tensor memory holds two such partial products of 256 columns, or four smaller ones.
//
// Warps: 0 TMA producer, 1-2 MMA issuers, 3 scales, 4-11 promotion and epilogue.
// Tiles as in gemm.cu: numbered on the device from `offsets`, expert-major, dealt round-robin to
// a persistent grid. Weight rows come in two halves (a TMA box each): consecutive rows, or with SwiGLU
// the gate rows and the up rows of the same columns.
//   Wide tile and pair: token rows are the MMA's M operand (128, or 256 over a pair of CTAs), weight rows its
//   N. A thread owns a token row and the same quarter of the columns out of either half, so that it finds a
//   gate value and its up value in its own registers; both scales are the same for all its columns of one
//   weight block, so a value costs half a packed multiply-add.
//   Few token rows: weight rows are the M (128), 32 token rows the N. A thread owns a weight row and 16
//   token rows: an eighth of the promotion, 4 KB of token rows to fetch and read instead of 16, and results
//   that go straight to memory, 32 columns of a row at a time. SwiGLU's up sums cross to the gates' warps
//   through shared memory. 8-bit results take 256 weight rows, so that a tile has its 128 columns' maximum.
//   (Token rows as M took 35.5 us for 8 tokens and 49.2 for 64, gate and up; this takes 31.3 and 43.5.)
//
// What bounds it. Few rows per expert: the weights' way from HBM (64 tokens, 268 MB of gate and up: 44 us,
// 6.1 TB/s), 3 us before the first ones arrive, and a last round of tiles, 3 to 4 us however few they are.
// Many rows: a block of 256 columns over two CTAs takes 0.43 us where the MMAs alone take 0.27, with shared
// memory busy for two thirds of it (by its bytes: 64 KB at 128 a clock), and the epilogues are a quarter
// of a launch of 16 blocks a tile; and, run for seconds, the GPU's power: 8192 tokens take 303 us in a
// burst of 2 ms, 344-361 us (from card to card) at 1.4 GHz and 990 W, of which the promotion's multiply-adds
// were 67 us. (The library's 8-bit product of the same size, one scale per matrix, no experts, no SwiGLU,
// takes 246 us at the same power.)
#include <cuda.h>
#include <cuda_fp8.h>

#include <atomic>
#include <string.h>
#include <type_traits>

#include "common.cuh"
#include "tensor_map.cuh"

namespace sy {

constexpr int G8_BLOCK = 128;                    // k per scale and per stage: one 128-byte swizzle atom
constexpr int G8_XR = 128;                       // token rows a CTA stages
constexpr int G8_XFEW = 32;                      // token rows of the small TMA box, for tiles with fewer rows
constexpr int G8_MAX_E = 256;
constexpr int G8_AHEAD = 7;                      // k blocks whose scales are on their way
constexpr int G8_SLOTS = 16;                     // k blocks whose scales are in shared memory or on their way
constexpr int G8_OUT_PITCH = 64 + 16;             // bytes per staged row of results: 32 columns, off the banks of the next
constexpr int G8_SLOT = G8_XR + 8;               // floats: the rows' scales, then the weights' two
constexpr int G8_HELPERS = 4;                    // warps before the promoters: TMA, two for MMA, scales
constexpr int G8_MOST = 0x7fff0000;              // rows and k: a tile's or a block's end is still a 32-bit number
constexpr float G8_LOG2E = 1.4426950408889634f, G8_MOST_EXP = 62.f;  // SwiGLU: exp(-g) is kept below 2^62
constexpr int G8_RING_BYTES = 192 * 1024;
constexpr int G8_SMEM = G8_RING_BYTES + 1024;    // room to align the ring to 1024

// The tiles. WIDE: 128 token rows (the MMA's M) by 256 weight rows (its N). PAIR: 256 by 256 over two CTAs. FEW:
// 128 weight rows as the MMA's M (with 8-bit results 256, as two MMAs: their columns are a block), by 32
// token rows as its N.
enum { G8_FEW = 1, G8_WIDE = 2, G8_PAIR = 3 };
template <int TILE, bool OUT8> struct Shape8 {
  static constexpr bool FEW = TILE == G8_FEW, PAIR = TILE == G8_PAIR;
  static constexpr int CTAS = PAIR ? 2 : 1;
  static constexpr int XR = FEW ? G8_XFEW : G8_XR;        // token rows a CTA stages
  static constexpr int BM = XR * CTAS;                    // token rows per tile
  static constexpr int WR = FEW && !OUT8 ? 128 : 256;     // weight rows per tile
  static constexpr int WRC = WR / CTAS;                   // weight rows a CTA stages
  static constexpr int WBOX = WR / 2;                     // weight rows per TMA box: a half of the tile
  static constexpr int W_BOXES = WRC / WBOX;              // PAIR: each CTA has one of the halves
  static constexpr int X_BYTES = XR * G8_BLOCK;
  static constexpr int STAGE_BYTES = X_BYTES + WRC * G8_BLOCK;
  // Even, and so is BUFS: a stage and a partial product are always the same MMA warp's. With an odd number
  // the two warps would take a stage's uses in turn, and the one that is ahead would find the phase it
  // waits for in the one before it, whose parity is the other's: a use of data not yet there.
  static constexpr int STAGES = G8_RING_BYTES / STAGE_BYTES / 2 * 2;
  static constexpr int MMAS = FEW ? WR / 128 : 1;         // per 32 k
  static constexpr int PART = FEW ? MMAS * XR : WR;       // columns of tensor memory of a partial product
  static constexpr int BUFS = FEW ? 4 : 2;                // partial products
  static_assert(STAGES % 2 == 0 && BUFS % 2 == 0, "two MMA warps");
  static constexpr int TMEM_COLS = BUFS * PART;
  static constexpr int PROMOTERS = 8;                     // warps
  static constexpr int THREADS = (G8_HELPERS + PROMOTERS) * 32;
  static constexpr int COLS = WR / 4;                     // columns a promoter thread has of either half (FEW: one)
  static constexpr int TOKENS = XR / 2;                   // FEW: token rows a promoter thread has
  // 128 accumulators: the helpers hand some of their registers to the promoters (88 / 208: 1-3 % slower)
  static constexpr bool SPLIT_REGS = !FEW;
};
constexpr int G8_REGS_LAUNCH = 168, G8_REGS_FEW = 72, G8_REGS_MANY = 216;
static_assert(G8_HELPERS * G8_REGS_FEW + 8 * G8_REGS_MANY <= (G8_HELPERS + 8) * G8_REGS_LAUNCH, "register split");

struct Gemm8Args {
  CUtensorMap wmap;   // [experts * halves * Nout, K] e4m3, box 128 k x WBOX
  CUtensorMap xmap;   // [rows, K] e4m3, box 128 k x 128 (not of the few-row tile)
  CUtensorMap xfew;   // the same, box 128 k x 32
  const float* xscale;  // [k blocks][rows]
  const float* wscale;  // [experts][halves * n blocks][k blocks]
  const int* offsets;   // [experts + 1]
  const void* scale;    // [rows] or null
  void* C;              // [rows, Nout]
  float* cscale;        // 8-bit results: [Nout blocks][rows]
  int experts, rows, Nout, K;
  int* status;
  unsigned long long wait_ns;
};

__device__ __forceinline__ void umma_f8(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t hi, uint32_t idesc,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "mov.b64 da, {%1, %3};\n\t"
      "mov.b64 db, {%2, %3};\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], da, db, %4, p;\n\t}" ::"r"(d),
      "r"(a_lo), "r"(b_lo), "r"(hi), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void umma_f8_pair(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t hi, uint32_t idesc,
                                             uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "mov.b64 da, {%1, %3};\n\t"
      "mov.b64 db, {%2, %3};\n\t"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], da, db, %4, p;\n\t}" ::"r"(d),
      "r"(a_lo), "r"(b_lo), "r"(hi), "r"(idesc), "r"(accumulate)
      : "memory");
}
// 32 lanes x 32 consecutive columns of tensor memory, and the wait for them in the same statement: the
// registers are not to be touched before it. (Two loads of 16: 32 registers in a row would have to be
// found otherwise.)
__device__ __forceinline__ void tmem_get_32(uint32_t addr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%32];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32 + 16];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_get_16(uint32_t addr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr)
      : "memory");
}
// 16 columns from either address.
__device__ __forceinline__ void tmem_get_16_16(uint32_t a, uint32_t b, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%32];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%33];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(a), "r"(b)
      : "memory");
}
__device__ __forceinline__ void cp_async_4(float* dst_smem, const float* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(dst_smem)), "l"(src) : "memory");
}
// acc += part * f for two float32 values at once. The accumulators are 64-bit values throughout, so
// that they stay in aligned register pairs.
__device__ __forceinline__ void fma2(uint64_t& acc, uint32_t lo, uint32_t hi, uint64_t ff) {
  asm("{\n\t.reg .b64 p;\n\t"
      "mov.b64 p, {%1, %2};\n\t"
      "fma.rn.f32x2 %0, p, %3, %0;\n\t}"
      : "+l"(acc)
      : "r"(lo), "r"(hi), "l"(ff));
}
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Two float32 values rounded to T, the first in the low half.
template <typename T> __device__ __forceinline__ uint32_t pack16(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack16<__half>(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return reinterpret_cast<const uint32_t&>(v);
}
template <> __device__ __forceinline__ uint32_t pack16<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return reinterpret_cast<const uint32_t&>(v);
}
__device__ __forceinline__ uint64_t pair64(float2 v) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(v.x), "f"(v.y));
  return r;
}
__device__ __forceinline__ float2 both(uint64_t v) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
  return f;
}
__device__ __forceinline__ uint64_t twice(float f) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %1};" : "=l"(r) : "f"(f));
  return r;
}

// Arrives on a barrier of the pair's leader. What it publishes is that tensor-memory reads are done,
// which tcgen05.wait::ld and the tcgen05 fence before it have settled; so it releases at CTA scope
// only. A release at cluster scope also waits for the thread's loads in flight (the next blocks'
// scales), which cost about 600 clocks per k block: 682 -> 425 us for 8192 tokens of the
// benchmark's layer.
__device__ __forceinline__ void arrive_leader(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}

__device__ __forceinline__ float max_nan(float a, float b) {  // NaN where either is
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
struct Tile8 {
  int e, cb, row0, nvalid;
};

// Tile t of the launch, found by a whole warp. `cursor` walks the experts; start[E] is the tiles' number.
template <int BM>
__device__ __forceinline__ Tile8 locate_tile8(int t, int& cursor, int E, const int* start, const int* begin, const int* end) {
  const int lane = threadIdx.x & 31;
  for (;;) {  // experts that end at or before t, 32 at a time
    const int e = cursor + 1 + lane;
    const unsigned past = __ballot_sync(0xffffffffu, e <= E && start[e] <= t);
    cursor += __popc(past);
    if (past != 0xffffffffu) break;
  }
  const int local = t - start[cursor], n = end[cursor] - begin[cursor], row_tiles = (n + BM - 1) / BM;
  // local / row_tiles: below 2^20 the float quotient of local + 1/2 cannot reach the next integer
  const int cb = local < (1 << 20) ? (int)(((float)local + 0.5f) * rcp_approx((float)row_tiles)) : local / row_tiles;
  Tile8 tile;
  tile.e = cursor;
  tile.cb = cb;
  tile.row0 = begin[cursor] + (local - cb * row_tiles) * BM;
  tile.nvalid = min(BM, end[cursor] - tile.row0);
  return tile;
}

// The exponent (to base 2) of what is left of exp(g) once 2^-62 is taken out, for gates below -43. Two
// roundings, written out: as one multiply-add the exponent is off by another 2^-18, and a row would
// have other bits in the tile whose form the compiler happens to contract.
__device__ __forceinline__ float swiglu_rest(float g) { return __fsub_rn(G8_MOST_EXP, __fmul_rn(g, -G8_LOG2E)); }

// up <- silu(gate) * up for N pairs of columns. The reciprocals of a pair's 1 + exp(-g) come from the one
// of their product (the special-function unit is what an epilogue waits for). exp and the
// reciprocal are the approximate ones, exp within 2^-22 and the rounding of its argument (2^-18 at
// g = -40): far inside the 16-bit rounding that follows. exp(-g) is kept below 2^62 so that the
// product stays finite. Where a gate is below that, at -43, the rest of exp(g) is a factor of its own:
// a thread asks for it once for all its columns (a branch per pair took 2-4 % of a launch). The bits are
// the same with PACKED products or single ones: 16-bit results are 1-2 % faster with the packed (65,536
// rows 257 -> 253 us), 8-bit results with the single ones (257, packed 260).
template <bool PACKED, int N> __device__ __forceinline__ void swiglu_pairs(const uint64_t (&gate)[N], uint64_t (&up)[N]) {
  constexpr float LOG2E = G8_LOG2E, MOST = G8_MOST_EXP;
  float most = 0.f;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const float2 g = both(gate[j]), u = both(up[j]);
    const float2 x = PACKED ? both(mul2(gate[j], twice(-LOG2E))) : make_float2(__fmul_rn(g.x, -LOG2E), __fmul_rn(g.y, -LOG2E));
    const float x0 = x.x, x1 = x.y;
    const float d0 = 1.f + exp2_approx(fminf(x0, MOST)), d1 = 1.f + exp2_approx(fminf(x1, MOST));
    const float r = rcp_approx(d0 * d1);
    if (PACKED) up[j] = mul2(mul2(gate[j], mul2(pair64(make_float2(d1, d0)), twice(r))), up[j]);
    else up[j] = pair64(make_float2(g.x * (r * d1) * u.x, g.y * (r * d0) * u.y));
    most = fmaxf(most, fmaxf(x0, x1));
  }
  if (__builtin_expect(most > MOST, 0)) {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const float2 g = both(gate[j]), v = both(up[j]);
      up[j] = pair64(make_float2(v.x * exp2_approx(fminf(swiglu_rest(g.x), 0.f)), v.y * exp2_approx(fminf(swiglu_rest(g.y), 0.f))));
    }
  }
}

// The same for one column per lane, the pair's other one the neighbouring lane's: the same bits.
__device__ __forceinline__ float swiglu_lane(float g, float u) {
  const float x = __fmul_rn(g, -G8_LOG2E), d = 1.f + exp2_approx(fminf(x, G8_MOST_EXP)), pair = __shfl_xor_sync(0xffffffffu, d, 1);
  const float v = g * (rcp_approx(d * pair) * pair) * u;
  return x > G8_MOST_EXP ? v * exp2_approx(swiglu_rest(g)) : v;
}

template <typename T, int TILE, bool SWIGLU>
__global__ void __launch_bounds__(Shape8<TILE, std::is_same<T, __nv_fp8_e4m3>::value>::THREADS, 1) gemm8_kernel(const __grid_constant__ Gemm8Args args) {
  using S = Shape8<TILE, std::is_same<T, __nv_fp8_e4m3>::value>;
  constexpr int WR = S::WR;
  constexpr bool PAIR = S::PAIR, FEW = S::FEW;
  constexpr bool OUT8 = std::is_same<T, __nv_fp8_e4m3>::value;
  static_assert(!OUT8 || SWIGLU, "a tile of SwiGLU columns is one block of 128");
  constexpr int STAGES = S::STAGES, BUFS = S::BUFS;
  extern __shared__ unsigned char smem_raw[];
  __shared__ __align__(8) uint64_t full_bar[STAGES];
  __shared__ __align__(8) uint64_t empty_bar[STAGES];
  __shared__ __align__(8) uint64_t part_full[BUFS];
  __shared__ __align__(8) uint64_t part_empty[BUFS];
  __shared__ uint32_t s_tmem;
  __shared__ int s_begin[G8_MAX_E], s_end[G8_MAX_E];
  __shared__ int s_tile_start[G8_MAX_E + 1];
  __shared__ __align__(16) float s_scale[G8_SLOTS][G8_SLOT];
  __shared__ float s_top[OUT8 ? 2 : 1][OUT8 ? 2 : 1][G8_XR];  // 8-bit results: largest magnitude of a row in the warp's columns
  __shared__ float s_up[FEW && SWIGLU && !OUT8 ? 4 : 1][S::TOKENS * (WR / 2)];  // sums of up rows on their way to the gates' warps
  __shared__ __align__(16) unsigned char s_out[FEW ? 1 : S::PROMOTERS][32 * G8_OUT_PITCH];

  // (uniform to the compiler, so that the roles are too)
  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  unsigned char* stages =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  int* status = args.status;
  const uint64_t wait_ns = args.wait_ns;
  const int E = args.experts, Nout = args.Nout;
  const int cr = PAIR ? (int)cluster_ctarank() : 0;
  const int unit = PAIR ? (int)blockIdx.x >> 1 : (int)blockIdx.x, units = PAIR ? (int)gridDim.x >> 1 : (int)gridDim.x;
  const int tile_cols = SWIGLU ? WR / 2 : WR;
  const int col_blocks = (Nout + tile_cols - 1) / tile_cols;
  const int k_blocks = (args.K + G8_BLOCK - 1) / G8_BLOCK;

  pdl_launch_dependents();
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int b = 0; b < BUFS; ++b) {
      mbar_init(&part_full[b], 2);                           // the MMAs, and this CTA's scales
      mbar_init(&part_empty[b], S::CTAS * S::PROMOTERS);  // PAIR: the leader's, for both CTAs
    }
    fence_barrier_init();
    prefetch_tensormap(&args.wmap);
    if (!FEW) prefetch_tensormap(&args.xmap);
    prefetch_tensormap(&args.xfew);
  }
  if (warp == 1) {
    if (PAIR) {
      tmem_alloc_pair(&s_tmem, S::TMEM_COLS);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(&s_tmem, S::TMEM_COLS);
      tmem_relinquish();
    }
  }
  pdl_wait();
  for (int e = threadIdx.x; e < E; e += S::THREADS) {
    // kept inside [0, rows] and ascending whatever the caller's offsets say
    const int b = min(max(args.offsets[e], 0), args.rows), n = min(args.offsets[e + 1], args.rows);
    s_begin[e] = b;
    s_end[e] = max(n, b);
  }
  __syncthreads();
  if (warp == 0) {  // exclusive prefix of tiles per expert
    int carry = 0;
    for (int base = 0; base < E; base += 32) {
      const int e = base + lane;
      const int tiles = e < E ? ((s_end[e] - s_begin[e] + S::BM - 1) / S::BM) * col_blocks : 0;
      int inc = tiles;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += y;
      }
      if (e < E) s_tile_start[e] = carry + inc - tiles;
      carry += __shfl_sync(0xffffffffu, inc, 31);
    }
    if (lane == 0) s_tile_start[E] = carry;
  }
  tc_fence_before_sync();
  __syncthreads();
  if (PAIR) cluster_sync_all();  // the other CTA's barriers exist before anything arrives on them
  tc_fence_after_sync();
  const uint32_t tmem = s_tmem;
  const int total_tiles = s_tile_start[E];

  if (warp < 4) {
    if (S::SPLIT_REGS) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(G8_REGS_FEW));
    if (warp == 0) {
      // -------------------------------------------------------------- TMA producer
      // Lane 0 waits for the slot and announces the stage's bytes; every box has its own lane.
      int it = 0, cursor = 0;
      bool alive = true;
      const uint64_t policy = l2_policy_evict_first();
      for (int t = unit; t < total_tiles && alive; t += units) {
        const Tile8 tile = locate_tile8<S::BM>(t, cursor, E, s_tile_start, s_begin, s_end);
        // Token rows: one box of 128 where the tile has that many, else boxes of 32 as far as there are rows.
        // What is multiplied in the others' place is never read.
        auto rows_of = [&](int c) { return min(max(tile.nvalid - c * S::XR, 0), S::XR); };
        auto boxes_of = [&](int n) { return (n + G8_XFEW - 1) / G8_XFEW; };  // of 32 rows
        const int mine = rows_of(cr), other = PAIR ? rows_of(cr ^ 1) : 0;
        const bool few = FEW || mine < G8_XR;
        const int x_boxes = few ? boxes_of(mine) : 1;
        const uint32_t bytes = WR * G8_BLOCK + (boxes_of(mine) + (PAIR ? boxes_of(other) : 0)) * (G8_XFEW * G8_BLOCK);  // of all CTAs
        const bool is_w = lane < S::W_BOXES, is_x = !is_w && lane - S::W_BOXES < x_boxes;
        const int b = is_w ? cr + lane : lane - S::W_BOXES;  // half of the weight rows, or box of token rows
        const int colbase = tile.cb * tile_cols;
        const int y = is_w ? (SWIGLU ? (tile.e * 2 + b) * Nout + colbase : tile.e * Nout + colbase + b * S::WBOX)
                           : tile.row0 + cr * S::XR + b * G8_XFEW;
        const int off = is_w ? S::X_BYTES + lane * (S::WBOX * G8_BLOCK) : b * (G8_XFEW * G8_BLOCK);
        const void* map = is_w ? static_cast<const void*>(&args.wmap)
                               : few ? static_cast<const void*>(&args.xfew) : static_cast<const void*>(&args.xmap);
        // Weights that no other tile reads make way in L2 first (64 tokens: gate-up 45.6 -> 44.5 us, down 26.8 -> 25.4;
        // 82 rows of 60 experts, the wide tile, 21.2 -> 20.5)
        const bool once = !PAIR && is_w && s_end[tile.e] - s_begin[tile.e] <= S::BM;
        for (int kb = 0; kb < k_blocks; ++kb, ++it) {
          const int s = it % STAGES, use = it / STAGES;
          int ok = 1;
          if (lane == 0) {
            if (use > 0) ok = (int)mbar_wait(&empty_bar[s], (use - 1) & 1, wait_ns);
            if (ok && cr == 0) mbar_arrive_expect_tx(&full_bar[s], bytes);
          }
          ok = __shfl_sync(0xffffffffu, ok, 0);
          if (!ok) {
            if (lane == 0) *status = DS_TIMEOUT_EMPTY;
            alive = false;
            break;
          }
          if (is_w || is_x) {
            unsigned char* dst = stages + (size_t)s * S::STAGE_BYTES + off;
            if (PAIR) tma_load_2d_pair(dst, map, kb * G8_BLOCK, y, cluster_map(&full_bar[s], 0));
            else if (once) tma_load_2d_hint(dst, map, kb * G8_BLOCK, y, &full_bar[s], policy);
            else tma_load_2d(dst, map, kb * G8_BLOCK, y, &full_bar[s]);
          }
        }
      }
      // The copies already issued land before the block can exit, whoever gave up on a wait. (PAIR: the other
      // CTA's count on the leader's barriers, and it does not leave before the leader; what it waits for
      // itself is the leader's last words on its own barriers.)
      if (lane == 0)
        for (int j = it > STAGES ? it - STAGES : 0; j < it; ++j)
          mbar_wait(cr == 0 ? &full_bar[j % STAGES] : &empty_bar[j % STAGES], (j / STAGES) & 1, 10000000ull);
    } else if (warp <= 2) {
      // -------------------------------------------------------------- MMA issuers (PAIR: the leader's, for both CTAs)
      // Two warps take the k blocks in turn: a wait costs its warp 100 to 250 clocks even when there is
      // nothing to wait for, and with one warp those came one after another, 750 clocks a block of 128
      // columns instead of 560. The whole warp walks the blocks (so that descriptors and loop counters stay in uniform
      // registers), one elected lane issues.
      if (cr == 0) {
        const uint32_t ring_lo = umma_desc_lo(smem_u32(stages));
        const uint32_t idesc = FEW ? umma_idesc(0, 128, S::XR) : umma_idesc(0, S::BM, WR);  // format 0 is e4m3 in this kind
        const int n = total_tiles > unit ? ((total_tiles - unit + units - 1) / units) * k_blocks : 0;
        int last = -1;
        for (int it = warp - 1; it < n; it += 2) {
          const int s = it % STAGES, buf = it % BUFS;
          const uint32_t d = tmem + buf * S::PART;
          if (!mbar_wait(&full_bar[s], (it / STAGES) & 1, wait_ns)) {
            *status = DS_TIMEOUT_FULL;
            break;
          }
          if (it >= BUFS && !mbar_wait(&part_empty[buf], (it / BUFS - 1) & 1, wait_ns)) {
            *status = DS_TIMEOUT_TMEM;
            break;
          }
          tc_fence_after_sync();
          const uint32_t x_lo = ring_lo + s * (S::STAGE_BYTES >> 4), w_lo = x_lo + (S::X_BYTES >> 4);
          if (elect_one()) {
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) {  // 32 k = 32 bytes inside the 128-byte rows
              if (FEW) {
                umma_f8(d, w_lo + ks * 2, x_lo + ks * 2, UMMA_DESC_HI_K_SW128, idesc, ks != 0);
                if (S::MMAS == 2)
                  umma_f8(d + S::XR, w_lo + (128 * G8_BLOCK >> 4) + ks * 2, x_lo + ks * 2, UMMA_DESC_HI_K_SW128, idesc, ks != 0);
                continue;
              }
              if (PAIR) umma_f8_pair(d, x_lo + ks * 2, w_lo + ks * 2, UMMA_DESC_HI_K_SW128, idesc, ks != 0);
              else umma_f8(d, x_lo + ks * 2, w_lo + ks * 2, UMMA_DESC_HI_K_SW128, idesc, ks != 0);
            }
            if (PAIR) {
              umma_commit_pair(&part_full[buf], 3);
              umma_commit_pair(&empty_bar[s], 3);
            } else {
              umma_commit(&part_full[buf]);
              umma_commit(&empty_bar[s]);
            }
          }
          __syncwarp();
          last = it;
        }
        if (last >= 0) mbar_wait(&empty_bar[last % STAGES], (last / STAGES) & 1, 10000000ull);  // nothing is left running
      }
    } else {
      // -------------------------------------------------------------- scales (and the rows of no expert)
      for (int r = (int)blockIdx.x, lo = s_begin[0], hi = s_end[E - 1]; r < lo + (args.rows - hi); r += (int)gridDim.x) {
        const size_t at = r < lo ? r : hi + (r - lo);
        uint4* row = reinterpret_cast<uint4*>(static_cast<T*>(args.C) + at * Nout);
        for (int c = lane; c < Nout / (16 / (int)sizeof(T)); c += 32) row[c] = make_uint4(0u, 0u, 0u, 0u);
        if constexpr (OUT8)
          for (int b = lane; b < (Nout + G8_BLOCK - 1) / G8_BLOCK; b += 32) args.cscale[(size_t)b * args.rows + at] = 0.f;
      }
      // Every block's scales are copied asynchronously, G8_AHEAD blocks before their turn: the first
      // ones come from DRAM, behind the weights. (Loads into registers are no ring: waiting for an
      // old one waits for the young ones too, 3000 clocks a block at the start of a launch.) When they
      // are there the block's partial product gets this warp's word, which is due only once the
      // block before in the same partial product has had its own: by then the block before that one
      // is promoted, so at most G8_AHEAD + 2 BUFS + 1 slots are in use.
      static_assert(G8_AHEAD + 2 * BUFS + 1 <= G8_SLOTS, "slots");
      const int n_blocks = (Nout + G8_BLOCK - 1) / G8_BLOCK;
      const int n = total_tiles > unit ? ((total_tiles - unit + units - 1) / units) * k_blocks : 0;
      int t = unit, kb = 0, cursor = 0, mine = 0, ahead = 0;
      const float *px = nullptr, *pw = nullptr;
      auto enter = [&]() {  // tile t
        const Tile8 tile = locate_tile8<S::BM>(t, cursor, E, s_tile_start, s_begin, s_end);
        mine = min(max(tile.nvalid - cr * S::XR, 0), S::XR);
        px = args.xscale + tile.row0 + cr * S::XR + lane;
        const int col = tile.cb * tile_cols;
        const int nb = SWIGLU ? (lane & 1) * n_blocks + col / G8_BLOCK
                              : min((col + (lane & 1) * (WR / 2)) / G8_BLOCK, n_blocks - 1);
        pw = args.wscale + ((size_t)tile.e * (SWIGLU ? 2 : 1) * n_blocks + nb) * k_blocks;  // lane parity: the half
      };
      auto fetch = [&]() {
        if (ahead < n) {
          float* slot = s_scale[ahead % G8_SLOTS];
#pragma unroll
          for (int r = 0; r < S::XR; r += 32)
            if (r + lane < mine) cp_async_4(slot + r + lane, px + r);
          if (lane < 2) cp_async_4(slot + G8_XR + lane, pw);
          px += args.rows, ++pw;
          if (++kb == k_blocks) {
            kb = 0, t += units;
            if (t < total_tiles) enter();
          }
        }
        ++ahead;
        cp_async_commit();
      };
      if (n) enter();
      for (int i = 0; i < G8_AHEAD; ++i) fetch();
      for (int it = 0; it < n; ++it) {
        const int buf = it % BUFS;
        if (it >= BUFS && !mbar_wait(&part_full[buf], (it / BUFS - 1) & 1, wait_ns)) {
          *status = DS_TIMEOUT_MMA;
          break;
        }
        __syncwarp();
        fetch();
        cp_async_wait<G8_AHEAD>();
        __syncwarp();
        if (lane == 0) mbar_arrive(&part_full[buf]);
      }
      cp_async_wait<0>();
    }
  } else if constexpr (FEW) {
    // ---------------------------------------------------------------- promotion and epilogue, few token rows
    // A thread owns a weight row (8-bit results: a gate row and its up row) and 16 token rows.
    constexpr int TOK = S::TOKENS, MMAS = S::MMAS;
    constexpr bool APART = SWIGLU && MMAS == 1;  // warps 0, 1 of a group have the gate rows, 2, 3 the up rows
    const int q = warp & 3, g = (warp - G8_HELPERS) >> 2;  // quarter of the weight rows; half of the token rows
    const uint32_t taddr = tmem + ((uint32_t)(q * 32) << 16) + g * TOK;
    int it = 0, cursor = 0, parity = 0;
    bool alive = true;
    for (int t = unit; t < total_tiles; t += units) {
      const Tile8 tile = locate_tile8<S::BM>(t, cursor, E, s_tile_start, s_begin, s_end);
      const int rows = tile.nvalid - g * TOK;  // token rows of the warp's
      uint64_t acc[MMAS][TOK / 2];
#pragma unroll
      for (int j = 0; j < TOK / 2; ++j)
        for (int h = 0; h < MMAS; ++h) acc[h][j] = 0;
#pragma unroll 1
      for (int kb = 0; kb < k_blocks; ++kb, ++it) {
        const int buf = it % BUFS;
        if (alive && !mbar_wait(&part_full[buf], (it / BUFS) & 1, wait_ns)) {
          *status = DS_TIMEOUT_MMA;
          alive = false;
        }
        __syncwarp();
        tc_fence_after_sync();
        const uint32_t from = taddr + buf * S::PART;
        const float* slot = s_scale[it % G8_SLOTS];
        uint32_t v[MMAS * TOK];
        uint64_t sx[TOK / 2];
        const uint64_t w0 = twice(slot[G8_XR + (APART && q >= 2 ? 1 : 0)]), w1 = twice(slot[G8_XR + 1]);
        if (rows > 0) {
          if constexpr (MMAS == 2) tmem_get_16_16(from, from + S::XR, v);
          else tmem_get_16(from, v);
#pragma unroll
          for (int j = 0; j < TOK / 2; j += 2) {
            const float4 f = *reinterpret_cast<const float4*>(slot + g * TOK + 2 * j);
            sx[j] = pair64(make_float2(f.x, f.y)), sx[j + 1] = pair64(make_float2(f.z, f.w));
          }
        }
        tc_fence_before_sync();
        __syncwarp();
        if (elect_one()) mbar_arrive(&part_empty[buf]);
        __syncwarp();
        if (rows > 0) {
#pragma unroll
          for (int j = 0; j < TOK / 2; ++j) {
            fma2(acc[0][j], v[2 * j], v[2 * j + 1], mul2(sx[j], w0));
            if constexpr (MMAS == 2) fma2(acc[1][j], v[TOK + 2 * j], v[TOK + 2 * j + 1], mul2(sx[j], w1));
          }
        }
      }
      alive = __all_sync(0xffffffffu, alive);
      if (rows <= 0 || (!alive && !OUT8 && !APART)) continue;
      const int col = tile.cb * tile_cols + (APART ? q & 1 : q) * 32 + lane;
      const size_t row0 = tile.row0 + g * TOK;
      float f[TOK];  // the results. Rows that the tile lacks are worked out too: a branch for each costs more
#pragma unroll
      for (int i = 0; i < TOK; ++i) {
        const float2 v = both(acc[0][i / 2]);
        f[i] = i & 1 ? v.y : v.x;
      }
      if constexpr (APART) {
        float* up = s_up[parity * 2 + g] + (q & 1) * 32 + lane;  // (two of them: a warp is at most a tile ahead)
        if (q >= 2) {
#pragma unroll
          for (int i = 0; i < TOK; ++i) up[i * (WR / 2)] = f[i];
        }
        named_barrier_sync(1 + g, 128);
        parity ^= 1;
        if (q >= 2 || !alive) continue;
#pragma unroll
        for (int i = 0; i < TOK; ++i) {
          if (i == TOK / 2 && rows <= TOK / 2) break;
          f[i] = swiglu_lane(f[i], up[i * (WR / 2)]);
        }
      } else if constexpr (SWIGLU) {
#pragma unroll
        for (int i = 0; i < TOK; ++i) {
          if (i == TOK / 2 && rows <= TOK / 2) break;
          const float2 u = both(acc[MMAS - 1][i / 2]);
          f[i] = swiglu_lane(f[i], i & 1 ? u.y : u.x);
        }
      } else if (args.scale) {
        const T* sc = static_cast<const T*>(args.scale) + row0;
        float r[TOK];
#pragma unroll
        for (int i = 0; i < TOK; ++i) r[i] = i < rows ? Elem<T>::to_f(sc[i]) : 0.f;
#pragma unroll
        for (int i = 0; i < TOK; ++i) f[i] *= r[i];
      }
      T* to = static_cast<T*>(args.C) + row0 * Nout + col;
      if constexpr (OUT8) {
        // As in the other tiles; the block's 128 columns are the four warps' lanes. Magnitudes as
        // integers order like floats, NaN above all.
        uint32_t most = 0;
#pragma unroll
        for (int i = 0; i < TOK; ++i) {
          const uint32_t m = __reduce_max_sync(0xffffffffu, col < Nout ? __float_as_uint(f[i]) & 0x7fffffffu : 0u);
          if (lane == i) most = m;
        }
        uint32_t* tops = reinterpret_cast<uint32_t*>(s_top[parity][g]);  // [warp][token row]
        if (lane < TOK) tops[q * TOK + lane] = most;
        named_barrier_sync(1 + g, 128);
#pragma unroll
        for (int i = 0; i < 4; ++i) most = max(most, tops[i * TOK + lane % TOK]);
        parity ^= 1;
        if (!alive) continue;
        const float top = most > 0x7f800000u ? __int_as_float(0x7fffffff) : fmaxf(__uint_as_float(most), 0x1p-96f);
        const float inv = 448.f / top;  // of token row `lane`
#pragma unroll
        for (int i = 0; i < TOK; ++i) {
          const float by = __shfl_sync(0xffffffffu, inv, i);
          if (i < rows && col < Nout)
            reinterpret_cast<__nv_fp8_storage_t*>(to)[(size_t)i * Nout] = __nv_cvt_float_to_fp8(f[i] * by, __NV_SATFINITE, __NV_E4M3);
        }
        if (q == 0 && lane < min(rows, TOK)) args.cscale[(size_t)tile.cb * args.rows + row0 + lane] = top / 448.f;
      } else {
#pragma unroll
        for (int i = 0; i < TOK; ++i)
          if (i < rows && col < Nout) to[(size_t)i * Nout] = Elem<T>::from_f(f[i]);
      }
    }
  } else {
    // ---------------------------------------------------------------- promotion and epilogue
    if (S::SPLIT_REGS) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(G8_REGS_MANY));
    const int q = warp & 3, g = (warp - G8_HELPERS) >> 2;  // quarter of the lanes; quarter of the columns: COLS of either half
    const int trow = cr * G8_XR + q * 32 + lane;
    const uint32_t taddr = tmem + ((uint32_t)(q * 32) << 16) + g * S::COLS;
    int it = 0, cursor = 0, parity = 0;
    bool alive = true;
    Tile8 next;
    if (unit < total_tiles) next = locate_tile8<S::BM>(unit, cursor, E, s_tile_start, s_begin, s_end);
    for (int t = unit; t < total_tiles; t += units) {
      const Tile8 tile = next;
      const bool busy = cr * G8_XR + q * 32 < tile.nvalid;  // the warp has rows of this tile
      float row_scale = 1.f;
      if constexpr (!SWIGLU)
        if (args.scale && trow < tile.nvalid) row_scale = Elem<T>::to_f(static_cast<const T*>(args.scale)[tile.row0 + trow]);
      uint64_t acc[2][S::COLS / 2];
#pragma unroll
      for (int j = 0; j < S::COLS / 2; ++j) acc[0][j] = acc[1][j] = 0;
#pragma unroll 1
      for (int kb = 0; kb < k_blocks; ++kb, ++it) {
        const int buf = it % BUFS;
        // (a warp that gave up goes on without waiting)
        if (alive && !mbar_wait(&part_full[buf], (it / BUFS) & 1, wait_ns)) {
          *status = DS_TIMEOUT_MMA;
          alive = false;
        }
        __syncwarp();
        tc_fence_after_sync();
        // All of the partial product is in registers: its buffer may be overwritten. The loads were
        // the whole warp's, so one lane's word is enough.
        auto close = [&]() {
          tc_fence_before_sync();
          if (elect_one()) {
            if (PAIR) arrive_leader(cluster_map(&part_empty[buf], 0));
            else mbar_arrive(&part_empty[buf]);
          }
          __syncwarp();
        };
        if (busy) {
          const uint32_t from = taddr + buf * WR;
          const float* slot = s_scale[it % G8_SLOTS];
          const float sx = slot[q * 32 + lane];
          const uint64_t f0 = twice(sx * slot[G8_XR]), f1 = twice(sx * slot[G8_XR + 1]);
          // as many columns at once as there are registers for
          constexpr int AT_ONCE = 32, GROUPS = 2 * S::COLS / AT_ONCE;
#pragma unroll
          for (int c = 0; c < GROUPS; ++c) {
            uint32_t v[AT_ONCE];
            tmem_get_32(from + (c * 32 / S::COLS) * (WR / 2) + c * 32 % S::COLS, v);
            if (c + 1 == GROUPS) close();
#pragma unroll
            for (int j = 0; j < AT_ONCE / 2; ++j) {
              const int at = c * AT_ONCE + 2 * j;  // of the thread's columns
              fma2(acc[at / S::COLS][at % S::COLS / 2], v[2 * j], v[2 * j + 1], at < S::COLS ? f0 : f1);
            }
          }
        } else {
          close();
        }
        if (kb == 0 && t + units < total_tiles)  // found while the next block is being multiplied
          next = locate_tile8<S::BM>(t + units, cursor, E, s_tile_start, s_begin, s_end);
      }
      alive = __all_sync(0xffffffffu, alive);
      if (!busy || (!alive && !OUT8)) continue;  // (8-bit results: the warp of the same rows waits at a barrier below)
      const int rows = tile.nvalid - (cr * G8_XR + q * 32), col = tile.cb * tile_cols + g * S::COLS;
      T* to = static_cast<T*>(args.C) + (size_t)(tile.row0 + cr * G8_XR + q * 32) * Nout + col;
      // 64 bytes of results per lane, its row's from column col + c on, to memory by way of shared memory:
      // a store then covers eight rows of 64 bytes, where a lane's own row would make it touch 32 lines.
      auto store64 = [&](int c, const uint32_t (&o)[16]) {
        constexpr int PART = 16 / sizeof(T);
        unsigned char* mine = s_out[warp - G8_HELPERS] + lane * G8_OUT_PITCH;
#pragma unroll
        for (int i = 0; i < 4; ++i) *reinterpret_cast<uint4*>(mine + i * 16) = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
        __syncwarp();
        const int part = lane & 3;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = i * 8 + (lane >> 2);
          const uint4 v = *reinterpret_cast<const uint4*>(s_out[warp - G8_HELPERS] + r * G8_OUT_PITCH + part * 16);
          if (r < rows && col + c + part * PART < Nout)
            *reinterpret_cast<uint4*>(to + (size_t)r * Nout + c + part * PART) = v;
        }
        __syncwarp();
      };
      // The same with 128 bytes of a row, half of the rows at a time: whole lines, where there are so many results
      // that the epilogues' writes are what waits (65,536 rows by 2048 columns, k 1024: 175 -> 167 us of
      // the wide tile, 170 -> 164 of the pair's; 8 rows per expert 26.4 -> 26.7; SwiGLU's half as many
      // results were no faster for it).
      auto store128 = [&](int c, const uint32_t (&o)[32]) {
        constexpr int PART = 16 / sizeof(T), PITCH = 128 + 16;
        static_assert(16 * PITCH <= sizeof(s_out[0]), "staging");
        unsigned char* half = s_out[warp - G8_HELPERS];
        const int part = lane & 7;
#pragma unroll
        for (int r0 = 0; r0 < 32; r0 += 16) {
          if ((lane & 16) == r0) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
              *reinterpret_cast<uint4*>(half + (lane & 15) * PITCH + i * 16) = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
          }
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int r = i * 4 + (lane >> 3);
            const uint4 v = *reinterpret_cast<const uint4*>(half + r * PITCH + part * 16);
            if (r0 + r < rows && col + c + part * PART < Nout)
              *reinterpret_cast<uint4*>(to + (size_t)(r0 + r) * Nout + c + part * PART) = v;
          }
          __syncwarp();
        }
      };
      if constexpr (OUT8) {
        // (Every operation per value counts: with two for the maximum and one for NaN, not two and three and
        // a bound, and packed products, a launch of 65,536 rows went from 276 to 260 us.)
        // The row's 128 columns are a block: its largest magnitude over this warp's 64 and, through shared
        // memory, over those of the warp that has the other half. A value is rounded from its product
        // with 448 / m; it comes out of float32 sums, so there are no midpoints to keep.
        swiglu_pairs<!OUT8>(acc[0], acc[1]);
        float top = 0.f;
        if (col + S::COLS <= Nout) {
#pragma unroll
          for (int j = 0; j < S::COLS / 2; ++j) {
            const float2 v = both(acc[1][j]);
            top = max_nan(max_nan(top, fabsf(v.x)), fabsf(v.y));
          }
        } else {
#pragma unroll
          for (int j = 0; j < S::COLS / 2; ++j) {
            const float2 v = both(acc[1][j]);
            if (col + 2 * j < Nout) top = max_nan(max_nan(top, fabsf(v.x)), fabsf(v.y));  // Nout is even
          }
        }
        float(*half)[G8_XR] = s_top[parity];
        half[g][q * 32 + lane] = top;
        named_barrier_sync(1 + q, 64);
        const float other = half[g ^ 1][q * 32 + lane];
        top = max_nan(max_nan(top, other), 0x1p-96f);
        parity ^= 1;
        if (!alive) continue;
        const uint64_t inv = twice(448.f / top);
        uint32_t o[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const float2 a = both(mul2(acc[1][2 * j], inv)), b = both(mul2(acc[1][2 * j + 1], inv));
          o[j] = (uint32_t)__nv_cvt_float2_to_fp8x2(a, __NV_SATFINITE, __NV_E4M3) |
                 ((uint32_t)__nv_cvt_float2_to_fp8x2(b, __NV_SATFINITE, __NV_E4M3) << 16);
        }
        store64(0, o);
        if (g == 0 && lane < rows)
          args.cscale[(size_t)(col / G8_BLOCK) * args.rows + tile.row0 + trow] = top / 448.f;
      } else if constexpr (SWIGLU) {
        swiglu_pairs<!OUT8>(acc[0], acc[1]);
#pragma unroll
        for (int c = 0; c < S::COLS; c += 32) {
          uint32_t o[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const float2 v = both(acc[1][c / 2 + j]);
            o[j] = pack16<T>(v.x, v.y);
          }
          store64(c, o);
        }
      } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t o[32];
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            const float2 v = both(acc[h][j]);
            o[j] = pack16<T>(v.x * row_scale, v.y * row_scale);
          }
          store128(h * (WR / 2), o);
        }
      }
    }
  }

  tc_fence_before_sync();
  __syncthreads();
  if (PAIR) cluster_sync_all();  // neither CTA leaves while the other may still signal or read it
  if (warp == 1) {
    tc_fence_after_sync();
    if (PAIR) tmem_dealloc_pair(tmem, S::TMEM_COLS);
    else tmem_dealloc(tmem, S::TMEM_COLS);
  }
}

// ---- host side ------------------------------------------------------------------------------
// How many blocks (pairs: clusters of two) fit the device at once; asked once per kernel and device.
template <typename T, int TILE, bool SWIGLU> static int units8(int sms, int* out) {
  static std::atomic<int> cached[MAX_DEVICES];
  int dev = 0;
  SY_CUDA(cudaGetDevice(&dev));
  int units = cached[dev].load(std::memory_order_acquire);
  if (!units) {
    auto kern = gemm8_kernel<T, TILE, SWIGLU>;
    SY_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, G8_SMEM));
    if (Shape8<TILE, std::is_same<T, __nv_fp8_e4m3>::value>::SPLIT_REGS) {
      // the promoters' register request waits for ever if the block was launched with fewer
      cudaFuncAttributes attr;
      SY_CUDA(cudaFuncGetAttributes(&attr, kern));
      if (attr.numRegs < G8_REGS_LAUNCH)
        return fail(SY_ERR_CUDA, "grouped_gemm_fp8: built with %d registers per thread, needs %d", attr.numRegs, G8_REGS_LAUNCH);
    }
    if (Shape8<TILE, std::is_same<T, __nv_fp8_e4m3>::value>::PAIR) {
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(sms & ~1);
      cfg.blockDim = dim3(Shape8<TILE, std::is_same<T, __nv_fp8_e4m3>::value>::THREADS);
      cfg.dynamicSmemBytes = G8_SMEM;
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = 2;
      attr[0].val.clusterDim.y = 1;
      attr[0].val.clusterDim.z = 1;
      cfg.attrs = attr;
      cfg.numAttrs = 1;
      SY_CUDA(cudaOccupancyMaxActiveClusters(&units, kern, &cfg));
      if (units > sms / 2) units = sms / 2;
    } else {
      int per_sm = 0;
      SY_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kern, Shape8<TILE, std::is_same<T, __nv_fp8_e4m3>::value>::THREADS, G8_SMEM));
      units = per_sm >= 1 ? sms : 0;
    }
    if (units < 1) return fail(SY_ERR_CUDA, "grouped_gemm_fp8: no block of the kernel fits on this device");
    cached[dev].store(units, std::memory_order_release);
  }
  *out = units;
  return SY_OK;
}

template <typename T, int TILE, bool SWIGLU>
static int launch8(Gemm8Args a, const void* x, const void* w, cudaStream_t stream) {
  using S = Shape8<TILE, std::is_same<T, __nv_fp8_e4m3>::value>;
  int sms = 0, units = 0;
  int rc = device_sm_count(&sms);
  if (rc != SY_OK) return rc;
  rc = units8<T, TILE, SWIGLU>(sms, &units);
  if (rc != SY_OK) return rc;
  const uint64_t w_rows = (uint64_t)a.experts * (SWIGLU ? 2 : 1) * a.Nout;
  rc = tensor_map_2d(&a.wmap, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, w, w_rows, (uint64_t)a.K, S::WBOX, G8_BLOCK);
  if (rc != SY_OK) return rc;
  if (!S::FEW) {
    rc = tensor_map_2d(&a.xmap, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, x, (uint64_t)a.rows, (uint64_t)a.K, G8_XR, G8_BLOCK);
    if (rc != SY_OK) return rc;
  }
  rc = tensor_map_2d(&a.xfew, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, x, (uint64_t)a.rows, (uint64_t)a.K, G8_XFEW, G8_BLOCK);
  if (rc != SY_OK) return rc;
  auto kern = gemm8_kernel<T, TILE, SWIGLU>;
  if (S::PAIR) return launch_cluster_kernel(kern, 2, 2 * units, S::THREADS, G8_SMEM, stream, "grouped_gemm_fp8 launch", a);
  return launch_kernel(kern, units, S::THREADS, G8_SMEM, stream, "grouped_gemm_fp8 launch", a);
}

template <typename T, bool SWIGLU>
static int dispatch8(const Gemm8Args& a, int tile, const void* x, const void* w, cudaStream_t s) {
  return tile == G8_FEW    ? launch8<T, G8_FEW, SWIGLU>(a, x, w, s)
         : tile == G8_WIDE ? launch8<T, G8_WIDE, SWIGLU>(a, x, w, s)
                           : launch8<T, G8_PAIR, SWIGLU>(a, x, w, s);
}

// Which tile a batch gets; the bits are the same. Measured on a B200 with the benchmark's layer (64 experts, top-8,
// gate and up 2048 x 2048 with SwiGLU, down 2048 x 1024), us for the few / wide / pair tile: the fastest of five
// graph replays of about 2 ms, 20 ms apart, over four weight sets (each larger than L2). Even routing, where
// not called skewed (the most popular expert has 4.9 times the mean, the least 0.4):
//   1 token     gate-up  9.5 / 13.4 / 14.0    down  6.6 /  8.8 /  8.7    8-bit results 11.5 / 13.7 / 14.6
//   8 tokens            31.3 / 35.7 / 45.6         17.7 / 20.4 / 28.1                  32.7 / 36.8 / 48.1
//   64 tokens           43.5 / 49.4 / 65.8         24.5 / 26.5 / 37.5                  45.9 / 50.2 / 67.9
//   160 tokens          44.3 / 49.0 / 66.1         25.6 / 26.1 / 38.2                  45.8 / 50.1 / 68.2   (20 rows per expert)
//      skewed           49.8 / 50.1 / 66.3         27.5 / 26.6 / 38.0                  48.9 / 50.8 / 68.4
//   192 tokens          48.1 / 50.3 / 66.3         26.9 / 26.4 / 38.3                  44.6 / 51.0 / 68.3
//      skewed           53.8 / 49.2 / 66.5         30.1 / 26.4 / 38.1                  51.0 / 50.4 / 68.6
//   256 tokens          61.4 / 50.2 / 66.9         34.4 / 26.3 / 38.3                  52.3 / 50.6 / 68.8
//   512 tokens                 51.5 / 69.7                26.9 / 39.7                         52.6 / 71.9
//   1024 tokens                67.1 / 71.6                40.1 / 45.8                         67.2 / 72.4
//   4096 tokens                 168 /  169                 101 /  103                          167 /  169
//   6144 tokens                 240 /  241                 144 /  149                          237 /  239   (768)
//      skewed                   241 /  235                 144 /  143                          237 /  234
//   8192 tokens                 312 /  303                 187 /  185                          309 /  303
// So: few up to 20 rows per expert (its 32 token rows are then seldom too few), pairs from 768, else wide.
// At 20 rows per expert of other layers: 8 experts, gate and up 1024 x 1024, 6.2 / 7.5 (few rows win up to 50 rows per
// expert, 6.7 / 7.5: the wide tiles do not fill the SMs); 16 experts 2048 x 2048, 15.7 / 16.0, skewed 17.7 / 15.9;
// 60 experts 992 x 1040, 18.7 / 17.1; 128 experts 1024 x 1024, 27.0 / 27.0, skewed 31.7 / 27.3.
static int choose_tile8(int rows, int experts) {
  return rows <= 20LL * experts ? G8_FEW : rows < 768LL * experts ? G8_WIDE : G8_PAIR;
}

}  // namespace sy

extern "C" int sy_grouped_gemm_fp8(const void* x, const float* x_scale, const void* w, const float* w_scale,
                                   const int32_t* offsets, int n_experts, int rows, int n_out, int k_dim, int swiglu,
                                   const void* scale, void* C, float* c_scale, int dtype, int tile, void* stream) {
  using namespace sy;
  SY_REQUIRE(rows >= 0 && rows <= G8_MOST, "grouped_gemm_fp8: 0..%d rows (got %d)", G8_MOST, rows);
  SY_REQUIRE(n_experts >= 1 && n_experts <= G8_MAX_E, "grouped_gemm_fp8: 1..%d experts (got %d)", G8_MAX_E,
             n_experts);
  SY_REQUIRE(k_dim > 0 && k_dim <= G8_MOST && k_dim % 16 == 0,
             "grouped_gemm_fp8: k_dim must be a multiple of 16, at most %d (got %d)", G8_MOST, k_dim);
  SY_REQUIRE(n_out > 0 && n_out % 8 == 0, "grouped_gemm_fp8: n_out must be a multiple of 8 (got %d)", n_out);
  SY_REQUIRE(!(swiglu && scale), "grouped_gemm_fp8: swiglu and scale are separate epilogues");
  SY_REQUIRE(c_scale || dtype == SY_DTYPE_F16 || dtype == SY_DTYPE_BF16, "grouped_gemm_fp8: dtype must be f16 or bf16");
  SY_REQUIRE(!c_scale || (swiglu && n_out % 16 == 0),
             "grouped_gemm_fp8: 8-bit results are SwiGLU's, of a multiple of 16 columns");
  SY_REQUIRE(tile >= 0 && tile <= 3, "grouped_gemm_fp8: tile 0..3 (got %d)", tile);
  SY_REQUIRE((int64_t)n_experts * 2 * n_out <= 0x7fffff00, "grouped_gemm_fp8: more than 2^31 weight rows");
  if (rows == 0) return SY_OK;
  SY_REQUIRE(x && x_scale && w && w_scale && offsets && C, "grouped_gemm_fp8: null pointer");
  SY_REQUIRE((uintptr_t)x % 16 == 0 && (uintptr_t)w % 16 == 0 && (uintptr_t)C % 16 == 0,
             "grouped_gemm_fp8: x, w and C must be 16-byte aligned");
  Gemm8Args a;
  memset(&a, 0, sizeof(a));
  a.xscale = x_scale;
  a.wscale = w_scale;
  a.offsets = offsets;
  a.scale = scale;
  a.C = C;
  a.cscale = c_scale;
  a.experts = n_experts;
  a.rows = rows;
  a.Nout = n_out;
  a.K = k_dim;
  a.status = device_status_word();
  if (!a.status) return SY_ERR_CUDA;
  a.wait_ns = wait_limit_ns();
  if (tile == 0) tile = choose_tile8(rows, n_experts);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (c_scale) return dispatch8<__nv_fp8_e4m3, true>(a, tile, x, w, s);
  if (dtype == SY_DTYPE_F16) return swiglu ? dispatch8<__half, true>(a, tile, x, w, s) : dispatch8<__half, false>(a, tile, x, w, s);
  return swiglu ? dispatch8<__nv_bfloat16, true>(a, tile, x, w, s) : dispatch8<__nv_bfloat16, false>(a, tile, x, w, s);
}
