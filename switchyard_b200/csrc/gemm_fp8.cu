// The experts' product in 8-bit floats: every expert's slice of the sorted rows times its weights,
// both e4m3 with float32 scales for blocks of 128 along k (1 x 128 for rows, 128 x 128 for weights):
//
//   acc[r, n] = sum_b sx[b, r] * sw[e, n / 128, b] * sum_{k in block b} x[r, k] * w[e, n, k]
//   C[r, n]   = round(acc[r, n] * scale[r])   or, with SwiGLU, round(silu(acc[r, gate n]) * acc[r, up n])
//
// Float32 scales cannot ride in the tensor core, so the inner sums of each block of 128 (four
// tcgen05.mma of k = 32) go to tensor memory on their own and eight warps multiply them by the
// two scales and add them up in float32 registers while the next block is being multiplied:
// tensor memory holds two such partial products. A thread owns a row of the tile and a half of its
// columns. Both factors of a step are the same for all of a thread's columns of one weight block,
// so the promotion costs one packed multiply-add per two values.
//
// Warps: 0 TMA producer, 1 MMA issuer, 2-3 spare (they clear rows that belong to no expert), 4-11 promotion and epilogue.
// Tiles as in gemm.cu: numbered on the device from `offsets`, expert-major, dealt round-robin to
// a persistent grid. Token rows are the MMA's M operand (128, or 256 over a pair of CTAs), weight
// rows its N operand, in two halves of WR / 2: consecutive rows, or with SwiGLU the gate rows and the
// up rows of the same columns. A thread takes the same quarter of the columns out of either half:
// it finds a gate value and its up value in its own registers, and each half of the tile is one
// TMA box (a box takes its thread about 130 clocks to issue, however small: six to eight boxes a
// stage took twice as long as the multiplication).
#include <cuda.h>

#include <atomic>
#include <string.h>
#include <type_traits>

#include "common.cuh"
#include "tensor_map.cuh"

namespace sy {

constexpr int G8_BLOCK = 128;                    // k per scale and per stage: one 128-byte swizzle atom
constexpr int G8_XR = 128;                       // token rows a CTA stages
constexpr int G8_XFEW = 32;                      // token rows of the small TMA box, for tiles of at most two of them
constexpr int G8_MAX_E = 256;
constexpr int G8_THREADS = 12 * 32;
constexpr int G8_PROMOTERS = 8;                  // warps
constexpr int G8_AHEAD = 6, G8_SLOTS = 8;        // k blocks that a scale is asked for before its use; slots of the ring
constexpr int G8_SLOT = 32 + 2;                  // a warp's scales of one k block: its rows' and the weights' two
constexpr int G8_RING_BYTES = 192 * 1024;
constexpr int G8_SMEM = G8_RING_BYTES + 1024;    // room to align the ring to 1024

// WR: weight rows per tile. PAIR: two CTAs share a tile (tcgen05 cta_group::2).
template <int WR, bool PAIR> struct Shape8 {
  static constexpr int CTAS = PAIR ? 2 : 1;
  static constexpr int BM = G8_XR * CTAS;                 // token rows per tile
  static constexpr int WRC = WR / CTAS;                   // weight rows a CTA stages
  static constexpr int WBOX = WR / 2;                     // weight rows per TMA box: a half of the tile
  static constexpr int W_BOXES = WRC / WBOX;              // PAIR: each CTA has one of the halves
  static constexpr int X_BYTES = G8_XR * G8_BLOCK;
  static constexpr int STAGE_BYTES = X_BYTES + WRC * G8_BLOCK;
  static constexpr int STAGES = G8_RING_BYTES / STAGE_BYTES;
  static constexpr int TMEM_COLS = 2 * WR;                // two partial products
  static constexpr int ACC = WR / 2;                      // columns per promoter thread
  // 128 accumulators need more registers than 65536 / 384: the four other warps hand theirs over
  static constexpr bool SPLIT_REGS = ACC > 64;
};
constexpr int G8_REGS_FEW = 72, G8_REGS_MANY = 216;       // 4 warps x 72 + 8 warps x 216 <= 12 warps x 168
constexpr int G8_REGS_LAUNCH = 168;
static_assert(4 * G8_REGS_FEW + 8 * G8_REGS_MANY <= 12 * G8_REGS_LAUNCH, "register split");

struct Gemm8Args {
  CUtensorMap wmap;   // [experts * halves * Nout, K] e4m3, box 128 k x WBOX
  CUtensorMap xmap;   // [rows, K] e4m3, box 128 k x 128
  CUtensorMap xfew;   // the same, box 128 k x 32
  const float* xscale;  // [k blocks][rows]
  const float* wscale;  // [experts][halves * n blocks][k blocks]
  const int* offsets;   // [experts + 1]
  const void* scale;    // [rows] or null
  void* C;              // [rows, Nout]
  int experts, rows, Nout, K, swiglu;
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
__device__ __forceinline__ void cp_async_4(float* dst_smem, const float* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(dst_smem)), "l"(src) : "memory");
}
// 32 lanes x 32 consecutive columns of tensor memory.
__device__ __forceinline__ void tmem_ld_x32(uint32_t addr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
      "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]),
        "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]),
        "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr)
      : "memory");
}
// Waits for this thread's tensor-memory loads. Naming the registers keeps their uses behind the wait.
__device__ __forceinline__ void tmem_ld_wait_x32(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                 "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                 "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
               :
               : "memory");
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

// Whether the barrier's phase is over; does not wait.
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.b32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}

struct Tile8 {
  int e, cb, row0, nvalid;
};

template <int BM>
__device__ __forceinline__ Tile8 locate_tile8(int t, int& cursor, const int* start, const int* begin, const int* end) {
  while (start[cursor + 1] <= t) ++cursor;
  const int local = t - start[cursor], n = end[cursor] - begin[cursor], row_tiles = (n + BM - 1) / BM;
  Tile8 tile;
  tile.e = cursor;
  tile.cb = local / row_tiles;
  tile.row0 = begin[cursor] + (local % row_tiles) * BM;
  tile.nvalid = min(BM, end[cursor] - tile.row0);
  return tile;
}

// silu(g) * u. exp and the division are the approximate ones: within about 2^-21, far inside the
// 16-bit rounding that follows.
__device__ __forceinline__ float swiglu32(float g, float u) { return __fdividef(g, 1.f + __expf(-g)) * u; }

template <typename T, int WR, bool PAIR>
__global__ void __launch_bounds__(G8_THREADS, 1) gemm8_kernel(const __grid_constant__ Gemm8Args args) {
  using S = Shape8<WR, PAIR>;
  constexpr int STAGES = S::STAGES, ACC = S::ACC;
  extern __shared__ unsigned char smem_raw[];
  __shared__ __align__(8) uint64_t full_bar[STAGES];
  __shared__ __align__(8) uint64_t empty_bar[STAGES];
  __shared__ __align__(8) uint64_t part_full[2];
  __shared__ __align__(8) uint64_t part_empty[2];
  __shared__ uint32_t s_tmem;
  __shared__ int s_begin[G8_MAX_E], s_end[G8_MAX_E];
  __shared__ int s_tile_start[G8_MAX_E + 2];
  __shared__ float s_scale[G8_PROMOTERS][G8_SLOTS][G8_SLOT];

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  unsigned char* stages =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  int* status = args.status;
  const uint64_t wait_ns = args.wait_ns;
  const int E = args.experts, Nout = args.Nout;
  const bool swiglu = args.swiglu != 0;
  const int cr = PAIR ? (int)cluster_ctarank() : 0;
  const int unit = PAIR ? (int)blockIdx.x >> 1 : (int)blockIdx.x, units = PAIR ? (int)gridDim.x >> 1 : (int)gridDim.x;
  const int tile_cols = swiglu ? WR / 2 : WR;
  const int col_blocks = (Nout + tile_cols - 1) / tile_cols;
  const int k_blocks = (args.K + G8_BLOCK - 1) / G8_BLOCK;

  pdl_launch_dependents();
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&part_full[b], 1);
      mbar_init(&part_empty[b], S::CTAS * G8_PROMOTERS);  // PAIR: the leader's, for both CTAs
    }
    fence_barrier_init();
    prefetch_tensormap(&args.wmap);
    prefetch_tensormap(&args.xmap);
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
  for (int e = threadIdx.x; e < E; e += G8_THREADS) {
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
    if (lane == 0) {
      s_tile_start[E] = carry;
      s_tile_start[E + 1] = 0x7fffffff;
    }
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
      for (int t = unit; t < total_tiles && alive; t += units) {
        const Tile8 tile = locate_tile8<S::BM>(t, cursor, s_tile_start, s_begin, s_end);
        // token rows: one box of 128, or one or two of 32 where the tile has no more
        auto rows_of = [&](int c) { return min(max(tile.nvalid - c * G8_XR, 0), G8_XR); };
        auto x_bytes = [&](int n) {
          return n > 2 * G8_XFEW ? S::X_BYTES : (n + G8_XFEW - 1) / G8_XFEW * (G8_XFEW * G8_BLOCK);
        };
        const int mine = rows_of(cr);
        const bool few = mine <= 2 * G8_XFEW;
        const int x_boxes = few ? (mine + G8_XFEW - 1) / G8_XFEW : 1;
        const uint32_t bytes = WR * G8_BLOCK + x_bytes(mine) + (PAIR ? x_bytes(rows_of(cr ^ 1)) : 0);  // of all CTAs of the tile
        const bool is_w = lane < S::W_BOXES, is_x = !is_w && lane - S::W_BOXES < x_boxes;
        const int b = is_w ? cr + lane : lane - S::W_BOXES;  // half of the weight rows, or box of token rows
        const int colbase = tile.cb * tile_cols;
        const int y = is_w ? (swiglu ? (tile.e * 2 + b) * Nout + colbase : tile.e * Nout + colbase + b * S::WBOX)
                           : tile.row0 + cr * G8_XR + b * G8_XFEW;
        const int off = is_w ? S::X_BYTES + lane * (S::WBOX * G8_BLOCK) : b * (G8_XFEW * G8_BLOCK);
        const void* map = is_w ? static_cast<const void*>(&args.wmap)
                               : few ? static_cast<const void*>(&args.xfew) : static_cast<const void*>(&args.xmap);
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
            else tma_load_2d(dst, map, kb * G8_BLOCK, y, &full_bar[s]);
          }
        }
      }
      if (!alive && cr == 0 && lane == 0)  // the copies already issued land before the block can exit
        for (int j = it > STAGES ? it - STAGES : 0; j < it; ++j) mbar_wait(&full_bar[j % STAGES], (j / STAGES) & 1, 10000000ull);
    } else if (warp == 1) {
      // -------------------------------------------------------------- MMA issuer (PAIR: the leader's, for both CTAs)
      // The whole warp walks the k blocks (so that descriptors and loop counters stay in uniform
      // registers), one elected lane issues; the next block's two barriers are looked at while this
      // block's MMAs are on their way.
      if (cr == 0) {
        const uint32_t ring_lo = umma_desc_lo(smem_u32(stages));
        const uint32_t idesc = umma_idesc(0, S::BM, WR);  // format 0 is e4m3 in this kind
        const int n = total_tiles > unit ? ((total_tiles - unit + units - 1) / units) * k_blocks : 0;
        int s = 0;
        uint32_t phase = 0;
        bool drained = true, filled = false;
        for (int it = 0; it < n; ++it) {
          const int buf = it & 1;
          if (!drained && !mbar_wait(&part_empty[buf], ((it >> 1) - 1) & 1, wait_ns)) {
            *status = DS_TIMEOUT_TMEM;
            break;
          }
          if (!filled && !mbar_wait(&full_bar[s], phase, wait_ns)) {
            *status = DS_TIMEOUT_FULL;
            break;
          }
          tc_fence_after_sync();
          const uint32_t x_lo = ring_lo + s * (S::STAGE_BYTES >> 4), w_lo = x_lo + (S::X_BYTES >> 4);
          const uint32_t d = tmem + buf * WR;
          const int s_next = s + 1 == STAGES ? 0 : s + 1;
          const uint32_t phase_next = s_next ? phase : phase ^ 1;
          if (elect_one()) {
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) {  // 32 k = 32 bytes inside the 128-byte rows
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
          drained = it < 1 || mbar_test(&part_empty[buf ^ 1], (((it + 1) >> 1) - 1) & 1);
          filled = mbar_test(&full_bar[s_next], phase_next);
          s = s_next, phase = phase_next;
        }
      }
    } else {
      // -------------------------------------------------------------- rows of no expert are zero
      const int lo = E ? s_begin[0] : 0, hi = E ? s_end[E - 1] : 0;
      const int vecs = Nout / 8, who = ((int)blockIdx.x * 2 + (warp - 2)), step = (int)gridDim.x * 2;
      for (int r = who; r < lo + (args.rows - hi); r += step) {
        uint4* row = reinterpret_cast<uint4*>(static_cast<T*>(args.C) + (size_t)(r < lo ? r : hi + (r - lo)) * Nout);
        for (int c = lane; c < vecs; c += 32) row[c] = make_uint4(0u, 0u, 0u, 0u);
      }
    }
  } else {
    // ---------------------------------------------------------------- promotion and epilogue
    if (S::SPLIT_REGS) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(G8_REGS_MANY));
    const int q = warp & 3, g = (warp - 4) >> 2;  // quarter of the lanes; half of the tile's columns
    const int trow = cr * G8_XR + q * 32 + lane;
    const int n_blocks = (Nout + G8_BLOCK - 1) / G8_BLOCK;
    const uint32_t taddr = tmem + ((uint32_t)(q * 32) << 16) + g * (ACC / 2);
    // accumulator columns 32 c, ... of the thread: a quarter of the tile's first half, then of its second
    auto column_of = [](int c) { return c < ACC / 64 ? c * 32 : WR / 2 + (c - ACC / 64) * 32; };
    // first output column of the thread's quarter of the tile's first half
    auto col_of = [&](const Tile8& tile) { return tile.cb * tile_cols + g * (ACC / 2); };
    // Scales: every thread copies its row's, two lanes the weights' two, into slots of the warp's own,
    // G8_AHEAD k blocks before they are used (across tiles), asynchronously and without registers.
    float (*slots)[G8_SLOT] = s_scale[warp - 4];
    Tile8 ptile;
    int pt = unit, pkb = 0, pcursor = 0, ahead = 0;
    const float *px = nullptr, *pw = nullptr;
    auto enter = [&]() {  // the scales of tile pt
      ptile = locate_tile8<S::BM>(pt, pcursor, s_tile_start, s_begin, s_end);
      px = args.xscale + ptile.row0 + (trow < ptile.nvalid ? trow : 0);
      const int col = col_of(ptile);
      const int nb = swiglu ? (lane & 1) * n_blocks + min(col / G8_BLOCK, n_blocks - 1)
                            : min((col + (lane & 1) * (WR / 2)) / G8_BLOCK, n_blocks - 1);
      pw = args.wscale + ((size_t)ptile.e * (swiglu ? 2 : 1) * n_blocks + nb) * k_blocks;
    };
    auto prefetch = [&]() {
      if (pt < total_tiles) {
        float* slot = slots[ahead & (G8_SLOTS - 1)];
        cp_async_4(slot + lane, px);
        if (lane < 2) cp_async_4(slot + 32 + lane, pw);
        px += args.rows, ++pw;
        if (++pkb == k_blocks) {
          pkb = 0, pt += units;
          if (pt < total_tiles) enter();
        }
      }
      ++ahead;
      cp_async_commit();
    };
    if (pt < total_tiles) enter();
    for (int i = 0; i < G8_AHEAD; ++i) prefetch();
    int it = 0, cursor = 0;
    bool alive = true;
    for (int t = unit; t < total_tiles; t += units) {
      const Tile8 tile = locate_tile8<S::BM>(t, cursor, s_tile_start, s_begin, s_end);
      const bool busy = cr * G8_XR + q * 32 < tile.nvalid;  // the warp has rows of this tile
      const bool valid = trow < tile.nvalid;
      const int row = tile.row0 + trow, col = col_of(tile);
      uint64_t acc[ACC / 2];
#pragma unroll
      for (int i = 0; i < ACC / 2; ++i) acc[i] = 0;
      // Waits for the partial product of k block `it`. A warp that gave up goes on without waiting.
      auto open = [&]() {
        if (alive && !mbar_wait(&part_full[it & 1], (it >> 1) & 1, wait_ns)) {
          *status = DS_TIMEOUT_MMA;
          alive = false;
        }
        __syncwarp();
        tc_fence_after_sync();
      };
      // All of it is in registers: the buffer may be overwritten.
      auto close = [&]() {
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) {
          if (PAIR) arrive_leader(cluster_map(&part_empty[it & 1], 0));
          else mbar_arrive(&part_empty[it & 1]);
        }
      };
      if (!busy) {
        for (int kb = 0; kb < k_blocks; ++kb, ++it) {
          prefetch();
          open();
          close();
        }
        continue;
      }
      uint32_t v[2][32];
      open();
      tmem_ld_x32(taddr + (it & 1) * WR + column_of(0), v[0]);
#pragma unroll 1
      for (int kb = 0; kb < k_blocks; ++kb, ++it) {
        prefetch();
        cp_async_wait<G8_AHEAD>();
        __syncwarp();
        const float* slot = slots[it & (G8_SLOTS - 1)];
        const float x = slot[lane];
        const uint64_t f0 = twice(x * slot[32]), f1 = twice(x * slot[33]);
        const uint32_t from = taddr + (it & 1) * WR;
#pragma unroll
        for (int c = 0; c < ACC / 32; ++c) {
          tmem_ld_wait_x32(v[c & 1]);
          if (c + 1 < ACC / 32) {
            tmem_ld_x32(from + column_of(c + 1), v[(c + 1) & 1]);
          } else {  // the next block's first columns are on their way during the last multiply-adds
            close();
            if (kb + 1 < k_blocks) {
              ++it;
              open();
              tmem_ld_x32(taddr + (it & 1) * WR + column_of(0), v[0]);
              --it;
            }
          }
          const uint64_t f = c < ACC / 64 ? f0 : f1;
#pragma unroll
          for (int j = 0; j < 16; ++j) fma2(acc[c * 16 + j], v[c & 1][2 * j], v[c & 1][2 * j + 1], f);
        }
      }
      if (!alive || !valid) continue;
      T* dst = static_cast<T*>(args.C) + (size_t)row * Nout + col;
      const float s = args.scale ? Elem<T>::to_f(static_cast<const T*>(args.scale)[row]) : 1.f;
      const bool wide = (reinterpret_cast<uintptr_t>(dst) & 31) == 0;
      constexpr int VALUES = 16;
      auto store16 = [&](int c, const float (&f)[VALUES]) {  // columns col + c, ...
        uint32_t o[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const T lo = Elem<T>::from_f(f[2 * j]), hi = Elem<T>::from_f(f[2 * j + 1]);
          o[j] = (uint32_t) reinterpret_cast<const uint16_t&>(lo) | ((uint32_t) reinterpret_cast<const uint16_t&>(hi) << 16);
        }
        if (wide && col + c + 16 <= Nout) {
          st_global_32(dst + c, o);
        } else {
          if (col + c < Nout) *reinterpret_cast<uint4*>(dst + c) = make_uint4(o[0], o[1], o[2], o[3]);
          if (col + c + 8 < Nout) *reinterpret_cast<uint4*>(dst + c + 8) = make_uint4(o[4], o[5], o[6], o[7]);
        }
      };
      if (swiglu) {
#pragma unroll
        for (int c = 0; c < ACC / 2; c += VALUES) {
          float f[VALUES];
#pragma unroll
          for (int j = 0; j < VALUES / 2; ++j) {
            const float2 gate = both(acc[c / 2 + j]), up = both(acc[ACC / 4 + c / 2 + j]);
            f[2 * j] = swiglu32(gate.x, up.x);
            f[2 * j + 1] = swiglu32(gate.y, up.y);
          }
          store16(c, f);
        }
      } else {
#pragma unroll
        for (int c = 0; c < ACC; c += VALUES) {
          float f[VALUES];
#pragma unroll
          for (int j = 0; j < VALUES / 2; ++j) {
            const float2 a = both(acc[c / 2 + j]);
            f[2 * j] = a.x * s;
            f[2 * j + 1] = a.y * s;
          }
          store16(c < ACC / 2 ? c : WR / 2 + c - ACC / 2, f);
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
template <typename T, int WR, bool PAIR> static int units8(int sms, int* out) {
  static std::atomic<int> cached[MAX_DEVICES];
  int dev = 0;
  SY_CUDA(cudaGetDevice(&dev));
  int units = cached[dev].load(std::memory_order_acquire);
  if (!units) {
    auto kern = gemm8_kernel<T, WR, PAIR>;
    SY_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, G8_SMEM));
    if (Shape8<WR, PAIR>::SPLIT_REGS) {
      // the promoters' register request waits for ever if the block was launched with fewer
      cudaFuncAttributes attr;
      SY_CUDA(cudaFuncGetAttributes(&attr, kern));
      if (attr.numRegs < G8_REGS_LAUNCH)
        return fail(SY_ERR_CUDA, "grouped_gemm_fp8: built with %d registers per thread, needs %d", attr.numRegs, G8_REGS_LAUNCH);
    }
    if (PAIR) {
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(sms & ~1);
      cfg.blockDim = dim3(G8_THREADS);
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
      SY_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kern, G8_THREADS, G8_SMEM));
      units = per_sm >= 1 ? sms : 0;
    }
    if (units < 1) return fail(SY_ERR_CUDA, "grouped_gemm_fp8: no block of the kernel fits on this device");
    cached[dev].store(units, std::memory_order_release);
  }
  *out = units;
  return SY_OK;
}

template <typename T, int WR, bool PAIR>
static int launch8(Gemm8Args a, const void* x, const void* w, cudaStream_t stream) {
  using S = Shape8<WR, PAIR>;
  int sms = 0, units = 0;
  int rc = device_sm_count(&sms);
  if (rc != SY_OK) return rc;
  rc = units8<T, WR, PAIR>(sms, &units);
  if (rc != SY_OK) return rc;
  const uint64_t w_rows = (uint64_t)a.experts * (a.swiglu ? 2 : 1) * a.Nout;
  rc = tensor_map_2d(&a.wmap, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, w, w_rows, (uint64_t)a.K, S::WBOX, G8_BLOCK);
  if (rc != SY_OK) return rc;
  rc = tensor_map_2d(&a.xmap, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, x, (uint64_t)a.rows, (uint64_t)a.K, G8_XR, G8_BLOCK);
  if (rc != SY_OK) return rc;
  rc = tensor_map_2d(&a.xfew, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, x, (uint64_t)a.rows, (uint64_t)a.K, G8_XFEW, G8_BLOCK);
  if (rc != SY_OK) return rc;
  auto kern = gemm8_kernel<T, WR, PAIR>;
  if (PAIR) return launch_cluster_kernel(kern, 2, 2 * units, G8_THREADS, G8_SMEM, stream, "grouped_gemm_fp8 launch", a);
  return launch_kernel(kern, units, G8_THREADS, G8_SMEM, stream, "grouped_gemm_fp8 launch", a);
}

template <typename T> static int dispatch8(const Gemm8Args& a, int tile, const void* x, const void* w, cudaStream_t s) {
  return tile == 1 ? launch8<T, 128, false>(a, x, w, s)
         : tile == 2 ? launch8<T, 256, false>(a, x, w, s)
                     : launch8<T, 256, true>(a, x, w, s);
}

}  // namespace sy

extern "C" int sy_grouped_gemm_fp8(const void* x, const float* x_scale, const void* w, const float* w_scale,
                                   const int32_t* offsets, int n_experts, int rows, int n_out, int k_dim, int swiglu,
                                   const void* scale, void* C, int dtype, int tile, void* stream) {
  using namespace sy;
  SY_REQUIRE(rows >= 0 && n_experts >= 1 && n_experts <= G8_MAX_E, "grouped_gemm_fp8: 1..%d experts (got %d)", G8_MAX_E,
             n_experts);
  SY_REQUIRE(k_dim > 0 && k_dim % 16 == 0, "grouped_gemm_fp8: k_dim must be a multiple of 16 (got %d)", k_dim);
  SY_REQUIRE(n_out > 0 && n_out % 8 == 0, "grouped_gemm_fp8: n_out must be a multiple of 8 (got %d)", n_out);
  SY_REQUIRE(!(swiglu && scale), "grouped_gemm_fp8: swiglu and scale are separate epilogues");
  SY_REQUIRE(dtype == SY_DTYPE_F16 || dtype == SY_DTYPE_BF16, "grouped_gemm_fp8: dtype must be f16 or bf16");
  SY_REQUIRE(tile >= 0 && tile <= 3, "grouped_gemm_fp8: tile 0..3 (got %d)", tile);
  SY_REQUIRE((int64_t)n_experts * 2 * n_out <= 0x7fffffff, "grouped_gemm_fp8: more than 2^31 weight rows");
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
  a.experts = n_experts;
  a.rows = rows;
  a.Nout = n_out;
  a.K = k_dim;
  a.swiglu = swiglu != 0;
  a.status = device_status_word();
  if (!a.status) return SY_ERR_CUDA;
  a.wait_ns = wait_limit_ns();
  if (tile == 0) tile = rows <= 64LL * n_experts ? 1 : rows < 256LL * n_experts ? 2 : 3;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == SY_DTYPE_F16 ? dispatch8<__half>(a, tile, x, w, s) : dispatch8<__nv_bfloat16>(a, tile, x, w, s);
}
