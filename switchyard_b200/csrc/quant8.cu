// 16- or 32-bit values to 8-bit floats (e4m3) with a float32 scale for each block: 1 x 128 for
// activations, 128 x 128 for weights.
//
// With m the largest magnitude of a block (at least 2^-96, so that a block of zeros has a finite
// scale) the stored values are scale = m / 448 and q = e4m3(448 x / m), 448 x and the quotient rounded
// to float32, ties to even throughout. 448 = 7 * 64, so 448 x is exact for 16-bit x, a quotient
// that lies midway between two e4m3 values comes out exactly midway, and any other is further
// from there than its rounding: q is the value nearest to the exact quotient. Of float32 x a quotient within
// two roundings (2^-23) of a midpoint may go to either neighbour. One product
// with 1/m sends about one value in a thousand of bf16 data to the other neighbour.
// A division per value is what the kernels would spend most of their time on (245 us for the
// benchmark's gate and up projections, with two thirds of the issue slots busy). So the value is
// bracketed by two products with 448/m, one a little small, one a little large (2^-21: more than
// the roundings between a product and the quotient can make, four of 2^-24, five of float32 x). Rounding is monotone: where
// both give the same e4m3 value it is the quotient's, and only where they differ, around the
// midpoints, the division decides.
// A NaN makes its block's scale NaN, an infinity makes it infinite: the products that use the block
// are then NaN, as in the input.
#include <cuda_fp8.h>

#include "common.cuh"
#include "rows.cuh"

namespace sy {

constexpr int Q8_BLOCK = 128;
constexpr int Q8_THREADS = 256;         // weights
constexpr int Q8_ROW_THREADS = 128;     // rows: small blocks that come and go (256: 36 us where this took 32, 8192 tokens)
constexpr int Q8_LANES = Q8_BLOCK / 16;  // threads that share a row of a block, 16 columns each
constexpr float Q8_TOP = 448.f;

// 16 consecutive elements (32 or 64 bytes from a 16-byte aligned address), as pairs of floats.
template <typename T> struct Sixteen {
  uint4 v[2];
  __device__ __forceinline__ void load(const T* p) {
    v[0] = __ldg(reinterpret_cast<const uint4*>(p));
    v[1] = __ldg(reinterpret_cast<const uint4*>(p) + 1);
  }
  __device__ __forceinline__ void zero() { v[0] = v[1] = make_uint4(0u, 0u, 0u, 0u); }
  __device__ __forceinline__ uint32_t word(int i) const {
    const uint4& q = v[i >> 2];
    return (i & 3) == 0 ? q.x : (i & 3) == 1 ? q.y : (i & 3) == 2 ? q.z : q.w;
  }
  __device__ __forceinline__ float2 pair(int i) const { return Elem<T>::pair_to_f2(word(i)); }
  // The largest magnitude's float32 bits. Bit patterns without their sign order like magnitudes,
  // infinities above every finite value and NaNs above those.
  __device__ __forceinline__ uint32_t magnitude() const {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = __vmaxu2(m, word(i) & 0x7fff7fffu);
    const float2 f = Elem<T>::pair_to_f2(m);
    return max(__float_as_uint(f.x), __float_as_uint(f.y));
  }
};
template <> struct Sixteen<float> {
  float4 v[4];
  __device__ __forceinline__ void load(const float* p) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __ldg(reinterpret_cast<const float4*>(p) + i);
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  __device__ __forceinline__ float2 pair(int i) const {
    return i & 1 ? make_float2(v[i >> 1].z, v[i >> 1].w) : make_float2(v[i >> 1].x, v[i >> 1].y);
  }
  __device__ __forceinline__ uint32_t magnitude() const {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 f = pair(i);
      m = max(m, max(__float_as_uint(f.x) & 0x7fffffffu, __float_as_uint(f.y) & 0x7fffffffu));
    }
    return m;
  }
};

struct BlockScale {
  float scale, den, low, high;  // m / 448, m * 2^-16, and 448 / m bracketed
  __device__ __forceinline__ explicit BlockScale(uint32_t magnitude) {
    const float m = __uint_as_float(max(magnitude, 0x0f800000u));  // 2^-96
    scale = m / Q8_TOP;
    den = m * 0x1p-16f;
    const float inv = Q8_TOP / m;
    low = inv * (1.f - 0x1p-21f), high = inv * (1.f + 0x1p-21f);
  }
};

__device__ __forceinline__ uint32_t e4m3_pair(float a, float b) {
  return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}

// x * f for two float32 values at once.
__device__ __forceinline__ float2 scaled(float2 x, float f) {
  float2 r;
  asm("{\n\t.reg .b64 a, b;\n\t"
      "mov.b64 a, {%2, %3};\n\t"
      "mov.b64 b, {%4, %4};\n\t"
      "mul.rn.f32x2 a, a, b;\n\t"
      "mov.b64 {%0, %1}, a;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(x.x), "f"(x.y), "f"(f));
  return r;
}

template <typename T> __device__ __forceinline__ uint4 quantize16(const Sixteen<T>& e, const BlockScale& s) {
  uint32_t r[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2 x = e.pair(i), l = scaled(x, s.low), h = scaled(x, s.high);
    r[i] = e4m3_pair(l.x, l.y);
    if (r[i] != e4m3_pair(h.x, h.y))  // (both sides carry 2^-16: no finite value overflows)
      r[i] = e4m3_pair(x.x * (Q8_TOP * 0x1p-16f) / s.den, x.y * (Q8_TOP * 0x1p-16f) / s.den);
  }
  return make_uint4(r[0] | (r[1] << 16), r[2] | (r[3] << 16), r[4] | (r[5] << 16), r[6] | (r[7] << 16));
}

// A token's row is quantised once and stored at its k places in expert order (pos_of), or at its
// own place (pos_of absent, k = 1). Bounded by the k stores: 8192 tokens, top-8, 2048 columns of bf16, 172 MB
// in 33 us (5.2 TB/s; 34 us a call of a loop), of which the scales' scattered four bytes are 3 us.
// Scales are [blocks][rows]: what a tile of the product reads for one block is contiguous.
template <typename T>
__global__ void __launch_bounds__(Q8_ROW_THREADS, 10)
quantize_rows_kernel(const T* __restrict__ x, const int* __restrict__ pos_of, const int* __restrict__ rows_used,
                     int n_tokens, int k, int H, int lanes, uint8_t* __restrict__ q, float* __restrict__ scale) {
  pdl_launch_dependents();
  pdl_wait();
  const int t = blockIdx.x * (Q8_ROW_THREADS / lanes) + threadIdx.x / lanes, lane = threadIdx.x % lanes;
  if (t >= n_tokens) return;  // whole warps: lanes is a multiple of 32
  const int m = n_tokens * k, blocks = (H + Q8_BLOCK - 1) / Q8_BLOCK;
  int pos[ROWS_MAX_K];
#pragma unroll
  for (int j = 0; j < ROWS_MAX_K; ++j) pos[j] = j >= k ? -1 : pos_of ? pos_of[(size_t)t * k + j] : t;
  for (int c0 = 0; c0 < blocks * Q8_LANES; c0 += lanes) {
    const int c = c0 + lane, col = c * 16;
    Sixteen<T> e;
    if (col < H) e.load(x + (size_t)t * H + col);
    else e.zero();
    uint32_t mag = e.magnitude();
#pragma unroll
    for (int o = Q8_LANES / 2; o; o >>= 1) mag = max(mag, __shfl_xor_sync(0xffffffffu, mag, o));
    const BlockScale s(mag);
    const uint4 v = quantize16<T>(e, s);
    if (col < H) {
#pragma unroll
      for (int j = 0; j < ROWS_MAX_K; ++j)
        if (pos[j] >= 0 && pos[j] < m) {
          *reinterpret_cast<uint4*>(q + (size_t)pos[j] * H + col) = v;
          if (c % Q8_LANES == 0) scale[(size_t)(c / Q8_LANES) * m + pos[j]] = s.scale;
        }
    }
  }
  if (rows_used)
    for (int r = max(t * k, *rows_used); r < (t + 1) * k; ++r) {  // rows without a choice
      for (int c = lane; c * 16 < H; c += lanes) *reinterpret_cast<uint4*>(q + (size_t)r * H + c * 16) = make_uint4(0u, 0u, 0u, 0u);
      for (int b = lane; b < blocks; b += lanes) scale[(size_t)b * m + r] = 0.f;
    }
}

// One block of threads per 128 x 128 block of a weight matrix, which stays in registers between
// the maximum and the division: every value crosses memory once (805 MB of bf16 in 140 us in a burst, 5.8 TB/s;
// 151 a call of a loop; issue slots two thirds busy). 512 threads a block: 174 us, 128: 197.
template <typename T>
__global__ void __launch_bounds__(Q8_THREADS)
quantize_weight_kernel(const T* __restrict__ w, int N, int K, uint8_t* __restrict__ q, float* __restrict__ scale) {
  constexpr int STEP = Q8_THREADS / Q8_LANES, EACH = Q8_BLOCK / STEP;
  __shared__ uint32_t s_mag[Q8_THREADS / 32];
  pdl_launch_dependents();
  pdl_wait();
  const int kb = blockIdx.x, nb = blockIdx.y;
  const size_t mat = blockIdx.z;
  const int col = kb * Q8_BLOCK + (threadIdx.x % Q8_LANES) * 16, row0 = nb * Q8_BLOCK + threadIdx.x / Q8_LANES;
  Sixteen<T> e[EACH];
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int row = row0 + i * STEP;
    if (row < N && col < K) e[i].load(w + (mat * N + row) * K + col);
    else e[i].zero();
  }
  uint32_t mag = 0;
#pragma unroll
  for (int i = 0; i < EACH; ++i) mag = max(mag, e[i].magnitude());
  mag = __reduce_max_sync(0xffffffffu, mag);
  if ((threadIdx.x & 31) == 0) s_mag[threadIdx.x >> 5] = mag;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < Q8_THREADS / 32; ++i) mag = max(mag, s_mag[i]);
  const BlockScale s(mag);
  if (threadIdx.x == 0) scale[(mat * gridDim.y + nb) * gridDim.x + kb] = s.scale;
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int row = row0 + i * STEP;
    if (row < N && col < K) *reinterpret_cast<uint4*>(q + (mat * N + row) * K + col) = quantize16<T>(e[i], s);
  }
}

template <typename T>
static int quantize_rows_launch(const void* x, const int32_t* pos_of, const int32_t* used, int n_tokens, int k, int H,
                                void* q, float* scale, cudaStream_t stream) {
  int lanes = 32;
  while (lanes * 16 < H && lanes < Q8_ROW_THREADS) lanes *= 2;
  const int tokens = Q8_ROW_THREADS / lanes;
  return launch_kernel(quantize_rows_kernel<T>, (n_tokens + tokens - 1) / tokens, Q8_ROW_THREADS, 0, stream,
                       "quantize_rows launch", static_cast<const T*>(x), pos_of, used, n_tokens, k, H, lanes,
                       static_cast<uint8_t*>(q), scale);
}

template <typename T>
static int quantize_weight_launch(const void* w, int mats, int N, int K, void* q, float* scale, cudaStream_t stream) {
  const dim3 grid((K + Q8_BLOCK - 1) / Q8_BLOCK, (N + Q8_BLOCK - 1) / Q8_BLOCK, mats);
  return launch_kernel(quantize_weight_kernel<T>, grid, Q8_THREADS, 0, stream, "quantize_weight launch",
                       static_cast<const T*>(w), N, K, static_cast<uint8_t*>(q), scale);
}

}  // namespace sy

extern "C" int sy_quantize_rows(const void* x, const int32_t* pos_of, const int32_t* offsets, int n_tokens, int top_k,
                                int n_experts, int hidden, int dtype, void* q, float* scale, void* stream) {
  using namespace sy;
  SY_REQUIRE(dtype == SY_DTYPE_F16 || dtype == SY_DTYPE_BF16 || dtype == SY_DTYPE_F32,
             "quantize_rows: dtype must be f16, bf16 or f32");
  SY_REQUIRE(n_tokens >= 0 && top_k >= 1 && top_k <= ROWS_MAX_K, "quantize_rows: top_k must be 1..%d (got %d)", ROWS_MAX_K,
             top_k);
  SY_REQUIRE(n_tokens <= ROWS_MOST / top_k, "quantize_rows: more than 2^31 - 256 rows");
  SY_REQUIRE(hidden > 0 && hidden <= WIDTH_MOST && hidden % 16 == 0,
             "quantize_rows: hidden must be a multiple of 16, at most %d (got %d)", WIDTH_MOST, hidden);
  if (n_tokens == 0) return SY_OK;
  SY_REQUIRE(pos_of || top_k == 1, "quantize_rows: rows kept in place have one place each");
  SY_REQUIRE(!pos_of || n_experts >= 1, "quantize_rows: at least one expert (got %d)", n_experts);
  SY_REQUIRE(x && q && scale && (offsets || !pos_of), "quantize_rows: null pointer");
  SY_REQUIRE((uintptr_t)x % 16 == 0 && (uintptr_t)q % 16 == 0, "quantize_rows: x and q must be 16-byte aligned");
  const int32_t* used = pos_of ? offsets + n_experts : nullptr;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == SY_DTYPE_F16    ? quantize_rows_launch<__half>(x, pos_of, used, n_tokens, top_k, hidden, q, scale, s)
         : dtype == SY_DTYPE_BF16 ? quantize_rows_launch<__nv_bfloat16>(x, pos_of, used, n_tokens, top_k, hidden, q, scale, s)
                                  : quantize_rows_launch<float>(x, pos_of, used, n_tokens, top_k, hidden, q, scale, s);
}

extern "C" int sy_quantize_weight(const void* w, int n_mats, int n_rows, int k_dim, int dtype, void* q, float* scale,
                                  void* stream) {
  using namespace sy;
  SY_REQUIRE(dtype == SY_DTYPE_F16 || dtype == SY_DTYPE_BF16 || dtype == SY_DTYPE_F32,
             "quantize_weight: dtype must be f16, bf16 or f32");
  SY_REQUIRE(n_mats >= 0 && n_mats <= 65535, "quantize_weight: at most 65535 matrices (got %d)", n_mats);
  SY_REQUIRE(n_rows > 0 && n_rows <= 65535 * Q8_BLOCK, "quantize_weight: 1..%d rows (got %d)", 65535 * Q8_BLOCK, n_rows);
  SY_REQUIRE(k_dim > 0 && k_dim <= WIDTH_MOST && k_dim % 16 == 0,
             "quantize_weight: k_dim must be a multiple of 16, at most %d (got %d)", WIDTH_MOST, k_dim);
  if (n_mats == 0) return SY_OK;
  SY_REQUIRE(w && q && scale, "quantize_weight: null pointer");
  SY_REQUIRE((uintptr_t)w % 16 == 0 && (uintptr_t)q % 16 == 0, "quantize_weight: w and q must be 16-byte aligned");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == SY_DTYPE_F16    ? quantize_weight_launch<__half>(w, n_mats, n_rows, k_dim, q, scale, s)
         : dtype == SY_DTYPE_BF16 ? quantize_weight_launch<__nv_bfloat16>(w, n_mats, n_rows, k_dim, q, scale, s)
                                  : quantize_weight_launch<float>(w, n_mats, n_rows, k_dim, q, scale, s);
}
