// 16- or 32-bit values to 8-bit floats (e4m3) with a float32 scale for each block: 1 x 128 for
// activations, 128 x 128 for weights.
//
// With m the largest magnitude of a block (at least 2^-96, so that a block of zeros has a finite
// scale) the stored values are scale = m / 448 and q = round(448 x / m), both from a correctly
// rounded division. 448 = 7 * 64, so 448 x is exact for 16-bit x, and a quotient that lies midway
// between two e4m3 values comes out exactly midway and rounds to even; a multiplication by 1/m
// would send about one value in a few thousand to the other neighbour. Both sides of the division
// carry a factor 2^-16 so that no finite float32 overflows. A NaN makes its block's scale NaN, an
// infinity makes it infinite: the products that use the block are then NaN, as in the input.
#include <cuda_fp8.h>

#include "common.cuh"
#include "rows.cuh"

namespace sy {

constexpr int Q8_BLOCK = 128;
constexpr int Q8_THREADS = 256;
constexpr float Q8_TOP = 448.f;

// 8 consecutive elements as floats (16 or 32 bytes; p is 16-byte aligned).
template <typename T> struct Eight {
  uint4 v;
  __device__ __forceinline__ void load(const T* p) { v = __ldg(reinterpret_cast<const uint4*>(p)); }
  __device__ __forceinline__ void zero() { v = make_uint4(0u, 0u, 0u, 0u); }
  __device__ __forceinline__ void get(float (&f)[8]) const { unpack8<T>(v, f); }
};
template <> struct Eight<float> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* p) {
    a = __ldg(reinterpret_cast<const float4*>(p));
    b = __ldg(reinterpret_cast<const float4*>(p) + 1);
  }
  __device__ __forceinline__ void zero() { a = b = make_float4(0.f, 0.f, 0.f, 0.f); }
  __device__ __forceinline__ void get(float (&f)[8]) const {
    f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
  }
};

// Largest magnitude as a bit pattern: orders like the magnitude, infinities above every finite
// value and NaNs above those, so that a maximum of integers keeps them.
template <typename T> __device__ __forceinline__ uint32_t magnitude8(const Eight<T>& e) {
  float f[8];
  e.get(f);
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(f[i]) & 0x7fffffffu);
  return m;
}

struct BlockScale {
  float scale, den;  // m / 448, and m * 2^-16
  __device__ __forceinline__ explicit BlockScale(uint32_t magnitude) {
    const float m = __uint_as_float(max(magnitude, 0x0f800000u));  // 2^-96
    scale = m / Q8_TOP;
    den = m * 0x1p-16f;
  }
};

template <typename T> __device__ __forceinline__ uint2 quantize8(const Eight<T>& e, float den) {
  float f[8];
  e.get(f);
  uint32_t r[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    r[i] = __nv_cvt_float2_to_fp8x2(make_float2(f[2 * i] * (Q8_TOP * 0x1p-16f) / den, f[2 * i + 1] * (Q8_TOP * 0x1p-16f) / den),
                                    __NV_SATFINITE, __NV_E4M3);
  return make_uint2(r[0] | (r[1] << 16), r[2] | (r[3] << 16));
}

// A token's row is quantised once and stored at its k places in expert order (pos_of), or at its
// own place (pos_of absent, k = 1). Sixteen lanes share a block of 128 columns, eight each.
// Scales are [blocks][rows]: what a tile of the product reads for one block is contiguous.
template <typename T>
__global__ void __launch_bounds__(Q8_THREADS)
quantize_rows_kernel(const T* __restrict__ x, const int* __restrict__ pos_of, const int* __restrict__ rows_used,
                     int n_tokens, int k, int H, int lanes, uint8_t* __restrict__ q, float* __restrict__ scale) {
  pdl_launch_dependents();
  pdl_wait();
  const int t = blockIdx.x * (Q8_THREADS / lanes) + threadIdx.x / lanes, lane = threadIdx.x % lanes;
  if (t >= n_tokens) return;  // whole warps: lanes is a multiple of 32
  const int m = n_tokens * k, blocks = (H + Q8_BLOCK - 1) / Q8_BLOCK;
  int pos[ROWS_MAX_K];
#pragma unroll
  for (int j = 0; j < ROWS_MAX_K; ++j) pos[j] = j >= k ? -1 : pos_of ? pos_of[(size_t)t * k + j] : t;
  for (int c0 = 0; c0 < blocks * 16; c0 += lanes) {
    const int c = c0 + lane, col = c * 8;
    Eight<T> e;
    if (col < H) e.load(x + (size_t)t * H + col);
    else e.zero();
    uint32_t mag = magnitude8<T>(e);
#pragma unroll
    for (int o = 8; o; o >>= 1) mag = max(mag, __shfl_xor_sync(0xffffffffu, mag, o));
    const BlockScale s(mag);
    const uint2 v = quantize8<T>(e, s.den);
#pragma unroll
    for (int j = 0; j < ROWS_MAX_K; ++j)
      if (pos[j] >= 0 && pos[j] < m) {
        if (col < H) *reinterpret_cast<uint2*>(q + (size_t)pos[j] * H + col) = v;
        if ((c & 15) == 0 && col < H) scale[(size_t)(c >> 4) * m + pos[j]] = s.scale;
      }
  }
  if (rows_used)
    for (int r = max(t * k, *rows_used); r < (t + 1) * k; ++r) {  // rows without a choice
      for (int c = lane; c * 8 < H; c += lanes) *reinterpret_cast<uint2*>(q + (size_t)r * H + c * 8) = make_uint2(0u, 0u);
      for (int b = lane; b < blocks; b += lanes) scale[(size_t)b * m + r] = 0.f;
    }
}

// One block of threads per 128 x 128 block of a weight matrix, which stays in registers between
// the maximum and the division: every value crosses memory once.
template <typename T>
__global__ void __launch_bounds__(Q8_THREADS)
quantize_weight_kernel(const T* __restrict__ w, int N, int K, uint8_t* __restrict__ q, float* __restrict__ scale) {
  constexpr int STEP = Q8_THREADS / 16, EACH = Q8_BLOCK / STEP;
  __shared__ uint32_t s_mag[Q8_THREADS / 32];
  pdl_launch_dependents();
  pdl_wait();
  const int kb = blockIdx.x, nb = blockIdx.y;
  const size_t mat = blockIdx.z;
  const int col = kb * Q8_BLOCK + (threadIdx.x & 15) * 8, row0 = nb * Q8_BLOCK + (threadIdx.x >> 4);
  Eight<T> e[EACH];
  uint32_t mag = 0;
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int row = row0 + i * STEP;
    if (row < N && col < K) e[i].load(w + (mat * N + row) * K + col);
    else e[i].zero();
  }
#pragma unroll
  for (int i = 0; i < EACH; ++i) mag = max(mag, magnitude8<T>(e[i]));
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
    if (row < N && col < K) *reinterpret_cast<uint2*>(q + (mat * N + row) * K + col) = quantize8<T>(e[i], s.den);
  }
}

template <typename T>
static int quantize_rows_launch(const void* x, const int32_t* pos_of, const int32_t* used, int n_tokens, int k, int H,
                                void* q, float* scale, cudaStream_t stream) {
  int lanes = 32;
  while (lanes * 8 < H && lanes < Q8_THREADS) lanes *= 2;
  const int tokens = Q8_THREADS / lanes;
  return launch_kernel(quantize_rows_kernel<T>, (n_tokens + tokens - 1) / tokens, Q8_THREADS, 0, stream,
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
  SY_REQUIRE(n_tokens <= 0x7fffffff / top_k, "quantize_rows: more than 2^31 rows");
  SY_REQUIRE(hidden > 0 && hidden % 16 == 0, "quantize_rows: hidden must be a multiple of 16 (got %d)", hidden);
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
  SY_REQUIRE(k_dim > 0 && k_dim % 16 == 0, "quantize_weight: k_dim must be a multiple of 16 (got %d)", k_dim);
  if (n_mats == 0) return SY_OK;
  SY_REQUIRE(w && q && scale, "quantize_weight: null pointer");
  SY_REQUIRE((uintptr_t)w % 16 == 0 && (uintptr_t)q % 16 == 0, "quantize_weight: w and q must be 16-byte aligned");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == SY_DTYPE_F16    ? quantize_weight_launch<__half>(w, n_mats, n_rows, k_dim, q, scale, s)
         : dtype == SY_DTYPE_BF16 ? quantize_weight_launch<__nv_bfloat16>(w, n_mats, n_rows, k_dim, q, scale, s)
                                  : quantize_weight_launch<float>(w, n_mats, n_rows, k_dim, q, scale, s);
}
