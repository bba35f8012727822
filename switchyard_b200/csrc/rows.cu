// Token rows into expert order and back, with the gradients of both.
//
//   permute_rows        x[pos_of[t, j], :] = h[t, :]
//   unpermute_rows      out[t, :] = sum_j w[t, j] * y[pos_of[t, j], :]     (w absent: plain sum)
//   unpermute_rows_grad dy[pos_of[t, j], :] = w[t, j] * dout[t, :],  dw[t, j] = <dout[t, :], y[pos_of[t, j], :]>
//
// The gradient of permute_rows is unpermute_rows without weights. Everything is laid out by token,
// not by sorted row: a token's k rows are then read or written by the threads that hold its own
// row, so h, out and dout cross memory once and not k times.
#include "common.cuh"
#include "rows.cuh"

namespace sy {

constexpr int ROWS_THREADS = 128;  // small blocks that come and go: 256 took 7 % longer for the gradient

// Which token a thread works on, and where in its row: `lanes` threads (a multiple of 32) share a
// token, ROWS_THREADS / lanes tokens share a block.
struct RowSplit {
  int lanes, tokens;
};
static RowSplit row_split(int vecs) {
  RowSplit s;
  s.lanes = 32;
  while (s.lanes < vecs && s.lanes < ROWS_THREADS) s.lanes *= 2;
  s.tokens = ROWS_THREADS / s.lanes;
  return s;
}

// Bounded by the k stores per load: 8192 tokens, top-8, 2048 columns of bf16, 302 MB in 50 us (6.0 TB/s,
// 0.92 of a copy's rate). Rows no choice was given (from offsets[n_experts] on, when the
// sort skipped invalid expert ids) are set to zero.
__global__ void __launch_bounds__(ROWS_THREADS)
permute_rows_kernel(const uint4* __restrict__ h, const int* __restrict__ pos_of, const int* __restrict__ rows_used,
                    int n_tokens, int k, int vecs, int lanes, uint4* __restrict__ x) {
  pdl_launch_dependents();
  pdl_wait();
  const int t = blockIdx.x * (ROWS_THREADS / lanes) + threadIdx.x / lanes, lane = threadIdx.x % lanes;
  if (t >= n_tokens) return;
  const int m = n_tokens * k, used = *rows_used;
  int pos[ROWS_MAX_K];
#pragma unroll
  for (int j = 0; j < ROWS_MAX_K; ++j) pos[j] = j < k ? pos_of[(size_t)t * k + j] : -1;
  for (int c = lane; c < vecs; c += lanes) {
    const uint4 v = __ldg(h + (size_t)t * vecs + c);
#pragma unroll
    for (int j = 0; j < ROWS_MAX_K; ++j)
      if (pos[j] >= 0 && pos[j] < m) x[(size_t)pos[j] * vecs + c] = v;
  }
  for (int r = max(t * k, used); r < (t + 1) * k; ++r)
    for (int c = lane; c < vecs; c += lanes) x[(size_t)r * vecs + c] = make_uint4(0u, 0u, 0u, 0u);
}

// A token's rows are added in ascending sorted row, which is ascending expert id, ties by slot:
// combine's order. float32 sum, one rounding. Bounded by reading the rows: the same 302 MB in 46-48 us.
template <typename T, typename W>
__global__ void __launch_bounds__(ROWS_THREADS)
unpermute_rows_kernel(const T* __restrict__ y, const W* __restrict__ w, const int* __restrict__ pos_of, int n_tokens,
                      int k, int vecs, int lanes, T* __restrict__ out) {
  constexpr int N = RowVec<T>::N;
  __shared__ int s_pos[ROWS_THREADS / 32][ROWS_MAX_K];
  __shared__ float s_w[ROWS_THREADS / 32][ROWS_MAX_K];
  pdl_launch_dependents();
  pdl_wait();
  const int slot = threadIdx.x / lanes, lane = threadIdx.x % lanes;
  const int t = blockIdx.x * (ROWS_THREADS / lanes) + slot;
  const int m = n_tokens * k;
  if (t < n_tokens && lane < k) {
    const int mine = pos_of[(size_t)t * k + lane];
    int rank = 0;
    for (int j = 0; j < k; ++j) {
      const int other = pos_of[(size_t)t * k + j];
      rank += other < mine || (other == mine && j < lane);
    }
    s_pos[slot][rank] = mine >= 0 && mine < m ? mine : -1;
    s_w[slot][rank] = w ? to_float(w[(size_t)t * k + lane]) : 1.f;
  }
  __syncthreads();
  if (t >= n_tokens) return;
  for (int c = lane; c < vecs; c += lanes) {
    uint4 v[ROWS_MAX_K];
#pragma unroll
    for (int j = 0; j < ROWS_MAX_K; ++j)
      if (j < k && s_pos[slot][j] >= 0) v[j] = __ldg(reinterpret_cast<const uint4*>(y) + (size_t)s_pos[slot][j] * vecs + c);
    float acc[N];
#pragma unroll
    for (int q = 0; q < N; ++q) acc[q] = 0.f;
#pragma unroll
    for (int j = 0; j < ROWS_MAX_K; ++j)
      if (j < k && s_pos[slot][j] >= 0) {
        float f[N];
        RowVec<T>::unpack(v[j], f);
        const float wj = s_w[slot][j];
#pragma unroll
        for (int q = 0; q < N; ++q) acc[q] = fmaf(wj, f[q], acc[q]);
      }
    reinterpret_cast<uint4*>(out)[(size_t)t * vecs + c] = RowVec<T>::pack(acc);
  }
}

// dy and dw in one pass over dout and y (either may be absent). The dot products are summed in
// float32 over a thread's columns, then over the lanes, then over the warps of the token, always
// in the same order. Bounded by HBM: 571 MB in 89.3 us (6.4 TB/s, 0.98 of a copy's rate); with all eight
// rows' loads in flight and the places in registers (110 of them) two blocks of 256 fitted an SM: 135 us.
template <typename T, typename W>
__global__ void __launch_bounds__(ROWS_THREADS, 8)
unpermute_rows_grad_kernel(const T* __restrict__ dout, const T* __restrict__ y, const W* __restrict__ w,
                           const int* __restrict__ pos_of, const int* __restrict__ rows_used, int n_tokens, int k,
                           int vecs, int lanes, T* __restrict__ dy, W* __restrict__ dw) {
  constexpr int N = RowVec<T>::N, AT_ONCE = 4;  // rows whose loads are in flight together
  __shared__ int s_pos[ROWS_THREADS / 32][ROWS_MAX_K];
  __shared__ float s_w[ROWS_THREADS / 32][ROWS_MAX_K];
  __shared__ float s_dot[ROWS_THREADS / 32][ROWS_MAX_K];
  pdl_launch_dependents();
  pdl_wait();
  const int slot = threadIdx.x / lanes, lane = threadIdx.x % lanes;
  const int t = blockIdx.x * (ROWS_THREADS / lanes) + slot;
  const int m = n_tokens * k;
  if (lane < ROWS_MAX_K) {
    int p = -1;
    float f = 1.f;
    if (t < n_tokens && lane < k) {
      p = pos_of[(size_t)t * k + lane];
      if (p >= m) p = -1;
      if (w) f = to_float(w[(size_t)t * k + lane]);
    }
    s_pos[slot][lane] = p;
    s_w[slot][lane] = f;
  }
  __syncthreads();
  float dot[ROWS_MAX_K];
#pragma unroll
  for (int j = 0; j < ROWS_MAX_K; ++j) dot[j] = 0.f;
  if (t < n_tokens) {
    for (int c = lane; c < vecs; c += lanes) {
      const uint4 d = __ldg(reinterpret_cast<const uint4*>(dout) + (size_t)t * vecs + c);
#pragma unroll
      for (int j0 = 0; j0 < ROWS_MAX_K; j0 += AT_ONCE) {
        if (j0 >= k) break;
        int pos[AT_ONCE];
        uint4 v[AT_ONCE];
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
          pos[i] = s_pos[slot][j0 + i];
          if (dw && pos[i] >= 0) v[i] = __ldg(reinterpret_cast<const uint4*>(y) + (size_t)pos[i] * vecs + c);
        }
        float g[N];
        RowVec<T>::unpack(d, g);
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
          if (pos[i] < 0) continue;
          if (dy) {
            const float wj = s_w[slot][j0 + i];
            float r[N];
#pragma unroll
            for (int q = 0; q < N; ++q) r[q] = wj * g[q];
            reinterpret_cast<uint4*>(dy)[(size_t)pos[i] * vecs + c] = RowVec<T>::pack(r);
          }
          if (dw) {
            float f[N];
            RowVec<T>::unpack(v[i], f);
#pragma unroll
            for (int q = 0; q < N; ++q) dot[j0 + i] = fmaf(g[q], f[q], dot[j0 + i]);
          }
        }
      }
    }
    if (dy) {
      const int used = *rows_used;
      for (int r = max(t * k, used); r < (t + 1) * k; ++r)
        for (int c = lane; c < vecs; c += lanes)
          reinterpret_cast<uint4*>(dy)[(size_t)r * vecs + c] = make_uint4(0u, 0u, 0u, 0u);
    }
  }
  if (!dw) return;
#pragma unroll
  for (int j = 0; j < ROWS_MAX_K; ++j)
    if (j < k) {
#pragma unroll
      for (int o = 16; o; o >>= 1) dot[j] += __shfl_xor_sync(0xffffffffu, dot[j], o);
      if ((threadIdx.x & 31) == 0) s_dot[threadIdx.x >> 5][j] = dot[j];
    }
  __syncthreads();
  if (t < n_tokens && lane < k) {
    const int first = slot * (lanes >> 5);
    float sum = s_dot[first][lane];
    for (int i = 1; i < lanes >> 5; ++i) sum += s_dot[first + i][lane];
    dw[(size_t)t * k + lane] = from_float<W>(sum);
  }
}

static int rows_check(const char* name, int n_tokens, int top_k, int hidden, int dtype, int* vecs) {
  SY_REQUIRE(dtype == SY_DTYPE_F16 || dtype == SY_DTYPE_BF16 || dtype == SY_DTYPE_F32, "%s: dtype must be f16, bf16 or f32",
             name);
  SY_REQUIRE(n_tokens >= 0 && top_k >= 1 && top_k <= ROWS_MAX_K, "%s: top_k must be 1..%d (got %d)", name, ROWS_MAX_K, top_k);
  SY_REQUIRE(n_tokens <= ROWS_MOST / top_k, "%s: more than 2^31 - 256 rows", name);
  const int per_vec = dtype == SY_DTYPE_F32 ? 4 : 8;
  SY_REQUIRE(hidden > 0 && hidden <= WIDTH_MOST && hidden % per_vec == 0,
             "%s: hidden must be a multiple of %d in this type, at most %d (got %d)", name, per_vec, WIDTH_MOST, hidden);
  *vecs = hidden / per_vec;
  return SY_OK;
}

static bool aligned16(const void* p) { return (uintptr_t)p % 16 == 0; }

template <typename T, typename W>
static int unpermute_launch(const void* y, const void* w, const int32_t* pos_of, int n_tokens, int k, int vecs, void* out,
                            cudaStream_t stream) {
  const RowSplit s = row_split(vecs);
  return launch_kernel(unpermute_rows_kernel<T, W>, (n_tokens + s.tokens - 1) / s.tokens, ROWS_THREADS, 0, stream,
                       "unpermute_rows launch", static_cast<const T*>(y), static_cast<const W*>(w), pos_of, n_tokens, k, vecs,
                       s.lanes, static_cast<T*>(out));
}

template <typename T, typename W>
static int grad_launch(const void* dout, const void* y, const void* w, const int32_t* pos_of, const int32_t* used,
                       int n_tokens, int k, int vecs, void* dy, void* dw, cudaStream_t stream) {
  const RowSplit s = row_split(vecs);
  return launch_kernel(unpermute_rows_grad_kernel<T, W>, (n_tokens + s.tokens - 1) / s.tokens, ROWS_THREADS, 0, stream,
                       "unpermute_rows_grad launch", static_cast<const T*>(dout), static_cast<const T*>(y),
                       static_cast<const W*>(w), pos_of, used, n_tokens, k, vecs, s.lanes, static_cast<T*>(dy),
                       static_cast<W*>(dw));
}

}  // namespace sy

// Calls `fn<T, W>` for the rows' type and the weights' type (float32 or the rows').
#define SY_ROWS_DISPATCH(fn, dtype, wdtype, ...)                                                      \
  ((dtype) == SY_DTYPE_F32  ? fn<float, float>(__VA_ARGS__)                                           \
   : (dtype) == SY_DTYPE_F16 ? ((wdtype) == SY_DTYPE_F32 ? fn<__half, float>(__VA_ARGS__)             \
                                                         : fn<__half, __half>(__VA_ARGS__))           \
                             : ((wdtype) == SY_DTYPE_F32 ? fn<__nv_bfloat16, float>(__VA_ARGS__)      \
                                                         : fn<__nv_bfloat16, __nv_bfloat16>(__VA_ARGS__)))

extern "C" int sy_permute_rows(const void* h, const int32_t* pos_of, const int32_t* offsets, int n_tokens, int top_k,
                               int n_experts, int hidden, int dtype, void* x, void* stream) {
  using namespace sy;
  int vecs = 0;
  const int rc = rows_check("permute_rows", n_tokens, top_k, hidden, dtype, &vecs);
  if (rc != SY_OK) return rc;
  SY_REQUIRE(n_experts >= 1, "permute_rows: at least one expert (got %d)", n_experts);
  if (n_tokens == 0) return SY_OK;
  SY_REQUIRE(h && pos_of && offsets && x, "permute_rows: null pointer");
  SY_REQUIRE(aligned16(h) && aligned16(x), "permute_rows: h and x must be 16-byte aligned");
  const RowSplit s = row_split(vecs);
  return launch_kernel(permute_rows_kernel, (n_tokens + s.tokens - 1) / s.tokens, ROWS_THREADS, 0,
                       static_cast<cudaStream_t>(stream), "permute_rows launch", static_cast<const uint4*>(h), pos_of,
                       offsets + n_experts, n_tokens, top_k, vecs, s.lanes, static_cast<uint4*>(x));
}

extern "C" int sy_unpermute_rows(const void* y, const void* w, int w_dtype, const int32_t* pos_of, int n_tokens, int top_k,
                                 int hidden, int dtype, void* out, void* stream) {
  using namespace sy;
  int vecs = 0;
  const int rc = rows_check("unpermute_rows", n_tokens, top_k, hidden, dtype, &vecs);
  if (rc != SY_OK) return rc;
  SY_REQUIRE(!w || w_dtype == dtype || w_dtype == SY_DTYPE_F32, "unpermute_rows: weights must be f32 or of the rows' type");
  if (n_tokens == 0) return SY_OK;
  SY_REQUIRE(y && pos_of && out, "unpermute_rows: null pointer");
  SY_REQUIRE(aligned16(y) && aligned16(out), "unpermute_rows: y and out must be 16-byte aligned");
  const int wd = w ? w_dtype : dtype;
  return SY_ROWS_DISPATCH(unpermute_launch, dtype, wd, y, w, pos_of, n_tokens, top_k, vecs, out,
                          static_cast<cudaStream_t>(stream));
}

extern "C" int sy_unpermute_rows_grad(const void* dout, const void* y, const void* w, int w_dtype, const int32_t* pos_of,
                                      const int32_t* offsets, int n_tokens, int top_k, int n_experts, int hidden, int dtype,
                                      void* dy, void* dw, void* stream) {
  using namespace sy;
  int vecs = 0;
  const int rc = rows_check("unpermute_rows_grad", n_tokens, top_k, hidden, dtype, &vecs);
  if (rc != SY_OK) return rc;
  SY_REQUIRE(n_experts >= 1, "unpermute_rows_grad: at least one expert (got %d)", n_experts);
  SY_REQUIRE((!w && !dw) || w_dtype == dtype || w_dtype == SY_DTYPE_F32,
             "unpermute_rows_grad: weights must be f32 or of the rows' type");
  if (n_tokens == 0 || (!dy && !dw)) return SY_OK;
  SY_REQUIRE(dout && pos_of && offsets && (y || !dw), "unpermute_rows_grad: null pointer");
  SY_REQUIRE(aligned16(dout) && aligned16(y) && aligned16(dy), "unpermute_rows_grad: dout, y and dy must be 16-byte aligned");
  const int wd = w || dw ? w_dtype : dtype;
  return SY_ROWS_DISPATCH(grad_launch, dtype, wd, dout, y, w, pos_of, offsets + n_experts, n_tokens, top_k, vecs, dy, dw,
                          static_cast<cudaStream_t>(stream));
}
