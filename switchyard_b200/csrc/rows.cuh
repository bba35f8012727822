// 16-byte pieces of rows in the three element types the row operators take.
#pragma once
#include "common.cuh"

namespace sy {

constexpr int ROWS_MAX_K = 8;  // most choices per token, as in route and combine
constexpr int ROWS_MOST = 0x7fffff00;   // rows, so that a block's last token is still a 32-bit number
constexpr int WIDTH_MOST = 0x7fff0000;  // columns, likewise

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v) { return Elem<T>::from_f(v); }
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }

template <typename T> struct RowVec {
  static constexpr int N = 8;
  static __device__ __forceinline__ void unpack(const uint4& v, float (&f)[8]) { unpack8<T>(v, f); }
  static __device__ __forceinline__ uint4 pack(const float (&f)[8]) {
    __align__(16) T r[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) r[q] = Elem<T>::from_f(f[q]);
    return *reinterpret_cast<const uint4*>(r);
  }
};
template <> struct RowVec<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void unpack(const uint4& v, float (&f)[4]) {
    f[0] = __uint_as_float(v.x), f[1] = __uint_as_float(v.y), f[2] = __uint_as_float(v.z), f[3] = __uint_as_float(v.w);
  }
  static __device__ __forceinline__ uint4 pack(const float (&f)[4]) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
};

}  // namespace sy
