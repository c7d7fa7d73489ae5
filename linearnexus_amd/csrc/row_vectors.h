// Rows of a norm in the registers of their threads: loads, stores and sums, for kernels whose rows belong to a part of a wave, a wave or a
// workgroup.
#pragma once

#include "mma_tiles.h"

namespace {

// The VN elements of a row that a thread holds: consecutive ones as 16-byte vectors (ES = 1), or, where widths or pointers do not allow
// that, ES = threads of the row apart, one at a time, so that a wave's loads are still whole lines (consecutive ones a lane touched every line
// VN times: 6435 rows of 4475, bf16 with an fp32 stream and a gate, forward 247 us, this way 128;
// 8751 rows of 3834 in fp32, backward 332 and 224).
template <int TPR, int VN, int ES> __device__ __forceinline__ int first_column(int k, int li) { return ES == 1 ? (k * TPR + li) * VN : k * TPR * VN + li; }

// VN elements of a row as fp32; those less than `left` from the first exist
template <typename E, int VN, int ES> __device__ __forceinline__ void load_row(const E* p, int left, float* f) {
  if constexpr (ES > 1) {
#pragma unroll
    for (int e = 0; e < VN; ++e) f[e] = e * ES < left ? to_f32(p[e * ES]) : 0.f;
  } else if constexpr (VN == Vec16<E>::N) {
    const typename Vec16<E>::V v = *reinterpret_cast<const typename Vec16<E>::V*>(p);
#pragma unroll
    for (int e = 0; e < VN; ++e) f[e] = to_f32(v[e]);
  } else {  // eight floats beside eight bf16
    const floatx4 a = load4(p), b = load4(p + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = a[e], f[e + 4] = b[e];
  }
}

template <typename E, int VN, int ES> __device__ __forceinline__ void store_row(E* p, int left, const float* f) {
  if constexpr (ES > 1) {
#pragma unroll
    for (int e = 0; e < VN; ++e)
      if (e * ES < left) p[e * ES] = from_f32<E>(f[e]);
  } else if constexpr (VN == Vec16<E>::N) {
    typename Vec16<E>::V v;
#pragma unroll
    for (int e = 0; e < VN; ++e) v[e] = from_f32<E>(f[e]);
    *reinterpret_cast<typename Vec16<E>::V*>(p) = v;
  } else {
    store4(p, floatx4{f[0], f[1], f[2], f[3]});
    store4(p + 4, floatx4{f[4], f[5], f[6], f[7]});
  }
}

// The same as it lies in memory, for a row that is fetched ahead of its use
template <typename E, int VN, int ES> struct RawRow {
  static constexpr int N = Vec16<E>::N;
  typename Vec16<E>::V v[VN / N];
  __device__ __forceinline__ void load(const E* p, int left) {
#pragma unroll
    for (int k = 0; k < VN / N; ++k) {
      v[k] = vec_zero<E>();
      if constexpr (ES == 1) {
        if (left > 0) v[k] = *reinterpret_cast<const typename Vec16<E>::V*>(p + k * N);
      } else {
#pragma unroll
        for (int e = 0; e < N; ++e)
          if ((k * N + e) * ES < left) v[k][e] = p[(k * N + e) * ES];
      }
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int k = 0; k < VN / N; ++k) v[k] = vec_zero<E>();
  }
  __device__ __forceinline__ float get(int e) const { return to_f32(v[e / N][e % N]); }
};

// Sums over the TPR threads of a row (a power of two from 4 on); all of them get them.  `red`: a slot per wave that nothing else uses until the
// next barrier but one (rows of up to 64 threads need none).
template <int TPR> __device__ __forceinline__ float lanes_sum(float x) {
  if constexpr (TPR == 4) return quad_sum(x);
  else if constexpr (TPR == 8) return quad_sum(x) + __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(quad_sum(x)), 0x141, 0xF, 0xF, true));  // the half row's other quad
  else if constexpr (TPR == 16) return row16_sum(x);
  else if constexpr (TPR == 32) return xor16_sum(row16_sum(x));
  else return wave_sum(x);
}
template <int TPR> __device__ __forceinline__ float row_sum(float x, float* red) {
  x = lanes_sum<TPR>(x);
  if constexpr (TPR <= 64) return x;
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
  lds_barrier();
  float s = red[0];
#pragma unroll
  for (int i = 1; i < TPR / 64; ++i) s += red[i];
  return s;
}
template <int TPR> __device__ __forceinline__ void row_sum2(float& x, float& y, float* red) {
  x = lanes_sum<TPR>(x);
  y = lanes_sum<TPR>(y);
  if constexpr (TPR <= 64) return;
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x, red[16 + (threadIdx.x >> 6)] = y;
  lds_barrier();
  x = red[0];
  y = red[16];
#pragma unroll
  for (int i = 1; i < TPR / 64; ++i) x += red[i], y += red[16 + i];
}
// Two or three of them, of rows of a wave and more by fewer exchanges: an exchange of rows of 16 lanes of two values leaves one sum, whose even rows are the
// first's and whose odd rows the second's, one of the halves of that and the third's the like, so that the last four steps are one value's
template <int TPR, int N> __device__ __forceinline__ void row_sums(float (&x)[N], float* red) {
  static_assert(N == 2 || N == 3, "rows of 16 lanes: 0, 1, 0, 1 or 0, 1, 2, 2");
  if constexpr (TPR < 64) {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = lanes_sum<TPR>(x[i]);
  } else {
    const auto two = __builtin_amdgcn_permlane16_swap(__float_as_uint(x[0]), __float_as_uint(x[1]), false, false);
    float s = __uint_as_float(two[0]) + __uint_as_float(two[1]);
    const auto all = __builtin_amdgcn_permlane32_swap(__float_as_uint(s), __float_as_uint(N == 2 ? s : xor16_sum(x[N - 1])), false, false);
    s = row16_sum(__uint_as_float(all[0]) + __uint_as_float(all[1]));
    if constexpr (TPR == 64) {
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(s), 16 * i));
    } else {
      const int lane = threadIdx.x & 63;
      if (lane % 16 == 0 && lane < 16 * N) red[lane + (threadIdx.x >> 6)] = s;
      lds_barrier();
#pragma unroll
      for (int i = 0; i < N; ++i) {
        x[i] = red[16 * i];
#pragma unroll
        for (int w = 1; w < TPR / 64; ++w) x[i] += red[16 * i + w];
      }
    }
  }
}

}  // namespace
