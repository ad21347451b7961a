// Helpers of the row-wise operators (layer norm, dropout): 16-byte pieces of rows of any alignment, sums over
// groups of lanes.
#pragma once
#include "bf16_util.h"

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

// Elements of T in 16 bytes.
template <typename T>
struct Piece {
  static constexpr int N = 16 / (int)sizeof(T);
};

__device__ __forceinline__ float to_f32(bf16_t h) { return bf16_to_f32(h); }
__device__ __forceinline__ float to_f32(float f) { return f; }
__device__ __forceinline__ void from_f32(float f, bf16_t &out) { out = (bf16_t)f32_to_bf16(f); }
__device__ __forceinline__ void from_f32(float f, float &out) { out = f; }

// The piece p[0..N), zero from element n on, as it is stored.  One 16-byte access when all N elements exist, whatever
// the alignment (global memory instructions take any on this target); element by element at the end of a row.
template <typename T>
__device__ __forceinline__ u32x4 load_raw(const T *__restrict__ p, int n) {
  constexpr int N = Piece<T>::N;
  u32x4 r = {0, 0, 0, 0};
  if (n >= N) {
    __builtin_memcpy(&r, p, 16);
  } else {
    T e[N];
#pragma unroll
    for (int i = 0; i < N; ++i) e[i] = i < n ? p[i] : (T)0;
    __builtin_memcpy(&r, e, 16);
  }
  return r;
}
template <typename T>
__device__ __forceinline__ void widen(const u32x4 &r, float (&v)[Piece<T>::N]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 2) {
      v[2 * i] = __uint_as_float(r[i] << 16);
      v[2 * i + 1] = __uint_as_float(r[i] & 0xffff0000u);
    } else {
      v[i] = __uint_as_float(r[i]);
    }
  }
}
template <typename T>
__device__ __forceinline__ void load_piece(const T *__restrict__ p, int n, float (&v)[Piece<T>::N]) {
  widen<T>(load_raw(p, n), v);
}
template <typename T>
__device__ __forceinline__ void store_piece(T *__restrict__ p, int n, const float (&v)[Piece<T>::N]) {
  constexpr int N = Piece<T>::N;
  T e[N];
  if constexpr (sizeof(T) == 2) {  // as pairs: one conversion instruction for two
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const bf16x2 h = __builtin_convertvector((f32x2{v[i], v[i + 1]}), bf16x2);
      __builtin_memcpy(e + i, &h, 4);
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) e[i] = v[i];
  }
  if (n >= N) {
    __builtin_memcpy(p, e, 16);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < n) p[i] = e[i];
  }
}

// Sum over the 16 lanes of a DPP row: four rotations, every lane gets the total.
__device__ __forceinline__ float row16_sum(float v) {
  v = lane_rot_sum4(lane_rot_sum8(v));
  v = keep_scalar(v);
  v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x122, 0xf, 0xf, true));
  v = keep_scalar(v);
  return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x121, 0xf, 0xf, true));
}
// Sum of a lane and the lane 16 / 32 further, in every lane the same terms in the same order (no LDS instruction).
__device__ __forceinline__ float pair_sum16(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float pair_sum32(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
// Sums of NS values over a group of G lanes (16, 32, 64, or the 256 of the workgroup); every lane gets the totals.
// G = 256: `red` holds 2 x NS x 4 floats and `phase` alternates between its halves, one barrier per sum.
template <int G, int NS>
__device__ __forceinline__ void group_sum(float (&v)[NS], float *red, int &phase) {
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    v[s] = row16_sum(v[s]);
    if (G > 16) v[s] = pair_sum16(v[s]);
    if (G > 32) v[s] = pair_sum32(v[s]);
  }
  if (G == 256) {
    float *r = red + phase * NS * 4;
    phase ^= 1;
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int s = 0; s < NS; ++s) r[s * 4 + (threadIdx.x >> 6)] = v[s];
    __syncthreads();
#pragma unroll
    for (int s = 0; s < NS; ++s) v[s] = (r[s * 4] + r[s * 4 + 1]) + (r[s * 4 + 2] + r[s * 4 + 3]);
  }
}
