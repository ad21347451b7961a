// Dropout whose mask is a function of (seed, offset, element), so that it is never stored: the backward, another
// storage type or another stride ask the same question and get the same answer.  The generator and the numbering
// are stated in include/unet_hip.h.
//
// out = residual + (kept ? x / (1 - p) : 0), in fp32, rounded once.
//
// Bound by HBM as long as the generator stays cheap: one Philox block (20 multiplications of 32 x 32 bits) makes the
// upper 16 bits of eight elements' numbers.  Those decide unless they equal the threshold's upper 16 bits, which
// happens to one element in 65536; only then the block of the lower 16 bits is computed.  So p has the resolution of
// 2^-32 at half the multiplications.  65536 rows of 1024 bf16 channels with a residual: 73 us, 5.5 TB/s (the 400 MB are
// partly in the last-level cache; a large copy reaches 4.9).
#include "rows_util.h"

namespace {

constexpr int E = 8;  // elements per thread and step: the eight numbers of one block

// Philox4x32-10: J. Salmon, M. Moraes, R. Dror, D. Shaw, "Parallel random numbers: as easy as 1, 2, 3" (2011).
__device__ __forceinline__ u32x4 philox(uint32_t c0, uint32_t c1, uint32_t c2, uint32_t c3, uint32_t k0, uint32_t k1) {
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const uint64_t a = (uint64_t)0xD2511F53u * c0, b = (uint64_t)0xCD9E8D57u * c2;
    c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
    c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
    c1 = (uint32_t)b;
    c3 = (uint32_t)a;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return u32x4{c0, c1, c2, c3};
}

template <typename T>
struct Args {
  const T *x, *res;
  T *out;
  i64 x_ld, res_ld, out_ld, total;  // total = rows * channels elements
  int C;
  uint32_t thr_hi, thr_lo;  // round(p * 2^32) = thr_hi * 2^16 + thr_lo; thr_hi = 2^16 at p = 1
  float scale;
  uint64_t seed, offset;
  const uint64_t *offset_device;
};

__device__ __forceinline__ void load8(const bf16_t *__restrict__ p, float (&v)[E]) { load_piece(p, E, v); }
__device__ __forceinline__ void load8(const float *__restrict__ p, float (&v)[E]) { __builtin_memcpy(v, p, 32); }
__device__ __forceinline__ void store8(bf16_t *__restrict__ p, const float (&v)[E]) { store_piece(p, E, v); }
__device__ __forceinline__ void store8(float *__restrict__ p, const float (&v)[E]) { __builtin_memcpy(p, v, 32); }

// FLAT: all strides equal the channel count (or there is one row), so an element's address is its number.
template <typename T, bool RES, bool FLAT>
__global__ __launch_bounds__(256) void dropout_kernel(const Args<T> a) {
  const uint64_t off = a.offset + (a.offset_device ? *a.offset_device : 0);
  const i64 blocks = (a.total + E - 1) / E;
  for (i64 b = (i64)blockIdx.x * 256 + threadIdx.x; b < blocks; b += (i64)gridDim.x * 256) {
    const i64 e0 = b * E;
    const int n = (int)min<i64>(E, a.total - e0);
    i64 row = 0, col = e0;
    if (!FLAT) {
      row = a.total <= 0xffffffffll ? (i64)((uint32_t)e0 / (uint32_t)a.C) : e0 / a.C;
      col = e0 - row * a.C;
    }
    // the thread's elements lie in one row, or in two (C >= 8: the second begins at element `left`), or anywhere (C < 8)
    const int left = FLAT ? E : (int)min<i64>(E, a.C - col);
    const bool whole = n == E && left == E;
    auto at = [&](const T *base, i64 ld, int i) __attribute__((always_inline)) {
      if (FLAT || a.C >= E) return base + row * ld + col + i + (i >= left ? ld - a.C : 0);
      const i64 r = (e0 + i) / a.C;
      return base + r * ld + (e0 + i - r * a.C);
    };
    float x[E], r[E];
    if (whole) {
      load8(a.x + row * a.x_ld + col, x);
      if (RES) load8(a.res + row * a.res_ld + col, r);
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i) {
        x[i] = i < n ? to_f32(*at(a.x, a.x_ld, i)) : 0.f;
        if (RES) r[i] = i < n ? to_f32(*at(a.res, a.res_ld, i)) : 0.f;
      }
    }
    const uint32_t b0 = (uint32_t)b, b1 = (uint32_t)((uint64_t)b >> 32);
    const u32x4 hi = philox(b0, b1, (uint32_t)off, (uint32_t)(off >> 32), (uint32_t)a.seed, (uint32_t)(a.seed >> 32));
    uint32_t h[E];
    bool tie = false;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      h[i] = (i & 1) ? hi[i >> 1] >> 16 : hi[i >> 1] & 0xffffu;
      tie |= h[i] == a.thr_hi;
    }
    bool keep[E];
#pragma unroll
    for (int i = 0; i < E; ++i) keep[i] = h[i] >= a.thr_hi;
    if (tie && a.thr_lo) {
      const u32x4 lo = philox(b0, b1 | 0x80000000u, (uint32_t)off, (uint32_t)(off >> 32), (uint32_t)a.seed,
                              (uint32_t)(a.seed >> 32));
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const uint32_t l = (i & 1) ? lo[i >> 1] >> 16 : lo[i >> 1] & 0xffffu;
        keep[i] = h[i] > a.thr_hi || (h[i] == a.thr_hi && l >= a.thr_lo);
      }
    }
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const float v = keep[i] ? x[i] * a.scale : 0.f;
      x[i] = RES ? r[i] + v : v;
    }
    if (whole) {
      store8(a.out + row * a.out_ld + col, x);
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i)
        if (i < n) from_f32(x[i], *const_cast<T *>(at(a.out, a.out_ld, i)));
    }
  }
}

template <typename T>
bool aligned(const void *p) { return ((uintptr_t)p & (sizeof(T) - 1)) == 0; }

template <typename T>
int dropout(const char *name, const T *x, i64 x_ld, const T *res, i64 res_ld, T *out, i64 out_ld, i64 rows, int C, double p,
            uint64_t seed, uint64_t offset, const uint64_t *offset_device, hipStream_t st) {
  UNET_REQUIRE(rows >= 0 && C >= 1, "%s: rows %lld, channels %d", name, (long long)rows, C);
  UNET_REQUIRE(p >= 0.0 && p <= 1.0, "%s: p = %g is not in [0, 1]", name, p);
  UNET_REQUIRE(x_ld >= C && out_ld >= C && (!res || res_ld >= C), "%s: a row stride is smaller than the %d channels", name, C);
  UNET_REQUIRE(rows <= INT64_MAX / 8 / C, "%s: %lld rows of %d channels are too many", name, (long long)rows, C);
  if (rows == 0) return UNET_OK;
  UNET_REQUIRE(x && out, "%s: NULL tensor", name);
  UNET_REQUIRE(aligned<T>(x) && aligned<T>(res) && aligned<T>(out) && aligned<uint64_t>(offset_device),
               "%s: misaligned pointer", name);
  const uint64_t thr = (uint64_t)llrint(p * 4294967296.0);
  const Args<T> a{x, res, out, x_ld, res_ld, out_ld, rows * C, C, (uint32_t)(thr >> 16), (uint32_t)(thr & 0xffff),
                  p < 1.0 ? (float)(1.0 / (1.0 - p)) : 0.f, seed, offset, offset_device};
  const bool flat = rows == 1 || (x_ld == C && out_ld == C && (!res || res_ld == C));
  const unsigned grid = ew_grid((a.total + E - 1) / E);
  if (res && flat) dropout_kernel<T, true, true><<<grid, 256, 0, st>>>(a);
  else if (res) dropout_kernel<T, true, false><<<grid, 256, 0, st>>>(a);
  else if (flat) dropout_kernel<T, false, true><<<grid, 256, 0, st>>>(a);
  else dropout_kernel<T, false, false><<<grid, 256, 0, st>>>(a);
  UNET_LAUNCH_CHECK(name);
  return UNET_OK;
}

}  // namespace

extern "C" {

int unet_dropout_f32(const float *inputs, int64_t in_ld, const float *residual, int64_t residual_ld, float *activations,
                     int64_t out_ld, int64_t rows, int channels, double p, uint64_t seed, uint64_t offset,
                     const uint64_t *offset_device, unet_stream_t stream) {
  return dropout<float>("dropout", inputs, in_ld, residual, residual_ld, activations, out_ld, rows, channels, p, seed, offset,
                        offset_device, as_stream(stream));
}
int unet_dropout_bf16(const uint16_t *inputs, int64_t in_ld, const uint16_t *residual, int64_t residual_ld,
                      uint16_t *activations, int64_t out_ld, int64_t rows, int channels, double p, uint64_t seed,
                      uint64_t offset, const uint64_t *offset_device, unet_stream_t stream) {
  return dropout<bf16_t>("dropout", inputs, in_ld, residual, residual_ld, activations, out_ld, rows, channels, p, seed, offset,
                         offset_device, as_stream(stream));
}
int unet_dropout_backward_f32(const float *grad_activations, int64_t grad_ld, float *grad_inputs, int64_t grad_in_ld,
                              int64_t rows, int channels, double p, uint64_t seed, uint64_t offset,
                              const uint64_t *offset_device, unet_stream_t stream) {
  return dropout<float>("dropout_backward", grad_activations, grad_ld, nullptr, 0, grad_inputs, grad_in_ld, rows, channels, p,
                        seed, offset, offset_device, as_stream(stream));
}
int unet_dropout_backward_bf16(const uint16_t *grad_activations, int64_t grad_ld, uint16_t *grad_inputs,
                               int64_t grad_in_ld, int64_t rows, int channels, double p, uint64_t seed, uint64_t offset,
                               const uint64_t *offset_device, unet_stream_t stream) {
  return dropout<bf16_t>("dropout_backward", grad_activations, grad_ld, nullptr, 0, grad_inputs, grad_in_ld, rows, channels, p,
                         seed, offset, offset_device, as_stream(stream));
}

}  // extern "C"
