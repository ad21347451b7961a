// Layer norm over the channels of each row, forward and backward (fp32 and bf16 storage).
//
//   xhat = (x - mean) * rstd,  y = gamma * xhat + beta
//   dx = rstd * (g - mean_c g - xhat * mean_c(g * xhat)) [+ skip],  g = gamma * dy
//   dgamma = sum_rows dy * xhat,  dbeta = sum_rows dy
//
// Bound by HBM: a few operations per element read or written.  So every tensor is passed over once: a row lives in
// the registers of a group of G lanes (16 lanes up to 32 pieces of 16 bytes, 32 or 64 up to 256, the workgroup up
// to 1024; longer rows are read again by the *_long kernels), which takes the statistics from the registers in two
// passes (mean, then squared deviations: no cancellation).  Groups walk over rows, gamma and beta stay on the CU
// across rows (in LDS: in registers they would cost half of the wavefronts), and the next row is requested before the
// current one is worked on.  65536 rows of 1024 bf16 channels: forward 47 us (5.7 TB/s; both tensors just fit the
// last-level cache), backward 77 us and 5 for the partial rows of the weight's gradient (4.9 TB/s, the rate of a large copy).
//
// The sums over rows (dgamma, dbeta) are kept per lane for the columns it owns, added up inside the workgroup in a
// fixed order and written as one partial row [2C] per workgroup; a last launch adds the partial rows, in double
// (it reads at most BWD_BLOCKS of them).  More than CHAIN rows a group (131072 rows and more) are taken by several
// launches, each adding to the partial rows, so that a sum over millions of rows is no chain of thousands.  No atomics,
// so equal calls give equal bits.
#include "rows_util.h"

namespace {

constexpr int FWD_BLOCKS = 2048;  // 8 workgroups of 4 wavefronts per CU: all resident for rows of up to 192 pieces; of longer
                                  // rows 6 to 2, whose gamma and beta take up to 64 KB of LDS
constexpr int BWD_BLOCKS = 512;   // 2 per CU: fewer partial rows for the second launch to read
constexpr int MOST_CHANNELS = 1 << 26;  // the column sums' launch has 32 threads a channel, of fewer than 2^32
constexpr int CHAIN = 256;        // rows of a group in one fp32 chain of the column sums
constexpr int LONG_SPLITS = 64;   // row ranges of the column sums of rows that do not fit registers

template <typename T>
struct FwdArgs {
  const T *x;
  T *y;
  const float *w;
  float *stats;
  i64 x_ld, y_ld, rows;
  int C;
  float eps;
};
template <typename T>
struct BwdArgs {
  const T *dy, *x, *skip;
  const float *stats, *w;
  T *dx;
  float *partials;  // [gridDim.x][2C], NULL: no weight gradient
  i64 dy_ld, x_ld, skip_ld, dx_ld, rows;
  int C;
  bool add;  // to the partials, which earlier rows have left
};

// gamma (and beta) of the row's columns in LDS, in the order in which the lanes take them: value i of piece v of lane l at
// [(v * N + i) / 4][l][i % 4], zero behind the last column.  In registers they would halve the wavefronts of a CU.
template <int N, int G, int NV, int STRIDE>
__device__ __forceinline__ void stage_weights(float *to, const float *w, int C, float none) {
  for (int i = threadIdx.x; i < G * NV * N; i += 256) {
    const int c = ((i / (4 * G) * 4) / N * G + i / 4 % G) * N + (i / (4 * G) * 4) % N + i % 4;
    to[i] = c >= C ? 0.f : w ? w[STRIDE * c] : none;
  }
}
template <int N, int G>
__device__ __forceinline__ f32x4 staged(const float *from, int v, int i, int lane) {
  return *reinterpret_cast<const f32x4 *>(from + ((v * N + i) / 4 * G + lane) * 4);
}

template <typename T, int G, int NV>
__global__ __launch_bounds__(256) void layer_norm_kernel(const FwdArgs<T> a) {
  constexpr int N = Piece<T>::N, COLS = G * NV * N;
  __shared__ float red[8];
  __shared__ __align__(16) float gamma[COLS], beta[COLS];
  stage_weights<N, G, NV, 2>(gamma, a.w, a.C, 1.f);
  stage_weights<N, G, NV, 2>(beta, a.w ? a.w + 1 : nullptr, a.C, 0.f);
  const int lane = threadIdx.x % G, per = 256 / G;
  int phase = 0, left[NV];
#pragma unroll
  for (int v = 0; v < NV; ++v) left[v] = a.C - (lane + v * G) * N;
  const float c = (float)a.C;
  const i64 step = (i64)gridDim.x * per;
  i64 row = (i64)blockIdx.x * per + threadIdx.x / G;
  u32x4 next[NV];
  auto load = [&](i64 r) __attribute__((always_inline)) {
    if (r < a.rows)
#pragma unroll
      for (int v = 0; v < NV; ++v) next[v] = load_raw(a.x + r * a.x_ld + (lane + v * G) * N, left[v]);
  };
  load(row);
  __syncthreads();
  for (; row < a.rows; row += step) {
    float x[NV][N], s[1] = {0.f};
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      widen<T>(next[v], x[v]);
#pragma unroll
      for (int i = 0; i < N; ++i) s[0] += x[v][i];
    }
    load(row + step);
    group_sum<G, 1>(s, red, phase);
    const float mean = s[0] / c;  // a true division: the mean of equal values is exact where their sum is
    s[0] = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int i = 0; i < N; ++i) {
        x[v][i] = i < left[v] ? x[v][i] - mean : 0.f;
        s[0] += x[v][i] * x[v][i];
      }
    group_sum<G, 1>(s, red, phase);
    const float rstd = 1.f / sqrtf(s[0] / c + a.eps);
    if (a.stats && lane == 0) {
      a.stats[2 * row] = mean;
      a.stats[2 * row + 1] = rstd;
    }
#pragma unroll
    for (int v = 0; v < NV; ++v) {
#pragma unroll
      for (int i = 0; i < N; i += 4) {
        const f32x4 g = staged<N, G>(gamma, v, i, lane), b = staged<N, G>(beta, v, i, lane);
#pragma unroll
        for (int j = 0; j < 4; ++j) x[v][i + j] = g[j] * (x[v][i + j] * rstd) + b[j];
      }
      store_piece(a.y + row * a.y_ld + (lane + v * G) * N, left[v], x[v]);
    }
  }
}

template <typename T, int G, int NV>
__global__ __launch_bounds__(256) void layer_norm_backward_kernel(const BwdArgs<T> a) {
  constexpr int N = Piece<T>::N, COLS = G * NV * N;
  __shared__ float red[16];
  __shared__ __align__(16) float gamma[COLS];
  __shared__ float sums[G < 256 ? 2 * COLS : 1];
  stage_weights<N, G, NV, 2>(gamma, a.w, a.C, 1.f);
  const int lane = threadIdx.x % G, per = 256 / G;
  int phase = 0, left[NV];
  float dga[NV][N], dbe[NV][N];
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    left[v] = a.C - (lane + v * G) * N;
#pragma unroll
    for (int i = 0; i < N; ++i) dga[v][i] = dbe[v][i] = 0.f;
  }
  const float inv_c = 1.f / (float)a.C;
  const i64 step = (i64)gridDim.x * per;
  i64 row = (i64)blockIdx.x * per + threadIdx.x / G;
  u32x4 nx[NV], nd[NV];
  float nmean = 0.f, nrstd = 0.f;
  auto load = [&](i64 r) __attribute__((always_inline)) {
    if (r < a.rows) {
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        nx[v] = load_raw(a.x + r * a.x_ld + (lane + v * G) * N, left[v]);
        nd[v] = load_raw(a.dy + r * a.dy_ld + (lane + v * G) * N, left[v]);
      }
      nmean = a.stats[2 * r];
      nrstd = a.stats[2 * r + 1];
    }
  };
  load(row);
  __syncthreads();
  for (; row < a.rows; row += step) {
    float x[NV][N], dy[NV][N], s[2] = {0.f, 0.f};
    const float mean = nmean, rstd = nrstd;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      widen<T>(nx[v], x[v]);
      widen<T>(nd[v], dy[v]);
    }
    load(row + step);
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int i = 0; i < N; i += 4) {
        const f32x4 g = staged<N, G>(gamma, v, i, lane);
#pragma unroll
        for (int j = i; j < i + 4; ++j) {
          x[v][j] = j < left[v] ? (x[v][j] - mean) * rstd : 0.f;
          dga[v][j] += dy[v][j] * x[v][j];
          dbe[v][j] += dy[v][j];
          dy[v][j] *= g[j - i];
          s[0] += dy[v][j];
          s[1] += dy[v][j] * x[v][j];
        }
      }
    if (a.dx) {
      group_sum<G, 2>(s, red, phase);
      const float m0 = s[0] * inv_c, m1 = s[1] * inv_c;
#pragma unroll
      for (int v = 0; v < NV; ++v) {
#pragma unroll
        for (int i = 0; i < N; ++i) dy[v][i] = rstd * (dy[v][i] - m0 - x[v][i] * m1);
        if (a.skip) {
          float skip[N];
          load_piece(a.skip + row * a.skip_ld + (lane + v * G) * N, left[v], skip);
#pragma unroll
          for (int i = 0; i < N; ++i) dy[v][i] += skip[i];
        }
        store_piece(a.dx + row * a.dx_ld + (lane + v * G) * N, left[v], dy[v]);
      }
    }
  }
  if (!a.partials) return;
  float *out = a.partials + (i64)blockIdx.x * 2 * a.C;
  if (G < 256) {  // the groups' sums, one group after the other
    for (int g = 0; g < per; ++g) {
      if (threadIdx.x / G == g)
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
          for (int i = 0; i < N; ++i) {
            const int c = 2 * ((lane + v * G) * N + i);
            sums[c] = g ? sums[c] + dga[v][i] : dga[v][i];
            sums[c + 1] = g ? sums[c + 1] + dbe[v][i] : dbe[v][i];
          }
      __syncthreads();
    }
    if (a.add)
      for (int c = threadIdx.x; c < 2 * a.C; c += 256) out[c] += sums[c];
    else
      for (int c = threadIdx.x; c < 2 * a.C; c += 256) out[c] = sums[c];
  } else {
    if (a.add)
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int c = 2 * min((lane + v * G) * N + i, a.C - 1);
          dga[v][i] += out[c];
          dbe[v][i] += out[c + 1];
        }
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (i < left[v]) {
          const int c = 2 * ((lane + v * G) * N + i);
          out[c] = dga[v][i];
          out[c + 1] = dbe[v][i];
        }
  }
}

// grad[c] = sum of partials[0..n)[c] for the 2C interleaved columns: 16 columns x 16 row classes per workgroup.
__global__ __launch_bounds__(256) void layer_norm_wgrad_kernel(const float *__restrict__ partials, int n, i64 cols,
                                                               float *__restrict__ grad) {
  __shared__ double red[16][17];
  const int tc = threadIdx.x & 15, tr = threadIdx.x >> 4;
  const i64 c = (i64)blockIdx.x * 16 + tc;
  double s = 0.0;
  if (c < cols)
#pragma unroll 8
    for (int r = tr; r < n; r += 16) s += (double)partials[(i64)r * cols + c];
  red[tr][tc] = s;
  __syncthreads();
  if (tr == 0 && c < cols) {
    for (int r = 1; r < 16; ++r) s += red[r][tc];
    grad[c] = (float)s;
  }
}

// Rows longer than the registers of a workgroup: one workgroup per row reads it once per pass.  A thread's share may be
// hundreds of thousands of elements, so it is added up in double (the passes wait for memory).
template <typename T>
__global__ __launch_bounds__(256) void layer_norm_long_kernel(const FwdArgs<T> a) {
  __shared__ float red[8];
  int phase = 0;
  for (i64 row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T *x = a.x + row * a.x_ld;
    T *y = a.y + row * a.y_ld;
    double t = 0.0;
    for (int c = threadIdx.x; c < a.C; c += 256) t += (double)to_f32(x[c]);
    float s[1] = {(float)t};
    group_sum<256, 1>(s, red, phase);
    const float mean = s[0] / (float)a.C;
    t = 0.0;
    for (int c = threadIdx.x; c < a.C; c += 256) {
      const double d = (double)(to_f32(x[c]) - mean);
      t += d * d;
    }
    s[0] = (float)t;
    group_sum<256, 1>(s, red, phase);
    const float rstd = 1.f / sqrtf(s[0] / (float)a.C + a.eps);
    if (a.stats && threadIdx.x == 0) {
      a.stats[2 * row] = mean;
      a.stats[2 * row + 1] = rstd;
    }
    for (int c = threadIdx.x; c < a.C; c += 256) {
      const float n = (to_f32(x[c]) - mean) * rstd;
      from_f32(a.w ? a.w[2 * (i64)c] * n + a.w[2 * (i64)c + 1] : n, y[c]);
    }
  }
}
template <typename T>
__global__ __launch_bounds__(256) void layer_norm_long_dx_kernel(const BwdArgs<T> a) {
  __shared__ float red[16];
  int phase = 0;
  for (i64 row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T *x = a.x + row * a.x_ld, *dy = a.dy + row * a.dy_ld;
    const float mean = a.stats[2 * row], rstd = a.stats[2 * row + 1];
    double t0 = 0.0, t1 = 0.0;
    for (int c = threadIdx.x; c < a.C; c += 256) {
      const float g = to_f32(dy[c]) * (a.w ? a.w[2 * (i64)c] : 1.f);
      t0 += (double)g;
      t1 += (double)g * (double)((to_f32(x[c]) - mean) * rstd);
    }
    float s[2] = {(float)t0, (float)t1};
    group_sum<256, 2>(s, red, phase);
    const float m0 = s[0] / (float)a.C, m1 = s[1] / (float)a.C;
    for (int c = threadIdx.x; c < a.C; c += 256) {
      const float g = to_f32(dy[c]) * (a.w ? a.w[2 * (i64)c] : 1.f), n = (to_f32(x[c]) - mean) * rstd;
      const float d = rstd * (g - m0 - n * m1);
      from_f32(a.skip ? d + to_f32(a.skip[row * a.skip_ld + c]) : d, a.dx[row * a.dx_ld + c]);
    }
  }
}
template <typename T>
__global__ __launch_bounds__(256) void layer_norm_long_columns_kernel(const BwdArgs<T> a, i64 rows_per) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= a.C) return;
  const i64 r0 = blockIdx.y * rows_per, r1 = min(a.rows, r0 + rows_per);
  double dga = 0.0, dbe = 0.0;
  for (i64 r = r0; r < r1; ++r) {
    const double dy = (double)to_f32(a.dy[r * a.dy_ld + c]);
    dga += dy * (double)((to_f32(a.x[r * a.x_ld + c]) - a.stats[2 * r]) * a.stats[2 * r + 1]);
    dbe += dy;
  }
  float *out = a.partials + (i64)blockIdx.y * 2 * a.C + 2 * (i64)c;
  out[0] = (float)dga;
  out[1] = (float)dbe;
}

// f(G, NV) with the lanes per row and 16-byte pieces per lane that hold a row of `pieces` pieces; false: too long.
// The smallest group that holds the row: the fewer lanes share a row, the fewer steps its sums take; three pieces a lane
// where two or four would leave more than a quarter of the lanes idle.
template <typename F>
bool with_row_shape(i64 pieces, F f) {
  using std::integral_constant;
  if (pieces <= 16) f(integral_constant<int, 16>(), integral_constant<int, 1>());
  else if (pieces <= 32) f(integral_constant<int, 16>(), integral_constant<int, 2>());
  else if (pieces <= 64) f(integral_constant<int, 64>(), integral_constant<int, 1>());
  else if (pieces <= 96) f(integral_constant<int, 32>(), integral_constant<int, 3>());
  else if (pieces <= 128) f(integral_constant<int, 64>(), integral_constant<int, 2>());
  else if (pieces <= 192) f(integral_constant<int, 64>(), integral_constant<int, 3>());
  else if (pieces <= 256) f(integral_constant<int, 64>(), integral_constant<int, 4>());
  else if (pieces <= 512) f(integral_constant<int, 256>(), integral_constant<int, 2>());
  else if (pieces <= 1024) f(integral_constant<int, 256>(), integral_constant<int, 4>());
  else return false;
  return true;
}
template <typename T>
i64 pieces_of(int C) { return ((i64)C + Piece<T>::N - 1) / Piece<T>::N; }

template <typename T>
bool aligned(const void *p) { return ((uintptr_t)p & (sizeof(T) - 1)) == 0; }

template <typename T>
int layer_norm(const T *x, i64 x_ld, T *y, i64 y_ld, const float *w, float *stats, i64 rows, int C, float eps,
               hipStream_t st) {
  UNET_REQUIRE(rows >= 0 && C >= 1 && C <= MOST_CHANNELS, "layer_norm: rows %lld, channels %d", (long long)rows, C);
  UNET_REQUIRE(eps >= 0.f, "layer_norm: eps %g is negative or NaN", (double)eps);
  UNET_REQUIRE(x_ld >= C && y_ld >= C, "layer_norm: a row stride (%lld, %lld) is smaller than the %d channels",
               (long long)x_ld, (long long)y_ld, C);
  if (rows == 0) return UNET_OK;
  UNET_REQUIRE(x && y, "layer_norm: NULL tensor");
  UNET_REQUIRE(aligned<T>(x) && aligned<T>(y) && aligned<float>(w) && aligned<float>(stats), "layer_norm: misaligned pointer");
  const FwdArgs<T> a{x, y, w, stats, x_ld, y_ld, rows, C, eps};
  const bool held = with_row_shape(pieces_of<T>(C), [&](auto g, auto nv) {
    const i64 blocks = (rows + 256 / g - 1) / (256 / g);
    layer_norm_kernel<T, decltype(g)::value, decltype(nv)::value>
        <<<(unsigned)(blocks < FWD_BLOCKS ? blocks : FWD_BLOCKS), 256, 0, st>>>(a);
  });
  if (!held) layer_norm_long_kernel<T><<<(unsigned)(rows < FWD_BLOCKS ? rows : FWD_BLOCKS), 256, 0, st>>>(a);
  UNET_LAUNCH_CHECK("layer_norm");
  return UNET_OK;
}

template <typename T>
int layer_norm_backward(const T *dy, i64 dy_ld, const T *x, i64 x_ld, const float *stats, const float *w, const T *skip,
                        i64 skip_ld, T *dx, i64 dx_ld, float *dw, i64 rows, int C, void *ws, size_t ws_bytes,
                        hipStream_t st) {
  UNET_REQUIRE(rows >= 0 && C >= 1 && C <= MOST_CHANNELS, "layer_norm_backward: rows %lld, channels %d", (long long)rows, C);
  UNET_REQUIRE(dy_ld >= C && x_ld >= C && (!skip || skip_ld >= C) && (!dx || dx_ld >= C),
               "layer_norm_backward: a row stride is smaller than the %d channels", C);
  UNET_REQUIRE(rows == 0 || (dy && x && stats), "layer_norm_backward: NULL tensor");
  UNET_REQUIRE(aligned<T>(dy) && aligned<T>(x) && aligned<T>(skip) && aligned<T>(dx) && aligned<float>(stats) &&
                   aligned<float>(w) && aligned<float>(dw),
               "layer_norm_backward: misaligned pointer");
  if (dw) {
    size_t need = 0;
    const int rc = unet_layer_norm_backward_workspace_bytes(rows, C, &need);
    if (rc != UNET_OK) return rc;
    UNET_REQUIRE(ws_bytes >= need && (ws || !need), "layer_norm_backward: workspace of %zu bytes, needs %zu", ws_bytes, need);
    UNET_REQUIRE(((uintptr_t)ws & 15) == 0, "layer_norm_backward: the workspace is not 16-byte aligned");
  }
  BwdArgs<T> a{dy, x, skip, stats, w, dx, dw ? (float *)ws : nullptr, dy_ld, x_ld, skip_ld, dx_ld, rows, C, false};
  if (!dw && (!dx || rows == 0)) return UNET_OK;
  int n = 0;  // partial rows written
  if (rows > 0) {
    const bool held = with_row_shape(pieces_of<T>(C), [&](auto g, auto nv) {
      const i64 most = dw ? (i64)CHAIN * BWD_BLOCKS * (256 / g) : rows;
      for (i64 done = 0; done < rows; done += most) {
        BwdArgs<T> b = a;
        b.dy += done * dy_ld, b.x += done * x_ld, b.stats += 2 * done, b.add = done > 0;
        if (skip) b.skip += done * skip_ld;
        if (dx) b.dx += done * dx_ld;
        b.rows = rows - done < most ? rows - done : most;
        const i64 blocks = (b.rows + 256 / g - 1) / (256 / g);
        const int grid = (int)(blocks < BWD_BLOCKS ? blocks : BWD_BLOCKS);
        if (!done) n = grid;
        layer_norm_backward_kernel<T, decltype(g)::value, decltype(nv)::value><<<grid, 256, 0, st>>>(b);
      }
    });
    if (!held) {
      if (dw) {  // before dx, which may overwrite what it reads
        n = (int)(rows < LONG_SPLITS ? rows : LONG_SPLITS);
        const i64 per = (rows + n - 1) / n;
        n = (int)((rows + per - 1) / per);
        layer_norm_long_columns_kernel<T><<<dim3(cdiv_u(C, 256), n), 256, 0, st>>>(a, per);
      }
      if (dx) layer_norm_long_dx_kernel<T><<<(unsigned)(rows < FWD_BLOCKS ? rows : FWD_BLOCKS), 256, 0, st>>>(a);
    }
  }
  if (dw) layer_norm_wgrad_kernel<<<cdiv_u(2 * (i64)C, 16), 256, 0, st>>>((const float *)ws, n, 2 * (i64)C, dw);
  UNET_LAUNCH_CHECK("layer_norm_backward");
  return UNET_OK;
}

}  // namespace

extern "C" {

int unet_layer_norm_backward_workspace_bytes(int64_t rows, int channels, size_t *bytes_host) {
  UNET_REQUIRE(bytes_host, "layer_norm_backward_workspace_bytes: NULL result");
  UNET_REQUIRE(rows >= 0 && channels >= 1 && channels <= MOST_CHANNELS, "layer_norm_backward_workspace_bytes: rows %lld, channels %d", (long long)rows,
               channels);
  *bytes_host = (size_t)(rows < BWD_BLOCKS ? rows : BWD_BLOCKS) * 2 * (size_t)channels * sizeof(float);
  return UNET_OK;
}

int unet_layer_norm_f32(const float *inputs, int64_t in_ld, float *activations, int64_t out_ld, const float *weights,
                        float *row_stats, int64_t rows, int channels, float eps, unet_stream_t stream) {
  return layer_norm<float>(inputs, in_ld, activations, out_ld, weights, row_stats, rows, channels, eps, as_stream(stream));
}
int unet_layer_norm_bf16(const uint16_t *inputs, int64_t in_ld, uint16_t *activations, int64_t out_ld,
                         const float *weights, float *row_stats, int64_t rows, int channels, float eps,
                         unet_stream_t stream) {
  return layer_norm<bf16_t>(inputs, in_ld, activations, out_ld, weights, row_stats, rows, channels, eps,
                            as_stream(stream));
}
int unet_layer_norm_backward_f32(const float *grad_activations, int64_t grad_ld, const float *inputs, int64_t in_ld,
                                 const float *row_stats, const float *weights, const float *grad_skip, int64_t skip_ld,
                                 float *grad_inputs, int64_t grad_in_ld, float *grad_weights, int64_t rows, int channels,
                                 void *workspace, size_t workspace_bytes, unet_stream_t stream) {
  return layer_norm_backward<float>(grad_activations, grad_ld, inputs, in_ld, row_stats, weights, grad_skip, skip_ld,
                                    grad_inputs, grad_in_ld, grad_weights, rows, channels, workspace, workspace_bytes,
                                    as_stream(stream));
}
int unet_layer_norm_backward_bf16(const uint16_t *grad_activations, int64_t grad_ld, const uint16_t *inputs,
                                  int64_t in_ld, const float *row_stats, const float *weights,
                                  const uint16_t *grad_skip, int64_t skip_ld, uint16_t *grad_inputs, int64_t grad_in_ld,
                                  float *grad_weights, int64_t rows, int channels, void *workspace,
                                  size_t workspace_bytes, unet_stream_t stream) {
  return layer_norm_backward<bf16_t>(grad_activations, grad_ld, inputs, in_ld, row_stats, weights, grad_skip, skip_ld,
                                     grad_inputs, grad_in_ld, grad_weights, rows, channels, workspace, workspace_bytes,
                                     as_stream(stream));
}

}  // extern "C"
