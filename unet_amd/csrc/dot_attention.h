// Dot-product attention over packed sequences, forward and backward (fp32 and bf16 storage; fp32 operands are taken as
// three bf16 numbers, see Parts).
//
//   S = scale Q K^T,  P = softmax over the visible keys,  out = P V,  lse = log sum exp S
//   delta = sum_d dout * out,  dP = dout V^T,  dS = P * (dP - delta)
//   dV = P^T dout,  dQ = scale dS K,  dK = scale dS^T Q
//
// Three kernels of one shape.  A wavefront keeps 32 "columns" in registers as matrix-core B operands (queries in the
// forward and in the dQ kernel, keys in the dK/dV kernel) and streams "rows" (keys, or queries) through LDS in
// tiles that the workgroup shares.  Scores are computed transposed, rows x columns, so that
//   - a column's scores lie in one lane (and in the lane 32 further): maxima, sums, masks and rescaling need no
//     exchange inside the loop;
//   - the 32x32 result layout (lane: column l % 32; rows 8 * (i / 4) + 4 * (l / 32) + i % 4, i < 16) is, 16 rows at a time,
//     a B operand again for the second product acc[d][column] += X^T[d][rows] W[rows][column], if the A operand takes its
//     rows in the same order: the softmax weights never leave the registers.
// Query heads that share a key/value head are packed into the row axis of that head: row r of a sequence is query
// r / G, head r % G of the group.  One tile of keys and values serves all of them, and the sums of dK and dV over the
// group are part of the loop.
//
// LDS holds a tile as rows of DP elements in 16-byte chunks, chunk c of row r at c ^ key(r): both the reads along a row
// (A operands of the scores) and the transposing reads down the rows (A operands of the second product) then
// spread over all banks.
//
// What bounds it, measured:
//   - long sequences: the matrix cores.  8192 tokens, 16/4 heads of 128, causal, bf16: forward 315 us (0.87 PFLOP/s of the
//     visible pairs), dQ 421, dK/dV 594, their join 23.5 (0.66 PFLOP/s on five products of two kernels that compute
//     seven; a large library product reaches 1.24).
//   - short ones: the latency of a few tiles.  16 x 256 tokens, 16 heads of 64, bf16: forward 13 us, dQ 21, dK/dV 20 for
//     34 to 50 MB each.
//   - few queries: HBM.  4 queries over 53386 keys, 32/4 heads of 128, bf16: 22 us (5.0 TB/s) and 4 for the join.
//   - fp32: the matrix cores and, beside them, the vector instructions that split operands into parts.  3525 tokens in 4
//     sequences, 8 heads of 64: forward 51 us, dQ 77, dK/dV 94, their join 10 (130, 129 and 141 TFLOP/s of the products that
//     they compute; a large library product in fp32 reaches 154); forward of one of 8192 tokens 731 us (188 TFLOP/s).
// (Medians of 20 calls in a kernel trace; cards differ by up to 5 %.)
#include <math.h>

#include "rows_util.h"

namespace {

typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));

constexpr int COLS = 32;            // columns (queries or keys) per wavefront
constexpr int WAVES = 4;
constexpr int BM = COLS * WAVES;    // columns per workgroup
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
// The running maximum follows a score only when that exceeds it by this much (in powers of two): until then nothing is
// rescaled.  The reference that the weights are taken from lies LAZY + ceil(log2 keys) above it, so that a sequence's weights
// add up to 1 at most and no finite value overflows on the way.  The final division makes up for both exactly.
constexpr float LAZY = 8.f;
constexpr unsigned NOWHERE = 0x80000000u;  // a byte offset behind the end of every buffer (a tile spans less than 2 GiB)

// Eight elements of a matrix operand.  An fp32 number is the sum of three bf16 numbers: its upper 16 bits, what they leave
// over (less than 2^-7 of it) rounded to bf16, and the rest, which has 8 bits and is at most 2^-15 of it.  Six products
// of parts make the product of two such numbers up to 2^-21 of it: what is left out is the middle part of one times the
// last part of the other, twice, with random signs (2^-25 on the average); the matrix cores do the six in 3/8 of the time of one
// fp32 product.
// (The upper part is cut off, not rounded: no finite number becomes infinite.  An infinity leaves NaN over, see below.)  3525
// tokens in 4 sequences, 8 heads of 64, forward and backward: 225 us, with fp32 matrix instructions 366; errors 5.3e-7 and 7.0e-7 of
// the result on the same inputs.
struct Parts {
  bf16x8 p[3];
};
template <typename T>
struct FragOf;
template <>
struct FragOf<bf16_t> { typedef bf16x8 type, raw; };
template <>
struct FragOf<float> { typedef Parts type; typedef f32x8 raw; };
template <typename T>
using Frag = typename FragOf<T>::type;
template <typename T>
using Raw = typename FragOf<T>::raw;  // the elements as they are stored
template <typename T>
constexpr int PARTS = sizeof(T) == 2 ? 1 : 3;

__device__ __forceinline__ bf16x8 as_frag(const bf16x8 &x) { return x; }
__device__ __forceinline__ Parts as_frag(const f32x8 &x) {
  uint32_t w[3][4];
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    const uint32_t u0 = __float_as_uint(x[j]), u1 = __float_as_uint(x[j + 1]);
    w[0][j / 2] = __builtin_amdgcn_perm(u1, u0, 0x07060302u);  // both upper halves
    const f32x2 r = {x[j] - __uint_as_float(u0 & 0xffff0000u), x[j + 1] - __uint_as_float(u1 & 0xffff0000u)};
    w[1][j / 2] = __builtin_bit_cast(uint32_t, __builtin_convertvector(r, bf16x2));
    const f32x2 l = {r[0] - __uint_as_float(w[1][j / 2] << 16), r[1] - __uint_as_float(w[1][j / 2] & 0xffff0000u)};
    w[2][j / 2] = __builtin_bit_cast(uint32_t, __builtin_convertvector(l, bf16x2));
  }
  Parts f;
  __builtin_memcpy(f.p, w, sizeof(w));
  return f;
}
__device__ __forceinline__ bf16x8 choose(bool c, const bf16x8 &a, const bf16x8 &b) { return c ? a : b; }
__device__ __forceinline__ Parts choose(bool c, const Parts &a, const Parts &b) {
  return Parts{{c ? a.p[0] : b.p[0], c ? a.p[1] : b.p[1], c ? a.p[2] : b.p[2]}};
}
// element j alone, zeros beside it; all zeros unless `c`
__device__ __forceinline__ bf16x8 alone(bool c, int j, bf16x8 a) {
#pragma unroll
  for (int x = 0; x < 8; ++x) a[x] = c && x == j ? a[x] : (bf16x8{})[0];
  return a;
}
__device__ __forceinline__ Parts alone(bool c, int j, const Parts &a) {
  return Parts{{alone(c, j, a.p[0]), alone(c, j, a.p[1]), alone(c, j, a.p[2])}};
}

// c += A B over 16 k: lane l holds A[l % 32][8 * (l / 32) + j] and B[8 * (l / 32) + j][l % 32], j < 8.
__device__ __forceinline__ f32x16 mma(bf16x8 a, bf16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma(const Parts &a, const Parts &b, f32x16 c) {
  c = mma(a.p[2], b.p[0], c);
  c = mma(a.p[0], b.p[2], c);
  c = mma(a.p[1], b.p[1], c);
  c = mma(a.p[1], b.p[0], c);
  c = mma(a.p[0], b.p[1], c);
  return mma(a.p[0], b.p[0], c);
}
// ---- fp32 with infinities --------------------------------------------------------------------------------
// An infinity, or a product that overflows, makes NaN of the six products, whatever it should have become: the parts that it
// leaves over are NaN, or infinite with the other sign.  So a workgroup of the fp32 kernels that ends with a sum that is not
// finite begins again with products that take infinities apart, two to three times as slow and slower yet at the edge of a
// mask: the first parts alone tell whether a sum is infinite or NaN, and which; where it is neither, it is the sum of the
// six products without the elements that are not finite (a finite sum has none).  Calls with finite results pay for the check
// and for larger kernels: 3525 tokens, 8 heads of 64, forward and backward 232 -> 234 us, one image of 256 48 -> 49, 4
// queries over 12000 keys, 16/4 heads of 128, 37 -> 39.
__device__ __forceinline__ f32x8 quiet(f32x8 x) {  // a signaling NaN's upper half alone could be an infinity
#pragma unroll
  for (int j = 0; j < 8; ++j) x[j] = __builtin_canonicalizef(x[j]);
  return x;
}
__device__ __forceinline__ bf16x8 quiet(const bf16x8 &x) { return x; }
__device__ __forceinline__ Parts finite_part(Parts f) {
  uint32_t w[3][4];
  __builtin_memcpy(w, f.p, sizeof(w));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    asm volatile("" : "+v"(w[0][i]));  // not to be taken out of a loop: kept beside the operand itself it would fill the registers
    const uint32_t keep = ((w[0][i] & 0x7f80u) != 0x7f80u ? 0xffffu : 0u) | ((w[0][i] & 0x7f800000u) != 0x7f800000u ? 0xffff0000u : 0u);
#pragma unroll
    for (int k = 0; k < 3; ++k) w[k][i] &= keep;
  }
  __builtin_memcpy(f.p, w, sizeof(w));
  return f;
}
// A sum of products: `first` of the first parts, `rest` of all.
// (A template so that the bf16 kernels, which have no use for it, leave it alone.)
template <bool CAREFUL>
struct Sum {
  f32x16 first, rest;
};
template <bool CAREFUL>
__device__ __forceinline__ void mma(const Parts &a, const Parts &b, Sum<CAREFUL> &c) {
  c.first = mma(a.p[0], b.p[0], c.first);
  c.rest = mma(finite_part(a), finite_part(b), c.rest);
  __builtin_amdgcn_sched_barrier(0);  // one after the other: the operands of several would not fit the registers
}
template <bool CAREFUL>
__device__ __forceinline__ f32x16 total(const Sum<CAREFUL> &c) {
  f32x16 r;
#pragma unroll
  for (int i = 0; i < 16; ++i) r[i] = fabsf(c.first[i]) < INFINITY ? c.rest[i] : c.first[i];
  return r;
}
__device__ __forceinline__ f32x16 zero16() {
  f32x16 z;
#pragma unroll
  for (int i = 0; i < 16; ++i) z[i] = 0.f;
  return z;
}
// Weights of 16 rows as a B operand; bf16 rounds them.  Each is off by at most 2^-8 of itself, so the sum by no more than
// rounding the output once costs, and by less where many keys have a part in it.
template <typename T, bool CAREFUL = false>
__device__ __forceinline__ Frag<T> pack8(const f32x16 &w, int t) {
  Raw<T> f;
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    if constexpr (sizeof(T) == 2) {  // as pairs: one conversion instruction for two
      const bf16x2 p = __builtin_convertvector((f32x2{w[8 * t + j], w[8 * t + j + 1]}), bf16x2);
      f[j] = p[0], f[j + 1] = p[1];
    } else {
      f[j] = w[8 * t + j], f[j + 1] = w[8 * t + j + 1];
    }
  }
  if constexpr (CAREFUL) f = quiet(f);
  return as_frag(f);
}

// ---- division by the group size (rows -> queries), by a multiplication -------------------------------
struct Div {
  uint32_t mul, shift, by;
};
inline Div make_div(uint32_t by) {
  uint32_t s = 0;
  while ((1ull << s) < by) ++s;
  return Div{(uint32_t)((((1ull << s) - by) << 32) / by + 1), s, by};
}
__device__ __forceinline__ int div_by(int r, const Div &d) {  // r < 2^31
  return (int)((__umulhi((uint32_t)r, d.mul) + (uint32_t)r) >> d.shift);
}

// The wavefront's number in its workgroup, in a scalar register.
__device__ __forceinline__ int wave_index() { return __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)); }

// ---- arguments ------------------------------------------------------------------------------------------
template <typename T>
struct Args {
  const T *q, *k, *v, *o, *dout;
  T *out, *dq, *dk, *dv;
  i64 q_ld, k_ld, v_ld, o_ld, dout_ld, out_ld, dq_ld, dk_ld, dv_ld;
  float *lse, *partials;
  float *rows;  // for the dK/dV kernel: lse in base 2, then -delta, [total_q][Hq] each
  const int *cu_q, *cu_k;
  int num_seqs, total_q, total_k, Hq, Hkv, D, causal, tiles, splits;
  Div G;
  float scale, scale2;  // scale * log2(e)
};

// Bounds of a sequence, inside [0, total] whatever the array holds.
__device__ __forceinline__ int bound_of(const int *cu, int s, int total) { return min(max(cu[s], 0), total); }

struct Seq {
  int q0, nq, k0, nk;  // first query / key and their numbers
};
// The sequence of tile `tile` and the tile's first row in it, where sequence s owns the tiles from
// floor(start(s) * g / TILE) + s on (start in queries, or in keys where KEYS): at least ceil(len * g / TILE) of them,
// without a prefix sum over the lengths.  Tiles in front of the first or behind the last row of their sequence are
// empty.  The lanes look at 64 sequences at once: up to 63 sequences cost the latency of one load.
template <int TILE, bool KEYS, typename A>
__device__ __forceinline__ Seq locate(const A &a, int g, int tile, int &row0) {
  const int lane = threadIdx.x & 63;
  int lo = 0, q0, q1, k0, k1;
  if (a.num_seqs < 64) {
    const int s = min(lane, a.num_seqs), vq = bound_of(a.cu_q, s, a.total_q), vk = bound_of(a.cu_k, s, a.total_k);
    // bounds do not decrease: the sequences that begin at or before the tile are the first lanes
    lo = __popcll(__ballot(lane == 0 || (lane < a.num_seqs && ((KEYS ? vk : vq) * g) / TILE + lane <= tile))) - 1;
    q0 = __builtin_amdgcn_readlane(vq, lo), q1 = __builtin_amdgcn_readlane(vq, lo + 1);
    k0 = __builtin_amdgcn_readlane(vk, lo), k1 = __builtin_amdgcn_readlane(vk, lo + 1);
  } else {
    const int *const cu = KEYS ? a.cu_k : a.cu_q, total = KEYS ? a.total_k : a.total_q;
    for (int n = a.num_seqs; n > 1;) {
      const int step = (n + 63) >> 6, s = lo + lane * step;
      const bool before = lane == 0 || (s < lo + n && (bound_of(cu, s, total) * g) / TILE + s <= tile);
      const int skip = (__popcll(__ballot(before)) - 1) * step;
      n = min(step, n - skip);
      lo += skip;
    }
    lo = __builtin_amdgcn_readfirstlane(lo);
    q0 = bound_of(a.cu_q, lo, a.total_q), q1 = bound_of(a.cu_q, lo + 1, a.total_q);
    k0 = bound_of(a.cu_k, lo, a.total_k), k1 = bound_of(a.cu_k, lo + 1, a.total_k);
  }
  row0 = (tile - (((KEYS ? k0 : q0) * g) / TILE + lo)) * TILE;
  return Seq{q0, max(q1 - q0, 0), k0, max(k1 - k0, 0)};
}

// ---- tiles in LDS ----------------------------------------------------------------------------------------
// DP: elements that are computed with, a multiple of 32 (rows of 96 are stored like rows of 128); NW: wavefronts of the
// workgroup.  fp32: 16 rows of the first parts, then the same rows of the second and of the third.
template <typename T, int DP, int ROWS, int NW = WAVES>
struct Tile {
  static constexpr int RB = (DP == 96 ? 128 : DP) * 2, NC = RB / 16, CH = 8;  // of one part; 8 elements are a chunk
  static constexpr int PART = 16 * RB, R16 = PARTS<T> * PART;
  static constexpr int BYTES = ROWS / 16 * R16, NT = 64 * NW, PER = ROWS * NC / NT;
  static_assert(ROWS % 32 == 0 && ROWS * NC % NT == 0, "whole sub-tiles, whole chunks per thread");
  // 16 rows at one chunk (the reads along rows, 16 lanes at a time) and 4 rows of 64 bytes (the transposing reads, 32
  // lanes at a time) both cover the 256 bytes of a bank line.
  static __device__ __forceinline__ int key(int row) {
    if constexpr (RB == 64) return (row >> 2) & 3;
    else if constexpr (RB == 128) return ((row & 2) << 1) | ((row >> 2) & 3);
    else return ((row & 3) << 2) | ((row >> 2) & 3);
  }
  // Lane offsets: reads along a row (lane l: row l % 32, elements 16 t + 8 (l / 32) + j) and down 16 rows (lane l:
  // element 32 db + l % 32 of the rows 4 (l / 32) + j and 8 + 4 (l / 32) + j, j < 4).  t and db change bits of the chunk
  // number alone, so they are exclusive-ored into the offset.
  struct Lane {
    int row, down[2];
  };
  static __device__ __forceinline__ Lane lane_offsets(int lane) {
    Lane o;
    const int h = lane >> 5, l = lane & 31;
    o.row = (l >> 4) * R16 + (l & 15) * RB + (h ^ key(l)) * 16;
    const int q = (lane & 15) >> 2, p = lane & 3;  // a 16-lane group transposes 4 rows x 16 elements
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = 8 * i + 4 * h + q;
      o.down[i] = r * RB + ((2 * ((lane >> 4) & 1) + (p >> 1)) ^ key(r)) * 16 + (p & 1) * 8;
    }
    return o;
  }
  // The same offsets, but not known to be the same as before: the exclusive-ors are then taken again where they are used
  // instead of being kept in registers over the whole loop.
  static __device__ __forceinline__ Lane forget(Lane o) {
    asm volatile("" : "+v"(o.row));
#pragma unroll
    for (int &d : o.down) asm volatile("" : "+v"(d));
    return o;
  }
  static __device__ __forceinline__ Frag<T> along(const unsigned char *rows32, const Lane &o, int t) {
    const unsigned char *const at = rows32 + (o.row ^ (t * 32));
    if constexpr (sizeof(T) == 2) {
      return *reinterpret_cast<const bf16x8 *>(at);
    } else {
      return Parts{{*reinterpret_cast<const bf16x8 *>(at), *reinterpret_cast<const bf16x8 *>(at + PART),
                    *reinterpret_cast<const bf16x8 *>(at + 2 * PART)}};
    }
  }
  static __device__ __forceinline__ Frag<T> down(const unsigned char *rows16, const Lane &o, int db) {
    const unsigned char *const a = rows16 + (o.down[0] ^ (db * 64)), *const b = rows16 + (o.down[1] ^ (db * 64));
    if constexpr (sizeof(T) == 2) return tr_read_pair(a, b);
    else return Parts{{tr_read_pair(a, b), tr_read_pair(a + PART, b + PART), tr_read_pair(a + 2 * PART, b + 2 * PART)}};
  }
  // ---- memory -> LDS, whole 16-byte chunks (FAST): direct loads, a wavefront moves 1 KB per instruction.  The swizzle is
  // on the side of the memory address: lane l of a wavefront's instruction i fills chunk `slot` of the tile.
  static constexpr int MOVES = BYTES / 1024 / NW;
  static __device__ __forceinline__ int slot(int i) { return ((int)(threadIdx.x >> 6) * MOVES + i) * 64 + (int)(threadIdx.x & 63); }
  static __device__ __forceinline__ int slot_row(int i) { return slot(i) / NC; }
  // byte offset of the slot's chunk in its row, or beyond any buffer where the head has no such elements
  static __device__ __forceinline__ unsigned slot_chunk(int i, int D) {
    const int c = (slot(i) % NC) ^ key(slot_row(i));
    return c * CH < D ? (unsigned)c * 16u : NOWHERE;
  }
  // offset[i]: the byte offsets of this lane's chunks from `base`; chunks at or beyond `bytes` become zeros.
  static __device__ __forceinline__ void move(const T *base, i64 bytes, const unsigned (&offset)[MOVES], unsigned lds_tile) {
    const uint64_t b = (uint64_t)base;
    const i32x4 rsrc = {__builtin_amdgcn_readfirstlane((int)(unsigned)b), __builtin_amdgcn_readfirstlane((int)(b >> 32)),
                        __builtin_amdgcn_readfirstlane((int)(unsigned)max(min(bytes, (i64)NOWHERE), (i64)0)), 0x00020000};
#pragma unroll
    for (int i = 0; i < MOVES; ++i) {
      const unsigned at = __builtin_amdgcn_readfirstlane(lds_tile + ((threadIdx.x >> 6) * MOVES + i) * 1024u);
      asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                   :
                   : "s"(at), "v"(offset[i]), "s"(rsrc));
    }
  }

  // ---- memory -> registers -> LDS, any alignment and head dimension.  This thread's chunks of a tile on their way; row r
  // of the tile is row first + r of a sequence of n rows.  Rows and elements that do not exist become zeros.
  struct Chunks {
    Raw<T> c[PER];
  };
  template <typename Row>
  static __device__ __forceinline__ void fetch(Chunks &to, int first, int n, int D, Row row_ptr) {
    const int e = (threadIdx.x % NC) * CH, r0 = first + threadIdx.x / NC;
#pragma unroll
    for (int i = 0; i < PER; ++i) to.c[i] = Raw<T>{};
    if (first >= n) return;
    if (e < D) {
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const T *p = row_ptr(min(r0 + i * (NT / NC), n - 1)) + e;
        if (e + CH <= D) {
          __builtin_memcpy(&to.c[i], p, sizeof(Raw<T>));
        } else {
          T tmp[CH];
#pragma unroll
          for (int x = 0; x < CH; ++x) tmp[x] = e + x < D ? p[x] : (T)0;
          __builtin_memcpy(&to.c[i], tmp, sizeof(tmp));
        }
      }
    }
    if (first + ROWS > n)
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (r0 + i * (NT / NC) >= n) to.c[i] = Raw<T>{};
  }
  template <bool CAREFUL = false>
  static __device__ __forceinline__ void put(const Chunks &from, unsigned char *tile) {
    const int chunk = threadIdx.x % NC;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int r = threadIdx.x / NC + i * (NT / NC);
      unsigned char *const at = tile + (r >> 4) * R16 + (r & 15) * RB + (chunk ^ key(r)) * 16;
      const Frag<T> f = as_frag(CAREFUL ? quiet(from.c[i]) : from.c[i]);
#pragma unroll
      for (int k = 0; k < PARTS<T>; ++k) *reinterpret_cast<bf16x8 *>(at + k * PART) = reinterpret_cast<const bf16x8 *>(&f)[k];
    }
  }
  // Whether any of 32 rows of the tile holds an infinity or NaN.
  static __device__ __forceinline__ bool not_finite(const unsigned char *rows32, const Lane &o) {
    u16x2 top = {};  // of the magnitudes (fp32: of their upper halves)
#pragma unroll
    for (int t = 0; t < DP / 16; ++t) {
      const bf16x8 f = *reinterpret_cast<const bf16x8 *>(rows32 + (o.row ^ (t * 32)));
      uint32_t w[4];
      __builtin_memcpy(w, &f, sizeof(f));
#pragma unroll
      for (int i = 0; i < 4; ++i) top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, w[i] & 0x7fff7fffu));
    }
    return __any(top[0] >= 0x7f80u || top[1] >= 0x7f80u);
  }
  // acc[d][column] += sum over 32 rows of X[row][d] W[row][column].  edge: some rows are hidden from some columns, with
  // weight 0.  If such rows hold infinities or NaN, 0 * inf must not reach a column that does not see them: then the
  // rows are added one at a time, the result taken by the columns that see the row, and the common product reads
  // zeros instead.  Rare, so slow is fine; what matters is that the accumulators stay where they are.
  // TWICE: a bf16 weight is taken as the sum of two bf16 numbers, its rounding and what that left over.
  static constexpr int ZEROS = sizeof(T) == 2 ? 2 * R16 : R16;
  template <bool TWICE = false, typename Sees>
  static __device__ __forceinline__ void add(f32x16 (&acc)[DP / 32], const unsigned char *rows32, const unsigned char *zeros,
                                             const Lane &o, const f32x16 &w, bool edge, Sees sees) {
    const Frag<T> b0 = pack8<T>(w, 0), b1 = pack8<T>(w, 1);
    Frag<T> c0, c1;
    if constexpr (TWICE) {
      f32x16 rest;
#pragma unroll
      for (int i = 0; i < 16; ++i) rest[i] = w[i] - (float)(i < 8 ? b0[i & 7] : b1[i & 7]);
      c0 = pack8<T>(rest, 0), c1 = pack8<T>(rest, 1);
    }
    const unsigned char *low = rows32, *high = rows32 + R16;  // (bf16: low + R16 throughout, an offset in the instruction)
    if (edge && not_finite(rows32, o)) {
      const int h = (threadIdx.x & 63) >> 5;
#pragma unroll 1
      for (int k = 0; k < 32; ++k) {
        const int j = ((k >> 3) & 1) * 4 + (k & 3);
        const bool mine = ((k >> 2) & 1) == h, seen = sees(k);
        const Frag<T> b = choose(k < 16, b0, b1);
        Frag<T> c;
        if constexpr (TWICE) c = choose(k < 16, c0, c1);
#pragma unroll
        for (int db = 0; db < DP / 32; ++db) {
          const Frag<T> f = alone(mine, j, down(rows32 + (k >> 4) * R16, o, db));
          f32x16 r = mma(f, b, zero16());
          if constexpr (TWICE) r = mma(f, c, r);
#pragma unroll
          for (int i = 0; i < 16; ++i) acc[db][i] += seen ? r[i] : 0.f;
        }
      }
      low = high = zeros;
    }
#pragma unroll
    for (int db = 0; db < DP / 32; ++db) {
      const Frag<T> x = down(low, o, db);
      acc[db] = mma(x, b0, acc[db]);
      if constexpr (TWICE) acc[db] = mma(x, c0, acc[db]);
    }
#pragma unroll
    for (int db = 0; db < DP / 32; ++db) {
      const Frag<T> x = down(ZEROS > R16 ? low + R16 : high, o, db);
      acc[db] = mma(x, b1, acc[db]);
      if constexpr (TWICE) acc[db] = mma(x, c1, acc[db]);
    }
  }
  // The same with products that take infinities apart; at the edge of a mask row by row.
  template <typename Sees>
  static __device__ __forceinline__ void add_careful(f32x16 (&acc)[DP / 32], const unsigned char *rows32, const Lane &o, const f32x16 &w,
                                                     bool edge, Sees sees) {
    const Parts b0 = pack8<T, true>(w, 0), b1 = pack8<T, true>(w, 1);
    const int h = (threadIdx.x & 63) >> 5;
#pragma unroll 1
    for (int k = 0; k < 32; k += edge ? 1 : 16) {
      const int j = ((k >> 3) & 1) * 4 + (k & 3);
      const bool mine = ((k >> 2) & 1) == h, seen = !edge || sees(k);
      Parts b = choose(k < 16, b0, b1);
      if (edge) b = alone(mine, j, b);
#pragma unroll
      for (int db = 0; db < DP / 32; ++db) {
        Parts f = down(rows32 + (k >> 4) * R16, o, db);
        if (edge) f = alone(mine, j, f);
        Sum<true> c = {zero16(), zero16()};
        mma(f, b, c);
        const f32x16 r = total(c);
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[db][i] += seen ? r[i] : 0.f;
      }
    }
  }
  static __device__ __forceinline__ void clear(unsigned char *zeros) {
    for (int i = threadIdx.x * 16; i < ZEROS; i += NT * 16) *reinterpret_cast<u32x4 *>(zeros + i) = u32x4{0, 0, 0, 0};
  }
};

// Eight consecutive elements p[e..e+8) of a row of D, zero from element D on, as (half of) a B operand.  WHOLE: D is a
// multiple of 8; then without branches, from the row's first elements where there are none.
template <typename T, bool WHOLE>
__device__ __forceinline__ Raw<T> load_eight(const T *p, int e, int D) {
  Raw<T> f;
  const int n = D - e;
  if constexpr (WHOLE) {
    __builtin_memcpy(&f, p + (n > 0 ? e : 0), sizeof(f));
    if (n <= 0) f = Raw<T>{};
  } else if (n >= 8) {
    __builtin_memcpy(&f, p + e, sizeof(f));
  } else {
    T x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = i < n ? p[e + i] : (T)0;
    __builtin_memcpy(&f, x, sizeof(f));
  }
  return f;
}
template <typename T, bool WHOLE>
__device__ __forceinline__ Frag<T> load_frag(const T *p, int e, int D) {
  return as_frag(quiet(load_eight<T, WHOLE>(p, e, D)));
}
// Four consecutive results p[0..4), as many as n allows.
template <typename T>
__device__ __forceinline__ void store4(T *p, int n, float a, float b, float c, float d) {
  T e[4];
  from_f32(a, e[0]);
  from_f32(b, e[1]);
  from_f32(c, e[2]);
  from_f32(d, e[3]);
  if (n >= 4) {
    __builtin_memcpy(p, e, sizeof(e));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < n) p[i] = e[i];
  }
}
// acc[d][column] * f -> p[d] of the lane's column
template <typename T, int DP>
__device__ __forceinline__ void store_column(T *p, int D, const f32x16 (&acc)[DP / 32], float f, int db0 = 0,
                                             int db1 = DP / 32) {
  const int h = (threadIdx.x & 63) >> 5;
#pragma unroll
  for (int db = 0; db < DP / 32; ++db)
    if (db >= db0 && db < db1)
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const int d = 32 * db + 8 * b + 4 * h;
        store4(p + d, D - d, acc[db][4 * b] * f, acc[db][4 * b + 1] * f, acc[db][4 * b + 2] * f, acc[db][4 * b + 3] * f);
      }
}

// The queries of a workgroup: what the forward and the dQ kernel share.
struct Rows {
  Seq s;
  int nrows, off, row, query, head, lim;  // lim: last visible key of the lane's query, negative: none
  bool live;
};
template <int BQ, typename T>
__device__ __forceinline__ bool rows_of(const Args<T> &a, int tile, int kvh, int wave, Rows &r, int &row0) {
  const int g = (int)a.G.by;
  r.s = locate<BQ, false>(a, g, tile, row0);
  r.nrows = r.s.nq * g;
  if (row0 < 0 || row0 >= r.nrows) return false;
  r.off = r.s.nk - r.s.nq;
  r.row = row0 + wave * COLS + (threadIdx.x & 31);
  r.live = r.row < r.nrows;
  const int rr = min(r.row, r.nrows - 1);
  r.query = div_by(rr, a.G);
  r.head = kvh * g + (rr - r.query * g);
  r.lim = a.causal ? min(r.query + r.off, r.s.nk - 1) : r.s.nk - 1;
  return true;
}

// Streamed rows per tile of the gradient kernels.  WK wavefronts that share queries take 32 rows each; else 64, or 32 for
// rows of 192 bytes and more
//   - that go through registers: a thread then holds 16 of them for the tile that is on its way, and with 64 rows the
//     kernels with two streamed matrices and 64 or 128 accumulators spill;
//   - in fp32, whose tiles are three times as large.  (With 128 elements dQ and dK/dV spill registers all the same: dQ 5
//     and, for WK = 2, 25, nearly all outside the loop over finite tiles; dK/dV 54, some of them inside.)
template <typename T, int DP, bool FAST, int WK>
constexpr int tile_rows() {
  return WK > 1 ? 32 * WK : DP * sizeof(T) >= 192 && !FAST ? 32 : 64;
}

// Runs step(tile, buffer) for the tiles [0, n), the next tiles on their way to other buffers (or, where there is one
// buffer, in registers).  One barrier per tile: behind it every wavefront has left the buffer that is written next, and
// sees the one that is read next.  One buffer: two barriers, in front of its filling and behind it.
//   FAST: move(t, buffer) starts the direct loads of tile t, at least PER of them per wavefront, into one of NB buffers;
//         tile t is waited for in front of its barrier, while the NB - 2 tiles behind it may be in flight.  The loop has
//         no other vector memory instructions: a wait of the compiler's for one of those would be for all direct loads
//         as well.
//   else: fetch(t) loads tile t to registers, put(buffer) writes them to a buffer.
// `how` (a std::bool_constant) is handed on to put and step in front of their arguments.  True (see Sum): each tile is loaded
// when its turn comes, so that its registers are free for the step.
template <bool FAST, int NB, int PER, typename Move, typename Fetch, typename Put, typename Step, typename How>
__device__ __forceinline__ void stream(int n, Move move, Fetch fetch, Put put, Step step, How how) {
  static_assert(NB == 2 || NB == (FAST ? 3 : 1), "two buffers, or three for direct loads, or one for loads by registers");
  if (n <= 0) return;
  if constexpr (FAST) {
    move(0, 0);
    if (NB == 3 && n > 1) move(1, 1);
    int buf = 0;
#pragma unroll 1
    for (int t = 0; t < n; ++t) {
      if (NB == 3 && t + 1 < n) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(PER) : "memory");
      else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      const int free = buf == 0 ? NB - 1 : buf - 1;
      if (t + NB - 1 < n) move(t + NB - 1, free);
      step(how, t, buf);
      buf = buf == NB - 1 ? 0 : buf + 1;
    }
  } else if constexpr (How::value) {
#pragma unroll 1
    for (int t = 0; t < n; ++t) {
      fetch(t);
      __syncthreads();
      put(how, 0);
      __syncthreads();
      step(how, t, 0);
    }
  } else if constexpr (NB == 1) {
    fetch(0);
#pragma unroll 1
    for (int t = 0; t < n; ++t) {
      if (t) __syncthreads();
      put(how, 0);
      __syncthreads();
      fetch(t + 1);
      step(how, t, 0);
    }
  } else {
    fetch(0);
    put(how, 0);
    fetch(1);
#pragma unroll 1
    for (int t = 0; t < n; ++t) {
      __syncthreads();
      if (t + 1 < n) {
        put(how, (t + 1) & 1);
        fetch(t + 2);
      }
      step(how, t, t & 1);
    }
  }
}
// Buffers: three where the LDS of two or three workgroups a CU has room for them.  Short sequences spend their time
// waiting for the first tiles: 16 x 256 tokens, 16 heads of 64, bf16, the backward's kernels together 40.7 us with three,
// 41.7 with two, and the forward 13.0 with either.  One for the long tiles of fp32 where wavefronts share queries: two
// workgroups a CU (3525 tokens, 8 heads of 64: forward 57 us, with two buffers and one workgroup 90; or no room for more).
template <typename T, int DP, bool FAST, int WK>
constexpr int buffers() { return FAST && DP <= 64 && WK < 4 ? 3 : sizeof(T) == 4 && WK > 1 ? 1 : 2; }

// Whether the registers are to be limited so that two workgroups fit a CU.  The LDS of WK = 4 at rows of 256 bytes and
// more, and the operands of fp32 at 96 elements and more, allow one.
template <typename T, int DP, int WK>
constexpr bool two_fit() { return sizeof(T) == 2 ? WK < 4 || DP <= 64 : WK <= 2 && DP <= 64; }

// The sums of the wavefronts that share queries, each times its factor, for the blocks [db0, db1) of 32 elements: `all`
// holds value i of block db of thread t at [(first + db * 16 + i) * NT + t], NT threads.
template <int NT, int DB>
__device__ __forceinline__ void leave_sums(float *mine, const f32x16 (&acc)[DB], int first) {
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int i = 0; i < 16; ++i) mine[(first + db * 16 + i) * NT] = acc[db][i];
}
template <int WK, int NT, int DB>
__device__ __forceinline__ void join_sums(f32x16 (&acc)[DB], const float *all, int first, const float (&f)[WK], int db0, int db1) {
#pragma unroll
  for (int db = 0; db < DB; ++db)
    if (db >= db0 && db < db1)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < WK; ++w) v += f[w] * all[(first + db * 16 + i) * NT + w * (NT / WK)];
        acc[db][i] = v;
      }
}

// LDS[lds + 4 * lane] = the number at byte offset `at` from base, 0 at NOWHERE.
__device__ __forceinline__ void direct_load_dword(const float *base, unsigned at, unsigned lds) {
  const uint64_t b = (uint64_t)base;
  const i32x4 rsrc = {__builtin_amdgcn_readfirstlane((int)(unsigned)b), __builtin_amdgcn_readfirstlane((int)(b >> 32)),
                      (int)NOWHERE, 0x00020000};
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds"
               :
               : "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(at), "s"(rsrc));
}
// 0, or NaN if a sum is not finite.
template <int DB>
__device__ __forceinline__ float finite_check(const f32x16 (&acc)[DB]) {
  float z[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int i = 0; i < 16; ++i) z[i & 3] += acc[db][i] * 0.f;
  return (z[0] + z[1]) + (z[2] + z[3]);
}
// Whether that is NaN in any thread of the workgroup.  Behind its barrier no tile is read any more.  `flags`: NW words of LDS
// for this alone, once a kernel.
template <int NW>
__device__ __forceinline__ bool anywhere(float z, int *flags) {
  flags[threadIdx.x >> 6] = __any(z != 0.f) ? 1 : 0;
  __syncthreads();
  int any = 0;
#pragma unroll
  for (int w = 0; w < NW; ++w) any |= flags[w];
  return __builtin_amdgcn_readfirstlane(any);
}
// Where a workgroup's LDS array begins, as the direct loads want it.
__device__ __forceinline__ unsigned lds_address(unsigned char *lds) {
  return (unsigned)(uintptr_t)(__attribute__((address_space(3))) unsigned char *)lds;
}

// Keys and values of a sequence, tile by tile, for the kernels that stream them.
template <typename T, typename TL, bool FAST>
struct KeyTiles {
  const T *k, *v;
  i64 k_ld, v_ld;
  int D;
  unsigned ko[TL::MOVES], vo[TL::MOVES];
  typename TL::Chunks ck, cv;
  __device__ __forceinline__ KeyTiles(const Args<T> &a, const Seq &s, int kvh)
      : k(a.k + (i64)s.k0 * a.k_ld + kvh * a.D), v(a.v + (i64)s.k0 * a.v_ld + kvh * a.D), k_ld(a.k_ld), v_ld(a.v_ld), D(a.D) {
    if constexpr (FAST)
#pragma unroll
      for (int i = 0; i < TL::MOVES; ++i) {
        const unsigned c = TL::slot_chunk(i, D);
        ko[i] = c == NOWHERE ? c : TL::slot_row(i) * (unsigned)k_ld * (unsigned)sizeof(T) + c;
        vo[i] = c == NOWHERE ? c : TL::slot_row(i) * (unsigned)v_ld * (unsigned)sizeof(T) + c;
      }
  }
  // the tile whose first key is `first`, keys [0, end)
  __device__ __forceinline__ void move(int first, int end, unsigned lds_k, unsigned lds_v) {
    const i64 rows = end - first - 1;  // behind the last row's elements, in front of the next row's
    TL::move(k + first * k_ld, rows < 0 ? 0 : (rows * k_ld + D) * (i64)sizeof(T), ko, lds_k);
    TL::move(v + first * v_ld, rows < 0 ? 0 : (rows * v_ld + D) * (i64)sizeof(T), vo, lds_v);
  }
  __device__ __forceinline__ void fetch(int first, int end) {
    TL::fetch(ck, first, end, D, [&](int j) __attribute__((always_inline)) { return k + j * k_ld; });
    TL::fetch(cv, first, end, D, [&](int j) __attribute__((always_inline)) { return v + j * v_ld; });
  }
  template <bool CAREFUL>
  __device__ __forceinline__ void put(unsigned char *lds_k, unsigned char *lds_v) {
    TL::template put<CAREFUL>(ck, lds_k);
    TL::template put<CAREFUL>(cv, lds_v);
  }
};

// Which keys the queries of a workgroup and of this wavefront see (all of them / at least one of them).
struct Span {
  int kend;                 // keys [0, kend) are seen by the workgroup
  int all;                  // keys [0, all] by every query of the workgroup
  int wave_all, wave_some;  // keys [0, wave_all] by every, [0, wave_some] by some query of the wavefront
};
template <int BQ, typename T>
__device__ __forceinline__ Span span_of(const Args<T> &a, const Rows &r, int row0, int wave) {
  const int last = r.s.nk - 1;
  if (!a.causal) return Span{r.s.nk, last, last, last};
  auto sees = [&](int row) __attribute__((always_inline)) { return min(div_by(min(row, r.nrows - 1), a.G) + r.off, last); };
  Span s;
  s.kend = max(sees(row0 + BQ - 1) + 1, 0);
  s.all = sees(row0);
  s.wave_all = sees(row0 + wave * COLS);
  s.wave_some = row0 + wave * COLS < r.nrows ? sees(row0 + wave * COLS + COLS - 1) : -1;
  return s;
}

// The forward.  WK wavefronts share the same 32 queries and take the 32-row pieces of a tile in turn: with WK = 1 a
// workgroup has 128 queries (every tile serves four times 32), with WK > 1 it has fewer, for calls that have too few
// queries to fill the GPU.  NW = 8: twice as many (see Plan for when).  splits > 1: the
// workgroup takes a share of the key tiles and leaves its sums to attention_join_kernel.
template <typename T, int DP, bool FAST, int WK, int NW = WAVES>
__global__ __launch_bounds__(64 * NW, (two_fit<T, DP, WK>() && (sizeof(T) == 2 || NW == WAVES) ? 2 : 1)) void attention_kernel(const Args<T> a) {
  constexpr int WQ = NW / WK, BQ = COLS * WQ, ROWS = sizeof(T) == 2 && WK == 1 ? 64 : tile_rows<T, DP, FAST, WK>();
  constexpr int NU = WK == 1 ? ROWS / 32 : 1, DB = DP / 32;
  typedef Tile<T, DP, ROWS, NW> TL;
  constexpr int NB = NW == 8 ? 2 : buffers<T, DP, FAST, WK>(), STAGE = 2 * TL::BYTES, MERGE = WK == 1 ? 0 : 64 * NW * (DB * 16 + 2) * 4;
  __shared__ __align__(16) unsigned char lds[(NB * STAGE > MERGE ? NB * STAGE : MERGE) + TL::ZEROS];
  __shared__ int flags[sizeof(T) == 4 ? NW : 1];
  unsigned char *const zeros = lds + sizeof(lds) - TL::ZEROS;
  const int lane = threadIdx.x & 63, h = lane >> 5, wave = wave_index(), wq = wave % WQ, wk = wave / WQ;
  const int kvh = blockIdx.x % a.Hkv, bs = blockIdx.x / a.Hkv, split = bs % a.splits, t0 = bs / a.splits;
  const int tile = a.causal ? a.tiles - 1 - t0 : t0;  // the queries with the most keys first
  Rows r;
  int row0;
  if (!rows_of<BQ>(a, tile, kvh, wq, r, row0)) return;
  TL::clear(zeros);
  const auto lo = TL::lane_offsets(lane);
  const Span span = span_of<BQ>(a, r, row0, wq);

  Frag<T> q[DP / 16];
  {
    const T *p = a.q + (i64)(r.s.q0 + r.query) * a.q_ld + r.head * a.D;
#pragma unroll
    for (int t = 0; t < DP / 16; ++t) q[t] = load_frag<T, FAST>(p, 16 * t + 8 * h, a.D);
  }
  f32x16 acc[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db) acc[db] = zero16();
  // m: the reference, at most `lift` above the largest score times scale2 (base 2); l: over this lane's rows only
  float m = -INFINITY, l = 0.f;
  const float lift = LAZY + (float)(32 - __builtin_clz(max(r.s.nk, 1)));

  int first = 0, n = (span.kend + ROWS - 1) / ROWS;  // key tiles
  if (a.splits > 1) {
    const int per = (n + a.splits - 1) / a.splits;
    first = min(split * per, n);
    n = min(per, n - first);
  }
  KeyTiles<T, TL, FAST> keys(a, r.s, kvh);
  const unsigned lds0 = lds_address(lds);
  const int end = min(span.kend, (first + n) * ROWS);
  auto move = [&](int t, int buf) __attribute__((always_inline)) {
    if constexpr (FAST) keys.move((first + t) * ROWS, end, lds0 + buf * STAGE, lds0 + buf * STAGE + TL::BYTES);
  };
  auto fetch = [&](int t) __attribute__((always_inline)) {
    if (!FAST) keys.fetch((first + t) * ROWS, end);
  };
  auto put = [&](auto careful, int buf) __attribute__((always_inline)) {
    if (!FAST) keys.template put<decltype(careful)::value>(lds + buf * STAGE, lds + buf * STAGE + TL::BYTES);
  };
  auto step = [&](auto careful, int t, int buf) __attribute__((always_inline)) {
    constexpr bool CAREFUL = decltype(careful)::value;
    const int key0 = (first + t) * ROWS + wk * 32;
    if (key0 > span.wave_some) return;
    const unsigned char *const ldsK = lds + buf * STAGE + wk * 2 * TL::R16, *const ldsV = ldsK + TL::BYTES;
    const bool edge = key0 + NU * 32 - 1 > span.wave_all;
    f32x16 s[NU];
    if constexpr (CAREFUL) {
#pragma unroll
      for (int u = 0; u < NU; ++u) {
        Sum<CAREFUL> c = {zero16(), zero16()};
#pragma unroll
        for (int x = 0; x < DP / 16; ++x) mma(TL::along(ldsK + u * 2 * TL::R16, lo, x), q[x], c);
        s[u] = total(c);
      }
    } else {
#pragma unroll
      for (int u = 0; u < NU; ++u) s[u] = zero16();
#pragma unroll
      for (int x = 0; x < DP / 16; ++x)  // the pieces in turn: no product waits for the one in front of it
#pragma unroll
        for (int u = 0; u < NU; ++u) s[u] = mma(TL::along(ldsK + u * 2 * TL::R16, lo, x), q[x], s[u]);
    }
    if (edge) {
#pragma unroll
      for (int u = 0; u < NU; ++u) {
        const int rel = r.lim - (key0 + u * 32) - 4 * h;
#pragma unroll
        for (int i = 0; i < 16; ++i) s[u][i] = 8 * (i / 4) + i % 4 <= rel ? s[u][i] : -INFINITY;
      }
    }
    float top = s[0][0];
#pragma unroll
    for (int u = 0; u < NU; ++u)
#pragma unroll
      for (int i = 0; i < 16; ++i) top = fmaxf(top, s[u][i]);
    top = top * a.scale2 + lift;
    if (__any(top > m + LAZY)) {
      const float m_new = fmaxf(m, fmaxf(top, __shfl_xor(top, 32, 64)));
      const float f = m_new == m ? 1.f : __builtin_amdgcn_exp2f(m - m_new);
      m = m_new;
      l *= f;
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[db][i] *= f;
    }
    const float base = m == -INFINITY ? 0.f : m;  // nothing but -inf so far: every weight is 0
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int u = 0; u < NU; ++u)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[u][i] = __builtin_amdgcn_exp2f(s[u][i] * a.scale2 - base);
        sum[i & 3] += s[u][i];
      }
    l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      const int kb = key0 + u * 32;
      auto sees = [&](int k) __attribute__((always_inline)) { return kb + k <= r.lim; };
      if constexpr (CAREFUL) TL::add_careful(acc, ldsV + u * 2 * TL::R16, lo, s[u], edge, sees);
      else TL::add(acc, ldsV + u * 2 * TL::R16, zeros, lo, s[u], edge && kb + 31 > span.wave_all, sees);
    }
  };
  stream<FAST, NB, 2 * TL::MOVES>(n, move, fetch, put, step, std::false_type());
  if constexpr (sizeof(T) == 4)
    if (anywhere<NW>(l * 0.f + finite_check(acc), flags)) {
#pragma unroll
      for (int db = 0; db < DB; ++db) acc[db] = zero16();
      m = -INFINITY, l = 0.f;
      stream<FAST, NB, 2 * TL::MOVES>(n, move, fetch, put, step, std::true_type());
    }
  l += __shfl_xor(l, 32, 64);
  int db0 = 0, db1 = DB;  // the blocks of 32 elements that this wavefront writes
  if constexpr (WK > 1) {
    // Join the sums of the wavefronts that share queries; each takes a part of the blocks.
    __syncthreads();
    float *const mine = reinterpret_cast<float *>(lds) + threadIdx.x;
    mine[0] = m;
    mine[64 * NW] = l;
    leave_sums<64 * NW>(mine, acc, 2);
    __syncthreads();
    const float *const all = reinterpret_cast<const float *>(lds) + wq * 64 + lane;
    float f[WK];
    m = -INFINITY, l = 0.f;
#pragma unroll
    for (int w = 0; w < WK; ++w) m = fmaxf(m, all[w * WQ * 64]);
#pragma unroll
    for (int w = 0; w < WK; ++w) {
      f[w] = __builtin_amdgcn_exp2f(all[w * WQ * 64] - (m == -INFINITY ? 0.f : m));
      l += f[w] * all[64 * NW + w * WQ * 64];
    }
    db0 = min(wk * ((DB + WK - 1) / WK), DB);
    db1 = min(db0 + (DB + WK - 1) / WK, DB);
    join_sums<WK, 64 * NW>(acc, all, 2, f, db0, db1);
  }
  if (!r.live) return;
  const i64 at = (i64)(r.s.q0 + r.query) * a.Hq + r.head;
  if (a.splits > 1) {
    const i64 plane = (i64)a.total_q * a.Hq;
    store_column<float, DP>(a.partials + (split * plane + at) * a.D, a.D, acc, 1.f, db0, db1);
    if (h == 0 && wk == 0) {
      float *const ml = a.partials + a.splits * plane * a.D + 2 * (split * plane + at);
      ml[0] = m;
      ml[1] = r.lim < 0 ? -1.f : l;  // a sum cannot be negative: the mark of a query that sees no key
    }
    return;
  }
  store_column<T, DP>(a.out + (i64)(r.s.q0 + r.query) * a.out_ld + r.head * a.D, a.D, acc, r.lim < 0 ? 0.f : 1.f / l, db0, db1);
  if (a.lse && h == 0 && wk == 0) a.lse[at] = r.lim < 0 ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * LN2;
}

// out and lse from the sums over the shares of the keys: one wavefront per query and head.
template <typename T>
__global__ __launch_bounds__(256) void attention_join_kernel(const Args<T> a) {
  const int q0 = bound_of(a.cu_q, 0, a.total_q), q1 = bound_of(a.cu_q, a.num_seqs, a.total_q), lane = threadIdx.x & 63;
  const i64 at = (i64)q0 * a.Hq + (i64)blockIdx.x * WAVES + (threadIdx.x >> 6), plane = (i64)a.total_q * a.Hq;
  if (at >= (i64)q1 * a.Hq) return;
  const float *const ml = a.partials + a.splits * plane * a.D + 2 * at;
  // lane s: the weight of share s (there are at most 64); then the lanes take the elements
  const float m_s = lane < a.splits ? ml[2 * lane * plane] : -INFINITY, l_s = lane < a.splits ? ml[2 * lane * plane + 1] : 0.f;
  const bool none = ml[1] < 0.f;
  float m = m_s;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
  const float f_s = __builtin_amdgcn_exp2f(m_s - (m == -INFINITY ? 0.f : m));
  const float l = wave_sum(f_s * l_s);
  float v0 = 0.f, v1 = 0.f;
  const float *p = a.partials + at * a.D;
  const int e0 = min(lane, a.D - 1), e1 = min(lane + 64, a.D - 1);
  for (int s0 = 0; s0 < a.splits; s0 += 8)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float f = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(f_s), s0 + j));
      const float *const ps = p + min(s0 + j, a.splits - 1) * (plane * a.D);
      const float x0 = f * ps[e0], x1 = f * ps[e1];
      v0 += s0 + j < a.splits ? x0 : 0.f;
      v1 += s0 + j < a.splits ? x1 : 0.f;
    }
  const i64 token = at / a.Hq, head = at - token * a.Hq;
  T *const o = a.out + token * a.out_ld + head * a.D;
  const float r = none ? 0.f : 1.f / l;
  if (lane < a.D) from_f32(none ? 0.f : v0 * r, o[lane]);
  if (lane + 64 < a.D) from_f32(none ? 0.f : v1 * r, o[lane + 64]);
  if (a.lse && lane == 0) a.lse[at] = none ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * LN2;
}

// dQ, and lse and delta for the kernel below.  WK and splits as in the forward.
template <typename T, int DP, bool FAST, int WK>
__global__ __launch_bounds__(256, (two_fit<T, DP, WK>() ? 2 : 1)) void attention_dq_kernel(const Args<T> a) {
  constexpr int WQ = WAVES / WK, BQ = COLS * WQ, ROWS = tile_rows<T, DP, FAST, WK>(), NU = WK == 1 ? ROWS / 32 : 1, DB = DP / 32;
  typedef Tile<T, DP, ROWS> TL;
  constexpr int NB = buffers<T, DP, FAST, WK>(), STAGE = 2 * TL::BYTES, MERGE = WK == 1 ? 0 : 256 * DB * 16 * 4;
  __shared__ __align__(16) unsigned char lds[(NB * STAGE > MERGE ? NB * STAGE : MERGE) + TL::ZEROS];
  __shared__ int flags[sizeof(T) == 4 ? WAVES : 1];
  unsigned char *const zeros = lds + sizeof(lds) - TL::ZEROS;
  const int lane = threadIdx.x & 63, h = lane >> 5, wave = wave_index(), wq = wave % WQ, wk = wave / WQ;
  const int kvh = blockIdx.x % a.Hkv, bs = blockIdx.x / a.Hkv, split = bs % a.splits, t0 = bs / a.splits;
  const int tile = a.causal ? a.tiles - 1 - t0 : t0;
  Rows r;
  int row0;
  if (!rows_of<BQ>(a, tile, kvh, wq, r, row0)) return;
  TL::clear(zeros);
  const auto lo = TL::lane_offsets(lane);
  const Span span = span_of<BQ>(a, r, row0, wq);

  Frag<T> q[DP / 16], dout[DP / 16];
  float delta = 0.f;
  {
    const i64 token = r.s.q0 + r.query;
    const T *p = a.q + token * a.q_ld + r.head * a.D, *pd = a.dout + token * a.dout_ld + r.head * a.D,
            *po = a.o + token * a.o_ld + r.head * a.D;
#pragma unroll
    for (int t = 0; t < DP / 16; ++t) {
      const int e = 16 * t + 8 * h;
      q[t] = load_frag<T, FAST>(p, e, a.D);
      const Raw<T> d = quiet(load_eight<T, FAST>(pd, e, a.D)), o = load_eight<T, FAST>(po, e, a.D);
      dout[t] = as_frag(d);
#pragma unroll
      for (int j = 0; j < 8; ++j) delta += (float)d[j] * (float)o[j];
    }
    delta += __shfl_xor(delta, 32, 64);
  }
  const float stored_delta = delta;
  const i64 at = (i64)(r.s.q0 + r.query) * a.Hq + r.head;
  const float lse2 = a.lse[at] * LOG2E;  // (a row that does not exist repeats the last one and is not stored)

  f32x16 acc[DP / 32];
#pragma unroll
  for (int db = 0; db < DP / 32; ++db) acc[db] = zero16();
  KeyTiles<T, TL, FAST> keys(a, r.s, kvh);
  const unsigned lds0 = lds_address(lds);
  int first = 0, n = (span.kend + ROWS - 1) / ROWS;  // key tiles
  if (a.splits > 1) {
    const int per = (n + a.splits - 1) / a.splits;
    first = min(split * per, n);
    n = min(per, n - first);
  }
  const int end = min(span.kend, (first + n) * ROWS);
  auto move = [&](int t, int buf) __attribute__((always_inline)) {
    if constexpr (FAST) keys.move((first + t) * ROWS, end, lds0 + buf * STAGE, lds0 + buf * STAGE + TL::BYTES);
  };
  auto fetch = [&](int t) __attribute__((always_inline)) {
    if (!FAST) keys.fetch((first + t) * ROWS, end);
  };
  auto put = [&](auto careful, int buf) __attribute__((always_inline)) {
    if (!FAST) keys.template put<decltype(careful)::value>(lds + buf * STAGE, lds + buf * STAGE + TL::BYTES);
  };
  auto step = [&](auto careful, int t, int buf) __attribute__((always_inline)) {
    constexpr bool CAREFUL = decltype(careful)::value;
    constexpr int UNROLL = sizeof(T) == 2 ? 2 : 1;
    const unsigned char *const ldsK = lds + buf * STAGE + wk * 2 * TL::R16, *const ldsV = ldsK + TL::BYTES;
#pragma unroll UNROLL  // two pieces share their addresses
    for (int u = 0; u < NU; ++u) {
      const int kb = (first + t) * ROWS + (wk + u) * 32;
      if (kb > span.wave_some) break;
      const unsigned char *const k32 = ldsK + u * 2 * TL::R16, *const v32 = ldsV + u * 2 * TL::R16;
      f32x16 s = zero16(), dp = zero16();
      if constexpr (CAREFUL) {
        Sum<CAREFUL> c = {s, s};
#pragma unroll
        for (int x = 0; x < DP / 16; ++x) mma(TL::along(k32, lo, x), q[x], c);
        s = total(c);
        c = {dp, dp};
#pragma unroll
        for (int x = 0; x < DP / 16; ++x) mma(TL::along(v32, lo, x), dout[x], c);
        dp = total(c);
      } else {
#pragma unroll
        for (int x = 0; x < DP / 16; ++x) {
          s = mma(TL::along(k32, lo, x), q[x], s);
          dp = mma(TL::along(v32, lo, x), dout[x], dp);
        }
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = __builtin_amdgcn_exp2f(s[i] * a.scale2 - lse2);
      const bool edge = kb + 31 > span.wave_all;
      if (edge) {
        const int rel = r.lim - kb - 4 * h;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          s[i] = 8 * (i / 4) + i % 4 <= rel ? s[i] : 0.f;
          dp[i] = 8 * (i / 4) + i % 4 <= rel ? dp[i] : 0.f;
        }
      }
      if (kb == 0 && span.wave_all < 32) {  // (the first query sees the fewest keys)
        // A query whose keys all lie here has its delta from the weights themselves: dout * out takes out as it was
        // stored, rounded, and with few keys, where out is large, that would be the largest error of dS.
        float d = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) d += s[i] * dp[i];
        d += __shfl_xor(d, 32, 64);
        delta = r.lim < 32 ? d : delta;
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] *= dp[i] - delta;
      // dS of a query adds up to zero, so its product with K loses the part that the keys have in common, but the
      // roundings of dS do not: with few elements (that part is then large beside the rest) they are kept out.  (16 x 256
      // tokens, 16 heads of 64: 21.2 us instead of 18.9, and an error of 1.0 instead of 1.45 output roundings.)
      auto sees = [&](int k) __attribute__((always_inline)) { return kb + k <= r.lim; };
      if constexpr (CAREFUL) TL::add_careful(acc, k32, lo, s, edge, sees);
      else TL::template add<sizeof(T) == 2 && DP <= 64>(acc, k32, zeros, lo, s, edge, sees);
    }
  };
  stream<FAST, NB, 2 * TL::MOVES>(n, move, fetch, put, step, std::false_type());
  if constexpr (sizeof(T) == 4)
    if (anywhere<WAVES>(finite_check(acc), flags)) {
#pragma unroll
      for (int db = 0; db < DP / 32; ++db) acc[db] = zero16();
      delta = stored_delta;
      stream<FAST, NB, 2 * TL::MOVES>(n, move, fetch, put, step, std::true_type());
    }
  int db0 = 0, db1 = DB;  // the blocks of 32 elements that this wavefront writes
  if constexpr (WK > 1) {
    __syncthreads();
    leave_sums<256>(reinterpret_cast<float *>(lds) + threadIdx.x, acc, 0);
    __syncthreads();
    float f[WK];
#pragma unroll
    for (int w = 0; w < WK; ++w) f[w] = 1.f;
    db0 = min(wk * ((DB + WK - 1) / WK), DB);
    db1 = min(db0 + (DB + WK - 1) / WK, DB);
    join_sums<WK, 256>(acc, reinterpret_cast<const float *>(lds) + wq * 64 + lane, 0, f, db0, db1);
  }
  if (!r.live) return;
  const i64 plane = (i64)a.total_q * a.Hq;
  if (h == 0 && wk == 0 && split == 0) {  // the wavefront that has seen the first keys
    a.rows[at] = lse2;
    a.rows[at + plane] = -delta;
  }
  if (a.splits > 1) {
    store_column<float, DP>(a.partials + (split * plane + at) * a.D, a.D, acc, a.scale, db0, db1);
    return;
  }
  store_column<T, DP>(a.dq + (i64)(r.s.q0 + r.query) * a.dq_ld + r.head * a.D, a.D, acc, a.scale, db0, db1);
}

// dQ from its sums over the shares of the keys, in their order.
template <typename T>
__global__ __launch_bounds__(256) void attention_dq_join_kernel(const Args<T> a) {
  const int q0 = bound_of(a.cu_q, 0, a.total_q), q1 = max(bound_of(a.cu_q, a.num_seqs, a.total_q), q0);
  const int cols = a.Hq * a.D;
  const i64 plane = (i64)a.total_q * cols, end = (i64)q1 * cols;
  for (i64 i = (i64)q0 * cols + (i64)blockIdx.x * 256 + threadIdx.x; i < end; i += (i64)gridDim.x * 256) {
    float dq = 0.f;
    for (int s = 0; s < a.splits; ++s) dq += a.partials[s * plane + i];
    const i64 query = i / cols;
    from_f32(dq, a.dq[query * a.dq_ld + i - query * cols]);
  }
}

// dK and dV: keys in registers, the packed queries of the group streamed.
template <typename T, int DP, bool FAST, int NW>
__global__ __launch_bounds__(64 * NW, (sizeof(T) == 2 || DP <= 64 ? 2 : 1)) void attention_dkv_kernel(const Args<T> a) {
  constexpr int ROWS = tile_rows<T, DP, FAST, 1>();
  typedef Tile<T, DP, ROWS, NW> TL;
  constexpr int STAGE = 2 * TL::BYTES + 2 * 64 * 4;  // Q, dout, lse (base 2), delta (64 values: a wavefront's direct load)
  constexpr int NB = sizeof(T) == 4 ? 1 : buffers<T, DP, FAST, 1>();
  // bf16, 128 elements: 128 accumulators, 32 scores and 32 of K leave no room for V in 256 registers.  Its operands, and
  // the last two of K, stay in LDS, each wavefront's own, in the order in which the lanes read them.  (With six more
  // registers in use one operand is reloaded from scratch memory in every step, behind the direct loads in flight: 25 %
  // slower.)  fp32 behind 32 elements: V's three parts, and one buffer, so that up to 64 elements two workgroups fit a CU
  // (3525 tokens, 8 heads of 64: backward 191 us with one, 174 with two; 2048 tokens, 8 heads of 128: 522 -> 371).
  constexpr bool ALL_REG = sizeof(T) == 2 ? DP < 128 : DP <= 32;
  constexpr int KT = DP / 16, K_REG = ALL_REG || sizeof(T) == 4 ? KT : KT - 2, V_REG = ALL_REG ? KT : 0;
  constexpr int OWN = (2 * KT - K_REG - V_REG) * 64 * (int)sizeof(Frag<T>);
  __shared__ __align__(16) unsigned char lds[NB * STAGE + TL::ZEROS + NW * OWN];
  __shared__ int flags[sizeof(T) == 4 ? NW : 1];
  unsigned char *const zeros = lds + NB * STAGE;
  const int kvh = blockIdx.x % a.Hkv, bs = blockIdx.x / a.Hkv, split = bs % a.splits;
  int key0;
  const Seq s = locate<COLS * NW, true>(a, 1, bs / a.splits, key0);
  if (key0 < 0 || key0 >= s.nk) return;
  TL::clear(zeros);
  const int lane = threadIdx.x & 63, h = lane >> 5, wave = wave_index();
  const auto lane_at = TL::lane_offsets(lane);
  const int g = (int)a.G.by, off = s.nk - s.nq;
  const int wkey = key0 + wave * COLS, key = wkey + (lane & 31);
  const bool live = key < s.nk;

  Frag<T> kr[K_REG], vr[V_REG ? V_REG : 1];
  Frag<T> *const own = reinterpret_cast<Frag<T> *>(lds + NB * STAGE + TL::ZEROS + wave * OWN) + lane;
  {
    const i64 token = s.k0 + min(key, s.nk - 1);
    const T *pk = a.k + token * a.k_ld + kvh * a.D, *pv = a.v + token * a.v_ld + kvh * a.D;
#pragma unroll
    for (int t = 0; t < KT; ++t) {
      const Frag<T> fk = load_frag<T, FAST>(pk, 16 * t + 8 * h, a.D), fv = load_frag<T, FAST>(pv, 16 * t + 8 * h, a.D);
      if (t < K_REG) kr[t] = fk;
      else own[64 * (KT - V_REG + t - K_REG)] = fk;
      if (t < V_REG) vr[t] = fv;
      else own[64 * (t - V_REG)] = fv;
    }
  }
  f32x16 dk[DP / 32], dv[DP / 32];
#pragma unroll
  for (int db = 0; db < DP / 32; ++db) dk[db] = dv[db] = zero16();

  // the rows that see a key: from the first query that sees the first key of the workgroup / the last one of the wavefront
  int first = a.causal ? min(max(key0 - off, 0), s.nq) * g : 0, nrows = s.nq * g;
  if (a.splits > 1) {  // this workgroup's share of them
    const int per = (((nrows - first + ROWS - 1) / ROWS + a.splits - 1) / a.splits) * ROWS;
    first = (int)min((i64)nrows, first + (i64)split * per);
    nrows = (int)min((i64)nrows, (i64)first + per);
  }
  const int wave_some = a.causal ? min(max(wkey - off, 0), s.nq) * g : 0;      // rows before it see none of the wavefront's keys
  const int wave_all = a.causal ? min(max(wkey + 31 - off, 0), s.nq) * g : 0;  // rows from it on see all of them
  const int lim = a.causal ? min(max(key - off, 0), s.nq) * g : 0;             // rows from it on see the lane's key
  auto row_of = [&](const T *base, i64 ld, int r) __attribute__((always_inline)) {
    const int query = div_by(r, a.G);
    return base + (i64)(s.q0 + query) * ld + (kvh * g + (r - query * g)) * a.D;
  };
  typename TL::Chunks cq, cd;
  float fl, fd;
  const unsigned lds0 = lds_address(lds);
  auto move = [&](int t, int buf) __attribute__((always_inline)) {
    if (!FAST) return;
    const int r0 = first + t * ROWS, query0 = div_by(r0, a.G);
    unsigned qo[TL::MOVES], dof[TL::MOVES];
#pragma unroll
    for (int i = 0; i < TL::MOVES; ++i) {
      const int r = r0 + TL::slot_row(i), query = div_by(r, a.G);
      const unsigned c = r < nrows ? TL::slot_chunk(i, a.D) : NOWHERE;
      const unsigned in_row = c + (unsigned)((r - query * g) * a.D * (int)sizeof(T));
      const unsigned by = (unsigned)(query - query0) * (unsigned)sizeof(T);
      qo[i] = c == NOWHERE ? c : by * (unsigned)a.q_ld + in_row;
      dof[i] = c == NOWHERE ? c : by * (unsigned)a.dout_ld + in_row;
    }
    const i64 token = s.q0 + query0;
    TL::move(a.q + token * a.q_ld + kvh * g * a.D, NOWHERE, qo, lds0 + buf * STAGE);
    TL::move(a.dout + token * a.dout_ld + kvh * g * a.D, NOWHERE, dof, lds0 + buf * STAGE + TL::BYTES);
    if (wave < 2) {  // lse, delta; zeros where there is no row: with Q and dout zero as well, it adds nothing
      const int r = r0 + lane, query = div_by(r, a.G);
      const unsigned at = lane < ROWS && r < nrows ? (unsigned)((query - query0) * a.Hq + (r - query * g)) * 4u : NOWHERE;
      direct_load_dword(a.rows + ((i64)wave * a.total_q + token) * a.Hq + kvh * g, at,
                        lds0 + buf * STAGE + 2 * TL::BYTES + wave * 256u);
    }
  };
  auto fetch = [&](int t) __attribute__((always_inline)) {
    const int r0 = first + t * ROWS;
    if (!FAST) {
      TL::fetch(cq, r0, nrows, a.D, [&](int r) __attribute__((always_inline)) { return row_of(a.q, a.q_ld, r); });
      TL::fetch(cd, r0, nrows, a.D, [&](int r) __attribute__((always_inline)) { return row_of(a.dout, a.dout_ld, r); });
    }
    fl = fd = 0.f;
    const int r = r0 + (int)threadIdx.x;
    if (!FAST && threadIdx.x < ROWS && r < nrows) {
      const int query = div_by(r, a.G);
      const i64 at = (i64)(s.q0 + query) * a.Hq + kvh * g + (r - query * g);
      fl = a.rows[at];
      fd = a.rows[at + (i64)a.total_q * a.Hq];
    }
  };
  auto put = [&](auto careful, int buf) __attribute__((always_inline)) {
    unsigned char *const st = lds + buf * STAGE;
    TL::template put<decltype(careful)::value>(cq, st);
    TL::template put<decltype(careful)::value>(cd, st + TL::BYTES);
    if (threadIdx.x < ROWS) {
      float *const f = reinterpret_cast<float *>(st + 2 * TL::BYTES) + threadIdx.x;
      f[0] = fl;
      f[64] = fd;
    }
  };
  auto step = [&](auto careful, int t, int buf) __attribute__((always_inline)) {
    constexpr bool CAREFUL = decltype(careful)::value;
    constexpr int UNROLL = sizeof(T) == 2 && DP < 128 ? 2 : 1;
    const unsigned char *const ldsQ = lds + buf * STAGE, *const ldsD = ldsQ + TL::BYTES;
    const float *const ldsL = reinterpret_cast<const float *>(ldsD + TL::BYTES), *const ldsDelta = ldsL + 64;
#pragma unroll UNROLL  // as above; at 128 elements every register counts
    for (int u = 0; u < ROWS / 32; ++u) {
      const int rb = first + t * ROWS + u * 32;
      if (rb >= nrows) break;
      if (rb + 31 < wave_some) continue;
      const unsigned char *const q32 = ldsQ + u * 2 * TL::R16, *const d32 = ldsD + u * 2 * TL::R16;
      const auto lo = sizeof(T) == 4 || DP < 128 ? lane_at : TL::forget(lane_at);
      f32x16 p = zero16(), ds;  // dP - delta: the accumulators begin with -delta
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const f32x4 d = *reinterpret_cast<const f32x4 *>(ldsDelta + u * 32 + 8 * b + 4 * h);
#pragma unroll
        for (int i = 0; i < 4; ++i) ds[4 * b + i] = d[i];
      }
      auto key_part = [&](int x) __attribute__((always_inline)) { return x < K_REG ? kr[x < K_REG ? x : 0] : own[64 * (KT - V_REG + x - K_REG)]; };
      auto value_part = [&](int x) __attribute__((always_inline)) { return x < V_REG ? vr[x < V_REG ? x : 0] : own[64 * (x - V_REG)]; };
      if constexpr (CAREFUL) {
        Sum<CAREFUL> c = {p, p};
#pragma unroll
        for (int x = 0; x < DP / 16; ++x) mma(TL::along(q32, lo, x), key_part(x), c);
        p = total(c);
        c = {zero16(), zero16()};
#pragma unroll
        for (int x = 0; x < DP / 16; ++x) mma(TL::along(d32, lo, x), value_part(x), c);
        ds += total(c);
      } else {
#pragma unroll
        for (int x = 0; x < DP / 16; ++x) p = mma(TL::along(q32, lo, x), key_part(x), p);
#pragma unroll
        for (int x = 0; x < DP / 16; ++x) ds = mma(TL::along(d32, lo, x), value_part(x), ds);
      }
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const f32x4 lse2 = *reinterpret_cast<const f32x4 *>(ldsL + u * 32 + 8 * b + 4 * h);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          p[4 * b + i] = __builtin_amdgcn_exp2f(p[4 * b + i] * a.scale2 - lse2[i]);
          ds[4 * b + i] *= p[4 * b + i];
        }
      }
      const bool edge = rb < wave_all;
      if (edge || rb + 32 > nrows) {  // (a row that does not exist is zeros, but with an infinite key they make NaN)
        const int rel = lim - rb - 4 * h, end = nrows - rb - 4 * h;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const bool seen = 8 * (i / 4) + i % 4 >= rel && 8 * (i / 4) + i % 4 < end;
          p[i] = seen ? p[i] : 0.f;
          ds[i] = seen ? ds[i] : 0.f;
        }
      }
      auto sees = [&](int i) __attribute__((always_inline)) { return rb + i >= lim; };
      if constexpr (CAREFUL) {
        TL::add_careful(dv, d32, lo, p, edge, sees);
        TL::add_careful(dk, q32, lo, ds, edge, sees);
      } else {
        TL::add(dv, d32, zeros, lo, p, edge, sees);
        TL::add(dk, q32, zeros, lo, ds, edge, sees);
      }
    }
  };
  const int n = (nrows - first + ROWS - 1) / ROWS;
  stream<FAST, NB, 2 * TL::MOVES>(n, move, fetch, put, step, std::false_type());
  if constexpr (sizeof(T) == 4)
    if (anywhere<NW>(finite_check(dk) + finite_check(dv), flags)) {
#pragma unroll
      for (int db = 0; db < DP / 32; ++db) dk[db] = dv[db] = zero16();
      stream<FAST, NB, 2 * TL::MOVES>(n, move, fetch, put, step, std::true_type());
    }
  if (!live) return;
  if (a.splits > 1) {
    const i64 at = ((i64)(s.k0 + key) * a.Hkv + kvh) * a.D, plane = (i64)a.total_k * a.Hkv * a.D;
    store_column<float, DP>(a.partials + (2 * split) * plane + at, a.D, dk, a.scale);
    store_column<float, DP>(a.partials + (2 * split + 1) * plane + at, a.D, dv, 1.f);
    return;
  }
  store_column<T, DP>(a.dk + (i64)(s.k0 + key) * a.dk_ld + kvh * a.D, a.D, dk, a.scale);
  store_column<T, DP>(a.dv + (i64)(s.k0 + key) * a.dv_ld + kvh * a.D, a.D, dv, 1.f);
}

// dK and dV from the partial sums of attention_dkv_kernel, in the order of the splits.
template <typename T>
__global__ __launch_bounds__(256) void attention_dkv_join_kernel(const Args<T> a) {
  const int k0 = bound_of(a.cu_k, 0, a.total_k), k1 = max(bound_of(a.cu_k, a.num_seqs, a.total_k), k0);
  const int cols = a.Hkv * a.D;
  const i64 plane = (i64)a.total_k * cols, end = (i64)k1 * cols;
  for (i64 i = (i64)k0 * cols + (i64)blockIdx.x * 256 + threadIdx.x; i < end; i += (i64)gridDim.x * 256) {
    float dk = 0.f, dv = 0.f;
    for (int s = 0; s < a.splits; ++s) {
      dk += a.partials[2 * s * plane + i];
      dv += a.partials[(2 * s + 1) * plane + i];
    }
    const i64 key = i / cols, c = i - key * cols;
    from_f32(dk, a.dk[key * a.dk_ld + c]);
    from_f32(dv, a.dv[key * a.dv_ld + c]);
  }
}

// ---- host ------------------------------------------------------------------------------------------------
template <typename T>
bool aligned(const void *p) { return ((uintptr_t)p & (sizeof(T) - 1)) == 0; }

inline int check_shape(const char *name, int num_seqs, i64 total_q, i64 total_k, int Hq, int Hkv, int D) {
  UNET_REQUIRE(num_seqs >= 0 && total_q >= 0 && total_k >= 0, "%s: num_seqs %d, total_q %lld, total_k %lld", name, num_seqs,
               (long long)total_q, (long long)total_k);
  UNET_REQUIRE(Hq >= 1 && Hkv >= 1 && Hq % Hkv == 0, "%s: %d query heads are no multiple of %d key/value heads", name, Hq, Hkv);
  UNET_REQUIRE(D >= 1, "%s: head_dim %d", name, D);
  if (D > 128) return unet_set_error(UNET_ERR_UNSUPPORTED, "%s: head_dim %d is larger than 128", name, D);
  // a token's elements and the rows are counted in 32 bits, and a launch has fewer than 2^32 threads (512 a workgroup at
  // most, splits only for few)
  UNET_REQUIRE((i64)Hq * D < (i64)1 << 31, "%s: %d heads of %d elements are too many", name, Hq, D);
  const i64 most = ((i64)1 << 31) - 256, groups = (i64)1 << 22, g = Hq / Hkv;
  UNET_REQUIRE(total_q <= most && total_k <= most && total_q * g <= most && total_q * g / BM + num_seqs <= groups / Hkv &&
                   total_k / BM + num_seqs <= groups / Hkv,
               "%s: too many tokens (%lld queries, %lld keys, %d and %d heads)", name, (long long)total_q, (long long)total_k,
               Hq, Hkv);
  return UNET_OK;
}
template <typename T>
int check_matrix(const char *name, const char *what, const T *p, i64 ld, i64 rows, i64 cols) {
  UNET_REQUIRE(p || rows == 0, "%s: %s is NULL", name, what);
  UNET_REQUIRE(ld >= cols, "%s: the stride of %s (%lld) is smaller than its %lld columns", name, what, (long long)ld,
               (long long)cols);
  UNET_REQUIRE(aligned<T>(p), "%s: %s is misaligned", name, what);
  return UNET_OK;
}
#define TRY(call)                    \
  do {                               \
    const int rc_ = (call);          \
    if (rc_ != UNET_OK) return rc_;  \
  } while (0)

template <typename T>
int common_args(const char *name, Args<T> &a, const T *q, i64 q_ld, const T *k, i64 k_ld, const T *v, i64 v_ld,
                const int32_t *cu_q, const int32_t *cu_k, int num_seqs, i64 total_q, i64 total_k, int Hq, int Hkv, int D,
                float scale, int causal) {
  TRY(check_shape(name, num_seqs, total_q, total_k, Hq, Hkv, D));
  UNET_REQUIRE(scale > 0.f && scale * LOG2E < INFINITY, "%s: scale %g is not positive and finite", name, (double)scale);
  UNET_REQUIRE(num_seqs == 0 || (cu_q && cu_k), "%s: cu_q or cu_k is NULL", name);
  UNET_REQUIRE(aligned<int>(cu_q) && aligned<int>(cu_k), "%s: cu_q or cu_k is misaligned", name);
  TRY(check_matrix(name, "q", q, q_ld, total_q, (i64)Hq * D));
  TRY(check_matrix(name, "k", k, k_ld, total_k, (i64)Hkv * D));
  TRY(check_matrix(name, "v", v, v_ld, total_k, (i64)Hkv * D));
  a.q = q, a.k = k, a.v = v, a.q_ld = q_ld, a.k_ld = k_ld, a.v_ld = v_ld;
  a.cu_q = cu_q, a.cu_k = cu_k, a.num_seqs = num_seqs, a.total_q = (int)total_q, a.total_k = (int)total_k;
  a.Hq = Hq, a.Hkv = Hkv, a.D = D, a.causal = causal != 0, a.G = make_div((uint32_t)(Hq / Hkv));
  a.scale = scale, a.scale2 = scale * LOG2E;
  return UNET_OK;
}

// How the kernels that keep queries share their work.
// wk (see attention_kernel): 128 queries a workgroup when that fills three quarters of the places (two a CU, one in fp32
// behind 64 elements), else 64, and 32 when it is a quarter or less: shorter workgroups fill the GPU evenly, but their
// tiles serve fewer wavefronts.  Forward in us with 128 / 64 / 32 queries: 512 workgroups of 128 (16 x 256 tokens, 16
// heads of 64, bf16) 12.6 / 17.4 / 23.6; 332 (8 sequences of up to 2049, 8/2 heads of 80, causal) 52.7 / 42.4 / 73; 224
// (fp32, 3525 tokens, 8 heads of 64) 65 / 47 / 108; 16 (256 tokens, 8 heads of 64) 10.0 / - / 6.6.  Under a causal mask
// twice as many before it is 128: workgroups that all run at once take as long as the longest (forward + backward in us
// with 128 / 64, 8 heads: one sequence of 6144, 64 elements, bf16 373 / 294, 128 elements 532 / 448; 8192, 64, fp32 1880 /
// 1697; 16 of 384, 128, bf16 85 / 91).  It does not change the splits, which come with the smallest number.
// splits: ranges of the keys (forward), when that is still too few, each of at least 512 keys on the average, 256 in fp32
// and for rows through registers
// (what a join costs more would not be won back; fp32, 4 queries over 12000 keys, 16/4 heads of 128: 59 us with 512, 37
// with 256, but one image of 256 tokens 11.7 whole and 13.2 in two).
// eight: 8 wavefronts and 128 queries a workgroup, one a CU (forward, fp32 rows of 33 to 64 elements, wk = 2): the tiles are
// split into parts by twice as many threads.  Where one round of workgroups does, or a single sequence leaves no empty
// workgroups among them; else a few CUs take two in a row.  us with 4 / 8 wavefronts, 8 heads of 64: 3525 tokens in 4 sequences
// 67 / 56; one of 5000 422 / 407, causal 204 / 198; 3 of 1024 60 / 49; but 16 of 256 25 / 37, 17 of 384, causal, 40 / 66, 4/2
// heads, 2 of 4086, 223 / 309.  (dQ gains nothing by it.  bf16 rows of 96 elements and more gain by 8 wavefronts and 256 queries
// only where the workgroups come out as whole rounds of the GPU: 8192 tokens, 16/4 heads of 128, causal, 294 -> 273 us; one
// sequence of 5000, 32 heads, 218 -> 231; 25 of 256, 16 heads, 33 -> 63.)
// dq_splits: the same for dQ, 256 keys at least in both types, at most 8 (backward in us: 3000 tokens, 2/1 heads of 128, fp32
// 463 whole, 344 in two; 976 tokens, 2 heads of 100, bf16 99 whole, 68 in three).
struct Plan {
  int wk, splits, dq_splits, tiles;  // tiles of queries: an upper bound
  bool eight;
};
template <typename T>
constexpr int most_shared(int DP) { return sizeof(T) == 2 || DP <= 64 ? 4 : 2; }  // what the LDS has room for
constexpr int padded_dim(int D) { return (D + 31) / 32 * 32; }
constexpr int MOST_SHARES = 64, MOST_DQ_SHARES = 8, MOST_RANGES = 16;  // of the keys (forward, dQ), of the rows (dK and dV)
template <typename T>
Plan make_plan(int num_seqs, i64 total_q, i64 total_k, int Hq, int Hkv, int D, bool causal) {
  // (a bf16 row that is no whole number of 16-byte chunks takes 128 queries a workgroup always)
  const int most = sizeof(T) == 2 && D % 8 ? 1 : most_shared<T>(padded_dim(D)), places = sizeof(T) == 2 || D <= 64 ? 512 : 256;
  const i64 rows = total_q * (Hq / Hkv);
  auto groups = [&](int bq) { const i64 t = (rows + bq - 1) / bq; return (t > num_seqs ? t : num_seqs) * Hkv; };
  Plan p;
  const i64 n = groups(BM);
  p.wk = n >= places * (causal ? 6 : 3) / 4 ? 1 : n > places / 4 ? 2 : 4;
  if (p.wk > most) p.wk = most;
  p.eight = sizeof(T) == 4 && p.wk == 2 && D > 32 && D <= 64 && (num_seqs == 1 || (rows / BM + num_seqs) * Hkv <= 256);
  auto shares = [&](i64 keys, i64 limit) {
    if (p.wk != most || num_seqs == 0) return 1;
    i64 s = 256 / groups(BM / p.wk);
    if (s > total_k / num_seqs / keys) s = total_k / num_seqs / keys;
    return (int)(s < 1 ? 1 : s > limit ? limit : s);
  };
  p.splits = shares(sizeof(T) == 2 && D % 8 == 0 ? 512 : 256, MOST_SHARES);
  p.dq_splits = shares(256, MOST_DQ_SHARES);
  p.tiles = (int)(rows / (BM / p.wk)) + num_seqs;
  return p;
}

// Wavefronts of a dK/dV workgroup.  bf16 rows of more than 96 elements: 8 wavefronts, 256 keys, share a tile of queries,
// because two workgroups of 4 would ask for 16 bytes of direct loads per clock and CU, which is all there is (forward and
// backward in us with 4 / 8, heads of 128: 8192 tokens, 16/4 heads, causal, 1807 / 1305; 8 of 512, 8 heads, 122 / 103; but 50 of 256, 16
// heads, 333 / 362).  Up to 96 elements they ask for less, and 128 keys leave less of a short sequence's last tile empty (heads
// of 96: 8192 tokens 1059 / 1057; 4 of 1024, 8 heads, 116 / 116; 16 of 256, 16 heads, 74 / 93; one of 256, 8 heads, 33 / 38).
template <typename T>
constexpr int dkv_waves(int DP) { return sizeof(T) == 2 && DP >= 128 ? 8 : WAVES; }
// Row ranges into which their sums are split when there are few key tiles: `fit` workgroups run at once (one of 8
// wavefronts a CU, one of fp32 behind 64 elements, else two), and where lengths differ as much as under a causal mask it
// takes twice as many to fill the GPU evenly, but 16 ranges only where 8 leave it empty (3 sequences, 3464 tokens, 8/1
// heads of 80, backward: 142 us with 8, 107 with 16; 8 sequences, 5289 tokens, 8/2 heads of 80, causal: 124 and 141).
// Each range costs a pass over fp32 dK and dV, so it should have 128 rows at least on the average, in bf16, and two of
// them are worth their join from 512 rows on (backward in us: 3 sequences, 1533 tokens, 4/1 heads of 40, causal: ranges of
// 256 rows 47, of 128 37; but 4 x 256 tokens, 8 heads of 128: whole 36, in ranges of 128 49); in fp32, where a row takes
// longer, 64 (one image of 256 tokens, 8 heads of 64: ranges of 256 46, 128 38, 64 34).
// A power of two, so that workgroups of one range and head keep to one XCD and its L2 (workgroups go round over
// the 8 XCDs): with 5 or 7 ranges the 8192 tokens above are 6 % slower than with 4; with one range they take 1.9 ms.
template <typename T>
int dkv_splits(int num_seqs, i64 total_q, i64 total_k, int Hq, int Hkv, int D, bool causal) {
  const int nw = dkv_waves<T>(padded_dim(D)), fit = nw == 4 && (sizeof(T) == 2 || D <= 64) ? 512 : 256;
  const i64 t = (total_k + COLS * nw - 1) / (COLS * nw), tiles = (t > num_seqs ? t : num_seqs) * Hkv;
  const i64 rows = num_seqs ? total_q * (Hq / Hkv) / num_seqs : 0, least = sizeof(T) == 2 ? 128 : 64;
  int s = 1;
  if (sizeof(T) == 2 && rows < 512) return s;
  while (s < MOST_RANGES && s * tiles < fit * (causal && s < 8 ? 6 : 3) / 4 && 2 * s * least <= rows) s *= 2;
  return s;
}
// What the shares of a plan take in the workspace: fp32 rows of D + 2 (forward), D (dQ) and 2 D (dK and dV) numbers.
inline i64 share_rows(i64 shares, i64 rows) { return shares > 1 ? shares * rows : 0; }
inline size_t forward_bytes(i64 rows, int D) { return (size_t)rows * (D + 2) * sizeof(float); }
inline size_t backward_bytes(i64 dq_rows, i64 dkv_rows, int D) {
  return (size_t)(dq_rows > 2 * dkv_rows ? dq_rows : 2 * dkv_rows) * D * sizeof(float);
}
// Rows enough for either storage type, with a causal mask or without, any number of sequences and no more queries and keys
// than these.  (Not those of the plan with these sizes: fewer tokens are cut into more shares.)
//   - make_plan has at most 256 / workgroups shares of the keys, and a workgroup has at most BM of the total_q * Hq rows:
//     together 256 * BM rows; a share has 256 keys at least on the average.
//   - dkv_splits doubles while shares * tiles < 3 / 2 fit, and a tile has 32 * waves of the total_k * Hkv keys: together less
//     than 3 * fit * 32 * waves rows, which is 3 * 512 * BM for 4 waves and for 8; a share has 64 rows at least.
inline i64 least_of(i64 a, i64 b) { return a < b ? a : b; }
inline i64 most_query_rows(i64 total_q, i64 total_k, int Hq, i64 shares) {
  return least_of(share_rows(least_of(shares, total_k / 256), total_q * Hq), 256 * BM);
}
inline i64 most_key_rows(i64 total_q, i64 total_k, int Hq, int Hkv) {
  return least_of(share_rows(least_of(MOST_RANGES, total_q * (Hq / Hkv) / 64), total_k * Hkv), 3 * 512 * BM);
}
inline size_t rows_bytes(i64 total_q, int Hq) { return ((size_t)total_q * Hq * 2 * sizeof(float) + 15) / 16 * 16; }

// f(DP, FAST) with the head dimension padded to the tile's, and whether the streamed rows are whole aligned chunks.
template <typename T, typename F>
void with_dim(int D, bool fast, F f) {
  auto padded = [&](auto dp) {
    if constexpr (sizeof(T) == 2)
      if (fast) return f(dp, std::true_type());
    f(dp, std::false_type());
  };
  if (D <= 32) padded(std::integral_constant<int, 32>());
  else if (D <= 64) padded(std::integral_constant<int, 64>());
  else if (D <= 96) padded(std::integral_constant<int, 96>());
  else padded(std::integral_constant<int, 128>());
}
// f(WK): bf16's shared kernels exist for whole chunks; other inputs take workgroups of 128 queries whatever their number.
template <typename T, int DP, bool FAST, typename F>
void with_shared(int wk, F f) {
  if constexpr (FAST || sizeof(T) == 4) {
    if constexpr (most_shared<T>(DP) == 4)
      if (wk == 4) return f(std::integral_constant<int, 4>());
    if constexpr (most_shared<T>(DP) >= 2)
      if (wk >= 2) return f(std::integral_constant<int, 2>());
  }
  f(std::integral_constant<int, 1>());
}
template <typename T>
bool whole_chunks(const T *p, i64 ld, int D) {
  // and a tile's span (at most 128 rows) stays below 2 GiB, the reach of the direct loads' offsets
  return ((uintptr_t)p & 15) == 0 && ld * sizeof(T) % 16 == 0 && D * sizeof(T) % 16 == 0 && ld <= (1 << 24) / (i64)sizeof(T);
}

template <typename T>
int forward(const T *q, i64 q_ld, const T *k, i64 k_ld, const T *v, i64 v_ld, T *out, i64 out_ld, float *lse,
            const int32_t *cu_q, const int32_t *cu_k, int num_seqs, i64 total_q, i64 total_k, int Hq, int Hkv, int D,
            float scale, int causal, void *ws, size_t ws_bytes, hipStream_t st) {
  const char *const name = "dot_attention";
  Args<T> a{};
  TRY(common_args(name, a, q, q_ld, k, k_ld, v, v_ld, cu_q, cu_k, num_seqs, total_q, total_k, Hq, Hkv, D, scale, causal));
  TRY(check_matrix(name, "out", out, out_ld, total_q, (i64)Hq * D));
  UNET_REQUIRE(aligned<float>(lse), "%s: lse is misaligned", name);
  if (num_seqs == 0 || total_q == 0) return UNET_OK;
  a.out = out, a.out_ld = out_ld, a.lse = lse;
  const bool whole = whole_chunks(k, k_ld, D) && whole_chunks(v, v_ld, D);
  const Plan plan = make_plan<T>(num_seqs, total_q, total_k, Hq, Hkv, D, a.causal);
  a.tiles = whole || sizeof(T) == 4 ? plan.tiles : (int)(total_q * (Hq / Hkv) / BM) + num_seqs;
  a.splits = plan.splits, a.partials = (float *)ws;
  if (plan.splits > 1) {
    const size_t need = forward_bytes(share_rows(plan.splits, total_q * Hq), D);
    UNET_REQUIRE(ws && ws_bytes >= need, "%s: workspace of %zu bytes, needs %zu", name, ws_bytes, need);
    UNET_REQUIRE(((uintptr_t)ws & 15) == 0, "%s: the workspace is not 16-byte aligned", name);
  }
  with_dim<T>(D, whole, [&](auto dp, auto fast) {
    constexpr int DP = decltype(dp)::value;
    constexpr bool FAST = decltype(fast)::value;
    with_shared<T, DP, FAST>(plan.wk, [&](auto wk) {
      constexpr int WK = decltype(wk)::value;
      if constexpr (sizeof(T) == 4 && DP == 64 && WK == 2)
        if (plan.eight) {
          a.tiles = (int)(total_q * (Hq / Hkv) / BM) + num_seqs;
          attention_kernel<T, DP, FAST, WK, 8><<<(unsigned)a.tiles * Hkv, 512, 0, st>>>(a);
          return;
        }
      attention_kernel<T, DP, FAST, WK><<<(unsigned)a.tiles * Hkv * a.splits, 256, 0, st>>>(a);
    });
  });
  if (a.splits > 1) attention_join_kernel<T><<<cdiv_u(total_q * Hq, WAVES), 256, 0, st>>>(a);
  UNET_LAUNCH_CHECK(name);
  return UNET_OK;
}

template <typename T>
int backward(const T *dout, i64 dout_ld, const T *q, i64 q_ld, const T *k, i64 k_ld, const T *v, i64 v_ld, const T *out,
             i64 out_ld, const float *lse, T *dq, i64 dq_ld, T *dk, i64 dk_ld, T *dv, i64 dv_ld, const int32_t *cu_q,
             const int32_t *cu_k, int num_seqs, i64 total_q, i64 total_k, int Hq, int Hkv, int D, float scale, int causal,
             void *ws, size_t ws_bytes, hipStream_t st) {
  const char *const name = "dot_attention_backward";
  Args<T> a{};
  TRY(common_args(name, a, q, q_ld, k, k_ld, v, v_ld, cu_q, cu_k, num_seqs, total_q, total_k, Hq, Hkv, D, scale, causal));
  TRY(check_matrix(name, "grad_out", dout, dout_ld, total_q, (i64)Hq * D));
  TRY(check_matrix(name, "out", out, out_ld, total_q, (i64)Hq * D));
  TRY(check_matrix(name, "grad_q", (const T *)dq, dq_ld, total_q, (i64)Hq * D));
  TRY(check_matrix(name, "grad_k", (const T *)dk, dk_ld, total_k, (i64)Hkv * D));
  TRY(check_matrix(name, "grad_v", (const T *)dv, dv_ld, total_k, (i64)Hkv * D));
  UNET_REQUIRE((lse || total_q == 0) && aligned<float>(lse), "%s: lse is NULL or misaligned", name);
  const Plan plan = make_plan<T>(num_seqs, total_q, total_k, Hq, Hkv, D, a.causal);
  const int dkv = dkv_splits<T>(num_seqs, total_q, total_k, Hq, Hkv, D, a.causal);
  const size_t need =
      rows_bytes(total_q, Hq) + backward_bytes(share_rows(plan.dq_splits, total_q * Hq), share_rows(dkv, total_k * Hkv), D);
  UNET_REQUIRE(ws_bytes >= need && (ws || !need), "%s: workspace of %zu bytes, needs %zu", name, ws_bytes, need);
  UNET_REQUIRE(((uintptr_t)ws & 15) == 0, "%s: the workspace is not 16-byte aligned", name);
  if (num_seqs == 0 || (total_q == 0 && total_k == 0)) return UNET_OK;
  a.dout = dout, a.o = out, a.dq = dq, a.dk = dk, a.dv = dv, a.lse = const_cast<float *>(lse), a.rows = (float *)ws;
  a.dout_ld = dout_ld, a.o_ld = out_ld, a.dq_ld = dq_ld, a.dk_ld = dk_ld, a.dv_ld = dv_ld;
  const bool whole =
      whole_chunks(q, q_ld, D) && whole_chunks(k, k_ld, D) && whole_chunks(v, v_ld, D) && whole_chunks(dout, dout_ld, D);
  a.tiles = whole || sizeof(T) == 4 ? plan.tiles : (int)(total_q * (Hq / Hkv) / BM) + num_seqs;
  const int nw = dkv_waves<T>(padded_dim(D));
  const unsigned key_tiles = (unsigned)(total_k / (COLS * nw)) + num_seqs;
  a.partials = (float *)((char *)ws + rows_bytes(total_q, Hq));
  a.splits = plan.dq_splits;
  with_dim<T>(D, whole, [&](auto dp, auto fast) {
    constexpr int DP = decltype(dp)::value, NW = dkv_waves<T>(DP);
    constexpr bool FAST = decltype(fast)::value;
    if (total_q)
      with_shared<T, DP, FAST>(plan.wk, [&](auto wk) {
        attention_dq_kernel<T, DP, FAST, decltype(wk)::value><<<(unsigned)a.tiles * Hkv * a.splits, 256, 0, st>>>(a);
      });
    if (total_q && a.splits > 1) attention_dq_join_kernel<T><<<ew_grid(total_q * Hq * D), 256, 0, st>>>(a);
    a.splits = dkv;
    if (total_k) attention_dkv_kernel<T, DP, FAST, NW><<<key_tiles * Hkv * a.splits, 64 * NW, 0, st>>>(a);
  });
  if (total_k && a.splits > 1) attention_dkv_join_kernel<T><<<ew_grid(total_k * Hkv * D), 256, 0, st>>>(a);
  UNET_LAUNCH_CHECK(name);
  return UNET_OK;
}

}  // namespace
