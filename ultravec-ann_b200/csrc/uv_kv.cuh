// uv_kv.cuh -- the cache held in 4 bits: its layout, its rotation, and the
// device helpers that the page, row and attention kernels share.
//
// Layout.  A page holds page_tokens tokens of every head of one layer:
//   pool[layer][page][head][page_tokens / 32][tile],
//   tile = 32 tokens of one head, 32 * (D + 8) bytes:
//     keys' codes    32 rows of D / 2 bytes; nibble i of a row is dimension i
//     keys' scales   32 f32
//     values' codes  16 pairs of D bytes: a row is D / 4 granules of 16 bits
//                    (4 dimensions each); tokens 2p and 2p + 1 alternate
//     values' scales 32 f32
// One tile is one bulk copy.  Its codes are what mma.m16n8k16 wants: a key is
// a row of the A operand whose K order is free, so a lane takes a quarter of a
// row as it lies; for the values A is transposed (rows are dimensions, K is
// the token), a half2 holds two tokens, and the interleaved granules give a
// lane one 32-bit word with 4 dimensions of both, so the same
// instructions unpack both.  A token never shares a byte pair with another:
// rows are written without reading their neighbours.
//
// Numbers.  y = R x, R the product over rounds of H diag(signs) / sqrt(D).  A
// row is held as levels l_i = n_i - 7.5 and one f32 scale s: y ~ s l, with
// s = |y|^2 / <l, y>, the trellis codec's rescaled estimator
// (src/trellis.rs:1517), for which <y, s l> = |y|^2.  The step that picks n is
// 0.3352 sigma, the best uniform 16-level step for a Gaussian.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "uv_common.cuh"
#include "uv_tc.cuh"

namespace uvb {
namespace kv {

constexpr int kTile = 32;
constexpr float kStep = 0.3352f;
constexpr int kMaxRounds = 3;

// Words of the cache's work buffer (Cache::work).
constexpr int kStatus = 0, kHint = 1, kUsed = 2, kMoves = 3, kWorkHead = 8;
// Status bits; the header names them UV_KV_*.
constexpr int kNoPages = 1, kBadSeq = 2, kTooLong = 4, kNotEmpty = 8, kShared = 16, kTimeout = 32;

struct Cache {
  int head_dim, heads, layers, page_tokens, n_pages, max_seqs, max_pages, rounds;
  uint32_t signs[kMaxRounds][8];  // set: negated; in the order that lane_signs reads
  uint8_t *pool;
  int32_t *table, *lens, *refs, *work;

  __host__ __device__ int tile_bytes() const { return kTile * (head_dim + 8); }
  __host__ __device__ int64_t page_bytes() const {
    return (int64_t)heads * (page_tokens / kTile) * tile_bytes();
  }
  // work: the head, then move sources, move targets (n_pages each), the
  // remap of a compaction, and a mark and an offset of every sequence.
  __host__ __device__ int64_t work_words() const {
    return kWorkHead + 3 * (int64_t)n_pages + 2 * (int64_t)max_seqs;
  }
  __device__ int32_t *move_src() const { return work + kWorkHead; }
  __device__ int32_t *move_dst() const { return move_src() + n_pages; }
  __device__ int32_t *remap() const { return move_dst() + n_pages; }
  __device__ int32_t *mark() const { return remap() + n_pages; }
  __device__ int32_t *offset() const { return mark() + max_seqs; }
  // A sequence's length, never more than its table row can hold.
  __device__ int length(int s) const {
    const int64_t cap = (int64_t)max_pages * page_tokens, n = lens[s];
    return n < 0 ? 0 : (int)(n < cap ? n : cap);
  }
  __device__ int page_at(int s, int column) const {
    const uint32_t p = (uint32_t)table[(int64_t)s * max_pages + column];
    return (int)(p < (uint32_t)n_pages ? p : (uint32_t)(n_pages - 1));
  }
  // Tile j (tokens 32 j ..) of sequence s, head h.
  __device__ uint8_t *tile_at(int layer, int page, int head, int sub) const {
    return pool + ((int64_t)layer * n_pages + page) * page_bytes() +
           ((int64_t)head * (page_tokens / kTile) + sub) * tile_bytes();
  }
};

// The rows of a call: sequence seqs[b] owns rows [starts[b], starts[b + 1])
// (one each without starts), its last tokens in order.  A negative sequence
// means that the entry is out of range and owns nothing.
struct Rows {
  const int32_t *seqs, *starts;
  int n, rows;
  __device__ int first(int b) const {
    if (starts == nullptr) return b;
    const int f = starts[b];
    return f < 0 ? 0 : (f < rows ? f : rows);
  }
  __device__ int count(int b) const {
    if (starts == nullptr) return 1;
    const int c = first(b + 1) - first(b);
    return c < 0 ? 0 : c;
  }
  __device__ int seq(int b, int max_seqs) const {
    const int s = seqs[b];
    return s >= 0 && s < max_seqs ? s : -1;
  }
};

__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

__device__ __forceinline__ void pdl_launch() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// ---- matrix instructions on registers ----
template <bool BF16>
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
  // (not volatile: independent products may be reordered between dependent ones)
  if (BF16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if (BF16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&v);
  }
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&v);
}
template <bool BF16>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
  if (BF16) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
  return __half22float2(*reinterpret_cast<const __half2 *>(&w));
}

// 8 nibbles of a word as 4 half2 of codes n, pair i = (nibble i, nibble i + 4):
// the bits as they stand are subnormal halves, n 2^-24 for i = 0, 2 and
// n 2^-20 for i = 1, 3, which the matrix instructions take exactly.
__device__ __forceinline__ void unpack8(uint32_t w, uint32_t (&out)[4]) {
  const uint32_t u = w >> 8;
  out[0] = w & 0x000f000fu;
  out[1] = w & 0x00f000f0u;
  out[2] = u & 0x000f000fu;
  out[3] = u & 0x00f000f0u;
}
// The same as levels n - 7.5 (0x6400 | n is the half 1024 + n, 0x6400 | 16 n is
// 1024 + 16 n).
__device__ __forceinline__ void unpack8_levels(uint32_t w, uint32_t (&out)[4]) {
  constexpr uint32_t lo = 0x000f000fu, hi = 0x00f000f0u, one = 0x64006400u;
  const uint32_t u = w >> 8;
  uint32_t r[4] = {(w & lo) | one, (w & hi) | one, (u & lo) | one, (u & hi) | one};
  constexpr uint32_t m1032 = 0xe408e408u, m715 = 0xd478d478u, sixteenth = 0x2c002c00u,
                     half = 0x38003800u;
#pragma unroll
  for (int i = 0; i < 4; i += 2) {
    uint32_t x;
    asm("add.f16x2 %0, %1, %2;" : "=r"(x) : "r"(r[i]), "r"(m1032));
    asm("add.f16x2 %0, %1, %2;" : "=r"(out[i]) : "r"(x), "r"(half));
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(out[i + 1]) : "r"(r[i + 1]), "r"(sixteenth), "r"(m715));
  }
}

// ---- the Hadamard transform of 16 rows by one warp ----
// Lane (g = lane / 4, t = lane % 4) owns dimensions [t D / 4, (t + 1) D / 4)
// of rows g and g + 8.  Four index bits (the lane's two and the element's
// lowest two) go through one m16n8k16 product with the +-1 matrix, whose
// output lands in the same owner; the other bits are butterflies in registers.
// An FWHT by shuffles spends about three times the instructions.
struct Hadamard {
  uint32_t b;  // the +-1 pair of this lane's column, as halves or bfloats
  template <bool BF16>
  __device__ static Hadamard make() {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const uint32_t one = BF16 ? 0x3f80u : 0x3c00u;
    const uint32_t s0 = (uint32_t)(__popc((2 * t) & g) & 1) << 15;
    const uint32_t s1 = (uint32_t)(__popc((2 * t + 1) & g) & 1) << 15;
    return {(one | s0) | ((one | s1) << 16)};
  }
};

// y[row][j] += H16 part of the packed pairs a[row][j / 2].
template <int D, bool BF16>
__device__ __forceinline__ void hadamard_mma(float (&y)[2][D / 4], const uint32_t (&a)[2][D / 8],
                                             Hadamard h) {
#pragma unroll
  for (int m = 0; m < D / 16; m++) {
#pragma unroll
    for (int nt = 0; nt < 2; nt++) {
      float c[4] = {y[0][4 * m + 2 * nt], y[0][4 * m + 2 * nt + 1], y[1][4 * m + 2 * nt],
                    y[1][4 * m + 2 * nt + 1]};
      mma16816<BF16>(c, a[0][2 * m], a[1][2 * m], a[0][2 * m + 1], a[1][2 * m + 1], h.b,
                     nt ? h.b ^ 0x80008000u : h.b);
      y[0][4 * m + 2 * nt] = c[0];
      y[0][4 * m + 2 * nt + 1] = c[1];
      y[1][4 * m + 2 * nt] = c[2];
      y[1][4 * m + 2 * nt + 1] = c[3];
    }
  }
}

// The remaining index bits, of both rows or of row g alone.
template <int D, int ROWS = 2>
__device__ __forceinline__ void hadamard_rest(float (&y)[2][D / 4]) {
#pragma unroll
  for (int h = 4; h < D / 4; h *= 2)
#pragma unroll
    for (int j = 0; j < D / 4; j++)
      if ((j & h) == 0)
#pragma unroll
        for (int r = 0; r < ROWS; r++) {
          const float u = y[r][j], v = y[r][j + h];
          y[r][j] = __fadd_rn(u, v);
          y[r][j + h] = __fsub_rn(u, v);
        }
}

template <int D>
__device__ __forceinline__ constexpr float inv_sqrt_d() {
  return D == 64 ? 0.125f : D == 128 ? 0.08838834764831845f : 0.0625f;
}

// y <- H y for f32 rows: each value as two or three bfloats that add up to it
// (to 2^-17 or 2^-25 of it), each part through the matrix product.
template <int D, int PARTS>
__device__ __forceinline__ void hadamard_f32(float (&y)[2][D / 4], Hadamard hb) {
  uint32_t part[PARTS][2][D / 8];
#pragma unroll
  for (int r = 0; r < 2; r++)
#pragma unroll
    for (int j = 0; j < D / 8; j++) {
      float lo = y[r][2 * j], hi = y[r][2 * j + 1];
#pragma unroll
      for (int p = 0; p < PARTS; p++) {
        const uint32_t w = pack2<true>(lo, hi);
        const float2 f = unpack2<true>(w);
        part[p][r][j] = w;
        lo = __fsub_rn(lo, f.x);
        hi = __fsub_rn(hi, f.y);
      }
      y[r][2 * j] = 0.0f;
      y[r][2 * j + 1] = 0.0f;
    }
#pragma unroll
  for (int p = PARTS - 1; p >= 0; p--) hadamard_mma<D, true>(y, part[p], hb);
  hadamard_rest<D>(y);
}

// The signs of this lane's dimensions in a round.  Word w covers dimensions
// t D / 4 + 32 w ..; bit j is dimension 2 j of them and bit 16 + j dimension
// 2 j + 1, so that one shift brings a pair's signs to bits 15 and 31.
template <int D>
__device__ __forceinline__ uint32_t lane_signs(const Cache &c, int round, int w) {
  const int t = threadIdx.x & 3;
  if (D == 64) return c.signs[round][t >> 1] >> ((t & 1) * 8);
  return c.signs[round][t * (D / 128) + w];
}
template <int D>
__device__ __forceinline__ void apply_signs(const Cache &c, int round, float (&y)[2][D / 4]) {
#pragma unroll
  for (int w = 0; w < (D + 127) / 128; w++) {
    const uint32_t s = lane_signs<D>(c, round, w);
#pragma unroll
    for (int j = 0; j < (D == 64 ? 8 : 16); j++)
#pragma unroll
      for (int i = 0; i < 2; i++) {
        const uint32_t flip = (s << ((i ? 15 : 31) - j)) & 0x80000000u;
        const int e = 32 * w + 2 * j + i;
        y[0][e] = __uint_as_float(__float_as_uint(y[0][e]) ^ flip);
        y[1][e] = __uint_as_float(__float_as_uint(y[1][e]) ^ flip);
      }
  }
}

// y = R x for 16 rows of packed halves or bfloats (a is consumed), or for rows
// g alone (ROWS = 1: the others are zero).  The products are exact and add up
// in f32; later rounds take f32 rows as three bfloats.  With SCALE = false the
// result is sqrt(D)^rounds times too large.
template <int D, bool BF16, int ROWS = 2, bool SCALE = true>
__device__ __forceinline__ void rotate_rows(const Cache &c, uint32_t (&a)[2][D / 8],
                                            float (&y)[2][D / 4]) {
#pragma unroll
  for (int w = 0; w < (D + 127) / 128; w++) {
    const uint32_t s = lane_signs<D>(c, 0, w);
#pragma unroll
    for (int j = 0; j < (D == 64 ? 8 : 16); j++) {
      const uint32_t flip = (s << (15 - j)) & 0x80008000u;
#pragma unroll
      for (int r = 0; r < ROWS; r++) a[r][16 * w + j] ^= flip;
    }
  }
#pragma unroll
  for (int j = 0; j < D / 4; j++) y[0][j] = y[1][j] = 0.0f;
  hadamard_mma<D, BF16>(y, a, Hadamard::make<BF16>());
  hadamard_rest<D, ROWS>(y);
  float scale = inv_sqrt_d<D>();
  for (int r = 1; r < c.rounds; r++) {
    apply_signs<D>(c, r, y);
    hadamard_f32<D, 3>(y, Hadamard::make<true>());
    scale = __fmul_rn(scale, inv_sqrt_d<D>());
  }
  if constexpr (SCALE) {
#pragma unroll
  for (int j = 0; j < D / 4; j++)
#pragma unroll
    for (int r = 0; r < ROWS; r++) y[r][j] = __fmul_rn(y[r][j], scale);
  }
}

// sqrt(D)^-rounds
template <int D>
__device__ __forceinline__ float rotation_scale(const Cache &c) {
  float scale = inv_sqrt_d<D>();
  for (int r = 1; r < c.rounds; r++) scale = __fmul_rn(scale, inv_sqrt_d<D>());
  return scale;
}

// x = sqrt(D)^rounds R^T y in place, for 16 f32 rows; the first transform takes
// PARTS bfloats a value, and may have been done already (first = false).
template <int D, int PARTS>
__device__ __forceinline__ void rotate_back(const Cache &c, float (&y)[2][D / 4], bool first) {
  for (int r = c.rounds - 1; r >= 0; r--) {
    if (first || r != c.rounds - 1) hadamard_f32<D, PARTS>(y, Hadamard::make<true>());
    apply_signs<D>(c, r, y);
  }
}

// The larger one, NaN if either is.
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
// 2^e as a float, e in [-126, 127].
__device__ __forceinline__ float exp2i(int e) { return __int_as_float((e + 127) << 23); }
// floor(log2 |x|) of a normal x (-127 for zero and subnormals, 128 for inf and NaN).
__device__ __forceinline__ int log2i(float x) {
  return (int)((__float_as_uint(x) >> 23) & 255u) - 127;
}

}  // namespace kv
}  // namespace uvb
