// kv_rows.cu -- rows into the cache held in 4 bits (rotate, quantise, write
// into the pages) and back out of it (levels, rotate back).
//
// A warp takes 16 consecutive token positions of one head, aligned to 16, of
// the keys or of the values: lane (g, t) holds a quarter of rows g and g + 8.
// The rotation's first four index bits go through the tensor core (16 m16n8k16
// for 16 rows of 128), the others are register butterflies; a row's sums cross
// 4 lanes.  Positions outside the call's rows are computed as zeros and not
// stored.
//
// Bound: HBM would allow 11 us each way for 14k tokens of 8 heads of 128 (2 D
// bytes of a row in, D / 2 + 4 out, and the reverse).  They take 37 and 29 us: 20
// instructions a value into the cache and 12 out of it (16 and 10 us of issue slots,
// had they no gaps), at three warps a scheduler, all that 160 registers leave, which
// do not cover the rows' loads.  For a token each it is latency (four dependent loads
// find the row's place).
#include "uv_kv.h"

namespace uvb {
namespace kv {

constexpr int kRowThreads = 128;

// Block u of 16 positions: its entry's sequence, the block's first position,
// the first position that a row has, and the row of position x, first + x.
// Entry b has starts[b + 1] / 16 - starts[b] / 16 + 2 blocks, never fewer than
// its rows can touch, so the map needs the starts alone.  blank: rows of the
// entry before the sequence's first token, told to its first block alone.
struct Block {
  int seq, len, pos0, begin, first, blank, row0;
};
__device__ __forceinline__ Block find_block(const Rows &r, const Cache &c, int64_t u) {
  int b;
  int64_t k = 0;
  if (r.starts == nullptr) {
    b = (int)u;
  } else {
    int lo = 0, hi = r.n - 1;  // the last entry whose first block is <= u
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (r.first(mid) / 16 + 2 * (int64_t)mid <= u) lo = mid;
      else hi = mid - 1;
    }
    b = lo;
    k = u - (r.first(b) / 16 + 2 * (int64_t)b);
  }
  Block x;
  x.seq = r.seq(b, c.max_seqs);
  x.row0 = r.first(b);
  const int n = r.count(b);
  x.len = x.seq < 0 ? 0 : c.length(x.seq);
  const int start = x.len - n;
  x.begin = max(start, 0);
  x.first = x.row0 - start;
  x.blank = k == 0 ? max(-start, 0) : 0;
  const int64_t p = (int64_t)(x.begin / 16 + k) * 16;
  x.pos0 = (int)min(p, (int64_t)x.len);  // past the end: no position
  return x;
}

// 8 f32 codes -> word; t[j] = code + 1.5 * 2^23 exactly.
__device__ __forceinline__ uint32_t pack_codes(const float *t) {
  uint32_t w = 0;
#pragma unroll
  for (int j = 7; j >= 0; j--) w = w * 16u + __float_as_uint(t[j]);
  // every term carried 0x4b400000: take the sum of its shifted copies out
  return w - 0x4b400000u * 0x11111111u;
}

// floor(log2) of the largest magnitude in a row of bfloats that four lanes hold (what
// exp2i takes, both ways: 126 at most), 0 where the row has an infinity or a NaN (which then stays what it is).
template <int D>
__device__ __forceinline__ int bfloat_exponent(const uint32_t (&a)[D / 8]) {
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < D / 8; j++) top = __vmaxu2(top, a[j] & 0x7fff7fffu);
  top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, 1));
  top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, 2));
  const int e = (int)(max(top >> 16, top & 0xffffu) >> 7);
  return e == 255 ? 0 : max(min(e, 253), 27) - 127;
}

// What an append must find before its first byte is written: sequences in range,
// none listed twice, and pages that nobody else holds (extend has made room).  One
// block, as the page operations decide; a lane looks at one entry's page or two, and
// where there are more (prompts) its warp shares them.  Beside the rows' own loads and
// rotations it costs 2 us of 67 (8 prompts), and a launch of 3 us where the host bounds
// the call.
constexpr int kCheckThreads = 1024;
__global__ void __launch_bounds__(kCheckThreads) append_check_kernel(Cache c, Rows rows) {
  __shared__ int errors;
  pdl_launch();
  const int before = c.work[kStatus];  // (looked at in the end: it waits for nothing)
  if (threadIdx.x == 0) errors = 0;
  __syncthreads();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int bad = 0;
  for (int i0 = 0; i0 < rows.n; i0 += kCheckThreads) {
    const int i = i0 + lane * (kCheckThreads / 32) + warp;  // a few long ones: a warp each
    int s = -1, from = 0, to = -1;  // columns that the rows lie in
    if (i < rows.n) {
      s = rows.seq(i, c.max_seqs);
      if (s < 0) {
        bad |= kBadSeq;
      } else {
        const int len = c.length(s), n = min(rows.count(i), len);
        if (n > 0) from = (len - n) / c.page_tokens, to = (len - 1) / c.page_tokens;
        if (atomicExch(&c.mark()[s], 1) != 0) bad |= kBadSeq;
      }
    }
    auto look = [&](int seq, int column) {
      if (c.refs[c.page_at(seq, column)] != 1) bad |= kShared;
    };
    if (from <= to) look(s, from);
    if (from < to) look(s, to);
    for (uint32_t more = __ballot_sync(0xffffffffu, to - from > 1); more; more &= more - 1) {
      const int who = __ffs(more) - 1;
      const int seq = __shfl_sync(0xffffffffu, s, who), lo = __shfl_sync(0xffffffffu, from, who);
      const int hi = __shfl_sync(0xffffffffu, to, who);
      for (int column = lo + 1 + lane; column < hi; column += 32) look(seq, column);
    }
  }
  if (bad) atomicOr(&errors, bad);
  __syncthreads();
  for (int i = threadIdx.x; i < rows.n; i += kCheckThreads) {
    const int s = rows.seq(i, c.max_seqs);
    if (s >= 0) c.mark()[s] = 0;
  }
  if (threadIdx.x == 0 && errors && before == 0) c.work[kStatus] = errors;
}

// A warp takes `each` of a block's 2 * heads parts (keys and values of a head),
// which share what finding the block took: four dependent loads.
template <int D, bool BF16>
__global__ void __launch_bounds__(kRowThreads) append_kernel(Cache c, int layer, Rows rows,
                                                             Strided kin, Strided vin, int64_t blocks,
                                                             int each) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int64_t item = (int64_t)blockIdx.x * (kRowThreads / 32) + (threadIdx.x >> 5);
  const int parts = 2 * c.heads, groups = (parts + each - 1) / each;
  if (item >= blocks * groups) return pdl_wait();
  const Block at = find_block(rows, c, item / groups);
  const int s = at.seq, len = at.len, pos0 = at.pos0, begin = at.begin, first = at.first;
  // (every block waits for the check, also to end: what follows is ordered behind both)
  if (pos0 >= len || begin >= len) return pdl_wait();  // no position, or an entry of no rows
  const int page = c.page_at(s, pos0 / c.page_tokens);
  const bool live[2] = {pos0 + g >= begin && pos0 + g < len, pos0 + g + 8 >= begin && pos0 + g + 8 < len};
  const int from = (int)(item % groups) * each, to_part = min(from + each, parts);
  for (int part = from; part < to_part; part++) {
    const int head = part >> 1;
    const bool value = part & 1;
    const Strided &in = value ? vin : kin;
    const uint16_t *src = (const uint16_t *)in.p + (int64_t)head * in.head + t * (D / 4);
    float y[2][D / 4], square[2], grow[2] = {1.0f, 1.0f};
    auto squares = [&](int r) {
      float some = 0.0f, more = 0.0f;
#pragma unroll
      for (int j = 0; j < D / 4; j += 2) {
        some = __fmaf_rn(y[r][j], y[r][j], some);
        more = __fmaf_rn(y[r][j + 1], y[r][j + 1], more);
      }
      some = __fadd_rn(some, more);
      some += __shfl_xor_sync(0xffffffffu, some, 1);
      some += __shfl_xor_sync(0xffffffffu, some, 2);
      square[r] = some;
    };
    uint32_t a[2][D / 8];
    auto load = [&] {
#pragma unroll
      for (int r = 0; r < 2; r++) {
        const uint4 *q = (const uint4 *)(src + (int64_t)(first + pos0 + g + 8 * r) * in.row);
#pragma unroll
        for (int i = 0; i < D / 32; i++) {
          const uint4 w = live[r] ? __ldg(q + i) : make_uint4(0, 0, 0, 0);
          a[r][4 * i] = w.x;
          a[r][4 * i + 1] = w.y;
          a[r][4 * i + 2] = w.z;
          a[r][4 * i + 3] = w.w;
        }
      }
    };
    load();
    rotate_rows<D, BF16, 2, false>(c, a, y);
    squares(0);
    squares(1);
    if (BF16 && __any_sync(0xffffffffu, !(square[0] < 0x1p80f && square[1] < 0x1p80f))) {
      // Bfloats may be so large that the transform passes the largest float: such
      // rows are taken again, with a power of two out of them first.
      load();
#pragma unroll
      for (int r = 0; r < 2; r++) {
        const int size = bfloat_exponent<D>(a[r]);  // (every lane: it shuffles)
        const int e = square[r] < 0x1p80f ? 0 : size;
        grow[r] = exp2i(e);
#pragma unroll
        for (int j = 0; j < D / 8; j++) {
          const float2 v = unpack2<true>(a[r][j]);
          a[r][j] = pack2<true>(__fmul_rn(v.x, exp2i(-e)), __fmul_rn(v.y, exp2i(-e)));
        }
      }
      rotate_rows<D, BF16, 2, false>(c, a, y);
      squares(0);
      squares(1);
    }
    if (part == from) {
      pdl_wait();
      // an extend failed, so that these rows have no place, or the check found an entry bad
      if (c.work[kStatus] != 0) return;
    }

    uint8_t *tile = c.tile_at(layer, page, head, pos0 % c.page_tokens / kTile) +
                    (value ? kTile * (D / 2 + 4) : 0);
    const int row0 = pos0 % kTile;
    const float shrink = rotation_scale<D>(c);
#pragma unroll
    for (int r = 0; r < 2; r++) {
      if (__any_sync(0xffffffffu, !(square[r] > 0x1p-80f && square[r] < 0x1p80f))) {
        // A power of two takes the row's size out, so that squares neither
        // overflow nor vanish (for the rows that need it: 1 for the others).
        float m = 0.0f;
#pragma unroll
        for (int j = 0; j < D / 4; j++) m = fmaxf(m, fabsf(y[r][j]));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
        const int e = square[r] > 0x1p-80f && square[r] < 0x1p80f ? 0 : max(-100, min(log2i(m), 126));
        grow[r] = __fmul_rn(grow[r], exp2i(e));
#pragma unroll
        for (int j = 0; j < D / 4; j++) y[r][j] = __fmul_rn(y[r][j], exp2i(-e));
        squares(r);
      }
      const float inv =
          square[r] > 0.0f ? __fdiv_rn(1.0f, __fmul_rn(kStep, __fsqrt_rn(__fmul_rn(square[r], 1.0f / D))))
                        : 0.0f;
      float ly = 0.0f, more = 0.0f;
      uint32_t w[D / 32];
#pragma unroll
      for (int i = 0; i < D / 32; i++) {
        float n[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
          const float z = fminf(fmaxf(__fmul_rn(y[r][8 * i + j], inv), -8.0f), 7.0f);
          n[j] = __fadd_rd(z, 12582920.0f);  // 1.5 * 2^23 + 8, rounded down: floor(z) + 8
          float &sum = j % 2 ? more : ly;
          sum = __fmaf_rn(__fadd_rn(__fsub_rn(n[j], 12582920.0f), 0.5f), y[r][8 * i + j], sum);
        }
        w[i] = pack_codes(n);
      }
      ly = __fadd_rn(ly, more);
      ly += __shfl_xor_sync(0xffffffffu, ly, 1);
      ly += __shfl_xor_sync(0xffffffffu, ly, 2);
      // |y| finite and not zero: ly > 0, since every level has its value's sign
      // (a row of zeros has the scale zero; one with an infinity or a NaN gets NaN)
      const float scale =
          square[r] == 0.0f ? 0.0f : __fmul_rn(__fmul_rn(__fdiv_rn(square[r], ly), shrink), grow[r]);
      const int row = row0 + g + 8 * r;
      if (live[r] && t == 0) ((float *)(tile + kTile * (D / 2)))[row] = scale;
      if (!value) {
        if (live[r]) {
          uint32_t *to = (uint32_t *)(tile + row * (D / 2)) + t * (D / 32);
          if (D == 128) {
            *(uint4 *)to = make_uint4(w[0], w[1], w[2], w[D / 32 - 1]);
          } else {
#pragma unroll
            for (int i = 0; i < D / 32; i++) to[i] = w[i];
          }
        }
        continue;
      }
      // Tokens 2p and 2p + 1 are lanes g and g ^ 1: the even one takes the
      // granules of dimensions 0..3 of each word, the odd one those of 4..7.
      const bool odd = g & 1;
      const bool other = __shfl_xor_sync(0xffffffffu, (int)live[r], 4);
      uint16_t *pair = (uint16_t *)(tile + (row >> 1) * D) + t * (D / 8);
#pragma unroll
      for (int i = 0; i < D / 32; i++) {
        const uint32_t x = __shfl_xor_sync(0xffffffffu, w[i], 4);
        if (live[r] && other) {
          ((uint32_t *)pair)[2 * i + odd] =
              odd ? (x >> 16) | (w[i] & 0xffff0000u) : (w[i] & 0xffffu) | (x << 16);
        } else if (live[r]) {
          pair[4 * i + odd] = (uint16_t)w[i];
          pair[4 * i + 2 + odd] = (uint16_t)(w[i] >> 16);
        }
      }
    }
  }
}

template <int D, bool BF16>
__global__ void __launch_bounds__(kRowThreads) read_kernel(Cache c, int layer, Rows rows,
                                                           uint16_t *kout, uint16_t *vout,
                                                           int64_t blocks, int each) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int64_t item = (int64_t)blockIdx.x * (kRowThreads / 32) + (threadIdx.x >> 5);
  const int parts = 2 * c.heads, groups = (parts + each - 1) / each;
  if (item >= blocks * groups) return;
  const Block at = find_block(rows, c, item / groups);
  const int s = at.seq, len = at.len, pos0 = at.pos0, begin = at.begin, first = at.first;
  const int from = (int)(item % groups) * each, to_part = min(from + each, parts);
  if (at.blank > 0)  // rows without a token read as zeros
    for (int part = from; part < to_part; part++)
      for (int i = lane; i < at.blank * (D / 8); i += 32)
        ((uint4 *)((part & 1 ? vout : kout) + ((int64_t)(at.row0 + i / (D / 8)) * c.heads + (part >> 1)) * D))
            [i % (D / 8)] = make_uint4(0, 0, 0, 0);
  if (pos0 >= len) return;
  const int page = c.page_at(s, pos0 / c.page_tokens);
  const int row0 = pos0 % kTile;
  const float shrink = rotation_scale<D>(c);
  for (int part = from; part < to_part; part++) {
    const int head = part >> 1;
    const bool value = part & 1;
    uint16_t *out = (value ? vout : kout) + head * D;
    const uint8_t *tile = c.tile_at(layer, page, head, pos0 % c.page_tokens / kTile) +
                          (value ? kTile * (D / 2 + 4) : 0);
    bool live[2];
    float scale[2];
    uint32_t w[2][D / 32];
#pragma unroll
    for (int r = 0; r < 2; r++) {
      const int row = row0 + g + 8 * r, p = pos0 + g + 8 * r;
      live[r] = p >= begin && p < len;
      scale[r] = live[r] ? __fmul_rn(((const float *)(tile + kTile * (D / 2)))[row], shrink) : 0.0f;
      if (!value) {
        const uint32_t *from_row = (const uint32_t *)(tile + row * (D / 2)) + t * (D / 32);
        if (D == 128) {
          const uint4 v = *(const uint4 *)from_row;
          w[r][0] = v.x, w[r][1] = v.y, w[r][2] = v.z, w[r][D / 32 - 1] = v.w;
        } else {
#pragma unroll
          for (int i = 0; i < D / 32; i++) w[r][i] = from_row[i];
        }
      } else {
        const bool odd = g & 1;
        const uint2 *pair = (const uint2 *)((const uint32_t *)(tile + (row >> 1) * D) + t * (D / 16));
#pragma unroll
        for (int i = 0; i < D / 32; i++) {
          const uint2 v = pair[i];
          w[r][i] = __byte_perm(v.x, v.y, odd ? 0x7632 : 0x5410);
        }
      }
    }
    // The levels are exact halves, so the first transform needs one product.
    // A half2 holds the nibbles i and i + 4 of a word: with the element's bits
    // renamed (2, 0, 1 for 0, 1, 2) the owner of every output stays the same.
    float y[2][D / 4];
#pragma unroll
    for (int j = 0; j < D / 4; j++) y[0][j] = y[1][j] = 0.0f;
    uint32_t a[2][D / 8];
#pragma unroll
    for (int r = 0; r < 2; r++)
#pragma unroll
      for (int i = 0; i < D / 32; i++) {
        uint32_t o[4];
        unpack8_levels(w[r][i], o);
#pragma unroll
        for (int k = 0; k < 4; k++) a[r][4 * i + k] = o[k];
      }
    hadamard_mma<D, false>(y, a, Hadamard::make<false>());
    hadamard_rest<D>(y);
#pragma unroll
    for (int r = 0; r < 2; r++)
#pragma unroll
      for (int i = 0; i < D / 32; i++) {  // element 2 k + h of a word -> k + 4 h
        float o[8];
#pragma unroll
        for (int k = 0; k < 8; k++) o[(k >> 1) + 4 * (k & 1)] = y[r][8 * i + k];
#pragma unroll
        for (int k = 0; k < 8; k++) y[r][8 * i + k] = __fmul_rn(o[k], scale[r]);
      }
    rotate_back<D, 3>(c, y, false);
#pragma unroll
    for (int r = 0; r < 2; r++) {
      if (!live[r]) continue;
      uint4 *to = (uint4 *)(out + (int64_t)(first + pos0 + g + 8 * r) * c.heads * D + t * (D / 4));
#pragma unroll
      for (int i = 0; i < D / 32; i++)
        __stcs(to + i, make_uint4(pack2<BF16>(y[r][8 * i], y[r][8 * i + 1]),
                                  pack2<BF16>(y[r][8 * i + 2], y[r][8 * i + 3]),
                                  pack2<BF16>(y[r][8 * i + 4], y[r][8 * i + 5]),
                                  pack2<BF16>(y[r][8 * i + 6], y[r][8 * i + 7])));
    }
  }
}

// Parts a warp takes: one while that leaves the card room (a token each), four
// where there are many blocks (14k tokens, in and out: 84 us with one, 72 with two, 67
// with four, 88 with eight).
static int parts_each(int64_t blocks, int heads) { return blocks * 2 * heads > 148 * 16 ? 4 : 1; }

static int64_t block_bound(const Rows &r) {
  return r.starts == nullptr ? r.n : r.rows / 16 + 2 * (int64_t)r.n;
}

template <int D, bool BF16>
static cudaError_t append_d(const Cache &c, int layer, const Rows &rows, const Strided &k,
                            const Strided &v, cudaStream_t st) {
  const int64_t blocks = block_bound(rows);
  const int each = parts_each(blocks, c.heads);
  const int64_t warps = blocks * ((2 * c.heads + each - 1) / each);
  const int64_t grid = (warps + kRowThreads / 32 - 1) / (kRowThreads / 32);
  append_check_kernel<<<1, kCheckThreads, 0, st>>>(c, rows);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  // finds its places while the check runs, and waits for it before it writes
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(kRowThreads);
  cfg.stream = st;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, append_kernel<D, BF16>, c, layer, rows, k, v, blocks, each);
}
template <int D, bool BF16>
static cudaError_t read_d(const Cache &c, int layer, const Rows &rows, void *k, void *v,
                          cudaStream_t st) {
  const int64_t blocks = block_bound(rows);
  const int each = parts_each(blocks, c.heads);
  const int64_t warps = blocks * ((2 * c.heads + each - 1) / each);
  const int64_t grid = (warps + kRowThreads / 32 - 1) / (kRowThreads / 32);
  read_kernel<D, BF16><<<(unsigned)grid, kRowThreads, 0, st>>>(c, layer, rows, (uint16_t *)k,
                                                               (uint16_t *)v, blocks, each);
  return cudaGetLastError();
}

cudaError_t append_launch(const Cache &c, int layer, const Rows &rows, const Strided &k,
                          const Strided &v, bool bf16, cudaStream_t st) {
  switch (c.head_dim) {
    case 64:
      return bf16 ? append_d<64, true>(c, layer, rows, k, v, st)
                  : append_d<64, false>(c, layer, rows, k, v, st);
    case 128:
      return bf16 ? append_d<128, true>(c, layer, rows, k, v, st)
                  : append_d<128, false>(c, layer, rows, k, v, st);
    default:
      return bf16 ? append_d<256, true>(c, layer, rows, k, v, st)
                  : append_d<256, false>(c, layer, rows, k, v, st);
  }
}
cudaError_t read_launch(const Cache &c, int layer, const Rows &rows, void *k, void *v, bool bf16,
                        cudaStream_t st) {
  switch (c.head_dim) {
    case 64:
      return bf16 ? read_d<64, true>(c, layer, rows, k, v, st)
                  : read_d<64, false>(c, layer, rows, k, v, st);
    case 128:
      return bf16 ? read_d<128, true>(c, layer, rows, k, v, st)
                  : read_d<128, false>(c, layer, rows, k, v, st);
    default:
      return bf16 ? read_d<256, true>(c, layer, rows, k, v, st)
                  : read_d<256, false>(c, layer, rows, k, v, st);
  }
}

}  // namespace kv
}  // namespace uvb
