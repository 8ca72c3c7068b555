// kv_attend.cu -- attention of one or more query rows a sequence over the
// cache held in 4 bits: for a query head with rotated row q and its key
// head's tokens j (scales s_j, levels l_j),
//   e_j = scale * s_j <q, l_j>,   out = R^T sum_j softmax(e)_j s'_j l'_j,
// over the tokens the row may see (its own position and those before it).
//
// Bound: HBM, D + 8 bytes a token and key head; the work behind each byte is
// unpacking (5 instructions for 8 codes) and two products with 8 columns.  64
// sequences of 1k to 20k tokens (448 MB of cache): 106 us, 4.2 TB/s; without any
// work on the tiles it takes 87.
// The columns of a block are (row, query head of the group) pairs of one
// sequence and key head, so the codes are read and unpacked once for the whole
// group.  Codes are the A operand of m16n8k16 (keys as rows for q k, dimensions
// as rows for p v): with 8 query columns no row of the product is padding,
// while a 128-row tcgen05 tile would be 94% padding on one side.
//
// Split: all tiles (32 tokens) of all (sequence, column tile, head) jobs lie in
// one line, cut into equal pieces, one for each block of a single wave,
// whatever the lengths are: the host need not know them.  A piece may hold the
// end of a job, whole jobs and the start of another; each part leaves its
// maximum, sum and output (divided by its sum) in scratch, and the block that finds all
// of a job's parts written joins them in order, rotates back and rounds.
//
// Numbers: q is rotated in f32 and rounded to a half, after a power of two that
// brings its row to size 1 (2^-11 relative, below the 4-bit keys' error by 2^6;
// where the rows are halves themselves the remainder goes along as a second
// half, so that the scores lose nothing against the output's own rounding).
// Codes enter the products as the integers that they are and their mean, 7.5
// times the sum, is taken off: from the scores at once, from the outputs every
// four tiles.  Scores, maxima and sums are f32.  The weights are rounded to halves
// after the multiplication by their token's value scale, itself divided by a power
// of two that follows the largest scale seen, but stays within 2^6 of the largest
// product of scale and weight (a large value that weighs nothing takes no bits from
// the others), so they neither overflow nor lose more than 2^-11: beside bf16 rows an eighth of the output's own rounding, beside
// halves as much again (0.00034 of the result's size off in all, where exact
// weights are 0.00021 off), so there the remainder goes along too; that product
// costs 8 rows over 4.5k tokens each 0.7 us of 23.  The running maximum moves only when a score exceeds it by
// 2^8, which keeps the weights below 2^8 and the rescaling of the sums rare.
#include <cfloat>

#include "uv_kv.h"

namespace uvb {
namespace kv {

constexpr int kWarps = 4, kAttendThreads = 32 * kWarps;
constexpr uint32_t kWaitLimit = 1u << 20;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kJump = 8.0f;     // log2 of what a score may exceed its reference by
constexpr float kSpread = 16.0f;  // what a value scale may exceed its reference by
constexpr int kAbove = 6;         // log2 of what that may exceed a scale times its weight by

// Blocks an SM: three where the sums and the query's fragments leave room in
// 168 registers, else two with the longer rings that then fit.
template <int D, int NT, bool BF16>
struct Fit {
  static constexpr int kParts = BF16 ? 1 : 2;  // halves for a query value, and for a weight
  static constexpr int kBlocks = D / 4 * NT + D / 8 * NT * kParts <= 64 ? 3 : 2;
  static constexpr int kStages = kBlocks == 3 ? 384 / D : D == 256 ? 2 : 640 / D;
  static constexpr int kTileBytes = kTile * (D + 8);
  static constexpr int kRing = kWarps * kStages * kTileBytes;  // the warps' rings of tiles
  static constexpr int kRow = D + 4, kJoin = 2 * 8 * NT * kRow * 4;  // two warps' outputs
  static constexpr int kBytes = kRing + kJoin;
};

// Scratch: one part for every (job + block): the sum grows with either along the
// line, so a part is one block's share of one job.  A part's flag holds the
// call's number once the part is written.
struct Parts {
  unsigned long long *flag;  // slots
  float *o;                  // slots x columns x D
  float2 *ml;                // slots x columns: maximum (log2) and sum
};
__host__ __device__ __forceinline__ int64_t flag_bytes(int64_t slots) {
  return (slots * 8 + 127) & ~127ll;
}
__device__ __forceinline__ Parts carve(void *p, int64_t slots, int cols, int D) {
  float *o = (float *)((char *)p + flag_bytes(slots));
  return {(unsigned long long *)p, o, (float2 *)(o + slots * cols * D)};
}
__device__ __forceinline__ void set_flag(unsigned long long *p, unsigned long long v) {
  asm volatile("st.release.gpu.global.u64 [%0], %1;" ::"l"(p), "l"(v) : "memory");
}
// Orders what comes before it against what comes after it, stores before loads
// among them, with every other such fence of the device.
__device__ __forceinline__ void fence_sc() { asm volatile("fence.sc.gpu;" ::: "memory"); }
__device__ __forceinline__ unsigned long long get_flag(const unsigned long long *p) {
  unsigned long long v;
  asm volatile("ld.acquire.gpu.global.u64 %0, [%1];" : "=l"(v) : "l"(p) : "memory");
  return v;
}

// What a job costs beside its tiles (its queries, the join of its parts), in
// tiles: the pieces of the line are equal in time, not in tiles.  64 sequences of
// 1k to 20k tokens take 119 us at 4, 113 at 14, 105 at 20, 107 at 32; 16 of 0.7k
// to 8k 37, 33, 35 and 31; drafts of 8 sequences of 33 to 4.5k 33, 25, 25 and 25.
constexpr int kJobCost = 20;

struct Job {
  int seq, first, n, len, tiles, col_tiles;
  __device__ int64_t units() const { return tiles == 0 ? 0 : tiles + kJobCost; }
};
__device__ __forceinline__ Job load_entry(const Cache &c, const Rows &r, int b, int group,
                                          int cols) {
  Job j;
  j.seq = r.seq(b, c.max_seqs);
  j.first = r.first(b);
  j.n = r.count(b);
  j.len = j.seq < 0 ? 0 : c.length(j.seq);
  j.tiles = (j.len + kTile - 1) / kTile;
  j.col_tiles = (int)(((int64_t)j.n * group + cols - 1) / cols);
  return j;
}

// a / b of numbers that are not negative: few are longer than 32 bits, whose
// division takes a fifth of the time
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
  if (((a | b) >> 32) == 0) return (uint32_t)a / (uint32_t)b;
  return a / b;
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void bulk_load(void *dst, const void *src, uint32_t bytes,
                                          uint64_t *bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::
          "r"(tc::smem_u32(dst)),
      "l"(src), "r"(bytes), "r"(tc::smem_u32(bar))
      : "memory");
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

template <int D>
struct Words {
  uint32_t w[D / 32];
};
template <int D>
__device__ __forceinline__ Words<D> load_words(const uint8_t *p) {
  Words<D> r;
  if (D == 64) {
    const uint2 v = *(const uint2 *)p;
    r.w[0] = v.x;
    r.w[1] = v.y;
  } else {
#pragma unroll
    for (int i = 0; i < D / 128; i++) {
      const uint4 v = ((const uint4 *)p)[i];
      r.w[4 * i] = v.x;
      r.w[4 * i + 1] = v.y;
      r.w[4 * i + 2] = v.z;
      r.w[4 * i + 3] = v.w;
    }
  }
  return r;
}

template <int D, int NT, bool BF16>
__global__ void __launch_bounds__(kAttendThreads, Fit<D, NT, BF16>::kBlocks)
    attend_kernel(Cache c, int layer, Rows rows, AttendArgs a, int64_t slots) {
  using F = Fit<D, NT, BF16>;
  constexpr int kCols = 8 * NT, kStages = F::kStages, kTileBytes = F::kTileBytes, kParts = F::kParts;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint64_t full[kWarps][kStages];
  __shared__ int64_t sums[2][kWarps];
  __shared__ int64_t begin[3];  // first entry of the piece, its first unit, its first job
  __shared__ Job first_job;
  __shared__ float join_m[kWarps][kCols], join_l[kWarps][kCols];
  __shared__ bool complete;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int group = a.q_heads / c.heads;
  const Parts sc = carve(a.scratch, slots, kCols, D);

  if (lane == 0)
    for (int i = 0; i < kStages; i++) tc::mbar_init(&full[warp][i], 1);
  tc::mbar_fence_init();

  // ---- this block's piece of the line of tiles ----
  const int per_thread = (rows.n + kAttendThreads - 1) / kAttendThreads;
  const int e0 = min(tid * per_thread, rows.n), e1 = min(e0 + per_thread, rows.n);
  int64_t my_units = 0, my_jobs = 0;
  for (int b = e0; b < e1; b++) {
    const Job j = load_entry(c, rows, b, group, kCols);
    const int64_t jobs = (int64_t)j.col_tiles * c.heads;
    my_jobs += jobs;
    my_units += jobs * j.units();
  }
  int64_t x = my_units, y = my_jobs;
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t u = __shfl_up_sync(0xffffffffu, x, o), v = __shfl_up_sync(0xffffffffu, y, o);
    if (lane >= o) x += u, y += v;
  }
  if (lane == 31) sums[0][warp] = x, sums[1][warp] = y;
  __syncthreads();
  int64_t total = 0, before_t = x - my_units, before_j = y - my_jobs;
  for (int w = 0; w < kWarps; w++) {
    total += sums[0][w];
    if (w < warp) before_t += sums[0][w], before_j += sums[1][w];
  }
  // at least one tile for every warp of a block
  const int64_t per = max(quotient(total + gridDim.x - 1, gridDim.x), (int64_t)kWarps);
  const int64_t T0 = per * blockIdx.x, T1 = min(T0 + per, total);
  // rows of sequences without a token
  for (int b = blockIdx.x; b < rows.n; b += gridDim.x) {
    const Job j = load_entry(c, rows, b, group, kCols);
    if (j.tiles != 0) continue;
    uint4 *to = (uint4 *)((uint16_t *)a.out + (int64_t)j.first * a.q_heads * D);
    for (int64_t i = tid; i < (int64_t)j.n * a.q_heads * (D / 8); i += kAttendThreads)
      to[i] = make_uint4(0, 0, 0, 0);
    if (a.lse != nullptr)
      for (int64_t i = tid; i < (int64_t)j.n * a.q_heads; i += kAttendThreads)
        a.lse[(int64_t)j.first * a.q_heads + i] = -INFINITY;
  }
  if (T0 >= T1) return;
  if (T0 >= before_t && T0 < before_t + my_units) {
    int64_t bt = before_t, bj = before_j;
    for (int b = e0; b < e1; b++) {
      const Job j = load_entry(c, rows, b, group, kCols);
      const int64_t jobs = (int64_t)j.col_tiles * c.heads;
      if (T0 < bt + jobs * j.units()) {
        begin[0] = b;
        begin[1] = bt;
        begin[2] = bj;
        first_job = j;
        break;
      }
      bt += jobs * j.units();
      bj += jobs;
    }
  }
  __syncthreads();
  int entry = (int)begin[0];
  int64_t base_t = begin[1], base_j = begin[2];
  Job job = first_job;

  uint8_t *ring = smem + warp * kStages * kTileBytes;
  int to_fill = 0, slot = 0;  // the ring's next slot to load, and to read
  uint32_t phase = 0;
  bool dead = false;

  // A segment: the part of a job that lies in this block's piece.
  struct Segment {
    Job job;
    int64_t number;           // of the job
    int first_block, blocks;  // that have a part of it
    int j0, todo, mine, c0, head;  // tiles j0 .. j0 + todo, every fourth this warp's
  };
  int64_t T = T0;
  auto next = [&](Segment *seg) {
    while (T < T1) {
      while (T >= base_t + (int64_t)job.col_tiles * c.heads * job.units()) {
        base_t += (int64_t)job.col_tiles * c.heads * job.units();
        base_j += (int64_t)job.col_tiles * c.heads;
        entry++;
        job = load_entry(c, rows, entry, group, kCols);
      }
      const int64_t local = T - base_t, units = job.units(), jl = quotient(local, units);
      const int off = (int)(local - jl * units);
      const int take = (int)min(units - off, T1 - T);
      T += take;
      const int j0 = max(0, off - kJobCost), j1 = max(0, off + take - kJobCost);
      if (j0 == j1) continue;
      const int ct = (int)(jl / c.heads);
      seg->job = job;
      const int64_t start = base_t + jl * units;
      seg->number = base_j + jl;
      seg->first_block = (int)quotient(start + kJobCost, per);
      seg->blocks = (int)quotient(start + units - 1, per) - seg->first_block + 1;
      seg->head = (int)(jl % c.heads);
      seg->c0 = ct * kCols;
      seg->j0 = j0;
      // tiles that the last of the columns sees something of
      const int lim = job.len - job.n + min((seg->c0 + kCols - 1) / group, job.n - 1) + 1;
      seg->todo = max(0, min(j1, (lim + kTile - 1) / kTile) - j0);
      seg->mine = seg->todo > warp ? (seg->todo - warp + kWarps - 1) / kWarps : 0;
      return true;
    }
    return false;
  };
  const int per_page = c.page_tokens / kTile;
  const uint8_t *src = nullptr;
  auto lookup = [&](const Segment &seg, int from) {  // this warp's tiles from .. from + 31, one a lane
    const int i = from + lane;
    if (i < seg.mine) {
      const int j = seg.j0 + warp + i * kWarps;
      src = c.tile_at(layer, c.page_at(seg.job.seq, j / per_page), seg.head, j % per_page);
    }
  };
  auto issue = [&](int i) {
    const uint8_t *p = (const uint8_t *)__shfl_sync(0xffffffffu, (unsigned long long)src, i & 31);
    if (lane == 0 && !dead) {
      tc::mbar_arrive_expect_tx(&full[warp][to_fill], kTileBytes);
      bulk_load(ring + to_fill * kTileBytes, p, kTileBytes, &full[warp][to_fill]);
    }
    if (++to_fill == kStages) to_fill = 0;
  };
  // Rows g and g + 8 of 16 of a segment's query columns, as they lie.
  auto load_queries = [&](const Segment &seg, int half, uint32_t (&raw)[2][D / 8]) {
#pragma unroll
    for (int r = 0; r < 2; r++) {
      const int col = seg.c0 + 16 * half + 8 * r + g;
      const bool live = 2 * half + r < NT && col < seg.job.n * group;
      const int row = seg.job.first + (live ? col / group : 0);
      const int hq = seg.head * group + (live ? col % group : 0);
      const uint4 *q = (const uint4 *)((const uint16_t *)a.q.p + (int64_t)row * a.q.row +
                                       (int64_t)hq * a.q.head + t * (D / 4));
#pragma unroll
      for (int i = 0; i < D / 32; i++) {
        const uint4 v = live ? __ldg(q + i) : make_uint4(0, 0, 0, 0);
        raw[r][4 * i] = v.x;
        raw[r][4 * i + 1] = v.y;
        raw[r][4 * i + 2] = v.z;
        raw[r][4 * i + 3] = v.w;
      }
    }
  };
  auto start = [&](const Segment &seg) {
    lookup(seg, 0);
    for (int i = 0; i < min(seg.mine, kStages); i++) issue(i);
  };

  // The first queries are asked for ahead of the tiles: behind a ring's worth
  // from every warp of the card they would wait for 3 us.
  uint32_t raw[2][D / 8];
  Segment seg, after;
  bool more = next(&seg);
  if (more) {
    load_queries(seg, 0, raw);
    start(seg);
  }
  while (more) {
    const Job &at = seg.job;
    const int ncol = at.n * group, c0 = seg.c0, head = seg.head, mine = seg.mine;
    const int offset = at.len - at.n;  // position of the entry's first row
    // the exclusive ends of what the tile's first and last rows may see
    const int lim_first = offset + c0 / group + 1;

    // ---- the query columns, rotated, as B fragments ----
    uint32_t qf[kParts][NT][D / 32][4];
    float cs[NT][2], hs[NT][2];  // of the columns 2t, 2t + 1 of each 8
    int lim[NT][2];
#pragma unroll
    for (int half = 0; half < (NT + 1) / 2; half++) {
      if (half > 0) load_queries(seg, half, raw);
      float y[2][D / 4];
      rotate_rows<D, BF16, NT == 1 ? 1 : 2>(c, raw, y);
#pragma unroll
      for (int r = 0; r < 2; r++) {
        if (2 * half + r >= NT) break;
        const int nt = 2 * half + r;
        float m = 0.0f;
#pragma unroll
        for (int j = 0; j < D / 4; j++) m = fmaxf(m, fabsf(y[r][j]));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
        const int e = max(-100, min(log2i(m), 126));
        const float down = exp2i(-e);
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < D / 32; w++)
#pragma unroll
          for (int i = 0; i < 4; i++) {
            // codes of even i come 16 times smaller out of unpack8
            const float f = __fmul_rn(down, i % 2 ? 1.0f : 16.0f);
            float lo = __fmul_rn(y[r][8 * w + i], f), hi = __fmul_rn(y[r][8 * w + i + 4], f);
#pragma unroll
            for (int part = 0; part < kParts; part++) {
              const uint32_t h = pack2<false>(lo, hi);
              const float2 v = unpack2<false>(h);
              sum = __fmaf_rn(__fadd_rn(v.x, v.y), i % 2 ? 1.0f : 0.0625f, sum);
              qf[part][nt][w][i] = h;
              lo = __fsub_rn(lo, v.x);
              hi = __fsub_rn(hi, v.y);
            }
          }
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        // the products give 2^-20 <q, n>, levels are n - 7.5
        const float h = __fmul_rn(-7.5f * 0x1p-20f, sum);
        const float cc = __fmul_rn(__fmul_rn(a.scale, kLog2e * 0x1p20f), exp2i(e));
#pragma unroll
        for (int k = 0; k < 2; k++) {
          hs[nt][k] = __shfl_sync(0xffffffffu, h, 4 * (2 * t + k));
          cs[nt][k] = __shfl_sync(0xffffffffu, cc, 4 * (2 * t + k));
          const int col = c0 + 8 * nt + 2 * t + k;
          lim[nt][k] = offset + min(col / group, at.n - 1) + 1;
        }
      }
    }

    // o: rows of even dimensions in units of 2^-24, of odd ones 2^-20
    float o[D / 16][NT][4], codes[NT][4], m[NT][2], l[NT][2];
    int ve[NT][2];         // a column's value scales are divided by 2^ve
    float down[NT][2];     // 2^-ve
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
#pragma unroll
      for (int mt = 0; mt < D / 16; mt++)
#pragma unroll
        for (int k = 0; k < 4; k++) o[mt][nt][k] = 0.0f;
#pragma unroll
      for (int k = 0; k < 4; k++) codes[nt][k] = 0.0f;
      m[nt][0] = m[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.0f;
      ve[nt][0] = ve[nt][1] = -100;
      down[nt][0] = down[nt][1] = exp2i(100);
    }

    // The codes 0 .. 15 stand for levels of mean zero: taking 7.5 times the
    // weights' sum (a product with ones) off every four tiles keeps the sums as
    // small as the levels' own, so that nothing cancels over a long sequence.
    auto recentre = [&] {
#pragma unroll
      for (int nt = 0; nt < NT; nt++) {
#pragma unroll
        for (int k = 0; k < 2; k++) {
          const float lo = __fmul_rn(codes[nt][k], 7.5f * 0x1p-24f);
          const float hi = __fmul_rn(codes[nt][k], 7.5f * 0x1p-20f);
#pragma unroll
          for (int mt = 0; mt < D / 16; mt++) {
            o[mt][nt][k] = __fsub_rn(o[mt][nt][k], lo);
            o[mt][nt][2 + k] = __fsub_rn(o[mt][nt][2 + k], hi);
          }
        }
#pragma unroll
        for (int k = 0; k < 4; k++) codes[nt][k] = 0.0f;
      }
    };
    // ---- one pass over the warp's tiles ----
    for (int i = 0; i < mine; i++) {
      uint64_t *bar = &full[warp][slot];
      if (!__all_sync(0xffffffffu, tc::mbar_try_wait(bar, phase)) &&
          !__all_sync(0xffffffffu, tc::mbar_wait(bar, phase, kWaitLimit))) {
        // give up: note it, let the copies in flight land, load no more
        if (lane == 0) atomicOr(&c.work[kStatus], kTimeout);
        for (int k = 0; k < min(kStages, mine - i); k++) {
          tc::mbar_wait(&full[warp][slot], phase, kWaitLimit);
          if (++slot == kStages) slot = 0, phase ^= 1;
        }
        dead = true;
      }
      if (dead) break;
      const uint8_t *tile = ring + slot * kTileBytes;
      const int key0 = (seg.j0 + warp + i * kWarps) * kTile;

      float s[2][NT][4];
      Words<D> kw[2][2];
#pragma unroll
      for (int sb = 0; sb < 2; sb++) {
#pragma unroll
        for (int r = 0; r < 2; r++)
          kw[sb][r] = load_words<D>(tile + (16 * sb + 8 * r + g) * (D / 2) + t * (D / 8));
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
          for (int k = 0; k < 4; k++) s[sb][nt][k] = hs[nt][k & 1];
      }
#pragma unroll
      for (int w = 0; w < D / 32; w++)
#pragma unroll
        for (int sb = 0; sb < 2; sb++) {
          uint32_t xa[4], xb[4];
          unpack8(kw[sb][0].w[w], xa);
          unpack8(kw[sb][1].w[w], xb);
#pragma unroll
          for (int k = 0; k < 4; k += 2)
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
              for (int part = 0; part < kParts; part++)
                mma16816<false>(s[sb][nt], xa[k], xb[k], xa[k + 1], xb[k + 1],
                                qf[part][nt][w][k], qf[part][nt][w][k + 1]);
        }
      float ks[2][2], vs[2][2];
      const float *kscale = (const float *)(tile + kTile * (D / 2));
      const float *vscale = (const float *)(tile + kTile * (D + 4));
      // every column sees every token
      const bool whole = __all_sync(0xffffffffu, key0 + kTile <= lim_first);
#pragma unroll
      for (int sb = 0; sb < 2; sb++)
#pragma unroll
        for (int r = 0; r < 2; r++) {
          ks[sb][r] = kscale[16 * sb + 8 * r + g];
          vs[sb][r] = vscale[16 * sb + 8 * r + g];
        }
      // Scores against the running maximum, in place.  Where every column sees
      // every token there is nothing to mask; elsewhere a token that a column
      // does not see neither weighs nor moves that column's references.
      auto seen = [&](int nt, int k, int sb, int r) {
        return key0 + 16 * sb + 8 * r + g < lim[nt][k];
      };
      bool jump = false;
#pragma unroll
      for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int k = 0; k < 2; k++) {
          const float base = m[nt][k] == -INFINITY ? 0.0f : -m[nt][k];
#pragma unroll
          for (int sb = 0; sb < 2; sb++)
#pragma unroll
            for (int r = 0; r < 2; r++)
              s[sb][nt][2 * r + k] =
                  __fmaf_rn(s[sb][nt][2 * r + k], __fmul_rn(cs[nt][k], ks[sb][r]), base);
        }
      if (whole) {
        const float vtop = fmaxf(fmaxf(vs[0][0], vs[0][1]), fmaxf(vs[1][0], vs[1][1]));
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
          for (int k = 0; k < 2; k++) {
            const float top = fmaxf(fmaxf(s[0][nt][k], s[0][nt][2 + k]), fmaxf(s[1][nt][k], s[1][nt][2 + k]));
            jump |= top > kJump || m[nt][k] == -INFINITY || !(__fmul_rn(vtop, down[nt][k]) <= kSpread);
          }
      } else {
        jump = true;
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
          for (int k = 0; k < 2; k++)
#pragma unroll
            for (int sb = 0; sb < 2; sb++)
#pragma unroll
              for (int r = 0; r < 2; r++)
                if (!seen(nt, k, sb, r)) s[sb][nt][2 * r + k] = -INFINITY;
      }
      if (__any_sync(0xffffffffu, jump)) {
        // new references, for the columns that need them
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
          for (int k = 0; k < 2; k++) {
            float top = max_nan(max_nan(s[0][nt][k], s[0][nt][2 + k]), max_nan(s[1][nt][k], s[1][nt][2 + k]));
#pragma unroll
            for (int x = 4; x < 32; x *= 2) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, x));
            const bool none = m[nt][k] == -INFINITY;
            const float up = none ? top : top > kJump ? top : 0.0f;  // what m grows by
            // the largest value scale, and the largest of them times its weight
            float vtop = 0.0f, wtop = 0.0f;
#pragma unroll
            for (int sb = 0; sb < 2; sb++)
#pragma unroll
              for (int r = 0; r < 2; r++)
                if ((whole || seen(nt, k, sb, r)) && vs[sb][r] <= FLT_MAX) {
                  vtop = fmaxf(vtop, vs[sb][r]);
                  wtop = fmaxf(wtop, __fmul_rn(exp2_fast(__fsub_rn(s[sb][nt][2 * r + k], up)),
                                               __fmul_rn(vs[sb][r], 0x1p-16f)));
                }
#pragma unroll
            for (int x = 4; x < 32; x *= 2) {
              vtop = fmaxf(vtop, __shfl_xor_sync(0xffffffffu, vtop, x));
              wtop = fmaxf(wtop, __shfl_xor_sync(0xffffffffu, wtop, x));
            }
            // What the sums hold shrinks with m, and the reference of their values
            // with it; it rises for values of weight, to 2^kAbove times them at most.
            const float grown = none ? 0.0f : up;
            const int kept = max(ve[nt][k] - (int)fminf(grown, 1000.0f), -100);
            const int risen = min(min(log2i(vtop), log2i(wtop) + 16 + kAbove), 126);
            const int ne = __fmul_rn(vtop, exp2i(-kept)) > kSpread ? max(kept, risen) : kept;
            // (a column that has seen nothing has sums of zero: any factor keeps them)
            const float f = exp2_fast(-grown);
            const float both = exp2_fast(__fsub_rn((float)(ve[nt][k] - ne), grown));
            if (none) m[nt][k] = top;
            else m[nt][k] = __fadd_rn(m[nt][k], up);
            ve[nt][k] = ne;
            down[nt][k] = exp2i(-ne);
            if (up != -INFINITY)
#pragma unroll
              for (int sb = 0; sb < 2; sb++)
#pragma unroll
                for (int r = 0; r < 2; r++) s[sb][nt][2 * r + k] = __fsub_rn(s[sb][nt][2 * r + k], up);
            l[nt][k] = __fmul_rn(l[nt][k], f);
            codes[nt][k] = __fmul_rn(codes[nt][k], both);
            codes[nt][2 + k] = __fmul_rn(codes[nt][2 + k], both);
#pragma unroll
            for (int mt = 0; mt < D / 16; mt++) {
              o[mt][nt][k] = __fmul_rn(o[mt][nt][k], both);
              o[mt][nt][2 + k] = __fmul_rn(o[mt][nt][2 + k], both);
            }
          }
      }
#pragma unroll
      for (int sb = 0; sb < 2; sb++) {
        uint32_t p[kParts][NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
          float w[4];
#pragma unroll
          for (int k = 0; k < 2; k++)
#pragma unroll
            for (int r = 0; r < 2; r++) {
              const float e = exp2_fast(s[sb][nt][2 * r + k]);
              l[nt][k] = __fadd_rn(l[nt][k], e);
              w[2 * r + k] = __fmul_rn(__fmul_rn(e, down[nt][k]), vs[sb][r]);
            }
          if (!whole)  // a token that is not seen weighs nothing even if its scale is no number
#pragma unroll
            for (int k = 0; k < 2; k++)
#pragma unroll
              for (int r = 0; r < 2; r++)
                if (!seen(nt, k, sb, r)) w[2 * r + k] = 0.0f;
#pragma unroll
          for (int part = 0; part < kParts; part++) {
#pragma unroll
            for (int r = 0; r < 2; r++) {
              const uint32_t h = pack2<false>(w[2 * r], w[2 * r + 1]);
              if (part + 1 < kParts) {
                const float2 v = unpack2<false>(h);
                w[2 * r] = __fsub_rn(w[2 * r], v.x);
                w[2 * r + 1] = __fsub_rn(w[2 * r + 1], v.y);
              }
              p[part][nt][r] = transpose8x8(h);
            }
            mma16816<false>(codes[nt], 0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u,
                            p[part][nt][0], p[part][nt][1]);
          }
        }
        const uint8_t *pairp = tile + kTile * (D / 2 + 4) + (8 * sb + t) * D + g * (D / 8);
        const Words<D> va = load_words<D>(pairp), vb = load_words<D>(pairp + 4 * D);
#pragma unroll
        for (int w = 0; w < D / 32; w++) {
          uint32_t xa[4], xb[4];
          unpack8(va.w[w], xa);
          unpack8(vb.w[w], xb);
#pragma unroll
          for (int k = 0; k < 2; k++)
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
              for (int part = 0; part < kParts; part++)
                mma16816<false>(o[2 * w + k][nt], xa[2 * k], xa[2 * k + 1], xb[2 * k], xb[2 * k + 1],
                                p[part][nt][0], p[part][nt][1]);
        }
      }
      if ((i & 3) == 3) recentre();
      __syncwarp();  // every lane has read the slot
      const int ahead = i + kStages;
      if (ahead < mine) {
        if ((ahead & 31) == 0) lookup(seg, ahead);
        issue(ahead);
      }
      if (++slot == kStages) slot = 0, phase ^= 1;
    }

    recentre();
    // the next segment's tiles are on their way while this one's parts join
    more = next(&after);
    if (more) {
      load_queries(after, 0, raw);
      start(after);
    }

    // ---- join the warps' parts: 2 and 3 leave theirs, 0 and 1 add to them ----
    // (maxima of maxima keep NaN: a column that has met nothing but NaN is not one
    // that has seen nothing)
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
      for (int k = 0; k < 2; k++) {
#pragma unroll
        for (int x = 4; x < 32; x *= 2)
          l[nt][k] = __fadd_rn(l[nt][k], __shfl_xor_sync(0xffffffffu, l[nt][k], x));
        if (g == 0) {
          join_m[warp][8 * nt + 2 * t + k] = m[nt][k];
          join_l[warp][8 * nt + 2 * t + k] = l[nt][k];
        }
      }
    __syncthreads();
    auto total_of = [&](int col, float *top) {
      float sum = 0.0f;
      *top = join_m[0][col];
      for (int v = 1; v < kWarps; v++) *top = max_nan(*top, join_m[v][col]);
      for (int v = 0; v < kWarps; v++)
        if (join_m[v][col] != -INFINITY)
          sum = __fmaf_rn(join_l[v][col], exp2_fast(__fsub_rn(join_m[v][col], *top)), sum);
      return sum;
    };
    // (divided by the block's sum at once: a mean of values is a float where their
    // sum may not be one)
    constexpr int kRow = F::kRow;
    float *out = (float *)(smem + F::kRing), *mine_out = out + (warp & 1) * kCols * kRow;
#pragma unroll
    for (int step = 0; step < 2; step++) {
      if (warp / 2 != step) {  // first 2 and 3
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
          for (int k = 0; k < 2; k++) {
            const int col = 8 * nt + 2 * t + k;
            float top;
            const float sum = total_of(col, &top);
            // a warp without a visible token adds nothing, whatever its sums hold
            const bool none = m[nt][k] == -INFINITY;
            const float f = __fdiv_rn(exp2_fast(__fsub_rn(m[nt][k], top)), sum);
            const float flo = __fmul_rn(f, 0x1p24f), fhi = __fmul_rn(f, 0x1p20f);
            const float unit = exp2i(ve[nt][k]);
#pragma unroll
            for (int mt = 0; mt < D / 16; mt++) {
              float2 *to = (float2 *)(mine_out + col * kRow + g * (D / 8) + 2 * mt);
              const float2 was = step == 0 ? make_float2(0.0f, 0.0f) : *to;
              const float u = none ? 0.0f : __fmul_rn(__fmul_rn(o[mt][nt][k], flo), unit);
              const float v = none ? 0.0f : __fmul_rn(__fmul_rn(o[mt][nt][2 + k], fhi), unit);
              *to = make_float2(__fadd_rn(was.x, u), __fadd_rn(was.y, v));
            }
          }
      }
      __syncthreads();
    }
    // ---- the job's result, or this block's part of it ----
    // (starts that do not rise give more jobs than rows allow: no slot, no part)
    const int64_t part = seg.number + blockIdx.x;
    const bool fits = seg.number + seg.first_block + seg.blocks <= slots;
    bool final = seg.blocks == 1 && fits;
    auto write_lse = [&](int col, float top, float sum) {
      const int x = c0 + col;
      if (a.lse != nullptr && x < ncol)
        a.lse[(int64_t)(at.first + x / group) * a.q_heads + head * group + x % group] =
            top == -INFINITY ? -INFINITY : __fmul_rn(__fadd_rn(top, __log2f(sum)), kLn2);
    };
    if (seg.blocks == 1) {
      for (int i = tid; i < kCols * (D / 4); i += kAttendThreads) {
        const int col = i / (D / 4), d4 = i % (D / 4);
        float4 *u = (float4 *)(out + col * kRow + 4 * d4);
        const float4 v = *(const float4 *)(out + (kCols + col) * kRow + 4 * d4), w = *u;
        *u = make_float4(__fadd_rn(w.x, v.x), __fadd_rn(w.y, v.y), __fadd_rn(w.z, v.z),
                         __fadd_rn(w.w, v.w));
        if (d4 == 0 && fits) {
          float top;
          const float sum = total_of(col, &top);
          write_lse(col, top, sum);
        }
      }
      __syncthreads();
    } else if (fits) {
      for (int i = tid; i < kCols * (D / 4); i += kAttendThreads) {
        const int col = i / (D / 4), d4 = i % (D / 4);
        const float4 u = *(const float4 *)(out + col * kRow + 4 * d4);
        const float4 v = *(const float4 *)(out + (kCols + col) * kRow + 4 * d4);
        __stcg((float4 *)(sc.o + (part * kCols + col) * D) + d4,
               make_float4(__fadd_rn(u.x, v.x), __fadd_rn(u.y, v.y), __fadd_rn(u.z, v.z),
                           __fadd_rn(u.w, v.w)));
      }
      if (tid < kCols) {
        float top;
        const float sum = total_of(tid, &top);
        __stcg(&sc.ml[part * kCols + tid], make_float2(top, sum));
      }
      __syncthreads();
      if (tid == 0) set_flag(&sc.flag[part], a.call);
      // Whoever finds every part written joins them, in their order.  Between a
      // block's own flag and its look at the others' stands a fence.sc (by the lane
      // that set the flag; the warp looks behind it): those fences have one order,
      // and the block whose fence is the last in it sees every flag (or zeros, from a
      // block that saw them all and joins).  Release and acquire alone would let two
      // blocks miss each other's.  Two that finish together may both join, and write
      // the same bytes.  Nothing waits, and no counter has to start at zero.
      const int64_t first = seg.number + seg.first_block;
      if (warp == 0) {
        if (lane == 0) fence_sc();
        __syncwarp();
        bool all = true;
        for (int i = lane; i < seg.blocks; i += 32) all = all && get_flag(&sc.flag[first + i]) == a.call;
        all = __all_sync(0xffffffffu, all);
        if (lane == 0) complete = all;
      }
      __syncthreads();
      final = complete;
      if (final) {
        // (a replayed graph makes the same call in the same scratch)
        for (int i = tid; i < seg.blocks; i += kAttendThreads) set_flag(&sc.flag[first + i], 0);
        constexpr int V = D / 32;
        for (int col = warp; col < kCols; col += kWarps) {
          auto load = [&](int i) {
            return i < seg.blocks ? __ldcg(&sc.ml[(first + i) * kCols + col])
                                  : make_float2(-INFINITY, 0.0f);
          };
          const float2 ml0 = load(lane);
          float top = ml0.x, sum = 0.0f, acc[V];
          for (int i = lane + 32; i < seg.blocks; i += 32) top = max_nan(top, load(i).x);
          for (int x = 16; x; x >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, x));
          // a part's sum against the largest maximum
          auto weight = [&](float2 ml) {
            return ml.x == -INFINITY ? 0.0f : __fmul_rn(ml.y, exp2_fast(__fsub_rn(ml.x, top)));
          };
          for (int i = lane; i < seg.blocks; i += 32)
            sum = __fadd_rn(sum, weight(i == lane ? ml0 : load(i)));
          for (int x = 16; x; x >>= 1) sum = __fadd_rn(sum, __shfl_xor_sync(0xffffffffu, sum, x));
          const float inv = top == -INFINITY ? 0.0f : __fdiv_rn(1.0f, sum);
#pragma unroll
          for (int v = 0; v < V; v++) acc[v] = 0.0f;
          for (int i0 = 0; i0 < seg.blocks; i0 += 32) {
            const float f = __fmul_rn(weight(i0 == 0 ? ml0 : load(i0 + lane)), inv);
            const int n = min(32, seg.blocks - i0);
#pragma unroll 4
            for (int i = 0; i < n; i++) {
              const float w = __shfl_sync(0xffffffffu, f, i);
              const float2 *from =
                  (const float2 *)(sc.o + ((first + i0 + i) * kCols + col) * D + lane * V);
#pragma unroll
              for (int v = 0; v < V; v += 2) {
                const float2 z = __ldcg(from + v / 2);
                acc[v] = __fmaf_rn(z.x, w, acc[v]);
                acc[v + 1] = __fmaf_rn(z.y, w, acc[v + 1]);
              }
            }
          }
#pragma unroll
          for (int v = 0; v < V; v++) out[col * kRow + lane * V + v] = acc[v];
          if (lane == 0) write_lse(col, top, sum);
        }
        __syncthreads();
      }
    }
    if (final) {
      for (int half = warp; half < (NT + 1) / 2; half += kWarps) {
        float y[2][D / 4];
        const float f = rotation_scale<D>(c);  // ahead: the transform then passes no float
#pragma unroll
        for (int r = 0; r < 2; r++)
#pragma unroll
          for (int j = 0; j < D / 4; j++) {
            const int col = 16 * half + 8 * r + g;
            y[r][j] = col < kCols ? __fmul_rn(out[(col < kCols ? col : 0) * kRow + t * (D / 4) + j], f) : 0.0f;
          }
        rotate_back<D, 2>(c, y, true);
#pragma unroll
        for (int r = 0; r < 2; r++) {
          const int col = 16 * half + 8 * r + g, x = c0 + col;
          if (col >= kCols || x >= ncol) continue;
          uint4 *to = (uint4 *)((uint16_t *)a.out +
                                ((int64_t)(at.first + x / group) * a.q_heads + head * group + x % group) * D +
                                t * (D / 4));
#pragma unroll
          for (int i = 0; i < D / 32; i++)
            to[i] = make_uint4(pack2<BF16>(y[r][8 * i], y[r][8 * i + 1]),
                               pack2<BF16>(y[r][8 * i + 2], y[r][8 * i + 3]),
                               pack2<BF16>(y[r][8 * i + 4], y[r][8 * i + 5]),
                               pack2<BF16>(y[r][8 * i + 6], y[r][8 * i + 7]));
        }
      }
    }
    __syncthreads();  // the join's bytes are free again
    seg = after;
  }
}

// ---- launches ----
// Columns of a tile: the fewest eights that hold a sequence's usual columns,
// so that one row of a group of 8 does not pay for 16; what is above the
// largest would not fit in registers.
static int column_eights(int D, int64_t cols) {
  if (D == 256 || cols <= 8) return 1;
  if (D == 128 || cols <= 16) return 2;
  return 4;
}

AttendPlan attend_plan(const Cache &c, int n, int rows, int most, int q_heads, int sms) {
  AttendPlan p;
  const int group = q_heads / c.heads;
  p.cols = 8 * column_eights(c.head_dim, (int64_t)group * most);
  p.jobs = ((int64_t)rows * group / p.cols + n) * c.heads;
  p.sms = sms;
  const int64_t slots = p.jobs + 3 * sms;
  p.bytes = flag_bytes(slots) + slots * p.cols * (c.head_dim + 2) * 4;
  return p;
}

template <int D, int NT, bool BF16>
static cudaError_t attend_nt(const Cache &c, int layer, const Rows &rows, const AttendArgs &a,
                             const AttendPlan &plan, cudaStream_t st) {
  const int64_t slots = plan.jobs + 3 * plan.sms;
  using F = Fit<D, NT, BF16>;
  const int smem = F::kBytes, workers = F::kBlocks * plan.sms;
  cudaError_t e = cudaFuncSetAttribute(attend_kernel<D, NT, BF16>,
                                       cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  attend_kernel<D, NT, BF16><<<workers, kAttendThreads, smem, st>>>(c, layer, rows, a, slots);
  return cudaGetLastError();
}

template <bool BF16>
static cudaError_t attend_t(const Cache &c, int layer, const Rows &rows, const AttendArgs &a,
                            const AttendPlan &p, cudaStream_t st) {
  if (c.head_dim == 256) return attend_nt<256, 1, BF16>(c, layer, rows, a, p, st);
  if (c.head_dim == 128)
    return p.cols == 8 ? attend_nt<128, 1, BF16>(c, layer, rows, a, p, st)
                       : attend_nt<128, 2, BF16>(c, layer, rows, a, p, st);
  if (p.cols == 8) return attend_nt<64, 1, BF16>(c, layer, rows, a, p, st);
  if (p.cols == 16) return attend_nt<64, 2, BF16>(c, layer, rows, a, p, st);
  return attend_nt<64, 4, BF16>(c, layer, rows, a, p, st);
}

cudaError_t attend_launch(const Cache &c, int layer, const Rows &rows, const AttendArgs &a,
                          const AttendPlan &plan, bool bf16, cudaStream_t st) {
  return bf16 ? attend_t<true>(c, layer, rows, a, plan, st)
              : attend_t<false>(c, layer, rows, a, plan, st);
}

}  // namespace kv
}  // namespace uvb
