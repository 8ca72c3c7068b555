// prompt.cu -- attention over whole prompts: packed sequences of different
// lengths, grouped heads, causal or not.  Sequence b owns query rows
// [starts_q[b], starts_q[b + 1]) and key rows [starts_k[b], starts_k[b + 1]);
// its queries are the last of its keys, so with a mask row i sees keys
// j <= i + (keys - queries).  out = softmax(scale q k^T) v, a row that sees
// nothing is zero.
//
// A tile is 128 query rows of one head.  Per 128 keys: S = Q K^T into TMEM
// (tcgen05, M = N = 128), a warpgroup with one row a thread takes S into
// registers (exponentials and sums without any shuffle), writes P back over S, and
// O += P V takes P from TMEM, its first 64 keys while the exponentials of the
// others still run.  Two tiles share an SM: while one is in its softmax the tensor
// core works for the other.  At D = 128 they are one block's, with the same keys
// (two heads of a group, or 256 consecutive rows where the group is odd); at
// D = 64 two blocks', each of which starts and writes out while the other works.
// (With a block for every piece of work, one long prompt of D = 128, 8192 tokens and
// 32 heads, took 562 us in the first form and 640 in the second, which has room for
// one tile of keys and one of values; 48 short texts of D = 64 took 66 and 49 us.)
//
//   warps 0-3 (, 4-7)  softmax and output of a tile
//   the next one       issues the products, owns the TMEM
//   the next one       finds the work, loads Q, K, V by TMA (one lane)
//   the next two       mend the values of blocks with masked keys (below)
//
// The grid has a block for every piece of work (its one or two tiles), and a block
// that has loaded its piece's last keys cancels one that has not started and does its
// work (the hardware hands them out in order): that piece's queries and first keys
// come, and its first scores are made, while this one's output goes out.  Beside a
// start and an end for every piece this took 7 packed prompts from 154 to 149 us and
// 48 texts from 45 to 43; what mattered more was code that runs once a piece, at some
// 10 cycles an instruction: the look over the values, the search, the output.
//
// Blocks of keys go from the last, masked ones to the first.  A row's weights
// stand against a reference, the maximum of the first keys that it sees, and no
// maximum is taken after that: as long as the sums of its weights stay below
// 2^14 times the reference's (2^7 of halves) it serves as well.  Where one does not, the row takes a new
// reference and its warp rescales O in TMEM.
//
// What a row does not see must not reach it, but a weight of zero times a value
// of infinity or NaN is a NaN.  So in blocks with a masked key such values are
// taken out (as are the next sequence's rows), and for every column the first
// key that held one is kept: rows that see that key get it added to their
// output.  Two warps look for the largest magnitude of a block (16 bits a value, two
// at a time) and go through it value by value only where there is one.
//
// Bound: per 128 x 128 tile and D = 128 the two products take 1024 cycles of
// the tensor core, the exponentials 1024 of the MUFU (16 a cycle), and their arguments,
// sums and packing about as many issue cycles.  (A polynomial in the FMA pipe for a
// quarter of them takes issue slots instead: texts 39.2 us with it and 33.7 without,
// 8192 tokens 543 and 542, packed prompts 124 and 123.)  A tile's chain (scores, 128
// exponentials a thread at about 7 cycles, product) takes 2300 cycles with the
// other tile beside it, so 3500 pass for two tiles, of which the tensor core
// works 2048: 1010 TFLOP/s for 8192 tokens and 32 heads (0.54 ms), at the 1.69 GHz
// that the power limit then leaves.
#include <cfloat>
#include <climits>
#include <cuda.h>

#include "capi_internal.h"
#include "uv_prompt.h"

namespace uvb {
namespace prompt {

constexpr int kRows = 128, kKeys = 128;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
// Barriers of mended values, in turn: the ring holds at most three blocks of values whose
// product is still to be issued, so none completes a second time before it was waited for.
// (An output waits for its piece's last one; by then at most the next piece's are mended,
// and 256 rows end within three blocks.)
constexpr int kMends = 4;
// A row's reference weighs 2^lift, and weights (sums of 32 of them) up to kGrow stay
// unanswered.  Halves are exact to 2^-25 at their small end: lifted by 8, a weight keeps
// 11 bits down to 2^-22 of its row's largest, and what the others may grow by, 2^7, is
// still beyond what the maximum of a row's first keys is usually passed by.  Bfloats
// have the exponents to spare: lowered by 20, the sums of a million of the largest
// values are floats.
template <bool BF16>
struct Weights {
  static constexpr float kLift = BF16 ? -20.0f : 8.0f;
  static constexpr float kGrow = BF16 ? 0x1p-6f : 0x1p15f;
};

__device__ __forceinline__ int bounded(int x, int hi) { return x < 0 ? 0 : (x < hi ? x : hi); }

using kv::max_nan;
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Half of a transpose over lanes: a of the lane without `bit` stays, b of the one with it.
__device__ __forceinline__ void trade(uint4 &a, uint4 &b, int bit) {
  const bool hi = threadIdx.x & bit;
  auto word = [&](uint32_t &x, uint32_t &y) {
    const uint32_t z = __shfl_xor_sync(0xffffffffu, hi ? x : y, bit);
    if (hi) x = z;
    else y = z;
  };
  word(a.x, b.x);
  word(a.y, b.y);
  word(a.z, b.z);
  word(a.w, b.w);
}

// ---- pairs of floats ----
using f2 = unsigned long long;
__device__ __forceinline__ f2 pair(float a, float b) {
  f2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 split(f2 v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) {
  f2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f2 add2(f2 a, f2 b) {
  f2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// ---- tensor core plumbing beside uv_tc.cuh ----
// A bounded wait (a second at most) whose polls sleep in hardware until the
// phase ends: polls that come back at once took two fifths of the issue slots
// from the warps that had work.
__device__ __forceinline__ bool wait_for(uint64_t *bar, int phase) {
  for (int i = 0; i < 1 << 16; i++) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, 20000;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(tc::smem_u32(bar)), "r"((uint32_t)phase & 1u)
        : "memory");
    if (done) return true;
  }
  return false;
}
// A wait for another role of the block, which may itself run into the limit first.
__device__ __forceinline__ bool wait_long(uint64_t *bar, int64_t phase) {
  bool done = false;
  for (int i = 0; i < 4 && !done; i++) done = wait_for(bar, phase);
  return done;
}
// Asks for the index of a block that has not started, to do its work here: the
// answer (16 bytes) arrives on `bar`.
__device__ __forceinline__ void ask_next(void *answer, uint64_t *bar) {
  tc::mbar_arrive_expect_tx(bar, 16);
  asm volatile(
      "clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128"
      " [%0], [%1];" ::"r"(tc::smem_u32(answer)),
      "r"(tc::smem_u32(bar))
      : "memory");
}
// The index, or -1 where none was left.
__device__ __forceinline__ int answer_of(const void *answer) {
  int block;
  asm volatile(
      "{\n\t.reg .b128 a;\n\t.reg .pred p;\n\t"
      "ld.shared.b128 a, [%1];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, a;\n\t"
      "mov.b32 %0, -1;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %0, a;\n\t}"
      : "=r"(block)
      : "r"(tc::smem_u32(answer))
      : "memory");
  return block;
}
// Whether any of the 64 threads that mend says so.
__device__ __forceinline__ bool any_of_64(bool x) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %1, 0;\n\t"
      "barrier.red.or.pred q, 1, 64, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"((uint32_t)x)
      : "memory");
  return r;
}
__device__ __forceinline__ void tma_load_3d(void *dst, const CUtensorMap *map, int x, int y, int z,
                                            uint64_t *bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(tc::smem_u32(dst)),
      "l"((uint64_t)map), "r"(tc::smem_u32(bar)), "r"(x), "r"(y), "r"(z)
      : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t *r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]),
      "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]),
      "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t *r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return __shfl_sync(0xffffffffu, x, 0); }
// D += A B, issued by the lane whose `leader` is set: A in TMEM (row i in lane
// i, K pairs low half first), or both in shared memory.
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc,
                                       bool accumulate, uint32_t leader) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate), "r"(leader)
      : "memory");
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                       bool accumulate, uint32_t leader) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate), "r"(leader)
      : "memory");
}
__device__ __forceinline__ void mma_commit(uint64_t *bar, uint32_t leader) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(
          tc::smem_u32(bar)),
      "r"(leader)
      : "memory");
}
// Descriptor of a B operand whose N index is contiguous (values as they lie:
// rows are keys): 64 columns (128 bytes, 128-byte swizzle) a block of N, blocks
// `block` bytes apart, 8 keys 1024 bytes apart.
__device__ __forceinline__ uint64_t sw128_desc_n(uint32_t addr, uint32_t block) {
  uint64_t d = 0;
  d |= (uint64_t)((addr >> 4) & 0x3FFFu);
  d |= (uint64_t)(block >> 4) << 16;
  d |= (uint64_t)(1024u >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}
// kind::f16 with f32 accumulators: format of A and B in [7,10) and [10,13)
// (1 = bfloat), bit 16: B's N index is the contiguous one.
__device__ __forceinline__ constexpr uint32_t idesc(int M, int N, bool bf16, bool b_n) {
  return tc::idesc_f16_f32(M, N) | (bf16 ? (1u << 7 | 1u << 10) : 0u) | (b_n ? 1u << 16 : 0u);
}

template <int D>
struct Shape {
  static constexpr int kTiles = D == 128 ? 2 : 1, kBlocks = 3 - kTiles;  // blocks an SM
  static constexpr int kSoftmaxWarps = 4 * kTiles, kThreads = 32 * (kSoftmaxWarps + 4);
  static constexpr int kSlots = kTiles == 2 ? 5 : 4;  // tiles of keys and values in turn
  static constexpr int kTile = 128 * D * 2;           // bytes of 128 rows
  static constexpr int kQ = 0, kRing = kTiles * kTile, kOdd = kRing + kSlots * kTile;
  static constexpr int kBars = kOdd + 3 * D * 4;
  static constexpr int kBytes = kBars + 320;
  // TMEM: S (then P) of the tiles, then their O
  static constexpr int kO = 128 * kTiles, kColumns = 256 * kTiles;
  // Registers of the softmax warps and of the others: they add up to what the
  // block was launched with (8 x 224 + 4 x 56 = 12 x 168, 4 x 208 + 4 x 48 = 8 x 128).
  static constexpr int kMore = kTiles == 2 ? 224 : 208, kLess = kTiles == 2 ? 56 : 48;
};

// What a block works on.
struct Item {
  int q0, nq, k0, nk;     // the sequence's rows
  int head[2], i0[2];     // a tile's head and first row in the sequence
  int blocks[2], n;       // key blocks of a tile, and of the longer one
  int whole;              // blocks below this one have no masked key
};

__device__ __forceinline__ int limit(const Args &a, const Item &it, int row) {
  return a.causal ? max(0, min(it.nk, row + it.nk - it.nq + 1)) : it.nk;
}

// A block's tiles are two heads of a group, or consecutive rows of one head.
template <int TILES>
__host__ __device__ __forceinline__ bool pairs_heads(const Args &a) {
  return TILES == 2 && a.q_heads / a.heads % 2 == 0;
}

// Fills in the tiles of rows i0 .. of entry b.
template <int TILES>
__device__ __forceinline__ void describe(const Args &a, int b, int64_t i0, int h, Item *it) {
  const bool twins = pairs_heads<TILES>(a);
  it->q0 = bounded(a.starts_q[b], a.rows_q);
  it->nq = bounded(a.starts_q[b + 1], a.rows_q) - it->q0;
  it->k0 = bounded(a.starts_k[b], a.rows_k);
  it->nk = max(0, bounded(a.starts_k[b + 1], a.rows_k) - it->k0);
  int first = INT_MAX;
  it->n = 0;
  for (int t = 0; t < TILES; t++) {
    it->head[t] = twins ? 2 * h + t : h;
    it->i0[t] = (int)i0 + (twins ? 0 : t * kRows);
    it->blocks[t] = 0;
    if (it->i0[t] < it->nq) {
      it->blocks[t] =
          (limit(a, *it, min(it->i0[t] + kRows, it->nq) - 1) + kKeys - 1) / kKeys;
      first = min(first, limit(a, *it, it->i0[t]));
    }
    it->n = max(it->n, it->blocks[t]);
  }
  it->whole = first / kKeys;
}

// One warp's search for a block's work.  Tiles go in the order of their key
// blocks, most first, so that no long one is left for the end: how many tiles of
// an entry have c blocks or more is a division, so the u-th tile is a binary
// search over c, with the entries over the lanes.  (One sequence of 6000 tokens
// ahead of 90 of 300, 8 heads of 128: 226 us in the order of the pack, from its
// end, 152 so.)  Past 128 entries the order is the pack's.
template <int TILES>
__device__ __forceinline__ bool find_item(const Args &a, int block, Item *it) {
  constexpr int kEach = 4;
  const bool twins = pairs_heads<TILES>(a);
  const int shift = !twins && TILES == 2 ? 8 : 7, rows = 1 << shift;
  const int heads = twins ? a.q_heads / 2 : a.q_heads;
  const int u = block / heads;
  const int h = block % heads, lane = threadIdx.x & 31;
  if (a.n > 32 * kEach) {
    // entry b has starts_q[b + 1] / rows - starts_q[b] / rows + 1 tiles
    const int64_t w = (int64_t)a.rows_q / rows + a.n - 1 - u;
    int lo = 0, hi = a.n - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (bounded(a.starts_q[mid], a.rows_q) / rows + mid <= w) lo = mid;
      else hi = mid - 1;
    }
    const int q0 = bounded(a.starts_q[lo], a.rows_q);
    const int64_t i0 = (w - (q0 / rows + lo)) * rows;
    if (i0 < 0 || i0 >= bounded(a.starts_q[lo + 1], a.rows_q) - q0) return false;
    if (lane == 0) describe<TILES>(a, lo, i0, h, it);
    return true;
  }
  int nq[kEach], nk[kEach], most = 0;
#pragma unroll
  for (int s = 0; s < kEach; s++) {
    const int b = 32 * s + lane;
    nq[s] = nk[s] = 0;
    if (b < a.n) {
      nq[s] = max(0, bounded(a.starts_q[b + 1], a.rows_q) - bounded(a.starts_q[b], a.rows_q));
      nk[s] = max(0, bounded(a.starts_k[b + 1], a.rows_k) - bounded(a.starts_k[b], a.rows_k));
    }
    most = max(most, (nk[s] + kKeys - 1) / kKeys);
  }
  // an entry's first tile whose last row sees something of key block c - 1
  auto begin = [&](int s, int c) {
    const int tiles = (nq[s] + rows - 1) >> shift;
    if (c == 0) return 0;
    const int x = (c - 1) * kKeys + (a.causal ? nq[s] - nk[s] : 0);
    if (!a.causal) return x < nk[s] ? 0 : tiles;
    return x >= nq[s] ? tiles : x < 0 ? 0 : x >> shift;
  };
  auto at_least = [&](int c) {  // tiles with c blocks or more, of all entries
    int sum = 0;
#pragma unroll
    for (int s = 0; s < kEach; s++)
      if (32 * s < a.n) sum += ((nq[s] + rows - 1) >> shift) - begin(s, c);
    return __reduce_add_sync(0xffffffffu, sum);
  };
  if (u >= at_least(0)) return false;
  int lo = 0, hi = __reduce_max_sync(0xffffffffu, most);
  while (lo < hi) {  // the largest c with more than u tiles
    const int mid = (lo + hi + 1) >> 1;
    if (at_least(mid) > u) lo = mid;
    else hi = mid - 1;
  }
  int v = u - at_least(lo + 1);  // among the tiles with exactly c blocks
#pragma unroll
  for (int s = 0; s < kEach; s++) {
    const int from = begin(s, lo), count = begin(s, lo + 1) - from;
    int before = count;
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, before, o);
      if (lane >= o) before += x;
    }
    const int sum = __shfl_sync(0xffffffffu, before, 31);
    before -= count;
    if (v >= before && v < before + count)
      describe<TILES>(a, 32 * s + lane, (int64_t)(from + v - before) * rows, h, it);
    v -= sum;
    if (v < 0) break;
  }
  return true;
}

// A piece of work that nobody will do: NaN rows, by one warp.
template <int TILES, int D>
__device__ __noinline__ void void_rows(uint32_t *out, float *lse, int q_heads, const Item &it) {
  const int lane = threadIdx.x & 31;
  for (int t = 0; t < TILES; t++)
    for (int row = it.i0[t]; row < min(it.i0[t] + kRows, it.nq); row++) {
      const int64_t at = (int64_t)(it.q0 + row) * q_heads + it.head[t];
      for (int i = lane; i < D / 2; i += 32) out[at * (D / 2) + i] = 0x7fff7fffu;
      if (lane == 0 && lse != nullptr) lse[at] = NAN;
    }
}

template <int D, bool BF16>
__global__ void __launch_bounds__(Shape<D>::kThreads, Shape<D>::kBlocks)
    prompt_kernel(const Args a, const __grid_constant__ CUtensorMap qmap,
                  const __grid_constant__ CUtensorMap kmap,
                  const __grid_constant__ CUtensorMap vmap) {
  using L = Shape<D>;
  constexpr int kTiles = L::kTiles, kSlots = L::kSlots, kSoftmaxWarps = L::kSoftmaxWarps;
  extern __shared__ __align__(1024) uint8_t sm[];
  int(*odd)[D] = (int(*)[D])(sm + L::kOdd);  // the first key whose value is NaN, +inf, -inf
  uint64_t *bars = (uint64_t *)(sm + L::kBars);
  uint64_t *q_full = bars, *kv_full = bars + 2, *kv_empty = kv_full + kSlots;
  uint64_t *s_full = kv_empty + kSlots, *p_ready = s_full + 2, *o_done = p_ready + 4;
  uint64_t *h_done = o_done + 2, *mended = h_done + 2, *drained = mended + kMends;
  uint64_t *q_empty = drained + 1, *item_full = q_empty + 2, *item_empty = item_full + 2;
  uint64_t *out_done = item_empty + 2, *asked = out_done + 1;
  uint32_t *tmem_s = (uint32_t *)(asked + 1);
  volatile int *abort_s = (volatile int *)(tmem_s + 1);

  // Pieces of work in turn, as the loading warp finds them: a block does its own
  // and then those of blocks that have not started.
  __shared__ Item items[2], lost;
  __shared__ int last_item[2], any_odd[2];  // no work left; values that are no numbers were found
  __shared__ __align__(16) uint4 answer;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < 2; i++) {
      tc::mbar_init(&q_full[i], 1);
      tc::mbar_init(&q_empty[i], 1);
      tc::mbar_init(&s_full[i], 1);
      tc::mbar_init(&o_done[i], 1);
      tc::mbar_init(&h_done[i], 1);
      tc::mbar_init(&item_full[i], 1);
      tc::mbar_init(&item_empty[i], kSoftmaxWarps + 3);
    }
    for (int i = 0; i < kSlots; i++) {
      tc::mbar_init(&kv_full[i], 1);
      tc::mbar_init(&kv_empty[i], 1);
    }
    for (int i = 0; i < 4; i++) tc::mbar_init(&p_ready[i], 4);
    for (int i = 0; i < kMends; i++) tc::mbar_init(&mended[i], 64);
    tc::mbar_init(drained, 1);
    tc::mbar_init(out_done, kSoftmaxWarps);
    tc::mbar_init(asked, 1);
    *abort_s = 0;
    tc::mbar_fence_init();
  }
  if (warp == kSoftmaxWarps) {
    tc::tmem_alloc(tmem_s, L::kColumns);
    tc::tmem_relinquish();
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = *tmem_s;
  // the k-th piece of work, once it is there
  auto take = [&](int k) {
    const bool there = __all_sync(0xffffffffu, wait_long(&item_full[k & 1], k >> 1));
    if (!there) *abort_s = 1;
    return there && !*(volatile int *)&last_item[k & 1];
  };
  auto release = [&](int k) {
    __syncwarp();
    if (lane == 0) tc::mbar_arrive(&item_empty[k & 1]);
  };

  if (warp < kSoftmaxWarps) {
    // ================= softmax: thread = row =================
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(L::kMore));
    const int t = warp >> 2;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_at = tmem + lanes + 128 * t, o_at = tmem + lanes + L::kO + 128 * t;
    const float c = __fmul_rn(a.scale, kLog2e);
    constexpr float kLift = Weights<BF16>::kLift, kGrow = Weights<BF16>::kGrow;
    bool ok = true;
    auto settle = [&](bool fine) {  // the warp goes on, or gives up as one
      ok = __all_sync(0xffffffffu, ok && fine);
      return ok;
    };
    // key blocks, pieces with one and mended blocks before this piece
    int past = 0, outs = 0, mends = 0;
#pragma unroll 1
    for (int k = 0; take(k); k++) {
      const Item &it = items[k & 1];
      const int row = it.i0[t] + (warp & 3) * 32 + lane;
      const int blocks = it.blocks[t], lim = limit(a, it, row), flagged = max(0, it.n - it.whole);
      const int first = limit(a, it, it.i0[t]);
      float m = -INFINITY;
      f2 l = 0;
      for (int j = blocks - 1, i = 0; j >= 0 && ok; j--, i++) {
        if (!settle(wait_for(&s_full[t], past + i))) break;
        tc::tc_fence_after();
        uint32_t r[4][32];
#pragma unroll
        for (int q = 0; q < 4; q++) tc::tmem_ld32(s_at + 32 * q, r[q]);
        tc::tmem_ld_wait();
        const bool masked = (j + 1) * kKeys > first;
        const int seen = lim - j * kKeys;  // columns of this block that the row sees
        if (masked) {
          asm volatile("");  // a branch, not 128 selects in every block
#pragma unroll
          for (int e = 0; e < 128; e++)
            if (e >= seen) r[e / 32][e % 32] = 0xff800000u;
        }
#pragma unroll
        for (int h = 0; h < 2; h++) {  // 64 keys
          f2 sum;
          uint32_t p[2][16];
          // a row without a reference needs its maximum first; a row that needs
          // none keeps its own, whoever shares its warp; `fresh` has taken its
          // reference from these keys, so that no weight is above the reference's
          bool need = m == -INFINITY, again = __any_sync(0xffffffffu, need), fresh = false;
          for (;;) {
            if (again) {
              // (opaque here, so that the maximum is not computed ahead of the branch)
#pragma unroll
              for (int e = 0; e < 64; e++) asm volatile("" : "+r"(r[2 * h + e / 32][e % 32]));
              float top[4];
#pragma unroll
              for (int q = 0; q < 4; q++) {
                const uint32_t *x = &r[2 * h + q / 2][16 * (q % 2)];
                top[q] = __uint_as_float(x[0]);
#pragma unroll
                for (int e = 1; e < 16; e++) top[q] = max_nan(top[q], __uint_as_float(x[e]));
              }
              const float nm =
                  max_nan(m, max_nan(max_nan(top[0], top[1]), max_nan(top[2], top[3])));
              // (what has seen nothing has sums of zero: any factor keeps them)
              const float f = need && m != -INFINITY && nm != -INFINITY
                                  ? exp2_fast(__fmul_rn(__fsub_rn(m, nm), c))
                                  : 1.0f;
              m = need ? nm : m;
              l = fma2(l, pair(f, f), 0);
              if (__any_sync(0xffffffffu, f != 1.0f)) {
                // O holds what the products before this half have added: those of
                // the block before are done (S came after them), those of this
                // block's first half say so
                if (h > 0 && !settle(wait_for(&h_done[t], past + i))) break;
                tc::tc_fence_after();
#pragma unroll 1
                for (int q = 0; q < D / 32; q++) {
                  uint32_t o[32];
                  tc::tmem_ld32(o_at + 32 * q, o);
                  tc::tmem_ld_wait();
#pragma unroll
                  for (int e = 0; e < 32; e++)
                    o[e] = __float_as_uint(__fmul_rn(__uint_as_float(o[e]), f));
                  tmem_st32(o_at + 32 * q, o);
                }
              }
            }
            // a row that sees a score of +inf or NaN is NaN
            const float base = m == -INFINITY ? 0.0f : m <= FLT_MAX ? __fmaf_rn(m, -c, kLift) : NAN;
            const f2 cc = pair(c, c), bb = pair(base, base);
            f2 b0 = 0, b1 = 0;
#pragma unroll
            for (int e = 0; e < 64; e += 2) {
              const uint32_t *x = &r[2 * h + e / 32][e % 32];
              const f2 z = fma2(pair(__uint_as_float(x[0]), __uint_as_float(x[1])), cc, bb);
              const float2 v = split(z);
              const float x0 = exp2_fast(v.x), x1 = exp2_fast(v.y);
              if (e % 4) b1 = add2(b1, pair(x0, x1));
              else b0 = add2(b0, pair(x0, x1));
              p[e / 32][e % 32 / 2] = kv::pack2<BF16>(x0, x1);
            }
            sum = add2(b0, b1);
            // weights beyond kGrow (or NaN): take a new reference and start over, once
            // at most for a row (also where the warp is here for another row's first keys)
            const float2 v = split(sum);
            fresh = fresh || need;
            need = !fresh && (!(v.x <= kGrow) || !(v.y <= kGrow));
            again = __any_sync(0xffffffffu, need);
            if (!again) break;
          }
          if (!ok) break;
          l = add2(l, sum);
          tmem_st16(s_at + 64 * h, p[0]);
          tmem_st16(s_at + 64 * h + 16, p[1]);
          tmem_st_wait();
          tc::tc_fence_before();
          __syncwarp();
          if (lane == 0) tc::mbar_arrive(&p_ready[2 * t + h]);
        }
      }
      if (!ok) *abort_s = 1;
      // ---- output ----
      const float2 ll = split(l);
      const float sum = __fadd_rn(ll.x, ll.y);
      past += blocks;
      mends += flagged;
      if (blocks > 0 && ok) settle(wait_for(&o_done[t], outs));
      if (flagged > 0 && ok) settle(wait_for(&mended[(mends - 1) % kMends], (mends - 1) / kMends));
      outs += blocks > 0;
      settle(!*abort_s);
      if (!ok) *abort_s = 1;
      tc::tc_fence_after();
      const bool none = blocks == 0 || lim == 0, live = row < it.nq;
      const bool odds = flagged > 0 && *(volatile int *)&any_odd[k & 1] != 0;
      // (the sums of a row that sees nothing are zeros: its keys' values are mended)
      // NaN: a wait gave up, or every score that the row sees is -inf
      const float inv = !ok ? NAN : none ? 0.0f : m == -INFINITY ? NAN : __fdiv_rn(1.0f, sum);
      uint16_t *to = (uint16_t *)a.out +
                     ((int64_t)(it.q0 + row - (lane & 3)) * a.q_heads + it.head[t]) * D + 8 * (lane & 3);
#pragma unroll 1
      for (int q = 0; q < D / 32; q++) {
        uint32_t o[32];
        if (blocks > 0 && ok) {
          tc::tmem_ld32(o_at + 32 * q, o);
          tc::tmem_ld_wait();
        } else {
#pragma unroll
          for (int e = 0; e < 32; e++) o[e] = 0;
        }
        float v[32];
#pragma unroll
        for (int e = 0; e < 32; e++) v[e] = __fmul_rn(__uint_as_float(o[e]), inv);
        if (odds && !none) {
#pragma unroll
          for (int e = 0; e < 32; e++) {
            const int d = 32 * q + e;
            if (odd[1][d] < lim) v[e] = __fadd_rn(v[e], INFINITY);
            if (odd[2][d] < lim) v[e] = __fadd_rn(v[e], -INFINITY);
            if (odd[0][d] < lim) v[e] = NAN;
          }
        }
        // four lanes trade their rows' 16-byte pieces, so that a store's lanes lie side
        // by side: row by row, 32 lanes' pieces are 32 lines
        uint4 x[4];
#pragma unroll
        for (int e = 0; e < 4; e++)
          x[e] = make_uint4(kv::pack2<BF16>(v[8 * e], v[8 * e + 1]),
                            kv::pack2<BF16>(v[8 * e + 2], v[8 * e + 3]),
                            kv::pack2<BF16>(v[8 * e + 4], v[8 * e + 5]),
                            kv::pack2<BF16>(v[8 * e + 6], v[8 * e + 7]));
        trade(x[0], x[2], 2);
        trade(x[1], x[3], 2);
        trade(x[0], x[1], 1);
        trade(x[2], x[3], 1);
#pragma unroll
        for (int e = 0; e < 4; e++)
          if (row - (lane & 3) + e < it.nq)
            *(uint4 *)(to + (int64_t)e * a.q_heads * D + 32 * q) = x[e];
      }
      if (live && a.lse != nullptr)
        a.lse[(int64_t)(it.q0 + row) * a.q_heads + it.head[t]] =
            none || m == -INFINITY ? -INFINITY
                 : ok ? __fmul_rn(__fmaf_rn(m, c, __log2f(sum) - kLift), kLn2) : NAN;
      tc::tc_fence_before();
      // (in this order: who finds piece k + 2 finds out_done past piece k, so that a
      // wait for piece k + 1 by its parity cannot take piece k's phase for it)
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(out_done);
      release(k);
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(L::kLess));
  }
  if (warp == kSoftmaxWarps) {
    // ================= products =================
    // The whole warp runs this on values that are the same in every lane, so
    // that addresses and descriptors stay in uniform registers; one lane issues.
    // (Run by one lane alone, the operands' way into uniform registers took
    // 70 to 160 cycles a product, and the tensor core idled for it.)
    constexpr uint32_t ds = idesc(128, 128, BF16, false), dp = idesc(128, D, BF16, true);
    const uint32_t leader = elect_one();
    const uint32_t tm = uniform(tmem), q_base = uniform(tc::smem_u32(sm + L::kQ));
    const uint64_t q_desc = tc::sw128_desc(q_base), k_desc = tc::sw128_desc(q_base + L::kRing);
    const uint64_t v_desc = sw128_desc_n(q_base + L::kRing, 128 * 128);
    bool ok = true;
    auto wait = [&](uint64_t *bar, int phase) {
      if (ok) ok = __all_sync(0xffffffffu, wait_for(bar, phase));
      return ok;
    };
    // block j's values (none for j = n), then block j - 1's scores
    int v_slot = 1, v_phase = 0, k_slot = 0, k_phase = 0;
    int past[2] = {0, 0}, queries[2] = {0, 0}, mends = 0;
#pragma unroll 1
    for (int k = 0; take(k); k++) {
      const int nu = uniform(items[k & 1].n), whole = uniform(items[k & 1].whole);
      const int nb[2] = {(int)uniform(items[k & 1].blocks[0]),
                         kTiles == 2 ? (int)uniform(items[k & 1].blocks[1]) : 0};
      release(k);
      for (int j = nu; j >= 0 && ok; j--) {
        if (j < nu) {
          if (!wait(&kv_full[v_slot], v_phase)) break;
          const int f = mends + nu - 1 - j;
          if (j >= whole && !wait(&mended[f % kMends], f / kMends)) break;
        }
        bool have_k = false;
#pragma unroll
        for (int t = 0; t < kTiles; t++) {
          if (j < nb[t]) {
            const uint64_t vd = v_desc + (uint64_t)(v_slot * (L::kTile >> 4));
#pragma unroll
            for (int h = 0; h < 2; h++) {
              if (!wait(&p_ready[2 * t + h], past[t] + nb[t] - 1 - j)) break;
              tc::tc_fence_after();
#pragma unroll
              for (int k = 4 * h; k < 4 * h + 4; k++)
                mma_ts(tm + L::kO + 128 * t, tm + 128 * t + 64 * h + 8 * (k & 3),
                       vd + (k * 16 * 128 >> 4), dp, k > 0 || j < nb[t] - 1, leader);
              if (h == 0) mma_commit(&h_done[t], leader);
            }
            if (!ok) break;
            if (j == 0) mma_commit(&o_done[t], leader);
          }
          if (j > 0 && j <= nb[t]) {
            if (!have_k && !wait(&kv_full[k_slot], k_phase)) break;
            have_k = true;
            if (j == nb[t] && !wait(&q_full[t], queries[t])) break;
            tc::tc_fence_after();
            const uint64_t kd = k_desc + (uint64_t)(k_slot * (L::kTile >> 4));
#pragma unroll
            for (int k = 0; k < D / 16; k++) {
              const uint32_t off = ((k >> 2) * (128 * 128) + (k & 3) * 32) >> 4;
              mma_ss(tm + 128 * t, q_desc + t * (L::kTile >> 4) + off, kd + off, ds, k > 0, leader);
            }
            mma_commit(&s_full[t], leader);
            if (j == 1) mma_commit(&q_empty[t], leader);
          }
        }
        if (!ok) break;
        if (j < nu) {
          mma_commit(&kv_empty[v_slot], leader);
          v_slot += 2;
          if (v_slot >= kSlots) v_slot -= kSlots, v_phase ^= 1;
        }
        if (j > 0) {
          mma_commit(&kv_empty[k_slot], leader);
          k_slot += 2;
          if (k_slot >= kSlots) k_slot -= kSlots, k_phase ^= 1;
        }
      }
      mends += max(0, nu - whole);
#pragma unroll
      for (int t = 0; t < kTiles; t++) {
        past[t] += nb[t];
        queries[t] += nb[t] > 0;
      }
      if (!ok) *abort_s = 1;
    }
    // every product done before the TMEM goes
    mma_commit(drained, leader);
    wait_for(drained, 0);
    __syncwarp();
  } else if (warp == kSoftmaxWarps + 1) {
    // ================= loads =================
    int block = blockIdx.x, k = 0;
    int answers = 0, queries[2] = {0, 0};
    int64_t issued = 0;
    bool waiting = true, stuck = false;
    if (lane == 0) ask_next(&answer, asked);
    for (;;) {
      if (k >= 2 && !__all_sync(0xffffffffu, wait_long(&item_empty[k & 1], (k >> 1) - 1))) {
        *abort_s = 1;
        stuck = true;
        break;
      }
      Item &it = items[k & 1];
      const bool some = block >= 0 && find_item<kTiles>(a, block, &it);
      __syncwarp();
      if (some || block < 0) {
        if (lane == 0) {
          last_item[k & 1] = block < 0;
          tc::mbar_arrive(&item_full[k & 1]);
        }
        k++;
      }
      if (block < 0) break;
      if (some && lane == 0 && !*abort_s) {
        const int n = it.n, kv_head = it.head[0] / (a.q_heads / a.heads);
        for (int i = 0; i < 2 * n; i++, issued++) {
          const int s = issued % kSlots, j = n - 1 - i / 2;
          if (!wait_for(&kv_empty[s], (issued / kSlots & 1) ^ 1) || *abort_s) {
            *abort_s = 1;
            break;
          }
          tc::mbar_arrive_expect_tx(&kv_full[s], L::kTile);
          for (int x = 0; x < D; x += 64)
            tma_load_3d(sm + L::kRing + s * L::kTile + x * 256, i & 1 ? &vmap : &kmap, x, kv_head,
                        it.k0 + j * kKeys, &kv_full[s]);
          if (i > 0) continue;
          // the first keys are there by the time that the last scores let go of the queries
          for (int t = 0; t < kTiles; t++) {
            if (it.blocks[t] == 0) continue;
            if (queries[t] > 0 && !wait_for(&q_empty[t], queries[t] - 1)) {
              *abort_s = 1;
              continue;
            }
            queries[t]++;
            tc::mbar_arrive_expect_tx(&q_full[t], L::kTile);
            for (int x = 0; x < D; x += 64)
              tma_load_3d(sm + L::kQ + t * L::kTile + x * 256, &qmap, x, it.head[t],
                          it.q0 + it.i0[t], &q_full[t]);
          }
        }
      }
      __syncwarp();
      block = -1;
      if (waiting && __all_sync(0xffffffffu, wait_for(asked, answers++))) block = answer_of(&answer);
      // (what was asked for is this block's to do, if only to say that it gave up)
      waiting = __all_sync(0xffffffffu, block >= 0 && !*abort_s);
      if (waiting && lane == 0) {
        tc::fence_async_smem();
        ask_next(&answer, asked);
      }
    }
    if (stuck) {
      // The piece in hand and the one asked for, whose answer is still to land, are
      // no other block's.
      const int next = waiting && __all_sync(0xffffffffu, wait_for(asked, answers)) ? answer_of(&answer) : -1;
      for (int i = 0; i < 2; i++) {
        const bool some = (i ? next : block) >= 0 && find_item<kTiles>(a, i ? next : block, &lost);
        __syncwarp();
        if (some) void_rows<kTiles, D>((uint32_t *)a.out, a.lse, a.q_heads, lost);
        __syncwarp();
      }
    }
    if (lane == 0 && *abort_s) {  // no copy may land after the block is gone
      for (int64_t i = issued > kSlots ? issued - kSlots : 0; i < issued; i++)
        wait_for(&kv_full[i % kSlots], (int)(i / kSlots));
      for (int t = 0; t < kTiles; t++)
        if (queries[t] > 0) wait_for(&q_full[t], queries[t] - 1);
    }
    __syncwarp();
  } else if (warp > kSoftmaxWarps + 1) {
    // ================= mending values =================
    const int id = tid - 32 * (kSoftmaxWarps + 2);
    int64_t tiles = 0;  // of keys and values before this piece
    int mends = 0;
#pragma unroll 1
    for (int k = 0; !any_of_64(!take(k)); k++) {  // (both warps, or none)
      const int n = items[k & 1].n, nk = items[k & 1].nk;
      const int flagged = max(0, n - items[k & 1].whole);
      bool marked = false;
      if (id == 0) any_odd[k & 1] = 0;
      for (int f = 0; f < flagged; f++, mends++) {
        const int64_t seq = tiles + 2 * f + 1;
        const int key0 = (n - 1 - f) * kKeys;
        bool ok = wait_for(&kv_full[seq % kSlots], seq / kSlots) && !*abort_s;
        if (any_of_64(!ok)) {
          *abort_s = 1;
          mends += flagged - f;
          break;
        }
        uint8_t *v = sm + L::kRing + (seq % kSlots) * L::kTile;
        // 16-byte pieces as they lie, 8 of them 64 columns of a row; first zeros for the
        // next sequence's rows (from each thread in the pieces that it looks at)
        const int from = 8 * min(nk - key0, 128);
        for (int x = 0; x < D; x += 64)
          for (int i = from + ((id - from) & 63); i < 128 * 8; i += 64)
            *(uint4 *)(v + x * 256 + i * 16) = make_uint4(0, 0, 0, 0);
        uint32_t top = 0;  // the largest magnitudes, as integers
#pragma unroll 4
        for (int i = 0; i < 128 * D * 2; i += 64 * 16) {
          const uint4 x = *(const uint4 *)(v + id * 16 + i);
          top = __vmaxu2(top, __vmaxu2(__vmaxu2(x.x & 0x7fff7fffu, x.y & 0x7fff7fffu),
                                       __vmaxu2(x.z & 0x7fff7fffu, x.w & 0x7fff7fffu)));
        }
        constexpr uint32_t kExp = BF16 ? 0x7f80u : 0x7c00u;  // infinity; NaNs are above
        const bool bad = (top & 0xffffu) >= kExp || top >> 16 >= kExp;
        if (any_of_64(bad)) {
          if (!marked) {  // the marks of the piece before have been read
            marked = true;
            if (any_of_64(k > 0 && !wait_long(out_done, k - 1))) *abort_s = 1;
            for (int i = id; i < 3 * D; i += 64) odd[i / D][i % D] = INT_MAX;
            if (id == 0) any_odd[k & 1] = 1;
            any_of_64(false);
          }
          for (int i = id; i < 128 * D; i += 64) {
            const int r = i / D, d = i % D;
            if (key0 + r >= nk) break;
            uint16_t *at = (uint16_t *)(v + tc::sw128_chunk_offset(r, d / 8, 128)) + d % 8;
            const uint32_t half = *at;
            if ((half & kExp) != kExp) continue;
            atomicMin(&odd[(half & 0x7fffu) != kExp ? 0 : half >> 15 ? 2 : 1][d],
                      key0 + r);
            *at = 0;
          }
        }
        tc::fence_async_smem();
        tc::mbar_arrive(&mended[mends % kMends]);
      }
      tiles += 2 * n;
      release(k);
    }
  }
  __syncthreads();
  if (warp == kSoftmaxWarps) {
    tc::tc_fence_after();
    tc::tmem_dealloc(tmem, L::kColumns);
  }
}

// ---- launch ----
using EncodeTiled = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *,
                                 const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                                 const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeTiled encoder() {
  static const EncodeTiled fn = [] {
    void *p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      p = nullptr;
    return (EncodeTiled)p;
  }();
  return fn;
}

// 128 rows of 64 columns of one head at a time
static bool tile_map(CUtensorMap *m, const kv::Strided &x, int rows, int heads, int D, bool bf16) {
  const cuuint64_t dim[3] = {(cuuint64_t)D, (cuuint64_t)heads, (cuuint64_t)rows};
  const cuuint64_t stride[2] = {(cuuint64_t)x.head * 2, (cuuint64_t)x.row * 2};
  const cuuint32_t box[3] = {64, 1, 128}, one[3] = {1, 1, 1};
  return encoder()(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                   const_cast<void *>(x.p), dim, stride, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                   CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D, bool BF16>
static cudaError_t launch_d(const Args &a, cudaStream_t st) {
  if (encoder() == nullptr) return cudaErrorNotSupported;
  CUtensorMap q, k, v;
  if (!tile_map(&q, a.q, a.rows_q, a.q_heads, D, BF16)) return cudaErrorInvalidValue;
  if (a.rows_k == 0) {
    k = v = q;  // never read
  } else if (!tile_map(&k, a.k, a.rows_k, a.heads, D, BF16) ||
             !tile_map(&v, a.v, a.rows_k, a.heads, D, BF16)) {
    return cudaErrorInvalidValue;
  }
  using L = Shape<D>;
  const int64_t grid = pairs_heads<L::kTiles>(a)
                           ? ((int64_t)a.rows_q / kRows + a.n) * (a.q_heads / 2)
                           : ((int64_t)a.rows_q / (L::kTiles * kRows) + a.n) * a.q_heads;
  if (grid > INT_MAX) return cudaErrorInvalidValue;
  const cudaError_t e = cudaFuncSetAttribute(
      prompt_kernel<D, BF16>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kBytes);
  if (e != cudaSuccess) return e;
  prompt_kernel<D, BF16><<<(unsigned)grid, L::kThreads, L::kBytes, st>>>(a, q, k, v);
  return cudaGetLastError();
}

cudaError_t launch(const Args &a, cudaStream_t st) {
  if (a.D == 64) return a.bf16 ? launch_d<64, true>(a, st) : launch_d<64, false>(a, st);
  return a.bf16 ? launch_d<128, true>(a, st) : launch_d<128, false>(a, st);
}

}  // namespace prompt
}  // namespace uvb
