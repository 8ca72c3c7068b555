// kv_pages.cu -- the page operations of the cache held in 4 bits: extending,
// forking, copying, truncating and compacting.  Everything they decide is
// decided on the device, so a serving step has no host wait and can be
// captured in a graph.
//
// A page is free when its reference count is zero and the lowest free pages
// are taken first, so the tables depend on the calls alone.  A call is all or
// nothing: its control kernel checks every entry and the free pages before it
// changes anything, and records what is wrong in the status word, which also
// stops later calls until the host has read it.
//
// What bounds them: the data kernel moves whole pages and is bound by HBM
// (twice the pages' bytes); the control kernels are bound by latency, a few
// dependent L2 accesses for each of their phases.  They run in one block
// (extend, copy, compact: an ordered prefix over the entries or the pages) or
// in one cluster of eight (fork, truncate: no order, many table entries).
#include <cooperative_groups.h>

#include "uv_kv.h"

namespace uvb {
namespace kv {

constexpr int kThreads = 1024;
constexpr int kCluster = 8;

__device__ __forceinline__ int pages_for(int64_t tokens, int page) {
  return (int)((tokens + page - 1) / page);
}

// Exclusive prefix of v over the block, in thread order; total in *sum.
template <class T>
__device__ __forceinline__ T block_prefix(T v, T *warp_sums, T *sum) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  T x = v;
  for (int o = 1; o < 32; o <<= 1) {
    const T y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  if (warp == 0) {
    T w = warp_sums[lane];
    for (int o = 1; o < 32; o <<= 1) {
      const T y = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += y;
    }
    warp_sums[lane] = w;
  }
  __syncthreads();
  *sum = warp_sums[31];
  return (warp ? warp_sums[warp - 1] : T(0)) + x - v;
}

// ---- extend and copy: pages for sequences, and what to copy into them ----
// Entry i grows sequence seqs[i] by counts[i] tokens (extend), or gives the
// empty sequence seqs[i] pages of its own for all of src[i]'s tokens (copy).
// In extend a last page that others hold too, and that the new tokens would
// write, is replaced by a copy.  Sharers that extend in the same call each
// copy: whether a page is shared is decided before the call's first change.
template <bool COPY>
__global__ void __launch_bounds__(kThreads) alloc_kernel(Cache c, const int32_t *seqs,
                                                         const int32_t *more, int n) {
  __shared__ int64_t sums[32];
  __shared__ int errors, next_hint;
  pdl_launch();
  if (threadIdx.x == 0) errors = 0, next_hint = c.n_pages;
  const int status = c.work[kStatus];
  __syncthreads();
  if (status != 0) {
    if (threadIdx.x == 0) c.work[kMoves] = 0;
    return;
  }
  const int page = c.page_tokens;
  const int per = (n + kThreads - 1) / kThreads;
  const int lo = min((int)threadIdx.x * per, n), hi = min(lo + per, n);
  // what every entry needs: pages in the low half, copies in the high half
  auto wants = [&](int i, int *bad) -> int64_t {
    const int s = seqs[i], m = more[i];
    if (s < 0 || s >= c.max_seqs || m < 0 || (COPY && m >= c.max_seqs)) {
      *bad |= kBadSeq;
      return 0;
    }
    const int len = c.length(s);
    if (COPY) {
      if (len != 0) *bad |= kNotEmpty;
      const int64_t pages = pages_for(c.length(m), page);
      return pages << 32 | pages;
    }
    if ((int64_t)len + m > (int64_t)c.max_pages * page) {
      *bad |= kTooLong;
      return 0;
    }
    const int have = pages_for(len, page);
    const int cow = m > 0 && len % page != 0 && c.refs[c.page_at(s, have - 1)] > 1;
    return pages_for((int64_t)len + m, page) - have + cow + ((int64_t)cow << 32);
  };
  int64_t need = 0;
  int bad = 0;
  for (int i = lo; i < hi; i++) {
    const int s = seqs[i];
    if (s >= 0 && s < c.max_seqs && atomicExch(&c.mark()[s], 1) != 0) bad |= kBadSeq;
    need += wants(i, &bad);
  }
  if (bad) atomicOr(&errors, bad);
  int64_t total2;
  int64_t off2 = block_prefix(need, sums, &total2);
  if (COPY) {  // a source must not be a target: it would change under the copy
    for (int i = lo; i < hi; i++) {
      const int from = more[i];
      if (from >= 0 && from < c.max_seqs && c.mark()[from] != 0) atomicOr(&errors, kBadSeq);
    }
    __syncthreads();
  }
  for (int i = lo; i < hi; i++)
    if (seqs[i] >= 0 && seqs[i] < c.max_seqs) c.mark()[seqs[i]] = 0;
  const int used = c.work[kUsed];
  const int64_t total = total2 & 0xffffffffll;
  if (threadIdx.x == 0) {
    if (total > c.n_pages - used) errors |= kNoPages;
    if (errors) c.work[kStatus] = errors;
    c.work[kMoves] = errors ? 0 : (int)(total2 >> 32);
  }
  __syncthreads();
  if (errors) return;

  // The `total` lowest free pages, in order, into the remap words.
  int32_t *fresh = c.remap();
  int64_t got = 0;
  for (int64_t at = c.work[kHint]; got < total && at < c.n_pages; at += 4 * kThreads) {
    const int64_t p = at + 4 * threadIdx.x;
    int free_mask = 0;
#pragma unroll
    for (int k = 0; k < 4; k++)
      if (p + k < c.n_pages && c.refs[p + k] == 0) free_mask |= 1 << k;
    int64_t found;
    int64_t rank = got + block_prefix<int64_t>(__popc(free_mask), sums, &found);
#pragma unroll
    for (int k = 0; k < 4; k++)
      if (free_mask >> k & 1) {
        if (rank < total) {
          fresh[rank] = (int)(p + k);
          if (rank == total - 1) next_hint = (int)(p + k) + 1;
        }
        rank++;
      }
    got += found;
    __syncthreads();
  }
  if (got < total) {  // the counts changed under the bookkeeping words
    if (threadIdx.x == 0) c.work[kStatus] = kNoPages, c.work[kMoves] = 0;
    return;
  }
  // Each entry's place among the fresh pages and the moves (the counts are
  // still those of the check, so it is the same sum again).  A thread serves its
  // entries itself where they take a page or so each; long ones go out by warps,
  // so that one prompt does not keep one thread busy.
  const bool short_ones = per == 1 && total <= 4 * (int64_t)n;
  int released = 0;
  auto serve = [&](int i, int64_t at, int64_t want, int first, int step) {
    const int s = seqs[i], len = c.length(s), have = pages_for(len, page);
    const int off = (int)(at & 0xffffffffll), take = (int)(want & 0xffffffffll);
    const int cow = COPY ? 0 : (int)(want >> 32);
    int32_t *row = c.table + (int64_t)s * c.max_pages;
    const int column = COPY ? 0 : have - cow;
    if (cow && first == 0) {
      const int old = c.page_at(s, column), move = (int)(at >> 32);
      c.move_src()[move] = old;
      c.move_dst()[move] = fresh[off];
      if (atomicSub(&c.refs[old], 1) == 1) {
        released++;
        atomicMin(&next_hint, old);
      }
    }
    for (int j = first; j < take; j += step) {
      const int p = fresh[off + j];
      if (COPY) {
        c.move_src()[off + j] = c.page_at(more[i], j);
        c.move_dst()[off + j] = p;
      }
      row[column + j] = p;
      c.refs[p] = 1;
    }
    return COPY ? c.length(more[i]) : len + more[i];
  };
  if (short_ones) {
    if (lo < hi) c.lens[seqs[lo]] = serve(lo, off2, need, 0, 1);
  } else {
    int ignore = 0;
    for (int i = lo; i < hi; i++) {
      const int64_t want = per == 1 ? need : wants(i, &ignore);
      c.offset()[i] = (int)(off2 & 0xffffffffll);
      c.mark()[i] = (int)(off2 >> 32) << 1 | (COPY ? 0 : (int)(want >> 32));
      off2 += want;
    }
    __syncthreads();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int i = warp; i < n; i += kThreads / 32) {
      const int s = seqs[i], len = c.length(s), have = pages_for(len, page), m = c.mark()[i];
      const int cow = m & 1;
      const int take = COPY ? pages_for(c.length(more[i]), page)
                            : pages_for((int64_t)len + more[i], page) - have + cow;
      const int now = serve(i, (int64_t)(m >> 1) << 32 | (uint32_t)c.offset()[i],
                            (int64_t)cow << 32 | take, lane, 32);
      __syncwarp();
      if (lane == 0) c.lens[s] = now;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kThreads) c.mark()[i] = 0;
  }
  if (released) atomicSub(&c.work[kUsed], released);
  __syncthreads();
  if (threadIdx.x == 0) {
    c.work[kUsed] += (int)total;
    if (total > 0) {
      const int hint = next_hint;
      c.work[kHint] = hint;
    }
  }
}

// ---- moving pages ----
// Copies the listed pages in every layer.  A unit is 16 KiB of one page, four
// 16-byte loads in flight for each of 256 threads: enough outstanding bytes
// over 8 blocks an SM to cover HBM's latency.  After a compaction the tables
// and counts follow (fix = 1): they share no byte with the pages' data.
constexpr int kMoveThreads = 256, kMoveUnit = kMoveThreads * 4;

__global__ void __launch_bounds__(kMoveThreads) move_kernel(Cache c, int fix) {
  pdl_wait();
  const int moves = c.work[kMoves];
  if (moves == 0) return;
  const int64_t vecs = c.page_bytes() / 16;
  const int units = (int)((vecs + kMoveUnit - 1) / kMoveUnit);
  const int64_t total = (int64_t)moves * c.layers * units;
  for (int64_t u = blockIdx.x; u < total; u += gridDim.x) {
    const int chunk = (int)(u % units);
    const int64_t item = u / units;
    const int layer = (int)(item % c.layers), m = (int)(item / c.layers);
    const int64_t base = (int64_t)layer * c.n_pages;
    const uint4 *from = (const uint4 *)(c.pool + (base + c.move_src()[m]) * c.page_bytes());
    uint4 *to = (uint4 *)(c.pool + (base + c.move_dst()[m]) * c.page_bytes());
    uint4 v[4];
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const int64_t i = (int64_t)chunk * kMoveUnit + k * kMoveThreads + threadIdx.x;
      if (i < vecs) v[k] = __ldcs(from + i);
    }
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const int64_t i = (int64_t)chunk * kMoveUnit + k * kMoveThreads + threadIdx.x;
      if (i < vecs) __stcs(to + i, v[k]);
    }
  }
  if (!fix) return;
  const int64_t all = (int64_t)gridDim.x * kMoveThreads, id = (int64_t)blockIdx.x * kMoveThreads + threadIdx.x;
  for (int64_t m = id; m < moves; m += all) {
    const int from = c.move_src()[m], to = c.move_dst()[m];
    c.refs[to] = c.refs[from];
    c.refs[from] = 0;
  }
  const int dense = c.work[kUsed];
  const int64_t entries = (int64_t)c.max_seqs * c.max_pages;
  for (int64_t i = id; i < entries; i += all) {
    const int p = c.table[i];
    if (p >= dense && p < c.n_pages) c.table[i] = c.remap()[p];
  }
}

// ---- fork and truncate ----
// One cluster: block 0 checks the entries, the others read its verdict
// through shared memory, then all warps share the entries' table columns in
// groups of 32.  One block does where each of its warps has one group at most
// (128 groups take 9.4 us in one block, 7.2 in a cluster of eight).
__global__ void __launch_bounds__(kThreads) fork_kernel(Cache c, const int32_t *src, const int32_t *dst, const int32_t *lens, int n) {
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  __shared__ int errors;
  if (threadIdx.x == 0) errors = 0;
  __syncthreads();
  if (cluster.block_rank() == 0) {
    int bad = c.work[kStatus] != 0 ? 1 << 30 : 0;
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const int s = src[i], d = dst[i];
      if (s < 0 || s >= c.max_seqs || d < 0 || d >= c.max_seqs) {
        bad |= kBadSeq;
        continue;
      }
      if (atomicExch(&c.mark()[d], 1) != 0) bad |= kBadSeq;
      if (c.length(d) != 0) bad |= kNotEmpty;
      if (lens != nullptr && lens[i] < 0) bad |= kBadSeq;
    }
    if (bad) atomicOr(&errors, bad);
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kThreads)
      if (src[i] >= 0 && src[i] < c.max_seqs && c.mark()[src[i]] != 0) atomicOr(&errors, kBadSeq);
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kThreads)
      if (dst[i] >= 0 && dst[i] < c.max_seqs) c.mark()[dst[i]] = 0;
    if (threadIdx.x == 0 && errors && !(errors >> 30)) c.work[kStatus] = errors;
  }
  cluster.sync();
  const int verdict = *cluster.map_shared_rank(&errors, 0);
  cluster.sync();
  if (verdict) return;
  const int lane = threadIdx.x & 31;
  const int warp = cluster.block_rank() * (kThreads / 32) + (threadIdx.x >> 5);
  const int groups = (c.max_pages + 31) / 32;
  for (int64_t u = warp; u < (int64_t)n * groups; u += (int64_t)cluster.num_blocks() * (kThreads / 32)) {
    const int i = (int)(u % n), col = (int)(u / n) * 32 + lane;
    const int s = src[i], d = dst[i];
    int len = c.length(s);
    if (lens != nullptr) len = min(len, lens[i]);
    if (col < pages_for(len, c.page_tokens)) {
      const int p = c.page_at(s, col);
      c.table[(int64_t)d * c.max_pages + col] = p;
      atomicAdd(&c.refs[p], 1);
    }
    if (col == 0) c.lens[d] = len;
  }
}

__global__ void __launch_bounds__(kThreads) truncate_kernel(Cache c, const int32_t *seqs, const int32_t *lens, int n) {
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  __shared__ int errors, released, low;
  if (threadIdx.x == 0) errors = 0, released = 0, low = c.n_pages;
  __syncthreads();
  if (cluster.block_rank() == 0) {
    int bad = c.work[kStatus] != 0 ? 1 << 30 : 0;
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const int s = seqs[i];
      if (s < 0 || s >= c.max_seqs) {
        bad |= kBadSeq;
        continue;
      }
      if (atomicExch(&c.mark()[s], 1) != 0) bad |= kBadSeq;
      if (lens != nullptr && lens[i] < 0) bad |= kBadSeq;
    }
    if (bad) atomicOr(&errors, bad);
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kThreads)
      if (seqs[i] >= 0 && seqs[i] < c.max_seqs) c.mark()[seqs[i]] = 0;
    if (threadIdx.x == 0 && errors && !(errors >> 30)) c.work[kStatus] = errors;
  }
  cluster.sync();
  const int verdict = *cluster.map_shared_rank(&errors, 0);
  cluster.sync();
  if (verdict) return;
  const int lane = threadIdx.x & 31;
  const int warp = cluster.block_rank() * (kThreads / 32) + (threadIdx.x >> 5);
  const int groups = (c.max_pages + 31) / 32;
  int freed = 0, least = c.n_pages;
  for (int64_t u = warp; u < (int64_t)n * groups; u += (int64_t)cluster.num_blocks() * (kThreads / 32)) {
    const int s = seqs[u % n], i = (int)(u % n), col = (int)(u / n) * 32 + lane;
    const int len = c.length(s), keep = lens != nullptr ? min(lens[i], len) : 0;
    if (col >= pages_for(keep, c.page_tokens) && col < pages_for(len, c.page_tokens)) {
      const int p = c.page_at(s, col);
      c.table[(int64_t)s * c.max_pages + col] = -1;
      if (atomicSub(&c.refs[p], 1) == 1) {
        freed++;
        least = min(least, p);
      }
    }
  }
  if (freed) {
    atomicAdd(&released, freed);
    atomicMin(&low, least);
  }
  // The lengths change after every warp of the cluster has read them.
  cluster.sync();
  for (int64_t i = (int64_t)cluster.block_rank() * kThreads + threadIdx.x; i < n;
       i += (int64_t)cluster.num_blocks() * kThreads) {
    const int s = seqs[i], len = c.length(s);
    c.lens[s] = lens != nullptr ? min(lens[i], len) : 0;
  }
  if (threadIdx.x == 0 && released) {
    atomicSub(&c.work[kUsed], released);
    atomicMin(&c.work[kHint], low);
  }
}

// ---- compact ----
// The k-th used page above the number of used pages goes to the k-th free one
// below it.  Sources and targets do not meet, so the moves need no order.
__global__ void __launch_bounds__(kThreads) compact_kernel(Cache c) {
  __shared__ int64_t sums[32];
  pdl_launch();
  const int status = c.work[kStatus], used = c.work[kUsed];
  if (status != 0) {
    if (threadIdx.x == 0) c.work[kMoves] = 0;
    return;
  }
  // a contiguous run of pages for each thread, in whole groups of four
  const int per = ((c.n_pages + kThreads - 1) / kThreads + 3) & ~3;
  const int64_t lo = min((int64_t)threadIdx.x * per, (int64_t)c.n_pages);
  const int64_t hi = min(lo + per, (int64_t)c.n_pages);
  int64_t count = 0;  // holes in the low half, strays in the high half
  for (int64_t p = lo; p < hi; p++) {
    const int r = c.refs[p];
    if (p < used) count += r == 0;
    else count += (int64_t)(r > 0) << 32;
  }
  int64_t total;
  int64_t at = block_prefix(count, sums, &total);
  for (int64_t p = lo; p < hi; p++) {
    const int r = c.refs[p];
    if (p < used && r == 0) {
      c.move_dst()[at & 0xffffffffll] = (int)p;
      at += 1;
    } else if (p >= used && r > 0) {
      c.move_src()[at >> 32] = (int)p;
      at += 1ll << 32;
    }
  }
  __syncthreads();
  const int moves = (int)min((int64_t)(total & 0xffffffff), (int64_t)(total >> 32));
  for (int k = threadIdx.x; k < moves; k += kThreads) c.remap()[c.move_src()[k]] = c.move_dst()[k];
  if (threadIdx.x == 0) {
    c.work[kMoves] = moves;
    c.work[kHint] = used;
  }
}

// ---- the bookkeeping words from the counts ----
__global__ void __launch_bounds__(kThreads) recount_kernel(Cache c) {
  __shared__ int64_t sums[32];
  int64_t used = 0, total;
  for (int p = threadIdx.x; p < c.n_pages; p += kThreads) used += c.refs[p] > 0;
  block_prefix(used, sums, &total);
  for (int s = threadIdx.x; s < c.max_seqs; s += kThreads) c.mark()[s] = 0;
  if (threadIdx.x < kWorkHead) c.work[threadIdx.x] = threadIdx.x == kUsed ? (int)total : 0;
}

// ---- launches ----
static cudaError_t move_launch(const Cache &c, int fix, int sms, cudaStream_t st) {
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(sms * 8);
  cfg.blockDim = dim3(kMoveThreads);
  cfg.stream = st;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, move_kernel, c, fix);
}

cudaError_t extend_launch(const Cache &c, const int32_t *seqs, const int32_t *counts, int n,
                          int sms, cudaStream_t st) {
  alloc_kernel<false><<<1, kThreads, 0, st>>>(c, seqs, counts, n);
  const cudaError_t e = cudaGetLastError();
  return e != cudaSuccess ? e : move_launch(c, 0, sms, st);
}
cudaError_t copy_launch(const Cache &c, const int32_t *src, const int32_t *dst, int n, int sms,
                        cudaStream_t st) {
  alloc_kernel<true><<<1, kThreads, 0, st>>>(c, dst, src, n);
  const cudaError_t e = cudaGetLastError();
  return e != cudaSuccess ? e : move_launch(c, 0, sms, st);
}
template <class... P, class... A>
static cudaError_t cluster_launch(void (*kernel)(P...), const Cache &c, int n, cudaStream_t st,
                                  A... args) {
  const int blocks = (int64_t)n * ((c.max_pages + 31) / 32) <= kThreads / 32 ? 1 : kCluster;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = blocks;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = st;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, c, args..., n);
}
cudaError_t fork_launch(const Cache &c, const int32_t *src, const int32_t *dst,
                        const int32_t *lens, int n, cudaStream_t st) {
  return cluster_launch(fork_kernel, c, n, st, src, dst, lens);
}
cudaError_t truncate_launch(const Cache &c, const int32_t *seqs, const int32_t *lens, int n,
                            cudaStream_t st) {
  return cluster_launch(truncate_kernel, c, n, st, seqs, lens);
}
cudaError_t compact_launch(const Cache &c, int sms, cudaStream_t st) {
  compact_kernel<<<1, kThreads, 0, st>>>(c);
  const cudaError_t e = cudaGetLastError();
  return e != cudaSuccess ? e : move_launch(c, 1, sms, st);
}
cudaError_t recount_launch(const Cache &c, cudaStream_t st) {
  recount_kernel<<<1, kThreads, 0, st>>>(c);
  return cudaGetLastError();
}

}  // namespace kv
}  // namespace uvb
