// prompt.cu -- attention over whole prompts: packed sequences of different
// lengths, grouped heads, causal or not.  Sequence b owns query rows
// [starts_q[b], starts_q[b + 1]) and key rows [starts_k[b], starts_k[b + 1]);
// its queries are the last of its keys, so with a mask row i sees keys
// j <= i + (keys - queries).  out = softmax(scale q k^T) v, a row that sees
// nothing is zero.
//
// A warp holds 16 query rows; scores, maxima and sums stay in registers (f32)
// over one pass of 64-key tiles in shared memory.
//
// What a row does not see must not reach it, but a weight of zero times a value
// of infinity or NaN is a NaN.  So in tiles with a masked key such values are
// taken out, and for every column the first key that held one is kept: rows
// that see that key get it added to their output.
#include <climits>

#include "uv_prompt.h"

namespace uvb {
namespace prompt {

using kv::mma16816;
using kv::pack2;

constexpr int kRows = 64, kKeys = 64, kThreads = 128;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], const void *p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(tc::smem_u32(p)));
}
__device__ __forceinline__ int bounded(int x, int hi) { return x < 0 ? 0 : (x < hi ? x : hi); }

template <int D, bool BF16>
__global__ void __launch_bounds__(kThreads) simple_kernel(Args a) {
  constexpr int kPitch = D + 8;  // halves: rows 16 bytes apart modulo 128
  __shared__ __align__(16) uint16_t ks[kKeys][kPitch], vs[kKeys][kPitch];
  __shared__ int odd[3][D];  // the first key whose value is NaN, +inf, -inf
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  // entry b has starts_q[b + 1] / 64 - starts_q[b] / 64 + 1 tiles
  const int64_t u = blockIdx.x;
  int lo = 0, hi = a.n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (bounded(a.starts_q[mid], a.rows_q) / kRows + mid <= u) lo = mid;
    else hi = mid - 1;
  }
  const int b = lo, q0 = bounded(a.starts_q[b], a.rows_q);
  const int nq = bounded(a.starts_q[b + 1], a.rows_q) - q0;
  const int i0 = (int)(u - (q0 / kRows + b)) * kRows;
  if (i0 >= nq) return;
  const int k0 = bounded(a.starts_k[b], a.rows_k);
  const int nk = max(0, bounded(a.starts_k[b + 1], a.rows_k) - k0);
  const int head = blockIdx.y, kh = head / (a.q_heads / a.heads);
  const uint16_t *kp = (const uint16_t *)a.k.p + (int64_t)kh * a.k.head;
  const uint16_t *vp = (const uint16_t *)a.v.p + (int64_t)kh * a.v.head;

  uint32_t qf[D / 16][4];
  const int row[2] = {i0 + 16 * warp + g, i0 + 16 * warp + g + 8};
#pragma unroll
  for (int s = 0; s < D / 16; s++)
#pragma unroll
    for (int r = 0; r < 4; r++) {
      const int i = row[r & 1];
      qf[s][r] = i < nq ? *(const uint32_t *)((const uint16_t *)a.q.p + (int64_t)(q0 + i) * a.q.row +
                                              (int64_t)head * a.q.head + 16 * s + 2 * t + 8 * (r >> 1))
                        : 0u;
    }
  float o[D / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
#pragma unroll
  for (int d = 0; d < D / 8; d++)
#pragma unroll
    for (int k = 0; k < 4; k++) o[d][k] = 0.0f;
  int lim[2];
#pragma unroll
  for (int r = 0; r < 2; r++) lim[r] = a.causal ? min(nk, row[r] + nk - nq + 1) : nk;
  const int end = a.causal ? min(nk, i0 + kRows + nk - nq) : nk;
  const float c = __fmul_rn(a.scale, kLog2e);
  for (int i = tid; i < 3 * D; i += kThreads) odd[i / D][i % D] = INT_MAX;

  for (int j0 = 0; j0 < end; j0 += kKeys) {
    __syncthreads();
    for (int i = tid; i < kKeys * (D / 8); i += kThreads) {
      const int j = i / (D / 8), d = i % (D / 8) * 8;
      uint4 x = make_uint4(0, 0, 0, 0), y = x;
      if (j0 + j < nk) {
        x = *(const uint4 *)(kp + (int64_t)(k0 + j0 + j) * a.k.row + d);
        y = *(const uint4 *)(vp + (int64_t)(k0 + j0 + j) * a.v.row + d);
      }
      *(uint4 *)&ks[j][d] = x;
      *(uint4 *)&vs[j][d] = y;
    }
    __syncthreads();
    if (a.causal ? j0 + kKeys > i0 + nk - nq + 1 : j0 + kKeys > nk) {  // some row does not see all
      constexpr uint16_t kExp = BF16 ? 0x7f80 : 0x7c00;
      for (int i = tid; i < kKeys * D; i += kThreads) {
        const uint16_t x = vs[i / D][i % D];
        if ((x & kExp) == kExp) {
          atomicMin(&odd[(x & 0x7fff) != kExp ? 0 : x >> 15 ? 2 : 1][i % D], j0 + i / D);
          vs[i / D][i % D] = 0;
        }
      }
      __syncthreads();
    }
    float s[kKeys / 8][4];
#pragma unroll
    for (int nt = 0; nt < kKeys / 8; nt++) {
#pragma unroll
      for (int k = 0; k < 4; k++) s[nt][k] = 0.0f;
#pragma unroll
      for (int k = 0; k < D / 16; k++)
        mma16816<BF16>(s[nt], qf[k][0], qf[k][1], qf[k][2], qf[k][3],
                       *(const uint32_t *)&ks[8 * nt + g][16 * k + 2 * t],
                       *(const uint32_t *)&ks[8 * nt + g][16 * k + 2 * t + 8]);
    }
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int nt = 0; nt < kKeys / 8; nt++)
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const int j = j0 + 8 * nt + 2 * t + (k & 1);
        s[nt][k] = j < lim[k >> 1] ? __fmul_rn(s[nt][k], c) : -INFINITY;
        top[k >> 1] = fmaxf(top[k >> 1], s[nt][k]);
      }
    float base[2];
#pragma unroll
    for (int r = 0; r < 2; r++) {
      top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
      top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
      const float nm = fmaxf(m[r], top[r]);
      base[r] = nm == -INFINITY ? 0.0f : nm;
      const float f = exp2_fast(__fsub_rn(m[r], base[r]));
      m[r] = nm;
      l[r] = __fmul_rn(l[r], f);
#pragma unroll
      for (int d = 0; d < D / 8; d++) {
        o[d][2 * r] = __fmul_rn(o[d][2 * r], f);
        o[d][2 * r + 1] = __fmul_rn(o[d][2 * r + 1], f);
      }
    }
#pragma unroll
    for (int kk = 0; kk < kKeys / 16; kk++) {
      uint32_t p[4];
#pragma unroll
      for (int h = 0; h < 2; h++)
#pragma unroll
        for (int r = 0; r < 2; r++) {
          const float x = exp2_fast(__fsub_rn(s[2 * kk + h][2 * r], base[r]));
          const float y = exp2_fast(__fsub_rn(s[2 * kk + h][2 * r + 1], base[r]));
          l[r] = __fadd_rn(l[r], __fadd_rn(x, y));
          p[2 * h + r] = pack2<BF16>(x, y);
        }
#pragma unroll
      for (int d = 0; d < D / 16; d++) {
        uint32_t f[4];
        ldsm4t(f, &vs[16 * kk + (lane & 15)][16 * d + 8 * (lane >> 4)]);
        mma16816<BF16>(o[2 * d], p[0], p[1], p[2], p[3], f[0], f[1]);
        mma16816<BF16>(o[2 * d + 1], p[0], p[1], p[2], p[3], f[2], f[3]);
      }
    }
  }
  __syncthreads();
  auto extra = [&](int r, int d) {
    float x = odd[1][d] < lim[r] ? INFINITY : 0.0f;
    if (odd[2][d] < lim[r]) x = __fadd_rn(x, -INFINITY);
    return odd[0][d] < lim[r] ? NAN : x;
  };
#pragma unroll
  for (int r = 0; r < 2; r++) {
    l[r] = __fadd_rn(l[r], __shfl_xor_sync(0xffffffffu, l[r], 1));
    l[r] = __fadd_rn(l[r], __shfl_xor_sync(0xffffffffu, l[r], 2));
    if (row[r] >= nq) continue;
    const bool none = m[r] == -INFINITY;
    const float inv = none ? 0.0f : __fdiv_rn(1.0f, l[r]);
    uint16_t *to = (uint16_t *)a.out + ((int64_t)(q0 + row[r]) * a.q_heads + head) * D;
#pragma unroll
    for (int d = 0; d < D / 8; d++)
      *(uint32_t *)(to + 8 * d + 2 * t) =
          none ? 0u
               : pack2<BF16>(__fmaf_rn(o[d][2 * r], inv, extra(r, 8 * d + 2 * t)),
                             __fmaf_rn(o[d][2 * r + 1], inv, extra(r, 8 * d + 2 * t + 1)));
    if (a.lse != nullptr && t == 0)
      a.lse[(int64_t)(q0 + row[r]) * a.q_heads + head] =
          none ? -INFINITY : __fmul_rn(__fadd_rn(m[r], __log2f(l[r])), kLn2);
  }
}

cudaError_t launch(const Args &a, int sms, cudaStream_t st) {
  (void)sms;
  const dim3 grid((unsigned)(a.rows_q / kRows + a.n), (unsigned)a.q_heads);
  if (a.D == 64)
    (a.bf16 ? simple_kernel<64, true> : simple_kernel<64, false>)<<<grid, kThreads, 0, st>>>(a);
  else
    (a.bf16 ? simple_kernel<128, true> : simple_kernel<128, false>)<<<grid, kThreads, 0, st>>>(a);
  return cudaGetLastError();
}

}  // namespace prompt
}  // namespace uvb
