// capi_kv.cu -- extern "C" entry points of the cache held in 4 bits and of
// the attention over prompts: argument checks and launches.  Every buffer is
// the caller's device memory; nothing here waits for the device except
// uv_kv_check.
#include <cfloat>

#include "capi_internal.h"
#include "uv_prompt.h"

using namespace uvb;
using namespace uvcapi;

namespace {

int on_device(const void *p, int device, const char *what) {
  if (p == nullptr) return fail(UV_EINVAL, std::string(what) + " is null");
  bool dev = false;
  UV_TRY(classify(p, device, &dev));
  if (!dev) return fail(UV_EINVAL, std::string(what) + " must be device memory");
  return UV_OK;
}

// bits 0, 2, 4, .. of x in the low half, 1, 3, 5, .. in the high half
uint32_t split_pairs(uint32_t x) {
  auto even = [](uint32_t v) {
    v &= 0x55555555u;
    v = (v | v >> 1) & 0x33333333u;
    v = (v | v >> 2) & 0x0f0f0f0fu;
    v = (v | v >> 4) & 0x00ff00ffu;
    return (v | v >> 8) & 0xffffu;
  };
  return even(x) | even(x >> 1) << 16;
}

int sizes(const uv_kv *kv) {
  if (kv == nullptr) return fail(UV_EINVAL, "null cache");
  if (kv->head_dim != 64 && kv->head_dim != 128 && kv->head_dim != 256)
    return fail(UV_EUNSUPPORTED, "head_dim must be 64, 128 or 256");
  if (kv->page_tokens != 32 && kv->page_tokens != 64 && kv->page_tokens != 128 &&
      kv->page_tokens != 256)
    return fail(UV_EUNSUPPORTED, "page_tokens must be 32, 64, 128 or 256");
  if (kv->kv_heads < 1 || kv->kv_heads > 4096 || kv->layers < 1 || kv->n_pages < 1 ||
      kv->max_seqs < 1 || kv->max_pages < 1 || kv->rounds < 1 || kv->rounds > 3)
    return fail(UV_EINVAL, "kv_heads, layers, n_pages, max_seqs, max_pages must be positive and "
                           "rounds 1 to 3");
  if ((int64_t)kv->max_seqs * kv->max_pages > INT32_MAX ||
      (int64_t)kv->max_pages * kv->page_tokens > INT32_MAX)
    return fail(UV_EINVAL, "the table has more than 2^31 entries or tokens a sequence");
  return UV_OK;
}

int open(const uv_kv *kv, kv::Cache *c) {
  UV_TRY(sizes(kv));
  UV_TRY(on_device(kv->pool, kv->device, "pool"));
  UV_TRY(on_device(kv->table, kv->device, "table"));
  UV_TRY(on_device(kv->lens, kv->device, "lens"));
  UV_TRY(on_device(kv->refs, kv->device, "refs"));
  UV_TRY(on_device(kv->work, kv->device, "work"));
  if ((uintptr_t)kv->pool % 16) return fail(UV_EINVAL, "pool must be 16-byte aligned");
  c->head_dim = kv->head_dim;
  c->heads = kv->kv_heads;
  c->layers = kv->layers;
  c->page_tokens = kv->page_tokens;
  c->n_pages = kv->n_pages;
  c->max_seqs = kv->max_seqs;
  c->max_pages = kv->max_pages;
  c->rounds = kv->rounds;
  for (int r = 0; r < kv::kMaxRounds; r++)
    for (int w = 0; w < 8; w++) c->signs[r][w] = split_pairs(kv->signs[r][w]);
  c->pool = (uint8_t *)kv->pool;
  c->table = kv->table;
  c->lens = kv->lens;
  c->refs = kv->refs;
  c->work = kv->work;
  return UV_OK;
}

// A list of sequences; at most one entry a sequence.
int listed(const uv_kv *kv, const int32_t *seqs, int32_t n, const char *what) {
  if (n < 0) return fail(UV_EINVAL, "negative count");
  if (n > kv->max_seqs) return fail(UV_EINVAL, "more entries than sequences");
  return n == 0 ? UV_OK : on_device(seqs, kv->device, what);
}

int packed(const uv_kv *kv, int32_t layer, const int32_t *seqs, const int32_t *starts, int32_t n,
           int32_t rows, kv::Rows *r) {
  if (layer < 0 || layer >= kv->layers) return fail(UV_EINVAL, "no such layer");
  UV_TRY(listed(kv, seqs, n, "seqs"));
  if (rows < 0) return fail(UV_EINVAL, "negative rows");
  if (n > 0 && starts != nullptr) UV_TRY(on_device(starts, kv->device, "starts"));
  if (starts == nullptr && rows != n)
    return fail(UV_EINVAL, "without starts every sequence has one row");
  *r = {seqs, starts, n, rows};
  return UV_OK;
}

int operand(const void *p, int64_t row, int64_t head, int device, const char *what,
            kv::Strided *out) {
  UV_TRY(on_device(p, device, what));
  if ((uintptr_t)p % 16 || row % 8 || head % 8 || row < 0 || head < 0)
    return fail(UV_EINVAL, std::string(what) +
                               ": 16-byte aligned rows wanted (strides multiples of 8 values)");
  *out = {p, row, head};
  return UV_OK;
}

// For a tensor map: a stride over one element is not read, but has to be one.
int mapped(kv::Strided *x, int rows, int heads, int dim, const char *what) {
  if (heads == 1) x->head = dim;
  if (rows == 1) x->row = (int64_t)heads * x->head;
  if (x->row == 0 || x->head == 0)
    return fail(UV_EINVAL, std::string(what) + ": strides must be positive");
  return UV_OK;
}

int dense(const void *p, int device, const char *what) {
  UV_TRY(on_device(p, device, what));
  if ((uintptr_t)p % 16) return fail(UV_EINVAL, std::string(what) + " must be 16-byte aligned");
  return UV_OK;
}

int typed(int32_t dtype) {
  if (dtype != UV_F16 && dtype != UV_BF16)
    return fail(UV_EUNSUPPORTED, "dtype must be UV_F16 or UV_BF16");
  return UV_OK;
}

}  // namespace

extern "C" {

int uv_kv_pool_bytes(const uv_kv *kv, int64_t *bytes) {
  UV_TRY(sizes(kv));
  if (bytes == nullptr) return fail(UV_EINVAL, "null result");
  *bytes = (int64_t)kv->layers * kv->n_pages * kv->kv_heads * kv->page_tokens * (kv->head_dim + 8);
  return UV_OK;
}

int uv_kv_work_words(const uv_kv *kv, int64_t *words) {
  UV_TRY(sizes(kv));
  if (words == nullptr) return fail(UV_EINVAL, "null result");
  *words = kv::kWorkHead + 3 * (int64_t)kv->n_pages + 2 * (int64_t)kv->max_seqs;
  return UV_OK;
}

int uv_kv_seed(uv_kv *kv, uint64_t seed) {
  UV_TRY(sizes(kv));
  const RotationHost rot = build_rotation(kv->head_dim, seed, kv->rounds);
  std::memset(kv->signs, 0, sizeof(kv->signs));
  for (int r = 0; r < kv->rounds; r++)
    for (int i = 0; i < kv->head_dim; i++)
      if (rot.signs[(size_t)r * kv->head_dim + i] < 0.0f)
        kv->signs[r][i / 32] |= 1u << (i % 32);
  return UV_OK;
}

int uv_kv_reset(const uv_kv *kv, void *stream) {
  kv::Cache c;
  UV_TRY(open(kv, &c));
  DeviceGuard g(kv->device);
  cudaStream_t st = (cudaStream_t)stream;
  UV_CK(cudaMemsetAsync(c.table, 0xff, (size_t)c.max_seqs * c.max_pages * 4, st));
  UV_CK(cudaMemsetAsync(c.lens, 0, (size_t)c.max_seqs * 4, st));
  UV_CK(cudaMemsetAsync(c.refs, 0, (size_t)c.n_pages * 4, st));
  UV_CK(cudaMemsetAsync(c.work, 0, (size_t)c.work_words() * 4, st));
  return UV_OK;
}

int uv_kv_recount(const uv_kv *kv, void *stream) {
  kv::Cache c;
  UV_TRY(open(kv, &c));
  DeviceGuard g(kv->device);
  UV_CK(kv::recount_launch(c, (cudaStream_t)stream));
  return UV_OK;
}

int uv_kv_check(const uv_kv *kv, int32_t *status, void *stream) {
  kv::Cache c;
  UV_TRY(open(kv, &c));
  if (status == nullptr) return fail(UV_EINVAL, "null result");
  DeviceGuard g(kv->device);
  cudaStream_t st = (cudaStream_t)stream;
  UV_CK(cudaMemcpyAsync(status, c.work + kv::kStatus, 4, cudaMemcpyDeviceToHost, st));
  UV_CK(cudaStreamSynchronize(st));
  if (*status != 0) UV_CK(cudaMemsetAsync(c.work + kv::kStatus, 0, 4, st));
  return UV_OK;
}

int uv_kv_extend(const uv_kv *kv, const int32_t *seqs, const int32_t *counts, int32_t n,
                 void *stream) {
  kv::Cache c;
  UV_TRY(open(kv, &c));
  UV_TRY(listed(kv, seqs, n, "seqs"));
  if (n == 0) return UV_OK;
  UV_TRY(on_device(counts, kv->device, "counts"));
  DeviceGuard g(kv->device);
  ProfScope ps("kv_extend", (cudaStream_t)stream);
  UV_CK(kv::extend_launch(c, seqs, counts, n, sm_count(kv->device), (cudaStream_t)stream));
  return UV_OK;
}

int uv_kv_fork(const uv_kv *kv, const int32_t *src, const int32_t *dst, const int32_t *lens,
               int32_t n, void *stream) {
  kv::Cache c;
  UV_TRY(open(kv, &c));
  UV_TRY(listed(kv, dst, n, "dst"));
  if (n == 0) return UV_OK;
  UV_TRY(on_device(src, kv->device, "src"));
  if (lens != nullptr) UV_TRY(on_device(lens, kv->device, "lens"));
  DeviceGuard g(kv->device);
  ProfScope ps("kv_fork", (cudaStream_t)stream);
  UV_CK(kv::fork_launch(c, src, dst, lens, n, (cudaStream_t)stream));
  return UV_OK;
}

int uv_kv_copy(const uv_kv *kv, const int32_t *src, const int32_t *dst, int32_t n, void *stream) {
  kv::Cache c;
  UV_TRY(open(kv, &c));
  UV_TRY(listed(kv, dst, n, "dst"));
  if (n == 0) return UV_OK;
  UV_TRY(on_device(src, kv->device, "src"));
  DeviceGuard g(kv->device);
  ProfScope ps("kv_copy", (cudaStream_t)stream);
  UV_CK(kv::copy_launch(c, src, dst, n, sm_count(kv->device), (cudaStream_t)stream));
  return UV_OK;
}

int uv_kv_truncate(const uv_kv *kv, const int32_t *seqs, const int32_t *lens, int32_t n,
                   void *stream) {
  kv::Cache c;
  UV_TRY(open(kv, &c));
  UV_TRY(listed(kv, seqs, n, "seqs"));
  if (n == 0) return UV_OK;
  if (lens != nullptr) UV_TRY(on_device(lens, kv->device, "lens"));
  DeviceGuard g(kv->device);
  ProfScope ps("kv_truncate", (cudaStream_t)stream);
  UV_CK(kv::truncate_launch(c, seqs, lens, n, (cudaStream_t)stream));
  return UV_OK;
}

int uv_kv_compact(const uv_kv *kv, void *stream) {
  kv::Cache c;
  UV_TRY(open(kv, &c));
  DeviceGuard g(kv->device);
  ProfScope ps("kv_compact", (cudaStream_t)stream);
  UV_CK(kv::compact_launch(c, sm_count(kv->device), (cudaStream_t)stream));
  return UV_OK;
}

int uv_kv_append(const uv_kv *kv, int32_t layer, const int32_t *seqs, const int32_t *starts,
                 int32_t n, int32_t rows, int32_t dtype, const void *k, int64_t k_row,
                 int64_t k_head, const void *v, int64_t v_row, int64_t v_head, void *stream) {
  kv::Cache c;
  kv::Rows r;
  kv::Strided ks, vs;
  UV_TRY(open(kv, &c));
  UV_TRY(packed(kv, layer, seqs, starts, n, rows, &r));
  UV_TRY(typed(dtype));
  if (n == 0 || rows == 0) return UV_OK;
  UV_TRY(operand(k, k_row, k_head, kv->device, "k", &ks));
  UV_TRY(operand(v, v_row, v_head, kv->device, "v", &vs));
  DeviceGuard g(kv->device);
  ProfScope ps("kv_append", (cudaStream_t)stream);
  UV_CK(kv::append_launch(c, layer, r, ks, vs, dtype == UV_BF16, (cudaStream_t)stream));
  return UV_OK;
}

int uv_kv_read(const uv_kv *kv, int32_t layer, const int32_t *seqs, const int32_t *starts,
               int32_t n, int32_t rows, int32_t dtype, void *k, void *v, void *stream) {
  kv::Cache c;
  kv::Rows r;
  UV_TRY(open(kv, &c));
  UV_TRY(packed(kv, layer, seqs, starts, n, rows, &r));
  UV_TRY(typed(dtype));
  if (n == 0 || rows == 0) return UV_OK;
  UV_TRY(dense(k, kv->device, "k"));
  UV_TRY(dense(v, kv->device, "v"));
  DeviceGuard g(kv->device);
  ProfScope ps("kv_read", (cudaStream_t)stream);
  UV_CK(kv::read_launch(c, layer, r, k, v, dtype == UV_BF16, (cudaStream_t)stream));
  return UV_OK;
}

int uv_kv_attend_bytes(const uv_kv *kv, int32_t n, int32_t rows, int32_t most, int32_t q_heads,
                       int64_t *bytes) {
  UV_TRY(sizes(kv));
  if (bytes == nullptr || n < 0 || rows < 0 || most < 1 || q_heads < 1 ||
      q_heads % kv->kv_heads != 0)
    return fail(UV_EINVAL, "q_heads must be a multiple of kv_heads, most at least 1");
  kv::Cache c = {};
  c.head_dim = kv->head_dim;
  c.heads = kv->kv_heads;
  *bytes = kv::attend_plan(c, n, rows, most, q_heads, sm_count(kv->device)).bytes;
  return UV_OK;
}

int uv_kv_attend(const uv_kv *kv, int32_t layer, const int32_t *seqs, const int32_t *starts,
                 int32_t n, int32_t rows, int32_t most, int32_t dtype, const void *q,
                 int64_t q_row, int64_t q_head, int32_t q_heads, float scale, void *out,
                 float *lse, void *scratch, int64_t scratch_bytes, void *stream) {
  kv::Cache c;
  kv::Rows r;
  kv::AttendArgs a;
  UV_TRY(open(kv, &c));
  UV_TRY(packed(kv, layer, seqs, starts, n, rows, &r));
  UV_TRY(typed(dtype));
  if (most < 1 || q_heads < 1 || q_heads % kv->kv_heads != 0)
    return fail(UV_EINVAL, "q_heads must be a multiple of kv_heads, most at least 1");
  if (!(scale > 0.0f) || scale > FLT_MAX) return fail(UV_EINVAL, "scale must be positive");
  if (n == 0 || rows == 0) return UV_OK;
  UV_TRY(operand(q, q_row, q_head, kv->device, "q", &a.q));
  UV_TRY(dense(out, kv->device, "out"));
  if (lse != nullptr) UV_TRY(on_device(lse, kv->device, "lse"));
  a.out = out;
  a.lse = lse;
  a.q_heads = q_heads;
  a.scale = scale;
  // Numbers that scratch memory does not hold by chance: mixed, never 0.
  static std::atomic<uint64_t> calls{0};
  uint64_t seed = calls.fetch_add(1) ^ 0x6b76617474656e64ull;
  a.call = splitmix64(&seed) | 1;
  const kv::AttendPlan plan =
      kv::attend_plan(c, n, rows, starts == nullptr ? 1 : most, q_heads, sm_count(kv->device));
  if (plan.jobs > INT32_MAX) return fail(UV_EINVAL, "too many rows for one call");
  DeviceGuard g(kv->device);
  Scratch sc((cudaStream_t)stream);
  if (scratch != nullptr) {
    if (scratch_bytes < plan.bytes) return fail(UV_EINVAL, "scratch is too small");
    UV_TRY(on_device(scratch, kv->device, "scratch"));
    if ((uintptr_t)scratch % 128) return fail(UV_EINVAL, "scratch must be 128-byte aligned");
    a.scratch = scratch;
  } else {
    uint8_t *p = nullptr;
    UV_TRY(sc.alloc(&p, (size_t)plan.bytes));
    a.scratch = p;
  }
  ProfScope ps("kv_attend", (cudaStream_t)stream);
  UV_CK(kv::attend_launch(c, layer, r, a, plan, dtype == UV_BF16, (cudaStream_t)stream));
  return UV_OK;
}

int uv_prompt_attention(int32_t device, const int32_t *starts_q, const int32_t *starts_k,
                        int32_t n, int32_t rows_q, int32_t rows_k, int32_t q_heads,
                        int32_t kv_heads, int32_t head_dim, int32_t causal, float scale,
                        int32_t dtype, const void *q, int64_t q_row, int64_t q_head, const void *k,
                        int64_t k_row, int64_t k_head, const void *v, int64_t v_row,
                        int64_t v_head, void *out, float *lse, void *stream) {
  if (n < 0 || rows_q < 0 || rows_k < 0) return fail(UV_EINVAL, "negative count");
  if (head_dim != 64 && head_dim != 128)
    return fail(UV_EUNSUPPORTED, "head_dim must be 64 or 128");
  if (kv_heads < 1 || q_heads < 1 || q_heads % kv_heads != 0 || q_heads > 65535)
    return fail(UV_EINVAL, "q_heads must be a multiple of kv_heads");
  UV_TRY(typed(dtype));
  if (!(scale > 0.0f) || scale > FLT_MAX) return fail(UV_EINVAL, "scale must be positive");
  if (n == 0 || rows_q == 0) return UV_OK;
  prompt::Args a;
  UV_TRY(on_device(starts_q, device, "starts_q"));
  if (starts_k == nullptr) {
    if (rows_k != rows_q) return fail(UV_EINVAL, "without starts_k keys and queries are as many");
    starts_k = starts_q;
  } else {
    UV_TRY(on_device(starts_k, device, "starts_k"));
  }
  UV_TRY(operand(q, q_row, q_head, device, "q", &a.q));
  UV_TRY(mapped(&a.q, rows_q, q_heads, head_dim, "q"));
  if (rows_k > 0) {
    UV_TRY(operand(k, k_row, k_head, device, "k", &a.k));
    UV_TRY(operand(v, v_row, v_head, device, "v", &a.v));
    UV_TRY(mapped(&a.k, rows_k, kv_heads, head_dim, "k"));
    UV_TRY(mapped(&a.v, rows_k, kv_heads, head_dim, "v"));
  } else {
    a.k = a.v = {q, 0, 0};  // never read
  }
  UV_TRY(dense(out, device, "out"));
  if (lse != nullptr) UV_TRY(on_device(lse, device, "lse"));
  a.starts_q = starts_q;
  a.starts_k = starts_k;
  a.n = n;
  a.rows_q = rows_q;
  a.rows_k = rows_k;
  a.q_heads = q_heads;
  a.heads = kv_heads;
  a.D = head_dim;
  a.causal = causal != 0;
  a.bf16 = dtype == UV_BF16;
  a.scale = scale;
  a.out = out;
  a.lse = lse;
  DeviceGuard g(device);
  ProfScope ps("prompt_attention", (cudaStream_t)stream);
  UV_CK(prompt::launch(a, (cudaStream_t)stream));
  return UV_OK;
}

}  // extern "C"
