// paged.cu — the paged 8-bit key/value cache: checks, rotation and append, reading back.
//
// Append, for one page and kv head, of rows x (k rotated to its position, or v):
//     need  = max |x| / 127 over the new rows        (finite elements only)
//     scale = max(old scale, need)                   (old scale: 0 when the page is new)
//     code  = 128 + clamp(rint(x * (1 / scale)), -127, 127)
// and, when the scale grew over rows already held, their codes become
//     128 + rint((code - 128) * (old scale * (1 / scale))),
// which adds at most half a step of the new scale; a page of 64 random rows grows about
// five times. Every product is rounded on its own (no contraction), so a page's contents
// depend on what was appended and in which steps, not on how a kernel is compiled.
#include <float.h>

#include <string>

#include "common.cuh"
#include "ops.cuh"
#include "paged.cuh"

namespace sq {
namespace paged {

__device__ unsigned g_paged_err;

unsigned *err_ptr() {
  static unsigned *ptrs[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return nullptr;
  if (!ptrs[dev]) {
    void *p = nullptr;
    if (cudaGetSymbolAddress(&p, g_paged_err) != cudaSuccess) return nullptr;
    ptrs[dev] = (unsigned *)p;
  }
  return ptrs[dev];
}

int check_cache(const sq_paged_cache *c, Cache *out, const char *what) {
  auto fail = [&](int code, const char *msg) { return sq::fail(code, std::string(what) + ": " + msg); };
  if (!c || !c->k || !c->v || !c->k_scale || !c->v_scale) return fail(SQ_ERR_ARG, "null cache pointer");
  if (c->n_pages <= 0 || c->n_kv_heads <= 0) return fail(SQ_ERR_SHAPE, "a cache has pages and kv heads");
  int shift = 4;
  while (shift < 8 && (1 << shift) != c->page) shift++;
  if ((1 << shift) != c->page) return fail(SQ_ERR_SHAPE, "a page holds 16, 32, 64, 128 or 256 positions");
  if (c->head_dim != 32 && c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256)
    return fail(SQ_ERR_SHAPE, "head_dim must be 32, 64, 128 or 256");
  if ((long long)c->n_pages * c->n_kv_heads * (c->page / 16) > INT32_MAX)
    return fail(SQ_ERR_SHAPE, "the cache's groups of 16 positions and kv heads must be countable in 31 bits");
  if (((uintptr_t)c->k | (uintptr_t)c->v) & 15 || ((uintptr_t)c->k_scale | (uintptr_t)c->v_scale) & 3)
    return fail(SQ_ERR_ALIGN, "codes must be 16-byte aligned, scales 4-byte");
  *out = {c->k, c->v, c->k_scale, c->v_scale, c->n_pages, c->n_kv_heads, c->page, shift, c->head_dim};
  return SQ_OK;
}

int check_batch(const sq_paged_batch *b, Batch *out, const char *what) {
  auto fail = [&](int code, const char *msg) { return sq::fail(code, std::string(what) + ": " + msg); };
  if (!b || !b->q_start || !b->kv_len || !b->page_table) return fail(SQ_ERR_ARG, "null batch pointer");
  if (b->n_seqs <= 0 || b->n_seqs > 65535) return fail(SQ_ERR_SHAPE, "1 to 65535 sequences");
  if (b->n_tokens < 0 || b->max_new < 0 || b->max_new > b->n_tokens || (b->n_tokens && !b->max_new) ||
      (long long)b->max_new * b->n_seqs < b->n_tokens)
    return fail(SQ_ERR_SHAPE, "max_new must be the most new tokens of one sequence");
  if (b->pages_per_seq <= 0) return fail(SQ_ERR_SHAPE, "a page table has columns");
  if (((uintptr_t)b->q_start | (uintptr_t)b->kv_len | (uintptr_t)b->page_table) & 3)
    return fail(SQ_ERR_ALIGN, "batch arrays must be 4-byte aligned");
  *out = {b->q_start, b->kv_len, b->page_table, b->n_seqs, b->n_tokens, b->max_new, b->pages_per_seq, nullptr};
  return SQ_OK;
}

int check_rows(const void *p, long long stride, long long width, int dtype, const char *what) {
  if (!p) return fail(SQ_ERR_ARG, std::string(what) + ": null pointer");
  if (stride < width) return fail(SQ_ERR_SHAPE, std::string(what) + ": rows overlap");
  const int item = dtype == SQ_F32 ? 4 : 2;
  if ((uintptr_t)p & 15 || stride * item & 15)
    return fail(SQ_ERR_ALIGN, std::string(what) + ": rows must start on 16-byte boundaries");
  return SQ_OK;
}

namespace {

constexpr int APPEND_THREADS = 128;
constexpr int Q_QUADS = 4;  // groups of four elements a thread of a query block takes

// One interleaved pair rotated as kernels/rope.rs:7-36 does: each product rounded.
__device__ __forceinline__ void spin(float &a, float &b, float c, float s) {
  const float x = __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s));
  b = __fadd_rn(__fmul_rn(a, s), __fmul_rn(b, c));
  a = x;
}
__device__ __forceinline__ float4 spin4(float4 x, const float *cos, const float *sin) {
  const float2 c = *reinterpret_cast<const float2 *>(cos), s = *reinterpret_cast<const float2 *>(sin);
  spin(x.x, x.y, c.x, s.x);
  spin(x.z, x.w, c.y, s.y);
  return x;
}
__device__ __forceinline__ float finite_abs(float x) {
  const float a = fabsf(x);
  return a <= FLT_MAX ? a : 0.f;  // NaN and infinities set no scale
}
// The conversion takes NaN to 0 and an infinity to the integer range's end.
__device__ __forceinline__ uint32_t code_of(float x, float inv) {
  return (uint32_t)(min(max(__float2int_rn(__fmul_rn(x, inv)), -127), 127) + 128);
}
__device__ __forceinline__ uint32_t codes_of(float4 x, float inv) {
  return code_of(x.x, inv) | code_of(x.y, inv) << 8 | code_of(x.z, inv) << 16 | code_of(x.w, inv) << 24;
}

template <typename T>
struct AppendArgs {
  Cache c;
  Batch b;
  const T *k, *v, *q;
  T *q_out;
  long long ks, vs, qs, qos;
  const float *cos, *sin;
  int rope_rows, n_heads;
  int touches;      // most pages one sequence's new tokens fall in
  int page_blocks;  // blocks that write pages; the rest rotate queries
  int q_parts;      // blocks of a query row
};

// Blocks [0, page_blocks): one (sequence, touched page, kv head, K or V) each, read twice
// (the maximum, then the codes; the second read comes from L1 / L2). The rest: one part
// of a query row each.
template <typename T>
__global__ void __launch_bounds__(APPEND_THREADS) k_paged_append(const AppendArgs<T> a) {
  const Cache &c = a.c;
  const int tid = threadIdx.x, half = c.hd / 2;
  pdl_wait();  // the rows and the batch come from earlier kernels, which may still read the cache
  pdl_trigger();
  if ((int)blockIdx.x >= a.page_blocks) {
    const int blk = blockIdx.x - a.page_blocks, t = blk / a.q_parts, part = blk % a.q_parts;
    const int b = seq_of_token(a.b, t);
    const Seq s = load_seq(a.b, c, b);
    const int pos = s.len - s.n + (t - s.first);
    const bool ok = t >= s.first && t < s.first + s.n && pos >= 0 && pos < a.rope_rows;
    if (!ok && tid == 0) flag(a.b.err, BAD_POSITION);
    const T *src = a.q + t * a.qs;
    T *dst = a.q_out + t * a.qos;
    const int quads = a.n_heads * c.hd / 4;
#pragma unroll
    for (int i = 0; i < Q_QUADS; i++) {
      const int quad = (part * Q_QUADS + i) * APPEND_THREADS + tid;
      if (quad >= quads) break;
      const int pair = (4 * quad & (c.hd - 1)) / 2;
      float4 x = load4(src + 4 * quad);
      if (ok) x = spin4(x, a.cos + (long long)pos * half + pair, a.sin + (long long)pos * half + pair);
      store4(dst + 4 * quad, x);
    }
    return;
  }
  int blk = blockIdx.x;
  const bool is_v = blk & 1;
  blk >>= 1;
  const int g = blk % c.kv_heads;
  blk /= c.kv_heads;
  const int b = blk / a.touches;
  const Seq s = load_seq(a.b, c, b);
  const int pos0 = s.len - s.n;  // position of the first new token
  const int end = min(s.len, a.rope_rows);
  if (tid == 0 && s.n && (pos0 < 0 || s.len > a.rope_rows)) flag(a.b.err, BAD_POSITION);
  const int from = max(pos0, 0), p = (from >> c.page_shift) + blk % a.touches, start = p << c.page_shift;
  if (!s.n || start >= end) return;
  const int page = load_page(a.b, c, b, start);
  if (page < 0) return;
  const int lo = max(start, from), rows = min(start + c.page, end) - lo, held = lo - start;
  const long long slot = (long long)page * c.kv_heads + g;
  float *scale_p = (is_v ? a.c.vs : a.c.ks) + slot;
  const float was = held ? *scale_p : 0.f;
  const T *src = (is_v ? a.v : a.k) + (s.first + (lo - pos0)) * (is_v ? a.vs : a.ks) + g * c.hd;
  const long long stride = is_v ? a.vs : a.ks;
  const int quads = c.hd / 4, qshift = 31 - __clz(quads), n = rows * quads;
  auto value = [&](int i) {
    const int r = i >> qshift, d = 4 * (i & (quads - 1));
    float4 x = load4(src + r * stride + d);
    if (!is_v) {
      const long long at = (long long)(lo + r) * half + d / 2;
      x = spin4(x, a.cos + at, a.sin + at);
    }
    return x;
  };

  float top = 0.f;
#pragma unroll 4
  for (int i = tid; i < n; i += APPEND_THREADS) {
    const float4 x = value(i);
    top = fmaxf(fmaxf(fmaxf(top, finite_abs(x.x)), finite_abs(x.y)), fmaxf(finite_abs(x.z), finite_abs(x.w)));
  }
  __shared__ unsigned tops[APPEND_THREADS / 32];
  const unsigned mine = __reduce_max_sync(0xffffffffu, __float_as_uint(top));  // ordered like the floats: none is negative
  if ((tid & 31) == 0) tops[tid >> 5] = mine;
  __syncthreads();
  unsigned all = tops[0];
#pragma unroll
  for (int w = 1; w < APPEND_THREADS / 32; w++) all = max(all, tops[w]);
  const float now = fmaxf(was, __uint_as_float(all) / 127.f);
  const float inv = now > 0.f ? fminf(1.f / now, FLT_MAX) : 0.f;
  uint8_t *codes = (is_v ? a.c.v : a.c.k) + slot * c.page * c.hd;
  if (held && now > was) {  // the earlier rows follow the new scale
    const float ratio = __fmul_rn(was, inv);
    uint32_t *w = reinterpret_cast<uint32_t *>(codes);
    for (int i = tid; i < held * quads; i += APPEND_THREADS) {
      const uint32_t u = w[i];
      const float4 x = make_float4((float)(int)(u & 255) - 128.f, (float)(int)(u >> 8 & 255) - 128.f,
                                   (float)(int)(u >> 16 & 255) - 128.f, (float)(int)(u >> 24) - 128.f);
      w[i] = codes_of(x, ratio);
    }
  }
  uint32_t *out = reinterpret_cast<uint32_t *>(codes + held * c.hd);
#pragma unroll 4
  for (int i = tid; i < n; i += APPEND_THREADS) out[i] = codes_of(value(i), inv);
  if (tid == 0) *scale_p = now;
}

constexpr int READ_THREADS = 256;
constexpr int READ_ROWS = 4;

// Block (x, y): READ_ROWS positions of sequence y.
template <typename T>
__global__ void __launch_bounds__(READ_THREADS)
    k_paged_read(const Cache c, const Batch b, const int *__restrict__ first, int count, T *__restrict__ k_out,
                 T *__restrict__ v_out) {
  pdl_wait();
  pdl_trigger();
  const Seq s = load_seq(b, c, blockIdx.y);
  const int quads = c.kv_heads * c.hd / 4, per_head = c.hd / 4;
  const int pos0 = first[blockIdx.y];
  for (int j = 0; j < READ_ROWS; j++) {
    const int i = blockIdx.x * READ_ROWS + j;
    if (i >= count) return;
    const long long pos = (long long)pos0 + i;
    const int page = pos >= 0 && pos < s.len ? load_page(b, c, blockIdx.y, (int)pos) : -1;
    const long long row = ((long long)blockIdx.y * count + i) * quads * 4;
    for (int q = threadIdx.x; q < quads; q += READ_THREADS) {
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f), y = x;
      if (page >= 0) {
        const int g = q / per_head;
        const long long slot = (long long)page * c.kv_heads + g;
        const long long at = (slot * c.page + (pos & (c.page - 1))) * c.hd + 4 * (q - g * per_head);
        const uchar4 u = *reinterpret_cast<const uchar4 *>(c.k + at), w = *reinterpret_cast<const uchar4 *>(c.v + at);
        const float ks = c.ks[slot], vs = c.vs[slot];
        x = make_float4(((float)u.x - 128.f) * ks, ((float)u.y - 128.f) * ks, ((float)u.z - 128.f) * ks,
                        ((float)u.w - 128.f) * ks);
        y = make_float4(((float)w.x - 128.f) * vs, ((float)w.y - 128.f) * vs, ((float)w.z - 128.f) * vs,
                        ((float)w.w - 128.f) * vs);
      }
      store4(k_out + row + 4 * q, x);
      store4(v_out + row + 4 * q, y);
    }
  }
}

template <typename T>
cudaError_t append(cudaStream_t s, const Cache &c, const Batch &b, const void *k, long long ks, const void *v,
                   long long vs, const float *cos, const float *sin, int rope_rows, const void *q, long long qs,
                   int n_heads, void *q_out, long long qos) {
  AppendArgs<T> a = {c,  b,  (const T *)k, (const T *)v, (const T *)q, (T *)q_out, ks, vs, qs,
                     qos, cos, sin,          rope_rows,    n_heads,      0,          0,  0};
  a.touches = (b.max_new - 1 + c.page - 1) / c.page + 1;
  const long long page_blocks = 2LL * b.n_seqs * a.touches * c.kv_heads;
  a.q_parts = q ? (n_heads * c.hd / 4 + APPEND_THREADS * Q_QUADS - 1) / (APPEND_THREADS * Q_QUADS) : 0;
  const long long blocks = page_blocks + (long long)b.n_tokens * a.q_parts;
  if (blocks > INT32_MAX) return cudaErrorInvalidConfiguration;
  a.page_blocks = (int)page_blocks;
  return launch_ex(k_paged_append<T>, dim3((unsigned)blocks), dim3(APPEND_THREADS), 0, s, pdl_enabled(), a);
}

}  // namespace
}  // namespace paged
}  // namespace sq

using namespace sq;

extern "C" int sq_paged_status(int clear) {
  unsigned v = 0, *p = paged::err_ptr();
  if (!p) return fail(SQ_ERR_CUDA, "paged_status: no current CUDA device");
  SQ_CUDA(cudaMemcpy(&v, p, sizeof(v), cudaMemcpyDeviceToHost));
  if (!v) return SQ_OK;
  if (clear) SQ_CUDA(cudaMemset(p, 0, sizeof(v)));
  if (v & paged::BAD_WAIT) return fail(SQ_ERR_TIMEOUT, "paged_status: a bounded wait expired");
  std::string what;
  if (v & paged::BAD_PAGE) what += "; a page id is outside the cache";
  if (v & paged::BAD_LENGTH) what += "; kv_len is negative or beyond the page table";
  if (v & paged::BAD_START) what += "; q_start does not ascend from 0 to n_tokens in steps of at most max_new";
  if (v & paged::BAD_POSITION) what += "; a new token's position is negative or past the rotation table";
  return fail(SQ_ERR_ARG, "paged_status: " + what.substr(2));
}

extern "C" int sq_paged_append(void *stream, const sq_paged_cache *cache, const sq_paged_batch *batch, int dtype,
                               const void *k, long long k_stride, const void *v, long long v_stride,
                               const float *rope_cos, const float *rope_sin, int rope_rows, const void *q,
                               long long q_stride, int n_heads, void *q_out, long long q_out_stride) {
  paged::Cache c;
  paged::Batch b;
  int st = paged::check_cache(cache, &c, "paged_append");
  if (!st) st = paged::check_batch(batch, &b, "paged_append");
  if (st) return st;
  if (dtype != SQ_F32 && dtype != SQ_BF16) return fail(SQ_ERR_INVALID_TYPE, "paged_append: rows must be F32 or BF16");
  if (!b.n_tokens) return SQ_OK;
  if (!rope_cos || !rope_sin) return fail(SQ_ERR_ARG, "paged_append: null rotation table");
  if (rope_rows <= 0) return fail(SQ_ERR_SHAPE, "paged_append: empty rotation table");
  if (((uintptr_t)rope_cos | (uintptr_t)rope_sin) & 7)
    return fail(SQ_ERR_ALIGN, "paged_append: rotation tables must be 8-byte aligned");
  const long long width = (long long)c.kv_heads * c.hd;
  st = paged::check_rows(k, k_stride, width, dtype, "paged_append: k");
  if (!st) st = paged::check_rows(v, v_stride, width, dtype, "paged_append: v");
  if (!st && q) {
    if (n_heads <= 0) return fail(SQ_ERR_SHAPE, "paged_append: n_heads must be positive");
    st = paged::check_rows(q, q_stride, (long long)n_heads * c.hd, dtype, "paged_append: q");
    if (!st) st = paged::check_rows(q_out, q_out_stride, (long long)n_heads * c.hd, dtype, "paged_append: q_out");
  }
  if (st) return st;
  if (!(b.err = paged::err_ptr())) return fail(SQ_ERR_CUDA, "paged_append: no current CUDA device");
  const auto run = dtype == SQ_F32 ? paged::append<float> : paged::append<__nv_bfloat16>;
  cudaError_t e = run((cudaStream_t)stream, c, b, k, k_stride, v, v_stride, rope_cos, rope_sin, rope_rows, q, q_stride,
                      n_heads, q_out, q_out_stride);
  return e == cudaSuccess ? SQ_OK : cuda_fail(e, "sq_paged_append");
}

extern "C" int sq_paged_read(void *stream, const sq_paged_cache *cache, const sq_paged_batch *batch,
                             const int32_t *first, int count, int dtype, void *k_out, void *v_out) {
  paged::Cache c;
  paged::Batch b;
  int st = paged::check_cache(cache, &c, "paged_read");
  if (!st) st = paged::check_batch(batch, &b, "paged_read");
  if (st) return st;
  if (dtype != SQ_F32 && dtype != SQ_BF16) return fail(SQ_ERR_INVALID_TYPE, "paged_read: rows must be F32 or BF16");
  if (count < 0) return fail(SQ_ERR_SHAPE, "paged_read: negative count");
  if (!count) return SQ_OK;
  if (!first) return fail(SQ_ERR_ARG, "paged_read: null pointer");
  const long long width = (long long)c.kv_heads * c.hd;
  st = paged::check_rows(k_out, width, width, dtype, "paged_read: k_out");
  if (!st) st = paged::check_rows(v_out, width, width, dtype, "paged_read: v_out");
  if (st) return st;
  if (!(b.err = paged::err_ptr())) return fail(SQ_ERR_CUDA, "paged_read: no current CUDA device");
  const dim3 grid((count + paged::READ_ROWS - 1) / paged::READ_ROWS, b.n_seqs), block(paged::READ_THREADS);
  const cudaError_t e =
      dtype == SQ_F32 ? launch_ex(paged::k_paged_read<float>, grid, block, 0, (cudaStream_t)stream, pdl_enabled(), c, b,
                                  first, count, (float *)k_out, (float *)v_out)
                      : launch_ex(paged::k_paged_read<__nv_bfloat16>, grid, block, 0, (cudaStream_t)stream, pdl_enabled(),
                                  c, b, first, count, (__nv_bfloat16 *)k_out, (__nv_bfloat16 *)v_out);
  if (e != cudaSuccess) return cuda_fail(e, "sq_paged_read");
  return SQ_OK;
}
