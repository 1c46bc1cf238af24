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

#include <algorithm>
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

int check_batch(const sq_paged_batch *b, const Cache &c, Batch *out, const char *what) {
  auto fail = [&](int code, const char *msg) { return sq::fail(code, std::string(what) + ": " + msg); };
  if (!b || !b->q_start || !b->kv_len || !b->page_table) return fail(SQ_ERR_ARG, "null batch pointer");
  if (b->n_seqs <= 0 || b->n_seqs > 65535) return fail(SQ_ERR_SHAPE, "1 to 65535 sequences");
  if (b->n_tokens < 0 || b->max_new < 0 || b->max_new > b->n_tokens || (b->n_tokens && !b->max_new) ||
      (long long)b->max_new * b->n_seqs < b->n_tokens)
    return fail(SQ_ERR_SHAPE, "max_new must be the most new tokens of one sequence");
  if (b->pages_per_seq <= 0) return fail(SQ_ERR_SHAPE, "a page table has columns");
  if ((long long)b->pages_per_seq * c.page > MAX_POSITIONS)
    return fail(SQ_ERR_SHAPE, "a page table names at most 2^30 positions of a sequence");
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

// Append moves 2 x (4 or 2) bytes an element of q, (4 or 2) + 1 of k and v. Threads take eight
// elements (16 or 32 bytes) at a time; a page block keeps HELD such chunks a thread in
// registers from the maximum to the codes, so that rows are read once. 24,465 tokens of 32
// and 8 heads of 64: f32 85.5 us, 6.2 TB/s, bound by that; bf16 85.8 us, 3.3 TB/s, bound by the
// instructions an element (rotation, maximum, rounding to a code), which are the same.
constexpr int HELD = 4;
constexpr int Q_CHUNKS = 4;  // chunks a thread of a query block takes

// One interleaved pair rotated as kernels/rope.rs:7-36 does: each product rounded.
__device__ __forceinline__ void spin(float &a, float &b, float c, float s) {
  const float x = __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s));
  b = __fadd_rn(__fmul_rn(a, s), __fmul_rn(b, c));
  a = x;
}
struct Eight {
  float x[8];
};
__device__ __forceinline__ Eight load8(const float *p) {
  const float4 a = load4(p), b = load4(p + 4);
  return {{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}};
}
__device__ __forceinline__ Eight load8(const __nv_bfloat16 *p) {
  const uint4 u = *reinterpret_cast<const uint4 *>(p);
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
  Eight e;
#pragma unroll
  for (int i = 0; i < 4; i++) e.x[2 * i] = __uint_as_float(w[i] << 16), e.x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  return e;
}
__device__ __forceinline__ void store8(float *p, const Eight &e) {
  store4(p, make_float4(e.x[0], e.x[1], e.x[2], e.x[3]));
  store4(p + 4, make_float4(e.x[4], e.x[5], e.x[6], e.x[7]));
}
__device__ __forceinline__ void store8(__nv_bfloat16 *p, const Eight &e) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(e.x[2 * i], e.x[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t *>(&h);
  }
  *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void spin8(Eight &e, const float *cos, const float *sin) {
  const float4 c = *reinterpret_cast<const float4 *>(cos), s = *reinterpret_cast<const float4 *>(sin);
  spin(e.x[0], e.x[1], c.x, s.x);
  spin(e.x[2], e.x[3], c.y, s.y);
  spin(e.x[4], e.x[5], c.z, s.z);
  spin(e.x[6], e.x[7], c.w, s.w);
}
__device__ __forceinline__ float finite_abs(float x) {
  const float a = fabsf(x);
  return a <= FLT_MAX ? a : 0.f;  // NaN and infinities set no scale
}
// The conversion takes NaN to 0 and an infinity to the integer range's end.
__device__ __forceinline__ uint32_t code_of(float x, float inv) {
  return (uint32_t)(min(max(__float2int_rn(__fmul_rn(x, inv)), -127), 127) + 128);
}
__device__ __forceinline__ uint32_t codes_of(const float *x, float inv) {
  return code_of(x[0], inv) | code_of(x[1], inv) << 8 | code_of(x[2], inv) << 16 | code_of(x[3], inv) << 24;
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

// Blocks [0, page_blocks): one (sequence, touched page, kv head, K or V) each. The rest: one part of a query row each.
template <typename T>
__global__ void __launch_bounds__(256) k_paged_append(const AppendArgs<T> a) {
  const Cache &c = a.c;
  const int tid = threadIdx.x, half = c.hd / 2, threads = blockDim.x;
  pdl_wait();  // the rows and the batch come from earlier kernels, which may still read the cache
  pdl_trigger();
  if ((int)blockIdx.x >= a.page_blocks) {
    const int blk = blockIdx.x - a.page_blocks, t = blk / a.q_parts, part = blk - t * a.q_parts;
    const int chunks = a.n_heads * c.hd / 8;
    const T *src = a.q + t * a.qs;
    T *dst = a.q_out + t * a.qos;
    Eight e[Q_CHUNKS];
#pragma unroll
    for (int i = 0; i < Q_CHUNKS; i++) {  // on their way while the position is looked up
      const int ch = (part * Q_CHUNKS + i) * threads + tid;
      if (ch < chunks) e[i] = load8(src + 8 * ch);
    }
    const Seq s = load_seq(a.b, c, seq_of_token(a.b, t));
    const int pos = s.len - s.n + (t - s.first);
    const bool ok = t >= s.first && t < s.first + s.n && pos >= 0 && pos < a.rope_rows;
    if (!ok && tid == 0) flag(a.b.err, BAD_POSITION);
#pragma unroll
    for (int i = 0; i < Q_CHUNKS; i++) {
      const int ch = (part * Q_CHUNKS + i) * threads + tid;
      if (ch < chunks) {
        const int pair = (8 * ch & (c.hd - 1)) / 2;
        if (ok) spin8(e[i], a.cos + (long long)pos * half + pair, a.sin + (long long)pos * half + pair);
        store8(dst + 8 * ch, e[i]);
      }
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
  const int from = max(pos0, 0), p = (from >> c.page_shift) + blk % a.touches;
  if (!s.n || p > (end - 1) >> c.page_shift) return;
  const int start = p << c.page_shift;
  const int lo = max(start, from), rows = min(start + c.page, end) - lo, held = lo - start;
  const long long stride = is_v ? a.vs : a.ks;
  const T *src = (is_v ? a.v : a.k) + (s.first + (lo - pos0)) * stride + g * c.hd;
  const int per_row = c.hd / 8, shift = 31 - __clz(per_row), n = rows * per_row;
  auto value = [&](int i) {
    const int r = i >> shift, d = 8 * (i & (per_row - 1));
    Eight e = load8(src + r * stride + d);
    if (!is_v) {
      const long long at = (long long)(lo + r) * half + d / 2;
      spin8(e, a.cos + at, a.sin + at);
    }
    return e;
  };
  auto top_of = [](const Eight &e, float top) {
#pragma unroll
    for (int i = 0; i < 8; i++) top = fmaxf(top, finite_abs(e.x[i]));
    return top;
  };
  Eight kept[HELD];
  float top = 0.f;
#pragma unroll
  for (int j = 0; j < HELD; j++)
    if (tid + j * threads < n) kept[j] = value(tid + j * threads);
  const int page = load_page(a.b, c, b, start);
#pragma unroll
  for (int j = 0; j < HELD; j++)
    if (tid + j * threads < n) top = top_of(kept[j], top);
  for (int i = tid + HELD * threads; i < n; i += threads) top = top_of(value(i), top);
  if (page < 0) return;
  const long long slot = (long long)page * c.kv_heads + g;
  float *scale_p = (is_v ? a.c.vs : a.c.ks) + slot;
  const float was = held ? *scale_p : 0.f;
  __shared__ unsigned tops[32];
  const unsigned mine = __reduce_max_sync(0xffffffffu, __float_as_uint(top));  // ordered like the floats: none is negative
  if ((tid & 31) == 0) tops[tid >> 5] = mine;
  __syncthreads();
  unsigned all = tops[0];
  for (int w = 1; w < threads / 32; w++) all = max(all, tops[w]);
  const float now = fmaxf(was, __uint_as_float(all) / 127.f);
  const float inv = now > 0.f ? fminf(1.f / now, FLT_MAX) : 0.f;
  uint8_t *codes = (is_v ? a.c.v : a.c.k) + slot * c.page * c.hd;
  if (held && now > was) {  // the earlier rows follow the new scale
    const float ratio = __fmul_rn(was, inv);
    uint32_t *w = reinterpret_cast<uint32_t *>(codes);
    for (int i = tid; i < held * c.hd / 4; i += threads) {
      const uint32_t u = w[i];
      const float x[4] = {(float)(int)(u & 255) - 128.f, (float)(int)(u >> 8 & 255) - 128.f,
                          (float)(int)(u >> 16 & 255) - 128.f, (float)(int)(u >> 24) - 128.f};
      w[i] = codes_of(x, ratio);
    }
  }
  uint2 *out = reinterpret_cast<uint2 *>(codes + held * c.hd);
#pragma unroll
  for (int j = 0; j < HELD; j++)
    if (tid + j * threads < n)
      out[tid + j * threads] = make_uint2(codes_of(kept[j].x, inv), codes_of(kept[j].x + 4, inv));
  for (int i = tid + HELD * threads; i < n; i += threads) {
    const Eight e = value(i);
    out[i] = make_uint2(codes_of(e.x, inv), codes_of(e.x + 4, inv));
  }
  if (tid == 0) *scale_p = now;
}

constexpr int READ_THREADS = 256;
constexpr int READ_ROWS = 4;

// Block (x, y): READ_ROWS positions of sequence y. A thread takes the same codes of each (4 for f32 values, 8 for bf16:
// 16 bytes stored), all of them on their way before the first is stored.
template <typename T>
__global__ void __launch_bounds__(READ_THREADS)
    k_paged_read(const Cache c, const Batch b, const int *first, int count, T *k_out,
                 T *v_out) {
  constexpr int N = 16 / sizeof(T), WORDS = N / 4;
  pdl_wait();
  pdl_trigger();
  const Seq s = load_seq(b, c, blockIdx.y);
  const int chunks = c.kv_heads * c.hd / N, per_head = c.hd / N, i0 = blockIdx.x * READ_ROWS;
  const long long pos0 = (long long)first[blockIdx.y] + i0;
  int page[READ_ROWS];
#pragma unroll
  for (int j = 0; j < READ_ROWS; j++) {
    const long long pos = pos0 + j;
    page[j] = i0 + j < count && pos >= 0 && pos < s.len ? load_page(b, c, blockIdx.y, (int)pos) : -1;
  }
  for (int q = threadIdx.x; q < chunks; q += READ_THREADS) {
    const int g = q / per_head, d = (q - g * per_head) * N;
    uint32_t u[READ_ROWS][2][WORDS];
    float scale[READ_ROWS][2];
#pragma unroll
    for (int j = 0; j < READ_ROWS; j++)
#pragma unroll
      for (int z = 0; z < 2; z++) {
        scale[j][z] = 0.f;
        if (page[j] >= 0) {
          const long long slot = (long long)page[j] * c.kv_heads + g;
          const uint8_t *codes = (z ? c.v : c.k) + (slot * c.page + ((pos0 + j) & (c.page - 1))) * c.hd + d;
          const uint32_t *src = reinterpret_cast<const uint32_t *>(codes);
          scale[j][z] = (z ? c.vs : c.ks)[slot];
          if constexpr (WORDS == 2) {
            const uint2 w = *reinterpret_cast<const uint2 *>(src);
            u[j][z][0] = w.x, u[j][z][WORDS - 1] = w.y;
          } else {
            u[j][z][0] = *src;
          }
        }
      }
#pragma unroll
    for (int j = 0; j < READ_ROWS; j++) {
      if (i0 + j >= count) break;
      T *dst[2] = {k_out, v_out};
#pragma unroll
      for (int z = 0; z < 2; z++) {
        T *p = dst[z] + (((long long)blockIdx.y * count + i0 + j) * chunks + q) * N;
        float x[N];
#pragma unroll
        for (int e = 0; e < N; e++)
          x[e] = page[j] >= 0 ? ((float)(int)(u[j][z][e / 4] >> (8 * (e & 3)) & 255) - 128.f) * scale[j][z] : 0.f;
        if constexpr (WORDS == 2) {
          store8(p, Eight{{x[0], x[1], x[2], x[3], x[N - 4], x[N - 3], x[N - 2], x[N - 1]}});
        } else {
          store4(p, make_float4(x[0], x[1], x[2], x[3]));
        }
      }
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
  // as many threads as a page's new rows have chunks for, up to HELD a thread
  const int chunks = std::min(c.page, b.max_new) * c.hd / 8;
  const int threads = std::min(std::max((chunks + HELD - 1) / HELD + 31 & ~31, 64), 256);
  a.q_parts = q ? (n_heads * c.hd / 8 + threads * Q_CHUNKS - 1) / (threads * Q_CHUNKS) : 0;
  const long long blocks = page_blocks + (long long)b.n_tokens * a.q_parts;
  if (blocks > INT32_MAX) return cudaErrorInvalidConfiguration;
  a.page_blocks = (int)page_blocks;
  return launch_ex(k_paged_append<T>, dim3((unsigned)blocks), dim3(threads), 0, s, pdl_enabled(), a);
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
  if (!st) st = paged::check_batch(batch, c, &b, "paged_append");
  if (st) return st;
  if (dtype != SQ_F32 && dtype != SQ_BF16) return fail(SQ_ERR_INVALID_TYPE, "paged_append: rows must be F32 or BF16");
  if (!b.n_tokens) return SQ_OK;
  if (!rope_cos || !rope_sin) return fail(SQ_ERR_ARG, "paged_append: null rotation table");
  if (rope_rows <= 0) return fail(SQ_ERR_SHAPE, "paged_append: empty rotation table");
  if (((uintptr_t)rope_cos | (uintptr_t)rope_sin) & 15)
    return fail(SQ_ERR_ALIGN, "paged_append: rotation tables must be 16-byte aligned");
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
  if (!st) st = paged::check_batch(batch, c, &b, "paged_read");
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
