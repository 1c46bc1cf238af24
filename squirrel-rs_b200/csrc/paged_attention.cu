// paged_attention.cu — causal grouped attention over the paged 8-bit cache.
#include <math.h>

#include <string>

#include "common.cuh"
#include "paged.cuh"

namespace sq {
namespace paged {
namespace {

template <typename T>
struct AttnArgs {
  Cache c;
  Batch b;
  const T *q;
  T *out;
  long long qs, os;
  int n_heads, group;
  float scale;
  int window, sinks;
};

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void put(float *p, float x) { *p = x; }
__device__ __forceinline__ void put(__nv_bfloat16 *p, float x) { *p = __float2bfloat16_rn(x); }

// One warp a query row and head; lanes share the dimensions, keys come one at a time.
template <typename T, int HD>
__global__ void __launch_bounds__(32) k_paged_attention(const AttnArgs<T> a) {
  constexpr int DPL = HD / 32;
  const int t = blockIdx.x, h = blockIdx.y, g = h / a.group, lane = threadIdx.x;
  const int b = seq_of_token(a.b, t);
  const Seq s = load_seq(a.b, a.c, b);
  const int pos = s.len - s.n + (t - s.first);
  float q[DPL], acc[DPL], m = -INFINITY, l = 0.f;
  for (int i = 0; i < DPL; i++) {
    q[i] = to_f(a.q[t * a.qs + h * HD + lane * DPL + i]) * a.scale;
    acc[i] = 0.f;
  }
  for (int j = 0; j <= pos && j < s.len; j++) {
    if (a.window && j <= pos - a.window && j >= a.sinks) {
      j = pos - a.window;
      continue;
    }
    const int page = load_page(a.b, a.c, b, j);
    if (page < 0) continue;
    const long long slot = (long long)page * a.c.kv_heads + g;
    const long long at = (slot * a.c.page + (j & (a.c.page - 1))) * HD + lane * DPL;
    float d = 0.f;
    for (int i = 0; i < DPL; i++) d = fmaf(q[i], (float)a.c.k[at + i] - 128.f, d);
    d = warp_sum(d) * a.c.ks[slot];
    const float mn = fmaxf(m, d), corr = expf(m - mn), p = expf(d - mn);
    l = l * corr + p;
    for (int i = 0; i < DPL; i++) acc[i] = acc[i] * corr + p * a.c.vs[slot] * ((float)a.c.v[at + i] - 128.f);
    m = mn;
  }
  for (int i = 0; i < DPL; i++) put(a.out + t * a.os + h * HD + lane * DPL + i, l == 0.f ? 0.f : acc[i] / l);
}

template <typename T>
cudaError_t attention(cudaStream_t s, const Cache &c, const Batch &b, const void *q, long long qs, int n_heads,
                      float scale, int window, int sinks, void *out, long long os) {
  const AttnArgs<T> a = {c, b, (const T *)q, (T *)out, qs, os, n_heads, n_heads / c.kv_heads, scale, window, sinks};
  const dim3 grid(b.n_tokens, n_heads);
  switch (c.hd) {
    case 32: k_paged_attention<T, 32><<<grid, 32, 0, s>>>(a); break;
    case 64: k_paged_attention<T, 64><<<grid, 32, 0, s>>>(a); break;
    case 128: k_paged_attention<T, 128><<<grid, 32, 0, s>>>(a); break;
    default: k_paged_attention<T, 256><<<grid, 32, 0, s>>>(a); break;
  }
  return cudaGetLastError();
}

size_t workspace_bytes(const Batch &, const Cache &, int) { return 256; }

int check_heads(const Cache &c, int n_heads, const char *what) {
  if (n_heads <= 0 || n_heads % c.kv_heads)
    return fail(SQ_ERR_SHAPE, std::string(what) + ": n_heads must be a positive multiple of n_kv_heads");
  return SQ_OK;
}

}  // namespace
}  // namespace paged
}  // namespace sq

using namespace sq;

extern "C" int sq_paged_attention_workspace(const sq_paged_cache *cache, const sq_paged_batch *batch, int n_heads,
                                            size_t *bytes) {
  paged::Cache c;
  int st = paged::check_cache(cache, &c, "paged_attention_workspace");
  paged::Batch b;
  if (!st) st = paged::check_batch(batch, &b, "paged_attention_workspace");
  if (!st && !bytes) st = fail(SQ_ERR_ARG, "paged_attention_workspace: null pointer");
  if (!st) st = paged::check_heads(c, n_heads, "paged_attention_workspace");
  if (st) return st;
  *bytes = paged::workspace_bytes(b, c, n_heads);
  return SQ_OK;
}

extern "C" int sq_paged_attention(void *stream, const sq_paged_cache *cache, const sq_paged_batch *batch, int dtype,
                                  const void *q, long long q_stride, int n_heads, float scale, int window, int sinks,
                                  void *out, long long out_stride, void *ws, size_t ws_bytes) {
  paged::Cache c;
  paged::Batch b;
  int st = paged::check_cache(cache, &c, "paged_attention");
  if (!st) st = paged::check_batch(batch, &b, "paged_attention");
  if (!st) st = paged::check_heads(c, n_heads, "paged_attention");
  if (st) return st;
  if (dtype != SQ_F32 && dtype != SQ_BF16)
    return fail(SQ_ERR_INVALID_TYPE, "paged_attention: rows must be F32 or BF16");
  if (window < 0 || sinks < 0) return fail(SQ_ERR_SHAPE, "paged_attention: negative window or sinks");
  if (!b.n_tokens) return SQ_OK;
  const long long width = (long long)n_heads * c.hd;
  st = paged::check_rows(q, q_stride, width, dtype, "paged_attention: q");
  if (!st) st = paged::check_rows(out, out_stride, width, dtype, "paged_attention: out");
  if (st) return st;
  if (!ws || ws_bytes < paged::workspace_bytes(b, c, n_heads))
    return fail(SQ_ERR_ARG, "paged_attention: the workspace is smaller than paged_attention_workspace says");
  if ((uintptr_t)ws & 255) return fail(SQ_ERR_ALIGN, "paged_attention: the workspace must be 256-byte aligned");
  if (!(b.err = paged::err_ptr())) return fail(SQ_ERR_CUDA, "paged_attention: no current CUDA device");
  const auto run = dtype == SQ_F32 ? paged::attention<float> : paged::attention<__nv_bfloat16>;
  cudaError_t e = run((cudaStream_t)stream, c, b, q, q_stride, n_heads, scale, window, sinks, out, out_stride);
  return e == cudaSuccess ? SQ_OK : cuda_fail(e, "sq_paged_attention");
}
