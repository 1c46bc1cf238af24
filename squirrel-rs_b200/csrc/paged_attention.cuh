// paged_attention.cuh — what the two kernels of the paged attention share: few query rows a
// kv head (paged_attention.cu) and many (paged_attention_tc.cu).
#pragma once
#include <math.h>

#include "common.cuh"
#include "paged.cuh"

namespace sq {
namespace paged {

constexpr float LOG2E = 1.4426950408889634f;

template <typename T>
struct AttnArgs {
  Cache c;
  Batch b;
  const T *q;
  T *out;
  long long qs, os;
  int n_heads, group;
  float scale;  // of the scores, times log2(e)
  int window, sinks;
  int few_rows;  // sequences with up to this many rows a kv head are the few-row kernel's, the others the many-row one's
  float *part;
  int *count;  // blocks that have left their part of a row tile; zero between calls
  int max_row_tiles;
  int withhold;  // failure-detection tests only: the many-row kernel's first block never gets its first piece
};

// Places on a line of work. The host refuses calls of LINE_END or more, taking the batch at its word; arrays that give
// rows to several sequences can still have more. Counts stop there, and such a call is recorded and left out: past
// 32 bits a thread block would look for its piece beyond the last sequence.
constexpr unsigned LINE_END = 1u << 30;
__device__ __forceinline__ unsigned line_add(unsigned a, unsigned b) { return min(a + b, LINE_END); }
__device__ __forceinline__ unsigned line_sum(unsigned v) {  // of the warp
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = line_add(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
template <int WARPS>
__device__ __forceinline__ int line_total(const int *warp_sums, unsigned *err) {  // 0 for a line that is too long
  unsigned v = 0;
#pragma unroll
  for (int w = 0; w < WARPS; w++) v = line_add(v, (unsigned)warp_sums[w]);
  if (v < LINE_END) return (int)v;
  if (threadIdx.x == 0) flag(err, BAD_START);
  return 0;
}

__device__ __forceinline__ uint32_t smem_addr(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void cp16(uint32_t dst, const void *src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ float ex2(float x) {  // relative error 2^-22; below 2^-126: 0
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t sub1152(uint32_t x) {  // two f16: 1024 + code -> code - 128
  uint32_t y;
  asm("sub.f16x2 %0, %1, %2;" : "=r"(y) : "r"(x), "r"(0x64806480u));
  return y;
}
// Codes (bytes 0, 1) and (2, 3) of a word as f16 pairs.
__device__ __forceinline__ uint32_t codes_lo(uint32_t w) { return sub1152(__byte_perm(w, 0x64646464u, 0x4140)); }
__device__ __forceinline__ uint32_t codes_hi(uint32_t w) { return sub1152(__byte_perm(w, 0x64646464u, 0x4342)); }
__device__ __forceinline__ uint32_t pack(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ float2 unpack(uint32_t x) { return __half22float2(*reinterpret_cast<const __half2 *>(&x)); }

// Power of two that takes a query row's largest magnitude to 2^10 .. 2^11 (as its
// exponent), and that factor; NaN for a row that holds NaN or an infinity, so that the
// row is NaN as a whole.
__device__ __forceinline__ int row_exp(float top) {
  return top > 0.f ? min(10 - ((int)(__float_as_uint(top) >> 23) - 127), 127) : 0;
}
__device__ __forceinline__ float row_factor(int e, bool finite) {
  return finite ? __uint_as_float((uint32_t)(e + 127) << 23) : __int_as_float(0x7fffffff);
}

// The exponent e of a page's V scale goes into its keys' scores: weights are 2^(s + e - max(s + e)), in f16's range where
// they count for the result, and the sum of the weights takes them times 2^-e. A key's exponent is not taken lower than
// V_EXP_SPAN below the largest met so far, so that no weight of the sum's first 50 bits vanishes, and at least
// V_EXP_MIN, so that the sum has room for 2^30 positions: what remains of such a scale counts as far as f16 goes.
constexpr int V_EXP_MIN = -80, V_EXP_SPAN = 80;
__device__ __forceinline__ int v_exp(float vs) {
  return min(max((int)(__float_as_uint(vs) >> 23 & 255) - 127, V_EXP_MIN), 126);
}
__device__ __forceinline__ float exp_inv(int e) { return __uint_as_float((uint32_t)(127 - e) << 23); }  // 2^-e
// v 2^x for a sum of weights: x may be below f32's exponents where v makes up for it.
__device__ __forceinline__ float scaled(float v, float x) { return v * ex2(fmaxf(x, -126.f)) * ex2(fminf(x + 126.f, 0.f)); }

// The many-row kernel (paged_attention_tc.cu).
bool many_supported(const Cache &c, int group);
template <typename T>
cudaError_t launch_many(cudaStream_t s, AttnArgs<T> a);
size_t many_partial_bytes(int head_dim);
int many_row_tiles(int max_new, int group);

}  // namespace paged
}  // namespace sq
