// speculative.cu — verification of drafted tokens against the target's probabilities.
//
// Token i of a sequence is accepted while u_i * q_i(x_i) < p_i(x_i), which happens with
// probability min(1, p / q). At the first rejection the next token is drawn from
// max(p - q, 0), after the last draft from p: the accepted tokens and the drawn one are
// then distributed as the target's own. The draw inverts the cumulated weights. Weights
// are whole numbers, trunc(2^38 * probability) in 64 bits, so their sum is the same in
// every order and the drawn index does not depend on how the row is split; 2^-38
// keeps the tail of a row that probabilities down to 4e-12 make up.
#include <string>

#include "common.cuh"
#include "status.h"

namespace sq {
namespace {

constexpr int VERIFY_THREADS = 1024;
constexpr int VERIFY_WARPS = VERIFY_THREADS / 32;
constexpr float WEIGHT_ONE = 274877906944.f;  // 2^38
constexpr int UNIFORM_BITS = 24;

struct VerifyArgs {
  const float *target, *draft, *uniform;
  const int *tokens, *n_draft;
  long long ts, ds;
  int max_draft, vocab;
  int *accepted, *out;
};

__device__ __forceinline__ unsigned long long weight_of(float x) {
  return x > 0.f ? (unsigned long long)(fminf(x, 1.f) * WEIGHT_ONE) : 0ull;  // NaN: no weight
}

__device__ __forceinline__ unsigned long long warp_sum_u64(unsigned long long v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// One block a sequence.
__global__ void __launch_bounds__(VERIFY_THREADS) k_verify(const VerifyArgs a) {
  __shared__ unsigned long long sums[VERIFY_WARPS];
  __shared__ int s_accepted;
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  const int K = a.max_draft, V = a.vocab;
  const int n = a.n_draft ? min(max(a.n_draft[b], 0), K) : K;
  const int *tok = a.tokens + (long long)b * K;
  const float *u = a.uniform + (long long)b * (K + 1);
  if (wid == 0) {
    int acc = n;
    for (int i0 = 0; i0 < n; i0 += 32) {
      const int i = i0 + lane;
      bool ok = true;
      if (i < n) {
        const int x = tok[i];
        ok = (unsigned)x < (unsigned)V;
        if (ok) {
          const float p = a.target[((long long)b * (K + 1) + i) * a.ts + x];
          const float q = a.draft ? a.draft[((long long)b * K + i) * a.ds + x] : 1.f;
          ok = __fmul_rn(u[i], q) < p;
        }
      }
      const unsigned bad = __ballot_sync(0xffffffffu, !ok);
      if (bad) {
        acc = i0 + __ffs(bad) - 1;
        break;
      }
    }
    if (lane == 0) s_accepted = acc;
  }
  __syncthreads();
  const int acc = s_accepted;
  const float *p = a.target + ((long long)b * (K + 1) + acc) * a.ts;
  const bool rejected = acc < n;
  const float *q = rejected && a.draft ? a.draft + ((long long)b * K + acc) * a.ds : nullptr;
  const int without = rejected && !a.draft ? tok[acc] : -1;
  const int seg = (V + VERIFY_WARPS - 1) / VERIFY_WARPS, lo = min(wid * seg, V), hi = min(lo + seg, V);
  int *out = a.out + (long long)b * (K + 1);
  for (int i = tid; i <= K; i += VERIFY_THREADS)
    if (i != acc) out[i] = i < acc ? tok[i] : -1;
  if (tid == 0) a.accepted[b] = acc;
  for (int pass = 0; pass < 2; pass++) {  // the remainder, then (if it has no mass) the target
    auto weight = [&](int i) {
      float x = p[i];
      if (pass == 0) {
        if (q) x = __fsub_rn(x, q[i]);
        if (i == without) x = 0.f;
      }
      return weight_of(x);
    };
    unsigned long long sum = 0;
    for (int i = lo + lane; i < hi; i += 32) sum += weight(i);
    sum = warp_sum_u64(sum);
    if (lane == 0) sums[wid] = sum;
    __syncthreads();
    unsigned long long total = 0, before = 0;
    for (int w = 0; w < VERIFY_WARPS; w++) {
      if (w == wid) before = total;
      total += sums[w];
    }
    __syncthreads();
    if (!total) {
      if (pass == 1 && tid == 0) out[acc] = -1;
      continue;
    }
    const float uf = fmaxf(u[K], 0.f) * (float)(1 << UNIFORM_BITS);
    const unsigned long long part = (unsigned long long)min((long long)uf, (1LL << UNIFORM_BITS) - 1);
    const unsigned long long goal =
        part * (total >> UNIFORM_BITS) + (part * (total & ((1ull << UNIFORM_BITS) - 1)) >> UNIFORM_BITS);
    if (goal < before || goal >= before + sum) return;
    for (int i0 = lo; i0 < hi; i0 += 32) {  // this warp's segment holds the drawn token
      const unsigned long long w = i0 + lane < hi ? weight(i0 + lane) : 0ull;
      unsigned long long run = w;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long y = __shfl_up_sync(0xffffffffu, run, o);
        if (lane >= o) run += y;
      }
      const unsigned over = __ballot_sync(0xffffffffu, before + run > goal);
      if (over) {
        if (lane == 0) out[acc] = i0 + __ffs(over) - 1;
        return;
      }
      before += __shfl_sync(0xffffffffu, run, 31);
    }
    return;
  }
}

}  // namespace
}  // namespace sq

using namespace sq;

extern "C" int sq_verify_drafts(void *stream, const float *target, long long target_stride, const float *draft,
                                long long draft_stride, const int32_t *tokens, const int32_t *n_draft,
                                const float *uniform, int n_seqs, int max_draft, int vocab, int32_t *n_accepted,
                                int32_t *out_tokens) {
  if (!target || !uniform || !n_accepted || !out_tokens || (max_draft > 0 && !tokens))
    return fail(SQ_ERR_ARG, "verify_drafts: null pointer");
  if (n_seqs < 0 || max_draft < 0 || vocab <= 0)
    return fail(SQ_ERR_SHAPE, "verify_drafts: negative counts or an empty vocabulary");
  if (target_stride < vocab || (draft && draft_stride < vocab))
    return fail(SQ_ERR_SHAPE, "verify_drafts: rows overlap");
  if (((uintptr_t)target | (uintptr_t)draft | (uintptr_t)tokens | (uintptr_t)n_draft | (uintptr_t)uniform) & 3)
    return fail(SQ_ERR_ALIGN, "verify_drafts: arrays must be 4-byte aligned");
  if (!n_seqs) return SQ_OK;
  const VerifyArgs a = {target, draft,     uniform, tokens,     n_draft,   target_stride, draft_stride,
                        max_draft, vocab, n_accepted, out_tokens};
  k_verify<<<n_seqs, VERIFY_THREADS, 0, (cudaStream_t)stream>>>(a);
  SQ_CHECK_LAUNCH("sq_verify_drafts");
  return SQ_OK;
}
