// speculative.cu — verification of drafted tokens against the target's probabilities.
//
// Token i of a sequence is accepted while u_i * q_i(x_i) < p_i(x_i), which happens with
// probability min(1, p / q). At the first rejection the next token is drawn from
// max(p - q, 0), after the last draft from p: the accepted tokens and the drawn one are
// then distributed as the target's own. The draw inverts the cumulated weights. Weights
// are whole numbers, trunc(2^38 * probability) in 64 bits, so their sum is the same in
// every order and the drawn index does not depend on how the row is split; 2^-38
// keeps the tail of a row that probabilities down to 4e-12 make up.
// One cluster of eight blocks a sequence: bound by reading the one or two rows that decide
// (1 MB at 128,256 tokens); a single block of 1,024 threads took 36 us for one sequence, the
// cluster takes 7.3. Each warp sums one piece of the rows, the blocks exchange their sums through
// distributed shared memory, and the warp whose piece holds the drawn weight reads its piece
// again (from L1) to find the token. No workspace, no atomics, no second launch.
#include <cooperative_groups.h>

#include <string>

#include "common.cuh"
#include "ops.cuh"
#include "status.h"

namespace sq {
namespace {

namespace cg = cooperative_groups;

// Four blocks of 512 threads an SM: all of 64 sequences' blocks run at once (20.5 us; with two an SM 25.5, with
// clusters of four 23.6), and one sequence still takes 7.3 us (clusters of four: 10.7).
constexpr int VERIFY_CLUSTER = 8, VERIFY_THREADS = 512, VERIFY_WARPS = VERIFY_THREADS / 32;
constexpr int UNIFORM_BITS = 24;

struct VerifyArgs {
  const float *target, *draft, *uniform;
  const int *tokens, *n_draft;
  long long ts, ds;
  int max_draft, vocab;
  int *accepted, *out;
};

// trunc(2^38 x) as 2^18 hi + lo, both with the bits of 2^23 on top (BIAS): additions that round towards zero
// cut the parts out at full rate, where a conversion to 64 bits runs at a fraction of it (64 x 128,256 tokens:
// 25.7 us with the conversion, 20.5 with these). NaN and negative x: 0; above 1: 1.
constexpr uint32_t BIAS = 0x4B000000u;
struct Parts {
  uint32_t hi, lo;
};
__device__ __forceinline__ Parts parts_of(float x) {
  const float y = fminf(fmaxf(x, 0.f), 1.f) * 1048576.f, t = __fadd_rz(y, 8388608.f);
  const float rest = __fsub_rn(y, __fsub_rn(t, 8388608.f));
  return {__float_as_uint(t), __float_as_uint(__fmaf_rz(rest, 262144.f, 8388608.f))};
}
__device__ __forceinline__ unsigned long long weight_of(Parts p) {
  return ((unsigned long long)(p.hi - BIAS) << 18) + (p.lo - BIAS);
}

__device__ __forceinline__ unsigned long long warp_sum_u64(unsigned long long v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

__device__ __forceinline__ unsigned long long warp_scan_u64(unsigned long long v) {  // inclusive
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned long long y = __shfl_up_sync(0xffffffffu, v, o);
    if ((threadIdx.x & 31) >= o) v += y;
  }
  return v;
}

// The weights of four consecutive tokens i .. i + 3 (those past `end`: 0). VEC: the rows allow 16-byte loads.
struct Row {
  const float *p, *q;  // target, draft (or null)
  int without;         // token left out (-1: none)
};
template <bool VEC>
__device__ __forceinline__ void weights4(const Row &r, int i, int end, Parts (&w)[4]) {
  float x[4] = {0.f, 0.f, 0.f, 0.f};
  if (VEC && i + 4 <= end) {
    const float4 a = *reinterpret_cast<const float4 *>(r.p + i);
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w;
    if (r.q) {
      const float4 b = *reinterpret_cast<const float4 *>(r.q + i);
      x[0] = __fsub_rn(x[0], b.x), x[1] = __fsub_rn(x[1], b.y), x[2] = __fsub_rn(x[2], b.z), x[3] = __fsub_rn(x[3], b.w);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; j++)
      if (i + j < end) x[j] = r.q ? __fsub_rn(r.p[i + j], r.q[i + j]) : r.p[i + j];
  }
#pragma unroll
  for (int j = 0; j < 4; j++) w[j] = parts_of(i + j == r.without ? 0.f : x[j]);
}

template <bool VEC>
__device__ __forceinline__ unsigned long long sum_piece(const Row &r, int lo, int hi) {
  constexpr int TURNS = 8;  // 32 tokens a lane: their sums fit 32 bits (hi 2^25, lo 2^23)
  unsigned long long sum = 0;
#pragma unroll 1
  for (int i0 = lo + 4 * (threadIdx.x & 31); i0 < hi; i0 += 128 * TURNS) {
    uint32_t his = 0, los = 0;
#pragma unroll
    for (int k = 0; k < TURNS; k++) {
      Parts w[4];
      weights4<VEC>(r, i0 + 128 * k, hi, w);
      his += (w[0].hi + w[1].hi) + (w[2].hi + w[3].hi);
      los += (w[0].lo + w[1].lo) + (w[2].lo + w[3].lo);
    }
    his -= 4 * TURNS * BIAS, los -= 4 * TURNS * BIAS;  // modulo 2^32
    sum += ((unsigned long long)his << 18) + los;
  }
  return warp_sum_u64(sum);
}

// The first token of the piece at which `before` plus the weights up to it exceeds `goal`.
template <bool VEC>
__device__ int find_token(const Row &r, int lo, int hi, unsigned long long before, unsigned long long goal) {
  const int lane = threadIdx.x & 31;
#pragma unroll 4
  for (int i0 = lo; i0 < hi; i0 += 128) {
    Parts parts[4];
    weights4<VEC>(r, i0 + 4 * lane, hi, parts);
    const unsigned long long w[4] = {weight_of(parts[0]), weight_of(parts[1]), weight_of(parts[2]), weight_of(parts[3])};
    const unsigned long long run = before + warp_scan_u64((w[0] + w[1]) + (w[2] + w[3]));
    const unsigned over = __ballot_sync(0xffffffffu, run > goal);
    if (over) {
      const int first = __ffs(over) - 1;
      unsigned long long at = run;  // less the weights after token j
      int j = 3;
#pragma unroll
      for (int k = 3; k > 0; k--) {
        at -= w[k];
        if (at > goal) j = k - 1;
        else break;
      }
      return __shfl_sync(0xffffffffu, i0 + 4 * lane + j, first);
    }
    before = __shfl_sync(0xffffffffu, run, 31);
  }
  return -1;  // not reached: the piece holds the goal
}

// A block's shared memory may be written by another only once the block runs: arrival when it starts, the wait
// before the first such write (by then the others have long arrived).
__device__ __forceinline__ void cluster_started() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait_started() { asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); }

__global__ void __cluster_dims__(VERIFY_CLUSTER, 1, 1) __launch_bounds__(VERIFY_THREADS, 4)
    k_verify(const VerifyArgs a) {
  __shared__ unsigned long long sums[VERIFY_WARPS], totals[2][VERIFY_CLUSTER];  // of the warps; of the cluster's blocks
  __shared__ int s_accepted;
  cg::cluster_group cluster = cg::this_cluster();
  cluster_started();
  const int rank = cluster.block_rank(), b = blockIdx.x / VERIFY_CLUSTER;
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  const int K = a.max_draft, V = a.vocab;
  pdl_wait();  // the probabilities come from earlier kernels
  pdl_trigger();
  const int n = a.n_draft ? min(max(a.n_draft[b], 0), K) : K;
  const int *tok = a.tokens + (long long)b * K;
  const float *u = a.uniform + (long long)b * (K + 1);
  if (wid == 0) {  // every block finds the first rejection itself
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
  const float uf = fmaxf(u[K], 0.f) * (float)(1 << UNIFORM_BITS);
  const unsigned long long part = (unsigned long long)min((long long)uf, (1LL << UNIFORM_BITS) - 1);
  __syncthreads();
  const int acc = s_accepted;
  const bool rejected = acc < n;
  Row row = {a.target + ((long long)b * (K + 1) + acc) * a.ts,
             rejected && a.draft ? a.draft + ((long long)b * K + acc) * a.ds : nullptr,
             rejected && !a.draft ? tok[acc] : -1};
  int *out = a.out + (long long)b * (K + 1);
  if (rank == 0) {
    for (int i = tid; i <= K; i += VERIFY_THREADS)
      if (i != acc) out[i] = i < acc ? tok[i] : -1;
    if (tid == 0) a.accepted[b] = acc;
  }
  // pieces of whole groups of four tokens, one a warp of the cluster
  const int seg = ((V + 3) / 4 + VERIFY_CLUSTER * VERIFY_WARPS - 1) / (VERIFY_CLUSTER * VERIFY_WARPS) * 4;
  const int lo = (int)min((long long)(rank * VERIFY_WARPS + wid) * seg, (long long)V), hi = min(lo + seg, V);
  for (int pass = 0; pass < 2; pass++) {  // the remainder, then (if it has no mass) the target
    if (pass) row.q = nullptr, row.without = -1;
    const bool vec = (((uintptr_t)row.p | (uintptr_t)row.q) & 15) == 0;
    const unsigned long long sum = vec ? sum_piece<true>(row, lo, hi) : sum_piece<false>(row, lo, hi);
    if (lane == 0) sums[wid] = sum;
    __syncthreads();
    if (!pass) cluster_wait_started();
    if (wid == 0) {
      const unsigned long long mine = warp_sum_u64(lane < VERIFY_WARPS ? sums[lane] : 0ull);
      if (lane < VERIFY_CLUSTER) *cluster.map_shared_rank(&totals[pass][rank], lane) = mine;
    }
    cluster.sync();
    unsigned long long total = 0, before = 0;
#pragma unroll
    for (int r = 0; r < VERIFY_CLUSTER; r++) {
      if (r == rank) before = total;
      total += totals[pass][r];
    }
    if (!total) {
      if (pass == 1 && rank == 0 && tid == 0) out[acc] = -1;
      continue;  // the whole cluster does
    }
#pragma unroll
    for (int w = 0; w < VERIFY_WARPS; w++)
      if (w < wid) before += sums[w];
    const unsigned long long goal =
        part * (total >> UNIFORM_BITS) + (part * (total & ((1ull << UNIFORM_BITS) - 1)) >> UNIFORM_BITS);
    if (goal >= before && goal < before + sum) {  // this warp's piece holds the drawn token
      const int x = vec ? find_token<true>(row, lo, hi, before, goal) : find_token<false>(row, lo, hi, before, goal);
      if (lane == 0) out[acc] = x;
    }
    return;  // no block reads another's shared memory past the exchange
  }
}

}  // namespace
}  // namespace sq

using namespace sq;

extern "C" int sq_verify_drafts(void *stream, const float *target, long long target_stride, const float *draft,
                                long long draft_stride, const int32_t *tokens, const int32_t *n_draft,
                                const float *uniform, int n_seqs, int max_draft, int vocab, int32_t *n_accepted,
                                int32_t *out_tokens) {
  // without sequences the arrays are empty, and an empty array may have no address
  if (n_seqs && (!target || !uniform || !n_accepted || !out_tokens || (max_draft > 0 && !tokens)))
    return fail(SQ_ERR_ARG, "verify_drafts: null pointer");
  if (n_seqs < 0 || n_seqs > INT32_MAX / VERIFY_CLUSTER || max_draft < 0 || max_draft == INT32_MAX || vocab <= 0 ||
      vocab > INT32_MAX - 4096)
    return fail(SQ_ERR_SHAPE, "verify_drafts: counts out of range or an empty vocabulary");
  if (target_stride < vocab || (draft && draft_stride < vocab))
    return fail(SQ_ERR_SHAPE, "verify_drafts: rows overlap");
  if (((uintptr_t)target | (uintptr_t)draft | (uintptr_t)tokens | (uintptr_t)n_draft | (uintptr_t)uniform) & 3)
    return fail(SQ_ERR_ALIGN, "verify_drafts: arrays must be 4-byte aligned");
  if (!n_seqs) return SQ_OK;
  const VerifyArgs a = {target, draft,     uniform, tokens,     n_draft,   target_stride, draft_stride,
                        max_draft, vocab, n_accepted, out_tokens};
  const cudaError_t e = launch_ex(k_verify, dim3(n_seqs * VERIFY_CLUSTER), dim3(VERIFY_THREADS), 0,
                                  (cudaStream_t)stream, pdl_enabled(), a);
  if (e != cudaSuccess) return cuda_fail(e, "sq_verify_drafts");
  return SQ_OK;
}
