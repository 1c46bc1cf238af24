// paged_attention.cu — causal grouped attention over the paged 8-bit cache, for few query
// rows a kv head (single tokens, drafted tokens): bound by reading the cache.
//
// out = softmax(scale * q.k) v over the keys a query sees, in one pass with a running
// maximum and sum. A row is one query token of one head; the rows of a kv head share its
// keys, so every code is read and converted once for all of them.
//
// The products run on mma.sync m16n8k16 (f16 in, f32 sums) rather than tcgen05: with at
// most 32 rows the tensor work is small, and the register fragments let a warp convert
// the codes it needs where it needs them, with no second pass through shared memory.
//   scores:  S[16 keys][8 rows]   = K[16 keys][dims] Q^T      (keys in the M rows)
//   output:  O[16 dims][8 rows]  += V^T[16 dims][keys] P      (dimensions in the M rows)
// Dimensions and keys are numbered inside the products so that a lane's K fragment is 16
// consecutive bytes of a key and its V fragment consecutive bytes of four keys; P goes
// from the scores' layout to the operand's by movmatrix.
//
// Precision. Codes are whole numbers up to 127: exact in f16. Query rows are scaled by a
// power of two; an f32 row takes two f16 terms (22 bits) and so two products, a bf16 row is
// exact in one. Weights, at most 2^10 (the maximum's), likewise: two terms for f32
// rows, one (11 bits, under the output's 8) for bf16 rows. The exponent of a page's V scale goes
// into its scores, the rest of it into the weights, so f16 neither overflows nor loses the
// weights of a page with small values beside one with large ones. With bf16
// rows K's codes enter as the f16 numbers code * 2^-24 (denormal, exact; one instruction a
// pair) and their bias leaves with the sum of the row, 128 sum(q): that costs a score two
// bits of 24 at most. With f32 rows the bias is taken off before the product (one
// instruction a pair more), and V's always is: an output is an average that may be a
// thousand times smaller than 128. The tensor core truncates its running sum (2^-25 of it a
// step on average): the scores of the query's two terms are summed apart, and f32 rows
// move their output sums every 8 groups of keys to f32 sums in shared memory. Measured
// with 4 x 131,072 positions of f32 rows: the bias taken off afterwards and one sum 66 us, error
// 1.4e-6 of the result; as it is 69 us, 8.2e-7; sums moved every 16 groups 0.7 us less, 1.0e-6
// (1,001 positions: 5.5e-7 and 8.1e-7, the plain f32 form 9.1e-7).
//
// Work is split evenly over the grid: the (sequence, kv head, row tile, key tile) space is
// one line, every block takes an equal piece of it, the four warps of a block take its key
// tiles in turn. A piece's ends move to the nearest end of a row tile's keys when that is
// at most SNAP tiles away: a cut costs about 6 us (partial results, the join, a second
// start), as long as the whole GPU reads some 20 tiles a block. A row tile that is cut
// leaves partial results in the workspace and the last block to arrive joins them, in block
// order (equal bits every call).
#include <float.h>
#include <limits.h>
#include <math.h>

#include <string>

#include "ops.cuh"
#include "paged_attention.cuh"

namespace sq {
namespace paged {
namespace {

constexpr int WARPS = 4, THREADS = WARPS * 32, STAGES = 2;
constexpr int BLOCKS_PER_SM = 3;
constexpr int MAX_BLOCKS = 160 * BLOCKS_PER_SM;  // and parts of a row tile
// What a row tile costs besides its keys (queries, look-ups, the join of the warps), in key tiles, when the work is
// shared out; these places hold no keys and a piece that would begin in them begins with the next row tile. 0 / 4 / 16:
// 64 x 5 drafts in up to 1,000 positions (f32, 64 dimensions) 49.1 / 43.1 / 43.2 us, 128 x up to 300 (bf16, 128) 25.0 / 22.4 /
// 24.0, 64 x up to 4,000 62.4 / 62.3 / 62.2, 16 x 5 drafts in up to 4,099 (f32) 37.6 / 38.7 / 42.5.
constexpr int JOB_COST = 4;
constexpr int MIN_TILES = WARPS;  // key tiles a block takes at least
constexpr int FLUSH_STEPS = 8;     // f32 rows: groups of 16 keys summed on the tensor core at a stretch
constexpr int SLOT_FLOATS = 2112;  // partial results of a row tile: 32 x 66 at most: maxima, sums, [row][head_dim]
constexpr size_t PARTIAL_BYTES = (size_t)MAX_BLOCKS * 2 * SLOT_FLOATS * 4;
constexpr float WEIGHT_EXP = 10.f;  // weights are 2^(s - max + 10)

__device__ __forceinline__ uint2 lds64(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
  return v;
}
// Codes (bytes 0, 2) and (1, 3) of a word as pairs of f16 numbers: code * 2^-24, or exact code - 128.
template <bool EXACT>
__device__ __forceinline__ uint32_t codes_02(uint32_t w) {
  return EXACT ? sub1152(w & 0x00FF00FFu | 0x64006400u) : w & 0x00FF00FFu;
}
template <bool EXACT>
__device__ __forceinline__ uint32_t codes_13(uint32_t w) {
  return EXACT ? sub1152(__byte_perm(w, 0x64646464u, 0x4341)) : __byte_perm(w, 0, 0x4341);
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <typename T, int HD_, int NT_>
struct Cfg {
  static constexpr int HD = HD_, NT = NT_;
  static constexpr bool SPLIT = sizeof(T) == 4;  // two f16 terms a row and weight
  static constexpr int TERMS = SPLIT ? 2 : 1;
  static constexpr int ROWS = NT * 8;
  static constexpr int TK = HD <= 64 ? 64 : 4096 / HD;   // keys a tile
  static constexpr int NG = TK / 16;                     // groups of 16 keys: each within one page
  static constexpr int TILE = TK * HD;                   // bytes of one operand's tile
  static constexpr int KS = HD / 16;                     // 16-dimension steps
  static constexpr int RING = WARPS * STAGES * 2 * TILE;
  static constexpr int SUMS = SPLIT ? WARPS * 32 * (HD / 16) * NT * 4 * 4 : 0;  // f32 rows: a lane's output sums
  static constexpr int SMEM = RING + SUMS;
  static constexpr int BATCH = 32 / NG;  // tiles whose pages a warp looks up at once
  static constexpr int SNAP = NT == 1 ? 16 : 8;  // tiles: 32 x 1,028 positions (bf16) 26 -> 21.5 us, 16 x 5 drafts (f32) 45 -> 38
  static constexpr int BLOCKS = NT <= 2 && 3 * SMEM <= 223 * 1024 ? BLOCKS_PER_SM : 2;
  static_assert(ROWS * (HD + 2) <= SLOT_FLOATS, "a row tile's partial results fit a slot");
  static_assert((MAX_BLOCKS * 8 + THREADS * 4) * 4 <= RING, "the factors of eight rows' parts fit the ring");
  static_assert(WARPS * ROWS * (HD + 2) * 4 <= RING, "the warps' results fit the ring");
};

// Byte offset of 16-byte chunk c of key r in a group of 16 keys. Chunks are permuted
// within 128-byte lines so that both fragment loads (K: 8 lanes on 2 keys, V: lanes on
// keys 0, 2, 4, 6) touch every bank once.
template <int HD>
__device__ __forceinline__ int chunk_at(int r, int c) {
  if constexpr (HD >= 128) {
    const int x = (r & 6) ^ ((r & 1) << 2);
    return r * HD + (c ^ x) * 16;  // x < 8 permutes inside lines of 8 chunks
  } else if constexpr (HD == 64) {
    const int line = r >> 1, i = (r & 1) * 4 + c;
    return line * 128 + (i ^ (2 * (line & 3))) * 16;
  } else {
    const int line = r >> 2, i = (r & 3) * 2 + c;
    return line * 128 + (i ^ (2 * (line & 1))) * 16;
  }
}

// A sequence's key tiles: those of the first `sinks` positions, then from the window's
// start (all of them without a window). A sequence with new tokens has one at least, seen
// or not, so that every row is written.
struct Span {
  int n;      // key tiles
  int n_sink;  // the first ones, counted from tile 0
  int skip;   // tile number minus index after them
};
template <int TK>
__device__ __forceinline__ Span key_span(const Seq &s, int window, int sinks) {
  Span p = {max((s.len + TK - 1) / TK, 1), 0, 0};
  if (window) {
    const int lo = max(s.len - s.n - window + 1, 0) / TK;  // tile of the first position in a window
    p.n_sink = min((min(sinks, s.len) + TK - 1) / TK, lo);
    p.skip = lo - p.n_sink;
    p.n -= p.skip;
  }
  return p;
}

template <class C, typename T>
__global__ void __launch_bounds__(THREADS, C::BLOCKS) k_paged_few(const AttnArgs<T> a) {
  constexpr int HD = C::HD, NT = C::NT, TK = C::TK, NG = C::NG, KS = C::KS, ROWS = C::ROWS, TERMS = C::TERMS, SNAP = C::SNAP;
  constexpr bool SPLIT = C::SPLIT;
  constexpr int MT = HD / 16;  // 16-dimension tiles of the output
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ int s_scan[WARPS + 1];
  __shared__ int s_end[2];
  __shared__ int s_last;
  __shared__ float s_sum[8];
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5, g = lane >> 2, t = lane & 3;
  const Cache &c = a.c;
  const int rows_of_token = a.group;
  pdl_wait();  // the batch, q and the cache come from earlier kernels
  pdl_trigger();

  auto tiles_of = [&](const Seq &s) -> int {
    if (!s.n || s.n * rows_of_token > a.few_rows) return 0;
    const int rt = (s.n * rows_of_token + ROWS - 1) / ROWS;
    return (key_span<TK>(s, a.window, a.sinks).n + JOB_COST) * rt * c.kv_heads;
  };
  // This block's piece [at, end) of the line of all tiles, and the sequence it starts in.
  const int first_n = tid < a.b.n_seqs ? tiles_of(load_seq(a.b, c, tid)) : 0;
  unsigned sum = first_n;
  for (int b = tid + THREADS; b < a.b.n_seqs; b += THREADS) sum = line_add(sum, tiles_of(load_seq(a.b, c, b)));
  sum = line_sum(sum);
  if (lane == 0) s_scan[wid] = (int)sum;
  if (tid < 2) s_end[tid] = -1;
  __syncthreads();
  const int total = line_total<WARPS>(s_scan, a.b.err);
  const int per = max((total + (int)gridDim.x - 1) / (int)gridDim.x, MIN_TILES);
  if (per * (int)blockIdx.x >= total) return;
  {
    int before = 0;  // tiles of the sequences before b0
#pragma unroll 1
    for (int b0 = 0; b0 < a.b.n_seqs; b0 += THREADS) {
      const int b = b0 + tid;
      int n = first_n, n_span = 0;
      if (b < a.b.n_seqs) {
        const Seq s = load_seq(a.b, c, b);
        n = tiles_of(s);
        n_span = key_span<TK>(s, a.window, a.sinks).n;
      } else {
        n = 0;
      }
      int run = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, run, o);
        if (lane >= o) run += y;
      }
      __syncthreads();
      if (lane == 31) s_scan[wid] = run;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < WARPS; w++) {
        if (w == wid) run += before;
        before += s_scan[w];
      }
      const int start = run - n;
#pragma unroll
      for (int i = 0; i < 2; i++) {  // this piece's start and the next one's
        const int x = per * ((int)blockIdx.x + i);
        if (x >= start && x < run) {  // one thread at most
          const int in_row_tile = (x - start) % (n_span + JOB_COST);
          s_end[i] = in_row_tile <= SNAP && in_row_tile <= n_span - in_row_tile ? x - in_row_tile
                     : n_span - in_row_tile <= SNAP                             ? x - in_row_tile + n_span + JOB_COST
                                                                                : x;
          if (i == 0) {
            s_last = b;
            s_scan[WARPS] = start;
          }
        }
      }
      if (before > per * ((int)blockIdx.x + 1)) break;
    }
    __syncthreads();
  }
  int at = s_end[0];
  const int end = s_end[1] < 0 ? total : s_end[1];
  if (at >= end) return;
  int b = s_last;                      // its sequence, or the one before where `at` moved to its end
  int b_start = s_scan[WARPS];  // first tile of sequence b
  __syncthreads();

  const uint32_t my_ring = smem_addr(ring) + wid * (STAGES * 2 * C::TILE);
  while (at < end) {
    Seq s = load_seq(a.b, c, b);
    int n_b = tiles_of(s);
    while (at >= b_start + n_b) {  // sequences without new tokens or positions hold no tiles
      b_start += n_b;
      s = load_seq(a.b, c, ++b);
      n_b = tiles_of(s);
    }
    const Span span = key_span<TK>(s, a.window, a.sinks);
    const int row_tiles = (s.n * rows_of_token + ROWS - 1) / ROWS;
    const int slots = span.n + JOB_COST, job = (at - b_start) / slots, head = job / row_tiles, rt = job - head * row_tiles;
    const int job_start = b_start + job * slots;
    const int t0 = at - job_start, t1 = min(span.n, end - job_start);
    const int pos0 = s.len - s.n;  // position of the first new token

    const int last_row = min((rt + 1) * ROWS, s.n * rows_of_token) - 1;
    const int min_pos = pos0 + rt * ROWS / rows_of_token, max_pos = pos0 + last_row / rows_of_token;

    float o[MT][NT][4], m[NT][2], l[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
#pragma unroll
      for (int j = 0; j < 2; j++) m[nt][j] = -INFINITY, l[nt][j] = 0.f;
#pragma unroll
      for (int mt = 0; mt < MT; mt++)
#pragma unroll
        for (int i = 0; i < 4; i++) o[mt][nt][i] = 0.f;
    }
    // f32 rows: sums[i][lane] += o every few tiles; `late` is what they have still to be multiplied by
    float *sums = reinterpret_cast<float *>(ring + C::RING) + wid * (32 * MT * NT * 4) + lane;
    float late[NT][2];
    if constexpr (SPLIT) {
#pragma unroll
      for (int nt = 0; nt < NT; nt++) late[nt][0] = late[nt][1] = 1.f;
#pragma unroll
      for (int i = 0; i < MT * NT * 4; i++) sums[i * 32] = 0.f;
    }
    auto flush = [&]() {
#pragma unroll
      for (int mt = 0; mt < MT; mt++)
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
          for (int i = 0; i < 4; i++) {
            float *p = sums + ((mt * NT + nt) * 4 + i) * 32;
            *p = fmaf(*p, late[nt][i & 1], o[mt][nt][i]);
            o[mt][nt][i] = 0.f;
          }
#pragma unroll
      for (int nt = 0; nt < NT; nt++) late[nt][0] = late[nt][1] = 1.f;
    };

    // ---- this warp's key tiles: the k-th is t0 + wid + k WARPS. Lane NG q + j of a batch of tiles holds the place (in
    // groups of 16 keys; -1: none) and the scales of group j of its tile q. A batch's table entries are loaded a batch
    // ahead, its scales half a batch ahead.
    auto tile_key = [&](int k) {
      const int i = t0 + wid + k * WARPS;
      return (i < span.n_sink ? i : i + span.skip) * TK;
    };
    const int n_tiles = t1 - t0 > wid ? (t1 - t0 - wid + WARPS - 1) / WARPS : 0;
    constexpr int BATCH = C::BATCH;
    const int low = a.window ? min_pos - a.window - 15 : -1;  // groups from there on are in a row's window
    auto entry_of = [&](int batch) {  // INT_MIN: no such group, or none that a row sees
      const int k = batch * BATCH + lane / NG, key = tile_key(k) + 16 * (lane % NG);
      if (k >= n_tiles || key >= s.len || (key <= low && key >= a.sinks)) return INT_MIN;
      return a.b.table[(long long)b * a.b.table_row + (key >> c.page_shift)];
    };
    auto place_of = [&](int batch, int entry) {
      if ((unsigned)entry >= (unsigned)c.n_pages) {
        if (entry != INT_MIN) flag(a.b.err, BAD_PAGE);
        return -1;
      }
      const int key = tile_key(batch * BATCH + lane / NG) + 16 * (lane % NG);
      return ((entry * c.kv_heads + head) << (c.page_shift - 4)) + ((key & (c.page - 1)) >> 4);
    };
    auto scale_of = [&](const float *scales, int place) { return place < 0 ? 0.f : scales[place >> (c.page_shift - 4)]; };
    // 16-byte pieces of a group of 16 keys: lane + 32 k, at lane_at(k) in the group's room in shared memory.
    auto lane_at = [&](int k) { return chunk_at<HD>((k * 32 + lane) / (HD / 16), (k * 32 + lane) % (HD / 16)); };
    const uint8_t *my_k = c.k + lane * 16, *my_v = c.v + lane * 16;
    auto load_tile = [&](int k, int place, int stage) {  // `place`: of the tile's batch
      if (k < n_tiles) {
        const uint32_t dst = my_ring + stage * (2 * C::TILE);
#pragma unroll
        for (int j = 0; j < NG; j++) {
          const int p = __shfl_sync(0xffffffffu, place, k % BATCH * NG + j);
          if (p < 0) continue;
          const uint8_t *ksrc = my_k + (long long)p * (16 * HD), *vsrc = my_v + (long long)p * (16 * HD);
#pragma unroll
          for (int q = 0; q < HD / 32; q++) {
            cp16(dst + j * 16 * HD + lane_at(q), ksrc + q * 512);
            cp16(dst + j * 16 * HD + lane_at(q) + C::TILE, vsrc + q * 512);
          }
        }
      }
      cp_commit();
    };
    int place = place_of(0, entry_of(0)), entry = entry_of(1), next_place = -1;
    float ks = scale_of(c.ks, place), vs = scale_of(c.vs, place), next_ks = 0.f, next_vs = 0.f, v_inv = 0.f, v_man = 0.f;
    int st = 0, v_top = V_EXP_MIN;
    if constexpr (BATCH >= STAGES) {
#pragma unroll
      for (int k = 0; k < STAGES; k++) load_tile(k, place, k);
    }
    // ---- query fragments (the first tiles are on their way): column g of tile nt = row 8 nt + g
    uint32_t qf[NT][KS][TERMS][2];
    float cf[NT][2], cb[NT][2];  // factor of the scores of the lane's columns 2t, 2t + 1, offset before it
    int pos[NT][2];              // and their rows' positions (-1: no such row)
    float4 qx[NT][KS];           // the lane's dimensions: 16 consecutive ones of each 64 (8 of 32)
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
      const int r = rt * ROWS + nt * 8 + g, tok = r / rows_of_token, h = r - tok * rows_of_token;
      const bool ok = tok < s.n;
      const T *src = a.q + (s.first + (ok ? tok : 0)) * a.qs + (head * rows_of_token + (ok ? h : 0)) * HD;
#pragma unroll
      for (int i = 0; i < KS; i++)
        qx[nt][i] = ok ? load4(src + (HD >= 64 ? (i >> 2) * 64 + t * 16 + (i & 3) * 4 : t * 8 + i * 4))
                       : make_float4(0.f, 0.f, 0.f, 0.f);
    }
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
      const int tok = (rt * ROWS + nt * 8 + g) / rows_of_token;
      const bool ok = tok < s.n;
      float x[KS * 4];
      float top = 0.f;
      bool finite = true;
#pragma unroll
      for (int i = 0; i < KS; i++)
        x[4 * i] = qx[nt][i].x, x[4 * i + 1] = qx[nt][i].y, x[4 * i + 2] = qx[nt][i].z, x[4 * i + 3] = qx[nt][i].w;
#pragma unroll
      for (int i = 0; i < KS * 4; i++) {
        top = fmaxf(top, fabsf(x[i]));
        finite &= fabsf(x[i]) <= FLT_MAX;
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      finite = (__ballot_sync(0xffffffffu, finite) >> (lane & 28) & 15) == 15;  // of the row's four lanes
      const int e = row_exp(top);
      const float up = row_factor(e, finite);
      const float down = scalbnf(a.scale, -e);
      float sum = 0.f;  // of the row, for the bias of the codes
#pragma unroll
      for (int i = 0; i < KS; i++) {
#pragma unroll
        for (int j = 0; j < 2; j++) {  // dimensions 4 i + j and 4 i + j + 2: bytes of a word two apart
          const float u = x[4 * i + j] * up, v = x[4 * i + j + 2] * up;
          qf[nt][i][0][j] = pack(u, v);
          const float2 hi = unpack(qf[nt][i][0][j]);
          if constexpr (SPLIT) qf[nt][i][1][j] = pack(u - hi.x, v - hi.y);
          else sum += hi.x + hi.y;
        }
      }
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
#pragma unroll
      for (int j = 0; j < 2; j++) {  // row 2t + j is held by the lanes of g = 2t + j
        const int from = (2 * t + j) * 4;
        const float d = __shfl_sync(0xffffffffu, down, from), q = __shfl_sync(0xffffffffu, sum, from);
        cf[nt][j] = d;
        cb[nt][j] = SPLIT ? 0.f : -128.f * q;
        pos[nt][j] = __shfl_sync(0xffffffffu, ok ? pos0 + tok : -1, from);
      }
    }
#pragma unroll 1
    for (int k = 0; k < n_tiles; k++, st ^= 1) {
      const int in_batch = k % BATCH;
      if (in_batch == 0) {
        if (k) place = next_place, ks = next_ks, vs = next_vs, entry = entry_of(k / BATCH + 1);
        const int e = v_exp(vs);
        v_top = max(v_top, __reduce_max_sync(0xffffffffu, e));
        v_inv = exp_inv(max(e, v_top - V_EXP_SPAN));
        v_man = vs * v_inv;
      }
      if (in_batch == BATCH / 2) {
        next_place = place_of(k / BATCH + 1, entry);
        next_ks = scale_of(c.ks, next_place);
        next_vs = scale_of(c.vs, next_place);
      }
      cp_wait<STAGES - 1>();
      __syncwarp();
      const int key0 = tile_key(k);
      const uint32_t kt = my_ring + st * (2 * C::TILE), vt = kt + C::TILE;

      // scores
      float sc[NG][NT][4];
#pragma unroll
      for (int j = 0; j < NG; j++) {
        float second[NT][4];  // of the second terms
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
          for (int x = 0; x < 4; x++) sc[j][nt][x] = second[nt][x] = 0.f;
        const uint32_t base = kt + j * 16 * HD;
        auto step = [&](uint32_t u, uint32_t w, int i) {  // 16 dimensions
          const uint32_t f[4] = {codes_02<SPLIT>(u), codes_02<SPLIT>(w), codes_13<SPLIT>(u), codes_13<SPLIT>(w)};
#pragma unroll
          for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int y = 0; y < TERMS; y++) mma(y ? second[nt] : sc[j][nt], f, qf[nt][i][y][0], qf[nt][i][y][1]);
        };
        if constexpr (HD >= 64) {
#pragma unroll
          for (int ch = 0; ch < HD / 64; ch++) {
            const uint4 u = lds128(base + chunk_at<HD>(g, ch * 4 + t)), w = lds128(base + chunk_at<HD>(g + 8, ch * 4 + t));
            step(u.x, w.x, ch * 4), step(u.y, w.y, ch * 4 + 1), step(u.z, w.z, ch * 4 + 2), step(u.w, w.w, ch * 4 + 3);
          }
        } else {
          const uint2 u = lds64(base + chunk_at<HD>(g, t >> 1) + (t & 1) * 8);
          const uint2 w = lds64(base + chunk_at<HD>(g + 8, t >> 1) + (t & 1) * 8);
          step(u.x, w.x, 0), step(u.y, w.y, 1);
        }
        if constexpr (SPLIT) {
#pragma unroll
          for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int x = 0; x < 4; x++) sc[j][nt][x] += second[nt][x];
        }
      }
      // in log2 units, with the exponents of the V scales
      float g_inv[NG];
#pragma unroll
      for (int j = 0; j < NG; j++) {
        const float gks = __shfl_sync(0xffffffffu, ks, in_batch * NG + j);
        g_inv[j] = __shfl_sync(0xffffffffu, v_inv, in_batch * NG + j);
        const float e = (float)(127 - (int)(__float_as_uint(g_inv[j]) >> 23));
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
          float f0 = cf[nt][0] * gks, f1 = cf[nt][1] * gks;
          const float b0 = SPLIT ? e : fmaf(cb[nt][0], f0, e), b1 = SPLIT ? e : fmaf(cb[nt][1], f1, e);
          if (!SPLIT) f0 *= 16777216.f, f1 *= 16777216.f;  // after the K scale: large rows have finite scores too
#pragma unroll
          for (int x = 0; x < 4; x++) sc[j][nt][x] = fmaf(sc[j][nt][x], x & 1 ? f1 : f0, x & 1 ? b1 : b0);
        }
      }
      const unsigned there = __ballot_sync(0xffffffffu, place >= 0) >> (in_batch * NG);
      if (key0 + TK - 1 > min_pos || (a.window && key0 <= max_pos - a.window && key0 + TK > a.sinks) ||
          (there & ((1u << NG) - 1)) != (1u << NG) - 1) {
#pragma unroll
        for (int j = 0; j < NG; j++)
#pragma unroll
          for (int x = 0; x < 4; x++) {
            const int key = key0 + 16 * j + g + (x >> 1) * 8;
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
              const int p = pos[nt][x & 1];
              const bool seen = key <= p && (!a.window || key > p - a.window || key < a.sinks) && (there >> j & 1);
              if (!seen) sc[j][nt][x] = -INFINITY;
            }
          }
      }
      // running maximum; the rows' earlier results move to it
      float corr[NT][2], ref[NT][2];
      bool moved = false;
#pragma unroll
      for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int j = 0; j < 2; j++) {
          float mx = m[nt][j];
#pragma unroll
          for (int x = 0; x < NG; x++) mx = fmaxf(mx, fmaxf(sc[x][nt][j], sc[x][nt][2 + j]));
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
          ref[nt][j] = mx == -INFINITY ? 0.f : mx - WEIGHT_EXP;
          corr[nt][j] = mx == m[nt][j] ? 0.f : m[nt][j] - mx;  // as an exponent
          moved |= corr[nt][j] != 0.f;
          m[nt][j] = mx;
        }
      if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
          const float f0 = ex2(corr[nt][0]), f1 = ex2(corr[nt][1]);  // 0 while nothing was seen
          l[nt][0] = scaled(l[nt][0], corr[nt][0]), l[nt][1] = scaled(l[nt][1], corr[nt][1]);
          if (SPLIT) late[nt][0] *= f0, late[nt][1] *= f1;
#pragma unroll
          for (int mt = 0; mt < MT; mt++) {
            o[mt][nt][0] *= f0, o[mt][nt][1] *= f1, o[mt][nt][2] *= f0, o[mt][nt][3] *= f1;
          }
        }
      }
      // weights, as the operand of the second product
      uint32_t pf[NG][NT][TERMS][2];
#pragma unroll
      for (int j = 0; j < NG; j++) {
        const float g_man = __shfl_sync(0xffffffffu, v_man, in_batch * NG + j);
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
          for (int x = 0; x < 2; x++) {
            float u = ex2(sc[j][nt][2 * x] - ref[nt][0]), v = ex2(sc[j][nt][2 * x + 1] - ref[nt][1]);
            l[nt][0] = fmaf(u, g_inv[j], l[nt][0]);
            l[nt][1] = fmaf(v, g_inv[j], l[nt][1]);
            u *= g_man;
            v *= g_man;
            const uint32_t f = pack(u, v);
            pf[j][nt][0][x] = transpose8x8(f);
            if constexpr (SPLIT) {
              const float2 hi = unpack(f);
              pf[j][nt][1][x] = transpose8x8(pack(u - hi.x, v - hi.y));
            }
          }
      }
      // output
#pragma unroll
      for (int j = 0; j < NG; j++) {
        const uint32_t base = vt + j * 16 * HD;
        constexpr int CH = HD >= 128 ? HD / 128 : 1;  // 16-byte pieces of the lane's dimensions
#pragma unroll
        for (int ch = 0; ch < CH; ch++) {
          constexpr int W = HD >= 128 ? 4 : HD / 32;  // words of a piece
          uint32_t w[4][W];  // keys 2t, 2t + 1, 2t + 8, 2t + 9
#pragma unroll
          for (int k = 0; k < 4; k++) {
            const int r = 2 * t + (k & 1) + (k >> 1) * 8;
            if constexpr (HD >= 128) {
              const uint4 u = lds128(base + chunk_at<HD>(r, ch * 8 + g));
              w[k][0] = u.x, w[k][1] = u.y, w[k][2] = u.z, w[k][3] = u.w;
            } else if constexpr (HD == 64) {
              const uint2 u = lds64(base + chunk_at<HD>(r, g >> 1) + (g & 1) * 8);
              w[k][0] = u.x, w[k][1] = u.y;
            } else {
              w[k][0] = lds32(base + chunk_at<HD>(r, g >> 2) + (g & 3) * 4);
            }
          }
#pragma unroll
          for (int x = 0; x < W; x++)
#pragma unroll
            for (int y = 0; y < 2; y++) {  // dimensions 4x + 2y, 4x + 2y + 1 of the piece
              const uint32_t u = __byte_perm(w[0][x], w[1][x], y ? 0x7362 : 0x5140);
              const uint32_t v = __byte_perm(w[2][x], w[3][x], y ? 0x7362 : 0x5140);
              const uint32_t f[4] = {codes_lo(u), codes_hi(u), codes_lo(v), codes_hi(v)};
#pragma unroll
              for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int z = 0; z < TERMS; z++)
                  mma(o[ch * 2 * W + 2 * x + y][nt], f, pf[j][nt][z][0], pf[j][nt][z][1]);
            }
        }
      }
      __syncwarp();  // every lane has read the stage that is loaded next
      load_tile(k + STAGES, (in_batch + STAGES < BATCH ? place : next_place), st);
      if constexpr (SPLIT) {
        if (k % (FLUSH_STEPS / NG) == FLUSH_STEPS / NG - 1) flush();
      }
    }
    if constexpr (SPLIT) flush();
    cp_wait<0>();
    __syncthreads();

    // ---- the warps' results joined: [warp][row]: maximum, sum, head_dim outputs
    float *mine = reinterpret_cast<float *>(ring) + wid * ROWS * (HD + 2);
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
      for (int j = 0; j < 2; j++) {
        float sum = l[nt][j];
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
        float *dst = mine + (nt * 8 + 2 * t + j) * (HD + 2);
        if (g == 0) *reinterpret_cast<float2 *>(dst) = make_float2(m[nt][j], sum);
#pragma unroll
        for (int mt = 0; mt < MT; mt++) {
          const float *sm = sums + ((mt * NT + nt) * 4 + j) * 32;
          const float2 v = SPLIT ? make_float2(sm[0], sm[64]) : make_float2(o[mt][nt][j], o[mt][nt][2 + j]);
          const int d = HD >= 128 ? (mt / 8) * 128 + g * 16 + (mt % 8) * 2 : g * (HD / 8) + mt * 2;
          *reinterpret_cast<float2 *>(dst + 2 + d) = v;
        }
      }
    __syncthreads();
    const bool whole = t0 == 0 && t1 == span.n;
    const int rows = last_row + 1 - rt * ROWS;
    auto put = [&](int row, int d, float4 v) {
      const int r = rt * ROWS + row, tok = r / rows_of_token, h = r - tok * rows_of_token;
      store4(a.out + (s.first + tok) * a.os + (head * rows_of_token + h) * HD + d, v);
    };
    // A block has two cut row tiles at most: the one its piece starts in (slot 0) and the one it ends in (slot 1).
    auto slot_of = [&](int block, bool first_part) { return a.part + (size_t)(2 * block + first_part) * SLOT_FLOATS; };
    constexpr int QUADS = HD / 4;
    float *slot = slot_of(blockIdx.x, t0 == 0);  // maxima, sums, outputs
    for (int e = tid; e < rows * QUADS; e += THREADS) {
      const int row = e / QUADS, d = e % QUADS * 4;
      const float *src = reinterpret_cast<const float *>(ring) + row * (HD + 2);
      float top = -INFINITY, sum = 0.f;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < WARPS; w++) top = fmaxf(top, src[w * ROWS * (HD + 2)]);
      const float at0 = top == -INFINITY ? 0.f : top;
#pragma unroll
      for (int w = 0; w < WARPS; w++) {
        const float *x = src + w * ROWS * (HD + 2);
        const float f = ex2(x[0] - at0);
        sum += scaled(x[1], x[0] - at0);
        v.x = fmaf(x[2 + d], f, v.x), v.y = fmaf(x[3 + d], f, v.y);
        v.z = fmaf(x[4 + d], f, v.z), v.w = fmaf(x[5 + d], f, v.w);
      }
      if (whole) {
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        put(row, d, sum == 0.f ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
      } else {
        *reinterpret_cast<float4 *>(slot + 2 * ROWS + row * HD + d) = v;
        if (d == 0) {
          slot[row] = top;
          slot[ROWS + row] = sum;
        }
      }
    }
    if (!whole) {
      // The last block to arrive joins all parts, in block order: every part's factors once, to shared memory, then
      // the threads share out rows, dimensions and (when there are few of those) slices of the parts.
      // The cuts are the multiples of `per` more than SNAP tiles inside its keys; the part before the first is the block's before.
      const int first = (job_start + SNAP) / per, parts = (job_start + span.n - SNAP - 1) / per - first + 1;
      int *count = a.count + (long long)(b * c.kv_heads + head) * a.max_row_tiles + rt;
      __syncthreads();
      if (tid == 0) {  // the block's stores before its arrival, the other blocks' arrivals before its loads
        __threadfence();
        s_last = atomicAdd(count, 1) == parts - 1;
        __threadfence();
      }
      __syncthreads();
      if (s_last) {
        auto part = [&](int i) { return slot_of(first + i, i == 0); };
        float *factor = reinterpret_cast<float *>(ring), *share_of = factor + MAX_BLOCKS * 8;  // [row of 8][part]; slices
        for (int r0 = 0; r0 < rows; r0 += 8) {
          const int nr = min(8, rows - r0);
          __syncthreads();
          for (int e = tid; e < nr * parts; e += THREADS) factor[e] = __ldcg(part(e % parts) + r0 + e / parts);
          __syncthreads();
          for (int r = wid; r < nr; r += WARPS) {  // a warp a row: maximum, factors, sum
            float *f = factor + r * parts, top = -INFINITY, sum = 0.f;
            for (int i = lane; i < parts; i += 32) top = fmaxf(top, f[i]);
            top = warp_max(top);
            const float at0 = top == -INFINITY ? 0.f : top;
            for (int i = lane; i < parts; i += 32) {
              const float x = f[i] - at0;
              f[i] = ex2(x);
              sum += scaled(__ldcg(part(i) + ROWS + r0 + r), x);
            }
            sum = warp_sum(sum);
            if (lane == 0) s_sum[r] = sum;
          }
          __syncthreads();
          const int items = nr * QUADS, slices = max(1, THREADS / items);
          for (int e0 = 0; e0 < items; e0 += THREADS) {
            const int item = slices > 1 ? tid % items : e0 + tid, slice = slices > 1 ? tid / items : 0;
            const int row = item / QUADS, d = item % QUADS * 4;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            if (item < items && slice < slices) {
              const float *f = factor + row * parts;
#pragma unroll 8
              for (int i = slice; i < parts; i += slices) {
                const float4 x = __ldcg(reinterpret_cast<const float4 *>(part(i) + 2 * ROWS + (r0 + row) * HD + d));
                const float y = f[i];
                v.x = fmaf(x.x, y, v.x), v.y = fmaf(x.y, y, v.y), v.z = fmaf(x.z, y, v.z), v.w = fmaf(x.w, y, v.w);
              }
              if (slice) *reinterpret_cast<float4 *>(share_of + 4 * tid) = v;
            }
            if (slices > 1) __syncthreads();
            if (item < items && slice == 0) {
              for (int i = 1; i < slices; i++) {
                const float4 x = *reinterpret_cast<const float4 *>(share_of + 4 * (tid + i * items));
                v.x += x.x, v.y += x.y, v.z += x.z, v.w += x.w;
              }
              const float sum = s_sum[row], inv = sum == 0.f ? 0.f : 1.f / sum;
              put(r0 + row, d,
                  sum == 0.f ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
            }
          }
        }
        if (tid == 0) *count = 0;
      }
    }
    at = t1 < span.n ? end : job_start + slots;
    __syncthreads();  // the ring is free again
  }
}

template <class C, typename T>
cudaError_t launch(cudaStream_t s, AttnArgs<T> &a) {
  static int blocks[64] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev >= 64) return cudaErrorInvalidDevice;
  if (!blocks[dev]) {
    int sms = 0, per_sm = 0;
    if ((e = cudaFuncSetAttribute(k_paged_few<C, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM)) !=
            cudaSuccess ||
        (e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev)) != cudaSuccess ||
        (e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, k_paged_few<C, T>, THREADS, C::SMEM)) !=
            cudaSuccess)
      return e;
    blocks[dev] = min(sms * max(per_sm, 1), MAX_BLOCKS);
  }
  a.max_row_tiles = (min(a.b.max_new * a.group, a.few_rows) + C::ROWS - 1) / C::ROWS;
  return launch_ex(k_paged_few<C, T>, dim3(blocks[dev]), dim3(THREADS), C::SMEM, s, pdl_enabled(), a);
}

// As few row tiles as the registers allow (8 rows and head_dim 256, 16 and 128, 32 below), and those as narrow as
// takes all rows.
template <typename T, int HD>
cudaError_t launch_few(cudaStream_t s, AttnArgs<T> &a) {
  const int rows = min(a.b.max_new * a.group, a.few_rows);
  constexpr int MOST = HD == 256 ? 1 : HD == 128 ? 2 : 4;
  const int tiles = (rows + 8 * MOST - 1) / (8 * MOST), nt = ((rows + tiles - 1) / tiles + 7) / 8;
  if (nt == 1) return launch<Cfg<T, HD, 1>>(s, a);
  if constexpr (MOST >= 2) {
    if (nt == 2) return launch<Cfg<T, HD, 2>>(s, a);
  }
  if constexpr (MOST == 4) return nt == 3 ? launch<Cfg<T, HD, 3>>(s, a) : launch<Cfg<T, HD, 4>>(s, a);
  return cudaErrorInvalidValue;
}

// Query rows a kv head. A call of up to ALONE_ROWS is this kernel's: 12 x up to 4,096 positions, this one / the other at
// 72 rows: f32 58 / 65 us (64 dimensions), 86 / 105 us (128), bf16 43 / 50 and 69 / 66 us; at 80 rows 73 / 65, 89 / 105,
// 53 / 50, 72 / 66: one number for all, 3 us late for bf16 of 128 dimensions, 16 us early for f32 of 128. Beyond, the other kernel takes the sequences of more than FEW_ROWS and this one the rest, one after
// the other: where all are long FEW_ROWS would only leave work for a second launch (a ragged batch of up to 96 rows:
// 16 or 32: 64 us, 48: 86, 64: 103), and single and drafted tokens beside prompts stay here.
constexpr int ALONE_ROWS = 72, FEW_ROWS = 32;

bool goes_many(const Cache &c, int max_new, int group) {
  return (long long)max_new * group > ALONE_ROWS && many_supported(c, group);
}

// Whether the (row tile, key tile) pairs of a call can be numbered below LINE_END by both kernels: 128 rows or
// more a tile and 64 keys for the many-row one, 4 rows and 16 keys at least for the other.
bool countable(const Batch &b, const Cache &c, int n_heads) {
  const int group = n_heads / c.kv_heads;
  const bool many = goes_many(c, b.max_new, group);
  const double keys = (double)b.table_row * c.page, tokens = b.n_tokens, seqs = b.n_seqs;
  const double few = many ? seqs * (FEW_ROWS / 4) : tokens * group / 4 + seqs;
  const double rest = many ? (tokens * group / 128 + seqs) * (keys / 64 + 16) : 0;
  return few * c.kv_heads * (keys / 16 + 32) < LINE_END && rest * c.kv_heads < LINE_END;
}

// Partial results of both kernels, then the counters of both.
struct Workspace {
  size_t many_part, few_count, many_count, bytes;
};
Workspace workspace(const Batch &b, const Cache &c, int n_heads) {
  const int group = n_heads / c.kv_heads;
  const bool many = goes_many(c, b.max_new, group);
  const size_t jobs = (size_t)b.n_seqs * c.kv_heads;
  const long long rows = many ? FEW_ROWS : (long long)b.max_new * group;
  Workspace w;
  w.many_part = PARTIAL_BYTES;
  w.few_count = w.many_part + (many ? many_partial_bytes(c.hd) : 0);
  w.many_count = w.few_count + jobs * ((rows + 7) / 8) * sizeof(int);  // row tiles have 8 rows at least
  w.bytes = w.many_count + (many ? jobs * many_row_tiles(b.max_new, group) * sizeof(int) : 0);
  return w;
}

template <typename T>
cudaError_t attention(cudaStream_t s, const Cache &c, const Batch &b, const void *q, long long qs, int n_heads,
                      float scale, int window, int sinks, void *out, long long os, void *ws) {
  const Workspace w = workspace(b, c, n_heads);
  uint8_t *p = (uint8_t *)ws;
  AttnArgs<T> a = {c,      b,     (const T *)q, (T *)out,  qs,      os, n_heads, n_heads / c.kv_heads, scale * LOG2E,
                   window, sinks, INT32_MAX,    (float *)p, (int *)(p + w.few_count), 0, 0};
  if (goes_many(c, b.max_new, a.group)) {
    AttnArgs<T> m = a;
    a.few_rows = m.few_rows = FEW_ROWS;
    m.part = (float *)(p + w.many_part);
    m.count = (int *)(p + w.many_count);
    const cudaError_t e = launch_many(s, m);
    // all sequences bring as many tokens as the longest: none is left for the other kernel
    if (e != cudaSuccess || (long long)b.max_new * b.n_seqs == b.n_tokens) return e;
  }
  switch (c.hd) {
    case 32: return launch_few<T, 32>(s, a);
    case 64: return launch_few<T, 64>(s, a);
    case 128: return launch_few<T, 128>(s, a);
    default: return launch_few<T, 256>(s, a);
  }
}

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
  if (!st) st = paged::check_batch(batch, c, &b, "paged_attention_workspace");
  if (!st && !bytes) st = fail(SQ_ERR_ARG, "paged_attention_workspace: null pointer");
  if (!st) st = paged::check_heads(c, n_heads, "paged_attention_workspace");
  if (st) return st;
  *bytes = paged::workspace(b, c, n_heads).bytes;
  return SQ_OK;
}

extern "C" int sq_paged_attention(void *stream, const sq_paged_cache *cache, const sq_paged_batch *batch, int dtype,
                                  const void *q, long long q_stride, int n_heads, float scale, int window, int sinks,
                                  void *out, long long out_stride, void *ws, size_t ws_bytes) {
  paged::Cache c;
  paged::Batch b;
  int st = paged::check_cache(cache, &c, "paged_attention");
  if (!st) st = paged::check_batch(batch, c, &b, "paged_attention");
  if (!st) st = paged::check_heads(c, n_heads, "paged_attention");
  if (st) return st;
  if (dtype != SQ_F32 && dtype != SQ_BF16)
    return fail(SQ_ERR_INVALID_TYPE, "paged_attention: rows must be F32 or BF16");
  if (window < 0 || sinks < 0) return fail(SQ_ERR_SHAPE, "paged_attention: negative window or sinks");
  if (!paged::countable(b, c, n_heads))
    return fail(SQ_ERR_SHAPE, "paged_attention: too many query rows for so long a page table in one call");
  if (!b.n_tokens) return SQ_OK;
  // a window that holds every position of the page table hides none; the kernels' sums with it fit 32 bits
  if (window >= (long long)b.table_row * c.page) window = 0;
  const long long width = (long long)n_heads * c.hd;
  st = paged::check_rows(q, q_stride, width, dtype, "paged_attention: q");
  if (!st) st = paged::check_rows(out, out_stride, width, dtype, "paged_attention: out");
  if (st) return st;
  if (!ws || ws_bytes < paged::workspace(b, c, n_heads).bytes)
    return fail(SQ_ERR_ARG, "paged_attention: the workspace is smaller than paged_attention_workspace says");
  if ((uintptr_t)ws & 255) return fail(SQ_ERR_ALIGN, "paged_attention: the workspace must be 256-byte aligned");
  if (!(b.err = paged::err_ptr())) return fail(SQ_ERR_CUDA, "paged_attention: no current CUDA device");
  const auto run = dtype == SQ_F32 ? paged::attention<float> : paged::attention<__nv_bfloat16>;
  cudaError_t e = run((cudaStream_t)stream, c, b, q, q_stride, n_heads, scale, window, sinks, out, out_stride, ws);
  return e == cudaSuccess ? SQ_OK : cuda_fail(e, "sq_paged_attention");
}
