// paged_attention_tc.cu — causal grouped attention over the paged 8-bit cache for many query
// rows a kv head (prompts): bound by the products and the exponentials. tcgen05, head_dim
// 64 and 128.
//
// A block works on 256 query rows of one kv head (row = token * group + head of the
// group), two tiles X of 128 that share every block of 64 keys, so that a code is
// converted once for 256 rows:
//   warps 8-11  codes of a block of keys, loaded a block ahead to registers and converted
//               to f16 (exact: whole numbers up to 127) into the
//               128-byte swizzled tiles of K [keys][dims] and V [keys][dims]
//   warps 12, 15 issue the products of tile 0 and 1, f32 sums in tensor memory (one warp for both spent
//               a third of its time on waits and commits between them):
//               S_X = Q_X K^T (K-major operands), O_X (+)= P_X V (V read MN-major as it
//               lies, P from tensor memory). A tile's scores have two buffers: those of
//               block j + 2 are issued right after P V of block j, so the softmax finds
//               the next block's scores ready (two blocks' scores in one product of 128
//               columns take a third less tensor time, but leave no second buffer: 694
//               -> 838 us for 2 x 4,096 rows of 8,000 positions, bf16, 128 dimensions)
//   warp 13     walks this block's share of the work, handed out piece by piece
//   warp 14     looks up pages and scales, eight blocks of keys at a time
//   warps 0-7   one thread a row (= tensor-memory lane): running maximum of its scores,
//               weights over the columns the scores leave, sum
// Loops are rolled where registers allow: with blocks of 128 keys in unrolled code (200
// KB) every role spent its time waiting for instructions.
//
// Precision, as in the few-row kernel: query rows scaled by powers of two, two f16 terms
// for f32 rows, one (exact) for bf16 rows. Scores s take the V scales' exponents on, weights are
// 2^(s - ref + 3), and ref follows the maximum only when it is passed by 2^6, so that f16 never overflows, loses
// no page with small values beside one with large ones, and outputs are seldom rescaled.
//   f32 rows:  weights in two terms; the O of four blocks of keys is summed in tensor memory and
//              added to f32 registers, because the tensor core truncates its running sum
//              (2^-25 of it a step: 500 steps would cost 1e-5). 2048 x 4,133 positions, 128
//              dimensions: every block 331 us (error 4.5e-7 of the result), every four 269 us
//              (7.5e-7), every eight 258 us (1.2e-6; the plain f32 form: 1.4e-6). With the V scales'
//              exponents in the scores every four takes 275 us (8.0e-7); a row's 128 sums leave too few
//              registers there (288 bytes of a thread's spill, 24 and less in the other forms).
//   bf16 rows: weights in one term (11 bits, under the output's 8); O stays in tensor memory.
//
// Work is split as in the few-row kernel: one line of (sequence, kv head, row tile, key
// block), an equal piece for every block, cut row tiles joined by the last block to arrive.
// Every wait is bounded: on expiry the block records it, stops, lets its products and
// copies finish, frees its tensor memory and returns.
#include <cuda.h>
#include <float.h>
#include <stdlib.h>

#include <atomic>

#include "ops.cuh"
#include "paged_attention.cuh"
#include "tc.cuh"

namespace sq {
namespace paged {
namespace {

using namespace tc;

constexpr int SOFTMAX_WARPS = 8, LOAD_WARPS = 4, MMA_WARP = SOFTMAX_WARPS + LOAD_WARPS;
constexpr int WARPS = 16;  // whole warpgroups: registers are shared out by them
constexpr int THREADS = WARPS * 32, LOADERS = LOAD_WARPS * 32;
constexpr int TILE_ROWS = 128, ROWS = 2 * TILE_ROWS;
constexpr int BATCH = 8, BATCHES = 2;  // blocks of keys looked up at once, and how many such batches are held
constexpr int PLAN_BYTES = 96;
constexpr int MAX_BLOCKS = 160;
// What a row tile costs besides its key blocks, in blocks (queries in, results out, the pipeline's start and end), when
// the work is shared out. 0 / 3 / 5 / 8 (bf16, 128 dimensions): 2 x 4,096 rows of 8,000 positions 776 / 718 /
// 696 / 696 us, 16 x 1,000 rows 260 / 222 / 213 / 218 us, 64 x 100 rows of 300 positions 136 / 105 / 101 / 102 us.
constexpr int TILE_COST = 5;
constexpr int MIN_BLOCKS = 2;  // key blocks a thread block takes at least
constexpr int MOVE = 4;        // f32 rows: blocks of keys summed in tensor memory at a stretch
constexpr float WEIGHT_EXP = 3.f, REF_LAG = 6.f, LARGE_SCORE = 4194304.f;
// Registers a thread: launched with 128 (512 x 128 = 65,536), then 256 x 184 + 128 x 80 + 128 x 64.
constexpr int SOFTMAX_REGS = 184, LOAD_REGS = 80, MMA_REGS = 64;

template <typename T, int HD_>
struct Cfg {
  static constexpr int HD = HD_;
  static constexpr bool SPLIT = sizeof(T) == 4;
  static constexpr int TERMS = SPLIT ? 2 : 1;
  static constexpr int BK = 64;                             // keys a block
  static constexpr int STAGES = SPLIT && HD == 128 ? 2 : 4;  // of K and V each
  static constexpr int NG = BK / 16;                        // groups of 16 keys: each within one page
  static constexpr int PANELS = HD / 64;                    // 64 dimensions = 128 bytes of f16
  static constexpr int Q_PANEL = TILE_ROWS * 128, KV_PANEL = BK * 128;
  static constexpr int Q_TILE = PANELS * Q_PANEL, KV_TILE = PANELS * KV_PANEL;
  static constexpr int ROW_CHUNKS = HD / 16;                      // 16-code chunks of a key
  static constexpr int STEP_ROWS = LOADERS / ROW_CHUNKS;          // keys the loading threads take at once: 16 or 32
  static constexpr int STEPS = BK / STEP_ROWS;
  static constexpr int OFF_Q = 0, OFF_K = OFF_Q + 2 * TERMS * Q_TILE, OFF_V = OFF_K + STAGES * KV_TILE,
                       OFF_SCALE = OFF_V + STAGES * KV_TILE,
                       OFF_BAR = OFF_SCALE + BATCHES * BATCH * PLAN_BYTES;
  static constexpr int SMEM = 1024 + OFF_BAR + 368;
  static constexpr int SLOT = ROWS * (HD + 2);  // floats of a cut row tile's partial result
  static_assert(SMEM <= 232448 - 256, "shared memory of a block");
};

// What is looked up for a block of 64 keys: of its four groups of 16 the place in the
// codes (in groups of 16 keys; -1: none), the K scale, the V scale 2^exp * man (f32 rows: exp is a whole
// number; bf16 rows: man is 1) and 2^-exp.
struct Plan {
  int place[4];
  float ks[4], exp[4], inv[4], man[4];
  uint32_t present, with_v;  // bit masks of groups: there at all; with a V scale that counts
  uint32_t pad[2];
};
static_assert(sizeof(Plan) == PLAN_BYTES, "room in shared memory");

constexpr int MAX_STAGES = 4;
// A wait tells a phase from the one before it only. So every barrier is one whose phase before is known to be done
// when a phase is waited for, and whose phase after cannot be: where a waiter may skip phases or lag behind, there
// is one for each buffer or place. Nothing else waits for tile 1's product warp in a piece that leaves tile 1
// without rows, so a piece is done, and its place and B_Q used again, only with that warp's arrival too.
enum : int {
  B_Q = 0,        // [4] both tiles' queries of a piece written
  B_K = 4,        // [stages] K written
  B_K_FREE = 8,   // [stages] scores of both tiles done
  B_V = 12,       // [stages]
  B_V_FREE = 16,  // [stages]
  B_S = 20,       // [2 tiles][2 buffers] scores done
  B_P = 24,       // [2 tiles][2 buffers] weights written
  B_PV = 28,      // [2 tiles][2 buffers] P V done
  B_PIECE = 32,   // [4] a piece handed out
  B_DONE = 36,    // [4] a piece's rows written, and tile 1's products issued
  B_PLAN = 40,    // [2] a batch of blocks looked up
  B_PLAN_FREE = 42,
  B_FIN = 44,
  N_BARS = 45
};
static_assert(8 * N_BARS <= 368, "room in shared memory");
// Columns: S, and P over it, of tile X and buffer B at 128 X + 64 B (P: first terms in 32, second terms
// in the next 32); O at 256 + 128 X.
constexpr uint32_t TM_O = 256, TM_COLS = 512;

// f16 operands, f32 sums; B K-major or (bit 16) MN-major.
constexpr uint32_t idesc_f16(int M, int N, bool b_mn) {
  return (1u << 4) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
// Descriptor of an MN-major operand in the 128-byte swizzled layout: a row of 128 bytes
// holds 64 consecutive MN elements of one K index, 8 rows (1,024 bytes) a swizzle atom,
// atoms of the next 8 K indices 1,024 bytes on (stride offset), the next 64 MN elements
// `panel` bytes on (leading offset).
__device__ __forceinline__ uint64_t mn_desc(uint32_t saddr, uint32_t panel) {
  return (uint64_t)((saddr & 0x3FFFFu) >> 4) | ((uint64_t)(panel >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
__device__ __forceinline__ void tmem_ld32(uint32_t a, float *v) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(a));
#pragma unroll
  for (int i = 0; i < 32; i++) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tmem_st32(uint32_t a, const uint32_t *r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(a),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r != 0;
}
// D[tmem] (+)= A B with A from shared memory, or from tensor memory (_ts).
__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)
      : "memory");
}
__device__ __forceinline__ void mma_f16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)
      : "memory");
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ uint32_t bf16_pair(float a, float b) {
  const __nv_bfloat162 x = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&x);
}
// Orders the uses of N loaded registers after the wait for them.
template <int N>
__device__ __forceinline__ void tmem_ready(float *v) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < N; i++) asm volatile("" : "+f"(v[i]));
}
__device__ __forceinline__ void sts128(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}

// Sum over i < n of floor((a i + b) / m), by Euclid's steps. It fits 32 bits for the row tiles of a sequence
// that has no more new tokens than positions: the host refuses calls whose line of key blocks would not.
__device__ __forceinline__ int floor_sum(unsigned n, unsigned m, unsigned a, unsigned b) {
  unsigned sum = 0;
  while (n) {
    if (a >= m) {
      sum += n * (n - 1) / 2 * (a / m);
      a %= m;
    }
    if (b >= m) {
      sum += n * (b / m);
      b %= m;
    }
    const unsigned y = a * n + b;
    if (y < m) break;
    n = y / m;
    b = y % m;
    const unsigned x = m;
    m = a;
    a = x;
  }
  return sum;
}

// Places of a sequence's row tiles on the line: key blocks, without a window the causal
// count of each (a little over for the last), with one (and where there are more new tokens
// than positions, whose first rows see nothing) the same for all, and TILE_COST
// more; what a tile does not have of them is empty.
template <int BK>
struct Line {
  int row_tiles, tokens;  // tokens of a row tile
  int flat;               // key blocks of every row tile, or 0
  int pos0, len;
  __device__ __forceinline__ void set(const Seq &s, int group, int window, int sinks, int few_rows) {
    tokens = ROWS / group;
    row_tiles = s.n * group > few_rows ? (s.n + tokens - 1) / tokens : 0;
    pos0 = max(s.len - s.n, 0);
    len = s.len;
    flat = 0;
    if (window && window < s.len)
      flat = min((min(sinks, s.len) + BK - 1) / BK + (window + tokens + BK - 3) / BK + 1, (s.len + BK - 1) / BK);
    else if (s.n > s.len)
      flat = max((s.len + BK - 1) / BK, 1);
  }
  __device__ __forceinline__ int before(int rt) const {  // key blocks of row tiles 0 .. rt - 1
    if (flat) return rt * (flat + TILE_COST);
    return rt * (1 + TILE_COST) + floor_sum(rt, BK, tokens, pos0 + tokens - 1);
  }
  __device__ __forceinline__ int of(int rt) const {
    return (flat ? flat : (pos0 + (rt + 1) * tokens - 1) / BK + 1) + TILE_COST;
  }
};

// One block's part of a row tile.
struct Piece {
  int b, head;
  int row0, n_rows;     // first token's row of the step, query rows in use (token * group + head of the group)
  int pos0, len;        // first token's position; positions held
  int t0, n;            // key blocks t0 .. t0 + n - 1 of the tile (n may be 0; -1: no more pieces)
  int n_sink, skip;     // tile index to block number, as in the few-row kernel
  int whole;
  int slot;             // of the partial results
  int first, parts;     // thread blocks first .. first + parts - 1 share the tile
  int late;             // block `first` began another tile before this one: its second slot
  long long counter;
  __device__ __forceinline__ int block(int i) const { return t0 + i + (t0 + i < n_sink ? 0 : skip); }
};
constexpr int PIECES = 4;

// Walks this thread block's piece of the line.
template <int BK>
struct Walk {
  int at, end, per;
  int seq_start;   // of sequence b on the line
  int tile_start;  // of the row tile (head, rt)
  int b, head, rt;
  bool found;  // the first row tile is looked up, the others follow
  Line<BK> line;
  Seq s;
  int per_head;

  template <typename T>
  __device__ __forceinline__ bool next(const AttnArgs<T> &a, Piece &p) {
#pragma unroll 1
    for (;;) {
      if (at >= end) return false;
      bool other = !found;
      if (found && ++rt == line.row_tiles) {
        rt = 0;
        if (++head == a.c.kv_heads) {
          head = 0;
          other = true;
          b++;
        }
      }
      if (other) {
#pragma unroll 1
        for (;; b++) {  // at < end: a sequence with row tiles follows
          s = load_seq(a.b, a.c, b);
          line.set(s, a.group, a.window, a.sinks, a.few_rows);
          if (line.row_tiles) break;
        }
      }
      if (!found) {
        per_head = line.before(line.row_tiles);
        head = (at - seq_start) / per_head;
        const int in_head = at - seq_start - head * per_head;
        // the row tile that holds in_head: 32 candidates at a time
        rt = 0;
#pragma unroll 1
        for (int width = line.row_tiles; width > 1;) {
          const int step = (width + 31) / 32, mine = rt + (threadIdx.x & 31) * step;
          const unsigned le = __ballot_sync(0xffffffffu, mine < rt + width && line.before(mine) <= in_head);
          const int k = 31 - __clz(le);  // lane 0 always holds
          rt += k * step;
          width = min(step, width - k * step);
        }
        tile_start = seq_start + head * per_head + line.before(rt);
        found = true;
      }
      const int slots = line.of(rt), first_tok = rt * line.tokens, toks = min(line.tokens, s.n - first_tok);
      p.b = b;
      p.head = head;
      p.row0 = s.first + first_tok;
      p.n_rows = toks * a.group;
      p.pos0 = s.len - s.n + first_tok;
      p.len = s.len;
      int real = max(p.pos0 + toks - 1, 0) / BK + 1;
      p.n_sink = p.skip = 0;
      if (a.window && a.window < s.len) {
        const int low = max(p.pos0 - a.window + 1, 0) / BK;
        p.n_sink = min((min(a.sinks, s.len) + BK - 1) / BK, low);
        p.skip = low - p.n_sink;
        real -= p.skip;
      }
      p.t0 = at - tile_start;
      const int t1 = min(slots, end - tile_start);
      p.n = min(t1, real) - p.t0;
      p.whole = p.n == real;
      p.first = tile_start / per;
      p.parts = (tile_start + real - 1) / per - p.first + 1;
      p.late = tile_start > per * p.first;
      p.slot = 2 * blockIdx.x + (tile_start > per * (int)blockIdx.x ? 1 : 0);
      p.counter = (long long)(b * a.c.kv_heads + head) * a.max_row_tiles + rt;
      at = tile_start + t1;
      tile_start += slots;
      if (p.n > 0) return true;
    }
  }
};

template <class C, typename T>
__global__ void __launch_bounds__(THREADS, 1) k_paged_many(const AttnArgs<T> a) {
  constexpr int HD = C::HD, BK = C::BK, NG = C::NG, TERMS = C::TERMS;
  constexpr bool SPLIT = C::SPLIT;
  extern __shared__ uint8_t smem_raw[];
  __shared__ int s_scan[WARPS + 2];
  __shared__ int s_seq, s_abort, s_last;
  __shared__ uint32_t s_tmem;
  __shared__ Piece s_pieces[PIECES];
  const uint32_t base = (smem_addr(smem_raw) + 1023u) & ~1023u;
  uint8_t *gen = smem_raw + (base - smem_addr(smem_raw));
  Plan *plans = reinterpret_cast<Plan *>(gen + C::OFF_SCALE);  // [batch][block]
  constexpr int STAGES = C::STAGES;
  auto bar = [&](int i) { return base + C::OFF_BAR + 8u * (uint32_t)i; };
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const Cache &c = a.c;
  pdl_wait();  // the batch, q and the cache come from earlier kernels
  pdl_trigger();

  // ---- this block's piece of the line
  auto blocks_of = [&](int b) -> int {
    Line<BK> l;
    l.set(load_seq(a.b, c, b), a.group, a.window, a.sinks, a.few_rows);
    return l.before(l.row_tiles) * c.kv_heads;
  };
  unsigned sum = 0;
  for (int b = tid; b < a.b.n_seqs; b += THREADS) sum = line_add(sum, blocks_of(b));
  sum = line_sum(sum);
  if (lane == 0) s_scan[warp] = (int)sum;
  __syncthreads();
  const int total = line_total<WARPS>(s_scan, a.b.err);
  Walk<BK> walk;
  walk.per = max((total + (int)gridDim.x - 1) / (int)gridDim.x, MIN_BLOCKS);
  if (walk.per * (long long)blockIdx.x >= total) return;
  walk.at = walk.per * blockIdx.x;
  walk.end = min(walk.at + walk.per, total);
  walk.b = 0;
  walk.seq_start = 0;
  for (int b0 = 0; b0 < a.b.n_seqs; b0 += THREADS) {
    const int n = b0 + tid < a.b.n_seqs ? blocks_of(b0 + tid) : 0;
    int run = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, run, o);
      if (lane >= o) run += y;
    }
    __syncthreads();
    if (lane == 31) s_scan[warp] = run;
    __syncthreads();
    int all = walk.seq_start;
    for (int w = 0; w < WARPS; w++) {
      if (w == warp) run += all;
      all += s_scan[w];
    }
    if (walk.at >= run - n && walk.at < run) {  // one thread at most
      s_seq = b0 + tid;
      s_scan[WARPS] = run - n;
    }
    __syncthreads();
    if (walk.at < all) {
      walk.b = s_seq;
      walk.seq_start = s_scan[WARPS];
      break;
    }
    walk.seq_start = all;
  }
  walk.found = false;

  if (tid == 0) {
    for (int i = 0; i < N_BARS; i++) {
      const auto is = [&](int first, int n) { return i >= first && i < first + n; };
      const unsigned count = is(B_Q, PIECES)                                      ? SOFTMAX_WARPS
                             : is(B_DONE, PIECES)                                 ? SOFTMAX_WARPS + 1
                             : is(B_P, 4)                                         ? SOFTMAX_WARPS / 2
                             : is(B_K, MAX_STAGES) || is(B_V, MAX_STAGES)         ? LOAD_WARPS
                             : is(B_K_FREE, MAX_STAGES) || is(B_V_FREE, MAX_STAGES) || is(B_PLAN_FREE, BATCHES) || i == B_FIN
                                 ? 2   // the warps of the products
                                 : 1;
      bar_init(bar(i), count);
    }
    s_abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncwarp();
  if (warp == MMA_WARP) tmem_alloc(smem_addr(&s_tmem), TM_COLS);
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = s_tmem;
  volatile int *abort_flag = &s_abort;
  // Every lane waits; bounded (about two seconds): false for the whole warp once any wait of the block has expired.
  auto wait = [&](int i, unsigned phase) -> bool {
    const uint32_t b = bar(i);
    bool ok = bar_try_wait(b, phase & 1u);
    if (!ok) {
      const unsigned t0 = (unsigned)clock();
      do ok = bar_try_wait_sleep(b, phase & 1u, 20000u);
      while (!ok && !*abort_flag && (unsigned)clock() - t0 < 4000000000u);
      if (!ok && !*abort_flag) {
        flag(a.b.err, BAD_WAIT);
        *abort_flag = 1;
      }
    }
    return __all_sync(0xffffffffu, ok);
  };

  if (warp >= MMA_WARP) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(MMA_REGS));
    if (warp == MMA_WARP + 1) {
      // ---------------- pieces ----------------
      bool more = true;
#pragma unroll 1
      for (unsigned k = 0; more; k++) {
        Piece p;
        more = walk.next(a, p);
        if (!more) p.n = -1;
        if (k >= PIECES && !wait(B_DONE + k % PIECES, k / PIECES - 1)) break;  // its place is free
        if (lane == 0 && !(a.withhold && blockIdx.x == 0 && k == 0)) {
          s_pieces[k % PIECES] = p;
          bar_arrive(bar(B_PIECE + k % PIECES));
        }
        __syncwarp();
      }
    } else if (warp == MMA_WARP + 2) {
      // ---------------- pages and scales ----------------
      unsigned batch = 0;
      bool ok = true;
#pragma unroll 1
      for (unsigned k = 0; ok; k++) {
        if (!(ok = wait(B_PIECE + k % PIECES, k / PIECES))) break;
        const Piece p = s_pieces[k % PIECES];
        if (p.n < 0) break;
        int v_top = V_EXP_MIN;
        const int j = lane & 3;  // lane: group j of block i
#pragma unroll 1
        for (int i0 = 0; i0 < p.n; i0 += BATCH, batch++) {
          const int i = i0 + (lane >> 2), key = p.block(i) * BK + 16 * j;
          const bool in = i < p.n;
          int page = -1;
          const bool seen = !a.window || key > p.pos0 - a.window - 15 || key < a.sinks;  // by a row at all
          if (in && key < p.len && seen) page = load_page(a.b, c, p.b, key);
          float ks = 0.f, vs = 0.f;
          if (page >= 0) {
            ks = c.ks[(long long)page * c.kv_heads + p.head];
            vs = c.vs[(long long)page * c.kv_heads + p.head];
          }
          const uint32_t present = __ballot_sync(0xffffffffu, page >= 0) >> (lane & 28) & 15;
          const int e = v_exp(vs);
          v_top = max(v_top, __reduce_max_sync(0xffffffffu, e));
          const int floor = max(v_top - V_EXP_SPAN, V_EXP_MIN);
          const uint32_t with_v = __ballot_sync(0xffffffffu, e > floor) >> (lane & 28) & 15;
          if (batch >= BATCHES && !(ok = wait(B_PLAN_FREE + batch % BATCHES, batch / BATCHES - 1))) break;
          Plan &plan = plans[batch % BATCHES * BATCH + (lane >> 2)];
          plan.place[j] = page < 0 ? -1 : ((page * c.kv_heads + p.head) << (c.page_shift - 4)) + ((key & (c.page - 1)) >> 4);
          plan.ks[j] = ks;
          if (SPLIT) {
            const int x = max(e, floor);
            plan.exp[j] = (float)x;
            plan.inv[j] = exp_inv(x);
            plan.man[j] = vs * exp_inv(x);
          } else {
            const float x = e > floor ? log2f(vs) : (float)floor;
            plan.exp[j] = x;
            plan.inv[j] = exp2f(-x);
          }
          if (j == 0) {
            plan.present = present;
            plan.with_v = with_v;
          }
          __syncwarp();
          if (lane == 0) bar_arrive(bar(B_PLAN + batch % BATCHES));
        }
      }
    } else {
      // ---------------- products of tile x ----------------
      const int x = warp == MMA_WARP ? 0 : 1;
      // The whole warp walks the loop, so that addresses and descriptors are uniform values; one elected thread
      // issues (with a single thread in the loop each product took 100 to 150 clocks to issue, twice its own time).
      const bool leader = elect_one();
      const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
      auto commit = [&](int i) {
        if (leader) mma_commit(bar(i));
      };
      unsigned done = 0, batch = 0, tile_done = 0;  // blocks in all, batches, blocks of the tile
      bool ok = true;
#pragma unroll 1
      for (unsigned k = 0; ok; k++) {
        if (!(ok = wait(B_PIECE + k % PIECES, k / PIECES))) break;
        const int n = __shfl_sync(0xffffffffu, s_pieces[k % PIECES].n, 0);
        const bool active = x == 0 || __shfl_sync(0xffffffffu, s_pieces[k % PIECES].n_rows, 0) > TILE_ROWS;
        if (n < 0) break;
        // An operand's place is the low bits of its descriptor, in units of 16 bytes: every one is a base and a sum.
        const uint64_t qd = sw128_desc(base + C::OFF_Q + x * TERMS * C::Q_TILE), kd = sw128_desc(base + C::OFF_K);
        const uint64_t vd = mn_desc(base + C::OFF_V, C::KV_PANEL);
        auto scores = [&](int buf, int st) {
          const uint64_t kk = kd + (uint32_t)(st * (C::KV_TILE >> 4));
          const uint32_t d = tm + x * 128 + buf * 64;
          if (leader) {
#pragma unroll
            for (int t = TERMS - 1; t >= 0; t--)  // second terms first: their sums are small when they are truncated
#pragma unroll
              for (int i = 0; i < HD / 16; i++)
                mma_f16(d, qd + ((t * C::Q_TILE + (i >> 2) * C::Q_PANEL + (i & 3) * 32) >> 4),
                        kk + (((i >> 2) * C::KV_PANEL + (i & 3) * 32) >> 4), idesc_f16(TILE_ROWS, BK, false),
                        t < TERMS - 1 || i);
            mma_commit(bar(B_S + 2 * x + buf));
          }
        };
        auto output = [&](int buf, int st, bool add) {
          const uint64_t v = vd + (uint32_t)(st * (C::KV_TILE >> 4));
          const uint32_t d = tm + TM_O + x * 128, w = tm + x * 128 + buf * 64;
          if (leader) {
#pragma unroll
            for (int t = TERMS - 1; t >= 0; t--)
#pragma unroll
              for (int i = 0; i < BK / 16; i++)
                mma_f16_ts(d, w + t * 32 + i * 8, v + (i * 2048 >> 4), idesc_f16(TILE_ROWS, HD, true),
                           t < TERMS - 1 || i || add);
            mma_commit(bar(B_PV + 2 * x + buf));
          }
        };
        if (!(ok = wait(B_Q + k % PIECES, k / PIECES))) break;
        // Turn i: P V of block i, then the scores of block i + 2 (turns -2 and -1: the first scores alone). A tile
        // without rows only gives its leave for each stage as it is filled.
#pragma unroll 1
        for (int i = -2; i < n; i++) {
          const unsigned now = done + i, ahead = now + 2, t = tile_done + i;  // the tile's buffer t % 2, its turn t / 2
          const int st = now % STAGES, st2 = ahead % STAGES, buf = t & 1;
          const bool more = i + 2 < n;
          // K of block i + 2 comes after V of block i + 1: one wait for both, well before it is needed
          if (!(ok = more ? wait(B_K + st2, ahead / STAGES) : i < 0 || wait(B_V + st, now / STAGES))) break;
          if (i >= 0) {
            if (active && !(ok = wait(B_P + 2 * x + buf, t / 2))) break;
            fence_after();
            if (active) output(buf, st, SPLIT ? i % MOVE : i);
            commit(B_V_FREE + st);
            if (i % BATCH == BATCH - 1 || i == n - 1) commit(B_PLAN_FREE + batch++ % BATCHES);
          }
          if (more) {
            fence_after();
            if (active) scores(buf, st2);
            commit(B_K_FREE + st2);
          }
        }
        done += n;
        if (active) tile_done += n;
        if (ok && x == 1 && lane == 0) bar_arrive(bar(B_DONE + k % PIECES));
      }
      // every product done before the columns are freed
      commit(B_FIN);
      if (x == 0) bar_drain(bar(B_FIN), 0u);
      __syncwarp();
    }
  } else if (warp >= SOFTMAX_WARPS) {
    // ---------------- codes to f16 tiles ----------------
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(LOAD_REGS));
    const int me = tid - SOFTMAX_WARPS * 32, r0 = me / C::ROW_CHUNKS, ch = me % C::ROW_CHUNKS;
    constexpr int STEP_GROUPS = C::STEP_ROWS / 16;  // groups of a step: a warp's keys are of one
    const int my_group = r0 >> 4;
    // Own chunks: keys r0 + STEP_ROWS k, codes 16 ch .. of the row; in the tile that row's 16-byte pieces 2 ch and
    // 2 ch + 1. With two panels a row's upper lanes start with their second piece, so that eight lanes meet
    // every bank once.
    const bool swap = HD == 128 && (ch & 4);
    const uint32_t row = (ch >> 2) * C::KV_PANEL + r0 * 128;
    const uint32_t piece0 = row + ((((ch & 3) * 2) + swap) ^ (r0 & 7)) * 16;
    const uint32_t piece1 = row + ((((ch & 3) * 2) + !swap) ^ (r0 & 7)) * 16;
    unsigned done = 0, batch = 0;  // blocks and batches so far
    bool ok = true;
    // Groups that are not there (or, for V, have a scale of 0) become zeros.
    auto fetch = [&](uint4 (&u)[C::STEPS], const int4 &place, uint32_t present, const uint8_t *codes) {
      const int at[4] = {place.x, place.y, place.z, place.w};
#pragma unroll
      for (int k = 0; k < C::STEPS; k++) {
        const int g0 = k * STEP_GROUPS, at_k = STEP_GROUPS == 1 ? at[g0] : (my_group ? at[(g0 + 1) & 3] : at[g0]);
        u[k] = make_uint4(0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u);
        if (present >> (g0 + my_group) & 1)
          u[k] = *reinterpret_cast<const uint4 *>(codes + (long long)at_k * (16 * HD));
      }
    };
    auto convert = [&](uint4 (&u)[C::STEPS], uint32_t tile) {
#pragma unroll
      for (int k = 0; k < C::STEPS; k++) {
        if (swap) {
          const uint4 x = u[k];
          u[k] = make_uint4(x.z, x.w, x.x, x.y);
        }
        const uint32_t to = tile + k * (C::STEP_ROWS * 128);
        sts128(to + piece0, codes_lo(u[k].x), codes_hi(u[k].x), codes_lo(u[k].y), codes_hi(u[k].y));
        sts128(to + piece1, codes_lo(u[k].z), codes_hi(u[k].z), codes_lo(u[k].w), codes_hi(u[k].w));
      }
    };
    const uint8_t *my_k = c.k + (r0 & 15) * HD + ch * 16, *my_v = c.v + (r0 & 15) * HD + ch * 16;
    // Turn i: block i is converted, block i + 1 fetched (turn -1: the first is fetched).
#pragma unroll 1
    for (unsigned k = 0; ok; k++) {
      if (!(ok = wait(B_PIECE + k % PIECES, k / PIECES))) break;
      const int n = s_pieces[k % PIECES].n;
      if (n < 0) break;
      uint4 ku[C::STEPS], vu[C::STEPS];
#pragma unroll 1
      for (int i = -1; ok && i < n; i++) {
        int4 place = {0, 0, 0, 0};
        uint32_t present = 0, with_v = 0;
        if (i + 1 < n) {
          const unsigned t = batch + (i + 1) / BATCH;
          if ((i + 1) % BATCH == 0 && !(ok = wait(B_PLAN + t % BATCHES, t / BATCHES))) break;
          const Plan &plan = plans[t % BATCHES * BATCH + (i + 1) % BATCH];
          place = *reinterpret_cast<const int4 *>(plan.place);
          present = plan.present;
          with_v = plan.with_v;
        }
        const unsigned at = done + i;
        const int st = at % STAGES;
        if (i >= 0) {
          if (at >= STAGES && !(ok = wait(B_K_FREE + st, at / STAGES - 1))) break;
          convert(ku, base + C::OFF_K + st * C::KV_TILE);
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) bar_arrive(bar(B_K + st));
        }
        if (i + 1 < n) fetch(ku, place, present, my_k);
        if (i >= 0) {
          if (at >= STAGES && !(ok = wait(B_V_FREE + st, at / STAGES - 1))) break;
          convert(vu, base + C::OFF_V + st * C::KV_TILE);
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) bar_arrive(bar(B_V + st));
        }
        if (i + 1 < n) fetch(vu, place, with_v, my_v);
      }
      done += n;
      batch += (n + BATCH - 1) / BATCH;
    }
  } else {
    // ---------------- softmax and output: one thread a row ----------------
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(SOFTMAX_REGS));
    const int x = warp >> 2, r = tid & (TILE_ROWS - 1), row = x * TILE_ROWS + r;
    const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
    const uint32_t s_tile = tmem + lanes + x * 128, o_col = tmem + lanes + TM_O + x * 128;
    auto all_ok = [&](bool v) -> bool {  // of the eight warps; also their barrier
      unsigned res;
      asm volatile(
          "{\n\t.reg .pred p, q;\n\t"
          "setp.ne.u32 p, %1, 0;\n\t"
          "bar.red.and.pred q, 1, %2, p;\n\t"
          "selp.u32 %0, 1, 0, q;\n\t}"
          : "=r"(res)
          : "r"((unsigned)v), "n"(SOFTMAX_WARPS * 32)
          : "memory");
      return res != 0;
    };
    unsigned batch = 0, tile_done = 0;  // batches so far, blocks of this tile
    const int per_group = (65536 + a.group - 1) / a.group;  // row / group = row * per_group >> 16 for rows < 256
#pragma unroll 1
    for (unsigned k = 0;; k++) {
      bool ok = wait(B_PIECE + k % PIECES, k / PIECES);
      const Piece &piece = s_pieces[k % PIECES];
      const int n = ok ? piece.n : -1;
      if (ok && n < 0) break;
      const int n_rows = piece.n_rows, row0 = piece.row0, h0 = piece.head * a.group, tok = row / a.group;
      const bool live = ok && row < n_rows, active = x == 0 || n_rows > TILE_ROWS;
      const int warp_row = x * TILE_ROWS + 32 * (warp & 3);  // first of the warp's 32 rows
      // Rows of the warp move in and out ROW_LANES lanes a row, 16 bytes a lane.
      constexpr int ROW_LANES = HD * (int)sizeof(T) / 16, AT_ONCE = 32 / ROW_LANES, PER16 = 16 / (int)sizeof(T);
      const int sub = lane / ROW_LANES, piece16 = lane % ROW_LANES;
      auto row_at = [&](const auto *rows, long long stride, int i) {  // the lane's part of the warp's row i
        const int q = warp_row + i, t = q * per_group >> 16;
        return rows + (long long)(row0 + t) * stride + (h0 + q - t * a.group) * HD + piece16 * PER16;
      };
      auto stage = [&](int i, int at) {  // 16-byte chunk `at` of the warp's row i, over the row's bytes in the query tile
        return base + C::OFF_Q + x * TERMS * C::Q_TILE + (at >> 3) * C::Q_PANEL + (32 * (warp & 3) + i) * 128 +
               ((at ^ i) & 7) * 16;
      };
      // ---- the queries: fetched into their tile, then replaced by their f16 terms
#pragma unroll 4
      for (int i = sub; i < 32; i += AT_ONCE) {
        if (ok && warp_row + i < n_rows) cp16(stage(i, piece16), row_at(a.q, a.qs, i));
        else sts128(stage(i, piece16), 0, 0, 0, 0);
      }
      cp_commit();
      cp_wait<0>();
      __syncwarp();
      // Each thread converts its own row in place: its largest magnitude (of the bits, so that NaN and infinities show),
      // then the terms, 8 elements a chunk, second terms in the panels after the first ones'.
      uint32_t most = 0;
#pragma unroll 8
      for (int j = 0; j < HD / PER16; j++) {
        const uint4 u = lds128(stage(lane, j));
        if constexpr (SPLIT) {
          most = max(max(most, max(u.x & 0x7FFFFFFFu, u.y & 0x7FFFFFFFu)), max(u.z & 0x7FFFFFFFu, u.w & 0x7FFFFFFFu));
        } else {
          most = __vmaxu2(most, __vmaxu2(__vmaxu2(u.x & 0x7FFF7FFFu, u.y & 0x7FFF7FFFu),
                                         __vmaxu2(u.z & 0x7FFF7FFFu, u.w & 0x7FFF7FFFu)));
        }
      }
      if (!SPLIT) most = max(most << 16, most & 0xFFFF0000u);
      const bool finite = most < 0x7F800000u;
      const int e = row_exp(finite ? __uint_as_float(most) : 0.f);
      // the sign of the scale goes into the row: the factor of its scores is then not negative and maxima commute
      const float up = row_factor(e, finite) * (a.scale < 0.f ? -1.f : 1.f), cf = scalbnf(fabsf(a.scale), -e);
      if constexpr (SPLIT) {
        uint32_t g[HD / 2];
#pragma unroll
        for (int j = 0; j < HD / 8; j++) {
          const uint4 u = lds128(stage(lane, 2 * j)), w = lds128(stage(lane, 2 * j + 1));
          const uint32_t x[8] = {u.x, u.y, u.z, u.w, w.x, w.y, w.z, w.w};
          uint32_t f[4];
#pragma unroll
          for (int z = 0; z < 4; z++) {
            const float y0 = __uint_as_float(x[2 * z]) * up, y1 = __uint_as_float(x[2 * z + 1]) * up;
            f[z] = pack(y0, y1);
            const float2 hi = unpack(f[z]);
            g[4 * j + z] = pack(y0 - hi.x, y1 - hi.y);
          }
          sts128(stage(lane, j), f[0], f[1], f[2], f[3]);
        }
#pragma unroll
        for (int j = 0; j < HD / 8; j++)
          sts128(stage(lane, HD / 8 + j), g[4 * j], g[4 * j + 1], g[4 * j + 2], g[4 * j + 3]);
      } else {
#pragma unroll 4
        for (int j = 0; j < HD / 8; j++) {
          const uint4 u = lds128(stage(lane, j));
          auto two = [&](uint32_t w) { return pack(__uint_as_float(w << 16) * up, __uint_as_float(w & 0xFFFF0000u) * up); };
          sts128(stage(lane, j), two(u.x), two(u.y), two(u.z), two(u.w));
        }
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) bar_arrive(bar(B_Q + k % PIECES));

      const int pos0 = piece.pos0, t0 = piece.t0, n_sink = piece.n_sink, skip = piece.skip;
      const int pos = live ? pos0 + tok : -1;
      const int low = a.window ? pos - a.window : -1;  // seen: low < key <= pos, or key < sinks
      const int sinks = a.window ? a.sinks : 0;
      const int min_pos = pos0 + warp_row / a.group, max_pos = pos0 + (warp_row + 31) / a.group;
      float o[SPLIT ? HD : 1], ref = -INFINITY, l = 0.f;
      if constexpr (SPLIT) {
#pragma unroll
        for (int d = 0; d < HD; d++) o[d] = 0.f;
      }
      // f32 rows: o += O
      auto add_output = [&]() {
        if constexpr (SPLIT) {
#pragma unroll
          for (int d = 0; d < HD; d += 32) {
            float v[32];
            tmem_ld32(o_col + d, v);
            tmem_ready<32>(v);
#pragma unroll
            for (int j = 0; j < 32; j++) o[d + j] += v[j];
          }
        }
      };
      // Products of the tile's block t (not every turn waits for them; those of t - 2 came before the scores of t).
      auto products_done = [&](unsigned t) { return wait(B_PV + 2 * x + (t & 1), t / 2); };
      // Turn i = n only takes the last output.
#pragma unroll 1
      for (int i = 0; ok && active && n && i <= n; i++) {
        if (i == n) {
          ok = products_done(tile_done + n - 1);
          fence_after();
          if (ok) add_output();
          break;
        }
        const unsigned t = tile_done + i, bt = batch + i / BATCH;
        const uint32_t s_col = s_tile + (t & 1) * 64;
        const Plan &plan = plans[bt % BATCHES * BATCH + i % BATCH];
        if (i % BATCH == 0 && !(ok = wait(B_PLAN + bt % BATCHES, bt / BATCHES))) break;
        if (!(ok = wait(B_S + 2 * x + (t & 1), t / 2))) break;
        fence_after();
        float v[64];
        tmem_ld32(s_col, v);
        tmem_ld32(s_col + 32, v + 32);
        const int key0 = (t0 + i + (t0 + i < n_sink ? 0 : skip)) * BK;
        const uint32_t present = plan.present;
        const float4 ks = *reinterpret_cast<const float4 *>(plan.ks), exp4 = *reinterpret_cast<const float4 *>(plan.exp);
        // the factors of the groups' scores; not 0, because hidden scores are -infinity
        float f[4] = {fmaxf(cf * ks.x, FLT_MIN), fmaxf(cf * ks.y, FLT_MIN), fmaxf(cf * ks.z, FLT_MIN),
                            fmaxf(cf * ks.w, FLT_MIN)};
        float exp[4] = {exp4.x, exp4.y, exp4.z, exp4.w};
        tmem_ready<64>(v);
        if (key0 + BK - 1 > min_pos || (a.window && key0 <= max_pos - a.window && key0 + BK > a.sinks) ||
            present != (1u << NG) - 1) {
          auto upto = [&](int end) -> uint64_t {  // bits of the block's keys < end
            const int m = min(max(end - key0, 0), 64);
            return m == 64 ? ~0ull : (1ull << m) - 1;
          };
          uint64_t see = upto(pos + 1) & (~upto(low + 1) | upto(sinks));
#pragma unroll
          for (int g = 0; g < NG; g++)
            if (!(present >> g & 1)) see &= ~(0xffffull << (16 * g));
          const uint32_t s0 = (uint32_t)see, s1 = (uint32_t)(see >> 32);
#pragma unroll
          for (int j = 0; j < 32; j++) {
            v[j] = s0 >> j & 1 ? v[j] : -INFINITY;
            v[32 + j] = s1 >> j & 1 ? v[32 + j] : -INFINITY;
          }
        }
        float mx = -INFINITY;
#pragma unroll
        for (int g = 0; g < NG; g++) {
          float m1 = fmaxf(v[16 * g], v[16 * g + 1]), m2 = fmaxf(v[16 * g + 2], v[16 * g + 3]);
#pragma unroll
          for (int j = 4; j < 16; j += 4) {
            m1 = max3(m1, v[16 * g + j], v[16 * g + j + 1]);
            m2 = max3(m2, v[16 * g + j + 2], v[16 * g + j + 3]);
          }
          mx = fmaxf(mx, fmaf(fmaxf(m1, m2), f[g], exp[g]));
        }
        // the reference follows the maximum: earlier results move along. A whole number, so that an f32 row's page
        // exponents are added to it exactly
        float alpha = 1.f;
        if (mx > ref + REF_LAG) {  // also the first key that a row sees: alpha = 0
          const float to = rintf(mx);
          alpha = ex2(ref - to);
          l = scaled(l, ref - to);
          ref = to;
        }
        const float shift = ref == -INFINITY ? 0.f : WEIGHT_EXP - ref;
        // The reference is a rounded score. Where a score's rounding is some octaves, they are all rounded before it is
        // taken off, or the largest weights would be off by as many.
        if (__any_sync(0xffffffffu, fabsf(shift) > LARGE_SCORE)) {
#pragma unroll
          for (int g = 0; g < NG; g++) {
#pragma unroll
            for (int j = 16 * g; j < 16 * g + 16; j++) v[j] = fmaf(v[j], f[g], exp[g]);
            f[g] = 1.f, exp[g] = 0.f;
          }
        }
        // weights, over the scores
        float sum = 0.f;
        uint32_t hi[32], lo[SPLIT ? 32 : 1];
#pragma unroll
        for (int g = 0; g < NG; g++) {
          const float sh = shift + exp[g], man = SPLIT ? plan.man[g] : 1.f;
          const f2x f2 = pk2(f[g], f[g]), sh2 = pk2(sh, sh), man2 = pk2(man, man);
          f2x gs = 0ull;
#pragma unroll
          for (int j = 0; j < 8; j++) {
            const float2 y = up2(ffma2(pk2(v[16 * g + 2 * j], v[16 * g + 2 * j + 1]), f2, sh2));
            f2x w = pk2(ex2(y.x), ex2(y.y));
            gs = fadd2(gs, w);
            if constexpr (SPLIT) w = fmul2(w, man2);
            const float2 z = up2(w);
            hi[8 * g + j] = pack(z.x, z.y);
            if constexpr (SPLIT) {
              const float2 h2 = unpack(hi[8 * g + j]);
              lo[8 * g + j] = pack(z.x - h2.x, z.y - h2.y);
            }
          }
          const float2 z = up2(gs);
          sum = fmaf(z.x + z.y, plan.inv[g], sum);
        }
        tmem_st32(s_col, hi);
        if constexpr (SPLIT) tmem_st32(s_col + 32, lo);
        l += sum;
        const bool take = SPLIT && i % MOVE == 0;  // the output so far is taken, this block's starts anew
        const bool any = i && __any_sync(0xffffffffu, alpha != 1.f);
        if (i && (take || any)) {  // the last block's P V is done before its output is read or moved
          if (!(ok = products_done(t - 1))) break;
          fence_after();
          if (take) {
            add_output();
          } else {
#pragma unroll 1
            for (int d = 0; d < HD; d += 32) {
              float y[32];
              tmem_ld32(o_col + d, y);
              tmem_ready<32>(y);
              uint32_t u[32];
#pragma unroll
              for (int j = 0; j < 32; j++) u[j] = __float_as_uint(y[j] * alpha);
              tmem_st32(o_col + d, u);
            }
          }
          if constexpr (SPLIT) {
            if (__any_sync(0xffffffffu, alpha != 1.f)) {
#pragma unroll
              for (int d = 0; d < HD; d++) o[d] *= alpha;
            }
          }
        }
        tmem_wait_st();
        fence_before();
        __syncwarp();
        if (lane == 0) bar_arrive(bar(B_P + 2 * x + (t & 1)));
      }
      if (!all_ok(ok)) break;
      if (active) tile_done += n;
      batch += (n + BATCH - 1) / BATCH;
      const bool none = !active || !n;  // nothing was computed: l = 0, O is not the tile's
      const bool whole = piece.whole;
      float *slot = a.part + (size_t)piece.slot * C::SLOT + row;  // [head_dim][rows], maxima, sums
      const float inv = l == 0.f ? 0.f : 1.f / l;
      // Results go out through the warp's own rows of the query tile (its products are done; other warps may be at
      // the next piece's queries): a thread writes its row, then ROW_LANES lanes a row store 16 bytes each.
      auto write = [&](int d, const float *v) {  // 32 values of the thread's row
#pragma unroll
        for (int j = 0; j < 32; j += PER16) {
          const uint32_t dst = stage(lane, (d + j) / PER16);
          if constexpr (SPLIT)
            sts128(dst, __float_as_uint(v[j]), __float_as_uint(v[j + 1]), __float_as_uint(v[j + 2]), __float_as_uint(v[j + 3]));
          else
            sts128(dst, bf16_pair(v[j], v[j + 1]), bf16_pair(v[j + 2], v[j + 3]), bf16_pair(v[j + 4], v[j + 5]),
                   bf16_pair(v[j + 6], v[j + 7]));
        }
      };
      auto flush = [&]() {
        __syncwarp();
#pragma unroll 4
        for (int i = sub; i < 32; i += AT_ONCE) {
          const uint4 u = lds128(stage(i, piece16));
          if (warp_row + i < n_rows) *reinterpret_cast<uint4 *>(const_cast<T *>(row_at(a.out, a.os, i))) = u;
        }
        __syncwarp();
      };
      auto put = [&](int d, float *v) {
        if (whole) {
#pragma unroll
          for (int j = 0; j < 32; j++) v[j] = l == 0.f ? 0.f : v[j] * inv;
          write(d, v);
        } else {
#pragma unroll
          for (int j = 0; j < 32; j++) slot[(d + j) * ROWS] = v[j];
        }
      };
      if constexpr (SPLIT) {
#pragma unroll
        for (int d = 0; d < HD; d += 32) put(d, o + d);
      } else {
#pragma unroll 1
        for (int d = 0; d < HD; d += 32) {
          float v[32];
          tmem_ld32(o_col + d, v);
          tmem_ready<32>(v);
#pragma unroll
          for (int j = 0; j < 32; j++) v[j] = none ? 0.f : v[j];
          put(d, v);
        }
      }
      if (whole) {
        flush();
      } else {  // the last block to arrive joins all parts, in block order
        slot[HD * ROWS] = ref;
        slot[(HD + 1) * ROWS] = l;
        int *count = a.count + piece.counter;
        const int parts = piece.parts, first = piece.first, late = piece.late;
        __threadfence();
        all_ok(true);
        if (tid == 0) s_last = atomicAdd(count, 1) == parts - 1;
        all_ok(true);
        if (s_last) {
          __threadfence();
          auto part = [&](int i) { return a.part + (size_t)(2 * (first + i) + (i == 0 ? late : 0)) * C::SLOT + row; };
          float top = -INFINITY, sum = 0.f;
#pragma unroll 1
          for (int i = 0; i < parts; i++) top = fmaxf(top, __ldcg(part(i) + HD * ROWS));
          const float at0 = top == -INFINITY ? 0.f : top;
#pragma unroll 1
          for (int i = 0; i < parts; i++)
            sum += scaled(__ldcg(part(i) + (HD + 1) * ROWS), __ldcg(part(i) + HD * ROWS) - at0);
          const float all_inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll 1
          for (int d = 0; d < HD; d += 32) {
            float v[32];
#pragma unroll
            for (int j = 0; j < 32; j++) v[j] = 0.f;
#pragma unroll 1
            for (int i = 0; i < parts; i++) {
              const float *src = part(i);
              const float f = ex2(__ldcg(src + HD * ROWS) - at0);
#pragma unroll
              for (int j = 0; j < 32; j++) v[j] = fmaf(__ldcg(src + (d + j) * ROWS), f, v[j]);
            }
#pragma unroll
            for (int j = 0; j < 32; j++) v[j] = sum == 0.f ? 0.f : v[j] * all_inv;
            write(d, v);
          }
          flush();
          if (tid == 0) *count = 0;
        }
      }
      __syncwarp();
      if (lane == 0) bar_arrive(bar(B_DONE + k % PIECES));
    }
  }
  fence_before();
  __syncthreads();
  if (warp == MMA_WARP) {
    fence_after();
    tmem_dealloc(tmem, TM_COLS);
  }
}

// Failure-detection tests only: SQ_TEST_WITHHOLD_PIECE=n (read at the process's first launch of this kernel) makes its
// n-th launch leave the first block's first piece unsaid, so that every wait of that block for it expires and the
// next status check reports a timeout.
int test_withhold() {
  static const long n = [] {
    const char *v = getenv("SQ_TEST_WITHHOLD_PIECE");
    return v ? strtol(v, nullptr, 10) : 0L;
  }();
  static std::atomic<long> launches{0};
  return n > 0 && ++launches == n ? 1 : 0;
}

template <class C, typename T>
cudaError_t launch(cudaStream_t s, AttnArgs<T> &a) {
  static int blocks[64] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev >= 64) return cudaErrorInvalidDevice;
  if (!blocks[dev]) {
    int sms = 0;
    if ((e = cudaFuncSetAttribute(k_paged_many<C, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM)) !=
            cudaSuccess ||
        (e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev)) != cudaSuccess)
      return e;
    blocks[dev] = min(sms, MAX_BLOCKS);
  }
  a.max_row_tiles = many_row_tiles(a.b.max_new, a.group);
  a.withhold = test_withhold();
  return launch_ex(k_paged_many<C, T>, dim3(blocks[dev]), dim3(THREADS), C::SMEM, s, pdl_enabled(), a);
}

}  // namespace

int many_row_tiles(int max_new, int group) {
  const int tokens = ROWS / group;
  return (max_new + tokens - 1) / tokens;
}
size_t many_partial_bytes(int head_dim) { return (size_t)MAX_BLOCKS * 2 * ROWS * (head_dim + 2) * sizeof(float); }

bool many_supported(const Cache &c, int group) {
  return (c.hd == 64 || c.hd == 128) && group <= TILE_ROWS;
}
template <typename T>
cudaError_t launch_many(cudaStream_t s, AttnArgs<T> a) {
  return a.c.hd == 64 ? launch<Cfg<T, 64>>(s, a) : launch<Cfg<T, 128>>(s, a);
}
template cudaError_t launch_many<float>(cudaStream_t, AttnArgs<float>);
template cudaError_t launch_many<__nv_bfloat16>(cudaStream_t, AttnArgs<__nv_bfloat16>);

}  // namespace paged
}  // namespace sq
