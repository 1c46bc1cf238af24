// paged_attention_tc.cu — causal grouped attention over the paged 8-bit cache for many query
// rows a kv head (prompts): bound by the products and the exponentials. tcgen05, head_dim
// 64 and 128.
//
// A block works on 256 query rows of one kv head (row = token * group + head of the
// group), two tiles X of 128 that share every key block, so that a code is converted once
// for 256 rows:
//   warps 8-10  codes of a block of keys to shared memory (cp.async, each thread its own
//               chunks), converted to f16 (exact: whole numbers up to 127) into the
//               128-byte swizzled tiles of K [keys][dims] and V [keys][dims]; two stages
//   warp 11     one thread issues the products, f32 sums in tensor memory:
//               S_X = Q_X K^T (K-major operands), O_X (+)= P_X V (V read MN-major as it
//               lies, P from tensor memory). Order: P V of one tile, its next S, then the
//               other tile: one tile's softmax runs under the other's products
//   warps 0-7   one thread a row (= tensor-memory lane): its scores to registers, running
//               maximum, weights back to the columns the scores left, sum
// Products issued by one thread complete in order, so a tile's S being done says that its
// last P V is done too: no further barriers between them.
//
// Precision, as in the few-row kernel: query rows scaled by powers of two, two f16 terms
// for f32 rows, one (exact) for bf16 rows. Weights are 2^(s - ref + 3); ref follows the
// maximum only when it is passed by 2^6, and the V scales go into the weights relative to
// a unit, so that f16 never overflows and outputs are seldom rescaled.
//   f32 rows:  weights in two terms; each block's O is summed on its own in tensor memory and
//              added to f32 registers, because the tensor core truncates its running sum
//              (2^-25 of it a step: 500 steps would cost 1e-5).
//   bf16 rows: weights in one term (11 bits, under the output's 8); O stays in tensor memory.
//
// Work is split as in the few-row kernel: one line of (sequence, kv head, row tile, key
// block), an equal piece for every block, cut row tiles joined by the last block to arrive.
// Every wait is bounded: on expiry the block records it, stops, lets its products and
// copies finish, frees its tensor memory and returns.
#include <cuda.h>
#include <float.h>

#include "paged_attention.cuh"
#include "tc.cuh"

namespace sq {
namespace paged {
namespace {

using namespace tc;

constexpr int SOFTMAX_WARPS = 8, LOAD_WARPS = 3, WARPS = SOFTMAX_WARPS + LOAD_WARPS + 1;
constexpr int THREADS = WARPS * 32, LOADERS = LOAD_WARPS * 32;
constexpr int TILE_ROWS = 128, ROWS = 2 * TILE_ROWS;
constexpr int STAGES = 2, SCALE_STAGES = 4;
constexpr int MAX_BLOCKS = 160;
constexpr int MIN_BLOCKS = 2;  // key blocks a thread block takes at least
constexpr float WEIGHT_EXP = 3.f, REF_LAG = 6.f, UNIT_LAG = 64.f;
// Registers a thread: launched with 168 (384 x 168 = 64,512), then 256 x 208 + 128 x 88.
constexpr int SOFTMAX_REGS = 208, OTHER_REGS = 88;

template <typename T, int HD_>
struct Cfg {
  static constexpr int HD = HD_;
  static constexpr bool SPLIT = sizeof(T) == 4;
  static constexpr int TERMS = SPLIT ? 2 : 1;
  static constexpr int BK = SPLIT && HD == 128 ? 64 : 128;  // keys a block; 64: two stages fit beside Q's two terms
  static constexpr int NG = BK / 16;                        // groups of 16 keys: each within one page
  static constexpr int PANELS = HD / 64;                    // 64 dimensions = 128 bytes of f16
  static constexpr int Q_PANEL = TILE_ROWS * 128, KV_PANEL = BK * 128;
  static constexpr int Q_TILE = PANELS * Q_PANEL, KV_TILE = PANELS * KV_PANEL;
  static constexpr int CHUNKS = BK * HD / 16;                     // 16-code chunks of a block
  static constexpr int PER_LOADER = (CHUNKS + LOADERS - 1) / LOADERS;
  static constexpr int RAW = PER_LOADER * LOADERS * 16;
  static constexpr int OFF_Q = 0, OFF_K = OFF_Q + 2 * TERMS * Q_TILE, OFF_V = OFF_K + STAGES * KV_TILE,
                       OFF_RAW = OFF_V + STAGES * KV_TILE, OFF_SCALE = OFF_RAW + 2 * RAW,
                       OFF_BAR = OFF_SCALE + SCALE_STAGES * 4 * 8 * 4;
  static constexpr int SMEM = 1024 + OFF_BAR + 256;
  static constexpr int SLOT = ROWS * (HD + 2);  // floats of a cut row tile's partial result
  static_assert(SMEM <= 232448 - 256, "shared memory of a block");
};

// A block's scales, read by the softmax threads: [group] K scale, V share, 1 / V share
// (bf16: log2 of the share), and in the last row: bit mask of present groups, unit.
struct Scales {
  float ks[8], share[8], inv[8];
  uint32_t present;
  float unit;
  float pad[6];
};
static_assert(sizeof(Scales) == 128, "four rows of eight words");

enum : int {
  B_Q = 0,       // both tiles' queries written
  B_K = 1,       // [2] a stage's K written
  B_K_FREE = 3,  // [2] S of both tiles done
  B_V = 5,       // [2]
  B_V_FREE = 7,  // [2]
  B_SCALE = 9,   // [4] a block's scales written
  B_S = 13,      // [2 tiles] scores done (and the tile's last P V)
  B_P = 15,      // [2 tiles] weights written
  B_O = 17,      // [2 tiles] the piece's last P V done
  B_FIN = 19,
  N_BARS = 20
};
constexpr uint32_t TM_O = 256, TM_COLS = 512;  // S / P of tile X at X * BK, O at 256 + 128 X

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

// Sum over i < n of floor((a i + b) / m), by Euclid's steps.
__device__ __forceinline__ long long floor_sum(long long n, int m, int a, long long b) {
  long long sum = 0;
  unsigned mm = m, aa = a;
  unsigned long long bb = b;
  while (n > 0) {
    if (aa >= mm) {
      sum += (n - 1) * n / 2 * (aa / mm);
      aa %= mm;
    }
    if (bb >= mm) {
      sum += n * (long long)(bb / mm);
      bb %= mm;
    }
    const unsigned long long y = (unsigned long long)aa * n + bb;
    if (y < mm) break;
    n = y / mm;
    bb = y % mm;
    const unsigned x = mm;
    mm = aa;
    aa = x;
  }
  return sum;
}

// Key blocks of a sequence's row tiles on the line: without a window the causal count of
// each (a little over for the last), with one the same for all; what a tile does not
// have of them is empty.
template <int BK>
struct Line {
  int row_tiles, tokens;  // tokens of a row tile
  int flat;               // key blocks of every row tile (window), or 0
  int pos0, len;
  __device__ __forceinline__ void set(const Seq &s, int group, int window, int sinks, int few_rows) {
    tokens = ROWS / group;
    row_tiles = s.n * group > few_rows ? (s.n + tokens - 1) / tokens : 0;
    pos0 = max(s.len - s.n, 0);
    len = s.len;
    flat = 0;
    if (window && window < s.len)
      flat = min((min(sinks, s.len) + BK - 1) / BK + (window + tokens + BK - 3) / BK + 1, (s.len + BK - 1) / BK);
  }
  __device__ __forceinline__ long long before(int rt) const {  // key blocks of row tiles 0 .. rt - 1
    if (flat) return (long long)rt * flat;
    return rt + floor_sum(rt, BK, tokens, pos0 + tokens - 1);
  }
  __device__ __forceinline__ int of(int rt) const {
    return flat ? flat : (int)((pos0 + (long long)(rt + 1) * tokens - 1) / BK) + 1;
  }
};

// One block's part of a row tile.
template <int BK>
struct Piece {
  int b, head, rt;
  Seq s;
  int first_tok, n_rows;     // tokens from first_tok on, rows in use
  int t0, n;                 // key blocks t0 .. t0 + n - 1 of the tile (n may be 0)
  int n_sink, skip;          // tile index to block number, as in the few-row kernel
  bool whole;
  int slot;                  // of the partial results
  long long first;           // blocks first .. first + parts - 1 share the tile
  int parts;
  bool late;                 // block `first` began another tile before this one: its second slot
  __device__ __forceinline__ int block(int i) const { return i < n_sink ? i : i + skip; }
};

// Walks this thread block's piece of the line; every warp does so on its own.
template <int BK>
struct Walk {
  long long at, end, per;
  long long seq_start;  // of sequence b on the line
  int b;
  Line<BK> line;
  Seq s;
  long long per_head;

  template <typename T>
  __device__ __forceinline__ void load(const AttnArgs<T> &a) {
    s = load_seq(a.b, a.c, b);
    line.set(s, a.group, a.window, a.sinks, a.few_rows);
    per_head = line.before(line.row_tiles);
  }
  template <typename T>
  __device__ __forceinline__ bool next(const AttnArgs<T> &a, Piece<BK> &p) {
    if (at >= end) return false;
    while (at >= seq_start + per_head * a.c.kv_heads) {
      seq_start += per_head * a.c.kv_heads;
      b++;
      load(a);
    }
    const long long in_seq = at - seq_start;
    p.head = (int)(in_seq / per_head);
    const long long in_head = in_seq - p.head * per_head;
    // the row tile that holds in_head: 32 candidates at a time
    int lo = 0, width = line.row_tiles;
    while (width > 1) {
      const int step = (width + 31) / 32, mine = lo + (threadIdx.x & 31) * step;
      const unsigned le = __ballot_sync(0xffffffffu, mine < lo + width && line.before(mine) <= in_head);
      const int k = 31 - __clz(le);  // lane 0 always holds
      lo += k * step;
      width = min(step, width - k * step);
    }
    p.rt = lo;
    p.b = b;
    p.s = s;
    const int slots = line.of(lo);
    const long long tile_start = seq_start + p.head * per_head + line.before(lo);
    p.first_tok = lo * line.tokens;
    const int toks = min(line.tokens, s.n - p.first_tok);
    p.n_rows = toks * a.group;
    const int min_pos = s.len - s.n + p.first_tok, max_pos = max(min_pos + toks - 1, 0);
    int real = max_pos / BK + 1;
    p.n_sink = p.skip = 0;
    if (line.flat) {
      const int low = max(min_pos - a.window + 1, 0) / BK;
      p.n_sink = min((min(a.sinks, s.len) + BK - 1) / BK, low);
      p.skip = low - p.n_sink;
      real -= p.skip;
    }
    p.t0 = (int)(at - tile_start);
    const int t1 = (int)min((long long)slots, end - tile_start);
    p.n = max(min(t1, real) - p.t0, 0);
    p.whole = p.t0 == 0 && t1 == slots;
    p.slot = 2 * blockIdx.x + (tile_start > per * blockIdx.x ? 1 : 0);
    p.first = tile_start / per;
    p.parts = (int)((tile_start + slots - 1) / per - p.first) + 1;
    p.late = tile_start > per * p.first;
    at = tile_start + t1;
    return true;
  }
};

template <class C, typename T>
__global__ void __launch_bounds__(THREADS, 1) k_paged_many(const AttnArgs<T> a) {
  constexpr int HD = C::HD, BK = C::BK, NG = C::NG, TERMS = C::TERMS;
  constexpr bool SPLIT = C::SPLIT;
  extern __shared__ uint8_t smem_raw[];
  __shared__ long long s_scan[WARPS + 2];
  __shared__ int s_seq, s_abort, s_last;
  __shared__ uint32_t s_tmem;
  const uint32_t base = (smem_addr(smem_raw) + 1023u) & ~1023u;
  uint8_t *gen = smem_raw + (base - smem_addr(smem_raw));
  Scales *scales = reinterpret_cast<Scales *>(gen + C::OFF_SCALE);
  auto bar = [&](int i) { return base + C::OFF_BAR + 8u * (uint32_t)i; };
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const Cache &c = a.c;

  // ---- this block's piece of the line
  auto blocks_of = [&](int b) -> long long {
    Line<BK> l;
    l.set(load_seq(a.b, c, b), a.group, a.window, a.sinks, a.few_rows);
    return l.before(l.row_tiles) * c.kv_heads;
  };
  long long total = 0;
  for (int b = tid; b < a.b.n_seqs; b += THREADS) total += blocks_of(b);
  total = warp_sum_ll(total);
  if (lane == 0) s_scan[warp] = total;
  __syncthreads();
  total = 0;
  for (int w = 0; w < WARPS; w++) total += s_scan[w];
  Walk<BK> walk;
  walk.per = max((total + gridDim.x - 1) / gridDim.x, (long long)MIN_BLOCKS);
  walk.at = walk.per * blockIdx.x;
  walk.end = min(walk.at + walk.per, total);
  if (walk.at >= walk.end) return;
  walk.b = 0;
  walk.seq_start = 0;
  for (int b0 = 0; b0 < a.b.n_seqs; b0 += THREADS) {
    const long long n = b0 + tid < a.b.n_seqs ? blocks_of(b0 + tid) : 0;
    long long run = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, run, o);
      if (lane >= o) run += y;
    }
    __syncthreads();
    if (lane == 31) s_scan[warp] = run;
    __syncthreads();
    long long all = walk.seq_start;
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
  walk.load(a);

  if (tid == 0) {
    for (int i = 0; i < N_BARS; i++) {
      const unsigned count = i == B_Q                          ? SOFTMAX_WARPS
                             : i >= B_P && i < B_P + 2         ? SOFTMAX_WARPS / 2
                             : i >= B_K && i < B_K + 2         ? LOAD_WARPS
                             : i >= B_V && i < B_V + 2         ? LOAD_WARPS
                                                               : 1;
      bar_init(bar(i), count);
    }
    s_abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncwarp();
  if (warp == WARPS - 1) tmem_alloc(smem_addr(&s_tmem), TM_COLS);
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = s_tmem;
  volatile int *abort_flag = &s_abort;
  // Bounded: false once any wait of the block has expired.
  auto wait = [&](int i, unsigned phase) -> bool {
    const uint32_t b = bar(i);
    if (bar_try_wait(b, phase & 1u)) return true;
    const long long t0 = clock64();
    while (!bar_try_wait_sleep(b, phase & 1u, 20000u)) {
      if (*abort_flag) return false;
      if (clock64() - t0 > WAIT_LIMIT) {
        flag(a.b.err, BAD_WAIT);
        *abort_flag = 1;
        return false;
      }
    }
    return true;
  };
  auto wait_warp = [&](int i, unsigned phase) -> bool {  // lane 0 waits, the warp follows
    int ok = 1;
    if (lane == 0) ok = wait(i, phase);
    ok = __shfl_sync(0xffffffffu, ok, 0);
    __syncwarp();
    return ok;
  };

  Piece<BK> p;
  if (warp >= SOFTMAX_WARPS) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(OTHER_REGS));
    if (warp < SOFTMAX_WARPS + LOAD_WARPS) {
      // ---------------- codes to f16 tiles ----------------
      const int me = tid - SOFTMAX_WARPS * 32;
      constexpr int ROW_CHUNKS = HD / 16;
      unsigned done = 0;  // blocks so far
      bool ok = true;
      while (ok && walk.next(a, p)) {
        float unit = 0.f;
        // Lane j < NG: page and scales of group j of a block.
        auto page_of = [&](int i) {
          const int key = p.block(p.t0 + i) * BK + 16 * lane;
          return i < p.n && lane < NG && key < p.s.len ? load_page(a.b, c, p.b, key) : -1;
        };
        auto fetch = [&](int i, int page, const uint8_t *codes, int raw) {
          if (i < p.n) {
            const int key0 = p.block(p.t0 + i) * BK;
#pragma unroll
            for (int k = 0; k < C::PER_LOADER; k++) {
              const int q = me + k * LOADERS, r = q / ROW_CHUNKS;
              const int pg = __shfl_sync(0xffffffffu, page, min(r >> 4, NG - 1));  // a warp's 32 chunks: one group
              if (q < C::CHUNKS && pg >= 0) {
                const long long at = (((long long)pg * c.kv_heads + p.head) * c.page + ((key0 + r) & (c.page - 1))) * HD;
                cp16(base + C::OFF_RAW + raw * C::RAW + q * 16, codes + at + (q % ROW_CHUNKS) * 16);
              }
            }
          }
          cp_commit();
        };
        // Own chunks: raw codes -> f16 in the swizzled tile; groups not in `present` become zeros.
        auto convert = [&](uint32_t present, int raw, uint32_t tile) {
#pragma unroll
          for (int k = 0; k < C::PER_LOADER; k++) {
            const int q = me + k * LOADERS, r = q / ROW_CHUNKS, ch = q % ROW_CHUNKS;
            if (q >= C::CHUNKS) break;
            uint4 u = lds128(base + C::OFF_RAW + raw * C::RAW + q * 16);
            if (!(present >> (r >> 4) & 1)) u = make_uint4(0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u);
            const uint32_t row = tile + (ch >> 2) * C::KV_PANEL + r * 128;
            const int at = (ch & 3) * 2;
            const bool swap = HD == 128 && (ch & 4);  // the second panel's lanes start with their odd chunk: no bank twice
            uint4 lo = make_uint4(codes_lo(u.x), codes_hi(u.x), codes_lo(u.y), codes_hi(u.y));
            uint4 hi = make_uint4(codes_lo(u.z), codes_hi(u.z), codes_lo(u.w), codes_hi(u.w));
            if (swap) {
              const uint4 x = lo;
              lo = hi;
              hi = x;
            }
            sts128(row + ((at + swap) ^ (r & 7)) * 16, lo.x, lo.y, lo.z, lo.w);
            sts128(row + ((at + !swap) ^ (r & 7)) * 16, hi.x, hi.y, hi.z, hi.w);
          }
        };
        int page = page_of(0);
        fetch(0, page, c.k, 0);
        fetch(0, page, c.v, 1);
        int next = page_of(1);
        for (int i = 0; i < p.n; i++, done++) {
          const int st = done % STAGES;
          const uint32_t present = __ballot_sync(0xffffffffu, page >= 0);
          float ks = 0.f, vs = 0.f;
          if (page >= 0) {
            ks = c.ks[(long long)page * c.kv_heads + p.head];
            vs = c.vs[(long long)page * c.kv_heads + p.head];
          }
          float top = vs;
#pragma unroll
          for (int o = 1; o < NG; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
          top = __shfl_sync(0xffffffffu, top, 0);
          if (SPLIT || top > unit * UNIT_LAG || unit == 0.f) unit = top;
          // the scales' slot was read out when P of block done - 2 was written, before this stage was freed
          if (done >= STAGES && !(ok = wait_warp(B_K_FREE + st, done / STAGES - 1))) break;
          if (warp == SOFTMAX_WARPS) {
            Scales &sc = scales[done % SCALE_STAGES];
            if (lane < NG) {
              const float share = vs > 0.f ? vs / unit : 0.f;
              sc.ks[lane] = ks;
              if (SPLIT) {
                sc.share[lane] = share;
              } else {  // as an exponent; below 2^-100 of the unit: as good as none
                const float e = share > 0.f ? fmaxf(log2f(share), -100.f) : 0.f;
                sc.share[lane] = e;
                sc.inv[lane] = share > 0.f ? exp2f(-e) : 1.f;
              }
            }
            if (lane == 0) {
              sc.present = present;
              sc.unit = unit;
            }
            __syncwarp();
            if (lane == 0) bar_arrive(bar(B_SCALE + done % SCALE_STAGES));
          }
          cp_wait<1>();
          convert(present, 0, base + C::OFF_K + st * C::KV_TILE);
          fetch(i + 1, next, c.k, 0);
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) bar_arrive(bar(B_K + st));
          if (done >= STAGES && !(ok = wait_warp(B_V_FREE + st, done / STAGES - 1))) break;
          cp_wait<1>();
          convert(present & __ballot_sync(0xffffffffu, vs > 0.f), 1, base + C::OFF_V + st * C::KV_TILE);
          fetch(i + 1, next, c.v, 1);
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) bar_arrive(bar(B_V + st));
          page = next;
          next = page_of(i + 2);
        }
        cp_wait<0>();
      }
    } else {
      // ---------------- products ----------------
      unsigned done = 0, pieces = 0, tile_done[2] = {0, 0};
      bool ok = true;
      while (ok && walk.next(a, p)) {
        if (lane == 0) {
          const int tiles = p.n_rows > TILE_ROWS ? 2 : 1;
          auto scores = [&](int x, int st) {
            uint32_t acc = 0;
#pragma unroll
            for (int t = 0; t < TERMS; t++)
#pragma unroll
              for (int k = 0; k < HD / 16; k++, acc = 1)
                mma_bf16(tmem + x * BK,
                         sw128_desc(base + C::OFF_Q + (x * TERMS + t) * C::Q_TILE + (k >> 2) * C::Q_PANEL + (k & 3) * 32),
                         sw128_desc(base + C::OFF_K + st * C::KV_TILE + (k >> 2) * C::KV_PANEL + (k & 3) * 32),
                         idesc_f16(TILE_ROWS, BK, false), acc);
            mma_commit(bar(B_S + x));
          };
          auto output = [&](int x, int st, bool first) {
            uint32_t acc = SPLIT || first ? 0 : 1;
#pragma unroll
            for (int t = 0; t < TERMS; t++)
#pragma unroll
              for (int k = 0; k < BK / 16; k++, acc = 1)
                mma_bf16_ts(tmem + TM_O + x * 128, tmem + x * BK + t * (BK / 2) + k * 8,
                            mn_desc(base + C::OFF_V + st * C::KV_TILE + k * 2048, C::KV_PANEL),
                            idesc_f16(TILE_ROWS, HD, true), acc);
          };
          ok = wait(B_Q, pieces);
          for (int i = 0; ok && i < p.n; i++, done++) {
            const int st = done % STAGES;
            if (i == 0) {
              if (!(ok = wait(B_K + st, done / STAGES))) break;
              fence_after();
              for (int x = 0; x < tiles; x++) scores(x, st);
              mma_commit(bar(B_K_FREE + st));
            }
            const int st1 = (done + 1) % STAGES;
            for (int x = 0; x < tiles; x++) {
              if (!(ok = wait(B_P + x, tile_done[x]))) break;
              tile_done[x]++;
              if (x == 0 && !(ok = wait(B_V + st, done / STAGES))) break;
              fence_after();
              output(x, st, i == 0);
              if (i + 1 < p.n) {
                if (x == 0 && !(ok = wait(B_K + st1, (done + 1) / STAGES))) break;
                fence_after();
                scores(x, st1);
              } else {
                mma_commit(bar(B_O + x));
              }
            }
            if (!ok) break;
            mma_commit(bar(B_V_FREE + st));
            if (i + 1 < p.n) mma_commit(bar(B_K_FREE + st1));
          }
          pieces++;
        }
        ok = __shfl_sync(0xffffffffu, ok, 0);
        __syncwarp();
      }
      if (lane == 0) {  // every product done before the columns are freed
        mma_commit(bar(B_FIN));
        bar_drain(bar(B_FIN), 0u);
      }
      __syncwarp();
    }
  } else {
    // ---------------- softmax and output: one thread a row ----------------
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(SOFTMAX_REGS));
    const int x = warp >> 2, r = tid & (TILE_ROWS - 1), row = x * TILE_ROWS + r;
    const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
    const uint32_t s_col = tmem + lanes + x * BK, o_col = tmem + lanes + TM_O + x * 128;
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
    unsigned done = 0, tile_done = 0, outs = 0;
    while (walk.next(a, p)) {
      // ---- the row's query as f16 terms in the swizzled tile
      const int tok = p.first_tok + row / a.group, h = p.head * a.group + row % a.group;
      const bool live = row < p.n_rows;
      const T *src = a.q + (long long)(p.s.first + (live ? tok : 0)) * a.qs + (live ? h : 0) * HD;
      const float sign = a.scale < 0.f ? -1.f : 1.f;  // the factor of the scores is then not negative: maxima commute
      float top = 0.f;
      bool finite = true;
#pragma unroll 8
      for (int d = 0; d < HD; d += 4) {
        const float4 v = live ? load4(src + d) : make_float4(0.f, 0.f, 0.f, 0.f);
        const float m4 = fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w)));
        top = fmaxf(top, m4);
        finite &= fabsf(v.x) <= FLT_MAX && fabsf(v.y) <= FLT_MAX && fabsf(v.z) <= FLT_MAX && fabsf(v.w) <= FLT_MAX;
      }
      const int e = row_exp(top);
      const float up = row_factor(e, finite) * sign, cf = scalbnf(fabsf(a.scale), -e);
#pragma unroll 4
      for (int d = 0; d < HD; d += 8) {
        const float4 v = live ? load4(src + d) : make_float4(0.f, 0.f, 0.f, 0.f);
        const float4 w = live ? load4(src + d + 4) : make_float4(0.f, 0.f, 0.f, 0.f);
        const float y[8] = {v.x * up, v.y * up, v.z * up, v.w * up, w.x * up, w.y * up, w.z * up, w.w * up};
        uint32_t f[4], g[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
          f[j] = pack(y[2 * j], y[2 * j + 1]);
          const float2 hi = unpack(f[j]);
          g[j] = pack(y[2 * j] - hi.x, y[2 * j + 1] - hi.y);
        }
        const uint32_t dst = base + C::OFF_Q + x * TERMS * C::Q_TILE + (d >> 6) * C::Q_PANEL + r * 128 +
                             (((d >> 3) & 7) ^ (r & 7)) * 16;
        sts128(dst, f[0], f[1], f[2], f[3]);
        if (SPLIT) sts128(dst + C::Q_TILE, g[0], g[1], g[2], g[3]);
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) bar_arrive(bar(B_Q));

      const bool active = x == 0 || p.n_rows > TILE_ROWS;
      const int pos = live ? p.s.len - p.s.n + tok : -1;
      const int warp_row = x * TILE_ROWS + 32 * (warp & 3);  // rows of the warp: for the test whether to mask
      const int min_pos = p.s.len - p.s.n + p.first_tok + warp_row / a.group;
      const int max_pos = p.s.len - p.s.n + p.first_tok + (warp_row + 31) / a.group;
      float o[SPLIT ? HD : 1], ref = -INFINITY, l = 0.f, unit = 0.f;
      if constexpr (SPLIT) {
#pragma unroll
        for (int d = 0; d < HD; d++) o[d] = 0.f;
      }
      bool ok = true;
      auto add_output = [&]() {  // f32 rows: o += unit * O of the last block
        if constexpr (SPLIT) {
#pragma unroll
          for (int d = 0; d < HD; d += 32) {
            float v[32];
            tmem_ld32(o_col + d, v);
            tmem_ready<32>(v);
#pragma unroll
            for (int j = 0; j < 32; j++) o[d + j] = fmaf(v[j], unit, o[d + j]);
          }
        }
      };
      for (int i = 0; i < p.n; i++, done++) {
        if (!active) continue;
        if (!(ok = wait_warp(B_SCALE + done % SCALE_STAGES, done / SCALE_STAGES))) break;
        if (!(ok = wait_warp(B_S + x, tile_done))) break;
        tile_done++;
        fence_after();
        if (SPLIT && i) add_output();
        const Scales &sc = scales[done % SCALE_STAGES];
        float s[BK];
#pragma unroll
        for (int k = 0; k < BK; k += 32) tmem_ld32(s_col + k, s + k);
        tmem_ready<BK>(s);
        const int key0 = p.block(p.t0 + i) * BK;
        const uint32_t present = sc.present;
        if (key0 + BK - 1 > min_pos || (a.window && key0 <= max_pos - a.window && key0 + BK > a.sinks) ||
            (present & ((1u << NG) - 1)) != (1u << NG) - 1) {
          const int low = a.window ? pos - a.window : -1;  // seen: low < key <= pos, or a sink
#pragma unroll
          for (int k = 0; k < BK; k++) {
            const int key = key0 + k;
            if (key > pos || (key <= low && key >= a.sinks) || !(present >> (k >> 4) & 1)) s[k] = -INFINITY;
          }
        }
        float mx = -INFINITY;
#pragma unroll
        for (int g = 0; g < NG; g++) {
          float m2[2] = {s[16 * g], s[16 * g + 1]};
#pragma unroll
          for (int k = 2; k < 16; k++) m2[k & 1] = fmaxf(m2[k & 1], s[16 * g + k]);
          const float m1 = fmaxf(m2[0], m2[1]);
          mx = fmaxf(mx, m1 == -INFINITY ? m1 : m1 * (cf * sc.ks[g]));
        }
        // the reference follows the maximum, the unit the block's: earlier results move along
        float alpha = 1.f;
        if (mx > ref + REF_LAG) {  // also the first key that a row sees: alpha = 0
          alpha = ex2(ref - mx);
          ref = mx;
        }
        float move = alpha;
        if (!SPLIT && unit != sc.unit) move *= sc.unit > 0.f ? unit / sc.unit : 0.f;
        unit = sc.unit;
        l *= alpha;
        if (i && __any_sync(0xffffffffu, move != 1.f)) {
          if constexpr (SPLIT) {
#pragma unroll
            for (int d = 0; d < HD; d++) o[d] *= move;
          } else {
#pragma unroll 1
            for (int d = 0; d < HD; d += 32) {
              float v[32];
              tmem_ld32(o_col + d, v);
              tmem_ready<32>(v);
              uint32_t u[32];
#pragma unroll
              for (int j = 0; j < 32; j++) u[j] = __float_as_uint(v[j] * move);
#pragma unroll
              for (int j = 0; j < 32; j += 8) tmem_st8(o_col + d + j, u + j);
            }
          }
        }
        const float shift = ref == -INFINITY ? 0.f : WEIGHT_EXP - ref;
        // weights into the columns that held the scores (this thread has read them all)
        float sum[2] = {0.f, 0.f};
#pragma unroll
        for (int g = 0; g < NG; g++) {
          const float f = fmaxf(cf * sc.ks[g], FLT_MIN), share = sc.share[g];  // not 0: hidden scores are -infinity
          uint32_t hi[8], lo[8];
          if constexpr (SPLIT) {
#pragma unroll
            for (int k = 0; k < 8; k++) {
              float u = ex2(fmaf(s[16 * g + 2 * k], f, shift)), v = ex2(fmaf(s[16 * g + 2 * k + 1], f, shift));
              sum[0] += u;
              sum[1] += v;
              u *= share;
              v *= share;
              hi[k] = pack(u, v);
              const float2 w = unpack(hi[k]);
              lo[k] = pack(u - w.x, v - w.y);
            }
            tmem_st8(s_col + 8 * g, hi);
            tmem_st8(s_col + BK / 2 + 8 * g, lo);
          } else {
            const float sh = shift + share;
            float gs[2] = {0.f, 0.f};
#pragma unroll
            for (int k = 0; k < 8; k++) {
              const float u = ex2(fmaf(s[16 * g + 2 * k], f, sh)), v = ex2(fmaf(s[16 * g + 2 * k + 1], f, sh));
              gs[0] += u;
              gs[1] += v;
              hi[k] = pack(u, v);
            }
            sum[0] = fmaf(gs[0] + gs[1], sc.inv[g], sum[0]);
            tmem_st8(s_col + 8 * g, hi);
          }
        }
        l += sum[0] + sum[1];
        tmem_wait_st();
        fence_before();
        __syncwarp();
        if (lane == 0) bar_arrive(bar(B_P + x));
      }
      // ---- the last block's output
      if (ok && active && p.n) {
        ok = wait_warp(B_O + x, outs);
        outs++;
        fence_after();
        if (ok) add_output();
      }
      if (!all_ok(ok)) break;
      const bool none = !active || !p.n;  // nothing was computed: l = 0, O is not the tile's
      T *dst = a.out + (long long)(p.s.first + tok) * a.os + h * HD;
      auto write = [&](int d, const float *v) {  // 32 values
        if (!live) return;
#pragma unroll
        for (int j = 0; j < 32; j += 4) store4(dst + d + j, make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]));
      };
      float *slot = a.part + (size_t)p.slot * C::SLOT;  // [head_dim][rows], maxima, sums
      const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
      for (int d = 0; d < HD; d += 32) {
        float v[32];
        if constexpr (SPLIT) {
#pragma unroll
          for (int j = 0; j < 32; j++) v[j] = o[d + j];
        } else {
          tmem_ld32(o_col + d, v);
          tmem_ready<32>(v);
#pragma unroll
          for (int j = 0; j < 32; j++) v[j] = none ? 0.f : v[j] * unit;
        }
        if (p.whole) {
#pragma unroll
          for (int j = 0; j < 32; j++) v[j] = l == 0.f ? 0.f : v[j] * inv;
          write(d, v);
        } else {
#pragma unroll
          for (int j = 0; j < 32; j++) slot[(d + j) * ROWS + row] = v[j];
        }
      }
      if (!p.whole) {  // the last block to arrive joins all parts, in block order
        slot[HD * ROWS + row] = ref;
        slot[(HD + 1) * ROWS + row] = l;
        int *count = a.count + ((long long)p.b * c.kv_heads + p.head) * a.max_row_tiles + p.rt;
        const int parts = p.parts;
        __threadfence();
        all_ok(true);
        if (tid == 0) s_last = atomicAdd(count, 1) == parts - 1;
        all_ok(true);
        if (s_last) {
          __threadfence();
          auto part = [&](int i) {
            return a.part + (size_t)(2 * (p.first + i) + (i == 0 && p.late ? 1 : 0)) * C::SLOT + row;
          };
          float top = -INFINITY, sum = 0.f;
          for (int i = 0; i < parts; i++) top = fmaxf(top, __ldcg(part(i) + HD * ROWS));
          const float at0 = top == -INFINITY ? 0.f : top;
          for (int i = 0; i < parts; i++)
            sum = fmaf(__ldcg(part(i) + (HD + 1) * ROWS), ex2(__ldcg(part(i) + HD * ROWS) - at0), sum);
          const float all_inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll 1
          for (int d = 0; d < HD; d += 32) {
            float v[32];
#pragma unroll
            for (int j = 0; j < 32; j++) v[j] = 0.f;
            for (int i = 0; i < parts; i++) {
              const float *x0 = part(i);
              const float f = ex2(__ldcg(x0 + HD * ROWS) - at0);
#pragma unroll
              for (int j = 0; j < 32; j++) v[j] = fmaf(__ldcg(x0 + (d + j) * ROWS), f, v[j]);
            }
#pragma unroll
            for (int j = 0; j < 32; j++) v[j] = sum == 0.f ? 0.f : v[j] * all_inv;
            write(d, v);
          }
          if (tid == 0) *count = 0;
        }
      }
    }
  }
  fence_before();
  __syncthreads();
  if (warp == WARPS - 1) {
    fence_after();
    tmem_dealloc(tmem, TM_COLS);
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
    int sms = 0;
    if ((e = cudaFuncSetAttribute(k_paged_many<C, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM)) !=
            cudaSuccess ||
        (e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev)) != cudaSuccess)
      return e;
    blocks[dev] = min(sms, MAX_BLOCKS);
  }
  a.max_row_tiles = many_row_tiles(a.b.max_new, a.group);
  k_paged_many<C, T><<<blocks[dev], THREADS, C::SMEM, s>>>(a);
  return cudaGetLastError();
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
