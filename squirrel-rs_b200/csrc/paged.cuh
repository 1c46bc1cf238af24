// paged.cuh — the paged 8-bit key/value cache as the kernels see it, and the reading of
// one step's batch with every index checked.
//
// A page holds `page` consecutive positions of one sequence for every kv head:
// codes [n_pages][n_kv_heads][page][head_dim], one f32 scale per page and kv head for K
// and one for V; value = (code - 128) * scale with codes 1..255. The codes are biased so
// that they become f16 numbers with one byte permute (0x6400 | code = 1024 + code) and
// one packed subtraction of 1152.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "status.h"

namespace sq {
namespace paged {

// What a kernel found wrong in device memory (the batch's arrays), where the host cannot
// look without waiting for the GPU. Kept in one word per device, read by sq_paged_status.
enum : unsigned {
  BAD_PAGE = 1,      // page id outside the cache: its positions count as masked
  BAD_LENGTH = 2,    // kv_len negative or beyond the page table's row
  BAD_START = 4,     // q_start not ascending from 0 to n_tokens, or more than max_new tokens of a sequence
  BAD_POSITION = 8,  // a new token before position 0 or past the rotation table
  BAD_WAIT = 16,     // a bounded wait gave up
};

struct Cache {
  uint8_t *k, *v;
  float *ks, *vs;
  int n_pages, kv_heads, page, page_shift, hd;
};
struct Batch {
  const int *q_start, *kv_len, *table;
  int n_seqs, n_tokens, max_new, table_row;
  unsigned *err;
};

struct Seq {
  int first;  // row of its first new token
  int n;      // new tokens
  int len;    // positions held after the step
};

__device__ __forceinline__ void flag(unsigned *err, unsigned what) { atomicOr(err, what); }

__device__ __forceinline__ Seq load_seq(const Batch &b, const Cache &c, int i) {
  Seq s;
  const int a = b.q_start[i], e = b.q_start[i + 1], l = b.kv_len[i];
  s.first = min(max(a, 0), b.n_tokens);
  s.n = min(max(min(e, b.n_tokens) - s.first, 0), b.max_new);
  s.len = (int)min((long long)max(l, 0), (long long)b.table_row << c.page_shift);
  // rows before the first sequence's or after the last one's would stay as they are
  if (s.first != a || s.n != e - a || (i == 0 && a != 0) || (i + 1 == b.n_seqs && e != b.n_tokens)) flag(b.err, BAD_START);
  if (s.len != l) flag(b.err, BAD_LENGTH);
  return s;
}

// Page that holds position `pos` of sequence i, or -1 (recorded) when the table names none.
__device__ __forceinline__ int load_page(const Batch &b, const Cache &c, int i, int pos) {
  const int p = b.table[(long long)i * b.table_row + (pos >> c.page_shift)];
  if ((unsigned)p < (unsigned)c.n_pages) return p;
  flag(b.err, BAD_PAGE);
  return -1;
}

// Sequence of token row t (rows ascend with the sequences; those without new tokens hold
// none). One new token a sequence, the decode step, is tried first.
__device__ __forceinline__ int seq_of_token(const Batch &b, int t) {
  if (t < b.n_seqs && b.q_start[t] == t && b.q_start[t + 1] == t + 1) return t;
  int lo = 0, hi = b.n_seqs - 1;  // the last sequence whose first row is <= t
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (b.q_start[mid] <= t) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// Four consecutive elements of a row, f32 or bf16, as f32.
__device__ __forceinline__ float4 load4(const float *p) { return *reinterpret_cast<const float4 *>(p); }
__device__ __forceinline__ float4 load4(const __nv_bfloat16 *p) {
  const uint2 u = *reinterpret_cast<const uint2 *>(p);
  return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xFFFF0000u), __uint_as_float(u.y << 16),
                     __uint_as_float(u.y & 0xFFFF0000u));
}
__device__ __forceinline__ void store4(float *p, float4 v) { *reinterpret_cast<float4 *>(p) = v; }
__device__ __forceinline__ void store4(__nv_bfloat16 *p, float4 v) {
  const __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
  *reinterpret_cast<uint2 *>(p) =
      make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
}

constexpr long long MAX_POSITIONS = 1 << 30;  // of a page table's row: sums of positions, tiles and pages fit 32 bits

unsigned *err_ptr();  // device address of the current device's word (null: no such device)
// Checked copies of the caller's structs (Batch::err left to the caller, who sets it to
// err_ptr() once every check that needs no GPU has passed); SQ_OK or the status.
int check_cache(const sq_paged_cache *c, Cache *out, const char *what);
int check_batch(const sq_paged_batch *b, const Cache &c, Batch *out, const char *what);
// Rows [n][width] of `dtype` at p with `stride` elements between them: 16-byte aligned throughout.
int check_rows(const void *p, long long stride, long long width, int dtype, const char *what);

}  // namespace paged
}  // namespace sq
