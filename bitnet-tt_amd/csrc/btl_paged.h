// The paged key-value cache and a batch of packed new tokens, shared by the
// kernels that write, read and attend over it.
//
// Pages: [P, Hkv, ps, D] bf16, or e4m3 codes with one exponent byte per page
// row ([P, Hkv, ps]).  Position p of sequence b is row p % ps of page
// table[b][p / ps].  ps is a multiple of 16, so 16 consecutive positions from
// a multiple of 16 lie in one page.  A contiguous cache [B, Hkv, S, D] is the
// special case ps = S with page b for sequence b.
//
// Batch: rows cu[b] .. cu[b+1] of the packed tensors are the newest tokens of
// sequence b, at positions len[b] - n .. len[b] - 1.  What the device arrays
// hold is not known on the host, so every kernel clamps it: no index leaves
// its buffer whatever they hold, and what had to be clamped sets the error
// word.
#pragma once

#include "btl_common.h"

namespace btl {

constexpr int kMaxPageSize = 1 << 20;
constexpr int kMaxRows = 1 << 24;  // packed rows of a batch
constexpr int kMaxSeqs = 1 << 20;

// n / d for n < 2^31 by a multiplication: m = ceil(2^(31+l) / d), l = ceil(log2 d);
// the excess e = m d - 2^(31+l) is below d <= 2^l, so n e < 2^(31+l) and the
// quotient is exact.
struct FastDiv {
  uint32_t d, m, s;
};
inline FastDiv fast_div(uint32_t d) {  // d >= 2
  uint32_t l = 1;
  while ((1ull << l) < d) ++l;
  return {d, (uint32_t)(((1ull << (31 + l)) + d - 1) / d), l - 1};
}
__host__ __device__ __forceinline__ uint32_t div_by(uint32_t n, const FastDiv& f) {
  return (uint32_t)(((uint64_t)n * f.m) >> 32) >> f.s;
}

struct Pages {
  uint8_t* k;
  uint8_t* v;
  uint8_t* ke;  // exponent bytes, 8-bit pages only
  uint8_t* ve;
  int P, Hkv;
  FastDiv ps;
};

struct Batch {
  const int32_t* cu;     // [B + 1]
  const int32_t* len;    // [B] (NULL: the new tokens are all there is)
  const int32_t* table;  // [B][max_pages]
  int B, T, max_pages;
};

// A sequence as the kernels use it: rows row0 .. row0 + n of the packed
// tensors, len positions; ok: nothing had to be clamped.
struct Seq {
  int row0, n, len;
  bool ok;
};
__host__ __device__ __forceinline__ int clampi(int x, int lo, int hi) { return x < lo ? lo : x > hi ? hi : x; }
// cap: the positions that the page table has room for; negative: no lengths are
// given, the sequence is its rows (as clamped: row0 + len is at most T).
__host__ __device__ __forceinline__ Seq clamp_seq(int lo, int hi, int len, int T, int64_t cap) {
  Seq s;
  s.row0 = clampi(lo, 0, T);
  s.n = clampi(hi, s.row0, T) - s.row0;
  s.ok = s.row0 == lo && s.row0 + s.n == hi;
  if (cap < 0) {
    s.len = s.n;
  } else {
    s.len = (len < 0 || len > cap) ? 0 : len;  // a length that cannot be: nothing is cached
    s.ok = s.ok && s.len == len;
  }
  return s;
}

// Where a position's row lies: index of its (page, head, row), or -1 where
// the table holds no page of the pool.
__host__ __device__ __forceinline__ int64_t page_row(int32_t page, int P, int Hkv, int hk, int ps, int row) {
  return (page < 0 || page >= P) ? -1 : ((int64_t)page * Hkv + hk) * ps + row;
}

// A run of rows in a pool: index of the first, how many there are (none behind
// kv_end, none in a page outside the pool).  Scalars, without a branch.
struct Run {
  int64_t row;
  uint32_t n;
};
__host__ __device__ __forceinline__ Run run_at(const Pages& pg, int hk, int at, int kv_end, int32_t page, int most, bool& bad) {
  const int left = clampi(kv_end - at, 0, most);
  const bool none = (uint32_t)page >= (uint32_t)pg.P;
  bad |= none & (left > 0);
  const uint32_t id = none ? 0u : (uint32_t)page, ps = pg.ps.d;
  const uint32_t in_page = (uint32_t)at - div_by((uint32_t)at, pg.ps) * ps;
  return {(int64_t)((uint64_t)id * (uint32_t)(pg.Hkv * ps)) + (uint32_t)(hk * ps + in_page), none ? 0u : (uint32_t)left};
}

// ---- e4m3 rows with a power of two ---------------------------------------
// Exponent of a row with largest magnitude a > 0: the least e >= -126 with
// a <= 448 * 2^e (448 = 1.75 * 2^8 is the largest code).  Scaling by a power
// of two is exact and costs an e4m3 code no precision, so a value is rounded
// once, and a code times 2^e has few enough bits to be a bf16 value.
__host__ __device__ __forceinline__ int row_exponent(float a) {
  const uint32_t u = __builtin_bit_cast(uint32_t, a);
  const int e = (int)(u >> 23) - 127;  // a = 1.f * 2^e (a subnormal a is below every bound)
  const int r = (u & 0x7fffffu) <= 0x600000u ? e - 8 : e - 7;
  return r < -126 ? -126 : r;
}

#if defined(__HIP_DEVICE_COMPILE__) || defined(__HIPCC__)
__device__ __forceinline__ void flag_error(int32_t* error) {
  __hip_atomic_store(error, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

__device__ __forceinline__ int uni(int x) { return __builtin_amdgcn_readfirstlane(x); }

// A word that no kernel running beside this one writes, at an index that is
// the same in every lane: a scalar load, which no vector load waits for.
__device__ __forceinline__ int32_t scalar_load(const int32_t* p, uint32_t i) {
  return ((const __attribute__((address_space(4))) int32_t*)p)[i];
}

__device__ __forceinline__ Seq load_seq(const Batch& bt, int b, int64_t cap) {
  const int lo = scalar_load(bt.cu, b), hi = scalar_load(bt.cu, b + 1);
  Seq s = clamp_seq(lo, hi, bt.len ? scalar_load(bt.len, b) : 0, bt.T, bt.len ? cap : -1);
  s.row0 = uni(s.row0);
  s.n = uni(s.n);
  s.len = uni(s.len);
  return s;
}

// Item x of the sequences' items, sequence b having ceil(n_b * per / of): the
// sequence and the item's number in it.  Every wave searches by itself, 64
// sequences a step.  False where there are fewer items.  A workgroup checks the sequences
// that it passes, item 0's all of them: one that gives no item has no other reader.
struct Item {
  int b, i, count;
};
__device__ __forceinline__ bool find_item(const Batch& bt, int per, int of, int x, Item& it, int32_t* error) {
  const int lane = __lane_id();
  int base = 0;
  bool found = false, ok = true;
  for (int c = 0; c < bt.B; c += 64) {
    const int b = c + lane;
    Seq s{0, 0, 0, true};
    if (b < bt.B) s = clamp_seq(bt.cu[b], bt.cu[b + 1], 0, bt.T, 0);
    ok &= s.ok;
    if (found) continue;
    const int n = s.n;
    const int cnt = (n * per + of - 1) / of;
    int inc = cnt;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int y = __shfl_up(inc, d);
      if (lane >= d) inc += y;
    }
    const int total = __builtin_amdgcn_readlane(inc, 63);
    if (x < base + total) {
      const int l = __builtin_ctzll(__ballot(base + inc > x));
      it.b = uni(c + l);
      it.count = __builtin_amdgcn_readlane(cnt, l);
      it.i = uni(x - base - (__builtin_amdgcn_readlane(inc, l) - it.count));
      found = true;
      if (x > 0) break;
    }
    base += total;
  }
  if (!ok) flag_error(error);
  return found;
}
#endif

// Host-side checks of the public structs (btl_paged.hip).
int check_pages(const char* who, const btl_pages_t* p, Pages* out);
int check_batch(const char* who, int64_t B, int64_t T, const int32_t* cu_q, const int32_t* kv_len,
                const int32_t* page_table, int64_t max_pages, Batch* out);

}  // namespace btl
