// Attention of packed rows: within prompts (keys and values of the same
// packed sequences), or over the pages of a cache.
//
//   out_i = sum_j softmax_j(c q_i.k_j) v_j,  j up to row i's own position (kCausal), of these
//   the last `window` and the first `sinks` (kWindow), or in two parts: the pages that every
//   sequence of the batch begins with, for the rows of all of them together (kShared), and
//   the positions behind those (kOwn)
//
// Rows of one sequence and key-value head are its tokens' G query heads, token
// by token (row r = token r / G, head r % G): they all read the same keys, so a
// tile of rows fetches a key once for the G heads, and a short chunk still
// fills a tile.
//
// Both kernels compute the transposed scores S^T = K Q^T: an MFMA's result
// then has one row of queries per lane column, so a lane holds many scores of
// one query, and the maximum and sum are sums in registers with one or two lane
// exchanges.  Its C layout is, up to the order of the positions, the B
// layout of P^T in O^T = V^T P^T: the probabilities never leave their lane, and
// the order is made up for where V is read (transposing LDS reads of row
// groups in the same order).
//
// Softmax in base 2: p = 2^(c' s - m), c' = c log2(e), in fp32; m, a whole number,
// is raised to the running maximum's ceiling only where that is more than kLazy
// above it (p then stays below 2^kLazy, which costs an fp32 sum nothing), and the
// factors that this puts on what has been summed are powers of two: exact.  p is
// rounded to bf16 for the second product, the matrix units' operand type, and the
// sum takes the same rounded values, so the weights that are used sum to one (few rows over bf16
// pages: 16 bits of p; not in the tiles of a shared prefix).  Two bf16 values of p in the tiles as well, a second product on the same values,
// measured: 4096 tokens 100 us, 136 so; 16001 415, 565; chunks of 4 users over up to 8000 139, 187; 67
// tokens over 40067 8-bit positions 62, 73.  Against 64 bits the one value costs 0.0020-0.0022 of the
// outputs' size where their own rounding has 0.0016.
//
// Rows of V behind the last position read as zero (whatever lies there), and a
// value that is not finite at a position that some of the tile's rows may not see is added
// to the rows that do see it and multiplied with none: 0 x inf is NaN.
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "btl.h"
#include "btl_act_row.h"
#include "btl_common.h"
#include "btl_fp8.h"
#include "btl_paged.h"

namespace btl {

typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef short v8s __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) uint8_t lds8;

enum { kDense = 0, kPagedBf16 = 1, kPagedFp8 = 2 };
enum { kCausal = 0, kWindow = 1, kShared = 2, kOwn = 3 };

constexpr float kLazy = 8.0f;
constexpr float kWhole = -1.0f;
constexpr float kNone = -2.0f;
constexpr float kNegInf = -__builtin_inff();

struct FlashArgs {
  const uint16_t* q;
  const uint16_t* k;  // dense
  const uint16_t* v;
  int64_t ldq, ldk, ldv, ldo;
  Pages pg;
  Batch bt;
  int H, Hkv, G;
  FastDiv g;        // G, where G > 1
  float c;          // scale * log2(e)
  uint16_t* out;
  int32_t* error;
  // splits > 1: workgroup z takes positions [z chunk, (z + 1) chunk), the last
  // split the rest, and leaves a partial per row; a sequence of at most chunk
  // positions is workgroup 0's alone, which writes the output and marks the row
  // (the sum of its first partial is kWhole)
  int splits, chunk;
  float* part_o;    // [splits][T][H][D]
  float2* part_ml;  // [splits][T][H]: exponents' offset, sum
  // kWindow: the row at position p sees (p - window, p] and, up to p, [0, sinks)
  int window, sinks;
  int neighbours;  // tiles of a head that run on one XCD, one after the other
  // kShared, kOwn: pages of the shared prefix (device).  Every row has shared_splits partials of
  // the prefix, then `splits` of its own positions; the sum of a row that sees nothing is kNone there.
  const int32_t* shared;
  int shared_splits, shared_chunk;
};

// What some of a tile's rows see through their windows, as one axis: the sinks (over pages, in whole
// steps), then from `lo`, the first position of the first row's window, on.  `gap` positions that no
// row sees lie between the two; they are not loaded, nor are their pages looked up.
struct Span {
  int lo, sinks, end;  // positions: end is behind the last
  int turn, gap;       // the axis leaves the sinks at `turn`
  // step: what `turn`, and align: what a step's first position must be a multiple of; powers of two
  __device__ __forceinline__ void init(const FlashArgs& p, int first_row, int end_, int step, int align) {
    lo = uni(max(0, first_row - p.window + 1));
    sinks = p.sinks;
    end = end_;
    turn = (sinks + step - 1) & -step;
    gap = uni(max(0, (lo & -align) - turn));
  }
  __device__ __forceinline__ int pos(int u) const { return u < turn ? u : u + gap; }
  // Whether a step has both sinks and positions of the windows (rows that are packed: any of them).
  __device__ __forceinline__ bool mixed(int u, int n) const { return gap > 0 && u < turn && u + n > turn; }
  // Where the positions that are to be loaded end, of n from `at`.
  __device__ __forceinline__ int end_of(int at, int n) const { return at + n <= lo ? sinks : end; }
};

// Positions of the shared prefix; not ok: no number of pages that a table row can hold.
__device__ __forceinline__ int shared_len(const FlashArgs& p, bool& ok) {
  const int pages = scalar_load(p.shared, 0);
  ok = pages >= 0 && pages <= p.bt.max_pages;
  return ok ? pages * (int)p.pg.ps.d : 0;
}

// A sequence as the kernels of a mode use it, `begin` the first position that its rows read.
template <int MODE>
__device__ __forceinline__ Seq mode_seq(const FlashArgs& p, int b, int& begin, bool first_group) {
  const int64_t cap = (int64_t)p.bt.max_pages * p.pg.ps.d;
  begin = 0;
  if (MODE == kShared) {  // every row of the batch; what is wrong with it is kOwn's to find
    bool ok;
    Seq s = clamp_seq(scalar_load(p.bt.cu, 0), scalar_load(p.bt.cu, p.bt.B), 0, p.bt.T, 0);
    s.row0 = uni(s.row0);
    s.n = uni(s.n);
    s.len = uni(shared_len(p, ok));
    return s;
  }
  Seq s = load_seq(p.bt, b, cap);
  if (MODE == kOwn) {
    bool ok;
    begin = uni(shared_len(p, ok));
    // rows before the prefix's end (but for padding, which sees nothing)
    s.ok &= ok & !(s.n > 0 && s.len > 0 && begin > 0 && s.len - s.n < begin);
  }
  if (!s.ok && first_group) flag_error(p.error);
  return s;
}

// The positions that a row sees end with `limit`; -1: it sees none.
template <int MODE>
__device__ __forceinline__ bool sees(const FlashArgs& p, int limit, int j) {
  return j <= limit && (MODE != kWindow || j > limit - p.window || j < p.sinks);
}
// Whether rows whose limits are in [lo, hi] all see, or some of them may see, positions a .. a + n - 1.
template <int MODE>
__device__ __forceinline__ bool all_see(const FlashArgs& p, int lo, int hi, int a, int n) {
  return a + n - 1 <= lo && (MODE != kWindow || a > hi - p.window || a + n <= p.sinks);
}
template <int MODE>
__device__ __forceinline__ bool some_see(const FlashArgs& p, int lo, int hi, int a, int n) {
  return a <= hi && (MODE != kWindow || a + n - 1 > lo - p.window || a < p.sinks);
}

// l plus both bf16 values of a pair, in 32 bits (one instruction).
__device__ __forceinline__ float sum_pair(uint32_t two, float l) {
  typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
  return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(v2bf, two), __builtin_bit_cast(v2bf, 0x3f803f80u), l, false);
}

// No score of a row so far (a NaN score leaves the maximum alone, not the sum).
__device__ __forceinline__ bool empty(float m, float l) { return m == kNegInf && l == 0.0f; }

__device__ __forceinline__ int row_token(int r, const FlashArgs& p) { return p.G > 1 ? (int)div_by(r, p.g) : r; }

__device__ __forceinline__ bool not_finite(uint32_t two) {
  return ((two & 0x7f80u) == 0x7f80u) | ((two & 0x7f800000u) == 0x7f800000u);
}
__device__ __forceinline__ bool any_not_finite(uint4 x) {
  return not_finite(x.x) | not_finite(x.y) | not_finite(x.z) | not_finite(x.w);
}
__device__ __forceinline__ uint32_t drop_not_finite(uint32_t x) {
  if ((x & 0x7f80u) == 0x7f80u) x &= 0xffff0000u;
  if ((x & 0x7f800000u) == 0x7f800000u) x &= 0x0000ffffu;
  return x;
}

// Loads through a buffer resource of `bytes` bytes at a scalar address; a piece behind them reads as zero.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buf_rsrc(const uint8_t* p, uint32_t bytes) {
  const uint64_t at = reinterpret_cast<uint64_t>(p);
  const uint32_t lo = (uint32_t)uni((int)(uint32_t)at), hi = (uint32_t)uni((int)(at >> 32));
  return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(((uint64_t)hi << 32) | lo), (short)0,
                                           uni((int)bytes), 0x00020000);
}
__device__ __forceinline__ uint4 buf_ld128(__amdgpu_buffer_rsrc_t r, uint32_t off) {
  const auto v = __builtin_amdgcn_raw_buffer_load_b128(r, (int)off, 0, 0);
  return make_uint4(v[0], v[1], v[2], v[3]);
}
__device__ __forceinline__ uint32_t buf_ld8(__amdgpu_buffer_rsrc_t r, uint32_t off) {
  return (uint8_t)__builtin_amdgcn_raw_buffer_load_b8(r, (int)off, 0, 0);
}

__device__ __forceinline__ uint4 lds_ld128(const lds8* p) {
  typedef uint32_t v4u __attribute__((ext_vector_type(4)));
  const v4u v = *(const __attribute__((address_space(3))) v4u*)p;
  return make_uint4(v[0], v[1], v[2], v[3]);
}
__device__ __forceinline__ uint2 lds_ld64(const lds8* p) {
  typedef uint32_t v2u __attribute__((ext_vector_type(2)));
  const v2u v = *(const __attribute__((address_space(3))) v2u*)p;
  return make_uint2(v[0], v[1]);
}
__device__ __forceinline__ v8bf lds_ld_bf8(const lds8* p) { return *(const __attribute__((address_space(3))) v8bf*)p; }
__device__ __forceinline__ void lds_st128(lds8* p, uint4 x) {
  typedef uint32_t v4u __attribute__((ext_vector_type(4)));
  *(__attribute__((address_space(3))) v4u*)p = (v4u){x.x, x.y, x.z, x.w};
}
__device__ __forceinline__ void lds_st64(lds8* p, uint2 x) {
  typedef uint32_t v2u __attribute__((ext_vector_type(2)));
  *(__attribute__((address_space(3))) v2u*)p = (v2u){x.x, x.y};
}
// ds_read_b64_tr_b16: in each group of 16 lanes, lane j receives, for r =
// 0..3, element j % 4 of the four 16-bit values that lane 4 r + j / 4 addresses:
// with lane 4 r + q at row r, columns 4 q .. 4 q + 3, lane j gets column j of rows 0..3.
__device__ __forceinline__ v4s lds_tr16(const lds8* p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s*)p);
}

// ======================================================================
// Tiles of 128 rows: 4 waves of 32 rows each, 64 positions a step.
//
// Keys and values are in LDS as bf16, two stages of each: 64 KiB at D = 128, so two
// workgroups share a CU.  Loads go to LDS directly (8-bit pages: through
// registers, converted), one barrier a step.  The scores run one step ahead: the
// MFMAs of step j + 1's scores are independent of step j's exponentials, so
// that a wave's vector work runs under its own matrix work, and not only under the other
// workgroup's.  (The second product one step behind as well, so that nothing
// in a step depends on anything else in it: the same speed, and 30 registers more than there are.)
//
// Bound by how far one wave's matrix work covers the other's vector work on a SIMD: at
// 16001 tokens of 20 / 5 heads of 128, 390-415 us, 980-1045 TFLOP/s (a large library
// product reaches 1360), the matrix units are busy 58% of the cycles and the vector units 47%;
// reading LDS alone would take 155 us.  Over pages, 8192 tokens: 1005 TFLOP/s; 8-bit
// pages, which are converted on the way, 955.  Measured beside it, in TFLOP/s: 64 rows a wave
// and one wave a SIMD, which halves the reading of LDS, 904 with 32 positions a
// step and 860 with 64; 32 rows and 32 positions 1018; all products of a step together and all
// exponentials after them 1003, with a raised priority for the products 980; 8 waves and 256
// rows a workgroup 998, the second wave of a SIMD a phase behind the first 994; keys and
// values through registers to LDS 843.  The clock under this work is 1.83 GHz, as under the
// library's product.
//
// 16-byte pieces of a row are stored at piece ^ f(row), for the LDS's 64 banks:
// the 16 rows that 16 lanes read a piece of, and the 4 rows x 64 bytes that 32 lanes
// of a transposing read cover, lie in different banks.
// ======================================================================
constexpr int kTileRows = 128;
constexpr int kStep = 64;

template <int D>
struct Tile {
  static constexpr int kBytes = kStep * D * 2;         // one stage of K, or of V
  static constexpr int kLoads = kBytes / (256 * 16);   // 16-byte pieces of a thread for it
  static __device__ __forceinline__ int k_swz(int row) { return D == 128 ? row & 15 : (row >> 1) & 7; }
  static __device__ __forceinline__ int v_swz(int row) { return D == 128 ? (row & 3) << 2 : (row & 2) << 1; }
};

// Where a step's rows come from: the sequence's packed rows, or its pages.
// A thread's rows of a step are i * kRpl + tid / kTpr for its loads i (kTpr threads
// to a row); a wave's rows of one load are in one run of 16 positions, and so in
// one page.  An address is a buffer resource at a scalar address plus a 32-bit
// offset that a thread keeps: no vector arithmetic per load (64-bit row addresses
// per load took half as many vector cycles again as the softmax).  Rows behind the
// end, and rows in no page, are out of the resource's range: they read as zeros.
template <int D, int KV, int MODE>
struct Source {
  static constexpr int kRowBytes = KV == kPagedFp8 ? D : 2 * D;
  static constexpr int kTpr = kRowBytes / 16;      // threads of a row
  static constexpr int kRpl = 256 / kTpr;          // rows of a load
  static constexpr int kN = kStep / kRpl;          // loads of a thread
  const uint8_t* k;                                // dense: the sequence's first row
  const uint8_t* v;
  int64_t ldk, ldv;                                // dense: bytes of a row
  const int32_t* table;
  int hk, kv_end, row0, my_row;                    // the wave's first row and the thread's row in the first load
  uint32_t off_k[kN], off_v[kN];                   // of the thread's pieces, from the step's first row
  bool one;                                        // pages of whole steps
  int32_t page_k[kN], page_v[kN];                  // pages of the runs of the keys and of the values to be loaded next
  bool bad;
  Span span;                                       // kWindow
  uint4 rk[kN], rv[kN];                            // 8-bit pages: a step on its way
  uint32_t ek[kN], ev[kN];

  __device__ __forceinline__ int end_of(int at, int n) const { return MODE == kWindow ? span.end_of(at, n) : kv_end; }
  __device__ __forceinline__ int pos(int u) const { return MODE == kWindow ? span.pos(u) : u; }

  __device__ __forceinline__ void init(const FlashArgs& p, const Seq& s, int b, int hk_, int kv_end_) {
    const int tid = threadIdx.x;
    hk = hk_;
    kv_end = kv_end_;
    bad = false;
    row0 = uni(tid) / kTpr;
    my_row = tid / kTpr;
    if (KV == kDense) {
      ldk = p.ldk * 2;
      ldv = p.ldv * 2;
      k = reinterpret_cast<const uint8_t*>(p.k + (int64_t)s.row0 * p.ldk + hk * D);
      v = reinterpret_cast<const uint8_t*>(p.v + (int64_t)s.row0 * p.ldv + hk * D);
    } else {
      table = p.bt.table + (int64_t)b * p.bt.max_pages;
      one = p.pg.ps.d % kStep == 0;
    }
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      // pieces land in LDS in the order of the lanes: the order f makes is made here
      const int row = i * kRpl + tid / kTpr, c = tid % kTpr;
      off_k[i] = row * (KV == kDense ? (uint32_t)ldk : kRowBytes) + 16 * (KV == kPagedFp8 ? c : c ^ Tile<D>::k_swz(row));
      off_v[i] = row * (KV == kDense ? (uint32_t)ldv : kRowBytes) + 16 * (KV == kPagedFp8 ? c : c ^ Tile<D>::v_swz(row));
    }
  }
  // The run of 16 rows that the wave's rows of load i are in.
  __device__ __forceinline__ int run_of(int i) const { return (i * kRpl + row0) & ~15; }
  __device__ __forceinline__ void fetch_pages(const FlashArgs& p, int u, int32_t (&page)[kN]) const {
    if (KV == kDense) return;
    const int kv = pos(u);
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int at = one ? kv : kv + run_of(i);
      page[i] = 0;
      if (at < end_of(at, one ? kStep : 16) && (i == 0 || !one)) page[i] = scalar_load(table, div_by(at, p.pg.ps));
    }
  }
  // The values follow the keys by a step; the keys' next pages, of the step at kv, are fetched.
  __device__ __forceinline__ void turn_pages(const FlashArgs& p, int kv) {
    if (KV == kDense) return;
#pragma unroll
    for (int i = 0; i < kN; ++i) page_v[i] = page_k[i];
    fetch_pages(p, kv, page_k);
  }
  // The step's keys (VAL: values) to LDS (8-bit pages: to registers).
  template <bool VAL>
  __device__ __forceinline__ void load(const FlashArgs& p, int u, lds8* at) {
    lds8* const dst = at + uni(threadIdx.x >> 6) * 1024;
    const int kv = pos(u);
    if (KV == kDense) {
      const uint32_t ld = (uint32_t)(VAL ? ldv : ldk);
      if (MODE == kWindow && span.mixed(u, kStep)) {
        const uint8_t* const rows = (VAL ? v : k) + u * (VAL ? ldv : ldk);
        const int sinks = span.turn - u;  // rows of the step
        const auto s = buf_rsrc(rows, (uint32_t)sinks * ld);
        const auto w = buf_rsrc(rows + span.gap * (VAL ? ldv : ldk), (uint32_t)min(span.end - span.gap - u, kStep) * ld);
#pragma unroll
        for (int i = 0; i < kN; ++i) {
          if (i * kRpl + my_row < sinks)
            piece<VAL>(s, i, dst);
          else
            piece<VAL>(w, i, dst);
        }
        return;
      }
      const int n = MODE == kWindow ? clampi(end_of(kv, kStep) - kv, 0, kStep) : min(kv_end - kv, kStep);
      const auto r = buf_rsrc((VAL ? v : k) + kv * (VAL ? ldv : ldk), (uint32_t)n * ld);
#pragma unroll
      for (int i = 0; i < kN; ++i) piece<VAL>(r, i, dst);
      return;
    }
    const uint8_t* const pool = VAL ? p.pg.v : p.pg.k;
    const uint8_t* const exps = VAL ? p.pg.ve : p.pg.ke;
    if (one) {
      const Run run = run_at(p.pg, hk, kv, end_of(kv, kStep), VAL ? page_v[0] : page_k[0], kStep, bad);
      const auto r = buf_rsrc(pool + run.row * kRowBytes, run.n * kRowBytes);
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        piece<VAL>(r, i, dst);
        if (KV == kPagedFp8) (VAL ? ev : ek)[i] = buf_ld8(buf_rsrc(exps + run.row, run.n), i * kRpl + my_row);
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      // a run's rows, by their offsets from the step's first
      const int r0 = run_of(i);
      const Run run = run_at(p.pg, hk, kv + r0, end_of(kv + r0, 16), VAL ? page_v[i] : page_k[i], 16, bad);
      const int64_t row = run.row - r0;
      const uint32_t n = run.n ? run.n + r0 : 0;
      piece<VAL>(buf_rsrc(pool + row * kRowBytes, n * kRowBytes), i, dst);
      if (KV == kPagedFp8) (VAL ? ev : ek)[i] = buf_ld8(buf_rsrc(exps + row, n), i * kRpl + my_row);
    }
  }
  template <bool VAL>
  __device__ __forceinline__ void piece(__amdgpu_buffer_rsrc_t r, int i, lds8* dst) {
    const uint32_t off = VAL ? off_v[i] : off_k[i];
    if (KV == kPagedFp8)
      (VAL ? rv : rk)[i] = buf_ld128(r, off);
    else
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, dst + i * 4096, 16, (int)off, 0, 0, 0);
  }
  // 8-bit pages: what load() brought, converted, to LDS.
  template <bool VAL>
  __device__ __forceinline__ void store(lds8* at) const {
    if (KV != kPagedFp8) return;
    const int c = threadIdx.x % kTpr;
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int row = i * kRpl + threadIdx.x / kTpr;
      const uint4 w = (VAL ? rv : rk)[i];
      const float f = exp_scale((VAL ? ev : ek)[i]);
      const int c0 = 2 * c ^ (VAL ? Tile<D>::v_swz(row) : Tile<D>::k_swz(row));
      lds_st128(at + row * 2 * D + c0 * 16, from_e4m3(make_uint2(w.x, w.y), f));
      lds_st128(at + row * 2 * D + (c0 ^ 1) * 16, from_e4m3(make_uint2(w.z, w.w), f));
    }
  }
};

template <int D>
struct TileState {
  v8bf q[D / 16];   // B operands: this lane's query row, dims 16 ks + 8 h ..
  v16f o[D / 32];   // O^T: element r of o[t] is dim 32 t + c_row(r) of the lane's row
  float m, l[2];    // the exponents' offset (a whole number; -inf: no score yet), this lane's share of the sum
  int limit;        // the last position that the lane's row sees, -1: none
  int lo, hi;       // of the wave's rows: least limit, greatest
};

__device__ __forceinline__ int c_row(int r, int h) { return 8 * (r >> 2) + 4 * h + (r & 3); }

// The larger of the two halves' values.
__device__ __forceinline__ float half_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// Key operands of a step: positions 32 t + r32, dims 16 k + 8 h .. + 7.
template <int D>
__device__ __forceinline__ v8bf tile_key(const lds8* ks, int t, int k) {
  const int lane = __lane_id(), h = lane >> 5, r32 = lane & 31;
  return lds_ld_bf8(ks + (32 * t + r32) * 2 * D + ((Tile<D>::k_swz(r32) ^ h ^ (2 * k)) * 16));
}
// The first of them, which are read ahead of whatever is issued before the products.
constexpr int kAhead = 2;
typedef v8bf TileKeys[kAhead][2];
template <int D>
__device__ __forceinline__ void tile_keys(const lds8* ks, TileKeys& a) {
#pragma unroll
  for (int k = 0; k < kAhead; ++k)
#pragma unroll
    for (int t = 0; t < 2; ++t) a[k][t] = tile_key<D>(ks, t, k);
}
// Scores of a step: element r of sc[t] is position 32 t + c_row(r).
template <int D>
__device__ __forceinline__ void tile_scores(const lds8* ks, TileKeys& a, const TileState<D>& s, v16f (&sc)[2]) {
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) sc[t][r] = 0.0f;
#pragma unroll
  for (int k = 0; k < D / 16; ++k)
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      sc[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[k % kAhead][t], s.q[k], sc[t], 0, 0, 0);
      if (k + kAhead < D / 16) a[k % kAhead][t] = tile_key<D>(ks, t, k + kAhead);
    }
}

// The lowest n bits (n <= 0: none, n >= 32: all).
__device__ __forceinline__ uint32_t low_bits(int n) { return n >= 32 ? ~0u : (1u << max(n, 0)) - 1u; }

// (kWindow: kv is a place on the axis.)
template <int D, int MODE>
__device__ __forceinline__ void tile_mask(const FlashArgs& p, const Span& span, const TileState<D>& s, int kv, v16f (&sc)[2]) {
  const int h = __lane_id() >> 5;
  if (MODE == kWindow) {  // a bit a position: three conditions a score would want more scalar registers than there are
    const int from = (span.gap > 0 ? span.turn : span.sinks) - kv - 4 * h;  // the windows' part of the axis
    const int sink = min(s.limit + 1, span.sinks) - kv - 4 * h;
    const int end = max(s.limit + 1 - span.gap - kv - 4 * h, 0);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const uint32_t see = low_bits(sink - 32 * t) |
                           (low_bits(end - 32 * t) & ~low_bits(end - p.window - 32 * t) & ~low_bits(from - 32 * t));
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int keep = __builtin_amdgcn_sbfe((int)see, c_row(r, 0), 1);
        sc[t][r] = __int_as_float((keep & __float_as_int(sc[t][r])) | (~keep & __float_as_int(kNegInf)));
      }
    }
    return;
  }
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r)
      if (kv + 32 * t + c_row(r, h) > s.limit) sc[t][r] = kNegInf;
}

// Raises the offset where the scores of the next step need it.
template <int D>
__device__ __forceinline__ void tile_raise(TileState<D>& s, float c, const v16f (&sc)[2]) {
  float mx = sc[0][0];
#pragma unroll
  for (int i = 1; i < 32; ++i) mx = fmaxf(mx, sc[i >> 4][i & 15]);
  mx = half_max(mx) * c;
  if (__any(mx - s.m > kLazy)) {  // (from -inf: any score is more)
    const float mn = fmaxf(s.m, __builtin_ceilf(mx));
    const float a = s.m == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(s.m - mn);
    s.m = mn;
    s.l[0] *= a;
    s.l[1] *= a;
#pragma unroll
    for (int t = 0; t < D / 32; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) s.o[t][r] *= a;
  }
}

// The probabilities of a step's scores, as operands.
template <int D>
__device__ __forceinline__ void tile_exp(TileState<D>& s, float c, const v16f (&sc)[2], v8bf (&pb)[4]) {
  const float mc = s.m == kNegInf ? 0.0f : -s.m;
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float e0 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t][8 * k + 2 * j], c, mc));
        const float e1 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t][8 * k + 2 * j + 1], c, mc));
        w[j] = f2bf_pair(e0, e1);
        s.l[k] = sum_pair(w[j], s.l[k]);
      }
      pb[2 * t + k] = __builtin_bit_cast(v8bf, make_uint4(w[0], w[1], w[2], w[3]));
    }
}

// (__restrict__: a transposing read carries no alias information of its own, and the compiler
// would wait for every load into LDS that is on its way before one.)
template <int D>
__device__ __forceinline__ void tile_values(const lds8* __restrict__ vs, TileState<D>& s, const v8bf (&pb)[4]) {
  const int lane = __lane_id(), h = lane >> 5, g1 = (lane >> 4) & 1, rr = (lane & 15) >> 2, qq = lane & 3;
  const int row = 4 * h + rr;
  const lds8* base = vs + row * 2 * D + (qq & 1) * 8;
  const int x = Tile<D>::v_swz(row), c0 = 2 * g1 + (qq >> 1);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
#pragma unroll
    for (int t = 0; t < D / 32; ++t) {
      // A operand: dim 32 t + 16 g1 + lane % 16 of positions 16 k + {4 h .. 4 h + 3, 8 + 4 h ..}
      const lds8* at = base + ((x ^ (4 * t + c0)) * 16) + 16 * k * 2 * D;
      const v4s a = lds_tr16(at), b = lds_tr16(at + 8 * 2 * D);
      const v8bf va = __builtin_bit_cast(v8bf, (v8s){a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w});
      s.o[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(va, pb[k], s.o[t], 0, 0, 0);
    }
  }
}

// A step some of whose positions some of the tile's rows may not see, with
// values that are not finite: those are added to the rows that see them, and
// then cleared for the product.
template <int D, int MODE>
__device__ __forceinline__ void add_not_finite(const FlashArgs& p, const Span& span, const lds8* vs, TileState<D>& s, int kv) {
  const int h = __lane_id() >> 5;
#pragma unroll 1
  for (int j = 0; j < kStep; ++j) {
    const bool seen = sees<MODE>(p, s.limit, MODE == kWindow ? span.pos(kv + j) : kv + j);
#pragma unroll
    for (int t = 0; t < D / 32; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        // dims 32 t + 8 i + 4 h .. + 3
        const uint2 x = lds_ld64(vs + j * 2 * D + ((4 * t + i) ^ Tile<D>::v_swz(j)) * 16 + 8 * h);
        if (seen && (not_finite(x.x) || not_finite(x.y))) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint16_t y = (uint16_t)((e < 2 ? x.x : x.y) >> (16 * (e & 1)));
            if ((y & 0x7f80u) == 0x7f80u) s.o[t][4 * i + e] += bf2f(y);
          }
        }
      }
  }
}

// The tile's part of it: whether there are such values is asked by all waves together.
template <int D, int MODE>
__device__ __forceinline__ void tile_not_finite(const FlashArgs& p, const Span& span, lds8* vs, int* s_flag, TileState<D>& s,
                                                int kv, bool mine) {
  const int tid = threadIdx.x;
  bool nf = false;
#pragma unroll
  for (int i = 0; i < Tile<D>::kLoads; ++i) nf |= any_not_finite(lds_ld128(vs + (i * 256 + tid) * 16));
  const bool any = __any(nf);
  if ((tid & 63) == 0) s_flag[uni(tid >> 6)] = any;
  lds_barrier();
  if (!(s_flag[0] | s_flag[1] | s_flag[2] | s_flag[3])) return;
  if (mine) add_not_finite<D, MODE>(p, span, vs, s, kv);
  lds_barrier();
#pragma unroll
  for (int i = 0; i < Tile<D>::kLoads; ++i) {
    lds8* const piece = vs + (i * 256 + tid) * 16;
    const uint4 x = lds_ld128(piece);
    lds_st128(piece, make_uint4(drop_not_finite(x.x), drop_not_finite(x.y), drop_not_finite(x.z), drop_not_finite(x.w)));
  }
  lds_barrier();
}

// LDS: keys in stages 0 and 1, values in 2 and 3; a flag per wave.  (One LDS object: the
// accesses to several get alias scopes, and reads then wait for the loads into LDS that are on their way.)
template <int D>
constexpr int kTileShared = 4 * Tile<D>::kBytes + 16;

// Item x (128 rows of a sequence; kShared: of the batch) and key-value head hk.
template <int D, int KV, int MODE>
__device__ __forceinline__ void tile_item(const FlashArgs& p, uint8_t* smem, int hk, int x, int split) {
  constexpr int kB = Tile<D>::kBytes;
  int* const s_flag = reinterpret_cast<int*>(smem + 4 * kB);
  const int tid = threadIdx.x, wv = uni(tid >> 6), lane = tid & 63, h = lane >> 5;
  Item it{0, x, 0};
  if (MODE != kShared && !find_item(p.bt, p.G, kTileRows, x, it, p.error)) return;
  int begin;
  const Seq sq = mode_seq<MODE>(p, it.b, begin, tid == 0);
  const int rows = sq.n * p.G, first = sq.len - sq.n;  // position of the first token
  if (MODE == kShared) {
    it.count = (rows + kTileRows - 1) / kTileRows;
    if (x >= it.count) return;
  }
  const int r0 = (it.count - 1 - it.i) * kTileRows;     // the longest tiles first
  const int t_last = uni(row_token(min(r0 + kTileRows, rows) - 1, p));
  // the last position that a token sees
  auto last_of = [&](int token) { return MODE == kShared ? sq.len - 1 : max(-1, first + token); };

  TileState<D> s;
  const int r = r0 + 32 * wv + (lane & 31);
  const int tok = row_token(min(r, rows - 1), p), head = hk * p.G + min(r, rows - 1) - tok * p.G;
  s.limit = r < rows ? last_of(tok) : -1;
  const int wr = r0 + 32 * wv;
  s.lo = wr < rows ? last_of(uni(row_token(wr, p))) : -1;
  s.hi = wr < rows ? last_of(uni(row_token(min(wr + 31, rows - 1), p))) : -1;
  {
    const uint16_t* q = p.q + (int64_t)(sq.row0 + tok) * p.ldq + head * D + 8 * h;
#pragma unroll
    for (int k = 0; k < D / 16; ++k)
      s.q[k] = __builtin_bit_cast(v8bf, *reinterpret_cast<const uint4*>(q + 16 * k));
  }
#pragma unroll
  for (int t = 0; t < D / 32; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) s.o[t][i] = 0.0f;
  s.m = kNegInf;
  s.l[0] = s.l[1] = 0.0f;

  const int wg_lo = last_of(uni(row_token(r0, p))), wg_hi = last_of(t_last);
  int kv_end = wg_hi + 1;
  int kv0 = begin;
  Source<D, KV, MODE> src;
  if (MODE == kWindow) {  // from here on steps are counted along the axis of what is seen
    src.span.init(p, first + uni(row_token(r0, p)), kv_end, KV == kDense ? 1 : kStep,
                  KV == kDense ? 1 : p.pg.ps.d % kStep == 0 ? kStep : 16);
    kv_end = max(0, kv_end - src.span.gap);
  }
  const int splits = MODE == kShared ? p.shared_splits : p.splits, chunk = MODE == kShared ? p.shared_chunk : p.chunk;
  const bool whole = MODE != kShared && MODE != kOwn && (splits == 1 || (MODE == kWindow ? kv_end : sq.len) <= chunk);
  if (whole && split > 0) return;
  if (!whole) {
    kv0 += split * chunk;
    if (split + 1 < splits) kv_end = min(kv_end, kv0 + chunk);
  }
  if (kv0 < kv_end) {
    lds8* const sm = (lds8*)smem;
    src.init(p, sq, it.b, hk, kv_end);
    // steps from whole_from on and up to whole_end: every row of the tile sees all of them
    const int gap = MODE == kWindow ? src.span.gap : 0;
    const int whole_from = MODE != kWindow ? kv0 : max(gap > 0 ? src.span.turn : 0, wg_hi - p.window + 1 - gap);
    const int whole_end = min(kv_end, wg_lo + 1 - gap);
    // step j at position kv; at: the parity of its stages, 0 where the whole steps begin
    int kv = kv0, at = MODE == kWindow ? (max(0, whole_from - kv0) + kStep - 1) / kStep & 1 : 0;
    auto arrived = [&] {
      __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): this thread's loads
      lds_barrier();                       // everyone's; and what the last step read is free
    };
    // the keys of two steps ahead, the values of the next
    auto load_ahead = [&](lds8* k_free, lds8* v_free) {
      if (kv + 2 * kStep < kv_end) src.template load<false>(p, kv + 2 * kStep, k_free);
      if (kv + kStep < kv_end) src.template load<true>(p, kv + kStep, v_free);
      src.turn_pages(p, kv + 3 * kStep);
    };
    auto store_ahead = [&](lds8* k_free, lds8* v_free) {
      if (kv + 2 * kStep < kv_end) src.template store<false>(k_free);
      if (kv + kStep < kv_end) src.template store<true>(v_free);
    };

    src.fetch_pages(p, kv0, src.page_k);
    src.template load<false>(p, kv0, sm + at * kB);
    src.template store<false>(sm + at * kB);
    src.turn_pages(p, kv0 + kStep);
    src.template load<true>(p, kv0, sm + (2 + at) * kB);
    src.template store<true>(sm + (2 + at) * kB);
    if (kv0 + kStep < kv_end) {
      src.template load<false>(p, kv0 + kStep, sm + (at ^ 1) * kB);
      src.template store<false>(sm + (at ^ 1) * kB);
    }
    src.turn_pages(p, kv0 + 2 * kStep);
    arrived();
    TileKeys keys;
    v16f sa[2], sb[2];
    // of rows whose limits are in [lo, hi]: whether all see all of the step at u, or some may see some of it
    auto all_of = [&](int lo, int hi, int u) {
      return !(MODE == kWindow && src.span.mixed(u, kStep)) && all_see<MODE>(p, lo, hi, src.pos(u), kStep);
    };
    auto some_of = [&](int lo, int hi, int u) {
      return (MODE == kWindow && src.span.mixed(u, kStep)) || some_see<MODE>(p, lo, hi, src.pos(u), kStep);
    };
    if (some_of(s.lo, s.hi, kv0)) {
      tile_keys<D>(sm + at * kB, keys);
      tile_scores<D>(sm + at * kB, keys, s, sa);
      if (!all_of(s.lo, s.hi, kv0)) tile_mask<D, MODE>(p, src.span, s, kv0, sa);
      tile_raise<D>(s, p.c, sa);
    }
    lds_barrier();  // the first keys are read: their stage is free

    // steps whose successor every row of the tile sees whole; a copy for each
    // parity, so that LDS addresses are constants and scores stay in their registers
    auto hot = [&](const lds8* ks, const lds8* vs, lds8* k_free, lds8* v_free, const v16f(&cur)[2], v16f(&nxt)[2]) {
      arrived();
      tile_keys<D>(ks, keys);
      load_ahead(k_free, v_free);
      v8bf pb[4];
      tile_scores<D>(ks, keys, s, nxt);
      tile_exp<D>(s, p.c, cur, pb);
      tile_values<D>(vs, s, pb);
      tile_raise<D>(s, p.c, nxt);
      store_ahead(k_free, v_free);
      kv += kStep;
    };
    // a wave without rows only loads (67 tokens at 40000 positions: 68.5 us, 65.5 so; windows, where this copy of the loads costs
    // the hot loop its registers: 67 tokens 24.4, 26.1, prompts of 16001 190, 247)
    if (MODE != kWindow && wr >= rows) {
      for (; kv + 2 * kStep <= whole_end; kv += kStep, at ^= 1) {
        arrived();
        load_ahead(sm + at * kB, sm + (3 - at) * kB);
        store_ahead(sm + at * kB, sm + (3 - at) * kB);
      }
    }
    // any step, of the wave's rows those that see some of it
    auto edge = [&] {
      const lds8* const ks = sm + (at ^ 1) * kB;
      lds8* const vs = sm + (2 + at) * kB;
      lds8 *const k_free = sm + at * kB, *const v_free = sm + (2 + (at ^ 1)) * kB;
      arrived();
      load_ahead(k_free, v_free);
      const bool mine = some_of(s.lo, s.hi, kv);  // some of the wave's rows see some of it
      const bool next = kv + kStep < kv_end && some_of(s.lo, s.hi, kv + kStep);
      if (!all_of(wg_lo, wg_hi, kv))  // some of the tile's rows do not see all of it
        tile_not_finite<D, MODE>(p, src.span, vs, s_flag, s, kv, mine);
      if (mine) {
        v8bf pb[4];
        tile_exp<D>(s, p.c, sa, pb);
        tile_values<D>(vs, s, pb);
      }
      if (next) {
        tile_keys<D>(ks, keys);
        tile_scores<D>(ks, keys, s, sa);
        if (!all_of(s.lo, s.hi, kv + kStep)) tile_mask<D, MODE>(p, src.span, s, kv + kStep, sa);
        tile_raise<D>(s, p.c, sa);
      }
      store_ahead(k_free, v_free);
      kv += kStep;
      at ^= 1;
    };
    if constexpr (MODE == kWindow)  // those that some rows do not see from their beginning
      while (kv < kv_end && kv < whole_from) edge();
    while (kv + 2 * kStep <= whole_end) {
      hot(sm + kB, sm + 2 * kB, sm, sm + 3 * kB, sa, sb);
      if (kv + 2 * kStep > whole_end) {
        at = 1;
#pragma unroll
        for (int t = 0; t < 2; ++t) sa[t] = sb[t];
        break;
      }
      hot(sm, sm + 3 * kB, sm + kB, sm + 2 * kB, sb, sa);
    }
    while (kv < kv_end) edge();
    if (KV != kDense && src.bad) flag_error(p.error);
  }

  const float l0 = s.l[0] + s.l[1], l = l0 + xor_partner<32>(l0);
  const int64_t row = sq.row0 + tok;
  if (!whole) {
    if (r >= rows) return;
    const int64_t at = ((int64_t)(split + (MODE == kOwn ? p.shared_splits : 0)) * p.bt.T + row) * p.H + head;
    if (h == 0) p.part_ml[at] = MODE == kOwn && s.limit < 0 ? make_float2(0.0f, kNone) : make_float2(s.m, l);
    if (empty(s.m, l)) return;
    float* o = p.part_o + at * D + 4 * h;
#pragma unroll
    for (int t = 0; t < D / 32; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<float4*>(o + 32 * t + 8 * i) =
            make_float4(s.o[t][4 * i], s.o[t][4 * i + 1], s.o[t][4 * i + 2], s.o[t][4 * i + 3]);
    return;
  }
  if (p.splits > 1 && h == 0 && r < rows) p.part_ml[row * p.H + head] = make_float2(0.0f, kWhole);
  const float inv = empty(s.m, l) ? 0.0f : 1.0f / l;
  // A wave's rows go through the stages, which are read, to leave in whole lines (16001 tokens, window 1 / 1024: 61 / 195 us from the
  // registers, 50 / 181 so; no window 396, 392).  Partials leave from the registers: their lines are shorter only by half,
  // and tiles of few rows would wait for this (drafts of 8 users 19.4, 21.1).
  lds_barrier();
  lds8* const mine = (lds8*)smem + wv * 32 * 2 * D;
#pragma unroll
  for (int t = 0; t < D / 32; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      lds_st64(mine + (lane & 31) * 2 * D + ((4 * t + i) ^ Tile<D>::k_swz(lane & 31)) * 16 + 8 * h,
               make_uint2(f2bf_pair(s.o[t][4 * i] * inv, s.o[t][4 * i + 1] * inv),
                          f2bf_pair(s.o[t][4 * i + 2] * inv, s.o[t][4 * i + 3] * inv)));
  __builtin_amdgcn_wave_barrier();
  const int64_t at = r < rows ? row * p.ldo + head * D : -1;
#pragma unroll
  for (int j = 0; j < D / 16; ++j) {
    const int x = 64 * j + lane, y = x / (D / 8), c = x % (D / 8);
    const int64_t to = __shfl(at, y);
    if (to >= 0) *reinterpret_cast<uint4*>(p.out + to + 8 * c) = lds_ld128(mine + y * 2 * D + (c ^ Tile<D>::k_swz(y)) * 16);
  }
}

// Workgroup x of units of `each` items that read the same keys and values: those are x's of one remainder by 8, which
// share an L2 (a workgroup's XCD is its number's remainder), close to one another in time.
constexpr int kXcds = 8;
struct UnitItem {
  int unit, item;
};
__host__ __device__ __forceinline__ UnitItem unit_item(int x, int each) {
  const int i = x / kXcds;
  return {i / each * kXcds + x % kXcds, i % each};
}
inline int64_t unit_groups(int64_t units, int64_t each) { return (units + kXcds - 1) / kXcds * kXcds * each; }

// kWindow: workgroup x's head and tile of it (any behind the last one), where units are `each` neighbouring tiles of a head.
struct HeadTile {
  int hk, x;
};
__host__ __device__ __forceinline__ HeadTile window_tile(int x, int Hkv, int each) {
  const UnitItem u = unit_item(x, each);
  return {u.unit % Hkv, u.unit / Hkv * each + u.item};
}

template <int D, int KV, int MODE>
__global__ __launch_bounds__(256, 2) void k_flash_tile(FlashArgs p) {
  __shared__ __attribute__((aligned(16))) uint8_t smem[kTileShared<D>];
  if (MODE == kWindow) {
    const HeadTile t = window_tile(blockIdx.x, p.Hkv, p.neighbours);
    tile_item<D, KV, MODE>(p, smem, uni(t.hk), uni(t.x), blockIdx.y);
  } else {
    tile_item<D, KV, MODE>(p, smem, uni(blockIdx.x % p.Hkv), blockIdx.x / p.Hkv, blockIdx.y);
  }
}
// kWindow: how many neighbouring tiles of a head, which see mostly the same positions, run on one XCD, one after the other: so
// many that each XCD has several such groups, up to 8.  20 / 5 heads of 128, window 1024, us with 1 / 2 / 4 / 8 / 16: 16001 tokens
// (2520 tiles of all heads) 198, 189, 186, 180, 188; 8000 (1270) 91.5, 85.5, 83.8, 86.6, 87.6; 4000 (640) 60.6, 57.9, 58.4, 60.6,
// 62; 2000 (320) 30.5, 30.4, 30.5, 30.9, 31.0; over pages, chunks of 4000 (640), window 2000: 130, 117, 116, 116, 116.  Splits
// read different positions, and want the XCDs evenly full: 500 rows at a window of 4096 in 4 (80 tiles), 1 / 8: 42, 46.
inline int window_neighbours(int64_t tiles, int splits) {
  int each = 1;
  while (splits == 1 && each < 8 && 2 * each * 5 * device_cus() <= 8 * tiles) each *= 2;
  return each;
}
inline int64_t window_groups(int64_t tiles, int64_t Hkv, int each) {
  return unit_groups((tiles / Hkv + each - 1) / each * Hkv, each);
}

// ======================================================================
// Few rows (up to 16 to a sequence and key-value head: single tokens, short
// drafts): bound by the bytes of keys and values.  4 waves share a context, a
// round of kPos positions each; a wave's keys go straight from memory to the
// MFMA's registers, its values through its own LDS.  The next round's loads are
// issued as soon as this one's registers are free (unconditionally: behind the end
// they are out of the resource's range and read nothing), so 16 KiB a wave (8 KiB of
// 8-bit pages) are on their way nearly all the time.  Page table entries are
// fetched a round ahead of that.  The waves' partials meet in LDS.
//
// Over bf16 pages p is two bf16 values, itself rounded and what that leaves, so 16 bits of it
// are used: the matrix units have the time (one user at 131001 positions 65.3 us, 65.7 so; 128 users at 2048
// 126.6, 126.9; 32 at 2048 35.5, 35.9).  The rests have a sum of their own (in one sum with the rest an infinite value
// that a row sees would become NaN), and the error against 64 bits is that of the output's own rounding.  8-bit
// pages, whose values have 4 bits, would pay 1 to 7% (128 users at 2048 70.2, 71.1; 32 at 2048 21.7, 23.3) and have one.
//
// 5 heads of 128: one user at 131001 positions 60 us (5.6 TB/s) and 5 of the merge, 128
// users at 2048 127 us (5.3 TB/s); 8-bit pages 70 us (4.8).  8 / 4 / 2 waves a workgroup, each
// at its best number of splits, in an early form of this kernel, 32 users of mixed lengths up to 4096,
// 8-bit pages: 38.5, 36.9, 36.2 us; one user at 512 positions: 10.7, 9.7, 13.0.
// ======================================================================
constexpr int kFewRows = 16;
constexpr int kFewWaves = 4;

// Pieces of a value row in LDS are at piece ^ few_swz(row): the 8 rows x 32 bytes
// that 32 lanes of a transposing read cover are in different banks.
template <int D>
__device__ __forceinline__ int few_swz(int row) {
  return D == 128 ? (2 * row) & 15 : row & 6;
}

template <int D, int NW = kFewWaves>
struct FewShared {
  union {
    uint8_t v[NW][32 * 2 * D];       // 32 value rows of a wave
    float o[NW][kFewRows][D];        // after the last round
  };
  float ml[NW][kFewRows][2];
};

template <int D, int KV, int MODE>
struct Few {
  static constexpr int kRowBytes = KV == kPagedFp8 ? D : 2 * D;
  static constexpr int kRuns = 2;                           // runs of 16 positions of a wave and round
  static constexpr int kPos = 16 * kRuns;
  static constexpr int kK = kRowBytes / 64;                 // key loads of a lane for a run
  static constexpr int kV = kRowBytes / 64;                 // value loads of a lane for a run
  static constexpr int kTpr = kRowBytes / 16;               // lanes of a value row
  static constexpr bool kRest = KV == kPagedBf16;           // p as two bf16 values
  uint4 k[kRuns][kK];
  uint4 v[kRuns][kV];
  uint32_t ke[kRuns], ve[kRuns][kV];
  int32_t page[kRuns];  // of the round to be loaded next
  bool one;             // pages of whole rounds
  Span span;            // kWindow

  __device__ __forceinline__ int pos(int u) const { return MODE == kWindow ? span.pos(u) : u; }
  // Page table entries of the round from position kv (any up to the table's end).
  __device__ __forceinline__ void fetch_pages(const FlashArgs& p, const int32_t* table, int u) {
    const int kv = pos(u);
#pragma unroll
    for (int t = 0; t < kRuns; ++t)
      if (t == 0 || !one)
        page[t] = scalar_load(table, min(div_by(kv + 16 * t, p.pg.ps), (uint32_t)p.bt.max_pages - 1));
  }
  // Run t's keys, from row `from` of n page rows at `row`.
  __device__ __forceinline__ void run_keys(const FlashArgs& p, int t, int64_t row, uint32_t n, int from) {
    const int lane = __lane_id(), r = from + (lane & 15);
    const auto rs = buf_rsrc(p.pg.k + row * kRowBytes, n * kRowBytes);
#pragma unroll
    for (int i = 0; i < kK; ++i) k[t][i] = buf_ld128(rs, r * kRowBytes + 64 * i + 16 * (lane >> 4));
    if (KV == kPagedFp8) ke[t] = buf_ld8(buf_rsrc(p.pg.ke + row, n), r);
  }
  __device__ __forceinline__ void run_values(const FlashArgs& p, int t, int64_t row, uint32_t n, int from) {
    const int lane = __lane_id();
    const auto rs = buf_rsrc(p.pg.v + row * kRowBytes, n * kRowBytes);
#pragma unroll
    for (int i = 0; i < kV; ++i) {
      v[t][i] = buf_ld128(rs, from * kRowBytes + 1024 * i + 16 * lane);
      if (KV == kPagedFp8) ve[t][i] = buf_ld8(buf_rsrc(p.pg.ve + row, n), from + (64 / kTpr) * i + lane / kTpr);
    }
  }
  // The round's keys (VAL: values) from position kv.
  template <bool VAL>
  __device__ __forceinline__ void load(const FlashArgs& p, int hk, int u, int kv_end, bool& bad) {
    const int kv = pos(u);
    auto end_of = [&](int at, int n) { return MODE == kWindow ? (u < kv_end ? span.end_of(at, n) : 0) : kv_end; };
    Run run;
    if (one) run = run_at(p.pg, hk, kv, end_of(kv, kPos), page[0], kPos, bad);
#pragma unroll
    for (int t = 0; t < kRuns; ++t) {
      if (!one) run = run_at(p.pg, hk, kv + 16 * t, end_of(kv + 16 * t, 16), page[t], 16, bad);
      if (VAL)
        run_values(p, t, run.row, run.n, one ? 16 * t : 0);
      else
        run_keys(p, t, run.row, run.n, one ? 16 * t : 0);
    }
  }
  // Key operand of run t, dims 32 k ..: 8-bit keys give a lane 16 dims of each 64.
  __device__ __forceinline__ v8bf key(int t, int i) const {
    if (KV != kPagedFp8) return __builtin_bit_cast(v8bf, k[t][i]);
    const uint4 w = k[t][i / 2];
    return __builtin_bit_cast(v8bf, from_e4m3(i & 1 ? make_uint2(w.z, w.w) : make_uint2(w.x, w.y), exp_scale(ke[t])));
  }
  // Value rows of runs t and t + 1 to the wave's LDS.
  __device__ __forceinline__ void store_values(lds8* vs, int t0) const {
    const int lane = __lane_id(), c = lane % kTpr;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < kV; ++i) {
        const int row = 16 * t + (64 / kTpr) * i + lane / kTpr;
        lds8* const at = vs + row * 2 * D;
        const uint4 w = v[t0 + t][i];
        if (KV == kPagedFp8) {
          const float f = exp_scale(ve[t0 + t][i]);
          const int c0 = 2 * c ^ few_swz<D>(row);
          lds_st128(at + c0 * 16, from_e4m3(make_uint2(w.x, w.y), f));
          lds_st128(at + (c0 ^ 1) * 16, from_e4m3(make_uint2(w.z, w.w), f));
        } else {
          lds_st128(at + (c ^ few_swz<D>(row)) * 16, w);
        }
      }
  }
};

// 32 value rows in LDS some of which some of the rows may not see: as
// add_not_finite, for this kernel's layout (lane r16: a query, its dims 16 t +
// 4 grp ..).
template <int D, int MODE>
__device__ __forceinline__ void few_not_finite(const FlashArgs& p, lds8* vs, v4f (&o)[D / 16], int at, int limit) {
  const int lane = __lane_id(), grp = lane >> 4;
  bool nf = false;
  for (int i = lane; i < 32 * D / 8; i += 64) nf |= any_not_finite(lds_ld128(vs + i * 16));
  if (!__any(nf)) return;
#pragma unroll 1
  for (int j = 0; j < 32; ++j)
#pragma unroll
    for (int t = 0; t < D / 16; ++t) {
      const uint2 x = lds_ld64(vs + j * 2 * D + ((2 * t + (grp >> 1)) ^ few_swz<D>(j)) * 16 + 8 * (grp & 1));
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint16_t y = (uint16_t)((i < 2 ? x.x : x.y) >> (16 * (i & 1)));
        if ((y & 0x7f80u) == 0x7f80u && sees<MODE>(p, limit, at + j)) o[t][i] += bf2f(y);
      }
    }
  __builtin_amdgcn_wave_barrier();
  for (int i = lane; i < 32 * D / 8; i += 64) {
    const uint4 x = lds_ld128(vs + i * 16);
    lds_st128(vs + i * 16, make_uint4(drop_not_finite(x.x), drop_not_finite(x.y), drop_not_finite(x.z),
                                      drop_not_finite(x.w)));
  }
  __builtin_amdgcn_wave_barrier();
}

// Sequence b (kShared: the batch as one) and key-value head hk.
template <int D, int KV, int MODE, int NW = kFewWaves>
__device__ __forceinline__ void few_item(const FlashArgs& p, FewShared<D, NW>& s, int hk, int b, int split) {
  using F = Few<D, KV, MODE>;
  constexpr int kRound = F::kPos * NW;
  const int tid = threadIdx.x, wv = uni(tid >> 6), lane = tid & 63, r16 = lane & 15, grp = lane >> 4;
  const int32_t* const table = p.bt.table + (int64_t)b * p.bt.max_pages;
  const int splits = MODE == kShared ? p.shared_splits : p.splits, chunk = MODE == kShared ? p.shared_chunk : p.chunk;
  const int part0 = MODE == kOwn ? p.shared_splits : 0;  // the mode's first partial
  int kv0 = splits > 1 ? split * chunk : 0, kv_first = kv0 + F::kPos * wv;
  F f;
  f.one = p.pg.ps.d % F::kPos == 0;
  if (MODE == kCausal || MODE == kShared) f.fetch_pages(p, table, kv_first);  // (does not wait for the lengths)
  int begin;
  const Seq sq = mode_seq<MODE>(p, b, begin, tid == 0);
  const int rows = sq.n * p.G, first = sq.len - sq.n;
  auto last_of = [&](int token) { return MODE == kShared ? sq.len - 1 : max(-1, first + token); };
  bool whole = MODE != kShared && MODE != kOwn && (splits == 1 || sq.len <= chunk);
  if (MODE != kWindow && whole && split > 0) return;
  if (MODE == kOwn) {
    kv0 += begin;
    kv_first += begin;
    f.fetch_pages(p, table, kv_first);
  }
  const int seq_end = whole || split + 1 == splits ? sq.len : min(sq.len, kv0 + chunk);
  bool bad = false;
  // one pass unless there are more rows than the caller said
  for (int r0 = 0; r0 < rows; r0 += kFewRows) {
    const int r = r0 + r16, rc = min(r, rows - 1);
    const int tok = row_token(rc, p), head = hk * p.G + rc - tok * p.G;
    const int limit = r < rows ? last_of(tok) : -1;
    const int lo = uni(last_of(row_token(r0, p))), hi = uni(last_of(row_token(min(r0 + kFewRows, rows) - 1, p)));
    int kv_end = min(seq_end, hi + 1);
    if (MODE == kWindow) {  // from here on rounds are counted along the axis of what is seen
      f.span.init(p, uni(first + row_token(r0, p)), hi + 1, F::kPos, f.one ? F::kPos : 16);
      kv_end = max(0, hi + 1 - f.span.gap);
      whole = splits == 1 || kv_end <= chunk;
      if (whole && split > 0) continue;
      if (!whole && split + 1 < splits) kv_end = min(kv_end, kv0 + chunk);
    }
    if (r0 > 0 || MODE == kWindow) f.fetch_pages(p, table, kv_first);
    v8bf q[D / 32];  // B operands, in the order of the keys' dims
    {
      const uint16_t* a = p.q + (int64_t)(sq.row0 + tok) * p.ldq + head * D;
#pragma unroll
      for (int k = 0; k < D / 32; ++k) {
        const int d = KV == kPagedFp8 ? 64 * (k / 2) + 16 * grp + 8 * (k & 1) : 32 * k + 8 * grp;
        q[k] = __builtin_bit_cast(v8bf, *reinterpret_cast<const uint4*>(a + d));
      }
    }
    f.template load<false>(p, hk, kv_first, kv_end, bad);
    f.template load<true>(p, hk, kv_first, kv_end, bad);
    f.fetch_pages(p, table, kv_first + kRound);
    v4f o[D / 16], o_rest[D / 16];
#pragma unroll
    for (int t = 0; t < D / 16; ++t) o[t] = o_rest[t] = (v4f){0.f, 0.f, 0.f, 0.f};
    float m = kNegInf, l = 0.0f;
    lds8* const vs = (lds8*)&s.v[wv][0];

    for (int kv = kv_first; kv < kv_end; kv += kRound) {
      // scores: positions 16 t + 4 grp + i of query r16
      v4f sc[F::kRuns];
#pragma unroll
      for (int t = 0; t < F::kRuns; ++t) {
        sc[t] = (v4f){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < D / 32; ++k)
          sc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f.key(t, k), q[k], sc[t], 0, 0, 0);
      }
      f.template load<false>(p, hk, kv + kRound, kv_end, bad);

      const int at = f.pos(kv);
      float mx = kNegInf;
#pragma unroll
      for (int t = 0; t < F::kRuns; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (!sees<MODE>(p, limit, at + 16 * t + 4 * grp + i)) sc[t][i] = kNegInf;
          mx = fmaxf(mx, sc[t][i]);
        }
      mx = fmaxf(mx, xor_partner<16>(mx));
      mx = fmaxf(mx, xor_partner<32>(mx)) * p.c;
      if (__any(mx - m > kLazy)) {
        const float mn = fmaxf(m, __builtin_ceilf(mx));
        const float a = m == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
        m = mn;
        l *= a;
#pragma unroll
        for (int t = 0; t < D / 16; ++t) {
          o[t] *= a;
          if (F::kRest) o_rest[t] *= a;
        }
      }
      const float mc = m == kNegInf ? 0.0f : -m;
      uint32_t w[F::kRuns][2], rest[F::kRuns][2];
#pragma unroll
      for (int t = 0; t < F::kRuns; ++t)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float e0 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t][2 * i], p.c, mc));
          const float e1 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t][2 * i + 1], p.c, mc));
          w[t][i] = f2bf_pair(e0, e1);
          if (F::kRest) {
            rest[t][i] = f2bf_pair(e0 - __uint_as_float(w[t][i] << 16), e1 - __uint_as_float(w[t][i] & 0xffff0000u));
            l += e0 + e1;
          } else {
            l = sum_pair(w[t][i], l);
          }
        }
#pragma unroll
      for (int t0 = 0; t0 < F::kRuns; t0 += 2) {
        __builtin_amdgcn_wave_barrier();  // reads done before the rows are written again
        f.store_values(vs, t0);
        if (t0 + 2 == F::kRuns) {
          f.template load<true>(p, hk, kv + kRound, kv_end, bad);
          f.fetch_pages(p, table, kv + 2 * kRound);
        }
        __builtin_amdgcn_wave_barrier();  // the wave's LDS rows are read back by other lanes
        if (!all_see<MODE>(p, lo, hi, at + 16 * t0, 32)) few_not_finite<D, MODE>(p, vs, o, at + 16 * t0, limit);
        const v8bf pb = __builtin_bit_cast(v8bf, make_uint4(w[t0][0], w[t0][1], w[t0 + 1][0], w[t0 + 1][1]));
        v8bf pr;
        if (F::kRest) pr = __builtin_bit_cast(v8bf, make_uint4(rest[t0][0], rest[t0][1], rest[t0 + 1][0], rest[t0 + 1][1]));
        // O^T += V^T P^T: dim 16 t + r16 of positions {4 grp .., 16 + 4 grp ..}
        const int rr = r16 >> 2, qq = r16 & 3, row = 4 * grp + rr;
        const lds8* const vb = vs + row * 2 * D + (qq & 1) * 8;
#pragma unroll
        for (int t = 0; t < D / 16; ++t) {
          const lds8* a = vb + (((2 * t + (qq >> 1)) ^ few_swz<D>(row)) * 16);
          const v4s x = lds_tr16(a), y = lds_tr16(a + 16 * 2 * D);
          const v8bf va = __builtin_bit_cast(v8bf, (v8s){x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w});
          o[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(va, pb, o[t], 0, 0, 0);
          if (F::kRest) o_rest[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(va, pr, o_rest[t], 0, 0, 0);
        }
      }
    }

    // What is left of p may be negative or zero, so that its product with an infinite value is no
    // part of the sum: where the product of the rounded p is not finite, that is the sum.
    if (F::kRest) {
#pragma unroll
      for (int t = 0; t < D / 16; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[t][i] += __builtin_isfinite(o[t][i]) ? o_rest[t][i] : 0.0f;
    }

    // the waves' partials, in wave order
    l += xor_partner<16>(l);
    l += xor_partner<32>(l);
    if (grp == 0) {
      s.ml[wv][r16][0] = m;
      s.ml[wv][r16][1] = l;
    }
    __syncthreads();  // every wave is done with its value rows
#pragma unroll
    for (int t = 0; t < D / 16; ++t) *reinterpret_cast<float4*>(&s.o[wv][r16][16 * t + 4 * grp]) =
        make_float4(o[t][0], o[t][1], o[t][2], o[t][3]);
    __syncthreads();
    const int live = min(kFewRows, rows - r0);
    for (int i = tid; i < live * (D / 4); i += 64 * NW) {
      const int x = i / (D / 4), d = 4 * (i % (D / 4));
      float M = kNegInf;
#pragma unroll
      for (int w = 0; w < NW; ++w) M = fmaxf(M, s.ml[w][x][0]);
      float L = 0.0f;
      v4f O = (v4f){0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const float mw = s.ml[w][x][0], lw = s.ml[w][x][1];
        const float4 ow = *reinterpret_cast<const float4*>(&s.o[w][x][d]);
        if (empty(mw, lw)) continue;
        const float e = __builtin_amdgcn_exp2f(mw - M);
        L += e * lw;
        O[0] += e * ow.x;
        O[1] += e * ow.y;
        O[2] += e * ow.z;
        O[3] += e * ow.w;
      }
      const int tk = row_token(r0 + x, p), hd = hk * p.G + r0 + x - tk * p.G;
      const int64_t row = sq.row0 + tk;
      if (!whole) {
        const int64_t at = ((int64_t)(split + part0) * p.bt.T + row) * p.H + hd;
        if (d == 0) p.part_ml[at] = MODE == kOwn && first + tk < 0 ? make_float2(0.0f, kNone) : make_float2(M, L);
        if (!empty(M, L)) *reinterpret_cast<float4*>(p.part_o + at * D + d) = make_float4(O[0], O[1], O[2], O[3]);
      } else {
        if (splits > 1 && d == 0) p.part_ml[row * p.H + hd] = make_float2(0.0f, kWhole);
        const float inv = empty(M, L) ? 0.0f : 1.0f / L;
        *reinterpret_cast<uint2*>(p.out + row * p.ldo + hd * D + d) =
            make_uint2(f2bf_pair(O[0] * inv, O[1] * inv), f2bf_pair(O[2] * inv, O[3] * inv));
      }
    }
    __syncthreads();  // before the next rows' values
  }
  if (bad) flag_error(p.error);
}

template <int D, int KV, int MODE>
__global__ __launch_bounds__(64 * kFewWaves, KV == kPagedFp8 ? 3 : 2) void k_flash_few(FlashArgs p) {
  __shared__ __attribute__((aligned(16))) FewShared<D> s;
  few_item<D, KV, MODE>(p, s, blockIdx.x, blockIdx.y, blockIdx.z);
}

// Windows over 8-bit pages, where the workgroups are no more than the CUs: 8 waves have twice the loads on their way, and the
// conversions of twice the positions run at once.  20 / 5 heads of 128, us with 4 / 8 waves: 32 users, window 100 / 500 / 1024: 9.6,
// 14.3, 19.4 / 9.1, 12.6, 15.3; 8 users, 4096: 18.3 / 17.1; one user, 4096: 14.8 / 14.0.  With more workgroups, 120 users, 1024: 44.9 / 51;
// 256: 75 / 89.  bf16 pages, which need no conversion: 8 users 15.5 / 16.5, one user, 4096: 15.5 / 16.4, 64 users 45.6 / 49.5.
template <int D>
__global__ __launch_bounds__(512, 2) void k_flash_few_wide(FlashArgs p) {
  __shared__ __attribute__((aligned(16))) FewShared<D, 8> s;
  few_item<D, kPagedFp8, kWindow, 8>(p, s, blockIdx.x, blockIdx.y, blockIdx.z);
}

// The splits' partials of a row, in an order that the number of splits fixes:
// a group of D / 4 threads sums every `groups`-th split of a row, then the first of a
// row's groups sums the groups.  Bound by latency: one pass with a running maximum (a pass
// for the maximum before it: 20 rows of 47 splits 6.7 us, 4.8 so).
struct MergeSum {
  float m = kNegInf, l = 0.0f;
  v4f o = (v4f){0.f, 0.f, 0.f, 0.f};
  __device__ __forceinline__ void add(float m2, float l2, float4 o2) {
    const bool none = empty(m2, l2);
    const float mn = fmaxf(m, m2), a = m == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
    const float f = none ? 0.0f : __builtin_amdgcn_exp2f(m2 - mn);
    m = mn;
    l = a * l + (none ? 0.0f : f * l2);
    o[0] = a * o[0] + (none ? 0.0f : f * o2.x);
    o[1] = a * o[1] + (none ? 0.0f : f * o2.y);
    o[2] = a * o[2] + (none ? 0.0f : f * o2.z);
    o[3] = a * o[3] + (none ? 0.0f : f * o2.w);
  }
};
template <int D, bool SHARED>
__global__ __launch_bounds__(256) void k_flash_merge(FlashArgs p, int groups) {
  constexpr int TG = D / 4, NG = 256 / TG;
  __shared__ float4 s_o[NG][TG];
  __shared__ float2 s_ml[NG];
  const int t = threadIdx.x % TG, g = threadIdx.x / TG, z0 = g % groups;
  const int n = p.bt.T * p.H, row = blockIdx.x * (NG / groups) + g / groups;  // (token, head)
  const int tok = (int)((uint32_t)row / (uint32_t)p.H), head = row - tok * p.H;
  const int parts = p.splits + (SHARED ? p.shared_splits : 0);
  bool live = tok >= max(0, p.bt.cu[0]) && tok < min(p.bt.T, p.bt.cu[p.bt.B]), some = live;
  if (live && SHARED) some = p.part_ml[(int64_t)p.shared_splits * n + row].y != kNone;
  if (live && !SHARED) live = some = p.part_ml[row].y != kWhole;
  MergeSum s;
  if (some) {
#pragma unroll 4
    for (int z = z0; z < parts; z += groups) {  // (an empty split's products are not read: any values)
      const int64_t at = (int64_t)z * n + row;
      const float2 ml = p.part_ml[at];
      s.add(ml.x, ml.y, *reinterpret_cast<const float4*>(p.part_o + at * D + 4 * t));
    }
  }
  s_o[g][t] = make_float4(s.o[0], s.o[1], s.o[2], s.o[3]);
  if (t == 0) s_ml[g] = make_float2(s.m, s.l);
  __syncthreads();
  if (!live || z0 != 0) return;
  for (int i = 1; i < groups; ++i) s.add(s_ml[g + i].x, s_ml[g + i].y, s_o[g + i][t]);
  const float inv = empty(s.m, s.l) ? 0.0f : 1.0f / s.l;
  *reinterpret_cast<uint2*>(p.out + tok * p.ldo + head * D + 4 * t) =
      make_uint2(f2bf_pair(s.o[0] * inv, s.o[1] * inv), f2bf_pair(s.o[2] * inv, s.o[3] * inv));
}

}  // namespace btl
