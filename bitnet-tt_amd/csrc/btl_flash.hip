// Causal attention of packed rows: within prompts (keys and values of the same
// packed sequences), or over the pages of a cache.
//
//   out_i = sum_j softmax_j(c q_i.k_j) v_j,  j up to row i's own position
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
// pages: 16 bits of p).  Two bf16 values of p in the tiles as well, a second product on the same values,
// measured: 4096 tokens 100 us, 136 so; 16001 415, 565; chunks of 4 users over up to 8000 139, 187; 67
// tokens over 40067 8-bit positions 62, 73.  Against 64 bits the one value costs 0.0020-0.0022 of the
// outputs' size where their own rounding has 0.0016.
//
// Rows of V behind the last position read as zero (whatever lies there), and a
// value that is not finite at a position that some of the tile's rows may not see is added
// to the rows that do see it and multiplied with none: 0 x inf is NaN.
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

constexpr float kLazy = 8.0f;
constexpr float kWhole = -1.0f;
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
};

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
template <int D, int KV>
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
  uint4 rk[kN], rv[kN];                            // 8-bit pages: a step on its way
  uint32_t ek[kN], ev[kN];

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
  __device__ __forceinline__ void fetch_pages(const FlashArgs& p, int kv, int32_t (&page)[kN]) const {
    if (KV == kDense) return;
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int at = one ? kv : kv + run_of(i);
      page[i] = 0;
      if (at < kv_end && (i == 0 || !one)) page[i] = scalar_load(table, div_by(at, p.pg.ps));
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
  __device__ __forceinline__ void load(const FlashArgs& p, int kv, lds8* at) {
    lds8* const dst = at + uni(threadIdx.x >> 6) * 1024;
    if (KV == kDense) {
      const uint32_t ld = (uint32_t)(VAL ? ldv : ldk);
      const auto r = buf_rsrc((VAL ? v : k) + kv * (VAL ? ldv : ldk), (uint32_t)min(kv_end - kv, kStep) * ld);
#pragma unroll
      for (int i = 0; i < kN; ++i) piece<VAL>(r, i, dst);
      return;
    }
    const uint8_t* const pool = VAL ? p.pg.v : p.pg.k;
    const uint8_t* const exps = VAL ? p.pg.ve : p.pg.ke;
    if (one) {
      const Run run = run_at(p.pg, hk, kv, kv_end, VAL ? page_v[0] : page_k[0], kStep, bad);
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
      const Run run = run_at(p.pg, hk, kv + r0, kv_end, VAL ? page_v[i] : page_k[i], 16, bad);
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

template <int D>
__device__ __forceinline__ void tile_mask(const TileState<D>& s, int kv, v16f (&sc)[2]) {
  const int h = __lane_id() >> 5;
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
template <int D>
__device__ __forceinline__ void add_not_finite(const lds8* vs, TileState<D>& s, int kv) {
  const int h = __lane_id() >> 5;
#pragma unroll 1
  for (int j = 0; j < kStep; ++j) {
    const bool sees = kv + j <= s.limit;
#pragma unroll
    for (int t = 0; t < D / 32; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        // dims 32 t + 8 i + 4 h .. + 3
        const uint2 x = lds_ld64(vs + j * 2 * D + ((4 * t + i) ^ Tile<D>::v_swz(j)) * 16 + 8 * h);
        if (sees && (not_finite(x.x) || not_finite(x.y))) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint16_t y = (uint16_t)((e < 2 ? x.x : x.y) >> (16 * (e & 1)));
            if ((y & 0x7f80u) == 0x7f80u) s.o[t][4 * i + e] += bf2f(y);
          }
        }
      }
  }
}

template <int D, int KV>
__global__ __launch_bounds__(256, 2) void k_flash_tile(FlashArgs p) {
  constexpr int kB = Tile<D>::kBytes;
  // Keys: stages 0 and 1, values: 2 and 3; a flag per wave.  (One LDS object: the
  // accesses to several get alias scopes, and reads then wait for the loads into LDS that are on their way.)
  __shared__ __attribute__((aligned(16))) uint8_t smem[4 * kB + 16];
  int* const s_flag = reinterpret_cast<int*>(smem + 4 * kB);
  const int tid = threadIdx.x, wv = uni(tid >> 6), lane = tid & 63, h = lane >> 5;
  const int hk = uni(blockIdx.x % p.Hkv), split = blockIdx.y;
  Item it;
  if (!find_item(p.bt, p.G, kTileRows, blockIdx.x / p.Hkv, it, p.error)) return;
  const Seq sq = load_seq(p.bt, it.b, (int64_t)p.bt.max_pages * p.pg.ps.d);
  if (!sq.ok && tid == 0) flag_error(p.error);
  const int rows = sq.n * p.G, first = sq.len - sq.n;  // position of the first token
  const int r0 = (it.count - 1 - it.i) * kTileRows;     // the longest tiles first
  const int t_last = uni(row_token(min(r0 + kTileRows, rows) - 1, p));

  TileState<D> s;
  const int r = r0 + 32 * wv + (lane & 31);
  const int tok = row_token(min(r, rows - 1), p), head = hk * p.G + min(r, rows - 1) - tok * p.G;
  s.limit = r < rows ? max(-1, first + tok) : -1;
  const int wr = r0 + 32 * wv;
  s.lo = wr < rows ? max(-1, first + uni(row_token(wr, p))) : -1;
  s.hi = wr < rows ? max(-1, first + uni(row_token(min(wr + 31, rows - 1), p))) : -1;
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

  const int wg_lo = max(-1, first + uni(row_token(r0, p)));
  int kv_end = max(0, first + t_last + 1);
  int kv0 = 0;
  const bool whole = p.splits == 1 || sq.len <= p.chunk;
  if (whole && split > 0) return;
  if (!whole) {
    kv0 = split * p.chunk;
    if (split + 1 < p.splits) kv_end = min(kv_end, kv0 + p.chunk);
  }
  if (kv0 < kv_end) {
    lds8* const sm = (lds8*)smem;
    Source<D, KV> src;
    src.init(p, sq, it.b, hk, kv_end);
    const int whole_end = min(kv_end, wg_lo + 1);  // every row of the tile sees the positions before it
    int kv = kv0, at = 0;  // step j at position kv; at: j's parity
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
    src.template load<false>(p, kv0, sm);
    src.template store<false>(sm);
    src.turn_pages(p, kv0 + kStep);
    src.template load<true>(p, kv0, sm + 2 * kB);
    src.template store<true>(sm + 2 * kB);
    if (kv0 + kStep < kv_end) {
      src.template load<false>(p, kv0 + kStep, sm + kB);
      src.template store<false>(sm + kB);
    }
    src.turn_pages(p, kv0 + 2 * kStep);
    arrived();
    TileKeys keys;
    v16f sa[2], sb[2];
    if (kv0 <= s.hi) {
      tile_keys<D>(sm, keys);
      tile_scores<D>(sm, keys, s, sa);
      if (kv0 + kStep - 1 > s.lo) tile_mask<D>(s, kv0, sa);
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
    if (wr >= rows) {  // a wave without rows only loads (67 tokens at 40000 positions: 68.5 us, 65.5 so)
      for (; kv + 2 * kStep <= whole_end; kv += kStep, at ^= 1) {
        arrived();
        load_ahead(sm + at * kB, sm + (3 - at) * kB);
        store_ahead(sm + at * kB, sm + (3 - at) * kB);
      }
    }
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
    for (; kv < kv_end; kv += kStep, at ^= 1) {
      const lds8* const ks = sm + (at ^ 1) * kB;
      lds8* const vs = sm + (2 + at) * kB;
      lds8 *const k_free = sm + at * kB, *const v_free = sm + (2 + (at ^ 1)) * kB;
      arrived();
      load_ahead(k_free, v_free);
      const bool mine = kv <= s.hi, next = kv + kStep < kv_end && kv + kStep <= s.hi;  // some of the wave's rows see some of it
      bool special = false;
      if (kv + kStep - 1 > wg_lo) {  // some of the tile's rows do not see all of it
        bool nf = false;
#pragma unroll
        for (int i = 0; i < Tile<D>::kLoads; ++i) nf |= any_not_finite(lds_ld128(vs + (i * 256 + tid) * 16));
        const bool any = __any(nf);
        if (lane == 0) s_flag[wv] = any;
        lds_barrier();
        special = s_flag[0] | s_flag[1] | s_flag[2] | s_flag[3];
      }
      if (special) {
        if (mine) add_not_finite<D>(vs, s, kv);
        lds_barrier();
#pragma unroll
        for (int i = 0; i < Tile<D>::kLoads; ++i) {
          lds8* const piece = vs + (i * 256 + tid) * 16;
          const uint4 x = lds_ld128(piece);
          lds_st128(piece, make_uint4(drop_not_finite(x.x), drop_not_finite(x.y), drop_not_finite(x.z),
                                      drop_not_finite(x.w)));
        }
        lds_barrier();
      }
      if (mine) {
        v8bf pb[4];
        tile_exp<D>(s, p.c, sa, pb);
        tile_values<D>(vs, s, pb);
      }
      if (next) {
        tile_keys<D>(ks, keys);
        tile_scores<D>(ks, keys, s, sa);
        if (kv + 2 * kStep - 1 > s.lo) tile_mask<D>(s, kv + kStep, sa);
        tile_raise<D>(s, p.c, sa);
      }
      store_ahead(k_free, v_free);
    }
    if (KV != kDense && src.bad) flag_error(p.error);
  }

  const float l0 = s.l[0] + s.l[1], l = l0 + xor_partner<32>(l0);
  if (r >= rows) return;
  const int64_t row = sq.row0 + tok;
  if (whole && p.splits > 1 && h == 0) p.part_ml[row * p.H + head] = make_float2(0.0f, kWhole);
  if (!whole) {
    const int64_t at = ((int64_t)split * p.bt.T + row) * p.H + head;
    if (h == 0) p.part_ml[at] = make_float2(s.m, l);
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
  const float inv = empty(s.m, l) ? 0.0f : 1.0f / l;
  uint16_t* o = p.out + row * p.ldo + head * D + 4 * h;
#pragma unroll
  for (int t = 0; t < D / 32; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      *reinterpret_cast<uint2*>(o + 32 * t + 8 * i) =
          make_uint2(f2bf_pair(s.o[t][4 * i] * inv, s.o[t][4 * i + 1] * inv),
                     f2bf_pair(s.o[t][4 * i + 2] * inv, s.o[t][4 * i + 3] * inv));
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

template <int D>
struct FewShared {
  union {
    uint8_t v[kFewWaves][32 * 2 * D];       // 32 value rows of a wave
    float o[kFewWaves][kFewRows][D];        // after the last round
  };
  float ml[kFewWaves][kFewRows][2];
};

template <int D, int KV>
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

  // Page table entries of the round from position kv (any up to the table's end).
  __device__ __forceinline__ void fetch_pages(const FlashArgs& p, const int32_t* table, int kv) {
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
  __device__ __forceinline__ void load(const FlashArgs& p, int hk, int kv, int kv_end, bool& bad) {
    Run run;
    if (one) run = run_at(p.pg, hk, kv, kv_end, page[0], kPos, bad);
#pragma unroll
    for (int t = 0; t < kRuns; ++t) {
      if (!one) run = run_at(p.pg, hk, kv + 16 * t, kv_end, page[t], 16, bad);
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
template <int D>
__device__ __forceinline__ void few_not_finite(lds8* vs, v4f (&o)[D / 16], int at, int limit) {
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
        if ((y & 0x7f80u) == 0x7f80u && at + j <= limit) o[t][i] += bf2f(y);
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

template <int D, int KV>
__global__ __launch_bounds__(64 * kFewWaves, KV == kPagedFp8 ? 3 : 2) void k_flash_few(FlashArgs p) {
  using F = Few<D, KV>;
  constexpr int kRound = F::kPos * kFewWaves;
  __shared__ __attribute__((aligned(16))) FewShared<D> s;
  const int tid = threadIdx.x, wv = uni(tid >> 6), lane = tid & 63, r16 = lane & 15, grp = lane >> 4;
  const int hk = blockIdx.x, b = blockIdx.y, split = blockIdx.z;
  const int32_t* const table = p.bt.table + (int64_t)b * p.bt.max_pages;
  const int kv0 = p.splits > 1 ? split * p.chunk : 0, kv_first = kv0 + F::kPos * wv;
  F f;
  f.one = p.pg.ps.d % F::kPos == 0;
  f.fetch_pages(p, table, kv_first);  // (does not wait for the lengths)
  const Seq sq = load_seq(p.bt, b, (int64_t)p.bt.max_pages * p.pg.ps.d);
  if (!sq.ok && tid == 0) flag_error(p.error);
  const int rows = sq.n * p.G, first = sq.len - sq.n;
  const bool whole = p.splits == 1 || sq.len <= p.chunk;
  if (whole && split > 0) return;
  const int seq_end = whole || split + 1 == p.splits ? sq.len : min(sq.len, kv0 + p.chunk);
  bool bad = false;
  // one pass unless there are more rows than the caller said
  for (int r0 = 0; r0 < rows; r0 += kFewRows) {
    const int r = r0 + r16, rc = min(r, rows - 1);
    const int tok = row_token(rc, p), head = hk * p.G + rc - tok * p.G;
    const int limit = r < rows ? max(-1, first + tok) : -1;
    const int lo = uni(max(-1, first + row_token(r0, p)));
    const int kv_end = uni(min(seq_end, max(0, first + row_token(min(r0 + kFewRows, rows) - 1, p) + 1)));
    if (r0 > 0) f.fetch_pages(p, table, kv_first);
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

      float mx = kNegInf;
#pragma unroll
      for (int t = 0; t < F::kRuns; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (kv + 16 * t + 4 * grp + i > limit) sc[t][i] = kNegInf;
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
        if (kv + 16 * t0 + 31 > lo) few_not_finite<D>(vs, o, kv + 16 * t0, limit);
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
    for (int i = tid; i < live * (D / 4); i += 64 * kFewWaves) {
      const int x = i / (D / 4), d = 4 * (i % (D / 4));
      float M = kNegInf;
#pragma unroll
      for (int w = 0; w < kFewWaves; ++w) M = fmaxf(M, s.ml[w][x][0]);
      float L = 0.0f;
      v4f O = (v4f){0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < kFewWaves; ++w) {
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
        const int64_t at = ((int64_t)split * p.bt.T + row) * p.H + hd;
        if (d == 0) p.part_ml[at] = make_float2(M, L);
        if (!empty(M, L)) *reinterpret_cast<float4*>(p.part_o + at * D + d) = make_float4(O[0], O[1], O[2], O[3]);
      } else {
        if (p.splits > 1 && d == 0) p.part_ml[row * p.H + hd] = make_float2(0.0f, kWhole);
        const float inv = empty(M, L) ? 0.0f : 1.0f / L;
        *reinterpret_cast<uint2*>(p.out + row * p.ldo + hd * D + d) =
            make_uint2(f2bf_pair(O[0] * inv, O[1] * inv), f2bf_pair(O[2] * inv, O[3] * inv));
      }
    }
    __syncthreads();  // before the next rows' values
  }
  if (bad) flag_error(p.error);
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
template <int D>
__global__ __launch_bounds__(256) void k_flash_merge(FlashArgs p, int groups) {
  constexpr int TG = D / 4, NG = 256 / TG;
  __shared__ float4 s_o[NG][TG];
  __shared__ float2 s_ml[NG];
  const int t = threadIdx.x % TG, g = threadIdx.x / TG, z0 = g % groups;
  const int n = p.bt.T * p.H, row = blockIdx.x * (NG / groups) + g / groups;  // (token, head)
  const int tok = (int)((uint32_t)row / (uint32_t)p.H), head = row - tok * p.H;
  const bool live = tok >= max(0, p.bt.cu[0]) && tok < min(p.bt.T, p.bt.cu[p.bt.B]) && p.part_ml[row].y != kWhole;
  MergeSum s;
  if (live) {
#pragma unroll 4
    for (int z = z0; z < p.splits; z += groups) {  // (an empty split's products are not read: any values)
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

// ---- host ---------------------------------------------------------------
struct FlashPlan {
  bool few;
  int64_t tiles;  // workgroups per split
  int splits, chunk;
};
// Few rows: the kernel of single tokens where a sequence's rows fit one of its tiles.
//
// Splits, by the workgroups that the rows alone give (`tiles`) and the longest
// context, measured on 256 CUs, 20 / 5 heads of 128, us a call; a chunk is at
// least kMinChunk positions and 256 of them a round.
//  - Tiles: two workgroups fit a CU, and a call's tiles are mostly of unlike
//    length, so as many as come nearest to two a CU.  1000 rows of one sequence at 9000
//    positions (160 workgroups), 1 / 2 / 3 / 4 splits: 173, 128, 110, 123; 4 x 320 at
//    8192 (220): 167, 141, 160, 150; 4 x 512 at 8192 (340): 234, 229, 224, 220; 2047 rows of
//    4 contexts of unlike length up to 8000 (339), 1 / 2 / 3 / 4: 172, 143, 165, 155.  Up to three
//    a CU two splits still even out the lengths, 1 / 2 / 3: 8 x 256 up to 8000 (360): 146, 132, 148;
//    16 x 128 (400): 163, 143, 155; 4000 rows of one at 8000 (630): 290, 271, 286.
//    But a split costs the merge's launch (4 us) and the writing and reading of its
//    partials, part = T H D 8 bytes at 4.8 TB/s each, and saves its share of the
//    longest workgroup's steps, whole = 0.75 us per 64 positions: the least of whole / n + n part is
//    at n = sqrt(whole / part), and n = 1 is better where that saves less than it costs.
//    Without this, with it: 2 x 512 rows at 512: 27.4, 17.8; 4 x 256 at 1024: 36.0, 26.8;
//    1000 at 1000: 28.9, 26.6; 512 at 2048: 34.9, 31.0; 256 at 1024: 23.2, 24.2.
//    The two rates are those of bf16 pages and D = 128; a step over 8-bit pages takes up to 1.4 times as long, one of
//    D = 64 0.8 times.  What the rule takes against the best of 1, 2, 3, 4, 6, 8, 12, 16, 32 splits:
//    67 rows at 40067 | 256 at 1024 | 512 at 2048 | 1000 at 9000 | 2047 of 4 up to 8000 | 2048 of 8 up to 7700,
//    D = 128, bf16: 64.3, 59.6 | 22.5, 21.2 | 29.7, 29.7 | 116, 111 | 140, 140 | 189, 176;
//    8-bit:         65.6, 61.5 | 25.6, 23.1 | 34.3, 33.8 | 122, 121 | 154, 154 | 206, 196;
//    4 / 2 heads of 64, bf16: 24.4, 24.4 | 12.6, 12.6 | 14.3, 14.2 | 31.9, 30.0 | 38.3, 38.3 | 41.4, 41.0;
//    8-bit:         26.5, 26.5 | 13.4, 13.3 | 14.9, 14.8 | 34.6, 32.0 | 41.7, 41.7 | 45.2, 44.7.
//  - Few rows: bound by memory, which one workgroup a CU saturates: as many
//    as there are CUs, from 1024 positions on.  bf16, 1 user at 16384, 16 / 25 / 51 / 102
//    splits: 20.1, 17.8, 16.5, 20.6; 8 users at 4096, 3 / 6 / 8: 24.3, 21.2, 24.6; 1 user at 1024,
//    1 / 4: 13.2, 11.2.
//    Up to 9/4 as many workgroups as CUs, some CUs have a long context more than others:
//    four splits from 2560 positions on.  Contexts of unlike length up to 4000, 1 / 2 / 3 / 4 / 6:
//    bf16, 36 users 53, 56, 49, 43, 49; 56: 100, 70, 65, 65, 66; 80: 107, 84, 85, 85, 87; 110: 125,
//    116, 115, 114, 116; 8-bit, 56: 48, 45, 40, 34, 37; 110: 84, 68, 69, 67, 68.  All of 4000,
//    bf16: 36: 69, 82, 82, 72, 76; 56: 138, 121, 117, 110, 110; 110: 227, 214, 209, 203, 207.  At 2048 positions,
//    1 / 4, unlike or alike, the gain is gone: bf16, 32 users 25.7, 27.2 or 33.7, 37.5;
//    140: 86, 86 or 134, 138.
//    Below one workgroup a CU the gain is that of 8-bit pages, and of some lengths: 1 / 2 / 3 / 4 splits, unlike
//    lengths up to 4096 (a quarter of it the least) or all of 4096, 32 users, bf16: 58, 65, 60, 59 or 65, 80, 71, 72;
//    8-bit: 37, 32, 31, 34 or 42, 46, 42, 42; 48 users, bf16: 68, 73, 69, 69 or 92, 97, 98, 98; 8-bit: 39, 39, 39,
//    37 or 50, 55, 56, 56; 80 users of 2 heads of 64, bf16: 28, 30, 27, 27 or 35, 43, 38, 38; 8-bit: 30, 25, 22, 19 or
//    31, 25, 23, 23.  (What would serve both: positions shared out by the lengths on the device.)
constexpr int64_t kMinChunk = 256;
constexpr int64_t kMaxSplits = 256;
// A hint behind this plans for as many positions as a page table may have room for: splits x
// chunk stays below 2^31, the kernels' positions.
constexpr int64_t kMaxPositions = INT32_MAX / 2;
inline FlashPlan flash_plan(int64_t T, int64_t H, int64_t Hkv, int64_t D, int64_t B, int64_t max_q, int64_t max_kv,
                            bool paged) {
  FlashPlan f{};
  const int64_t G = H / Hkv, cus = device_cus();
  max_q = std::min(max_q, T);
  max_kv = std::min(max_kv, kMaxPositions);
  f.few = paged && max_q * G <= kFewRows;
  f.tiles = (f.few ? B : T * G / kTileRows + (B < T ? B : T)) * Hkv;
  f.splits = 1;
  f.chunk = (int)round_up(max_kv > 0 ? max_kv : 1, kMinChunk);
  if (!paged || max_kv < (f.few ? 4 : 2) * kMinChunk) return f;
  int64_t n;
  if (f.few) {
    n = cus / f.tiles;
    if (n <= 1 && 4 * f.tiles <= 9 * cus && max_kv >= 10 * kMinChunk) n = 4;
  } else {
    n = std::max((4 * cus + f.tiles) / (2 * f.tiles), (int64_t)(f.tiles <= 3 * cus ? 2 : 1));
    const double whole = 0.0117 * (double)max_kv, part = 1.67e-6 * (double)(T * H * D);  // us
    n = std::min(n, (int64_t)(std::sqrt(whole / part) + 0.5));
    if (n > 1 && whole - whole / (double)n <= 4.0 + part * (double)n) n = 1;
  }
  if (n > max_kv / kMinChunk) n = max_kv / kMinChunk;
  if (n > kMaxSplits) n = kMaxSplits;
  if (n > 1) {
    f.chunk = (int)round_up((max_kv + n - 1) / n, kMinChunk);
    f.splits = (int)((max_kv + f.chunk - 1) / f.chunk);
  }
  return f;
}

inline int64_t flash_scratch(const FlashPlan& f, int64_t T, int64_t H, int64_t D) {
  return f.splits > 1 ? (int64_t)f.splits * T * H * (D + 2) * 4 : 0;
}

inline bool flash_heads(int64_t T, int64_t H, int64_t Hkv) {
  return H > 0 && Hkv > 0 && H <= 1024 && H % Hkv == 0 && H / Hkv <= 64 && T <= INT32_MAX / 2 / H;
}
// Sizes of calls with rows: those that the entry point takes, so that nothing planned from them overflows.
inline bool flash_sizes(int64_t T, int64_t H, int64_t Hkv, int64_t D, int64_t B, int64_t max_q, int64_t max_kv) {
  return T > 0 && T <= kMaxRows && B > 0 && B <= kMaxSeqs && (D == 64 || D == 128) && flash_heads(T, H, Hkv) &&
         max_q > 0 && max_kv > 0;
}

// Checks shared by both entry points; fills what they share.
int flash_args(const char* who, const uint16_t* q, int64_t ldq, int64_t T, int64_t H, int64_t Hkv, int64_t D,
               float scale, uint16_t* out, int64_t ldo, int32_t* error, FlashArgs* a) {
  if (D != 64 && D != 128)
    return set_error(BTL_ERR_SHAPE, "%s: head dim %lld (64 and 128 supported)", who, (long long)D);
  if (!flash_heads(T, H, Hkv))
    return set_error(BTL_ERR_SHAPE, "%s: T=%lld H=%lld Hkv=%lld (H / Hkv <= 64)", who, (long long)T, (long long)H,
                     (long long)Hkv);
  if (!(scale > 0.0f) || !(scale < __builtin_inff()))
    return set_error(BTL_ERR_ARG, "%s: scale %g (positive and finite)", who, (double)scale);
  if (T > 0 && (!q || !out || !error)) return set_error(BTL_ERR_NULL, "%s: NULL pointer", who);
  if (ldq < H * D || ldo < H * D) return set_error(BTL_ERR_SHAPE, "%s: row stride smaller than a row", who);
  if (!aligned(q, 16) || !aligned(out, 16) || !aligned(error, 4) || ldq % 8 || ldo % 8)
    return set_error(BTL_ERR_ALIGN, "%s: misaligned buffer or row stride", who);
  a->q = q;
  a->ldq = ldq;
  a->ldo = ldo;
  a->H = (int)H;
  a->Hkv = (int)Hkv;
  a->G = (int)(H / Hkv);
  a->g = a->G > 1 ? fast_div((uint32_t)a->G) : FastDiv{1, 0, 0};
  a->c = scale * 1.44269504088896340736f;
  a->out = out;
  a->error = error;
  return BTL_OK;
}

}  // namespace btl

using namespace btl;

extern "C" {

int btl_prompt_attention(const uint16_t* q, int64_t ldq, const uint16_t* k, int64_t ldk, const uint16_t* v,
                         int64_t ldv, int64_t T, int64_t H, int64_t Hkv, int64_t D, const int32_t* cu_q, int64_t B,
                         float scale, int64_t max_q, uint16_t* out, int64_t ldo, int32_t* error_word,
                         btl_stream_t stream) {
  const char* who = "btl_prompt_attention";
  clear_error();
  FlashArgs a{};
  int rc = check_batch(who, B, T, cu_q, nullptr, nullptr, 0, &a.bt);
  if (rc != BTL_OK) return rc;
  rc = flash_args(who, q, ldq, T, H, Hkv, D, scale, out, ldo, error_word, &a);
  if (rc != BTL_OK) return rc;
  if (max_q < 0) return set_error(BTL_ERR_SHAPE, "%s: max_q=%lld", who, (long long)max_q);
  if (T == 0) return BTL_OK;
  if (!k || !v) return set_error(BTL_ERR_NULL, "%s: NULL pointer", who);
  if (ldk < Hkv * D || ldv < Hkv * D) return set_error(BTL_ERR_SHAPE, "%s: row stride smaller than a row", who);
  if (ldk > (1 << 24) || ldv > (1 << 24))  // a step's rows within a 32-bit range
    return set_error(BTL_ERR_SHAPE, "%s: row stride over %d elements", who, 1 << 24);
  if (!aligned(k, 16) || !aligned(v, 16) || ldk % 8 || ldv % 8)
    return set_error(BTL_ERR_ALIGN, "%s: misaligned buffer or row stride", who);
  a.k = k;
  a.v = v;
  a.ldk = ldk;
  a.ldv = ldv;
  a.splits = 1;
  const FlashPlan f = flash_plan(T, H, Hkv, D, B, T, T, false);
  const dim3 grid((unsigned)f.tiles);
  if (D == 128)
    hipLaunchKernelGGL((k_flash_tile<128, kDense>), grid, dim3(256), 0, (hipStream_t)stream, a);
  else
    hipLaunchKernelGGL((k_flash_tile<64, kDense>), grid, dim3(256), 0, (hipStream_t)stream, a);
  return check_launch("prompt attention");
}

int64_t btl_paged_attention_scratch_bytes(int64_t T, int64_t H, int64_t Hkv, int64_t D, int64_t B, int64_t max_q,
                                          int64_t max_kv) {
  if (!flash_sizes(T, H, Hkv, D, B, max_q, max_kv)) return 0;
  return flash_scratch(flash_plan(T, H, Hkv, D, B, max_q, max_kv, true), T, H, D);
}

int btl_paged_attention_plan(int64_t T, int64_t H, int64_t Hkv, int64_t D, int64_t B, int64_t max_q, int64_t max_kv,
                             int64_t* plan) {
  if (!plan || !flash_sizes(T, H, Hkv, D, B, max_q, max_kv)) return 0;
  const FlashPlan f = flash_plan(T, H, Hkv, D, B, max_q, max_kv, true);
  plan[0] = f.few;
  plan[1] = f.splits;
  plan[2] = f.chunk;
  return 1;
}

int btl_paged_attention(const uint16_t* q, int64_t ldq, int64_t T, int64_t H, const btl_pages_t* pages,
                        const int32_t* page_table, int64_t max_pages, const int32_t* cu_q, const int32_t* kv_len,
                        int64_t B, float scale, int64_t max_q, int64_t max_kv, uint16_t* out, int64_t ldo,
                        void* scratch, size_t scratch_bytes, int32_t* error_word, btl_stream_t stream) {
  const char* who = "btl_paged_attention";
  clear_error();
  FlashArgs a{};
  int rc = check_pages(who, pages, &a.pg);
  if (rc != BTL_OK) return rc;
  const int64_t Hkv = pages->num_kv_heads, D = pages->head_dim;
  rc = check_batch(who, B, T, cu_q, kv_len, page_table, max_pages, &a.bt);
  if (rc != BTL_OK) return rc;
  rc = flash_args(who, q, ldq, T, H, Hkv, D, scale, out, ldo, error_word, &a);
  if (rc != BTL_OK) return rc;
  if (max_q <= 0 || max_kv <= 0 || max_pages <= 0 || max_pages * pages->page_size > kMaxPositions)
    return set_error(BTL_ERR_SHAPE, "%s: max_q=%lld max_kv=%lld max_pages=%lld", who, (long long)max_q,
                     (long long)max_kv, (long long)max_pages);
  if (T == 0) return BTL_OK;
  if (!page_table || !kv_len) return set_error(BTL_ERR_NULL, "%s: NULL pointer", who);
  const bool fp8 = pages->k_exp != nullptr;
  const FlashPlan f = flash_plan(T, H, Hkv, D, B, max_q, max_kv, true);
  if (f.few && B > 65535) return set_error(BTL_ERR_SHAPE, "%s: %lld sequences", who, (long long)B);
  const int64_t need = flash_scratch(f, T, H, D);
  if (need > 0) {
    if (!scratch || (int64_t)scratch_bytes < need)
      return set_error(BTL_ERR_WORKSPACE, "%s: scratch %zu < %lld bytes", who, scratch ? scratch_bytes : 0,
                       (long long)need);
    if (!aligned(scratch, 16)) return set_error(BTL_ERR_ALIGN, "%s: misaligned scratch", who);
  }
  a.splits = f.splits;
  a.chunk = f.chunk;
  a.part_o = static_cast<float*>(scratch);
  a.part_ml = reinterpret_cast<float2*>(a.part_o + (f.splits > 1 ? (int64_t)f.splits * T * H * D : 0));
  if (f.few) {
    const dim3 grid((unsigned)Hkv, (unsigned)B, (unsigned)f.splits);
    auto* kern = D == 128 ? (fp8 ? k_flash_few<128, kPagedFp8> : k_flash_few<128, kPagedBf16>)
                          : (fp8 ? k_flash_few<64, kPagedFp8> : k_flash_few<64, kPagedBf16>);
    hipLaunchKernelGGL(kern, grid, dim3(64 * kFewWaves), 0, (hipStream_t)stream, a);
  } else {
    const dim3 grid((unsigned)f.tiles, (unsigned)f.splits);
    auto* kern = D == 128 ? (fp8 ? k_flash_tile<128, kPagedFp8> : k_flash_tile<128, kPagedBf16>)
                          : (fp8 ? k_flash_tile<64, kPagedFp8> : k_flash_tile<64, kPagedBf16>);
    hipLaunchKernelGGL(kern, grid, dim3(256), 0, (hipStream_t)stream, a);
  }
  if (f.splits > 1) {
    rc = check_launch("paged attention");
    if (rc != BTL_OK) return rc;
    // up to four splits for a group of threads
    const int ng = D == 128 ? 8 : 16;
    int groups = 1;
    while (groups < ng && 4 * groups < f.splits) groups *= 2;
    const dim3 grid((unsigned)((T * H * groups + ng - 1) / ng));
    if (D == 128)
      hipLaunchKernelGGL(k_flash_merge<128>, grid, dim3(256), 0, (hipStream_t)stream, a, groups);
    else
      hipLaunchKernelGGL(k_flash_merge<64>, grid, dim3(256), 0, (hipStream_t)stream, a, groups);
  }
  return check_launch("paged attention");
}

}  // extern "C"
