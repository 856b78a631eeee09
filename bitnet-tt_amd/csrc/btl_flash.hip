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
// Softmax in base 2: p = 2^(c' s - c' m), c' = c log2(e), in fp32; m is a running
// maximum that is only raised, and the output rescaled, where a row's maximum
// grew by more than 2^kLazy (p then stays below 2^kLazy, which costs an fp32 sum
// nothing).  p is rounded to bf16 for the second product, the matrix units'
// operand type; the sum takes p unrounded.
//
// Rows of V behind the last position read as zero (whatever lies there), and a
// value that is not finite at a position that some of the tile's rows may not see is added
// to the rows that do see it and multiplied with none: 0 x inf is NaN.
#include <hip/hip_runtime.h>

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
  // split the rest, and leaves a partial per row
  int splits, chunk;
  float* part_o;    // [splits][T][H][D]
  float2* part_ml;  // [splits][T][H]: maximum (in score units), sum
};

__device__ const uint4 g_zero_row[16] = {};  // 256 bytes that read as zero

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

// Loads from memory, not from LDS: a flat load would count as both.
__device__ __forceinline__ uint4 mem_ld128(const uint8_t* p) {
  typedef uint32_t v4u __attribute__((ext_vector_type(4)));
  const v4u v = *(const __attribute__((address_space(1))) v4u*)p;
  return make_uint4(v[0], v[1], v[2], v[3]);
}
__device__ __forceinline__ uint32_t mem_ld8(const uint8_t* p) { return *(const __attribute__((address_space(1))) uint8_t*)p; }

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
// Keys and values go to LDS as bf16, two stages of each: 64 KiB at D = 128, so two
// workgroups share a CU and one's softmax runs under the other's MFMAs.  A step's
// loads are issued one step ahead of their use; one barrier a step.  16-byte pieces of a row are
// stored at piece ^ f(row): for K, f = row, so that 8 lanes that read the same
// piece of 8 rows hit different banks; for V, f = 2 row, so that the 4 rows x 32
// bytes of a transposing read do.
// ======================================================================
constexpr int kTileRows = 128;
constexpr int kStep = 64;

template <int D>
struct Tile {
  static constexpr int kPieces = D / 8;                // 16-byte pieces of a bf16 row
  static constexpr int kBytes = kStep * D * 2;         // one stage of K, or of V
  static constexpr int kLoads = kBytes / (256 * 16);   // 16-byte loads of a thread for it
  static constexpr int kRowsLoad = 256 / kPieces;      // rows that one load of every thread covers
  static __device__ __forceinline__ int k_swz(int row) { return row & (kPieces - 1); }
  static __device__ __forceinline__ int v_swz(int row) { return (2 * row) & (kPieces - 1); }
};

// Where a step's rows come from: the sequence's packed rows, or its pages.
// A thread's rows of a step are i * RPL + tid / TPR for its loads i (TPR threads
// to a row); each run of 16 rows is in one page.
template <int D, int KV>
struct Source {
  static constexpr int kRowBytes = KV == kPagedFp8 ? D : 2 * D;
  static constexpr int kTpr = kRowBytes / 16;      // threads of a row
  static constexpr int kRpl = 256 / kTpr;          // rows of a load
  static constexpr int kN = kStep / kRpl;          // loads of a thread
  int32_t page[kN];                                // pages of the next step's row runs
  const uint8_t* k;
  const uint8_t* v;
  int64_t ldk, ldv;   // bytes
  const int32_t* table;
  int hk, kv_end;
  bool bad;

  __device__ __forceinline__ void init(const FlashArgs& p, const Seq& s, int b, int hk_, int kv_end_) {
    hk = hk_;
    kv_end = kv_end_;
    bad = false;
    if (KV == kDense) {
      ldk = p.ldk * 2;
      ldv = p.ldv * 2;
      k = reinterpret_cast<const uint8_t*>(p.k + (int64_t)s.row0 * p.ldk + hk * D);
      v = reinterpret_cast<const uint8_t*>(p.v + (int64_t)s.row0 * p.ldv + hk * D);
    } else {
      table = p.bt.table + (int64_t)b * p.bt.max_pages;
    }
  }
  // Run of 16 rows that this wave's rows of load i lie in.
  __device__ __forceinline__ int run(int kv, int i) const {
    return kv + i * kRpl + (uni(threadIdx.x) / kTpr & ~15);
  }
  __device__ __forceinline__ void fetch_pages(const FlashArgs& p, int kv) {
    if (KV == kDense) return;
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int at = run(kv, i);
      page[i] = 0;
      if (at < kv_end) page[i] = scalar_load(table, div_by(at, p.pg.ps));
    }
  }
  // The row of load i as (address of its first byte in k, in v, exponent index);
  // a row behind the end or in no page reads zeros.
  __device__ __forceinline__ void row(const FlashArgs& p, int kv, int i, const uint8_t*& rk, const uint8_t*& rv,
                                      int64_t& at) {
    const int pos = kv + i * kRpl + (int)threadIdx.x / kTpr;
    at = -1;
    if (KV == kDense) {
      rk = k + (int64_t)pos * ldk;
      rv = v + (int64_t)pos * ldv;
    } else {
      const int r0 = run(kv, i);
      const int32_t id = page[i];
      const int64_t base = page_row(id, p.pg.P, p.pg.Hkv, hk, p.pg.ps.d,
                                    r0 - (int)div_by(r0, p.pg.ps) * (int)p.pg.ps.d);
      if (base < 0 && r0 < kv_end) bad = true;
      at = base < 0 ? -1 : base + (pos - r0);
      rk = at < 0 ? reinterpret_cast<const uint8_t*>(g_zero_row) : p.pg.k + at * kRowBytes;
      rv = at < 0 ? reinterpret_cast<const uint8_t*>(g_zero_row) : p.pg.v + at * kRowBytes;
    }
    if (pos >= kv_end) {
      rk = rv = reinterpret_cast<const uint8_t*>(g_zero_row);
      at = -1;
    }
  }
};

// A step's rows on their way from memory to LDS.  (Through registers: loads
// into LDS directly would cost none, but the compiler takes every LDS read
// to depend on them, and would wait for the next step's rows before reading this one's.)
template <int N>
struct Staged {
  uint4 k[N], v[N];
  uint32_t ke[N], ve[N];  // exponent bytes (8-bit pages)
};

template <int D, int KV>
__device__ __forceinline__ void load_step(const FlashArgs& p, Source<D, KV>& src, int kv,
                                          Staged<Source<D, KV>::kN>& st) {
  using S = Source<D, KV>;
  const int c = threadIdx.x % S::kTpr;
#pragma unroll
  for (int i = 0; i < S::kN; ++i) {
    const uint8_t *rk, *rv;
    int64_t at;
    src.row(p, kv, i, rk, rv, at);
    st.k[i] = mem_ld128(rk + 16 * c);
    st.v[i] = mem_ld128(rv + 16 * c);
    if (KV == kPagedFp8) {
      st.ke[i] = st.ve[i] = 127;
      if (at >= 0) {
        st.ke[i] = mem_ld8(p.pg.ke + at);
        st.ve[i] = mem_ld8(p.pg.ve + at);
      }
    }
  }
}

template <int D, int KV>
__device__ __forceinline__ void store_step(lds8* ks, lds8* vs, const Staged<Source<D, KV>::kN>& st) {
  using S = Source<D, KV>;
  const int c = threadIdx.x % S::kTpr;
#pragma unroll
  for (int i = 0; i < S::kN; ++i) {
    const int r = i * S::kRpl + threadIdx.x / S::kTpr;
    lds8 *const k = ks + r * 2 * D, *const v = vs + r * 2 * D;
    if (KV == kPagedFp8) {
      const float fk = exp_scale(st.ke[i]), fv = exp_scale(st.ve[i]);
      const int k0 = 2 * c ^ Tile<D>::k_swz(r), v0 = 2 * c ^ Tile<D>::v_swz(r);
      lds_st128(k + k0 * 16, from_e4m3(make_uint2(st.k[i].x, st.k[i].y), fk));
      lds_st128(k + (k0 ^ 1) * 16, from_e4m3(make_uint2(st.k[i].z, st.k[i].w), fk));
      lds_st128(v + v0 * 16, from_e4m3(make_uint2(st.v[i].x, st.v[i].y), fv));
      lds_st128(v + (v0 ^ 1) * 16, from_e4m3(make_uint2(st.v[i].z, st.v[i].w), fv));
    } else {
      lds_st128(k + (c ^ Tile<D>::k_swz(r)) * 16, st.k[i]);
      lds_st128(v + (c ^ Tile<D>::v_swz(r)) * 16, st.v[i]);
    }
  }
}

template <int D>
struct TileState {
  v8bf q[D / 16];   // B operands: this lane's query row, dims 16 ks + 8 h ..
  v16f o[D / 32];   // O^T: element r of o[t] is dim 32 t + acc_row(r) of the lane's row
  float m, l;       // running maximum (score units), this lane's share of the sum
  int limit;        // the last position that the lane's row sees, -1: none
  int lo, hi;       // of the wave's rows: least limit, greatest
};

__device__ __forceinline__ int c_row(int r, int h) { return 8 * (r >> 2) + 4 * h + (r & 3); }

// Scores of the step, softmax, and the probabilities as operands.
template <int D, bool MASK>
__device__ __forceinline__ void step_scores(const lds8* ks, TileState<D>& s, float c, int kv, v8bf (&pb)[4]) {
  const int lane = __lane_id(), h = lane >> 5, r32 = lane & 31;
  v16f sc[2];
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) sc[t][r] = 0.0f;
  const lds8* row = ks + r32 * 2 * D;
  const int x = Tile<D>::k_swz(r32) ^ h;
#pragma unroll
  for (int k = 0; k < D / 16; ++k) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const v8bf a = lds_ld_bf8(row + t * 32 * 2 * D + ((x ^ (2 * k)) * 16));
      sc[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, s.q[k], sc[t], 0, 0, 0);
    }
  }
  if (MASK) {
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (kv + 32 * t + c_row(r, h) > s.limit) sc[t][r] = kNegInf;
  }
  float mx = sc[0][0];
#pragma unroll
  for (int i = 1; i < 32; ++i) mx = fmaxf(mx, sc[i >> 4][i & 15]);
  mx = fmaxf(mx, xor_partner<32>(mx));
  if (__any(mx > s.m && (mx - s.m) * c > kLazy)) {  // (m = -inf: any score is more)
    const float mn = fmaxf(s.m, mx);
    const float a = s.m == kNegInf ? 0.0f : __builtin_amdgcn_exp2f((s.m - mn) * c);
    s.m = mn;
    s.l *= a;
#pragma unroll
    for (int t = 0; t < D / 32; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) s.o[t][r] *= a;
  }
  const float mc = s.m == kNegInf ? 0.0f : -s.m * c;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float e0 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t][8 * k + 2 * j], c, mc));
        const float e1 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t][8 * k + 2 * j + 1], c, mc));
        s.l += e0 + e1;
        w[j] = f2bf_pair(e0, e1);
      }
      pb[2 * t + k] = __builtin_bit_cast(v8bf, make_uint4(w[0], w[1], w[2], w[3]));
    }
  }
}

template <int D>
__device__ __forceinline__ void step_values(const lds8* vs, TileState<D>& s, const v8bf (&pb)[4]) {
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
__device__ __forceinline__ void add_not_finite(lds8* vs, TileState<D>& s, int kv) {
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
  __shared__ __attribute__((aligned(16))) uint8_t smem[4 * Tile<D>::kBytes];
  __shared__ int s_flag[4];
  const int tid = threadIdx.x, wv = uni(tid >> 6), lane = tid & 63, h = lane >> 5;
  const int hk = blockIdx.x % p.Hkv, split = blockIdx.y;
  Item it;
  if (!find_item(p.bt, p.G, kTileRows, blockIdx.x / p.Hkv, it)) return;
  const int64_t cap = (int64_t)p.bt.max_pages * p.pg.ps.d;
  const Seq sq = load_seq(p.bt, it.b, cap);
  if (!sq.ok && tid == 0) flag_error(p.error);
  const int rows = sq.n * p.G, first = sq.len - sq.n;  // position of the first token
  const int r0 = (it.count - 1 - it.i) * kTileRows;     // the longest tiles first
  const int t_last = row_token(min(r0 + kTileRows, rows) - 1, p);

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
  s.l = 0.0f;

  const int wg_lo = max(-1, first + row_token(r0, p));
  int kv_end = max(0, first + t_last + 1);
  int kv0 = 0;
  if (p.splits > 1) {
    kv0 = split * p.chunk;
    if (split + 1 < p.splits) kv_end = min(kv_end, kv0 + p.chunk);
  }
  if (kv0 < kv_end) {
    lds8* const sm = (lds8*)smem;
    Source<D, KV> src;
    Staged<Source<D, KV>::kN> st;
    src.init(p, sq, it.b, hk, kv_end);
    src.fetch_pages(p, kv0);
    load_step<D, KV>(p, src, kv0, st);
    src.fetch_pages(p, kv0 + kStep);
    store_step<D, KV>(sm, sm + Tile<D>::kBytes, st);
    int kv = kv0, at = 0;  // the step's rows are in stage `at` (keys, then values), the next step's go to the other
    // steps that every row of the tile sees whole
    for (; kv < kv_end && kv + kStep - 1 <= wg_lo; kv += kStep, at ^= 1) {
      lds8* const ks = sm + at * 2 * Tile<D>::kBytes;
      lds8* const kn = sm + (at ^ 1) * 2 * Tile<D>::kBytes;
      lds_barrier();  // the step's rows are in LDS, and the other stage is free
      const bool more = kv + kStep < kv_end;
      if (more) {
        load_step<D, KV>(p, src, kv + kStep, st);
        src.fetch_pages(p, kv + 2 * kStep);
      }
      v8bf pb[4];
      step_scores<D, false>(ks, s, p.c, kv, pb);
      step_values<D>(ks + Tile<D>::kBytes, s, pb);
      if (more) store_step<D, KV>(kn, kn + Tile<D>::kBytes, st);
    }
    for (; kv < kv_end; kv += kStep, at ^= 1) {
      lds8* const ks = sm + at * 2 * Tile<D>::kBytes;
      lds8* const vs = ks + Tile<D>::kBytes;
      lds8* const kn = sm + (at ^ 1) * 2 * Tile<D>::kBytes;
      lds_barrier();
      const bool more = kv + kStep < kv_end;
      if (more) {
        load_step<D, KV>(p, src, kv + kStep, st);
        src.fetch_pages(p, kv + 2 * kStep);
      }
      bool nf = false;
#pragma unroll
      for (int i = 0; i < Tile<D>::kLoads; ++i) nf |= any_not_finite(lds_ld128(vs + (i * 256 + tid) * 16));
      const bool any = __any(nf);
      if (lane == 0) s_flag[wv] = any;
      lds_barrier();
      const bool special = s_flag[0] | s_flag[1] | s_flag[2] | s_flag[3];
      const bool mine = kv <= s.hi;  // some of the wave's rows see some of it
      v8bf pb[4];
      if (mine) step_scores<D, true>(ks, s, p.c, kv, pb);
      if (special) {
        if (mine) add_not_finite<D>(vs, s, kv);
        lds_barrier();
#pragma unroll
        for (int i = 0; i < Tile<D>::kLoads; ++i) {
          lds8* const at = vs + (i * 256 + tid) * 16;
          const uint4 x = lds_ld128(at);
          lds_st128(at, make_uint4(drop_not_finite(x.x), drop_not_finite(x.y), drop_not_finite(x.z),
                                   drop_not_finite(x.w)));
        }
        lds_barrier();
      }
      if (mine) step_values<D>(vs, s, pb);
      if (more) store_step<D, KV>(kn, kn + Tile<D>::kBytes, st);
    }
    if (KV != kDense && src.bad) flag_error(p.error);
  }

  const float l = s.l + xor_partner<32>(s.l);
  if (r >= rows) return;
  const int64_t row = sq.row0 + tok;
  if (p.splits > 1) {
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
// drafts): bound by the bytes of keys and values.  8 waves share a context,
// 32 positions each a round; a wave's keys go straight from memory to the MFMA's
// registers, its values through its own 8 KiB of LDS, and the next round's
// loads are issued before this one is computed, so 256 KiB a CU are on their way.
// The waves' partials meet in LDS.
// ======================================================================
constexpr int kFewRows = 16;
constexpr int kFewWaves = 8;
constexpr int kFewPos = 32;  // positions of a wave and round

template <int D>
struct FewShared {
  union {
    uint8_t v[kFewWaves][kFewPos * 2 * D];
    float o[kFewWaves][kFewRows][D];  // after the last round
  };
  float ml[kFewWaves][kFewRows][2];
};

template <int D, int KV>
struct FewRound {
  static constexpr int kRowBytes = KV == kPagedFp8 ? D : 2 * D;
  static constexpr int kK = kRowBytes / 64;                 // key loads of a lane per 16 rows
  static constexpr int kV = kFewPos * kRowBytes / 1024;     // value loads of a lane
  uint4 k[2][kK];
  uint4 v[kV];
  uint32_t ke[2], ve[kV];
};

template <int D, int KV>
__device__ __forceinline__ void few_load(const FlashArgs& p, const int32_t* table, int hk, int kv, int kv_end,
                                         FewRound<D, KV>& r, bool& bad) {
  using R = FewRound<D, KV>;
  const int lane = __lane_id();
  int64_t base[2];  // page row of each run of 16 positions
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int at = kv + 16 * t;
    base[t] = -1;
    if (at < kv_end) {
      const uint32_t pi = div_by(at, p.pg.ps);
      base[t] = page_row(scalar_load(table, pi), p.pg.P, p.pg.Hkv, hk, p.pg.ps.d, at - (int)pi * (int)p.pg.ps.d);
      if (base[t] < 0) bad = true;
    }
  }
  const uint8_t* const zero = reinterpret_cast<const uint8_t*>(g_zero_row);
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int row = lane & 15;
    const bool ok = base[t] >= 0 && kv + 16 * t + row < kv_end;
    const int64_t at = base[t] + row;
    const uint8_t* a = ok ? p.pg.k + at * R::kRowBytes : zero;
#pragma unroll
    for (int i = 0; i < R::kK; ++i) r.k[t][i] = mem_ld128(a + 64 * i + 16 * (lane >> 4));
    r.ke[t] = 127;
    if (KV == kPagedFp8 && ok) r.ke[t] = mem_ld8(p.pg.ke + at);
  }
  constexpr int TPR = R::kRowBytes / 16, RPL = 64 / TPR;
#pragma unroll
  for (int i = 0; i < R::kV; ++i) {
    const int row = i * RPL + lane / TPR, t = (i * RPL) / 16;  // RPL <= 16: a load's rows are in one run
    const bool ok = base[t] >= 0 && kv + row < kv_end;
    const int64_t at = base[t] + row - 16 * t;
    const uint8_t* a = ok ? p.pg.v + at * R::kRowBytes : zero;
    r.v[i] = mem_ld128(a + 16 * (lane % TPR));
    r.ve[i] = 127;
    if (KV == kPagedFp8 && ok) r.ve[i] = mem_ld8(p.pg.ve + at);
  }
}

template <int D, int KV>
__global__ __launch_bounds__(64 * kFewWaves, 2) void k_flash_few(FlashArgs p) {
  using R = FewRound<D, KV>;
  __shared__ __attribute__((aligned(16))) FewShared<D> s;
  const int tid = threadIdx.x, wv = uni(tid >> 6), lane = tid & 63, r16 = lane & 15, grp = lane >> 4;
  const int hk = blockIdx.x, b = blockIdx.y, split = blockIdx.z;
  const Seq sq = load_seq(p.bt, b, (int64_t)p.bt.max_pages * p.pg.ps.d);
  if (!sq.ok && tid == 0) flag_error(p.error);
  const int rows = sq.n * p.G, first = sq.len - sq.n;
  const int32_t* const table = p.bt.table + (int64_t)b * p.bt.max_pages;
  int seq_end = sq.len, kv0 = 0;
  if (p.splits > 1) {
    kv0 = split * p.chunk;
    if (split + 1 < p.splits) seq_end = min(seq_end, kv0 + p.chunk);
  }
  constexpr int PC = D / 8;  // 16-byte pieces of a bf16 row
  bool bad = false;
  // one pass unless there are more rows than the caller said
  for (int r0 = 0; r0 < rows; r0 += kFewRows) {
    const int r = r0 + r16, rc = min(r, rows - 1);
    const int tok = row_token(rc, p), head = hk * p.G + rc - tok * p.G;
    const int limit = r < rows ? max(-1, first + tok) : -1;
    const int lo = max(-1, first + row_token(r0, p));
    const int kv_end = min(seq_end, max(0, first + row_token(min(r0 + kFewRows, rows) - 1, p) + 1));
    FewRound<D, KV> cur;
    int kv = kv0 + kFewPos * wv;
    if (kv < kv_end) few_load<D, KV>(p, table, hk, kv, kv_end, cur, bad);
    // B operands: bf16 keys give a lane 8 dims of each 32, 8-bit keys 16 of each 64
    v8bf q[D / 32];
    {
      const uint16_t* a = p.q + (int64_t)(sq.row0 + tok) * p.ldq + head * D;
#pragma unroll
      for (int k = 0; k < D / 32; ++k) {
        const int d = KV == kPagedFp8 ? 64 * (k / 2) + 16 * grp + 8 * (k & 1) : 32 * k + 8 * grp;
        q[k] = __builtin_bit_cast(v8bf, *reinterpret_cast<const uint4*>(a + d));
      }
    }
    v4f o[D / 16];
#pragma unroll
    for (int t = 0; t < D / 16; ++t) o[t] = (v4f){0.f, 0.f, 0.f, 0.f};
    float m = kNegInf, l = 0.0f;
    lds8* const vs = (lds8*)&s.v[wv][0];

    for (; kv < kv_end; kv += kFewPos * kFewWaves) {
      // scores: positions 16 t + 4 grp + i of query r16
      v4f sc[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        sc[t] = (v4f){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < D / 32; ++k) {
          uint4 a;
          if (KV == kPagedFp8) {
            const uint4 w = cur.k[t][k / 2];
            a = from_e4m3(k & 1 ? make_uint2(w.z, w.w) : make_uint2(w.x, w.y), exp_scale(cur.ke[t]));
          } else {
            a = cur.k[t][k];
          }
          sc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), q[k], sc[t], 0, 0, 0);
        }
      }
      // this round's value rows to LDS (pieces at piece ^ 2 row, for the transposing reads)
      bool nf = false;
      {
        constexpr int TPR = R::kRowBytes / 16, RPL = 64 / TPR;
#pragma unroll
        for (int i = 0; i < R::kV; ++i) {
          const int row = i * RPL + lane / TPR, c = lane % TPR;
          if (KV == kPagedFp8) {
            const float f = exp_scale(cur.ve[i]);
            const uint4 a = from_e4m3(make_uint2(cur.v[i].x, cur.v[i].y), f);
            const uint4 e = from_e4m3(make_uint2(cur.v[i].z, cur.v[i].w), f);
            const int c0 = 2 * c ^ Tile<D>::v_swz(row);
            lds_st128(vs + row * 2 * D + c0 * 16, a);
            lds_st128(vs + row * 2 * D + (c0 ^ 1) * 16, e);
            nf |= any_not_finite(a) | any_not_finite(e);
          } else {
            lds_st128(vs + row * 2 * D + (c ^ Tile<D>::v_swz(row)) * 16, cur.v[i]);
            nf |= any_not_finite(cur.v[i]);
          }
        }
      }
      const int at = kv;
      if (kv + kFewPos * kFewWaves < kv_end)
        few_load<D, KV>(p, table, hk, kv + kFewPos * kFewWaves, kv_end, cur, bad);

      float mx = kNegInf;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (at + 16 * t + 4 * grp + i > limit) sc[t][i] = kNegInf;
          mx = fmaxf(mx, sc[t][i]);
        }
      mx = fmaxf(mx, xor_partner<16>(mx));
      mx = fmaxf(mx, xor_partner<32>(mx));
      if (__any(mx > m)) {
        const float mn = fmaxf(m, mx);
        const float a = m == kNegInf ? 0.0f : __builtin_amdgcn_exp2f((m - mn) * p.c);
        m = mn;
        l *= a;
#pragma unroll
        for (int t = 0; t < D / 16; ++t) o[t] *= a;
      }
      const float mc = m == kNegInf ? 0.0f : -m * p.c;
      uint32_t w[4];
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float e0 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t][2 * i], p.c, mc));
          const float e1 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t][2 * i + 1], p.c, mc));
          l += e0 + e1;
          w[2 * t + i] = f2bf_pair(e0, e1);
        }
      const v8bf pb = __builtin_bit_cast(v8bf, make_uint4(w[0], w[1], w[2], w[3]));
      __builtin_amdgcn_wave_barrier();  // the wave's LDS rows are read back by other lanes
      if (at + kFewPos - 1 > lo && __any(nf)) {
        for (int j = 0; j < kFewPos; ++j)
#pragma unroll
          for (int t = 0; t < D / 16; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int d = 16 * t + 4 * grp + i;
              const uint16_t x = *(const __attribute__((address_space(3))) uint16_t*)(
                  vs + j * 2 * D + ((d / 8) ^ Tile<D>::v_swz(j)) * 16 + (d % 8) * 2);
              if ((x & 0x7f80u) == 0x7f80u && at + j <= limit) o[t][i] += bf2f(x);
            }
        __builtin_amdgcn_wave_barrier();
        for (int i = lane; i < kFewPos * PC; i += 64) {
          const uint4 x = lds_ld128(vs + i * 16);
          lds_st128(vs + i * 16, make_uint4(drop_not_finite(x.x), drop_not_finite(x.y), drop_not_finite(x.z),
                                            drop_not_finite(x.w)));
        }
        __builtin_amdgcn_wave_barrier();
      }
      // O^T += V^T P^T: dim 16 t + r16 of positions {4 grp .., 16 + 4 grp ..}
      const int rr = r16 >> 2, qq = r16 & 3, row = 4 * grp + rr;
      const lds8* const vb = vs + row * 2 * D + (qq & 1) * 8;
#pragma unroll
      for (int t = 0; t < D / 16; ++t) {
        const lds8* a = vb + (((2 * t + (qq >> 1)) ^ Tile<D>::v_swz(row)) * 16);
        const v4s x = lds_tr16(a), y = lds_tr16(a + 16 * 2 * D);
        const v8bf va = __builtin_bit_cast(v8bf, (v8s){x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w});
        o[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(va, pb, o[t], 0, 0, 0);
      }
      __builtin_amdgcn_wave_barrier();  // reads done before the rows are written again
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
        if (empty(mw, lw)) continue;
        const float f = __builtin_amdgcn_exp2f((mw - M) * p.c);
        L += f * lw;
#pragma unroll
        for (int j = 0; j < 4; ++j) O[j] += f * s.o[w][x][d + j];
      }
      const int tk = row_token(r0 + x, p), hd = hk * p.G + r0 + x - tk * p.G;
      const int64_t row = sq.row0 + tk;
      if (p.splits > 1) {
        const int64_t at = ((int64_t)split * p.bt.T + row) * p.H + hd;
        if (d == 0) p.part_ml[at] = make_float2(M, L);
        if (!empty(M, L)) *reinterpret_cast<float4*>(p.part_o + at * D + d) = make_float4(O[0], O[1], O[2], O[3]);
      } else {
        const float inv = empty(M, L) ? 0.0f : 1.0f / L;
        *reinterpret_cast<uint2*>(p.out + row * p.ldo + hd * D + d) =
            make_uint2(f2bf_pair(O[0] * inv, O[1] * inv), f2bf_pair(O[2] * inv, O[3] * inv));
      }
    }
    __syncthreads();  // before the next rows' values
  }
  if (bad) flag_error(p.error);
}

// The splits' partials of a row, in split order; D / 4 threads a row.
template <int D>
__global__ __launch_bounds__(256) void k_flash_merge(FlashArgs p) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, row = i / (D / 4);  // row: (token, head)
  const int d = 4 * (int)(i % (D / 4));
  const int tok = (int)(row / p.H), head = (int)(row - (int64_t)tok * p.H);
  if (tok < max(0, p.bt.cu[0]) || tok >= min(p.bt.T, p.bt.cu[p.bt.B])) return;
  const int64_t n = (int64_t)p.bt.T * p.H;
  float M = kNegInf;
  for (int z = 0; z < p.splits; ++z) M = fmaxf(M, p.part_ml[z * n + row].x);
  float L = 0.0f;
  v4f O = (v4f){0.f, 0.f, 0.f, 0.f};
  for (int z = 0; z < p.splits; ++z) {
    const float2 ml = p.part_ml[z * n + row];
    if (empty(ml.x, ml.y)) continue;
    const float f = __builtin_amdgcn_exp2f((ml.x - M) * p.c);
    const float4 o = *reinterpret_cast<const float4*>(p.part_o + (z * n + row) * D + d);
    L += f * ml.y;
    O[0] += f * o.x;
    O[1] += f * o.y;
    O[2] += f * o.z;
    O[3] += f * o.w;
  }
  const float inv = empty(M, L) ? 0.0f : 1.0f / L;
  *reinterpret_cast<uint2*>(p.out + tok * p.ldo + head * D + d) =
      make_uint2(f2bf_pair(O[0] * inv, O[1] * inv), f2bf_pair(O[2] * inv, O[3] * inv));
}

// ---- host ---------------------------------------------------------------
struct FlashPlan {
  bool few;
  int64_t tiles;  // workgroups per split
  int splits;
  int64_t chunk;
};
// Few rows: the kernel of single tokens where a sequence's rows fit one of its
// tiles.  Splits: enough workgroups for the chip where the rows alone give
// too few, each of at least kMinChunk positions.
constexpr int64_t kMinChunk = 512;
constexpr int64_t kMaxSplits = 256;
inline FlashPlan flash_plan(int64_t T, int64_t H, int64_t Hkv, int64_t B, int64_t max_q, int64_t max_kv, bool paged) {
  FlashPlan f{};
  const int64_t G = H / Hkv;
  f.few = paged && max_q * G <= kFewRows;
  f.tiles = (f.few ? B : T * G / kTileRows + (B < T ? B : T)) * Hkv;
  f.splits = 1;
  f.chunk = round_up(max_kv > 0 ? max_kv : 1, 256);
  const int64_t slots = (int64_t)device_cus() * (f.few ? 1 : 2);
  if (paged && 2 * f.tiles <= slots && max_kv > kMinChunk) {
    int64_t n = slots / f.tiles;
    if (n > max_kv / kMinChunk) n = max_kv / kMinChunk;
    if (n > kMaxSplits) n = kMaxSplits;
    if (n > 1) {
      f.chunk = round_up((max_kv + n - 1) / n, 256);
      f.splits = (int)((max_kv + f.chunk - 1) / f.chunk);
    }
  }
  return f;
}

inline int64_t flash_scratch(const FlashPlan& f, int64_t T, int64_t H, int64_t D) {
  return f.splits > 1 ? (int64_t)f.splits * T * H * (D + 2) * 4 : 0;
}

// Checks shared by both entry points; fills what they share.
int flash_args(const char* who, const uint16_t* q, int64_t ldq, int64_t T, int64_t H, int64_t Hkv, int64_t D,
               float scale, uint16_t* out, int64_t ldo, int32_t* error, FlashArgs* a) {
  if (D != 64 && D != 128)
    return set_error(BTL_ERR_SHAPE, "%s: head dim %lld (64 and 128 supported)", who, (long long)D);
  if (H <= 0 || Hkv <= 0 || H > 1024 || H % Hkv || H / Hkv > 64 || T * H > INT32_MAX / 2)
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
  if (!aligned(k, 16) || !aligned(v, 16) || ldk % 8 || ldv % 8)
    return set_error(BTL_ERR_ALIGN, "%s: misaligned buffer or row stride", who);
  a.k = k;
  a.v = v;
  a.ldk = ldk;
  a.ldv = ldv;
  a.splits = 1;
  const FlashPlan f = flash_plan(T, H, Hkv, B, T, T, false);
  const dim3 grid((unsigned)f.tiles);
  if (D == 128)
    hipLaunchKernelGGL((k_flash_tile<128, kDense>), grid, dim3(256), 0, (hipStream_t)stream, a);
  else
    hipLaunchKernelGGL((k_flash_tile<64, kDense>), grid, dim3(256), 0, (hipStream_t)stream, a);
  return check_launch("prompt attention");
}

int64_t btl_paged_attention_scratch_bytes(int64_t T, int64_t H, int64_t Hkv, int64_t D, int64_t B, int64_t max_q,
                                          int64_t max_kv) {
  if (T <= 0 || H <= 0 || Hkv <= 0 || H % Hkv || B <= 0 || max_q <= 0 || max_kv <= 0) return 0;
  return flash_scratch(flash_plan(T, H, Hkv, B, max_q, max_kv, true), T, H, D);
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
  if (max_q <= 0 || max_kv <= 0 || max_pages <= 0 || max_pages * pages->page_size > INT32_MAX / 2)
    return set_error(BTL_ERR_SHAPE, "%s: max_q=%lld max_kv=%lld max_pages=%lld", who, (long long)max_q,
                     (long long)max_kv, (long long)max_pages);
  if (T == 0) return BTL_OK;
  if (!page_table || !kv_len) return set_error(BTL_ERR_NULL, "%s: NULL pointer", who);
  const FlashPlan f = flash_plan(T, H, Hkv, B, max_q, max_kv, true);
  if (f.few && B > 65535) return set_error(BTL_ERR_SHAPE, "%s: %lld sequences", who, (long long)B);
  const int64_t need = flash_scratch(f, T, H, D);
  if (need > 0) {
    if (!scratch || (int64_t)scratch_bytes < need)
      return set_error(BTL_ERR_WORKSPACE, "%s: scratch %zu < %lld bytes", who, scratch ? scratch_bytes : 0,
                       (long long)need);
    if (!aligned(scratch, 16)) return set_error(BTL_ERR_ALIGN, "%s: misaligned scratch", who);
  }
  a.splits = f.splits;
  a.chunk = (int)f.chunk;
  a.part_o = static_cast<float*>(scratch);
  a.part_ml = reinterpret_cast<float2*>(a.part_o + (f.splits > 1 ? (int64_t)f.splits * T * H * D : 0));
  const bool fp8 = pages->k_exp != nullptr;
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
    const dim3 grid((unsigned)((T * H * (D / 4) + 255) / 256));
    if (D == 128)
      hipLaunchKernelGGL(k_flash_merge<128>, grid, dim3(256), 0, (hipStream_t)stream, a);
    else
      hipLaunchKernelGGL(k_flash_merge<64>, grid, dim3(256), 0, (hipStream_t)stream, a);
  }
  return check_launch("paged attention");
}

}  // extern "C"
