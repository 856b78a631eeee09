// Products of 8-bit integers with a scale for each row (token) and each column (channel):
//
//   out[m, n] = (sum_k a[m, k] w[n, k]) sa[m] sw[n]
//
// The sum is exact in 32 bits (K up to 16384: below 2^28); it becomes fp32 (one rounding from 2^24 on),
// is multiplied by the row's scale and then the column's, each rounded to fp32, and rounded to
// bf16 where that is the output.
//
// Weights are laid out once: blocks of 16 columns x 64 k, 1 KiB, [ceil(N/16)][ceil(K/64)], a
// lane's 16 bytes being those that v_mfma_i32_16x16x64_i8 takes from it (column lane % 16, k
// 16 (lane / 16) ..), zeros behind N and K.  A wave's operand is one coalesced load, from
// memory to registers or to LDS.  Weights are the MFMA's first operand, so that a lane holds four
// neighbouring columns of one row.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "btl.h"
#include "btl_act_row.h"
#include "btl_common.h"
#include "btl_mfma.h"

namespace btl {

typedef __attribute__((address_space(3))) uint8_t lds8;

struct Int8Args {
  const int8_t* a;
  int64_t lda;
  const float* sa;
  const uint8_t* w;
  const float* sw;
  int M, K, N, KB, NT;  // KB, NT: blocks of 64 k, of 16 columns
  void* out;
  int64_t ldo;
  int f32, vec;  // vec: rows of out are 16-byte aligned
  // few rows, the head: out may be missing; the first index of each row's largest output
  int32_t* tokens;
  uint64_t* keys;   // [M], zero at first
  uint32_t* count;  // workgroups that are done, zero at first
};

// An output's place in the order (value, then the lower index); 0: a NaN.
__device__ __forceinline__ uint64_t arg_key(float y, int col) {
  const uint32_t u = __float_as_uint(y + 0.0f);  // (both zeros alike)
  const uint32_t order = (u & 0x80000000u) ? ~u : u | 0x80000000u;
  return y == y ? ((uint64_t)order << 32) | (0xffffffffu - (uint32_t)col) : 0u;
}
__device__ __forceinline__ uint64_t arg_max(uint64_t a, uint64_t b) { return a > b ? a : b; }
__device__ __forceinline__ int32_t arg_col(uint64_t key) { return key ? (int32_t)(0xffffffffu - (uint32_t)key) : -1; }

__device__ __forceinline__ int uni8(int x) { return __builtin_amdgcn_readfirstlane(x); }

// A buffer resource at a scalar address; a piece behind its `bytes` reads as zeros and costs no traffic.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc8(const void* p, uint32_t bytes) {
  const uint64_t at = reinterpret_cast<uint64_t>(p);
  const uint32_t lo = (uint32_t)uni8((int)(uint32_t)at), hi = (uint32_t)uni8((int)(at >> 32));
  return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(((uint64_t)hi << 32) | lo), (short)0,
                                           uni8((int)bytes), 0x00020000);
}
__device__ __forceinline__ v4i buf128(__amdgpu_buffer_rsrc_t r, uint32_t off) {
  return __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(r, (int)off, 0, 0));
}

__device__ __forceinline__ float scaled(int acc, float sa, float sw) { return (float)acc * sa * sw; }

// ======================================================================
// Few rows: a stream of weights.  A workgroup takes groups of CT column blocks, its 8 waves the
// blocks of 64 k in turn (wave w: w, w + 8, ...); the waves' sums meet in LDS.  A wave has two sets of U x CT
// loads: while it works on one, the other's are on their way, across the sums of a group as well.  ONCE: a
// wave's blocks are one set (K <= 512 U), so that its rows stay in registers for all groups.
//
// Bound by the weights' bytes: 128256 columns of 2560 to bf16, 1 / 16 / 32 / 64 rows 57 / 62 / 66 / 74 us, 5.7 / 5.4 / 5.1 / 4.6
// TB/s (a large copy reaches 5.2); rows loaded again for each group 64 / 82 / 108 / 144.  Few columns: by latency, 3840 of
// 2560 4.1-5.7 us.
// ======================================================================
constexpr int kI8Waves = 8;

template <int RB, int CT, int U, bool ONCE>
__global__ __launch_bounds__(64 * kI8Waves, 2) void k_int8_stream(Int8Args p, int groups) {
  constexpr int kPart = 4 * 68;  // words of a block's sums: 16 rows of four columns, four times, and what keeps those in other banks
  __shared__ __attribute__((aligned(16))) int red[kI8Waves][RB][CT][kPart];
  const int tid = threadIdx.x, lane = tid & 63, wv = uni8(tid >> 6);
  const int rounds = ONCE ? 1 : ((p.KB + kI8Waves - 1) / kI8Waves + U - 1) / U;
  const int mine = (groups - (int)blockIdx.x + (int)gridDim.x - 1) / (int)gridDim.x;
  const int chunks = mine * rounds;

  // rows behind M: the last one's values, never written; k behind K: any values, the weights are zero there
  const auto ra = rsrc8(p.a, 0x7fffffff);
  uint32_t row_off[RB];
#pragma unroll
  for (int r = 0; r < RB; ++r) row_off[r] = (uint32_t)(min(16 * r + (lane & 15), p.M - 1) * p.lda);

  v4i b[2][U][CT], a[ONCE ? 1 : 2][U][RB];
  auto issue_rows = [&](int set, int k0) {
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int r = 0; r < RB; ++r)
        a[set][u][r] = buf128(ra, row_off[r] + min((k0 + kI8Waves * u) * 64 + 16 * (lane >> 4), p.K - 16));
  };
  auto issue = [&](int set, int c) {
    const int g = blockIdx.x + min(c / rounds, mine - 1) * gridDim.x, k0 = c % rounds * U * kI8Waves + wv;
#pragma unroll
    for (int t = 0; t < CT; ++t) {
      const int nt = min(g * CT + t, p.NT - 1);
      const auto rw = rsrc8(p.w + (int64_t)nt * p.KB * 1024, c < chunks ? p.KB * 1024 : 0);
#pragma unroll
      for (int u = 0; u < U; ++u) b[set][u][t] = buf128(rw, (k0 + kI8Waves * u) * 1024 + lane * 16);
    }
    if (!ONCE) issue_rows(set, k0);
  };
  v4i acc[RB][CT];
  auto clear = [&] {
#pragma unroll
    for (int r = 0; r < RB; ++r)
#pragma unroll
      for (int t = 0; t < CT; ++t) acc[r][t] = (v4i){0, 0, 0, 0};
  };
  auto consume = [&](int set) {
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int r = 0; r < RB; ++r)
#pragma unroll
        for (int t = 0; t < CT; ++t)
          acc[r][t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(b[set][u][t], a[ONCE ? 0 : set][u][r], acc[r][t], 0, 0, 0);
  };
  static_assert(RB * CT * 64 <= 64 * kI8Waves, "a thread has the same row in every group");
  uint64_t best = 0;
  auto finish = [&](int c) {  // the group of chunk c is complete
    const int g = blockIdx.x + c / rounds * gridDim.x;
#pragma unroll
    for (int r = 0; r < RB; ++r)
#pragma unroll
      for (int t = 0; t < CT; ++t) *reinterpret_cast<v4i*>(&red[wv][r][t][4 * lane + 4 * (lane >> 4)]) = acc[r][t];
    lds_barrier();
    // a thread's four columns of a row
    for (int e = tid; e < RB * CT * 64; e += 64 * kI8Waves) {  // (once)
      const int q = e % (4 * CT), m = e / (4 * CT), at = 4 * (16 * (q & 3) + (m & 15)) + 4 * (q & 3);
      v4i sum = (v4i){0, 0, 0, 0};
#pragma unroll
      for (int w = 0; w < kI8Waves; ++w) sum += *reinterpret_cast<const v4i*>(&red[w][m >> 4][q >> 2][at]);
      const int col = g * 16 * CT + 4 * q;
      if (m >= p.M) continue;
      const float sa = p.sa[m];
      float y[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] = scaled(sum[i], sa, p.sw[min(col + i, p.N - 1)]);
      if (p.tokens)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (col + i < p.N) best = arg_max(best, arg_key(y[i], col + i));
      if (!p.out) continue;
      if (p.f32) {
        float* const o = static_cast<float*>(p.out) + m * p.ldo + col;
        if (p.vec && col + 4 <= p.N)
          *reinterpret_cast<float4*>(o) = make_float4(y[0], y[1], y[2], y[3]);
        else
          for (int i = 0; i < 4; ++i)
            if (col + i < p.N) o[i] = y[i];
      } else {
        uint16_t* const o = static_cast<uint16_t*>(p.out) + m * p.ldo + col;
        if (p.vec && col + 4 <= p.N)
          *reinterpret_cast<uint2*>(o) = make_uint2(f2bf_pair(y[0], y[1]), f2bf_pair(y[2], y[3]));
        else
          for (int i = 0; i < 4; ++i)
            if (col + i < p.N) o[i] = f2bf(y[i]);
      }
    }
    lds_barrier();
    clear();
  };

  clear();
  issue(0, 0);
  if (ONCE) issue_rows(0, wv);
  issue(1, 1);
  for (int c = 0; c < chunks; c += 2) {
    consume(0);
    issue(0, c + 2);
    if (ONCE || (c + 1) % rounds == 0) finish(c);
    if (c + 1 >= chunks) break;
    consume(1);
    issue(1, c + 3);
    if (ONCE || (c + 2) % rounds == 0) finish(c + 1);
  }
  if (!p.tokens) return;

  // the best of a row: over the 4 CT threads that have its columns here, then over the workgroups; the last of
  // those to end writes the indexes
#pragma unroll
  for (int off = 1; off < 4 * CT; off <<= 1) best = arg_max(best, __shfl_xor(best, off, 64));
  const int row = tid / (4 * CT);
  if (tid < RB * CT * 64 && tid % (4 * CT) == 0 && row < p.M && best)
    __hip_atomic_fetch_max(p.keys + row, best, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  wait_memory();  // this workgroup's maxima are performed before it counts itself done
  int* const last = &red[0][0][0][0];
  lds_barrier();
  if (tid == 0) *last = atomicAdd(p.count, 1u) + 1u == gridDim.x;
  lds_barrier();
  if (!*last) return;
  if (tid < p.M) p.tokens[tid] = arg_col(ld_coherent(p.keys + tid));
}

// The best of part blockIdx.x of row blockIdx.y; a row of one part is done.  Parts of at least 2048 columns, about four workgroups a
// CU.  Bound by latency, a thread having few loads of 4 bytes on their way: 128256 columns, 128 rows 28 us (2.4 TB/s) and 5 of the
// join, 1024 rows 293 (1.8 TB/s), beside 74 and 356 of the product.
__global__ __launch_bounds__(256) void k_int8_argmax(const float* y, int64_t ldo, int N, int each, uint64_t* keys, int32_t* tokens) {
  __shared__ uint64_t s_best[4];
  const int row = blockIdx.y, end = min(N, ((int)blockIdx.x + 1) * each);
  const float* const at = y + (int64_t)row * ldo;
  uint64_t best = 0;
  for (int c = blockIdx.x * each + threadIdx.x; c < end; c += 256) best = arg_max(best, arg_key(at[c], c));
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) best = arg_max(best, __shfl_xor(best, off, 64));
  if ((threadIdx.x & 63) == 0) s_best[threadIdx.x >> 6] = best;
  __syncthreads();
  if (threadIdx.x != 0) return;
  best = arg_max(arg_max(s_best[0], s_best[1]), arg_max(s_best[2], s_best[3]));
  if (gridDim.x == 1)
    tokens[row] = arg_col(best);
  else
    keys[(int64_t)row * gridDim.x + blockIdx.x] = best;
}

__global__ __launch_bounds__(64) void k_int8_argmax_parts(const uint64_t* keys, int parts, int32_t* tokens) {
  uint64_t best = 0;
  for (int i = threadIdx.x; i < parts; i += 64) best = arg_max(best, keys[(int64_t)blockIdx.x * parts + i]);
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) best = arg_max(best, __shfl_xor(best, off, 64));
  if (threadIdx.x == 0) tokens[blockIdx.x] = arg_col(best);
}

// ======================================================================
// Many rows: tiles of BM x BN, S stages of KG x SUB x 64 k in LDS, filled without registers.  The waves are KG groups
// of WM x WN; a group takes its blocks of 64 k of every stage, and the groups' sums meet in LDS.
//
// Large tiles: the matrix units are busy 50% (K = 2560) to 59% (8192) of the cycles; what remains is a tile's first loads, its
// outputs, and the wait for operands that 256 x 256 x 128 k take in (64 KiB a step through each CU).  8192^3: 445-468 us, 2.35-2.47
// POP/s (a large library product 2.12); 4096 x 2560 x 13824: 142-151 us, 1.92-2.04.  Small tiles: bound by the operands that pass
// through each CU, at 37-50 B/ns a CU, and by latency, so that they have several stages on their way and the waves of a
// workgroup share a small tile's k (511 x 2560 x 3840: 10.7 us).  The next tile's first stage loaded before the outputs are
// stored, by workgroups of several tiles each: 1-3% slower (474 -> 482); weights two steps ahead, in a third stage: no gain.
// ======================================================================
// 16 rows of a wave's TN blocks through its own LDS, so that they leave in whole lines: a lane has four columns
// (4 (lane / 16) ..) of one row (lane % 16) of each block.
template <typename T>
__device__ __forceinline__ void put4(T* at, const float* y);
template <>
__device__ __forceinline__ void put4<float>(float* at, const float* y) {
  *reinterpret_cast<float4*>(at) = make_float4(y[0], y[1], y[2], y[3]);
}
template <>
__device__ __forceinline__ void put4<uint16_t>(uint16_t* at, const float* y) {
  *reinterpret_cast<uint2*>(at) = make_uint2(f2bf_pair(y[0], y[1]), f2bf_pair(y[2], y[3]));
}
template <int TN, typename T>
__device__ __forceinline__ void store_block(const Int8Args& p, const v4i (&acc)[TN], float sa, const float (&sw)[TN][4], T* mine,
                                            int row0, int col0) {
  constexpr int kCols = 16 * TN, kLd = kCols + 16 / (int)sizeof(T);  // elements of a row in LDS
  const int lane = threadIdx.x & 63;
  __builtin_amdgcn_wave_barrier();
#pragma unroll
  for (int j = 0; j < TN; ++j) {
    float y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = scaled(acc[j][e], sa, sw[j][e]);
    put4(mine + (lane & 15) * kLd + 16 * j + 4 * (lane >> 4), y);
  }
  __builtin_amdgcn_wave_barrier();
  T* const out = static_cast<T*>(p.out) + (int64_t)row0 * p.ldo + col0;
  const int rows = min(16, p.M - row0), cols = min(kCols, p.N - col0);
  if (p.vec && cols == kCols) {
    constexpr int kPiece = 16 / (int)sizeof(T), kPer = kCols / kPiece;  // pieces of a row
#pragma unroll
    for (int q = 0; q < 16 * kPer / 64; ++q) {
      const int piece = q * 64 + lane, r = piece / kPer, c = piece % kPer * kPiece;
      const uint4 v = *reinterpret_cast<const uint4*>(mine + r * kLd + c);
      if (r < rows) *reinterpret_cast<uint4*>(out + r * p.ldo + c) = v;
    }
  } else {
    for (int r = 0; r < rows; ++r)
      for (int c = lane; c < cols; c += 64) out[r * p.ldo + c] = mine[r * kLd + c];
  }
}

template <int BM, int BN, int WM, int WN, int KG, int SUB, int S>
struct TileShape {
  static constexpr int kWaves = WM * WN * KG, kB = BN / 16, kK = KG * SUB;  // kK: blocks of 64 k of a stage
  static constexpr int kRowKiB = kK * BM / 16, kStage = kRowKiB + kK * kB;  // KiB of a stage: the rows', all
  static constexpr int TM = BM / WM / 16, TN = BN / WN / 16;                // a wave's blocks
  static constexpr int kOutBytes = 16 * (TN * 16 + 4) * 4, kSums = KG > 1 ? BM * BN * 4 * (KG - 1) : 0;
  static constexpr int kBytes = std::max(S * kStage * 1024, std::max(kWaves * kOutBytes, kSums));
};

// The tile whose first row is m0 and first block of columns nt0.
template <int BM, int BN, int WM, int WN, int KG, int SUB, int S>
__device__ __forceinline__ void int8_tile(const Int8Args& p, uint8_t* smem, int m0, int nt0) {
  using Shape = TileShape<BM, BN, WM, WN, KG, SUB, S>;
  constexpr int kWaves = Shape::kWaves, kB = Shape::kB, kK = Shape::kK, kRowKiB = Shape::kRowKiB, kStage = Shape::kStage;
  constexpr int TM = Shape::TM, TN = Shape::TN, kOutBytes = Shape::kOutBytes;
  constexpr int kLoads = kStage / kWaves;
  static_assert(kK % 2 == 0 && kStage % kWaves == 0 && kRowKiB % kWaves == 0 && TM % KG == 0, "loads and sums of a wave");
  lds8* const sm = (lds8*)smem;
  const int tid = threadIdx.x, lane = tid & 63, wv = uni8(tid >> 6);
  const int steps = (p.KB + kK - 1) / kK;

  // Rows: 8 of them x 128 k a KiB, so that whole lines of memory are asked for; 16-byte pieces of a row are at piece ^ row % 8,
  // for the banks that 8 lanes read at once.  Columns: their blocks as they lie in memory.
  const auto ra = rsrc8(p.a + (int64_t)m0 * p.lda, 0x7fffffff);
  const auto rw = rsrc8(p.w + (int64_t)nt0 * p.KB * 1024, (uint32_t)min(kB, p.NT - nt0) * p.KB * 1024);
  constexpr int kLa = kRowKiB / kWaves;  // a wave's loads of rows, then those of columns
  uint32_t off[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int x = wv + kWaves * i;
    off[i] = i < kLa ? (uint32_t)(min(x % (BM / 8) * 8 + (lane >> 3), p.M - 1 - m0) * p.lda)
                     : (uint32_t)((x - kRowKiB) % kB) * p.KB * 1024 + lane * 16;
  }
  auto issue = [&](int step, lds8* at) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int x = wv + kWaves * i;
      lds8* const dst = at + x * 1024;
      if (i < kLa) {  // k behind K: any values of the row, the weights are zero there
        const int k = step * kK * 64 + x / (BM / 8) * 128 + 16 * ((lane & 7) ^ (lane >> 3));
        __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, dst, 16, (int)(off[i] + min(k, p.K - 16)), 0, 0, 0);
      } else {  // blocks behind the last read as zeros
        const int kb = step * kK + (x - kRowKiB) / kB;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rw, dst, 16, kb < p.KB ? (int)(off[i] + kb * 1024) : -1, 0, 0, 0);
      }
    }
  };
  const int kg = wv / (WM * WN), wm = wv % WM, wn = wv / WM % WN;
  constexpr int kRows = TM / KG;  // of a wave's row blocks, those that it finishes
  const int col0 = (nt0 + wn * TN) * 16, row0 = m0 + (wm * TM + kg * kRows) * 16;
  // (now: a load between the stores of the outputs would wait for those)
  float sa[kRows], sw[TN][4];
#pragma unroll
  for (int i = 0; i < kRows; ++i) sa[i] = p.sa[min(row0 + 16 * i + (lane & 15), p.M - 1)];
#pragma unroll
  for (int j = 0; j < TN; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) sw[j][e] = p.sw[min(col0 + 16 * j + 4 * (lane >> 4) + e, p.N - 1)];

  v4i acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = (v4i){0, 0, 0, 0};

#pragma unroll
  for (int s = 0; s < S - 1; ++s) issue(s, sm + s * kStage * 1024);
  int at = 0;
  for (int step = 0; step < steps; ++step) {
    constexpr int kLeft = (S - 2) * kLoads;  // loads that may still be on their way
    __builtin_amdgcn_s_waitcnt(0x0f70 | (kLeft & 15) | ((kLeft >> 4) << 14));
    lds_barrier();
    issue(step + S - 1, sm + (at == 0 ? S - 1 : at - 1) * kStage * 1024);
#pragma unroll
    for (int u = 0; u < SUB; ++u) {
      const int kb = kg * SUB + u;
      const lds8* const as = sm + at * kStage * 1024 + kb / 2 * BM * 128 + (wm * TM * 16 + (lane & 15)) * 128 +
                             16 * ((4 * (kb & 1) + (lane >> 4)) ^ (lane & 7));
      const lds8* const bs = sm + (at * kStage + kRowKiB + kb * kB + wn * TN) * 1024 + lane * 16;
      v4i x[TM], y[TN];
#pragma unroll
      for (int j = 0; j < TN; ++j) y[j] = *(const __attribute__((address_space(3))) v4i*)(bs + j * 1024);
#pragma unroll
      for (int i = 0; i < TM; ++i) x[i] = *(const __attribute__((address_space(3))) v4i*)(as + i * 2048);
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(y[j], x[i], acc[i][j], 0, 0, 0);
    }
    at = at + 1 == S ? 0 : at + 1;
  }
  __builtin_amdgcn_s_waitcnt(0x0f70);  // nothing may land in LDS any more
  lds_barrier();                       // every wave is done with the stages: their place takes sums and outputs

  if (KG > 1) {
    v4i* const sums = reinterpret_cast<v4i*>(smem);
    // place of (owner, which of the others, row block, column block) of this wave's part of the tile
    auto place = [&](int owner, int other, int i, int j) {
      return ((((owner * (KG - 1) + other) * kRows + i) * TN + j) * (WM * WN) + wv % (WM * WN)) * 64 + lane;
    };
#pragma unroll
    for (int o = 0; o < KG; ++o)
      if (o != kg)
#pragma unroll
        for (int i = 0; i < kRows; ++i)
#pragma unroll
          for (int j = 0; j < TN; ++j) sums[place(o, kg - (kg > o), i, j)] = acc[o * kRows + i][j];
    lds_barrier();
#pragma unroll
    for (int o = 0; o < KG; ++o)
      if (o == kg)
#pragma unroll
        for (int i = 0; i < kRows; ++i)
#pragma unroll
          for (int j = 0; j < TN; ++j) {
            v4i v = acc[o * kRows + i][j];
#pragma unroll
            for (int x = 0; x < KG - 1; ++x) v += sums[place(o, x, i, j)];
            acc[i][j] = v;
          }
    lds_barrier();
  }
  uint8_t* const mine = smem + wv * kOutBytes;
  if (col0 >= p.N) return;
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    if (row0 + 16 * i >= p.M) break;
    if (p.f32)
      store_block<TN, float>(p, acc[i], sa[i], sw, reinterpret_cast<float*>(mine), row0 + 16 * i, col0);
    else
      store_block<TN, uint16_t>(p, acc[i], sa[i], sw, reinterpret_cast<uint16_t*>(mine), row0 + 16 * i, col0);
  }
}

// Tiles in strips of `strip` rows of them, column by column; a workgroup's XCD is its number's remainder by 8, and takes a part of
// that order, so that what it works on at a time is nearly square, and its L2 reads few rows and columns.  Numbers as they come,
// down the rows / strips of 2 / 4 / 8 / 16: 4096 x 2560 x 13824 150, 152, 142, 143, 146 us; 1024 x 2560 x 6912 27.0, 24.0, 23.4, 24.6, 24.6;
// 300 x 2560 x 128256 (fp32) 183, 182, 165, 160, 164; 511 x 2560 x 3840 11.1, 10.8, 10.7, 10.8, 10.8; 128 x 6912 x 2560, two rows of
// tiles, 12.7, 13.2, 13.1, 13.1, 13.1.
constexpr int kXcds8 = 8;
struct TileAt {
  int m, n;
};
__device__ __forceinline__ TileAt tile_at(int t, int ngm, int ngn, int strip) {
  const int s = t / (strip * ngn), in = t - s * strip * ngn, h = min(strip, ngm - s * strip);
  return {uni8(s * strip + in % h), uni8(in / h)};
}
// Workgroup x's place of `tiles`; -1: none.
__device__ __forceinline__ int xcd_place(int x, int tiles) {
  const int each = (tiles + kXcds8 - 1) / kXcds8, t = x % kXcds8 * each + x / kXcds8;
  return x / kXcds8 < each && t < tiles ? t : -1;
}
inline int xcd_groups(int tiles) { return (tiles + kXcds8 - 1) / kXcds8 * kXcds8; }

template <int BM, int BN, int WM, int WN, int KG, int SUB, int S, int PER_CU>
__global__ __launch_bounds__(64 * WM * WN * KG, PER_CU) void k_int8_tile(Int8Args p, int ngm, int ngn, int strip) {
  __shared__ __attribute__((aligned(16))) uint8_t smem[TileShape<BM, BN, WM, WN, KG, SUB, S>::kBytes];
  const int t = xcd_place(blockIdx.x, ngm * ngn);
  if (t < 0) return;
  const TileAt at = tile_at(t, ngm, ngn, strip);
  int8_tile<BM, BN, WM, WN, KG, SUB, S>(p, smem, at.m * BM, at.n * (BN / 16));
}

// Tiles of 256 x 256, the last ones (from `full` on) as two of 128 rows each: they fill the CUs once more where
// whole tiles would fill half of them for twice as long.
__global__ __launch_bounds__(512, 1) void k_int8_large(Int8Args p, int ngm, int ngn, int full, int strip) {
  constexpr int kBytes = std::max(TileShape<256, 256, 2, 4, 1, 2, 2>::kBytes, TileShape<128, 256, 2, 4, 1, 2, 3>::kBytes);
  __shared__ __attribute__((aligned(16))) uint8_t smem[kBytes];
  const int whole = (full + kXcds8 - 1) / kXcds8 * kXcds8, x = (int)blockIdx.x - whole;
  if (x < 0) {
    const int t = xcd_place(blockIdx.x, full);
    if (t < 0) return;
    const TileAt at = tile_at(t, ngm, ngn, strip);
    int8_tile<256, 256, 2, 4, 1, 2, 2>(p, smem, at.m * 256, at.n * 16);
  } else {
    const TileAt at = tile_at(full + x / 2, ngm, ngn, strip);
    const int m0 = at.m * 256 + (x & 1) * 128;
    if (m0 < p.M) int8_tile<128, 256, 2, 4, 1, 2, 3>(p, smem, m0, at.n * 16);
  }
}

// ---- weights (once, when they are loaded) ---------------------------------------------------------------
__global__ void k_int8_layout(const int8_t* w, int64_t ldw, int N, int K, int KB, int64_t total, uint4* out) {
  const int64_t g = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (g >= total) return;
  const int lane = (int)(g & 63);
  const int64_t blk = g >> 6;
  const int64_t n = blk / KB * 16 + (lane & 15);
  const int k = (int)(blk % KB) * 64 + 16 * (lane >> 4);
  uint4 v = make_uint4(0u, 0u, 0u, 0u);
  if (n < N && k < K) v = *reinterpret_cast<const uint4*>(w + n * ldw + k);
  out[g] = v;
}

// Channel n of float weights: scale = max|w| / 127 (1 where that is 0), codes round(w / scale) to even, on a wave.  The
// quotient is the correctly rounded one, so a code is off by half a step and 127 is reached, never passed.
template <typename T>
__device__ __forceinline__ float weight_at(const T* w, int64_t i);
template <>
__device__ __forceinline__ float weight_at<float>(const float* w, int64_t i) { return w[i]; }
template <>
__device__ __forceinline__ float weight_at<uint16_t>(const uint16_t* w, int64_t i) { return bf2f(w[i]); }

template <typename T>
__global__ __launch_bounds__(256) void k_int8_quantise(const T* w, int64_t ldw, int N, int K, int KB, uint8_t* out, float* scale) {
  const int lane = threadIdx.x & 63;
  const int64_t n = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);  // up to the end of the last block
  if (n >= (int64_t)(N + 15) / 16 * 16) return;
  const T* const row = w + n * ldw;
  float m = 0.0f;
  bool bad = false;
  if (n < N)
    for (int k = lane; k < K; k += 64) {
      const float x = weight_at(row, k);
      bad |= !__builtin_isfinite(x);
      m = fmaxf(m, fabsf(x));
    }
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) m = fmaxf(m, __shfl_xor(m, off, 64));
  bad = __any(bad);
  // a tiny row's m / 127 could be a subnormal of few bits, and w / scale pass 127: below it the codes are zero
  const bool none = m < 0x1p-119f;
  const float s = none ? 1.0f : m / 127.0f;
  if (n < N && lane == 0) scale[n] = bad ? __builtin_nanf("") : s;
  uint8_t* const col = out + n / 16 * KB * 1024 + (n & 15) * 16;
  for (int k = lane; k < KB * 64; k += 64) {
    int q = 0;
    if (n < N && k < K && !bad && !none) q = min(127, max(-127, (int)__builtin_rintf(weight_at(row, k) / s)));
    col[(int64_t)(k >> 6) * 1024 + ((k & 63) >> 4) * 256 + (k & 15)] = (uint8_t)(int8_t)q;
  }
}

// ---- host ------------------------------------------------------------------
// btl_act.hip
int launch_act(const uint16_t* x, int64_t M, int64_t K, int64_t ldx, const uint16_t* gamma, float norm_eps,
               int8_t* xa, float* a_dq, int32_t* rowsum, float* act_scale, int8_t* xq_rm, uint16_t* y_rm,
               uint32_t* zero_words, int n_zero_words, hipStream_t stream);
int check_act_args(const char* who, const uint16_t* x, int64_t M, int64_t K, int64_t ldx, const uint16_t* gamma);

inline int check_int8_shape(const char* who, int64_t N, int64_t K) {
  if (N <= 0 || N > (1 << 24)) return set_error(BTL_ERR_SHAPE, "%s: N=%lld", who, (long long)N);
  if (K <= 0 || K % 16 || K > BTL_MAX_K)
    return set_error(BTL_ERR_SHAPE, "%s: K=%lld (a multiple of 16 up to %d)", who, (long long)K, BTL_MAX_K);
  return BTL_OK;
}
inline int64_t int8_kb(int64_t K) { return (K + 63) / 64; }
inline int64_t int8_nt(int64_t N) { return (N + 15) / 16; }

template <int RB, int CT>
static void launch_stream(const Int8Args& a, int groups, dim3 grid, hipStream_t s) {
  const int each = (a.KB + kI8Waves - 1) / kI8Waves;
  if (each <= 2)
    hipLaunchKernelGGL((k_int8_stream<RB, CT, 2, true>), grid, dim3(64 * kI8Waves), 0, s, a, groups);
  else if (each <= 5)
    hipLaunchKernelGGL((k_int8_stream<RB, CT, 5, true>), grid, dim3(64 * kI8Waves), 0, s, a, groups);
  else
    hipLaunchKernelGGL((k_int8_stream<RB, CT, RB == 4 ? 2 : 4, false>), grid, dim3(64 * kI8Waves), 0, s, a, groups);
}

constexpr int kStrip = 4;  // rows of tiles

template <int BM, int BN, int WM, int WN, int KG, int SUB, int S, int PER_CU>
static void launch_tile(const Int8Args& a, hipStream_t s) {
  const int ngm = (a.M + BM - 1) / BM, ngn = (a.NT * 16 + BN - 1) / BN;
  hipLaunchKernelGGL((k_int8_tile<BM, BN, WM, WN, KG, SUB, S, PER_CU>), dim3((unsigned)xcd_groups(ngm * ngn)),
                     dim3(64 * WM * WN * KG), 0, s, a, ngm, ngn, kStrip);
}

// Of `tiles` large ones, how many go as halves: a last round that fills at most half of the CUs.  4096 x 2560 x 13824 (864 tiles)
// 155 us, 146 so; 8192 x 2560 x 2560 (320) 84, 64.
static int64_t large_halves(int64_t tiles, int64_t cus) { return tiles > cus && 2 * (tiles % cus) <= cus ? tiles % cus : 0; }

static void launch_large(const Int8Args& a, int halves, hipStream_t s) {
  const int ngm = (a.M + 255) / 256, ngn = (a.NT + 15) / 16, tiles = ngm * ngn;
  hipLaunchKernelGGL(k_int8_large, dim3((unsigned)(xcd_groups(tiles - halves) + 2 * halves)), dim3(512), 0, s, a, ngm, ngn,
                     tiles - halves, kStrip);
}

// The tile of the least time, us: rounds of workgroups over the CUs x what a workgroup takes, for a start (and an end) and for
// each 128 k; alone on its CU, or beside another one.  Fitted to 69 shapes, 65-8192 rows, K 576-6912, 640-128256
// columns, with tiles in plain rows; in strips, as they are now, the rule takes the best of the five for 68 of them and 4% more for the
// other, and for 46 others drawn at random (65-6000 rows, K 320-6912, 300-40000 columns) the best for 44, 5% and 0.2% more for two.  Us of
// each, in this order: 4096 x 2560 x 13824: 148, 175, 232, 312, 270; 1024 x 2560 x 6912: 36, 26, 29, 36, 36; 256 x 2560 x
// 13824: 36, 24, 19, 26, 26; 511 x 2560 x 3840: 34, 21, 14, 10.8, 12.3; 128 x 6912 x 2560: 78, 46, 28, 19, 13; 400 x 640 x 2560: 13,
// 9, 7.0, 5.9, 6.0.  (128 x 128 as two a CU is never more than 2% better, 64 x 64 as one of 8 stages never better.)
struct TileCost {
  int bm, bn, per_cu;
  double start, step;          // one on a CU
  double start_two, step_two;  // per_cu 2
};
constexpr TileCost kTiles[] = {
    {256, 256, 1, 8.0, 1.60, 0, 0}, {128, 256, 1, 5.5, 0.95, 0, 0},    {128, 128, 1, 4.2, 0.56, 0, 0},
    {128, 64, 1, 3.0, 0.35, 0, 0},  {64, 64, 2, 2.8, 0.20, 3.5, 0.45},
};
static int tile_choice(int64_t M, int64_t N, int64_t K, int cus) {
  const double steps = (double)((K + 127) / 128);
  int best = 0;
  double least = 0;
  for (int i = 0; i < (int)(sizeof(kTiles) / sizeof(kTiles[0])); ++i) {
    const TileCost& t = kTiles[i];
    const int64_t tiles = (M + t.bm - 1) / t.bm * ((N + t.bn - 1) / t.bn), slots = (int64_t)cus * t.per_cu;
    const bool two = t.per_cu == 2 && tiles > cus;
    double rounds = (double)((tiles + slots - 1) / slots);
    if (i == 0 && large_halves(tiles, cus)) rounds -= 0.5;
    const double us = rounds * (two ? t.start_two + t.step_two * steps : t.start + t.step * steps);
    if (i == 0 || us < least) best = i, least = us;
  }
  return best;
}

constexpr int kFewRows8 = 64;     // that the weight stream can take
constexpr int kHeadRows = 65535;  // a grid's second dimension
constexpr int kHeadWords = kFewRows8 * 2 + 1;  // few rows: keys and count, which the quantisation clears

// A head call's scratch: byte offsets (few rows: the cleared words first), parts of a row for its argmax.
struct HeadScratch {
  int64_t codes, blocked, scale, keys, total, parts;
};
static HeadScratch head_scratch(int64_t M, int64_t K, int64_t N) {
  HeadScratch h;
  h.codes = 1024;
  h.blocked = round_up(h.codes + M * K, 256);
  h.scale = round_up(h.blocked + btl_act_bytes(M, K), 256);
  h.keys = round_up(h.scale + round_up(M, 32) * 4, 256);
  // about four workgroups a CU
  h.parts = std::max((int64_t)1, std::min((4 * (int64_t)device_cus() + M - 1) / M, (N + 2047) / 2048));
  h.total = h.keys + (h.parts > 1 ? M * h.parts * 8 : 0);
  return h;
}

// Checks that the entry points share; fills what they share.
static int int8_args(const char* who, const int8_t* a, int64_t lda, const float* a_scale, int64_t M, int64_t K, int64_t N,
                     const uint8_t* wdev, const float* w_scale, void* out, int64_t ldo, int out_f32, Int8Args* p) {
  const int rc = check_int8_shape(who, N, K);
  if (rc != BTL_OK) return rc;
  if (M < 0 || M > (1 << 24)) return set_error(BTL_ERR_SHAPE, "%s: M=%lld", who, (long long)M);
  if (lda < K || lda > (1 << 22) || (out && ldo < N))
    return set_error(BTL_ERR_SHAPE, "%s: lda=%lld ldo=%lld", who, (long long)lda, (long long)ldo);
  if (M == 0) return BTL_OK;
  if (!a || !a_scale || !wdev || !w_scale) return set_error(BTL_ERR_NULL, "%s: NULL pointer", who);
  if (!aligned(a, 16) || lda % 16 || !aligned(wdev, 16) || !aligned(a_scale, 4) || !aligned(w_scale, 4) ||
      !aligned(out, out_f32 ? 4 : 2))
    return set_error(BTL_ERR_ALIGN, "%s: misaligned buffer or row stride", who);
  if ((M + 63) / 64 * ((N + 63) / 64) > INT32_MAX)
    return set_error(BTL_ERR_SHAPE, "%s: M=%lld N=%lld", who, (long long)M, (long long)N);
  *p = Int8Args{a, lda, a_scale, wdev, w_scale, (int)M, (int)K, (int)N, (int)int8_kb(K), (int)int8_nt(N), out, ldo, out_f32 != 0,
                aligned(out, 16) && ldo % (out_f32 ? 4 : 8) == 0, nullptr, nullptr, nullptr};
  return BTL_OK;
}

// Whether the weight stream takes it; where a few rows' argmax is wanted without logits in any case, as tiles need them (whole head
// calls, K = 6912, 40000 columns, 17 / 32 / 48 / 64 rows: 58 / 71 / 84 / 98 us so, with logits, in tiles from 17 rows on, 58 / 60 / 64 /
// 69; 4096 x 128256, 17 / 32 / 64: 107 / 126 / 189, 108 / 112 / 128; 6912 x 3840: 19 / 24 / 29, 24 / 24 / 25).  Us of the stream / of tiles,
// K = 2560, 16 rows: 640 columns 3.9 / 6.4, 3840: 4.7 / 7.1, 13824: 10.2 / 10.6, 128256: 66 / 71; 32 rows: 5.0 / 6.7, 5.8 / 7.1,
// 11.9 / 11.1, 70 / 74; 64 rows: 7.3 / 6.9, 8.5 / 7.3, 14.7 / 11.7, 76 / 78.  K = 6912, where rows are loaded again for each group
// of columns, 16 rows: 640: 8.9 / 12.9, 3840: 9.5 / 13.2, 13824: 34 / 21, 40000: 64 / 59; 32 rows: 14.1 / 12.8, 14.6 / 13.2, 48 / 22,
// 80 / 59.
static bool streams_once(int64_t K) { return int8_kb(K) <= 5 * kI8Waves; }
static bool few_rows(int64_t M, int64_t N, int64_t K, bool tokens, int cus) {
  if (tokens) return true;
  return streams_once(K) ? M <= 32 : M <= 16 && int8_nt(N) <= cus;
}

// How a product is done: the weight stream in groups of `ct` column blocks (0: not so), or a tile of kTiles, of which `halves`
// large ones go as two.
struct Int8Plan {
  int ct, tile, halves;
};
static Int8Plan int8_plan(int64_t M, int64_t N, int64_t K, bool tokens) {
  const int cus = device_cus();
  // pairs of column blocks share the rows' registers and the sums' barriers: 128256 columns of 2560, 1 / 16 / 64 rows, alone 59 /
  // 66 / 79 us, in pairs 57 / 62 / 74; 27648 columns 16.3 / 17.2 / 22.9, 16.9 / 17.5 / 23.8, as the last round is less even
  if (few_rows(M, N, K, tokens, cus)) return {int8_nt(N) > 8 * cus ? 2 : 1, 0, 0};
  const int tile = tile_choice(M, N, K, cus);
  return {0, tile, tile ? 0 : (int)large_halves((M + 255) / 256 * ((N + 255) / 256), cus)};
}

static int int8_launch(const char* who, const Int8Args& p, hipStream_t s) {
  const Int8Plan plan = int8_plan(p.M, p.N, p.K, p.tokens != nullptr);
  if (plan.ct) {
    const int ct = plan.ct, groups = (p.NT + ct - 1) / ct;
    const dim3 grid((unsigned)std::min(groups, device_cus()));
    if (p.M <= 16)
      ct == 1 ? launch_stream<1, 1>(p, groups, grid, s) : launch_stream<1, 2>(p, groups, grid, s);
    else if (p.M <= 32)
      ct == 1 ? launch_stream<2, 1>(p, groups, grid, s) : launch_stream<2, 2>(p, groups, grid, s);
    else
      ct == 1 ? launch_stream<4, 1>(p, groups, grid, s) : launch_stream<4, 2>(p, groups, grid, s);
    return check_launch(who);
  }
  switch (plan.tile) {
    case 0: launch_large(p, plan.halves, s); break;
    case 1: launch_tile<128, 256, 2, 4, 1, 2, 3, 1>(p, s); break;
    case 2: launch_tile<128, 128, 2, 2, 2, 1, 4, 1>(p, s); break;
    case 3: launch_tile<128, 64, 2, 2, 2, 1, 6, 1>(p, s); break;
    default: launch_tile<64, 64, 2, 2, 2, 1, 4, 2>(p, s); break;
  }
  return check_launch(who);
}

}  // namespace btl

using namespace btl;

extern "C" {

int64_t btl_int8_weight_bytes(int64_t N, int64_t K) {
  if (N <= 0 || N > (1 << 24) || K <= 0 || K % 16 || K > BTL_MAX_K) return 0;
  return int8_nt(N) * int8_kb(K) * 1024;
}

int btl_int8_weight_layout(const int8_t* w, int64_t ldw, int64_t N, int64_t K, uint8_t* wdev, btl_stream_t stream) {
  const char* who = "btl_int8_weight_layout";
  clear_error();
  const int rc = check_int8_shape(who, N, K);
  if (rc != BTL_OK) return rc;
  if (!w || !wdev) return set_error(BTL_ERR_NULL, "%s: NULL pointer", who);
  if (ldw < K) return set_error(BTL_ERR_SHAPE, "%s: row stride smaller than a row", who);
  if (!aligned(w, 16) || !aligned(wdev, 16) || ldw % 16) return set_error(BTL_ERR_ALIGN, "%s: 16-byte alignment", who);
  const int64_t total = int8_nt(N) * int8_kb(K) * 64;
  hipLaunchKernelGGL(k_int8_layout, dim3((unsigned)((total + 255) / 256)), dim3(256), 0, (hipStream_t)stream, w, ldw, (int)N,
                     (int)K, (int)int8_kb(K), total, reinterpret_cast<uint4*>(wdev));
  return check_launch(who);
}

int btl_int8_weight_quantise(const void* w, int bf16, int64_t ldw, int64_t N, int64_t K, uint8_t* wdev, float* scale,
                             btl_stream_t stream) {
  const char* who = "btl_int8_weight_quantise";
  clear_error();
  const int rc = check_int8_shape(who, N, K);
  if (rc != BTL_OK) return rc;
  if (!w || !wdev || !scale) return set_error(BTL_ERR_NULL, "%s: NULL pointer", who);
  if (ldw < K) return set_error(BTL_ERR_SHAPE, "%s: row stride smaller than a row", who);
  if (!aligned(w, bf16 ? 2 : 4) || !aligned(wdev, 16) || !aligned(scale, 4))
    return set_error(BTL_ERR_ALIGN, "%s: misaligned buffer", who);
  const dim3 grid((unsigned)(int8_nt(N) * 4));
  if (bf16)
    hipLaunchKernelGGL(k_int8_quantise<uint16_t>, grid, dim3(256), 0, (hipStream_t)stream, static_cast<const uint16_t*>(w), ldw,
                       (int)N, (int)K, (int)int8_kb(K), wdev, scale);
  else
    hipLaunchKernelGGL(k_int8_quantise<float>, grid, dim3(256), 0, (hipStream_t)stream, static_cast<const float*>(w), ldw,
                       (int)N, (int)K, (int)int8_kb(K), wdev, scale);
  return check_launch(who);
}

int btl_int8_matmul(const int8_t* a, int64_t lda, const float* a_scale, int64_t M, int64_t K, int64_t N, const uint8_t* wdev,
                    const float* w_scale, void* out, int64_t ldo, int out_f32, btl_stream_t stream) {
  const char* who = "btl_int8_matmul";
  clear_error();
  Int8Args p{};
  const int rc = int8_args(who, a, lda, a_scale, M, K, N, wdev, w_scale, out, ldo, out_f32, &p);
  if (rc != BTL_OK || M == 0) return rc;
  if (!out) return set_error(BTL_ERR_NULL, "%s: NULL pointer", who);
  return int8_launch(who, p, (hipStream_t)stream);
}

int btl_int8_matmul_plan(int64_t M, int64_t K, int64_t N, int64_t* plan) {
  if (!plan || M <= 0 || M > (1 << 24) || N <= 0 || N > (1 << 24) || K <= 0 || K % 16 || K > BTL_MAX_K ||
      (M + 63) / 64 * ((N + 63) / 64) > INT32_MAX)
    return 0;
  const Int8Plan f = int8_plan(M, N, K, false);
  plan[0] = f.ct;
  plan[1] = f.ct ? 0 : kTiles[f.tile].bm;
  plan[2] = f.ct ? 0 : kTiles[f.tile].bn;
  plan[3] = f.halves;
  return 1;
}

int64_t btl_int8_head_scratch_bytes(int64_t M, int64_t K, int64_t N) {
  if (M <= 0 || M > kHeadRows || K <= 0 || K % 32 || K > BTL_MAX_K || N <= 0 || N > (1 << 24)) return 0;
  return head_scratch(M, K, N).total;
}

int btl_int8_head(const uint16_t* x, int64_t M, int64_t K, int64_t N, const uint16_t* gamma, float norm_eps, const uint8_t* wdev,
                  const float* w_scale, uint16_t* normed, float* logits, int32_t* tokens, void* scratch, size_t scratch_bytes,
                  btl_stream_t stream) {
  const char* who = "btl_int8_head";
  clear_error();
  if (M < 0 || M > kHeadRows) return set_error(BTL_ERR_SHAPE, "%s: M=%lld (up to %d)", who, (long long)M, kHeadRows);
  int rc = check_int8_shape(who, N, K);
  if (rc != BTL_OK || M == 0) return rc;
  rc = check_act_args(who, x, M, K, K, gamma);
  if (rc != BTL_OK) return rc;
  if (!gamma || !wdev || !w_scale || !tokens || !scratch || (!logits && M > kFewRows8))
    return set_error(BTL_ERR_NULL, "%s: NULL pointer", who);
  if (!aligned(tokens, 4) || !aligned(normed, 16) || !aligned(scratch, 256))
    return set_error(BTL_ERR_ALIGN, "%s: misaligned buffer", who);
  const HeadScratch h = head_scratch(M, K, N);
  if ((int64_t)scratch_bytes < h.total)
    return set_error(BTL_ERR_WORKSPACE, "%s: scratch %zu < %lld bytes", who, scratch_bytes, (long long)h.total);
  char* const at = static_cast<char*>(scratch);
  int8_t* const codes = reinterpret_cast<int8_t*>(at + h.codes);
  float* const a_scale = reinterpret_cast<float*>(at + h.scale);
  Int8Args p{};
  rc = int8_args(who, codes, K, a_scale, M, K, N, wdev, w_scale, logits, N, 1, &p);
  if (rc != BTL_OK) return rc;
  // (with logits: where rows are loaded again for each group of columns, tiles and the argmax behind them are faster)
  const bool few = M <= kFewRows8 && (!logits || M <= 16 || streams_once(K));
  hipStream_t s = (hipStream_t)stream;
  rc = launch_act(x, M, K, K, gamma, norm_eps, reinterpret_cast<int8_t*>(at + h.blocked), a_scale, nullptr, nullptr, codes, normed,
                  reinterpret_cast<uint32_t*>(at), few ? kHeadWords : 0, s);
  if (rc != BTL_OK) return rc;
  if (few) {
    p.tokens = tokens;
    p.keys = reinterpret_cast<uint64_t*>(at);
    p.count = reinterpret_cast<uint32_t*>(at + kFewRows8 * 8);
    return int8_launch(who, p, s);
  }
  rc = int8_launch(who, p, s);
  if (rc != BTL_OK) return rc;
  uint64_t* const keys = reinterpret_cast<uint64_t*>(at + h.keys);
  const int each = (int)((N + h.parts - 1) / h.parts), parts = (int)((N + each - 1) / each);
  hipLaunchKernelGGL(k_int8_argmax, dim3((unsigned)parts, (unsigned)M), dim3(256), 0, s, logits, N, (int)N, each, keys, tokens);
  if (parts > 1) {
    rc = check_launch(who);
    if (rc != BTL_OK) return rc;
    hipLaunchKernelGGL(k_int8_argmax_parts, dim3((unsigned)M), dim3(64), 0, s, keys, parts, tokens);
  }
  return check_launch(who);
}

}  // extern "C"
