// The plan of an attention call (which kernel, how contexts are split) and the checks that the entry
// points share: host only.
#pragma once

#include "btl_flash_body.h"

namespace btl {

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
// Us, of the tiles' rule: all steps of the longest workgroup, the partials of a split.
inline double split_whole(int64_t positions) { return 0.0117 * (double)positions; }
inline double split_part(int64_t T, int64_t H, int64_t D) { return 1.67e-6 * (double)(T * H * D); }
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
    const double whole = split_whole(max_kv), part = split_part(T, H, D);
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

// Checks that the entry points share; fills what they share.
inline int flash_args(const char* who, const uint16_t* q, int64_t ldq, int64_t T, int64_t H, int64_t Hkv, int64_t D,
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

// Of btl_flash.hip: the merge of a call's partials (shared: of both parts), a planned causal prompt.
int launch_merge(const char* what, const FlashArgs& a, int64_t T, int64_t H, int64_t D, bool shared, int parts,
                 hipStream_t stream);
int launch_causal_prompt(const FlashArgs& a, int64_t tiles, int64_t D, hipStream_t stream);

// Checks of a prompt's attention: everything but its launch.  T == 0 leaves *a without keys.
inline int prompt_args(const char* who, const uint16_t* q, int64_t ldq, const uint16_t* k, int64_t ldk, const uint16_t* v,
                       int64_t ldv, int64_t T, int64_t H, int64_t Hkv, int64_t D, const int32_t* cu_q, int64_t B, float scale,
                       int64_t max_q, uint16_t* out, int64_t ldo, int32_t* error_word, FlashArgs* a) {
  int rc = check_batch(who, B, T, cu_q, nullptr, nullptr, 0, &a->bt);
  if (rc != BTL_OK) return rc;
  rc = flash_args(who, q, ldq, T, H, Hkv, D, scale, out, ldo, error_word, a);
  if (rc != BTL_OK) return rc;
  if (max_q < 0) return set_error(BTL_ERR_SHAPE, "%s: max_q=%lld", who, (long long)max_q);
  if (T == 0) return BTL_OK;
  if (!k || !v) return set_error(BTL_ERR_NULL, "%s: NULL pointer", who);
  if (ldk < Hkv * D || ldv < Hkv * D) return set_error(BTL_ERR_SHAPE, "%s: row stride smaller than a row", who);
  if (ldk > (1 << 24) || ldv > (1 << 24))  // a step's rows within a 32-bit range
    return set_error(BTL_ERR_SHAPE, "%s: row stride over %d elements", who, 1 << 24);
  if (!aligned(k, 16) || !aligned(v, 16) || ldk % 8 || ldv % 8)
    return set_error(BTL_ERR_ALIGN, "%s: misaligned buffer or row stride", who);
  a->k = k;
  a->v = v;
  a->ldk = ldk;
  a->ldv = ldv;
  a->splits = 1;
  return BTL_OK;
}

// The same over pages.
inline int paged_args(const char* who, const uint16_t* q, int64_t ldq, int64_t T, int64_t H, const btl_pages_t* pages,
                      const int32_t* page_table, int64_t max_pages, const int32_t* cu_q, const int32_t* kv_len, int64_t B,
                      float scale, int64_t max_q, int64_t max_kv, uint16_t* out, int64_t ldo, int32_t* error_word,
                      FlashArgs* a) {
  int rc = check_pages(who, pages, &a->pg);
  if (rc != BTL_OK) return rc;
  rc = check_batch(who, B, T, cu_q, kv_len, page_table, max_pages, &a->bt);
  if (rc != BTL_OK) return rc;
  rc = flash_args(who, q, ldq, T, H, pages->num_kv_heads, pages->head_dim, scale, out, ldo, error_word, a);
  if (rc != BTL_OK) return rc;
  if (max_q <= 0 || max_kv <= 0 || max_pages <= 0 || max_pages * pages->page_size > kMaxPositions)
    return set_error(BTL_ERR_SHAPE, "%s: max_q=%lld max_kv=%lld max_pages=%lld", who, (long long)max_q,
                     (long long)max_kv, (long long)max_pages);
  if (T > 0 && (!page_table || !kv_len)) return set_error(BTL_ERR_NULL, "%s: NULL pointer", who);
  return BTL_OK;
}

// The call's partials in its scratch.
inline int partials(const char* who, void* scratch, size_t bytes, int64_t need, int64_t rows, FlashArgs* a) {
  if (need > 0) {
    if (!scratch || (int64_t)bytes < need)
      return set_error(BTL_ERR_WORKSPACE, "%s: scratch %zu < %lld bytes", who, scratch ? bytes : 0, (long long)need);
    if (!aligned(scratch, 16)) return set_error(BTL_ERR_ALIGN, "%s: misaligned scratch", who);
  }
  a->part_o = static_cast<float*>(scratch);
  a->part_ml = reinterpret_cast<float2*>(a->part_o + rows);
  return BTL_OK;
}

template <int MODE>
inline int launch_prompt(const char* what, FlashArgs a, int64_t tiles, int64_t D, hipStream_t stream) {
  a.neighbours = window_neighbours(tiles, 1);
  const dim3 grid((unsigned)(MODE == kWindow ? window_groups(tiles, a.Hkv, a.neighbours) : tiles));
  if (D == 128)
    hipLaunchKernelGGL((k_flash_tile<128, kDense, MODE>), grid, dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL((k_flash_tile<64, kDense, MODE>), grid, dim3(256), 0, stream, a);
  return check_launch(what);
}

// Windows over 8-bit pages: whether the kernel of few rows has 8 waves.
inline bool few_wide(const FlashPlan& f) { return f.tiles * f.splits <= device_cus(); }

// A planned call over pages, the merge included.
template <int MODE>
inline int launch_paged(const char* who, const char* what, const FlashPlan& f, FlashArgs* a, int64_t T, int64_t H, int64_t D,
                        bool fp8, void* scratch, size_t scratch_bytes, hipStream_t stream) {
  const int64_t B = a->bt.B;
  if (f.few && B > 65535) return set_error(BTL_ERR_SHAPE, "%s: %lld sequences", who, (long long)B);
  const int rc = partials(who, scratch, scratch_bytes, flash_scratch(f, T, H, D), f.splits > 1 ? (int64_t)f.splits * T * H * D : 0, a);
  if (rc != BTL_OK) return rc;
  a->splits = f.splits;
  a->chunk = f.chunk;
  if (f.few) {
    const dim3 grid((unsigned)a->Hkv, (unsigned)B, (unsigned)f.splits);
    auto* kern = D == 128 ? (fp8 ? k_flash_few<128, kPagedFp8, MODE> : k_flash_few<128, kPagedBf16, MODE>)
                          : (fp8 ? k_flash_few<64, kPagedFp8, MODE> : k_flash_few<64, kPagedBf16, MODE>);
    int threads = 64 * kFewWaves;
    if constexpr (MODE == kWindow) {
      if (fp8 && few_wide(f)) {
        threads = 512;
        kern = D == 128 ? k_flash_few_wide<128> : k_flash_few_wide<64>;
      }
    }
    hipLaunchKernelGGL(kern, grid, dim3(threads), 0, stream, *a);
  } else {
    a->neighbours = window_neighbours(f.tiles, f.splits);
    const dim3 grid((unsigned)(MODE == kWindow ? window_groups(f.tiles, a->Hkv, a->neighbours) : f.tiles), (unsigned)f.splits);
    auto* kern = D == 128 ? (fp8 ? k_flash_tile<128, kPagedFp8, MODE> : k_flash_tile<128, kPagedBf16, MODE>)
                          : (fp8 ? k_flash_tile<64, kPagedFp8, MODE> : k_flash_tile<64, kPagedBf16, MODE>);
    hipLaunchKernelGGL(kern, grid, dim3(256), 0, stream, *a);
  }
  const int launched = check_launch(what);
  if (launched != BTL_OK || f.splits == 1) return launched;
  return launch_merge(what, *a, T, H, D, false, f.splits, stream);
}

}  // namespace btl
