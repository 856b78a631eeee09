// Attention of rows that see a window of the last positions and the first few ("sinks"), within packed
// prompts and over the pages of a cache: the entry points.
#include "btl_flash_plan.h"

namespace btl {

// The plan of a call over pages, by `seen`, the positions of the longest axis that a workgroup walks: those of its rows' windows
// (`tokens` of them side by side), the sinks, and what both are rounded to.  Windows are alike in length, so that a split
// only pays where the CUs are not full; measured on 256 of them, 20 / 5 heads of 128, us, chunks in positions:
//  - Few rows: as many workgroups as CUs, a chunk at least a round of 4 waves, up to 36 of them (the merge).  One user, bf16, window
//    4096, 128 / 256 / 512 / one: 12.3, 13.5, 15.6, 47.6; 8000: 16.8, 13.7, 15.1, 77.6; 4 users, 2000 (a CU each at
//    256): 16.1, 13.8, 15.7, 27.4; 8 users, 8-bit, 1024 (256): 13.5, 12.4, 13.7, 14.3.  Where it shortens the longest workgroup
//    by less than 576 positions the merge's launch costs more, 25 users, 1024, 640 / one: 8-bit 16.7, 14.8; bf16 20.0, 19.5.  From a
//    workgroup on every other CU on: as without a window.
//  - Tiles: up to two workgroups a CU on every XCD, by the rule on what a split costs (FlashPlan), a chunk not below 192.
//    bf16, 1 / 2 / 3 / 4 / 6 / 8 splits: 500 rows of one user, 4096 (80 tiles of rows and heads): -, 54, 43, 42, 44, 54; 250, 4096
//    (40): -, 52, 40, 34, 29.5, 33; 1000, 4096 (160): -, 71, 67, 84, 78, 84; 20 users of 10, 2000 (100): 50, 36, 33, 30.5, 34;
//    4 users' 2047 rows, 2000 (340): 68, 69.  8-bit, 8 users of 1-10 rows, 1024 (40), chunks of 192 / 256 / 512: 18.6, 19.1,
//    24.2.
constexpr int64_t kWindowSplits = 36;
constexpr int64_t kWindowGain = 576;
constexpr int64_t kWindowChunk = 192;
inline FlashPlan window_plan(int64_t T, int64_t H, int64_t Hkv, int64_t D, int64_t B, int64_t max_q, int64_t max_kv,
                             int64_t window, int64_t sinks) {
  const int64_t G = H / Hkv, cus = device_cus();
  const int64_t tokens = std::min(std::min(max_q, T), (int64_t)kTileRows / G + 2);
  const int64_t all = std::min(window, kMaxPositions) + tokens + kStep + round_up(std::min(sinks, kMaxPositions), kStep);
  const int64_t seen = std::min(std::min(max_kv, all), kMaxPositions);
  FlashPlan f = flash_plan(T, H, Hkv, D, B, max_q, 1, true);  // one split
  f.chunk = (int)round_up(seen, kMinChunk);
  int64_t n, chunk;
  if (f.few) {
    n = std::min(cus / f.tiles, kWindowSplits);
    if (n <= 1) return flash_plan(T, H, Hkv, D, B, max_q, seen, true);
    chunk = round_up((seen + n - 1) / n, 32 * kFewWaves);
    if (seen - chunk < kWindowGain) return f;
  } else {
    const int64_t tiles = std::min(f.tiles, B * ((std::min(max_q, T) * G + kTileRows - 1) / kTileRows) * Hkv);  // (if the hint holds)
    const double whole = split_whole(seen), part = split_part(T, H, D);
    n = std::min(2 * cus / kXcds / ((tiles + kXcds - 1) / kXcds), (int64_t)(std::sqrt(whole / part) + 0.5));
    if (n <= 1 || whole - whole / (double)n <= 4.0 + part * (double)n) return f;
    chunk = std::max(kWindowChunk, round_up((seen + n - 1) / n, kStep));
    if (chunk >= seen) return f;
  }
  f.chunk = (int)chunk;
  f.splits = (int)((seen + chunk - 1) / chunk);
  return f;
}

static int check_window(const char* who, int64_t window, int64_t sinks, FlashArgs* a) {
  if (window < 1 || sinks < 0)
    return set_error(BTL_ERR_ARG, "%s: window=%lld sinks=%lld", who, (long long)window, (long long)sinks);
  a->window = (int)std::min(window, kMaxPositions);
  a->sinks = (int)std::min(sinks, kMaxPositions);
  return BTL_OK;
}

}  // namespace btl

using namespace btl;

extern "C" {

int btl_prompt_attention_window(const uint16_t* q, int64_t ldq, const uint16_t* k, int64_t ldk, const uint16_t* v,
                                int64_t ldv, int64_t T, int64_t H, int64_t Hkv, int64_t D, const int32_t* cu_q, int64_t B,
                                float scale, int64_t max_q, int64_t window, int64_t sinks, uint16_t* out, int64_t ldo,
                                int32_t* error_word, btl_stream_t stream) {
  const char* who = "btl_prompt_attention_window";
  clear_error();
  FlashArgs a{};
  int rc = prompt_args(who, q, ldq, k, ldk, v, ldv, T, H, Hkv, D, cu_q, B, scale, max_q, out, ldo, error_word, &a);
  if (rc == BTL_OK) rc = check_window(who, window, sinks, &a);
  if (rc != BTL_OK || T == 0) return rc;
  const int64_t tiles = flash_plan(T, H, Hkv, D, B, T, T, false).tiles;
  if (window >= T)  // every row sees all of its sequence: the causal kernel, and its bits
    return launch_causal_prompt(a, tiles, D, (hipStream_t)stream);
  return launch_prompt<kWindow>("prompt attention in a window", a, tiles, D, (hipStream_t)stream);
}

int64_t btl_paged_attention_window_scratch_bytes(int64_t T, int64_t H, int64_t Hkv, int64_t D, int64_t B, int64_t max_q,
                                                 int64_t max_kv, int64_t window, int64_t sinks) {
  if (!flash_sizes(T, H, Hkv, D, B, max_q, max_kv) || window < 1 || sinks < 0) return 0;
  return flash_scratch(window_plan(T, H, Hkv, D, B, max_q, max_kv, window, sinks), T, H, D);
}

int btl_paged_attention_window_plan(int64_t T, int64_t H, int64_t Hkv, int64_t D, int64_t B, int64_t max_q, int64_t max_kv,
                                    int64_t window, int64_t sinks, int64_t* plan) {
  if (!plan || !flash_sizes(T, H, Hkv, D, B, max_q, max_kv) || window < 1 || sinks < 0) return 0;
  const FlashPlan f = window_plan(T, H, Hkv, D, B, max_q, max_kv, window, sinks);
  plan[0] = f.few;
  plan[1] = f.splits;
  plan[2] = f.chunk;
  return 1;
}

int64_t btl_attention_window_tile(int64_t tiles, int64_t splits, int64_t Hkv, int64_t x, int64_t* tile) {
  if (!tile || Hkv <= 0 || Hkv > 1024 || tiles <= 0 || tiles > (1 << 26) || tiles % Hkv || splits <= 0) return 0;
  const int each = window_neighbours(tiles, splits > 1 ? 2 : 1);
  const int64_t groups = window_groups(tiles, Hkv, each);
  if (x < 0 || x >= groups) return 0;
  const HeadTile t = window_tile((int)x, (int)Hkv, each);
  tile[0] = each;
  tile[1] = t.hk;
  tile[2] = t.x;
  return groups;
}

int btl_paged_attention_window(const uint16_t* q, int64_t ldq, int64_t T, int64_t H, const btl_pages_t* pages,
                               const int32_t* page_table, int64_t max_pages, const int32_t* cu_q, const int32_t* kv_len,
                               int64_t B, float scale, int64_t max_q, int64_t max_kv, int64_t window, int64_t sinks,
                               uint16_t* out, int64_t ldo, void* scratch, size_t scratch_bytes, int32_t* error_word,
                               btl_stream_t stream) {
  const char* who = "btl_paged_attention_window";
  clear_error();
  FlashArgs a{};
  int rc = paged_args(who, q, ldq, T, H, pages, page_table, max_pages, cu_q, kv_len, B, scale, max_q, max_kv, out, ldo,
                      error_word, &a);
  if (rc == BTL_OK) rc = check_window(who, window, sinks, &a);
  if (rc != BTL_OK || T == 0) return rc;
  const FlashPlan f = window_plan(T, H, pages->num_kv_heads, pages->head_dim, B, max_q, max_kv, window, sinks);
  return launch_paged<kWindow>(who, "paged attention in a window", f, &a, T, H, pages->head_dim, pages->k_exp != nullptr,
                               scratch, scratch_bytes, (hipStream_t)stream);
}

}  // extern "C"
