// Attention of rows that see a window of the last positions and the first few ("sinks"), within packed
// prompts and over the pages of a cache: the entry points.
#include "btl_flash_plan.h"

namespace btl {

// Positions of the longest axis that a workgroup walks: those of its rows' windows (`tokens` of them
// side by side), the sinks, and what both are rounded to.
inline FlashPlan window_plan(int64_t T, int64_t H, int64_t Hkv, int64_t D, int64_t B, int64_t max_q, int64_t max_kv,
                             int64_t window, int64_t sinks) {
  const int64_t G = H / Hkv;
  const int64_t tokens = std::min(std::min(max_q, T), (int64_t)kTileRows / G + 2);
  const int64_t seen = std::min(window, kMaxPositions) + tokens + kStep + round_up(std::min(sinks, kMaxPositions), kStep);
  return flash_plan(T, H, Hkv, D, B, max_q, std::min(max_kv, seen), true);
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
