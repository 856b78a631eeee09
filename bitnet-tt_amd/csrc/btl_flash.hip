// Causal attention within packed prompts and over the pages of a cache: the entry points.
// (The kernels: btl_flash_body.h; how contexts are split: btl_flash_plan.h.)
#include "btl_flash_plan.h"

namespace btl {

int launch_merge(const char* what, const FlashArgs& a, int64_t T, int64_t H, int64_t D, bool shared, int parts,
                 hipStream_t stream) {
  // up to four splits for a group of threads
  const int ng = D == 128 ? 8 : 16;
  int groups = 1;
  while (groups < ng && 4 * groups < parts) groups *= 2;
  const dim3 grid((unsigned)((T * H * groups + ng - 1) / ng));
  auto* kern = D == 128 ? (shared ? k_flash_merge<128, true> : k_flash_merge<128, false>)
                        : (shared ? k_flash_merge<64, true> : k_flash_merge<64, false>);
  hipLaunchKernelGGL(kern, grid, dim3(256), 0, stream, a, groups);
  return check_launch(what);
}

int launch_causal_prompt(const FlashArgs& a, int64_t tiles, int64_t D, hipStream_t stream) {
  return launch_prompt<kCausal>("prompt attention", a, tiles, D, stream);
}

}  // namespace btl

using namespace btl;

extern "C" {

int btl_prompt_attention(const uint16_t* q, int64_t ldq, const uint16_t* k, int64_t ldk, const uint16_t* v,
                         int64_t ldv, int64_t T, int64_t H, int64_t Hkv, int64_t D, const int32_t* cu_q, int64_t B,
                         float scale, int64_t max_q, uint16_t* out, int64_t ldo, int32_t* error_word,
                         btl_stream_t stream) {
  clear_error();
  FlashArgs a{};
  const int rc = prompt_args("btl_prompt_attention", q, ldq, k, ldk, v, ldv, T, H, Hkv, D, cu_q, B, scale, max_q, out, ldo,
                             error_word, &a);
  if (rc != BTL_OK || T == 0) return rc;
  return launch_causal_prompt(a, flash_plan(T, H, Hkv, D, B, T, T, false).tiles, D, (hipStream_t)stream);
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
  const int rc = paged_args(who, q, ldq, T, H, pages, page_table, max_pages, cu_q, kv_len, B, scale, max_q, max_kv, out, ldo,
                            error_word, &a);
  if (rc != BTL_OK || T == 0) return rc;
  const FlashPlan f = flash_plan(T, H, pages->num_kv_heads, pages->head_dim, B, max_q, max_kv, true);
  return launch_paged<kCausal>(who, "paged attention", f, &a, T, H, pages->head_dim, pages->k_exp != nullptr, scratch,
                               scratch_bytes, (hipStream_t)stream);
}

}  // extern "C"
