// Attention of a batch whose sequences begin with the same pages: the entry points.
//
//   out_i = (e_p o_p + sum_z e_z o_z) / (e_p l_p + sum_z e_z l_z),   e = 2^(m - max m)
//
// where (m, l, o) are maximum, sum and product of a part of the positions that row i sees.  The rows
// of all sequences together (their G query heads of a key-value head) attend to the shared positions,
// so that those are read once for 128 rows and not once for each sequence; each sequence's rows attend to
// its own positions as everywhere else.  Both are workgroups of one launch, the shared ones
// first; the merge is a second one.
//
// p of the shared positions is one bf16 value in tiles, also where a call without a prefix would have the two of
// few rows (single tokens over bf16 pages): two would cost a tile a third of its rate.  32 users of 8192 + 500, against 64 bits:
// 0.0023 of the outputs' size, 0.0017 without a prefix, which is their own rounding.  Up to 16 rows of heads in all, and
// every sequence's own positions, keep two.
#include <type_traits>

#include "btl_flash_plan.h"

namespace btl {

// FEW: the kernel of few rows for a part, else tiles of 128 rows.
template <int D, int KV, bool SHARED_FEW, bool OWN_FEW>
__global__ __launch_bounds__(256, 2) void k_flash_shared(FlashArgs p, int shared_items, int own_items) {
  constexpr int kFewBytes = (int)sizeof(FewShared<D>);
  constexpr int kBytes = SHARED_FEW && OWN_FEW ? kFewBytes : kFewBytes > kTileShared<D> ? kFewBytes : kTileShared<D>;
  __shared__ __attribute__((aligned(16))) uint8_t smem[kBytes];
  const int units = p.Hkv * p.shared_splits, shared = (units + kXcds - 1) / kXcds * kXcds * shared_items;
  int x = blockIdx.x;
  if (x < shared) {
    // the tiles of a head's split read the same pages
    const UnitItem u = unit_item(x, shared_items);
    if (u.unit >= units) return;
    const int hk = uni(u.unit % p.Hkv), split = uni(u.unit / p.Hkv), item = uni(u.item);
    if constexpr (SHARED_FEW)
      few_item<D, KV, kShared>(p, *reinterpret_cast<FewShared<D>*>(smem), hk, 0, split);
    else
      tile_item<D, KV, kShared>(p, smem, hk, item, split);
  } else {
    x -= shared;
    const int hk = uni(x % p.Hkv), y = x / p.Hkv, item = uni(y % own_items), split = uni(y / own_items);
    if constexpr (OWN_FEW)
      few_item<D, KV, kOwn>(p, *reinterpret_cast<FewShared<D>*>(smem), hk, item, split);
    else
      tile_item<D, KV, kOwn>(p, smem, hk, item, split);
  }
}

constexpr int64_t kSharedSplits = 64;  // of tiles

struct SharedPlan {
  bool shared_few;
  int64_t shared_items, own_items;  // of a key-value head
  int shared_splits, shared_chunk;
  FlashPlan own;
};

// max_kv: positions of the longest sequence, max_shared of them shared (max_kv or more: not known).
//  - The shared positions in tiles: the split of the least time, in units of a step of a workgroup that has its CU alone (among
//    the tiles): steps x 1, or 1.4 where two share a CU, by the workgroups of an XCD, which has a unit's all (unit_item), in
//    rounds; and 2.4 times what a split's partials take, as the merge reads them with the rest.  Against the best of up to 27 splits
//    in 26 shapes it is 3% above in the mean, 14% at most (128 users of up to 2000 behind 16384, 8-bit, whose own positions keep
//    the CUs busy besides; their work in the rule gains nothing unless it knows the pages' type).  20 / 5 heads of 128, bf16, us
//    by splits: 200 rows of 8 users behind 16000 (7 tiles a head): 5: 88, 6: 77, 7: 84, 10: 73, 13: 60, 16: 74; 400 of
//    4 (13): 5: 118, 6: 105, 7: 138, 12: 105; 32 users behind 8192 (1): 11: 26, 22: 22.5, 32: 24.5, 64: 26.6; 64 of 65536,
//    8-bit (2): 16: 125, 25: 92, 32: 91, 36: 85, 64: 99.  A chunk is at least two steps.
//  - Few rows in all: as for a call without a prefix.
//  - Their own positions: the merge's launch is paid in any case, so that splits that fill two workgroups a CU pay from 512
//    positions on: 16 users of 8192 + 1000, n = 1 / 2: 21.7, 19.5; 16 x 5 rows of 16000 + 1000, 1 / 2 / 4: 41, 39, 34.
//    Where the shared positions are not known they are planned for all of max_kv: 4 users of 1024 + 16000 39 us (with one
//    position of their own 147, known 34), 32 of 8192 + 500 23.6 (known 22.2), 16 of 2048 + 4000 30.5 (known 35).
inline SharedPlan shared_plan(int64_t T, int64_t H, int64_t Hkv, int64_t D, int64_t B, int64_t max_q, int64_t max_kv,
                              int64_t max_shared) {
  SharedPlan s{};
  const int64_t G = H / Hkv, cus = device_cus();
  // (both parts' ends together stay below 2^31)
  max_shared = std::max(std::min(max_shared, kMaxPositions), (int64_t)1);
  // a prefix as long as the sequences is no known length: their own positions may be all of theirs
  const int64_t own = std::min(max_shared < max_kv ? max_kv - max_shared : max_kv, kMaxPositions / 2);
  s.own = flash_plan(T, H, Hkv, D, B, max_q, own, true);
  s.own_items = s.own.few ? B : s.own.tiles / Hkv;
  s.shared_few = T * G <= kFewRows && s.own.few;
  s.shared_items = s.shared_few ? 1 : (T * G + kTileRows - 1) / kTileRows;
  const int64_t tiles = s.shared_items * Hkv;
  if (s.shared_few) {
    const FlashPlan f = flash_plan(T, H, Hkv, D, 1, 1, max_shared, true);
    s.shared_splits = f.splits;
    s.shared_chunk = f.chunk;
  } else {
    const double part = 2.4 * split_part(T, H, D);
    const int64_t place = std::max(cus / kXcds, (int64_t)1);  // an XCD's CUs
    double least = 0;
    for (int64_t n = 1; n <= std::max((int64_t)1, std::min(max_shared / (2 * kStep), kSharedSplits)); ++n) {
      const int64_t groups = (Hkv * n + kXcds - 1) / kXcds * s.shared_items, full = (groups - 1) / (2 * place);
      const int64_t chunk = round_up((max_shared + n - 1) / n, kStep);
      const double step = 1.4 * (double)full + (groups - full * 2 * place > place ? 1.4 : 1.0);
      const double t = step * (double)(chunk / kStep) + part * (double)n;
      if (n > 1 && t >= least) continue;
      least = t;
      s.shared_chunk = (int)chunk;
    }
    s.shared_splits = (int)((max_shared + s.shared_chunk - 1) / s.shared_chunk);
  }
  const int64_t rest = (2 * cus - tiles * s.shared_splits) / (s.own_items * Hkv);
  const int64_t n = std::min(rest, std::min(own / kMinChunk, kMaxSplits));
  if (n > s.own.splits) {
    s.own.chunk = (int)round_up((own + n - 1) / n, kMinChunk);
    s.own.splits = (int)((own + s.own.chunk - 1) / s.own.chunk);
  }
  return s;
}

inline int64_t shared_scratch(const SharedPlan& s, int64_t T, int64_t H, int64_t D) {
  return (int64_t)(s.shared_splits + s.own.splits) * T * H * (D + 2) * 4;
}

inline bool shared_sizes(int64_t T, int64_t H, int64_t Hkv, int64_t D, int64_t B, int64_t max_q, int64_t max_kv,
                         int64_t max_shared) {
  return flash_sizes(T, H, Hkv, D, B, max_q, max_kv) && max_shared >= 0;
}

}  // namespace btl

using namespace btl;

extern "C" {

int64_t btl_shared_prefix_attention_scratch_bytes(int64_t T, int64_t H, int64_t Hkv, int64_t D, int64_t B, int64_t max_q,
                                                  int64_t max_kv, int64_t max_shared) {
  if (!shared_sizes(T, H, Hkv, D, B, max_q, max_kv, max_shared)) return 0;
  return shared_scratch(shared_plan(T, H, Hkv, D, B, max_q, max_kv, max_shared), T, H, D);
}

int btl_shared_prefix_attention_plan(int64_t T, int64_t H, int64_t Hkv, int64_t D, int64_t B, int64_t max_q, int64_t max_kv,
                                     int64_t max_shared, int64_t* plan) {
  if (!plan || !shared_sizes(T, H, Hkv, D, B, max_q, max_kv, max_shared)) return 0;
  const SharedPlan s = shared_plan(T, H, Hkv, D, B, max_q, max_kv, max_shared);
  plan[0] = s.shared_few;
  plan[1] = s.shared_splits;
  plan[2] = s.shared_chunk;
  plan[3] = s.own.few;
  plan[4] = s.own.splits;
  plan[5] = s.own.chunk;
  return 1;
}

int btl_shared_prefix_attention(const uint16_t* q, int64_t ldq, int64_t T, int64_t H, const btl_pages_t* pages,
                                const int32_t* page_table, int64_t max_pages, const int32_t* cu_q, const int32_t* kv_len,
                                const int32_t* shared_pages, int64_t B, float scale, int64_t max_q, int64_t max_kv,
                                int64_t max_shared, uint16_t* out, int64_t ldo, void* scratch, size_t scratch_bytes,
                                int32_t* error_word, btl_stream_t stream) {
  const char* who = "btl_shared_prefix_attention";
  clear_error();
  FlashArgs a{};
  int rc = paged_args(who, q, ldq, T, H, pages, page_table, max_pages, cu_q, kv_len, B, scale, max_q, max_kv, out, ldo,
                      error_word, &a);
  if (rc != BTL_OK) return rc;
  if (max_shared < 0) return set_error(BTL_ERR_SHAPE, "%s: max_shared=%lld", who, (long long)max_shared);
  if (T == 0) return BTL_OK;
  if (!shared_pages) return set_error(BTL_ERR_NULL, "%s: NULL pointer", who);
  if (!aligned(shared_pages, 4)) return set_error(BTL_ERR_ALIGN, "%s: misaligned shared_pages", who);
  const int64_t Hkv = a.Hkv, D = pages->head_dim;
  const bool fp8 = pages->k_exp != nullptr;
  const SharedPlan s = shared_plan(T, H, Hkv, D, B, max_q, max_kv, max_shared);
  const int parts = s.shared_splits + s.own.splits;
  const int64_t groups = unit_groups(s.shared_splits * Hkv, s.shared_items) + s.own_items * s.own.splits * Hkv;
  if (groups > INT32_MAX) return set_error(BTL_ERR_SHAPE, "%s: T=%lld B=%lld", who, (long long)T, (long long)B);
  rc = partials(who, scratch, scratch_bytes, shared_scratch(s, T, H, D), (int64_t)parts * T * H * D, &a);
  if (rc != BTL_OK) return rc;
  a.shared = shared_pages;
  a.shared_splits = s.shared_splits;
  a.shared_chunk = s.shared_chunk;
  a.splits = s.own.splits;
  a.chunk = s.own.chunk;
  auto pick = [&](auto d, auto kv) {
    constexpr int kD = decltype(d)::value, kKV = decltype(kv)::value;
    return s.shared_few ? k_flash_shared<kD, kKV, true, true>
           : s.own.few  ? k_flash_shared<kD, kKV, false, true>
                        : k_flash_shared<kD, kKV, false, false>;
  };
  using std::integral_constant;
  auto* kern = D == 128 ? (fp8 ? pick(integral_constant<int, 128>(), integral_constant<int, kPagedFp8>())
                               : pick(integral_constant<int, 128>(), integral_constant<int, kPagedBf16>()))
                        : (fp8 ? pick(integral_constant<int, 64>(), integral_constant<int, kPagedFp8>())
                               : pick(integral_constant<int, 64>(), integral_constant<int, kPagedBf16>()));
  hipLaunchKernelGGL(kern, dim3((unsigned)groups), dim3(256), 0, (hipStream_t)stream, a, (int)s.shared_items,
                     (int)s.own_items);
  rc = check_launch("shared prefix attention");
  if (rc != BTL_OK) return rc;
  return launch_merge("shared prefix attention", a, T, H, D, true, parts, (hipStream_t)stream);
}

}  // extern "C"
