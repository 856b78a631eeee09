// Writing and reading the paged key-value cache.
//
// k_rope_write: the fused QKV rows of a batch of packed tokens -> rotated
// queries, and rotated keys and values in their pages (src/bitnet_tt/layers/
// attention.py:1088-1171 does the same for one token per user).  Per head row
//   (y_a, y_b) = (x_a c - x_b s, x_b c + x_a s),  c, s = cos, sin(position x freq_i)
// over the first R dims: pairs (i, i + R/2), or (2i, 2i + 1).  8-bit pages: per
// row e = the least exponent with max|y| <= 448 2^e, codes e4m3(y 2^-e).
//
// Bound by memory (and, for a decode step's few rows, by the chain table entry
// -> position -> angle -> store).  A thread takes 16 values of a head row, as
// two 16-byte pieces that hold both members of its pairs, so a row is D / 16
// neighbouring lanes and its maximum three lane exchanges.  A workgroup takes
// whole tokens: one where there are few, so that every row has a workgroup,
// else 8, which looks the sequences up once for 1920 pieces of the 2B heads.
// 32 single tokens of 20 / 5 heads of 128 4.0 us; prompts of 8191 tokens to 8-bit pages 27.8 us,
// 120 MB at 4.3 TB/s.  (Ordinary stores: what is written is read by the attention next.)
//
// k_read_pages: rows of pages -> a contiguous [B, Hkv, S, D] bf16 cache, a copy
// (or one conversion per two values).  Bound by memory: small workgroups whose
// threads have one key and one value piece each, so that all of a workgroup's
// loads leave at once after one page lookup, and stores past the caches, which
// hold nothing of the copy that is read again soon.  32 users x 4096 positions of 5
// heads of 128, 8-bit pages, workgroups of 64 / 32 / 16 rows: 80.6, 70.4, 60.1 us (5.5
// TB/s; with ordinary stores 86.2, 78.0 at 64, 32); bf16 pages 87.7, 82.3, 80.7 us.
#include <hip/hip_runtime.h>

#include "btl.h"
#include "btl_act_row.h"
#include "btl_common.h"
#include "btl_fp8.h"
#include "btl_paged.h"

namespace btl {

constexpr int kRopeThreads = 256;
constexpr int kRopeTokens = 8;  // tokens of a workgroup where there are many

struct RopeArgs {
  const uint16_t* qkv;
  int64_t ldx;
  int H, Hkv, R, S, adjacent;
  const float* rcos;  // [S][R / 2]
  const float* rsin;
  Batch bt;
  Pages pg;  // k == NULL: none
  int fp8;
  uint16_t* q;  // [T][H D], row stride ldq
  int64_t ldq;
  uint16_t* ko;  // [T][Hkv D], row stride ldk, or NULL
  int64_t ldk;
  int32_t* error;
  FastDiv heads;  // H + 2 Hkv
  int tokens;     // of a workgroup
};

// 16 values of a head row at dims o0 .. o0 + 7 and o1 .. o1 + 7.
struct Piece {
  uint4 a, b;
};

template <int D>
__global__ __launch_bounds__(kRopeThreads) void k_rope_write(RopeArgs p) {
  constexpr int U = D / 16;  // pieces of a head row
  __shared__ int s_pos[kRopeTokens];   // -1: no position (zero rows), -2: not a row of the batch
  __shared__ int s_page[kRopeTokens];  // -1: nothing to write
  __shared__ int s_row[kRopeTokens];
  const int tid = threadIdx.x, t0 = blockIdx.x * p.tokens;
  const int nt = min(p.tokens, p.bt.T - t0), items = nt * (int)p.heads.d * U;
  const int u = tid & (U - 1);

  // piece `idx` of the workgroup: token t, head row h
  auto where = [&](int idx, int& t, int& h, int& o0, int& o1) {
    const uint32_t r = idx / U;
    t = div_by(r, p.heads);
    h = r - t * p.heads.d;
    const bool halves = !p.adjacent && h < p.H + p.Hkv && 16 * u < p.R;
    o0 = halves ? 8 * u : 16 * u;
    o1 = halves ? 8 * u + p.R / 2 : 16 * u + 8;
  };
  auto load = [&](int t, int h, int o0, int o1) {
    const uint16_t* x = p.qkv + (int64_t)(t0 + t) * p.ldx + h * D;
    return Piece{*reinterpret_cast<const uint4*>(x + o0), *reinterpret_cast<const uint4*>(x + o1)};
  };
  int t = 0, h = 0, o0 = 0, o1 = 0;
  Piece x{};
  const bool any = tid < items;
  if (any) {  // the first piece does not wait for the lookup
    where(tid, t, h, o0, o1);
    x = load(t, h, o0, o1);
  }

  if (tid < 64) {  // one wave looks the tokens up, 64 sequences at a time
    int mine = -1, first = 0, n = 0;
    bool ok = true;
    for (int c = 0; c < p.bt.B; c += 64) {
      const int b = c + tid;
      Seq s{0, 0, 0, true};
      if (b < p.bt.B) s = clamp_seq(p.bt.cu[b], p.bt.cu[b + 1], 0, p.bt.T, 0);
      ok = ok && s.ok;
      for (int i = 0; i < nt; ++i) {
        const uint64_t hit = __ballot(t0 + i >= s.row0 && t0 + i < s.row0 + s.n);
        if (hit) {
          const int l = __builtin_ctzll(hit);
          const int r0 = __builtin_amdgcn_readlane(s.row0, l), rn = __builtin_amdgcn_readlane(s.n, l);
          if (tid == i && mine < 0) {
            mine = c + l;
            first = r0;
            n = rn;
          }
        }
      }
    }
    if (tid < nt) {
      int pos = -2, page = -1, row = 0;
      if (mine >= 0) {
        const int64_t cap = p.pg.k ? min((int64_t)p.bt.max_pages * p.pg.ps.d, (int64_t)INT32_MAX) : INT32_MAX;
        const int len = p.bt.len ? p.bt.len[mine] : n;
        if (len < 0 || len > cap) {
          ok = false;
          pos = -1;
        } else {
          pos = max(-1, len - n + (t0 + tid - first));
        }
        if (pos >= p.S) {
          ok = false;
          pos = -1;
        }
        if (pos >= 0 && p.pg.k) {
          const uint32_t pi = div_by(pos, p.pg.ps);
          row = pos - pi * p.pg.ps.d;
          page = p.bt.table[(int64_t)mine * p.bt.max_pages + pi];
          if (page < 0 || page >= p.pg.P) {
            ok = false;
            page = -1;
          }
        }
      }
      s_pos[tid] = pos;
      s_page[tid] = page;
      s_row[tid] = row;
    }
    if (!ok) flag_error(p.error);
  }
  __syncthreads();

  for (int idx = tid; idx < items; idx += kRopeThreads) {
    if (idx != tid) {
      where(idx, t, h, o0, o1);
      x = load(t, h, o0, o1);
    }
    const int pos = s_pos[t], page = s_page[t];
    if (pos == -2) continue;  // behind the last sequence: left as it is (all of a row's lanes alike)
    const uint16_t* xa = reinterpret_cast<const uint16_t*>(&x.a);
    const uint16_t* xb = reinterpret_cast<const uint16_t*>(&x.b);
    float y[16];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      y[j] = bf2f(xa[j]);
      y[8 + j] = bf2f(xb[j]);
    }
    const bool is_v = h >= p.H + p.Hkv, is_k = h >= p.H && !is_v;
    if (!is_v && pos < 0) {
#pragma unroll
      for (int j = 0; j < 16; ++j) y[j] = 0.0f;
    } else if (!is_v && 16 * u < p.R) {
      float c[8], s[8];
      const int64_t at = (int64_t)pos * (p.R / 2) + 8 * u;
      *reinterpret_cast<float4*>(c) = *reinterpret_cast<const float4*>(p.rcos + at);
      *reinterpret_cast<float4*>(c + 4) = *reinterpret_cast<const float4*>(p.rcos + at + 4);
      *reinterpret_cast<float4*>(s) = *reinterpret_cast<const float4*>(p.rsin + at);
      *reinterpret_cast<float4*>(s + 4) = *reinterpret_cast<const float4*>(p.rsin + at + 4);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (p.adjacent) {
          const float a = y[2 * j], b = y[2 * j + 1];
          y[2 * j] = a * c[j] - b * s[j];
          y[2 * j + 1] = b * c[j] + a * s[j];
        } else {
          const float a = y[j], b = y[8 + j];
          y[j] = a * c[j] - b * s[j];
          y[8 + j] = b * c[j] + a * s[j];
        }
      }
    }
    Piece o;
    o.a = make_uint4(f2bf_pair(y[0], y[1]), f2bf_pair(y[2], y[3]), f2bf_pair(y[4], y[5]), f2bf_pair(y[6], y[7]));
    o.b = make_uint4(f2bf_pair(y[8], y[9]), f2bf_pair(y[10], y[11]), f2bf_pair(y[12], y[13]), f2bf_pair(y[14], y[15]));
    if (!is_k && !is_v) {
      uint16_t* d = p.q + (int64_t)(t0 + t) * p.ldq + h * D;
      *reinterpret_cast<uint4*>(d + o0) = o.a;
      *reinterpret_cast<uint4*>(d + o1) = o.b;
      continue;
    }
    const int hk = is_k ? h - p.H : h - p.H - p.Hkv;
    if (is_k && p.ko) {
      uint16_t* d = p.ko + (int64_t)(t0 + t) * p.ldk + hk * D;
      *reinterpret_cast<uint4*>(d + o0) = o.a;
      *reinterpret_cast<uint4*>(d + o1) = o.b;
    }
    const int64_t at = page_row(page, p.pg.P, p.Hkv, hk, p.pg.ps.d, s_row[t]);
    if (at < 0) continue;
    uint8_t* const pages = is_k ? p.pg.k : p.pg.v;
    if (!p.fp8) {
      uint16_t* d = reinterpret_cast<uint16_t*>(pages) + at * D;
      *reinterpret_cast<uint4*>(d + o0) = o.a;
      *reinterpret_cast<uint4*>(d + o1) = o.b;
      continue;
    }
    // the row's largest magnitude as bits: NaN is above infinity, infinity above the rest
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 16; ++j) m = max(m, __float_as_uint(y[j]) & 0x7fffffffu);
    if (U == 8) m = max(m, xor_partner_u<4>(m));
    m = max(m, xor_partner_u<2>(m));
    m = max(m, xor_partner_u<1>(m));
    uint2 ca, cb;
    int e = 0;
    if (m >= 0x7f800000u) {  // a value that is not finite: the row reads as NaN
      ca = cb = make_uint2(0x7f7f7f7fu, 0x7f7f7f7fu);
    } else {
      e = row_exponent(__uint_as_float(m));
      ca = to_e4m3(y, -e);
      cb = to_e4m3(y + 8, -e);
    }
    uint8_t* d = pages + at * D;
    *reinterpret_cast<uint2*>(d + o0) = ca;
    *reinterpret_cast<uint2*>(d + o1) = cb;
    if (u == 0) (is_k ? p.pg.ke : p.pg.ve)[at] = (uint8_t)(e + 127);
  }
}

struct ReadArgs {
  Batch bt;
  Pages pg;
  int fp8, S;
  uint16_t* k;  // [B, Hkv, S, D]
  uint16_t* v;
  int32_t* error;
};
// Rows of a workgroup: a thread takes 8 values of a key row and of its value row.
constexpr int read_rows(int D) { return 2048 / D; }

template <int D, bool FP8>
__global__ __launch_bounds__(256) void k_read_pages(ReadArgs p) {
  constexpr int C = D / 8;
  const int b = blockIdx.z, hk = blockIdx.y, r0 = blockIdx.x * read_rows(D);
  const int64_t cap = min((int64_t)p.bt.max_pages * p.pg.ps.d, (int64_t)p.S);
  const int len = p.bt.len[b];
  if (len < 0 || len > cap) {
    if (r0 == 0 && hk == 0 && threadIdx.x == 0) flag_error(p.error);
    return;
  }
  const int row = r0 + threadIdx.x / C, c = threadIdx.x % C;
  if (row >= len) return;
  const uint32_t pi = div_by(row, p.pg.ps);
  const int64_t at =
      page_row(p.bt.table[(int64_t)b * p.bt.max_pages + pi], p.pg.P, p.pg.Hkv, hk, p.pg.ps.d, row - pi * p.pg.ps.d);
  uint4 x[2] = {};
  uint32_t e[2] = {127, 127};
  if (at >= 0) {
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      const uint8_t* src = (kv ? p.pg.v : p.pg.k) + (at * C + c) * (FP8 ? 8 : 16);
      if (FP8) {
        const uint2 w = *reinterpret_cast<const uint2*>(src);
        x[kv] = make_uint4(w.x, w.y, 0, 0);
        e[kv] = (kv ? p.pg.ve : p.pg.ke)[at];
      } else {
        x[kv] = *reinterpret_cast<const uint4*>(src);
      }
    }
  } else {
    flag_error(p.error);
  }
  typedef uint32_t v4u __attribute__((ext_vector_type(4)));
  const int64_t to = (((int64_t)b * p.pg.Hkv + hk) * p.S + row) * D + 8 * c;
#pragma unroll
  for (int kv = 0; kv < 2; ++kv) {
    const uint4 y = FP8 ? from_e4m3(make_uint2(x[kv].x, x[kv].y), exp_scale(e[kv])) : x[kv];
    __builtin_nontemporal_store(__builtin_bit_cast(v4u, y), reinterpret_cast<v4u*>((kv ? p.v : p.k) + to));
  }
}

int check_pages(const char* who, const btl_pages_t* p, Pages* out) {
  if (!p) return set_error(BTL_ERR_NULL, "%s: pages is NULL", who);
  if (p->head_dim != 64 && p->head_dim != 128)
    return set_error(BTL_ERR_SHAPE, "%s: head dim %lld (64 and 128 supported)", who, (long long)p->head_dim);
  if (p->num_pages <= 0 || p->num_pages > INT32_MAX || p->num_kv_heads <= 0 || p->num_kv_heads > 1024 ||
      p->page_size < 16 || p->page_size > kMaxPageSize || p->page_size % 16)
    return set_error(BTL_ERR_SHAPE, "%s: %lld pages of %lld heads x %lld rows (rows a multiple of 16, up to %d)", who,
                     (long long)p->num_pages, (long long)p->num_kv_heads, (long long)p->page_size, kMaxPageSize);
  if (!p->k || !p->v || !p->k_exp != !p->v_exp) return set_error(BTL_ERR_NULL, "%s: NULL page pointer", who);
  if (!aligned(p->k, 16) || !aligned(p->v, 16)) return set_error(BTL_ERR_ALIGN, "%s: pages must be 16-byte aligned", who);
  *out = Pages{static_cast<uint8_t*>(p->k), static_cast<uint8_t*>(p->v), p->k_exp, p->v_exp, (int)p->num_pages,
               (int)p->num_kv_heads, fast_div((uint32_t)p->page_size)};
  return BTL_OK;
}

int check_batch(const char* who, int64_t B, int64_t T, const int32_t* cu_q, const int32_t* kv_len,
                const int32_t* page_table, int64_t max_pages, Batch* out) {
  if (B <= 0 || B > kMaxSeqs || T < 0 || T > kMaxRows || max_pages < 0 || max_pages > (1 << 24))
    return set_error(BTL_ERR_SHAPE, "%s: B=%lld T=%lld max_pages=%lld", who, (long long)B, (long long)T,
                     (long long)max_pages);
  if (!cu_q && T > 0) return set_error(BTL_ERR_NULL, "%s: cu_q is NULL", who);
  if (!aligned(cu_q, 4) || !aligned(kv_len, 4) || !aligned(page_table, 4))
    return set_error(BTL_ERR_ALIGN, "%s: misaligned int32 array", who);
  *out = Batch{cu_q, kv_len, page_table, (int)B, (int)T, (int)max_pages};
  return BTL_OK;
}

}  // namespace btl

using namespace btl;

extern "C" {

int64_t btl_page_row(int64_t page, int64_t num_pages, int64_t num_kv_heads, int64_t kv_head, int64_t page_size,
                     int64_t position) {
  if (page_size < 16 || page_size > kMaxPageSize || num_pages > INT32_MAX || page > INT32_MAX || page < INT32_MIN ||
      position < 0 || position > INT32_MAX)
    return -1;
  const FastDiv f = fast_div((uint32_t)page_size);
  return page_row((int32_t)page, (int)num_pages, (int)num_kv_heads, (int)kv_head, (int)page_size,
                  (int)(position - (int64_t)div_by((uint32_t)position, f) * page_size));
}

int btl_page_run(int64_t page, int64_t num_pages, int64_t num_kv_heads, int64_t kv_head, int64_t page_size, int64_t position,
                 int64_t end, int64_t most, int64_t* run) {
  if (!run || page_size < 16 || page_size > kMaxPageSize || num_pages <= 0 || num_pages > INT32_MAX || page > INT32_MAX ||
      page < INT32_MIN || num_kv_heads <= 0 || num_kv_heads > 1024 || kv_head < 0 || kv_head >= num_kv_heads || position < 0 ||
      position > INT32_MAX || end < 0 || end > INT32_MAX || most < 0 || most > INT32_MAX)
    return -1;
  Pages pg{};
  pg.P = (int)num_pages;
  pg.Hkv = (int)num_kv_heads;
  pg.ps = fast_div((uint32_t)page_size);
  bool bad = false;
  const Run r = run_at(pg, (int)kv_head, (int)position, (int)end, (int32_t)page, (int)most, bad);
  run[0] = r.row;
  run[1] = r.n;
  return bad ? 1 : 0;
}

int btl_clamp_seq(int64_t lo, int64_t hi, int64_t len, int64_t T, int64_t cap, int64_t* seq) {
  if (!seq) return 0;
  const Seq s = clamp_seq((int)lo, (int)hi, (int)len, (int)T, cap);
  seq[0] = s.row0;
  seq[1] = s.n;
  seq[2] = s.len;
  return s.ok ? 1 : 0;
}

int btl_row_exponent(float largest) { return row_exponent(largest); }

int btl_rope_write(const uint16_t* qkv, int64_t T, int64_t ldx, int64_t H, int64_t Hkv, int64_t D,
                   const float* rope_cos, const float* rope_sin, int64_t R, int64_t S, int rope_adjacent,
                   const int32_t* cu_q, const int32_t* kv_len, int64_t B, uint16_t* q_out, int64_t ldq,
                   uint16_t* k_out, int64_t ldk, const btl_pages_t* pages, const int32_t* page_table,
                   int64_t max_pages, int32_t* error_word, btl_stream_t stream) {
  const char* who = "btl_rope_write";
  clear_error();
  RopeArgs a{};
  if (D != 64 && D != 128)
    return set_error(BTL_ERR_SHAPE, "%s: head dim %lld (64 and 128 supported)", who, (long long)D);
  if (H <= 0 || Hkv <= 0 || H > 1024 || Hkv > 1024 || H % Hkv)
    return set_error(BTL_ERR_SHAPE, "%s: H=%lld Hkv=%lld", who, (long long)H, (long long)Hkv);
  if (R < 16 || R > D || R % 16 || S <= 0 || S > INT32_MAX)
    return set_error(BTL_ERR_SHAPE, "%s: %lld rotated dims of %lld (a multiple of 16), %lld positions", who,
                     (long long)R, (long long)D, (long long)S);
  int rc = check_batch(who, B, T, cu_q, kv_len, page_table, max_pages, &a.bt);
  if (rc != BTL_OK) return rc;
  if (pages) {
    rc = check_pages(who, pages, &a.pg);
    if (rc != BTL_OK) return rc;
    if (pages->num_kv_heads != Hkv || pages->head_dim != D)
      return set_error(BTL_ERR_SHAPE, "%s: pages of %lld heads x %lld, the rows have %lld x %lld", who,
                       (long long)pages->num_kv_heads, (long long)pages->head_dim, (long long)Hkv, (long long)D);
    if (!page_table || max_pages <= 0) return set_error(BTL_ERR_NULL, "%s: pages without a page table", who);
    a.fp8 = pages->k_exp != nullptr;
  }
  if (T == 0) return BTL_OK;
  if (!qkv || !rope_cos || !rope_sin || !q_out || !error_word) return set_error(BTL_ERR_NULL, "%s: NULL pointer", who);
  if (ldx < (H + 2 * Hkv) * D || ldq < H * D || (k_out && ldk < Hkv * D))
    return set_error(BTL_ERR_SHAPE, "%s: row stride smaller than a row", who);
  if (!aligned(qkv, 16) || !aligned(q_out, 16) || !aligned(k_out, 16) || !aligned(rope_cos, 16) ||
      !aligned(rope_sin, 16) || !aligned(error_word, 4) || ldx % 8 || ldq % 8 || ldk % 8)
    return set_error(BTL_ERR_ALIGN, "%s: misaligned buffer or row stride", who);
  a.qkv = qkv;
  a.ldx = ldx;
  a.H = (int)H;
  a.Hkv = (int)Hkv;
  a.R = (int)R;
  a.S = (int)S;
  a.adjacent = rope_adjacent ? 1 : 0;
  a.rcos = rope_cos;
  a.rsin = rope_sin;
  a.q = q_out;
  a.ldq = ldq;
  a.ko = k_out;
  a.ldk = ldk;
  a.error = error_word;
  a.heads = fast_div((uint32_t)(H + 2 * Hkv));
  a.tokens = T <= 1024 ? 1 : kRopeTokens;
  const dim3 grid((unsigned)((T + a.tokens - 1) / a.tokens));
  if (D == 128)
    hipLaunchKernelGGL(k_rope_write<128>, grid, dim3(kRopeThreads), 0, (hipStream_t)stream, a);
  else
    hipLaunchKernelGGL(k_rope_write<64>, grid, dim3(kRopeThreads), 0, (hipStream_t)stream, a);
  return check_launch("rope write");
}

int btl_read_pages(const btl_pages_t* pages, const int32_t* page_table, int64_t B, int64_t max_pages,
                   const int32_t* kv_len, int64_t S, uint16_t* k, uint16_t* v, int32_t* error_word,
                   btl_stream_t stream) {
  const char* who = "btl_read_pages";
  clear_error();
  ReadArgs a{};
  int rc = check_pages(who, pages, &a.pg);
  if (rc != BTL_OK) return rc;
  rc = check_batch(who, B, 0, nullptr, kv_len, page_table, max_pages, &a.bt);
  if (rc != BTL_OK) return rc;
  // no row behind the page table's room is ever read
  const int64_t room = max_pages * pages->page_size, rows = S < room ? S : room, each = read_rows((int)pages->head_dim);
  if (S <= 0 || S > INT32_MAX - 64 || rows > (1 << 27) || B > 65535 || max_pages <= 0)
    return set_error(BTL_ERR_SHAPE, "%s: B=%lld S=%lld max_pages=%lld", who, (long long)B, (long long)S,
                     (long long)max_pages);
  if (!page_table || !kv_len || !k || !v || !error_word) return set_error(BTL_ERR_NULL, "%s: NULL pointer", who);
  if (!aligned(k, 16) || !aligned(v, 16) || !aligned(error_word, 4))
    return set_error(BTL_ERR_ALIGN, "%s: misaligned buffer", who);
  a.fp8 = pages->k_exp != nullptr;
  a.S = (int)S;
  a.k = k;
  a.v = v;
  a.error = error_word;
  const dim3 grid((unsigned)((rows + each - 1) / each), (unsigned)pages->num_kv_heads, (unsigned)B);
  auto* kern = pages->head_dim == 128 ? (a.fp8 ? k_read_pages<128, true> : k_read_pages<128, false>)
                                      : (a.fp8 ? k_read_pages<64, true> : k_read_pages<64, false>);
  hipLaunchKernelGGL(kern, grid, dim3(256), 0, (hipStream_t)stream, a);
  return check_launch("read pages");
}

}  // extern "C"
