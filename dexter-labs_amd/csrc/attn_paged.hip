// Attention over pages of a KV cache: the plan and the C entry points (the
// kernels: attn_paged_kernels.h).
#include "attn_paged.h"

#include <algorithm>
#include <cmath>

namespace dx {
namespace {

// Rows of 32 to a wave, one or four waves of them. Four single-wave streams for up to
// 32 rows: 30.4 and 32.3 us against 33.0 and 34.9 with one stream (4 x 16 and 4 x 32 queries
// of 24 heads over 300 to 3,000 rows; 64 decoded tokens over 0 to 100 rows 19.4 against
// 21.9; alike where memory bounds it, 32 tokens of 8 K/V heads over 300 to 3,000). For 40
// and 64 rows, two items of one wave read the keys twice: 46.8 and 47.2 against 33.9 and 36.6.
int row_waves(int64_t rows) { return rows <= 32 ? 1 : 4; }

// Own keys of one row tile per sequence and head, 16-bit, no prefix: up to this many
// 32-key tiles the items are not cut, and there is nothing to join. Cut or whole, us,
// over 0 to so many tiles, bf16, D 128:
//                               8            16           32           48           64
//   4 tokens, 8 K/V heads    15.8/ 9.2    15.2/11.8    16.4/16.9    16.6/21.6    16.2/25.7
//   64 tokens                22.8/14.3    30.5/24.8    40.7/35.6    54.1/47.6    64.0/61.0
//   256 tokens               53.8/44.5    69.2/61.8     114/105      159/151      206/202
//   4 x 83, 24 heads         21.6/15.6    24.6/22.2    25.7/33.3    27.2/42.9    30.3/55.8
//   16 x 83                  34.1/22.0    39.6/30.4    50.1/44.2    58.1/57.4    70.2/73.3
// Longer ragged ones leave workgroups idle (128 tokens over 300 to 3,000 rows: 169/179).
// D 256 runs half as many workgroups, each twice as long: 16 x 83 74.9/64.8 at 16 tiles, but
// 256 tokens 201/212 at 32, 16 x 83 160/175 at 64. In fp32 a tile takes four times as long:
// 4 x 99 over 16 tiles 45.8/79.5.
int64_t whole_tiles(int64_t items, int64_t D, int64_t slots) {
  return D > 128 ? 16 : std::min<int64_t>(64, std::max<int64_t>(16, 64 * items / slots));
}

// Key ranges per item of a split line: `tiles` per item, rounds of `slots`
// workgroups, each with the cost of some tiles for its start and end, and the join. The
// smallest of the counts that are within 2% of the best. 16 x 83 rows of 24 heads over
// 8,217 shared ones: 3, 5 and 7 ranges take 220, 212 and 218 us (it says 5). 1, 2 and 3
// ranges under a causal mask over 400 to 1,000 cached rows: 2 x 1,500 queries, 16 heads of
// 8, 80, 92 and 92 us (it says 1), half of them 60, 50 and 49 (2).
int range_count(int64_t items, int64_t tiles, int64_t slots) {
  auto cost = [&](int64_t s) {
    const int64_t rounds = (items * s + slots - 1) / slots;
    return double(rounds) * (double((tiles + s - 1) / s) + 8) + (s > 1 ? 8 : 0);
  };
  double best = cost(1);
  const int64_t most = std::min<int64_t>(64, std::max<int64_t>(1, tiles / 8));
  for (int64_t s = 2; s <= most; ++s) best = std::min(best, cost(s));
  int s = 1;
  while (cost(s) > 1.02 * best) ++s;
  return s;
}

PagedPlan plan_paged(int64_t B, int64_t Lq, int64_t Lk, int64_t H, int64_t Hkv, int64_t D,
                     int64_t dtype, int64_t own_rows, int64_t pre_rows, bool prefix, int cus) {
  PagedPlan p{};
  const int64_t R = Lq * (H / Hkv);
  auto row_tiles = [](int64_t rows, int rw) { return (rows + 32 * rw - 1) / (32 * rw); };
  auto tiles = [](int64_t rows) { return (rows + kPN - 1) / kPN; };
  p.rw_own = row_waves(R);
  p.own_items = B * Hkv * row_tiles(R, p.rw_own);
  const int64_t own_tiles = tiles(own_rows) + std::max<int64_t>(tiles(Lk), 1);
  p.own_work = p.own_items * (own_tiles + kMaxItemCost);
  int64_t pre_tiles = 0;
  if (prefix) {
    p.rw_pre = row_waves(B * R);
    p.pre_items = Hkv * row_tiles(B * R, p.rw_pre);
    pre_tiles = std::max<int64_t>(tiles(pre_rows), 1);
    p.pre_work = p.pre_items * (pre_tiles + kMaxItemCost);
  }
  // Workgroups that run at once. Lines of more than one row tile per sequence and head are
  // never cut (range_count is at least 1): the kernel's cut lines rely on it.
  const int64_t slots = (D == 256 ? 1 : 2) * int64_t(cus);
  if (prefix && row_tiles(B * R, p.rw_pre) > 1) p.pre_splits = range_count(p.pre_items, pre_tiles, slots);
  const bool halves = dtype != DX_F32;
  if (row_tiles(R, p.rw_own) > 1 || (B == 1 && halves && !prefix))
    p.own_splits = range_count(p.own_items, own_tiles, slots);
  else if (halves && !prefix && own_tiles <= whole_tiles(p.own_items, D, slots) &&
           grid_fits(p.own_items, kPagedThreads))
    p.own_splits = 1;
  // A cut line: no more of them than it has tiles and items.
  p.own_n = p.own_splits ? p.own_items * p.own_splits : std::min(slots, p.own_items * (own_tiles + 1));
  const int64_t pre_n = p.pre_splits ? p.pre_items * p.pre_splits
                                     : std::min(slots, p.pre_items * (pre_tiles + 1));
  p.grid = p.own_n;
  if (prefix) {
    p.grid = p.own_splits || p.pre_splits ? p.own_n + pre_n
                                          : std::max<int64_t>(2, std::min(slots, p.own_n + pre_n));
    p.own_slots = p.own_splits ? p.own_n : p.own_items + p.grid;
    p.pre_slots = p.pre_splits ? pre_n : p.pre_items + p.grid;
    p.own_recs = p.own_items;
    p.pre_recs = p.pre_items;
    p.merge = true;
  } else if (p.own_splits) {
    p.merge = p.own_splits > 1;
    p.own_slots = p.merge ? p.own_n : 0;
    p.own_recs = p.merge ? p.own_items : 0;
  } else {
    p.merge = true;
    p.own_slots = 2 * p.grid;
    p.own_recs = std::min(p.grid, p.own_items);
  }
  return p;
}

// two: partials have a second sum (log-sum-exps in 16 bits).
int64_t slot_bytes(int rw, int64_t D, bool two) { return 32 * int64_t(rw) * (D * 4 + (two ? 12 : 8)); }
int64_t plan_bytes(const PagedPlan& p, int64_t D, bool two) {
  return p.own_slots * slot_bytes(p.rw_own, D, two) + p.pre_slots * slot_bytes(p.rw_pre, D, two) +
         (p.own_recs + p.pre_recs) * int64_t(sizeof(Record));
}

constexpr int64_t kMaxRows = int64_t(1) << 30;  // rows of a sequence or prefix, and keys

// Sizes that the kernels' 32-bit arithmetic and one launch hold.
int check_sizes(const char* what, int64_t B, int64_t Lq, int64_t Lk, int64_t H, int64_t Hkv,
                int64_t D, int64_t dtype, int64_t page_rows, int64_t width, int64_t prefix_width) {
  DX_CHECK_ARG(dtype == DX_BF16 || dtype == DX_F16 || dtype == DX_F32,
               "%s: dtype code %lld unsupported", what, (long long)dtype);
  DX_CHECK_ARG(D == 64 || D == 128 || (D == 256 && dtype != DX_F32),
               "%s: head_dim %lld (supported: 64, 128, and 256 in 16 bits)", what, (long long)D);
  DX_CHECK_ARG(B >= 0 && Lq >= 0 && Lk >= 0 && H > 0 && Hkv > 0 && width >= 0 && prefix_width >= 0,
               "%s: bad shape", what);
  DX_CHECK_ARG(H % Hkv == 0, "%s: %lld query heads are not a multiple of %lld k/v heads", what,
               (long long)H, (long long)Hkv);
  DX_CHECK_ARG(page_rows > 0 && page_rows % 16 == 0 && page_rows <= 1024,
               "%s: pages of %lld rows (supported: multiples of 16 up to 1024)", what,
               (long long)page_rows);
  DX_CHECK_ARG(Lq < kMaxRows && Lk < kMaxRows && width < kMaxRows / page_rows &&
                   prefix_width < kMaxRows / page_rows && H < kMaxRows && B < kMaxRows,
               "%s: sequences must hold fewer than 2^30 rows", what);
  const int64_t group = H / Hkv;
  DX_CHECK_ARG(B == 0 || Lq == 0 || (group < kMaxRows / Lq && Lq * group < kMaxRows / B),
               "%s: %lld x %lld queries of %lld heads exceed one launch", what, (long long)B,
               (long long)Lq, (long long)group);
  return DX_OK;
}

// What a call reads and writes besides: the queries' log-sum-exps, cached rows in 4 bits.
struct Form {
  bool prefix, fp4, with_lse;
  void* lse;
};

int paged_entry(const char* what, const dx_paged_call* call, Form form) {
  const bool prefix = form.prefix;
  DX_CHECK_ARG(call, "%s: null call", what);
  dx_paged_call c = *call;
  DX_CHECK_ARG(!form.fp4 || c.dtype == DX_BF16 || c.dtype == DX_F16,
               "%s: dtype code %lld unsupported (a 4-bit cache serves bf16 and f16)", what,
               (long long)c.dtype);
  if (!prefix) {
    c.prefix_table = c.prefix_len = nullptr;
    c.prefix_width = 0;
  }
  const int bad = check_sizes(what, c.B, c.Lq, c.Lk, c.H, c.Hkv, c.D, c.dtype, c.page_rows, c.width,
                              c.prefix_width);
  if (bad) return bad;
  DX_CHECK_ARG(c.n_pages >= 0 && c.n_pages < (int64_t(1) << 31), "%s: bad page count", what);
  DX_CHECK_ARG(c.n_blocks >= 0 && c.n_blocks < kMaxRows &&
                   (c.starts_dtype == DX_I32 || c.starts_dtype == DX_I64),
               "%s: bad block starts", what);
  DX_CHECK_ARG(c.n_blocks == 0 || c.block_starts, "%s: null block starts", what);
  DX_CHECK_ARG(c.Lk == c.Lq || (!c.causal && c.n_blocks == 0),
               "%s: k/v length %lld must equal q length %lld with block starts or causal", what,
               (long long)c.Lk, (long long)c.Lq);
  const float scale_log2 = float(c.softmax_scale * 1.4426950408889634);
  DX_CHECK_ARG(std::isfinite(scale_log2), "%s: softmax scale must be finite", what);
  if (c.B == 0 || c.Lq == 0) return DX_OK;
  const int64_t es = c.dtype == DX_F32 ? 4 : 2, per16 = 16 / es;
  auto al = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; };
  DX_CHECK_ARG(c.q && c.out, "%s: null pointer", what);
  DX_CHECK_ARG(c.Lk == 0 || (c.k && c.v), "%s: null k or v", what);
  DX_CHECK_ARG(c.width == 0 || (c.block_table && c.cache_lens), "%s: null block table or lengths", what);
  DX_CHECK_ARG(!prefix || c.prefix_len, "%s: null prefix length", what);
  DX_CHECK_ARG(c.prefix_width == 0 || c.prefix_table, "%s: null prefix table", what);
  DX_CHECK_ARG(c.n_pages == 0 || c.pages, "%s: null pages", what);
  DX_CHECK_ARG(!form.with_lse || (form.lse && (reinterpret_cast<uintptr_t>(form.lse) & 3u) == 0),
               "%s: null or misaligned lse", what);
  DX_CHECK_ARG(al(c.q) && al(c.k) && al(c.v) && al(c.pages) && al(c.out),
               "%s: pointers must be 16-byte aligned", what);
  // A pool's element size; one in 4 bits is bytes, with its rows where the format has them.
  const int64_t pe = form.fp4 ? 1 : es;
  if (form.fp4) c.p_sr = c.D / 2;
  for (const int64_t s : {c.q_sb, c.q_sl, c.q_sh, c.k_sb, c.k_sl, c.k_sh, c.v_sb, c.v_sl, c.v_sh,
                          c.o_sb, c.o_sl, c.o_sh})
    DX_CHECK_ARG(s % per16 == 0, "%s: strides must keep head rows 16-byte aligned", what);
  for (const int64_t s : {c.p_plane, c.p_sp, c.p_sr, c.p_sh})
    DX_CHECK_ARG(s % (16 / pe) == 0, "%s: strides must keep head rows 16-byte aligned", what);
  // 16 rows of keys lie within one buffer descriptor (below 2^31 bytes).
  for (const int64_t s : {c.p_sr, c.k_sl, c.v_sl})
    DX_CHECK_ARG(s >= 0 && s * es < (int64_t(1) << 26), "%s: row stride %lld out of range", what,
                 (long long)s);

  const PagedPlan p = plan_paged(c.B, c.Lq, c.Lk, c.H, c.Hkv, c.D, c.dtype, c.width * c.page_rows,
                                 c.prefix_width * c.page_rows, prefix, device_cus());
  const bool two = form.with_lse && c.dtype != DX_F32;
  const int64_t need = plan_bytes(p, c.D, two);
  if (need > c.workspace_bytes || (need > 0 && !c.workspace)) {
    set_error("%s: workspace of %lld bytes, %lld needed", what, (long long)(c.workspace ? c.workspace_bytes : 0),
              (long long)need);
    return DX_EWORKSPACE;
  }
  DX_CHECK_ARG(al(c.workspace), "%s: workspace must be 16-byte aligned", what);
  const int64_t group = c.H / c.Hkv, R = c.Lq * group;
  // Item numbers and slots are 32-bit; the merge takes a workgroup per item.
  // Lines are counted in 32 bits.
  DX_CHECK_ARG(p.own_work < (int64_t(1) << 31) && p.pre_work < (int64_t(1) << 31),
               "%s: too many queries and keys for one launch", what);
  DX_CHECK_ARG((p.own_splits || p.own_items == c.B * c.Hkv) &&
                   (!prefix || p.pre_splits || p.pre_items == c.Hkv),
               "%s: a line of several row tiles was to be cut", what);
  DX_CHECK_ARG(grid_fits(p.own_recs, 256) && grid_fits(p.grid, kPagedThreads) && p.own_items < (int64_t(1) << 30) &&
                   p.pre_items < (int64_t(1) << 30),
               "%s: the call exceeds one launch", what);
  PagedArgs a{};
  a.q = static_cast<const char*>(c.q); a.q_sb = c.q_sb * es; a.q_sl = c.q_sl * es; a.q_sh = c.q_sh * es;
  a.k = static_cast<const char*>(c.k); a.k_sb = c.k_sb * es; a.k_sl = c.k_sl * es; a.k_sh = c.k_sh * es;
  a.v = static_cast<const char*>(c.v); a.v_sb = c.v_sb * es; a.v_sl = c.v_sl * es; a.v_sh = c.v_sh * es;
  a.pk = static_cast<const char*>(c.pages); a.pv = a.pk + c.p_plane * pe;
  a.p_sp = c.p_sp * pe; a.p_sr = c.p_sr * pe; a.p_sh = c.p_sh * pe;
  a.lse = static_cast<float*>(form.lse);
  a.out = static_cast<char*>(c.out); a.o_sb = c.o_sb * es; a.o_sl = c.o_sl * es; a.o_sh = c.o_sh * es;
  a.table = static_cast<const int32_t*>(c.block_table); a.t_sb = c.t_sb;
  a.lens = static_cast<const int32_t*>(c.cache_lens);
  a.ptable = static_cast<const int32_t*>(c.prefix_table);
  a.plen = prefix ? static_cast<const int32_t*>(c.prefix_len) : nullptr;
  a.width = int(c.width); a.pwidth = int(c.prefix_width);
  a.n_pages = int(c.n_pages); a.page_rows = int(c.page_rows);
  const uint64_t per = uint64_t(c.page_rows / 16);
  a.page_magic = per == 1 ? 0u : uint32_t(((uint64_t(1) << 32) + per - 1) / per);
  a.starts = c.block_starts; a.starts_i64 = c.starts_dtype == DX_I64; a.n_blocks = int(c.n_blocks);
  a.B = int(c.B); a.H = int(c.H); a.Hkv = int(c.Hkv); a.group = int(group);
  a.Lq = int(c.Lq); a.Lk = int(c.Lk); a.causal = c.causal != 0;
  a.R = int(R);
  a.scale_log2 = scale_log2;
  a.own.splits = p.own_splits;
  a.own.by_item = p.own_recs == p.own_items;  // no records: nothing is left to join
  a.pre.by_item = p.pre_recs > 0;
  a.pre.splits = p.pre_splits;
  a.own_n = int(p.own_n);
  char* ws = static_cast<char*>(c.workspace);
  auto take = [&](int64_t bytes) {
    char* const at = ws;
    ws += bytes;
    return at;
  };
  a.own.o = reinterpret_cast<float*>(take(p.own_slots * 32 * p.rw_own * c.D * 4));
  a.pre.o = reinterpret_cast<float*>(take(p.pre_slots * 32 * p.rw_pre * c.D * 4));
  a.own.ml = reinterpret_cast<float*>(take(p.own_slots * 32 * p.rw_own * (two ? 12 : 8)));
  a.pre.ml = reinterpret_cast<float*>(take(p.pre_slots * 32 * p.rw_pre * (two ? 12 : 8)));
  a.own.rec = reinterpret_cast<Record*>(take(p.own_recs * int64_t(sizeof(Record))));
  a.pre.rec = reinterpret_cast<Record*>(take(p.pre_recs * int64_t(sizeof(Record))));
  const hipStream_t st = static_cast<hipStream_t>(c.stream);
  const int D = int(c.D);
  const bool bf16 = c.dtype == DX_BF16;
  hipError_t e;
  if (form.fp4 && form.with_lse)
    e = bf16 ? launch_paged_bf16_fp4_lse(a, p, D, st) : launch_paged_f16_fp4_lse(a, p, D, st);
  else if (form.fp4)
    e = bf16 ? launch_paged_bf16_fp4(a, p, D, st) : launch_paged_f16_fp4(a, p, D, st);
  else if (form.with_lse)
    e = c.dtype == DX_F32 ? launch_paged_f32_lse(a, p, D, st)
        : bf16            ? launch_paged_bf16_lse(a, p, D, st)
                          : launch_paged_f16_lse(a, p, D, st);
  else
    e = c.dtype == DX_F32 ? launch_paged_f32(a, p, D, st)
        : bf16            ? launch_paged_bf16(a, p, D, st)
                          : launch_paged_f16(a, p, D, st);
  if (e != hipSuccess) {
    set_error("%s: launch failed: %s", what, hipGetErrorString(e));
    return DX_ELAUNCH;
  }
  return DX_OK;
}

}  // namespace
}  // namespace dx

using namespace dx;

namespace {
int64_t workspace_bytes(int dtype, int64_t B, int64_t Lq, int64_t Lk, int64_t H, int64_t Hkv, int64_t D,
                        int64_t page_rows, int64_t width, int has_prefix, int64_t prefix_width, bool lse) {
  const int bad = check_sizes("paged_attention", B, Lq, Lk, H, Hkv, D, dtype, page_rows, width,
                              prefix_width);
  if (bad) return -bad;
  if (B == 0 || Lq == 0) return 0;
  const PagedPlan p = plan_paged(B, Lq, Lk, H, Hkv, D, dtype, width * page_rows,
                                 prefix_width * page_rows, has_prefix != 0, device_cus());
  return plan_bytes(p, D, lse && dtype != DX_F32);
}
}  // namespace

extern "C" int64_t dx_paged_attention_workspace_bytes(int dtype, int64_t B, int64_t Lq, int64_t Lk,
                                                      int64_t H, int64_t Hkv, int64_t D,
                                                      int64_t page_rows, int64_t width,
                                                      int has_prefix, int64_t prefix_width) {
  return workspace_bytes(dtype, B, Lq, Lk, H, Hkv, D, page_rows, width, has_prefix, prefix_width, false);
}

extern "C" int64_t dx_paged_attention_lse_workspace_bytes(int dtype, int64_t B, int64_t Lq, int64_t Lk,
                                                          int64_t H, int64_t Hkv, int64_t D,
                                                          int64_t page_rows, int64_t width,
                                                          int has_prefix, int64_t prefix_width) {
  return workspace_bytes(dtype, B, Lq, Lk, H, Hkv, D, page_rows, width, has_prefix, prefix_width, true);
}

extern "C" int dx_paged_attention(const dx_paged_call* call) {
  return paged_entry("paged_attention", call, {false, false, false, nullptr});
}

extern "C" int dx_shared_prefix_attention(const dx_paged_call* call) {
  return paged_entry("shared_prefix_attention", call, {true, false, false, nullptr});
}

extern "C" int dx_paged_attention_lse(const dx_paged_call* call, void* lse) {
  return paged_entry("paged_attention", call, {false, false, true, lse});
}

extern "C" int dx_shared_prefix_attention_lse(const dx_paged_call* call, void* lse) {
  return paged_entry("shared_prefix_attention", call, {true, false, true, lse});
}

extern "C" int dx_paged_attention_fp4(const dx_paged_call* call, void* lse) {
  return paged_entry("paged_attention_fp4", call, {false, true, lse != nullptr, lse});
}

extern "C" int dx_shared_prefix_attention_fp4(const dx_paged_call* call, void* lse) {
  return paged_entry("shared_prefix_attention_fp4", call, {true, true, lse != nullptr, lse});
}
