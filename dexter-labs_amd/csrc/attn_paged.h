// Launch arguments, plan and launchers of attention over pages: shared by the
// entry points (attn_paged.hip) and the kernels (attn_paged_kernels.h), which are
// compiled once per element type (attn_paged_bf16.hip, _f16.hip, _f32.hip).
#pragma once

#include "attn_common.h"

namespace dx {

constexpr int kPN = 32;  // keys per tile of the line
constexpr int kPagedThreads = 256;

// Where an item's parts are: slot of the first, and their number (one after the
// other; 0: none, its result is written). By item; or, where a cut line without
// a prefix has more items than workgroups, by workgroup: the item it leaves broken.
struct Record { int item, slot, parts, pad; };

// A line of work: its partials and records.
struct Line {
  float* o;     // [slot][32 RW rows][D]: unnormalised sums
  float* ml;    // [slot][32 RW rows]: {m, l}
  Record* rec;
  int splits;   // key ranges per item; 0: the line is cut into pieces
  int by_item;  // the records are, and there are some
};

struct PagedArgs {
  const char* q; int64_t q_sb, q_sl, q_sh;  // strides in bytes, here and below
  const char* k; int64_t k_sb, k_sl, k_sh;
  const char* v; int64_t v_sb, v_sl, v_sh;
  const char* pk; const char* pv; int64_t p_sp, p_sr, p_sh;
  char* out; int64_t o_sb, o_sl, o_sh;
  const int32_t* table; int64_t t_sb; const int32_t* lens;  // own cached rows
  const int32_t* ptable; const int32_t* plen;               // the prefix (null: none)
  int width, pwidth;            // table entries per sequence, of the prefix
  int n_pages, page_rows;
  uint32_t page_magic;          // ceil(2^32 / (page_rows / 16)); 0: pages of 16 rows
  const void* starts; int starts_i64, n_blocks;
  int B, H, Hkv, group, Lq, Lk, causal;
  int R;                        // rows of a (sequence, K/V head): Lq * group
  float scale_log2;             // signed
  int own_n;                    // workgroups for the own line at most, where it alone is cut
  Line own, pre;
};

constexpr int64_t kMaxItemCost = 16;  // kItemCost at most

struct PagedPlan {
  int rw_own, rw_pre;            // row waves of a workgroup; rw_pre 0: no prefix
  int own_splits, pre_splits;    // 0: the line is cut
  int64_t own_items, pre_items;
  int64_t own_work, pre_work;    // lengths of the lines at most, at the largest row counts
  int64_t own_n, grid;           // workgroups
  int64_t own_slots, pre_slots;  // partials of 32 rw rows
  int64_t own_recs, pre_recs;
  bool merge;
};

// Launch the plan (head dims: attn_paged.hip's checks).
hipError_t launch_paged_bf16(const PagedArgs& a, const PagedPlan& p, int D, hipStream_t st);
hipError_t launch_paged_f16(const PagedArgs& a, const PagedPlan& p, int D, hipStream_t st);
hipError_t launch_paged_f32(const PagedArgs& a, const PagedPlan& p, int D, hipStream_t st);

}  // namespace dx
