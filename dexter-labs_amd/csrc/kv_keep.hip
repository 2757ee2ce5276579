// Which rows of a cache to keep by the weight they received, and moving them, on gfx950.
//
// kv_keep_rows. Of a sequence's n rows, per K/V head: c = min(n, keep) are kept, the last
// min(recent, c) of them always, and of the m rows before those the k = c - min(recent, c)
// with the largest weights; ties go to the lowest row, NaN counts as the lowest weight. The
// k-th largest is found digit by digit: weights as integers of the same order, largest
// first, a histogram of 11, 11, then 10 bits of those that agree with the digits found
// before. One more pass counts per wave what lies above it and at it, a last one writes the
// rows in order. One workgroup per (sequence, head): five passes over 4 n bytes, which
// stay in its XCD's L2 (128 KB of 32,768 rows); latency bounds it, each pass a round trip.
//
// kv_page_gather. Row i of a head becomes row rows[i], which is i at least and ascending in
// i. A workgroup moves a column of the rows of one (sequence, head, plane), kRows rows at a
// time and in order: all loads of a step are done (a barrier) before its first store, and
// what later steps read lies behind the rows that this one writes. So it may run in place,
// on the pages it reads. Bound by memory: kept rows are read and written once.
#include "kv_fp4.h"

#include <algorithm>

namespace dx {
namespace {

constexpr int kKeepThreads = 1024, kKeepWaves = kKeepThreads / 64;
constexpr int kBits = 11, kBins = 1 << kBits;

struct KeepArgs {
  const float* w; int64_t w_sb, w_sh;
  const int32_t* lens;
  int32_t* rows;  // [B, H, keep]
  int H, width, keep, recent;
};

// Unsigned integers in the weights' order, -0 as 0, NaN as the lowest.
__device__ __forceinline__ uint32_t rank_of(float x) {
  const uint32_t u = __float_as_uint(x);
  if ((u & 0x7fffffffu) > 0x7f800000u) return 0x007fffffu;  // that of -inf
  if (u == 0x80000000u) return 0x80000000u;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__global__ __launch_bounds__(kKeepThreads) void kv_keep_rows_kernel(KeepArgs a) {
  __shared__ uint32_t hist[kBins];
  __shared__ uint32_t found[2];               // digit, how many are left to find among its rows
  __shared__ uint32_t above[kKeepWaves], at[kKeepWaves];
  const int tid = int(threadIdx.x), lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int bh = int(blockIdx.x), b = bh / a.H, h = bh - b * a.H;
  const float* const w = a.w + b * a.w_sb + h * a.w_sh;
  int32_t* const out = a.rows + int64_t(bh) * a.keep;
  const int n = min(max(a.lens[b], 0), a.width);
  const int c = min(n, a.keep), last = min(a.recent, c), m = n - last;
  const uint32_t k = uint32_t(c - last);
  for (int i = c + tid; i < a.keep; i += kKeepThreads) out[i] = -1;
  for (int i = tid; i < last; i += kKeepThreads) out[int(k) + i] = m + i;
  if (k == 0) return;
  if (int(k) == m) {
    for (int i = tid; i < m; i += kKeepThreads) out[i] = i;
    return;
  }

  // The k-th largest: `prefix` are its bits found so far, `want` its place among those.
  uint32_t prefix = 0, mask = 0, want = k;
#pragma unroll 1
  for (int shift = 21; ; shift = shift == 21 ? 10 : 0) {
    const int bits = shift ? kBits : 10;
    for (int i = tid; i < kBins; i += kKeepThreads) hist[i] = 0;
    __syncthreads();
    for (int i = tid; i < m; i += kKeepThreads) {
      const uint32_t x = rank_of(w[i]);
      if ((x & mask) == prefix) atomicAdd(&hist[(x >> shift) & ((1u << bits) - 1)], 1u);
    }
    __syncthreads();
    // From the largest digit down: the first whose rows and all above reach `want`. A
    // wave takes it, 32 bins to a lane.
    if (wave == 0) {
      constexpr int per = kBins / 64;
      const int top = kBins - 1 - lane * per;  // this lane's bins: top, top - 1, ...
      uint32_t mine = 0;
      for (int j = 0; j < per; ++j) mine += hist[top - j];
      uint32_t upto = mine;
#pragma unroll
      for (int d = 1; d < 64; d *= 2) {
        const uint32_t y = __shfl_up(upto, d);
        if (lane >= d) upto += y;
      }
      const uint64_t hit = __ballot(upto >= want);
      if (lane == __builtin_ctzll(hit)) {
        uint32_t before = upto - mine;
        int j = 0;
        while (before + hist[top - j] < want) before += hist[top - j++];
        found[0] = uint32_t(top - j);
        found[1] = want - before;
      }
    }
    __syncthreads();
    prefix |= found[0] << shift;
    mask |= ((1u << bits) - 1) << shift;
    want = found[1];
    if (shift == 0) break;
  }

  // Rows above it, and the first `want` of those at it. A wave takes a run of rows.
  const int run = (m + kKeepThreads - 1) / kKeepThreads * 64;
  const int from = min(wave * run, m), to = min(from + run, m);
  uint32_t n_above = 0, n_at = 0;
  for (int i = from; i < to; i += 64) {
    const uint32_t x = i + lane < to ? rank_of(w[i + lane]) : 0u;
    n_above += uint32_t(__popcll(__ballot(x > prefix)));
    n_at += uint32_t(__popcll(__ballot(i + lane < to && x == prefix)));
  }
  if (lane == 0) {
    above[wave] = n_above;
    at[wave] = n_at;
  }
  __syncthreads();
  uint32_t pos = 0, seen = 0;  // kept and met at it before this wave's run
  for (int i = 0; i < wave; ++i) {
    pos += above[i];
    seen += at[i];
  }
  pos += min(seen, want);
  const uint64_t below = (uint64_t(1) << lane) - 1;
  for (int i = from; i < to; i += 64) {
    const uint32_t x = i + lane < to ? rank_of(w[i + lane]) : 0u;
    const uint64_t same = __ballot(i + lane < to && x == prefix);
    const bool take = x > prefix || (same >> lane & 1 && seen + uint32_t(__popcll(same & below)) < want);
    const uint64_t taken = __ballot(take);
    if (take) out[pos + uint32_t(__popcll(taken & below))] = i + lane;
    pos += uint32_t(__popcll(taken));
    seen += uint32_t(__popcll(same));
  }
}

constexpr int kGatherThreads = 256, kChunks = 8;  // 16-byte chunks of a thread in a step

struct GatherArgs {
  char* pages; int64_t p_plane, p_sp, p_sr, p_sh;  // bytes
  const int32_t* src; int64_t s_sb;
  const int32_t* dst; int64_t d_sb;
  const int32_t* rows;             // [B, H, keep]
  float* w; int64_t w_sb, w_sh;    // null: none
  int H, keep, width, dst_width, n_pages, page_rows, w_width;
  int chunks, slice;               // 16-byte chunks of a row; of a workgroup's column (a power of two)
  int slices;                      // columns of a plane; a 4-bit one's last holds its scales
  int tail;                        // scale bytes of a row (0: a 16- or 32-bit pool)
};

// Where row r of a table's pages lies: the page, or none.
__device__ __forceinline__ int page_at(const int32_t* table, int r, int rows, int width, int n_pages) {
  if (uint32_t(r) >= uint32_t(width) * uint32_t(rows)) return -1;
  const int page = table[r / rows];
  return uint32_t(page) < uint32_t(n_pages) ? page : -1;
}

// One step after the other: UNIT bytes of a row to a lane at a time.
template <typename U, int N>
__device__ __forceinline__ void move_column(const GatherArgs& a, char* plane, const int32_t* rows,
                                            const int32_t* src, const int32_t* dst, int64_t head,
                                            int64_t first, int64_t row_bytes, int per, int units) {
  // `units` a row in this column; `per` (a power of two, units at least) lanes to a row.
  const int step = N * kGatherThreads / per;
  const int lr = int(threadIdx.x) / per, lu = int(threadIdx.x) % per;
#pragma unroll 1
  for (int i0 = 0; i0 < a.keep; i0 += step) {
    U x[N];
    char* to[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int i = i0 + j * (kGatherThreads / per) + lr;
      to[j] = nullptr;
      if (i >= a.keep || lu >= units) continue;
      const int r = rows[i];
      if (r < 0) continue;
      const int from = page_at(src, r, a.page_rows, a.width, a.n_pages);
      const int into = page_at(dst, i, a.page_rows, a.dst_width, a.n_pages);
      if (from < 0 || into < 0) continue;
      const char* const p = plane + from * a.p_sp + head + first + (r % a.page_rows) * row_bytes + lu * int(sizeof(U));
      char* const q = plane + into * a.p_sp + head + first + (i % a.page_rows) * row_bytes + lu * int(sizeof(U));
      if (p == q) continue;  // (another sequence may read it)
      x[j] = *reinterpret_cast<const U*>(p);
      to[j] = q;
    }
    wait_vmcnt<0>();  // every load of this wave has returned,
    __syncthreads();  // and of the others
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (to[j]) *reinterpret_cast<U*>(to[j]) = x[j];
  }
}

__global__ __launch_bounds__(kGatherThreads) void kv_page_gather_kernel(GatherArgs a) {
  const int bh = int(blockIdx.y), b = bh / a.H, h = bh - b * a.H;
  const int32_t* const rows = a.rows + int64_t(bh) * a.keep;
  int col = int(blockIdx.x);
  if (col == 2 * a.slices) {  // the weights: kept ones to the front, 0 behind
    float* const w = a.w + b * a.w_sb + h * a.w_sh;
#pragma unroll 1
    for (int i0 = 0; i0 < a.w_width; i0 += 4 * kGatherThreads) {
      float x[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = i0 + j * kGatherThreads + int(threadIdx.x);
        const int r = i < a.keep ? rows[i] : -1;
        x[j] = uint32_t(r) < uint32_t(a.w_width) ? w[r] : 0.f;
      }
      wait_vmcnt<0>();
      __syncthreads();
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = i0 + j * kGatherThreads + int(threadIdx.x);
        if (i < a.w_width) w[i] = x[j];
      }
    }
    return;
  }
  char* const plane = a.pages + (col >= a.slices ? a.p_plane : 0);
  col = col >= a.slices ? col - a.slices : col;
  const int32_t* const src = a.src + b * a.s_sb;
  const int32_t* const dst = a.dst + b * a.d_sb;
  const int64_t head = h * a.p_sh;
  if (a.tail && col == a.slices - 1) {
    // Scales, 2 bytes at a time (a row has 2, 4 or 8), behind the page's codes.
    const int units = a.tail / 2;
    move_column<uint16_t, kChunks>(a, plane, rows, src, dst, head, int64_t(a.page_rows) * a.p_sr, a.tail, units, units);
  } else {
    move_column<u32x4, kChunks>(a, plane, rows, src, dst, head, int64_t(col) * a.slice * 16, a.p_sr, a.slice,
                                min(a.slice, a.chunks - col * a.slice));
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
constexpr int64_t kMax = (int64_t(1) << 31) - 1;
constexpr int64_t kMaxRows = int64_t(1) << 30;

}  // namespace
}  // namespace dx

using namespace dx;

extern "C" int dx_kv_keep_rows(const void* weights, int64_t w_sb, int64_t w_sh, int64_t width,
                               const void* lens, int64_t keep, int64_t recent, void* rows,
                               int64_t B, int64_t H, void* stream) {
  const char* const what = "kv_keep_rows";
  DX_CHECK_ARG(B >= 0 && H > 0 && width >= 0 && keep >= 0 && recent >= 0, "%s: bad shape", what);
  DX_CHECK_ARG(width < kMaxRows && keep < kMaxRows, "%s: fewer than 2^30 rows are taken", what);
  DX_CHECK_ARG(H <= kMax && B <= ((int64_t(1) << 32) / kKeepThreads - 1) / H,
               "%s: %lld sequences of %lld heads exceed one launch", what, (long long)B, (long long)H);
  if (B == 0 || keep == 0) return DX_OK;
  DX_CHECK_ARG(lens && rows && (weights || width == 0), "%s: null pointer", what);
  KeepArgs a{};
  a.w = static_cast<const float*>(weights); a.w_sb = w_sb; a.w_sh = w_sh;
  a.lens = static_cast<const int32_t*>(lens);
  a.rows = static_cast<int32_t*>(rows);
  a.H = int(H); a.width = int(width); a.keep = int(keep);
  a.recent = int(std::min<int64_t>(recent, keep));
  hipLaunchKernelGGL(kv_keep_rows_kernel, dim3(unsigned(B * H)), dim3(kKeepThreads), 0,
                     static_cast<hipStream_t>(stream), a);
  DX_CHECK_LAUNCH(what);
  return DX_OK;
}

extern "C" int dx_kv_page_gather(void* pages, int64_t p_plane, int64_t p_sp, int64_t p_sr, int64_t p_sh,
                                 int dtype, int64_t n_pages, int64_t page_rows, const void* src_table,
                                 int64_t s_sb, int64_t width, const void* dst_table, int64_t d_sb,
                                 int64_t dst_width, const void* rows, int64_t keep, void* weights,
                                 int64_t w_sb, int64_t w_sh, int64_t w_width, int64_t B, int64_t H,
                                 int64_t D, void* stream) {
  const char* const what = "kv_page_gather";
  const bool fp4 = dtype == DX_FP4;
  const int64_t es = dtype == DX_F32 ? 4 : dtype == DX_BF16 || dtype == DX_F16 ? 2 : fp4 ? 1 : 0;
  DX_CHECK_ARG(es != 0, "%s: dtype code %d unsupported", what, dtype);
  DX_CHECK_ARG(B >= 0 && H > 0 && D > 0 && n_pages >= 0 && page_rows > 0 && width >= 0 && dst_width >= 0 &&
                   keep >= 0 && w_width >= 0, "%s: bad shape", what);
  DX_CHECK_ARG(!fp4 || D == 64 || D == 128 || D == 256, "%s: head_dim %lld (4 bits: 64, 128 and 256)", what,
               (long long)D);
  DX_CHECK_ARG(!fp4 || (page_rows % 16 == 0 && page_rows <= 1024),
               "%s: pages of %lld rows (4 bits: multiples of 16 up to 1024)", what, (long long)page_rows);
  DX_CHECK_ARG(D <= 4096 && D * es % 16 == 0, "%s: head_dim must fill 16-byte chunks (4096 elements at most)", what);
  DX_CHECK_ARG(n_pages <= kMax && page_rows < kMaxRows && width < kMaxRows / page_rows &&
                   dst_width < kMaxRows / page_rows && keep < kMaxRows && w_width < kMaxRows,
               "%s: sequences must hold fewer than 2^30 rows", what);
  DX_CHECK_ARG(B < 65536 && H < 65536 && B * H < 65536, "%s: %lld sequences of %lld heads exceed one launch",
               what, (long long)B, (long long)H);
  if (B == 0 || (keep == 0 && !weights)) return DX_OK;
  DX_CHECK_ARG((rows || keep == 0) && (src_table || width == 0) && (dst_table || dst_width == 0),
               "%s: null pointer", what);
  DX_CHECK_ARG(pages || n_pages == 0, "%s: null pages", what);
  DX_CHECK_ARG(aligned16(pages), "%s: pages must be 16-byte aligned", what);
  if (fp4) p_sr = D / 2;
  DX_CHECK_ARG(p_plane * es % 16 == 0 && p_sp * es % 16 == 0 && p_sr * es % 16 == 0 && p_sh * es % 16 == 0,
               "%s: strides must keep head rows 16-byte aligned", what);
  GatherArgs a{};
  a.pages = static_cast<char*>(pages);
  a.p_plane = p_plane * es; a.p_sp = p_sp * es; a.p_sr = p_sr * es; a.p_sh = p_sh * es;
  a.src = static_cast<const int32_t*>(src_table); a.s_sb = s_sb;
  a.dst = static_cast<const int32_t*>(dst_table); a.d_sb = d_sb;
  a.rows = static_cast<const int32_t*>(rows);
  a.w = static_cast<float*>(weights); a.w_sb = w_sb; a.w_sh = w_sh;
  a.H = int(H); a.keep = int(keep); a.width = int(width); a.dst_width = int(dst_width);
  a.n_pages = int(n_pages); a.page_rows = int(page_rows); a.w_width = int(w_width);
  a.chunks = int(fp4 ? D / 32 : D * es / 16);
  a.tail = int(fp4 ? D / 32 : 0);
  // Columns of 4 chunks (64 bytes), of less where a row has less: of one long sequence of
  // few heads there would be too few workgroups otherwise.
  a.slice = std::min(4, a.chunks);
  while (a.slice & (a.slice - 1)) --a.slice;
  a.slices = (a.chunks + a.slice - 1) / a.slice + (fp4 ? 1 : 0);
  hipLaunchKernelGGL(kv_page_gather_kernel, dim3(unsigned(2 * a.slices + (weights ? 1 : 0)), unsigned(B * H)),
                     dim3(kGatherThreads), 0, static_cast<hipStream_t>(stream), a);
  DX_CHECK_LAUNCH(what);
  return DX_OK;
}
