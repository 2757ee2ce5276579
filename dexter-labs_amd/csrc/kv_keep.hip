// Which rows of a cache to keep by the weight they received, and moving them, on gfx950.
//
// kv_keep_rows. Of a sequence's n rows, per K/V head: c = min(n, keep) are kept, the last
// min(recent, c) of them always, and of the m rows before those the k = c - min(recent, c)
// with the largest weights; ties go to the lowest row, NaN counts as the lowest weight. The
// k-th largest is found digit by digit: weights as integers of the same order, largest
// first, a histogram of 11, 11, then 10 bits of those that agree with the digits found
// before, until a digit's rows are wanted all. Then the rows above it and at it are counted per
// wave and written in order. One workgroup per (sequence, head), whose weights stay in
// LDS (up to 32,768 rows): they are read once. (In registers the unrolled passes over 32
// of them are 30 KB of code, which takes longer to fetch than to run.) Bound by one compute
// unit's passes over a head's weights, four steps that wait for each other: 8,192 of 32,768
// rows for 96 heads take 22 us (15.7 MB: 0.7 TB/s; 23.6 with other weights each time), 1,024 of
// 300 to 3,000 for 256 heads 8.7 (9.1). Past 32,768 rows each pass reads the weights again, one load
// at a time: 8,192 of 40,000 for 96 heads 40 us, of 65,536 62, of 131,072 for 24 heads 111.
// A second histogram for odd lanes, to halve what meets in one digit, changed nothing.
//
// kv_page_gather. Row i of a head becomes row rows[i], which is i at least and ascending in
// i. A workgroup moves a column of the rows of one (sequence, head, plane), step by step in
// their order: all loads of a step are done (a barrier) before its first store, and what
// later steps read lies behind the rows that this one writes. So it may run in place, on the
// pages it reads. Bound by memory: kept rows are read and written once; the next step's loads
// are under way while one is stored, and the lookups of 1,024 rows are made at once. 8,192 of
// 32,768 rows of 24 heads (bf16, D 128, in place): 47 us, 4.3 TB/s, when the same rows come again,
// and 77 with others, 2.7; of four such sequences 244 us, 3.3 TB/s; 1,024 of 300 to 3,000 rows of 32
// x 8 heads in 4 bits to new pages: 17 and 22 us.
#include "attn_common.h"
#include "kv_fp4.h"

#include <algorithm>

namespace dx {
namespace {

constexpr int kKeepThreads = 1024, kKeepWaves = kKeepThreads / 64;
constexpr int kBits = 11, kBins = 1 << kBits;
constexpr int kHeld = 32 * kKeepThreads;  // weights in LDS at most: 128 KB

struct KeepArgs {
  const float* w; int64_t w_sb, w_sh;
  const int32_t* lens;
  int32_t* rows;  // [B, H, keep]
  int H, width, keep, recent;
  int held;       // weights that fit in LDS
};

// Unsigned integers in the weights' order, -0 as 0, NaN as the lowest. Never 0.
__device__ __forceinline__ uint32_t rank_of(float x) {
  const uint32_t u = __float_as_uint(x);
  if ((u & 0x7fffffffu) > 0x7f800000u) return 0x007fffffu;  // that of -inf
  if (u == 0x80000000u) return 0x80000000u;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Inclusive sums over a wave: shifts by 1, 2, 4, 8 within rows of 16 lanes, then each
// row's last to the next row, and the first half's to the second.
template <int kCtrl, int kRows>
__device__ __forceinline__ uint32_t scan_add(uint32_t x) {
  return x + uint32_t(__builtin_amdgcn_update_dpp(0, int(x), kCtrl, kRows, 0xf, false));
}
__device__ __forceinline__ uint32_t scan64(uint32_t x) {
  x = scan_add<0x111, 0xf>(x);
  x = scan_add<0x112, 0xf>(x);
  x = scan_add<0x114, 0xf>(x);
  x = scan_add<0x118, 0xf>(x);
  x = scan_add<0x142, 0xa>(x);
  return scan_add<0x143, 0xc>(x);
}

__global__ __launch_bounds__(kKeepThreads) void kv_keep_rows_kernel(KeepArgs a) {
  __shared__ uint32_t hist[kBins];
  __shared__ uint32_t found[3];     // digit, how many are left to find among its rows, its rows
  __shared__ uint32_t above[kKeepWaves], at[kKeepWaves];
  const int tid = int(threadIdx.x), lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int bh = int(blockIdx.x), b = bh / a.H, h = bh - b * a.H;
  const float* const w = a.w + b * a.w_sb + h * a.w_sh;
  int32_t* const out = a.rows + int64_t(bh) * a.keep;
  const int n = __builtin_amdgcn_readfirstlane(min(max(a.lens[b], 0), a.width));
  const int c = min(n, a.keep), last = min(a.recent, c), m = n - last;
  const uint32_t k = uint32_t(c - last);
  for (int i = c + tid; i < a.keep; i += kKeepThreads) out[i] = -1;
  for (int i = tid; i < last; i += kKeepThreads) out[int(k) + i] = m + i;
  if (k == 0) return;
  if (int(k) == m) {
    for (int i = tid; i < m; i += kKeepThreads) out[i] = i;
    return;
  }

  // A wave has a run of `steps` 256 rows, as integers in LDS, 0 past the end (its own, so no
  // barrier), of which a lane has four that lie side by side. Longer sequences than fit are
  // read again each time.
  const int steps = (m + 4 * kKeepThreads - 1) / (4 * kKeepThreads);
  const int from = wave * steps * 256 + 4 * lane;
  extern __shared__ __attribute__((aligned(16))) uint32_t held[];
  const bool hold = 4 * steps * kKeepThreads <= a.held;
  const bool wide = (reinterpret_cast<uintptr_t>(w) & 15u) == 0 && m >= 4;
  // Rows row.. of the sequence, whatever stands there instead past its end.
  auto load = [&](int row) __attribute__((always_inline)) {
    if (wide) return *reinterpret_cast<const f32x4*>(w + min(row, (m & ~3) - 4));
    f32x4 f;
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = w[min(row + j, m - 1)];
    return f;
  };
  auto ranks = [&](f32x4 f, int row) __attribute__((always_inline)) {
    if (wide && row < m && row + 4 > m) {  // the last, that are no four
#pragma unroll
      for (int j = 0; j < 3; ++j) f[j] = w[min(row + j, m - 1)];
    }
    u32x4 x;
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = row + j < m ? rank_of(f[j]) : 0u;
    return x;
  };
  auto each = [&](auto&& fn) __attribute__((always_inline)) {
#pragma unroll 1
    for (int s = 0; s < steps; ++s) {
      const int row = from + 256 * s;
      fn(hold ? *reinterpret_cast<const u32x4*>(held + row) : ranks(load(row), row), row);
    }
  };
  if (hold) {
    constexpr int N = 4;  // loads under way
#pragma unroll 1
    for (int s = 0; s < steps; s += N) {
      f32x4 f[N];
#pragma unroll
      for (int j = 0; j < N; ++j) f[j] = load(from + 256 * (s + j));
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (s + j < steps)
          *reinterpret_cast<u32x4*>(held + from + 256 * (s + j)) = ranks(f[j], from + 256 * (s + j));
    }
  }

  // The k-th largest: `prefix` are its bits found so far, `want` its place among those.
  uint32_t prefix = 0, mask = 0, want = k;
#pragma unroll 1
  for (int shift = 21; ; shift = shift == 21 ? 10 : 0) {
    const uint32_t digits = shift ? kBins - 1 : (1u << 10) - 1;
    for (int i = tid; i < kBins; i += kKeepThreads) hist[i] = 0;
    __syncthreads();
    each([&](u32x4 v, int) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (v[j] != 0u && (v[j] & mask) == prefix) atomicAdd(&hist[(v[j] >> shift) & digits], 1u);
    });
    __syncthreads();
    // From the largest digit down: the first whose rows and all above reach `want`. Lanes
    // take 32 digits each, then the lanes' scan its 32.
    if (wave == 0) {
      const int group = 63 - lane;
      uint32_t mine = 0;
#pragma unroll
      for (int j = 0; j < 32; ++j) mine += hist[32 * group + ((j + lane) & 31)];  // (banks apart)
      const uint32_t upto = scan64(mine);
      const int l = __builtin_ctzll(__ballot(upto >= want));
      const uint32_t before = __shfl(upto - mine, l);
      const uint32_t one = lane < 32 ? hist[32 * (63 - l) + 31 - lane] : 0u;
      const uint32_t in = before + scan64(one);
      if (lane == __builtin_ctzll(__ballot(in >= want))) {
        found[0] = uint32_t(32 * (63 - l) + 31 - lane);
        found[1] = want - (in - one);
        found[2] = one;
      }
    }
    __syncthreads();
    prefix |= found[0] << shift;
    mask |= digits << shift;
    want = found[1];
    if (found[2] == want) {  // all of these: whatever is at least as large as the digits found
      prefix -= 1;
      want = 0;
      break;
    }
    if (shift == 0) break;
  }

  // Rows above it, and the first `want` of those at it. Two counts of a step's 256 rows
  // in one number: those above it in the low half, those at it in the high one.
  auto count = [&](u32x4 v) __attribute__((always_inline)) {
    uint32_t n = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) n += (v[j] > prefix ? 1u : 0u) + (v[j] == prefix ? 1u << 16 : 0u);
    return n;
  };
  uint32_t n_above = 0, n_at = 0;
  each([&](u32x4 v, int) __attribute__((always_inline)) {
    const uint32_t n = count(v);
    n_above += n & 0xffffu;
    n_at += n >> 16;
  });
  n_above = scan64(n_above);
  n_at = scan64(n_at);
  if (lane == 63) {
    above[wave] = n_above;
    at[wave] = n_at;
  }
  __syncthreads();
  uint32_t pos = 0, seen = 0;  // above, and at it, before this wave's next step
  for (int i = 0; i < wave; ++i) {
    pos += above[i];
    seen += at[i];
  }
  each([&](u32x4 v, int row) __attribute__((always_inline)) {
    const uint32_t n = count(v), upto = scan64(n), before = upto - n;
    uint32_t s = seen + (before >> 16), p = pos + (before & 0xffffu) + min(s, want);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bool same = v[j] == prefix;
      if (v[j] > prefix || (same && s < want)) out[p++] = row + j;
      s += same ? 1u : 0u;
    }
    const uint32_t all = uint32_t(__builtin_amdgcn_readlane(int(upto), 63));
    pos += all & 0xffffu;
    seen += all >> 16;
  });
}

constexpr int kUnits = 4;  // of a thread in a step, and of a row in a column

struct GatherArgs {
  char* pages; int64_t p_plane, p_sp, p_sr, p_sh;  // bytes
  const int32_t* src; int64_t s_sb;
  const int32_t* dst; int64_t d_sb;
  const int32_t* rows;             // [B, H, keep]
  float* w; int64_t w_sb, w_sh;    // null: none
  int BH, H, keep, width, dst_width, n_pages, page_rows, w_width;
  int chunks, slice;               // 16-byte chunks of a row; of a workgroup's column (a power of two)
  int slices;                      // columns of a plane; a 4-bit one's last holds its scales
  int tail;                        // scale bytes of a row (0: a 16- or 32-bit pool)
};

// Where a row goes from and to, in bytes from a plane's head; from < 0: it does not move.
struct Place { int64_t from, to; };

// Byte offset of row r of a table's pages, or -1.
__device__ __forceinline__ int64_t place_of(const GatherArgs& a, const int32_t* table, int r, int width,
                                            int64_t row_bytes) {
  if (uint32_t(r) >= uint32_t(width) * uint32_t(a.page_rows)) return -1;
  const int e = int(uint32_t(r) / uint32_t(a.page_rows));
  const int page = table[e];
  if (uint32_t(page) >= uint32_t(a.n_pages)) return -1;
  return page * a.p_sp + (r - e * a.page_rows) * row_bytes;
}

// A column of the rows, `units` Us of each; `per` (a power of two, units at least, kUnits at
// most) lanes to a row. kThreads rows to a step. Their places are looked up (two reads that
// wait for one another) by a thread each, one step ahead; a step's loads go out before the
// last one's stores: its rows lie behind those that are written then. No wave stores a step
// before all have read it.
template <int kThreads, typename U>
__device__ __forceinline__ void move_column(const GatherArgs& a, Place (*list)[kThreads], char* column,
                                            const int32_t* rows, const int32_t* src, const int32_t* dst,
                                            int64_t row_bytes, int per, int units) {
  const int tid = int(threadIdx.x), lr = tid / per, lu = tid % per, row_step = kThreads / per;
  auto number = [&](int i) __attribute__((always_inline)) { return i < a.keep ? rows[i] : -1; };
  auto look = [&](int r, int i) __attribute__((always_inline)) {
    Place p{-1, -1};
    if (r >= 0) {
      p.from = place_of(a, src, r, a.width, row_bytes);
      p.to = place_of(a, dst, i, a.dst_width, row_bytes);
      if (p.to < 0 || p.from == p.to) p.from = -1;  // (what stays may be another sequence's too)
    }
    return p;
  };
  U x[2][kUnits];
  int64_t to[2][kUnits];  // below 0: nothing
  auto load = [&](const Place* l, U (&y)[kUnits], int64_t (&t)[kUnits]) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < kUnits; ++j) {
      t[j] = -1;
      if (j < per && lu < units) {
        const Place p = l[j * row_step + lr];
        if (p.from >= 0) {
          y[j] = *reinterpret_cast<const U*>(column + p.from + lu * int(sizeof(U)));
          t[j] = p.to;
        }
      }
    }
  };
  list[0][tid] = look(number(tid), tid);
  int r = number(kThreads + tid);
  __syncthreads();
  load(list[0], x[0], to[0]);
#pragma unroll 1
  for (int i0 = 0; i0 < a.keep; i0 += 2 * kThreads) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int next = i0 + (u + 1) * kThreads;  // first row of the next step
      if (next - kThreads >= a.keep) break;
      list[1 - u][tid] = look(r, next + tid);
      r = number(next + kThreads + tid);
      wait_vmcnt<0>();  // this wave's loads have returned,
      __syncthreads();  // and the others'
      if (next < a.keep) load(list[1 - u], x[1 - u], to[1 - u]);
#pragma unroll
      for (int j = 0; j < kUnits; ++j)
        if (to[u][j] >= 0) *reinterpret_cast<U*>(column + to[u][j] + lu * int(sizeof(U))) = x[u][j];
    }
  }
}

template <int kThreads>
__global__ __launch_bounds__(kThreads) void kv_page_gather_kernel(GatherArgs a) {
  __shared__ Place list[2][kThreads];
  // The columns of a plane's head on one XCD (workgroup i runs on XCD i % 8), whose L2 then
  // has the other half of each line that one of them reads.
  uint32_t i = blockIdx.x, plane = 0;
  uint32_t bh, col;
  const uint32_t planes = 2u * uint32_t(a.BH), moves = planes * uint32_t(a.slices);
  const bool weights = i >= moves;
  if (weights) {
    bh = i - moves;
    col = 0;
  } else {
    const uint32_t in8 = planes % 8 == 0 ? 8u : 1u, at = i / in8;
    plane = at / uint32_t(a.slices);
    col = at - plane * uint32_t(a.slices);
    plane = plane * in8 + i % in8;
    bh = plane >> 1;
  }
  const int b = int(bh / uint32_t(a.H)), h = int(bh) - b * a.H;
  const int32_t* const rows = a.rows + int64_t(bh) * a.keep;
  if (weights) {  // kept ones to the front, 0 behind
    float* const w = a.w + b * a.w_sb + h * a.w_sh;
    constexpr int N = 8;
#pragma unroll 1
    for (int i0 = 0; i0 < a.w_width; i0 += N * kThreads) {
      float x[N];
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const int i = i0 + j * kThreads + int(threadIdx.x);
        const int r = i < a.keep ? rows[i] : -1;
        x[j] = uint32_t(r) < uint32_t(a.w_width) ? w[r] : 0.f;
      }
      wait_vmcnt<0>();
      __syncthreads();
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const int i = i0 + j * kThreads + int(threadIdx.x);
        if (i < a.w_width) w[i] = x[j];
      }
    }
    return;
  }
  char* column = a.pages + (plane & 1 ? a.p_plane : 0) + h * a.p_sh;
  const int32_t* const src = a.src + b * a.s_sb;
  const int32_t* const dst = a.dst + b * a.d_sb;
  if (a.tail && int(col) == a.slices - 1) {
    // Scales, 2, 4 or 8 bytes of a row, behind the page's codes.
    column += int64_t(a.page_rows) * a.p_sr;
    if (a.tail == 2)
      move_column<kThreads, uint16_t>(a, list, column, rows, src, dst, 2, 1, 1);
    else
      move_column<kThreads, uint32_t>(a, list, column, rows, src, dst, a.tail, a.tail / 4, a.tail / 4);
  } else {
    move_column<kThreads, u32x4>(a, list, column + int64_t(col) * a.slice * 16, rows, src, dst, a.p_sr, a.slice,
                       min(a.slice, a.chunks - int(col) * a.slice));
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
  a.held = int(std::min<int64_t>(kHeld, (width + 4 * kKeepThreads - 1) / (4 * kKeepThreads) * (4 * kKeepThreads)));
  const hipError_t e = opt_in_lds(reinterpret_cast<const void*>(&kv_keep_rows_kernel), kHeld * 4);
  if (e != hipSuccess) {
    set_error("%s: %s", what, hipGetErrorString(e));
    return DX_ELAUNCH;
  }
  hipLaunchKernelGGL(kv_keep_rows_kernel, dim3(unsigned(B * H)), dim3(kKeepThreads), a.held * 4,
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
  a.BH = int(B * H); a.H = int(H); a.keep = int(keep); a.width = int(width); a.dst_width = int(dst_width);
  a.n_pages = int(n_pages); a.page_rows = int(page_rows); a.w_width = int(w_width);
  a.chunks = int(fp4 ? D / 32 : D * es / 16);
  a.tail = int(fp4 ? D / 32 : 0);
  // Columns of 4 chunks (64 bytes), of less where a row has less: of one long sequence of
  // few heads there would be too few workgroups otherwise.
  a.slice = std::min(kUnits, a.chunks);
  while (a.slice & (a.slice - 1)) --a.slice;
  a.slices = (a.chunks + a.slice - 1) / a.slice + (fp4 ? 1 : 0);
  const int64_t blocks = (2 * a.slices + (weights ? 1 : 0)) * B * H;
  DX_CHECK_ARG(grid_fits(blocks, 1024), "%s: the call exceeds one launch", what);
  const dim3 grid{unsigned(blocks)};
  const hipStream_t st = static_cast<hipStream_t>(stream);
  // Few columns: as many rows to a step as a workgroup has threads, since a step waits for
  // its lookups. Two and more to a compute unit: short steps, whose waits overlap. With 256 and
  // with 1,024 threads, us a call of 1,024 of 3,000 rows: 4 x 8 heads (256 columns, bf16) 14.3
  // and 13.7; 16 x 8 (1,024 columns) 24.3 and 30.1; 32 x 8 in 4 bits (1,024) 18.6 and 21.6; 24
  // heads, 8,192 of 32,768 rows (192) 57.1 and 48.7, of four sequences (768) 241 and 242.
  if (2 * a.slices * B * H <= 2 * device_cus())
    hipLaunchKernelGGL(kv_page_gather_kernel<1024>, grid, dim3(1024), 0, st, a);
  else
    hipLaunchKernelGGL(kv_page_gather_kernel<256>, grid, dim3(256), 0, st, a);
  DX_CHECK_LAUNCH(what);
  return DX_OK;
}
