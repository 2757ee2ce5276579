// Pages of a KV cache on gfx950: writing a chunk into a batch's pages, and
// copying pages (forks, compaction).
//
// A pool is [2, P, R, H, D]: plane 0 K, plane 1 V, P pages of R rows. Row r of
// sequence b lies in page table[b][r / R] at row r % R. Both kernels move bits
// (16-byte loads and stores) and are bound by memory traffic: what they read
// and write once each is all there is. Append of 4 x 1,826 rows of 40 heads (f16,
// D 128): 57.5 us, 5.2 TB/s; of one token of 64 sequences 3.9 us, its latency. Copy
// of 16 pages (32 rows of 24 heads, bf16, D 128) in 30 pools: 76 us, 5.0 TB/s; of one
// page in 16 pools (a fork) 3.9 us.
//
//  * kv_page_append_kernel: one wave per piece of a token row (128 16-byte
//    chunks of k and of v, so four loads are in flight per lane); its page is
//    looked up once, in scalar registers. A row that has no page (a start
//    below 0, a row past the table, an entry that names no page of the pool)
//    is not written and sets the status word.
//  * kv_page_copy_kernel: workgroups take pieces of (pool, plane, pair); the
//    pools' addresses and the page pairs travel in the kernel arguments, so a
//    fork of every layer is one launch and needs no device list.
#include "dx_common.h"

#include <algorithm>
#include <exception>
#include <vector>

namespace dx {
namespace {

constexpr int kAppendWaves = 4;   // waves per workgroup of the append
constexpr int kAppendChunks = 2;  // 16-byte chunks of k (and of v) per lane

struct PageAppendArgs {
  const uint8_t* k; int64_t k_sb, k_sl, k_sh;  // strides in bytes
  const uint8_t* v; int64_t v_sb, v_sl, v_sh;
  uint8_t* pk; uint8_t* pv; int64_t p_sp, p_sr, p_sh;
  const int32_t* table; int64_t t_sb;
  const int32_t* starts;
  int32_t* status;
  int64_t items;         // (sequence, token, piece of its row)
  int n, parts;          // tokens per sequence, pieces per row
  int chunks, head_chunks;  // 16-byte chunks per row and per head
  int width, n_pages, page_rows;
};

__global__ __launch_bounds__(64 * kAppendWaves) void kv_page_append_kernel(PageAppendArgs a) {
  const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) >> 6);
  const int lane = int(threadIdx.x) & 63;
  const int64_t item = int64_t(blockIdx.x) * kAppendWaves + wave;
  if (item >= a.items) return;
  // items < 2^31 (the host's check), so the decode is 32-bit.
  const uint32_t row = uint32_t(item) / uint32_t(a.parts);
  const int part = int(uint32_t(item) - row * uint32_t(a.parts));
  const int b = int(row / uint32_t(a.n)), t = int(row - uint32_t(b) * uint32_t(a.n));
  const int64_t at = int64_t(a.starts[b]) + t;
  int page = -1;
  if (at >= 0 && at < int64_t(a.width) * a.page_rows)
    page = a.table[b * a.t_sb + at / a.page_rows];
  if (uint32_t(page) >= uint32_t(a.n_pages)) {
    if (a.status && lane == 0) a.status[0] = 1;
    return;
  }
  const uint8_t* const k = a.k + b * a.k_sb + t * a.k_sl;
  const uint8_t* const v = a.v + b * a.v_sb + t * a.v_sl;
  const int64_t dst = page * a.p_sp + (at % a.page_rows) * a.p_sr;
  u32x4 kx[kAppendChunks], vx[kAppendChunks];
  int64_t off[kAppendChunks];
#pragma unroll
  for (int i = 0; i < kAppendChunks; ++i) {
    const int c = (part * kAppendChunks + i) * 64 + lane;
    off[i] = -1;
    if (c < a.chunks) {
      const int h = int(uint32_t(c) / uint32_t(a.head_chunks));
      const int64_t in_head = 16 * int64_t(c - h * a.head_chunks);
      kx[i] = *reinterpret_cast<const u32x4*>(k + h * a.k_sh + in_head);
      vx[i] = *reinterpret_cast<const u32x4*>(v + h * a.v_sh + in_head);
      off[i] = dst + h * a.p_sh + in_head;
    }
  }
#pragma unroll
  for (int i = 0; i < kAppendChunks; ++i)
    if (off[i] >= 0) {
      *reinterpret_cast<u32x4*>(a.pk + off[i]) = kx[i];
      *reinterpret_cast<u32x4*>(a.pv + off[i]) = vx[i];
    }
}

constexpr int kCopyPools = 64;   // pools per launch
constexpr int kCopyPairs = 256;  // page pairs per launch
constexpr int kCopyThreads = 256, kCopyChunks = 4;
constexpr int kCopyPiece = kCopyThreads * kCopyChunks;  // 16-byte chunks per workgroup

struct PageCopyArgs {
  uint8_t* pool[kCopyPools];  // plane 0
  int src[kCopyPairs], dst[kCopyPairs];
  int64_t plane, p_sp, p_sr, p_sh;  // bytes
  int pairs, pieces;                // page pairs, workgroups per (pool, plane, pair)
  int chunks;                       // 16-byte chunks of a page in one plane
  int row_chunks, head_chunks;      // of a row and of a head; row_chunks 0: a page is one run
};

__global__ __launch_bounds__(kCopyThreads) void kv_page_copy_kernel(PageCopyArgs a) {
  uint32_t i = blockIdx.x;
  const uint32_t group = i / uint32_t(a.pieces);
  const int piece = int(i - group * uint32_t(a.pieces));
  const uint32_t pool2 = group / uint32_t(a.pairs);
  const int pair = int(group - pool2 * uint32_t(a.pairs));
  uint8_t* const base = a.pool[pool2 >> 1] + (pool2 & 1) * a.plane;
  const uint8_t* const from = base + a.src[pair] * a.p_sp;
  uint8_t* const to = base + a.dst[pair] * a.p_sp;
  u32x4 x[kCopyChunks];
  int64_t off[kCopyChunks];
#pragma unroll
  for (int u = 0; u < kCopyChunks; ++u) {
    const int c = piece * kCopyPiece + u * kCopyThreads + int(threadIdx.x);
    off[u] = -1;
    if (c < a.chunks) {
      if (a.row_chunks == 0) {
        off[u] = 16 * int64_t(c);
      } else {
        const uint32_t r = uint32_t(c) / uint32_t(a.row_chunks);
        const uint32_t in_row = uint32_t(c) - r * uint32_t(a.row_chunks);
        const uint32_t h = in_row / uint32_t(a.head_chunks);
        off[u] = r * a.p_sr + h * a.p_sh + 16 * int64_t(in_row - h * uint32_t(a.head_chunks));
      }
      x[u] = *reinterpret_cast<const u32x4*>(from + off[u]);
    }
  }
#pragma unroll
  for (int u = 0; u < kCopyChunks; ++u)
    if (off[u] >= 0) *reinterpret_cast<u32x4*>(to + off[u]) = x[u];
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Element size of a dtype code, 0 for none.
int64_t elem_size(int dtype) {
  return dtype == DX_F32 ? 4 : dtype == DX_BF16 || dtype == DX_F16 ? 2 : 0;
}

}  // namespace
}  // namespace dx

using namespace dx;

extern "C" int dx_kv_page_append(const void* k, int64_t k_sb, int64_t k_sl, int64_t k_sh,
                                 const void* v, int64_t v_sb, int64_t v_sl, int64_t v_sh,
                                 void* pages, int64_t p_plane, int64_t p_sp, int64_t p_sr,
                                 int64_t p_sh, int dtype, int64_t n_pages, int64_t page_rows,
                                 const void* block_table, int64_t t_sb, int64_t width,
                                 const void* starts, void* status, int64_t B, int64_t n,
                                 int64_t H, int64_t D, void* stream) {
  const int64_t es = elem_size(dtype);
  DX_CHECK_ARG(es != 0, "kv_page_append: dtype code %d unsupported", dtype);
  DX_CHECK_ARG(B >= 0 && n >= 0 && H > 0 && D > 0 && n_pages >= 0 && page_rows > 0 && width >= 0,
               "kv_page_append: bad shape");
  const int64_t per16 = 16 / es;
  DX_CHECK_ARG(D % per16 == 0, "kv_page_append: head_dim must fill 16-byte chunks");
  constexpr int64_t kMax = (int64_t(1) << 31) - 1;
  DX_CHECK_ARG(n_pages <= kMax && page_rows <= kMax && width <= kMax && n <= kMax,
               "kv_page_append: sizes must be below 2^31");
  if (B == 0 || n == 0) return DX_OK;
  DX_CHECK_ARG(k && v && block_table && starts, "kv_page_append: null pointer");
  DX_CHECK_ARG(pages || n_pages == 0, "kv_page_append: null pages");
  DX_CHECK_ARG(aligned16(k) && aligned16(v) && aligned16(pages),
               "kv_page_append: pointers must be 16-byte aligned");
  DX_CHECK_ARG(k_sb % per16 == 0 && k_sl % per16 == 0 && k_sh % per16 == 0 &&
                   v_sb % per16 == 0 && v_sl % per16 == 0 && v_sh % per16 == 0 &&
                   p_plane % per16 == 0 && p_sp % per16 == 0 && p_sr % per16 == 0 &&
                   p_sh % per16 == 0,
               "kv_page_append: strides must keep head rows 16-byte aligned");
  PageAppendArgs a{};
  a.k = static_cast<const uint8_t*>(k); a.k_sb = k_sb * es; a.k_sl = k_sl * es; a.k_sh = k_sh * es;
  a.v = static_cast<const uint8_t*>(v); a.v_sb = v_sb * es; a.v_sl = v_sl * es; a.v_sh = v_sh * es;
  a.pk = static_cast<uint8_t*>(pages);
  a.pv = static_cast<uint8_t*>(pages) + p_plane * es;
  a.p_sp = p_sp * es; a.p_sr = p_sr * es; a.p_sh = p_sh * es;
  a.table = static_cast<const int32_t*>(block_table); a.t_sb = t_sb;
  a.starts = static_cast<const int32_t*>(starts);
  a.status = static_cast<int32_t*>(status);
  const int64_t chunks = H * (D / per16);
  DX_CHECK_ARG(H <= kMax && D <= kMax && chunks <= kMax, "kv_page_append: rows too long");
  const int64_t parts = (chunks + 64 * kAppendChunks - 1) / (64 * kAppendChunks);
  // Workgroups below 2^31 and threads below 2^32, 32-bit item numbers.
  DX_CHECK_ARG(B <= kMax && n <= kMax / B && parts <= kMax / (B * n) && B * n * parts <= (1 << 26) - 1,
               "kv_page_append: %lld x %lld rows exceed one launch", (long long)B, (long long)n);
  a.items = B * n * parts;
  a.n = int(n); a.parts = int(parts);
  a.chunks = int(chunks); a.head_chunks = int(D / per16);
  a.width = int(width); a.n_pages = int(n_pages); a.page_rows = int(page_rows);
  const int64_t blocks = (a.items + kAppendWaves - 1) / kAppendWaves;
  hipLaunchKernelGGL(kv_page_append_kernel, dim3(unsigned(blocks)), dim3(64 * kAppendWaves), 0,
                     static_cast<hipStream_t>(stream), a);
  DX_CHECK_LAUNCH("kv_page_append");
  return DX_OK;
}

extern "C" int dx_kv_page_copy(const void* const* pools, int64_t n_pools, int64_t p_plane,
                               int64_t p_sp, int64_t p_sr, int64_t p_sh, int dtype,
                               int64_t n_pages, int64_t page_rows, int64_t H, int64_t D,
                               const int64_t* src, const int64_t* dst, int64_t pairs,
                               void* stream) {
  const int64_t es = elem_size(dtype);
  DX_CHECK_ARG(es != 0, "kv_page_copy: dtype code %d unsupported", dtype);
  DX_CHECK_ARG(n_pools >= 0 && pairs >= 0 && n_pages >= 0 && page_rows > 0 && H > 0 && D > 0,
               "kv_page_copy: bad shape");
  const int64_t per16 = 16 / es;
  DX_CHECK_ARG(D % per16 == 0, "kv_page_copy: head_dim must fill 16-byte chunks");
  DX_CHECK_ARG(p_plane % per16 == 0 && p_sp % per16 == 0 && p_sr % per16 == 0 && p_sh % per16 == 0,
               "kv_page_copy: strides must keep head rows 16-byte aligned");
  if (pairs == 0) return DX_OK;
  DX_CHECK_ARG(src && dst, "kv_page_copy: null page list");
  for (int64_t i = 0; i < pairs; ++i)
    DX_CHECK_ARG(src[i] >= 0 && src[i] < n_pages && dst[i] >= 0 && dst[i] < n_pages,
                 "kv_page_copy: page %lld -> %lld outside a pool of %lld", (long long)src[i],
                 (long long)dst[i], (long long)n_pages);
  // No order is defined between the copies of one call, so a page that is
  // written may be neither read nor written by another of them.
  try {
    std::vector<int64_t> to(dst, dst + pairs), from(src, src + pairs);
    std::sort(to.begin(), to.end());
    const auto twice = std::adjacent_find(to.begin(), to.end());
    DX_CHECK_ARG(twice == to.end(), "kv_page_copy: page %lld is written twice",
                 (long long)*twice);
    for (const int64_t p : from)
      DX_CHECK_ARG(!std::binary_search(to.begin(), to.end(), p),
                   "kv_page_copy: page %lld is both read and written", (long long)p);
  } catch (const std::exception&) {  // bad_alloc, length_error
    set_error("kv_page_copy: out of host memory");
    return DX_EINVAL;
  }
  if (n_pools == 0) return DX_OK;
  DX_CHECK_ARG(pools, "kv_page_copy: null pool list");
  for (int64_t i = 0; i < n_pools; ++i)
    DX_CHECK_ARG(pools[i] && aligned16(pools[i]), "kv_page_copy: pools must be 16-byte aligned");
  constexpr int64_t kMax = (int64_t(1) << 31) - 1;
  const int64_t head_chunks = D / per16;
  DX_CHECK_ARG(H <= kMax / head_chunks && page_rows <= kMax / (H * head_chunks) &&
                   page_rows * H * head_chunks <= kMax - kCopyPiece && n_pages <= kMax,
               "kv_page_copy: a page must hold fewer than 2^31 16-byte chunks");
  PageCopyArgs a{};
  a.plane = p_plane * es; a.p_sp = p_sp * es; a.p_sr = p_sr * es; a.p_sh = p_sh * es;
  a.chunks = int(page_rows * H * head_chunks);
  const bool one_run = (H == 1 || p_sh == D) && (page_rows == 1 || p_sr == H * D);
  a.row_chunks = one_run ? 0 : int(H * head_chunks);
  a.head_chunks = int(head_chunks);
  a.pieces = (a.chunks + kCopyPiece - 1) / kCopyPiece;
  for (int64_t l0 = 0; l0 < n_pools; l0 += kCopyPools) {
    const int64_t nl = std::min<int64_t>(kCopyPools, n_pools - l0);
    for (int64_t i = 0; i < nl; ++i) a.pool[i] = static_cast<uint8_t*>(const_cast<void*>(pools[l0 + i]));
    // Pairs per launch: below 2^24 workgroups (2^32 threads).
    const int64_t most = std::max<int64_t>(
        1, std::min<int64_t>(kCopyPairs, ((int64_t(1) << 24) - 1) / (2 * nl * a.pieces)));
    DX_CHECK_ARG(2 * nl * a.pieces < (int64_t(1) << 24), "kv_page_copy: pages too large");
    for (int64_t p0 = 0; p0 < pairs; p0 += most) {
      a.pairs = int(std::min<int64_t>(most, pairs - p0));
      for (int i = 0; i < a.pairs; ++i) {
        a.src[i] = int(src[p0 + i]);
        a.dst[i] = int(dst[p0 + i]);
      }
      hipLaunchKernelGGL(kv_page_copy_kernel, dim3(unsigned(2 * nl * a.pairs * a.pieces)),
                         dim3(kCopyThreads), 0, static_cast<hipStream_t>(stream), a);
      DX_CHECK_LAUNCH("kv_page_copy");
    }
  }
  return DX_OK;
}
