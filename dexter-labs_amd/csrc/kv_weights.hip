// The softmax weight that each cached row received, on gfx950: what a cache that forgets
// goes by.
//
//   w[b][hk][r] (+)= sum over queries t and the query heads h of K/V head hk of
//                    exp(scale q[b][t][h] . k[b][r][hk] - lse[b][t][h])
//
// with the log-sum-exp that attention over the same keys returned, so that each
// term is the probability which that query gave the row. Every cached row is seen by
// every query of its sequence, so there is no mask; K is read once, V not at all.
//
// S = Q K^T on 32 x 32 MFMAs with the queries on M and the keys on N: a lane holds one
// key and 16 queries, so a key's sum stays in its lane, in fp32, in one order (no
// atomics: the same call gives the same bits), and two lanes meet at the end. Each wave
// keeps 32 NK keys in registers, for 4 bits converted there (CodedRow), while the
// queries, all rows of a (sequence, K/V head), pass through LDS for four waves. 64 keys
// a wave halve the LDS reads per product, which at 32 would take the LDS as long as the
// products take the matrix units.
//
// What it takes (in a captured stream): a chunk of 83 over 32,768 rows of 24 heads (D 128) 43 us
// in bf16 when the same rows come again, 4.7 TB/s, and 58 with others, 3.6; 32 us in 4 bits; 199
// in fp32, whose products are a thirteenth of the rate; one token of 32 prompts of 300 to 3,000
// rows 14.5 us in 4 bits, most of it first loads, and 30 in 16; 2 x 1,500 queries, 16 heads
// over 8, over 4,000 to 10,000 rows 120 us, 600 TFLOP/s, exponentials and products in turn, and 158
// over a table of twice the width: workgroups that find no row there take a place among the
// others, and CUs get uneven shares. Long workgroups that walk several blocks of keys gained
// nothing at 3 to 1,000 workgroups per compute unit.
#include "attn_common.h"
#include "attn_tile.h"
#include "kv_fp4.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace dx {
namespace {

constexpr int kWaves = 4, kThreads = 64 * kWaves;
constexpr float kNone = 0x1.fffffep127f;  // for a log-sum-exp: of a query that gives nothing

struct WeightArgs {
  const char* q; int64_t q_sb, q_sl, q_sh;  // bytes
  const float* lse;                         // [B, Lq, H]
  const char* pk; int64_t p_sp, p_sr, p_sh; // plane 0
  const int32_t* table; int64_t t_sb;
  const int32_t* lens;
  float* w; int64_t w_sb, w_sh;             // [B, Hkv, width * page_rows]
  int add;                                  // 0: rows past a length become 0
  int width, n_pages, page_rows;
  uint32_t page_magic;                      // as PagedArgs'
  int Hkv, H, group, Lq, R;
  float scale_log2;
};

template <typename T, int D, bool FP4> struct Form {
  static constexpr int es = sizeof(T), RB = D * es, KS = RB / 32;
  static constexpr int NK = RB <= 256 ? 2 : 1;  // 32-key tiles of a wave
  static constexpr int QT = RB <= 256 ? 64 : 32;       // query rows in LDS
  static constexpr int keys = 32 * NK * kWaves;        // of a workgroup
};

// 16-byte chunk c of query row r in LDS sits at c ^ swz(r): reads of 32 rows at one chunk
// meet no bank twice.
template <int RB> __device__ __forceinline__ constexpr int swz(int r) {
  return RB == 128 ? ((r >> 2) ^ (4 * ((r >> 1) & 1))) & 7 : (r & 15) ^ ((r >> 4) & 1);
}

template <typename T, int D, bool FP4>
__global__ __launch_bounds__(kThreads) void paged_key_weights_kernel(WeightArgs a) {
  using F = Form<T, D, FP4>;
  constexpr int RB = F::RB, KS = F::KS, NK = F::NK, QT = F::QT, CR = RB / 16;
  constexpr bool F32 = F::es == 4;
  // One array, the tile at a multiple of RB in it: chunks are addressed by XOR into a row's start.
  struct Shared {
    __attribute__((aligned(512))) char tile[QT * RB];
    __attribute__((aligned(16))) float stat[QT];
  };
  __shared__ Shared shared;
  static_assert(512 % RB == 0 && alignof(Shared) % RB == 0 && __builtin_offsetof(Shared, tile) == 0,
                "a row's chunks by XOR");
  char* const tile = shared.tile;
  float* const stat = shared.stat;
  const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) >> 6), lane = int(threadIdx.x) & 63;
  const int g = lane >> 5, nl = lane & 31;
  const int bh = int(blockIdx.y), b = bh / a.Hkv, hk = bh - b * a.Hkv;
  // (Without queries no row is looked at: what stands in for missing ones is a query.)
  const int rows = a.width * a.page_rows, len = a.R > 0 ? min(max(a.lens[b], 0), rows) : 0;
  const int key0 = int(blockIdx.x) * F::keys + wave * 32 * NK;
  float* const w = a.w + b * a.w_sb + hk * a.w_sh;
  if (int(blockIdx.x) * F::keys >= len) {  // nothing here
    if (!a.add)
      for (int r = int(threadIdx.x); r < F::keys; r += kThreads)
        if (int(blockIdx.x) * F::keys + r < rows) w[int(blockIdx.x) * F::keys + r] = 0.f;
    return;
  }

  // Queries on their way into LDS: this thread's chunks of rows row0.., and a row's lse. The
  // first ones are read before all else, then the page numbers, whatever the length: what a
  // workgroup waits for at its start are two reads one after the other, not four (a chunk of 83
  // over 32,768 rows of 24 heads in bf16, the same rows again: 50 us in the other order).
  constexpr int NQ = QT * CR / kThreads;
  static_assert(QT * CR % kThreads == 0 && QT <= kThreads, "whole shares");
  u32x4 qx[NQ];
  float lx;
  auto read_queries = [&](int row0) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < NQ; ++e) {
      const int u = e * kThreads + int(threadIdx.x), row = min(row0 + u / CR, a.R - 1);
      const int t = int(uint32_t(row) / uint32_t(a.group)), h = hk * a.group + row - t * a.group;
      qx[e] = *reinterpret_cast<const u32x4*>(a.q + b * a.q_sb + t * a.q_sl + h * a.q_sh + 16 * (u % CR));
    }
    const int row = min(row0 + int(threadIdx.x) % QT, a.R - 1);
    const int t = int(uint32_t(row) / uint32_t(a.group)), h = hk * a.group + row - t * a.group;
    lx = a.lse[(int64_t(b) * a.Lq + t) * a.H + h];
  };
  auto write_queries = [&](int row0) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < NQ; ++e) {
      const int u = e * kThreads + int(threadIdx.x), r = u / CR, c = u % CR;
      *reinterpret_cast<u32x4*>(tile + r * RB + 16 * (c ^ swz<RB>(r))) = qx[e];
    }
    // A query that saw no key, and one past the last, gives nothing, whatever its scores.
    const bool none = row0 + int(threadIdx.x) % QT >= a.R || lx == -INFINITY;
    if (int(threadIdx.x) < QT) stat[threadIdx.x] = none ? kNone : lx * 1.4426950408889634f;
  };
  read_queries(0);  // (there are some: without any there are no rows either, see len)

  // This lane's keys: half of the dims of each, chunks 8 (s / 4) + 4 g + s % 4, which in
  // 4 bits are whole blocks. Rows without a page or past the length read a query instead
  // (2 or 4 D bytes) and are not written. (4-bit rows are converted here: kept as codes they
  // take fewer registers, but 1,500 queries then take 134 us for 118.)
  u32x4 kf[NK][KS];
  bool there[NK];
  int page[NK];
  auto entry_of = [&](uint32_t r) __attribute__((always_inline)) {
    return a.page_magic ? uint32_t((uint64_t(r >> 4) * a.page_magic) >> 32) : r >> 4;
  };
#pragma unroll
  for (int x = 0; x < NK; ++x)
    page[x] = a.table[b * a.t_sb + entry_of(uint32_t(min(key0 + 32 * x + nl, rows - 1)))];
#pragma unroll
  for (int x = 0; x < NK; ++x) {
    const int r = key0 + 32 * x + nl;
    there[x] = r < len && uint32_t(page[x]) < uint32_t(a.n_pages);
    const uint32_t in_page = uint32_t(r) - entry_of(uint32_t(r)) * uint32_t(a.page_rows);
    const char* const head = a.pk + int64_t(page[x]) * a.p_sp + hk * a.p_sh;
    if constexpr (FP4) {
      const char* const codes = there[x] ? head + in_page * uint32_t(D / 2) : a.q;
      const char* const scales = there[x] ? head + uint32_t(a.page_rows) * (D / 2) + in_page * uint32_t(D / 32) : a.q;
      u32x4 c[D / 64];
      uint8_t sb[D / 64];
#pragma unroll
      for (int i = 0; i < D / 64; ++i) {
        c[i] = *reinterpret_cast<const u32x4*>(codes + 32 * i + 16 * g);
        sb[i] = *reinterpret_cast<const uint8_t*>(scales + 2 * i + g);
      }
#pragma unroll
      for (int s = 0; s < KS; ++s) kf[x][s] = fp4_values<T>(c[s / 4][s % 4], fp4_scale(sb[s / 4]));
    } else {
      const char* const row = there[x] ? head + int64_t(in_page) * a.p_sr : a.q;
#pragma unroll
      for (int s = 0; s < KS; ++s)
        kf[x][s] = *reinterpret_cast<const u32x4*>(row + 16 * (8 * (s / 4) + 4 * g + s % 4));
    }
  }

  float sum[NK] = {};
  const uint32_t base = lds_addr(tile);
  for (int row0 = 0; row0 < a.R; row0 += QT) {
    if (row0) {
      read_queries(row0);
      __syncthreads();  // the last rows are read
    }
    write_queries(row0);
    __syncthreads();
#pragma unroll 1
    for (int m0 = 0; m0 < QT && row0 + m0 < a.R; m0 += 32) {
      f32x16 s[NK];
#pragma unroll
      for (int x = 0; x < NK; ++x) s[x] = f32x16{};
      const uint32_t qa = base + (m0 + nl) * RB + 16 * ((4 * g) ^ swz<RB>(nl));  // (the same for m0 + nl)
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        const u32x4 qf = lds_read_b128_at(qa ^ (16u * (8 * (i / 4) + i % 4)));
#pragma unroll
        for (int x = 0; x < NK; ++x) {
          if constexpr (F32) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              s[x] = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(qf[e]), __uint_as_float(kf[x][i][e]), s[x], 0, 0, 0);
          } else {
            s[x] = Mfma<T>::run(qf, kf[x][i], s[x]);
          }
        }
      }
      // Register r: query m0 + 8 (r / 4) + 4 g + r % 4. Their sum as a tree, then one
      // addition: of many queries the running sum takes a rounding per 32. (An infinite score
      // or NaN less kNone is no 0: where a query that saw no key is among them, such terms are
      // taken out. What stands behind the last query is that one again, whose own term is as
      // infinite then.)
      auto add_up = [&](auto some) __attribute__((always_inline)) {
#pragma unroll
        for (int x = 0; x < NK; ++x) {
          float part[4];
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const f32x4 l = *reinterpret_cast<const f32x4*>(&stat[m0 + 8 * u + 4 * g]);
            float p[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              p[e] = fast_exp2(__builtin_fmaf(s[x][4 * u + e], a.scale_log2, -l[e]));
              if constexpr (decltype(some)::value) p[e] = l[e] == kNone ? 0.f : p[e];
            }
            part[u] = (p[0] + p[1]) + (p[2] + p[3]);
          }
          sum[x] += (part[0] + part[1]) + (part[2] + part[3]);
        }
      };
      if (__ballot(stat[m0 + nl] == kNone && row0 + m0 + nl < a.R))
        add_up(std::integral_constant<bool, true>{});
      else
        add_up(std::integral_constant<bool, false>{});
    }
  }
#pragma unroll
  for (int x = 0; x < NK; ++x) {
    const float total = xor32_sum(sum[x]);
    const int r = key0 + 32 * x + nl;
    if (g == 0 && r < rows) {
      if (there[x])
        w[r] = a.add ? w[r] + total : total;
      else if (!a.add)
        w[r] = 0.f;
    }
  }
}

template <typename T, int D, bool FP4>
hipError_t launch(const WeightArgs& a, int64_t bh, hipStream_t st) {
  const int64_t rows = int64_t(a.width) * a.page_rows;
  const int64_t blocks = (rows + Form<T, D, FP4>::keys - 1) / Form<T, D, FP4>::keys;
  hipLaunchKernelGGL((paged_key_weights_kernel<T, D, FP4>), dim3(unsigned(blocks), unsigned(bh)),
                     dim3(kThreads), 0, st, a);
  return hipGetLastError();
}

int weights_entry(const dx_weights_call* call) {
  const char* const what = "paged_key_weights";
  DX_CHECK_ARG(call, "%s: null call", what);
  const dx_weights_call& c = *call;
  const bool fp4 = c.fp4 != 0;
  DX_CHECK_ARG(c.dtype == DX_BF16 || c.dtype == DX_F16 || (c.dtype == DX_F32 && !fp4),
               "%s: dtype code %lld unsupported%s", what, (long long)c.dtype,
               fp4 ? " (a 4-bit cache serves bf16 and f16)" : "");
  DX_CHECK_ARG(c.D == 64 || c.D == 128 || (c.D == 256 && c.dtype != DX_F32),
               "%s: head_dim %lld (supported: 64, 128, and 256 in 16 bits)", what, (long long)c.D);
  DX_CHECK_ARG(c.B >= 0 && c.Lq >= 0 && c.H > 0 && c.Hkv > 0 && c.width >= 0 && c.n_pages >= 0 &&
                   c.n_pages < (int64_t(1) << 31), "%s: bad shape", what);
  DX_CHECK_ARG(c.H % c.Hkv == 0, "%s: %lld query heads are not a multiple of %lld k/v heads", what,
               (long long)c.H, (long long)c.Hkv);
  DX_CHECK_ARG(c.page_rows > 0 && c.page_rows % 16 == 0 && c.page_rows <= 1024,
               "%s: pages of %lld rows (supported: multiples of 16 up to 1024)", what, (long long)c.page_rows);
  constexpr int64_t kMaxRows = int64_t(1) << 30;
  DX_CHECK_ARG(c.width < kMaxRows / c.page_rows && c.H < kMaxRows && c.Lq < kMaxRows / c.H,
               "%s: a sequence must hold fewer than 2^30 rows and query rows", what);
  // Grid dimensions: y below 2^16, threads in all below 2^32.
  const int64_t blocks = (c.width * c.page_rows + 127) / 128;
  DX_CHECK_ARG(c.B < 65536 && c.Hkv < 65536 && c.B * c.Hkv < 65536,
               "%s: %lld sequences of %lld heads exceed one launch", what, (long long)c.B, (long long)c.Hkv);
  DX_CHECK_ARG(grid_fits(blocks * std::max<int64_t>(c.B * c.Hkv, 1), kThreads), "%s: the call exceeds one launch", what);
  const float scale_log2 = float(c.softmax_scale * 1.4426950408889634);
  DX_CHECK_ARG(std::isfinite(scale_log2), "%s: softmax scale must be finite", what);
  if (c.B == 0 || c.width == 0) return DX_OK;
  const int64_t es = c.dtype == DX_F32 ? 4 : 2, pe = fp4 ? 1 : es;
  auto al = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; };
  DX_CHECK_ARG(c.Lq == 0 || (c.q && c.lse), "%s: null q or lse", what);
  DX_CHECK_ARG(c.block_table && c.cache_lens && c.weights, "%s: null pointer", what);
  DX_CHECK_ARG(c.n_pages == 0 || c.pages, "%s: null pages", what);
  DX_CHECK_ARG(al(c.q) && al(c.pages), "%s: pointers must be 16-byte aligned", what);
  for (const int64_t s : {c.q_sb, c.q_sl, c.q_sh})
    DX_CHECK_ARG(s * es % 16 == 0, "%s: strides must keep head rows 16-byte aligned", what);
  const int64_t p_sr = fp4 ? c.D / 2 : c.p_sr;
  for (const int64_t s : {c.p_sp, p_sr, c.p_sh})
    DX_CHECK_ARG(s * pe % 16 == 0, "%s: strides must keep head rows 16-byte aligned", what);
  WeightArgs a{};
  a.q = static_cast<const char*>(c.q); a.q_sb = c.q_sb * es; a.q_sl = c.q_sl * es; a.q_sh = c.q_sh * es;
  a.lse = static_cast<const float*>(c.lse);
  a.pk = static_cast<const char*>(c.pages);
  a.p_sp = c.p_sp * pe; a.p_sr = p_sr * pe; a.p_sh = c.p_sh * pe;
  a.table = static_cast<const int32_t*>(c.block_table); a.t_sb = c.t_sb;
  a.lens = static_cast<const int32_t*>(c.cache_lens);
  a.w = static_cast<float*>(c.weights); a.w_sb = c.w_sb; a.w_sh = c.w_sh;
  a.add = c.add != 0;
  a.width = int(c.width); a.n_pages = int(c.n_pages); a.page_rows = int(c.page_rows);
  const uint64_t per = uint64_t(c.page_rows / 16);
  a.page_magic = per == 1 ? 0u : uint32_t(((uint64_t(1) << 32) + per - 1) / per);
  a.Hkv = int(c.Hkv); a.H = int(c.H); a.group = int(c.H / c.Hkv); a.Lq = int(c.Lq);
  a.R = int(c.Lq * (c.H / c.Hkv));
  a.scale_log2 = scale_log2;
  if (c.Lq == 0 && a.add) return DX_OK;
  const hipStream_t st = static_cast<hipStream_t>(c.stream);
  const int64_t bh = c.B * c.Hkv;
  auto by_dim = [&](auto t, auto f) {
    using T = decltype(t);
    constexpr bool FP4 = decltype(f)::value;
    if (c.D == 64) return launch<T, 64, FP4>(a, bh, st);
    if (c.D == 128) return launch<T, 128, FP4>(a, bh, st);
    if constexpr (sizeof(T) == 2) return launch<T, 256, FP4>(a, bh, st);
    return hipErrorInvalidValue;
  };
  using Yes = std::integral_constant<bool, true>;
  using No = std::integral_constant<bool, false>;
  const hipError_t e = c.dtype == DX_F32    ? by_dim(float{}, No{})
                       : c.dtype == DX_BF16 ? (fp4 ? by_dim(bf16_t{}, Yes{}) : by_dim(bf16_t{}, No{}))
                                            : (fp4 ? by_dim(f16_t{}, Yes{}) : by_dim(f16_t{}, No{}));
  if (e != hipSuccess) {
    set_error("%s: launch failed: %s", what, hipGetErrorString(e));
    return DX_ELAUNCH;
  }
  return DX_OK;
}

}  // namespace
}  // namespace dx

extern "C" int dx_paged_key_weights(const dx_weights_call* call) { return dx::weights_entry(call); }
