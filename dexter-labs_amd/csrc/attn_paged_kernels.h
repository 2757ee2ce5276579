// Attention over pages of a KV cache on gfx950, and over a prefix that a whole
// batch shares.
//
// Keys of sequence b, in this order: the prefix's rows (shared_prefix_attention
// only), the sequence's own cached rows, its chunk's new keys k[b]. Cached rows
// lie in pages of a pool [2, P, R, H, D] (R a multiple of 16), found through a
// table of page numbers that the kernels read when they run; row counts are
// device integers too, clamped to what the table holds. Masks are those of
// attn_common.h, over the new keys.
//
// Mathematics. Each part p of a row's keys (the prefix, the own keys, and key
// splits of either) gives
//   m_p = max_j s_j,  l_p = sum_j 2^(s_j - m_p),  acc_p = sum_j 2^(s_j - m_p) v_j
// with s_j = (scale log2 e) q.k_j over its visible keys, and the parts join as
//   out = sum_p 2^(m_p - m) acc_p / sum_p 2^(m_p - m) l_p,   m = max_p m_p.
// So the prefix is one attention problem whose rows are the queries of every
// sequence (and, as everywhere here, of every query head of a K/V head): its
// K and V are read once for 32 RW rows, whatever sequence they belong to.
//
// Work. The unit is a 32-key tile of a work item (32 RW rows of one K/V head, of
// one sequence or, for the prefix, of the whole batch). There are two lines of
// items, the own keys' and the prefix's, in one launch, and two ways to deal one
// (attn_paged.hip chooses):
//  * Cut (items that share no keys: one row tile per sequence and head, or for
//    the prefix per head). All tiles of all items form one line, which is cut into
//    equal pieces, one per workgroup, whatever the lengths are: the device cuts it,
//    by the lengths as they are. A piece covers whole items, whose results it writes
//    itself, and at most two broken ones, whose partials paged_merge_kernel joins.
//  * Split (several row tiles read the same keys): every item in S equal ranges
//    of keys, a workgroup each, those of one head next to each other on one XCD,
//    so that they read a key tile at about the same time, through one L2. 16 x 83
//    queries over a shared 8,217-row prefix (24 heads) took 205 us so, and 242 cut
//    (every workgroup at a place of its own in the keys), both with the join.
// With a prefix every row has parts of both lines, and the merge joins them all.
//
// Kernel. A wave owns 32 rows (S^T = K Q^T on 32 x 32 MFMAs, the formulation of
// attn_fwd.hip: a lane holds one row and 16 keys, P^T is the B operand of
// O^T += V^T P^T as it is). A workgroup is RW waves of rows times KW streams,
// which take alternate tiles; the streams' results meet in LDS at the end.
// Tiles land by LDS DMA, 16 rows to a descriptor: pages are multiples of 16
// rows, so 16 rows lie in one page, the page's 64-bit address is scalar
// arithmetic, and rows past the end (or of a table entry that names no page)
// come back as zeros from the descriptor's bound.
//
// What it takes (medians; bf16, D 128 where not said; kernel alone, the join 4-8 us
// more where not said):
//   32 tokens, 8 K/V heads, 300 to 3,000 cached rows each   48 us, 4.4 TB/s
//   the same at D 256                                        84 us, 5.1 TB/s
//   83 queries, 24 heads, 32,768 cached rows                 84 us, 4.8 TB/s
//   64 tokens, 8 K/V heads, 1 to 500 rows, prefix of 4,001   26 us, 3.2 TB/s
//   the same at D 256                                        62 us, 2.6 TB/s
//   the same in fp32                                         95 us, 1.7 TB/s
//   16 x 83, 24 heads, 0 to 332 rows, prefix of 8,217        200 us, 690 TFLOP/s (join 20)
//   8 x 83, 24 heads, D 256, 0 to 332 rows, prefix of 4,001  185 us, 373 TFLOP/s (join 17)
//   4 x 99 in fp32, 24 heads, 0 to 332 rows, prefix of 2,000 157 us, 69 TFLOP/s (join 10)
//   2 x 1,500 causal, 8 K/V heads, 400 to 1,000 rows         79 us, 418 TFLOP/s (no join)
//   the same at D 256                                        178 us, 369 TFLOP/s (join 23)
//   4 x 99 in fp32, 24 heads, 0 to 1,245 rows                62 us, 48 TFLOP/s
// Many keys to a row tile: bound by memory. Otherwise by the chain of a tile (scores,
// softmax, product) in the few waves that registers allow, and by the 4 to 8 us from
// a workgroup's start to its first product: lengths, table, keys and queries, one
// after the other.
#pragma once

#include "attn_paged.h"
#include "attn_tile.h"

#include <float.h>
#include <limits.h>

#include <type_traits>

namespace dx {
namespace {

// The launch arguments where they lie. reread() hides where a pointer to them
// comes from: what is read through its result is read there, and not kept in
// scalar registers from the kernel's start on (they hold a third of what the
// compiler would keep, and spilled the tile loop's).
typedef __attribute__((address_space(4))) const PagedArgs Args;
__device__ __forceinline__ Args* reread(Args* a) {
  asm volatile("" : "+s"(a));
  return a;
}

template <typename T> struct Elem { static constexpr int bytes = 2; };
template <> struct Elem<float> { static constexpr int bytes = 4; };

// Tile rows of RB bytes in LDS: 16-byte chunk c of row r sits at c ^ kswz(r)
// (K) or c ^ vswz(r) (V). K: the swizzles of attn_fwd.hip and attn_wide.hip,
// conflict-free for 32 rows at one chunk. V: 64-byte groups move for the
// transposing 16-bit reads; for 4-byte reads of rows r and r + 4 by the two
// halves of a wave the groups of the odd rows-of-four move by 128 bytes.
template <int RB> __device__ __forceinline__ constexpr int kswz(int r) {
  return RB == 128 ? ((r >> 2) ^ (4 * ((r >> 1) & 1))) & 7 : (r & 15) ^ ((r >> 4) & 1);
}
template <int RB, bool F32> __device__ __forceinline__ constexpr int vswz(int r) {
  if (F32) return 8 * ((r >> 2) & 1);
  return 4 * (RB == 128 ? ((r >> 1) ^ (r >> 2)) & 1 : (r & 3) ^ ((r >> 2) & 1));
}

constexpr int kThreads = kPagedThreads, kWaves = kThreads / 64;

// A workgroup's shape for RW row waves.
template <typename T, int D, int RW> struct Shape {
  static constexpr int RB = D * Elem<T>::bytes;      // bytes of a row
  // Four waves and half of a CU's LDS, so that two workgroups share a CU and one
  // starts, ends or waits while the other computes. One row wave: streams of one
  // wave, as many as fit, 32 keys at a time, whose K and V are single (the next
  // K goes out when S is done, the next V when PV is done). Four: one stream,
  // two stages of 64 keys (each wave then fetches 16 rows, which one page
  // holds), or of 32 where registers and LDS hold no more.
  // Head dim 256 (queries and sums of a wave alone take 192 registers) has a CU
  // to itself: registers for one wave per SIMD (two leave 256, which spill).
  static constexpr int per_cu = D == 256 ? 1 : 2;
  static constexpr int TK = RW == 1 || RB >= 512 ? 32 : 64;
  static constexpr int KW = RW == 1 ? (RB * per_cu >= 1024 ? 2 : 4) : kWaves / RW;
  static constexpr int tile = TK * RB;               // bytes of a K or V tile
  static constexpr int stages = RW == 1 ? 1 : 2;
  static constexpr int stream = stages * 2 * tile;
  // Results on their way between waves: [wave][D' / 8 vectors][64 lanes] of 16
  // bytes, a vector's row padded by 16 (reads across vectors then hit all
  // banks), and {m, l} of 32 rows. D' = D, or half of it where that fits.
  static constexpr int DP = D > 128 ? 128 : D;
  static constexpr int vec = 1040;
  static constexpr int area = DP / 8 * vec + 256;
  static constexpr int body = KW * stream > RW * KW * area ? KW * stream : RW * KW * area;
  // Behind them: which 16-row groups of each stage's tile have no page, and
  // whether a wave's sums hold what is no number.
  static constexpr int flags = body;
  static constexpr int votes = flags + kWaves * 2 * 16;
  static constexpr int lds = votes + 16;
  static_assert(lds * per_cu <= 160 * 1024, "the LDS of a CU");
};

__device__ __forceinline__ int tiles_of(int rows) { return (rows + kPN - 1) / kPN; }

__device__ __forceinline__ uint32_t scan(uint32_t x, int lane) {  // inclusive, over a wave
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const uint32_t y = __shfl_up(x, d);
    if (lane >= d) x += y;
  }
  return x;
}
__device__ __forceinline__ uint32_t lane_of(uint32_t x, int lane) {
  return uint32_t(__builtin_amdgcn_readlane(int(x), lane));
}
__device__ __forceinline__ uint64_t uniform(uint64_t x) {
  return uint64_t(uint32_t(__builtin_amdgcn_readfirstlane(int(x)))) |
         uint64_t(uint32_t(__builtin_amdgcn_readfirstlane(int(x >> 32)))) << 32;
}
__device__ __forceinline__ uint32_t uniform(uint32_t x) {
  return uint32_t(__builtin_amdgcn_readfirstlane(int(x)));
}
__device__ __forceinline__ int own_rows(Args& a, int b) {
  return a.width == 0 ? 0 : min(max(a.lens[b], 0), a.width * a.page_rows);
}
__device__ __forceinline__ int prefix_rows(Args& a) {
  return a.plen ? min(max(*a.plen, 0), a.pwidth * a.page_rows) : 0;
}

// Work on a line is counted in tiles; an item adds `kItemCost` to its tiles, for
// its queries and its result (what a piece of so many tiles costs: half, this and
// twice it take 24.4, 22.0 and 22.8 us at 4 x 99 queries of 24 heads over 0 to 1,245
// rows, 30.6, 30.4 and 32.2 with the join at 4 x 16 over 300 to 3,000). A cut that
// falls among those is taken as one behind the item.
template <typename T, int D, int RW>
constexpr uint32_t kItemCost = Shape<T, D, RW>::KW * Shape<T, D, RW>::TK / kPN * 2;
static_assert(kItemCost<float, 64, 1> <= kMaxItemCost && kItemCost<uint16_t, 64, 1> <= kMaxItemCost,
              "the host's bound of a line's length");

// A line of `total` cut into n pieces, the first `longer` of them q + 1 long.
struct Cut {
  uint32_t q, longer;
  __device__ __forceinline__ Cut(uint32_t total, uint32_t n) : q(total / n), longer(total - q * n) {}
  __device__ __forceinline__ uint32_t start(uint32_t w) const { return w * q + min(w, longer); }
  // The piece that holds position x.
  __device__ __forceinline__ uint32_t piece(uint32_t x) const {
    const uint32_t y = longer * (q + 1);
    return x < y ? x / (q + 1) : longer + (x - y) / q;
  }
};

// The line of the own keys: items (sequence, K/V head), in this order, all rows of one in
// one row tile (attn_paged.hip cuts no other line). The host holds its length below 2^31.
struct OwnLine {
  uint32_t fresh;  // an item's tiles of new keys that some row sees (at least 1, so that it has a
                   // tile and a workgroup), and its cost
  uint32_t total;
  __device__ __forceinline__ void init(Args& a, int lane, uint32_t cost) {
    fresh = uniform(uint32_t(max(tiles_of(end_bounds(a, 0, a.Lq - 1).hi), 1)) + cost);
    uint32_t cached = 0;
    if (a.B == 1) {
      cached = uint32_t(tiles_of(own_rows(a, 0)));
    } else {
      for (int b0 = 0; b0 < a.B; b0 += 64)
        cached += lane_of(scan(b0 + lane < a.B ? tiles_of(own_rows(a, b0 + lane)) : 0, lane), 63);
    }
    total = uniform(uint32_t(a.Hkv) * (cached + uint32_t(a.B) * fresh));
  }
  // The item that holds position `at` of the line, and the place in it.
  __device__ __forceinline__ void locate(Args& a, int lane, uint32_t at, int& b, int& hk, int& t) const {
    b = 0;
    uint32_t before = 0;  // what the sequences before b have, per head
    if (a.B > 1) {
      const uint32_t want = at / uint32_t(a.Hkv);
      uint32_t cached = 0;
      for (int b0 = 0; b0 < a.B; b0 += 64) {
        const uint32_t own = b0 + lane < a.B ? tiles_of(own_rows(a, b0 + lane)) : 0;
        const uint32_t upto = cached + scan(own, lane);
        // Up to and with this lane's sequence.
        const uint32_t end = upto + uint32_t(b0 + lane + 1) * fresh;
        const uint64_t hit = __ballot(b0 + lane < a.B && end > want);
        if (hit) {
          const int j = __builtin_ctzll(hit);
          b = b0 + j;
          before = lane_of(end, j) - lane_of(own, j) - fresh;
          break;
        }
        cached = lane_of(upto, 63);
      }
    }
    b = __builtin_amdgcn_readfirstlane(b);
    const uint32_t in_seq = at - before * uint32_t(a.Hkv);
    const uint32_t per_head = uniform(uint32_t(tiles_of(own_rows(a, b)))) + fresh;
    hk = int(in_seq / per_head);
    t = int(in_seq - uint32_t(hk) * per_head);
  }
};

// One wave's S tile (TK / 32 blocks of 32 keys), softmax step and PV product.
template <typename T, int D, int NS>
struct Tile {
  static constexpr bool F32 = Elem<T>::bytes == 4;
  static constexpr int RB = D * Elem<T>::bytes, KS = RB / 32, DT = D / 32;
  f32x16 acc[DT];
  float m, l;

  __device__ __forceinline__ void reset() {
#pragma unroll
    for (int d = 0; d < DT; ++d) acc[d] = f32x16{};
    m = -INFINITY;
    l = 0.f;
  }
  // S^T = K Q^T of the tile, K fragments read W ahead of the products that use
  // them: left alone the compiler reads each right before its product, which
  // then waits out the LDS latency.
  static __device__ __forceinline__ void scores(uint32_t ka, const u32x4 (&qr)[KS], f32x16 (&s)[NS]) {
    constexpr int N = KS * NS, W = F32 ? 2 : 4;
    auto frag = [&](int i) __attribute__((always_inline)) {
      return lds_read_b128_at((ka ^ (32u * (i / NS))) + 32 * RB * (i % NS));
    };
    __builtin_amdgcn_sched_barrier(0);
    u32x4 kf[W];
#pragma unroll
    for (int i = 0; i < W; ++i) kf[i] = frag(i);
#pragma unroll
    for (int x = 0; x < NS; ++x) s[x] = f32x16{};
#pragma unroll
    for (int i = 0; i < N; ++i) {
      f32x16& sx = s[i % NS];
      if constexpr (F32) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          sx = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(kf[i % W][e]),
                                                    __uint_as_float(qr[i / NS][e]), sx, 0, 0, 0);
      } else {
        sx = Mfma<T>::run(kf[i % W], qr[i / NS], sx);
      }
      if (i + W < N) kf[i % W] = frag(i + W);
    }
    constexpr int kMfma = 0x008, kDsRead = 0x100;
    __builtin_amdgcn_sched_group_barrier(kDsRead, W, 0);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      __builtin_amdgcn_sched_group_barrier(kMfma, F32 ? 4 : 1, 0);
      if (i + W < N) __builtin_amdgcn_sched_group_barrier(kDsRead, 1, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
  }
  // Mask, follow the maximum, exponentials in place. lim: rows of the tile
  // below it are seen (already less 4 g); bad: 16-row groups without a page.
  __device__ __forceinline__ void softmax(f32x16 (&s)[NS], bool masked, int lim, uint32_t bad, float c) {
    if (masked) {
      asm volatile("" : "+v"(lim));
#pragma unroll
      for (int x = 0; x < NS; ++x)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (key_hidden(x, r, lim)) s[x][r] = -INFINITY;
    }
    if (bad) {
#pragma unroll
      for (int x = 0; x < NS; ++x)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (bad >> (2 * x + r / 8) & 1) s[x][r] = -INFINITY;
    }
    float tm[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
    for (int x = 0; x < NS; ++x)
#pragma unroll
      for (int r = 0; r < 16; ++r) tm[r % 4] = fmaxf(tm[r % 4], s[x][r]);
    const float m_new = fmaxf(m, xor32_max(fmaxf(fmaxf(tm[0], tm[1]), fmaxf(tm[2], tm[3]))));
    // The reference may lag behind the maximum by up to 2^8 (what is summed is
    // then up to 2^8 times larger, and divided out): most tiles rescale nothing.
    if (__any((m_new - m) * c > 8.0f)) {
      if (!__all(m == -INFINITY)) {
        const float corr = m == -INFINITY ? 0.f : fast_exp2((m - m_new) * c);
        l *= corr;
#pragma unroll
        for (int d = 0; d < DT; ++d) acc[d] *= corr;
      }
      m = m_new;
    }
    const float mb = m == -INFINITY ? 0.f : m * c;
#pragma unroll
    for (int x = 0; x < NS; ++x)
#pragma unroll
      for (int r = 0; r < 16; ++r) s[x][r] = fast_exp2(__builtin_fmaf(s[x][r], c, -mb));
  }
  __device__ __forceinline__ void pv(uint32_t va, const f32x16 (&s)[NS]) {
    if constexpr (F32) {
      float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int x = 0; x < NS; ++x)
#pragma unroll
        for (int r = 0; r < 16; ++r) part[r % 4] += s[x][r];
      l += (part[0] + part[1]) + (part[2] + part[3]);
      // V read W ahead of the products, as K is in scores().
      constexpr int N = 16 * NS * DT, W = 8;
      auto frag = [&](int i) __attribute__((always_inline)) {
        typedef __attribute__((address_space(3))) float lds_f32;
        const int x = i / DT / 16, r = i / DT % 16;
        return *reinterpret_cast<const lds_f32*>((va ^ (128u * (i % DT))) +
                                                 (32 * x + 8 * (r / 4) + r % 4) * RB);
      };
      __builtin_amdgcn_sched_barrier(0);
      float vf[W];
#pragma unroll
      for (int i = 0; i < W; ++i) vf[i] = frag(i);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        acc[i % DT] = __builtin_amdgcn_mfma_f32_32x32x2f32(vf[i % W], s[i / DT / 16][i / DT % 16],
                                                           acc[i % DT], 0, 0, 0);
        if (i + W < N) vf[i % W] = frag(i + W);
      }
      __builtin_amdgcn_sched_group_barrier(0x100, W, 0);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        if (i + W < N) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
    } else {
      // Probabilities in 16 bits: a lane's scores are then, packed, the operand of the
      // 16-bit product as they lie. Kept in 32 they would need fp32 products, a sixteenth of
      // the peak rate, or a second product of what the rounding left. l sums the rounded ones, so
      // that a row's weights still add up to 1. Against 64 bits, relative to the
      // outputs' norm: 0.0023 in bf16 and 2.9e-4 in f16, of which the result's own rounding
      // is 0.0017 and 2.1e-4.
      u32x4 pk[2 * NS];
      float part[2] = {0.f, 0.f};
#pragma unroll
      for (int u = 0; u < 2 * NS; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t p = Mfma<T>::pack(s[u / 2][8 * (u % 2) + 2 * e], s[u / 2][8 * (u % 2) + 2 * e + 1]);
          pk[u][e] = p;
          part[e & 1] = Mfma<T>::sum2(p, part[e & 1]);
        }
      l += part[0] + part[1];
#pragma unroll
      for (int u = 0; u < 2 * NS; ++u)
#pragma unroll
        for (int d = 0; d < DT; ++d) acc[d] = Mfma<T>::run(v_frag(va, u, d), pk[u], acc[d]);
    }
  }
  // V^T operand: dims 32 d + lane % 32 of keys 16 u + {4 g .. 4 g + 3, 8 + 4 g .. 8 + 4 g + 3}.
  static __device__ __forceinline__ u32x4 v_frag(uint32_t va, int u, int d) {
    const uint32_t vu = (va ^ (64u * d)) + 16 * u * RB;
    const u32x2 lo = lds_read_tr16_at(vu);
    const u32x2 hi = lds_read_tr16_at(vu + 8 * RB);
    return u32x4{lo[0], lo[1], hi[0], hi[1]};
  }

  // An infinity or NaN in V that some rows do not see. Their weight for it is 0, and
  // 0 times that is NaN in the product. Sums with such a value in them (wild_sums) of an
  // item whose rows do not all see the same keys send its workgroup through the item once
  // more, carefully: it looks through the tiles that some rows do not see to their end
  // (poisoned), the rows that see what is no number take it key by key on the vector
  // units (take_poison), it is cleared in LDS (clear_poison), and the product goes on
  // without it. Slow, rolled and in place: rare, and another product beside pv() would
  // cost the loop its registers. Looking through those tiles always cost 5 us of 76 (2 x
  // 1,500 causal queries over 400 to 1,000 cached rows, 16 heads).
  static __device__ __forceinline__ bool poisoned(uint32_t v0, int lane) {
    // Any order does; not unrolled further, to keep its registers few.
    typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
    uint32_t top = 0;
#pragma unroll 4
    for (int i = 0; i < 32 * NS * RB; i += 1024) {
      const u32x4 x = lds_read_b128_at(v0 + i + 16 * lane);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if constexpr (F32)
          top = max(top, x[e] & 0x7fffffffu);
        else
          top = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(
                    __builtin_bit_cast(u16x2, top), __builtin_bit_cast(u16x2, x[e] & 0x7fff7fffu)));
      }
    }
    if constexpr (F32) return __any(top >= 0x7f800000u);
    constexpr uint32_t kInf = std::is_same<T, f16_t>::value ? 0x7c00u : 0x7f80u;
    return __any((top & 0xffffu) >= kInf || top >> 16 >= kInf);
  }
  static __device__ __forceinline__ bool wild(float x) {
    return (__float_as_uint(x) & 0x7f800000u) == 0x7f800000u;
  }
  __device__ __forceinline__ bool wild_sums() const {
    uint32_t top = 0;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) top = max(top, __float_as_uint(acc[d][r]) & 0x7f800000u);
    return top == 0x7f800000u;
  }
  // seen[x]: rows of 32-key block x below it are seen (the same in both lanes of a row).
  __device__ __forceinline__ void take_poison(uint32_t v0, const f32x16 (&s)[NS], const int (&seen)[NS],
                                              int lane) {
    const int g = lane >> 5;
#pragma unroll 1
    for (int k = 0; k < 32 * NS; ++k) {
      // Key k's probability: register 4 (k / 8) + k % 4 of its block, lanes of half (k / 4) % 2.
      const int at = 16 * (k >> 5) + 4 * ((k >> 3) & 3) + (k & 3);
      float p = 0.f;
      int end = 0;
#pragma unroll
      for (int x = 0; x < NS; ++x) {
        end = x == k >> 5 ? seen[x] : end;
#pragma unroll
        for (int r = 0; r < 16; ++r) p = 16 * x + r == at ? s[x][r] : p;
      }
      p = __shfl(p, (lane & 31) + 8 * (k & 4));
      p = (k & 31) < end ? p : -1.f;  // not seen
      const uint32_t row = v0 + k * RB;
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          __builtin_amdgcn_sched_barrier(0);  // one read at a time: few registers
          float v[4];
          if constexpr (F32) {
            const u32x4 x = lds_read_b128_at(row + 16 * ((8 * d + 2 * u + g) ^ vswz<RB, true>(k)));
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = __uint_as_float(x[e]);
          } else {
            typedef __attribute__((address_space(3))) const u32x2 lds_u32x2;
            const u32x2 x = *reinterpret_cast<lds_u32x2*>(row + 16 * ((4 * d + u) ^ vswz<RB, false>(k)) + 8 * g);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = to_f32(T{uint16_t(x[e / 2] >> (16 * (e % 2)))});
          }
#pragma unroll
          for (int e = 0; e < 4; ++e)
            acc[d][4 * u + e] += wild(v[e]) && !(p < 0.f) ? p * v[e] : 0.f;
        }
    }
  }
  // Bytes [from, to) of the tile, a wave's share.
  static __device__ __forceinline__ void clear_poison(uint32_t v0, int from, int to, int lane) {
#pragma unroll 1
    for (int i = from; i < to; i += 1024) {
      u32x4 x = lds_read_b128_at(v0 + i + 16 * lane);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if constexpr (F32) {
          x[e] = wild(__uint_as_float(x[e])) ? 0u : x[e];
        } else {
          constexpr uint32_t kInf = std::is_same<T, f16_t>::value ? 0x7c00u : 0x7f80u;
          x[e] = (x[e] & kInf) == kInf ? x[e] & 0xffff0000u : x[e];
          x[e] = (x[e] >> 16 & kInf) == kInf ? x[e] & 0xffffu : x[e];
        }
      }
      typedef __attribute__((address_space(3))) u32x4 lds_u32x4_w;
      *reinterpret_cast<lds_u32x4_w*>(v0 + i + 16 * lane) = x;
    }
  }
};

// Where an item's keys lie, in scalar registers.
struct Keys {
  uint64_t pk, pv, nk, nv, table;  // pages and new keys of this head; the sequence's table
  int64_t p_sp;
  int p_sr, k_sl, v_sl;
  uint32_t magic;
  int page_rows, n_pages;
  int len, fresh;  // cached rows, new rows that some row of the item sees
  int n_ct;        // 32-key tiles of the cached rows; the new ones' follow

  // The 16 rows from row r0 of the cached ones, or of the new ones: addresses,
  // and how many exist. True where the table names no page for them.
  __device__ __forceinline__ bool find(bool cached, int r0, uint64_t& k, uint64_t& v, int& rows) const {
    rows = max(min((cached ? len : fresh) - r0, 16), 0);
    bool gone = false;
    if (cached) {
      // Entry of these rows (the table has one for every row below len).
      const uint32_t x16 = uint32_t(r0) >> 4;
      uint32_t e = magic ? uint32_t((uint64_t(x16) * magic) >> 32) : x16;
      e = rows > 0 ? e : 0;
      const int page = rows > 0 ? ((const_i32*)table)[e] : 0;
      gone = uint32_t(page) >= uint32_t(n_pages);
      rows = gone ? 0 : rows;
      const uint64_t off = uint64_t(page * p_sp) + uint64_t(uint32_t(r0) - e * uint32_t(page_rows)) * uint32_t(p_sr);
      k = pk + off;
      v = pv + off;
    } else {
      k = nk + uint64_t(uint32_t(r0)) * uint32_t(k_sl);
      v = nv + uint64_t(uint32_t(r0)) * uint32_t(v_sl);
    }
    k = uniform(k);
    v = uniform(v);
    rows = __builtin_amdgcn_readfirstlane(rows);
    return gone;
  }
};

// DMA of `pieces` pieces (RPP rows each) of a 16-row group at `from`, `rows` of
// which exist, into LDS bytes from `to`; r0: the first row within the group, tr0:
// within the tile (multiples of RPP). K swizzle or V swizzle.
template <int RB, bool F32, bool K>
__device__ __forceinline__ void send_rows(uint64_t from, int rows, int step, uint32_t to, int r0, int tr0,
                                          int pieces, int lane) {
  constexpr int CR = RB / 16, RPP = 64 / CR;
  const int lr = lane / CR, lx = lane % CR;  // row and physical chunk within a piece
  const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
      reinterpret_cast<char*>(from), (short)0, rows > 0 ? (rows - 1) * step + RB : 0, kBufWord3);
#pragma unroll
  for (int p = 0; p < pieces; ++p) {
    const int r = r0 + p * RPP + lr, tr = tr0 + p * RPP + lr;
    const uint32_t past = r < rows ? 0u : 0x80000000u;  // past every bound: zeros
    const int swz = K ? kswz<RB>(tr) : vswz<RB, F32>(tr);
    dma_piece_at(rs, to + p * 1024, (uint32_t(r * step) + 16u * (lx ^ swz)) | past);
  }
}

// One workgroup's share of a line: workgroup w of n.
template <typename T, int D, int RW, bool PREFIX, bool SHARED>
__device__ __forceinline__ void run_line(Args* args, char* smem, uint32_t w, uint32_t n,
                                         uint32_t total, uint32_t line_fresh) {
  using Sh = Shape<T, D, RW>;
  constexpr int RB = Sh::RB, KW = Sh::KW, TK = Sh::TK, CR = RB / 16, RPP = 64 / CR;
  using Ti = Tile<T, D, TK / 32>;
  constexpr bool F32 = Ti::F32;
  constexpr int KS = Ti::KS;
  constexpr int UT = TK / kPN;  // 32-key tiles that a stream takes at a time
  const int wid = __builtin_amdgcn_readfirstlane(int(threadIdx.x) >> 6);
  const int stream = wid / RW, wave = wid % RW, lane = int(threadIdx.x) & 63;
  const int g = lane >> 5, nl = lane & 31;

  // Cut: piece w of the line, from tile t0 of an item on. Split: range t0 (for
  // now) of an item.
  const Cut cut(total, n);
  constexpr uint32_t kCost = kItemCost<T, D, RW>;
  uint32_t at = 0;
  int todo = 1;  // what is left of the piece
  int b = 0, hk = 0, rt = 0, t0 = 0;
  int n_rt, splits;
  {
    Args& a = *reread(args);
    const int nrows = PREFIX ? a.B * a.R : a.R;
    n_rt = __builtin_amdgcn_readfirstlane((nrows + 32 * RW - 1) / (32 * RW));
    splits = __builtin_amdgcn_readfirstlane(PREFIX ? a.pre.splits : a.own.splits);
    if (splits == 0) {
      at = uniform(cut.start(w));
      todo = __builtin_amdgcn_readfirstlane(int(cut.start(w + 1) - at));
      if (todo > 0) {
        if (PREFIX) {
          const uint32_t weight = uint32_t(max(tiles_of(prefix_rows(a)), 1)) + kCost;
          hk = int(at / weight);
          t0 = int(at - uint32_t(hk) * weight);
        } else {
          OwnLine{line_fresh, total}.locate(a, lane, at, b, hk, t0);
        }
      }
    } else {
      // Groups (sequence and head) to XCDs in runs; there, range by range of the
      // keys, group by group, late row tiles (most keys under a causal mask) first.
      const uint32_t G = uint32_t(PREFIX ? a.Hkv : a.B * a.Hkv);
      uint32_t grp0 = 0, groups = G, i = w;
      if (G % 8 == 0) {
        groups = G / 8;
        grp0 = w % 8 * groups;
        i = w / 8;
      }
      const uint32_t range = i / (groups * uint32_t(n_rt));
      i -= range * (groups * uint32_t(n_rt));
      const uint32_t grp = i / uint32_t(n_rt);
      rt = n_rt - 1 - int(i - grp * uint32_t(n_rt));
      t0 = int(range);
      b = int((grp0 + grp) / uint32_t(a.Hkv));
      hk = int(grp0 + grp) - b * a.Hkv;
      if (PREFIX) b = 0;
    }
  }
  Record left{0, 0, 0, 0};

  while (todo > 0) {
    // The item and this share's tiles [t0, t1) of it, in scalar registers.
    b = __builtin_amdgcn_readfirstlane(b);
    hk = __builtin_amdgcn_readfirstlane(hk);
    rt = __builtin_amdgcn_readfirstlane(rt);
    t0 = __builtin_amdgcn_readfirstlane(t0);
    const int row0 = rt * 32 * RW;
    Keys keys;
    u32x4 qr[KS];
    float c;
    int my_end = 0, full_end, t1, weight, nt, iters, item;
    uint32_t slot;
    const bool first = t0 == 0;  // this share holds the item's first tile: it leaves the record
    bool active, behind = false;
    int history;  // what the masks call the cache
    {
      Args& a = *reread(args);
      const int nrows = PREFIX ? a.B * a.R : a.R;
      const int pre_len = __builtin_amdgcn_readfirstlane(prefix_rows(a));
      const int own_len = PREFIX ? 0 : __builtin_amdgcn_readfirstlane(own_rows(a, b));
      history = pre_len + own_len;
      EndBounds eb{0, 0};
      if (!PREFIX) eb = end_bounds(a, row0 / a.group, (min(row0 + 32 * RW, nrows) - 1) / a.group);
      full_end = eb.lo;
      keys.len = PREFIX ? pre_len : own_len;
      keys.fresh = __builtin_amdgcn_readfirstlane(eb.hi);
      keys.n_ct = tiles_of(keys.len);
      weight = max(keys.n_ct, 1);
      if (!PREFIX) weight = keys.n_ct + max(tiles_of(keys.fresh), 1);
      item = PREFIX ? hk * n_rt + rt : (b * a.Hkv + hk) * n_rt + rt;
      if (splits == 0) {
        behind = t0 >= weight;  // the piece begins behind the item's tiles
        t1 = __builtin_amdgcn_readfirstlane(max(min(weight - t0, todo), 0) + t0);
        // Without a prefix a workgroup breaks two items at most; with one, every
        // item has parts, and (workgroup, item) grow together.
        slot = SHARED ? w + uint32_t(item) : 2 * w + uint32_t(first);
      } else {
        slot = uint32_t(item) * uint32_t(splits) + uint32_t(t0);
        t1 = int(uint64_t(weight) * uint32_t(t0 + 1) / uint32_t(splits));
        t0 = __builtin_amdgcn_readfirstlane(int(uint64_t(weight) * uint32_t(t0) / uint32_t(splits)));
        t1 = __builtin_amdgcn_readfirstlane(t1);
      }
      const int count = __builtin_amdgcn_readfirstlane(
          max(min(t1, keys.n_ct + tiles_of(keys.fresh)) - t0, 0));  // tiles that exist
      iters = (count + KW * UT - 1) / (KW * UT);  // barrier rounds
      // How many tiles this stream takes (the last may be past t1: it is masked).
      nt = stream < KW && count > stream * UT ? (count - stream * UT + KW * UT - 1) / (KW * UT) : 0;
      keys.pk = reinterpret_cast<uint64_t>(a.pk) + uint64_t(hk * a.p_sh);
      keys.pv = reinterpret_cast<uint64_t>(a.pv) + uint64_t(hk * a.p_sh);
      keys.nk = reinterpret_cast<uint64_t>(a.k) + uint64_t(b * a.k_sb + hk * a.k_sh);
      keys.nv = reinterpret_cast<uint64_t>(a.v) + uint64_t(b * a.v_sb + hk * a.v_sh);
      keys.table = reinterpret_cast<uint64_t>(PREFIX ? a.ptable : a.table + b * a.t_sb);
      keys.p_sp = a.p_sp;
      keys.p_sr = int(a.p_sr);
      keys.k_sl = int(a.k_sl);
      keys.v_sl = int(a.v_sl);
      keys.magic = a.page_magic;
      keys.page_rows = a.page_rows;
      keys.n_pages = a.n_pages;
      c = fmaxf(fabsf(a.scale_log2), FLT_MIN);

      active = row0 + wave * 32 < nrows && stream < KW;  // wave-uniform
    }
    // This lane's row: query head hq of query qi of sequence bq; its queries, and
    // how many of the new keys it sees. Called once the first tiles are on their
    // way: one wait is both's.
    auto load_queries = [&]() __attribute__((always_inline)) {
      Args& a = *reread(args);
      const int nrows = PREFIX ? a.B * a.R : a.R;
      const int row = row0 + wave * 32 + nl;
      const bool rvalid = row < nrows;
      int bq = b;
      const uint32_t r = uint32_t(rvalid ? row : nrows - 1);
      uint32_t rr = r;
      if (PREFIX) {
        bq = int(r / uint32_t(a.R));
        rr = r - uint32_t(bq) * uint32_t(a.R);
      }
      const int qi = int(rr / uint32_t(a.group));
      const int hq = hk * a.group + int(rr - uint32_t(qi) * uint32_t(a.group));
      const char* const qp = a.q + bq * a.q_sb + qi * a.q_sl + hq * a.q_sh + 16 * g;
      const uint32_t flip = a.scale_log2 < 0.f ? (F32 ? 0x80000000u : 0x80008000u) : 0u;
#pragma unroll
      for (int s = 0; s < KS; ++s) qr[s] = *reinterpret_cast<const u32x4*>(qp + 32 * s) ^ flip;
      if (!PREFIX && rvalid) my_end = visible_end(a, qi, history);  // new keys seen
    };

    const uint32_t base = lds_addr(smem) + stream * Sh::stream;
    const uint32_t ka = base + nl * RB + 16 * (g ^ kswz<RB>(nl));
    uint32_t va;
    if (F32) {
      va = base + Sh::tile + 4 * g * RB + 4 * nl + 128 * g;
    } else {
      const int j = lane & 15, r0 = 4 * g + (j >> 2);
      va = base + Sh::tile + r0 * RB + 32 * ((lane >> 4) & 1) + 8 * (j & 3) + 16 * vswz<RB, F32>(r0);
    }
    // A stream's i-th 32-key tile. A 64-key one may begin with the last cached
    // tile and end with the first new one: its halves are found one by one.
    auto tile_at = [&](int i) __attribute__((always_inline)) { return t0 + (KW * i + stream) * UT; };
    Ti ti;
    // Mask of tile i: rows of it that are seen, less 4 g, per 32-key block; all
    // of it where `masked` comes back false.
    auto limits = [&](int t, bool& masked) __attribute__((always_inline)) {
      const bool cached = t < keys.n_ct;
      const int j0 = (cached ? t : t - keys.n_ct) * kPN;
      masked = t >= t1 || (cached ? j0 + kPN > keys.len : j0 + kPN > full_end);
      return t >= t1 ? -64 : (cached ? keys.len : my_end) - j0 - 4 * g;
    };
    // Carefully the second time, if there is one: some sum is no number, and may come
    // from a key that its row does not see. A share behind the item's tiles sums nothing and
    // casts no vote: what keeps the next item's votes behind this one's reads is the
    // barriers of the results' way out, which such a share does not take.
    const bool partly = !PREFIX && !behind && full_end < keys.fresh;
    for (bool careful = false;; careful = true) {
    ti.reset();
    if constexpr (RW == 1) {
      // Streams of one wave: no barriers, each wave waits for its own pieces.
      constexpr int HP = 16 / RPP;  // pieces of a 16-row group
      uint64_t k0, v0, k1, v1;
      int rows0, rows1, sv = 0;
      uint32_t gone = 0;
      auto find = [&](int t) __attribute__((always_inline)) {
        const bool cached = t < keys.n_ct;
        const int r0 = (cached ? t : t - keys.n_ct) * kPN;
        gone = keys.find(cached, r0, k0, v0, rows0) ? 1 : 0;
        gone |= keys.find(cached, r0 + 16, k1, v1, rows1) ? 2 : 0;
        const int sk = __builtin_amdgcn_readfirstlane(cached ? keys.p_sr : keys.k_sl);
        sv = __builtin_amdgcn_readfirstlane(cached ? keys.p_sr : keys.v_sl);
        send_rows<RB, F32, true>(k0, rows0, sk, base, 0, 0, HP, lane);
        send_rows<RB, F32, true>(k1, rows1, sk, base + 16 * RB, 0, 16, HP, lane);
      };
      auto send_v = [&]() __attribute__((always_inline)) {
        send_rows<RB, F32, false>(v0, rows0, sv, base + Sh::tile, 0, 0, HP, lane);
        send_rows<RB, F32, false>(v1, rows1, sv, base + Sh::tile + 16 * RB, 0, 16, HP, lane);
      };
      if (nt > 0) {
        find(tile_at(0));
        send_v();
      }
      if (!careful) load_queries();
      for (int i = 0; i < nt; ++i) {
        const bool more = i + 1 < nt;
        const uint32_t bad = gone;
        wait_vmcnt<2 * HP>();  // K of tile i (its V was sent last)
        f32x16 s[1];
        Ti::scores(ka, qr, s);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // K is read: its place is free
        if (more) find(tile_at(i + 1));
        bool masked;
        const int lim = limits(tile_at(i), masked);
        ti.softmax(s, masked, lim, bad, c);
        if (more) wait_vmcnt<2 * HP>();  // V of tile i (the next K was sent last)
        else wait_vmcnt<0>();
        if (!PREFIX && careful && masked && tile_at(i) >= keys.n_ct && Ti::poisoned(base + Sh::tile, lane)) {
          ti.take_poison(base + Sh::tile, s, {lim + 4 * g}, lane);
          Ti::clear_poison(base + Sh::tile, 0, Sh::tile, lane);
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
        ti.pv(va, s);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if (more) send_v();
      }
    } else {
      // Each wave of a stream fetches TK / RW rows of a tile, all in one page.
      constexpr int WR = TK / RW;
      static_assert(16 % WR == 0 && WR % RPP == 0, "a wave's rows lie in one 16-row group");
      uint32_t* const flags = reinterpret_cast<uint32_t*>(smem + Sh::flags) + stream * 2 * 4;
      auto send_tile = [&](int i) __attribute__((always_inline)) {
        const int st = i & 1;
        const int tr = wave * WR;                 // this wave's first row of the tile
        const int t = tile_at(i) + tr / kPN;      // 32-key tile it lies in
        // Past t1: rows that do not exist (seen rows of the next part may hold
        // infinities, which have no weight of 0 here).
        const bool cached = t < min(keys.n_ct, t1);
        const int r0 = t < t1 ? (cached ? t : t - keys.n_ct) * kPN + tr % kPN / 16 * 16 : INT_MAX;
        uint64_t k, v;
        int rows;
        const bool gone = keys.find(cached, r0, k, v, rows);
        if (lane == 0) flags[4 * st + wave] = gone ? 1u : 0u;
        const int sk = __builtin_amdgcn_readfirstlane(cached ? keys.p_sr : keys.k_sl);
        const int sv = __builtin_amdgcn_readfirstlane(cached ? keys.p_sr : keys.v_sl);
        const uint32_t to = base + st * 2 * Sh::tile + tr * RB;
        send_rows<RB, F32, true>(k, rows, sk, to, tr % 16, tr, WR / RPP, lane);
        send_rows<RB, F32, false>(v, rows, sv, to + Sh::tile, tr % 16, tr, WR / RPP, lane);
      };
      if (nt > 0) send_tile(0);
      if (!careful) load_queries();
      for (int i = 0; i < iters; ++i) {
        // This wave's pieces of tile i have landed; past the barrier the tile
        // is whole, and reads of the stage that is sent to next have returned.
        wait_vmcnt<0>();
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (i + 1 < nt) send_tile(i + 1);
        if (i >= nt) continue;
        const uint32_t st = uint32_t(i & 1) * 2 * Sh::tile;
        const int t = tile_at(i);
        bool masked, masked1 = false;
        int lim = limits(t, masked), lim1 = 0;
        if (UT == 2) lim1 = limits(t + 1, masked1);
        const uint32_t v0 = base + st + Sh::tile;
        // Some row does not see all of the tile's new keys: the whole workgroup looks
        // through its V.
        const bool poison =
            !PREFIX && careful && (masked || masked1) && t + UT > keys.n_ct && Ti::poisoned(v0, lane);
        auto clear = [&]() __attribute__((always_inline)) {
          // Every wave has looked and taken its rows' share, then each clears its
          // part, then all go on.
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
          __builtin_amdgcn_s_barrier();
          asm volatile("" ::: "memory");
          Ti::clear_poison(v0, wave * (Sh::tile / RW), (wave + 1) * (Sh::tile / RW), lane);
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
          __builtin_amdgcn_s_barrier();
          asm volatile("" ::: "memory");
        };
        if (!active) {
          if (poison) clear();
          continue;
        }
        f32x16 s[UT];
        Ti::scores(ka + st, qr, s);
        const u32x4 fl = *reinterpret_cast<const u32x4*>(flags + 4 * (i & 1));
        int seen[UT];
        seen[0] = masked ? lim + 4 * g : kPN;
        if constexpr (UT == 2) {
          seen[1] = masked1 ? lim1 + 4 * g : kPN;
          // Each block by its own limit (its rows count from 0 in both).
          if (masked || masked1) {
            if (!masked) lim = kPN;
            if (!masked1) lim1 = kPN;
            asm volatile("" : "+v"(lim), "+v"(lim1));
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              if (key_hidden(0, r, lim)) s[0][r] = -INFINITY;
              if (key_hidden(0, r, lim1)) s[1][r] = -INFINITY;
            }
          }
          masked = false;
        }
        uint32_t bad = 0;
        if (__builtin_amdgcn_readfirstlane(int(fl[0] | fl[1] | fl[2] | fl[3]))) {
#pragma unroll
          for (int x = 0; x < 4; ++x) bad |= fl[x] << (x * WR / 16);
          bad = uint32_t(__builtin_amdgcn_readfirstlane(int(bad)));
        }
        ti.softmax(s, masked, lim, bad, c);
        if (poison) {
          ti.take_poison(v0, s, seen, lane);
          clear();
        }
        ti.pv(va + st, s);
      }
    }
    if (!partly || careful) break;
    const uint32_t vote = __any(ti.wild_sums()) ? 1u : 0u;
    if (lane == 0) reinterpret_cast<uint32_t*>(smem + Sh::votes)[wid] = vote;
    __syncthreads();
    const u32x4 all = *reinterpret_cast<const u32x4*>(smem + Sh::votes);
    if (__builtin_amdgcn_readfirstlane(int(all[0] | all[1] | all[2] | all[3])) == 0) break;
    }

    if (!behind) {
    // The streams' results meet in LDS. Thread j of a row takes 8 of its
    // values: it reads them from every stream and weighs them by its maximum.
    const bool whole = first && t1 == weight && splits <= 1;
    const float mref = ti.m == -INFINITY ? -INFINITY : ti.m * c;
    const float lsum = xor32_sum(ti.l);
    Args& a = *reread(args);
    const int nrows = PREFIX ? a.B * a.R : a.R;
#pragma unroll
    for (int pass = 0; pass < D / Sh::DP; ++pass) {
      __syncthreads();  // tile reads, or the last pass's reads, are done
      if (stream < KW) {
        char* const area = smem + wid * Sh::area;
#pragma unroll
        for (int d = 0; d < Sh::DP / 32; ++d)
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const f32x16& v = ti.acc[pass * (Sh::DP / 32) + d];
            *reinterpret_cast<f32x4*>(area + (4 * d + u) * Sh::vec + 16 * lane) =
                f32x4{v[4 * u], v[4 * u + 1], v[4 * u + 2], v[4 * u + 3]};
          }
        if (g == 0)
          *reinterpret_cast<f32x2*>(area + Sh::DP / 8 * Sh::vec + 8 * nl) = f32x2{mref, lsum};
      }
      __syncthreads();
      constexpr int CD = Sh::DP / 8;  // 8-value chunks of a row in this pass
#pragma unroll 1
      for (int e = 0; e < (RW * 32 * CD + kThreads - 1) / kThreads; ++e) {
        const int u = e * kThreads + int(threadIdx.x);
        const int r = u / CD, ch = u % CD;  // row of the item, chunk
        if (r < 32 * RW && row0 + r < nrows) {
          const char* const area = smem + (r / 32) * Sh::area;
          f32x2 ml[KW];
          float mm = -INFINITY;
#pragma unroll
          for (int s = 0; s < KW; ++s) {
            ml[s] = *reinterpret_cast<const f32x2*>(area + s * RW * Sh::area + CD * Sh::vec + 8 * (r % 32));
            mm = fmaxf(mm, ml[s][0]);
          }
          const float ref = mm == -INFINITY ? 0.f : mm;
          float l = 0.f;
          f32x4 o[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
          for (int s = 0; s < KW; ++s) {
            const float wt = fast_exp2(ml[s][0] - ref);
            l = __builtin_fmaf(ml[s][1], wt, l);
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const f32x4 v = *reinterpret_cast<const f32x4*>(area + s * RW * Sh::area + ch * Sh::vec +
                                                              16 * (r % 32 + 32 * x));
#pragma unroll
              for (int y = 0; y < 4; ++y) o[x][y] = __builtin_fmaf(v[y], wt, o[x][y]);
            }
          }
          const int col = pass * Sh::DP + 8 * ch;
          if (!SHARED && whole) {
            // The result. No visible key: 0 * inf = NaN, as the reference's softmax.
            const float inv = 1.0f / l;
            const uint32_t rr = uint32_t(row0 + r);
            const int qo = int(rr / uint32_t(a.group));
            const int ho = hk * a.group + int(rr - uint32_t(qo) * uint32_t(a.group));
            char* const op = a.out + b * a.o_sb + qo * a.o_sl + ho * a.o_sh + col * Elem<T>::bytes;
            if constexpr (F32) {
              reinterpret_cast<f32x4*>(op)[0] = o[0] * inv;
              reinterpret_cast<f32x4*>(op)[1] = o[1] * inv;
            } else {
              *reinterpret_cast<u32x4*>(op) =
                  u32x4{Mfma<T>::pack(o[0][0] * inv, o[0][1] * inv), Mfma<T>::pack(o[0][2] * inv, o[0][3] * inv),
                        Mfma<T>::pack(o[1][0] * inv, o[1][1] * inv), Mfma<T>::pack(o[1][2] * inv, o[1][3] * inv)};
            }
          } else {
            const int64_t at_row = int64_t(slot) * (32 * RW) + r;
            f32x4* const po = reinterpret_cast<f32x4*>((PREFIX ? a.pre.o : a.own.o) + at_row * D + col);
            po[0] = o[0];
            po[1] = o[1];
            if (col == 0)
              *reinterpret_cast<f32x2*>((PREFIX ? a.pre.ml : a.own.ml) + at_row * 2) = f32x2{mm, l};
          }
        }
      }
    }
    if (first) {
      // Parts up to the workgroup that holds the item's last tile.
      const int parts = splits ? splits : int(cut.piece(at + uint32_t(weight) - 1)) - int(w) + 1;
      left = Record{item, int(slot), !SHARED && whole ? 0 : parts, 0};
      if ((PREFIX ? a.pre.by_item : a.own.by_item) && threadIdx.x == 0)
        (PREFIX ? a.pre.rec : a.own.rec)[item] = left;
    }
    if (splits) return;
    __syncthreads();  // the results are read: tiles may land again
    }
    const int used = weight + int(kCost) - t0;  // to the next item
    at += uint32_t(used);
    todo = __builtin_amdgcn_readfirstlane(todo - used);
    t0 = 0;
    if (++hk == reread(args)->Hkv) {
      hk = 0;
      ++b;
    }
  }
  if (!SHARED && splits == 0 && !args->own.by_item && threadIdx.x == 0) args->own.rec[w] = left;
}

template <typename T, int D, int RWP, int RWO>
__global__ __launch_bounds__(kThreads, (Shape<T, D, RWO>::per_cu)) void paged_attn_kernel(PagedArgs) {
  Args* const args = (Args*)(uint64_t)__builtin_amdgcn_kernarg_segment_ptr();
  // Touch every line of the arguments up front: one wait instead of one for
  // each line at its first use.
  {
    const uint32_t* const x = (const uint32_t*)(uint64_t)args;
    static_assert(sizeof(PagedArgs) > 5 * 64 && sizeof(PagedArgs) <= 7 * 64, "lines of the arguments");
    typedef __attribute__((address_space(4))) const uint32_t const_u32;
    const_u32* const l = (const_u32*)(uint64_t)x;
    const uint32_t l0 = l[0], l1 = l[16], l2 = l[32], l3 = l[48], l4 = l[64], l5 = l[80],
                   l6 = l[sizeof(PagedArgs) / 4 - 1];
    asm volatile("" ::"s"(l0), "s"(l1), "s"(l2), "s"(l3), "s"(l4), "s"(l5), "s"(l6));
  }
  Args& a = *reread(args);
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int lane = int(threadIdx.x) & 63;
  constexpr uint32_t kCostO = kItemCost<T, D, RWO>, kCostP = kItemCost<T, D, RWP ? RWP : 1>;
  const uint32_t grid = gridDim.x;
  // Workgroups of a cut line: one for what an item costs besides its tiles.
  auto wanted = [&](uint32_t total, uint32_t least, uint32_t most) __attribute__((always_inline)) {
    return min((total + least - 1) / least, most);
  };
  // Workgroup i runs on XCD i % 8: consecutive pieces of a cut line, which may
  // share keys, go to one XCD's L2.
  auto in_runs = [](uint32_t i, uint32_t n) __attribute__((always_inline)) {
    const uint32_t n8 = n & ~7u;
    return i < n8 ? i % 8 * (n8 / 8) + i / 8 : i;
  };
  // The prefix's workgroups come first.
  uint32_t w = blockIdx.x, n_pre = 0, pre_total = 0;
  if constexpr (RWP > 0) {
    if (a.pre.splits) {
      n_pre = uint32_t(a.Hkv) * (uint32_t(a.B * a.R + 32 * RWP - 1) / (32 * RWP)) * uint32_t(a.pre.splits);
      if (w < n_pre) {
        run_line<T, D, RWP, true, true>(args, smem, w, n_pre, 0, 0);
        return;
      }
    } else {
      pre_total = uniform(uint32_t(a.Hkv) * (uint32_t(max(tiles_of(prefix_rows(a)), 1)) + kCostP));
    }
  }
  OwnLine own{};
  uint32_t n_own;
  if (a.own.splits) {
    n_own = uint32_t(a.B * a.Hkv) * (uint32_t(a.R + 32 * RWO - 1) / (32 * RWO)) * uint32_t(a.own.splits);
  } else {
    own.init(a, lane, kCostO);
    n_own = wanted(own.total, kCostO, uint32_t(a.own_n));
  }
  if constexpr (RWP > 0) {
    if (a.pre.splits == 0) {
      n_pre = wanted(pre_total, kCostP, grid);
      if (a.own.splits == 0 && n_pre + n_own > grid) {
        // Both are cut: in proportion to their work. A tile takes four row waves 1.5 times
        // as long as single ones (64 and 128 decoded tokens over prompts of 4,001 and 2,000
        // rows, 8 and 24 K/V heads: 28.4 and 68.4 us counted alike, 26.9 and 59.8 so, 27.0
        // and 57.6 counted double, which a prompt of 12,000 rows pays with 36.6 for 32.4).
        const float pre_work = (RWP > RWO ? 1.5f : 1.0f) * float(pre_total);
        const float part = pre_work / (pre_work + float(own.total));
        n_pre = uint32_t(part * float(grid) + 0.5f);
        n_pre = min(max(n_pre, 1u), grid - 1);
        n_own = grid - n_pre;
      }
      n_pre = uniform(n_pre);
      if (w < n_pre) {
        run_line<T, D, RWP, true, true>(args, smem, in_runs(w, n_pre), n_pre, pre_total, 0);
        return;
      }
    }
  }
  n_own = uniform(n_own);
  w -= n_pre;
  if (w >= n_own) {
    if (RWP == 0 && !a.own.by_item && threadIdx.x == 0) a.own.rec[w] = Record{0, 0, 0, 0};
    return;
  }
  if (a.own.splits == 0) w = in_runs(w, n_own);
  run_line<T, D, RWO, false, (RWP > 0)>(args, smem, w, n_own, own.total, own.fresh);
}

// Join the parts of 8 rows of an item, 64 of their values (blockIdx.z): a lane
// holds 8 values of a row, and the four waves take every fourth part each, so
// that a long list of parts is no long chain of loads; their sums meet in LDS.
// Bound by memory: 20.4 us for the 106 MB of 16 x 83 rows of 24 heads in six parts, 5.2
// TB/s; by its latency, 4-5 us, for decoded tokens.
// blockIdx.x is a record. Prefix items are over all sequences' rows, so the rows
// here may be those of two. A part that saw nothing has l = 0.
template <typename T, int D, int RWP, int RWO>
__global__ __launch_bounds__(256) void paged_merge_kernel(PagedArgs a) {
  __shared__ f32x4 sums[3][64][2];
  __shared__ f32x2 stats[3][64];
  const Record rec = a.own.rec[blockIdx.x];
  if (rec.parts == 0) return;
  const uint32_t n_rt = uint32_t(a.R + 32 * RWO - 1) / (32 * RWO);
  constexpr int CD = 8;  // 8-value chunks of a row here: 64 values
  const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) >> 6), lane = int(threadIdx.x) & 63;
  const int ch = int(blockIdx.z) * CD + lane % CD;
  const int in_item = int(blockIdx.y) * 8 + lane / CD;
  const uint32_t bh = uint32_t(rec.item) / n_rt, rt = uint32_t(rec.item) - bh * n_rt;
  const int b = int(bh / uint32_t(a.Hkv)), hk = int(bh) - b * a.Hkv;
  const int row = int(rt) * 32 * RWO + in_item;
  if (int(rt) * 32 * RWO + int(blockIdx.y) * 8 >= a.R) return;  // no row of this workgroup exists
  const bool valid = row < a.R;
  float m = -INFINITY, l = 0.f;
  f32x4 o[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
  auto add = [&](const f32x2 ml, const f32x4 (&v)[2], float ref) __attribute__((always_inline)) {
    const float wt = fast_exp2(ml[0] - ref);
    l = __builtin_fmaf(ml[1], wt, l);
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int y = 0; y < 4; ++y) o[x][y] = __builtin_fmaf(v[x][y], wt, o[x][y]);
  };
  auto rescale = [&](float mm) __attribute__((always_inline)) {
    const float ref = mm == -INFINITY ? 0.f : mm, keep = fast_exp2(m - ref);
    l *= keep;
    o[0] *= keep;
    o[1] *= keep;
    m = mm;
    return ref;
  };
  if (valid) {
    // The row's parts of the prefix, then those of its own keys.
    int pre_parts = 0;
    int64_t pre_row = 0;
    if constexpr (RWP > 0) {
      const uint32_t pr = uint32_t(b) * uint32_t(a.R) + uint32_t(row);
      const uint32_t pre_rt = uint32_t(a.B * a.R + 32 * RWP - 1) / (32 * RWP);
      const Record p = a.pre.rec[uint32_t(hk) * pre_rt + pr / (32 * RWP)];
      pre_parts = p.parts;
      pre_row = int64_t(p.slot) * (32 * RWP) + pr % (32 * RWP);
    }
    // Of a cut line without a prefix, a broken item's first part is its
    // workgroup's odd slot, the others are the next workgroups' even ones.
    const bool broken = RWP == 0 && a.own.splits == 0;
    const int64_t own_row = int64_t(rec.slot) * (32 * RWO) + in_item;
    const int parts = pre_parts + rec.parts;
    // This wave's parts, four at a time: their loads do not wait for one another.
    for (int p0 = wave; p0 < parts; p0 += 16) {
      f32x2 ml[4];
      f32x4 v[4][2];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int p = p0 + 4 * x, q = p - pre_parts;
        ml[x] = f32x2{-INFINITY, 0.f};
        v[x][0] = v[x][1] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (p < parts) {
          const bool pre = RWP > 0 && q < 0;
          const int64_t at = pre ? pre_row + int64_t(p) * (32 * RWP)
                                 : own_row + int64_t(broken ? (q ? 2 * q - 1 : 0) : q) * (32 * RWO);
          ml[x] = *reinterpret_cast<const f32x2*>((pre ? a.pre.ml : a.own.ml) + at * 2);
          const f32x4* const from = reinterpret_cast<const f32x4*>((pre ? a.pre.o : a.own.o) + at * D + 8 * ch);
          v[x][0] = from[0];
          v[x][1] = from[1];
        }
      }
      float mm = m;
#pragma unroll
      for (int x = 0; x < 4; ++x) mm = fmaxf(mm, ml[x][0]);
      const float ref = rescale(mm);
#pragma unroll
      for (int x = 0; x < 4; ++x) add(ml[x], v[x], ref);
    }
  }
  if (wave > 0) {
    stats[wave - 1][lane] = f32x2{m, l};
    sums[wave - 1][lane][0] = o[0];
    sums[wave - 1][lane][1] = o[1];
  }
  __syncthreads();
  if (wave > 0 || !valid) return;
  float mm = m;
#pragma unroll
  for (int x = 0; x < 3; ++x) mm = fmaxf(mm, stats[x][lane][0]);
  const float ref = rescale(mm);
#pragma unroll
  for (int x = 0; x < 3; ++x) add(stats[x][lane], sums[x][lane], ref);
  const float inv = 1.0f / l;  // no visible key: 0 * inf = NaN
  const int qi = int(uint32_t(row) / uint32_t(a.group)), hq = hk * a.group + row - qi * a.group;
  char* const op = a.out + b * a.o_sb + qi * a.o_sl + hq * a.o_sh + 8 * ch * Elem<T>::bytes;
  if constexpr (Elem<T>::bytes == 4) {
    reinterpret_cast<f32x4*>(op)[0] = o[0] * inv;
    reinterpret_cast<f32x4*>(op)[1] = o[1] * inv;
  } else {
    *reinterpret_cast<u32x4*>(op) =
        u32x4{Mfma<T>::pack(o[0][0] * inv, o[0][1] * inv), Mfma<T>::pack(o[0][2] * inv, o[0][3] * inv),
              Mfma<T>::pack(o[1][0] * inv, o[1][1] * inv), Mfma<T>::pack(o[1][2] * inv, o[1][3] * inv)};
  }
}

template <typename T, int D, int RWP, int RWO>
hipError_t launch_form(const PagedArgs& a, const PagedPlan& p, hipStream_t st) {
  constexpr int lds_own = Shape<T, D, RWO>::lds, lds_pre = RWP ? Shape<T, D, RWP ? RWP : 1>::lds : 0;
  constexpr int lds = lds_own > lds_pre ? lds_own : lds_pre;
  const void* fn = reinterpret_cast<const void*>(&paged_attn_kernel<T, D, RWP, RWO>);
  hipError_t e = opt_in_lds(fn, lds);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((paged_attn_kernel<T, D, RWP, RWO>), dim3(unsigned(p.grid)), dim3(kThreads), lds,
                     st, a);
  e = hipGetLastError();
  if (e != hipSuccess || !p.merge) return e;
  hipLaunchKernelGGL((paged_merge_kernel<T, D, RWP, RWO>), dim3(unsigned(p.own_recs), 4 * RWO, D / 64),
                     dim3(256), 0, st, a);
  return hipGetLastError();
}

template <typename T, int D>
hipError_t launch_paged(const PagedArgs& a, const PagedPlan& p, hipStream_t st) {
  if (p.rw_pre == 0)
    return p.rw_own == 1 ? launch_form<T, D, 0, 1>(a, p, st) : launch_form<T, D, 0, 4>(a, p, st);
  if (p.rw_pre == 1) return launch_form<T, D, 1, 1>(a, p, st);
  return p.rw_own == 1 ? launch_form<T, D, 4, 1>(a, p, st) : launch_form<T, D, 4, 4>(a, p, st);
}

}  // namespace
}  // namespace dx
