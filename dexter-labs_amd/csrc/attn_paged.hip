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
// Kernel. A wave owns 32 rows (S^T = K Q^T on 32 x 32 MFMAs, the formulation of
// attn_fwd.hip: a lane holds one row and 16 keys, P^T is the B operand of
// O^T += V^T P^T as it is). A workgroup is RW waves of rows times KW streams,
// which take alternate 32-key tiles; the streams' results meet in LDS at the
// end. Tiles land by LDS DMA, 16 rows to a descriptor: pages are multiples of
// 16 rows, so 16 rows lie in one page, the page's 64-bit address is scalar
// arithmetic, and rows past the end (or of a table entry that names no page)
// come back as zeros from the descriptor's bound.
#include "attn_tile.h"

#include <float.h>

#include <algorithm>
#include <cmath>

namespace dx {
namespace {

constexpr int kPN = 32;  // keys per tile

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
  // Partials, by parts: of the own keys ([unit][split], a unit being 32 rows of
  // a (K/V head, sequence)) and of the prefix (a unit being 32 of all B R rows
  // of a K/V head). ws_o: [64 lanes] x 16 bytes per 32 x 8 block, in
  // accumulator order; ws_ml: {m, l} per row.
  float* own_o; float* own_ml; int own_splits, own_blocks;  // blocks: units per (head, sequence)
  float* pre_o; float* pre_ml; int pre_splits, pre_blocks;
};

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

template <typename T, int D, int RW> struct Shape {
  static constexpr int RB = D * Elem<T>::bytes;      // bytes of a row
  static constexpr int KW = RB >= 512 ? 2 : RW == 4 ? 2 : 4;
  static constexpr int NW = RW * KW;
  static constexpr int stages = 2;
  static constexpr int tile = kPN * RB;              // bytes of a K or V tile
  static constexpr int stage = 2 * tile;
  static constexpr int stream = stages * stage;
  static constexpr int hand = (1 + D / 8) * 1024;    // bytes a wave hands over: m, l and acc
  static constexpr int lds = KW * stream > KW / 2 * RW * hand ? KW * stream : KW / 2 * RW * hand;
};

// Where a 16-row group of keys lies, and how many of its rows exist.
struct Rows16 {
  const char* k; const char* v;
  int rows;
};

template <typename T, int D, int RW, bool PREFIX>
__global__ __launch_bounds__((64 * Shape<T, D, RW>::NW), 1) void paged_attn_kernel(PagedArgs a) {
  using Sh = Shape<T, D, RW>;
  constexpr bool F32 = Elem<T>::bytes == 4;
  constexpr int RB = Sh::RB, KW = Sh::KW, ST = Sh::stages;
  constexpr int KS = RB / 32, DT = D / 32, CR = RB / 16, RPP = 64 / CR;
  constexpr int PW = kPN / RPP / RW;  // DMA pieces (of K, and of V) a wave sends per tile
  static_assert(PW >= 1, "every wave sends whole pieces");
  extern __shared__ __attribute__((aligned(16))) char smem[];

  // Work item: (sequence and K/V head, row tile, key split); late row tiles,
  // which see the most keys under a causal mask, first. Workgroup i runs on
  // XCD i % 8: with a multiple of 8 groups each XCD takes a run of them, so
  // that what reads the same keys goes through one L2.
  const int splits = PREFIX ? a.pre_splits : a.own_splits;
  const int nrows = PREFIX ? a.B * a.R : a.R;
  const int n_rt = (nrows + 32 * RW - 1) / (32 * RW);
  int b, hk, rt, split;
  {
    const uint32_t i = blockIdx.x, G = uint32_t(PREFIX ? a.Hkv : a.B * a.Hkv);
    uint32_t grp, rank;
    if (G % 8 == 0) {
      const uint32_t g8 = G / 8, slot = i / 8;
      rank = slot / g8;
      grp = i % 8 * g8 + (slot - rank * g8);
    } else {
      rank = i / G;
      grp = i - rank * G;
    }
    const uint32_t t = rank / uint32_t(splits);
    split = int(rank - t * uint32_t(splits));
    rt = n_rt - 1 - int(t);
    b = PREFIX ? 0 : int(grp / uint32_t(a.Hkv));
    hk = int(grp) - b * a.Hkv;
  }
  const int wid = __builtin_amdgcn_readfirstlane(int(threadIdx.x) >> 6);
  const int stream = wid / RW, wave = wid % RW, lane = int(threadIdx.x) & 63;
  const int g = lane >> 5, n = lane & 31;
  const int row0 = rt * 32 * RW;                   // first row of the item
  const int row = row0 + wave * 32 + n;
  const bool rvalid = row < nrows;
  const bool active = row0 + wave * 32 < nrows;    // wave-uniform

  // Key range: cached tiles, then tiles of the new keys; a tile never straddles.
  const int pre_len = a.plen ? min(max(*a.plen, 0), a.pwidth * a.page_rows) : 0;
  const int own_len = PREFIX || a.width == 0 ? 0 : min(max(a.lens[b], 0), a.width * a.page_rows);
  const int len = __builtin_amdgcn_readfirstlane(PREFIX ? pre_len : own_len);
  const int history = pre_len + own_len;           // what the masks call the cache
  EndBounds eb{0, 0};
  if (!PREFIX) eb = end_bounds(a, row0 / a.group, (min(row0 + 32 * RW, nrows) - 1) / a.group);
  const int n_ct = (len + kPN - 1) / kPN;
  const int n_tiles = n_ct + (eb.hi + kPN - 1) / kPN;
  const int t_begin = int(uint32_t(split) * uint32_t(n_tiles) / uint32_t(splits));
  const int t_end = int(uint32_t(split + 1) * uint32_t(n_tiles) / uint32_t(splits));
  const int iters = (t_end - t_begin + KW - 1) / KW;             // barrier rounds
  const int nt = (t_end - t_begin - stream + KW - 1) / KW;       // this stream's tiles

  // This lane's row: query head h0 + gq of query qi of sequence bq.
  int bq = b, qi = 0, hq = 0;
  {
    const uint32_t r = uint32_t(rvalid ? row : nrows - 1);
    uint32_t rr = r;
    if (PREFIX) {
      bq = int(r / uint32_t(a.R));
      rr = r - uint32_t(bq) * uint32_t(a.R);
    }
    qi = int(rr / uint32_t(a.group));
    hq = hk * a.group + int(rr - uint32_t(qi) * uint32_t(a.group));
  }
  u32x4 qr[KS];
  {
    const char* const qp = a.q + bq * a.q_sb + qi * a.q_sl + hq * a.q_sh + 16 * g;
    const uint32_t flip = a.scale_log2 < 0.f ? (F32 ? 0x80000000u : 0x80008000u) : 0u;
#pragma unroll
    for (int s = 0; s < KS; ++s) qr[s] = *reinterpret_cast<const u32x4*>(qp + 32 * s) ^ flip;
  }
  const int my_end = PREFIX || !rvalid ? 0 : visible_end(a, qi, history);  // new keys seen

  const int32_t* const table = PREFIX ? a.ptable : a.table + b * a.t_sb;
  // Page number of the 16 cached rows from r0 (a multiple of 16 below len),
  // and the first of them within it.
  auto page_at = [&](int r0, int& in_page) __attribute__((always_inline)) {
    const uint32_t x = uint32_t(r0) >> 4;
    const uint32_t e = a.page_magic ? uint32_t((uint64_t(x) * a.page_magic) >> 32) : x;
    in_page = r0 - int(e) * a.page_rows;
    return ((const_i32*)reinterpret_cast<uint64_t>(table))[e];
  };
  const uint32_t base = lds_addr(smem) + stream * Sh::stream;
  const int lr = lane / CR, lx = lane % CR;  // row and physical chunk within a piece
  uint32_t gone = 0;  // two bits per stage: halves of its tile whose table entry names no page
  // Send this wave's pieces of the stream's tile i: rows [32 / RW wave, ...).
  auto send = [&](int i) __attribute__((always_inline)) {
    const int t = t_begin + KW * i + stream;
    const int st = i % ST;
    const bool cached = t < n_ct;
    const int first = (cached ? t : t - n_ct) * kPN;
    const int count = (cached ? len : eb.hi) - first;  // rows of the tile that exist
    Rows16 h[2];
    uint32_t bad = 0;
    if (cached) {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        h[x] = {a.q, a.q, 0};
        const int rows = min(count - 16 * x, 16);
        if (rows > 0) {
          int in_page;
          const int page = page_at(first + 16 * x, in_page);
          if (uint32_t(page) < uint32_t(a.n_pages)) {
            const int64_t off = page * a.p_sp + in_page * a.p_sr + hk * a.p_sh;
            h[x] = {a.pk + off, a.pv + off, rows};
          } else {
            bad |= 1u << x;
          }
        }
      }
    } else {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int64_t r = first + 16 * x;
        h[x] = {a.k + b * a.k_sb + hk * a.k_sh + r * a.k_sl,
                a.v + b * a.v_sb + hk * a.v_sh + r * a.v_sl, max(min(count - 16 * x, 16), 0)};
      }
    }
    gone = (gone & ~(3u << (2 * st))) | bad << (2 * st);
    const int sk = int(cached ? a.p_sr : a.k_sl), sv = int(cached ? a.p_sr : a.v_sl);
    const uint32_t at = base + st * Sh::stage;
#pragma unroll
    for (int p = 0; p < PW; ++p) {
      const int piece = wave * PW + p;                 // of the tile's PW * RW
      const int x = piece * RPP / 16;                  // half it lies in
      const Rows16 hx = x ? h[1] : h[0];
      const int r = piece * RPP % 16 + lr;             // this lane's row of the half
      const __amdgpu_buffer_rsrc_t rk = __builtin_amdgcn_make_buffer_rsrc(
          const_cast<char*>(hx.k), (short)0, hx.rows > 0 ? (hx.rows - 1) * sk + RB : 0, kBufWord3);
      const __amdgpu_buffer_rsrc_t rv = __builtin_amdgcn_make_buffer_rsrc(
          const_cast<char*>(hx.v), (short)0, hx.rows > 0 ? (hx.rows - 1) * sv + RB : 0, kBufWord3);
      const int tr = piece * RPP + lr;                 // row of the tile
      const uint32_t past = r < hx.rows ? 0u : 0x80000000u;  // past every bound: zeros
      dma_piece_at(rk, at + piece * 1024, (uint32_t(r * sk) + 16u * (lx ^ kswz<RB>(tr))) | past);
      dma_piece_at(rv, at + Sh::tile + piece * 1024,
                   (uint32_t(r * sv) + 16u * (lx ^ vswz<RB, F32>(tr))) | past);
    }
  };
  for (int i = 0; i < ST - 1 && i < nt; ++i) send(i);

  // c > 0: masked scores are -inf and exp2(-inf c) has to be 0 (a zero scale
  // weighs every visible key alike: exp2(~0)).
  const float c = fmaxf(fabsf(a.scale_log2), FLT_MIN);
  const uint32_t ka = base + n * RB + 16 * (g ^ kswz<RB>(n));
  uint32_t va;
  if (F32) {
    va = base + Sh::tile + 4 * g * RB + 4 * n + 128 * g;
  } else {
    const int j = lane & 15, r0 = 4 * g + (j >> 2);
    va = base + Sh::tile + r0 * RB + 32 * ((lane >> 4) & 1) + 8 * (j & 3) + 16 * vswz<RB, F32>(r0);
  }

  f32x16 acc[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d) acc[d] = f32x16{};
  float m = -INFINITY, l = 0.f;
  for (int i = 0; i < iters; ++i) {
    // This wave's pieces of tile i have landed; past the barrier the tile is
    // whole, and reads of the stage that is sent to next have returned.
    wait_vmcnt<0>();
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (i + ST - 1 < nt) send(i + ST - 1);
    if (i >= nt || !active) continue;
    const uint32_t st = uint32_t(i % ST) * Sh::stage;
    f32x16 s = f32x16{};
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      const u32x4 kf = lds_read_b128_at((ka + st) ^ (32u * k));
      if constexpr (F32) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          s = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(kf[e]),
                                                   __uint_as_float(qr[k][e]), s, 0, 0, 0);
      } else {
        s = Mfma<T>::run(kf, qr[k], s);
      }
    }
    const int t = t_begin + KW * i + stream;
    const bool cached = t < n_ct;
    const int j0 = (cached ? t : t - n_ct) * kPN;
    const uint32_t bad = gone >> (2 * (i % ST)) & 3;
    if (cached ? j0 + kPN > len : j0 + kPN > eb.lo) {
      int lim = (cached ? len : my_end) - j0 - 4 * g;
      asm volatile("" : "+v"(lim));
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (key_hidden(0, r, lim)) s[r] = -INFINITY;
    }
    if (bad) {
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (bad >> (r / 8) & 1) s[r] = -INFINITY;
    }
    float tm[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
    for (int r = 0; r < 16; ++r) tm[r % 4] = fmaxf(tm[r % 4], s[r]);
    const float m_new = fmaxf(m, xor32_max(fmaxf(fmaxf(tm[0], tm[1]), fmaxf(tm[2], tm[3]))));
    if (__any(m_new > m)) {
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
    for (int r = 0; r < 16; ++r) s[r] = fast_exp2(__builtin_fmaf(s[r], c, -mb));
    if constexpr (F32) {
      float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int r = 0; r < 16; ++r) part[r % 4] += s[r];
      l += (part[0] + part[1]) + (part[2] + part[3]);
#pragma unroll
      for (int r = 0; r < 16; ++r)
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          typedef __attribute__((address_space(3))) float lds_f32;
          const float vf = *reinterpret_cast<const lds_f32*>(
              ((va + st) ^ (128u * d)) + (8 * (r / 4) + r % 4) * RB);
          acc[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(vf, s[r], acc[d], 0, 0, 0);
        }
    } else {
      u32x4 pk[2];
      float part[2] = {0.f, 0.f};
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t p = Mfma<T>::pack(s[8 * u + 2 * e], s[8 * u + 2 * e + 1]);
          pk[u][e] = p;
          part[e & 1] = Mfma<T>::sum2(p, part[e & 1]);
        }
      l += part[0] + part[1];
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          const uint32_t vu = ((va + st) ^ (64u * d)) + 16 * u * RB;
          const u32x2 lo = lds_read_tr16_at(vu);
          const u32x2 hi = lds_read_tr16_at(vu + 8 * RB);
          acc[d] = Mfma<T>::run(u32x4{lo[0], lo[1], hi[0], hi[1]}, pk[u], acc[d]);
        }
    }
  }

  // The streams' results meet: in each round the upper half hands (m, l, acc)
  // to the lower, lane by lane ([vector][lane], whole 1 KB rows).
  float mref = m == -INFINITY ? -INFINITY : m * c;
  f32x4* const x = reinterpret_cast<f32x4*>(smem);
#pragma unroll
  for (int half = KW / 2; half >= 1; half /= 2) {
    __syncthreads();  // tile reads, or the last round's reads, are done
    f32x4* const hand = x + ((stream % half) * RW + wave) * (Sh::hand / 16) + lane;
    if (stream >= half && stream < 2 * half) {
      hand[0] = f32x4{mref, l, 0.f, 0.f};
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int u = 0; u < 4; ++u)
          hand[64 * (1 + 4 * d + u)] =
              f32x4{acc[d][4 * u], acc[d][4 * u + 1], acc[d][4 * u + 2], acc[d][4 * u + 3]};
    }
    __syncthreads();
    if (stream < half) {
      const f32x4 o = hand[0];
      const float mm = fmaxf(mref, o[0]), ref = mm == -INFINITY ? 0.f : mm;
      const float w0 = fast_exp2(mref - ref), w1 = fast_exp2(o[0] - ref);
      l = __builtin_fmaf(l, w0, o[1] * w1);
      mref = mm;
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const f32x4 v = hand[64 * (1 + 4 * d + u)];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            acc[d][4 * u + e] = __builtin_fmaf(acc[d][4 * u + e], w0, v[e] * w1);
        }
    }
  }
  if (stream != 0 || !active) return;
  l = xor32_sum(l);

  float* const part_o = PREFIX ? a.pre_o : a.own_o;
  if (part_o == nullptr) {
    // The only part: the result. No visible key: 0 * inf = NaN, as the
    // reference's softmax.
    if (!rvalid) return;
    const float inv = 1.0f / l;
    char* const op = a.out + bq * a.o_sb + qi * a.o_sl + hq * a.o_sh + 4 * g * Elem<T>::bytes;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const f32x4 r = {acc[d][4 * u] * inv, acc[d][4 * u + 1] * inv, acc[d][4 * u + 2] * inv,
                         acc[d][4 * u + 3] * inv};
        if constexpr (F32)
          *reinterpret_cast<f32x4*>(op + 128 * d + 32 * u) = r;
        else
          *reinterpret_cast<u32x2*>(op + 64 * d + 16 * u) =
              u32x2{Mfma<T>::pack(r[0], r[1]), Mfma<T>::pack(r[2], r[3])};
      }
    return;
  }
  const int blk = rt * RW + wave;
  const int64_t unit = (PREFIX ? int64_t(hk) * a.pre_blocks + blk
                               : (int64_t(hk) * a.B + b) * a.own_blocks + blk) * splits + split;
  float* const part_ml = (PREFIX ? a.pre_ml : a.own_ml) + unit * 64;
  if (g == 0) *reinterpret_cast<f32x2*>(part_ml + 2 * n) = f32x2{mref, l};
  if (__all(l == 0.f)) return;  // nothing seen: the merge does not read acc where l is 0
  f32x4* const po = reinterpret_cast<f32x4*>(part_o) + unit * (8 * D) + lane;
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int u = 0; u < 4; ++u)
      po[64 * (4 * d + u)] =
          f32x4{acc[d][4 * u], acc[d][4 * u + 1], acc[d][4 * u + 2], acc[d][4 * u + 3]};
}

// Join the parts of 32 rows of one (K/V head, sequence), 32 of their D values
// per workgroup (blockIdx.y): thread (u, lane) holds 4 values of row lane % 32.
// Prefix parts are numbered over all sequences' rows, so a unit's rows may
// begin in the middle of one. A part that saw nothing has l = 0 and is not read.
template <typename T, int D>
__global__ __launch_bounds__(256) void paged_merge_kernel(PagedArgs a) {
  const int lane = int(threadIdx.x) & 63, u = int(threadIdx.x) >> 6, d = int(blockIdx.y);
  const int g = lane >> 5, n = lane & 31;
  uint32_t i = blockIdx.x;
  const int blk = int(i % uint32_t(a.own_blocks));
  i /= uint32_t(a.own_blocks);
  const int b = int(i % uint32_t(a.B)), hk = int(i / uint32_t(a.B));
  const int row = blk * 32 + n;
  if (row >= a.R) return;
  const int64_t own = ((int64_t(hk) * a.B + b) * a.own_blocks + blk) * a.own_splits;
  const uint32_t pr = uint32_t(b) * uint32_t(a.R) + uint32_t(row);
  const int64_t pre = (int64_t(hk) * a.pre_blocks + (pr >> 5)) * a.pre_splits;
  const int pn = int(pr & 31);
  const f32x2* const own_ml = reinterpret_cast<const f32x2*>(a.own_ml) + own * 32 + n;
  const f32x2* const pre_ml = reinterpret_cast<const f32x2*>(a.pre_ml) + pre * 32 + pn;
  float m = -INFINITY;
  for (int s = 0; s < a.own_splits; ++s) m = fmaxf(m, own_ml[32 * s][0]);
  for (int s = 0; s < a.pre_splits; ++s) m = fmaxf(m, pre_ml[32 * s][0]);
  const f32x4* const own_o = reinterpret_cast<const f32x4*>(a.own_o) + own * (8 * D) +
                             64 * (4 * d + u) + lane;
  const f32x4* const pre_o = reinterpret_cast<const f32x4*>(a.pre_o) + pre * (8 * D) +
                             64 * (4 * d + u) + 32 * g + pn;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  float l = 0.f;
  auto join = [&](const f32x2 ml, const f32x4* o) __attribute__((always_inline)) {
    if (ml[1] == 0.f) return;
    const float w = fast_exp2(ml[0] - m);
    l = __builtin_fmaf(ml[1], w, l);
    const f32x4 v = *o;
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] = __builtin_fmaf(v[e], w, acc[e]);
  };
  for (int s = 0; s < a.pre_splits; ++s) join(pre_ml[32 * s], pre_o + int64_t(s) * (8 * D));
  for (int s = 0; s < a.own_splits; ++s) join(own_ml[32 * s], own_o + int64_t(s) * (8 * D));
  const float inv = 1.0f / l;  // no visible key: 0 * inf = NaN
  const int qi = row / a.group, hq = hk * a.group + row % a.group;
  char* const op = a.out + b * a.o_sb + qi * a.o_sl + hq * a.o_sh +
                   (32 * d + 8 * u + 4 * g) * Elem<T>::bytes;
  const f32x4 r = {acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv};
  if constexpr (Elem<T>::bytes == 4)
    *reinterpret_cast<f32x4*>(op) = r;
  else
    *reinterpret_cast<u32x2*>(op) = u32x2{Mfma<T>::pack(r[0], r[1]), Mfma<T>::pack(r[2], r[3])};
}

// ---------------------------------------------------------------------------
// Host side: the plan and the launches.
// ---------------------------------------------------------------------------
struct PagedPlan {
  int rw_own, rw_pre;        // row waves of a workgroup
  int own_splits, pre_splits;  // pre_splits 0: no prefix
  int64_t own_blocks, pre_blocks;
  int64_t own_units, pre_units;  // 32-row partials (0: the kernel writes the result)
};

int row_waves(int64_t rows) { return rows <= 32 ? 1 : rows <= 64 ? 2 : 4; }

constexpr int kPagedMaxSplits = 64;

int split_count(int64_t items, int64_t tiles, int cus) {
  const int64_t want = (cus + items - 1) / std::max<int64_t>(items, 1);
  return int(std::max<int64_t>(1, std::min({want, tiles / 8, int64_t(kPagedMaxSplits)})));
}

PagedPlan plan_paged(int64_t B, int64_t Lq, int64_t Lk, int64_t H, int64_t Hkv, int64_t own_rows,
                     int64_t pre_rows, bool prefix, int cus) {
  PagedPlan p{};
  const int64_t R = Lq * (H / Hkv);
  auto tiles = [](int64_t rows) { return (rows + kPN - 1) / kPN; };
  auto row_tiles = [](int64_t rows, int rw) { return (rows + 32 * rw - 1) / (32 * rw); };
  p.rw_own = row_waves(R);
  p.own_blocks = (R + 31) / 32;
  p.own_splits = split_count(B * Hkv * row_tiles(R, p.rw_own), tiles(own_rows) + tiles(Lk), cus);
  if (prefix) {
    p.rw_pre = row_waves(B * R);
    p.pre_blocks = (B * R + 31) / 32;
    p.pre_splits = split_count(Hkv * row_tiles(B * R, p.rw_pre), tiles(pre_rows), cus);
    p.pre_units = Hkv * p.pre_blocks * p.pre_splits;
  }
  if (prefix || p.own_splits > 1) p.own_units = Hkv * B * p.own_blocks * p.own_splits;
  return p;
}

int64_t unit_bytes(int64_t D) { return 32 * D * 4 + 32 * 8; }

template <typename T, int D, int RW, bool PREFIX>
hipError_t launch_part(const PagedArgs& a, int64_t items, hipStream_t st) {
  using Sh = Shape<T, D, RW>;
  const void* fn = reinterpret_cast<const void*>(&paged_attn_kernel<T, D, RW, PREFIX>);
  const hipError_t e = opt_in_lds(fn, Sh::lds);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((paged_attn_kernel<T, D, RW, PREFIX>), dim3(unsigned(items)),
                     dim3(64 * Sh::NW), Sh::lds, st, a);
  return hipGetLastError();
}

template <typename T, int D, bool PREFIX>
hipError_t launch_rows(const PagedArgs& a, int rw, int64_t items, hipStream_t st) {
  switch (rw) {
    case 1: return launch_part<T, D, 1, PREFIX>(a, items, st);
    case 2: return launch_part<T, D, 2, PREFIX>(a, items, st);
    default: return launch_part<T, D, 4, PREFIX>(a, items, st);
  }
}

template <typename T, int D>
hipError_t launch_paged(const PagedArgs& a, const PagedPlan& p, hipStream_t st) {
  auto row_tiles = [](int64_t rows, int rw) { return (rows + 32 * rw - 1) / (32 * rw); };
  if (p.pre_splits) {
    const hipError_t e = launch_rows<T, D, true>(
        a, p.rw_pre, int64_t(a.Hkv) * row_tiles(int64_t(a.B) * a.R, p.rw_pre) * p.pre_splits, st);
    if (e != hipSuccess) return e;
  }
  const hipError_t e = launch_rows<T, D, false>(
      a, p.rw_own, int64_t(a.B) * a.Hkv * row_tiles(a.R, p.rw_own) * p.own_splits, st);
  if (e != hipSuccess || p.own_units == 0) return e;
  hipLaunchKernelGGL((paged_merge_kernel<T, D>), dim3(unsigned(a.Hkv * a.B * p.own_blocks), D / 32),
                     dim3(256), 0, st, a);
  return hipGetLastError();
}

struct PagedCall {
  const void* q; int64_t q_sb, q_sl, q_sh;
  const void* k; int64_t k_sb, k_sl, k_sh;
  const void* v; int64_t v_sb, v_sl, v_sh;
  const void* pages; int64_t p_plane, p_sp, p_sr, p_sh, n_pages, page_rows;
  const void* prefix_table; int64_t prefix_width; const void* prefix_len;
  const void* table; int64_t t_sb, width; const void* lens;
  void* out; int64_t o_sb, o_sl, o_sh;
  int dtype; int64_t B, Lq, Lk, H, Hkv, D;
  const void* starts; int starts_dtype; int64_t n_blocks; int causal; float scale;
  void* ws; int64_t ws_bytes;
};

constexpr int64_t kMaxRows = int64_t(1) << 30;  // rows of a sequence or prefix, and keys

// Sizes that the kernels' 32-bit arithmetic and one launch hold.
int check_sizes(const char* what, int64_t B, int64_t Lq, int64_t Lk, int64_t H, int64_t Hkv,
                int64_t D, int dtype, int64_t page_rows, int64_t width, int64_t prefix_width) {
  DX_CHECK_ARG(dtype == DX_BF16 || dtype == DX_F16 || dtype == DX_F32,
               "%s: dtype code %d unsupported", what, dtype);
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

int paged_entry(const char* what, const PagedCall& c, bool prefix, void* stream) {
  const int bad = check_sizes(what, c.B, c.Lq, c.Lk, c.H, c.Hkv, c.D, c.dtype, c.page_rows, c.width,
                              c.prefix_width);
  if (bad) return bad;
  DX_CHECK_ARG(c.n_pages >= 0 && c.n_pages < (int64_t(1) << 31), "%s: bad page count", what);
  DX_CHECK_ARG(c.n_blocks >= 0 && c.n_blocks < kMaxRows &&
                   (c.starts_dtype == DX_I32 || c.starts_dtype == DX_I64),
               "%s: bad block starts", what);
  DX_CHECK_ARG(c.n_blocks == 0 || c.starts, "%s: null block starts", what);
  DX_CHECK_ARG(c.Lk == c.Lq || (!c.causal && c.n_blocks == 0),
               "%s: k/v length %lld must equal q length %lld with block starts or causal", what,
               (long long)c.Lk, (long long)c.Lq);
  DX_CHECK_ARG(std::isfinite(c.scale), "%s: softmax scale must be finite", what);
  if (c.B == 0 || c.Lq == 0) return DX_OK;
  const int64_t es = c.dtype == DX_F32 ? 4 : 2, per16 = 16 / es;
  auto al = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; };
  DX_CHECK_ARG(c.q && c.out, "%s: null pointer", what);
  DX_CHECK_ARG(c.Lk == 0 || (c.k && c.v), "%s: null k or v", what);
  DX_CHECK_ARG(c.width == 0 || (c.table && c.lens), "%s: null block table or lengths", what);
  DX_CHECK_ARG(!prefix || c.prefix_len, "%s: null prefix length", what);
  DX_CHECK_ARG(c.prefix_width == 0 || c.prefix_table, "%s: null prefix table", what);
  DX_CHECK_ARG(c.n_pages == 0 || c.pages, "%s: null pages", what);
  DX_CHECK_ARG(al(c.q) && al(c.k) && al(c.v) && al(c.pages) && al(c.out),
               "%s: pointers must be 16-byte aligned", what);
  for (const int64_t s : {c.q_sb, c.q_sl, c.q_sh, c.k_sb, c.k_sl, c.k_sh, c.v_sb, c.v_sl, c.v_sh,
                          c.p_plane, c.p_sp, c.p_sr, c.p_sh, c.o_sb, c.o_sl, c.o_sh})
    DX_CHECK_ARG(s % per16 == 0, "%s: strides must keep head rows 16-byte aligned", what);
  // 16 rows of keys lie within one buffer descriptor (below 2^31 bytes).
  for (const int64_t s : {c.p_sr, c.k_sl, c.v_sl})
    DX_CHECK_ARG(s >= 0 && s * es < (int64_t(1) << 26), "%s: row stride %lld out of range", what,
                 (long long)s);

  const PagedPlan p = plan_paged(c.B, c.Lq, c.Lk, c.H, c.Hkv, c.width * c.page_rows,
                                 c.prefix_width * c.page_rows, prefix, device_cus());
  const int64_t need = (p.own_units + p.pre_units) * unit_bytes(c.D);
  if (need > c.ws_bytes || (need > 0 && !c.ws)) {
    set_error("%s: workspace of %lld bytes, %lld needed", what, (long long)c.ws_bytes,
              (long long)need);
    return DX_EWORKSPACE;
  }
  DX_CHECK_ARG(al(c.ws), "%s: workspace must be 16-byte aligned", what);
  const int64_t group = c.H / c.Hkv, R = c.Lq * group;
  DX_CHECK_ARG(grid_fits(c.B * c.Hkv * p.own_blocks * p.own_splits, 512) &&
                   grid_fits(c.Hkv * p.pre_blocks * std::max(p.pre_splits, 1), 512),
               "%s: the call exceeds one launch", what);
  PagedArgs a{};
  a.q = static_cast<const char*>(c.q); a.q_sb = c.q_sb * es; a.q_sl = c.q_sl * es; a.q_sh = c.q_sh * es;
  a.k = static_cast<const char*>(c.k); a.k_sb = c.k_sb * es; a.k_sl = c.k_sl * es; a.k_sh = c.k_sh * es;
  a.v = static_cast<const char*>(c.v); a.v_sb = c.v_sb * es; a.v_sl = c.v_sl * es; a.v_sh = c.v_sh * es;
  a.pk = static_cast<const char*>(c.pages); a.pv = a.pk + c.p_plane * es;
  a.p_sp = c.p_sp * es; a.p_sr = c.p_sr * es; a.p_sh = c.p_sh * es;
  a.out = static_cast<char*>(c.out); a.o_sb = c.o_sb * es; a.o_sl = c.o_sl * es; a.o_sh = c.o_sh * es;
  a.table = static_cast<const int32_t*>(c.table); a.t_sb = c.t_sb;
  a.lens = static_cast<const int32_t*>(c.lens);
  a.ptable = static_cast<const int32_t*>(c.prefix_table);
  a.plen = prefix ? static_cast<const int32_t*>(c.prefix_len) : nullptr;
  a.width = int(c.width); a.pwidth = int(c.prefix_width);
  a.n_pages = int(c.n_pages); a.page_rows = int(c.page_rows);
  const uint64_t per = uint64_t(c.page_rows / 16);
  a.page_magic = per == 1 ? 0u : uint32_t(((uint64_t(1) << 32) + per - 1) / per);
  a.starts = c.starts; a.starts_i64 = c.starts_dtype == DX_I64; a.n_blocks = int(c.n_blocks);
  a.B = int(c.B); a.H = int(c.H); a.Hkv = int(c.Hkv); a.group = int(group);
  a.Lq = int(c.Lq); a.Lk = int(c.Lk); a.causal = c.causal != 0;
  a.R = int(R);
  a.scale_log2 = c.scale * 1.4426950408889634f;
  a.own_splits = p.own_splits; a.own_blocks = int(p.own_blocks);
  a.pre_splits = p.pre_splits; a.pre_blocks = int(p.pre_blocks);
  if (p.own_units) {
    a.own_o = static_cast<float*>(c.ws);
    a.pre_o = a.own_o + p.own_units * 32 * c.D;
    a.own_ml = a.pre_o + p.pre_units * 32 * c.D;
    a.pre_ml = a.own_ml + p.own_units * 64;
  }
  const hipStream_t st = static_cast<hipStream_t>(stream);
  hipError_t e;
  if (c.dtype == DX_F32)
    e = c.D == 64 ? launch_paged<float, 64>(a, p, st) : launch_paged<float, 128>(a, p, st);
  else if (c.dtype == DX_BF16)
    e = c.D == 64    ? launch_paged<bf16_t, 64>(a, p, st)
        : c.D == 128 ? launch_paged<bf16_t, 128>(a, p, st)
                     : launch_paged<bf16_t, 256>(a, p, st);
  else
    e = c.D == 64    ? launch_paged<f16_t, 64>(a, p, st)
        : c.D == 128 ? launch_paged<f16_t, 128>(a, p, st)
                     : launch_paged<f16_t, 256>(a, p, st);
  if (e != hipSuccess) {
    set_error("%s: launch failed: %s", what, hipGetErrorString(e));
    return DX_ELAUNCH;
  }
  return DX_OK;
}

}  // namespace
}  // namespace dx

using namespace dx;

extern "C" int64_t dx_paged_attention_workspace_bytes(int dtype, int64_t B, int64_t Lq, int64_t Lk,
                                                      int64_t H, int64_t Hkv, int64_t D,
                                                      int64_t page_rows, int64_t width,
                                                      int has_prefix, int64_t prefix_width) {
  const int bad = check_sizes("paged_attention", B, Lq, Lk, H, Hkv, D, dtype, page_rows, width,
                              prefix_width);
  if (bad) return -bad;
  if (B == 0 || Lq == 0) return 0;
  const PagedPlan p = plan_paged(B, Lq, Lk, H, Hkv, width * page_rows, prefix_width * page_rows,
                                 has_prefix != 0, device_cus());
  return (p.own_units + p.pre_units) * unit_bytes(D);
}

extern "C" int dx_paged_attention(
    const void* q, int64_t q_sb, int64_t q_sl, int64_t q_sh,
    const void* k, int64_t k_sb, int64_t k_sl, int64_t k_sh,
    const void* v, int64_t v_sb, int64_t v_sl, int64_t v_sh,
    const void* pages, int64_t p_plane, int64_t p_sp, int64_t p_sr, int64_t p_sh,
    int64_t n_pages, int64_t page_rows,
    const void* block_table, int64_t t_sb, int64_t width, const void* cache_lens,
    void* out, int64_t o_sb, int64_t o_sl, int64_t o_sh,
    int dtype, int64_t B, int64_t Lq, int64_t Lk, int64_t H, int64_t Hkv, int64_t D,
    const void* block_starts, int starts_dtype, int64_t n_blocks, int causal, float softmax_scale,
    void* workspace, int64_t workspace_bytes, void* stream) {
  const PagedCall c{q, q_sb, q_sl, q_sh, k, k_sb, k_sl, k_sh, v, v_sb, v_sl, v_sh,
                    pages, p_plane, p_sp, p_sr, p_sh, n_pages, page_rows, nullptr, 0, nullptr,
                    block_table, t_sb, width, cache_lens, out, o_sb, o_sl, o_sh,
                    dtype, B, Lq, Lk, H, Hkv, D, block_starts, starts_dtype, n_blocks, causal,
                    softmax_scale, workspace, workspace_bytes};
  return paged_entry("paged_attention", c, false, stream);
}

extern "C" int dx_shared_prefix_attention(
    const void* q, int64_t q_sb, int64_t q_sl, int64_t q_sh,
    const void* k, int64_t k_sb, int64_t k_sl, int64_t k_sh,
    const void* v, int64_t v_sb, int64_t v_sl, int64_t v_sh,
    const void* pages, int64_t p_plane, int64_t p_sp, int64_t p_sr, int64_t p_sh,
    int64_t n_pages, int64_t page_rows,
    const void* prefix_table, int64_t prefix_width, const void* prefix_len,
    const void* block_table, int64_t t_sb, int64_t width, const void* cache_lens,
    void* out, int64_t o_sb, int64_t o_sl, int64_t o_sh,
    int dtype, int64_t B, int64_t Lq, int64_t Lk, int64_t H, int64_t Hkv, int64_t D,
    const void* block_starts, int starts_dtype, int64_t n_blocks, int causal, float softmax_scale,
    void* workspace, int64_t workspace_bytes, void* stream) {
  const PagedCall c{q, q_sb, q_sl, q_sh, k, k_sb, k_sl, k_sh, v, v_sb, v_sl, v_sh,
                    pages, p_plane, p_sp, p_sr, p_sh, n_pages, page_rows,
                    prefix_table, prefix_width, prefix_len,
                    block_table, t_sb, width, cache_lens, out, o_sb, o_sl, o_sh,
                    dtype, B, Lq, Lk, H, Hkv, D, block_starts, starts_dtype, n_blocks, causal,
                    softmax_scale, workspace, workspace_bytes};
  return paged_entry("shared_prefix_attention", c, true, stream);
}
