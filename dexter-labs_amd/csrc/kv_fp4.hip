// Pages of a KV cache in 4 bits on gfx950: writing a chunk into a batch's pages, and
// reading rows back (kv_fp4.h has the format).
//
// Writing: four lanes hold a block, 8 elements (16 bytes) of k and 8 of v each.
// The block's largest magnitude is found among them in the values' own bits (an
// exchange of lanes 1 and 2 apart), its exponent is integer arithmetic on those, and
// the conversion instruction rounds to the codes, ties to even. Reading is the
// conversion the other way. Both are bound by memory, and by latency for few rows: 4 x
// 1,826 rows of 40 heads (f16, D 128; 150 MB of values, 40 of pages) are written in 45 us, 4.2
// TB/s, and read back in 31 us, 6.1 TB/s from caches that still hold them; one row of 64
// sequences of 8 heads takes 3.4 and 2.9 us.
//
// Work: a sequence's rows are (head, token), tokens fastest, so that a wave's rows lie
// side by side in a page, whose codes and scales are then written in runs: 16 rows of
// a head are 1 KB and 64 bytes (D 128). Of one token they are its heads.
#include "kv_fp4.h"

#include <algorithm>

namespace dx {
namespace {

constexpr int kWaves = 4;  // waves per workgroup

struct Fp4Args {
  const char* k; int64_t k_sb, k_sl, k_sh;  // 16-bit rows, strides in bytes
  const char* v; int64_t v_sb, v_sl, v_sh;
  char* pages; int64_t p_plane, p_sp, p_sh;
  const int32_t* table; int64_t t_sb;
  const int32_t* starts;
  int32_t* status;
  int64_t per_seq;           // lanes' pieces of a sequence: n * H * D / 8
  int B, n, H;
  int waves;                 // per sequence
  int width, n_pages, page_rows;
};

// This lane's piece: 8 elements of a row of a head, and its place in the pages.
template <int D>
struct Piece {
  int b, t, h, part;        // part: of the row's D / 8
  int64_t codes, scales;    // byte offsets in a plane; codes < 0: the row has no page
  bool there;

  __device__ __forceinline__ Piece(const Fp4Args& a) {
    constexpr int P = D / 8;
    const int lane = int(threadIdx.x) & 63;
    const uint32_t w = uint32_t(__builtin_amdgcn_readfirstlane(int(blockIdx.x) * kWaves + (int(threadIdx.x) >> 6)));
    b = int(w / uint32_t(a.waves));
    const int64_t at = int64_t(w - uint32_t(b) * uint32_t(a.waves)) * 64 + lane;
    there = b < a.B && at < a.per_seq;
    const uint32_t row = there ? uint32_t(at / P) : 0u;
    part = int(at % P);
    h = int(row / uint32_t(a.n));
    t = int(row - uint32_t(h) * uint32_t(a.n));
    codes = -1;
    scales = 0;
    if (!there) return;
    const int64_t r = int64_t(a.starts[b]) + t;
    int page = -1;
    if (r >= 0 && r < int64_t(a.width) * a.page_rows) page = a.table[b * a.t_sb + r / a.page_rows];
    if (uint32_t(page) >= uint32_t(a.n_pages)) {
      if (a.status) a.status[0] = 1;
      return;
    }
    const int in_page = int(r % a.page_rows);
    codes = page * a.p_sp + h * a.p_sh;
    scales = codes + int64_t(a.page_rows) * (D / 2) + int64_t(in_page) * (D / 32) + part / 4;
    codes += int64_t(in_page) * (D / 2) + part * 4;
  }
};

// The scale byte of a block whose magnitudes are at most that with bits `top` (of fp32):
// 7 * 2^e holds m 2^E for e = E - 2 up to m = 7 / 4, above that for E - 1.
template <typename T>
__device__ __forceinline__ uint32_t scale_byte(uint32_t top) {
  if (top >= 0x7f800000u) return 255u;
  const int byte = int((top + 0x1fffffu) >> 23) - 2;
  return uint32_t(min(max(byte, Fp4Range<T>::lo), Fp4Range<T>::hi));
}

// Two values to two codes, in byte 0 of what is returned; both exact as fp32.
__device__ __forceinline__ uint32_t fp4_codes(float lo, float hi, float scale) {
  return uint32_t(__builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, lo, hi, scale, 0)) & 255u;
}

template <typename T>
__device__ __forceinline__ void write_piece(char* plane, int64_t codes, int64_t scales, int part, const u32x4& x) {
  float f[8];
  uint32_t top = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    f[e] = to_f32(T{uint16_t(x[e / 2] >> (16 * (e % 2)))});
    top = max(top, __float_as_uint(f[e]) & 0x7fffffffu);
  }
  top = max(top, uint32_t(__builtin_amdgcn_update_dpp(0, int(top), 0xb1, 0xf, 0xf, false)));
  top = max(top, uint32_t(__builtin_amdgcn_update_dpp(0, int(top), 0x4e, 0xf, 0xf, false)));
  const uint32_t byte = scale_byte<T>(top);
  const float scale = fp4_scale(byte);
  uint32_t out = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) out |= fp4_codes(f[2 * e], f[2 * e + 1], scale) << (8 * e);
  if (codes < 0) return;
  *reinterpret_cast<uint32_t*>(plane + codes) = byte == 255u ? 0u : out;
  if (part % 4 == 0) *reinterpret_cast<uint8_t*>(plane + scales) = uint8_t(byte);
}

template <typename T, int D>
__global__ __launch_bounds__(64 * kWaves) void kv_page_append_fp4_kernel(Fp4Args a) {
  const Piece<D> p(a);
  u32x4 k{0, 0, 0, 0}, v{0, 0, 0, 0};
  if (p.there) {
    k = *reinterpret_cast<const u32x4*>(a.k + p.b * a.k_sb + p.t * a.k_sl + p.h * a.k_sh + 16 * p.part);
    v = *reinterpret_cast<const u32x4*>(a.v + p.b * a.v_sb + p.t * a.v_sl + p.h * a.v_sh + 16 * p.part);
  }
  write_piece<T>(a.pages, p.codes, p.scales, p.part, k);
  write_piece<T>(a.pages + a.p_plane, p.codes, p.scales, p.part, v);
}

// k and v are written here, both contiguous.
template <typename T, int D>
__global__ __launch_bounds__(64 * kWaves) void kv_page_read_fp4_kernel(Fp4Args a) {
  const Piece<D> p(a);
  if (!p.there) return;
  u32x4 k{0, 0, 0, 0}, v{0, 0, 0, 0};
  if (p.codes >= 0) {
    const uint32_t kc = *reinterpret_cast<const uint32_t*>(a.pages + p.codes);
    const uint32_t vc = *reinterpret_cast<const uint32_t*>(a.pages + a.p_plane + p.codes);
    const uint32_t ks = *reinterpret_cast<const uint8_t*>(a.pages + p.scales);
    const uint32_t vs = *reinterpret_cast<const uint8_t*>(a.pages + a.p_plane + p.scales);
    k = fp4_values<T>(kc, fp4_scale(ks));
    v = fp4_values<T>(vc, fp4_scale(vs));
  }
  *reinterpret_cast<u32x4*>(const_cast<char*>(a.k) + p.b * a.k_sb + p.t * a.k_sl + p.h * a.k_sh + 16 * p.part) = k;
  *reinterpret_cast<u32x4*>(const_cast<char*>(a.v) + p.b * a.v_sb + p.t * a.v_sl + p.h * a.v_sh + 16 * p.part) = v;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <typename T, bool READ>
void launch(const Fp4Args& a, int64_t D, unsigned blocks, hipStream_t st) {
  auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(blocks), dim3(64 * kWaves), 0, st, a); };
  if constexpr (READ)
    go(D == 64 ? kv_page_read_fp4_kernel<T, 64> : D == 128 ? kv_page_read_fp4_kernel<T, 128> : kv_page_read_fp4_kernel<T, 256>);
  else
    go(D == 64 ? kv_page_append_fp4_kernel<T, 64> : D == 128 ? kv_page_append_fp4_kernel<T, 128> : kv_page_append_fp4_kernel<T, 256>);
}

template <bool READ>
int fp4_entry(const char* what, const void* k, int64_t k_sb, int64_t k_sl, int64_t k_sh,
              const void* v, int64_t v_sb, int64_t v_sl, int64_t v_sh, const void* pages,
              int64_t p_plane, int64_t p_sp, int64_t p_sh, int dtype, int64_t n_pages,
              int64_t page_rows, const void* block_table, int64_t t_sb, int64_t width,
              const void* starts, void* status, int64_t B, int64_t n, int64_t H, int64_t D,
              void* stream) {
  DX_CHECK_ARG(dtype == DX_BF16 || dtype == DX_F16, "%s: dtype code %d unsupported", what, dtype);
  DX_CHECK_ARG(D == 64 || D == 128 || D == 256, "%s: head_dim %lld (supported: 64, 128 and 256)", what,
               (long long)D);
  DX_CHECK_ARG(B >= 0 && n >= 0 && H > 0 && n_pages >= 0 && width >= 0, "%s: bad shape", what);
  DX_CHECK_ARG(page_rows > 0 && page_rows % 16 == 0 && page_rows <= 1024,
               "%s: pages of %lld rows (supported: multiples of 16 up to 1024)", what, (long long)page_rows);
  constexpr int64_t kMax = (int64_t(1) << 31) - 1;
  DX_CHECK_ARG(n_pages <= kMax && width <= kMax && n <= kMax && H <= kMax && B <= kMax,
               "%s: sizes must be below 2^31", what);
  if (B == 0 || n == 0) return DX_OK;
  DX_CHECK_ARG(k && v && starts && (block_table || width == 0), "%s: null pointer", what);
  DX_CHECK_ARG(pages || n_pages == 0, "%s: null pages", what);
  DX_CHECK_ARG(aligned16(k) && aligned16(v) && aligned16(pages), "%s: pointers must be 16-byte aligned", what);
  DX_CHECK_ARG(k_sb % 8 == 0 && k_sl % 8 == 0 && k_sh % 8 == 0 && v_sb % 8 == 0 && v_sl % 8 == 0 &&
                   v_sh % 8 == 0 && p_plane % 16 == 0 && p_sp % 16 == 0 && p_sh % 16 == 0,
               "%s: strides must keep head rows 16-byte aligned", what);
  // Rows of a sequence in 32 bits, waves in 32, threads of a launch below 2^32.
  DX_CHECK_ARG(n <= kMax / H, "%s: %lld rows of %lld heads exceed one launch", what, (long long)n, (long long)H);
  const int64_t per_seq = n * H * (D / 8), waves = (per_seq + 63) / 64;
  DX_CHECK_ARG(waves <= ((int64_t(1) << 26) - kWaves) / B, "%s: %lld x %lld rows exceed one launch", what,
               (long long)B, (long long)n);
  Fp4Args a{};
  a.k = static_cast<const char*>(k); a.k_sb = 2 * k_sb; a.k_sl = 2 * k_sl; a.k_sh = 2 * k_sh;
  a.v = static_cast<const char*>(v); a.v_sb = 2 * v_sb; a.v_sl = 2 * v_sl; a.v_sh = 2 * v_sh;
  a.pages = static_cast<char*>(const_cast<void*>(pages));
  a.p_plane = p_plane; a.p_sp = p_sp; a.p_sh = p_sh;
  a.table = static_cast<const int32_t*>(block_table); a.t_sb = t_sb;
  a.starts = static_cast<const int32_t*>(starts);
  a.status = static_cast<int32_t*>(status);
  a.per_seq = per_seq; a.waves = int(waves);
  a.B = int(B); a.n = int(n); a.H = int(H);
  a.width = int(width); a.n_pages = int(n_pages); a.page_rows = int(page_rows);
  const unsigned blocks = unsigned((B * waves + kWaves - 1) / kWaves);
  if (dtype == DX_BF16)
    launch<bf16_t, READ>(a, D, blocks, static_cast<hipStream_t>(stream));
  else
    launch<f16_t, READ>(a, D, blocks, static_cast<hipStream_t>(stream));
  DX_CHECK_LAUNCH(what);
  return DX_OK;
}

}  // namespace
}  // namespace dx

using namespace dx;

extern "C" int dx_kv_page_append_fp4(const void* k, int64_t k_sb, int64_t k_sl, int64_t k_sh,
                                     const void* v, int64_t v_sb, int64_t v_sl, int64_t v_sh,
                                     void* pages, int64_t p_plane, int64_t p_sp, int64_t p_sh,
                                     int dtype, int64_t n_pages, int64_t page_rows,
                                     const void* block_table, int64_t t_sb, int64_t width,
                                     const void* starts, void* status, int64_t B, int64_t n,
                                     int64_t H, int64_t D, void* stream) {
  return fp4_entry<false>("kv_page_append_fp4", k, k_sb, k_sl, k_sh, v, v_sb, v_sl, v_sh, pages, p_plane,
                          p_sp, p_sh, dtype, n_pages, page_rows, block_table, t_sb, width, starts, status,
                          B, n, H, D, stream);
}

extern "C" int dx_kv_page_read_fp4(const void* pages, int64_t p_plane, int64_t p_sp, int64_t p_sh,
                                   int dtype, int64_t n_pages, int64_t page_rows,
                                   const void* block_table, int64_t t_sb, int64_t width,
                                   const void* starts, void* status, void* k, void* v, int64_t B,
                                   int64_t n, int64_t H, int64_t D, void* stream) {
  const int64_t sl = D > 0 && H > 0 && H < (int64_t(1) << 31) && D <= 256 ? H * D : 0;
  const int64_t sb = sl && n >= 0 && n <= ((int64_t(1) << 31) - 1) ? n * sl : 0;
  return fp4_entry<true>("kv_page_read_fp4", k, sb, sl, D, v, sb, sl, D, pages, p_plane, p_sp, p_sh, dtype,
                         n_pages, page_rows, block_table, t_sb, width, starts, status, B, n, H, D, stream);
}
