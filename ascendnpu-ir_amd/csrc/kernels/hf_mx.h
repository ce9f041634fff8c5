// Block-scaled (microscaling) codes: hfusion.quantize_mx and its inverse.
//
// 32 consecutive elements along the blocked axis share the scale 2^E, held as
// the byte E + 127 (e8m0); a code stands for code * 2^E.
//   E    = floor(log2 max|x|) - EMAX, at least -127   (EMAX: the exponent of
//          the format's largest binade, so the block's largest element lands
//          in it; a block of zeros has the byte 0)
//   code = x * 2^-E rounded to the nearest code, ties to even, values past the
//          largest finite code becoming that code
// A block that holds an infinity or a NaN has the byte 255 (its values are
// NaN whatever the codes) and codes 0.
// floor(log2 max|x|) is the exponent field of the largest magnitude, which
// integer maxima of the bits without the sign find (NaN and infinity compare
// above every number), and x * 2^-E is exact or far below the smallest code,
// so the only rounding is the conversion's own.
#pragma once
#include "hf_row.h"

namespace hf {

// element types of the values
enum MxElem : int { EL_F32 = 0, EL_BF16 = 1, EL_F16 = 2 };
// formats of the codes (the matrix core's numbers)
enum MxFormat : int { MX_E4M3 = 0, MX_E5M2 = 1, MX_E2M1 = 4 };
template <int EL> constexpr int el_bytes = EL == EL_F32 ? 4 : 2;
template <int FMT> constexpr int mx_emax = FMT == MX_E4M3 ? 8 : FMT == MX_E5M2 ? 15 : 2;
template <int FMT> constexpr float mx_top = FMT == MX_E4M3 ? 448.0f : FMT == MX_E5M2 ? 57344.0f : 6.0f;
// values of one 16-byte access, lanes that share a block of 32, bytes of the
// codes of one access
template <int EL> constexpr int mx_vals = 16 / el_bytes<EL>;
template <int EL> constexpr int mx_lanes = 32 / mx_vals<EL>;
template <int EL, int FMT> constexpr int mx_bytes = FMT == MX_E2M1 ? mx_vals<EL> / 2 : mx_vals<EL>;

// ---------------------------------------------------------------- 16 bytes of values
template <int EL> struct Pack { uint32_t w[4]; };

// (accesses at any element: rows of odd lengths start anywhere)
typedef u32x4 u32x4_any __attribute__((aligned(1)));
typedef u32x2 u32x2_any __attribute__((aligned(1)));
typedef uint32_t u32_any __attribute__((aligned(1)));
typedef uint16_t u16_any __attribute__((aligned(1)));

template <int EL, bool ONCE = true> __device__ __forceinline__ Pack<EL> pack_load(const void *p) {
  const u32x4_any *q = reinterpret_cast<const u32x4_any *>(p);
  const u32x4 v = ONCE ? __builtin_nontemporal_load(q) : *q;
  return Pack<EL>{{v.x, v.y, v.z, v.w}};
}
// The end of a row of D values: a lane whose access would pass it reads the
// row's last 16 bytes instead (`behind` values before its own first one) and
// moves its values to the front, zeros behind them, when it needs them: a load
// per value, each waiting for the one before, made a short odd row slow (the
// gradient of [45, 4441] 13.9 us, 7.7 so).  Rows of less than
// 16 bytes are read value by value.
template <int EL, int64_t D, bool ONCE = true>
__device__ __forceinline__ Pack<EL> pack_load_row(const void *base, int64_t row, int64_t c) {
  constexpr int V = mx_vals<EL>;
  if constexpr (D >= V) {
    return pack_load<EL, ONCE>((const char *)base + (row * D + (c < D - V ? c : D - V)) * el_bytes<EL>);
  } else {
    Pack<EL> o{};
    const char *p = (const char *)base + row * D * el_bytes<EL>;
#pragma unroll
    for (int i = 0; i < (int)D; ++i) {
      if constexpr (EL == EL_F32) o.w[i] = reinterpret_cast<const uint32_t *>(p)[i];
      else o.w[i / 2] |= (uint32_t)reinterpret_cast<const uint16_t *>(p)[i] << (16 * (i % 2));
    }
    return o;
  }
}
// what pack_load_row read, put right: the values at column c, a multiple of
// the pack's (so the one lane that holds the row's end has a fixed distance)
template <int EL, int64_t D> __device__ __forceinline__ void pack_at(Pack<EL> &o, int64_t c) {
  constexpr int V = mx_vals<EL>, END = (int)(D % V), DOWN = END ? (V - END) * el_bytes<EL> : 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (D >= V && END != 0) {
      const int k = i + DOWN / 4; // (words further up are read before they are written)
      const uint32_t lo = k < 4 ? o.w[k] : 0, hi = k < 3 ? o.w[k + 1] : 0;
      const uint32_t end = DOWN % 4 ? lo >> 16 | hi << 16 : lo;
      o.w[i] = c > D - V ? end : o.w[i];
    }
    o.w[i] = c >= D ? 0 : o.w[i];
  }
}
template <int EL> __device__ __forceinline__ void pack_store(void *p, const Pack<EL> &o) {
  __builtin_nontemporal_store(u32x4{o.w[0], o.w[1], o.w[2], o.w[3]}, reinterpret_cast<u32x4_any *>(p));
}
template <int EL> __device__ __forceinline__ void pack_store_part(void *p, const Pack<EL> &o, int n) {
#pragma unroll
  for (int i = 0; i < mx_vals<EL>; ++i) {
    if (i >= n) break;
    if constexpr (EL == EL_F32) reinterpret_cast<uint32_t *>(p)[i] = o.w[i];
    else reinterpret_cast<uint16_t *>(p)[i] = (uint16_t)(o.w[i / 2] >> (16 * (i % 2)));
  }
}
template <int EL> __device__ __forceinline__ float word_get(const uint32_t *w, int i) {
  if constexpr (EL == EL_F32) return u2f(w[i]);
  else if constexpr (EL == EL_BF16) return u2f(i % 2 ? w[i / 2] & 0xFFFF0000u : w[i / 2] << 16);
  else return f16_to_f32((uint16_t)(w[i / 2] >> (16 * (i % 2))));
}
template <int EL> __device__ __forceinline__ float pack_get(const Pack<EL> &o, int i) { return word_get<EL>(o.w, i); }
// two neighbouring values rounded to nearest even
template <int EL> __device__ __forceinline__ void pack_set2(Pack<EL> &o, int i, float a, float b) {
  if constexpr (EL == EL_F32) o.w[i] = f2u(a), o.w[i + 1] = f2u(b);
  else if constexpr (EL == EL_BF16) o.w[i / 2] = (uint32_t)f32_to_bf16_rne(a) | (uint32_t)f32_to_bf16_rne(b) << 16;
  else {
    // (a product and its conversion would become one multiply-add with +0,
    // which loses the sign of a product that is -0)
    asm("" : "+v"(a), "+v"(b));
    o.w[i / 2] = (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)a) | (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)b) << 16;
  }
}

// ---------------------------------------------------------------- magnitudes
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
}
__device__ __forceinline__ uint32_t max_u32(uint32_t a, uint32_t b) { return a > b ? a : b; }
// f32 bits of a 16-bit magnitude (bits without the sign)
template <int EL> __device__ __forceinline__ uint32_t mag_f32(uint32_t half) {
  if constexpr (EL == EL_BF16) return half << 16;
  else return f2u(f16_to_f32((uint16_t)half));
}
// f32 bits of the largest magnitude of a pack
template <int EL> __device__ __forceinline__ uint32_t pack_amax(const Pack<EL> &o) {
  if constexpr (EL == EL_F32) {
    uint32_t m = o.w[0] & 0x7FFFFFFFu;
#pragma unroll
    for (int i = 1; i < 4; ++i) m = max_u32(m, o.w[i] & 0x7FFFFFFFu);
    return m;
  } else {
    uint32_t m = o.w[0] & 0x7FFF7FFFu;
#pragma unroll
    for (int i = 1; i < 4; ++i) m = max_u16x2(m, o.w[i] & 0x7FFF7FFFu);
    return mag_f32<EL>(max_u32(m & 0xFFFFu, m >> 16));
  }
}
// over the lanes that share a block
template <int EL> __device__ __forceinline__ uint32_t block_max(uint32_t m) {
  m = max_u32(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0xB1, 0xF, 0xF, true)); // lanes 1 0 3 2
  m = max_u32(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x4E, 0xF, 0xF, true)); // lanes 2 3 0 1
  if constexpr (mx_lanes<EL> == 8)
    m = max_u32(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x141, 0xF, 0xF, true)); // eight lanes mirrored
  return m;
}

// ---------------------------------------------------------------- codes
// the scale byte of a block whose largest magnitude has these f32 bits
template <int FMT> __device__ __forceinline__ uint32_t mx_scale_byte(uint32_t amax) {
  const int e = (int)(amax >> 23);
  return e == 255 ? 255u : (uint32_t)(e > mx_emax<FMT> ? e - mx_emax<FMT> : 0);
}
// 2^-E of a scale byte (any number for 255, whose codes are zeros)
__device__ __forceinline__ float mx_inverse(uint32_t byte) { return u2f((254u - (byte > 253u ? 253u : byte)) << 23); }
// 2^E; the byte 0 is a subnormal, 255 NaN
__device__ __forceinline__ float mx_scale(uint32_t byte) {
  return u2f(byte == 0 ? 0x00400000u : byte == 255 ? 0x7FC00000u : byte << 23);
}
template <int FMT> __device__ __forceinline__ float mx_clamp(float v) {
  return __builtin_amdgcn_fmed3f(v, -mx_top<FMT>, mx_top<FMT>);
}
// two codes into half h (16 bits) of w
template <int FMT> __device__ __forceinline__ uint32_t mx_pair8(float a, float b, uint32_t w, bool hi) {
  static_assert(FMT != MX_E2M1);
  a = mx_clamp<FMT>(a), b = mx_clamp<FMT>(b);
  if constexpr (FMT == MX_E4M3) return (uint32_t)(hi ? __builtin_amdgcn_cvt_pk_fp8_f32(a, b, (int)w, true) : __builtin_amdgcn_cvt_pk_fp8_f32(a, b, (int)w, false));
  else return (uint32_t)(hi ? __builtin_amdgcn_cvt_pk_bf8_f32(a, b, (int)w, true) : __builtin_amdgcn_cvt_pk_bf8_f32(a, b, (int)w, false));
}
// two e2m1 codes into byte B of w, a in the low half
template <int B> __device__ __forceinline__ uint32_t mx_pair4(float a, float b, uint32_t w) {
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, mx_clamp<MX_E2M1>(a), mx_clamp<MX_E2M1>(b), 1.0f, B);
}
// the codes of a pack, in as many low bytes as they take
template <int EL, int FMT> __device__ __forceinline__ u32x2 mx_encode(const Pack<EL> &o, float inv, bool finite) {
  u32x2 c = {0, 0};
  auto v = [&](int i) { return pack_get<EL>(o, i) * inv; };
  if constexpr (FMT == MX_E2M1) {
    c.x = mx_pair4<0>(v(0), v(1), c.x);
    c.x = mx_pair4<1>(v(2), v(3), c.x);
    if constexpr (mx_vals<EL> == 8) {
      c.x = mx_pair4<2>(v(4), v(5), c.x);
      c.x = mx_pair4<3>(v(6), v(7), c.x);
    }
  } else {
    c.x = mx_pair8<FMT>(v(0), v(1), c.x, false);
    c.x = mx_pair8<FMT>(v(2), v(3), c.x, true);
    if constexpr (mx_vals<EL> == 8) {
      c.y = mx_pair8<FMT>(v(4), v(5), c.y, false);
      c.y = mx_pair8<FMT>(v(6), v(7), c.y, true);
    }
  }
  return finite ? c : u32x2{0, 0};
}
typedef float f32x2 __attribute__((ext_vector_type(2)));
// codes 2 i, 2 i + 1 of a word
template <int FMT> __device__ __forceinline__ f32x2 mx_decode2(uint32_t w, int i) {
  if constexpr (FMT == MX_E4M3) return i ? __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true) : __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
  else if constexpr (FMT == MX_E5M2) return i ? __builtin_amdgcn_cvt_pk_f32_bf8((int)w, true) : __builtin_amdgcn_cvt_pk_f32_bf8((int)w, false);
  else
    return i == 0   ? __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 0)
           : i == 1 ? __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 1)
           : i == 2 ? __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 2)
                    : __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 3);
}
template <int EL, int FMT> __device__ __forceinline__ void mx_decode(u32x2 c, float scale, float (&f)[mx_vals<EL>]) {
#pragma unroll
  for (int i = 0; i < mx_vals<EL> / 2; ++i) {
    const f32x2 v = FMT == MX_E2M1 ? mx_decode2<FMT>(c.x, i) : mx_decode2<FMT>(i < 2 ? c.x : c.y, i % 2);
    f[2 * i] = v.x * scale, f[2 * i + 1] = v.y * scale;
  }
}
template <int EL, int FMT> __device__ __forceinline__ void codes_store(void *p, u32x2 c) {
  constexpr int B = mx_bytes<EL, FMT>;
  if constexpr (B == 8) __builtin_nontemporal_store(c, reinterpret_cast<u32x2_any *>(p));
  else if constexpr (B == 4) __builtin_nontemporal_store(c.x, reinterpret_cast<u32_any *>(p));
  else __builtin_nontemporal_store((uint16_t)c.x, reinterpret_cast<u16_any *>(p));
}
// the codes of the first n values (n even for e2m1)
template <int EL, int FMT> __device__ __forceinline__ void codes_store_part(uint8_t *p, u32x2 c, int n) {
  const int bytes = FMT == MX_E2M1 ? n / 2 : n;
#pragma unroll
  for (int i = 0; i < mx_bytes<EL, FMT>; ++i) {
    if (i >= bytes) break;
    p[i] = (uint8_t)((i < 4 ? c.x : c.y) >> (8 * (i % 4)));
  }
}
template <int EL, int FMT> __device__ __forceinline__ u32x2 codes_load(const void *p) {
  constexpr int B = mx_bytes<EL, FMT>;
  if constexpr (B == 8) return __builtin_nontemporal_load(reinterpret_cast<const u32x2_any *>(p));
  else if constexpr (B == 4) return u32x2{__builtin_nontemporal_load(reinterpret_cast<const u32_any *>(p)), 0};
  else return u32x2{__builtin_nontemporal_load(reinterpret_cast<const u16_any *>(p)), 0};
}
// as pack_load_row and pack_at, of a row of codes (D even for e2m1)
template <int EL, int FMT, int64_t D> __device__ __forceinline__ u32x2 codes_load_row(const void *base, int64_t row, int64_t c) {
  constexpr int V = mx_vals<EL>, P = FMT == MX_E2M1 ? 2 : 1;
  if constexpr (D >= V) {
    return codes_load<EL, FMT>((const uint8_t *)base + (row * D + (c < D - V ? c : D - V)) / P);
  } else {
    const uint8_t *p = (const uint8_t *)base + row * D / P;
    u32x2 o = {0, 0};
#pragma unroll
    for (int i = 0; i < (int)D / P; ++i) {
      if (i < 4) o.x |= (uint32_t)p[i] << (8 * i);
      else o.y |= (uint32_t)p[i] << (8 * (i - 4));
    }
    return o;
  }
}
template <int EL, int FMT, int64_t D> __device__ __forceinline__ u32x2 codes_at(u32x2 o, int64_t c) {
  constexpr int V = mx_vals<EL>, P = FMT == MX_E2M1 ? 2 : 1, END = (int)(D % V), DOWN = END ? 8 * ((V - END) / P) : 0;
  uint64_t w = ((uint64_t)o.y << 32) | o.x;
  if constexpr (D >= V && END != 0) w = c > D - V ? w >> DOWN : w;
  w = c >= D ? 0 : w;
  return u32x2{(uint32_t)w, (uint32_t)(w >> 32)};
}

// One scale byte a block: lane l holds block `blk`, which counts up by one
// every mx_lanes lanes.  Of 16-bit values the four blocks of 16 lanes leave
// as one word where all four exist.
template <int EL> __device__ __forceinline__ void scales_store(uint8_t *__restrict__ scales, int64_t blk, int64_t nblk, uint32_t byte) {
  const int lane = threadIdx.x & 15;
  if (mx_lanes<EL> == 4 && (blk | 3) < nblk) { // (a row of lanes starts at a multiple of 4)
    uint32_t w = byte;
    w |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)byte, 0x104, 0xF, 0xF, true) << 8;  // lane + 4
    w |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)byte, 0x108, 0xF, 0xF, true) << 16; // lane + 8
    w |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)byte, 0x10C, 0xF, 0xF, true) << 24; // lane + 12
    if (lane == 0) *reinterpret_cast<u32_any *>(scales + blk) = w;
  } else if ((lane & (mx_lanes<EL> - 1)) == 0) {
    scales[blk] = (uint8_t)byte;
  }
}

// ---------------------------------------------------------------- blocks along a row
// x [R, K] -> codes [R, K] (e2m1: [R, K/2]), scales [R, ceil(K/32)].  A lane
// takes 16-byte accesses of values, four (f32: eight) neighbouring lanes a
// block; a workgroup's accesses are consecutive, U of them a thread in flight.
// Bound by HBM: [8192, 4096] bf16 to 8 bits moves 101.7 MB in 17.6 us (5.8 TB/s;
// a large copy runs at 5.4).
// Access `it` of the rows: row and column of its first value, its block, and
// how many of its values exist.  Accesses past the last are the last one
// again, of which nothing is written.
template <int EL, int64_t K> struct RowAccess {
  int64_t row, c, blk;
  int cnt;
  __device__ __forceinline__ RowAccess(int64_t it, int64_t n) {
    constexpr int V = mx_vals<EL>, L = mx_lanes<EL>;
    constexpr int64_t NB = (K + 31) / 32;
    const int64_t at = it < n ? it : n - 1;
    blk = it / L;
    if constexpr (K % 32 == 0) { // whole accesses only: rows follow each other
      row = 0;
      c = at * V;
      cnt = it < n ? V : 0;
    } else {
      row = at / (NB * L);
      c = (at - row * (NB * L)) * V;
      cnt = it >= n || c >= K ? 0 : K - c < V ? (int)(K - c) : V;
    }
  }
};

template <int EL, int FMT, int64_t K, int U>
__device__ __forceinline__ void mx_quantize_rows(const void *__restrict__ x, void *__restrict__ codes, void *__restrict__ scales,
                                                 int64_t R) {
  constexpr int V = mx_vals<EL>;
  const int64_t nblk = R * ((K + 31) / 32), n = nblk * mx_lanes<EL>;
  for (int64_t it0 = (int64_t)blockIdx.x * (blockDim.x * U); it0 < n; it0 += (int64_t)gridDim.x * (blockDim.x * U)) {
    Pack<EL> o[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const RowAccess<EL, K> a(it0 + u * (int64_t)blockDim.x + threadIdx.x, n);
      if constexpr (K % 32 == 0) o[u] = pack_load<EL>((const char *)x + a.c * el_bytes<EL>);
      else o[u] = pack_load_row<EL, K>(x, a.row, a.c);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const RowAccess<EL, K> a(it0 + u * (int64_t)blockDim.x + threadIdx.x, n);
      if constexpr (K % 32 != 0) pack_at<EL, K>(o[u], a.c);
      const uint32_t byte = mx_scale_byte<FMT>(block_max<EL>(pack_amax<EL>(o[u])));
      const u32x2 c = mx_encode<EL, FMT>(o[u], mx_inverse(byte), byte != 255);
      uint8_t *dst = (uint8_t *)codes + (a.row * K + a.c) / (FMT == MX_E2M1 ? 2 : 1);
      if (a.cnt == V) codes_store<EL, FMT>(dst, c);
      else codes_store_part<EL, FMT>(dst, c, a.cnt);
      if (a.blk < nblk) scales_store<EL>((uint8_t *)scales, a.blk, nblk, byte);
    }
  }
}

// codes -> values, the same layout; f32 products are exact, the one rounding
// is to the result's type
template <int EL, int FMT, int64_t K, int U>
__device__ __forceinline__ void mx_dequantize_rows(const void *__restrict__ codes, const void *__restrict__ scales, void *__restrict__ out,
                                                   int64_t R) {
  constexpr int V = mx_vals<EL>;
  const int64_t nblk = R * ((K + 31) / 32), n = nblk * mx_lanes<EL>;
  for (int64_t it0 = (int64_t)blockIdx.x * (blockDim.x * U); it0 < n; it0 += (int64_t)gridDim.x * (blockDim.x * U)) {
    u32x2 c[U];
    uint32_t byte[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const RowAccess<EL, K> a(it0 + u * (int64_t)blockDim.x + threadIdx.x, n);
      if constexpr (K % 32 == 0) c[u] = codes_load<EL, FMT>((const uint8_t *)codes + a.c / (FMT == MX_E2M1 ? 2 : 1));
      else c[u] = codes_load_row<EL, FMT, K>(codes, a.row, a.c);
      byte[u] = ((const uint8_t *)scales)[a.blk < nblk ? a.blk : nblk - 1];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const RowAccess<EL, K> a(it0 + u * (int64_t)blockDim.x + threadIdx.x, n);
      float f[V];
      if constexpr (K % 32 != 0) c[u] = codes_at<EL, FMT, K>(c[u], a.c);
      mx_decode<EL, FMT>(c[u], mx_scale(byte[u]), f);
      Pack<EL> o;
#pragma unroll
      for (int i = 0; i < V; i += 2) pack_set2<EL>(o, i, f[i], f[i + 1]);
      char *dst = (char *)out + (a.row * K + a.c) * el_bytes<EL>;
      if (a.cnt == V) pack_store<EL>(dst, o);
      else pack_store_part<EL>(dst, o, a.cnt);
    }
  }
}

// ---------------------------------------------------------------- blocks down a column
// x [K, N] -> codes [K, N] (e2m1: [K/2, N], two k a byte), scales
// [N, ceil(K/32)].  A lane owns four columns of one block (32 k-rows), a wave
// 256 columns, and the eight waves of a workgroup eight blocks, whose scale
// bytes leave together: eight consecutive bytes of every column.
constexpr int MXC_COLS = 256, MXC_BLOCKS = 8;

template <int EL> struct Quad4 { uint32_t w[el_bytes<EL>]; }; // four values of a k-row
template <int EL, bool FOUR> __device__ __forceinline__ Quad4<EL> quad_load(const char *p, int n) {
  Quad4<EL> q{};
  if constexpr (FOUR) {
    if constexpr (EL == EL_F32) {
      const u32x4 v = __builtin_nontemporal_load(reinterpret_cast<const u32x4_any *>(p));
      q.w[0] = v.x, q.w[1] = v.y, q.w[2] = v.z, q.w[3] = v.w;
    } else {
      const u32x2 v = __builtin_nontemporal_load(reinterpret_cast<const u32x2_any *>(p));
      q.w[0] = v.x, q.w[1] = v.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      if constexpr (EL == EL_F32) q.w[i] = reinterpret_cast<const uint32_t *>(p)[i < n ? i : 0];
      else q.w[i / 2] |= (uint32_t)reinterpret_cast<const uint16_t *>(p)[i < n ? i : 0] << (16 * (i % 2));
    }
  }
  return q;
}
template <int EL> __device__ __forceinline__ float quad_get(const Quad4<EL> &q, int i) { return word_get<EL>(q.w, i); }
template <bool FOUR> __device__ __forceinline__ void bytes_store(uint8_t *p, uint32_t w, int n) {
  if constexpr (FOUR) {
    __builtin_nontemporal_store(w, reinterpret_cast<u32_any *>(p));
  } else {
#pragma unroll
    for (int i = 0; i < 3; ++i)
      if (i < n) p[i] = (uint8_t)(w >> (8 * i));
  }
}

// The tile of a workgroup and the four columns of a lane: the last lanes of a
// row of N columns take its last four again (they write the same bytes); a
// matrix of less than four columns has them one by one.
template <int64_t K, int64_t N> struct ColTile {
  static constexpr bool FOUR = N >= 4;
  static constexpr int64_t NB = (K + 31) / 32, CT = (N + MXC_COLS - 1) / MXC_COLS;
  int64_t n0, n, kb0, kb, k0;
  int rows;
  __device__ __forceinline__ ColTile() {
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / 64);
    n0 = (int64_t)(blockIdx.x % CT) * MXC_COLS;
    n = n0 + 4 * lane;
    if (n > N - 4) n = FOUR ? N - 4 : 0;
    kb0 = (int64_t)(blockIdx.x / CT) * MXC_BLOCKS;
    kb = kb0 + wave;
    k0 = kb * 32;
    rows = (int)(K - k0 < 32 ? K - k0 : 32);
  }
};

template <int EL, int FMT, int64_t K, int64_t N>
__device__ __forceinline__ void mx_quantize_cols(const void *__restrict__ x, void *__restrict__ codes, void *__restrict__ scales) {
  using Tile = ColTile<K, N>;
  constexpr int64_t NB = Tile::NB;
  constexpr bool FOUR = Tile::FOUR;
  __shared__ uint8_t sc[MXC_COLS][MXC_BLOCKS];
  const Tile t;
  if (t.kb < NB) {
    Quad4<EL> q[32];
    const char *src = (const char *)x + (t.k0 * N + t.n) * el_bytes<EL>;
#pragma unroll
    for (int i = 0; i < 32; ++i) q[i] = quad_load<EL, FOUR>(src + (int64_t)(i < t.rows ? i : 0) * N * el_bytes<EL>, (int)N);
    if (K % 32 != 0 && t.rows < 32) {
#pragma unroll
      for (int i = 1; i < 32; ++i)
        if (i >= t.rows) q[i] = Quad4<EL>{};
    }
    uint32_t m[4];
    if constexpr (EL == EL_F32) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        m[j] = 0;
#pragma unroll
        for (int i = 0; i < 32; ++i) m[j] = max_u32(m[j], q[i].w[j] & 0x7FFFFFFFu);
      }
    } else {
      uint32_t a = 0, b = 0;
#pragma unroll
      for (int i = 0; i < 32; ++i) a = max_u16x2(a, q[i].w[0] & 0x7FFF7FFFu), b = max_u16x2(b, q[i].w[1] & 0x7FFF7FFFu);
      m[0] = mag_f32<EL>(a & 0xFFFFu), m[1] = mag_f32<EL>(a >> 16);
      m[2] = mag_f32<EL>(b & 0xFFFFu), m[3] = mag_f32<EL>(b >> 16);
    }
    float inv[4];
    uint32_t keep = 0; // bytes of the columns whose block is finite
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t byte = mx_scale_byte<FMT>(m[j]);
      inv[j] = mx_inverse(byte);
      keep |= byte == 255 ? 0u : 0xFFu << (8 * j);
      const int64_t c = t.n - t.n0 + j; // (before the tile: another's column)
      if (c >= 0) sc[c][t.kb - t.kb0] = (uint8_t)byte;
    }
    if constexpr (FMT == MX_E2M1) {
      uint8_t *dst = (uint8_t *)codes + (t.k0 / 2) * N + t.n;
#pragma unroll
      for (int i = 0; i < 32; i += 2) {
        uint32_t w = 0;
        auto v = [&](int d, int j) { return quad_get<EL>(q[i + d], j) * inv[j]; };
        w = mx_pair4<0>(v(0, 0), v(1, 0), w);
        w = mx_pair4<1>(v(0, 1), v(1, 1), w);
        w = mx_pair4<2>(v(0, 2), v(1, 2), w);
        w = mx_pair4<3>(v(0, 3), v(1, 3), w);
        if (i < t.rows) bytes_store<FOUR>(dst + (int64_t)(i / 2) * N, w & keep, (int)N);
      }
    } else {
      uint8_t *dst = (uint8_t *)codes + t.k0 * N + t.n;
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        auto v = [&](int j) { return quad_get<EL>(q[i], j) * inv[j]; };
        uint32_t w = mx_pair8<FMT>(v(0), v(1), 0, false);
        w = mx_pair8<FMT>(v(2), v(3), w, true);
        if (i < t.rows) bytes_store<FOUR>(dst + (int64_t)i * N, w & keep, (int)N);
      }
    }
  }
  __syncthreads();
  const int64_t col = t.n0 + threadIdx.x;
  if (threadIdx.x < MXC_COLS && col < N) {
    uint8_t *dst = (uint8_t *)scales + col * NB + t.kb0;
    const u32x2 v = *reinterpret_cast<const u32x2 *>(sc[threadIdx.x]);
    if (t.kb0 + MXC_BLOCKS <= NB) {
      *reinterpret_cast<u32x2_any *>(dst) = v;
    } else {
      for (int i = 0; i < (int)(NB - t.kb0); ++i) dst[i] = (uint8_t)((i < 4 ? v.x : v.y) >> (8 * (i % 4)));
    }
  }
}

template <int EL, int FMT, int64_t K, int64_t N>
__device__ __forceinline__ void mx_dequantize_cols(const void *__restrict__ codes, const void *__restrict__ scales, void *__restrict__ out) {
  using Tile = ColTile<K, N>;
  constexpr int64_t NB = Tile::NB;
  constexpr bool FOUR = Tile::FOUR;
  __shared__ uint8_t sc[MXC_COLS][MXC_BLOCKS];
  const Tile t;
  const int64_t col = t.n0 + threadIdx.x;
  if (threadIdx.x < MXC_COLS && col < N) {
    const uint8_t *p = (const uint8_t *)scales + col * NB + t.kb0;
    u32x2 v = {0, 0};
    if (t.kb0 + MXC_BLOCKS <= NB) {
      v = *reinterpret_cast<const u32x2_any *>(p);
    } else {
#pragma unroll
      for (int i = 0; i < MXC_BLOCKS; ++i) {
        const uint32_t b = p[t.kb0 + i < NB ? i : 0];
        if (i < 4) v.x |= b << (8 * i);
        else v.y |= b << (8 * (i - 4));
      }
    }
    *reinterpret_cast<u32x2 *>(sc[threadIdx.x]) = v;
  }
  constexpr int P = FMT == MX_E2M1 ? 2 : 1; // k-rows a byte
  const uint8_t *src = (const uint8_t *)codes + (t.k0 / P) * N + t.n;
  char *dst = (char *)out + (t.k0 * N + t.n) * el_bytes<EL>;
  uint32_t w[32 / P];
#pragma unroll
  for (int i = 0; i < 32 / P; ++i) {
    const uint8_t *p = src + (t.kb < NB && i * P < t.rows ? (int64_t)i * N : t.kb < NB ? 0 : -(t.k0 / P) * N);
    if constexpr (FOUR) {
      w[i] = __builtin_nontemporal_load(reinterpret_cast<const u32_any *>(p));
    } else {
      w[i] = 0;
#pragma unroll
      for (int j = 0; j < 3; ++j) w[i] |= (uint32_t)p[j < N ? j : 0] << (8 * j);
    }
  }
  __syncthreads();
  if (t.kb >= NB) return;
  // (the row's last four columns may begin before the tile: their scales are
  // another tile's)
  float s[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int64_t c = t.n - t.n0 + j;
    s[j] = mx_scale(c >= 0 && c < MXC_COLS ? sc[c][t.kb - t.kb0] : ((const uint8_t *)scales)[(t.n + (FOUR || j < N ? j : 0)) * NB + t.kb]);
  }
  auto put = [&](int k, float a, float b, float c, float d) {
    if (k >= t.rows) return;
    a *= s[0], b *= s[1], c *= s[2], d *= s[3];
    char *p = dst + (int64_t)k * N * el_bytes<EL>;
    Pack<EL> o{};
    pack_set2<EL>(o, 0, a, b);
    pack_set2<EL>(o, 2, c, d);
    if constexpr (!FOUR) {
      pack_store_part<EL>(p, o, (int)N);
    } else if constexpr (EL == EL_F32) {
      __builtin_nontemporal_store(u32x4{o.w[0], o.w[1], o.w[2], o.w[3]}, reinterpret_cast<u32x4_any *>(p));
    } else {
      __builtin_nontemporal_store(u32x2{o.w[0], o.w[1]}, reinterpret_cast<u32x2_any *>(p));
    }
  };
#pragma unroll
  for (int i = 0; i < 32 / P; ++i) {
    if constexpr (FMT == MX_E2M1) {
      // byte j of the word is column j's two k
      const f32x2 a = mx_decode2<FMT>(w[i], 0), b = mx_decode2<FMT>(w[i], 1), c = mx_decode2<FMT>(w[i], 2), d = mx_decode2<FMT>(w[i], 3);
      put(2 * i, a.x, b.x, c.x, d.x);
      put(2 * i + 1, a.y, b.y, c.y, d.y);
    } else {
      const f32x2 a = mx_decode2<FMT>(w[i], 0), b = mx_decode2<FMT>(w[i], 1);
      put(i, a.x, a.y, b.x, b.y);
    }
  }
}

} // namespace hf
