// Attention over the paged 8-bit cache (hf_kv.h; hfusion.paged_attention).
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q k_j - max),  over the positions
//   j in (pos - WINDOW, pos] of the row's sequence whose blocks the table has
// in one pass with the running maximum and sum (f32); a row that sees nothing
// is zeros.  The matrix core takes 16-bit operands and sums in f32; codes are
// exact in both types.  Of bf16 queries, p_j times its block's value scale is
// rounded to bf16.  f16 has not the range for that: p_j is rounded by itself and
// the codes are scaled to a running reference exponent, exactly; a tile with
// blocks that lie further apart takes p_j as the sum of two bf16 numbers.
//
// Transposed products, so that nothing moves between lanes: S^T = K Q^T leaves
// a lane with four tokens' scores of one row, and these are the B operand of
// O^T = V^T P^T as they lie.  Which tokens the rows of a K tile are is free: a
// lane group g (16 lanes) is given tokens 16 g .. 16 g + 15 of 64, whose codes
// of one channel are 16 consecutive bytes of the cache's values.  Codes go from
// memory to registers and become 16-bit there.
#pragma once
#include "hf_kv.h"
#include "hf_mmsk.h"
#include "hf_mmwx.h"

namespace hf {

// eight codes times a power of two, as bf16 or as f16
template <int EL, int FMT> __device__ __forceinline__ v4i attn_decode8(uint32_t w0, uint32_t w1, float scale) {
  if constexpr (EL == EL_BF16) {
    return wx_decode8<FMT>(w0, w1, scale);
  } else {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    auto bits = [](h2 v) { return __builtin_bit_cast(int, v); };
    if constexpr (FMT == MX_E4M3)
      return v4i{bits(__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w0, scale, false)), bits(__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w0, scale, true)),
                 bits(__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w1, scale, false)), bits(__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w1, scale, true))};
    else
      return v4i{bits(__builtin_amdgcn_cvt_scalef32_pk_f16_bf8(w0, scale, false)), bits(__builtin_amdgcn_cvt_scalef32_pk_f16_bf8(w0, scale, true)),
                 bits(__builtin_amdgcn_cvt_scalef32_pk_f16_bf8(w1, scale, false)), bits(__builtin_amdgcn_cvt_scalef32_pk_f16_bf8(w1, scale, true))};
  }
}
// eight f32 rounded to bf16, or to f16
template <int EL> __device__ __forceinline__ v4i attn_round8(const float *p) {
  v4i o;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if constexpr (EL == EL_BF16) o[w] = (int)((uint32_t)f32_to_bf16_rne(p[2 * w]) | (uint32_t)f32_to_bf16_rne(p[2 * w + 1]) << 16);
    else
      o[w] = (int)((uint32_t)__builtin_bit_cast(uint16_t, (_Float16)p[2 * w]) | (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)p[2 * w + 1]) << 16);
  }
  return o;
}
// over the four lane groups that share a row
__device__ __forceinline__ float group_max(float v) {
  v = __builtin_fmaxf(v, __shfl_xor(v, 16));
  return __builtin_fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float group_add(float v) {
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}

// What a group of this op knows when it is compiled.  Sixteen matrix-core
// rows are GT heads of a kv head's group times N tokens of a sequence.
template <int EL_, int FMT_, int HQ_, int HK_, int D_, int BLOCK_, int64_t SLOTS_, int64_t PER_, int64_t NBLK_, int WINDOW_> struct Paged {
  static constexpr int EL = EL_, FMT = FMT_, HQ = HQ_, HK = HK_, D = D_, BLOCK = BLOCK_, WINDOW = WINDOW_;
  static constexpr int64_t SLOTS = SLOTS_, PER = PER_, NBLK = NBLK_, FAR = PER * BLOCK;
  static constexpr int G = HQ / HK, GT = G < 16 ? G : 16, GTILES = (G + 15) / 16, N = 16 / GT;
  static constexpr int KS = D / 32, DT = D / 16;
  static_assert(HQ % HK == 0 && D % 32 == 0 && D <= 256 && BLOCK % 16 == 0 && BLOCK <= 128 && (BLOCK & (BLOCK - 1)) == 0);
  __device__ static __forceinline__ bool inside(int s, int p) { return s >= 0 && s < SLOTS && p >= 0 && p < FAR; }
  // whether row t begins a group of tokens, and how many follow it there: rows
  // of a sequence with positions p, p + 1, ... up to a multiple of N
  __device__ static __forceinline__ int tokens(const int *seq, const int *pos, int64_t t, int64_t T) {
    const int s = seq[t], p = pos[t];
    if (!inside(s, p)) return 0;
    if (N == 1) return 1;
    if (t > 0 && p % N != 0 && seq[t - 1] == s && pos[t - 1] == p - 1) return 0;
    int n = 1;
#pragma unroll
    for (int i = 1; i < N; ++i)
      if (n == i && t + i < T && (p + i) % N != 0 && p + i < FAR && seq[t + i] == s && pos[t + i] == p + i) ++n;
    return n;
  }
};

struct PagedArgs {
  const uint16_t *q;
  const uint8_t *k, *ks, *v, *vs;
  const int *seq, *pos, *table;
  uint16_t *out;
  float scale; // of the scores, times log2 e
};

// Running state of 16 rows in a wave: lane l holds row l % 16, of O^T channels
// 16 dt + 4 (l / 16) + i; m is the same in the row's four lanes, sum each lane's own.
template <typename S> struct PagedState {
  v4f o[S::DT];
  float m, sum;
  uint32_t ref; // f16: o is in units of 2^(ref - 127)
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < S::DT; ++i) o[i] = v4f{0, 0, 0, 0};
    m = -__builtin_inff(), sum = 0, ref = S::EL == EL_BF16 ? 127 : 0;
  }
  __device__ __forceinline__ void times(float by) {
#pragma unroll
    for (int i = 0; i < S::DT; ++i) o[i] *= by;
  }
};

// Codes of 64 tokens of one kv head: keys as K tile u's rows (lane l: token 16
// (l % 16 / 4) + 4 u + l % 4), values as V^T tile dt's (lane l: channel 16 dt + l %
// 16, tokens 16 (l / 16) ..).
template <typename S> struct PagedTile {
  u32x4 k[4][(S::KS + 1) / 2], v[S::DT];
  uint32_t ks, vs; // scale bytes of the lane group's tokens
  bool there;      // their block is in the table
  __device__ __forceinline__ void load(const PagedArgs &a, int seq, int h, int b0) {
    const int lane = threadIdx.x % 64, r = lane % 16, g = lane / 16;
    const int *row = a.table + (int64_t)seq * S::PER;
    auto block = [&](int tok) {
      const int i = tok / S::BLOCK;
      return i < S::PER ? row[i] : -1;
    };
    const int bv = block(b0 + 16 * g), bk = S::BLOCK >= 64 ? bv : block(b0 + 16 * (r / 4));
    there = bv >= 0 && bv < S::NBLK;
    const int64_t pv = (int64_t)(there ? bv : 0) * S::HK + h, pk = (int64_t)(bk >= 0 && bk < S::NBLK ? bk : 0) * S::HK + h;
    ks = a.ks[pv], vs = a.vs[pv];
    const uint8_t *kp = a.k + pk * (S::BLOCK * S::D);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const uint8_t *p = kp + (b0 + 16 * (r / 4) + 4 * u + r % 4) % S::BLOCK * S::D;
#pragma unroll
      for (int c = 0; c < S::KS / 2; ++c) k[u][c] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_any *>(p + 64 * c + 16 * g));
      if constexpr (S::KS % 2 != 0) {
        const u32x2 w = __builtin_nontemporal_load(reinterpret_cast<const u32x2_any *>(p + 32 * (S::KS - 1) + 8 * g));
        k[u][S::KS / 2] = u32x4{w.x, w.y, 0, 0};
      }
    }
    const uint8_t *vp = a.v + pv * (S::BLOCK * S::D) + (b0 + 16 * g) % S::BLOCK;
#pragma unroll
    for (int dt = 0; dt < S::DT; ++dt) v[dt] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_any *>(vp + (16 * dt + r) * S::BLOCK));
  }
};

// The queries as the B operand: row r's channels in the order that the keys'
// codes have them (eight of step c: 64 (c / 2) + 16 g + 8 (c % 2), of an odd last
// step 32 c + 8 g).
template <typename S> __device__ __forceinline__ void paged_query(const PagedArgs &a, int64_t t, int n, int h, int gt, v4i (&q)[S::KS]) {
  const int lane = threadIdx.x % 64, r = lane % 16, g = lane / 16;
  const int i = r / S::GT, head = gt * 16 + r % S::GT;
  const bool ok = i < n && head < S::G;
  const uint16_t *p = a.q + ((t + (ok ? i : 0)) * S::HQ + h * S::G + (ok ? head : 0)) * S::D;
#pragma unroll
  for (int c = 0; c < S::KS; ++c) {
    const int d = S::KS % 2 != 0 && c == S::KS - 1 ? 32 * c + 8 * g : 64 * (c / 2) + 16 * g + 8 * (c % 2);
    const u32x4 w = *reinterpret_cast<const u32x4_any *>(p + d);
    q[c] = ok ? v4i{(int)w.x, (int)w.y, (int)w.z, (int)w.w} : v4i{0, 0, 0, 0};
  }
}

// One tile of 64 tokens from b0 on.  pos: the lane's row's position (-1: no
// row), lo and hi: the first and last of the tile's rows.
template <typename S> __device__ __forceinline__ void paged_step(PagedState<S> &st, PagedTile<S> &t, const v4i (&q)[S::KS], const PagedArgs &a, int b0,
                                                                  int pos, int lo, int hi) {
  const int g = threadIdx.x % 64 / 16;
  v4f s[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    s[u] = v4f{0, 0, 0, 0};
#pragma unroll
    for (int c = 0; c < S::KS; ++c) {
      const u32x4 w = t.k[u][c / 2];
      const v4i kf = c % 2 ? attn_decode8<S::EL, S::FMT>(w.z, w.w, 1.0f) : attn_decode8<S::EL, S::FMT>(w.x, w.y, 1.0f);
      s[u] = Mfma16<(S::EL == EL_BF16 ? MK_BF16 : MK_F16)>::run(kf, q[c], s[u]);
    }
  }
  const float f = a.scale * mx_scale(t.ks);
#pragma unroll
  for (int u = 0; u < 4; ++u)
#pragma unroll
    for (int i = 0; i < 4; ++i) s[u][i] *= f;
  // tokens that some row does not see
  const int at = b0 + 16 * g;
  const bool whole = __all(t.there && b0 + 63 <= lo && (S::WINDOW == 0 || b0 > hi - S::WINDOW));
  auto sees = [&](int tok) { return t.there && tok <= pos && (S::WINDOW == 0 || tok > pos - S::WINDOW); };
  if (!whole) {
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[u][i] = sees(at + 4 * u + i) ? s[u][i] : -__builtin_inff();
    // (behind the last position the cache may hold anything, NaN too)
    const int n = t.there ? hi + 1 - at : 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const uint32_t keep = n >= 4 * w + 4 ? 0xFFFFFFFFu : n <= 4 * w ? 0u : 0xFFFFFFFFu >> (8 * (4 * w + 4 - n));
#pragma unroll
      for (int dt = 0; dt < S::DT; ++dt) t.v[dt][w] &= keep;
    }
  }
  float top = s[0][0];
#pragma unroll
  for (int u = 0; u < 4; ++u)
#pragma unroll
    for (int i = 0; i < 4; ++i) top = __builtin_fmaxf(top, s[u][i]);
  top = __builtin_fmaxf(st.m, group_max(top));
  const float m = top == -__builtin_inff() ? 0.0f : top; // (a row that has seen nothing)
  const float was = st.m == top ? 1.0f : __builtin_amdgcn_exp2f(st.m - m);
  st.m = top;
  float sum = 0;
  float p[16];
#pragma unroll
  for (int u = 0; u < 4; ++u)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      p[4 * u + i] = __builtin_amdgcn_exp2f(s[u][i] - m);
      sum += p[4 * u + i];
    }
  st.sum = st.sum * was + sum;
  auto scaled = [&](float by) { // (a scale may be NaN, also of what is not seen)
#pragma unroll
    for (int i = 0; i < 16; ++i) p[i] *= by;
    if (!whole)
#pragma unroll
      for (int i = 0; i < 16; ++i) p[i] = sees(at + i) ? p[i] : 0.0f;
  };
  if constexpr (S::EL == EL_BF16) {
    if (!__all(was == 1.0f)) st.times(was);
    scaled(mx_scale(t.vs));
    const v4i p0 = attn_round8<EL_BF16>(p), p1 = attn_round8<EL_BF16>(p + 8);
#pragma unroll
    for (int dt = 0; dt < S::DT; ++dt) {
      st.o[dt] = Mfma16<MK_BF16>::run(wx_decode8<S::FMT>(t.v[dt].x, t.v[dt].y, 1.0f), p0, st.o[dt]);
      st.o[dt] = Mfma16<MK_BF16>::run(wx_decode8<S::FMT>(t.v[dt].z, t.v[dt].w, 1.0f), p1, st.o[dt]);
    }
    return;
  }
  // the exponents of the blocks that are read
  const bool read = t.there && at <= hi;
  const bool bad = __any(read && t.vs == 255);
  uint32_t big = read && t.vs != 255 ? t.vs : 0, small = read ? t.vs : 255;
  if constexpr (S::BLOCK < 64) {
#pragma unroll
    for (int k = 16; k < 64; k *= 2) big = max_u32(big, (uint32_t)__shfl_xor((int)big, k)), small = 255 - max_u32(255 - small, 255 - (uint32_t)__shfl_xor((int)small, k));
  }
  big = __builtin_amdgcn_readfirstlane(big), small = __builtin_amdgcn_readfirstlane(small);
  const uint32_t ref = max_u32(st.ref, big);
  const float by = ref - st.ref > 126 ? 0.0f : u2f((127 - (ref - st.ref)) << 23);
  st.ref = ref;
  if (!__all(was * by == 1.0f)) st.times(was * by);
  if (!bad && (int)(ref - small) <= 8) {
    const float vs = read ? u2f((127 - (ref - t.vs)) << 23) : 1.0f;
    const v4i p0 = attn_round8<EL_F16>(p), p1 = attn_round8<EL_F16>(p + 8);
#pragma unroll
    for (int dt = 0; dt < S::DT; ++dt) {
      st.o[dt] = Mfma16<MK_F16>::run(attn_decode8<EL_F16, S::FMT>(t.v[dt].x, t.v[dt].y, vs), p0, st.o[dt]);
      st.o[dt] = Mfma16<MK_F16>::run(attn_decode8<EL_F16, S::FMT>(t.v[dt].z, t.v[dt].w, vs), p1, st.o[dt]);
    }
    return;
  }
  scaled(t.vs == 255 ? __builtin_nanf("") : ref - t.vs > 126u && t.vs < ref ? 0.0f : u2f((127 + t.vs - ref) << 23));
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const v4i p0 = attn_round8<EL_BF16>(p), p1 = attn_round8<EL_BF16>(p + 8);
#pragma unroll
    for (int dt = 0; dt < S::DT; ++dt) {
      st.o[dt] = Mfma16<MK_BF16>::run(wx_decode8<S::FMT>(t.v[dt].x, t.v[dt].y, 1.0f), p0, st.o[dt]);
      st.o[dt] = Mfma16<MK_BF16>::run(wx_decode8<S::FMT>(t.v[dt].z, t.v[dt].w, 1.0f), p1, st.o[dt]);
    }
    // what the rounding left
#pragma unroll
    for (int i = 0; i < 16; ++i) p[i] -= bf16_to_f32(f32_to_bf16_rne(p[i]));
  }
}

// Rows of a few tokens: a workgroup has the rows of one group of tokens of a
// kv head, its four waves take its tiles in turn and meet in LDS.
template <typename S> __device__ __forceinline__ void paged_rows(const PagedArgs &a, int64_t T) {
  constexpr int HEADS = S::HK * S::GTILES, PITCH = S::D + 4, CH = S::D / 8;
  __shared__ __attribute__((aligned(16))) float so[4][16][PITCH];
  __shared__ float sm[4][16], ss[4][16];
  const int64_t t = blockIdx.x / HEADS;
  const int h = blockIdx.x % HEADS / S::GTILES, gt = blockIdx.x % S::GTILES;
  const int n = S::tokens(a.seq, a.pos, t, T);
  if (n == 0) return;
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, r = lane % 16, g = lane / 16;
  const int seq = a.seq[t], lo = a.pos[t], hi = lo + n - 1;
  v4i q[S::KS];
  paged_query<S>(a, t, n, h, gt, q);
  const int pos = r / S::GT < n ? lo + r / S::GT : -1;
  PagedState<S> st;
  st.clear();
  int b = S::WINDOW && lo >= S::WINDOW ? (lo - S::WINDOW + 1) / 64 * 64 : 0;
  for (b += 64 * wave; b <= hi; b += 256) {
    PagedTile<S> tile;
    tile.load(a, seq, h, b);
    paged_step<S>(st, tile, q, a, b, pos, lo, hi);
  }
  if constexpr (S::EL != EL_BF16) st.times(mx_scale(st.ref));
  const float sum = group_add(st.sum);
  if (g == 0) sm[wave][r] = st.m, ss[wave][r] = sum;
#pragma unroll
  for (int dt = 0; dt < S::DT; ++dt) *reinterpret_cast<v4f *>(&so[wave][r][16 * dt + 4 * g]) = st.o[dt];
  __syncthreads();
  for (int i = threadIdx.x; i < 16 * CH; i += 256) {
    const int row = i / CH, d = i % CH * 8, tok = row / S::GT, head = gt * 16 + row % S::GT;
    if (tok >= n || head >= S::G) continue;
    float m = sm[0][row];
#pragma unroll
    for (int w = 1; w < 4; ++w) m = __builtin_fmaxf(m, sm[w][row]);
    float f[8] = {0, 0, 0, 0, 0, 0, 0, 0}, l = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float by = m == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(sm[w][row] - m);
      l += ss[w][row] * by;
#pragma unroll
      for (int k = 0; k < 8; ++k) f[k] += so[w][row][d + k] * by;
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] = l == 0 ? 0.0f : f[k] / l;
    store8<S::EL>(a.out + ((t + tok) * S::HQ + h * S::G + head) * S::D + d, f);
  }
}

} // namespace hf
