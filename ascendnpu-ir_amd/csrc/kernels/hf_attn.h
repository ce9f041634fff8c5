// Attention over the paged 8-bit cache (hf_kv.h; hfusion.paged_attention).
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q k_j - max),  over the positions
//   j in (pos - WINDOW, pos] of the row's sequence whose blocks the table has
// in one pass with the running maximum and sum (f32); a row that sees nothing
// is zeros.  The matrix core takes 16-bit operands and sums in f32; codes are
// exact in both types.  A probability is rounded once to the queries' type, which
// costs a result some half of a step of its own; the sum of a few tokens' row takes
// it unrounded, of a prompt's rounded.  Of f16, which has not the range for
// values' scales, see where they are applied.
//
// Which kernel by the row count (the compiler has the bounds and both sides'
// times): up to a group of tokens a sequence, rows of a few tokens, whose cost is
// the cache's bytes; more of them a prompt's rows, whose cost is arithmetic.
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
    using T = std::conditional_t<EL == EL_BF16, __bf16, _Float16>;
    typedef T t2 __attribute__((ext_vector_type(2)));
    o[w] = __builtin_bit_cast(int, __builtin_convertvector(f32x2{p[2 * w], p[2 * w + 1]}, t2));
  }
  return o;
}
// c and the two 16-bit numbers in w
template <int EL> __device__ __forceinline__ float attn_sum2(int w, float c) {
  using T = std::conditional_t<EL == EL_BF16, __bf16, _Float16>;
  typedef T t2 __attribute__((ext_vector_type(2)));
  if constexpr (EL == EL_BF16) return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(t2, w), __builtin_bit_cast(t2, 0x3F803F80), c, false);
  else return __builtin_amdgcn_fdot2(__builtin_bit_cast(t2, w), __builtin_bit_cast(t2, 0x3C003C00), c, false);
}
// the value of the lane 16 or 32 lanes away, combined with this one's
template <int BY, typename F> __device__ __forceinline__ float with_lane(float v, F f) {
  typedef unsigned u2 __attribute__((ext_vector_type(2)));
  const u2 r = __builtin_bit_cast(u2, BY == 16 ? __builtin_amdgcn_permlane16_swap(f2u(v), f2u(v), false, false) : __builtin_amdgcn_permlane32_swap(f2u(v), f2u(v), false, false));
  return f(u2f(r.x), u2f(r.y));
}
__device__ __forceinline__ float max2(float a, float b) { return __builtin_fmaxf(a, b); }
// over the four lane groups that share a row
__device__ __forceinline__ float group_max(float v) { return with_lane<32>(with_lane<16>(v, max2), max2); }
__device__ __forceinline__ float group_add(float v) {
  auto add = [](float a, float b) { return a + b; };
  return with_lane<32>(with_lane<16>(v, add), add);
}

// What a group of this op knows when it is compiled.  Sixteen matrix-core
// rows are GT heads of a kv head's group times N tokens of a sequence.
template <int EL_, int FMT_, int HQ_, int HK_, int D_, int BLOCK_, int64_t SLOTS_, int64_t PER_, int64_t NBLK_, int WINDOW_> struct Paged {
  static constexpr int EL = EL_, FMT = FMT_, HQ = HQ_, HK = HK_, D = D_, BLOCK = BLOCK_, WINDOW = WINDOW_;
  static constexpr int64_t SLOTS = SLOTS_, PER = PER_, NBLK = NBLK_, FAR = PER * BLOCK;
  static constexpr int G = HQ / HK, GT = G < 16 ? G : 16, GTILES = (G + 15) / 16, N = 16 / GT;
  static constexpr int KS = D / 32, DT = D / 16;
  // Probabilities and their sums are in units of 2^-LIFT: a prompt's are up to 2^6,
  // and f16, which ends at 2^16, has all bits of a number from 2^-14 on
  static constexpr float LIFT = EL == EL_F16 ? 9 : 0;
  static_assert(HQ % HK == 0 && D % 32 == 0 && D <= 256 && BLOCK % 16 == 0 && BLOCK <= 128 && (BLOCK & (BLOCK - 1)) == 0);
  __device__ static __forceinline__ bool inside(int s, int p) { return s >= 0 && s < SLOTS && p >= 0 && p < FAR; }
  // whether row t begins a group of tokens, and how many follow it there: rows
  // of a sequence with positions p, p + 1, ... up to a multiple of N
  // (all of them are asked for at once)
  __device__ static __forceinline__ int tokens(const int *seq, const int *pos, int64_t t, int64_t T, int &s, int &p) {
    int sn[N], pn[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int64_t at = t + i < T ? t + i : T - 1;
      sn[i] = seq[at], pn[i] = pos[at];
    }
    const int64_t up = t > 0 ? t - 1 : 0;
    const int su = N > 1 ? seq[up] : 0, pu = N > 1 ? pos[up] : 0;
    s = sn[0], p = pn[0];
    if (!inside(s, p) || (N > 1 && t > 0 && p % N != 0 && su == s && pu == p - 1)) return 0;
    int n = 1;
#pragma unroll
    for (int i = 1; i < N; ++i)
      if (n == i && t + i < T && (p + i) % N != 0 && p + i < FAR && sn[i] == s && pn[i] == p + i) ++n;
    return n;
  }
  // whether row t, of sequence s at p, is one of at most FEW that follow each
  // other in the batch (all rows about it are asked for at once)
  static constexpr int FEW = N > 4 ? N : 4;
  __device__ static __forceinline__ bool few(const int *seq, const int *pos, int64_t t, int64_t T, int s, int p) {
    int before = 0, after = 0;
#pragma unroll
    for (int i = 1; i <= FEW; ++i) {
      const int64_t b = t - i < 0 ? 0 : t - i, e = t + i < T ? t + i : T - 1;
      const bool up = seq[b] == s && pos[b] == p - i, down = seq[e] == s && pos[e] == p + i;
      before += before == i - 1 && t - i >= 0 && p - i >= 0 && up;
      after += after == i - 1 && t + i < T && p + i < FAR && down;
    }
    return before + after < FEW;
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
  // the blocks of the lane's keys and values
  __device__ static __forceinline__ void blocks(const PagedArgs &a, int seq, int b0, int &bk, int &bv) {
    const int lane = threadIdx.x % 64;
    const int *row = a.table + (int64_t)seq * S::PER;
    auto block = [&](int tok) {
      const int i = tok / S::BLOCK;
      return i < S::PER ? row[i] : -1;
    };
    bv = block(b0 + 16 * (lane / 16)), bk = S::BLOCK >= 64 ? bv : block(b0 + 16 * (lane % 16 / 4));
  }
  __device__ __forceinline__ void load(const PagedArgs &a, int h, int b0, int bk, int bv) {
    const int lane = threadIdx.x % 64, r = lane % 16, g = lane / 16;
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

// The largest scale byte, 2^16, whose unit a row's sums are held in while it may
// see small values alone: those keep their bits down to 2^-110.
constexpr uint32_t kTopScale = 143;

// Whether rows at lo .. hi see some of the sixteen positions from `at` on.
// Elsewhere, behind the last row's position and before the first one's window,
// the cache may hold anything, NaN and any scale.
template <typename S> __device__ __forceinline__ bool some_seen(int at, int lo, int hi) { return at <= hi && (S::WINDOW == 0 || at + 15 > lo - S::WINDOW); }
// the codes in word w of sixteen that are among the first n, less the first `gone`
template <typename S> __device__ __forceinline__ uint32_t kept_codes(int w, int n, int gone) {
  uint32_t keep = n >= 4 * w + 4 ? 0xFFFFFFFFu : n <= 4 * w ? 0u : 0xFFFFFFFFu >> (8 * (4 * w + 4 - n));
  if constexpr (S::WINDOW != 0) keep &= gone <= 4 * w ? 0xFFFFFFFFu : gone >= 4 * w + 4 ? 0u : 0xFFFFFFFFu << (8 * (gone - 4 * w));
  return keep;
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
  const int to = pos - at, from = to - S::WINDOW; // (compares with constants)
  auto sees = [&](int i) { return t.there && i <= to && (S::WINDOW == 0 || i > from); };
  if (!whole) {
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[u][i] = sees(4 * u + i) ? s[u][i] : -__builtin_inff();
    const int n = t.there ? hi + 1 - at : 0, gone = lo - S::WINDOW + 1 - at;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const uint32_t keep = kept_codes<S>(w, n, gone);
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
      p[4 * u + i] = __builtin_amdgcn_exp2f(s[u][i] - (m - S::LIFT));
      sum += p[4 * u + i];
    }
  st.sum = st.sum * was + sum;
  auto scaled = [&](float by) { // (a scale may be NaN, also of what is not seen)
#pragma unroll
    for (int i = 0; i < 16; ++i) p[i] *= by;
    if (!whole)
#pragma unroll
      for (int i = 0; i < 16; ++i) p[i] = sees(i) ? p[i] : 0.0f;
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
  // f16: p by itself, and the codes scaled to a running reference exponent, that
  // of the largest block up to kTopScale (a row may see small ones alone); where
  // a block lies above it, or further below than f16 reaches, p times its scale as
  // the sum of two bf16 numbers
  // (a tile of one block is read)
  const bool read = t.there && (S::BLOCK >= 64 || some_seen<S>(at, lo, hi));
  const bool bad = __any(read && t.vs == 255);
  uint32_t big = read && t.vs != 255 ? t.vs : 0, small = read ? t.vs : 255;
  if constexpr (S::BLOCK < 64) {
#pragma unroll
    for (int k = 16; k < 64; k *= 2) big = max_u32(big, (uint32_t)__shfl_xor((int)big, k)), small = 255 - max_u32(255 - small, 255 - (uint32_t)__shfl_xor((int)small, k));
  }
  big = __builtin_amdgcn_readfirstlane(big), small = __builtin_amdgcn_readfirstlane(small);
  const uint32_t ref = max_u32(st.ref, big < kTopScale ? big : kTopScale);
  const float by = ref - st.ref > 126 ? 0.0f : u2f((127 - (ref - st.ref)) << 23);
  st.ref = ref;
  if (!__all(was * by == 1.0f)) st.times(was * by);
  if (!bad && big <= ref && (int)(ref - small) <= 8) {
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

// ---------------------------------------------------------------- rows of a few tokens
// A unit is the rows of one group of tokens and one kv head (of a group of more
// than 16 query heads, 16 of them); its tiles are those that hold a visible
// position.  16-row products: a kv head's query heads share its codes, and the
// tokens of a sequence that follow each other.  Memory bounds long caches: one
// row over 32768 positions 19.9 us (67 MB; 16.9 of it the pieces at 4.0 TB/s, 4
// the join), 48 rows over up to 8100 85.7 (405 MB, 4.7 TB/s).  Eight sequences of
// four tokens over up to 500 positions take 7.4: positions, table, codes and
// eight tiles in a row for the longest, each waiting for the one before.
template <typename S> struct PagedUnits {
  static constexpr int HEADS = S::HK * S::GTILES, ROWS = S::GT * S::N, CH = S::D / 8;
  __device__ static __forceinline__ int first(int lo) { return S::WINDOW && lo >= S::WINDOW ? (lo - S::WINDOW + 1) / 64 : 0; }
  // tiles of a group of n tokens from position lo on
  __device__ static __forceinline__ int tiles(int lo, int n) { return (lo + n - 1) / 64 - first(lo) + 1; }
};
// What WV waves share when they join their states.
template <typename S, int WV> struct PagedJoin {
  float o[WV][16][S::D + 4], m[WV][16], sum[WV][16];
};

// Tiles t0 .. t1 - 1 of the unit of n tokens from row t on (sequence seq,
// positions from lo on), by the workgroup's WV waves in turn, joined in LDS: the
// rows' results to out, or as a part (not divided by the sum; the running
// maximum and the sum in stats, two of each row) to o and stats.
template <typename S, int WV>
__device__ __forceinline__ void paged_part(const PagedArgs &a, PagedJoin<S, WV> &join, int64_t t, int n, int seq, int lo, int hh, int t0, int t1,
                                           float *o, float *stats) {
  using U = PagedUnits<S>;
  const int h = hh / S::GTILES, gt = hh % S::GTILES;
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, r = lane % 16, g = lane / 16;
  const int hi = lo + n - 1;
  v4i q[S::KS];
  paged_query<S>(a, t, n, h, gt, q);
  const int pos = r / S::GT < n ? lo + r / S::GT : -1;
  PagedState<S> st;
  st.clear();
  int bk = 0, bv = 0;
  if (t0 + wave < t1) PagedTile<S>::blocks(a, seq, 64 * (t0 + wave), bk, bv);
  for (int i = t0 + wave; i < t1; i += WV) {
    PagedTile<S> tile;
    tile.load(a, h, 64 * i, bk, bv);
    // (the next tile's blocks are asked for ahead, its codes are not: their
    // registers cost a third of the waves, and the other waves' codes are on
    // their way instead)
    if (i + WV < t1) PagedTile<S>::blocks(a, seq, 64 * (i + WV), bk, bv);
    paged_step<S>(st, tile, q, a, 64 * i, pos, lo, hi);
  }
  if constexpr (S::EL != EL_BF16) st.times(mx_scale(st.ref));
  const float sum = group_add(st.sum);
  if (g == 0) join.m[wave][r] = st.m, join.sum[wave][r] = sum;
#pragma unroll
  for (int dt = 0; dt < S::DT; ++dt) *reinterpret_cast<v4f *>(&join.o[wave][r][16 * dt + 4 * g]) = st.o[dt];
  __syncthreads();
  for (int i = threadIdx.x; i < U::ROWS * U::CH; i += 64 * WV) {
    const int row = i / U::CH, d = i % U::CH * 8, tok = row / S::GT, head = gt * 16 + row % S::GT;
    if (tok >= n || head >= S::G) continue;
    float m = join.m[0][row];
#pragma unroll
    for (int w = 1; w < WV; ++w) m = __builtin_fmaxf(m, join.m[w][row]);
    float f[8] = {0, 0, 0, 0, 0, 0, 0, 0}, l = 0;
#pragma unroll
    for (int w = 0; w < WV; ++w) {
      // (a wave that has seen nothing; its sum may be NaN)
      const float by = join.m[w][row] == m ? 1.0f : __builtin_amdgcn_exp2f(join.m[w][row] - m);
      l += join.sum[w][row] * by;
#pragma unroll
      for (int k = 0; k < 8; ++k) f[k] += join.o[w][row][d + k] * by;
    }
    if (o) {
      *reinterpret_cast<v4f *>(o + row * S::D + d) = v4f{f[0], f[1], f[2], f[3]};
      *reinterpret_cast<v4f *>(o + row * S::D + d + 4) = v4f{f[4], f[5], f[6], f[7]};
      if (d == 0) stats[2 * row] = m, stats[2 * row + 1] = l;
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) f[k] = l == 0 ? 0.0f : f[k] / l;
      store8<S::EL>(a.out + ((t + tok) * S::HQ + h * S::G + head) * S::D + d, f);
    }
  }
  __syncthreads(); // (join is written again)
}

// A workgroup a unit.
template <typename S, int WV> __device__ __forceinline__ void paged_rows(const PagedArgs &a, int64_t T) {
  using U = PagedUnits<S>;
  __shared__ __attribute__((aligned(16))) PagedJoin<S, WV> join;
  const int64_t t = blockIdx.x / U::HEADS;
  int seq, lo;
  const int n = S::tokens(a.seq, a.pos, t, T, seq, lo);
  if (n == 0) return;
  const int t0 = U::first(lo);
  paged_part<S, WV>(a, join, t, n, seq, lo, blockIdx.x % U::HEADS, t0, t0 + U::tiles(lo, n), nullptr, nullptr);
}

// The rows beside a prompt's that come a few at a time (Paged::few): PagedPrompt
// would take a tile's sequences one after another, a workgroup here takes one
// unit.  BLOCKS workgroups, each a head and every STEP-th row of the batch, so
// that neighbours are different workgroups'.  flags: of the first TILES tiles
// of PagedPrompt, whether they have such rows (of 10495 rows of prompts alone
// this launch takes 5 us, 7 where each workgroup reads every row's neighbours).
// us of a call, tokens of 63 sequences of 100 to 8100 positions beside a prompt
// of 300, 2000 and 4000 rows: 156, 193, 299; the tokens alone 108, the prompts
// 20, 76, 159.  512 workgroups: three tokens a sequence beside 1000 rows 289,
// 237 so.
template <typename S> struct PagedFew {
  using U = PagedUnits<S>;
  static constexpr int STEP = 1024 / U::HEADS, BLOCKS = STEP * U::HEADS, TILES = 4096;
  static_assert(U::HEADS <= 1024);
  __device__ static __forceinline__ void rows(const PagedArgs &a, int64_t T, const int *flags, int block) {
    __shared__ __attribute__((aligned(16))) PagedJoin<S, 4> join;
    __shared__ uint64_t found[4];
    const int tid = threadIdx.x, hh = block % U::HEADS;
    for (int64_t base = block / U::HEADS; base < T; base += 256 * STEP) {
      const int64_t mine = base + tid * STEP, tile = mine / (128 / S::GT);
      int seq, lo;
      bool one = mine < T && (tile >= TILES || flags[tile]);
      if (!__syncthreads_or(one)) continue;
      one = one && S::tokens(a.seq, a.pos, mine, T, seq, lo) > 0 && S::few(a.seq, a.pos, mine, T, seq, lo);
      const uint64_t some = __ballot(one);
      if (tid % 64 == 0) found[tid / 64] = some;
      __syncthreads();
      for (int w = 0; w < 4; ++w)
        for (uint64_t left = found[w]; left; left &= left - 1) {
          const int64_t t = base + (64 * w + __builtin_ctzll(left)) * STEP;
          const int n = S::tokens(a.seq, a.pos, t, T, seq, lo), t0 = U::first(lo);
          paged_part<S, 4>(a, join, t, n, seq, lo, hh, t0, t0 + U::tiles(lo, n), nullptr, nullptr);
        }
      __syncthreads(); // (found is written again)
    }
  }
};

// Units of different lengths: one is cut into pieces of at most `run` tiles, a
// workgroup a piece, the longest first; units of several pieces leave parts,
// which join() adds in order.  run makes as many pieces as fill the chip with
// the units that stay whole: PIECES less the units, LEAST to SHARED of them.  us of
// a call, with 512, 768 (taken), 1536 (of 2048 in all) at most: one row over 32768
// positions 19.8, 19.8, 24.1; over 131072 49, 53, 57; 48 rows over up to 8100 90, 85,
// 79 (a workgroup a unit 114, as long as the longest takes); 4 over up to 4000 14.7,
// 14.8, 14.9 (30.7).
// Up to MOST rows: every workgroup adds up the units' tiles itself, which takes
// it some 2 us.
// ws: the number of records, one a token of a unit in parts; then for each part
// the rows' maximum and sum, and the rows.
template <typename S, int WV> struct PagedSplit {
  using U = PagedUnits<S>;
  static constexpr int MOST = 1024, PIECES = 1024, LEAST = 256, SHARED = 768, THREADS = 64 * WV, PER = (MOST + THREADS - 1) / THREADS;
  // (a unit has at most 2^20 tiles, less than the longest `run`)
  static_assert(S::FAR <= 1 << 26 && (int64_t)MOST * U::HEADS < (int64_t(1) << 30));
  struct Record { // a token (row t, `token` of its unit) of a unit in parts
    int t, token, hh, part, parts, pad[3];
  };
  // units in parts are at most SHARED, and have at most SHARED parts more than that
  static constexpr int64_t STATS = 32 + SHARED * S::N * sizeof(Record), ROWS = STATS + 2 * SHARED * U::ROWS * 8, BYTES = ROWS + 2ll * SHARED * U::ROWS * S::D * 4;
  __device__ static __forceinline__ float *stats(char *ws, int part) { return reinterpret_cast<float *>(ws + STATS) + part * (U::ROWS * 2); }
  __device__ static __forceinline__ float *part(char *ws, int part) { return reinterpret_cast<float *>(ws + ROWS) + (int64_t)part * (U::ROWS * S::D); }

  // sums of M values over the threads before this one, and over all
  template <int M> __device__ static __forceinline__ void before(int (&v)[M], int (&total)[M], int (*tops)[WV]) {
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    int sum[M];
    auto step = [](int a, auto ctrl, auto rows) { return a + __builtin_amdgcn_update_dpp(0, a, decltype(ctrl)::value, decltype(rows)::value, 0xF, false); };
    using All = std::integral_constant<int, 0xF>;
#pragma unroll
    for (int j = 0; j < M; ++j) {
      sum[j] = step(v[j], std::integral_constant<int, 0x111>{}, All{});                                // one lane up in its row of sixteen
      sum[j] = step(sum[j], std::integral_constant<int, 0x112>{}, All{});                              // two
      sum[j] = step(sum[j], std::integral_constant<int, 0x114>{}, All{});                              // four
      sum[j] = step(sum[j], std::integral_constant<int, 0x118>{}, All{});                              // eight
      sum[j] = step(sum[j], std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xA>{}); // a row's last lane to the next row
      sum[j] = step(sum[j], std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xC>{}); // lane 31 to the upper half
      if (lane == 63) tops[j][wave] = sum[j];
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < M; ++j) {
      sum[j] -= v[j], total[j] = 0;
#pragma unroll
      for (int w = 0; w < WV; ++w) {
        sum[j] += w < wave ? tops[j][w] : 0;
        total[j] += tops[j][w];
      }
      v[j] = sum[j];
    }
  }

  // grid: T * HEADS + SHARED
  __device__ static __forceinline__ void rows(const PagedArgs &a, int64_t T, char *ws) {
    __shared__ __attribute__((aligned(16))) PagedJoin<S, WV> join;
    __shared__ int tops[6][WV];
    struct Found {
      int t, n, seq, lo, tiles, in, shared, part;
    };
    __shared__ Found found;
    // a thread has PER rows, one after another
    const int tid = threadIdx.x, per = (int)((T + THREADS - 1) / THREADS);
    int tiles[PER], n[PER], seq[PER], lo[PER], size[2] = {0, 0}, sizes[2];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int64_t t = tid * per + i;
      n[i] = i < per && t < T ? S::tokens(a.seq, a.pos, t, T, seq[i], lo[i]) : 0;
      tiles[i] = n[i] ? U::tiles(lo[i], n[i]) : 0;
      size[0] += tiles[i], size[1] += n[i] > 0;
    }
    before(size, sizes, tops);
    const int64_t all = (int64_t)sizes[0] * U::HEADS;
    int want = PIECES - sizes[1] * U::HEADS;
    want = want < LEAST ? LEAST : want > SHARED ? SHARED : want;
    // (every wave as many; a batch of padding alone has none)
    int64_t few = ((all + want - 1) / want + WV - 1) / WV * WV;
    few = few < WV ? WV : few > 1 << 24 ? 1 << 24 : few;
    const int run = (int)few;
    // pieces of `run` tiles, shorter ones, tokens of units in parts, and parts, of the thread's rows
    int count[4] = {0, 0, 0, 0}, counts[4];
    auto add = [&](int i) {
      const int full = tiles[i] / run, rest = tiles[i] % run != 0, c = full + rest;
      count[0] += full, count[1] += rest, count[2] += c > 1 ? n[i] : 0, count[3] += c > 1 ? c : 0;
    };
#pragma unroll
    for (int i = 0; i < PER; ++i) add(i);
    before(count, counts, tops + 2);
    if (blockIdx.x == 0 && tid == 0) *reinterpret_cast<int *>(ws) = counts[2] * U::HEADS;
    // the longest pieces first: those that start last are short
    int piece = (int)blockIdx.x;
    const bool shorter = piece >= counts[0] * U::HEADS;
    if (shorter) piece -= counts[0] * U::HEADS;
    if (shorter && piece >= counts[1] * U::HEADS) return;
    // the row whose piece this is: the thread that has it says so
    const int x = piece / U::HEADS;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int b = shorter ? count[1] : count[0], shared = count[2], part = count[3];
      add(i);
      if (b <= x && x < (shorter ? count[1] : count[0])) found = Found{tid * per + i, n[i], seq[i], lo[i], tiles[i], piece - b * U::HEADS, shared, part};
    }
    __syncthreads();
    auto one = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
    const int w = one(found.tiles), full = w / run, cuts = full + (w % run != 0), in = one(found.in);
    // (a head's pieces lie together)
    const int hh = shorter ? in : in / full, k = shorter ? full : in % full, t0 = U::first(one(found.lo)), b = k * run, e = b + run < w ? b + run : w;
    const int slot = one(found.part) * U::HEADS + hh * cuts + k;
    if (cuts > 1 && k == 0 && tid < found.n)
      reinterpret_cast<Record *>(ws + 32)[(found.shared + tid) * U::HEADS + hh] = Record{found.t + tid, tid, hh, slot, cuts, {0, 0, 0}};
    paged_part<S, WV>(a, join, one(found.t), one(found.n), one(found.seq), one(found.lo), hh, t0 + b, t0 + e, cuts > 1 ? part(ws, slot) : nullptr,
                      stats(ws, slot));
  }

  // The tokens of units in parts: a workgroup a head, its four waves a quarter
  // of the parts each.
  static constexpr int BLOCKS = 1024;
  __device__ static __forceinline__ void join(const PagedArgs &a, const char *ws_) {
    constexpr int L = S::D / 4, GROUPS = 64 / L; // lanes a part, parts at once
    __shared__ __attribute__((aligned(16))) v4f sums[4][64];
    __shared__ float by[4][SHARED / 4 + 1];
    char *ws = const_cast<char *>(ws_);
    const int count = *reinterpret_cast<const int *>(ws) * S::GT, lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    for (int i = blockIdx.x; i < count; i += BLOCKS) {
      const Record rec = reinterpret_cast<const Record *>(ws + 32)[i / S::GT];
      const int row = rec.token * S::GT + i % S::GT, gt = rec.hh % S::GTILES, h = rec.hh / S::GTILES, head = gt * 16 + i % S::GT;
      if (head >= S::G) continue;
      float m = -__builtin_inff(), l = 0;
      for (int k = lane; k < rec.parts; k += 64) m = __builtin_fmaxf(m, stats(ws, rec.part + k)[2 * row]);
#pragma unroll
      for (int k = 1; k < 64; k *= 2) m = __builtin_fmaxf(m, __shfl_xor(m, k));
      for (int k = lane; k < rec.parts; k += 64) {
        const float *st = stats(ws, rec.part + k) + 2 * row;
        const float f = st[0] == m ? 1.0f : __builtin_amdgcn_exp2f(st[0] - m);
        l += st[1] * f;
        if (k % 4 == wave) by[wave][k / 4] = f;
      }
#pragma unroll
      for (int k = 1; k < 64; k *= 2) l += __shfl_xor(l, k);
      v4f o = {0, 0, 0, 0};
      if (lane < GROUPS * L) {
#pragma unroll 4
        for (int k = lane / L; 4 * k + wave < rec.parts; k += GROUPS)
          o += *reinterpret_cast<const v4f *>(part(ws, rec.part + 4 * k + wave) + row * S::D + lane % L * 4) * by[wave][k];
      }
      sums[wave][lane] = o;
      __syncthreads();
      if (wave == 0 && lane < L) {
        o = v4f{0, 0, 0, 0};
#pragma unroll
        for (int v = 0; v < 4; ++v)
#pragma unroll
          for (int k = 0; k < GROUPS; ++k) o += sums[v][k * L + lane];
        uint16_t e[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float v = l == 0 ? 0.0f : o[k] / l;
          e[k] = S::EL == EL_BF16 ? f32_to_bf16_rne(v) : __builtin_bit_cast(uint16_t, (_Float16)v);
        }
        *reinterpret_cast<u32x2_any *>(a.out + (rec.t * (int64_t)S::HQ + h * S::G + head) * S::D + lane * 4) =
            u32x2{(uint32_t)e[0] | (uint32_t)e[1] << 16, (uint32_t)e[2] | (uint32_t)e[3] << 16};
      }
      __syncthreads();
    }
  }
};

// ---------------------------------------------------------------- rows of prompts
// A workgroup has TOKENS rows of the batch and one kv head (of a group of more
// than 16 query heads, 16 of them): 128 matrix-core rows, 32 a wave.  Its rows'
// sequences are taken one after another; of each, tiles of 64 tokens are
// decoded to 16 bits into LDS, keys by token and values by channel, for all
// four waves, while the tile before is worked on.
// As above the products are transposed, here 32x32x16: a lane's 16 scores of a K
// tile of 32 tokens are tokens 16 (i / 8) + 8 (lane / 32) + i % 8 of one row, eight at a
// time the B operand of the second product as they lie, if row r of the K tile
// is the token with bits 2 and 3 of r exchanged.
// The running maximum is only raised, and what is summed only scaled, when a
// row's new scores exceed it by 2^6: numbers up to that are as good as up to 1.
//
// A tile's two halves of 32 tokens go through in turn, so that a half's
// exponentials have products of the other beside them, and each product's
// operand is read one stage ahead: scores of the first half; those of the
// second beside the first's exponentials; the first's values beside the
// second's exponentials; the second's values.  10495 rows of four prompts (276
// Gflop) take 345 to 368 us a call by box, 750 to 800 Tflop/s; beside 342 both
// halves at once took 355, reads ordered by the compiler 412.  A large library product of bf16 reaches 1215 on this card.
// A SIMD's two waves have some 250 vector instructions for each 32 products,
// which issue half the time, the matrix core 35 to 40 %; a third of a wave's
// time goes to waits and barriers.
template <typename S> struct PagedPrompt {
  static constexpr int TOKENS = 128 / S::GT, HEADS = S::HK * S::GTILES, KP = S::D + 8, VP = 64 + 8;
  static constexpr int CHUNKS = 4 * S::D, N = (CHUNKS + 255) / 256; // 16-byte pieces of a tile's keys, a thread
  static constexpr int QF = S::D / 16, OT = S::D / 32;
  union Lds {
    struct {
      __attribute__((aligned(16))) uint16_t k[2][64 * KP], v[2][S::D * VP];
    };
    PagedJoin<S, 4> join;
  };

  __device__ static __forceinline__ v16f mfma(v4i a, v4i b, v16f c) {
    if constexpr (S::EL == EL_BF16) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
  }
  // a tile's four groups of 16 tokens, group lane % 4 in a lane
  struct Groups {
    int block;      // of the cache, -1 for none
    uint32_t ks, vs; // scale bytes
  };
  // What the tile's values are scaled to: o is in units of 2^(ref - 127), of
  // about the largest block of the tile, but no less than 2^-60 of the largest
  // so far (`peak`; o would pass f32's range).  bf16 has the range for codes
  // 2^100 below it, f16 for 2^8 (DOWN).  Blocks further apart cannot share a
  // product, and one above kTopScale not the sums (`apart`, a peak past all bytes),
  // since a row may see the small ones alone: what rows that have met such a tile
  // come to is dropped, and they go by paged_part.
  struct Mode {
    uint32_t ref, peak;
    __device__ __forceinline__ bool apart() const { return peak > 255; }
  };
  static constexpr uint32_t DOWN = S::EL == EL_BF16 ? 100 : 8;

  const PagedArgs &a;
  Lds &lds;
  const int seq, h, lo, hi;
  u32x4 kx[N], vx[N];

  __device__ __forceinline__ int block(int tile) const {
    const int i = (64 * tile + 16 * (int)(threadIdx.x % 4)) / S::BLOCK;
    const int b = i < S::PER ? a.table[(int64_t)seq * S::PER + i] : -1;
    return b >= 0 && b < S::NBLK ? b : -1;
  }
  __device__ __forceinline__ Groups groups(int b) const {
    const int64_t at = (int64_t)(b < 0 ? 0 : b) * S::HK + h;
    return Groups{b, a.ks[at], a.vs[at]};
  }
  __device__ __forceinline__ void load(const Groups &gr, int tile) {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const int c = (int)threadIdx.x + 256 * e;
      if (CHUNKS % 256 != 0 && c >= CHUNKS) break;
      const int tok = c / (S::D / 16), part = c % (S::D / 16), d = c / 4, g = c % 4;
      if constexpr (S::BLOCK >= 64) { // (one block: its place is a scalar)
        const int b = __builtin_amdgcn_readfirstlane(gr.block), off = 64 * tile % S::BLOCK;
        const int64_t at = ((int64_t)(b < 0 ? 0 : b) * S::HK + h) * (S::BLOCK * S::D);
        kx[e] = *reinterpret_cast<const u32x4_any *>(a.k + at + off * S::D + (tok * S::D + 16 * part));
        vx[e] = *reinterpret_cast<const u32x4_any *>(a.v + at + off + (d * S::BLOCK + 16 * g));
      } else {
        const int bk = __shfl(gr.block, tok / 16), bv = __shfl(gr.block, g); // (lane i of the first four holds group i)
        const uint8_t *kp = a.k + ((int64_t)(bk < 0 ? 0 : bk) * S::HK + h) * (S::BLOCK * S::D), *vp = a.v + ((int64_t)(bv < 0 ? 0 : bv) * S::HK + h) * (S::BLOCK * S::D);
        kx[e] = *reinterpret_cast<const u32x4_any *>(kp + (64 * tile + tok) % S::BLOCK * S::D + 16 * part);
        vx[e] = *reinterpret_cast<const u32x4_any *>(vp + d * S::BLOCK + (64 * tile + 16 * g) % S::BLOCK);
      }
    }
  }
  __device__ __forceinline__ Mode mode(const Groups &gr, int tile, const Mode &was) const {
    // the tile's largest scale byte, and 255 less the smallest (a tile has one of
    // blocks of 64 tokens and more)
    typedef uint16_t u2 __attribute__((ext_vector_type(2)));
    const bool read = gr.block >= 0 && gr.vs != 255 && (S::BLOCK >= 64 || some_seen<S>(64 * tile + 16 * (int)(threadIdx.x % 4), lo, hi));
    uint32_t both = read ? gr.vs << 16 | (255 - gr.vs) : 0u;
    if constexpr (S::BLOCK < 64) {
      auto most = [](uint32_t a, uint32_t b) { return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u2, a), __builtin_bit_cast(u2, b))); };
      both = most(both, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)both, 0xB1, 0xF, 0xF, true));
      both = most(both, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)both, 0x4E, 0xF, 0xF, true));
    }
    both = (uint32_t)__builtin_amdgcn_readfirstlane((int)both);
    const uint32_t big = both >> 16, up = both & 0xFFFF, peak = max_u32(was.peak, big);
    uint32_t now = big > was.ref || (big && big + 4 < was.ref) ? big : was.ref; // (a little lower is near enough)
    now = now + 60 < peak ? peak - 60 : now;
    return Mode{now, now > kTopScale || now + up > 255 + DOWN ? 512u : peak};
  }
  __device__ __forceinline__ void stage(const Groups &gr, const Mode &mo, int tile, int buf) {
    const bool whole = 64 * tile + 63 <= hi && (S::WINDOW == 0 || 64 * tile > lo - S::WINDOW) && __all(gr.block >= 0);
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const int c = (int)threadIdx.x + 256 * e;
      if (CHUNKS % 256 != 0 && c >= CHUNKS) break;
      const int tok = c / (S::D / 16), part = c % (S::D / 16), d = c / 4, g = c % 4;
      v4i *kd = reinterpret_cast<v4i *>(&lds.k[buf][tok * KP + 16 * part]), *vd = reinterpret_cast<v4i *>(&lds.v[buf][d * VP + 16 * g]);
      kd[0] = attn_decode8<S::EL, S::FMT>(kx[e].x, kx[e].y, 1.0f), kd[1] = attn_decode8<S::EL, S::FMT>(kx[e].z, kx[e].w, 1.0f);
      const uint32_t vs = S::BLOCK >= 64 ? (uint32_t)__builtin_amdgcn_readfirstlane((int)gr.vs) : (uint32_t)__shfl((int)gr.vs, g);
      bool used = true;
      if (!whole) {
        // (what no row sees, and where there is no block, zeros)
        const int at = 64 * tile + 16 * g, n = __shfl(gr.block, g) >= 0 ? hi + 1 - at : 0, gone = lo - S::WINDOW + 1 - at;
        used = n > 0 && (S::WINDOW == 0 || gone < 16);
#pragma unroll
        for (int w = 0; w < 4; ++w) vx[e][w] &= kept_codes<S>(w, n, gone);
      }
      const uint32_t down = mo.ref - vs < DOWN ? mo.ref - vs : DOWN;
      const float by = !used || vs == 255 ? 1.0f : u2f((127 - down) << 23);
      vd[0] = attn_decode8<S::EL, S::FMT>(vx[e].x, vx[e].y, by), vd[1] = attn_decode8<S::EL, S::FMT>(vx[e].z, vx[e].w, by);
    }
  }

  v16f o[OT];
  float m, sum;
  uint32_t ref;
  v4i q[QF];

  __device__ __forceinline__ void times(float by) {
#pragma unroll
    for (int i = 0; i < OT; ++i) o[i] *= by;
  }
  // tile from LDS; pos: the lane's row's position (-1: no row), first and last:
  // the wave's rows'
  __device__ __forceinline__ void step(const Groups &gr, const Mode &mo, int tile, int buf, int pos, int first, int last) {
    const int lane = threadIdx.x % 64, r = lane % 32, half = lane / 32, key = (r & 0x13) | (r & 4) << 1 | (r & 8) >> 1;
    if (mo.ref != ref) {
      const int by = (int)ref - (int)mo.ref; // -143 .. 60
      // (a power of two that far below 1 is none of f32)
      if (by < -120) times(0x1p-40f);
      times(u2f((uint32_t)(127 + (by < -120 ? by + 40 : by)) << 23));
      ref = mo.ref;
    }
    constexpr int GS = S::BLOCK >= 64 ? 1 : 4; // groups of tokens whose blocks may differ
    float f[GS];
    uint32_t there = 0;
    bool odd = false; // (a factor that is zero or NaN, with which -inf is no zero)
#pragma unroll
    for (int g = 0; g < GS; ++g) {
      // (a block of values that are NaN makes NaN of the rows that see it: by their scores)
      const uint32_t ks = (uint32_t)__builtin_amdgcn_readlane((int)gr.ks, g), vs = (uint32_t)__builtin_amdgcn_readlane((int)gr.vs, g);
      f[g] = __builtin_fabsf(a.scale) * mx_scale(vs == 255 ? 255 : ks);
      odd |= !(f[g] > 0);
      there |= (uint32_t)(__builtin_amdgcn_readlane(gr.block, g) >= 0) << g;
    }
    const bool whole = there == (1u << GS) - 1 && 64 * tile + 63 <= first && (S::WINDOW == 0 || 64 * tile > last - S::WINDOW);
    // (tokens by their distance from the lane's first: compares with constants)
    const int to = pos - (64 * tile + 8 * half), from = to - S::WINDOW;
    v16f s[2] = {};
    auto hide = [&](int u, float with) {
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const int end = there >> ((2 * u + g) * GS / 4) & 1 ? to : -1;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int at = 32 * u + 16 * g + i;
          s[u][8 * g + i] = at <= end && (S::WINDOW == 0 || at > from) ? s[u][8 * g + i] : with;
        }
      }
    };
    // scores of half u: hidden, and the maximum raised where it has to be
    auto scored = [&](int u) {
      if (!whole) hide(u, -__builtin_inff());
      float top = -__builtin_inff();
#pragma unroll
      for (int g = 0; g < (GS + 1) / 2; ++g) {
        constexpr int W = GS == 1 ? 16 : 8;
        float t = -__builtin_inff();
#pragma unroll
        for (int i = W * g; i < W * (g + 1); i += 2) t = __builtin_fmaxf(__builtin_fmaxf(t, s[u][i]), s[u][i + 1]);
        top = __builtin_fmaxf(top, t * f[GS == 1 ? 0 : 2 * u + g]); // (f is not negative)
      }
      top = with_lane<32>(top, max2);
      if (__any(top > m + 6.0f)) {
        const float now = __builtin_fmaxf(m, top), was = m == now ? 1.0f : __builtin_amdgcn_exp2f(m - now);
        m = now;
        sum *= was;
        times(was);
        if (u == 1) s[0] *= was; // (probabilities by now)
      }
    };
    float part[4] = {0, 0, 0, 0};
    // probabilities of half u, a share of them; then what the values are multiplied by
    float mu = 0;
    auto exps = [&](int u, int c) {
#pragma unroll
      for (int i = 16 * c / QF; i < 16 * (c + 1) / QF; ++i) s[u][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][i], f[GS == 1 ? 0 : 2 * u + i / 8], -mu));
    };
    auto rounded = [&](int u, v4i (&pf)[2]) {
      if (odd && !whole) hide(u, 0.0f);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float p[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = s[u][8 * k + i];
        pf[k] = attn_round8<S::EL>(p);
        // (the sum of the rounded: half the additions, and its rounding and that
        // of what the values are multiplied by go together)
#pragma unroll
        for (int w = 0; w < 4; ++w) part[w] = attn_sum2<S::EL>(pf[k][w], part[w]);
      }
    };
    auto keys = [&](int u, int c) { return *reinterpret_cast<const v4i *>(&lds.k[buf][(32 * u + key) * KP + 16 * c + 8 * half]); };
    auto values = [&](int u, int c) { return *reinterpret_cast<const v4i *>(&lds.v[buf][(32 * (c % OT) + r) * VP + 32 * u + 16 * (c / OT) + 8 * half]); };
    auto limit = [] { __builtin_amdgcn_sched_barrier(0); };
    v4i w[QF], pf[2];
#pragma unroll
    for (int c = 0; c < QF; ++c) w[c] = keys(0, c);
    limit();
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int c = 0; c < QF; ++c) {
      s[0] = mfma(w[c], q[c], s[0]);
      w[c] = keys(1, c);
      limit();
    }
    __builtin_amdgcn_s_setprio(0);
    scored(0);
    mu = (m == -__builtin_inff() ? 0.0f : m) - S::LIFT; // (a row that has seen nothing)
#pragma unroll
    for (int c = 0; c < QF; ++c) {
      s[1] = mfma(w[c], q[c], s[1]);
      w[c] = values(0, c);
      exps(0, c);
      limit();
    }
    scored(1);
    mu = (m == -__builtin_inff() ? 0.0f : m) - S::LIFT;
    rounded(0, pf);
#pragma unroll
    for (int c = 0; c < QF; ++c) {
      o[c % OT] = mfma(w[c], pf[c / OT], o[c % OT]);
      w[c] = values(1, c);
      exps(1, c);
      limit();
    }
    rounded(1, pf);
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int c = 0; c < QF; ++c) o[c % OT] = mfma(w[c], pf[c / OT], o[c % OT]);
    __builtin_amdgcn_s_setprio(0);
    sum += (part[0] + part[1]) + (part[2] + part[3]);
  }

  // The tiles of a piece of the rows; whether it has all of them.
  template <bool PARTS> __device__ __forceinline__ bool range(int piece, int pieces, int &begin, int &end) const {
    begin = PagedUnits<S>::first(lo), end = hi / 64 + 1;
    if constexpr (!PARTS) return true;
    int cut = (end - begin + pieces - 1) / pieces;
    cut = cut < CUT ? CUT : cut;
    const bool alone = end - begin <= cut;
    begin += piece * cut;
    end = begin + cut < end ? begin + cut : end;
    return alone;
  }
  // Rows t .. t + n - 1, of a sequence's positions lo .. hi; t0: the tile's first
  // row.  PARTS: piece `piece` of `pieces` of their tiles, at least CUT tiles
  // long, to part and stats.
  // (false: a tile's blocks are too far apart, and split() has these rows to do)
  template <bool PARTS> __device__ __forceinline__ bool run(int64_t t0, int64_t t, int n, int gt, int piece, int pieces, float *part, float *stats) {
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, r = lane % 32, half = lane / 32;
    const int row = 32 * wave + r, tok = row / S::GT, head = gt * 16 + row % S::GT, skip = (int)(t - t0);
    const bool ok = tok >= skip && tok < skip + n && head < S::G && row < TOKENS * S::GT;
    const int pos = ok ? lo + tok - skip : -1;
    int begin, end;
    // one piece has all of them: the result, and the mark DONE for a sum
    const bool alone = range<PARTS>(piece, pieces, begin, end);
    if (PARTS && begin >= end) {
      if (ok && half == 0) stats[2 * row] = -__builtin_inff(), stats[2 * row + 1] = 0;
      return true;
    }
    // the wave's rows' positions
    const int a0 = 32 * wave / S::GT, a1 = (32 * wave + 31) / S::GT;
    const int first = lo + (a0 > skip ? a0 - skip : 0), last = a1 < skip ? -1 : lo + (a1 - skip < n ? a1 - skip : n - 1);
    const int seen = a0 >= skip + n ? -1 : last; // (-1: the wave has no rows)
    const uint16_t *qp = a.q + ((t0 + (ok ? tok : skip)) * S::HQ + h * S::G + (ok ? head : 0)) * S::D + 8 * half;
#pragma unroll
    for (int c = 0; c < QF; ++c) {
      const u32x4 w = *reinterpret_cast<const u32x4_any *>(qp + 16 * c);
      // (a negative scale's sign goes to the queries: a maximum is one before and after)
      const int turn = a.scale < 0 ? (int)0x80008000u : 0;
      q[c] = ok ? v4i{(int)w.x ^ turn, (int)w.y ^ turn, (int)w.z ^ turn, (int)w.w ^ turn} : v4i{0, 0, 0, 0};
    }
#pragma unroll
    for (int i = 0; i < OT; ++i) o[i] = v16f{};
    m = -__builtin_inff(), sum = 0, ref = 0;
    Groups gr = groups(block(begin));
    load(gr, begin);
    Mode mo = mode(gr, begin, Mode{0, 0});
    int next = block(begin + 1);
    stage(gr, mo, begin, begin & 1);
    __syncthreads();
    for (int i = begin; i < end; ++i) {
      Groups gn = gr;
      if (i + 1 < end) {
        gn = groups(next);
        load(gn, i + 1);
        next = block(i + 2);
      }
      __builtin_amdgcn_sched_barrier(0);
      if (64 * i <= seen && (S::WINDOW == 0 || 64 * i + 63 > first - S::WINDOW)) step(gr, mo, i, i & 1, pos, first, last);
      if (i + 1 < end) {
        mo = mode(gn, i + 1, mo);
        stage(gn, mo, i + 1, (i + 1) & 1);
        gr = gn;
      }
      __syncthreads();
    }
    if (mo.apart()) return false;
    times(mx_scale(ref));
    sum = with_lane<32>(sum, [](float x, float y) { return x + y; });
    if (!ok) return true;
    if (PARTS && alone && half == 0) stats[2 * row + 1] = DONE;
    if (PARTS && !alone) {
      if (half == 0) stats[2 * row] = m, stats[2 * row + 1] = sum;
      float *dst = part + row * S::D + 4 * half;
#pragma unroll
      for (int dt = 0; dt < OT; ++dt)
#pragma unroll
        for (int k = 0; k < 4; ++k)
          *reinterpret_cast<v4f *>(dst + 32 * dt + 8 * k) = v4f{o[dt][4 * k], o[dt][4 * k + 1], o[dt][4 * k + 2], o[dt][4 * k + 3]};
      return true;
    }
    const float by = sum == 0 ? 0.0f : 1.0f / sum;
    uint16_t *dst = a.out + ((t0 + tok) * (int64_t)S::HQ + h * S::G + head) * S::D + 4 * half;
#pragma unroll
    for (int dt = 0; dt < OT; ++dt)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        uint16_t e[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float v = o[dt][4 * k + j] * by;
          e[j] = S::EL == EL_BF16 ? f32_to_bf16_rne(v) : __builtin_bit_cast(uint16_t, (_Float16)v);
        }
        *reinterpret_cast<u32x2_any *>(dst + 32 * dt + 8 * k) = u32x2{(uint32_t)e[0] | (uint32_t)e[1] << 16, (uint32_t)e[2] | (uint32_t)e[3] << 16};
      }
    return true;
  }
  // The same rows and piece, N tokens at a time, by paged_part, which takes
  // blocks any distance apart.
  template <bool PARTS> __device__ __forceinline__ void split(int64_t t0, int64_t t, int n, int gt, int piece, int pieces, float *part, float *stats) {
    int begin, end;
    const bool alone = range<PARTS>(piece, pieces, begin, end);
    for (int i = 0; i < n; i += S::N) {
      const int k = n - i < S::N ? n - i : S::N, row = (int)(t - t0 + i) * S::GT, b = PagedUnits<S>::first(lo + i), e = (lo + i + k - 1) / 64 + 1;
      paged_part<S, 4>(a, lds.join, t + i, k, seq, lo + i, h * S::GTILES + gt, b < begin ? begin : b, e < end ? e : end,
                       alone ? nullptr : part + row * S::D, alone ? nullptr : stats + 2 * row);
      if (PARTS && alone && (int)threadIdx.x < k * S::GT) stats[2 * (row + threadIdx.x) + 1] = DONE;
    }
  }

  __device__ static __forceinline__ int64_t tiles(int64_t T) { return (T + TOKENS - 1) / TOKENS; }
  // The units of a tile and a head in `pieces` pieces each, first all units'
  // first ones: few units leave most of the chip idle, and those of a prompt's
  // last rows take longest.  us of a call: 512 rows behind 7000 positions whole
  // 226, in eight pieces 107, in four, which all run at once, 92; two times 900
  // rows behind 4000 and 7000 whole 336, in two pieces 300; a prompt of 2048 whole
  // 73.5, in two 70; 1001 rows over a window of 4096 in pieces of at least 4, 8 and
  // 12 tiles 63, 61, 64, of 16 53.
  // ws: PagedFew's flags, the pieces' statistics (two of each of 128 rows), then
  // their rows.
  static constexpr int PIECES = 1024, CUT = 16;
  static constexpr float DONE = -1; // (no sum is negative)
  __device__ static __forceinline__ int pieces(int64_t T) {
    // (four and more that all run at once, or twice as many workgroups as do)
    const int64_t units = tiles(T) * HEADS, once = PIECES / 2 / units, n = once >= 4 ? once : PIECES / units;
    return n > 16 ? 16 : n < 1 ? 1 : (int)n;
  }
  __device__ static __forceinline__ float *stats_of(char *ws, int64_t piece) { return reinterpret_cast<float *>(ws) + PagedFew<S>::TILES + piece * 256; }
  __device__ static __forceinline__ float *part_of(char *ws, int64_t piece) { return stats_of(ws, PIECES) + piece * (128 * S::D); }

  // grid: tiles(T) * HEADS, PARTS: PIECES; the last rows, which see most, first
  template <bool PARTS> __device__ static __forceinline__ void rows(const PagedArgs &a, int64_t T, char *ws) {
    __shared__ Lds lds;
    const int cuts = PARTS ? pieces(T) : 1, units = (int)tiles(T) * HEADS, piece = PARTS ? (int)blockIdx.x / units : 0;
    if (piece >= cuts) return;
    const int64_t t0 = (tiles(T) - 1 - (blockIdx.x - piece * units) / HEADS) * TOKENS;
    const int hh = (int)(blockIdx.x - piece * units) % HEADS, h = hh / S::GTILES, gt = hh % S::GTILES, lane = threadIdx.x % 64;
    const int tokens = (int)(T - t0 < TOKENS ? T - t0 : TOKENS);
    auto uniform = [](uint64_t v) {
      return (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)v);
    };
    // a row and those that follow it
    auto follow = [&](int at, int s, int p) {
      const int64_t t = t0 + at;
      int n = 0;
#pragma unroll
      for (int k = 0; k < TOKENS; k += 64) {
        const int i = k + lane;
        const uint64_t other = __ballot(!(i < tokens - at && p + i < S::FAR && a.seq[t + i] == s && a.pos[t + i] == p + i));
        if (n == k) n += other ? __builtin_ctzll(other) : 64;
      }
      return n;
    };
    auto part = [&]() -> float * { return PARTS ? part_of(ws, blockIdx.x) : nullptr; };
    auto stats = [&]() -> float * { return PARTS ? stats_of(ws, blockIdx.x) : nullptr; };
    int few = 0;
    // rows that run() has left, done behind all others: beside its loop they would
    // take registers (f16 heads of 256 channels 12 % slower)
    __shared__ uint64_t apart[2];
    if (threadIdx.x < 2) apart[threadIdx.x] = 0;
    for (int at = 0; at < tokens;) {
      const int64_t t = t0 + at;
      const int s = a.seq[t], p = a.pos[t];
      if (!S::inside(s, p)) {
        ++at;
        continue;
      }
      const int n = follow(at, s, p);
      if (n <= S::FEW && S::few(a.seq, a.pos, t, T, s, p)) { // PagedFew's
        if (PARTS && piece == 0)
          for (int i = threadIdx.x; i < n * S::GT; i += 256) stats()[2 * (at * S::GT + i) + 1] = DONE;
        at += n, few = 1;
        continue;
      }
      const bool done = PagedPrompt{a, lds, s, h, p, p + n - 1}.template run<PARTS>(t0, t, n, gt, piece, cuts, part(), stats());
      if (!done && (int)threadIdx.x == at / 64) apart[at / 64] |= 1ull << at % 64;
      at += n;
    }
    auto end = [&] {
      if (piece == 0 && hh == 0 && threadIdx.x == 0 && t0 / TOKENS < PagedFew<S>::TILES) reinterpret_cast<int *>(ws)[t0 / TOKENS] = few;
    };
    __syncthreads();
    if (__builtin_expect(uniform(apart[0] | apart[1]) == 0, 1)) return end();
    for (int w = 0; w < 2; ++w)
      for (uint64_t left = uniform(apart[w]); left; left &= left - 1) {
        const int at = 64 * w + __builtin_ctzll(left), s = a.seq[t0 + at], p = a.pos[t0 + at], n = follow(at, s, p);
        PagedPrompt{a, lds, s, h, p, p + n - 1}.template split<PARTS>(t0, t0 + at, n, gt, piece, cuts, part(), stats());
      }
    end();
  }

  // The second launch: PagedFew's workgroups, and PARTS behind them PIECES / 2 *
  // 4 that add the rows' pieces in order, eight lanes a row, a quarter of a
  // unit's rows each.
  template <bool PARTS> __device__ static __forceinline__ void finish(const PagedArgs &a, int64_t T, const char *ws_) {
    const int block = (int)blockIdx.x - PagedFew<S>::BLOCKS;
    if (block < 0) return PagedFew<S>::rows(a, T, reinterpret_cast<const int *>(ws_), (int)blockIdx.x);
    if constexpr (PARTS) join(a, T, ws_, block);
  }
  __device__ static __forceinline__ void join(const PagedArgs &a, int64_t T, const char *ws_, int block) {
    char *ws = const_cast<char *>(ws_);
    const int cuts = pieces(T), unit = block / 4, hh = unit % HEADS, h = hh / S::GTILES, gt = hh % S::GTILES;
    const int64_t t0 = (tiles(T) - 1 - unit / HEADS) * TOKENS, units = tiles(T) * HEADS;
    if (t0 < 0) return;
    const int row = block % 4 * 32 + threadIdx.x / 8, tok = row / S::GT, head = gt * 16 + row % S::GT;
    if (row >= TOKENS * S::GT || t0 + tok >= T || head >= S::G || !S::inside(a.seq[t0 + tok], a.pos[t0 + tok])) return;
    auto piece = [&](int i) { return i * units + unit; };
    if (stats_of(ws, piece(0))[2 * row + 1] == DONE) return;
    float m = -__builtin_inff(), l = 0, by[16];
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (i < cuts) m = __builtin_fmaxf(m, by[i] = stats_of(ws, piece(i))[2 * row]);
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (i < cuts) {
        const float sum = stats_of(ws, piece(i))[2 * row + 1];
        by[i] = sum == 0 ? 0.0f : by[i] == m ? 1.0f : __builtin_amdgcn_exp2f(by[i] - m);
        l += sum * by[i];
      }
    const float over = l == 0 ? 0.0f : 1.0f / l;
    for (int d = threadIdx.x % 8 * 4; d < S::D; d += 32) {
      v4f o = {0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < 16; ++i) // (what saw nothing may not have been written)
        if (i < cuts && by[i] != 0) o += *reinterpret_cast<const v4f *>(part_of(ws, piece(i)) + row * S::D + d) * by[i];
      uint16_t e[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) e[k] = S::EL == EL_BF16 ? f32_to_bf16_rne(o[k] * over) : __builtin_bit_cast(uint16_t, (_Float16)(o[k] * over));
      *reinterpret_cast<u32x2_any *>(a.out + ((t0 + tok) * (int64_t)S::HQ + h * S::G + head) * S::D + d) =
          u32x2{(uint32_t)e[0] | (uint32_t)e[1] << 16, (uint32_t)e[2] | (uint32_t)e[3] << 16};
    }
  }
};

} // namespace hf
