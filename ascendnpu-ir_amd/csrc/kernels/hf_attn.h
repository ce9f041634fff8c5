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

// ---------------------------------------------------------------- rows of a few tokens
// A unit is the rows of one group of tokens and one kv head (of a group of more
// than 16 query heads, 16 of them); its tiles are those that hold a visible
// position.
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

// Units of different lengths: one is cut into pieces of at most `run` tiles, a
// workgroup a piece, the longest first; units of several pieces leave parts,
// which join() adds in order.  run makes as many pieces as fill the chip with
// the units that stay whole: PIECES less the units, LEAST to SHARED of them.  us of
// a call, with 512, 768 (taken), 1536 at most: one row over 32768 positions 19.5,
// 19.6, 23; over 131072 49, 53, 58; 48 rows over up to 8100 90, 80, 87 (5.1 TB/s;
// a workgroup a unit 114, as long as the longest takes).
// Up to MOST rows: every workgroup adds up the units' tiles itself, which takes
// it some 2 us.
// ws: the number of records, one a token of a unit in parts; then for each part
// the rows' maximum and sum, and the rows.
template <typename S, int WV> struct PagedSplit {
  using U = PagedUnits<S>;
  static constexpr int MOST = 1024, PIECES = 1024, LEAST = 256, SHARED = 768, THREADS = 64 * WV, PER = (MOST + THREADS - 1) / THREADS;
  static_assert((S::FAR / 64 + 1) * MOST < (int64_t(1) << 31) && (int64_t)MOST * U::HEADS < (int64_t(1) << 30));
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
    const int run = ((int)((all + want - 1) / want) + WV - 1) / WV * WV; // (every wave as many)
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

} // namespace hf
