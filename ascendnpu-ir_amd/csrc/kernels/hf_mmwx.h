// bf16 rows times a block-scaled weight, few rows (hfusion.linear_mx):
//   C[m, n] = sum_k A[m, k] w[n, k] 2^E[n, k / 32]
// A [M, K] bf16, w [N, K] 8-bit codes or [N, K/2] bytes of two e2m1 codes,
// one e8m0 byte per 32 k of a row.  Such a call reads every weight once and
// multiplies little: what counts is that the whole chip has its share of the
// weights in flight at once.
//
// A workgroup owns 16 MT rows and 16 NT columns of C and its NW waves split K,
// so no sum crosses workgroups; the waves' partial sums meet in LDS, added in
// wave order.  The order of k within a matrix-core step is free as long as
// both operands agree on it: a lane takes KPL consecutive k of its row and of
// its column (one or two whole scale blocks, 32 bytes of codes) and feeds
// them eight at a time.  The codes become bf16 pairs, scale included, in one
// instruction; code times scale fits bf16's significand, so f32 sums are the
// only rounding before the epilogue's.
#pragma once
#include "hf_mmsk.h"
#include "hf_mx.h"

namespace hf {

// eight codes of w (words w0, w1 of 8-bit codes; w0 of e2m1) times the scale
template <int FMT> __device__ __forceinline__ v4i wx_decode8(uint32_t w0, uint32_t w1, float scale) {
  typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
  auto bits = [](bf2 v) { return __builtin_bit_cast(int, v); };
  if constexpr (FMT == MX_E2M1)
    return v4i{bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w0, scale, 0)), bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w0, scale, 1)),
               bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w0, scale, 2)), bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w0, scale, 3))};
  else if constexpr (FMT == MX_E4M3)
    return v4i{bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, scale, false)), bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, scale, true)),
               bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, scale, false)), bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, scale, true))};
  else
    return v4i{bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(w0, scale, false)), bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(w0, scale, true)),
               bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(w1, scale, false)), bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(w1, scale, true))};
}

template <int FMT, typename Epi, int MT, int NT, int NW, int64_t K, typename Args>
__device__ __forceinline__ void linear_wx(const uint16_t *__restrict__ A, const uint8_t *__restrict__ W, const uint8_t *__restrict__ S,
                                          typename Epi::out_t *__restrict__ out, int64_t M, int64_t N, const Args &P) {
  static_assert(K % 32 == 0);
  constexpr int BLK = FMT == MX_E2M1 ? 2 : 1;    // scale blocks a lane takes of a step
  constexpr int KPL = 32 * BLK, KS = 4 * KPL;    // k a lane, a step of the wave
  constexpr int64_t WP = FMT == MX_E2M1 ? K / 2 : K, SP = K / 32;
  constexpr int ns = (int)((K + KS - 1) / KS);
  constexpr bool RAGGED = K % KS != 0;
  __shared__ v4f red[NW * MT * NT * 64];
  const int64_t tn = (N + 16 * NT - 1) / (16 * NT);
  const int64_t m0 = (int64_t)(blockIdx.x / tn) * (16 * MT), n0 = (int64_t)(blockIdx.x % tn) * (16 * NT);
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / 64), lane = threadIdx.x % 64;
  const int q = lane / 16, j = lane % 16;
  // rows and columns past the end re-read the last one; their results are not stored
  const uint16_t *ap[MT];
  const uint8_t *wp[NT], *sp[NT];
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    const int64_t m = m0 + 16 * t + j;
    ap[t] = A + (m < M ? m : M - 1) * K + q * KPL;
  }
#pragma unroll
  for (int u = 0; u < NT; ++u) {
    const int64_t n = n0 + 16 * u + j, nn = n < N ? n : N - 1;
    wp[u] = W + nn * WP + q * 32;
    sp[u] = S + nn * SP + q * BLK;
  }
  struct Step {
    u32x4 a[MT][KPL / 8], w[NT][2];
    uint32_t s[NT][BLK];
  };
  // the operands of step i; blocks past K become zeros
  auto load = [&](int i, Step &st) {
    const bool tail = RAGGED && i == ns - 1;
#pragma unroll
    for (int b = 0; b < BLK; ++b) {
      const bool in = !tail || i * KS + q * KPL + 32 * b < K;
      if (in) {
#pragma unroll
        for (int u = 0; u < NT; ++u) {
          st.s[u][b] = sp[u][i * (4 * BLK) + b];
          if constexpr (BLK == 2) {
            st.w[u][b] = *reinterpret_cast<const u32x4 *>(wp[u] + i * 128 + 16 * b);
          } else {
            st.w[u][0] = *reinterpret_cast<const u32x4 *>(wp[u] + i * 128);
            st.w[u][1] = *reinterpret_cast<const u32x4 *>(wp[u] + i * 128 + 16);
          }
        }
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
          for (int c = 0; c < 4; ++c) st.a[t][4 * b + c] = *reinterpret_cast<const u32x4 *>(ap[t] + i * KS + 32 * b + 8 * c);
      } else {
#pragma unroll
        for (int u = 0; u < NT; ++u) {
          st.s[u][b] = 127;
          if constexpr (BLK == 2) st.w[u][b] = u32x4{0, 0, 0, 0};
          else st.w[u][0] = st.w[u][1] = u32x4{0, 0, 0, 0};
        }
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
          for (int c = 0; c < 4; ++c) st.a[t][4 * b + c] = u32x4{0, 0, 0, 0};
      }
    }
  };
  v4f acc[MT][NT];
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int u = 0; u < NT; ++u) acc[t][u] = v4f{0, 0, 0, 0};
  auto multiply = [&](const Step &st) {
#pragma unroll
    for (int c = 0; c < KPL / 8; ++c) {
      v4i b[NT];
#pragma unroll
      for (int u = 0; u < NT; ++u) {
        const float scale = u2f(st.s[u][c / 4] << 23);
        if constexpr (FMT == MX_E2M1) b[u] = wx_decode8<FMT>(st.w[u][c / 4][c % 4], 0, scale);
        else b[u] = wx_decode8<FMT>(st.w[u][c / 2][2 * (c % 2)], st.w[u][c / 2][2 * (c % 2) + 1], scale);
      }
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int u = 0; u < NT; ++u) acc[t][u] = Mfma16<MK_BF16>::run(__builtin_bit_cast(v4i, st.a[t][c]), b[u], acc[t][u]);
    }
  };
  Step cur, nxt;
  if (wave < ns) load(wave, cur);
#pragma unroll 1
  for (int i = wave; i < ns; i += NW) {
    if (i + NW < ns) load(i + NW, nxt);
    multiply(cur);
    cur = nxt;
  }
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int u = 0; u < NT; ++u) red[((wave * MT + t) * NT + u) * 64 + lane] = acc[t][u];
  __syncthreads();
  // one output element per thread and step, consecutive threads on
  // consecutive columns
  const float *rs = reinterpret_cast<const float *>(red);
  constexpr int TM = 16 * MT, TN = 16 * NT;
#pragma unroll 4
  for (int o = threadIdx.x; o < TM * TN; o += NW * 64) {
    const int r = o / TN, c = o % TN, rr = r % 16;
    const int64_t m = m0 + r, nn = n0 + c;
    if (m >= M || nn >= N) continue;
    const int at = ((r / 16 * NT + c / 16) * 64 + rr / 4 * 16 + c % 16) * 4 + rr % 4;
    float s = rs[at];
#pragma unroll
    for (int w = 1; w < NW; ++w) s += rs[w * MT * NT * 256 + at];
    out[m * N + nn] = Epi::apply(s, m, nn, Epi::row(m, P), Epi::col(nn, P), P);
  }
}

} // namespace hf
