// Layer norm over the last axis, and its gradient.
//
//   mu = mean(x), r = 1 / sqrt(mean((x - mu)^2) + eps), y = (x - mu) r gamma + beta
//   xh = (x - mu) r, g = dy gamma
//   dx = r (g - mean(g) - xh mean(g xh)),  dgamma = sum over rows dy xh,  dbeta = sum over rows dy
// All sums are f32, in an order that the sizes alone decide.  The variance
// is the sum of squared distances from the mean found first (both over
// values that stay in registers): a sum of squares less the squared mean
// loses what a row's offset takes from it.
// An 8-bit checkpoint of x (hf_mx.h's codes along the row) is written by the
// forward pass and read by the gradient in place of x.
//
// A row group of T threads owns a row, NCH chunks of eight consecutive
// elements a thread (chunk j at column (j T + thread) * 8, so a group's
// accesses are consecutive and four neighbouring lanes hold a block of 32).
#pragma once
#include "hf_mx.h"

namespace hf {

// Sum over a wave: 16 lanes by DPP, then the four rows of lanes in order.
__device__ __forceinline__ float wave_sum(float v) {
  auto dpp = [](float a, auto ctrl) {
    return u2f((uint32_t)__builtin_amdgcn_update_dpp(0, (int)f2u(a), decltype(ctrl)::value, 0xF, 0xF, true));
  };
  v += dpp(v, std::integral_constant<int, 0xB1>{});  // quad 1 0 3 2
  v += dpp(v, std::integral_constant<int, 0x4E>{});  // quad 2 3 0 1
  v += dpp(v, std::integral_constant<int, 0x141>{}); // mirrored half row
  v += dpp(v, std::integral_constant<int, 0x140>{}); // mirrored row
  auto lane = [&](int l) { return u2f((uint32_t)__builtin_amdgcn_readlane((int)f2u(v), l)); };
  return (lane(0) + lane(16)) + (lane(32) + lane(48));
}

// Sums of N values over the row group; slots: N * T / 64 floats of the group.
template <int T, int N> __device__ __forceinline__ void group_sum(float (&v)[N], float *slots) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = wave_sum(v[i]);
  if constexpr (T > 64) {
    constexpr int W = T / 64;
    const int wave = (threadIdx.x % T) / 64;
    if (threadIdx.x % 64 == 0)
#pragma unroll
      for (int i = 0; i < N; ++i) slots[i * W + wave] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float s = slots[i * W];
#pragma unroll
      for (int w = 1; w < W; ++w) s += slots[i * W + w];
      v[i] = s;
    }
  }
}

// valid elements of the chunk at column c
template <int64_t D> __device__ __forceinline__ int ln_count(int64_t c) {
  return (int)(D - c <= 0 ? 0 : D - c < 8 ? D - c : 8);
}
template <int EL, bool FULL> __device__ __forceinline__ Oct<EL> ln_load(const void *base, int64_t e, int n) {
  const char *p = (const char *)base + e * el_bytes<EL>;
  if (FULL || n == 8) return oct_load<EL>(p);
  return oct_load_part<EL>(p, n);
}

// AFF: 0 neither weight nor bias, 1 gamma, 2 gamma and beta (of type PEL).
// CK: format of the checkpoint, -1 for none.  RPB row groups a workgroup.
// mean and rstd may be null.
template <int EL, int PEL, int AFF, int CK, int T, int NCH, int RPB, int64_t D>
__device__ __forceinline__ void ln_forward(const void *__restrict__ x, const void *__restrict__ gamma, const void *__restrict__ beta,
                                           void *__restrict__ y, float *__restrict__ mean, float *__restrict__ rstd,
                                           void *__restrict__ codes, void *__restrict__ scales, int64_t R, float eps) {
  static_assert((int64_t)T * NCH * 8 >= D && (T == 64 || RPB == 1));
  constexpr bool FULL = (int64_t)T * NCH * 8 == D;
  constexpr int64_t NB = (D + 31) / 32;
  __shared__ float slots[2][T / 64];
  const int lt = threadIdx.x % T, group = threadIdx.x / T;
  Oct<PEL> gm[NCH], bt[NCH];
#pragma unroll
  for (int j = 0; j < NCH; ++j) {
    const int64_t c = ((int64_t)j * T + lt) * 8;
    if constexpr (AFF >= 1) gm[j] = ln_load<PEL, FULL>(gamma, c, ln_count<D>(c));
    if constexpr (AFF >= 2) bt[j] = ln_load<PEL, FULL>(beta, c, ln_count<D>(c));
  }
  for (int64_t row = (int64_t)blockIdx.x * RPB + group; row < R; row += (int64_t)gridDim.x * RPB) {
    Oct<EL> v[NCH];
    float s[1] = {0}, q[1] = {0};
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
      const int64_t c = ((int64_t)j * T + lt) * 8;
      v[j] = ln_load<EL, FULL>(x, row * D + c, ln_count<D>(c));
    }
#pragma unroll
    for (int j = 0; j < NCH; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) s[0] += oct_get<EL>(v[j], i);
    group_sum<T>(s, slots[0]);
    const float mu = s[0] / (float)D;
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
      const int n = FULL ? 8 : ln_count<D>(((int64_t)j * T + lt) * 8);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float d = oct_get<EL>(v[j], i) - mu;
        if (FULL || i < n) q[0] = __builtin_fmaf(d, d, q[0]);
      }
    }
    group_sum<T>(q, slots[1]);
    const float r = 1.0f / __builtin_sqrtf(q[0] / (float)D + eps);
    if (lt == 0) {
      if (mean) mean[row] = mu;
      if (rstd) rstd[row] = r;
    }
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
      const int64_t c = ((int64_t)j * T + lt) * 8;
      const int n = FULL ? 8 : ln_count<D>(c);
      Oct<EL> o{};
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        float a[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          a[k] = (oct_get<EL>(v[j], i + k) - mu) * r;
          if constexpr (AFF == 1) a[k] *= oct_get<PEL>(gm[j], i + k);
          if constexpr (AFF == 2) a[k] = __builtin_fmaf(a[k], oct_get<PEL>(gm[j], i + k), oct_get<PEL>(bt[j], i + k));
        }
        oct_set2<EL>(o, i, a[0], a[1]);
      }
      char *dst = (char *)y + (row * D + c) * el_bytes<EL>;
      if (FULL || n == 8) oct_store<EL>(dst, o);
      else oct_store_part<EL>(dst, o, n);
      if constexpr (CK >= 0) {
        // (zeros behind the row's end do not change a block's maximum)
        const uint32_t byte = mx_scale_byte<CK>(quad_max(oct_amax<EL>(v[j])));
        const u32x2 w = mx_encode<EL, CK>(v[j], mx_inverse(byte), byte != 255);
        uint8_t *cd = (uint8_t *)codes + row * D + c;
        if (FULL || n == 8) codes_store<CK>(cd, w);
        else codes_store_part<CK>(cd, w, n);
        if ((lt & 3) == 0 && (FULL || n > 0)) ((uint8_t *)scales)[row * NB + c / 32] = (uint8_t)byte;
      }
    }
  }
}

// Row groups walk the rows with a stride and keep their columns' part of
// dgamma and dbeta in registers; each leaves one row of part [2][D] behind
// (ln_grad_columns adds them in order).
template <int EL, int PEL, int AFF, int CK, int T, int NCH, int RPB, int64_t D>
__device__ __forceinline__ void ln_grad_rows(const void *__restrict__ dy, const void *__restrict__ x, const void *__restrict__ scales,
                                             const void *__restrict__ gamma, const float *__restrict__ mean,
                                             const float *__restrict__ rstd, void *__restrict__ dx, float *__restrict__ part, int64_t R) {
  static_assert((int64_t)T * NCH * 8 >= D && (T == 64 || RPB == 1));
  constexpr bool FULL = (int64_t)T * NCH * 8 == D;
  constexpr int64_t NB = (D + 31) / 32;
  __shared__ float slots[2][2 * (T / 64)];
  const int lt = threadIdx.x % T, group = threadIdx.x / T;
  Oct<PEL> gm[NCH];
  float dg[NCH][8], db[NCH][8];
#pragma unroll
  for (int j = 0; j < NCH; ++j) {
    const int64_t c = ((int64_t)j * T + lt) * 8;
    if constexpr (AFF >= 1) gm[j] = ln_load<PEL, FULL>(gamma, c, ln_count<D>(c));
#pragma unroll
    for (int i = 0; i < 8; ++i) dg[j][i] = db[j][i] = 0;
  }
  const int64_t first = (int64_t)blockIdx.x * RPB + group, stride = (int64_t)gridDim.x * RPB;
  int parity = 0;
  for (int64_t row = first; row < R; row += stride) {
    Oct<EL> vd[NCH];
    float xv[NCH][8];
    const float mu = mean[row], r = rstd[row];
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
      const int64_t c = ((int64_t)j * T + lt) * 8;
      const int n = ln_count<D>(c);
      vd[j] = ln_load<EL, FULL>(dy, row * D + c, n);
      if constexpr (CK >= 0) {
        const uint8_t *p = (const uint8_t *)x + row * D + c;
        const u32x2 w = FULL || n == 8 ? codes_load<CK>(p) : codes_load_part<CK>(p, n);
        const uint32_t byte = FULL || n > 0 ? ((const uint8_t *)scales)[row * NB + c / 32] : 0;
        mx_decode<CK>(w, mx_scale(byte), xv[j]);
      } else {
        const Oct<EL> o = ln_load<EL, FULL>(x, row * D + c, n);
#pragma unroll
        for (int i = 0; i < 8; ++i) xv[j][i] = oct_get<EL>(o, i);
      }
    }
    float s[2] = {0, 0};
#pragma unroll
    for (int j = 0; j < NCH; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float d = oct_get<EL>(vd[j], i), xh = (xv[j][i] - mu) * r;
        const float g = AFF >= 1 ? d * oct_get<PEL>(gm[j], i) : d;
        // (behind the row's end dy and gamma are zeros)
        s[0] += g;
        s[1] = __builtin_fmaf(g, xh, s[1]);
        xv[j][i] = xh;
        dg[j][i] = __builtin_fmaf(d, xh, dg[j][i]);
        db[j][i] += d;
      }
    group_sum<T>(s, slots[parity]);
    parity ^= 1;
    const float m0 = s[0] / (float)D, m1 = s[1] / (float)D;
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
      const int64_t c = ((int64_t)j * T + lt) * 8;
      const int n = FULL ? 8 : ln_count<D>(c);
      Oct<EL> o{};
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        float a[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const float d = oct_get<EL>(vd[j], i + k);
          const float g = AFF >= 1 ? d * oct_get<PEL>(gm[j], i + k) : d;
          a[k] = r * ((g - m0) - xv[j][i + k] * m1);
        }
        oct_set2<EL>(o, i, a[0], a[1]);
      }
      char *dst = (char *)dx + (row * D + c) * el_bytes<EL>;
      if (FULL || n == 8) oct_store<EL>(dst, o);
      else oct_store_part<EL>(dst, o, n);
    }
  }
  if constexpr (AFF >= 1) {
    if (first >= R) return; // (only the first min(groups, R) rows of `part` are read)
    float *p = part + first * (AFF * D);
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
      const int64_t c = ((int64_t)j * T + lt) * 8;
      const int n = FULL ? 8 : ln_count<D>(c);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (i >= n) break;
        p[c + i] = dg[j][i];
        if constexpr (AFF >= 2) p[D + c + i] = db[j][i];
      }
    }
  }
}

// dgamma and dbeta: column c of part [P][AFF D] summed over its rows, 64
// columns a workgroup, the rows dealt to SL slices of threads.
template <int PEL, int AFF, int SL, int64_t D>
__device__ __forceinline__ void ln_grad_columns(const float *__restrict__ part, int64_t P, void *__restrict__ dgamma, void *__restrict__ dbeta) {
  __shared__ float s[SL][64];
  const int lane = threadIdx.x % 64, sl = threadIdx.x / 64;
  const int64_t c = (int64_t)blockIdx.x * 64 + lane;
  float a = 0;
  if (c < AFF * D)
#pragma unroll 8
    for (int64_t p = sl; p < P; p += SL) a += part[p * (AFF * D) + c];
  s[sl][lane] = a;
  __syncthreads();
  if (sl != 0 || c >= AFF * D) return;
#pragma unroll
  for (int i = 1; i < SL; ++i) a += s[i][lane];
  void *out = c < D ? dgamma : dbeta;
  const int64_t i = c < D ? c : c - D;
  if constexpr (PEL == EL_F32) ((float *)out)[i] = a;
  else if constexpr (PEL == EL_BF16) ((uint16_t *)out)[i] = f32_to_bf16_rne(a);
  else ((uint16_t *)out)[i] = __builtin_bit_cast(uint16_t, (_Float16)a);
}

} // namespace hf
