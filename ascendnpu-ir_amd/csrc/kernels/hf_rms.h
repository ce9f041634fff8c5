// Root-mean-square norm of a residual stream, into 8-bit codes (hfusion.rms_norm).
//
//   s = x + residual, rounded once to the rows' type (no residual: s = x)
//   r = f32(1 / sqrt(mean(s^2) + eps)), the squares summed in 64 bits
//   y = (s r) gamma, each product rounded to f32
//   int8:  scale = max|y| f32(1/127) of the row, code = y / scale to the nearest even
//          (a scale that is zero, infinite or NaN: codes 0)
//   8-bit floats: hf_mx.h's codes of y, 32 columns a block
// The sum of squares in 64 bits makes r the same in any order of the additions
// but for one row in some 2^28, and with it the codes: they equal those of a
// serial program, and each row's do not depend on how many rows a launch has.
//
// Rows, accesses and workgroups are the layer norm's (hf_ln.h): a row group of
// T threads keeps a row in registers and loads the next one ahead.  Each row is
// read once and its sum, codes and scale written once, so memory bounds it: bf16
// [8192, 4096] with a residual to int8 43.5 us (235 MB, 5.4 TB/s; a copy of that
// size 5.1), f16 [2003, 8192] to e4m3 21.4 (5.4), f32 [777, 5003] without to e5m2
// 6.9, whose rows end off 16 bytes.  16 rows of 4096 take 3.4 us on the device:
// one load, two reductions and one store, each waiting for the one before.
#pragma once
#include "hf_ln.h"

namespace hf {

// Sum over the lanes of a row group, or of the wave where a row has more.
template <int T> __device__ __forceinline__ double lane_sum64(double v) {
  auto dpp = [](double a, auto ctrl) {
    const uint64_t b = __builtin_bit_cast(uint64_t, a);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, decltype(ctrl)::value, 0xF, 0xF, true);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(b >> 32), decltype(ctrl)::value, 0xF, 0xF, true);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
  };
  v += dpp(v, std::integral_constant<int, 0xB1>{});  // quad 1 0 3 2
  v += dpp(v, std::integral_constant<int, 0x4E>{});  // quad 2 3 0 1
  v += dpp(v, std::integral_constant<int, 0x141>{}); // eight lanes mirrored
  if constexpr (T == 8) return v;
  v += dpp(v, std::integral_constant<int, 0x140>{}); // sixteen lanes mirrored
  if constexpr (T == 16) return v;
  auto lane = [&](int l) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)b, l), hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(b >> 32), l);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
  };
  return (lane(0) + lane(16)) + (lane(32) + lane(48));
}
// Largest of the lanes' unsigned values, as lane_sum64.
template <int T> __device__ __forceinline__ uint32_t lane_max(uint32_t v) {
  auto dpp = [](uint32_t a, auto ctrl) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)a, decltype(ctrl)::value, 0xF, 0xF, true);
  };
  v = max_u32(v, dpp(v, std::integral_constant<int, 0xB1>{}));
  v = max_u32(v, dpp(v, std::integral_constant<int, 0x4E>{}));
  v = max_u32(v, dpp(v, std::integral_constant<int, 0x141>{}));
  if constexpr (T == 8) return v;
  v = max_u32(v, dpp(v, std::integral_constant<int, 0x140>{}));
  if constexpr (T == 16) return v;
  auto lane = [&](int l) { return (uint32_t)__builtin_amdgcn_readlane((int)v, l); };
  return max_u32(max_u32(lane(0), lane(16)), max_u32(lane(32), lane(48)));
}

// int8 codes of four quotients a / b, |a / b| < 127.5, r = RN(1 / b) a normal
// number: a r is within 2^-17 of the quotient, so where the conversions of a r +
// 128 less and plus 2^-15 agree, both are the quotient's; elsewhere (one
// element in some 2^13) the division decides.
__device__ __forceinline__ uint32_t rms_codes4(const float *a, float b, float r) {
  constexpr float W = 0x1p-15f;
  uint32_t lo = 0, hi = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    lo = __builtin_amdgcn_cvt_pk_u8_f32(__builtin_fmaf(a[i], r, 128.0f - W), i, lo);
    hi = __builtin_amdgcn_cvt_pk_u8_f32(__builtin_fmaf(a[i], r, 128.0f + W), i, hi);
  }
  uint32_t w = lo ^ 0x80808080u;
  if (__builtin_expect(lo != hi, 0)) {
    w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) w |= ((uint32_t)(int)__builtin_rintf(a[i] / b) & 0xFFu) << (8 * i);
  }
  return w;
}

// RES: with a residual, whose sum is kept.  OUT: -1 int8 codes with one f32
// scale a row, else the format of the block-scaled codes.  `sum` may be the
// residual's own buffer: a row is read whole before any of it is written.
template <int EL, int PEL, bool RES, int OUT, int T, int NCH, int RPB, int64_t D>
__device__ __forceinline__ void rms_rows(const void *x, const void *residual, const void *gamma, void *sum, void *codes, void *scales, int64_t R,
                                         double eps) {
  constexpr int V = mx_vals<EL>, W = T > 64 ? T / 64 : 1;
  static_assert((int64_t)T * NCH * V >= D);
  constexpr bool FULL = (int64_t)T * NCH * V == D;
  constexpr int64_t NB = (D + 31) / 32;
  __shared__ double sums[2][RPB * W];
  __shared__ uint32_t tops[RPB * W];
  const int lt = threadIdx.x % T, group = threadIdx.x / T, wave = lt / 64;
  auto col = [&](int j) { return ((int64_t)j * T + lt) * V; };
  if ((int64_t)blockIdx.x * RPB >= R) return;
  struct Row {
    Pack<EL> x[NCH], r[RES ? NCH : 1];
  };
  // (a row past the last is the last one again, of which nothing is written)
  auto load = [&](int64_t row, Row &v) {
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
      v.x[j] = pack_load_row<EL, D>(x, row < R ? row : R - 1, col(j));
      if constexpr (RES) v.r[j] = pack_load_row<EL, D>(residual, row < R ? row : R - 1, col(j));
    }
  };
  const int64_t step = (int64_t)gridDim.x * RPB;
  Row va, vb;
  LnParam<PEL, V, D> gm[NCH];
#pragma unroll
  for (int j = 0; j < NCH; ++j) gm[j].load(gamma, col(j));
  load((int64_t)blockIdx.x * RPB + group, va);
  if constexpr (!FULL)
#pragma unroll
    for (int j = 0; j < NCH; ++j) gm[j].put_right(col(j));
  int parity = 0;
  auto work = [&](int64_t row, Row &v) {
    Pack<EL> s[NCH];
    double q = 0;
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
      if constexpr (!FULL) {
        pack_at<EL, D>(v.x[j], col(j));
        if constexpr (RES) pack_at<EL, D>(v.r[j], col(j));
      }
      if constexpr (RES) {
#pragma unroll
        for (int i = 0; i < V; i += 2)
          pack_set2<EL>(s[j], i, pack_get<EL>(v.x[j], i) + pack_get<EL>(v.r[j], i), pack_get<EL>(v.x[j], i + 1) + pack_get<EL>(v.r[j], i + 1));
      } else {
        s[j] = v.x[j];
      }
      // (zeros behind the row's end add nothing)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const double d = pack_get<EL>(s[j], i);
        q = __builtin_fma(d, d, q);
      }
    }
    q = lane_sum64<T>(q);
    if constexpr (T > 64) {
      double *slot = sums[parity] + group * W;
      parity ^= 1;
      if (threadIdx.x % 64 == 0) slot[wave] = q;
      __syncthreads();
      q = slot[0];
#pragma unroll
      for (int w = 1; w < W; ++w) q += slot[w];
    }
    const float r = (float)(1.0 / __builtin_sqrt(q / (double)D + eps));
    float y[NCH][V];
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
      const int n = ln_count<D, V, FULL>(col(j), row < R);
      // (behind the row's end y is zero, but NaN where r is infinite; a block of
      // 32 columns that has an infinity has the byte 255 either way)
      const bool all = OUT >= 0 || (int64_t)(j + 1) * T * V <= D;
      uint32_t most = 0;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float u = pack_get<EL>(s[j], i) * r;
        y[j][i] = u * gm[j].get(i);
        most = max_u32(most, all || i < n ? f2u(y[j][i]) & 0x7FFFFFFFu : 0u);
      }
      if constexpr (RES) {
        char *dst = (char *)sum + (row * D + col(j)) * el_bytes<EL>;
        if (n == V) pack_store<EL>(dst, s[j]);
        else if (!FULL) pack_store_part<EL>(dst, s[j], n);
      }
      if constexpr (OUT < 0) {
        top = max_u32(top, most);
      } else {
        const uint32_t byte = mx_scale_byte<(OUT < 0 ? 0 : OUT)>(block_max<EL>(most));
        const float inv = mx_inverse(byte);
        u32x2 w = {0, 0};
        w.x = mx_pair8<(OUT < 0 ? 0 : OUT)>(y[j][0] * inv, y[j][1] * inv, w.x, false);
        w.x = mx_pair8<(OUT < 0 ? 0 : OUT)>(y[j][2] * inv, y[j][3] * inv, w.x, true);
        if constexpr (V == 8) {
          w.y = mx_pair8<(OUT < 0 ? 0 : OUT)>(y[j][4] * inv, y[j][5] * inv, w.y, false);
          w.y = mx_pair8<(OUT < 0 ? 0 : OUT)>(y[j][6] * inv, y[j][7] * inv, w.y, true);
        }
        if (byte == 255) w = u32x2{0, 0};
        uint8_t *cd = (uint8_t *)codes + row * D + col(j);
        if (n == V) codes_store<EL, MX_E4M3>(cd, w);
        else if (!FULL) codes_store_part<EL, MX_E4M3>(cd, w, n);
        if (lt % mx_lanes<EL> == 0 && n > 0) ((uint8_t *)scales)[row * NB + col(j) / 32] = (uint8_t)byte;
      }
    }
    if constexpr (OUT < 0) {
      top = lane_max<T>(top);
      if constexpr (T > 64) {
        uint32_t *slot = tops + group * W;
        if (threadIdx.x % 64 == 0) slot[wave] = top;
        __syncthreads();
        top = slot[0];
#pragma unroll
        for (int w = 1; w < W; ++w) top = max_u32(top, slot[w]);
      }
      const float scale = u2f(top) * (1.0f / 127.0f);
      if (lt == 0 && row < R) ((float *)scales)[row] = scale;
      const bool ok = scale > 0 && scale < __builtin_inff();
      // (far from 1 the reciprocal is no normal number, or the quotient passes
      // 127.5 because a subnormal scale is a rough one)
      const bool slow = !(scale > 0x1p-100f && scale < 0x1p100f);
      const float inv = 1.0f / scale;
#pragma unroll
      for (int j = 0; j < NCH; ++j) {
        const int n = ln_count<D, V, FULL>(col(j), row < R);
        u32x2 w = {0, 0};
        if (__builtin_expect(slow, 0)) {
          if (ok)
#pragma unroll
            for (int i = 0; i < V; ++i) {
              const float c = __builtin_amdgcn_fmed3f(__builtin_rintf(y[j][i] / scale), -127.0f, 127.0f);
              w[i / 4] |= ((uint32_t)(int)c & 0xFFu) << (8 * (i % 4));
            }
        } else {
          w.x = rms_codes4(y[j], scale, inv);
          if constexpr (V == 8) w.y = rms_codes4(y[j] + 4, scale, inv);
        }
        uint8_t *cd = (uint8_t *)codes + row * D + col(j);
        if (n == V) codes_store<EL, MX_E4M3>(cd, w);
        else if (!FULL) codes_store_part<EL, MX_E4M3>(cd, w, n);
      }
    }
  };
  int64_t row0 = (int64_t)blockIdx.x * RPB;
  for (; row0 + step < R; row0 += step) {
    load(row0 + step + group, vb);
    __builtin_amdgcn_sched_barrier(0);
    work(row0 + group, va);
    va = vb;
  }
  work(row0 + group, va);
}

} // namespace hf
