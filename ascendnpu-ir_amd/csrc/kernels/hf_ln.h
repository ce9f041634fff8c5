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
// A row group of T threads owns a row, NCH 16-byte accesses a thread (access
// j at column (j T + thread) * V, so a group's accesses are consecutive and
// neighbouring lanes hold a block of 32).  RPB row groups share a workgroup
// and take their rows in step; a row is loaded while the one before it is
// worked on.
#pragma once
#include "hf_mx.h"

namespace hf {

typedef float v4f_ln __attribute__((ext_vector_type(4)));

// Sums over the lanes of a row group, or of the wave where a row has more:
// up to 16 lanes by DPP, then the four rows of lanes in order.
template <int T> __device__ __forceinline__ float lane_sum(float v) {
  auto dpp = [](float a, auto ctrl) {
    return u2f((uint32_t)__builtin_amdgcn_update_dpp(0, (int)f2u(a), decltype(ctrl)::value, 0xF, 0xF, true));
  };
  v += dpp(v, std::integral_constant<int, 0xB1>{});  // quad 1 0 3 2
  v += dpp(v, std::integral_constant<int, 0x4E>{});  // quad 2 3 0 1
  v += dpp(v, std::integral_constant<int, 0x141>{}); // eight lanes mirrored
  if constexpr (T == 8) return v;
  v += dpp(v, std::integral_constant<int, 0x140>{}); // sixteen lanes mirrored
  if constexpr (T == 16) return v;
  auto lane = [&](int l) { return u2f((uint32_t)__builtin_amdgcn_readlane((int)f2u(v), l)); };
  return (lane(0) + lane(16)) + (lane(32) + lane(48));
}

// Sums of N values over each row group; slots: N * T / 64 floats a group.
template <int T, int N> __device__ __forceinline__ void group_sum(float (&v)[N], float *slots) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = lane_sum<T>(v[i]);
  if constexpr (T > 64) {
    constexpr int W = T / 64;
    slots += threadIdx.x / T * (N * W);
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

// Weight and bias of a thread's columns: V values of type PEL as they lie,
// zeros behind the row's end (put there by put_right).
template <int PEL, int V, int64_t D> struct LnParam {
  static constexpr int PV = mx_vals<PEL>, N = V / PV > 0 ? V / PV : 1;
  Pack<PEL> p[N];
  __device__ __forceinline__ float get(int i) const { return pack_get<PEL>(p[i / PV], i % PV); }
  __device__ __forceinline__ void load(const void *base, int64_t c) {
#pragma unroll
    for (int k = 0; k < N; ++k) p[k] = pack_load_row<PEL, D, false>(base, 0, c + k * PV);
  }
  __device__ __forceinline__ void put_right(int64_t c) {
#pragma unroll
    for (int k = 0; k < N; ++k) pack_at<PEL, D>(p[k], c + k * PV);
  }
};

// valid elements of the access at column c
template <int64_t D, int V, bool FULL> __device__ __forceinline__ int ln_count(int64_t c, bool ok) {
  if (!ok) return 0;
  return FULL ? V : (int)(D - c <= 0 ? 0 : D - c < V ? D - c : V);
}

// AFF: 0 neither weight nor bias, 1 gamma, 2 gamma and beta (of type PEL).
// CK: format of the checkpoint, -1 for none.  mean and rstd may be null.
template <int EL, int PEL, int AFF, int CK, int T, int NCH, int RPB, int64_t D>
__device__ __forceinline__ void ln_forward(const void *__restrict__ x, const void *__restrict__ gamma, const void *__restrict__ beta,
                                           void *__restrict__ y, float *__restrict__ mean, float *__restrict__ rstd,
                                           void *__restrict__ codes, void *__restrict__ scales, int64_t R, float eps) {
  constexpr int V = mx_vals<EL>, W = T > 64 ? T / 64 : 1;
  static_assert((int64_t)T * NCH * V >= D);
  constexpr bool FULL = (int64_t)T * NCH * V == D;
  constexpr int64_t NB = (D + 31) / 32;
  __shared__ float slots[2][RPB * W];
  const int lt = threadIdx.x % T, group = threadIdx.x / T;
  auto col = [&](int j) { return ((int64_t)j * T + lt) * V; };
  if ((int64_t)blockIdx.x * RPB >= R) return;
  // (a row past the last is the last one again, of which nothing is written)
  auto load = [&](int64_t row, Pack<EL> (&v)[NCH]) {
#pragma unroll
    for (int j = 0; j < NCH; ++j) v[j] = pack_load_row<EL, D>(x, row < R ? row : R - 1, col(j));
  };
  const int64_t step = (int64_t)gridDim.x * RPB;
  Pack<EL> va[NCH], vb[NCH];
  LnParam<PEL, V, D> gm[NCH], bt[NCH];
#pragma unroll
  for (int j = 0; j < NCH; ++j) {
    if constexpr (AFF >= 1) gm[j].load(gamma, col(j));
    if constexpr (AFF >= 2) bt[j].load(beta, col(j));
  }
  load((int64_t)blockIdx.x * RPB + group, va);
#pragma unroll
  for (int j = 0; j < NCH; ++j) {
    if constexpr (AFF >= 1 && !FULL) gm[j].put_right(col(j));
    if constexpr (AFF >= 2 && !FULL) bt[j].put_right(col(j));
  }
  auto work = [&](int64_t row, Pack<EL> (&v)[NCH]) {
    float s[1] = {0}, q[1] = {0};
    if constexpr (!FULL)
#pragma unroll
      for (int j = 0; j < NCH; ++j) pack_at<EL, D>(v[j], col(j));
#pragma unroll
    for (int j = 0; j < NCH; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) s[0] += pack_get<EL>(v[j], i);
    group_sum<T>(s, slots[0]);
    const float mu = s[0] / (float)D;
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
      const int n = ln_count<D, V, FULL>(col(j), true);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float d = pack_get<EL>(v[j], i) - mu;
        if (FULL || i < n) q[0] = __builtin_fmaf(d, d, q[0]);
      }
    }
    group_sum<T>(q, slots[1]);
    const float r = 1.0f / __builtin_sqrtf(q[0] / (float)D + eps);
    if (lt == 0 && row < R) {
      if (mean) mean[row] = mu;
      if (rstd) rstd[row] = r;
    }
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
      const int n = ln_count<D, V, FULL>(col(j), row < R);
      Pack<EL> o{};
#pragma unroll
      for (int i = 0; i < V; i += 2) {
        float a[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          a[k] = (pack_get<EL>(v[j], i + k) - mu) * r;
          if constexpr (AFF == 1) a[k] *= gm[j].get(i + k);
          if constexpr (AFF == 2) a[k] = __builtin_fmaf(a[k], gm[j].get(i + k), bt[j].get(i + k));
        }
        pack_set2<EL>(o, i, a[0], a[1]);
      }
      char *dst = (char *)y + (row * D + col(j)) * el_bytes<EL>;
      if (n == V) pack_store<EL>(dst, o);
      else if (!FULL) pack_store_part<EL>(dst, o, n);
      if constexpr (CK >= 0) {
        // (zeros behind the row's end do not change a block's maximum)
        const uint32_t byte = mx_scale_byte<CK>(block_max<EL>(pack_amax<EL>(v[j])));
        const u32x2 w = mx_encode<EL, CK>(v[j], mx_inverse(byte), byte != 255);
        uint8_t *cd = (uint8_t *)codes + row * D + col(j);
        if (n == V) codes_store<EL, CK>(cd, w);
        else if (!FULL) codes_store_part<EL, CK>(cd, w, n);
        if (lt % mx_lanes<EL> == 0 && n > 0) ((uint8_t *)scales)[row * NB + col(j) / 32] = (uint8_t)byte;
      }
    }
  };
  // (the last rows apart: a load that only some turns make would have the wait
  // for the row at hand wait for the next one too, and one that reads no new
  // row had all workgroups read the last row: [777, 5003] f32 11.9 us for 8.0)
  int64_t row0 = (int64_t)blockIdx.x * RPB;
  for (; row0 + step < R; row0 += step) {
    load(row0 + step + group, vb);
    __builtin_amdgcn_sched_barrier(0);
    work(row0 + group, va);
#pragma unroll
    for (int j = 0; j < NCH; ++j) va[j] = vb[j];
  }
  work(row0 + group, va);
}

// Row groups walk the rows with a stride and keep their columns' part of
// dgamma and dbeta in registers; the groups of a workgroup add theirs in LDS
// and leave one row of part [AFF][D] behind (ln_grad_columns adds those).
template <int EL, int PEL, int AFF, int CK, int T, int NCH, int RPB, int64_t D, bool SUMS>
__device__ __forceinline__ void ln_grad_rows(const void *__restrict__ dy, const void *__restrict__ x, const void *__restrict__ scales,
                                             const void *__restrict__ gamma, const float *__restrict__ mean,
                                             const float *__restrict__ rstd, void *__restrict__ dx, float *__restrict__ part, int64_t R, uint32_t block,
                                             uint32_t blocks) {
  constexpr int V = mx_vals<EL>, W = T > 64 ? T / 64 : 1;
  static_assert((int64_t)T * NCH * V >= D);
  constexpr bool FULL = (int64_t)T * NCH * V == D;
  constexpr int64_t NB = (D + 31) / 32;
  constexpr int CAP = T * NCH * V; // columns of a row group
  // (a workgroup of 1024 threads has no registers for the next row of the widest f32 rows)
  constexpr bool AHEAD = T * RPB < 1024 || NCH <= 2;
  __shared__ float slots[2][RPB * 2 * W];
  __shared__ __attribute__((aligned(16))) float sums[SUMS && RPB > 1 ? RPB * CAP : 4];
  const int lt = threadIdx.x % T, group = threadIdx.x / T;
  auto col = [&](int j) { return ((int64_t)j * T + lt) * V; };
  if ((int64_t)block * RPB >= R) return; // (its row of `part` is not read)
  LnParam<PEL, V, D> gm[NCH];
  float dg[NCH][V], db[NCH][V];
#pragma unroll
  for (int j = 0; j < NCH; ++j) {
#pragma unroll
    for (int i = 0; i < V; ++i) dg[j][i] = db[j][i] = 0;
  }
  struct Row {
    Pack<EL> d[NCH], x[NCH];
    u32x2 code[NCH];
    uint32_t byte[NCH];
    float mu, r;
  };
  // (a row past the last is the last one again: its dy counts as zeros)
  auto load = [&](int64_t row, Row &v) {
    row = row < R ? row : R - 1;
    v.mu = mean[row], v.r = rstd[row];
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
      v.d[j] = pack_load_row<EL, D>(dy, row, col(j));
      if constexpr (CK >= 0) {
        const int64_t b = col(j) / 32;
        v.code[j] = codes_load_row<EL, CK, D>(x, row, col(j));
        v.byte[j] = ((const uint8_t *)scales)[row * NB + (FULL || b < NB ? b : NB - 1)];
      } else {
        v.x[j] = pack_load_row<EL, D>(x, row, col(j));
      }
    }
  };
  auto put_right = [&](bool ok, Row &v) {
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
      if constexpr (!FULL) {
        pack_at<EL, D>(v.d[j], col(j));
        if constexpr (CK >= 0) v.code[j] = codes_at<EL, CK, D>(v.code[j], col(j));
        else pack_at<EL, D>(v.x[j], col(j));
      }
      if (RPB > 1 && !ok) {
        v.d[j] = Pack<EL>{};
        if constexpr (CK >= 0) v.code[j] = u32x2{0, 0}, v.byte[j] = 0;
        else v.x[j] = Pack<EL>{};
      }
    }
    if (RPB > 1 && !ok) v.mu = v.r = 0;
  };
  const int64_t step = (int64_t)blocks * RPB;
  Row ra, rb;
  int parity = 0;
#pragma unroll
  for (int j = 0; j < NCH; ++j)
    if constexpr (AFF >= 1) gm[j].load(gamma, col(j));
  load((int64_t)block * RPB + group, ra);
#pragma unroll
  for (int j = 0; j < NCH; ++j)
    if constexpr (AFF >= 1 && !FULL) gm[j].put_right(col(j));
  auto work = [&](int64_t row, Row &cur) {
    put_right(row < R, cur);
    float xh[NCH][V], s[2] = {0, 0};
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
      if constexpr (CK >= 0) mx_decode<EL, CK>(cur.code[j], mx_scale(cur.byte[j]), xh[j]);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float d = pack_get<EL>(cur.d[j], i);
        xh[j][i] = ((CK >= 0 ? xh[j][i] : pack_get<EL>(cur.x[j], i)) - cur.mu) * cur.r;
        const float g = AFF >= 1 ? d * gm[j].get(i) : d;
        // (behind the row's end, and in rows past the last, dy is zero)
        s[0] += g;
        s[1] = __builtin_fmaf(g, xh[j][i], s[1]);
        if constexpr (SUMS) {
          dg[j][i] = __builtin_fmaf(d, xh[j][i], dg[j][i]);
          db[j][i] += d;
        }
      }
    }
    group_sum<T>(s, slots[parity]);
    parity ^= 1;
    const float m0 = s[0] / (float)D, m1 = s[1] / (float)D;
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
      const int n = ln_count<D, V, FULL>(col(j), row < R);
      Pack<EL> o{};
#pragma unroll
      for (int i = 0; i < V; i += 2) {
        float a[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const float d = pack_get<EL>(cur.d[j], i + k);
          const float g = AFF >= 1 ? d * gm[j].get(i + k) : d;
          a[k] = cur.r * ((g - m0) - xh[j][i + k] * m1);
        }
        pack_set2<EL>(o, i, a[0], a[1]);
      }
      char *dst = (char *)dx + (row * D + col(j)) * el_bytes<EL>;
      if (n == V) pack_store<EL>(dst, o);
      else if (!FULL) pack_store_part<EL>(dst, o, n);
    }
  };
  int64_t row0 = (int64_t)block * RPB;
  for (; row0 + step < R; row0 += step) {
    if constexpr (AHEAD) {
      load(row0 + step + group, rb);
      __builtin_amdgcn_sched_barrier(0);
    }
    work(row0 + group, ra);
    if constexpr (AHEAD) ra = rb;
    else load(row0 + step + group, ra);
  }
  work(row0 + group, ra);
  if constexpr (SUMS) {
    float *p = part + (int64_t)block * (AFF * D);
#pragma unroll
    for (int a = 0; a < AFF; ++a) {
      float(&mine)[NCH][V] = a == 0 ? dg : db;
      if constexpr (RPB == 1) {
#pragma unroll
        for (int j = 0; j < NCH; ++j) {
          const int n = ln_count<D, V, FULL>(col(j), true);
#pragma unroll
          for (int i = 0; i < V; ++i)
            if (FULL || i < n) p[a * D + col(j) + i] = mine[j][i];
        }
      } else {
        if (a > 0) __syncthreads();
#pragma unroll
        for (int j = 0; j < NCH; ++j)
#pragma unroll
          for (int i = 0; i < V; i += 4)
            *reinterpret_cast<v4f_ln *>(&sums[group * CAP + col(j) + i]) = v4f_ln{mine[j][i], mine[j][i + 1], mine[j][i + 2], mine[j][i + 3]};
        __syncthreads();
        for (int c = threadIdx.x; c < (int)D; c += T * RPB) {
          float t = sums[c];
#pragma unroll
          for (int k = 1; k < RPB; ++k) t += sums[k * CAP + c];
          p[a * D + c] = t;
        }
      }
    }
  }
}

// dgamma and dbeta: column c of part [P][AFF D], P at most LNC_ROWS, summed
// over its rows: 32 columns a workgroup, the rows dealt to 32 slices of
// threads, whose loads are all in flight at once.
template <int PEL> __device__ __forceinline__ void param_store(void *out, int64_t i, float a) {
  if constexpr (PEL == EL_F32) ((float *)out)[i] = a;
  else if constexpr (PEL == EL_BF16) ((uint16_t *)out)[i] = f32_to_bf16_rne(a);
  else ((uint16_t *)out)[i] = __builtin_bit_cast(uint16_t, (_Float16)a);
}
constexpr int LNC_COLS = 32, LNC_SLICES = 32, LNC_ROWS = 256;
template <int PEL, int AFF, int64_t D>
__device__ __forceinline__ void ln_grad_columns(const float *__restrict__ part, int64_t P, void *__restrict__ dgamma, void *__restrict__ dbeta) {
  __shared__ float s[LNC_SLICES][LNC_COLS + 1];
  const int lane = threadIdx.x % LNC_COLS, sl = threadIdx.x / LNC_COLS;
  const int64_t c = (int64_t)blockIdx.x * LNC_COLS + lane;
  float v[LNC_ROWS / LNC_SLICES], a = 0;
#pragma unroll
  for (int i = 0; i < LNC_ROWS / LNC_SLICES; ++i) {
    const int64_t p = sl + i * LNC_SLICES;
    v[i] = p < P && c < AFF * D ? part[p * (AFF * D) + c] : 0.0f;
  }
#pragma unroll
  for (int i = 0; i < LNC_ROWS / LNC_SLICES; ++i) a += v[i];
  s[sl][lane] = a;
  __syncthreads();
  if (sl != 0 || c >= AFF * D) return;
#pragma unroll
  for (int i = 1; i < LNC_SLICES; ++i) a += s[i][lane];
  param_store<PEL>(c < D ? dgamma : dbeta, c < D ? c : c - D, a);
}

// Few rows: dgamma and dbeta need no row's sums, only its mean and rstd, so
// that one launch does all: the first workgroups own 32 columns each and read
// dy and x of every row of them, the others make dx.  Lanes of 16 bytes side
// by side, the rest of the threads down the rows, four of them in flight;
// lanes of the same columns are added first, then the waves in order.
// [64, 1024] f32: 3.6 us, 4.7 + 2.9 in two launches; [777, 2048] bf16 6.9.
template <int EL, int PEL, int AFF, int CK, int BT, int64_t D, int COLS>
__device__ __forceinline__ void ln_grad_slab(const void *__restrict__ dy, const void *__restrict__ x, const void *__restrict__ scales,
                                             const float *__restrict__ mean, const float *__restrict__ rstd, void *__restrict__ dgamma,
                                             void *__restrict__ dbeta, int64_t R, uint32_t block) {
  constexpr int V = mx_vals<EL>, CL = COLS / V, RL = BT / CL, U = 4, W = BT / 64;
  constexpr int64_t NB = (D + 31) / 32;
  __shared__ float sums[AFF][W][COLS];
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const int64_t c0 = (int64_t)block * COLS, c = c0 + threadIdx.x % CL * V;
  float dg[V], db[V];
#pragma unroll
  for (int i = 0; i < V; ++i) dg[i] = db[i] = 0;
  for (int64_t row0 = threadIdx.x / CL; row0 < R; row0 += U * RL) {
    Pack<EL> d[U], xv[U];
    u32x2 code[U];
    uint32_t byte[U];
    float mu[U], r[U];
#pragma unroll
    for (int u = 0; u < U; ++u) { // (a row past the last is the last one again, its dy counts as zeros)
      const int64_t row = row0 + u * RL < R ? row0 + u * RL : R - 1;
      mu[u] = mean[row], r[u] = rstd[row];
      d[u] = pack_load_row<EL, D, false>(dy, row, c);
      if constexpr (CK >= 0) {
        code[u] = codes_load_row<EL, CK, D>(x, row, c);
        byte[u] = ((const uint8_t *)scales)[row * NB + c0 / 32];
      } else {
        xv[u] = pack_load_row<EL, D, false>(x, row, c);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool ok = row0 + u * RL < R;
      if constexpr (D % COLS != 0) {
        pack_at<EL, D>(d[u], c);
        if constexpr (CK >= 0) code[u] = codes_at<EL, CK, D>(code[u], c);
        else pack_at<EL, D>(xv[u], c);
      }
      float xh[V];
      if constexpr (CK >= 0) mx_decode<EL, CK>(code[u], mx_scale(byte[u]), xh);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float g = pack_get<EL>(d[u], i), h = ((CK >= 0 ? xh[i] : pack_get<EL>(xv[u], i)) - mu[u]) * r[u];
        dg[i] = ok ? __builtin_fmaf(g, h, dg[i]) : dg[i];
        db[i] = ok ? db[i] + g : db[i];
      }
    }
  }
#pragma unroll
  for (int a = 0; a < AFF; ++a)
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float v = a == 0 ? dg[i] : db[i];
#pragma unroll
      for (int k = CL; k < 64; k *= 2) v += __shfl_xor(v, k);
      if (lane < CL) sums[a][wave][lane * V + i] = v;
    }
  __syncthreads();
  const int a = threadIdx.x / COLS, at = threadIdx.x % COLS;
  const int64_t to = c0 + at;
  if (a >= AFF || to >= D) return;
  float v = sums[a][0][at];
#pragma unroll
  for (int w = 1; w < W; ++w) v += sums[a][w][at];
  param_store<PEL>(a == 0 ? dgamma : dbeta, to, v);
}
template <int EL, int PEL, int AFF, int CK, int T, int NCH, int RPB, int64_t D, int COLS>
__device__ __forceinline__ void ln_grad_once(const void *__restrict__ dy, const void *__restrict__ x, const void *__restrict__ scales,
                                             const void *__restrict__ gamma, const float *__restrict__ mean,
                                             const float *__restrict__ rstd, void *__restrict__ dx, void *__restrict__ dgamma,
                                             void *__restrict__ dbeta, int64_t R) {
  // (workgroup b runs on XCD b % 8: neighbouring slabs, which share cache
  // lines, on the same one)
  constexpr uint32_t CB = (uint32_t)((D + COLS - 1) / COLS), EACH = (CB + 7) / 8;
  const uint32_t slab = blockIdx.x % 8 * EACH + blockIdx.x / 8;
  if (blockIdx.x >= 8 * EACH)
    ln_grad_rows<EL, PEL, AFF, CK, T, NCH, RPB, D, false>(dy, x, scales, gamma, mean, rstd, dx, nullptr, R, blockIdx.x - 8 * EACH,
                                                          gridDim.x - 8 * EACH);
  else if (slab < CB) ln_grad_slab<EL, PEL, AFF, CK, T * RPB, D, COLS>(dy, x, scales, mean, rstd, dgamma, dbeta, R, slab);
}

} // namespace hf
