// bf16 rows times a block-scaled weight, few rows (hfusion.linear_mx):
//   C[m, n] = sum_k A[m, k] w[n, k] 2^E[n, k / 32]
// A [M, K] bf16, w [N, K] 8-bit codes or [N, K/2] bytes of two e2m1 codes,
// one e8m0 byte per 32 k of a row.  Such a call reads every weight once and
// multiplies little: what counts is how fast every CU pulls its share of the
// weights, and of the rows that go with them, through its L1.
//
// A workgroup owns 8 MD rows and 16 NT columns of C and its NW waves split K,
// so no sum crosses workgroups; the waves' partial sums meet in LDS, added in
// wave order.  Each wave has a slot of its own in LDS, filled by LDS DMA: 64
// bytes of codes of every column (KS k) and the same k of every row; while one
// wave multiplies, the others' slots fill (rings of two to four slots a wave
// took the same time).  The order of k within a matrix-core step is free as
// long as both operands agree on it: a lane takes 16 bytes of codes of its
// column, 16 (8-bit) or 32 (e2m1) consecutive k, and feeds them eight at a
// time.  Codes become bf16 pairs, scale included, in one instruction; code
// times scale fits bf16's significand, so f32 sums are the only rounding
// before the epilogue's, but at the ends of bf16's range (2^128 and more is
// infinite, what is no multiple of 2^-133 is rounded to one).
// What bounds it: at N = K = 4096 and 8-bit codes M = 1 takes 5.4 us (16.8 MB of
// codes are 3.1 us at the rate of a large copy; an empty launch is 2.3), M = 48
// 7.5, M = 128 11, M = 512 28; e2m1 3.3, 6.5, 9.5, 27 us.  The codes cross HBM at
// 4 to 4.5 TB/s, and past a few rows the rows' way through the L1s (16 bytes a
// lane of DMA, about 120 GB/s a CU) is added to that.
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

// LDS slot: the rows' k as pieces of 128 bytes, 16-byte granule g of row r at
// position g ^ ((r >> 1) & 7); 64 bytes of codes a column, at g ^ ((r >> 2) &
// 3): the 16 rows of a fragment read hit 16 bank groups.
template <int FMT, typename Epi, int MD, int NT, int NW, int64_t K, typename Args>
__device__ __forceinline__ void linear_wx(const uint16_t *__restrict__ A, const uint8_t *__restrict__ W, const uint8_t *__restrict__ Sc,
                                          typename Epi::out_t *__restrict__ out, int64_t M, int64_t N, const Args &P) {
  static_assert(K % 32 == 0);
  constexpr int MT = (MD + 1) / 2, TM = 16 * MT, TN = 16 * NT;
  constexpr int CPB = FMT == MX_E2M1 ? 2 : 1;        // codes a byte
  constexpr int KS = 64 * CPB, NA = CPB;             // k a slice, 128-byte pieces of an A row
  constexpr int STEPS = 2 * CPB;                     // matrix-core steps of a slice
  constexpr int64_t WP = K / CPB;
  constexpr int SP = (int)(K / 32);                  // scale bytes of a column
  constexpr int ns = (int)((K + KS - 1) / KS);
  constexpr bool RAGGED = K % KS != 0;
  constexpr int SLOT = (NA * MD + NT) * 1024;        // (a DMA instruction fills 1 KiB)
  constexpr int SPITCH = TN + 4;                     // scales in LDS, one row a block of k
  constexpr int PIECES = (TN * SP + NW * 512 - 1) / (NW * 512); // 8-byte pieces of them a thread
  constexpr int SLOTS = NW * SLOT, SUMS = NW * MT * NT * 1024, SCALES = SLOTS > SUMS ? SLOTS : SUMS;
  // (past K and past the last column, bytes of other scales or none are read and not used)
  __shared__ __attribute__((aligned(1024))) char lds[SCALES + (SP + 8) * SPITCH];
  // workgroup b runs on XCD b % 8: the row tiles of a column tile follow each
  // other there, so that one L2 fetches its codes for all of them.  Grid: row
  // tiles * column tiles, these rounded up to eight.
  const uint32_t tn = (uint32_t)((N + TN - 1) / TN), rt = (uint32_t)((M + 8 * MD - 1) / (8 * MD));
  const uint32_t ct = blockIdx.x / 8 / rt * 8 + blockIdx.x % 8;
  if (ct >= tn) return;
  const int64_t m0 = (int64_t)(blockIdx.x / 8 % rt) * (8 * MD), n0 = (int64_t)ct * TN;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / 64), lane = threadIdx.x % 64;
  const uint32_t base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)&lds[0];
  const uint32_t slot = base + (uint32_t)(wave * SLOT), scl = base + (uint32_t)SCALES;

  // the output elements of a thread, consecutive threads on consecutive
  // columns, and what the epilogue reads of their rows and columns: asked for
  // first (one after another at the end, those loads took as long as the
  // product: 9.5 us at M = 48, N = 5003, 8-bit codes, K = 4096)
  constexpr int OUTS = (8 * MD * TN + NW * 64 - 1) / (NW * 64);
  typename Epi::row_t erow[OUTS];
  typename Epi::col_t ecol[OUTS];
#pragma unroll
  for (int e = 0; e < OUTS; ++e) {
    const int o = (int)threadIdx.x + e * NW * 64;
    const int64_t m = m0 + o / TN, nn = n0 + o % TN;
    erow[e] = Epi::row(m < M ? m : M - 1, P);
    ecol[e] = Epi::col(nn < N ? nn : N - 1, P);
  }

  // the scales of the workgroup's columns lie together
  const uint8_t *const s0 = Sc + n0 * SP;
  const int sbytes = (int)(N - n0 < TN ? N - n0 : TN) * SP;
  u32x2 piece[PIECES];
#pragma unroll
  for (int e = 0; e < PIECES; ++e) {
    const int at = 8 * ((int)threadIdx.x + e * NW * 64);
    piece[e] = u32x2{0, 0};
    if (at + 8 <= sbytes) piece[e] = *reinterpret_cast<const u32x2_any *>(s0 + at);
    else
      for (int i = 0; at + i < sbytes; ++i) {
        if (i < 4) piece[e].x |= (uint32_t)s0[at + i] << (8 * i);
        else piece[e].y |= (uint32_t)s0[at + i] << (8 * (i - 4));
      }
  }

  // this lane's source of each DMA instruction as an offset from the slice's
  // first byte (rows and columns past the end re-read the last one, whose
  // results are not stored; in the last slice, what lies past K re-reads the
  // slice's first 16 bytes and is not multiplied)
  uint32_t arow[MD], wrow[NT];
  int wg[NT];
#pragma unroll
  for (int d = 0; d < MD; ++d) {
    const int r = 8 * d + lane / 8;
    const int64_t m = m0 + r < M ? r : M - 1 - m0;
    arow[d] = (uint32_t)(m * K * 2);
  }
  const int ag = (lane % 8) ^ ((lane / 16) & 3); // ((r >> 1) & 7 of row 8 d + lane / 8: bit 2 is d & 1)
#pragma unroll
  for (int d = 0; d < NT; ++d) {
    const int r = 16 * d + lane / 4;
    wg[d] = (lane % 4) ^ ((r >> 2) & 3);
    const int64_t c = n0 + r < N ? r : N - 1 - n0;
    wrow[d] = (uint32_t)(c * WP);
  }
  const char *const a0 = (const char *)(A + m0 * K), *const w0 = (const char *)(W + n0 * WP);
  auto issue = [&](int s) { // slice s into the wave's slot
    const int left = (int)(K - (int64_t)s * KS); // k from the slice's start
#pragma unroll
    for (int b = 0; b < NA; ++b)
#pragma unroll
      for (int d = 0; d < MD; ++d) {
        const int g = ag ^ (4 * (d & 1));
        uint32_t k2 = (uint32_t)(b * 128 + g * 16); // byte of the slice's row
        if (RAGGED && (int)k2 >= 2 * left) k2 = 0;
        mmd_dma16_off(a0 + (int64_t)s * (KS * 2), arow[d] + k2, __builtin_amdgcn_readfirstlane(slot + (uint32_t)((b * MD + d) * 1024)));
      }
#pragma unroll
    for (int d = 0; d < NT; ++d) {
      uint32_t kb = (uint32_t)(wg[d] * 16);
      if (RAGGED && (int)kb * CPB >= left) kb = 0;
      mmd_dma16_off(w0 + (int64_t)s * 64, wrow[d] + kb, __builtin_amdgcn_readfirstlane(slot + (uint32_t)((NA * MD + d) * 1024)));
    }
  };
  if (wave < ns) issue(wave);
  // scales by block, then column: the lanes of a fragment read neighbouring
  // bytes (as they lie, the columns of a power-of-two K share two banks: 19.2
  // us, 7.8 of them those reads, at M = 48, N = 5003, K = 16384)
#pragma unroll
  for (int e = 0; e < PIECES; ++e)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int at = 8 * ((int)threadIdx.x + e * NW * 64) + i;
      if (at < TN * SP) lds[SCALES + at % SP * SPITCH + at / SP] = (char)((i < 4 ? piece[e].x : piece[e].y) >> (8 * (i % 4)));
    }
  __syncthreads();

  const int q = lane / 16, j = lane % 16;
  typedef __attribute__((address_space(3))) const v4i *lds16;
  typedef __attribute__((address_space(3))) const uint8_t *lds1;
  v4f acc[MT][NT];
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int u = 0; u < NT; ++u) acc[t][u] = v4f{0, 0, 0, 0};
#pragma unroll 1
  for (int s = wave; s < ns; s += NW) {
    mmd_wait_vm<0>();
    v4i fw[NT], fa[MT][STEPS];
    uint32_t sb[NT];
#pragma unroll
    for (int u = 0; u < NT; ++u) {
      const int r = 16 * u + j;
      fw[u] = *(lds16)(uintptr_t)(slot + (uint32_t)(NA * MD * 1024 + r * 64 + (q ^ ((r >> 2) & 3)) * 16));
      sb[u] = *(lds1)(uintptr_t)(scl + (uint32_t)((s * (KS / 32) + q * CPB / 2) * SPITCH + r));
    }
#pragma unroll
    for (int c = 0; c < STEPS; ++c) {
      const int k = 16 * CPB * q + 8 * c, b = k / 64, g = k % 64 / 8;
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        const int r = 16 * t + j;
        // (an odd number of eight-row pieces: the last eight rows are another tile's, and are not stored)
        const int rr = MD % 2 != 0 && r >= 8 * MD ? r - 8 : r;
        fa[t][c] = *(lds16)(uintptr_t)(slot + (uint32_t)(b * MD * 1024 + rr * 128 + (g ^ ((rr >> 1) & 7)) * 16));
      }
    }
    if (RAGGED && s == ns - 1) {
      const bool in = (int64_t)s * KS + 16 * CPB * q < K;
#pragma unroll
      for (int u = 0; u < NT; ++u) fw[u] = in ? fw[u] : v4i{0, 0, 0, 0}, sb[u] = in ? sb[u] : 127;
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int c = 0; c < STEPS; ++c) fa[t][c] = in ? fa[t][c] : v4i{0, 0, 0, 0};
    }
    if (s + NW < ns) {
      // the slot has been read (the fragments are in registers) before it is filled again
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      issue(s + NW);
    }
#pragma unroll
    for (int c = 0; c < STEPS; ++c) {
      v4i b[NT];
#pragma unroll
      for (int u = 0; u < NT; ++u) {
        const float scale = u2f(sb[u] << 23);
        if constexpr (FMT == MX_E2M1) b[u] = wx_decode8<FMT>((uint32_t)fw[u][c], 0, scale);
        else b[u] = wx_decode8<FMT>((uint32_t)fw[u][2 * c], (uint32_t)fw[u][2 * c + 1], scale);
      }
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int u = 0; u < NT; ++u) acc[t][u] = Mfma16<MK_BF16>::run(fa[t][c], b[u], acc[t][u]);
    }
  }
  __syncthreads(); // every wave is done with its slot
  v4f *red = reinterpret_cast<v4f *>(lds);
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int u = 0; u < NT; ++u) red[((wave * MT + t) * NT + u) * 64 + lane] = acc[t][u];
  __syncthreads();
  const float *rs = reinterpret_cast<const float *>(lds);
  float sum[OUTS];
#pragma unroll
  for (int e = 0; e < OUTS; ++e) {
    const int o = (int)threadIdx.x + e * NW * 64, r = o / TN, c = o % TN, rr = r % 16;
    const int at = OUTS * NW * 64 == 8 * MD * TN || r < 8 * MD ? ((r / 16 * NT + c / 16) * 64 + rr / 4 * 16 + c % 16) * 4 + rr % 4 : 0;
    sum[e] = rs[at];
#pragma unroll
    for (int w = 1; w < NW; ++w) sum[e] += rs[w * MT * NT * 256 + at];
  }
#pragma unroll
  for (int e = 0; e < OUTS; ++e) {
    const int o = (int)threadIdx.x + e * NW * 64;
    const int64_t m = m0 + o / TN, nn = n0 + o % TN;
    if (o < 8 * MD * TN && m < M && nn < N) out[m * N + nn] = Epi::apply(sum[e], m, nn, erow[e], ecol[e], P);
  }
}

} // namespace hf
