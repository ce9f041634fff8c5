// The paged 8-bit cache of keys and values, and appending to it
// (hfusion.append_kv).
//
// Cache: keys [blocks, kv heads, BLOCK, D], values [blocks, kv heads, D,
// BLOCK] (so that the tokens that a matrix-core step sums over lie together),
// one e8m0 byte for each block and head of either.  A row of the batch is a
// token at position p of a sequence; it lies in block table[seq][p / BLOCK] at p
// % BLOCK.
//   E    = the smallest exponent with |values| <= TOP 2^E (TOP: the format's
//          largest value), of all the block's tokens: the byte only grows while
//          a block fills, so one append of many tokens and many appends of one
//          leave the same scale
//   code = value 2^-E to nearest even; where E grows, the codes that are there
//          are rounded again, which loses nothing but below the smallest
//          normal code
// Infinities and NaN make the block's byte 255 (its values are NaN) and its
// codes 0.
#pragma once
#include "hf_mx.h"

namespace hf {

// ---------------------------------------------------------------- eight values
template <int EL> __device__ __forceinline__ void load8(const void *p, float (&f)[8]) {
  constexpr int V = mx_vals<EL>;
#pragma unroll
  for (int k = 0; k < 8 / V; ++k) {
    const Pack<EL> o = pack_load<EL, false>((const char *)p + 16 * k);
#pragma unroll
    for (int i = 0; i < V; ++i) f[k * V + i] = pack_get<EL>(o, i);
  }
}
template <int EL> __device__ __forceinline__ void store8(void *p, const float (&f)[8]) {
  constexpr int V = mx_vals<EL>;
#pragma unroll
  for (int k = 0; k < 8 / V; ++k) {
    Pack<EL> o{};
#pragma unroll
    for (int i = 0; i < V; i += 2) pack_set2<EL>(o, i, f[k * V + i], f[k * V + i + 1]);
    pack_store<EL>((char *)p + 16 * k, o);
  }
}

// Rotation of a head's first ROT channels by `turn` (ROT / 2 cosines, then
// sines): channel i with i + ROT / 2, or (PAIRS) 2 i with 2 i + 1.  Two products
// and an addition, each rounded to f32.  A head's channels as slots of 16 that
// turn among themselves, two runs of eight each: the first at at(slot), the
// second next(slot) behind it.
template <int ROT, bool PAIRS> struct Turn {
  static constexpr int HALF = ROT / 2, TURNED = ROT / 16; // slots that turn
  float c[8], s[8];
  __device__ static __forceinline__ int at(int slot) { return PAIRS || slot >= TURNED ? 16 * slot : 8 * slot; }
  __device__ static __forceinline__ int next(int slot) { return PAIRS || slot >= TURNED ? 8 : HALF; }
  __device__ __forceinline__ void load(const float *turn, int slot) {
    if (slot >= TURNED) return;
    load8<EL_F32>(turn + 8 * slot, c);
    load8<EL_F32>(turn + HALF + 8 * slot, s);
  }
  __device__ __forceinline__ void apply(int slot, float (&a)[8], float (&b)[8]) const {
    if (slot >= TURNED) return;
    float f[16];
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = a[i], f[8 + i] = b[i];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float x = PAIRS ? f[2 * i] : f[i], y = PAIRS ? f[2 * i + 1] : f[8 + i];
      const float u = x * c[i] - y * s[i], v = y * c[i] + x * s[i];
      if constexpr (PAIRS) (i < 4 ? a : b)[2 * i % 8] = u, (i < 4 ? a : b)[(2 * i + 1) % 8] = v;
      else a[i] = u, b[i] = v;
    }
  }
};

// ---------------------------------------------------------------- scales
// the byte of a block whose largest magnitude has these f32 bits (TOP is 1.75
// times a power of two in both formats)
template <int FMT> __device__ __forceinline__ uint32_t kv_scale_byte(uint32_t amax) {
  const int e = (int)(amax >> 23), b = e - mx_emax<FMT> + ((amax & 0x7FFFFFu) > 0x600000u);
  return e == 255 ? 255u : (uint32_t)(b > 0 ? b : 0);
}
__device__ __forceinline__ float kv_inverse(uint32_t byte) { return u2f(byte < 254 ? (254u - byte) << 23 : 0x00400000u); }
// codes of eight values under a scale byte
template <int FMT> __device__ __forceinline__ u32x2 kv_encode(const float (&f)[8], uint32_t byte) {
  const float inv = kv_inverse(byte);
  u32x2 w = {0, 0};
  w.x = mx_pair8<FMT>(f[0] * inv, f[1] * inv, w.x, false);
  w.x = mx_pair8<FMT>(f[2] * inv, f[3] * inv, w.x, true);
  w.y = mx_pair8<FMT>(f[4] * inv, f[5] * inv, w.y, false);
  w.y = mx_pair8<FMT>(f[6] * inv, f[7] * inv, w.y, true);
  return byte == 255 ? u32x2{0, 0} : w;
}
// codes under the byte `old` as codes under the larger byte `now`
template <int FMT> __device__ __forceinline__ u32x2 kv_rescale(u32x2 w, uint32_t old, uint32_t now) {
  const int d = (int)old - (int)now;
  const float by = d < -126 ? 0.0f : u2f((uint32_t)(127 + d) << 23);
  u32x2 o = {0, 0};
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const f32x2 a = mx_decode2<FMT>(k ? w.y : w.x, 0), b = mx_decode2<FMT>(k ? w.y : w.x, 1);
    uint32_t t = mx_pair8<FMT>(a.x * by, a.y * by, 0, false);
    t = mx_pair8<FMT>(b.x * by, b.y * by, t, true);
    o[k] = t;
  }
  return now == 255 ? u32x2{0, 0} : o;
}

// ---------------------------------------------------------------- append
// qkv [T, (HQ + 2 HK) D]: queries, keys and values of a token's heads, which
// leave as q [T, HQ, D] and codes.  A tile of C rows owns the blocks whose
// first new row is one of them (that row's neighbour above lies in another
// block or sequence); a workgroup takes one head's keys or values of them, the
// tile's other QB workgroups its queries, HB heads a thread that turn alike.
// Rows with a sequence or position out of range, and blocks out of range, are
// left alone.
// A block's rows are read once, kept in registers until its largest magnitude is
// known, and written as codes (values turned around in LDS, so that a channel's
// tokens leave together); codes that are there already are read again only where
// the scale grows.  No atomics: a block has one owner.  Memory bounds long
// batches: three prompts, 8561 rows of 32 heads over 8 of 128 channels, 40.1 us
// (226 MB, of which 32 are rotations that each XCD reads, 5.6 TB/s; with a tile's
// workgroups on one XCD 45.9); a decoding step of 64 rows takes 5.6 us on the device, the
// chain of positions, table, scale, rows, and the block rounded again.
// Two rows of one place, or a sequence in two pieces that share a block, write
// it at once: codes and scale of its tokens, earlier ones too, need not belong
// together then.  Other blocks are not touched.
template <int EL, int FMT, int HQ, int HK, int D, int ROT, bool PAIRS, int BLOCK, int64_t SLOTS, int64_t PER, int64_t FAR, int64_t NBLK, int C, int QB, int HB>
__device__ __forceinline__ void kv_append(const void *__restrict__ qkv, const float *__restrict__ rot, const int *__restrict__ seq,
                                          const int *__restrict__ pos, const int *__restrict__ table, void *__restrict__ q,
                                          uint8_t *__restrict__ kc, uint8_t *__restrict__ ks, uint8_t *__restrict__ vc,
                                          uint8_t *__restrict__ vs, int64_t T) {
  constexpr int E = el_bytes<EL>, SUBS = 2 * HK + QB, W = (HQ + 2 * HK) * D;
  static_assert(C <= 64 && D % 32 == 0 && ROT % 16 == 0 && ROT <= D && BLOCK % 16 == 0 && BLOCK <= 128);
  const int64_t t0 = (int64_t)(blockIdx.x / SUBS) * C;
  const int sub = blockIdx.x % SUBS, tid = threadIdx.x;
  auto inside = [](int s, int p) { return s >= 0 && s < SLOTS && p >= 0 && p < FAR; };
  using R = Turn<ROT, PAIRS>;
  constexpr int SLOT = D / 16, PARTS = (HQ + HB - 1) / HB;
  if (sub >= 2 * HK) {
    const int n = (int)(T - t0 < C ? T - t0 : C) * (PARTS * SLOT);
    for (int i = (sub - 2 * HK) * 256 + tid; i < n; i += QB * 256) {
      const int64_t t = t0 + i / (PARTS * SLOT);
      const int slot = i % SLOT, h0 = i / SLOT % PARTS * HB, p = pos[t];
      if (!inside(seq[t], p)) continue;
      R turn;
      turn.load(rot + (int64_t)p * ROT, slot);
      const char *src = (const char *)qkv + (t * W + h0 * D + R::at(slot)) * E;
      char *dst = (char *)q + ((t * HQ + h0) * D + R::at(slot)) * E;
#pragma unroll
      for (int h = 0; h < HB; ++h) {
        if (HQ % HB != 0 && h0 + h >= HQ) break;
        float a[8], b[8];
        load8<EL>(src + h * D * E, a);
        load8<EL>(src + (h * D + R::next(slot)) * E, b);
        turn.apply(slot, a, b);
        store8<EL>(dst + h * D * E, a);
        store8<EL>(dst + (h * D + R::next(slot)) * E, b);
      }
    }
    return;
  }
  const bool values = sub >= HK;
  const int h = values ? sub - HK : sub;
  uint8_t *const codes = values ? vc : kc, *const scales = values ? vs : ks;
  constexpr int RPP = 256 / SLOT, NP = (BLOCK + RPP - 1) / RPP; // tokens a pass, passes
  constexpr int PITCH = BLOCK + 8;
  __shared__ uint32_t tops[4];
  __shared__ __attribute__((aligned(16))) uint8_t turned[D * PITCH]; // the values' codes by channel
  const int lane = tid % 64;
  const int64_t mine = t0 + lane;
  bool first = false;
  if (lane < C && mine < T) {
    const int s = seq[mine], p = pos[mine];
    first = inside(s, p) && (mine == 0 || seq[mine - 1] != s || pos[mine - 1] != p - 1 || p % BLOCK == 0);
  }
  for (uint64_t left = __ballot(first); left; left &= left - 1) {
    const int64_t t = t0 + __builtin_ctzll(left);
    const int s = seq[t], p = pos[t], off = p % BLOCK;
    const int blk = table[s * PER + p / BLOCK];
    if (blk < 0 || blk >= NBLK) continue;
    // the block's new rows follow each other
    int most = BLOCK - off;
    if (T - t < most) most = (int)(T - t);
    if (FAR - p < most) most = (int)(FAR - p);
    int n = 0;
#pragma unroll
    for (int k = 0; k < BLOCK; k += 64) {
      const int i = k + lane;
      const uint64_t other = __ballot(!(i < most && seq[t + i] == s && pos[t + i] == p + i));
      if (n == k) n += other ? __builtin_ctzll(other) : 64;
    }
    const int64_t at = ((int64_t)blk * HK + h) * (BLOCK * D);
    const uint32_t old = off > 0 ? scales[(int64_t)blk * HK + h] : 0;
    float f[NP][2][8];
    uint32_t top = 0;
    const int slot = tid % SLOT, r0 = tid / SLOT, c0 = R::at(slot), c1 = c0 + R::next(slot);
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int r = i * RPP + r0;
      if (r0 < RPP && r < n) {
        const char *head = (const char *)qkv + ((t + r) * W + (values ? HQ + HK + h : HQ + h) * D) * E;
        load8<EL>(head + c0 * E, f[i][0]);
        load8<EL>(head + c1 * E, f[i][1]);
        if (!values) {
          R turn;
          turn.load(rot + (int64_t)(p + r) * ROT, slot);
          turn.apply(slot, f[i][0], f[i][1]);
        }
#pragma unroll
        for (int k = 0; k < 16; ++k) top = max_u32(top, f2u(f[i][k / 8][k % 8]) & 0x7FFFFFFFu);
      }
    }
#pragma unroll
    for (int k = 1; k < 64; k *= 2) top = max_u32(top, (uint32_t)__shfl_xor((int)top, k));
    if (lane == 0) tops[tid / 64] = top;
    __syncthreads();
    top = max_u32(max_u32(tops[0], tops[1]), max_u32(tops[2], tops[3]));
    const uint32_t now = max_u32(old, kv_scale_byte<FMT>(top));
    if (tid == 0) scales[(int64_t)blk * HK + h] = (uint8_t)now;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int r = i * RPP + r0;
      if (r0 < RPP && r < n) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const u32x2 w = kv_encode<FMT>(f[i][k], now);
          const int c = k ? c1 : c0;
          if (!values) {
            *reinterpret_cast<u32x2_any *>(codes + at + (off + r) * D + c) = w;
          } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) turned[(c + j) * PITCH + off + r] = (uint8_t)(w[j / 4] >> (8 * (j % 4)));
          }
        }
      }
    }
    if (values) {
      // rows of BLOCK tokens a channel: pieces of eight, whole where all eight are new
      __syncthreads();
      const int b0 = off / 8, b1 = (off + n + 7) / 8;
      for (int i = tid; i < D * (b1 - b0); i += 256) {
        const int d = i / (b1 - b0), b = 8 * (b0 + i % (b1 - b0));
        uint8_t *dst = codes + at + d * BLOCK + b;
        const uint8_t *src = turned + d * PITCH + b;
        if (b >= off && b + 8 <= off + n) {
          *reinterpret_cast<u32x2_any *>(dst) = *reinterpret_cast<const u32x2 *>(src);
        } else {
#pragma unroll
          for (int k = 0; k < 8; ++k)
            if (b + k >= off && b + k < off + n) dst[k] = src[k];
        }
      }
    }
    if ((now != old || now == 255) && off > 0) {
      if (!values) {
        for (int i = tid; i < off * (D / 8); i += 256) {
          u32x2_any *w = reinterpret_cast<u32x2_any *>(codes + at + 8 * i);
          *w = kv_rescale<FMT>(*w, old, now);
        }
      } else {
        const int pieces = (off + 7) / 8;
        for (int i = tid; i < D * pieces; i += 256) {
          const int d = i / pieces, b = 8 * (i % pieces);
          uint8_t *dst = codes + at + d * BLOCK + b;
          if (b + 8 <= off) {
            u32x2_any *w = reinterpret_cast<u32x2_any *>(dst);
            *w = kv_rescale<FMT>(*w, old, now);
          } else {
            // (the piece that the new tokens begin in: theirs are being written)
#pragma unroll
            for (int k = 0; k < 8; ++k)
              if (b + k < off) dst[k] = (uint8_t)kv_rescale<FMT>(u32x2{dst[k], 0}, old, now).x;
          }
        }
      }
    }
    __syncthreads(); // (tops and turned are written again)
  }
}

} // namespace hf
