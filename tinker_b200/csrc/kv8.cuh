// The 8-bit KV cache: its block format, the quantiser of one block, and the register fragments that the
// attention kernels read. Shared by the append kernel (kv8_append.cu) and the attention (kv8_attention.cu).
//
// Format. A sequence's keys and values of one kv head are kept in blocks of 32 tokens. With a = the largest
// magnitude of the block's keys (values), not less than 2^-60, and M = 448 (e4m3) or 127 (int8):
//     scale = a / M,   code = rn(x * (M * (1 / a)))       (fp32, ties to even)
// so |code| <= M and code * scale is within half a code step of x. A block that holds a NaN or an infinity gets
// the scale NaN and codes 0: every result that reads it is NaN, none is silently wrong. The block that is still
// open (pos / 32) keeps its rows in 16 bits in `tail`; a block is quantised once, when its last row arrives, so
// no code is ever rounded twice and the contents do not depend on how the tokens were split into calls.
//
// Layout. The codes of a block are stored in the order in which a warp's m16n8k16 products take them, so that
// one 16-byte load per lane, fully coalesced, is one operand fragment:
//   keys   [j = 4][h = D/64][lane = 4n + q][16]: token 8(n/2) + 2j + n%2, columns 64h + 16q .. + 15
//   values [m = D/16][lane = 4r + q][e = 2][8]:  column 16m + 8e + r, tokens 8q .. 8q + 7
// In Q K^T the contraction order is free, so a lane takes 16 neighbouring columns for four steps of k; the
// columns of n-tile j are the tokens 8q + 2j + {0, 1} of lane q, so the probabilities leave the accumulators as
// the A operand of P V with its tokens 8q .. 8q + 7 in the lane that holds the same tokens of V.
#pragma once

#include <math.h>

#include "tk_common.cuh"

namespace tk {
namespace kv8 {

constexpr int BLOCK = 32;

template <int FMT> struct Code;
template <> struct Code<TK_KV8_E4M3> {
  static constexpr float LIMIT = 448.f;
};
template <> struct Code<TK_KV8_INT8> {
  static constexpr float LIMIT = 127.f;
};

__device__ __forceinline__ uint32_t h2_u32(__half2 v) { return *reinterpret_cast<const uint32_t*>(&v); }
__device__ __forceinline__ __half2 u32_h2(uint32_t v) { return *reinterpret_cast<const __half2*>(&v); }

// Codes of four values, lowest byte first. int8: 1.5 * 2^23 + v has v, rounded to even, in its low byte, in two's
// complement (a conversion runs at a quarter of the rate: 16 x 4001 rows of 8 heads of 128 took 85.5 us, now 75.2).
template <int FMT>
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
  if constexpr (FMT == TK_KV8_E4M3) {
    uint16_t lo, hi;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
    return static_cast<uint32_t>(lo) | (static_cast<uint32_t>(hi) << 16);
  } else {
    constexpr float MAGIC = 12582912.f;
    const uint32_t lo = __byte_perm(__float_as_uint(__fadd_rn(a, MAGIC)), __float_as_uint(__fadd_rn(b, MAGIC)), 0x0040);
    const uint32_t hi = __byte_perm(__float_as_uint(__fadd_rn(c, MAGIC)), __float_as_uint(__fadd_rn(d, MAGIC)), 0x0040);
    return __byte_perm(lo, hi, 0x5410);
  }
}

// Four codes as two f16 pairs; both types are exact in f16. int8: 0x64xx is 1024 + xx, so the byte with its sign
// bit flipped gives 1024 + (v + 128), and one packed subtraction leaves v.
template <int FMT>
__device__ __forceinline__ void decode4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (FMT == TK_KV8_E4M3) {
    asm("{\n\t.reg .b16 a, b;\n\t"
        "mov.b32 {a, b}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, a;\n\t"
        "cvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(w));
  } else {
    const uint32_t u = w ^ 0x80808080u;
    const __half2 off = __half2half2(__ushort_as_half(0x6480));  // 1152
    lo = h2_u32(__hsub2(u32_h2(__byte_perm(u, 0x64646464u, 0x4140)), off));
    hi = h2_u32(__hsub2(u32_h2(__byte_perm(u, 0x64646464u, 0x4342)), off));
  }
}

// The least pattern of a magnitude that is infinite or NaN.
template <int DT>
__device__ __forceinline__ constexpr uint32_t not_finite_bits() {
  return DT == TK_F16 ? 0x7c00u : 0x7f80u;
}

// Scale of a block from the 16-bit pattern of its largest magnitude; `inv` is what its values are multiplied by.
template <int DT, int FMT>
__device__ __forceinline__ float block_scale(uint32_t amax_bits, float& inv) {
  const bool fine = amax_bits < not_finite_bits<DT>();
  const unsigned short b = static_cast<unsigned short>(amax_bits);
  float a;
  if constexpr (DT == TK_F16) a = __half2float(__ushort_as_half(b));
  else a = __uint_as_float(static_cast<uint32_t>(b) << 16);
  a = fmaxf(a, 0x1p-60f);
  inv = fine ? __fmul_rn(__fdiv_rn(1.f, a), Code<FMT>::LIMIT) : 0.f;
  return fine ? __fdiv_rn(a, Code<FMT>::LIMIT) : __uint_as_float(0x7fc00000u);
}

// The power of two, at most 2^60, that brings `amax` (fp32 bits of a magnitude) to [2^14, 2^15); 1 if it is not finite.
// (A tile of zeros has the inverse of the factor as its scale, and sums of that have to stay finite.)
__device__ __forceinline__ float to_f16_range(uint32_t amax_bits) {
  const int e = static_cast<int>(amax_bits >> 23);
  if (e >= 255) return 1.f;
  return __uint_as_float(static_cast<uint32_t>(min(187, 268 - e)) << 23);
}

// The power of two that 16-bit values are multiplied by before they are operands in f16; from the 16-bit pattern of their
// largest magnitude. It belongs to the weights' exponent as a block's scale does, so it has to bring the tile near the
// codes' magnitudes: with f16 values of 0.05 taken as they are, a dominant token of this tile left the weights of encoded
// blocks 2^-13 lower than its own, below what f16 holds. f16 goes up only, which is exact, and by 2^15 at most, so that one
// packed product does it.
template <int DT>
__device__ __forceinline__ float value_factor(uint32_t amax_bits) {
  if constexpr (DT == TK_F16) {
    const float a = __half2float(__ushort_as_half(static_cast<unsigned short>(amax_bits)));
    return fminf(fmaxf(to_f16_range(__float_as_uint(a)), 1.f), 32768.f);
  } else {
    return to_f16_range(amax_bits << 16);
  }
}

template <int DT>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
  return Dt<DT>::unpack(*reinterpret_cast<const typename Dt<DT>::T2*>(&w));
}
template <int DT>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  const typename Dt<DT>::T2 h = Dt<DT>::pack(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// value * inv with a zero for everything in a block that is not finite (0 * inf would be NaN).
template <int FMT>
__device__ __forceinline__ uint32_t encode_words(float2 a, float2 b, float inv) {
  if (inv == 0.f) return 0u;
  return encode4<FMT>(__fmul_rn(a.x, inv), __fmul_rn(a.y, inv), __fmul_rn(b.x, inv), __fmul_rn(b.y, inv));
}

// Largest magnitude of packed 16-bit pairs, as bit patterns (they order like the magnitudes, NaN above inf).
__device__ __forceinline__ uint32_t amax2(uint32_t m, uint32_t w) { return __vmaxu2(m, w & 0x7fff7fffu); }
__device__ __forceinline__ uint32_t amax2_warp(uint32_t m) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, o));
  return max(m & 0xffffu, m >> 16);
}

// Whether a 16-byte chunk holds a NaN or an infinity.
template <int DT>
__device__ __forceinline__ bool not_finite(uint4 x) {
  const uint32_t m = amax2(amax2(amax2(amax2(0u, x.x), x.y), x.z), x.w);
  return max(m & 0xffffu, m >> 16) >= not_finite_bits<DT>();
}

// A warp's 16-bit tile in shared memory: 32 rows of D elements in 16-byte chunks, chunk c of row t at c ^ swz(t),
// which keeps both the column fragments (rows 8a + e) and the row fragments free of bank conflicts.
__device__ __forceinline__ int swz(int t) { return (t & 1) | (((t >> 3) & 3) << 1); }
template <int D>
__device__ __forceinline__ uint32_t tile_off(int t, int c) {
  return static_cast<uint32_t>(t * (2 * D) + ((c ^ swz(t)) << 4));
}

__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

// Columns 8n .. 8n + 7 of a 16-bit tile: lane 4r + q gets the pairs (8q + 2u, 8q + 2u + 1), u = 0..3, of column
// 8n + r.
template <int D>
__device__ __forceinline__ void load_column_tokens(uint32_t tile, int n, int lane, uint32_t (&r)[4]) {
  const int t = 8 * ((lane & 7) >> 1) + 2 * (lane >> 3) + (lane & 1);
  ldmatrix_x4_trans(tile + tile_off<D>(t, n), r);
}

// Rotate 16 neighbouring columns (8 interleaved pairs, the angles of table columns i0 .. i0 + 7) of one row in
// place, every product and sum rounded on its own, the results rounded to DT.
template <int DT>
__device__ __forceinline__ void rope_chunk(uint4& x, const float* cos_row, const float* sin_row) {
  const float4 c = __ldg(reinterpret_cast<const float4*>(cos_row)), s = __ldg(reinterpret_cast<const float4*>(sin_row));
  const float cc[4] = {c.x, c.y, c.z, c.w}, ss[4] = {s.x, s.y, s.z, s.w};
  uint32_t* w = reinterpret_cast<uint32_t*>(&x);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = unpack2<DT>(w[i]);
    w[i] = pack2<DT>(__fsub_rn(__fmul_rn(f.x, cc[i]), __fmul_rn(f.y, ss[i])),
                     __fadd_rn(__fmul_rn(f.x, ss[i]), __fmul_rn(f.y, cc[i])));
  }
}

// Quantise a block of keys: `piece(token, c)` loads 16-byte chunk c of a token's row, `finish(x, token, c)` completes it
// when all loads are on their way. One warp; returns the scale.
template <int DT, int FMT, int D, typename F, typename G>
__device__ __forceinline__ float encode_keys(uint8_t* block, int lane, F piece, G finish) {
  constexpr int H = D / 64;
  const int n = lane >> 2, q = lane & 3;
  uint4 x[4][H][2];
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int h = 0; h < H; ++h)
#pragma unroll
      for (int e = 0; e < 2; ++e) x[j][h][e] = piece(8 * (n >> 1) + 2 * j + (n & 1), 8 * h + 2 * q + e);
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int h = 0; h < H; ++h)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        finish(x[j][h][e], 8 * (n >> 1) + 2 * j + (n & 1), 8 * h + 2 * q + e);
        m = amax2(amax2(amax2(amax2(m, x[j][h][e].x), x[j][h][e].y), x[j][h][e].z), x[j][h][e].w);
      }
  float inv;
  const float scale = block_scale<DT, FMT>(amax2_warp(m), inv);
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int h = 0; h < H; ++h) {
      uint4 y;
      y.x = encode_words<FMT>(unpack2<DT>(x[j][h][0].x), unpack2<DT>(x[j][h][0].y), inv);
      y.y = encode_words<FMT>(unpack2<DT>(x[j][h][0].z), unpack2<DT>(x[j][h][0].w), inv);
      y.z = encode_words<FMT>(unpack2<DT>(x[j][h][1].x), unpack2<DT>(x[j][h][1].y), inv);
      y.w = encode_words<FMT>(unpack2<DT>(x[j][h][1].z), unpack2<DT>(x[j][h][1].w), inv);
      *reinterpret_cast<uint4*>(block + ((j * H + h) * 32 + lane) * 16) = y;
    }
  return scale;
}

// Quantise a block of values from a complete 16-bit tile in shared memory. One warp; returns the scale.
template <int DT, int FMT, int D>
__device__ __forceinline__ float encode_values(uint8_t* block, int lane, uint32_t tile, uint32_t amax_bits) {
  float inv;
  const float scale = block_scale<DT, FMT>(amax_bits, inv);
#pragma unroll
  for (int m = 0; m < D / 16; ++m) {
    uint32_t a[4], b[4];
    load_column_tokens<D>(tile, 2 * m, lane, a);
    load_column_tokens<D>(tile, 2 * m + 1, lane, b);
    uint4 y;
    y.x = encode_words<FMT>(unpack2<DT>(a[0]), unpack2<DT>(a[1]), inv);
    y.y = encode_words<FMT>(unpack2<DT>(a[2]), unpack2<DT>(a[3]), inv);
    y.z = encode_words<FMT>(unpack2<DT>(b[0]), unpack2<DT>(b[1]), inv);
    y.w = encode_words<FMT>(unpack2<DT>(b[2]), unpack2<DT>(b[3]), inv);
    *reinterpret_cast<uint4*>(block + (m * 32 + lane) * 16) = y;
  }
  return scale;
}

}  // namespace kv8
}  // namespace tk
