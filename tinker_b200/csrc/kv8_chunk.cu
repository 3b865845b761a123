// Attention of many new tokens (a chunk of a prompt) against an 8-bit KV cache, on tcgen05 tensor cores. What it
// computes is described in kv8_attention.cu; this is the form for enough query rows that the products are the work
// (4 D Hq S len flops against 2 D Hkv len bytes of codes), with the position known on the host.
//
// 1. kv8_expand_kernel lays the operands out for the tensor cores, once for all query tiles, in f16:
//      q   [sequence, kv head, token * groups + head, D], rotated in fp32, times a power of two that brings the row to
//          [2^14, 2^15), with the row's factor (scale log2 e / that power) beside it
//      k   [sequence, kv head, position, D], v [sequence, kv head, D, position]: codes as they are, rows of the open
//          block and of the call times a power of two for each 32 tokens (f16 keys as they are), zeros to the end of the
//          last 128-key tile; with (scale_k, log2 scale_v, 1 / scale_v) of each 32 tokens beside them.
//    Codes and scaled rows are exact in f16; q is rounded to 11 bits, 2^-12 of each of a score's terms. Under a bf16
//    result (2^-9) that does not show; for an fp16 result it would double the error (4.3e-4 instead of 2.1e-4 relative
//    on 8-bit keys with strong channels), so there the remainder q - f16(q) is laid out too and has a product of its
//    own. The weights are rounded to f16 once, 2^-12 of a weight, in both. They go up to 2^15, so one is lost to f16's
//    smallest number, 2^-24, only 2^36 below the largest.
// 2. kv8_chunk_kernel: a CTA takes two 128-row query tiles (fp16: one and its remainder) of one (sequence, kv head) -
//    rows of all the heads that share it, so a key tile is loaded once for them - and a range of the 128-key tiles. One
//    thread feeds a ring of K and V tiles by TMA, one issues S = Q K^T and O += P V as tcgen05.mma with S and O in
//    tensor memory, two warpgroups (thread = query row) turn S into weights: x = s * (factor * scale_k) + log2 scale_v
//    for each 32 keys, w = 2^(x - m + HEADROOM), l += sum w / scale_v, P = f16(w) to shared memory. m moves only when a
//    tile raises it by more than 2^4. The scales cost nothing per score: the FMA of the softmax takes them as its factor
//    and addend.
// 3. With the key axis split (few query tiles), kv8_join_kernel merges the parts in their order.
// Bound by the softmax's latency: products and exponentials take some 2000 cycles each for a pair of tiles at D = 128, a
// step some 6000 (8 softmax warps on 4 schedulers, 29 % of the issue slots filled). 512 tokens of 32 heads of 128 at
// 7001: 124 us in all, 100 of them here (128 CTAs), the rest the expansion, the join and the append; 154 us for fp16,
// whose second warpgroup has no tile. kv8_attention.cu takes 739 us.
#include <algorithm>
#include <cmath>
#include <string>
#include <type_traits>

#include "kv8.cuh"
#include "kv8_host.h"
#include "tk_host.h"

namespace tk {
namespace kv8 {
namespace chunk {

constexpr int BQ = 128;
constexpr int BKV = 128;
constexpr int SOFTMAX_WARPS = 8;
constexpr int TMA_WARP = 8, MMA_WARP = 9;
constexpr int THREADS = 12 * 32;  // the last two warps only make up a warpgroup
constexpr float LAZY_RESCALE_LOG2 = 4.f;
constexpr float HEADROOM = 11.f;  // log2 of a weight at the maximum; with what that may lag behind, 15: the top of f16

template <int D>
struct Smem {
  static constexpr int Q_BYTES = BQ * D * 2;
  static constexpr int T_BYTES = BKV * D * 2;
  static constexpr int STAGES = D == 64 ? 4 : 3;
  static constexpr int P_BYTES = BQ * BKV * 2;
  static constexpr int RING_OFF = 2 * Q_BYTES;
  static constexpr int P_OFF = RING_OFF + STAGES * T_BYTES;
  static constexpr int BAR_OFF = P_OFF + 2 * P_BYTES;
  static constexpr int NUM_BARS = 20;
  static constexpr int TOTAL = 1024 + BAR_OFF + NUM_BARS * 8 + 16;
  // S_a: columns 0-127, S_b: 128-255, O_a: 256.., O_b: 256 + D..
  static constexpr uint32_t TMEM_COLS = 512;
};

enum : int { B_Q_FULL = 0, B_FULL = 1, B_EMPTY = 5, B_S_FULL = 9, B_P_FULL = 11, B_PV_DONE = 13, B_S_FREE = 15 };

struct Params {
  // inputs of the expansion
  const void* q;
  int64_t qs;
  const void* k;
  int64_t ks;
  const void* v;
  int64_t vs;
  const uint8_t* kc;
  const uint8_t* vc;
  const float* scales;
  const void* tail;
  int num_blocks;
  const float* cos_t;
  const float* sin_t;
  int start, seq, num_kv_heads, groups, rows, batch;
  float scale_log2;
  // what it writes
  __half* qx;     // [batch, num_kv_heads, rows, D], then the remainders in the same layout
  float* qf;      // [batch, num_kv_heads, rows]
  __half* kx;     // [batch, num_kv_heads, keys, D]
  __half* vx;     // [batch, num_kv_heads, D, keys]
  float4* sx;     // [batch, num_kv_heads, keys / 32]: scale_k, log2 scale_v, 1 / scale_v, tokens to be NaN (bits)
  int keys;       // start + seq, rounded up to whole key tiles
  int q_ctas;     // expansion CTAs that lay out q
  // the attention
  void* out;
  int64_t os;
  int n_qtiles, splits;
  float2* part_ml;  // [batch, num_kv_heads, rows, splits]
  float* part_o;    // [batch, num_kv_heads, rows, splits, D]
};

// fp16: a query tile's remainder takes the place of the second tile
template <int DT> constexpr bool REMAINDER = DT == TK_F16;
// The values' scales may lie so far apart that a weight is below fp32's range and its share of the denominator, weight /
// scale_v, is not: see kv8_attention.cu. Here the shares of 32 keys whose scale is 2^SPREAD below the greatest are
// exponentials of their own, in a loop that only CTAs with values of 2^20 and more take (a branch in the one loop cost
// 3 %).
template <int DT> constexpr bool WIDE = DT == TK_BF16;
constexpr float SPREAD = 80.f, LSV_LOW = -69.f;  // the least log2 scale_v: 2^-60 / 448

constexpr int EXPAND_WARPS = 8;  // 4 for keys, 4 for values

template <int DT, int FMT, int D>
__global__ void __launch_bounds__(EXPAND_WARPS * 32, 2) kv8_expand_kernel(const Params p) {
  extern __shared__ __align__(128) uint8_t smem[];
  using T = typename Dt<DT>::T;
  constexpr int C16 = D / 8;
  constexpr int H = D / 64;
  pdl_wait();
  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int kvh = blockIdx.y, b = blockIdx.z;
  const int64_t bh = static_cast<int64_t>(b) * p.num_kv_heads + kvh;

  if (static_cast<int>(blockIdx.x) < p.q_ctas) {  // D / 16 lanes for a query row, 16 columns each
    constexpr int LANES = D / 16, ROWS_WARP = 32 / LANES;
    const int row = (blockIdx.x * EXPAND_WARPS + warp) * ROWS_WARP + lane / LANES, part = lane % LANES;
    const bool valid = row < p.rows;
    const int s = valid ? row / p.groups : 0, head = kvh * p.groups + (valid ? row - s * p.groups : 0);
    const T* src = reinterpret_cast<const T*>(p.q) + (static_cast<int64_t>(b) * p.seq + s) * p.qs +
                   static_cast<int64_t>(head) * D + part * 16;
    float f[16];
    float amax = 0.f;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const uint4 x = __ldcg(reinterpret_cast<const uint4*>(src) + e);
      const uint32_t w[4] = {x.x, x.y, x.z, x.w};
      float cc[4] = {1.f, 1.f, 1.f, 1.f}, ss[4] = {0.f, 0.f, 0.f, 0.f};
      if (p.cos_t) {
        const int64_t ang = (static_cast<int64_t>(p.start) + s) * (D / 2) + part * 8 + e * 4;
        const float4 a = __ldg(reinterpret_cast<const float4*>(p.cos_t + ang));
        const float4 d = __ldg(reinterpret_cast<const float4*>(p.sin_t + ang));
        cc[0] = a.x, cc[1] = a.y, cc[2] = a.z, cc[3] = a.w;
        ss[0] = d.x, ss[1] = d.y, ss[2] = d.z, ss[3] = d.w;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 v = unpack2<DT>(w[i]);
        f[8 * e + 2 * i] = v.x * cc[i] - v.y * ss[i];
        f[8 * e + 2 * i + 1] = v.x * ss[i] + v.y * cc[i];
        amax = fmaxf(amax, fmaxf(fabsf(f[8 * e + 2 * i]), fabsf(f[8 * e + 2 * i + 1])));
      }
    }
#pragma unroll
    for (int o = 1; o < LANES; o <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    const float up = to_f16_range(__float_as_uint(amax));
    uint32_t y[8], z[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const __half2 hi = __floats2half2_rn(f[2 * i] * up, f[2 * i + 1] * up);
      const float2 g = __half22float2(hi);
      y[i] = h2_u32(hi);
      z[i] = h2_u32(__floats2half2_rn(f[2 * i] * up - g.x, f[2 * i + 1] * up - g.y));
    }
    if (valid) {
      if constexpr (REMAINDER<DT>) {
        const int64_t all = static_cast<int64_t>(p.batch) * p.num_kv_heads;
        uint4* lo = reinterpret_cast<uint4*>(p.qx + ((all + bh) * p.rows + row) * D + part * 16);
        lo[0] = make_uint4(z[0], z[1], z[2], z[3]);
        lo[1] = make_uint4(z[4], z[5], z[6], z[7]);
      }
      uint4* dst = reinterpret_cast<uint4*>(p.qx + (bh * p.rows + row) * D + part * 16);
      dst[0] = make_uint4(y[0], y[1], y[2], y[3]);
      dst[1] = make_uint4(y[4], y[5], y[6], y[7]);
      if (part == 0) p.qf[bh * p.rows + row] = p.scale_log2 / up;
    }
    return;
  }

  const int block = (blockIdx.x - p.q_ctas) * (EXPAND_WARPS / 2) + warp % (EXPAND_WARPS / 2);
  const bool values = warp >= EXPAND_WARPS / 2;
  if (block >= p.keys / BLOCK) return;
  const int n8 = p.start / BLOCK, open = p.start % BLOCK;
  const int r = lane >> 2, q = lane & 3;
  __half* kx = p.kx + (bh * p.keys + static_cast<int64_t>(block) * BLOCK) * D;
  __half* vx = p.vx + bh * D * p.keys + static_cast<int64_t>(block) * BLOCK;
  float* sx = reinterpret_cast<float*>(p.sx + bh * (p.keys / BLOCK) + block);
  auto decode16 = [](uint4 x, uint4& lo, uint4& hi) {
    decode4<FMT>(x.x, lo.x, lo.y);
    decode4<FMT>(x.y, lo.z, lo.w);
    decode4<FMT>(x.z, hi.x, hi.y);
    decode4<FMT>(x.w, hi.z, hi.w);
  };
  if (block < n8) {
    const int64_t at = (bh * p.num_blocks + block) * (BLOCK * D);
    if (!values) {
      uint4 x[4 * H];
#pragma unroll
      for (int i = 0; i < 4 * H; ++i) x[i] = __ldcg(reinterpret_cast<const uint4*>(p.kc + at) + i * 32 + lane);
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int h = 0; h < H; ++h) {
          uint4 lo, hi;
          decode16(x[j * H + h], lo, hi);
          uint4* dst = reinterpret_cast<uint4*>(kx + (8 * (r >> 1) + 2 * j + (r & 1)) * D + 64 * h + 16 * q);
          dst[0] = lo;
          dst[1] = hi;
        }
      if (lane == 0) {
        const float2 sc = __ldcg(reinterpret_cast<const float2*>(p.scales) + bh * p.num_blocks + block);
        *reinterpret_cast<float4*>(sx) = make_float4(sc.x, __log2f(sc.y), 1.f / sc.y, 0.f);
      }
    } else {
      uint4 x[D / 16];
#pragma unroll
      for (int m = 0; m < D / 16; ++m) x[m] = __ldcg(reinterpret_cast<const uint4*>(p.vc + at) + m * 32 + lane);
#pragma unroll
      for (int m = 0; m < D / 16; ++m) {
        uint4 lo, hi;
        decode16(x[m], lo, hi);
        *reinterpret_cast<uint4*>(vx + static_cast<int64_t>(16 * m + r) * p.keys + 8 * q) = lo;
        *reinterpret_cast<uint4*>(vx + static_cast<int64_t>(16 * m + 8 + r) * p.keys + 8 * q) = hi;
      }
    }
    return;
  }
  // rows in 16 bits: the open block from the tail, the call's own, zeros behind them
  const T* tail = reinterpret_cast<const T*>(p.tail) + (bh * 2 + (values ? 1 : 0)) * BLOCK * D;
  const T* in = reinterpret_cast<const T*>(values ? p.v : p.k) + static_cast<int64_t>(kvh) * D;
  const int64_t stride = values ? p.vs : p.ks;
  const int row0 = (block - n8) * BLOCK - open;  // the call's row of the block's first token
  uint8_t* tile = smem + warp * (BLOCK * D * 2);
  uint32_t m = 0;
  uint4 x[C16];
#pragma unroll
  for (int i = 0; i < C16; ++i) {  // all loads in flight, then the rotations
    const int idx = lane + 32 * i, t = idx / C16, c = idx % C16, s = row0 + t;
    const T* src = s < 0 ? tail + t * D : in + (static_cast<int64_t>(b) * p.seq + min(s, p.seq - 1)) * stride;
    x[i] = s < p.seq ? __ldcg(reinterpret_cast<const uint4*>(src) + c) : make_uint4(0, 0, 0, 0);
  }
#pragma unroll
  for (int i = 0; i < C16; ++i) {
    const int idx = lane + 32 * i, t = idx / C16, c = idx % C16, s = row0 + t;
    if (!values && p.cos_t && s >= 0 && s < p.seq) {
      const int64_t ang = (static_cast<int64_t>(p.start) + s) * (D / 2) + c * 4;
      rope_chunk<DT>(x[i], p.cos_t + ang, p.sin_t + ang);
    }
    m = amax2(amax2(amax2(amax2(m, x[i].x), x[i].y), x[i].z), x[i].w);
    *reinterpret_cast<uint4*>(tile + tile_off<D>(t, c)) = x[i];
  }
  uint32_t amax = amax2_warp(m), bad = 0;
  __syncwarp();
  if (amax >= not_finite_bits<DT>()) {
    // A token that is not finite makes the rows that see it NaN, by its scores, and must not reach the others, neither as
    // 0 * NaN nor by the range of its 32 tokens: a key becomes NaN throughout, values become 0 and their bit does the same.
#pragma unroll 1
    for (int idx = lane; idx < BLOCK * C16; idx += 32)
      if (not_finite<DT>(*reinterpret_cast<const uint4*>(tile + tile_off<D>(idx / C16, idx % C16))))
        bad |= 1u << (idx / C16);
    bad = __reduce_or_sync(0xffffffffu, bad);
    const uint32_t w = values ? 0u : 0x7fff7fffu;
    m = 0;
#pragma unroll 1
    for (int idx = lane; idx < BLOCK * C16; idx += 32) {
      uint4* y = reinterpret_cast<uint4*>(tile + tile_off<D>(idx / C16, idx % C16));
      if (bad >> (idx / C16) & 1) *y = make_uint4(w, w, w, w);
      else m = amax2(amax2(amax2(amax2(m, y->x), y->y), y->z), y->w);
    }
    amax = amax2_warp(m);
    __syncwarp();
  }
  const float up = values ? value_factor<DT>(amax) : DT == TK_F16 ? 1.f : to_f16_range(amax << 16);
  auto to_half = [&](uint32_t w) -> uint32_t {
    const float2 v = unpack2<DT>(w);
    return h2_u32(__floats2half2_rn(v.x * up, v.y * up));
  };
  if (!values) {
#pragma unroll 4
    for (int i = 0; i < C16; ++i) {
      const int idx = lane + 32 * i, t = idx / C16, c = idx % C16;
      const uint4 x = *reinterpret_cast<const uint4*>(tile + tile_off<D>(t, c));
      *(reinterpret_cast<uint4*>(kx + t * D) + c) = make_uint4(to_half(x.x), to_half(x.y), to_half(x.z), to_half(x.w));
    }
    if (lane == 0) sx[0] = 1.f / up;
  } else {
#pragma unroll 4
    for (int n = 0; n < D / 8; ++n) {
      uint32_t x[4];
      load_column_tokens<D>(smem_u32(tile), n, lane, x);
      *reinterpret_cast<uint4*>(vx + static_cast<int64_t>(8 * n + r) * p.keys + 8 * q) =
          make_uint4(to_half(x[0]), to_half(x[1]), to_half(x[2]), to_half(x[3]));
    }
    if (lane == 0) sx[1] = -__log2f(up), sx[2] = up, sx[3] = __uint_as_float(bad);
  }
}

template <int DT, int D>
__global__ void __launch_bounds__(THREADS, 1)
    kv8_chunk_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                     const __grid_constant__ CUtensorMap tv, const Params p) {
  using S = Smem<D>;
  using Dx = Dt<DT>;
  constexpr int NS = S::STAGES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* ring = smem + S::RING_OFF;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::BAR_OFF);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + S::NUM_BARS);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  constexpr bool LO = REMAINDER<DT>;
  const int n_pairs = LO ? p.n_qtiles : (p.n_qtiles + 1) >> 1;
  const int pair = n_pairs - 1 - static_cast<int>(blockIdx.z) / p.splits;  // the longest first
  const int split = static_cast<int>(blockIdx.z) % p.splits;
  const int kvh = blockIdx.x, b = blockIdx.y;
  const int64_t bh = static_cast<int64_t>(b) * p.num_kv_heads + kvh;
  // key tiles that query tile x sees (0 if there is none), and this CTA's part of them
  auto first_row = [&](int x) { return (LO ? pair : 2 * pair + x) * BQ; };
  auto tiles_of = [&](int x) {
    const int first = first_row(x);
    if (first >= p.rows || (LO && x == 1)) return 0;
    return (p.start + (min(p.rows, first + BQ) - 1) / p.groups) / BKV + 1;
  };
  const int all_a = tiles_of(0), all_b = tiles_of(1), all = max(all_a, all_b);
  const int lo = static_cast<int>(static_cast<int64_t>(all) * split / p.splits);
  const int hi = static_cast<int>(static_cast<int64_t>(all) * (split + 1) / p.splits);
  const int n_a = max(0, min(hi, all_a) - lo), n_b = max(0, min(hi, all_b) - lo);
  const int n_kv = max(n_a, n_b);

  if (tid == 0) {
    mbar_init(bars + B_Q_FULL, 1);
    for (int i = 0; i < NS; ++i) {
      mbar_init(bars + B_FULL + i, 1);
      mbar_init(bars + B_EMPTY + i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(bars + B_S_FULL + i, 1);
      mbar_init(bars + B_P_FULL + i, 128);
      mbar_init(bars + B_PV_DONE + i, 1);
      mbar_init(bars + B_S_FREE + i, 128);
    }
    fence_mbar_init();
  }
  if (warp == MMA_WARP) {
    tmem_alloc(tmem_slot, S::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == TMA_WARP) {
    if (lane == 0) {
      pdl_launch_dependents();
      prefetch_tmap(&tq);
      prefetch_tmap(&tk);
      prefetch_tmap(&tv);
      pdl_wait();  // the operands are written by the expansion
      const int n_q = n_kv == 0 ? 0 : LO || all_b > 0 ? 2 : 1;  // no copy that nobody waits for
      const int bhi = static_cast<int>(bh), all_bh = p.batch * p.num_kv_heads;
      if (n_q > 0) mbar_arrive_expect_tx(bars + B_Q_FULL, n_q * S::Q_BYTES);
      for (int t = 0; t < n_q; ++t)
#pragma unroll
        for (int cb = 0; cb < D / 64; ++cb)
          tma_load_3d(smem + t * S::Q_BYTES + cb * 128 * 128, &tq, bars + B_Q_FULL, cb * 64, first_row(t),
                      bhi + (LO ? t * all_bh : 0));
      for (int i = 0; i < 2 * n_kv; ++i) {
        const int slot = i % NS;
        if (i >= NS && !mbar_wait(bars + B_EMPTY + slot, ((i / NS) - 1) & 1)) break;
        uint8_t* dst = ring + slot * S::T_BYTES;
        const int key = (lo + (i >> 1)) * BKV;
        mbar_arrive_expect_tx(bars + B_FULL + slot, S::T_BYTES);
        if (i & 1) {  // V: two halves of 64 keys, D rows each
#pragma unroll
          for (int kb = 0; kb < 2; ++kb)
            tma_load_3d(dst + kb * D * 128, &tv, bars + B_FULL + slot, key + kb * 64, 0, bhi);
        } else {
#pragma unroll
          for (int cb = 0; cb < D / 64; ++cb)
            tma_load_3d(dst + cb * 128 * 128, &tk, bars + B_FULL + slot, cb * 64, key, bhi);
        }
      }
    }
  } else if (warp == MMA_WARP) {
    if (lane == 0) {
      constexpr uint32_t idesc_s = make_idesc_f16(Dt<TK_F16>::umma_fmt, BQ, BKV, 0, 0);
      constexpr uint32_t idesc_o = make_idesc_f16(Dt<TK_F16>::umma_fmt, BQ, D, 0, 0);
      auto issue_s = [&](uint64_t q_desc, uint64_t k_desc, uint32_t t_s) {
#pragma unroll
        for (int lo = 0; lo <= (LO ? 1 : 0); ++lo)
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const uint64_t off16 = static_cast<uint64_t>(((kk >> 2) * (128 * 128) + (kk & 3) * 32) >> 4);
            umma_f16_ss(t_s, q_desc + static_cast<uint64_t>(lo * S::Q_BYTES / 16) + off16, k_desc + off16, idesc_s,
                        lo + kk != 0);
          }
      };
      auto issue_pv = [&](uint64_t p_desc, uint64_t v_desc, uint32_t t_o, bool acc) {
#pragma unroll
        for (int kk = 0; kk < BKV / 16; ++kk) {
          const uint64_t poff = static_cast<uint64_t>(((kk >> 2) * (128 * 128) + (kk & 3) * 32) >> 4);
          const uint64_t voff = static_cast<uint64_t>(((kk >> 2) * (D * 128) + (kk & 3) * 32) >> 4);
          umma_f16_ss(t_o, p_desc + poff, v_desc + voff, idesc_o, (acc || kk > 0) ? 1u : 0u);
        }
      };
      auto full = [&](int i) { return mbar_wait(bars + B_FULL + i % NS, (i / NS) & 1); };
      auto desc = [&](int i) { return make_sw128_desc(smem_u32(ring + (i % NS) * S::T_BYTES), 0, 1024); };
      const uint64_t qd_a = make_sw128_desc(smem_u32(smem), 0, 1024);
      const uint64_t qd_b = make_sw128_desc(smem_u32(smem + S::Q_BYTES), 0, 1024);
      const uint64_t pd_a = make_sw128_desc(smem_u32(smem + S::P_OFF), 0, 1024);
      const uint64_t pd_b = make_sw128_desc(smem_u32(smem + S::P_OFF + S::P_BYTES), 0, 1024);
      const uint32_t t_sa = tmem_base, t_sb = tmem_base + 128;
      const uint32_t t_oa = tmem_base + 256, t_ob = tmem_base + 256 + D;
      bool ok = n_kv > 0 && mbar_wait(bars + B_Q_FULL, 0) && full(0);
      if (ok) {
        tc_fence_after();
        if (n_a > 0) {
          issue_s(qd_a, desc(0), t_sa);
          umma_commit(bars + B_S_FULL + 0);
        }
        if (n_b > 0) {
          issue_s(qd_b, desc(0), t_sb);
          umma_commit(bars + B_S_FULL + 1);
        }
        umma_commit(bars + B_EMPTY + 0);
      }
      for (int j = 0; ok && j < n_kv; ++j) {
        const int iv = 2 * j + 1;
        if (j + 1 < n_kv) {  // the next S of a tile as soon as its softmax has read this one
          if (!full(iv + 1)) break;
          if (j + 1 < n_a) {
            if (!mbar_wait(bars + B_S_FREE + 0, j & 1)) break;
            tc_fence_after();
            issue_s(qd_a, desc(iv + 1), t_sa);
            umma_commit(bars + B_S_FULL + 0);
          }
          if (j + 1 < n_b) {
            if (!mbar_wait(bars + B_S_FREE + 1, j & 1)) break;
            tc_fence_after();
            issue_s(qd_b, desc(iv + 1), t_sb);
            umma_commit(bars + B_S_FULL + 1);
          }
          umma_commit(bars + B_EMPTY + (iv + 1) % NS);
        }
        if (!full(iv)) break;
        if (j < n_a) {
          if (!mbar_wait(bars + B_P_FULL + 0, j & 1)) break;
          tc_fence_after();
          issue_pv(pd_a, desc(iv), t_oa, j > 0);
          umma_commit(bars + B_PV_DONE + 0);
        }
        if (j < n_b) {
          if (!mbar_wait(bars + B_P_FULL + 1, j & 1)) break;
          tc_fence_after();
          issue_pv(pd_b, desc(iv), t_ob, j > 0);
          umma_commit(bars + B_PV_DONE + 1);
        }
        umma_commit(bars + B_EMPTY + iv % NS);
      }
    }
  } else if (warp < SOFTMAX_WARPS) {
    const int x = warp >> 2, r = tid & 127;
    const int row = first_row(x) + r;
    const int n_x = x == 0 ? n_a : n_b;
    const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t t_s = tmem_base + x * 128, t_o = tmem_base + 256 + x * D;
    uint8_t* sp = smem + S::P_OFF + x * S::P_BYTES;
    bool ok = true;
    float m_run = -INFINITY, l_run = 0.f;
    if ((x == 0 ? all_a : all_b) > 0) {
      pdl_wait();  // the factors are written by the expansion
      const bool valid = row < p.rows;
      const float cq = valid ? __ldcg(p.qf + bh * p.rows + row) : 0.f;
      const int qpos = p.start + (valid ? row : p.rows - 1) / p.groups;
      const int rows16 = p.start / BLOCK * BLOCK;  // the first position that is kept in 16 bits; no row's own is below it
      const float4* sx = p.sx + bh * (p.keys / BLOCK) + static_cast<int64_t>(lo) * (BKV / BLOCK);
      auto tiles = [&](auto wide, float top) {  // top: the greatest log2 scale_v of the CTA's keys
        for (int j = 0; ok && j < n_x; ++j) {
          float4 sc[4];  // from L1: one line holds two tiles' and the line after it is on its way
#pragma unroll
          for (int i = 0; i < 4; ++i) sc[i] = sx[4 * j + i];
          if (lane == 0 && j + 3 < n_x) prefetch_l1(sx + 4 * (j + 3));
          if (!mbar_wait(bars + B_S_FULL + x, j & 1)) { ok = false; break; }
          tc_fence_after();
          float sv[BKV];
          tmem_load128(t_s + lane_off, sv);
          tc_fence_before();
          mbar_arrive(bars + B_S_FREE + x);
          const int key = (lo + j) * BKV;
          if (key + BKV > rows16) {  // the open block and the call's own tokens: the mask, and tokens that are NaN
#pragma unroll
            for (int c = 0; c < BKV; ++c) {
              if (__float_as_uint(sc[c >> 5].w) >> (c & 31) & 1) sv[c] = __uint_as_float(0x7fc00000u);
              if (key + c > qpos) sv[c] = -INFINITY;
            }
          }
          // the maximum of x: for each 32 keys that of the raw products, times their factor
          float f[4], mx = -INFINITY;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float m2[2] = {sv[32 * i], sv[32 * i + 1]};
#pragma unroll
            for (int c = 2; c < 32; ++c) m2[c & 1] = fmaxf(m2[c & 1], sv[32 * i + c]);
            f[i] = cq * sc[i].x;
            if (f[i] < 1e-30f) f[i] = 1e-30f;  // not 0, which times a masked -inf is NaN
            const float raw = fmaxf(m2[0], m2[1]);
            mx = fmaxf(mx, fmaf(raw, f[i], sc[i].y));
          }
          float m_use = m_run, root = 1.f, alpha = 1.f;
          if (mx > m_run + LAZY_RESCALE_LOG2) {
            m_use = mx;
            if constexpr (WIDE<DT>) root = exp2_approx(0.5f * (m_run - mx));
            alpha = WIDE<DT> ? root * root : exp2_approx(m_run - mx);
          }
          const float base = m_use == -INFINITY ? 0.f : m_use - HEADROOM;  // no key of this row so far
          float rs = 0.f;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if constexpr (decltype(wide)::value) {
              if (sc[i].y < top - SPREAD) {
#pragma unroll
                for (int c = 32 * i; c < 32 * i + 32; ++c) rs += exp2_approx(fmaf(sv[c], f[i], -base));
                sc[i].z = 0.f;
              }
            }
            const uint64_t f2 = pack_f32x2(f[i], f[i]), a2 = pack_f32x2(sc[i].y - base, sc[i].y - base);
            uint64_t s2[2] = {0, 0};
#pragma unroll
            for (int c = 32 * i; c < 32 * i + 32; c += 2) {
              float e0, e1;
              unpack_f32x2(fma_f32x2(pack_f32x2(sv[c], sv[c + 1]), f2, a2), e0, e1);
              sv[c] = exp2_approx(e0);
              sv[c + 1] = exp2_approx(e1);
              s2[(c >> 1) & 1] = add_f32x2(s2[(c >> 1) & 1], pack_f32x2(sv[c], sv[c + 1]));
            }
            float a, c2, d, e;
            unpack_f32x2(s2[0], a, c2);
            unpack_f32x2(s2[1], d, e);
            rs = fmaf((a + c2) + (d + e), sc[i].z, rs);
          }
          l_run = (WIDE<DT> ? l_run * root * root : l_run * alpha) + rs;
          m_run = m_use;
          if (j > 0) {  // P and O are still in use by the P V before
            if (!mbar_wait(bars + B_PV_DONE + x, (j - 1) & 1)) { ok = false; break; }
            tc_fence_after();
          }
#pragma unroll
          for (int c = 0; c < BKV / 8; ++c) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = h2_u32(__floats2half2_rn(sv[c * 8 + 2 * i], sv[c * 8 + 2 * i + 1]));
            *reinterpret_cast<uint4*>(sp + (c >> 3) * (128 * 128) + r * 128 + (((c & 7) ^ (r & 7)) * 16)) =
                make_uint4(w[0], w[1], w[2], w[3]);
          }
          if (j > 0 && __any_sync(0xffffffffu, alpha != 1.0f)) {
#pragma unroll
            for (int c = 0; c < D; c += 32) {
              float o[32];
              tmem_load32(t_o + lane_off + c, o);
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] *= alpha;
              tmem_st32(t_o + lane_off + c, o);
            }
          }
          fence_proxy_async_smem();
          tc_fence_before();
          mbar_arrive(bars + B_P_FULL + x);
        }
      };
      if constexpr (WIDE<DT>) {
        float top = -INFINITY;
        for (int i = lane; i < n_x * (BKV / BLOCK); i += 32) top = fmaxf(top, sx[i].y);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        if (top > LSV_LOW + SPREAD) tiles(std::true_type(), top);
        else tiles(std::false_type(), top);
      } else {
        tiles(std::false_type(), 0.f);
      }
      const int64_t slot = (bh * p.rows + row) * p.splits + split;
      if (ok && n_x > 0) ok = mbar_wait(bars + B_PV_DONE + x, (n_x - 1) & 1);
      if (ok) {
        tc_fence_after();
        const float inv_l = 1.0f / l_run;
        using T = typename Dx::T;
        const int s = valid ? row / p.groups : 0, head = kvh * p.groups + (valid ? row - s * p.groups : 0);
        T* dst = reinterpret_cast<T*>(p.out) + (static_cast<int64_t>(b) * p.seq + s) * p.os + static_cast<int64_t>(head) * D;
        if (p.splits > 1 && valid) p.part_ml[slot] = make_float2(m_run, n_x > 0 ? l_run : 0.f);
        if (n_x > 0) {
#pragma unroll
          for (int c = 0; c < D; c += 32) {
            float o[32];
            tmem_load32(t_o + lane_off + c, o);
            if (!valid) continue;
            if (p.splits > 1) {
#pragma unroll
              for (int i = 0; i < 8; ++i)
                reinterpret_cast<float4*>(p.part_o + slot * D + c)[i] =
                    make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
            } else {
#pragma unroll
              for (int i = 0; i < 4; ++i)
                reinterpret_cast<uint4*>(dst + c)[i] =
                    make_uint4(pack2<DT>(o[8 * i] * inv_l, o[8 * i + 1] * inv_l),
                               pack2<DT>(o[8 * i + 2] * inv_l, o[8 * i + 3] * inv_l),
                               pack2<DT>(o[8 * i + 4] * inv_l, o[8 * i + 5] * inv_l),
                               pack2<DT>(o[8 * i + 6] * inv_l, o[8 * i + 7] * inv_l));
            }
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == MMA_WARP) {
    tc_fence_after();
    tmem_dealloc(tmem_base, S::TMEM_COLS);
  }
}

// The parts of every row, a warp for each.
template <int DT, int D>
__global__ void __launch_bounds__(256) kv8_join_kernel(const Params p) {
  using T = typename Dt<DT>::T;
  constexpr int E = D / 32;
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, row = blockIdx.x * 8 + (threadIdx.x >> 5);
  if (row >= p.rows) return;
  const int64_t bh = static_cast<int64_t>(blockIdx.z) * p.num_kv_heads + blockIdx.y;
  const int64_t slot = (bh * p.rows + row) * p.splits;
  float M = -INFINITY, L = 0.f, acc[E] = {};
  const float* from = p.part_o + slot * D + lane * E;
  for (int i = 0; i < p.splits; ++i) {
    const float2 ml = __ldcg(p.part_ml + slot + i);
    if (ml.x == -INFINITY && ml.y == 0.f) continue;  // no key of this row in the part
    const float mn = fmaxf(M, ml.x);
    const float ra = exp2_approx(0.5f * (M - mn)), re = exp2_approx(0.5f * (ml.x - mn)), a = ra * ra, e = re * re;
    L = L * ra * ra + ml.y * re * re;
    if constexpr (E == 4) {
      const float4 o = __ldcg(reinterpret_cast<const float4*>(from + static_cast<int64_t>(i) * D));
      acc[0] = acc[0] * a + o.x * e;
      acc[1] = acc[1] * a + o.y * e;
      acc[2] = acc[2] * a + o.z * e;
      acc[3] = acc[3] * a + o.w * e;
    } else {
      const float2 o = __ldcg(reinterpret_cast<const float2*>(from + static_cast<int64_t>(i) * D));
      acc[0] = acc[0] * a + o.x * e;
      acc[1] = acc[1] * a + o.y * e;
    }
    M = mn;
  }
  const float inv = 1.f / L;
  const int s = row / p.groups, head = blockIdx.y * p.groups + row - s * p.groups;
  T* dst = reinterpret_cast<T*>(p.out) + (static_cast<int64_t>(blockIdx.z) * p.seq + s) * p.os +
           static_cast<int64_t>(head) * D + lane * E;
#pragma unroll
  for (int c = 0; c < E; c += 2) *reinterpret_cast<uint32_t*>(dst + c) = pack2<DT>(acc[c] * inv, acc[c + 1] * inv);
}

int64_t up256(int64_t x) { return (x + 255) / 256 * 256; }

struct Plan {
  int n_qtiles, splits;
  int64_t keys;
  int64_t qx, qf, kx, vx, sx, ml, o, total;  // offsets in the workspace
};

// Splits of the key axis: as many as CTAs fit on the GPU at once, with four key tiles or more each.
Plan make_plan(int batch, int num_kv_heads, int64_t rows, int64_t len, int head_dim, bool remainder, int sm_count) {
  Plan pl{};
  pl.n_qtiles = static_cast<int>((rows + BQ - 1) / BQ);
  pl.keys = (len + BKV - 1) / BKV * BKV;
  const int64_t units = int64_t(batch) * num_kv_heads * (remainder ? pl.n_qtiles : (pl.n_qtiles + 1) / 2);
  pl.splits = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(sm_count / units, pl.keys / BKV / 4)));
  const int64_t bh = int64_t(batch) * num_kv_heads;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t x = at;
    at += up256(bytes);
    return x;
  };
  pl.qx = take(bh * rows * head_dim * (remainder ? 4 : 2));
  pl.qf = take(bh * rows * 4);
  pl.kx = take(bh * pl.keys * head_dim * 2);
  pl.vx = take(bh * pl.keys * head_dim * 2);
  pl.sx = take(bh * (pl.keys / BLOCK) * 16);
  pl.ml = take(pl.splits > 1 ? bh * rows * pl.splits * 8 : 0);
  pl.o = take(pl.splits > 1 ? bh * rows * pl.splits * head_dim * 4 : 0);
  pl.total = at;
  return pl;
}

template <int DT, int FMT, int D>
int launch(Params& p, const Plan& pl, cudaStream_t st) {
  const uint64_t bh = uint64_t(p.batch) * p.num_kv_heads;
  CUtensorMap tq, tk_, tv;
  const uint64_t q_parts = REMAINDER<DT> ? 2 * bh : bh;
  if (int rc = tensor_map_3d(&tq, p.qx, TK_F16, D, p.rows, q_parts, D, uint64_t(p.rows) * D, 64, BQ, 1)) return rc;
  if (int rc = tensor_map_3d(&tk_, p.kx, TK_F16, D, p.keys, bh, D, uint64_t(p.keys) * D, 64, BKV, 1)) return rc;
  if (int rc = tensor_map_3d(&tv, p.vx, TK_F16, p.keys, D, bh, p.keys, uint64_t(p.keys) * D, 64, D, 1)) return rc;
  auto kern = kv8_chunk_kernel<DT, D>;
  auto expand = kv8_expand_kernel<DT, FMT, D>;
  constexpr int EXPAND_SMEM = EXPAND_WARPS * BLOCK * D * 2;
  static bool configured[64] = {};
  DeviceInfo dev;
  if (int rc = current_device_info(&dev)) return rc;
  if (!configured[dev.device]) {
    if (int rc = check_cuda(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Smem<D>::TOTAL),
                            "cudaFuncSetAttribute(kv8_chunk)"))
      return rc;
    if (int rc = check_cuda(cudaFuncSetAttribute(expand, cudaFuncAttributeMaxDynamicSharedMemorySize, EXPAND_SMEM),
                            "cudaFuncSetAttribute(kv8_expand)"))
      return rc;
    configured[dev.device] = true;
  }
  const int rows_cta = EXPAND_WARPS * 32 / (D / 16);
  p.q_ctas = (p.rows + rows_cta - 1) / rows_cta;
  const int k_ctas = (p.keys / BLOCK + EXPAND_WARPS / 2 - 1) / (EXPAND_WARPS / 2);
  if (int rc = launch_kernel(expand, dim3(p.q_ctas + k_ctas, p.num_kv_heads, p.batch), dim3(EXPAND_WARPS * 32),
                             EXPAND_SMEM, st, 1, "kv8_expand", p))
    return rc;
  const int query_ctas = REMAINDER<DT> ? p.n_qtiles : (p.n_qtiles + 1) / 2;
  if (int rc = launch_kernel(kern, dim3(p.num_kv_heads, p.batch, query_ctas * p.splits), dim3(THREADS), Smem<D>::TOTAL, st, 1,
                             "kv8_chunk", tq, tk_, tv, p))
    return rc;
  if (p.splits == 1) return TK_OK;
  return launch_kernel(kv8_join_kernel<DT, D>, dim3((p.rows + 7) / 8, p.num_kv_heads, p.batch), dim3(256), 0, st, 1,
                       "kv8_join", p);
}

template <int DT, int FMT>
int launch(Params& p, const Plan& pl, int head_dim, cudaStream_t st) {
  return head_dim == 64 ? launch<DT, FMT, 64>(p, pl, st) : launch<DT, FMT, 128>(p, pl, st);
}

}  // namespace chunk

// Workspace of a plan, whichever the type.
static int64_t chunk_total(int batch, int num_kv_heads, int64_t rows, int64_t len, int head_dim, int sm_count) {
  return std::max(chunk::make_plan(batch, num_kv_heads, rows, len, head_dim, true, sm_count).total,
                  chunk::make_plan(batch, num_kv_heads, rows, len, head_dim, false, sm_count).total);
}

// Sequences whose operands are laid out at once: the workspace stays below a gigabyte unless one alone needs more.
static int sequences_at_once(int batch, int num_kv_heads, int64_t rows, int64_t len, int head_dim, int sm_count) {
  const int64_t one = chunk_total(1, num_kv_heads, rows, len, head_dim, sm_count);
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(batch, (int64_t(1) << 30) / std::max<int64_t>(one, 1))));
}

// One new token never: laying out the whole cache costs more than its step, and that one appends as it goes.
bool chunk_fits(int batch, int num_heads, int num_kv_heads, int seq, int64_t len) {
  const int64_t rows = int64_t(num_heads / num_kv_heads) * seq;
  return seq > 1 && rows >= CHUNK_MIN_ROWS && rows < (1 << 20) && len < (1 << 30) && batch <= 65535 &&
         int64_t(batch) * num_kv_heads < (1 << 30);
}

int64_t chunk_workspace(int batch, int num_heads, int num_kv_heads, int head_dim, int seq, int64_t len, int sm_count) {
  // the largest over all lengths up to `len`: fewer sequences at once may need more than more of a shorter length
  const int64_t rows = int64_t(num_heads / num_kv_heads) * seq;
  const int n = sequences_at_once(batch, num_kv_heads, rows, len, head_dim, sm_count);
  const int64_t here = chunk_total(n, num_kv_heads, rows, len, head_dim, sm_count);
  return n < batch ? std::max(here, int64_t(1) << 30) : here;
}

int chunk_launches(int batch, int num_heads, int num_kv_heads, int head_dim, int seq, int64_t len, int dtype,
                   int sm_count) {
  const int64_t rows = int64_t(num_heads / num_kv_heads) * seq;
  const int at_once = sequences_at_once(batch, num_kv_heads, rows, len, head_dim, sm_count);
  int n = 0;
  for (int b = 0; b < batch; b += at_once) {
    const int m = std::min(at_once, batch - b);
    n += chunk::make_plan(m, num_kv_heads, rows, len, head_dim, dtype == TK_F16, sm_count).splits > 1 ? 3 : 2;
  }
  return n;
}

int chunk_attention(const Cache& c, const void* q, int64_t qs, const void* k, int64_t ks, const void* v, int64_t vs,
                    const float* cos_t, const float* sin_t, void* out, int64_t os, int batch, int seq, int num_heads,
                    int num_kv_heads, int head_dim, int start_pos, void* workspace, int dtype, int sm_count,
                    cudaStream_t st) {
  using namespace chunk;
  Params p{};
  p.groups = num_heads / num_kv_heads;
  p.rows = p.groups * seq;
  const int64_t len = int64_t(start_pos) + seq;
  const int at_once = sequences_at_once(batch, num_kv_heads, p.rows, len, head_dim, sm_count);
  p.qs = qs, p.ks = ks, p.vs = vs, p.os = os;
  p.num_blocks = c.num_blocks;
  p.cos_t = cos_t, p.sin_t = sin_t;
  p.start = start_pos;
  p.seq = seq;
  p.num_kv_heads = num_kv_heads;
  p.scale_log2 = static_cast<float>((1.0 / std::sqrt(double(head_dim))) * 1.4426950408889634);
  for (int b = 0; b < batch; b += at_once) {
    p.batch = std::min(at_once, batch - b);
    const Plan pl = make_plan(p.batch, num_kv_heads, p.rows, len, head_dim, dtype == TK_F16, sm_count);
    const int64_t tok = int64_t(b) * seq, bh = int64_t(b) * num_kv_heads, block = int64_t(BLOCK) * head_dim;
    p.q = static_cast<const char*>(q) + tok * qs * 2;
    p.k = static_cast<const char*>(k) + tok * ks * 2;
    p.v = static_cast<const char*>(v) + tok * vs * 2;
    p.out = static_cast<char*>(out) + tok * os * 2;
    p.kc = static_cast<const uint8_t*>(c.k) + bh * c.num_blocks * block;
    p.vc = static_cast<const uint8_t*>(c.v) + bh * c.num_blocks * block;
    p.scales = c.scales + bh * c.num_blocks * 2;
    p.tail = static_cast<const char*>(c.tail) + bh * 2 * block * 2;
    char* ws = static_cast<char*>(workspace);
    p.qx = reinterpret_cast<__half*>(ws + pl.qx);
    p.qf = reinterpret_cast<float*>(ws + pl.qf);
    p.kx = reinterpret_cast<__half*>(ws + pl.kx);
    p.vx = reinterpret_cast<__half*>(ws + pl.vx);
    p.sx = reinterpret_cast<float4*>(ws + pl.sx);
    p.part_ml = reinterpret_cast<float2*>(ws + pl.ml);
    p.part_o = reinterpret_cast<float*>(ws + pl.o);
    p.keys = static_cast<int>(pl.keys);
    p.n_qtiles = pl.n_qtiles;
    p.splits = pl.splits;
    int rc;
    if (dtype == TK_F16)
      rc = c.format == TK_KV8_E4M3 ? launch<TK_F16, TK_KV8_E4M3>(p, pl, head_dim, st)
                                   : launch<TK_F16, TK_KV8_INT8>(p, pl, head_dim, st);
    else
      rc = c.format == TK_KV8_E4M3 ? launch<TK_BF16, TK_KV8_E4M3>(p, pl, head_dim, st)
                                   : launch<TK_BF16, TK_KV8_INT8>(p, pl, head_dim, st);
    if (rc) return rc;
  }
  return TK_OK;
}

}  // namespace kv8
}  // namespace tk
