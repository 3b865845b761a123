// Attention of new tokens against an 8-bit KV cache (format: kv8.cuh), and their append.
//
// What it computes. Sequence b has `start` tokens in its cache; its S new tokens sit at start .. start + S - 1. Query
// row t attends to the keys 0 .. t: those of complete blocks as code * scale, the rows of the open block and the
// call's own rows in 16 bits. q is rotated in fp32 and not rounded, k is rotated and rounded to the model type (what
// the cache keeps), o = softmax(q k^T / sqrt(D)) v, rounded once. Then the new rows are appended.
//
// One launch for the attention: a CTA takes a range of 32-key tiles of one (sequence, kv head, 8 query rows). Each of
// its warps runs the products of its own tiles on m16n8k16 with f16 operands and fp32 sums:
//   * codes are exact in f16, so are 16-bit rows times a power of two that brings the tile's largest magnitude to
//     [2^14, 2^15) (bf16; its 8 bits stay whole for 28 binades below that);
//   * the 8 query rows fill rows 0-7 of the A operand with f16(q), rows 8-15 with the remainder q - f16(q), likewise
//     the probabilities: the products lose nothing to 16-bit operands and the rows that GQA leaves unused are free;
//   * the scale of a block's values goes into the exponent: with x = s * scale_k / sqrt(D) * log2 e, a weight is
//     w = 2^(x + log2 scale_v - m), m the running maximum of that sum, O = sum w * code, and the softmax's
//     denominator is sum w / scale_v. So O needs no pass per block, w stays in [0, 1], and the rounding of log2
//     scale_v cancels between numerator and denominator.
// The warps' (m, l, O) rows are merged in shared memory; with the key axis split over CTAs, each stores its rows
// and the last to arrive (a counter, which it returns to zero) merges them in the order of the chunks, so results do
// not depend on the order of arrival. For S = 1 the warp that holds the open block also appends the row, or encodes
// the block if the row completes it (no CTA of the launch reads that block from the cache); for S > 1 a second launch
// appends, since other CTAs still read the tail.
#include <algorithm>
#include <string>

#include "kv8.cuh"
#include "kv8_host.h"
#include "tk_host.h"

namespace tk {
namespace kv8 {

constexpr int WARPS = 4;
constexpr int THREADS = WARPS * 32;
constexpr int ROWS = 8;         // query rows of a CTA
constexpr int CHUNK_TILES = 8;  // tiles of a CTA at the finest split of the key axis

struct AttnParams {
  const void* q;
  int64_t qs;
  const void* k;
  int64_t ks;
  const void* v;
  int64_t vs;
  uint8_t* kc;
  uint8_t* vc;
  float* scales;
  void* tail;
  int num_blocks;
  const float* cos_t;  // [table_rows, D / 2]; NULL: q and k are rotated already
  const float* sin_t;
  int64_t table_rows;
  void* out;
  int64_t os;
  int seq, num_kv_heads, groups, rows;  // rows = groups * seq
  int start_pos;
  const int* start_dev;
  int start_step;
  int n_rb, n_chunks;
  float scale_log2;
  int* counters;
  float2* part_ml;
  float* part_o;
};

__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, "
      "%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// f16(x), f16(y) and the remainders
__device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(x, y);
  const float2 f = __half22float2(h);
  hi = h2_u32(h);
  lo = h2_u32(__floats2half2_rn(x - f.x, y - f.y));
}

// The power of two that brings `amax` (fp32 bits of a magnitude) to [2^14, 2^15); 1 if it is not finite.
__device__ __forceinline__ float to_f16_range(uint32_t amax_bits) {
  const int e = static_cast<int>(amax_bits >> 23);
  if (e >= 255) return 1.f;
  return __uint_as_float(static_cast<uint32_t>(min(254, 268 - e)) << 23);
}

// State of a warp's 8 query rows: lane 4r + q holds row r; m and l of that row (l: this lane's share), O columns
// 8n + 2q + {0, 1} of it in o[n][0..1] and the part that comes from the probabilities' remainders in o[n][2..3].
template <int D>
struct Rows {
  float m, l;
  float o[D / 8][4];
};

// One tile: K(j, h, w) and V(m, w) give code words (w = 0..7: f16 pairs of the lane's fragment, kv8.cuh), `sk` the
// factor of the raw products, `lsv` = log2 of the values' scale, `isv` its inverse, allowed(token) the mask.
template <int D, bool MASK, typename KF, typename VF, typename AF>
__device__ __forceinline__ void attend_tile(Rows<D>& st, const uint32_t (&qf)[D / 64 * 4][4], float sk, float lsv,
                                            float isv, int lane, KF key_words, VF value_words, AF allowed) {
  constexpr int H = D / 64;
  const int q = lane & 3;
  float s[4][2];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int h = 0; h < H; ++h) {
      uint32_t w[8];
      key_words(j, h, w);
#pragma unroll
      for (int t = 0; t < 4; ++t)
        mma16816(c, qf[h * 4 + t][0], qf[h * 4 + t][1], qf[h * 4 + t][2], qf[h * 4 + t][3], w[2 * t], w[2 * t + 1]);
    }
    s[j][0] = fmaf(c[0] + c[2], sk, lsv);
    s[j][1] = fmaf(c[1] + c[3], sk, lsv);
    if (MASK) {
      if (!allowed(8 * q + 2 * j)) s[j][0] = -INFINITY;
      if (!allowed(8 * q + 2 * j + 1)) s[j][1] = -INFINITY;
    }
  }
  float mx = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[1][0], s[1][1])),
                   fmaxf(fmaxf(s[2][0], s[2][1]), fmaxf(s[3][0], s[3][1])));
  mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
  mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
  const float mn = fmaxf(st.m, mx);
  if (__any_sync(0xffffffffu, mn > st.m)) {
    const float a = mn == -INFINITY ? 1.f : exp2_approx(st.m - mn);
    st.l *= a;
#pragma unroll
    for (int n = 0; n < D / 8; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) st.o[n][i] *= a;
    st.m = mn;
  }
  const float base = mn == -INFINITY ? 0.f : mn;  // a row that has seen no key yet: all weights 0
  uint32_t hi[4], lo[4];
  float sum = 0.f;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float w0 = exp2_approx(s[j][0] - base), w1 = exp2_approx(s[j][1] - base);
    sum += w0 + w1;
    split2(w0, w1, hi[j], lo[j]);
  }
  st.l = fmaf(sum, isv, st.l);
#pragma unroll
  for (int m = 0; m < D / 16; ++m) {
    uint32_t w[8];
    value_words(m, w);
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int i = 0; i < 2; ++i)
        mma16816(st.o[2 * m + e], hi[2 * i], lo[2 * i], hi[2 * i + 1], lo[2 * i + 1], w[4 * e + 2 * i],
                 w[4 * e + 2 * i + 1]);
  }
}

template <int D>
struct Smem {
  static constexpr int TILE = BLOCK * D * 2;             // a 16-bit tile of keys or values
  static constexpr int STAGE = 2 * TILE;                 // per warp
  static constexpr int ML = WARPS * ROWS * 8;            // merge, over the stages: float2 [WARPS][ROWS]
  static constexpr int O = ML;                           // float [WARPS][ROWS][D]
  static constexpr int FLAG = WARPS * STAGE;
  static constexpr int TOTAL = FLAG + 16;
  static_assert(O + WARPS * ROWS * D * 4 <= FLAG, "the merge must fit in the stages");
};

template <int DT, int FMT, int D>
__global__ void __launch_bounds__(THREADS) kv8_attention_kernel(const AttnParams p) {
  extern __shared__ __align__(128) uint8_t smem[];
  using S = Smem<D>;
  using T = typename Dt<DT>::T;
  constexpr int C16 = D / 8;
  constexpr int H = D / 64;
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int kvh = blockIdx.y / p.n_rb, rb = blockIdx.y % p.n_rb, b = blockIdx.z;
  const int unit = blockIdx.z * gridDim.y + blockIdx.y;
  const int start = p.start_dev ? __ldcg(p.start_dev + static_cast<int64_t>(b) * p.start_step) : p.start_pos;
  const int64_t end = static_cast<int64_t>(start) + p.seq;
  if (start < 0 || end > static_cast<int64_t>(p.num_blocks) * BLOCK || (p.cos_t && end > p.table_rows)) {
    if (threadIdx.x == 0 && blockIdx.x == 0 && blockIdx.y == 0) record_device_error(TK_DEVERR_POSITION);
    return;
  }
  const int open = start % BLOCK, n8 = start / BLOCK;
  const int n_tiles = n8 + (open + p.seq + BLOCK - 1) / BLOCK;
  const int n_chunks = min(p.n_chunks, (n_tiles + CHUNK_TILES - 1) / CHUNK_TILES);
  const int chunk = blockIdx.x;
  if (chunk >= n_chunks) return;
  const int lo = static_cast<int>(static_cast<int64_t>(n_tiles) * chunk / n_chunks);
  const int hi = static_cast<int>(static_cast<int64_t>(n_tiles) * (chunk + 1) / n_chunks);
  const int64_t bh = static_cast<int64_t>(b) * p.num_kv_heads + kvh;
  const uint8_t* kc = p.kc + bh * p.num_blocks * (BLOCK * D);
  const uint8_t* vc = p.vc + bh * p.num_blocks * (BLOCK * D);
  const float2* scales = reinterpret_cast<const float2*>(p.scales) + bh * p.num_blocks;

  // this lane's share of query row r: rotated, brought to the f16 range, split in two
  const int r = lane >> 2, q = lane & 3;
  const int gr = rb * ROWS + r;
  int qpos = -1;  // a padding row sees no key of the 16-bit tiles, and its zeros harm nothing in the others
  uint32_t qf[H * 4][4];
  float cq;
  {
    float f[H][16];
    float amax = 0.f;
#pragma unroll
    for (int h = 0; h < H; ++h)
#pragma unroll
      for (int i = 0; i < 16; ++i) f[h][i] = 0.f;
    if (gr < p.rows) {
      const int s = gr / p.groups, head = kvh * p.groups + gr % p.groups;
      qpos = start + s;
      const T* row = reinterpret_cast<const T*>(p.q) + (static_cast<int64_t>(b) * p.seq + s) * p.qs +
                     static_cast<int64_t>(head) * D;
#pragma unroll
      for (int h = 0; h < H; ++h)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int c = 8 * h + 2 * q + e;
          const uint4 x = __ldcg(reinterpret_cast<const uint4*>(row) + c);
          const uint32_t w[4] = {x.x, x.y, x.z, x.w};
          float cc[4] = {1.f, 1.f, 1.f, 1.f}, ss[4] = {0.f, 0.f, 0.f, 0.f};
          if (p.cos_t) {
            const int64_t at = static_cast<int64_t>(qpos) * (D / 2) + c * 4;
            const float4 a = __ldg(reinterpret_cast<const float4*>(p.cos_t + at));
            const float4 d = __ldg(reinterpret_cast<const float4*>(p.sin_t + at));
            cc[0] = a.x, cc[1] = a.y, cc[2] = a.z, cc[3] = a.w;
            ss[0] = d.x, ss[1] = d.y, ss[2] = d.z, ss[3] = d.w;
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 v = unpack2<DT>(w[i]);
            f[h][8 * e + 2 * i] = v.x * cc[i] - v.y * ss[i];
            f[h][8 * e + 2 * i + 1] = v.x * ss[i] + v.y * cc[i];
          }
        }
    }
#pragma unroll
    for (int h = 0; h < H; ++h)
#pragma unroll
      for (int i = 0; i < 16; ++i) amax = fmaxf(amax, fabsf(f[h][i]));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    const float up = to_f16_range(__float_as_uint(amax));
    cq = p.scale_log2 / up;
#pragma unroll
    for (int h = 0; h < H; ++h)
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        split2(f[h][4 * t] * up, f[h][4 * t + 1] * up, qf[h * 4 + t][0], qf[h * 4 + t][1]);
        split2(f[h][4 * t + 2] * up, f[h][4 * t + 3] * up, qf[h * 4 + t][2], qf[h * 4 + t][3]);
      }
  }

  Rows<D> st;
  st.m = -INFINITY;
  st.l = 0.f;
#pragma unroll
  for (int n = 0; n < D / 8; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) st.o[n][i] = 0.f;

  // complete blocks: the next block's keys are loaded once this one's are used, likewise its values
  const int hi8 = min(hi, n8);
  const int first = lo + warp;
  uint4 kr[4][H], vr[D / 16];
  float2 sc = make_float2(1.f, 1.f);
  auto load_keys = [&](int t) {
    const uint4* src = reinterpret_cast<const uint4*>(kc + static_cast<int64_t>(t) * (BLOCK * D)) + lane;
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int h = 0; h < H; ++h) kr[j][h] = __ldcg(src + (j * H + h) * 32);
  };
  auto load_values = [&](int t) {
    const uint4* src = reinterpret_cast<const uint4*>(vc + static_cast<int64_t>(t) * (BLOCK * D)) + lane;
#pragma unroll
    for (int m = 0; m < D / 16; ++m) vr[m] = __ldcg(src + m * 32);
  };
  if (first < hi8) {
    sc = __ldcg(scales + first);
    load_keys(first);
    load_values(first);
  }
  for (int t = first; t < hi8; t += WARPS) {
    const float2 now = sc;
    const int next = t + WARPS;
    const bool more = next < hi8;
    if (more) sc = __ldcg(scales + next);
    attend_tile<D, false>(
        st, qf, cq * now.x, __log2f(now.y), 1.f / now.y, lane,
        [&](int j, int h, uint32_t (&w)[8]) {
          decode4<FMT>(kr[j][h].x, w[0], w[1]);
          decode4<FMT>(kr[j][h].y, w[2], w[3]);
          decode4<FMT>(kr[j][h].z, w[4], w[5]);
          decode4<FMT>(kr[j][h].w, w[6], w[7]);
          if (j == 3 && h == H - 1 && more) load_keys(next);
        },
        [&](int m, uint32_t (&w)[8]) {
          decode4<FMT>(vr[m].x, w[0], w[1]);
          decode4<FMT>(vr[m].y, w[2], w[3]);
          decode4<FMT>(vr[m].z, w[4], w[5]);
          decode4<FMT>(vr[m].w, w[6], w[7]);
          if (m == D / 16 - 1 && more) load_values(next);
        },
        [](int) { return true; });
  }

  // the open block and the new rows
  for (int t = first; t < hi; t += WARPS) {
    if (t < n8) continue;
    const uint32_t ktile = smem_u32(smem) + warp * S::STAGE, vtile = ktile + S::TILE;
    uint8_t* kp = smem + warp * S::STAGE;
    uint8_t* vp = kp + S::TILE;
    const T* tail = reinterpret_cast<const T*>(p.tail) + bh * 2 * BLOCK * D;
    const int n_rows = min(BLOCK, static_cast<int>(end - static_cast<int64_t>(t) * BLOCK));
    uint32_t km = 0, vm = 0;
    __syncwarp();
#pragma unroll 4
    for (int i = 0; i < C16; ++i) {
      const int idx = lane + 32 * i, row = idx / C16, c = idx % C16;
      const int s = (t - n8) * BLOCK + row - open;  // the call's row, or one of the tail
      uint4 kx = make_uint4(0, 0, 0, 0), vx = kx;
      if (row < n_rows) {
        if (s < 0) {
          kx = __ldcg(reinterpret_cast<const uint4*>(tail + row * D) + c);
          vx = __ldcg(reinterpret_cast<const uint4*>(tail + (BLOCK + row) * D) + c);
        } else {
          const int64_t tok = static_cast<int64_t>(b) * p.seq + s;
          kx = __ldcg(reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(p.k) + tok * p.ks +
                                                     static_cast<int64_t>(kvh) * D) + c);
          vx = __ldcg(reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(p.v) + tok * p.vs +
                                                     static_cast<int64_t>(kvh) * D) + c);
          if (p.cos_t) {
            const int64_t at = (static_cast<int64_t>(start) + s) * (D / 2) + c * 4;
            rope_chunk<DT>(kx, p.cos_t + at, p.sin_t + at);
          }
        }
      }
      km = amax2(amax2(amax2(amax2(km, kx.x), kx.y), kx.z), kx.w);
      vm = amax2(amax2(amax2(amax2(vm, vx.x), vx.y), vx.z), vx.w);
      *reinterpret_cast<uint4*>(kp + tile_off<D>(row, c)) = kx;
      *reinterpret_cast<uint4*>(vp + tile_off<D>(row, c)) = vx;
    }
    km = amax2_warp(km);
    vm = amax2_warp(vm);
    __syncwarp();

    // f16 takes its own rows as they are; bf16 rows are brought to its range
    const float fk = DT == TK_F16 ? 1.f : to_f16_range(km << 16), fv = DT == TK_F16 ? 1.f : to_f16_range(vm << 16);
    auto to_half = [](uint32_t w, float f) -> uint32_t {
      if constexpr (DT == TK_F16) {
        return w;
      } else {
        const float2 v = unpack2<DT>(w);
        return h2_u32(__floats2half2_rn(v.x * f, v.y * f));
      }
    };
    attend_tile<D, true>(
        st, qf, cq / fk, -__log2f(fv), fv, lane,
        [&](int j, int h, uint32_t (&w)[8]) {
          const int row = 8 * (r >> 1) + 2 * j + (r & 1);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const uint4 x = *reinterpret_cast<const uint4*>(kp + tile_off<D>(row, 8 * h + 2 * q + e));
            w[4 * e] = to_half(x.x, fk);
            w[4 * e + 1] = to_half(x.y, fk);
            w[4 * e + 2] = to_half(x.z, fk);
            w[4 * e + 3] = to_half(x.w, fk);
          }
        },
        [&](int m, uint32_t (&w)[8]) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            uint32_t x[4];
            load_column_tokens<D>(vtile, 2 * m + e, lane, x);
#pragma unroll
            for (int i = 0; i < 4; ++i) w[4 * e + i] = to_half(x[i], fv);
          }
        },
        [&](int token) { return t * BLOCK + token <= qpos; });

    if (p.seq == 1 && rb == 0) {  // the append of a decode step
      T* to = reinterpret_cast<T*>(p.tail) + bh * 2 * BLOCK * D;
      if (open < BLOCK - 1) {
        for (int c = lane; c < 2 * C16; c += 32) {
          const bool val = c >= C16;
          const int cc = val ? c - C16 : c;
          *(reinterpret_cast<uint4*>(to + ((val ? BLOCK : 0) + open) * D) + cc) =
              *reinterpret_cast<const uint4*>((val ? vp : kp) + tile_off<D>(open, cc));
        }
      } else {
        const int64_t block = bh * p.num_blocks + t;
        const float sk = encode_keys<DT, FMT, D>(p.kc + block * (BLOCK * D), lane, [&](int tok, int c) {
          return *reinterpret_cast<const uint4*>(kp + tile_off<D>(tok, c));
        });
        const float sv = encode_values<DT, FMT, D>(p.vc + block * (BLOCK * D), lane, vtile, vm);
        if (lane == 0) reinterpret_cast<float2*>(p.scales)[block] = make_float2(sk, sv);
      }
    }
  }
  pdl_launch_dependents();

  // merge the warps' rows in shared memory, over the stages
  st.l += __shfl_xor_sync(0xffffffffu, st.l, 1);
  st.l += __shfl_xor_sync(0xffffffffu, st.l, 2);
  __syncthreads();
  float2* ml_s = reinterpret_cast<float2*>(smem);
  float* o_s = reinterpret_cast<float*>(smem + S::O);
  int* last_s = reinterpret_cast<int*>(smem + S::FLAG);
  if (q == 0) ml_s[warp * ROWS + r] = make_float2(st.m, st.l);
#pragma unroll
  for (int n = 0; n < D / 8; ++n)
    *reinterpret_cast<float2*>(o_s + (warp * ROWS + r) * D + 8 * n + 2 * q) =
        make_float2(st.o[n][0] + st.o[n][2], st.o[n][1] + st.o[n][3]);
  __syncthreads();

  constexpr int D4 = D / 4;
  auto fold = [](float& M, float& L, float (&acc)[4], float2 ml, float4 ov) {
    const float mn = fmaxf(M, ml.x);
    const float a = exp2_approx(M - mn), e = exp2_approx(ml.x - mn);
    L = L * a + ml.y * e;
    acc[0] = acc[0] * a + ov.x * e;
    acc[1] = acc[1] * a + ov.y * e;
    acc[2] = acc[2] * a + ov.z * e;
    acc[3] = acc[3] * a + ov.w * e;
    M = mn;
  };
  auto store = [&](int g, int d, float L, const float (&acc)[4]) {
    const float inv = 1.f / L;
    const int s = g / p.groups, head = kvh * p.groups + g % p.groups;
    T* dst = reinterpret_cast<T*>(p.out) + (static_cast<int64_t>(b) * p.seq + s) * p.os +
             static_cast<int64_t>(head) * D + d;
    *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<DT>(acc[0] * inv, acc[1] * inv),
                                                pack2<DT>(acc[2] * inv, acc[3] * inv));
  };
  for (int idx = threadIdx.x; idx < ROWS * D4; idx += THREADS) {
    const int lr = idx / D4, d = (idx % D4) * 4, g = rb * ROWS + lr;
    if (g >= p.rows) continue;
    float M = -INFINITY, L = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float2 ml = ml_s[w * ROWS + lr];
      if (ml.x == -INFINITY && ml.y == 0.f) continue;  // no key of this row in the warp's tiles
      fold(M, L, acc, ml, *reinterpret_cast<const float4*>(o_s + (w * ROWS + lr) * D + d));
    }
    if (n_chunks == 1) {
      store(g, d, L, acc);
    } else {
      const int64_t slot = (static_cast<int64_t>(unit) * p.n_chunks + chunk) * ROWS + lr;
      if (d == 0) p.part_ml[slot] = make_float2(M, L);
      *reinterpret_cast<float4*>(p.part_o + slot * D + d) = make_float4(acc[0], acc[1], acc[2], acc[3]);
    }
  }
  if (n_chunks == 1) return;

  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) *last_s = atomicAdd(p.counters + unit, 1) == n_chunks - 1;
  __syncthreads();
  if (!*last_s) return;
  __threadfence();
  for (int idx = threadIdx.x; idx < ROWS * D4; idx += THREADS) {
    const int lr = idx / D4, d = (idx % D4) * 4, g = rb * ROWS + lr;
    if (g >= p.rows) continue;
    float M = -INFINITY, L = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
    for (int c = 0; c < n_chunks; ++c) {
      const int64_t slot = (static_cast<int64_t>(unit) * p.n_chunks + c) * ROWS + lr;
      const float2 ml = __ldcg(p.part_ml + slot);
      if (ml.x == -INFINITY && ml.y == 0.f) continue;
      fold(M, L, acc, ml, __ldcg(reinterpret_cast<const float4*>(p.part_o + slot * D + d)));
    }
    store(g, d, L, acc);
  }
  if (threadIdx.x == 0) p.counters[unit] = 0;
}

// The arrival counters come first and in a fixed size (a split needs fewer than two units for every SM), so calls
// of different shapes that follow one another on a stream can share one workspace.
constexpr int64_t COUNTERS = 4096;

struct Plan {
  int n_rb, n_chunks;
  int64_t units;
  size_t ml_bytes, o_bytes;
  size_t bytes() const { return n_chunks > 1 ? COUNTERS + ml_bytes + o_bytes : 0; }
};

size_t round_up(size_t x, size_t a) { return (x + a - 1) / a * a; }

// Chunks of the key axis: enough CTAs for two on every SM, each with CHUNK_TILES tiles or more. Never fewer for a
// longer cache, so that a workspace sized for the capacity serves every position.
Plan make_plan(int batch, int num_kv_heads, int rows, int max_kv, int head_dim, int sm_count) {
  Plan pl{};
  pl.n_rb = (rows + ROWS - 1) / ROWS;
  pl.units = static_cast<int64_t>(batch) * num_kv_heads * pl.n_rb;
  const int tiles = max_kv / BLOCK + 1;
  const int64_t most = (tiles + CHUNK_TILES - 1) / CHUNK_TILES;
  const int64_t want = (2 * static_cast<int64_t>(std::max(sm_count, 1)) + pl.units - 1) / pl.units;
  pl.n_chunks = static_cast<int>(std::max<int64_t>(1, std::min(most, want)));
  if (pl.units * static_cast<int64_t>(sizeof(int)) > COUNTERS) pl.n_chunks = 1;
  const size_t slots = static_cast<size_t>(pl.units) * pl.n_chunks * ROWS;
  pl.ml_bytes = round_up(slots * sizeof(float2), 256);
  pl.o_bytes = slots * head_dim * sizeof(float);
  return pl;
}

template <int DT, int FMT, int D>
int launch(const AttnParams& p, dim3 grid, cudaStream_t st) {
  auto kern = kv8_attention_kernel<DT, FMT, D>;
  static bool configured[64] = {};
  DeviceInfo dev;
  if (int rc = current_device_info(&dev)) return rc;
  if (!configured[dev.device]) {
    if (int rc = check_cuda(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Smem<D>::TOTAL),
                            "cudaFuncSetAttribute(kv8_attention)"))
      return rc;
    configured[dev.device] = true;
  }
  return launch_kernel(kern, grid, dim3(THREADS), Smem<D>::TOTAL, st, 1, "kv8_attention", p);
}

template <int DT, int FMT>
int launch(const AttnParams& p, int head_dim, dim3 grid, cudaStream_t st) {
  return head_dim == 64 ? launch<DT, FMT, 64>(p, grid, st) : launch<DT, FMT, 128>(p, grid, st);
}

}  // namespace kv8
}  // namespace tk

extern "C" int64_t tk_kv8_attention_workspace(int batch, int num_heads, int num_kv_heads, int head_dim, int seq,
                                              int max_kv) {
  using namespace tk;
  if (batch <= 0 || seq <= 0 || num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads || max_kv <= 0)
    return 0;
  DeviceInfo di;
  if (current_device_info(&di)) return -1;
  const int64_t rows = int64_t(num_heads / num_kv_heads) * seq;
  if (rows > INT32_MAX) return 0;
  return static_cast<int64_t>(
      kv8::make_plan(batch, num_kv_heads, static_cast<int>(rows), max_kv, head_dim, di.sm_count).bytes());
}

extern "C" int tk_kv8_attention(const void* q, int64_t q_tok_stride, const void* k, int64_t k_tok_stride,
                                const void* v, int64_t v_tok_stride, void* k_cache, void* v_cache, float* scales,
                                void* tail, int num_blocks, int format, const float* cos_table,
                                const float* sin_table, int64_t table_rows, void* out, int64_t out_tok_stride,
                                int batch, int seq, int num_heads, int num_kv_heads, int head_dim, int start_pos,
                                const int* start_pos_device, int start_pos_step, void* workspace,
                                int64_t workspace_bytes, int dtype, void* stream) {
  using namespace tk;
  using namespace tk::kv8;
  const Cache c{k_cache, v_cache, scales, tail, num_blocks, format};
  if (int rc = check_cache("kv8_attention", c, batch, seq, num_heads, num_kv_heads, head_dim, dtype)) return rc;
  if (q_tok_stride < int64_t(num_heads) * head_dim || k_tok_stride < int64_t(num_kv_heads) * head_dim ||
      v_tok_stride < int64_t(num_kv_heads) * head_dim || out_tok_stride < int64_t(num_heads) * head_dim)
    return fail_invalid("kv8_attention: token stride smaller than heads * head_dim");
  if (q_tok_stride % 8 || k_tok_stride % 8 || v_tok_stride % 8 || out_tok_stride % 8)
    return fail_invalid("kv8_attention: token strides must be multiples of 8 elements");
  if ((cos_table == nullptr) != (sin_table == nullptr))
    return fail_invalid("kv8_attention: give both RoPE tables or neither");
  const int64_t capacity = int64_t(num_blocks) * BLOCK;
  if (!start_pos_device) {
    if (start_pos < 0) return fail_invalid("kv8_attention: start_pos must be >= 0");
    if (int64_t(start_pos) + seq > capacity) return fail_invalid("kv8_attention: start_pos + seq exceeds the cache");
    if (cos_table && int64_t(start_pos) + seq > table_rows)
      return fail_invalid("kv8_attention: start_pos + seq exceeds the RoPE table length");
  } else if (start_pos_step != 0 && start_pos_step != 1) {
    return fail_invalid("kv8_attention: start_pos_step must be 0 or 1");
  }
  if (batch == 0 || seq == 0) return TK_OK;
  if (!q || !k || !v || !out) return fail_invalid("kv8_attention: NULL pointer");
  for (const void* ptr : {q, k, v, static_cast<const void*>(out), static_cast<const void*>(cos_table),
                          static_cast<const void*>(sin_table)})
    if (!aligned16(ptr)) return fail_invalid("kv8_attention: pointers must be 16-byte aligned");
  DeviceInfo di;
  if (int rc = current_device_info(&di)) return rc;
  const int64_t rows = int64_t(num_heads / num_kv_heads) * seq;
  const int max_kv = start_pos_device ? static_cast<int>(std::min<int64_t>(capacity, INT32_MAX)) : start_pos + seq;
  if (rows > (int64_t(65535) / num_kv_heads) * ROWS)
    return fail_invalid("kv8_attention: too many query rows per kv head");
  const Plan pl = make_plan(batch, num_kv_heads, static_cast<int>(rows), max_kv, head_dim, di.sm_count);
  if (pl.bytes() > 0) {
    if (!workspace || workspace_bytes < static_cast<int64_t>(pl.bytes()))
      return fail_invalid("kv8_attention: workspace missing or smaller than tk_kv8_attention_workspace()");
    if (!aligned16(workspace)) return fail_invalid("kv8_attention: workspace must be 16-byte aligned");
  }
  AttnParams p{};
  p.q = q;
  p.qs = q_tok_stride;
  p.k = k;
  p.ks = k_tok_stride;
  p.v = v;
  p.vs = v_tok_stride;
  p.kc = static_cast<uint8_t*>(k_cache);
  p.vc = static_cast<uint8_t*>(v_cache);
  p.scales = scales;
  p.tail = tail;
  p.num_blocks = num_blocks;
  p.cos_t = cos_table;
  p.sin_t = sin_table;
  p.table_rows = table_rows;
  p.out = out;
  p.os = out_tok_stride;
  p.seq = seq;
  p.num_kv_heads = num_kv_heads;
  p.groups = num_heads / num_kv_heads;
  p.rows = static_cast<int>(rows);
  p.start_pos = start_pos;
  p.start_dev = start_pos_device;
  p.start_step = start_pos_step;
  p.n_rb = pl.n_rb;
  p.n_chunks = pl.n_chunks;
  p.scale_log2 = static_cast<float>((1.0 / std::sqrt(double(head_dim))) * 1.4426950408889634);
  if (pl.bytes() > 0) {
    char* ws = static_cast<char*>(workspace);
    p.counters = reinterpret_cast<int*>(ws);
    p.part_ml = reinterpret_cast<float2*>(ws + COUNTERS);
    p.part_o = reinterpret_cast<float*>(ws + COUNTERS + pl.ml_bytes);
  }
  const dim3 grid(pl.n_chunks, num_kv_heads * pl.n_rb, batch);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  int rc;
  if (dtype == TK_F16)
    rc = format == TK_KV8_E4M3 ? launch<TK_F16, TK_KV8_E4M3>(p, head_dim, grid, st)
                               : launch<TK_F16, TK_KV8_INT8>(p, head_dim, grid, st);
  else
    rc = format == TK_KV8_E4M3 ? launch<TK_BF16, TK_KV8_E4M3>(p, head_dim, grid, st)
                               : launch<TK_BF16, TK_KV8_INT8>(p, head_dim, grid, st);
  if (rc || seq == 1) return rc;
  return append(c, k, k_tok_stride, v, v_tok_stride, cos_table, sin_table, table_rows, batch, seq, num_kv_heads,
                head_dim, start_pos, start_pos_device, start_pos_step, dtype, st);
}
