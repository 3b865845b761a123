// Attention of new tokens against an 8-bit KV cache (format: kv8.cuh), and their append.
//
// What it computes. Sequence b has `start` tokens in its cache; its S new tokens sit at start .. start + S - 1. Query
// row t attends to the keys 0 .. t: those of complete blocks as code * scale, the rows of the open block and the
// call's own rows in 16 bits. q is rotated in fp32 and not rounded, k is rotated and rounded to the model type (what
// the cache keeps), o = softmax(q k^T / sqrt(D)) v, rounded once. Then the new rows are appended.
//
// Products: m16n8k16 with f16 operands and fp32 sums, a warp for each tile of 32 keys, with the keys (and the columns
// of V) as the 16 rows of the product and the query rows as its 8 columns:
//   * codes are exact in f16, so are 16-bit rows times a power of two that brings the tile's largest magnitude to
//     [2^14, 2^15) (bf16; its 8 bits stay whole for 28 binades below that; f16 keys are taken as they are);
//   * a query row takes two columns, f16(q) and the remainder q - f16(q), likewise its probabilities, whose sum stays
//     in one lane: 22 bits of each. Four query rows fill the 8 columns, which is what GQA with up to four heads for each
//     kv head needs; eight rows (NG = 2) take every product twice;
//   * the scale of a block's values goes into the exponent: with x = s * scale_k / sqrt(D) * log2 e, a weight is
//     w = 2^(x + log2 scale_v - m + HEADROOM), m the running maximum of x + log2 scale_v, O = sum w * code, and the
//     softmax's denominator is sum w / scale_v. So O needs no pass per block, and the rounding of log2 scale_v cancels
//     between numerator and denominator. w goes up to 2^15, the top of f16's range, so that a weight is lost to its
//     smallest number, 2^-24, only 2^40 below the largest: a million of them are still 2^-20 of the result. With bf16 the
//     scales of two blocks can be 2^188 apart (zeros beside values of 2^120), so w can leave fp32's range below while w /
//     scale_v counts in the denominator: where a lane's keys are all 2^60 below m it takes their shares of the denominator
//     as exponentials of their own, and sums of shares are scaled in two steps, by the root of the factor (an f16 cache's
//     scales are 2^76 apart at most, so what is lost of w is below 2^-126 2^76 of the denominator).
// (The keys as columns, with f16(q) and remainder as two halves of the 16 rows, took 274 instead of 231 instructions
// for a tile of 64 columns and four rows, twice the accumulators, and 20.5 us instead of 18.7 us for 64 sequences of 4
// kv heads at 2047.)
//
// Bound by HBM at D = 128 (16 x 16001 positions of 8 kv heads: 87 us, 6.0 TB/s). At D = 64 by latency and balance: a warp
// goes copies - products - maximum - products tile by tile, and the instructions fill a third to a half of the issue slots
// (64 x 2047 of 4 kv heads, one CTA a unit: 18.6 us, 31 %; 48 ragged sequences of 8 kv heads, int8: 45.6 us, 4.5 TB/s, 45 %;
// 2 x 100003 with 7 heads a kv head, int8: 26.6 us, 28 %). For little work by the chain position - copies - products - merge
// (7 us for one sequence of 4 kv heads at 127). int8 costs some 97 instructions a tile more than e4m3.
//
// Division of the work: all units' tiles in one line (beginning a unit counts UNIT_WEIGHT, a 16-bit tile TAIL_WEIGHT),
// cut into equal pieces, one for each warp that fits on the GPU at once. So long and short sequences, few units and
// many, keep every SM busy to the end, and no CTA waits for another. A piece covers parts of one or more units. The
// parts of a unit that lie in one CTA are merged in shared memory when its warps are done; where a unit lies in
// several CTAs, the last of them to arrive (counters, which it returns to zero) merges their parts in the order of the
// pieces, so results do not depend on the order of arrival; above 16 CTAs in two steps, the first over aligned groups of
// 16, so that no warp reads hundreds of parts. With little work a unit gets CTAs of its own, PIECE_MIN for each warp.
// A warp copies its tiles ahead into a ring of its own in shared memory (cp.async), and the first tiles of its next
// unit before it puts the last one's rows away. For S = 1 the warp that holds the open block also appends the row, or
// encodes the block if the row completes it (nothing in the launch reads that block from the cache); for S > 1 a
// second launch appends, since other warps still read the tail. Many rows at a position known on the host take
// kv8_chunk.cu.
#include <algorithm>
#include <string>
#include <type_traits>

#include "kv8.cuh"
#include "kv8_host.h"
#include "tk_host.h"

namespace tk {
namespace kv8 {

constexpr int WARPS = 4;
constexpr int THREADS = WARPS * 32;
constexpr int TAIL_WEIGHT = 4;  // tiles that one 16-bit tile takes as long as
constexpr int UNIT_WEIGHT = 1;  // and beginning a unit
constexpr int PIECE_MIN = 4;    // weight of a piece when there is little work
constexpr int MERGE_COST = 8;   // weight that a warp could take while the parts of two CTAs are merged
constexpr int GROUP = 16;       // CTAs that are merged in one step
constexpr float HEADROOM = 15.f;  // log2 of the largest weight

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
  int n_rb, batch;
  int most_ctas;  // CTAs that each unit can have for its own
  float scale_log2;
  int* counters;    // [CTAs][3], zero between launches
  // [CTAs][2: the unit that goes on from the CTA before, the one that the next goes on with][NG][...]
  float2* part_ml;  // [4 rows]
  float* part_o;    // [D / 8][32 lanes]
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

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

// 8 x 8 16-bit matrix transposed: lane 4i + q gives row i, columns 2q and 2q + 1, and takes them of the transpose.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// State of a warp's 4 NG query rows; lane 4r + q has row 4g + q, of that row m, and its own keys' share of l, and the
// columns 16n + r and 16n + 8 + r of O as sums of two parts, o[g][n][0] + [1] and [2] + [3].
template <int D, int NG>
struct Rows {
  float m[NG], l[NG];
  float o[NG][D / 16][4];
};

// N tiles in one step (independent products and one maximum, so that a warp that has a scheduler to itself waits
// less): key_words(u, j, h, w) and value_words(u, m, w) give the f16 pairs w[0..7] of the lane's fragment of tile u
// (kv8.cuh), `sk` the factor of the raw products, `lsv` log2 of the values' scale, `isv` its inverse, allowed(g, token)
// the mask. qf[g][k step] is the fragment of the query rows. WIDE: the values' scales may lie far apart (bf16).
template <int D, int NG, int N, bool MASK, bool WIDE, typename KF, typename VF, typename AF>
__device__ __forceinline__ void attend_tiles(Rows<D, NG>& st, const uint32_t (&qf)[NG][D / 16][2],
                                             const float (&sk)[NG][N], const float (&lsv)[N], const float (&isv)[N],
                                             int lane, KF key_words, VF value_words, AF allowed) {
  constexpr int H = D / 64;
  const int r = lane >> 2;
  float s[NG][N][4];
#pragma unroll
  for (int u = 0; u < N; ++u)
#pragma unroll
    for (int jj = 0; jj < 2; ++jj) {
      float c[NG][4];
#pragma unroll
      for (int g = 0; g < NG; ++g) c[g][0] = c[g][1] = c[g][2] = c[g][3] = 0.f;
#pragma unroll
      for (int h = 0; h < H; ++h) {
        uint32_t w0[8], w1[8];
        key_words(u, 2 * jj, h, w0);
        key_words(u, 2 * jj + 1, h, w1);
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int g = 0; g < NG; ++g)
            mma16816(c[g], w0[2 * t], w1[2 * t], w0[2 * t + 1], w1[2 * t + 1], qf[g][h * 4 + t][0], qf[g][h * 4 + t][1]);
      }
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        s[g][u][2 * jj] = fmaf(c[g][0] + c[g][1], sk[g][u], lsv[u]);
        s[g][u][2 * jj + 1] = fmaf(c[g][2] + c[g][3], sk[g][u], lsv[u]);
        if (MASK) {
          const int tok = 8 * (r >> 1) + 4 * jj + (r & 1);
          if (!allowed(g, tok)) s[g][u][2 * jj] = -INFINITY;
          if (!allowed(g, tok + 2)) s[g][u][2 * jj + 1] = -INFINITY;
        }
      }
    }
  float mn[NG], own[NG][N];
  bool grown = false;
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    float mx = -INFINITY;
#pragma unroll
    for (int u = 0; u < N; ++u) {
      own[g][u] = fmaxf(fmaxf(s[g][u][0], s[g][u][1]), fmaxf(s[g][u][2], s[g][u][3]));
      mx = fmaxf(mx, own[g][u]);
    }
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    mn[g] = fmaxf(st.m[g], mx);
    grown |= mn[g] > st.m[g];
  }
  if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      // O's columns are the rows' weights in two parts, in this lane those of row q: the factor is the lane's own
      const float root = mn[g] == -INFINITY ? 1.f : exp2_approx(0.5f * (st.m[g] - mn[g])), a = root * root;
      st.l[g] = st.l[g] * root * root;
#pragma unroll
      for (int n = 0; n < D / 16; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) st.o[g][n][i] *= a;
      st.m[g] = mn[g];
    }
  }
#pragma unroll
  for (int u = 0; u < N; ++u) {
    uint32_t pf[NG][4];
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const float base = mn[g] == -INFINITY ? 0.f : mn[g] - HEADROOM;  // a row that has seen no key yet: all weights 0
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float w = exp2_approx(s[g][u][j] - base);
        sum += w;
        pf[g][j] = transpose8(h2_u32(__floats2half2_rn(w, w - __half2float(__float2half_rn(w)))));
      }
      if (WIDE && own[g][u] < mn[g] - 60.f) {
        sum = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) sum += exp2_approx((s[g][u][j] - lsv[u]) - base);
        st.l[g] += sum;
      } else {
        st.l[g] = fmaf(sum, isv[u], st.l[g]);
      }
    }
#pragma unroll
    for (int n = 0; n < D / 16; ++n) {
      uint32_t w[8];
      value_words(u, n, w);
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int g = 0; g < NG; ++g)
          mma16816(st.o[g][n], w[2 * i], w[4 + 2 * i], w[2 * i + 1], w[4 + 2 * i + 1], pf[g][2 * i], pf[g][2 * i + 1]);
    }
  }
}

// a / b for small non-negative numbers, without the latency of an integer division
__device__ __forceinline__ int quotient(int a, int b) {
  if (a >= 1 << 22) return a / b;
  int x = static_cast<int>(__fdividef(static_cast<float>(a), static_cast<float>(b)));
  const int rem = a - x * b;
  return x + (rem >= b) - (rem < 0);
}

template <int D, int NG>
struct Smem {
  static constexpr int ROWS = 4 * NG;                                        // query rows of a unit
  static constexpr int CTAS_SM = D == 64 ? (NG == 1 ? 4 : 3) : 2;
  static constexpr int SPLIT_COST = D == 64 ? 40 : 20;
  static constexpr int STAGES = D == 64 && NG == 2 ? 4 : 3;
  static constexpr int PAIR = D == 64 && NG == 2 ? 2 : 1;                      // blocks of a step
  static constexpr int HALF = BLOCK * D;                                     // a block's keys or values
  static constexpr int STAGE = 2 * HALF;        // a block, or the keys or the values of a 16-bit tile
  static constexpr int RING = STAGES * STAGE;   // of one warp
  static constexpr int PART = ROWS * D * 4 + ROWS * 8;  // a warp's rows of a unit: O, then (m, l)
  static constexpr int HEAD = WARPS * RING;     // parts of units that go on from the piece before, one for each warp
  static constexpr int INFO = HEAD + WARPS * PART;
  static constexpr int TOTAL = INFO + WARPS * 2 * 32;
  static_assert(PART <= RING, "the other parts lie over the rings");
};

__device__ __forceinline__ int tiles16(int start, int seq) { return (start % BLOCK + seq + BLOCK - 1) / BLOCK; }

// What a unit weighs on the line; `step` > 1: rounded up to whole pieces.
__device__ __forceinline__ int unit_weight(int start, int seq, int step) {
  const int w = UNIT_WEIGHT + start / BLOCK + TAIL_WEIGHT * tiles16(start, seq);
  return step == 1 ? w : quotient(w + step - 1, step) * step;
}

// A position that does not fit gives -1 (no weight): its sequence is left out.
__device__ __forceinline__ int position_of(const AttnParams& p, int b) {
  const int start = p.start_dev ? __ldcg(p.start_dev + static_cast<int64_t>(b) * p.start_step) : p.start_pos;
  const int64_t end = static_cast<int64_t>(start) + p.seq;
  return start < 0 || end > static_cast<int64_t>(p.num_blocks) * BLOCK || (p.cos_t && end > p.table_rows) ? -1 : start;
}

// A warp's part of one unit.
struct Segment {
  int b, kvh, rb, start;
  int t16_lo, t16_hi, lo, hi;  // 16-bit tiles and blocks
  int first, last;             // the warps whose pieces the unit lies in
};

struct PartInfo {  // what a warp left in shared memory
  int valid, b, kvh, rb, first, last;
};

// Merged rows of a unit: lane 4r + q has row 4g + q, columns 8n + r.
template <int D, int NG>
struct Merged {
  float m[NG], l[NG];
  float o[NG][D / 8];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      m[g] = -INFINITY, l[g] = 0.f;
#pragma unroll
      for (int n = 0; n < D / 8; ++n) o[g][n] = 0.f;
    }
  }
  __device__ __forceinline__ void fold(const float2 (&ml)[NG], const float (&v)[NG][D / 8]) {
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const float mn = fmaxf(m[g], ml[g].x);
      const float base = mn == -INFINITY ? 0.f : mn;  // nothing but rows without a key so far
      // by the roots of the factors: a denominator can count where the factor itself is below fp32's range
      const float ra = exp2_approx(0.5f * (m[g] - base)), re = exp2_approx(0.5f * (ml[g].x - base));
      const float a = ra * ra, e = re * re;
      l[g] = l[g] * ra * ra + ml[g].y * re * re;
#pragma unroll
      for (int n = 0; n < D / 8; ++n) o[g][n] = o[g][n] * a + v[g][n] * e;
      m[g] = mn;
    }
  }
};

// RAGGED: every sequence has a position of its own.
template <int DT, int FMT, int D, int NG, bool RAGGED>
__global__ void __launch_bounds__(THREADS, Smem<D, NG>::CTAS_SM) kv8_attention_kernel(const AttnParams p) {
  extern __shared__ __align__(128) uint8_t smem[];
  using S = Smem<D, NG>;
  constexpr int ROWS = S::ROWS;
  using T = typename Dt<DT>::T;
  constexpr int C16 = D / 8;
  constexpr int H = D / 64;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int r = lane >> 2, q = lane & 3;
  const int per_b = p.num_kv_heads * p.n_rb;
  const int me = blockIdx.x * WARPS + warp;
  PartInfo* info = reinterpret_cast<PartInfo*>(smem + S::INFO);  // [WARPS][2]
  uint8_t* ring = smem + warp * S::RING;
  const uint32_t ring_u = smem_u32(ring);
  pdl_wait();

  // the line and this warp's piece (all warps do the same sums). `step` > 1: units are rounded up to whole CTAs
  const int common = RAGGED ? 0 : position_of(p, 0);
  const int n_units = p.batch * per_b, ctas = gridDim.x;
  int total, piece, step;
  bool bad = false;
  if constexpr (!RAGGED) {
    bad = common < 0;
    const int w = bad ? 0 : unit_weight(common, p.seq, 1);
    total = w * n_units;
    piece = quotient(total + ctas * WARPS - 1, ctas * WARPS);
    step = 1;
    if (n_units <= ctas) {
      // A unit in CTAs of its own begins at once, and in one CTA is merged without leaving the SM; equal pieces balance
      // better, but end with a merge through L2 that takes as long as SPLIT_COST weights on an SM. 64 sequences of 4
      // kv heads (256 units) at 511: 15.1 us in equal pieces, 9.6 us with a CTA for each unit; at 8184 52 and 55 us.
      // Several CTAs for a unit pay where they save a warp more than MERGE_COST weights.
      int own = max(PIECE_MIN, quotient(w + p.most_ctas * WARPS - 1, p.most_ctas * WARPS));
      const int alone = (w + WARPS - 1) / WARPS;
      if (alone <= own + MERGE_COST) own = max(PIECE_MIN, alone);
      const int per_unit = quotient(w + own * WARPS - 1, own * WARPS);
      const int sms = ctas / S::CTAS_SM;
      if (quotient(n_units * per_unit + sms - 1, sms) * (own * WARPS) <= quotient(total, sms) + S::SPLIT_COST) {
        piece = own;
        step = own * WARPS;
        total = n_units * per_unit * step;
      }
    }
  } else {
    int exact = 0, padded = 0;
    for (int b = lane; b < p.batch; b += 32) {
      const int s = position_of(p, b);
      bad |= s < 0;
      exact += s < 0 ? 0 : unit_weight(s, p.seq, 1);
      padded += s < 0 ? 0 : unit_weight(s, p.seq, WARPS * PIECE_MIN);
    }
    exact = __reduce_add_sync(0xffffffffu, exact) * per_b;
    padded = __reduce_add_sync(0xffffffffu, padded) * per_b;
    const bool whole = padded <= ctas * WARPS * PIECE_MIN;
    total = whole ? padded : exact;
    piece = whole ? PIECE_MIN : (exact + ctas * WARPS - 1) / (ctas * WARPS);
    step = whole ? WARPS * PIECE_MIN : 1;
  }
  if (__any_sync(0xffffffffu, bad)) {
    if (me == 0) record_device_error(TK_DEVERR_POSITION);
    // a sequence that is left out gives rows of NaN
    const int row_chunks = p.num_kv_heads * p.groups * C16;
    for (int64_t row = me; row < static_cast<int64_t>(p.batch) * p.seq; row += static_cast<int64_t>(ctas) * WARPS) {
      if (position_of(p, static_cast<int>(row / p.seq)) >= 0) continue;
      uint4* dst = reinterpret_cast<uint4*>(reinterpret_cast<T*>(p.out) + row * p.os);
      for (int c = lane; c < row_chunks; c += 32) dst[c] = make_uint4(0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu);
    }
  }
  if (static_cast<int64_t>(piece) * (blockIdx.x * WARPS) >= total) return;  // nothing for the whole CTA
  const int from = static_cast<int>(min(static_cast<int64_t>(piece) * me, static_cast<int64_t>(total)));
  const int to = static_cast<int>(min(static_cast<int64_t>(from) + piece, static_cast<int64_t>(total)));

  // the sequence that `from` lies in, and where it begins
  int b = 0, at = 0;
  if (from >= to) {
  } else if constexpr (!RAGGED) {
    const int w = unit_weight(common, p.seq, step) * per_b;
    b = quotient(from, w);
    at = b * w;
  } else {
    for (int b0 = 0;; b0 += 32) {
      const int s = b0 + lane < p.batch ? position_of(p, b0 + lane) : -1;
      const int mine = s < 0 ? 0 : unit_weight(s, p.seq, step) * per_b;
      int upto = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
      }
      const uint32_t past = __ballot_sync(0xffffffffu, at + upto > from);
      if (past) {
        const int i = __ffs(past) - 1;
        b = b0 + i;
        at += __shfl_sync(0xffffffffu, upto - mine, i);
        break;
      }
      at += __shfl_sync(0xffffffffu, upto, 31);
    }
  }

  auto token_of = [&](int row) { return p.seq == 1 ? 0 : quotient(row, p.groups); };
  int here = from;
  auto next_segment = [&](Segment& g) {  // false: the piece is done
    if (here >= to) return false;
    int start, w;
    for (;;) {
      start = RAGGED ? position_of(p, b) : common;
      w = start < 0 ? 0 : unit_weight(start, p.seq, step);
      if (here < at + w * per_b) break;
      at += w * per_b;  // a sequence without a valid position has no weight
      ++b;
    }
    const int y = quotient(here - at, w), unit = at + y * w;
    const int n8 = start / BLOCK, n16 = tiles16(start, p.seq), w16 = TAIL_WEIGHT * n16;
    const int lo_w = max(here - unit - UNIT_WEIGHT, 0), hi_w = max(min(to - unit, w) - UNIT_WEIGHT, 0);
    here = min(to, unit + w);
    g.b = b;
    g.kvh = p.n_rb == 1 ? y : quotient(y, p.n_rb);
    g.rb = y - g.kvh * p.n_rb;
    g.start = start;
    // 16-bit tiles whose first weight lies in the piece, then blocks
    g.t16_lo = min(n16, (lo_w + TAIL_WEIGHT - 1) / TAIL_WEIGHT);
    g.t16_hi = min(n16, (hi_w + TAIL_WEIGHT - 1) / TAIL_WEIGHT);
    g.lo = min(n8, max(lo_w - w16, 0));
    g.hi = min(n8, max(hi_w - w16, 0));
    g.first = quotient(unit, piece);
    g.last = quotient(unit + w - 1, piece);
    return true;
  };

  // slot j of a segment's ring: the keys and the values of its 16-bit tiles, then its blocks
  auto issue = [&](const Segment& g, int j) {
    const int64_t bh = static_cast<int64_t>(g.b) * p.num_kv_heads + g.kvh;
    const uint32_t dst = ring_u + (j % S::STAGES) * S::STAGE;
    const int n16 = 2 * (g.t16_hi - g.t16_lo), t = g.lo + j - n16;
    if (j < n16) {
      // the open block's rows from the tail, the call's own (not rotated yet) from its tensors
      const int open = g.start % BLOCK, row0 = (g.t16_lo + j / 2) * BLOCK - open;  // the call's row of the first token
      const T* old = reinterpret_cast<const T*>(p.tail) + (bh * 2 + (j & 1)) * (BLOCK * D);
      const int64_t stride = j & 1 ? p.vs : p.ks;
      const T* fresh = reinterpret_cast<const T*>(j & 1 ? p.v : p.k) + static_cast<int64_t>(g.b) * p.seq * stride +
                       static_cast<int64_t>(g.kvh) * D;
      const int rows = min(BLOCK, p.seq - row0);
#pragma unroll 1
      for (int idx = lane; idx < rows * C16; idx += 32) {
        const int row = idx / C16, c = idx % C16, s = row0 + row;
        cp_async16(dst + tile_off<D>(row, c), (s < 0 ? old + row * D : fresh + s * stride) + c * 8);
      }
    } else if (t < g.hi) {
      const int64_t block = (bh * p.num_blocks + t) * S::HALF + lane * 16;
#pragma unroll
      for (int i = 0; i < S::HALF / 512; ++i) cp_async16(dst + lane * 16 + i * 512, p.kc + block + i * 512);
#pragma unroll
      for (int i = 0; i < S::HALF / 512; ++i) cp_async16(dst + S::HALF + lane * 16 + i * 512, p.vc + block + i * 512);
    }
    cp_async_commit();
  };
  auto load_scale = [&](const Segment& g, int t) {
    const int64_t bh = static_cast<int64_t>(g.b) * p.num_kv_heads + g.kvh;
    return t + lane < g.hi ? __ldcg(reinterpret_cast<const float2*>(p.scales) + bh * p.num_blocks + t + lane)
                           : make_float2(0.f, 1.f);
  };

  Segment g;
  bool more = next_segment(g);
  float2 sc = make_float2(0.f, 1.f);
  uint4 q_raw[NG][H][2];  // this lane's share of query rows 4g + r / 2
  auto begin = [&]() {    // what a unit needs first, all in flight at once
#pragma unroll 1
    for (int j = 0; j < S::STAGES - 1; ++j) issue(g, j);
    sc = load_scale(g, g.lo);
#pragma unroll
    for (int cg = 0; cg < NG; ++cg) {
      const int gr = g.rb * ROWS + 4 * cg + (r >> 1), s = token_of(gr), head = g.kvh * p.groups + gr - s * p.groups;
      const T* row = reinterpret_cast<const T*>(p.q) + (static_cast<int64_t>(g.b) * p.seq + s) * p.qs +
                     static_cast<int64_t>(head) * D;
#pragma unroll
      for (int h = 0; h < H; ++h)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          q_raw[cg][h][e] = gr < p.rows ? __ldcg(reinterpret_cast<const uint4*>(row) + 8 * h + 2 * q + e)
                                        : make_uint4(0, 0, 0, 0);
    }
  };
  if (more) begin();
  if (lane == 0) info[2 * warp].valid = info[2 * warp + 1].valid = 0;

  auto store = [&](const Merged<D, NG>& mg, int b_, int kvh_, int rb_) {
#pragma unroll
    for (int cg = 0; cg < NG; ++cg) {
      const int row = rb_ * ROWS + 4 * cg + q;
      const float inv = 1.f / mg.l[cg];
      const int s = token_of(row), head = kvh_ * p.groups + row - s * p.groups;
      T* dst = reinterpret_cast<T*>(p.out) + (static_cast<int64_t>(b_) * p.seq + s) * p.os +
               static_cast<int64_t>(head) * D + (r & 1 ? 8 + r - 1 : r);
#pragma unroll
      for (int n = 0; n < D / 16; ++n) {  // neighbouring columns lie in neighbouring r: a pair for each lane
        const float v0 = mg.o[cg][2 * n] * inv, v1 = mg.o[cg][2 * n + 1] * inv;
        const float other = __shfl_xor_sync(0xffffffffu, r & 1 ? v0 : v1, 4);
        if (row < p.rows)
          *reinterpret_cast<uint32_t*>(dst + 16 * n) = r & 1 ? pack2<DT>(other, v1) : pack2<DT>(v0, other);
      }
    }
  };

  while (more) {
    const int64_t bh = static_cast<int64_t>(g.b) * p.num_kv_heads + g.kvh;
    // query rows: rotated, brought to the f16 range; even lanes r take f16(q), odd ones the remainder
    uint32_t qf[NG][H * 4][2];
    float cq[NG];
    int qpos[NG];
#pragma unroll
    for (int cg = 0; cg < NG; ++cg) {
      const int gr = g.rb * ROWS + 4 * cg + (r >> 1);
      const int pos = gr < p.rows ? g.start + token_of(gr) : -1;  // a padding row sees no key of the 16-bit tiles, and
      float f[H][16];                                             // its zeros harm nothing in the others
      float amax = 0.f;
#pragma unroll
      for (int h = 0; h < H; ++h)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint4 x = q_raw[cg][h][e];
          const uint32_t w[4] = {x.x, x.y, x.z, x.w};
          float cc[4] = {1.f, 1.f, 1.f, 1.f}, ss[4] = {0.f, 0.f, 0.f, 0.f};
          if (p.cos_t && pos >= 0) {
            const int64_t ang = static_cast<int64_t>(pos) * (D / 2) + (8 * h + 2 * q + e) * 4;
            const float4 a = __ldg(reinterpret_cast<const float4*>(p.cos_t + ang));
            const float4 d = __ldg(reinterpret_cast<const float4*>(p.sin_t + ang));
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
#pragma unroll
      for (int h = 0; h < H; ++h)
#pragma unroll
        for (int i = 0; i < 16; ++i) amax = fmaxf(amax, fabsf(f[h][i]));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
      const float up = to_f16_range(__float_as_uint(amax));
      // after the products lane 4r + q has row q, whose factor and position are in the lanes with r = 2q
      cq[cg] = __shfl_sync(0xffffffffu, p.scale_log2 / up, 8 * q);
      qpos[cg] = __shfl_sync(0xffffffffu, pos, 8 * q);
#pragma unroll
      for (int h = 0; h < H; ++h)
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            uint32_t hi, lo;
            split2(f[h][4 * t + 2 * e] * up, f[h][4 * t + 2 * e + 1] * up, hi, lo);
            qf[cg][h * 4 + t][e] = r & 1 ? lo : hi;
          }
    }

    Rows<D, NG> st;
#pragma unroll
    for (int cg = 0; cg < NG; ++cg) {
      st.m[cg] = -INFINITY;
      st.l[cg] = 0.f;
#pragma unroll
      for (int n = 0; n < D / 16; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) st.o[cg][n][i] = 0.f;
    }

    int j = 0;  // the slot that is read next; slots up to j + STAGES - 2 are on their way
    const int open = g.start % BLOCK, n8 = g.start / BLOCK;
#pragma unroll 1
    for (int t = g.t16_lo; t < g.t16_hi; ++t, j += 2) {  // the open block and the new rows
      uint8_t* ktile = ring + (j % S::STAGES) * S::STAGE;
      uint8_t* vtile = ring + ((j + 1) % S::STAGES) * S::STAGE;
      const int n_rows = min(BLOCK, open + p.seq - t * BLOCK);
      const int row0 = t == 0 ? open : 0;  // the first row that the call brings
      cp_async_wait<S::STAGES - 3>();  // both slots
      __syncwarp();
#pragma unroll 1
      for (int idx = row0 * C16 + lane; idx < BLOCK * C16; idx += 32) {  // rotate its keys, clear what is behind them
        const int row = idx / C16, c = idx % C16;
        uint4* kx = reinterpret_cast<uint4*>(ktile + tile_off<D>(row, c));
        if (row >= n_rows) {
          *kx = make_uint4(0, 0, 0, 0);
          *reinterpret_cast<uint4*>(vtile + tile_off<D>(row, c)) = make_uint4(0, 0, 0, 0);
        } else if (p.cos_t) {
          const int64_t ang = (static_cast<int64_t>(n8 + t) * BLOCK + row) * (D / 2) + c * 4;
          rope_chunk<DT>(*kx, p.cos_t + ang, p.sin_t + ang);
        }
      }
      __syncwarp();
      uint32_t km = 0, vm = 0;
#pragma unroll 4
      for (int i = 0; i < C16; ++i) {  // any order of the tile's chunks
        const uint4 kx = *reinterpret_cast<const uint4*>(ktile + (lane + 32 * i) * 16);
        const uint4 vx = *reinterpret_cast<const uint4*>(vtile + (lane + 32 * i) * 16);
        km = amax2(amax2(amax2(amax2(km, kx.x), kx.y), kx.z), kx.w);
        vm = amax2(amax2(amax2(amax2(vm, vx.x), vx.y), vx.z), vx.w);
      }
      km = amax2_warp(km);
      vm = amax2_warp(vm);
      // A token that is not finite makes the rows that see it NaN: its scores are. One token's rows see all of the tile.
      const bool broken = max(km, vm) >= not_finite_bits<DT>();
      if (broken && p.seq > 1) {
        // It must not reach the rows that do not see it, neither as 0 * NaN nor by the tile's range: its key becomes NaN,
        // which the mask hides from those rows, its values 0.
        uint32_t bad = 0;
#pragma unroll 1
        for (int idx = lane; idx < BLOCK * C16; idx += 32) {
          const uint32_t off = tile_off<D>(idx / C16, idx % C16);
          if (not_finite<DT>(*reinterpret_cast<const uint4*>(ktile + off)) ||
              not_finite<DT>(*reinterpret_cast<const uint4*>(vtile + off)))
            bad |= 1u << (idx / C16);
        }
        bad = __reduce_or_sync(0xffffffffu, bad);
        km = vm = 0;
#pragma unroll 1
        for (int idx = lane; idx < BLOCK * C16; idx += 32) {
          uint4* kx = reinterpret_cast<uint4*>(ktile + tile_off<D>(idx / C16, idx % C16));
          uint4* vx = reinterpret_cast<uint4*>(vtile + tile_off<D>(idx / C16, idx % C16));
          if (bad >> (idx / C16) & 1) {
            *kx = make_uint4(0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu);
            *vx = make_uint4(0, 0, 0, 0);
          } else {
            km = amax2(amax2(amax2(amax2(km, kx->x), kx->y), kx->z), kx->w);
            vm = amax2(amax2(amax2(amax2(vm, vx->x), vx->y), vx->z), vx->w);
          }
        }
        km = amax2_warp(km);
        vm = amax2_warp(vm);
        __syncwarp();
      }

      const float fk = DT == TK_F16 ? 1.f : to_f16_range(km << 16), fv = value_factor<DT>(vm);
      auto to_half = [](uint32_t w, float f) -> uint32_t {
        if constexpr (DT == TK_F16) {
          return h2_u32(__hmul2(u32_h2(w), __float2half2_rn(f)));
        } else {
          const float2 v = unpack2<DT>(w);
          return h2_u32(__floats2half2_rn(v.x * f, v.y * f));
        }
      };
      float sk1[NG][1];
#pragma unroll
      for (int cg = 0; cg < NG; ++cg)
        sk1[cg][0] = broken && p.seq == 1 ? __uint_as_float(0x7fc00000u) : cq[cg] / fk;
      const float lsv1[1] = {-__log2f(fv)}, isv1[1] = {fv};
      attend_tiles<D, NG, 1, true, DT == TK_BF16>(
          st, qf, sk1, lsv1, isv1, lane,
          [&](int, int jj, int h, uint32_t (&w)[8]) {
            const int row = 8 * (r >> 1) + 2 * jj + (r & 1);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const uint4 x = *reinterpret_cast<const uint4*>(ktile + tile_off<D>(row, 8 * h + 2 * q + e));
              w[4 * e] = DT == TK_F16 ? x.x : to_half(x.x, fk);
              w[4 * e + 1] = DT == TK_F16 ? x.y : to_half(x.y, fk);
              w[4 * e + 2] = DT == TK_F16 ? x.z : to_half(x.z, fk);
              w[4 * e + 3] = DT == TK_F16 ? x.w : to_half(x.w, fk);
            }
          },
          [&](int, int m, uint32_t (&w)[8]) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              uint32_t x[4];
              load_column_tokens<D>(smem_u32(vtile), 2 * m + e, lane, x);
#pragma unroll
              for (int i = 0; i < 4; ++i) w[4 * e + i] = to_half(x[i], fv);
            }
          },
          [&](int cg, int token) { return (n8 + t) * BLOCK + token <= qpos[cg]; });

      if (p.seq == 1 && g.rb == 0) {  // the append of a decode step
        T* to_row = reinterpret_cast<T*>(p.tail) + bh * 2 * BLOCK * D;
        if (open < BLOCK - 1) {
          for (int c = lane; c < 2 * C16; c += 32) {
            const bool val = c >= C16;
            const int cc = val ? c - C16 : c;
            *(reinterpret_cast<uint4*>(to_row + ((val ? BLOCK : 0) + open) * D) + cc) =
                *reinterpret_cast<const uint4*>((val ? vtile : ktile) + tile_off<D>(open, cc));
          }
        } else {
          const int64_t block = bh * p.num_blocks + n8;
          const float sk = encode_keys<DT, FMT, D>(p.kc + block * S::HALF, lane, [&](int tok, int c) {
            return *reinterpret_cast<const uint4*>(ktile + tile_off<D>(tok, c));
          }, [](uint4&, int, int) {});
          const float sv = encode_values<DT, FMT, D>(p.vc + block * S::HALF, lane, smem_u32(vtile), vm);
          if (lane == 0) reinterpret_cast<float2*>(p.scales)[block] = make_float2(sk, sv);
        }
      }
      __syncwarp();  // both slots are written again
#pragma unroll 1
      for (int i = S::STAGES - 1; i <= S::STAGES; ++i) issue(g, j + i);
    }

    // complete blocks, PAIR of them in a step; lane i keeps the scales of the i-th block of each 32
    float lv_l = 0.f, iv_l = 0.f;
    auto blocks = [&](auto count, int t) {
      constexpr int N = decltype(count)::value;
      const int i = (t - g.lo) & 31;
      if (i == 0) {
        if (t > g.lo) sc = load_scale(g, t);
        lv_l = __log2f(sc.y);
        iv_l = 1.f / sc.y;
      }
      issue(g, j + S::STAGES - 1);
      cp_async_wait<S::STAGES - N>();
      __syncwarp();  // every lane's copies of the blocks have landed
      float sk[NG][N], lsv[N], isv[N];
#pragma unroll
      for (int u = 0; u < N; ++u) {
        const float x = __shfl_sync(0xffffffffu, sc.x, i + u);
#pragma unroll
        for (int cg = 0; cg < NG; ++cg) sk[cg][u] = cq[cg] * x;
        lsv[u] = __shfl_sync(0xffffffffu, lv_l, i + u);
        isv[u] = __shfl_sync(0xffffffffu, iv_l, i + u);
      }
      const uint8_t* slot[N];
#pragma unroll
      for (int u = 0; u < N; ++u) slot[u] = ring + ((j + u) % S::STAGES) * S::STAGE + lane * 16;
      attend_tiles<D, NG, N, false, DT == TK_BF16>(
          st, qf, sk, lsv, isv, lane,
          [&](int u, int jj, int h, uint32_t (&w)[8]) {
            const uint4 x = *reinterpret_cast<const uint4*>(slot[u] + (jj * H + h) * 512);
            decode4<FMT>(x.x, w[0], w[1]);
            decode4<FMT>(x.y, w[2], w[3]);
            decode4<FMT>(x.z, w[4], w[5]);
            decode4<FMT>(x.w, w[6], w[7]);
          },
          [&](int u, int m, uint32_t (&w)[8]) {
            const uint4 x = *reinterpret_cast<const uint4*>(slot[u] + S::HALF + m * 512);
            decode4<FMT>(x.x, w[0], w[1]);
            decode4<FMT>(x.y, w[2], w[3]);
            decode4<FMT>(x.z, w[4], w[5]);
            decode4<FMT>(x.w, w[6], w[7]);
          },
          [](int, int) { return true; });
      __syncwarp();  // the slots are written again by the next copies
      if constexpr (N == 2) issue(g, j + S::STAGES);
      j += N;
    };
    int t = g.lo;
    if constexpr (S::PAIR == 2) {
#pragma unroll 1
      for (; t + 1 < g.hi; t += 2) blocks(std::integral_constant<int, 2>(), t);
    }
#pragma unroll 1
    for (; t < g.hi; ++t) blocks(std::integral_constant<int, 1>(), t);

    // the next unit's first copies, then this unit's rows
    const Segment done = g;
    more = next_segment(g);
    if (more) begin();

    Merged<D, NG> mg;
#pragma unroll
    for (int cg = 0; cg < NG; ++cg) {
      mg.m[cg] = st.m[cg];
      mg.l[cg] = st.l[cg];
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) mg.l[cg] += __shfl_xor_sync(0xffffffffu, mg.l[cg], o);
#pragma unroll
      for (int n = 0; n < D / 16; ++n) {
        mg.o[cg][2 * n] = st.o[cg][n][0] + st.o[cg][n][1];
        mg.o[cg][2 * n + 1] = st.o[cg][n][2] + st.o[cg][n][3];
      }
    }
    if (done.first == done.last) {
      store(mg, done.b, done.kvh, done.rb);
    } else {
      // a unit that goes on from the piece before is this warp's first; any other is its last, when the ring is free
      const int k = me == done.first;
      uint8_t* part = k ? ring : smem + S::HEAD + warp * S::PART;
#pragma unroll
      for (int cg = 0; cg < NG; ++cg) {
#pragma unroll
        for (int n = 0; n < D / 8; ++n)
          *reinterpret_cast<float*>(part + ((cg * (D / 8) + n) * 32 + lane) * 4) = mg.o[cg][n];
        if (r == 0)
          *reinterpret_cast<float2*>(part + ROWS * D * 4 + (4 * cg + q) * 8) = make_float2(mg.m[cg], mg.l[cg]);
      }
      if (lane == 0) info[2 * warp + k] = PartInfo{1, done.b, done.kvh, done.rb, done.first, done.last};
    }
  }
  pdl_launch_dependents();
  __syncthreads();

  // the parts of a unit in this CTA: merged by the warp in which the unit begins; those of the unit that goes on from
  // the CTA before by a warp in which none begins, if there is one
  const int cta = blockIdx.x;
  int head_by = 0;
#pragma unroll
  for (int w = WARPS - 1; w >= 0; --w)
    if (!info[2 * w + 1].valid) head_by = w;
#pragma unroll 1
  for (int k = 1; k >= 0; --k) {
    const int w0 = k ? warp : 0;  // where the unit's parts begin
    const PartInfo u = info[2 * w0 + k];
    if (!u.valid || (k == 0 && warp != head_by)) continue;
    Merged<D, NG> mg;
    mg.clear();
    for (int w = w0; w < WARPS; ++w) {
      const int kk = w == w0 ? k : 0;
      if (w > w0 && blockIdx.x * WARPS + w > u.last) break;
      const uint8_t* part = kk ? smem + w * S::RING : smem + S::HEAD + w * S::PART;
      float2 ml[NG];
      float v[NG][D / 8];
#pragma unroll
      for (int cg = 0; cg < NG; ++cg) {
        ml[cg] = *reinterpret_cast<const float2*>(part + ROWS * D * 4 + (4 * cg + q) * 8);
#pragma unroll
        for (int n = 0; n < D / 8; ++n)
          v[cg][n] = *reinterpret_cast<const float*>(part + ((cg * (D / 8) + n) * 32 + lane) * 4);
      }
      mg.fold(ml, v);
    }
    const int c_first = u.first / WARPS, c_last = u.last / WARPS;
    if (c_first != c_last) {
      auto slot_of = [&](int c) { return 2 * static_cast<int64_t>(c) + (c == c_first); };
      auto put = [&](int c) {
        const int64_t slot = slot_of(c);
#pragma unroll
        for (int cg = 0; cg < NG; ++cg) {
          if (r == 0) p.part_ml[(slot * NG + cg) * 4 + q] = make_float2(mg.m[cg], mg.l[cg]);
#pragma unroll
          for (int n = 0; n < D / 8; ++n) p.part_o[((slot * NG + cg) * (D / 8) + n) * 32 + lane] = mg.o[cg][n];
        }
      };
      auto arrive = [&](int* counter, int count) {  // whether this warp is the last of `count`
        int last = 0;
        __syncwarp();
        if (lane == 0) {
          __threadfence();
          last = atomicAdd(counter, 1) == count - 1;
          if (last) {
            *counter = 0;
            __threadfence();
          }
        }
        last = __shfl_sync(0xffffffffu, last, 0);
        __syncwarp();
        return last != 0;
      };
      auto gather = [&](int count, auto cta_of) {  // parts of CTAs cta_of(0 .. count - 1), in this order
        constexpr int AHEAD = 256 / (D * NG);
        mg.clear();
#pragma unroll 1
        for (int i0 = 0; i0 < count; i0 += AHEAD) {
          float2 ml[AHEAD][NG];
          float v[AHEAD][NG][D / 8];
#pragma unroll
          for (int i = 0; i < AHEAD; ++i) {
            const int64_t slot = slot_of(cta_of(min(i0 + i, count - 1)));
#pragma unroll
            for (int cg = 0; cg < NG; ++cg) {
              ml[i][cg] = __ldcg(p.part_ml + (slot * NG + cg) * 4 + q);
#pragma unroll
              for (int n = 0; n < D / 8; ++n)
                v[i][cg][n] = __ldcg(p.part_o + ((slot * NG + cg) * (D / 8) + n) * 32 + lane);
            }
          }
#pragma unroll
          for (int i = 0; i < AHEAD; ++i)
            if (i0 + i < count) mg.fold(ml[i], v[i]);
        }
      };
      const int g_lo = c_first / GROUP, g_hi = c_last / GROUP, mine = cta / GROUP;
      auto leader = [&](int grp) { return max(c_first, grp * GROUP); };  // the group's parts end up in its slot
      const int c_lo = leader(mine), n_in = min(c_last, mine * GROUP + GROUP - 1) - c_lo + 1;
      put(cta);
      if (n_in > 1) {
        if (!arrive(p.counters + slot_of(c_lo), n_in)) continue;
        gather(n_in, [&](int i) { return c_lo + i; });
      }
      if (g_lo != g_hi) {
        if (n_in > 1) put(c_lo);
        if (!arrive(p.counters + 2 * gridDim.x + c_first, g_hi - g_lo + 1)) continue;
        gather(g_hi - g_lo + 1, [&](int i) { return leader(g_lo + i); });
      }
    }
    store(mg, u.b, u.kvh, u.rb);
  }
}

// The arrival counters come first, then two slots of rows for each CTA: one size for all shapes of a head_dim, so
// calls that follow one another on a stream can share one workspace.
int64_t counter_bytes(int sm_count) { return (int64_t(4) * sm_count * 3 * sizeof(int) + 255) / 256 * 256; }
template <int D, int NG>
int64_t parts_bytes(int sm_count) {
  return int64_t(Smem<D, NG>::CTAS_SM) * sm_count * 2 * Smem<D, NG>::PART;
}
int64_t workspace_bytes_for(int head_dim, int sm_count) {
  sm_count = std::max(sm_count, 1);
  return counter_bytes(sm_count) + (head_dim == 64 ? std::max(parts_bytes<64, 1>(sm_count), parts_bytes<64, 2>(sm_count))
                                                   : std::max(parts_bytes<128, 1>(sm_count), parts_bytes<128, 2>(sm_count)));
}

template <int DT, int FMT, int D, int NG, bool RAGGED>
int launch(AttnParams& p, void* workspace, const DeviceInfo& dev, cudaStream_t st) {
  using S = Smem<D, NG>;
  auto kern = kv8_attention_kernel<DT, FMT, D, NG, RAGGED>;
  static bool configured[64] = {};
  if (!configured[dev.device]) {
    if (int rc = check_cuda(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, S::TOTAL),
                            "cudaFuncSetAttribute(kv8_attention)"))
      return rc;
    configured[dev.device] = true;
  }
  const int ctas = S::CTAS_SM * std::max(dev.sm_count, 1);
  p.n_rb = (p.rows + S::ROWS - 1) / S::ROWS;
  // the line of tiles is counted in 32 bits
  const int64_t units = int64_t(p.batch) * p.num_kv_heads * p.n_rb;
  const int64_t longest = UNIT_WEIGHT + p.num_blocks + int64_t(TAIL_WEIGHT) * (p.seq / BLOCK + 2) + WARPS * PIECE_MIN;
  if (units > INT32_MAX / longest) return fail_invalid("kv8_attention: too many query rows for one call");
  p.most_ctas = static_cast<int>(std::max<int64_t>(1, ctas / units));
  char* ws = static_cast<char*>(workspace);
  p.counters = reinterpret_cast<int*>(ws);
  ws += counter_bytes(dev.sm_count);
  p.part_ml = reinterpret_cast<float2*>(ws);
  ws += int64_t(ctas) * 2 * S::ROWS * sizeof(float2);
  p.part_o = reinterpret_cast<float*>(ws);
  return launch_kernel(kern, dim3(ctas), dim3(THREADS), S::TOTAL, st, 1, "kv8_attention", p);
}

template <int DT, int FMT, int D>
int launch(AttnParams& p, void* workspace, const DeviceInfo& dev, cudaStream_t st) {
  const bool ragged = p.start_dev && p.start_step;
  if (p.rows <= 4)
    return ragged ? launch<DT, FMT, D, 1, true>(p, workspace, dev, st) : launch<DT, FMT, D, 1, false>(p, workspace, dev, st);
  return ragged ? launch<DT, FMT, D, 2, true>(p, workspace, dev, st) : launch<DT, FMT, D, 2, false>(p, workspace, dev, st);
}

template <int DT, int FMT>
int launch(AttnParams& p, int head_dim, void* workspace, const DeviceInfo& dev, cudaStream_t st) {
  return head_dim == 64 ? launch<DT, FMT, 64>(p, workspace, dev, st) : launch<DT, FMT, 128>(p, workspace, dev, st);
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
  int64_t need = kv8::workspace_bytes_for(head_dim, di.sm_count);
  if (kv8::chunk_fits(batch, num_heads, num_kv_heads, seq, max_kv))
    need += kv8::chunk_workspace(batch, num_heads, num_kv_heads, head_dim, seq, max_kv, di.sm_count);
  return need;
}

extern "C" int tk_kv8_attention_launches(int batch, int num_heads, int num_kv_heads, int head_dim, int seq, int start_pos,
                                         int dtype) {
  using namespace tk;
  if (batch <= 0 || seq <= 0 || num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads) return 0;
  if (seq == 1) return 1;
  const int64_t len = int64_t(start_pos) + seq;
  if (start_pos < 0 || !kv8::chunk_fits(batch, num_heads, num_kv_heads, seq, len)) return 2;
  DeviceInfo di;
  if (current_device_info(&di)) return -1;
  return kv8::chunk_launches(batch, num_heads, num_kv_heads, head_dim, seq, len, dtype, di.sm_count) + 1;
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
  if (rows > INT32_MAX) return fail_invalid("kv8_attention: too many query rows for one call");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int64_t small = workspace_bytes_for(head_dim, di.sm_count);
  // with the position in device memory the length, and so the tiles, are not known here
  const bool chunk = !start_pos_device && chunk_fits(batch, num_heads, num_kv_heads, seq, int64_t(start_pos) + seq);
  const int64_t need = small + (chunk ? chunk_workspace(batch, num_heads, num_kv_heads, head_dim, seq,
                                                        int64_t(start_pos) + seq, di.sm_count) : 0);
  if (!workspace || workspace_bytes < need)
    return fail_invalid("kv8_attention: workspace missing or smaller than tk_kv8_attention_workspace()");
  if (!aligned16(workspace)) return fail_invalid("kv8_attention: workspace must be 16-byte aligned");
  if (chunk) {
    // behind the counters and parts of the other form, which have to stay as they are
    if (int rc = chunk_attention(c, q, q_tok_stride, k, k_tok_stride, v, v_tok_stride, cos_table, sin_table, out,
                                 out_tok_stride, batch, seq, num_heads, num_kv_heads, head_dim, start_pos,
                                 static_cast<char*>(workspace) + small, dtype, di.sm_count, st))
      return rc;
    return append(c, k, k_tok_stride, v, v_tok_stride, cos_table, sin_table, table_rows, batch, seq, num_kv_heads,
                  head_dim, start_pos, nullptr, 0, dtype, st);
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
  p.batch = batch;
  p.scale_log2 = static_cast<float>((1.0 / std::sqrt(double(head_dim))) * 1.4426950408889634);
  int rc;
  if (dtype == TK_F16)
    rc = format == TK_KV8_E4M3 ? launch<TK_F16, TK_KV8_E4M3>(p, head_dim, workspace, di, st)
                               : launch<TK_F16, TK_KV8_INT8>(p, head_dim, workspace, di, st);
  else
    rc = format == TK_KV8_E4M3 ? launch<TK_BF16, TK_KV8_E4M3>(p, head_dim, workspace, di, st)
                               : launch<TK_BF16, TK_KV8_INT8>(p, head_dim, workspace, di, st);
  if (rc || seq == 1) return rc;
  return append(c, k, k_tok_stride, v, v_tok_stride, cos_table, sin_table, table_rows, batch, seq, num_kv_heads,
                head_dim, start_pos, start_pos_device, start_pos_step, dtype, st);
}
