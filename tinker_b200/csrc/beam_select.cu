// One step of beam search: the best n of beams x vocabulary for every sequence.
//
//   c[b, k, v] = score[b, k] + logit[b, k, v] - logsumexp_v(logit[b, k, :])
//
// ordered by c, ties by the lower k * V + v. Within a beam the order is that of the logits themselves (exact), across
// beams that of c in fp64. A finished beam has one candidate, the end token at its score unchanged; everything else of
// it, and everything of a beam whose score is -inf or NaN, is -inf. A NaN logit counts as -inf, +inf as the largest
// finite value of the type; a beam without a finite logit is -inf throughout.
//
// Two launches, the logits are read once:
//   1. a CTA takes a segment of one row. The first vectors stay in registers (as they come, 16-bit pairs) and give a
//      reference m (their maximum) and a first threshold: of the threads' maxima each of the 8 warps takes its
//      ceil(n / 8)-th largest, and the least of those is a value that at least n elements reach. What exceeds it (some
//      2 n elements) is collected in shared memory and ranked by counting; what equals it fills up the rest in order
//      of index, found by a scan from the start (a masked vocabulary has thousands of equal values). The rest of the
//      segment streams by: an element costs a conversion, an FMA, one ex2 and an addition, and half a comparison with
//      the value of the n-th best so far; vectors that hold a larger one are put aside and, every STRIDE vectors,
//      ranked with the best n, which raises the threshold. Equal elements that come later lose in any case.
//      An exponential is 2^(x L - b) with L = log2 e and b = m L rounded; the sum is corrected by 2^(b - m L), the
//      rounding that all its terms share. Where the reference proves too far off (a masked beginning) or is above 2^20
//      (the rounding grows with it), the sum is taken again. A segment with a NaN or +inf, or with more candidates than
//      the lists hold, is done again in the plain way: cleaned, its maximum, the sum of e^(x - m), n rounds of a maximum
//      over (value, index).
//   2. a CTA for each sequence joins the segments' sums to a logsumexp for each beam, takes a threshold from the heads of
//      the segments' lists in the same way, walks each list down to it and ranks what it finds, with c in fp64.
// Sums are taken in an order that depends on element numbers alone, so equal rows give equal sums wherever they lie.
// For many rows bound by the first launch's order: its CTAs all fit at once and go through the same prologue (load,
// threshold, collect, rank) together, so that 57 % of the issue slots are filled and the logits come at 2.7 TB/s (256
// rows of 151936, a quarter finished: 28.5 us; the logits alone 8.9 us, the exponentials 7 us, all instructions 11 us;
// all live 38.4 us, fp32 53.7 us). For few by the latency of the two launches (4 rows of 32000: 9.4 us).
// Slow, not wrong: rows that do not begin on 16 bytes (an odd vocabulary, for 7 of 8 rows of 16-bit logits) are read
// element by element (256 rows of 50257: 33.4 us, of 50264: 25.7 us); a round of STRIDE steps with more than HITS vectors
// above the threshold (a masked beginning of 8192 16-bit logits before unmasked ones, steadily rising logits) sends the
// segment to the plain way (256 rows of 151936: 900 us).
#include <math.h>

#include <algorithm>
#include <string>

#include "tk_common.cuh"
#include "tk_host.h"

namespace tk {
namespace beam {

constexpr int THREADS = 256;
constexpr int WARPS = THREADS / 32;
constexpr int MAX_N = 64;
constexpr int CAP = 512;  // candidates that are ranked by counting
constexpr int HITS = 256;  // vectors that hold them
constexpr int STRIDE = 8;  // streamed vectors of a thread between two rankings
constexpr float L2E = 1.4426950408889634f;

template <int DT> struct Logit {
  using T = typename Dt<DT>::T;
  __device__ static __forceinline__ float to_f(T v) { return Dt<DT>::to_f(v); }
};
template <> struct Logit<TK_F32> {
  using T = float;
  __device__ static __forceinline__ float to_f(float v) { return v; }
};

struct Entry {
  float x;
  int idx;
};

struct Params {
  const void* logits;
  int64_t row_stride;
  const float* scores;
  const uint8_t* finished;
  int64_t eos;
  int beams, vocab, n, splits, segment;
  float2* part_ms;   // [rows, splits]: a reference m, sum of e^(x - m)
  Entry* part_top;   // [rows, splits, n], missing ones with idx -1
  float* out_scores;
  int64_t* out_beams;
  int64_t* out_tokens;
};

// Larger for the larger value; equal for equal values (-0 and 0 are).
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return u ^ (static_cast<uint32_t>(static_cast<int32_t>(u) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t k) {  // key 0 (none) gives NaN
  return __uint_as_float(k ^ (k >> 31 ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ uint64_t key_of(double x) {
  const uint64_t u = static_cast<uint64_t>(__double_as_longlong(x + 0.0));
  return u ^ (static_cast<uint64_t>(static_cast<int64_t>(u) >> 63) | 0x8000000000000000ull);
}

// The beam gives no candidates of its own: finished, or dead (score -inf or NaN).
__device__ __forceinline__ bool is_still(const Params& p, int row) {
  const float score = p.scores[row];
  const bool done = p.finished && p.finished[row];
  return done || !(score > -INFINITY);
}

// A key that at least n of the keys of the first `warps` warps' threads reach (0 if there are too few of them): see the
// head of this file. All threads call it.
__device__ __forceinline__ uint32_t reach_of(uint32_t mine, int n, int warps, uint32_t* warp_key) {
  const int lane = threadIdx.x & 31;
  uint32_t left = mine, kth = 0;
  const int rounds = warps > 0 ? (n + warps - 1) / warps : 33;
  for (int i = 0; i < min(rounds, 32); ++i) {
    kth = __reduce_max_sync(0xffffffffu, left);
    const uint32_t who = __ballot_sync(0xffffffffu, left == kth);
    if (lane == __ffs(who) - 1) left = 0;
  }
  if (lane == 0) warp_key[threadIdx.x >> 5] = kth;
  __syncthreads();
  if (rounds > 32) return 0;
  uint32_t t = warp_key[0];
#pragma unroll
  for (int w = 1; w < WARPS; ++w)
    if (w < warps) t = min(t, warp_key[w]);
  return t;
}

// Largest (key, ~index) over the CTA; all threads get it. `box` holds one value for each warp.
__device__ __forceinline__ ulonglong2 best_of(ulonglong2 v, ulonglong2* box) {
  auto better = [](ulonglong2 a, ulonglong2 b) { return a.x > b.x || (a.x == b.x && a.y > b.y); };
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const ulonglong2 u = make_ulonglong2(__shfl_xor_sync(0xffffffffu, v.x, o), __shfl_xor_sync(0xffffffffu, v.y, o));
    if (better(u, v)) v = u;
  }
  __syncthreads();  // the box may still be read from the round before
  if ((threadIdx.x & 31) == 0) box[threadIdx.x >> 5] = v;
  __syncthreads();
  v = box[0];
#pragma unroll
  for (int w = 1; w < WARPS; ++w)
    if (better(box[w], v)) v = box[w];
  return v;
}

struct ChunkSmem {
  float red[WARPS], red2[WARPS];
  uint32_t warp_key[WARPS];
  ulonglong2 box[WARPS];
  ulonglong2 cand2[CAP / 2];  // key << 32 | ~index: larger is better
  uint4 hit[HITS];
  int hit_at[HITS];
  int n_cand, n_hit;
  __device__ uint64_t* cand() { return reinterpret_cast<uint64_t*>(cand2); }
  __device__ float value(int i) { return value_of(static_cast<uint32_t>(cand()[i] >> 32)); }
  __device__ int index(int i) { return static_cast<int>(~static_cast<uint32_t>(cand()[i])); }
};

// A segment in the plain way, element tid, tid + THREADS, ... for a thread.
template <int DT>
__device__ __forceinline__ void plain_segment(const Params& p, const typename Logit<DT>::T* src, int lo, int hi,
                                              int64_t part, ChunkSmem& sm) {
  constexpr float TOP = DT == TK_F16 ? 65504.f : DT == TK_BF16 ? 3.3895313892515355e38f : 3.4028234663852886e38f;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  auto get = [&](int at) { return fminf(fmaxf(Logit<DT>::to_f(src[at]), -INFINITY), TOP); };  // fmaxf turns NaN into -inf
  float mx = -INFINITY;
#pragma unroll 1
  for (int at = lo + tid; at < hi; at += THREADS) mx = fmaxf(mx, get(at));
  for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  __syncthreads();
  if (lane == 0) sm.red[warp] = mx;
  __syncthreads();
  for (int w = 0; w < WARPS; ++w) mx = fmaxf(mx, sm.red[w]);
  const float m = mx == -INFINITY ? 0.f : mx;
  float sum = 0.f;
#pragma unroll 1
  for (int at = lo + tid; at < hi; at += THREADS) sum += exp2_approx((get(at) - m) * L2E);
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) sm.red2[warp] = sum;
  __syncthreads();
  sum = 0.f;
  for (int w = 0; w < WARPS; ++w) sum += sm.red2[w];
  if (tid == 0) p.part_ms[part] = make_float2(mx, sum);
  Entry* top = p.part_top + part * p.n;
  ulonglong2 last = make_ulonglong2(~0ull, ~0ull);
#pragma unroll 1
  for (int i = 0; i < p.n; ++i) {
    ulonglong2 v = make_ulonglong2(0, 0);
#pragma unroll 1
    for (int at = lo + tid; at < hi; at += THREADS) {
      const uint64_t k = key_of(get(at)), t = static_cast<uint32_t>(~at);
      if ((k < last.x || (k == last.x && t < last.y)) && (k > v.x || (k == v.x && t > v.y))) v = make_ulonglong2(k, t);
    }
    last = best_of(v, sm.box);
    if (tid == 0)
      top[i] = last.x ? Entry{value_of(static_cast<uint32_t>(last.x)), static_cast<int>(~static_cast<uint32_t>(last.y))}
                      : Entry{-INFINITY, -1};
  }
}

// The best min(n, c) of the c candidates, in order, to the front of the list; every other thread's view is the same
// after the call. At least n candidates: the n-th value is the new threshold.
__device__ __forceinline__ void rank_candidates(ChunkSmem& sm, int c, int n) {
  constexpr int EACH = CAP / THREADS;
  const int tid = threadIdx.x;
  if (tid == 0 && (c & 1)) sm.cand()[c] = 0;  // read in pairs
  __syncthreads();
  uint64_t k[EACH];
  int rank[EACH];
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    const int i = tid + THREADS * e;
    rank[e] = n;
    if (i < c) {
      k[e] = sm.cand()[i];
      rank[e] = 0;
#pragma unroll 4
      for (int o = 0; 2 * o < c; ++o) {
        const ulonglong2 x = sm.cand2[o];
        rank[e] += (x.x > k[e]) + (x.y > k[e]);
      }
    }
  }
  __syncthreads();
#pragma unroll
  for (int e = 0; e < EACH; ++e)
    if (rank[e] < n) sm.cand()[rank[e]] = k[e];
  if (tid == 0) sm.n_cand = min(c, n);
  __syncthreads();
}

// NV: vectors that stay in registers; STREAM: more follow. 64 registers leave four CTAs on an SM: while one waits for
// its loads or at a barrier, the others compute.
template <int DT, int NV, bool STREAM>
__global__ void __launch_bounds__(THREADS, 4) beam_chunk_kernel(const Params p) {
  using T = typename Logit<DT>::T;
  constexpr int VE = 16 / sizeof(T);  // elements of a vector
  constexpr int STEP = THREADS * VE;
  __shared__ ChunkSmem sm;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int row = blockIdx.y, split = blockIdx.x;
  if (tid == 0) sm.n_cand = sm.n_hit = 0;
  pdl_wait();
  pdl_launch_dependents();
  if (is_still(p, row)) return;
  const T* src = static_cast<const T*>(p.logits) + static_cast<int64_t>(row) * p.row_stride;
  const int lo = split * p.segment;
  const int hi = static_cast<int>(min(static_cast<int64_t>(p.vocab), static_cast<int64_t>(lo) + p.segment));
  const bool aligned = (reinterpret_cast<uintptr_t>(src) & 15) == 0;
  const int64_t part = static_cast<int64_t>(row) * p.splits + split;

  auto get = [](const uint4& v, int i) {
    if constexpr (DT == TK_F32) return reinterpret_cast<const float*>(&v)[i];
    else return Logit<DT>::to_f(reinterpret_cast<const T*>(&v)[i]);
  };
  // the vector at element `at`, -inf behind the segment; a thread has the same elements however the row lies
  auto load = [&](int64_t at) {
    if (aligned && at + VE <= hi) return __ldcs(reinterpret_cast<const uint4*>(src + at));
    uint4 v;
#pragma unroll
    for (int i = 0; i < VE; ++i) {
      const float x = at + i < hi ? Logit<DT>::to_f(src[at + i]) : -INFINITY;
      if constexpr (DT == TK_F32) reinterpret_cast<float*>(&v)[i] = x;
      else reinterpret_cast<T*>(&v)[i] = Dt<DT>::from_f(x);
    }
    return v;
  };
  auto exceeds = [&](const uint4& v, float t) {
    if constexpr (DT == TK_F32) {
      return fmaxf(fmaxf(get(v, 0), get(v, 1)), fmaxf(get(v, 2), get(v, 3))) > t;
    } else {
      const auto* w = reinterpret_cast<const typename Dt<DT>::T2*>(&v);
      const float2 f = Dt<DT>::unpack(__hmax2(__hmax2(w[0], w[1]), __hmax2(w[2], w[3])));
      return fmaxf(f.x, f.y) > t;
    }
  };
  auto add = [&](float& sum, const uint4& v, float nb) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (DT == TK_F32) {
        sum += exp2_approx(fmaf(__uint_as_float(w[i]), L2E, nb));
      } else {
        float2 f;
        if constexpr (DT == TK_BF16) f = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
        else f = Dt<DT>::unpack(*reinterpret_cast<const typename Dt<DT>::T2*>(&w[i]));
        sum += exp2_approx(fmaf(f.x, L2E, nb));
        sum += exp2_approx(fmaf(f.y, L2E, nb));
      }
    }
  };
  auto push = [&](float x, int at) {
    const int slot = atomicAdd(&sm.n_cand, 1);
    if (slot < CAP) sm.cand()[slot] = static_cast<uint64_t>(key_of(x)) << 32 | static_cast<uint32_t>(~at);
  };
  auto put_aside = [&](const uint4& v, int at) {
    const int slot = atomicAdd(&sm.n_hit, 1);
    if (slot < HITS) {
      sm.hit[slot] = v;
      sm.hit_at[slot] = at;
    }
  };
  // the elements above t of the vectors put aside become candidates, one element for each thread
  auto sift = [&](float t) {
    __syncthreads();
    const int hits = min(sm.n_hit, HITS);
    for (int e = tid; e < hits * VE; e += THREADS) {
      const float x = Logit<DT>::to_f(reinterpret_cast<const T*>(sm.hit)[e]);
      if (x > t) push(x, sm.hit_at[e / VE] + e % VE);
    }
    __syncthreads();
  };

  uint4 raw[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) raw[j] = load(static_cast<int64_t>(lo) + STEP * j + tid * VE);
  uint4 ahead[2];
  if constexpr (STREAM) {
#pragma unroll
    for (int j = 0; j < 2; ++j) ahead[j] = load(static_cast<int64_t>(lo) + STEP * (NV + j) + tid * VE);
  }

  float mine, mx;  // the maximum; a NaN does not show in it
  if constexpr (DT == TK_F32) {
    mine = -INFINITY;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < VE; ++i) mine = fmaxf(mine, get(raw[j], i));
  } else {
    using T2 = typename Dt<DT>::T2;
    T2 m2 = Dt<DT>::pack(-INFINITY, -INFINITY);
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) m2 = __hmax2(m2, reinterpret_cast<const T2*>(&raw[j])[i]);
    const float2 f = Dt<DT>::unpack(m2);
    mine = fmaxf(f.x, f.y);
  }
  mx = mine;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  if (lane == 0) sm.red[warp] = mx;
  constexpr uint32_t LOWEST = 0x007fffffu;  // the key of -inf
  const int warps = min(WARPS, (hi - lo) / (32 * VE));  // those whose threads all have elements of their own
  float reach = value_of(max(reach_of(key_of(mine), p.n, warps, sm.warp_key), LOWEST));  // synchronises
  mx = sm.red[0];
#pragma unroll
  for (int w = 1; w < WARPS; ++w) mx = fmaxf(mx, sm.red[w]);
  // far below zero it may be the value of a mask: the sum is then taken relative to 1
  float ref = mx > -1000.f ? mx : 0.f, b = ref * L2E;
  float sum = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    add(sum, raw[j], -b);
    asm volatile("" : "+f"(sum));  // a vector at a time: all converted at once would take twice the registers
  }
  auto collect = [&]() {
    if (mine > reach) {
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (exceeds(raw[j], reach)) put_aside(raw[j], lo + STEP * j + tid * VE);
    }
    sift(reach);
  };
  collect();
  if (sm.n_hit > HITS || sm.n_cand > CAP) {
    // the best elements lie in few threads' hands (most of the vocabulary is masked): the n-th largest value itself,
    // bit by bit
    uint32_t t = 0;
#pragma unroll 1
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t probe = t | 1u << bit;
      int count = 0;
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < VE; ++i) count += key_of(get(raw[j], i)) >= probe && lo + STEP * j + tid * VE + i < hi;
      count = __reduce_add_sync(0xffffffffu, count);
      __syncthreads();
      if (lane == 0) sm.warp_key[warp] = count;
      __syncthreads();
      count = 0;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) count += static_cast<int>(sm.warp_key[w]);
      if (count >= p.n) t = probe;
    }
    reach = value_of(max(t, LOWEST));
    __syncthreads();
    if (tid == 0) sm.n_cand = sm.n_hit = 0;
    __syncthreads();
    collect();
  }
  const int above = sm.n_cand;
  bool plain = sm.n_hit > HITS;  // a NaN at most
  __syncthreads();
  if (above < p.n && !plain) {  // equal ones in order of index: vector by vector, thread by thread
    int need = p.n - above;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (need > 0) {
        const int at = lo + STEP * j + tid * VE;
        int mine_eq = 0;
#pragma unroll
        for (int i = 0; i < VE; ++i) mine_eq += get(raw[j], i) == reach && at + i < hi;
        int upto = mine_eq;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int v = __shfl_up_sync(0xffffffffu, upto, o);
          if (lane >= o) upto += v;
        }
        if (lane == 31) sm.warp_key[warp] = upto;
        __syncthreads();
        int before = upto - mine_eq, all = 0;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
          if (w < warp) before += static_cast<int>(sm.warp_key[w]);
          all += static_cast<int>(sm.warp_key[w]);
        }
#pragma unroll
        for (int i = 0; i < VE; ++i)
          if (get(raw[j], i) == reach && at + i < hi && before++ < need) push(reach, at + i);
        need -= all;
        __syncthreads();
      }
    }
  }
  plain |= sm.n_cand > CAP;
  if (!plain) rank_candidates(sm, sm.n_cand, p.n);

  if constexpr (STREAM) {
    const int steps = (hi - lo + STEP - 1) / STEP, full = aligned ? (hi - lo) / STEP : 0;
    const uint4* from = reinterpret_cast<const uint4*>(src + lo) + tid;
#pragma unroll 1
    for (int it = NV; it < steps && !plain;) {
      __syncthreads();  // the counters of the last round have been read
      if (tid == 0) sm.n_hit = 0;
      const float t = sm.value(p.n - 1);
      __syncthreads();
      const int stop = min(steps, it + STRIDE);
      const float nb = -b;
#pragma unroll 1
      for (; it < stop; it += 2) {
        uint4 v[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) v[e] = ahead[e];
        if (it + 3 < full) {
#pragma unroll
          for (int e = 0; e < 2; ++e) ahead[e] = __ldcs(from + (it + 2 + e) * THREADS);
        } else {
#pragma unroll
          for (int e = 0; e < 2; ++e) ahead[e] = load(static_cast<int64_t>(lo) + STEP * (it + 2 + e) + tid * VE);
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {  // what is behind the segment is -inf and adds nothing
          if (exceeds(v[e], t)) put_aside(v[e], lo + STEP * (it + e) + tid * VE);
          add(sum, v[e], nb);
        }
      }
      sift(t);
      plain = sm.n_hit > HITS || sm.n_cand > CAP;
      if (plain || sm.n_cand == p.n) continue;
      rank_candidates(sm, sm.n_cand, p.n);
      const float best = sm.value(0);
      if (best > ref + 16.f && best < INFINITY) {  // far above the reference: the sum goes by it from here on
        const float nb = best * L2E;
        sum *= exp2_approx(b - nb);
        ref = best;
        b = nb;
      }
    }
  }

  auto total = [&](float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (lane == 0) sm.red2[warp] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) v += sm.red2[w];
    __syncthreads();
    return v;
  };
  sum = total(sum);
  const float best = sm.n_cand > 0 && !plain ? sm.value(0) : INFINITY;
  if (plain || !(sum <= INFINITY) || !(best < INFINITY)) {  // the second is true of NaN
    plain_segment<DT>(p, src, lo, hi, part, sm);
    return;
  }
  if (best == -INFINITY) {
    ref = -INFINITY;
  } else if (sum == INFINITY || best < ref - 60.f || fabsf(ref) > 0x1p20f) {
    // The reference was too far off, or so large that the rounding of b alone takes the terms out of fp32's range (ref L
    // beyond 2^30: half a step of b is 64): once more with the maximum, subtracted before the product.
    sum = 0.f;
#pragma unroll 1
    for (int at = lo + tid * VE; at < hi; at += STEP) {
      const uint4 v = load(at);
#pragma unroll
      for (int i = 0; i < VE; ++i) sum += exp2_approx((get(v, i) - best) * L2E);
    }
    ref = best;
    sum = total(sum);
  } else {
    sum *= exp2_approx(-fmaf(ref, L2E, -b));
  }
  if (tid == 0) p.part_ms[part] = make_float2(ref, sum);
  Entry* top = p.part_top + part * p.n;
  for (int i = tid; i < p.n; i += THREADS)  // a segment shorter than n has fewer
    top[i] = i < sm.n_cand ? Entry{sm.value(i), sm.index(i)} : Entry{-INFINITY, -1};
}

// Candidate j of a still beam: the end token of a finished one first, then -inf at its lowest tokens.
__device__ __forceinline__ int still_token(const Params& p, bool done, int j) {
  if (!done) return j;
  if (j == 0) return static_cast<int>(p.eos);
  return j - 1 < p.eos ? j - 1 : j;
}

__global__ void __launch_bounds__(THREADS) beam_merge_kernel(const Params p) {
  extern __shared__ float4 beam[];  // [beams]: maximum, log of the sum, score, kind (0 live, 1 dead, 2 finished)
  __shared__ uint32_t warp_key[WARPS];
  __shared__ ulonglong2 box[WARPS];
  __shared__ uint64_t cand_key[CAP];
  __shared__ uint64_t cand_at[CAP];  // beam, then token
  __shared__ int n_cand;
  constexpr int FIRST = 8;  // candidates that a thread keeps in registers
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, b = blockIdx.x;
  if (tid == 0) n_cand = 0;
  pdl_wait();
  pdl_launch_dependents();
  const int per = p.splits * p.n;  // candidates of a beam (a still one has n)
  const int total = p.beams * per;
  const int2* top = reinterpret_cast<const int2*>(p.part_top) + static_cast<int64_t>(b) * total;
  // Candidate i is that of rank i / (beams * splits) in chunk (i / beams) % splits of beam i % beams, so that the
  // threads' maxima are spread over the beams and a threshold from them is high whatever their scores.
  const float beams_inv = 1.f / static_cast<float>(p.beams), splits_inv = 1.f / static_cast<float>(p.splits);
  auto split = [](int i, int d, float inv, int& rem) {  // i / d for i < 2^30
    int x = static_cast<int>(static_cast<float>(i) * inv);
    rem = i - x * d;
    while (rem >= d) ++x, rem -= d;  // off by one at most for small numbers, by a few for large ones
    while (rem < 0) --x, rem += d;
    return x;
  };
  auto place = [&](int i, int& k) {  // beam and number in its list
    int s;
    const int r = split(split(i, p.beams, beams_inv, k), p.splits, splits_inv, s);
    return s * p.n + r;
  };
  auto load = [&](int i) {
    int k;
    const int j = place(i, k);
    return __ldcg(top + k * per + j);
  };
  int2 raw[FIRST];
#pragma unroll
  for (int e = 0; e < FIRST; ++e) raw[e] = tid + THREADS * e < total ? load(tid + THREADS * e) : make_int2(0, -1);
  for (int k = warp; k < p.beams; k += WARPS) {
    const int row = b * p.beams + k;
    const float score = p.scores[row];
    const bool done = p.finished && p.finished[row], live = !done && score > -INFINITY;
    const float2* ms = p.part_ms + static_cast<int64_t>(row) * p.splits;
    float2 v = lane < p.splits ? __ldcg(ms + lane) : make_float2(-INFINITY, 0.f);
    if (!live) {  // its chunks wrote nothing
      if (lane == 0) beam[k] = make_float4(0.f, 0.f, score, done && score > -INFINITY ? 2.f : 1.f);
      continue;
    }
    for (int s = lane + 32; s < p.splits; s += 32) {  // more than 32 chunks: join a lane's own first
      const float2 u = __ldcg(ms + s);
      const float m = fmaxf(v.x, u.x);
      if (m > -INFINITY) v = make_float2(m, v.y * exp2_approx((v.x - m) * L2E) + u.y * exp2_approx((u.x - m) * L2E));
    }
    float m = v.x;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    float sum = v.x > -INFINITY ? v.y * exp2_approx((v.x - m) * L2E) : 0.f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) beam[k] = m == -INFINITY ? make_float4(0.f, 0.f, score, 0.f) : make_float4(m, logf(sum), score, 0.f);
  }
  __syncthreads();

  // candidate j of beam k (as its chunk wrote it): its value and place; false if there is none
  auto value_at = [&](int k, int j, int2 t, double& c, uint64_t& at) {
    const float4 f = beam[k];
    int token = t.y;
    if (f.w != 0.f) {
      const bool done = f.w == 2.f;
      token = j < p.n && j < p.vocab ? still_token(p, done, j) : -1;
      c = done && j == 0 ? static_cast<double>(f.z) : -INFINITY;
    } else {
      const float x = __int_as_float(t.x);
      const double below = static_cast<double>(x) - static_cast<double>(f.x) - static_cast<double>(f.y);
      c = x == -INFINITY ? -INFINITY : static_cast<double>(f.z) + below;
    }
    at = static_cast<uint64_t>(k) << 32 | static_cast<uint32_t>(token);
    return token >= 0;
  };
  auto value = [&](int i, int2 t, double& c, uint64_t& at) {
    int k;
    const int j = place(i, k);
    return value_at(k, j, t, c, at);
  };
  // rounding to fp32 keeps the order of unequal values or makes them equal, so a threshold on it keeps all of the best
  uint32_t mine = 0;
  auto look = [&](int i, int2 t) {
    double c;
    uint64_t at;
    if (value(i, t, c, at)) mine = max(mine, key_of(static_cast<float>(c)));
  };
  // All candidates in registers, or the first ranks of many lists. (32 sequences of 8 beams, 3 segments each: 28.6 us with
  // all in registers, 32.8 us with the walk; 8 beams of 38 segments: 24.4 and 11.6 us.)
  const bool few = total <= THREADS * FIRST;
#pragma unroll
  for (int e = 0; e < FIRST; ++e)
    if (tid + THREADS * e < total && (few || e < 2)) look(tid + THREADS * e, raw[e]);
  const uint32_t reach = max(reach_of(mine, p.n, WARPS, warp_key), 1u);
  auto keep = [&](double c, uint64_t at) {
    const int slot = atomicAdd(&n_cand, 1);
    if (slot < CAP) {
      cand_key[slot] = key_of(c);
      cand_at[slot] = at;
    }
  };
  double c0;
  uint64_t at0;
  if (few) {
    if (mine >= reach) {
#pragma unroll
      for (int e = 0; e < FIRST; ++e)
        if (tid + THREADS * e < total && value(tid + THREADS * e, raw[e], c0, at0) &&
            key_of(static_cast<float>(c0)) >= reach)
          keep(c0, at0);
    }
  } else {  // a segment's list is in order: a thread walks it down to the threshold
    for (int l = tid; l < p.beams * p.splits; l += THREADS) {
      int k;
      const int s = split(l, p.beams, beams_inv, k), from = k * per + s * p.n;
      for (int r = 0; r < p.n; ++r) {
        if (!value_at(k, s * p.n + r, __ldcg(top + from + r), c0, at0) || key_of(static_cast<float>(c0)) < reach) break;
        keep(c0, at0);
      }
    }
  }
  __syncthreads();
  auto put = [&](int rank, uint64_t k, uint64_t at) {
    const int64_t to = static_cast<int64_t>(b) * p.n + rank;
    const uint64_t bits = k ^ (k >> 63 ? 0x8000000000000000ull : ~0ull);
    p.out_scores[to] = static_cast<float>(__longlong_as_double(static_cast<long long>(bits)));
    p.out_beams[to] = static_cast<int64_t>(at >> 32);
    p.out_tokens[to] = static_cast<int64_t>(at & 0xffffffffu);
  };
  int c = n_cand;
  if (c <= CAP) {
    if (c > THREADS / 4) {  // beams of very different scores leave a low threshold: once more among the candidates
      uint64_t k[CAP / THREADS], at[CAP / THREADS];
      uint32_t best = 0;
#pragma unroll
      for (int e = 0; e < CAP / THREADS; ++e) {
        const int i = tid + THREADS * e;
        k[e] = i < c ? cand_key[i] : 0;
        at[e] = i < c ? cand_at[i] : 0;
        best = max(best, static_cast<uint32_t>(k[e] >> 32));
      }
      __syncthreads();
      if (tid == 0) n_cand = 0;
      const uint32_t high = max(reach_of(best, p.n, WARPS, warp_key), 1u);
#pragma unroll
      for (int e = 0; e < CAP / THREADS; ++e)
        if (k[e] >> 32 >= high) {
          const int slot = atomicAdd(&n_cand, 1);
          cand_key[slot] = k[e];
          cand_at[slot] = at[e];
        }
      __syncthreads();
      c = n_cand;
    }
    for (int i = tid; i < c; i += THREADS) {
      const uint64_t k = cand_key[i], at = cand_at[i];
      int rank = 0;
#pragma unroll 4
      for (int o = 0; o < c; ++o) rank += cand_key[o] > k || (cand_key[o] == k && cand_at[o] < at);
      if (rank < p.n) put(rank, k, at);
    }
    return;
  }
  ulonglong2 last = make_ulonglong2(~0ull, ~0ull);
  for (int i = 0; i < p.n; ++i) {
    ulonglong2 v = make_ulonglong2(0, 0);
    for (int e = tid; e < total; e += THREADS) {
      double cv;
      uint64_t at;
      if (!value(e, load(e), cv, at)) continue;
      const uint64_t k = key_of(cv), t = ~at;
      if ((k < last.x || (k == last.x && t < last.y)) && (k > v.x || (k == v.x && t > v.y))) v = make_ulonglong2(k, t);
    }
    last = best_of(v, box);
    if (tid == 0) put(i, last.x, ~last.y);
  }
}

// Vectors that a thread keeps in registers and the segment of a CTA. Segments of 1, 2 or 4 vectors a thread (8 to 32
// 16-bit logits) where that gives up to two CTAs for every SM: 4 rows of 32000 make 64 CTAs of 2048 elements. More work
// streams: segments of equal length, as many as it takes to fill the four CTAs that an SM holds once (256 rows of
// 151936: 3 segments each, 49 us with 10 segments in registers, 28 us streamed).
struct Plan {
  int vectors, splits, segment;
  bool stream;
  size_t ms_bytes, top_bytes;
};
Plan make_plan(int64_t rows, int vocab, int n, int dtype, int sm_count) {
  Plan pl{};
  const int step = THREADS * (dtype == TK_F32 ? 4 : 8), vectors = (vocab + step - 1) / step;
  const int64_t slots = 4 * static_cast<int64_t>(std::max(sm_count, 1));
  pl.vectors = 4;
  const int64_t fill = (slots + rows - 1) / rows;  // segments of a row that fill the GPU once
  const int64_t each = (vectors + fill - 1) / fill;
  if (each <= 4) {
    pl.vectors = each <= 1 ? 1 : each <= 2 ? 2 : 4;
    pl.segment = pl.vectors * step;
  } else {
    pl.stream = true;
    pl.segment = static_cast<int>(each) * step;
  }
  pl.splits = (vocab + pl.segment - 1) / pl.segment;
  pl.ms_bytes = (static_cast<size_t>(rows) * pl.splits * sizeof(float2) + 255) / 256 * 256;
  pl.top_bytes = static_cast<size_t>(rows) * pl.splits * n * sizeof(Entry);
  return pl;
}

template <int DT>
int launch_chunks(const Params& p, const Plan& pl, dim3 grid, cudaStream_t st) {
  if (pl.stream) return launch_kernel(beam_chunk_kernel<DT, 4, true>, grid, dim3(THREADS), 0, st, 1, "beam_select", p);
  switch (pl.vectors) {
    case 1: return launch_kernel(beam_chunk_kernel<DT, 1, false>, grid, dim3(THREADS), 0, st, 1, "beam_select", p);
    case 2: return launch_kernel(beam_chunk_kernel<DT, 2, false>, grid, dim3(THREADS), 0, st, 1, "beam_select", p);
    default: return launch_kernel(beam_chunk_kernel<DT, 4, false>, grid, dim3(THREADS), 0, st, 1, "beam_select", p);
  }
}

}  // namespace beam
}  // namespace tk

extern "C" int64_t tk_beam_select_workspace(int batch, int beams, int vocab, int num_select, int dtype) {
  using namespace tk;
  if (batch <= 0 || beams <= 0 || vocab <= 0 || num_select <= 0 || !valid_dtype(dtype)) return 0;
  DeviceInfo di;
  if (current_device_info(&di)) return -1;
  const beam::Plan pl = beam::make_plan(int64_t(batch) * beams, vocab, num_select, dtype, di.sm_count);
  return static_cast<int64_t>(pl.ms_bytes + pl.top_bytes);
}

extern "C" int tk_beam_select(const void* logits, int64_t row_stride, const float* scores, const uint8_t* finished,
                              int64_t eos_token, float* out_scores, int64_t* out_beams, int64_t* out_tokens,
                              int batch, int beams, int vocab, int num_select, void* workspace,
                              int64_t workspace_bytes, int dtype, void* stream) {
  using namespace tk;
  using namespace tk::beam;
  if (!valid_dtype(dtype)) return fail_invalid("beam_select: dtype must be F16, BF16 or F32");
  if (batch < 0 || beams <= 0 || vocab <= 0) return fail_invalid("beam_select: invalid sizes");
  if (num_select < 1 || num_select > MAX_N)
    return set_error(TK_ERR_UNSUPPORTED, "beam_select: num_select must be 1.." + std::to_string(MAX_N));
  if (num_select > int64_t(beams) * vocab) return fail_invalid("beam_select: num_select exceeds beams * vocab");
  if (beams > 1024) return set_error(TK_ERR_UNSUPPORTED, "beam_select: more than 1024 beams");
  if (vocab > (1 << 30)) return set_error(TK_ERR_UNSUPPORTED, "beam_select: vocab above 2^30");
  if (row_stride < vocab) return fail_invalid("beam_select: row stride smaller than vocab");
  if (int64_t(batch) * beams > 65535) return fail_invalid("beam_select: more than 65535 rows");
  if (finished && (eos_token < 0 || eos_token >= vocab))
    return fail_invalid("beam_select: finished beams need an eos_token inside the vocabulary");
  if (batch == 0) return TK_OK;
  if (!logits || !scores || !out_scores || !out_beams || !out_tokens) return fail_invalid("beam_select: NULL pointer");
  DeviceInfo di;
  if (int rc = current_device_info(&di)) return rc;
  const int rows = batch * beams;
  const Plan pl = make_plan(rows, vocab, num_select, dtype, di.sm_count);
  if (!workspace || workspace_bytes < static_cast<int64_t>(pl.ms_bytes + pl.top_bytes))
    return fail_invalid("beam_select: workspace missing or smaller than tk_beam_select_workspace()");
  if (!aligned16(workspace)) return fail_invalid("beam_select: workspace must be 16-byte aligned");
  if (int64_t(beams) * pl.splits * num_select > (1 << 30))
    return set_error(TK_ERR_UNSUPPORTED, "beam_select: too many candidates for one sequence");
  Params p{};
  p.logits = logits;
  p.row_stride = row_stride;
  p.scores = scores;
  p.finished = finished;
  p.eos = eos_token;
  p.beams = beams;
  p.vocab = vocab;
  p.n = num_select;
  p.splits = pl.splits;
  p.segment = pl.segment;
  p.part_ms = static_cast<float2*>(workspace);
  p.part_top = reinterpret_cast<Entry*>(static_cast<char*>(workspace) + pl.ms_bytes);
  p.out_scores = out_scores;
  p.out_beams = out_beams;
  p.out_tokens = out_tokens;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const dim3 grid(pl.splits, rows);
  int rc = dtype == TK_F16    ? launch_chunks<TK_F16>(p, pl, grid, st)
           : dtype == TK_BF16 ? launch_chunks<TK_BF16>(p, pl, grid, st)
                              : launch_chunks<TK_F32>(p, pl, grid, st);
  if (rc) return rc;
  return launch_kernel(beam_merge_kernel, dim3(batch), dim3(THREADS), beams * sizeof(float4), st, 1,
                       "beam_select merge", p);
}
