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
//   1. a CTA takes a chunk of one row into registers: its maximum m, sum of e^(x - m), and its best n. Of the threads' maxima each of the 8 warps takes its ceil(n / 8)-th largest; the least of those is a
//      value that at least n elements reach, so the best n are among the elements that reach it (some 2 n of them),
//      which are collected in shared memory and ranked by counting. Where ties make them too many (a masked
//      vocabulary), n rounds of a maximum over (value, index) take over.
//   2. a CTA for each sequence joins the chunks' sums to a logsumexp for each beam and picks the best n of the chunks'
//      candidates the same way, with c in fp64.
// Sums are taken in an order that depends on element numbers alone, so equal rows give equal sums wherever they lie.
// Bound by HBM for many rows (one read of the logits; one exponential for each element is the next limit), by the
// latency of the two launches for few.
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
  int beams, vocab, n, splits;
  float2* part_ms;   // [rows, splits]: maximum, sum of e^(x - maximum)
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
__device__ __forceinline__ uint64_t key_of(double x) {
  const uint64_t u = static_cast<uint64_t>(__double_as_longlong(x + 0.0));
  return u ^ (static_cast<uint64_t>(static_cast<int64_t>(u) >> 63) | 0x8000000000000000ull);
}

// The beam gives no candidates of its own: finished, or dead (score -inf or NaN).
__device__ __forceinline__ bool is_still(const Params& p, int row) {
  return (p.finished && p.finished[row]) || !(p.scores[row] > -INFINITY);
}

// A key that at least n of the threads' keys reach, for n <= 8 * 32: see the head of this file. All threads call it.
__device__ __forceinline__ uint32_t reach_of(uint32_t mine, int n, uint32_t* warp_key) {
  const int lane = threadIdx.x & 31;
  uint32_t left = mine, kth = 0;
  for (int i = 0; i < (n + WARPS - 1) / WARPS; ++i) {
    kth = __reduce_max_sync(0xffffffffu, left);
    const uint32_t who = __ballot_sync(0xffffffffu, left == kth);
    if (lane == __ffs(who) - 1) left = 0;
  }
  if (lane == 0) warp_key[threadIdx.x >> 5] = kth;
  __syncthreads();
  uint32_t t = warp_key[0];
#pragma unroll
  for (int w = 1; w < WARPS; ++w) t = min(t, warp_key[w]);
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

template <int DT, int NV>
__global__ void __launch_bounds__(THREADS) beam_chunk_kernel(const Params p) {
  using T = typename Logit<DT>::T;
  constexpr int VE = 16 / sizeof(T);  // elements of a vector
  constexpr int CHUNK = THREADS * NV * VE;
  __shared__ float red[WARPS], red2[WARPS];
  __shared__ uint32_t warp_key[WARPS];
  __shared__ ulonglong2 box[WARPS];
  __shared__ uint32_t cand_key[CAP];
  __shared__ int cand_idx[CAP];
  __shared__ int n_cand;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int row = blockIdx.y, split = blockIdx.x;
  if (tid == 0) n_cand = 0;
  pdl_wait();
  pdl_launch_dependents();
  if (is_still(p, row)) return;
  const T* src = static_cast<const T*>(p.logits) + static_cast<int64_t>(row) * p.row_stride;
  const int lo = split * CHUNK;
  const bool aligned = (reinterpret_cast<uintptr_t>(src) & 15) == 0;

  float x[NV][VE];
  if (aligned && lo + CHUNK <= p.vocab) {
    uint4 raw[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) raw[j] = __ldcs(reinterpret_cast<const uint4*>(src + lo) + tid + THREADS * j);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const T* e = reinterpret_cast<const T*>(&raw[j]);
#pragma unroll
      for (int i = 0; i < VE; ++i) x[j][i] = Logit<DT>::to_f(e[i]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < VE; ++i) {
        const int64_t at = static_cast<int64_t>(lo) + (tid + THREADS * j) * VE + i;
        x[j][i] = at < p.vocab ? Logit<DT>::to_f(src[at]) : -INFINITY;
      }
  }
  constexpr float TOP = DT == TK_F16 ? 65504.f : DT == TK_BF16 ? 3.3895313892515355e38f : 3.4028234663852886e38f;
  float mx = -INFINITY;
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int i = 0; i < VE; ++i) {
      x[j][i] = fminf(fmaxf(x[j][i], -INFINITY), TOP);  // fmaxf turns NaN into -inf
      mx = fmaxf(mx, x[j][i]);
    }
  const float mine = mx;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  if (lane == 0) red[warp] = mx;
  const uint32_t reach = reach_of(key_of(mine), p.n, warp_key);  // synchronises
  mx = red[0];
#pragma unroll
  for (int w = 1; w < WARPS; ++w) mx = fmaxf(mx, red[w]);
  const float base = mx == -INFINITY ? 0.f : mx;  // subtracted first: m log2 e may be past the largest float
  float sum = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int i = 0; i < VE; ++i) sum += exp2_approx((x[j][i] - base) * L2E);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) red2[warp] = sum;

  if (key_of(mine) >= reach) {
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < VE; ++i) {
        const int at = lo + (tid + THREADS * j) * VE + i;
        const uint32_t k = key_of(x[j][i]);
        if (k >= reach && at < p.vocab) {
          const int slot = atomicAdd(&n_cand, 1);
          if (slot < CAP) {
            cand_key[slot] = k;
            cand_idx[slot] = at;
          }
        }
      }
  }
  __syncthreads();
  const int64_t part = static_cast<int64_t>(row) * p.splits + split;
  if (tid == 0) {
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) s += red2[w];
    p.part_ms[part] = make_float2(mx, s);
  }
  auto value = [](uint32_t k) { return __uint_as_float(k ^ (k >> 31 ? 0x80000000u : 0xffffffffu)); };
  Entry* top = p.part_top + part * p.n;
  const int c = n_cand;
  if (c <= CAP) {
    for (int i = tid; i < c; i += THREADS) {
      const uint32_t k = cand_key[i];
      const int at = cand_idx[i];
      int rank = 0;
      for (int o = 0; o < c; ++o) rank += cand_key[o] > k || (cand_key[o] == k && cand_idx[o] < at);
      if (rank < p.n) top[rank] = Entry{value(k), at};
    }
    for (int i = c + tid; i < p.n; i += THREADS) top[i] = Entry{-INFINITY, -1};  // a chunk shorter than n
    return;
  }
  ulonglong2 last = make_ulonglong2(~0ull, ~0ull);
  for (int i = 0; i < p.n; ++i) {
    ulonglong2 v = make_ulonglong2(0, 0);
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        const int at = lo + (tid + THREADS * j) * VE + e;
        const uint64_t k = key_of(x[j][e]), t = static_cast<uint32_t>(~at);
        if (at < p.vocab && (k < last.x || (k == last.x && t < last.y)) && (k > v.x || (k == v.x && t > v.y)))
          v = make_ulonglong2(k, t);
      }
    last = best_of(v, box);
    if (tid == 0)
      top[i] = last.x ? Entry{value(static_cast<uint32_t>(last.x)), static_cast<int>(~static_cast<uint32_t>(last.y))}
                      : Entry{-INFINITY, -1};
  }
}

// Candidate j of a still beam: the end token of a finished one first, then -inf at its lowest tokens.
__device__ __forceinline__ int still_token(const Params& p, bool done, int j) {
  if (!done) return j;
  if (j == 0) return static_cast<int>(p.eos);
  return j - 1 < p.eos ? j - 1 : j;
}

__global__ void __launch_bounds__(THREADS) beam_merge_kernel(const Params p) {
  extern __shared__ double2 norm[];  // [beams]: maximum, log of the sum
  __shared__ uint32_t warp_key[WARPS];
  __shared__ ulonglong2 box[WARPS];
  __shared__ uint64_t cand_key[CAP];
  __shared__ int64_t cand_at[CAP];
  __shared__ int n_cand;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, b = blockIdx.x;
  if (tid == 0) n_cand = 0;
  pdl_wait();
  pdl_launch_dependents();
  for (int k = warp; k < p.beams; k += WARPS) {
    const int row = b * p.beams + k;
    if (is_still(p, row)) continue;
    const float2* ms = p.part_ms + static_cast<int64_t>(row) * p.splits;
    float m = -INFINITY;
    for (int s = lane; s < p.splits; s += 32) m = fmaxf(m, __ldcg(ms + s).x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    double sum = 0.0;
    for (int s = lane; s < p.splits; s += 32) {
      const float2 v = __ldcg(ms + s);
      if (v.x > -INFINITY) sum += static_cast<double>(v.y) * exp(static_cast<double>(v.x) - static_cast<double>(m));
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) norm[k] = m == -INFINITY ? make_double2(0.0, 0.0) : make_double2(m, log(sum));
  }
  __syncthreads();

  const int per = p.splits * p.n;  // candidates of a beam (a still one has n)
  const int64_t total = static_cast<int64_t>(p.beams) * per;
  // candidate i: its value and flat place beam * V + token, -1 if there is none
  auto get = [&](int64_t i, double& c, int64_t& at) {
    const int k = static_cast<int>(i / per), j = static_cast<int>(i - static_cast<int64_t>(k) * per);
    const int row = b * p.beams + k;
    const float score = p.scores[row];
    if (is_still(p, row)) {
      const bool done = p.finished && p.finished[row] && score > -INFINITY;
      at = j < p.n && j < p.vocab ? static_cast<int64_t>(k) * p.vocab + still_token(p, done, j) : -1;
      c = done && j == 0 ? static_cast<double>(score) : -INFINITY;
      return;
    }
    const int2 raw = __ldcg(reinterpret_cast<const int2*>(p.part_top + static_cast<int64_t>(row) * per + j));
    const float x = __int_as_float(raw.x);
    at = raw.y < 0 ? -1 : static_cast<int64_t>(k) * p.vocab + raw.y;
    c = x == -INFINITY ? -INFINITY : static_cast<double>(score) + ((static_cast<double>(x) - norm[k].x) - norm[k].y);
  };
  // rounding to fp32 keeps the order of unequal values or makes them equal, so a threshold on it keeps all of the best
  uint32_t mine = 0;
  for (int64_t i = tid; i < total; i += THREADS) {
    double c;
    int64_t at;
    get(i, c, at);
    if (at >= 0) mine = max(mine, key_of(static_cast<float>(c)));
  }
  const uint32_t reach = max(reach_of(mine, p.n, warp_key), 1u);
  if (mine >= reach) {
    for (int64_t i = tid; i < total; i += THREADS) {
      double c;
      int64_t at;
      get(i, c, at);
      if (at < 0 || key_of(static_cast<float>(c)) < reach) continue;
      const int slot = atomicAdd(&n_cand, 1);
      if (slot < CAP) {
        cand_key[slot] = key_of(c);
        cand_at[slot] = at;
      }
    }
  }
  __syncthreads();
  auto put = [&](int rank, uint64_t k, int64_t at) {
    const int64_t to = static_cast<int64_t>(b) * p.n + rank;
    const uint64_t bits = k ^ (k >> 63 ? 0x8000000000000000ull : ~0ull);
    p.out_scores[to] = static_cast<float>(__longlong_as_double(static_cast<long long>(bits)));
    p.out_beams[to] = at / p.vocab;
    p.out_tokens[to] = at % p.vocab;
  };
  const int c = n_cand;
  if (c <= CAP) {
    for (int i = tid; i < c; i += THREADS) {
      const uint64_t k = cand_key[i];
      const int64_t at = cand_at[i];
      int rank = 0;
      for (int o = 0; o < c; ++o) rank += cand_key[o] > k || (cand_key[o] == k && cand_at[o] < at);
      if (rank < p.n) put(rank, k, at);
    }
    return;
  }
  ulonglong2 last = make_ulonglong2(~0ull, ~0ull);
  for (int i = 0; i < p.n; ++i) {
    ulonglong2 v = make_ulonglong2(0, 0);
    for (int64_t e = tid; e < total; e += THREADS) {
      double cv;
      int64_t at;
      get(e, cv, at);
      if (at < 0) continue;
      const uint64_t k = key_of(cv), t = ~static_cast<uint64_t>(at);
      if ((k < last.x || (k == last.x && t < last.y)) && (k > v.x || (k == v.x && t > v.y))) v = make_ulonglong2(k, t);
    }
    last = best_of(v, box);
    if (tid == 0) put(i, last.x, static_cast<int64_t>(~last.y));
  }
}

// Elements a thread takes (8, 16 or 32): the most that still gives two CTAs for every SM, 8 if none does. A row of
// 32000 and 4 rows: 8 gives 64 CTAs; 256 rows of 151936: 32.
struct Plan {
  int per_thread, splits;
  size_t ms_bytes, top_bytes;
};
Plan make_plan(int64_t rows, int vocab, int n, int sm_count) {
  Plan pl{};
  for (pl.per_thread = 32;; pl.per_thread /= 2) {
    pl.splits = (vocab + THREADS * pl.per_thread - 1) / (THREADS * pl.per_thread);
    if (pl.per_thread == 8 || rows * pl.splits >= 2 * static_cast<int64_t>(sm_count)) break;
  }
  pl.ms_bytes = (static_cast<size_t>(rows) * pl.splits * sizeof(float2) + 255) / 256 * 256;
  pl.top_bytes = static_cast<size_t>(rows) * pl.splits * n * sizeof(Entry);
  return pl;
}

template <int DT>
int launch_chunks(const Params& p, int per_thread, dim3 grid, cudaStream_t st) {
  constexpr int VE = DT == TK_F32 ? 4 : 8;
  switch (per_thread) {
    case 8: return launch_kernel(beam_chunk_kernel<DT, 8 / VE>, grid, dim3(THREADS), 0, st, 1, "beam_select", p);
    case 16: return launch_kernel(beam_chunk_kernel<DT, 16 / VE>, grid, dim3(THREADS), 0, st, 1, "beam_select", p);
    default: return launch_kernel(beam_chunk_kernel<DT, 32 / VE>, grid, dim3(THREADS), 0, st, 1, "beam_select", p);
  }
}

}  // namespace beam
}  // namespace tk

extern "C" int64_t tk_beam_select_workspace(int batch, int beams, int vocab, int num_select) {
  using namespace tk;
  if (batch <= 0 || beams <= 0 || vocab <= 0 || num_select <= 0) return 0;
  DeviceInfo di;
  if (current_device_info(&di)) return -1;
  const beam::Plan pl = beam::make_plan(int64_t(batch) * beams, vocab, num_select, di.sm_count);
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
  const Plan pl = make_plan(rows, vocab, num_select, di.sm_count);
  if (!workspace || workspace_bytes < static_cast<int64_t>(pl.ms_bytes + pl.top_bytes))
    return fail_invalid("beam_select: workspace missing or smaller than tk_beam_select_workspace()");
  if (!aligned16(workspace)) return fail_invalid("beam_select: workspace must be 16-byte aligned");
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
  p.part_ms = static_cast<float2*>(workspace);
  p.part_top = reinterpret_cast<Entry*>(static_cast<char*>(workspace) + pl.ms_bytes);
  p.out_scores = out_scores;
  p.out_beams = out_beams;
  p.out_tokens = out_tokens;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const dim3 grid(pl.splits, rows);
  int rc = dtype == TK_F16    ? launch_chunks<TK_F16>(p, pl.per_thread, grid, st)
           : dtype == TK_BF16 ? launch_chunks<TK_BF16>(p, pl.per_thread, grid, st)
                              : launch_chunks<TK_F32>(p, pl.per_thread, grid, st);
  if (rc) return rc;
  return launch_kernel(beam_merge_kernel, dim3(batch), dim3(THREADS), beams * sizeof(double2), st, 1,
                       "beam_select merge", p);
}
