// Appending rows to an 8-bit KV cache (format and layout: kv8.cuh): the fill after a prompt's tensor-core
// attention, and the second launch of kv8_attention for more than one new token.
//
// Rows start .. start + S - 1 of one (sequence, kv head) touch the open block, then whole blocks, then the new open
// block. A warp quantises the keys or the values of one block that the call completes: rows before `start` come
// from the tail, the others from the input. The warp of the first such block also copies the rows of the new open
// block into the tail, after its own reads of the tail (its warp-wide maximum depends on all of them), so no other
// warp reads or writes the rows of the tail and nothing races. Nothing but these rows is written.
//
// Bound by HBM: 4 * D bytes read and 2 * D written per row and kv head (16 x 4001 rows of 8 heads of 128: 66.5 us,
// 5.9 TB/s; 16 x 8001 of 8 heads of 64: 62.5 us, 6.3 TB/s).
#include <algorithm>
#include <string>

#include "kv8.cuh"
#include "kv8_host.h"
#include "tk_host.h"

namespace tk {
namespace kv8 {

struct AppendParams {
  const void* k;  // [batch * seq, ...] rows, head j at column j * D
  int64_t ks;
  const void* v;
  int64_t vs;
  uint8_t* kc;  // [batch, num_kv_heads, num_blocks, 32 * D]
  uint8_t* vc;
  float* scales;  // [batch, num_kv_heads, num_blocks, 2]
  void* tail;     // [batch, num_kv_heads, 2, 32, D]
  const float* cos_t;  // if set, k is rotated at its position
  const float* sin_t;
  int64_t table_rows;
  int num_blocks, seq, num_kv_heads, start_pos;
  const int* start_dev;
  int start_step;
};

constexpr int PAIRS = 4;  // warps for keys, and as many for values, of one CTA

// 128 registers leave two CTAs on an SM at D = 128 (the keys alone need 64 for a block): 16 x 4001 rows of 8 heads of 128
// take 66.6 us (5.9 TB/s) instead of 101.4 us with one.
template <int DT, int FMT, int D>
__global__ void __launch_bounds__(PAIRS * 64, D == 64 ? 3 : 2) kv8_append_kernel(const AppendParams p) {
  extern __shared__ __align__(128) uint8_t smem[];
  using T = typename Dt<DT>::T;
  constexpr int C16 = D / 8;
  pdl_wait();
  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool values = warp >= PAIRS;
  const int head = blockIdx.y, b = blockIdx.z;
  const int start = p.start_dev ? __ldcg(p.start_dev + static_cast<int64_t>(b) * p.start_step) : p.start_pos;
  const int64_t end = static_cast<int64_t>(start) + p.seq;
  if (start < 0 || end > static_cast<int64_t>(p.num_blocks) * BLOCK || (p.cos_t && end > p.table_rows)) {
    if (threadIdx.x == 0 && blockIdx.x == 0 && head == 0) record_device_error(TK_DEVERR_POSITION);
    return;
  }
  const int open = start % BLOCK, first = start / BLOCK;
  const int whole = (open + p.seq) / BLOCK, rest = (open + p.seq) % BLOCK;
  const int task = blockIdx.x * PAIRS + warp % PAIRS;
  if (task >= max(whole, 1)) return;

  const int64_t bh = static_cast<int64_t>(b) * p.num_kv_heads + head;
  T* tail = reinterpret_cast<T*>(p.tail) + (bh * 2 + (values ? 1 : 0)) * BLOCK * D;
  const T* in = reinterpret_cast<const T*>(values ? p.v : p.k) + static_cast<int64_t>(head) * D;
  const int64_t stride = values ? p.vs : p.ks;
  const int row0 = task * BLOCK - open;  // the input row of the block's first token
  // 16-byte chunk c of input row s, rotated if it is a key
  auto fresh = [&](int s, int c) {
    return __ldcg(reinterpret_cast<const uint4*>(in + (static_cast<int64_t>(b) * p.seq + s) * stride) + c);
  };
  auto rotate = [&](uint4& x, int s, int c) {
    if (!values && p.cos_t && s >= 0) {
      const int64_t at = (static_cast<int64_t>(start) + s) * (D / 2) + c * 4;
      rope_chunk<DT>(x, p.cos_t + at, p.sin_t + at);
    }
  };
  auto piece = [&](int t, int c) {  // one load whatever its source, so that a lane's loads are all in flight at once
    const int s = row0 + t;
    const T* src = s < 0 ? tail + t * D : in + (static_cast<int64_t>(b) * p.seq + s) * stride;
    return __ldcg(reinterpret_cast<const uint4*>(src) + c);
  };

  if (whole > 0) {
    const int64_t block = bh * p.num_blocks + first + task;
    float scale;
    if (!values) {
      scale = encode_keys<DT, FMT, D>(p.kc + block * (BLOCK * D), lane, piece,
                                       [&](uint4& x, int t, int c) { rotate(x, row0 + t, c); });
    } else {
      uint8_t* tile = smem + (warp - PAIRS) * (BLOCK * D * 2);
      uint32_t m = 0;
      uint4 x[C16];
#pragma unroll
      for (int i = 0; i < C16; ++i) x[i] = piece((lane + 32 * i) / C16, (lane + 32 * i) % C16);
#pragma unroll
      for (int i = 0; i < C16; ++i) {
        const int idx = lane + 32 * i, t = idx / C16, c = idx % C16;
        m = amax2(amax2(amax2(amax2(m, x[i].x), x[i].y), x[i].z), x[i].w);
        *reinterpret_cast<uint4*>(tile + tile_off<D>(t, c)) = x[i];
      }
      const uint32_t amax = amax2_warp(m);
      __syncwarp();
      scale = encode_values<DT, FMT, D>(p.vc + block * (BLOCK * D), lane, smem_u32(tile), amax);
    }
    if (lane == 0) p.scales[block * 2 + (values ? 1 : 0)] = scale;
  }
  if (task == 0) {  // the rows of the block that stays open
    const int n = whole > 0 ? rest : p.seq, to = whole > 0 ? 0 : open, from = p.seq - n;
    for (int idx = lane; idx < n * C16; idx += 32) {
      const int t = idx / C16, c = idx % C16;
      uint4 x = fresh(from + t, c);
      rotate(x, from + t, c);
      *(reinterpret_cast<uint4*>(tail + (to + t) * D) + c) = x;
    }
  }
}

template <int DT, int FMT, int D>
int launch_append(const AppendParams& p, int batch, cudaStream_t st) {
  const int most = std::max(1, (BLOCK - 1 + p.seq) / BLOCK);  // blocks that a call may complete
  const dim3 grid((most + PAIRS - 1) / PAIRS, p.num_kv_heads, batch);
  return launch_kernel(kv8_append_kernel<DT, FMT, D>, grid, dim3(PAIRS * 64), PAIRS * BLOCK * D * 2, st, 1,
                       "kv8_append", p);
}

template <int DT, int FMT>
int launch_append(const AppendParams& p, int batch, int head_dim, cudaStream_t st) {
  return head_dim == 64 ? launch_append<DT, FMT, 64>(p, batch, st) : launch_append<DT, FMT, 128>(p, batch, st);
}

int append(const Cache& c, const void* k, int64_t ks, const void* v, int64_t vs, const float* cos_t,
           const float* sin_t, int64_t table_rows, int batch, int seq, int num_kv_heads, int head_dim, int start_pos,
           const int* start_dev, int start_step, int dtype, cudaStream_t st) {
  AppendParams p{};
  p.k = k;
  p.ks = ks;
  p.v = v;
  p.vs = vs;
  p.kc = static_cast<uint8_t*>(c.k);
  p.vc = static_cast<uint8_t*>(c.v);
  p.scales = c.scales;
  p.tail = c.tail;
  p.cos_t = cos_t;
  p.sin_t = sin_t;
  p.table_rows = table_rows;
  p.num_blocks = c.num_blocks;
  p.seq = seq;
  p.num_kv_heads = num_kv_heads;
  p.start_pos = start_pos;
  p.start_dev = start_dev;
  p.start_step = start_step;
  if (dtype == TK_F16)
    return c.format == TK_KV8_E4M3 ? launch_append<TK_F16, TK_KV8_E4M3>(p, batch, head_dim, st)
                                   : launch_append<TK_F16, TK_KV8_INT8>(p, batch, head_dim, st);
  return c.format == TK_KV8_E4M3 ? launch_append<TK_BF16, TK_KV8_E4M3>(p, batch, head_dim, st)
                                 : launch_append<TK_BF16, TK_KV8_INT8>(p, batch, head_dim, st);
}

int check_cache(const char* what, const Cache& c, int batch, int seq, int num_heads, int num_kv_heads, int head_dim,
                int dtype) {
  const std::string w(what);
  if (!half_dtype(dtype)) return fail_invalid(w + ": dtype must be F16 or BF16");
  if (c.format != TK_KV8_E4M3 && c.format != TK_KV8_INT8)
    return fail_invalid(w + ": cache format must be TK_KV8_E4M3 or TK_KV8_INT8");
  if (head_dim != 64 && head_dim != 128) return set_error(TK_ERR_UNSUPPORTED, w + ": head_dim must be 64 or 128");
  if (batch < 0 || seq < 0 || num_heads <= 0 || num_kv_heads <= 0 || c.num_blocks < 0)
    return fail_invalid(w + ": invalid sizes");
  if (num_heads % num_kv_heads != 0) return fail_invalid(w + ": num_heads must be a multiple of num_kv_heads");
  if (batch > 65535 || num_kv_heads > 65535) return fail_invalid(w + ": too many sequences or kv heads");
  if (c.num_blocks > (1 << 26) - 1) return fail_invalid(w + ": the cache is longer than 2^31 positions");
  if (batch == 0 || seq == 0) return TK_OK;
  if (!c.k || !c.v || !c.scales || !c.tail) return fail_invalid(w + ": NULL cache pointer");
  if (!aligned16(c.k) || !aligned16(c.v) || !aligned16(c.tail) || reinterpret_cast<uintptr_t>(c.scales) % 8)
    return fail_invalid(w + ": cache pointers must be 16-byte aligned (scales: 8)");
  return TK_OK;
}

}  // namespace kv8
}  // namespace tk

extern "C" int tk_kv8_append(const void* k, int64_t k_tok_stride, const void* v, int64_t v_tok_stride, void* k_cache,
                             void* v_cache, float* scales, void* tail, int num_blocks, int format, int batch, int seq,
                             int num_kv_heads, int head_dim, int start_pos, int dtype, void* stream) {
  using namespace tk;
  using namespace tk::kv8;
  const Cache c{k_cache, v_cache, scales, tail, num_blocks, format};
  if (int rc = check_cache("kv8_append", c, batch, seq, num_kv_heads, num_kv_heads, head_dim, dtype)) return rc;
  if (k_tok_stride < int64_t(num_kv_heads) * head_dim || v_tok_stride < int64_t(num_kv_heads) * head_dim)
    return fail_invalid("kv8_append: token stride smaller than num_kv_heads * head_dim");
  if (k_tok_stride % 8 || v_tok_stride % 8)
    return fail_invalid("kv8_append: token strides must be multiples of 8 elements");
  if (start_pos < 0 || int64_t(start_pos) + seq > int64_t(num_blocks) * BLOCK)
    return fail_invalid("kv8_append: start_pos + seq exceeds the cache");
  if (batch == 0 || seq == 0) return TK_OK;
  if (!k || !v) return fail_invalid("kv8_append: NULL pointer");
  if (!aligned16(k) || !aligned16(v)) return fail_invalid("kv8_append: pointers must be 16-byte aligned");
  return append(c, k, k_tok_stride, v, v_tok_stride, nullptr, nullptr, 0, batch, seq, num_kv_heads, head_dim,
                start_pos, nullptr, 0, dtype, static_cast<cudaStream_t>(stream));
}
