// Reordering a cache's rows after a beam search step, in place: row g * beams + i becomes what row
// g * beams + parents[g, i] was. Only the filled positions move, and rows that stay their own parent are not touched.
//
// A thread owns the same bytes of all rows of a group: it loads the parents' bytes of every row that changes, then
// stores them. No other thread touches these bytes, so no order of rows, no second buffer and no barrier is needed,
// whatever cycles the parents form. A parent of several rows is read from HBM once (the thread's later loads hit L1).
// Bound by HBM: one read for each row that is a parent of another, one write for each row that changes (16 layers of 8 x
// 8 beams, 8 heads of 64 in 8 bits at 2001: 469 us, 6.2 TB/s; 18 layers of 4 beams, 4 heads of 64 at 301: 5.3 us).
#include <algorithm>
#include <string>

#include "tk_common.cuh"
#include "tk_host.h"

namespace tk {
namespace reorder {

constexpr int THREADS = 256;
constexpr int MAX_ITEMS = 4;

struct Item {
  char* base;
  int64_t row_stride, layer_stride, head_stride;  // bytes
  int layers, heads;
  int unit_bytes, unit_tokens;
  int rest;       // 0: the length / unit_tokens whole units, 1: the length % unit_tokens units that follow
  int pieces;     // CTAs along one (layer, head)'s bytes at the greatest length
  int first_cta;  // of this item
};

struct Params {
  Item item[MAX_ITEMS];
  int n_items, beams;
  const int64_t* parents;  // [groups, beams]
  int length, max_length;
  const int* length_dev;
};

template <int BEAMS, typename V>
__device__ __forceinline__ void move_bytes(char* at, int64_t row_stride, int64_t off, const int (&parent)[BEAMS],
                                           uint32_t moved) {
  V x[BEAMS];
#pragma unroll
  for (int i = 0; i < BEAMS; ++i)
    if (moved >> i & 1) x[i] = *reinterpret_cast<const V*>(at + parent[i] * row_stride + off);
#pragma unroll
  for (int i = 0; i < BEAMS; ++i)
    if (moved >> i & 1) *reinterpret_cast<V*>(at + i * row_stride + off) = x[i];
}

template <int BEAMS>
__global__ void __launch_bounds__(THREADS) reorder_kernel(const Params p) {
  pdl_wait();
  pdl_launch_dependents();
  const int group = blockIdx.y;
  const int length = p.length_dev ? __ldcg(p.length_dev) : p.length;
  if (length < 0 || length > p.max_length) {
    if (threadIdx.x == 0 && blockIdx.x == 0 && group == 0) record_device_error(TK_DEVERR_POSITION);
    return;
  }
  int parent[BEAMS];
  uint32_t moved = 0;
  bool bad = false;
#pragma unroll
  for (int i = 0; i < BEAMS; ++i) {
    const int64_t a = i < p.beams ? __ldg(p.parents + static_cast<int64_t>(group) * p.beams + i) : i;
    bad |= i < p.beams && (a < 0 || a >= p.beams);
    parent[i] = static_cast<int>(a);
    if (i < p.beams && a != i) moved |= 1u << i;
  }
  if (bad) {  // a group with a parent outside it stays as it is
    if (threadIdx.x == 0 && blockIdx.x == 0) record_device_error(TK_DEVERR_PARENT);
    return;
  }
  if (!moved) return;
  int n = 0;
#pragma unroll
  for (int i = 1; i < MAX_ITEMS; ++i)
    if (i < p.n_items && static_cast<int>(blockIdx.x) >= p.item[i].first_cta) n = i;
  const Item& it = p.item[n];
  const int c = blockIdx.x - it.first_cta;
  const int piece = c % it.pieces, lh = c / it.pieces;
  const int units = it.rest ? length % it.unit_tokens : length / it.unit_tokens;
  const int64_t bytes = static_cast<int64_t>(units) * it.unit_bytes;
  char* at = it.base + static_cast<int64_t>(lh / it.heads) * it.layer_stride + (lh % it.heads) * it.head_stride +
             static_cast<int64_t>(group) * p.beams * it.row_stride;
  if (it.unit_bytes % 16 == 0) {
    const int64_t off = (static_cast<int64_t>(piece) * THREADS + threadIdx.x) * 16;
    if (off < bytes) {
      if constexpr (BEAMS <= 16) {
        move_bytes<BEAMS, uint4>(at, it.row_stride, off, parent, moved);
      } else {  // 16 bytes of 32 rows do not fit in a thread's registers
        move_bytes<BEAMS, uint2>(at, it.row_stride, off, parent, moved);
        move_bytes<BEAMS, uint2>(at, it.row_stride, off + 8, parent, moved);
      }
    }
  } else {  // a block's two scales
    const int64_t off = (static_cast<int64_t>(piece) * THREADS + threadIdx.x) * 8;
    if (off < bytes) move_bytes<BEAMS, uint2>(at, it.row_stride, off, parent, moved);
  }
}

template <int BEAMS>
int launch(const Params& p, int ctas, int groups, cudaStream_t st) {
  return launch_kernel(reorder_kernel<BEAMS>, dim3(ctas, groups), dim3(THREADS), 0, st, 1, "kv_reorder", p);
}

// Add a tensor [layers, rows, heads, units, unit_bytes], contiguous, of at most `units` units.
void add_item(Params& p, int64_t& ctas, void* base, int layers, int rows, int heads, int units, int unit_bytes,
              int unit_tokens, bool rest, int max_length) {
  Item& it = p.item[p.n_items];
  it.base = static_cast<char*>(base);
  it.head_stride = int64_t(units) * unit_bytes;
  it.row_stride = heads * it.head_stride;
  it.layer_stride = rows * it.row_stride;
  it.layers = layers;
  it.heads = heads;
  it.unit_bytes = unit_bytes;
  it.unit_tokens = unit_tokens;
  it.rest = rest;
  const int64_t most = rest ? std::min<int64_t>(max_length, unit_tokens - 1) : max_length / unit_tokens;
  const int64_t each = unit_bytes % 16 == 0 ? 16 : 8;
  it.pieces = static_cast<int>((most * unit_bytes + THREADS * each - 1) / (THREADS * each));
  if (it.pieces == 0) return;
  it.first_cta = static_cast<int>(std::min<int64_t>(ctas, INT32_MAX));
  ctas += int64_t(it.pieces) * layers * heads;
  ++p.n_items;
}

int check(const char* what, int layers, int groups, int beams, int heads, int head_dim, int64_t capacity, int length,
          const int* length_dev) {
  const std::string w(what);
  if (layers < 0 || groups < 0 || beams <= 0 || heads <= 0 || head_dim <= 0 || capacity < 0)
    return fail_invalid(w + ": invalid sizes");
  if (beams > 32) return set_error(TK_ERR_UNSUPPORTED, w + ": more than 32 beams");
  if (groups > 65535) return fail_invalid(w + ": too many groups");
  if (head_dim % 8) return set_error(TK_ERR_UNSUPPORTED, w + ": head_dim must be a multiple of 8");
  if (capacity > INT32_MAX) return fail_invalid(w + ": the cache is longer than 2^31 positions");
  if (!length_dev && (length < 0 || length > capacity)) return fail_invalid(w + ": length outside the cache");
  return TK_OK;
}

int run(Params& p, int64_t ctas, int groups, cudaStream_t st) {
  if (ctas == 0 || groups == 0 || p.beams == 1) return TK_OK;
  if (ctas > INT32_MAX) return fail_invalid("kv_reorder: the cache is too large for one launch");
  const int n = static_cast<int>(ctas);
  if (p.beams <= 4) return launch<4>(p, n, groups, st);
  if (p.beams <= 8) return launch<8>(p, n, groups, st);
  if (p.beams <= 16) return launch<16>(p, n, groups, st);
  return launch<32>(p, n, groups, st);
}

}  // namespace reorder
}  // namespace tk

extern "C" int tk_kv_reorder(void* k_cache, void* v_cache, const int64_t* parents, int layers, int groups, int beams,
                             int num_kv_heads, int capacity, int head_dim, int length, const int* length_device,
                             int dtype, void* stream) {
  using namespace tk;
  using namespace tk::reorder;
  if (!half_dtype(dtype)) return fail_invalid("kv_reorder: dtype must be F16 or BF16");
  if (int rc = check("kv_reorder", layers, groups, beams, num_kv_heads, head_dim, capacity, length, length_device))
    return rc;
  if (layers == 0 || groups == 0) return TK_OK;
  if (!k_cache || !v_cache || !parents) return fail_invalid("kv_reorder: NULL pointer");
  if (!aligned16(k_cache) || !aligned16(v_cache)) return fail_invalid("kv_reorder: caches must be 16-byte aligned");
  Params p{};
  p.beams = beams;
  p.parents = parents;
  p.length = length;
  p.length_dev = length_device;
  p.max_length = capacity;
  const int most = length_device ? capacity : length;
  int64_t ctas = 0;
  for (void* t : {k_cache, v_cache})
    add_item(p, ctas, t, layers, groups * beams, num_kv_heads, capacity, head_dim * 2, 1, false, most);
  return run(p, ctas, groups, static_cast<cudaStream_t>(stream));
}

extern "C" int tk_kv8_reorder(void* k_cache, void* v_cache, float* scales, void* tail, const int64_t* parents,
                              int layers, int groups, int beams, int num_kv_heads, int num_blocks, int head_dim,
                              int length, const int* length_device, void* stream) {
  using namespace tk;
  using namespace tk::reorder;
  const int64_t capacity = int64_t(num_blocks) * 32;
  if (int rc = check("kv8_reorder", layers, groups, beams, num_kv_heads, head_dim, capacity, length, length_device))
    return rc;
  if (layers == 0 || groups == 0) return TK_OK;
  if (!k_cache || !v_cache || !scales || !tail || !parents) return fail_invalid("kv8_reorder: NULL pointer");
  if (!aligned16(k_cache) || !aligned16(v_cache) || !aligned16(tail) || reinterpret_cast<uintptr_t>(scales) % 8)
    return fail_invalid("kv8_reorder: caches must be 16-byte aligned (scales: 8)");
  Params p{};
  p.beams = beams;
  p.parents = parents;
  p.length = length;
  p.length_dev = length_device;
  p.max_length = static_cast<int>(capacity);
  const int most = length_device ? static_cast<int>(capacity) : length;
  const int rows = groups * beams;
  int64_t ctas = 0;
  for (void* t : {k_cache, v_cache})
    add_item(p, ctas, t, layers, rows, num_kv_heads, num_blocks, 32 * head_dim, 32, false, most);
  add_item(p, ctas, scales, layers, rows, num_kv_heads, num_blocks, 8, 32, false, most);
  add_item(p, ctas, tail, layers, rows, 2 * num_kv_heads, 32, head_dim * 2, 32, true, most);
  return run(p, ctas, groups, static_cast<cudaStream_t>(stream));
}
