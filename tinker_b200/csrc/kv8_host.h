// Host-side pieces that the 8-bit KV cache entry points share.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace tk {
namespace kv8 {

// The tensors of one layer's 8-bit cache (kv8.cuh).
struct Cache {
  void* k;
  void* v;
  float* scales;
  void* tail;
  int num_blocks;
  int format;
};

int check_cache(const char* what, const Cache& c, int batch, int seq, int num_heads, int num_kv_heads, int head_dim,
                int dtype);

// Append launch; with cos_t the keys are rotated at their positions. The position is start_pos, or
// start_dev[b * start_step] of sequence b.
int append(const Cache& c, const void* k, int64_t ks, const void* v, int64_t vs, const float* cos_t,
           const float* sin_t, int64_t table_rows, int batch, int seq, int num_kv_heads, int head_dim, int start_pos,
           const int* start_dev, int start_step, int dtype, cudaStream_t st);

// The tensor-core form for many query rows (kv8_chunk.cu); appends nothing.
constexpr int CHUNK_MIN_ROWS = 64;  // query rows of a kv head, of two new tokens or more
bool chunk_fits(int batch, int num_heads, int num_kv_heads, int seq, int64_t len);
int64_t chunk_workspace(int batch, int num_heads, int num_kv_heads, int head_dim, int seq, int64_t len, int sm_count);
int chunk_launches(int batch, int num_heads, int num_kv_heads, int head_dim, int seq, int64_t len, int dtype,
                   int sm_count);
int chunk_attention(const Cache& c, const void* q, int64_t qs, const void* k, int64_t ks, const void* v, int64_t vs,
                    const float* cos_t, const float* sin_t, void* out, int64_t os, int batch, int seq, int num_heads,
                    int num_kv_heads, int head_dim, int start_pos, void* workspace, int dtype, int sm_count,
                    cudaStream_t st);

}  // namespace kv8
}  // namespace tk
