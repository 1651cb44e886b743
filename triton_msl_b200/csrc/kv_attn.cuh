// What the two kernels of attention over the 4-bit cache share (kv_attn.cu,
// kv_attn_mma.cu).
#pragma once
#include <cuda_runtime.h>
#include <cstddef>
#include <cstdint>

#include "decoder.cuh"

namespace b2 {

struct AttnArgs {
  const void* q;
  void* o;
  const uint8_t *k_codes, *v_codes;
  const uint32_t *k_scales, *v_scales;
  const int32_t *page_table, *lengths;
  long long qb, qn, qh, ob, on, oh, table_stride;
  int B, N, Hq, H, G, page_size, num_pages, max_pages;
  int rows;        // N * G rows share a key head
  int row_blocks;  // of 4, 8 or 16 rows
  FastDiv page_div;  // by page_size
  int q_vec;       // q may be read 16 bytes at a time
  float scale_log2;
  float* partials;
  uint32_t* status;
};

size_t kv_attn_mma_workspace(int64_t rows, int64_t D);
int kv_attn_mma_launch(AttnArgs& a, int D, int group, int dtype, cudaStream_t st);

}  // namespace b2
