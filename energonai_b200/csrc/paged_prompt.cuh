// What paged_attention.cu and paged_prompt.cu tell each other.
#pragma once

#include "paged.cuh"

namespace eb {

struct PromptParams {
  PagedBatch batch;
  const void *q;
  void *o;
  long long ldq, ldo;
  const void *k_pages, *v_pages;
  const float *k_scale, *v_scale;
  int kv_heads, group, window, few;      // few: sequences with no more rows (tokens x group) than this are left to the step kernel
  float scale_log2;
  float *part;                           // [batch][kv_heads][blocks][splits][256][D + 2], or null: one split
  int splits, split_tiles;
  int q_tma;                             // the heads of a group divide a row tile: queries come by tensor map
};
struct PromptPlan {
  int blocks, splits, split_tiles;       // CTAs of 256 rows per key / value head, splits of so many key tiles
};
PromptPlan prompt_plan(int batch, int kv_heads, int rows_per_head, long long keys);
int paged_prompt(PromptParams p, const PromptPlan &s, int head_dim, int dtype, cudaStream_t st);

}  // namespace eb
