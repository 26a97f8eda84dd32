// What the kernels of prompt_attn and shared_prefix_attn share: the segments of a call, the plan of their work and
// the partial results.
//
// A call is a list of SEGMENTS: a run of consecutive query tokens that attend to the same pages.  prompt_attn has
// one per sequence (causal); shared_prefix_attn one per sequence (its own pages) and one per group (the prefix, no
// mask).  With G query heads per KV head, the rows of a segment for one KV head are its tokens x G, packed, so a
// K/V page is read once for all of them.
// Segments of at most 8 (or 16) rows go to the row kernel (a warp-level tensor-core tile of as many rows; bound by reading
// K and V): all their (KV head, page) units in one line, cut into equal runs, one per warp of the GPU.  Longer
// segments go to the tile kernel in tiles of up to 256 rows; where there are fewer of those than the GPU runs at once,
// the keys are cut into chunks too.  Partial (reference, sum, accumulator) triples are joined by the merge kernel.
#pragma once
#include "common.cuh"

namespace twl {

constexpr int kFewRows = 16;  // most rows of a segment of the row kernel

// The largest weight of a row, as a power of two: weights 2^(x - reference) go to the tensor cores in the model type, and fp16 rounds
// those below 2^-14 in steps of 2^-24 and drops those below 2^-25.  Up here n weights are off by at most n 2^-40 of the largest one
// altogether (n 2^-25 with the largest at 1: a step of fp16 from 32K keys on).  bf16 has the exponents of fp32.
template <typename T>
constexpr float kTopWeight = 15.f;
template <>
inline constexpr float kTopWeight<__nv_bfloat16> = 0.f;

struct Segment {
  int32_t tok0, ntok;     // query tokens
  int32_t kvbase, npages; // its part of kv_indices (or of the prefix's)
  int32_t len;            // tokens of the pages
  int32_t units;          // row kernel: pages of a KV head; 0 for the tile kernel's segments
  int32_t chunks;         // tile kernel: key chunks of every tile
  int32_t chunk_pages;    // and their pages
  int32_t second;         // 1: pages of the prefix table
  int32_t few;            // 1: the row kernel's
  int64_t start;          // row kernel: its first unit in the line
  int64_t pbase;          // first partial row, or -1 where tiles write the output themselves
};

struct PlanHeader {
  int64_t units;         // of the row kernel
  int32_t per_warp;      // units of a warp
  int32_t tile_items;    // per KV head
  int32_t merge;         // some output row is joined from partial results
  int32_t next_tile;     // work counter of the tile kernel
};

struct AttnParams {
  const void *q, *k_pages, *v_pages;
  void* out;
  float* lse;
  int64_t q_ts, o_ts;  // token strides in elements; heads are 128 apart
  // segments 0..n_first-1: table 1; n_first.. : table 2 (the prefix)
  const int32_t *qo1, *indptr1, *indices1, *last1;  // qo1 null: one token per segment
  const int32_t *qo2, *indptr2, *indices2, *last2;
  int32_t n_first, n_second, causal, always_partial;
  // block lists (prompt_attn): rows of kvh of query block j of sequence b at slot qo1[b]/query_block + b + j
  const int32_t *block_pages, *block_npages;
  int32_t max_k, query_block;
  int32_t num_tokens, Hq, Hkv, G, num_pages_total, tok_tile;
  int32_t row_warps, tile_target, row_tile;
  float scale_log2;
  // workspace
  PlanHeader* hdr;
  Segment* segs;
  int4* tile_list;  // {segment, first token, tokens, chunk}
  int32_t tile_cap;
  float* part_acc;  // [rows][128]
  float2* part_ml;  // [rows] {reference in log2 units, sum of the weights}
  int64_t part_cap;
  int32_t* status;
};

// pages that rows up to token `tok` (of the segment) may see
__device__ __forceinline__ int pages_seen(const Segment& s, int tok, int causal) {
  if (!causal) return s.npages;
  const int pos = s.len - s.ntok + tok;
  return pos < 0 ? 0 : min(s.npages, (pos >> 4) + 1);
}

int tile_attention_launch(const AttnParams& p, int dtype, cudaStream_t st);

}  // namespace twl
