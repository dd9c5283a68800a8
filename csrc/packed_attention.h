// Kernel-side interface of the packed attention (see packed_attention_sm100.cu).
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

namespace appcorr {

constexpr int kPaRows = 256;                // query rows of one tile: two 128-row halves
constexpr int kPaSlotsPerBlock = 2;         // partial results a block may leave behind

struct PackedAttnParams {
  int B, N;            // requests; packed rows of q / o
  int H, Hv, ng;       // query heads; key heads times sub-groups; sub-groups per key head
  int G, TT;           // query heads of a sub-group; tokens of a 128-row half tile (128 / G)
  const int* q_start;  // [B + 1]
  const int* kv_len;   // [B]
  const int* table;    // [B, W] pages (prefix pass: the prefix's page list), nullptr: packed rows
  long ld_table;
  int W;
  const int* k_start;  // [B] first key row of packed keys
  int pages;           // whole pages of the pool
  int key_rows;        // rows of k / v
  int shared_len;      // prefix pass: keys of the shared prefix, all visible to every token
  float scale_log2;
  __nv_bfloat16* o;
  long ldo;
  float* lse;          // [N, H] natural log-sum-exp or nullptr
  float* prior;        // [N, H, D] normalised result of the prefix pass and its
  float* prior_lse;    // [N, H] log2-sum-exp: written by the prefix pass, joined by the other (nullptr: none)
  float* slots;        // [2 * blocks, 256, D] partial results, [2 * blocks, 256, 2] their max and sum
  float* slot_ml;
  int* counters;       // [blocks, 8] arrivals at a cut tile; zero between launches
  int* err;
};

// Blocks launched (one per SM) and bytes of the three workspace parts.
int packed_attention_blocks();
void launch_packed_attention(int head_dim, bool prefix_pass, const CUtensorMap& q, const CUtensorMap& q1,
                             const CUtensorMap& k, const CUtensorMap& v, const PackedAttnParams& p, cudaStream_t stream);

}  // namespace appcorr
