// Kernel-side interface of the packed attention (see packed_attention_sm100.cu).
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

namespace appcorr {

constexpr int kPaRows = 256;                // query rows of one tile: two 128-row halves
constexpr int kPaSlotsPerBlock = 2;         // partial results a block may leave behind

struct CutTile {  // a tile whose keys several blocks share, noted by the one that began it
  int parts;      // which blocks (< 0: none)
  int tok0, ntok, hv;
};

struct PackedAttnParams {
  int B, N;            // requests; packed rows of q / o
  int H, Hv, ng;       // query heads; key heads times sub-groups; sub-groups per key head
  int G, TT;           // query heads of a sub-group; tokens of a 128-row half tile (128 / G)
  const int* q_start;  // [B + 1]
  const int* kv_len;   // [B]
  const int* table;    // [B, W] pages, nullptr: packed key rows
  long ld_table;
  int W;
  const int* k_start;  // [B] first key row of packed keys
  int pages;           // whole pages of the pool
  int key_rows;        // rows of k / v
  const int* prefix;   // pages of the shared prefix, how many, and its keys (0: no prefix)
  int prefix_pages;
  int shared_len;
  float scale_log2;
  __nv_bfloat16* o;
  long ldo;
  float* lse;          // [N, H] natural log-sum-exp or nullptr
  float* slots;        // [2 * blocks, 256, D] parts of cut tiles, [2 * blocks, 256, 2] their max and sum
  float* slot_ml;
  CutTile* cuts;       // [blocks]
  float* row_o;        // with a prefix: [2, N, H, D] results of whole tiles (own keys, prefix),
  float* row_ml;       // [2, N, H, 2] their max and sum,
  int* row_parts;      // [2, N, H] the row's parts
  int* err;
};

int packed_attention_blocks();  // one per SM
void launch_packed_attention(int head_dim, const CUtensorMap& q, const CUtensorMap& q1, const CUtensorMap& k,
                             const CUtensorMap& v, const PackedAttnParams& p, cudaStream_t stream);

}  // namespace appcorr
