// Launch parameters of the drafted-token tree kernels (qd_tree_attention.hip,
// qd_tree_rows.hip, qd_tree_verify.hip), between them and the C ABI (qd_tree.cpp).
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

namespace qd {

// Rows of a tree's nodes, and of the cache they follow.  Strides in halves.
struct TreeRopeParams {
  const uint16_t* qkv;      // [nodes][(heads + 2 kv_heads) * 128]
  const uint16_t* bias;     // [(heads + 2 kv_heads) * 128] or null
  const int* depth;
  uint16_t* q_out;
  uint16_t* k_tree;
  uint16_t* v_tree;
  const float2* rope_cs;    // [max_seqlen][64] (cos, sin)
  long long qkv_stride, q_stride, row_stride, head_stride;
  int prefix, nodes, heads, kv_heads, max_seqlen;
};
hipError_t launch_tree_rope(const TreeRopeParams& p, hipStream_t stream);

struct TreeCommitParams {
  const uint16_t* src[2];   // node rows of K and of V
  uint16_t* dst[2];         // the caches
  long long src_layer, src_row, src_head;
  long long dst_layer, dst_row, dst_head;
  const int* path;
  const int* count;
  int prefix, nodes, layers, kv_heads, max_seqlen;
  int in_place;             // the node rows are the cache's own from prefix on
};
hipError_t launch_tree_commit(const TreeCommitParams& p, hipStream_t stream);

struct TreeAttnParams {
  const uint16_t* q;        // [nodes][heads][128]
  const uint16_t* k;        // cache rows [0, prefix)
  const uint16_t* v;
  const uint16_t* kt;       // node rows
  const uint16_t* vt;
  const uint64_t* mask;     // [nodes][ceil(nodes / 64)]
  uint16_t* out;
  long long q_stride, out_stride;
  long long row_stride, head_stride;      // cache
  long long trow_stride, thead_stride;    // node rows
  int prefix, nodes, kv_heads;
  int group;                // query heads per cache head
  float scale_log2;         // log2(e) / sqrt(128)
  int splits, rounds, block_rows;   // TreeAttnPlan
  // Partials, when splits > 1, per (block, cache head, split): the block's accumulators as
  // fragments [block_rows / 16][8][64 lanes], and its rows' (log2 reference, denominator).
  float __attribute__((ext_vector_type(4)))* part_o;
  float2* part_ml;
};

// Launch plan: blocks of block_rows query rows per cache head (a cache head's query rows are
// its nodes x the heads that share it), `splits` workgroups of eight waves for each, of which
// key_waves take different tiles of keys.
struct TreeAttnPlan {
  int block_rows, key_waves, blocks, splits, rounds;   // rounds: tiles of a key wave, at most
};

// max_splits: what the workspace is sized for, at any prefix.
//
// Block rows: the smallest of 16, 32 and 64 that holds all query rows, else 128-row blocks
// unless 64-row blocks leave fewer rows empty (192 rows, 32 query heads on 8 cache heads over
// 16001 rows: 32.4 us in 64-row blocks, 33.7 in 128-row ones).
// Splits: at most one workgroup per CU, and no more than the rounds need: a key wave takes a
// tile per round, and every further split adds partials to write and fold (16 cache heads, 64
// nodes over 4096 rows, 3 rounds: 18.6 us at 12 splits, 19.5 at 16; 27 nodes over 4096 rows,
// 2 rounds: 13.3 at 9, 14.0 at 16).  One split, without the second launch, where its rounds
// cost no more than that launch (5 nodes over 512 rows, 3 rounds: 7.6 against 7.9 us, and one
// launch less for the host; over 1024 rows, 5 rounds: 9.1 against 8.3).
inline TreeAttnPlan tree_attn_plan(int nodes, int heads, int kv_heads, int prefix, int num_cus, int* max_splits) {
  TreeAttnPlan plan;
  const int rows = nodes * (heads / kv_heads);
  const bool wide = (rows + 127) / 128 * 2 == (rows + 63) / 64;
  plan.block_rows = rows <= 16 ? 16 : rows <= 32 ? 32 : wide ? 128 : 64;
  plan.key_waves = rows <= 32 ? 8 : wide ? 2 : 4;
  plan.blocks = (rows + plan.block_rows - 1) / plan.block_rows;
  const int most = num_cus / (plan.blocks * kv_heads);
  *max_splits = most < 1 ? 1 : most;
  const int tiles = (prefix + 31) / 32 + (nodes + 31) / 32;
  const int groups = (tiles + plan.key_waves - 1) / plan.key_waves;   // rounds of one split
  plan.rounds = (groups + *max_splits - 1) / *max_splits;
  plan.splits = (groups + plan.rounds - 1) / plan.rounds;
  if (groups <= (plan.key_waves == 8 ? 3 : 2)) {
    plan.splits = 1;
    plan.rounds = groups;
  }
  return plan;
}
hipError_t launch_tree_attention(const TreeAttnParams& p, const TreeAttnPlan& plan, hipStream_t stream);

// Logits of a row per chunk of the verification's passes, and chunks per workgroup: as many as
// leave four workgroups per CU (5 rows of 151936 logits, argmax pass, 3.8 us at 1 chunk, 5.8 at
// 4, which leaves CUs empty; 64 rows, sums of weights, 14.7 us at 1, 14.1 at 4), at most 16.
constexpr int kVerifyChunk = 2048;
constexpr int kVerifyRuns = 16;
inline int verify_runs(int nodes, int chunks) {
  const long long n = (long long)nodes * chunks / 1024;
  return n < 1 ? 1 : n > kVerifyRuns ? kVerifyRuns : (int)n;
}

struct TreeVerifyParams {
  const uint16_t* target;   // [nodes][vocab]
  const uint16_t* draft;    // the drafter's, or null
  const int* tokens;
  const int* parents;
  const float* accept_u;
  const float* sample_u;
  int* path;
  int* emitted;
  int* count;
  // Workspace.  A group is the chunks of one workgroup; per side (target, draft), node and group
  // the largest logit and the sum of weights relative to it (greedy: the argmax and its logit),
  // per chunk its part of that sum; then per round, node and chunk the sums of max(p - A q, 0).
  double* sums;             // [2][nodes][chunks]
  double* group_sums;       // [2][nodes][groups]
  double* rounds;           // [max_children][nodes][chunks]
  float* maxes;             // [2][nodes][groups]
  int* args;                // [nodes][groups]
  long long ldt, ldd;
  double scale_log2;        // 32 log2(e) / temperature
  int nodes, vocab, chunks, runs, groups, max_children;   // groups: workgroups per row
  int greedy;
};
hipError_t launch_tree_verify(const TreeVerifyParams& p, hipStream_t stream);

}  // namespace qd
