// Rows of a tree of drafted tokens (gfx950): QKV bias + rotate-half RoPE of its
// nodes, and the copy of an accepted path's K/V rows into the caches.
//
// Both are bound by a launch's own time at the sizes a step has (a few hundred
// KB), so each is one launch with 16-byte accesses and nothing shared between
// threads (MI355X: 5 nodes 2.9 us, 250 nodes of 32 + 16 heads 3.6 us; 4 and 60
// rows into 24 layers of 16 heads 3.9 and 8.0 us, the latter 24 MB moved at 3.0
// TB/s).  The rotation is qd_qkv_bias_rope_cache's, operation for operation: fp32
// products, rounded once each (no contraction), cos and sin from the context's
// table.
#include "qd_device.h"
#include "qd_internal.h"
#include "qd_tree.h"

namespace qd {
namespace {

// A thread takes eight rotation pairs (i, i + 64) of one head of one node, or
// the same elements of a V head.  Sections of a row: Q heads, K heads, V heads.
__global__ __launch_bounds__(256) void tree_rope_kernel(TreeRopeParams p) {
#pragma clang fp contract(off)
  const int per_node = (p.heads + 2 * p.kv_heads) * 8;
  const int gid = blockIdx.x * 256 + threadIdx.x;
  const int sec = gid >> 3;                        // head of the row
  const int i0 = 8 * (gid & 7);
  const int t = blockIdx.y;
  if (gid >= per_node) return;
  const _Float16* src = reinterpret_cast<const _Float16*>(p.qkv) + t * p.qkv_stride + sec * 128 + i0;
  const f16x8 a = *reinterpret_cast<const f16x8*>(src);
  const f16x8 b = *reinterpret_cast<const f16x8*>(src + 64);
  f16x8 x1 = a, x2 = b;
  if (p.bias) {
    const _Float16* bias = reinterpret_cast<const _Float16*>(p.bias) + sec * 128 + i0;
    const f16x8 b1 = *reinterpret_cast<const f16x8*>(bias), b2 = *reinterpret_cast<const f16x8*>(bias + 64);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x1[e] = (_Float16)((float)a[e] + (float)b1[e]);
      x2[e] = (_Float16)((float)b[e] + (float)b2[e]);
    }
  }
  const int depth = p.depth[t];
  const long long pos = (long long)p.prefix + depth;
  const bool ok = depth >= 0 && pos < p.max_seqlen;
  _Float16* dst;
  if (sec < p.heads)
    dst = reinterpret_cast<_Float16*>(p.q_out) + t * p.q_stride + sec * 128 + i0;
  else if (sec < p.heads + p.kv_heads)
    dst = reinterpret_cast<_Float16*>(p.k_tree) + t * p.row_stride + (sec - p.heads) * p.head_stride + i0;
  else
    dst = reinterpret_cast<_Float16*>(p.v_tree) + t * p.row_stride + (sec - p.heads - p.kv_heads) * p.head_stride + i0;
  if (!ok) {                                       // no such position: NaN shows the mistake
#pragma unroll
    for (int e = 0; e < 8; ++e) x1[e] = x2[e] = (_Float16)__builtin_nanf("");
  } else if (sec < p.heads + p.kv_heads) {
    const float4* cs = reinterpret_cast<const float4*>(p.rope_cs + pos * 64 + i0);   // two pairs each
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float4 c = cs[j];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int e = 2 * j + u;
        const float co = u ? c.z : c.x, si = u ? c.w : c.y;
        const float v1 = (float)x1[e], v2 = (float)x2[e];
        const float v1c = v1 * co, v2s = v2 * si, v2c = v2 * co, v1s = v1 * si;
        x1[e] = to_f16(v1c - v2s);
        x2[e] = to_f16(v2c + v1s);
      }
    }
  }
  *reinterpret_cast<f16x8*>(dst) = x1;
  *reinterpret_cast<f16x8*>(dst + 64) = x2;
}

// A thread moves one 16-byte column of the path's rows of one layer, K or V, in
// batches of kRows rows: the loads of a batch are in flight together, then its
// stores.  In place, one thread walks all batches of its column in order: a
// batch's destinations i <= path[i] lie below every later batch's sources (path
// ascending), so no row is overwritten before it is read.  Apart, each batch is
// a workgroup of its own (blockIdx.y).
constexpr int kCommitRows = 8;
__global__ __launch_bounds__(256) void tree_commit_kernel(TreeCommitParams p) {
  const int cols = p.kv_heads * 16;                // 16-byte chunks of a row
  const int col = blockIdx.x * 256 + threadIdx.x;
  if (col >= cols) return;
  const int layer = blockIdx.z >> 1, kv = blockIdx.z & 1;
  const int h = col >> 4, d = 8 * (col & 15);
  const int n = min(min(*p.count, p.nodes), p.max_seqlen - p.prefix);
  const uint16_t* src = p.src[kv] + layer * p.src_layer + h * p.src_head + d;
  uint16_t* dst = p.dst[kv] + layer * p.dst_layer + p.prefix * p.dst_row + h * p.dst_head + d;
  const int step = p.in_place ? kCommitRows : (int)gridDim.y * kCommitRows;
  for (int i0 = p.in_place ? 0 : (int)blockIdx.y * kCommitRows; i0 < n; i0 += step) {
    int row[kCommitRows];
    f16x8 x[kCommitRows];
#pragma unroll
    for (int i = 0; i < kCommitRows; ++i) {
      row[i] = i0 + i < n ? p.path[i0 + i] : -1;
      if (row[i] >= p.nodes) row[i] = -1;
      if (row[i] >= 0) x[i] = *reinterpret_cast<const f16x8*>(src + row[i] * p.src_row);
    }
#pragma unroll
    for (int i = 0; i < kCommitRows; ++i)
      if (row[i] >= 0) *reinterpret_cast<f16x8*>(dst + (long long)(i0 + i) * p.dst_row) = x[i];
  }
}

}  // namespace

hipError_t launch_tree_rope(const TreeRopeParams& p, hipStream_t stream) {
  const int per_node = (p.heads + 2 * p.kv_heads) * 8;
  hipLaunchKernelGGL(tree_rope_kernel, dim3((per_node + 255) / 256, p.nodes), dim3(256), 0, stream, p);
  return hipGetLastError();
}

hipError_t launch_tree_commit(const TreeCommitParams& p, hipStream_t stream) {
  const int cols = p.kv_heads * 16;
  const int batches = p.in_place ? 1 : (p.nodes + kCommitRows - 1) / kCommitRows;
  hipLaunchKernelGGL(tree_commit_kernel, dim3((cols + 255) / 256, batches, 2 * p.layers), dim3(256), 0, stream, p);
  return hipGetLastError();
}

}  // namespace qd
