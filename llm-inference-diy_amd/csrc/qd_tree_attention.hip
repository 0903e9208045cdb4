// Attention of a tree of drafted tokens over a KV cache (gfx950).
#include "qd_device.h"
#include "qd_internal.h"
#include "qd_tree.h"

namespace qd {
namespace {

// One workgroup per (node, head); its four waves take rows in turn.  Lane l
// holds dims 2 l and 2 l + 1.
__global__ __launch_bounds__(256) void tree_attention_kernel(TreeAttnParams p) {
  __shared__ float so[4][128], sm[4], sl[4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int h = blockIdx.x % p.heads, t = blockIdx.x / p.heads;
  const int kh = h / (p.heads / p.kv_heads);
  const int words = (p.nodes + 63) / 64;
  const f16x2 qv = *reinterpret_cast<const f16x2*>(p.q + t * p.q_stride + h * 128 + 2 * lane);
  float m = -__builtin_inff(), l = 0.0f, o0 = 0.0f, o1 = 0.0f;
  for (int j = wave; j < p.prefix + p.nodes; j += 4) {
    const int n = j - p.prefix;
    if (n >= 0 && !((p.mask[(long long)t * words + n / 64] >> (n % 64)) & 1)) continue;
    const uint16_t* k = n < 0 ? p.k + j * p.row_stride + kh * p.head_stride : p.kt + n * p.trow_stride + kh * p.thead_stride;
    const uint16_t* v = n < 0 ? p.v + j * p.row_stride + kh * p.head_stride : p.vt + n * p.trow_stride + kh * p.thead_stride;
    const f16x2 kv = *reinterpret_cast<const f16x2*>(k + 2 * lane);
    const f16x2 vv = *reinterpret_cast<const f16x2*>(v + 2 * lane);
    const float s = wave64_sum((float)qv[0] * (float)kv[0] + (float)qv[1] * (float)kv[1]) * p.scale_log2;
    const float mn = fmaxf(m, s);
    const float a = m == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
    const float w = mn == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(s - mn);
    l = l * a + w;
    o0 = o0 * a + w * (float)vv[0];
    o1 = o1 * a + w * (float)vv[1];
    m = mn;
  }
  so[wave][2 * lane] = o0;
  so[wave][2 * lane + 1] = o1;
  if (lane == 0) {
    sm[wave] = m;
    sl[wave] = l;
  }
  __syncthreads();
  if (threadIdx.x < 128) {
    float mx = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3])), acc = 0.0f, den = 0.0f;
    for (int w = 0; w < 4; ++w) {
      const float a = sm[w] == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(sm[w] - mx);
      acc += a * so[w][threadIdx.x];
      den += a * sl[w];
    }
    reinterpret_cast<_Float16*>(p.out)[t * p.out_stride + h * 128 + threadIdx.x] =
        to_f16(den > 0.0f || den != den ? acc / den : 0.0f);
  }
}

}  // namespace

hipError_t launch_tree_attention(const TreeAttnParams& p, hipStream_t stream) {
  hipLaunchKernelGGL(tree_attention_kernel, dim3(p.nodes * p.heads), dim3(256), 0, stream, p);
  return hipGetLastError();
}

}  // namespace qd
