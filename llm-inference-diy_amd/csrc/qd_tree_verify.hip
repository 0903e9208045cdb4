// Verification of a tree of drafted tokens against the target's logits (gfx950).
//
// Everything a decision depends on is held in 64 bits: weights
//   w(v) = 2^((l(v) - M) log2(e) / temperature),  M the row's largest logit,
// their sums, and the residuals max(p - A q, 0).  A decision compares a random
// number with a ratio of such sums, and the last token is the first index whose
// cumulative weight passes a random share of the total: with a vocabulary of
// 150 thousand, fp32 sums would move the chosen index.  (fp64 fused multiply-adds
// issue at the fp32 rate on this part, so this costs little.)
//
// Residuals of drawn drafts in closed form: with p normalised, A_0 = 0, S_0 = 1,
// the distribution after j rejections is max(p - A_j q, 0) / S_j, where
//   A_{j+1} = A_j + S_j,   S_{j+1} = sum_v max(p(v) - A_{j+1} q(v), 0),
// since max(p - A_j q, 0)/S_j - q = (p - (A_j + S_j) q)/S_j wherever it is positive.
//
// Passes: (1) every (row, chunk of kVerifyChunk logits) gives its largest logit
// and its sum of weights relative to it, or its argmax; (2) with drawn drafts,
// per round j <= max_children, the chunks' sums of S_j, for every node with at
// least j children; (3) one workgroup reduces the rows' partials, decides every
// node's children (a node's decisions do not depend on how it was reached), walks
// from node 0, and takes the last token from one chunk.
#include "qd_device.h"
#include "qd_internal.h"
#include "qd_tree.h"
#include "qdiy/decode.h"

namespace qd {
namespace {

typedef _Float16 f16x8u __attribute__((ext_vector_type(8), aligned(2)));   // rows need not be 16-byte aligned

constexpr int kNodes = QD_TREE_MAX_NODES;

// 2^x for x <= 0, relative error below 1e-12: 2^n times the Taylor series of
// exp(f ln 2) to degree 10 on |f| <= 1/2 (remainder (ln2/2)^11 / 11! = 2e-13).
// Below 2^-1000: 0.
__device__ __forceinline__ double exp2_neg(double x) {
  const double n = __builtin_rint(x);
  const double f = (x - n) * 0.6931471805599453;
  double r = 1.0 / 3628800.0;
  r = __builtin_fma(r, f, 1.0 / 362880.0);
  r = __builtin_fma(r, f, 1.0 / 40320.0);
  r = __builtin_fma(r, f, 1.0 / 5040.0);
  r = __builtin_fma(r, f, 1.0 / 720.0);
  r = __builtin_fma(r, f, 1.0 / 120.0);
  r = __builtin_fma(r, f, 1.0 / 24.0);
  r = __builtin_fma(r, f, 1.0 / 6.0);
  r = __builtin_fma(r, f, 0.5);
  r = __builtin_fma(r, f, 1.0);
  r = __builtin_fma(r, f, 1.0);
  return x > -1000.0 ? __builtin_ldexp(r, (int)fmax(n, -1100.0)) : 0.0;
}

// Weight of logit l in a row (or chunk) whose largest logit is m; NaN counts as
// -inf.  The largest itself weighs 1, also where it is infinite.
__device__ __forceinline__ double weight(float l, float m, double scale) {
  if (l != l) l = -__builtin_inff();
  return l == m ? 1.0 : exp2_neg(((double)l - (double)m) * scale);
}

__device__ __forceinline__ double wave_sum(double x) {
#pragma unroll
  for (int d = 32; d; d >>= 1) x += __shfl_xor(x, d);
  return x;
}

// Eight logits from index v on; -inf past the row's end.
__device__ __forceinline__ void load8(const uint16_t* row, int v, int vocab, float (&x)[8]) {
  if (v + 8 <= vocab) {
    const f16x8u a = *reinterpret_cast<const f16x8u*>(row + v);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = (float)a[e];
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      x[e] = v + e < vocab ? (float)reinterpret_cast<const _Float16*>(row)[v + e] : -__builtin_inff();
  }
}

constexpr int kThreads = 256;
constexpr int kRuns = kVerifyChunk / (8 * kThreads);   // runs of 8 logits per thread

// (1) Sampled: blockIdx = (chunk, node, side).
__global__ __launch_bounds__(kThreads) void verify_stats_kernel(TreeVerifyParams p) {
  __shared__ float sm[kThreads / 64];
  __shared__ double ss[kThreads / 64];
  const int t = blockIdx.y, side = blockIdx.z, c = blockIdx.x;
  const uint16_t* row = side ? p.draft + t * p.ldd : p.target + t * p.ldt;
  const int v0 = c * kVerifyChunk + 8 * threadIdx.x;
  float x[kRuns][8];
  float m = -__builtin_inff();
#pragma unroll
  for (int r = 0; r < kRuns; ++r) {
    load8(row, v0 + 8 * kThreads * r, p.vocab, x[r]);
#pragma unroll
    for (int e = 0; e < 8; ++e) m = fmaxf(m, x[r][e]);            // fmaxf passes NaN over
  }
  m = wave64_max(m);
  if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) m = fmaxf(m, sm[w]);
  double s = 0.0;
#pragma unroll
  for (int r = 0; r < kRuns; ++r)
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (v0 + 8 * kThreads * r + e < p.vocab) s += weight(x[r][e], m, p.scale_log2);
  s = wave_sum(s);
  if ((threadIdx.x & 63) == 0) ss[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kThreads / 64; ++w) s += ss[w];
    const long long at = ((long long)side * p.nodes + t) * p.chunks + c;
    p.maxes[at] = m;
    p.sums[at] = s;
  }
}

// (1) Greedy: the chunk's largest logit and its lowest index; no number, no index
// (INT_MAX).
__device__ __forceinline__ void better(float& m, int& i, float m2, int i2) {
  if (m2 > m || (m2 == m && i2 < i)) {
    m = m2;
    i = i2;
  }
}
__global__ __launch_bounds__(kThreads) void verify_argmax_kernel(TreeVerifyParams p) {
  __shared__ float sm[kThreads / 64];
  __shared__ int si[kThreads / 64];
  const int t = blockIdx.y, c = blockIdx.x;
  const uint16_t* row = p.target + t * p.ldt;
  const int v0 = c * kVerifyChunk + 8 * threadIdx.x;
  float m = -__builtin_inff();
  int at = 0x7fffffff;
#pragma unroll
  for (int r = 0; r < kRuns; ++r) {
    float x[8];
    const int v = v0 + 8 * kThreads * r;
    load8(row, v, p.vocab, x);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (v + e < p.vocab && x[e] == x[e]) better(m, at, x[e], v + e);
  }
#pragma unroll
  for (int d = 32; d; d >>= 1) better(m, at, __shfl_xor(m, d), __shfl_xor(at, d));
  if ((threadIdx.x & 63) == 0) {
    sm[threadIdx.x >> 6] = m;
    si[threadIdx.x >> 6] = at;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kThreads / 64; ++w) better(m, at, sm[w], si[w]);
    p.maxes[(long long)t * p.chunks + c] = m;
    p.args[(long long)t * p.chunks + c] = at;
  }
}

// A row's largest logit and its sum of weights relative to it, by one wave.
__device__ __forceinline__ void row_stats(const TreeVerifyParams& p, int side, int t, int lane, float& m, double& z) {
  const long long at = ((long long)side * p.nodes + t) * p.chunks;
  m = -__builtin_inff();
  for (int c = lane; c < p.chunks; c += 64) m = fmaxf(m, p.maxes[at + c]);
  m = wave64_max(m);
  z = 0.0;
  for (int c = lane; c < p.chunks; c += 64) z += p.sums[at + c] * weight(p.maxes[at + c], m, p.scale_log2);
  z = wave_sum(z);
}

// The sum over chunks of round r (from 1) of node t, by one wave.
__device__ __forceinline__ double round_total(const TreeVerifyParams& p, int r, int t, int lane) {
  const double* s = p.rounds + ((long long)(r - 1) * p.nodes + t) * p.chunks;
  double z = 0.0;
  for (int c = lane; c < p.chunks; c += 64) z += s[c];
  return wave_sum(z);
}

// A and S of a node after `rejected` rejections (rounds whose sum is 0 change
// nothing), and the last round that counted (0: p itself).
struct Residual {
  double a, s;
  int round;
};
__device__ __forceinline__ Residual residual(const TreeVerifyParams& p, int t, int rejected, int lane) {
  Residual r{0.0, 1.0, 0};
  for (int j = 1; j <= rejected; ++j) {
    const double s = round_total(p, j, t, lane);
    if (s > 0.0) {
      r.a += r.s;
      r.s = s;
      r.round = j;
    } else {
      break;                 // p stays as it was, and so does every later round's sum: 0
    }
  }
  return r;
}

// (2) Round `round` of drawn drafts: blockIdx = (chunk, node).
__global__ __launch_bounds__(kThreads) void verify_round_kernel(TreeVerifyParams p, int round) {
  __shared__ double ss[kThreads / 64];
  __shared__ int kids[kThreads / 64];
  const int t = blockIdx.y, c = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int n = 0;
  for (int s = t + 1 + threadIdx.x; s < p.nodes; s += kThreads) n += p.parents[s] == t;
#pragma unroll
  for (int d = 32; d; d >>= 1) n += __shfl_xor(n, d);
  if (lane == 0) kids[wave] = n;
  __syncthreads();
  n = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) n += kids[w];
  if (n < round) return;                             // uniform over the workgroup
  float mp, mq;
  double zp, zq;
  row_stats(p, 0, t, lane, mp, zp);
  row_stats(p, 1, t, lane, mq, zq);
  const Residual r = residual(p, t, round - 1, lane);
  const bool kept = r.round != round - 1;            // an earlier round's sum was 0
  const double a = (r.a + r.s) / zq, ip = 1.0 / zp;
  const uint16_t* rp = p.target + t * p.ldt;
  const uint16_t* rq = p.draft + t * p.ldd;
  double s = 0.0;
  if (!kept) {
    for (int i = 0; i < kRuns; ++i) {
      const int v = c * kVerifyChunk + 8 * (threadIdx.x + kThreads * i);
      float x[8], y[8];
      load8(rp, v, p.vocab, x);
      load8(rq, v, p.vocab, y);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (v + e < p.vocab) s += fmax(weight(x[e], mp, p.scale_log2) * ip - weight(y[e], mq, p.scale_log2) * a, 0.0);
    }
  }
  s = wave_sum(s);
  if (lane == 0) ss[wave] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kThreads / 64; ++w) s += ss[w];
    p.rounds[((long long)(round - 1) * p.nodes + t) * p.chunks + c] = s;
  }
}

__device__ __forceinline__ float logit(const uint16_t* row, int v) {
  return (float)reinterpret_cast<const _Float16*>(row)[v];
}

// (3) One workgroup.
constexpr int kWalkThreads = 1024;
constexpr int kWalkWaves = kWalkThreads / 64;
constexpr int kPer = kVerifyChunk / kWalkThreads;      // 8 logits of the last chunk per thread
static_assert(kPer == 8, "the last token's chunk is one run of 8 logits per thread");

struct WalkShared {
  int parent[kNodes], token[kNodes], next[kNodes], path[kNodes], best[kNodes];
  float mp[kNodes], mq[kNodes];
  double zp[kNodes], zq[kNodes];
  double wave[kWalkWaves];
  unsigned gone[kVerifyChunk / 32];                    // rejected tokens of one chunk
  int count, chunk, last;
  double before, total;
};

// Sum over the workgroup; every thread receives it.
__device__ __forceinline__ double block_sum(double x, WalkShared& sh) {
  x = wave_sum(x);
  __syncthreads();                                     // sh.wave may still be read
  if ((threadIdx.x & 63) == 0) sh.wave[threadIdx.x >> 6] = x;
  __syncthreads();
  double s = 0.0;
#pragma unroll
  for (int w = 0; w < kWalkWaves; ++w) s += sh.wave[w];
  return s;
}

__global__ __launch_bounds__(kWalkThreads) void verify_walk_kernel(TreeVerifyParams p) {
  __shared__ WalkShared sh;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const bool drawn = !p.greedy && p.draft != nullptr;
  for (int t = tid; t < p.nodes; t += kWalkThreads) {
    sh.parent[t] = t ? p.parents[t] : -1;
    if (t && sh.parent[t] >= t) sh.parent[t] = -1;      // never reached
    sh.token[t] = t ? p.tokens[t] : -1;
    sh.next[t] = -1;
  }
  for (int t = wave; t < p.nodes; t += kWalkWaves) {
    if (p.greedy) {
      float m = -__builtin_inff();
      int at = 0x7fffffff;
      for (int c = lane; c < p.chunks; c += 64)
        better(m, at, p.maxes[(long long)t * p.chunks + c], p.args[(long long)t * p.chunks + c]);
#pragma unroll
      for (int d = 32; d; d >>= 1) better(m, at, __shfl_xor(m, d), __shfl_xor(at, d));
      if (lane == 0) sh.best[t] = at == 0x7fffffff ? 0 : at;
    } else {
      float m;
      double z;
      row_stats(p, 0, t, lane, m, z);
      if (lane == 0) {
        sh.mp[t] = m;
        sh.zp[t] = z;
      }
      if (drawn) {
        row_stats(p, 1, t, lane, m, z);
        if (lane == 0) {
          sh.mq[t] = m;
          sh.zq[t] = z;
        }
      }
    }
  }
  __syncthreads();

  // Every node's children, a wave per node.
  for (int t = wave; t < p.nodes; t += kWalkWaves) {
    const uint16_t* rp = p.target + t * p.ldt;
    const uint16_t* rq = drawn ? p.draft + t * p.ldd : nullptr;
    double left = p.greedy ? 0.0 : sh.zp[t];           // point drafts: weight not yet rejected
    int rejected = 0;
    Residual r{0.0, 1.0, 0};
    for (int s = t + 1; s < p.nodes; ++s) {
      if (sh.parent[s] != t) continue;
      const int x = sh.token[s];
      const bool in = x >= 0 && x < p.vocab;
      bool ok = false;
      if (p.greedy) {
        ok = x == sh.best[t];
      } else if (!drawn) {
        bool fresh = in;                               // a sibling's token that was rejected has no weight left
        for (int b = t + 1; b < s && fresh; ++b) fresh = !(sh.parent[b] == t && sh.token[b] == x);
        const double w = fresh ? weight(logit(rp, x), sh.mp[t], p.scale_log2) : 0.0;
        ok = (double)p.accept_u[s] * left < w;
        left = fmax(left - w, 0.0);
      } else {
        if (rejected == p.max_children) break;
        const double pw = in ? weight(logit(rp, x), sh.mp[t], p.scale_log2) / sh.zp[t] : 0.0;
        const double qw = in ? weight(logit(rq, x), sh.mq[t], p.scale_log2) / sh.zq[t] : 0.0;
        ok = (double)p.accept_u[s] * qw * r.s < fmax(pw - r.a * qw, 0.0);
        if (!ok) r = residual(p, t, rejected + 1, lane);
      }
      if (ok) {
        if (lane == 0) sh.next[t] = s;
        break;
      }
      ++rejected;
    }
  }
  __syncthreads();

  if (tid == 0) {
    int n = 0, t = 0;
    for (; t >= 0; t = sh.next[t]) sh.path[n++] = t;
    sh.count = n;
  }
  __syncthreads();
  const int count = sh.count, node = sh.path[count - 1];

  if (p.greedy) {
    if (tid == 0) sh.last = sh.best[node];
    __syncthreads();
  } else {
    // The last token: choose a chunk, then the index in it.  What is left of
    // the distribution: chunk sums in a global array, or for point drafts
    // computed again without the rejected tokens (subtracting their weights
    // would leave rounding where nothing is left).
    const uint16_t* rp = p.target + node * p.ldt;
    const float mp = sh.mp[node];
    int children = 0;
    for (int s = node + 1; s < p.nodes; ++s) children += sh.parent[s] == node;
    Residual r{0.0, 1.0, 0};
    if (drawn) r = residual(p, node, min(children, p.max_children), lane);
    const double a = r.round ? r.a / sh.zq[node] : 0.0, ip = 1.0 / sh.zp[node];
    const uint16_t* rq = r.round ? p.draft + node * p.ldd : nullptr;
    const double* rs = r.round ? p.rounds + ((long long)(r.round - 1) * p.nodes + node) * p.chunks : nullptr;

    auto mark = [&](int c) {                            // the chunk's rejected tokens
      for (int i = tid; i < kVerifyChunk / 32; i += kWalkThreads) sh.gone[i] = 0u;
      __syncthreads();
      if (!drawn)
        for (int s = node + 1 + tid; s < p.nodes; s += kWalkThreads) {
          const int x = sh.token[s] - c * kVerifyChunk;
          if (sh.parent[s] == node && sh.token[s] >= 0 && x >= 0 && x < kVerifyChunk) atomicOr(&sh.gone[x >> 5], 1u << (x & 31));
        }
      __syncthreads();
    };
    auto weights = [&](int c, double (&w)[kPer]) {      // this thread's eight of chunk c
      const int i0 = kPer * tid, v = c * kVerifyChunk + i0;
      float x[8], y[8];
      load8(rp, v, p.vocab, x);
      if (rq) load8(rq, v, p.vocab, y);
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        w[e] = 0.0;
        if (v + e < p.vocab && !((sh.gone[(i0 + e) >> 5] >> ((i0 + e) & 31)) & 1u)) {
          w[e] = weight(x[e], mp, p.scale_log2) * ip;
          if (rq) w[e] = fmax(w[e] - weight(y[e], sh.mq[node], p.scale_log2) * a, 0.0);
        }
      }
    };
    auto chunk_sum = [&](int c) -> double {
      if (rs) return rs[c];
      bool touched = false;
      if (!drawn)
        for (int s = node + 1; s < p.nodes; ++s)
          touched |= sh.parent[s] == node && sh.token[s] >= 0 && sh.token[s] / kVerifyChunk == c;
      if (!touched) return p.sums[(long long)node * p.chunks + c] * weight(p.maxes[(long long)node * p.chunks + c], mp, p.scale_log2) * ip;
      double w[kPer];
      mark(c);
      weights(c, w);
      double s = 0.0;
#pragma unroll
      for (int e = 0; e < kPer; ++e) s += w[e];
      return block_sum(s, sh);
    };
    double total = 0.0;
    for (int c = 0; c < p.chunks; ++c) total += chunk_sum(c);
    const double goal = (double)*p.sample_u * total;
    double before = 0.0;
    int chunk = -1;                                      // the first chunk whose end passes the goal, else the last with weight
    double chunk_before = 0.0;
    for (int c = 0; c < p.chunks; ++c) {
      const double s = chunk_sum(c);
      if (s > 0.0) {
        chunk = c;
        chunk_before = before;
      }
      before += s;
      if (s > 0.0 && before > goal) break;
    }
    if (chunk < 0) {                                     // every child was rejected and nothing else has weight
      if (tid == 0) sh.last = 0;
    } else {
      double w[kPer];
      mark(chunk);
      weights(chunk, w);
      if (tid == 0) sh.last = -1;
      double run = 0.0;
#pragma unroll
      for (int e = 0; e < kPer; ++e) run += w[e];
      double incl = run;                                 // inclusive scan over the wave, then over the waves
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const double y = __shfl_up(incl, d);
        if (lane >= d) incl += y;
      }
      __syncthreads();
      if (lane == 63) sh.wave[wave] = incl;
      __syncthreads();
      double base = chunk_before;
      for (int i = 0; i < wave; ++i) base += sh.wave[i];
      double cum = base + (incl - run);
      int hit = 0x7fffffff, tail = -1;
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        cum += w[e];
        if (w[e] > 0.0) {
          tail = kPer * tid + e;
          if (cum > goal && hit == 0x7fffffff) hit = kPer * tid + e;
        }
      }
      __shared__ int first, final_;
      if (tid == 0) {
        first = 0x7fffffff;
        final_ = -1;
      }
      __syncthreads();
      if (hit != 0x7fffffff) atomicMin(&first, hit);
      if (tail >= 0) atomicMax(&final_, tail);
      __syncthreads();
      if (tid == 0) sh.last = chunk * kVerifyChunk + (first != 0x7fffffff ? first : max(final_, 0));
    }
    __syncthreads();
  }

  for (int i = tid; i < p.nodes; i += kWalkThreads) {
    p.path[i] = i < count ? sh.path[i] : -1;
    p.emitted[i] = i < count - 1 ? sh.token[sh.path[i + 1]] : i == count - 1 ? sh.last : -1;
  }
  if (tid == 0) *p.count = count;
}

}  // namespace

hipError_t launch_tree_verify(const TreeVerifyParams& p, hipStream_t stream) {
  if (p.greedy) {
    hipLaunchKernelGGL(verify_argmax_kernel, dim3(p.chunks, p.nodes), dim3(kThreads), 0, stream, p);
  } else {
    hipLaunchKernelGGL(verify_stats_kernel, dim3(p.chunks, p.nodes, p.draft ? 2 : 1), dim3(kThreads), 0, stream, p);
    if (p.draft)
      for (int r = 1; r <= p.max_children; ++r)
        hipLaunchKernelGGL(verify_round_kernel, dim3(p.chunks, p.nodes), dim3(kThreads), 0, stream, p, r);
  }
  hipLaunchKernelGGL(verify_walk_kernel, dim3(1), dim3(kWalkThreads), 0, stream, p);
  return hipGetLastError();
}

}  // namespace qd
