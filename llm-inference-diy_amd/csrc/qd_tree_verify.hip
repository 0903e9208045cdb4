// Verification of a tree of drafted tokens against the target's logits (gfx950).
//
// Everything a decision depends on is held in 64 bits: weights
//   w(v) = 2^((l(v) - M) log2(e) / temperature),  M the row's largest logit,
// their sums, and the residuals max(p - A q, 0).  A decision compares a random
// number with a ratio of such sums, and the last token is the first index whose
// cumulative weight passes a random share of the total: with a vocabulary of
// 150 thousand, fp32 sums would move the chosen index.
//
// Residuals of drawn drafts in closed form: with p normalised, A_0 = 0, S_0 = 1,
// the distribution after j rejections is max(p - A_j q, 0) / S_j, where
//   A_{j+1} = A_j + S_j,   S_{j+1} = sum_v max(p(v) - A_{j+1} q(v), 0),
// since max(p - A_j q, 0)/S_j - q = (p - (A_j + S_j) q)/S_j wherever it is positive.
//
// Passes: (1) every (row, chunk of logits) gives its largest logit and its sum of weights
// relative to it, or its argmax; (2) with drawn drafts, per round j <= max_children, the
// chunks' sums of S_j, for every node whose first j children are all rejected; (3) one
// workgroup reduces the rows' partials, decides every node's children (a node's decisions do
// not depend on how it was reached), walks from node 0, and takes the last token from one
// chunk.  A single pass cannot do: p needs its row's whole sum, and S_j the sums before it.
//
// Measured on MI355X: 64 rows of 151936 logits 13 us (25 instructions per logit are 15 of its 25
// thousand cycles; the loads' and LDS latency at its two ends the rest) and the one workgroup
// 11; 27 rows of drawn drafts over 32003 logits 5, four rounds of 5.5-6.9 and 10; the greedy
// check of 5 rows 4.0 and 4.0.
#include "qd_device.h"
#include "qd_internal.h"
#include "qd_tree.h"
#include "qdiy/decode.h"

namespace qd {
namespace {

typedef _Float16 f16x8u __attribute__((ext_vector_type(8), aligned(2)));   // rows need not be 16-byte aligned

constexpr int kNodes = QD_TREE_MAX_NODES;
constexpr int kThreads = 256;                          // of the passes over chunks: 8 logits per thread and chunk
static_assert(kVerifyChunk == 8 * kThreads, "a chunk is one run of 8 logits per thread");

// Touches the argument block's cache lines at once: on its own the compiler loads each argument
// where it is first used, and waits for a line each time.
__device__ __forceinline__ void load_arguments(const TreeVerifyParams& p) {
  static_assert(sizeof(TreeVerifyParams) > 128 && sizeof(TreeVerifyParams) <= 192, "three 64-byte lines");
  asm volatile("" ::"s"(p.target), "s"(p.sums), "s"(p.groups));
}

// Weight of a logit in a row (or chunk): `m` its largest logit, `scale` 32 log2(e) / temperature
// (exponents are counted in 32nds).
struct Scale {
  float m;
  double md, scale;
};
__device__ __forceinline__ Scale make_scale(float m, double scale) { return Scale{m, (double)m, scale}; }
constexpr double kLeast = -28800.0;                    // 2^-900
// What a sum may hold of weights that should be 0 (2^24 of 2^-900) counts as 0.
constexpr double kNothing = 1e-250;

// 2^(j / 32) for j < 32 as the bits of a double, with j << 15 taken off the high word: adding n << 15
// to it gives 2^(n / 32) for n = 32 q + j.  Formed by the compiler from the exponential's series (the
// terms left out are below 2^-70).
struct Pow32 {
  unsigned long long bits[32];
};
constexpr Pow32 make_pow32() {
  Pow32 t{};
  for (int j = 0; j < 32; ++j) {
    const double x = j * 0.6931471805599453 / 32;      // j ln2 / 32
    double r = 1.0;
    for (int k = 20; k > 0; --k) r = 1.0 + r * x / k;
    t.bits[j] = __builtin_bit_cast(unsigned long long, r) - ((unsigned long long)j << 47);
  }
  return t;
}
__device__ constexpr Pow32 kPow32 = make_pow32();

// 2^(x / 32), kLeast <= x <= 0, to a relative 2e-12, by a table of a few powers as in P. T. P. Tang,
// "Table-driven implementation of the exponential function in IEEE floating-point arithmetic" (ACM
// TOMS 15, 1989): 2^(n/32) times the series of 2^(f/32) to degree 4 on |f| <= 1/2 (remainder
// (ln2/64)^5 / 5! = 1.3e-12).
// Rounding to n by adding 1.5 * 2^52 leaves it in the low word.  (A series on |f| <= 1/2 of a whole
// exponent, without the table, takes six fp64 instructions more: the pass over 64 rows of 151936
// logits 14.2 us against 13.9.)
// table: the workgroup's copy of kPow32 in LDS, 256 bytes: one entry per pair of banks, so
// lanes never conflict.
__device__ __forceinline__ double exp2_32nds(double x, const unsigned long long* table) {
  const double t = x + 0x1.8p52;
  const double f = x - (t - 0x1.8p52);
  const unsigned n = (unsigned)__builtin_bit_cast(unsigned long long, t);
  const unsigned long long bits = table[n & 31];
  const double base = __builtin_bit_cast(double, ((unsigned long long)((unsigned)(bits >> 32) + (n << 15)) << 32) | (unsigned)bits);
  double r = 9.172562701824643e-09;                    // (ln2 / 32)^k / k!, k = 4 .. 1
  r = __builtin_fma(r, f, 1.6938509724371819e-06);
  r = __builtin_fma(r, f, 0.00023459619820224677);
  r = __builtin_fma(r, f, 0.02166084939249829);
  return __builtin_fma(base, r * f, base);
}
// The weight where m is finite, for sums: a NaN, and what weighs less than 2^-900, counts as
// 2^-900.  (The difference of two halves is exact.)
__device__ __forceinline__ double weight_finite(float l, const Scale& s, const unsigned long long* table) {
  return exp2_32nds(fmax(((double)l - s.md) * s.scale, kLeast), table);
}
// For any m, and 0 where there is no weight: the largest logits weigh 1 also where they are
// infinite.
__device__ __forceinline__ double weight(float l, const Scale& s, const unsigned long long* table) {
  if (fabsf(s.m) < __builtin_inff()) {
    const double x = ((double)l - s.md) * s.scale;
    return x > kLeast ? exp2_32nds(x, table) : 0.0;    // 0 where x is NaN, too
  }
  if (l != l) l = -__builtin_inff();
  return l == s.m ? 1.0 : 0.0;
}
// The same as a function of its own, where few lanes have one weight each: the time there is that
// of fetching instructions that run once, and an inlined weight is 40 of them.
__device__ __attribute__((noinline)) double weight_call(float l, float m, double scale, const unsigned long long* table) {
  return weight(l, make_scale(m, scale), table);
}

// Reductions and scans by row operations and lane reads; every lane has to be there.  (Shuffles
// go through LDS, at some 100 cycles a step and two of them for 64 bits: the four rounds over 27
// rows of 32003 logits took 6.0 to 7.1 us with them, 5.3 to 6.4 without, the one-workgroup
// kernel 12.9 and 10.9.)
template <int Ctrl>
__device__ __forceinline__ double dpp_mov64(double x) {
  const unsigned long long b = __builtin_bit_cast(unsigned long long, x);
  const unsigned lo = __builtin_amdgcn_update_dpp(0, (int)(unsigned)b, Ctrl, 0xF, 0xF, true);
  const unsigned hi = __builtin_amdgcn_update_dpp(0, (int)(b >> 32), Ctrl, 0xF, 0xF, true);
  return __builtin_bit_cast(double, ((unsigned long long)hi << 32) | lo);
}
// The value of lane `at`, which is the same in all lanes.
__device__ __forceinline__ float lane_value(float x, int at) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), at));
}
__device__ __forceinline__ double lane_value(double x, int at) {
  const unsigned long long b = __builtin_bit_cast(unsigned long long, x);
  const unsigned lo = __builtin_amdgcn_readlane((int)(unsigned)b, at), hi = __builtin_amdgcn_readlane((int)(b >> 32), at);
  return __builtin_bit_cast(double, ((unsigned long long)hi << 32) | lo);
}
// Over the 16 lanes of a row; all of them receive it.
__device__ __forceinline__ double row16_sum64(double x) {
  x += dpp_mov64<kDppQuadSwap1>(x);
  x += dpp_mov64<kDppQuadSwap2>(x);
  x += dpp_mov64<kDppHalfMirror>(x);
  x += dpp_mov64<kDppMirror>(x);
  return x;
}
__device__ __forceinline__ double wave_sum(double x) {
  x = row16_sum64(x);
  return (lane_value(x, 0) + lane_value(x, 16)) + (lane_value(x, 32) + lane_value(x, 48));
}
__device__ __forceinline__ float wave_max(float x) {
  x = row16_max(x);
  return fmaxf(fmaxf(lane_value(x, 0), lane_value(x, 16)), fmaxf(lane_value(x, 32), lane_value(x, 48)));
}
// Inclusive.  Lanes without a partner to the left add 0.
__device__ __forceinline__ double wave_scan(double x, int lane) {
  x += dpp_mov64<0x111>(x);                            // row_shr:1, 2, 4, 8
  x += dpp_mov64<0x112>(x);
  x += dpp_mov64<0x114>(x);
  x += dpp_mov64<0x118>(x);
  const double r0 = lane_value(x, 15), r1 = r0 + lane_value(x, 31), r2 = r1 + lane_value(x, 47);
  const double before = lane < 32 ? (lane < 16 ? 0.0 : r0) : lane < 48 ? r1 : r2;
  return x + before;
}

// Eight logits from index v on; -inf past the row's end.  In two steps, so that several runs'
// loads are in flight together: fetch8 has no branch (it moves a run that passes the end back
// into the row), expand8 reads such a run again, one by one.
__device__ __forceinline__ f16x8u fetch8(const uint16_t* row, int v, int vocab) {
  if (vocab < 8) return f16x8u{};                      // uniform: expand8 reads them all
  return *reinterpret_cast<const f16x8u*>(row + min(v, vocab - 8));
}
__device__ __forceinline__ void expand8(const f16x8u& raw, const uint16_t* row, int v, int vocab, float (&x)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = (float)raw[e];
  if (v + 8 > vocab) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      x[e] = v + e < vocab ? (float)reinterpret_cast<const _Float16*>(row)[v + e] : -__builtin_inff();
  }
}

// Their weights; 0 past the row's end.
__device__ __forceinline__ void weights8(const float (&x)[8], int v, int vocab, const Scale& s, const unsigned long long* table,
                                         double (&w)[8]) {
  if (fabsf(s.m) < __builtin_inff()) {                 // uniform over a chunk
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = weight_finite(x[e], s, table);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = v + e < vocab ? weight(x[e], s, table) : 0.0;
  }
}

// (1) Sampled: blockIdx = (p.runs chunks, node, side).  The drafter's rows of nodes without
// children are not read: the buffer may end before them.  Each wave sums each run of 512 logits relative to the run's own
// largest, so that its work on one run stands behind that run's load alone; one wave puts the
// sums on a common base at the end.
constexpr int kWaves = kThreads / 64;
static_assert(kVerifyRuns * kWaves <= 64, "a workgroup's parts are one wave's lanes");
__global__ __launch_bounds__(kThreads) void verify_stats_kernel(TreeVerifyParams p) {
  __shared__ unsigned long long table[32];
  __shared__ float sm[64];                             // [run][wave]
  __shared__ double ss[64];
  load_arguments(p);
  const int t = blockIdx.y, side = blockIdx.z, c = blockIdx.x * p.runs, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint16_t* row = side ? p.draft + t * p.ldd : p.target + t * p.ldt;
  const int v0 = c * kVerifyChunk + 8 * threadIdx.x;
  if (side) {                                          // before any load: the row need not be there
    bool child = false;
    for (int s = t + 1 + threadIdx.x; s < p.nodes; s += kThreads) child |= p.parents[s] == t;
    if (!__syncthreads_or(child)) return;
  }
  f16x8u raw = fetch8(row, v0, p.vocab);
  if (lane < 32) table[lane] = kPow32.bits[lane];      // every wave writes it all, and needs no barrier to read it
#pragma unroll 1
  for (int r = 0; r < p.runs; ++r) {
    const int v = v0 + kVerifyChunk * r;
    float x[8], m = -__builtin_inff();
    double w[8];
    const f16x8u cur = raw;
    raw = fetch8(row, v + kVerifyChunk, p.vocab);
    expand8(cur, row, v, p.vocab, x);
#pragma unroll
    for (int e = 0; e < 8; ++e) m = fmaxf(m, x[e]);    // fmaxf passes NaN over
    m = wave_max(m);
    weights8(x, v, p.vocab, make_scale(m, p.scale_log2), table, w);
    const double s = wave_sum(((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7])));
    if (lane == 0) {
      sm[r * kWaves + wave] = m;
      ss[r * kWaves + wave] = s;
    }
  }
  __syncthreads();
  if (wave == 0) {
    const int parts = p.runs * kWaves;
    const float m = lane < parts ? sm[lane] : -__builtin_inff(), mg = wave_max(m);
    double s = lane < parts ? ss[lane] * weight(m, make_scale(mg, p.scale_log2), table) : 0.0;
    static_assert(kWaves == 4, "a run's parts are four lanes");
    s += dpp_mov64<kDppQuadSwap1>(s);
    s += dpp_mov64<kDppQuadSwap2>(s);                  // the run's, in each of its lanes
    const double all = wave_sum(lane % kWaves == 0 ? s : 0.0);    // 0 past the row's end
    const long long row_at = (long long)side * p.nodes + t;
    if (lane % kWaves == 0 && lane < parts && c + lane / kWaves < p.chunks) p.sums[row_at * p.chunks + c + lane / kWaves] = s;
    if (lane == 0) {
      p.maxes[row_at * p.groups + blockIdx.x] = mg;
      p.group_sums[row_at * p.groups + blockIdx.x] = all;
    }
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
  load_arguments(p);
  const int t = blockIdx.y, c = blockIdx.x;
  const uint16_t* row = p.target + t * p.ldt;
  const int v0 = c * p.runs * kVerifyChunk + 8 * threadIdx.x;
  f16x8u raw = fetch8(row, v0, p.vocab);
  float m = -__builtin_inff();
  int at = 0x7fffffff;
#pragma unroll 1
  for (int r = 0; r < p.runs; ++r) {
    const int v = v0 + kVerifyChunk * r;
    const f16x8u cur = raw;
    raw = fetch8(row, v + kVerifyChunk, p.vocab);
    float x[8];
    expand8(cur, row, v, p.vocab, x);
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
    p.maxes[(long long)t * p.groups + c] = m;
    p.args[(long long)t * p.groups + c] = at;
  }
}

// A row's groups as 16 lanes load them, two each, and from them and the rest of a long row its
// largest logit and its sum of weights relative to it.  In two steps, so that other loads are in
// flight with these.  The rounds and the one-workgroup kernel form both alike, so that they take
// the same decisions.
struct Groups {
  long long at;
  float m[2];
  double s[2];
};
__device__ __forceinline__ Groups fetch_groups(const TreeVerifyParams& p, int side, int t, int c) {
  Groups g;
  g.at = ((long long)side * p.nodes + t) * p.groups;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const bool in = c + 16 * i < p.groups;
    g.m[i] = in ? p.maxes[g.at + c + 16 * i] : -__builtin_inff();
    g.s[i] = in ? p.group_sums[g.at + c + 16 * i] : 0.0;
  }
  return g;
}
__device__ __forceinline__ void row_stats(const TreeVerifyParams& p, const unsigned long long* table, const Groups& g, int c, float& m,
                                          double& z) {
  m = fmaxf(g.m[0], g.m[1]);
#pragma unroll 4
  for (int i = c + 32; i < p.groups; i += 16) m = fmaxf(m, p.maxes[g.at + i]);
  m = row16_max(m);
  z = 0.0;
  float m0 = g.m[0], m1 = g.m[1];
  double s0 = g.s[0], s1 = g.s[1];
#pragma unroll 1
  for (int i = 0; i < p.groups; i += 16) {             // the same for all lanes
    const bool in = i + c + 32 < p.groups;
    const float m2 = in ? p.maxes[g.at + i + c + 32] : -__builtin_inff();
    const double s2 = in ? p.group_sums[g.at + i + c + 32] : 0.0;
    z += s0 * weight_call(m0, m, p.scale_log2, table);
    m0 = m1;
    s0 = s1;
    m1 = m2;
    s1 = s2;
  }
  z = row16_sum64(z);
}

// The first 64 chunks' sums of a node's rounds 1 to 3, a chunk per lane, loaded before it is
// known which will be needed (of rounds that are not: whatever is there).
struct Ahead {
  double r1, r2, r3;
};
__device__ __forceinline__ Ahead fetch_rounds(const TreeVerifyParams& p, int rounds, int t, int lane) {
  const double* s = p.rounds + (long long)t * p.chunks + lane;
  const long long next = (long long)p.nodes * p.chunks;
  const bool in = lane < p.chunks;
  return Ahead{in && rounds > 0 ? s[0] : 0.0, in && rounds > 1 ? s[next] : 0.0, in && rounds > 2 ? s[2 * next] : 0.0};
}
// The sum over chunks of round r (from 1) of node t, by one wave.
__device__ __forceinline__ double round_total(const TreeVerifyParams& p, int r, int t, int lane, const Ahead& first) {
  const double* s = p.rounds + ((long long)(r - 1) * p.nodes + t) * p.chunks;
  double z = r == 1 ? first.r1 : r == 2 ? first.r2 : first.r3;
  if (r > 3) z = lane < p.chunks ? s[lane] : 0.0;
  for (int c = lane + 64; c < p.chunks; c += 64) z += s[c];
  return wave_sum(z);
}

// The remaining distribution of a node with drawn drafts, max(p - a q, 0) / s, and the last
// round that changed it (0: p itself).  A round whose sum is 0 changes nothing, nor does any
// later one.
struct Residual {
  double a, s;
  int round;
};
__device__ __forceinline__ void reject(const TreeVerifyParams& p, int t, int rejected, int lane, const Ahead& first, Residual& r) {
  if (r.round != rejected - 1) return;
  const double s = round_total(p, rejected, t, lane, first);
  if (s > kNothing) r = Residual{r.a + r.s, s, rejected};
}

__device__ __forceinline__ float logit(const uint16_t* row, int v) {
  return (float)reinterpret_cast<const _Float16*>(row)[v];
}
// (2) Round `round` of drawn drafts: blockIdx = (chunk, node).  Each wave finds out for itself
// whether the node's first `round` children are all rejected; all that it takes for that but
// the children's tokens and their logits, and the chunk's logits, is loaded at once.
__global__ __launch_bounds__(kThreads) void verify_round_kernel(TreeVerifyParams p, int round) {
  __shared__ unsigned long long table[32];
  __shared__ double ss[kVerifyRuns][kWaves];
  load_arguments(p);
  const int t = blockIdx.y, c = blockIdx.x * p.runs, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint16_t* rp = p.target + t * p.ldt;
  const uint16_t* rq = p.draft + t * p.ldd;
  const Groups g = fetch_groups(p, (lane >> 4) & 1, t, lane & 15);   // target and drafter, twice
  const Ahead first = fetch_rounds(p, round - 1, t, lane);
  int child = -1, found = 0;                           // lane k: the node's child k (from 0), k < round
  for (int s0 = t + 1; s0 < p.nodes && found < round; s0 += 64) {
    const int s = s0 + lane;
    unsigned long long hits = __ballot(s < p.nodes && p.parents[s] == t);
    for (; hits && found < round; hits &= hits - 1, ++found)
      if (lane == found) child = s0 + __builtin_ctzll(hits);
  }
  if (found < round) return;                           // the same in every wave
  const int v0 = c * kVerifyChunk + 8 * threadIdx.x;
  const int tok = child >= 0 ? p.tokens[child] : -1;
  const float u = child >= 0 ? p.accept_u[child] : 0.0f;
  f16x8u xr = fetch8(rp, v0, p.vocab), yr = fetch8(rq, v0, p.vocab);
  if (threadIdx.x < 32) table[threadIdx.x] = kPow32.bits[threadIdx.x];
  const bool in = tok >= 0 && tok < p.vocab;
  const float lp = in ? logit(rp, tok) : 0.0f, lq = in ? logit(rq, tok) : 0.0f;
  __syncthreads();
  float m;
  double z;
  row_stats(p, table, g, lane & 15, m, z);
  const float mp = lane_value(m, 0), mq = lane_value(m, 16);
  const double zp = lane_value(z, 0), zq = lane_value(z, 16);
  const Scale sp = make_scale(mp, p.scale_log2), sq = make_scale(mq, p.scale_log2);
  const double pw = in ? weight(lp, sp, table) / zp : 0.0, qw = in ? weight(lq, sq, table) / zq : 0.0, uq = (double)u * qw;
  Residual r{0.0, 1.0, 0};
  for (int k = 0; k < round; ++k) {
    const bool ok = lane_value(uq, k) * r.s < fmax(lane_value(pw, k) - r.a * lane_value(qw, k), 0.0);
    if (ok) return;                                    // a child stands: no later round is looked at
    if (k + 1 < round) reject(p, t, k + 1, lane, first, r);
  }
  const double a = (r.a + r.s) / zq, ip = 1.0 / zp;
#pragma unroll 1
  for (int i = 0; i < p.runs; ++i) {
    double s = 0.0;
    const int v = v0 + kVerifyChunk * i;
    const f16x8u xc = xr, yc = yr;
    xr = fetch8(rp, v + kVerifyChunk, p.vocab);
    yr = fetch8(rq, v + kVerifyChunk, p.vocab);
    if (r.round == round - 1) {                        // else an earlier round's sum was 0
      float x[8], y[8];
      double wp[8], wq[8];
      expand8(xc, rp, v, p.vocab, x);
      expand8(yc, rq, v, p.vocab, y);
      weights8(x, v, p.vocab, sp, table, wp);
      weights8(y, v, p.vocab, sq, table, wq);
#pragma unroll
      for (int e = 0; e < 8; ++e) s += fmax(wp[e] * ip - wq[e] * a, 0.0);
    }
    s = wave_sum(s);
    if (lane == 0) ss[i][wave] = s;
  }
  __syncthreads();
  if ((int)threadIdx.x < p.runs && c + (int)threadIdx.x < p.chunks) {
    double s = ss[threadIdx.x][0];
    for (int w = 1; w < kThreads / 64; ++w) s += ss[threadIdx.x][w];
    p.rounds[((long long)(round - 1) * p.nodes + t) * p.chunks + c + threadIdx.x] = s;
  }
}

// (3) One workgroup.
constexpr int kWalkThreads = 1024;
constexpr int kWalkWaves = kWalkThreads / 64;
constexpr int kMaxChunks = (1 << 24) / kVerifyChunk;   // of the largest vocabulary

struct WalkShared {
  unsigned long long table[32];
  int parent[kNodes], token[kNodes], next[kNodes], path[kNodes], best[kNodes], round[kNodes];
  float mp[kNodes], mq[kNodes], u[kNodes];
  double zp[kNodes], zq[kNodes];
  double a[kNodes], s[kNodes];                         // with round: what a node's children left, if all are rejected
  double pw[kNodes], qw[kNodes];                       // a node's token in its parent's distributions
  double wave[kWalkWaves];
  unsigned gone[kVerifyChunk / 32];                       // rejected tokens of one chunk
  double sums[kMaxChunks];                             // of the last token's row
  int hit[kWalkWaves], tail[kWalkWaves];
  int count, chunk;
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
  load_arguments(p);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const bool drawn = !p.greedy && p.draft != nullptr;
  const float sample_u = p.greedy ? 0.0f : *p.sample_u;
  if (!p.greedy && tid < 32) sh.table[tid] = kPow32.bits[tid];
  // Thread t: node t and, on their way while the rows are summed, its token's logits in its
  // parent's rows.
  static_assert(kWalkThreads >= kNodes, "a thread per node");
  int parent = -1, token = -1;
  float lp = 0.0f, lq = 0.0f;
  if (tid < p.nodes) {
    const int above = tid ? p.parents[tid] : -1;
    parent = above < tid ? above : -1;                 // otherwise never reached
    token = tid ? p.tokens[tid] : -1;
    sh.u[tid] = tid && !p.greedy ? p.accept_u[tid] : 0.0f;
    sh.parent[tid] = parent;
    sh.token[tid] = token;
  }
  const bool in = !p.greedy && parent >= 0 && token >= 0 && token < p.vocab;
  if (in) {
    lp = logit(p.target + parent * p.ldt, token);
    if (drawn) lq = logit(p.draft + parent * p.ldd, token);
  }
  __syncthreads();
  for (int t0 = 4 * wave; t0 < p.nodes; t0 += 4 * kWalkWaves) {   // four rows per wave, 16 lanes each
    const int c0 = lane & 15, t = min(t0 + (lane >> 4), p.nodes - 1);
    if (p.greedy) {
      float m = -__builtin_inff();
      int at = 0x7fffffff;
      for (int g0 = 0; g0 < p.groups; g0 += 64) {      // four loads at once; a group may be met twice
        float gm[4];
        int gi[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const long long g = (long long)t * p.groups + min(g0 + 16 * i + c0, p.groups - 1);
          gm[i] = p.maxes[g];
          gi[i] = p.args[g];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) better(m, at, gm[i], gi[i]);
      }
#pragma unroll
      for (int d = 8; d; d >>= 1) better(m, at, __shfl_xor(m, d), __shfl_xor(at, d));
      if (c0 == 0) sh.best[t] = at == 0x7fffffff ? 0 : at;
    } else {
      float m, mq = 0.0f;
      double z, zq = 1.0;
      const Groups gp = fetch_groups(p, 0, t, c0), gq = drawn ? fetch_groups(p, 1, t, c0) : Groups{};
      row_stats(p, sh.table, gp, c0, m, z);
      if (drawn) row_stats(p, sh.table, gq, c0, mq, zq);     // of a node without children: not written, not used
      if (c0 == 0) {
        sh.mp[t] = m;
        sh.zp[t] = z;
        sh.mq[t] = mq;
        sh.zq[t] = zq;
      }
    }
  }
  __syncthreads();
  if (!p.greedy) {
    if (tid < p.nodes) {
      double pw = 0.0, qw = 0.0;
      if (in) {
        pw = weight_call(lp, sh.mp[parent], p.scale_log2, sh.table) / sh.zp[parent];
        if (drawn) {
          qw = weight_call(lq, sh.mq[parent], p.scale_log2, sh.table) / sh.zq[parent];
        } else {                                       // a sibling's token that was rejected has nothing left
          for (int b = parent + 1; b < tid; ++b)
            if (sh.parent[b] == parent && sh.token[b] == token) pw = 0.0;
        }
      }
      sh.pw[tid] = pw;
      sh.qw[tid] = qw;
    }
    __syncthreads();
  }

  // Every node's children in order, a wave per node.  Lanes hold a block of 64 nodes (read once
  // where there are no more), and lane i the decision on the wave's node i.
  static_assert(kNodes == 64 * kWalkWaves, "a lane per node of a wave");
  int block = -1, above = -1, next = -1, round = 0;
  double u = 0.0, pw = 0.0, qw = 0.0, ra = 0.0, rs = 1.0;
  for (int t = wave; t < p.nodes; t += kWalkWaves) {
    double left = 1.0;                                 // point drafts: what the rejected siblings leave
    int rejected = 0, taken = -1;
    Residual r{0.0, 1.0, 0};
    Ahead first{0.0, 0.0, 0.0};
    for (int s0 = t & ~63; s0 < p.nodes && taken < 0; s0 += 64) {
      if (s0 != block) {
        const int s = s0 + lane;
        const bool there = s < p.nodes;
        block = s0;
        above = there ? sh.parent[s] : -1;
        u = there ? (double)sh.u[s] : 0.0;
        pw = there ? sh.pw[s] : 0.0;
        qw = there ? sh.qw[s] : 0.0;
      }
      const bool mine = above == t;
      unsigned long long hits = __ballot(mine);
      if (!hits) continue;
      if (drawn) {
        if (rejected == 0) first = fetch_rounds(p, p.max_children, t, lane);
        for (; hits && taken < 0 && rejected < p.max_children; hits &= hits - 1) {
          const int c = __builtin_ctzll(hits);
          const double q = lane_value(qw, c);
          if (lane_value(u, c) * q * r.s < fmax(lane_value(pw, c) - r.a * q, 0.0)) {
            taken = s0 + c;
          } else {
            reject(p, t, rejected + 1, lane, first, r);
            ++rejected;
          }
        }
        continue;
      }
      bool ok;
      if (p.greedy) {
        ok = mine && sh.token[s0 + lane] == sh.best[t];
      } else {
        const double w = mine ? pw : 0.0, upto = wave_scan(w, lane);
        // At least the token's own share: rounding may have taken a little of it.
        ok = u * fmax(left - (upto - w), w) < w;
        left -= lane_value(upto, 63);
      }
      const unsigned long long good = __ballot(ok);
      if (good) taken = s0 + __builtin_ctzll(good);
    }
    if (lane == t / kWalkWaves) {
      next = taken;
      ra = r.a;
      rs = r.s;
      round = r.round;
    }
  }
  if (wave + kWalkWaves * lane < p.nodes) {
    const int t = wave + kWalkWaves * lane;
    sh.next[t] = next;
    sh.a[t] = ra;
    sh.s[t] = rs;
    sh.round[t] = round;
  }
  __syncthreads();

  if (tid == 0) {
    int n = 0, t = 0;
    for (; t >= 0; t = sh.next[t]) sh.path[n++] = t;
    sh.count = n;
    sh.chunk = -1;
  }
  __syncthreads();
  const int count = sh.count, node = sh.path[count - 1];

  int last = 0;
  if (p.greedy) {
    last = sh.best[node];
  } else {
    // The last token: choose a chunk by the chunks' sums of what is left of the distribution,
    // then the index in it.
    const uint16_t* rp = p.target + node * p.ldt;
    const float mp = sh.mp[node];
    const double ip = 1.0 / sh.zp[node];
    const Residual r{sh.a[node], sh.s[node], sh.round[node]};
    int children = 0;
    for (int s0 = node + 1; s0 < p.nodes; s0 += 64)
      children += __builtin_popcountll(__ballot(s0 + lane < p.nodes && sh.parent[min(s0 + lane, kNodes - 1)] == node));
    const double a = r.round ? r.a / sh.zq[node] : 0.0;
    const uint16_t* rq = r.round ? p.draft + node * p.ldd : nullptr;
    const float mq = r.round ? sh.mq[node] : 0.0f;
    const double* rs = r.round ? p.rounds + ((long long)(r.round - 1) * p.nodes + node) * p.chunks : nullptr;
    const bool holes = !drawn && children;             // rejected tokens of point drafts

    // This thread's two of chunk c, without the rejected tokens.
    constexpr int kEach = kVerifyChunk / kWalkThreads;
    auto chunk_weights = [&](int c, double (&w)[kEach]) {
      float x[kEach], y[kEach];
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        const int v = min(c * kVerifyChunk + kEach * tid + e, p.vocab - 1);
        x[e] = logit(rp, v);
        y[e] = rq ? logit(rq, v) : 0.0f;
      }
      if (holes) {
        __syncthreads();                               // sh.gone may still be read
        if (tid < kVerifyChunk / 32) sh.gone[tid] = 0u;
        __syncthreads();
        for (int s = node + 1 + tid; s < p.nodes; s += kWalkThreads) {
          const int x = sh.token[s] - c * kVerifyChunk;
          if (sh.parent[s] == node && sh.token[s] >= 0 && x >= 0 && x < kVerifyChunk) atomicOr(&sh.gone[x >> 5], 1u << (x & 31));
        }
        __syncthreads();
      }
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        const int i = kEach * tid + e;
        w[e] = weight_call(x[e], mp, p.scale_log2, sh.table) * ip;
        if (rq) w[e] = fmax(w[e] - weight_call(y[e], mq, p.scale_log2, sh.table) * a, 0.0);
        if (c * kVerifyChunk + i >= p.vocab || (holes && (sh.gone[i >> 5] >> (i & 31)) & 1u)) w[e] = 0.0;
      }
    };

    // Chunk sums.  Point drafts: without the rejected tokens' weights, subtracted where enough is
    // left that the rounding of the subtraction does not matter, else summed again.
    double* sums = sh.sums;
    for (int c = tid; c < p.chunks; c += kWalkThreads) {
      const long long at = (long long)node * p.chunks + c;
      double s = rs ? rs[c] : p.sums[at] * weight_call(p.maxes[(long long)node * p.groups + c / p.runs], mp, p.scale_log2, sh.table) * ip;
      if (holes) {
        const double all = s;
        for (int k = node + 1; k < p.nodes; ++k)
          if (sh.parent[k] == node && sh.token[k] >= 0 && sh.token[k] / kVerifyChunk == c) s -= sh.pw[k];
        if (s < 1e-3 * all) s = -1.0;                  // to be summed again
      }
      sums[c] = s >= 0.0 && s < kNothing ? 0.0 : s;
    }
    __syncthreads();
    if (holes)
      for (int k = node + 1; k < p.nodes; ++k) {       // only these chunks can be marked
        if (sh.parent[k] != node || sh.token[k] < 0 || sh.token[k] >= p.vocab) continue;
        const int c = sh.token[k] / kVerifyChunk;
        if (sums[c] >= 0.0) continue;                  // uniform: nothing is written between the barriers
        double w[kEach];
        chunk_weights(c, w);
        static_assert(kEach == 2, "the sum of two");
        const double s = block_sum(w[0] + w[1], sh);
        if (tid == 0) sums[c] = s;
        __syncthreads();
      }
    // Wave 0: the total, then the first chunk whose end passes the goal, else the last with weight.
    if (wave == 0) {
      double total = 0.0;
      for (int c = lane; c < p.chunks; c += 64) total += sums[c];
      total = wave_sum(total);
      const double goal = (double)sample_u * total;
      double before = 0.0, chunk_before = 0.0;
      int chunk = -1;
      bool passed = false;
      for (int c0 = 0; c0 < p.chunks && !passed; c0 += 64) {
        const double s = c0 + lane < p.chunks ? sums[c0 + lane] : 0.0;
        const double end = wave_scan(s, lane);
        const unsigned long long some = __ballot(s > 0.0), past = __ballot(s > 0.0 && before + end > goal);
        if (some) {
          const int at = past ? __builtin_ctzll(past) : 63 - __builtin_clzll(some);
          chunk = c0 + at;
          chunk_before = before + lane_value(end - s, at);
          passed = past != 0;
        }
        before += lane_value(end, 63);
      }
      if (lane == 0) {
        sh.chunk = chunk;
        sh.before = chunk_before;
        sh.total = total;
      }
    }
    __syncthreads();
    const int chunk = sh.chunk;
    if (chunk >= 0) {                                  // else all is rejected and nothing has weight: token 0
      const double goal = (double)sample_u * sh.total;
      double w[kEach];
      chunk_weights(chunk, w);
      const double run = w[0] + w[1];
      const double end = wave_scan(run, lane);         // then over the waves
      __syncthreads();                                 // sh.wave may still be read
      if (lane == 63) sh.wave[wave] = end;
      __syncthreads();
      double ahead = lane < wave ? sh.wave[lane] : 0.0;  // the waves before this one
      ahead = lane_value(row16_sum64(ahead), 0);
      double cum = sh.before + ahead + (end - run);
      int hit = -1, tail = -1;                         // the thread's first past the goal, and last with weight
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        cum += w[e];
        if (w[e] > 0.0) {
          tail = kEach * tid + e;
          if (cum > goal && hit < 0) hit = kEach * tid + e;
        }
      }
      // The first hit in index order, else the last tail.  (Not by LDS atomics: over a wave's
      // lanes those run one lane at a time.)
      const unsigned long long hits = __ballot(hit >= 0), tails = __ballot(tail >= 0);
      const int h = __builtin_amdgcn_readlane(hit, hits ? __builtin_ctzll(hits) : 0);
      const int tl = __builtin_amdgcn_readlane(tail, tails ? 63 - __builtin_clzll(tails) : 0);
      if (lane == 0) {
        sh.hit[wave] = hits ? h : -1;
        sh.tail[wave] = tails ? tl : -1;
      }
      __syncthreads();
      const int wh = lane < kWalkWaves ? sh.hit[lane] : -1, wt = lane < kWalkWaves ? sh.tail[lane] : -1;
      const unsigned long long whits = __ballot(wh >= 0), wtails = __ballot(wt >= 0);
      const int at = whits ? __builtin_amdgcn_readlane(wh, __builtin_ctzll(whits))
                     : wtails ? __builtin_amdgcn_readlane(wt, 63 - __builtin_clzll(wtails)) : 0;
      last = chunk * kVerifyChunk + at;
    }
  }

  for (int i = tid; i < p.nodes; i += kWalkThreads) {
    p.path[i] = i < count ? sh.path[i] : -1;
    p.emitted[i] = i < count - 1 ? sh.token[sh.path[i + 1]] : i == count - 1 ? last : -1;
  }
  if (tid == 0) *p.count = count;
}

}  // namespace

hipError_t launch_tree_verify(const TreeVerifyParams& p, hipStream_t stream) {
  if (p.greedy) {
    hipLaunchKernelGGL(verify_argmax_kernel, dim3(p.groups, p.nodes), dim3(kThreads), 0, stream, p);
  } else {
    hipLaunchKernelGGL(verify_stats_kernel, dim3(p.groups, p.nodes, p.draft ? 2 : 1), dim3(kThreads), 0, stream, p);
    if (p.draft)
      for (int r = 1; r <= p.max_children; ++r)
        hipLaunchKernelGGL(verify_round_kernel, dim3(p.groups, p.nodes), dim3(kThreads), 0, stream, p, r);
  }
  hipLaunchKernelGGL(verify_walk_kernel, dim3(1), dim3(kWalkThreads), 0, stream, p);
  return hipGetLastError();
}

}  // namespace qd
