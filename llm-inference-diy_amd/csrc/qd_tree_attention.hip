// Attention of a tree of drafted tokens over a KV cache, on the matrix cores (gfx950
// v_mfma_f32_16x16x32_f16).
//
// The query rows of one cache head -- `nodes` times the query heads that share it -- are
// handled together, so every K/V row is read once for up to 128 of them; with few rows a step
// is bound by the cache's bytes.  The keys form tiles of 32 rows: those of the cache, then the
// node rows, which alone are masked.  A workgroup takes one block of 16 kQ kQW query rows (16 to
// 128) of one cache head and every splits-th group of kKW tiles, a tile per key wave; its key
// waves keep a softmax state each over all of the block's rows and are folded through LDS at the
// end.  Several splits leave fp32 partials in the workspace, which a second launch folds.
//
//   S^T = K Q^T     (M = 16 keys, two tiles; N = 16 queries; K = 128 dims in four steps)
//   O^T += V^T P^T  (M = 16 dims, eight tiles; N = 16 queries; K = 32 keys)
// Operand lanes (c = l % 16, g = l / 16): A[c][8 g + e], B[8 g + e][c]; accumulator
// D[4 g + r][c].  Loads take whole rows, four per instruction (16 bytes per lane, chunk c of
// row 4 j + g): a K operand read straight from memory would touch a row per lane, which the
// load path takes at one lane per clock.  K rows therefore go through LDS.  A lane's V rows
// 4 j + g are P^T's operand slots as they are, when the K operands' rows are dealt so that
// S^T leaves the lane the scores of the same eight keys; V^T's operand then is, per dim, the
// lane's own eight rows, transposed by byte permutations (32 per 8 x 8 halves x 4).  The dims
// tile e takes dim 8 c + e of every lane, so lane (g, c) ends with dims 32 g .. 32 g + 31 of
// query c, and stores rows of its own.
//
// With more than 32 query rows the tiles are shared: 2 or 4 waves of 32 rows each (query waves)
// read every K and V tile from LDS, into which they loaded it together.
//
// Weights are rounded to fp16 for the second product, and the denominator sums the rounded
// weights on the matrix core (an all-ones A operand), so an output is a weighted mean of V
// rows.  A query's reference maximum moves only when a score passes it by more than 2^kLazy:
// weights stay below 2^kLazy, and the accumulators are scaled in few tiles.
//
// Measured on MI355X, 16 cache heads, scan + fold of the splits (kernel time in a trace, medians of
// 24 calls, us; a trace adds some 0.5 to the shortest):
//   5 nodes over 512 rows     8.4, one launch: latency (arguments, rows, fold, store)
//   27 nodes over 8191 rows   16.1 + 4.1; 67 MB of cache at 4.2 TB/s
//   64 nodes over 32700 rows  54.6 + 4.9; 268 MB at 4.9 TB/s (a large copy reaches 4.9)
//   250 nodes over 4001 rows  23.0 + 5.9; 378 TFLOP/s: a round of two tiles takes ~2850 cycles,
//     of them 1088 on the matrix cores and ~1300 in LDS; half of the rest are the start (two
//     loads' latency), the fold through LDS (4500 cycles) and the partials (16 MB)
// Half a round's shift between the two waves of a SIMD, so that one's products run beside the
// other's softmax, measured no better (62.9 against 58.0 us, 250 nodes over 16384 rows).
#include "qd_device.h"
#include "qd_internal.h"
#include "qd_tree.h"

namespace qd {
namespace {

constexpr int kKeys = 32;
constexpr float kLazy = 8.0f;            // log2 of the largest softmax weight before a rescale
__device__ constexpr float kNone = -__builtin_inff();

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

// What a lane holds of a V tile: dims 8 c .. 8 c + 7 of rows 4 j + g.
struct Rows {
  u32x4 x[8];
};

// Operand slot j: dim e of row j.
__device__ __forceinline__ f16x8 v_column(const u32x4 (&v)[8], int e) {
  u32x4 r;
  const unsigned sel = e & 1 ? 0x07060302u : 0x05040100u;   // high or low halves of (second, first)
#pragma unroll
  for (int j = 0; j < 4; ++j) r[j] = __builtin_amdgcn_perm(v[2 * j + 1][e >> 1], v[2 * j][e >> 1], sel);
  return __builtin_bit_cast(f16x8, r);
}

// A descriptor of wave-uniform values, held in scalar registers.
__device__ __forceinline__ i32x4 wave_rsrc(const void* base, unsigned bytes) {
  i32x4 r = buffer_rsrc(base, bytes);
  r[0] = __builtin_amdgcn_readfirstlane(r[0]);
  r[1] = __builtin_amdgcn_readfirstlane(r[1]);
  r[2] = __builtin_amdgcn_readfirstlane(r[2]);
  return r;
}

// Whether any half of x is an infinity or a NaN; x with those halves cleared.
__device__ __forceinline__ bool has_nonfinite(u32x4 x) {
  bool bad = false;
#pragma unroll
  for (int d = 0; d < 4; ++d) bad |= (x[d] & 0x7c00u) == 0x7c00u || (x[d] & 0x7c000000u) == 0x7c000000u;
  return bad;
}
__device__ __forceinline__ u32x4 finite_halves(u32x4 x) {
#pragma unroll
  for (int d = 0; d < 4; ++d) {
    unsigned keep = (x[d] & 0x7c00u) == 0x7c00u ? 0xffff0000u : 0xffffffffu;
    if ((x[d] & 0x7c000000u) == 0x7c000000u) keep &= 0x0000ffffu;
    x[d] &= keep;
  }
  return x;
}

// Touches the argument block's three cache lines at once: on its own the compiler loads each
// argument where it is first used, and waits for a line three times in a row.
__device__ __forceinline__ void load_arguments(const TreeAttnParams& p) {
  static_assert(sizeof(TreeAttnParams) > 128 && sizeof(TreeAttnParams) <= 192, "three 64-byte lines");
  asm volatile("" ::"s"(p.q), "s"(p.q_stride), "s"(p.part_o));
}

// Node of query row r (row = node * group + head of the group): exact for rows below 2^22 (the
// reciprocal's estimate is off by at most one).
__device__ __forceinline__ int row_node(int r, int group) {
  int t = (int)((float)r * __builtin_amdgcn_rcpf((float)group));
  if (t * group > r) --t;
  if ((t + 1) * group <= r) ++t;
  return t;
}

// Outputs that are no numbers: dims 32 g + 8 i + e of query row r, for a whole wave.  The weight of
// a seen row may have rounded to 0 (its own, or its split's), which makes NaN of an infinity in V:
// where V holds infinities or NaN that the row sees, the output is their sum, whatever their
// weights.  weighed: the row's weights are numbers, and not all 0.  (Runs for such rows alone: a
// wave reads a column of the cache, 64 rows at a time.)
__device__ __forceinline__ bool no_number(f32x4 y) {     // (sums of weighted halves are far from overflow)
  return !(fabsf((y[0] + y[1]) + (y[2] + y[3])) < __builtin_inff());
}
__device__ __forceinline__ float infinity_at(const uint16_t* v) {
  const float y = (float)*reinterpret_cast<const _Float16*>(v);
  return fabsf(y) < __builtin_inff() ? 0.0f : y;
}
__device__ __forceinline__ f32x4 with_infinities(const TreeAttnParams& p, f32x4 y, int kh, int r, int e, bool weighed) {
  const int lane = threadIdx.x & 63, g = lane >> 4;
  const uint64_t* mask = p.mask + (long long)row_node(r, p.group) * ((p.nodes + 63) / 64);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const bool odd = weighed && !(fabsf(y[i]) < __builtin_inff());
    unsigned long long todo = __ballot(odd);
#pragma unroll 1
    while (todo) {                                         // dim by dim: the 16 lanes of one g
      const int of = __builtin_ctzll(todo) >> 4, d = 32 * of + 8 * i + e;
      todo &= ~(0xffffull << (16 * of));
      const uint16_t* v = p.v + kh * p.head_stride + d;
      float x = 0.0f;
#pragma unroll 4
      for (int j = lane; j < p.prefix; j += 64) x += infinity_at(v + j * p.row_stride);
#pragma unroll
      for (int s = 32; s; s >>= 1) x += __shfl_xor(x, s);
      if (odd && g == of) {
        const uint16_t* vt = p.vt + kh * p.thead_stride + d;
#pragma unroll 1
        for (int j = 0; j < p.nodes; ++j)
          if ((mask[j >> 6] >> (j & 63)) & 1u) x += infinity_at(vt + j * p.trow_stride);
        if (x != 0.0f) y[i] = x;                           // NaN, too
      }
    }
  }
  return y;
}

template <int kQ, int kQW, int kKW>
__global__ __launch_bounds__(kQW * kKW * 64) void tree_attention_kernel(TreeAttnParams p) {
  constexpr int kRows = 16 * kQ * kQW;                   // query rows of the block
  constexpr int kThreads = kQW * kKW * 64;
  // K (and shared V) tiles during the scan, the waves' accumulators afterwards.
  constexpr size_t kTiles = (size_t)(kQW == 1 ? 1 : 4) * kKW * kKeys * 256;
  constexpr size_t kFold = (size_t)kKW * kRows * (128 * 4 + 8) + kQW * kKW * 4;
  __shared__ __align__(16) char smem[kTiles > kFold ? kTiles : kFold];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int kw = wave / kQW, wq0 = 16 * kQ * (wave % kQW);   // key group, first row in the block
  const int c = lane & 15, g = lane >> 4;
  load_arguments(p);
  const int split = blockIdx.x, kh = blockIdx.y;
  const int r0 = blockIdx.z * kRows;                     // the block's first query row
  const int group = p.group;
  const int rows = p.nodes * group;
  const int words = (p.nodes + 63) / 64;

  // Query rows past the last repeat it; they are not stored.  (Loaded before the first tiles: a
  // wait for rows loaded later would hold up the tiles' loads in every round of the loop.)
  f16x8 qb[kQ][4];
  const unsigned* mask_row[kQ];
#pragma unroll
  for (int u = 0; u < kQ; ++u) {
    const int r = min(r0 + wq0 + 16 * u + c, rows - 1), t = row_node(r, group);
    const uint16_t* q = p.q + t * p.q_stride + (kh * group + (r - t * group)) * 128 + 8 * g;
    mask_row[u] = reinterpret_cast<const unsigned*>(p.mask + (long long)t * words);
#pragma unroll
    for (int s = 0; s < 4; ++s) qb[u][s] = *reinterpret_cast<const f16x8*>(q + 32 * s);
  }

  // Per query, in log2 units: the reference maximum (0 while there is none), and the score that
  // moves it (any score while there is none).
  float m[kQ], lim[kQ];
  f32x4 ls[kQ], o[kQ][8];
#pragma unroll
  for (int u = 0; u < kQ; ++u) {
    m[u] = 0.0f;
    lim[u] = kNone;
    ls[u] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int e = 0; e < 8; ++e) o[u][e] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }
  f16x8 ones;
#pragma unroll
  for (int e = 0; e < 8; ++e) ones[e] = (_Float16)1.0f;

  auto scores = [&](const u32x4 (&k)[8], f32x4 (&st)[kQ][2]) {
#pragma unroll
    for (int u = 0; u < kQ; ++u)
#pragma unroll
      for (int a = 0; a < 2; ++a) st[u][a] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
      for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int u = 0; u < kQ; ++u)
          st[u][a] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, k[4 * a + s]), qb[u][s], st[u][a], 0, 0, 0);
  };
  // Scores to weights; moves the reference maxima and scales the accumulators where needed.
  auto weights = [&](f32x4 (&st)[kQ][2], f16x8 (&pb)[kQ]) {
    // Each lane tests its own eight scores against the bound; only when some lane's pass it
    // are maxima formed across the four lanes of a query.  (Scaled first: a maximum of values
    // that were just computed needs no instruction to quiet NaN inputs.)
    float lm[kQ];
    bool grow = false;
#pragma unroll
    for (int u = 0; u < kQ; ++u) {
#pragma unroll
      for (int a = 0; a < 2; ++a) st[u][a] *= p.scale_log2;
      lm[u] = fmaxf(fmaxf(fmaxf(st[u][0][0], st[u][0][1]), fmaxf(st[u][0][2], st[u][0][3])),
                    fmaxf(fmaxf(st[u][1][0], st[u][1][1]), fmaxf(st[u][1][2], st[u][1][3])));
      grow |= lm[u] > lim[u];
    }
    if (__any(grow)) {
#pragma unroll
      for (int u = 0; u < kQ; ++u) {
        float bm = fmaxf(lm[u], __shfl_xor(lm[u], 16));
        bm = fmaxf(bm, __shfl_xor(bm, 32));
        if (bm > lim[u]) {
          const float alpha = lim[u] == kNone ? 0.0f : __builtin_amdgcn_exp2f(m[u] - bm);
          ls[u] *= alpha;
#pragma unroll
          for (int e = 0; e < 8; ++e) o[u][e] *= alpha;
          m[u] = bm;
          lim[u] = bm + kLazy;
        }
      }
    }
#pragma unroll
    for (int u = 0; u < kQ; ++u) {
#pragma unroll
      for (int e = 0; e < 8; ++e) pb[u][e] = (_Float16)__builtin_amdgcn_exp2f(st[u][e / 4][e % 4] - m[u]);
      ls[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, pb[u], ls[u], 0, 0, 0);
    }
  };
  auto products = [&](const Rows& v, const f16x8 (&pb)[kQ]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const f16x8 va = v_column(v.x, e);
#pragma unroll
      for (int u = 0; u < kQ; ++u) o[u][e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, pb[u], o[u][e], 0, 0, 0);
    }
  };

  // The tiles: the cache's rows, then the node rows, each in tiles of their own.  A load reads
  // four whole rows: instruction j of a tile row 4 j + g, 16-byte chunk c of it.  A tile's descriptor
  // ends with the last row that is there, so that rows past it (and tiles past the last) come as
  // zeros without being read: the loops have no branch around a load, and their waits count
  // exactly the loads that they need.
  const int cache_tiles = (p.prefix + kKeys - 1) / kKeys;
  const int tiles = cache_tiles + (p.nodes + kKeys - 1) / kKeys;
  const int step = p.splits * kKW;                         // tiles from one of a wave's to its next
  int tile = split * kKW + kw;
  struct Source {
    i32x4 k, v;
    unsigned off, row4;
  };
  // Descriptors of tile t; called for the wave's tiles in turn.  The cache's whole tiles lie a
  // constant apart.
  const int full = p.prefix / kKeys;
  const uint16_t* k_next = p.k + kh * p.head_stride + (long long)tile * kKeys * p.row_stride;
  const uint16_t* v_next = p.v + kh * p.head_stride + (long long)tile * kKeys * p.row_stride;
  const long long hop = (long long)step * kKeys * p.row_stride;
  auto source = [&](int t) {
    const uint16_t *kb = k_next, *vb = v_next;
    unsigned row_bytes = (unsigned)(p.row_stride * 2), bytes = 0xffffffffu;
    if (t >= full) {
      const bool node = t >= cache_tiles;
      const int row = (node ? t - cache_tiles : t) * kKeys, left = (node ? p.nodes : p.prefix) - row;
      if (node) {
        kb = p.kt + kh * p.thead_stride + row * p.trow_stride;
        vb = p.vt + kh * p.thead_stride + row * p.trow_stride;
        row_bytes = (unsigned)(p.trow_stride * 2);
      }
      bytes = t >= tiles ? 0u : (unsigned)(min(left, kKeys) - 1) * row_bytes + 256u;
    }
    k_next += hop;
    v_next += hop;
    Source x;
    x.k = wave_rsrc(kb, bytes);
    x.v = wave_rsrc(vb, bytes);
    x.off = (unsigned)g * row_bytes + 16u * c;
    x.row4 = 4u * row_bytes;
    return x;
  };
  auto load_k = [&](const Source& x, int j) {
    return __builtin_bit_cast(u32x4, raw_buffer_load_b128(x.k, (int)(x.off + j * x.row4), 0, 0));
  };
  auto load_v = [&](const Source& x, int j) {
    return __builtin_bit_cast(u32x4, raw_buffer_load_b128(x.v, (int)(x.off + j * x.row4), 0, 0));
  };
  // K rows in LDS: chunk q of row r at position q ^ (r % 16), so that neither the writes (whole
  // rows) nor the operand reads (one chunk of 16 rows) meet on a bank.  V rows as they are.
  auto put_k = [&](char* lk, int j, u32x4 x) {
    const int r = 4 * j + g;
    *reinterpret_cast<u32x4*>(lk + r * 256 + 16 * (c ^ (r & 15))) = x;
  };
  // K operand a, row c: key 16 a + 4 (c % 4) + c / 4, so that the accumulator's row 4 g + r is
  // key 4 (4 a + r) + g: the weights of a lane are those of the V rows that it loads.
  const int krow = 4 * (c & 3) + (c >> 2);
  auto get_k = [&](const char* lk, u32x4 (&k)[8]) {
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
      for (int s = 0; s < 4; ++s)
        k[4 * a + s] = *reinterpret_cast<const u32x4*>(lk + (16 * a + krow) * 256 + 16 * ((4 * s + g) ^ krow));
  };
  // Weights of tile t from its K rows in LDS.
  auto weigh = [&](int t, const char* lk, f16x8 (&pb)[kQ]) {
    f32x4 st[kQ][2];
    {
      u32x4 k[8];
      get_k(lk, k);
      scores(k, st);
    }
    if ((t + 1) * kKeys > p.prefix) {                      // node rows, or the cache's last rows
      const bool node = t >= cache_tiles;
      const int n = node ? p.nodes - (t - cache_tiles) * kKeys : p.prefix - t * kKeys;
      const unsigned rows_here = n >= kKeys ? ~0u : (1u << n) - 1u;
#pragma unroll
      for (int u = 0; u < kQ; ++u) {
        const unsigned bits = ((node ? mask_row[u][t - cache_tiles] : ~0u) & rows_here) >> g;
#pragma unroll
        for (int j = 0; j < 8; ++j) st[u][j / 4][j % 4] = (bits >> (4 * j)) & 1u ? st[u][j / 4][j % 4] : kNone;
      }
    }
    weights(st, pb);
  };
  // A weight of 0 keeps a finite V row out of a product, but not an infinity or a NaN: in a node
  // tile, whose rows may be unseen, such elements count as 0, and the fold adds them where they are
  // seen.  (The cache's rows are all seen: with_infinities finds what became of theirs.)
  bool nonfinite = false;
  auto make_finite = [&](auto& v) {
    constexpr int n = sizeof(v) / sizeof(u32x4);
    bool bad = false;
#pragma unroll
    for (int i = 0; i < n; ++i) bad |= has_nonfinite(v[i]);
    if (!__any(bad)) return;
    nonfinite = true;
#pragma unroll
    for (int i = 0; i < n; ++i) v[i] = finite_halves(v[i]);
  };

  if constexpr (kQW == 1) {
    // A wave's own tiles: K through its own LDS rows (in order within the wave, no barrier),
    // V straight to registers.
    char* lk = smem + wave * kKeys * 256;
    u32x4 kr[8];
    Rows v;
    {
      const Source x = source(tile);
#pragma unroll
      for (int j = 0; j < 8; ++j) kr[j] = load_k(x, j);
#pragma unroll
      for (int j = 0; j < 8; ++j) v.x[j] = load_v(x, j);
    }
    for (; tile < tiles; tile += step) {
#pragma unroll
      for (int j = 0; j < 8; ++j) put_k(lk, j, kr[j]);
      const Source next = source(tile + step);
#pragma unroll
      for (int j = 0; j < 8; ++j) kr[j] = load_k(next, j);
      f16x8 pb[kQ];
      weigh(tile, lk, pb);
      if (tile >= cache_tiles) make_finite(v.x);
      products(v, pb);
#pragma unroll
      for (int j = 0; j < 8; ++j) v.x[j] = load_v(next, j);
    }
  } else {
    // The key group's query waves share its tiles: each loads its part of the rows, two tiles
    // ahead, and puts them into one of two LDS buffers; one barrier per tile (a buffer is
    // written again only after the barrier behind its readers).  All key groups run the
    // same number of rounds.
    constexpr int kPart = 8 / kQW;
    constexpr int kTile = kKeys * 256;                     // bytes of a K or V tile
    const int qw = wave % kQW;
    const bool active = r0 + wq0 < rows;
    u32x4 kr[2][kPart], vr[2][kPart];
    auto fetch = [&](int t, u32x4 (&k)[kPart], u32x4 (&v)[kPart]) {
      const Source x = source(t);
#pragma unroll
      for (int j = 0; j < kPart; ++j) k[j] = load_k(x, kPart * qw + j);
#pragma unroll
      for (int j = 0; j < kPart; ++j) v[j] = load_v(x, kPart * qw + j);
    };
    auto round = [&](int t, int buf, u32x4 (&kx)[kPart], u32x4 (&vx)[kPart]) {
      char* lk = smem + (buf * kKW + kw) * 2 * kTile;
      char* lv = lk + kTile;
      if (t >= cache_tiles) make_finite(vx);
#pragma unroll
      for (int j = 0; j < kPart; ++j) {
        put_k(lk, kPart * qw + j, kx[j]);
        *reinterpret_cast<u32x4*>(lv + (4 * (kPart * qw + j) + g) * 256 + 16 * c) = vx[j];
      }
      fetch(t + 2 * step, kx, vx);
      __syncthreads();
      if (active && t < tiles) {
        f16x8 pb[kQ];
        weigh(t, lk, pb);
        Rows v;
#pragma unroll
        for (int j = 0; j < 8; ++j) v.x[j] = *reinterpret_cast<const u32x4*>(lv + (4 * j + g) * 256 + 16 * c);
        products(v, pb);
      }
    };
    fetch(tile, kr[0], vr[0]);
    fetch(tile + step, kr[1], vr[1]);
    for (int it = 0; it < p.rounds; it += 2) {
      round(tile, 0, kr[0], vr[0]);
      if (it + 1 == p.rounds) break;
      round(tile + step, 1, kr[1], vr[1]);
      tile += 2 * step;
    }
  }
  // Fold the key waves.  Every wave leaves its accumulators in LDS as they lie in its registers
  // (fragment (u, e): 16 bytes of each lane); then each wave folds its share of the fragments
  // and, of several splits, writes them out the same way.
  __syncthreads();                                         // the tiles' LDS is taken over
  constexpr int kWaves = kQW * kKW, kFrags = kQW * kQ * 8;
  f32x4* frag = reinterpret_cast<f32x4*>(smem);            // [kKW][kFrags][64]
  float2* state = reinterpret_cast<float2*>(frag + kKW * kFrags * 64);   // [kKW][kRows]
  int* bad = reinterpret_cast<int*>(state + kKW * kRows);  // [kWaves]
#pragma unroll
  for (int u = 0; u < kQ; ++u) {
#pragma unroll
    for (int e = 0; e < 8; ++e) frag[(kw * kFrags + (wave % kQW * kQ + u) * 8 + e) * 64 + lane] = o[u][e];
    if (g == 0) state[kw * kRows + wq0 + 16 * u + c] = float2{lim[u] == kNone ? kNone : m[u], ls[u][0]};
  }
  if (lane == 0) bad[wave] = nonfinite;
  __syncthreads();
  bool any_bad = false;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) any_bad |= bad[w] != 0;
  const int slot = (blockIdx.z * p.kv_heads + kh) * p.splits + split;
  // A wave's fragments belong to one tile of 16 rows: the key waves' weights are formed once.
  constexpr int kOwn = kFrags / kWaves;
  static_assert(8 % kOwn == 0, "a wave's fragments lie in one row tile");
  const int f0 = wave * kOwn, q = 16 * (f0 >> 3) + c;      // the lane's row in the block
  float mx = kNone, l = 0.0f, a[kKW];
#pragma unroll
  for (int w = 0; w < kKW; ++w) mx = fmaxf(mx, state[w * kRows + q].x);
#pragma unroll
  for (int w = 0; w < kKW; ++w) {
    const float2 ml = state[w * kRows + q];
    a[w] = ml.x == mx ? 1.0f : __builtin_amdgcn_exp2f(ml.x - mx);   // -inf: saw no row
    l += a[w] * ml.y;
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  const bool live = r0 + q < rows;
  if (any_bad) {
    // Add the infinities and NaN of this workgroup's node tiles that the row sees, to the
    // accumulators of a key wave whose weight is 1.
    int one = 0;
#pragma unroll
    for (int w = 0; w < kKW; ++w) one = a[w] == 1.0f ? w : one;
    const uint64_t* mask = p.mask + (long long)row_node(min(r0 + q, rows - 1), group) * words;
#pragma unroll 1
    for (int j = 0; j < p.nodes; ++j) {
      if ((cache_tiles + j / kKeys) % step / kKW != split || !((mask[j >> 6] >> (j & 63)) & 1u)) continue;
#pragma unroll 1
      for (int f = f0; f < f0 + kOwn; ++f) {
        const uint16_t* v = p.vt + kh * p.thead_stride + j * p.trow_stride + 32 * g + (f & 7);
        f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float y = (float)*reinterpret_cast<const _Float16*>(v + 8 * i);
          x[i] = fabsf(y) < __builtin_inff() ? 0.0f : y;
        }
        frag[(one * kFrags + f) * 64 + lane] += x;
      }
    }
  }
  if (p.splits > 1 && live && (f0 & 7) == 0 && g == 0) p.part_ml[(long long)slot * kRows + q] = float2{mx, l};
  unsigned odd = 0;                                        // the wave's fragments with no numbers in them
#pragma unroll
  for (int n = 0; n < kOwn; ++n) {
    const int f = f0 + n;
    f32x4 acc = a[0] * frag[f * 64 + lane];
#pragma unroll
    for (int w = 1; w < kKW; ++w) acc += a[w] * frag[(w * kFrags + f) * 64 + lane];
    if (p.splits > 1) {
      if (live) p.part_o[((long long)slot * kFrags + f) * 64 + lane] = acc;
    } else {
      frag[f * 64 + lane] = l == 0.0f ? f32x4{0.0f, 0.0f, 0.0f, 0.0f} : acc * inv;   // read by this wave alone
      odd |= (__any(no_number(acc)) ? 1u : 0u) << n;
    }
  }
  if (p.splits > 1) return;
  for (; odd; odd &= odd - 1) {
    const int f = f0 + __builtin_ctz(odd);
    frag[f * 64 + lane] = with_infinities(p, frag[f * 64 + lane], kh, min(r0 + q, rows - 1), f & 7, l == l && l != 0.0f);
  }
  __syncthreads();
  const float* folded = reinterpret_cast<const float*>(frag);
  for (int i = threadIdx.x; i < kRows * 16; i += kThreads) {
    const int q = i >> 4, d = 8 * (i & 15), r = r0 + q;    // dims d + e: fragment e, group d / 32, element d / 8 % 4
    if (r >= rows) break;
    f16x8 y;
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = (_Float16)folded[(((q >> 4) * 8 + e) * 64 + 16 * (d >> 5) + (q & 15)) * 4 + ((d >> 3) & 3)];
    const int t = row_node(r, group);
    *reinterpret_cast<f16x8*>(p.out + t * p.out_stride + (kh * group + (r - t * group)) * 128 + d) = y;
  }
}

// Folds the splits of 16 query rows of one cache head: a wave for the fragments 2 x and 2 x + 1
// of a block's row tile, so that a few rows are spread over many CUs; kBatch splits' loads are
// in flight together.  (Rows that are not there: whatever the workspace holds, in lanes that
// store nothing.)
template <int kBatch>
__global__ __launch_bounds__(64) void tree_attention_merge_kernel(TreeAttnParams p) {
  const int lane = threadIdx.x, c = lane & 15, g = lane >> 4;
  load_arguments(p);
  const int pair = blockIdx.x & 3, tile = blockIdx.x >> 2, tiles = p.block_rows >> 4, kh = blockIdx.y;
  const int group = p.group;
  const int r = (blockIdx.z * tiles + tile) * 16 + c;
  const long long slot = (long long)(blockIdx.z * p.kv_heads + kh) * p.splits;
  const f32x4* po = p.part_o + ((slot * tiles + tile) * 8 + 2 * pair) * 64 + lane;   // a split: tiles * 512
  const float2* ml = p.part_ml + (slot * tiles + tile) * 16 + c;                     // a split: tiles * 16
  float mx = kNone, l = 0.0f;
  f32x4 a0 = {0.0f, 0.0f, 0.0f, 0.0f}, a1 = a0;
  for (int s0 = 0; s0 < p.splits; s0 += kBatch) {
    float2 w[kBatch];
    f32x4 x[kBatch], y[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const int s = min(s0 + j, p.splits - 1);
      w[j] = ml[s * tiles * 16];
      x[j] = po[s * tiles * 512];
      y[j] = po[s * tiles * 512 + 64];
    }
    float mn = mx;
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      if (s0 + j >= p.splits) {                            // no such split: no row seen
        w[j] = float2{kNone, 0.0f};
        x[j] = y[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      }
      mn = fmaxf(mn, w[j].x);
    }
    const float keep = mn == mx ? 1.0f : __builtin_amdgcn_exp2f(mx - mn);
    l *= keep;
    a0 *= keep;
    a1 *= keep;
    mx = mn;
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const float a = w[j].x == mx ? 1.0f : __builtin_amdgcn_exp2f(w[j].x - mx);   // -inf: saw no row
      l += a * w[j].y;
      a0 += a * x[j];
      a1 += a * y[j];
    }
  }
  const bool live = r < p.nodes * group;
  if (__any(live && no_number(a0 + a1))) {
#pragma unroll 1
    for (int k = 0; k < 2; ++k) {                          // a0, then a1
      const f32x4 y = with_infinities(p, a0, kh, min(r, p.nodes * group - 1), 2 * pair + k, live && l == l && l != 0.0f);
      a0 = a1;
      a1 = y;
    }
  }
  if (!live) return;
  const int t = row_node(r, group);
  const float inv = 1.0f / l;
  _Float16* out = reinterpret_cast<_Float16*>(p.out) + t * p.out_stride + (kh * group + (r - t * group)) * 128 + 32 * g + 2 * pair;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f16x2 v;
    v[0] = (_Float16)(l == 0.0f ? 0.0f : a0[i] * inv);
    v[1] = (_Float16)(l == 0.0f ? 0.0f : a1[i] * inv);
    *reinterpret_cast<f16x2*>(out + 8 * i) = v;
  }
}

template <int kQ, int kQW, int kKW>
hipError_t launch(const TreeAttnParams& p, int blocks, hipStream_t stream) {
  hipLaunchKernelGGL((tree_attention_kernel<kQ, kQW, kKW>), dim3(p.splits, p.kv_heads, blocks), dim3(kQW * kKW * 64), 0,
                     stream, p);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_tree_attention(const TreeAttnParams& p, const TreeAttnPlan& plan, hipStream_t stream) {
  hipError_t e;
  switch (plan.block_rows) {
    case 16: e = launch<1, 1, 8>(p, plan.blocks, stream); break;
    case 32: e = launch<2, 1, 8>(p, plan.blocks, stream); break;
    case 64: e = launch<2, 2, 4>(p, plan.blocks, stream); break;
    default: e = launch<2, 4, 2>(p, plan.blocks, stream); break;
  }
  if (e != hipSuccess || plan.splits == 1) return e;
  const dim3 grid(4 * (plan.block_rows / 16), p.kv_heads, plan.blocks);
  if (plan.splits <= 4)
    hipLaunchKernelGGL(tree_attention_merge_kernel<4>, grid, dim3(64), 0, stream, p);
  else if (plan.splits <= 8)
    hipLaunchKernelGGL(tree_attention_merge_kernel<8>, grid, dim3(64), 0, stream, p);
  else
    hipLaunchKernelGGL(tree_attention_merge_kernel<16>, grid, dim3(64), 0, stream, p);
  return hipGetLastError();
}

}  // namespace qd
