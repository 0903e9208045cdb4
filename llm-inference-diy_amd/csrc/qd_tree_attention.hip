// Attention of a tree of drafted tokens over a KV cache, on the matrix cores (gfx950
// v_mfma_f32_16x16x32_f16).
//
// The query rows of one cache head -- `nodes` times the query heads that share it -- are
// handled together, so every K/V row is read once for up to 64 of them; with few rows a step
// is bound by the cache's bytes.  The keys form tiles of 32 rows: those of the cache, then the
// node rows, which alone are masked.  A workgroup takes one block of 16 kQ query rows of one
// cache head and every splits-th group of kW tiles, a tile per wave; its waves keep a softmax
// state each over all of the block's rows and are folded through LDS at the end.  Several
// splits leave fp32 partials in the workspace, which a second launch folds.
//
// Nothing goes through LDS on the way to the products:
//   S^T = K Q^T     (M = 16 keys, two tiles; N = 16 queries; K = 128 dims in four steps)
//   O^T += V^T P^T  (M = 16 dims, eight tiles; N = 16 queries; K = 32 keys)
// Operand lanes (c = l % 16, g = l / 16): A[c][8 g + e], B[8 g + e][c]; accumulator
// D[4 g + r][c].  K rows feed A as loaded, 16 bytes a lane.  S^T leaves lane (g, c) the
// scores of keys 16 a + 4 g + r of query c, which become P^T's B operand in place: its slot
// 8 g + 4 a + r stands for key 16 a + 4 g + r.  V^T's A operand then needs, per dim, those
// eight keys: a lane loads dims 8 c .. 8 c + 7 of its group's eight V rows (an instruction
// reads four whole rows) and transposes the 8 x 8 halves with 32 byte permutations; the dims
// tile e takes dim 8 c + e of every lane, so lane (g, c) ends with dims 32 g .. 32 g + 31 of
// query c, and stores rows of its own.
//
// Weights are rounded to fp16 for the second product, and the denominator sums the rounded
// weights on the matrix core (an all-ones A operand), so an output is a weighted mean of V
// rows.  A query's reference maximum moves only when a score passes it by more than 2^kLazy:
// weights stay below 2^kLazy, and the accumulators are scaled in few tiles.
#include "qd_device.h"
#include "qd_internal.h"
#include "qd_tree.h"

namespace qd {
namespace {

constexpr int kKeys = 32;
constexpr float kLazy = 8.0f;            // log2 of the largest softmax weight before a rescale
constexpr int kFoldRow = 132;            // floats of a query's O row in LDS: 128, and 4 to spread the banks
__device__ constexpr float kNone = -__builtin_inff();

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));

// Eight keys x eight dims of V as loaded, row 4 a + i of the group: va[e] slot 4 a + i is its
// dim e.
__device__ __forceinline__ f16x8 v_column(const u32x4 (&v)[8], int e) {
  u32x4 r;
  const unsigned sel = e & 1 ? 0x07060302u : 0x05040100u;   // high or low halves of (second, first)
#pragma unroll
  for (int j = 0; j < 4; ++j) r[j] = __builtin_amdgcn_perm(v[2 * j + 1][e >> 1], v[2 * j][e >> 1], sel);
  return __builtin_bit_cast(f16x8, r);
}

__device__ __forceinline__ bool any_nonfinite(const u32x4 (&v)[8]) {
  u16x2 m = {0, 0};
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, v[i][j] & 0x7fff7fffu));
  return m[0] >= 0x7c00 || m[1] >= 0x7c00;
}

// A descriptor of wave-uniform values, held in scalar registers.
__device__ __forceinline__ i32x4 wave_rsrc(const void* base, unsigned bytes) {
  i32x4 r = buffer_rsrc(base, bytes);
  r[0] = __builtin_amdgcn_readfirstlane(r[0]);
  r[1] = __builtin_amdgcn_readfirstlane(r[1]);
  r[2] = __builtin_amdgcn_readfirstlane(r[2]);
  return r;
}

template <int kQ, int kQW, int kKW>
__global__ __launch_bounds__(kQW * kKW * 64) void tree_attention_kernel(TreeAttnParams p) {
  constexpr int kRows = 16 * kQ * kQW;                   // query rows of the block
  constexpr int kThreads = kQW * kKW * 64;
  // K (and shared V) tiles during the scan, the waves' accumulators afterwards.
  constexpr size_t kTiles = kQW == 1 ? (size_t)kKW * kKeys * 256 : (size_t)2 * kKW * kKeys * 512;
  constexpr size_t kFold = (size_t)kKW * kRows * (kFoldRow + 2) * 4;
  __shared__ __align__(16) char smem[kTiles > kFold ? kTiles : kFold];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int kw = wave / kQW, wq0 = 16 * kQ * (wave % kQW);   // key group, first row in the block
  const int c = lane & 15, g = lane >> 4;
  const int split = blockIdx.x % p.splits;
  const int kh = (blockIdx.x / p.splits) % p.kv_heads;
  const int r0 = (blockIdx.x / p.splits / p.kv_heads) * kRows;   // the block's first query row
  const int group = p.heads / p.kv_heads;
  const int rows = p.nodes * group;
  const int words = (p.nodes + 63) / 64;

  // Query rows past the last repeat it; they are not stored.
  f16x8 qb[kQ][4];
  const unsigned* mask_row[kQ];
#pragma unroll
  for (int u = 0; u < kQ; ++u) {
    const int r = min(r0 + wq0 + 16 * u + c, rows - 1), t = r / group;
    const uint16_t* q = p.q + t * p.q_stride + (kh * group + r % group) * 128 + 8 * g;
    mask_row[u] = reinterpret_cast<const unsigned*>(p.mask + (long long)t * words);
#pragma unroll
    for (int s = 0; s < 4; ++s) qb[u][s] = *reinterpret_cast<const f16x8*>(q + 32 * s);
  }

  float m[kQ];
  f32x4 ls[kQ], o[kQ][8];
#pragma unroll
  for (int u = 0; u < kQ; ++u) {
    m[u] = kNone;
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
  auto weights = [&](const f32x4 (&st)[kQ][2], f16x8 (&pb)[kQ]) {
    // Each lane tests its own eight scores against the bound; only when some lane's pass it
    // are maxima formed across the four lanes of a query.
    float lm[kQ];
    bool grow = false;
#pragma unroll
    for (int u = 0; u < kQ; ++u) {
      lm[u] = fmaxf(fmaxf(fmaxf(st[u][0][0], st[u][0][1]), fmaxf(st[u][0][2], st[u][0][3])),
                    fmaxf(fmaxf(st[u][1][0], st[u][1][1]), fmaxf(st[u][1][2], st[u][1][3])));
      grow |= lm[u] * p.scale_log2 > m[u] + kLazy;         // -inf + kLazy is -inf: the first score grows it
    }
    if (__any(grow)) {
#pragma unroll
      for (int u = 0; u < kQ; ++u) {
        float bm = fmaxf(lm[u], __shfl_xor(lm[u], 16));
        bm = fmaxf(bm, __shfl_xor(bm, 32)) * p.scale_log2;
        const float mn = bm > m[u] + kLazy ? bm : m[u];
        const float alpha = mn == m[u] ? 1.0f : __builtin_amdgcn_exp2f(m[u] - mn);
        ls[u] *= alpha;
#pragma unroll
        for (int e = 0; e < 8; ++e) o[u][e] *= alpha;
        m[u] = mn;
      }
    }
#pragma unroll
    for (int u = 0; u < kQ; ++u) {
      const float nref = m[u] == kNone ? 0.0f : -m[u];     // no row yet: every weight is 0
#pragma unroll
      for (int e = 0; e < 8; ++e)
        pb[u][e] = (_Float16)__builtin_amdgcn_exp2f(__builtin_fmaf(st[u][e / 4][e % 4], p.scale_log2, nref));
      ls[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, pb[u], ls[u], 0, 0, 0);
    }
  };
  auto products = [&](const u32x4 (&v)[8], const f16x8 (&pb)[kQ]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const f16x8 va = v_column(v, e);
#pragma unroll
      for (int u = 0; u < kQ; ++u) o[u][e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, pb[u], o[u][e], 0, 0, 0);
    }
  };

  // The tiles in the order that they are dealt out: the masked ones (node rows, and the
  // cache's last rows if they do not fill a tile), then the cache's whole tiles.
  const int full = p.prefix / kKeys, part = p.prefix % kKeys;
  const int node_tiles = (p.nodes + kKeys - 1) / kKeys;
  const int masked = node_tiles + (part ? 1 : 0);
  const int step = p.splits * kKW;
  int tile = r0 + wq0 < rows ? split * kKW + kw : full + masked;   // a wave without rows takes no tile
  for (; tile < masked; tile += step) {
    const bool node = tile < node_tiles;
    const int j0 = kKeys * (node ? tile : full), n = node ? p.nodes : p.prefix;
    const uint16_t* kb = node ? p.kt + kh * p.thead_stride : p.k + kh * p.head_stride;
    const uint16_t* vb = node ? p.vt + kh * p.thead_stride : p.v + kh * p.head_stride;
    const long long stride = node ? p.trow_stride : p.row_stride;
    u32x4 k[8], v[8];
#pragma unroll
    for (int a = 0; a < 2; ++a) {                          // rows past the last are zeros
      const int row = j0 + 16 * a + c;
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        k[4 * a + s] = u32x4{0u, 0u, 0u, 0u};
        if (row < n) k[4 * a + s] = *reinterpret_cast<const u32x4*>(kb + row * stride + 32 * s + 8 * g);
      }
    }
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = j0 + 16 * a + 4 * g + i;
        v[4 * a + i] = u32x4{0u, 0u, 0u, 0u};
        if (row < n) v[4 * a + i] = *reinterpret_cast<const u32x4*>(vb + row * stride + 8 * c);
      }
    f32x4 st[kQ][2];
    scores(k, st);
    unsigned bits[kQ];
    const unsigned rows_here = n - j0 >= kKeys ? ~0u : (1u << (n - j0)) - 1u;
#pragma unroll
    for (int u = 0; u < kQ; ++u) {
      bits[u] = (node ? mask_row[u][tile] : ~0u) & rows_here;
#pragma unroll
      for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int r = 0; r < 4; ++r) st[u][a][r] = (bits[u] >> (16 * a + 4 * g + r)) & 1u ? st[u][a][r] : kNone;
    }
    f16x8 pb[kQ];
    weights(st, pb);
    // A weight of 0 keeps a finite V row out of a product, but not an infinity or a NaN: where
    // the tile holds one, such elements are taken out of the product and added, with the
    // weights of the queries that see their row.
    if (__any(any_nonfinite(v))) {
      for (int j = 0; j < kKeys && j0 + j < n; ++j) {
        const _Float16* row = reinterpret_cast<const _Float16*>(vb + (j0 + j) * stride + 32 * g);
        const int slot = 4 * (j >> 4) + (j & 3), from = c + 16 * ((j & 15) >> 2);
#pragma unroll
        for (int u = 0; u < kQ; ++u) {
          float w = 0.0f;
#pragma unroll
          for (int e = 0; e < 8; ++e) w = e == slot ? (float)pb[u][e] : w;
          w = __shfl(w, from);
          if ((bits[u] >> j) & 1u) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                const float x = (float)row[8 * i + e];
                if (!(fabsf(x) < __builtin_inff())) o[u][e][i] = __builtin_fmaf(w, x, o[u][e][i]);
              }
          }
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          const unsigned x = v[i][d];
          if ((x & 0x7c00u) == 0x7c00u) v[i][d] &= 0xffff0000u;
          if ((x & 0x7c000000u) == 0x7c000000u) v[i][d] &= 0x0000ffffu;
        }
    }
    products(v, pb);
  }

  // Whole tiles.  Loads read whole rows, four per instruction (instruction j: row 4 j + g,
  // 16-byte chunk c of it); past the last tile the buffer is empty and they return zeros
  // without reading, so the loops have no branch around a load and their waits count exactly
  // the loads that they need.
  const unsigned row_bytes = (unsigned)(p.row_stride * 2);   // 32 rows stay below 4 GiB where a tile is full
  const unsigned off0 = (unsigned)g * row_bytes + 16u * c;
  auto load = [&](const uint16_t* base, int t, int j) {
    const i32x4 rsrc = wave_rsrc(base + kh * p.head_stride + (long long)t * kKeys * p.row_stride, t < full ? 0xffffffffu : 0u);
    return __builtin_bit_cast(u32x4, raw_buffer_load_b128(rsrc, (int)(off0 + 4u * j * row_bytes), 0, 0));
  };
  // K rows in LDS: chunk q of row r at position q ^ (r % 16), so that neither the writes (whole
  // rows) nor the operand reads (one chunk of 16 rows) meet on a bank.  V rows as they are.
  auto put_k = [&](char* lk, int j, u32x4 x) {
    const int r = 4 * j + g;
    *reinterpret_cast<u32x4*>(lk + r * 256 + 16 * (c ^ (r & 15))) = x;
  };
  auto get_k = [&](const char* lk, u32x4 (&k)[8]) {
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
      for (int s = 0; s < 4; ++s)
        k[4 * a + s] = *reinterpret_cast<const u32x4*>(lk + (16 * a + c) * 256 + 16 * ((4 * s + g) ^ c));
  };
  tile -= masked;
  if constexpr (kQW == 1) {
    // A wave's own tiles: K through its own LDS rows (in order within the wave, no barrier),
    // V straight to registers: instruction 4 a + i of a lane is row 16 a + 4 g + i.
    char* lk = smem + wave * kKeys * 256;
    const unsigned voff = (unsigned)(4 * g) * row_bytes + 16u * c;
    auto load_v = [&](int t, u32x4 (&v)[8]) {
      const i32x4 rsrc = wave_rsrc(p.v + kh * p.head_stride + (long long)t * kKeys * p.row_stride, t < full ? 0xffffffffu : 0u);
#pragma unroll
      for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          v[4 * a + i] = __builtin_bit_cast(u32x4, raw_buffer_load_b128(rsrc, (int)(voff + (16u * a + i) * row_bytes), 0, 0));
    };
    if (tile < full) {
      u32x4 kr[8], v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) kr[j] = load(p.k, tile, j);
      load_v(tile, v);
      for (; tile < full; tile += step) {
        u32x4 k[8];
        f32x4 st[kQ][2];
        f16x8 pb[kQ];
#pragma unroll
        for (int j = 0; j < 8; ++j) put_k(lk, j, kr[j]);
#pragma unroll
        for (int j = 0; j < 8; ++j) kr[j] = load(p.k, tile + step, j);
        get_k(lk, k);
        scores(k, st);
        weights(st, pb);
        products(v, pb);
        load_v(tile + step, v);
      }
    }
  } else {
    // The key group's query waves share its tiles: each loads its part of the rows, two tiles
    // ahead, and puts them into one of two LDS buffers; one barrier per tile (a buffer is
    // written again only after the barrier behind its readers).  All key groups run the
    // same number of rounds.
    constexpr int kPart = 8 / kQW;
    const int qw = wave % kQW;
    int rounds = 0;
    for (int w = 0; w < kKW; ++w) {
      int t = split * kKW + w;
      if (t < masked) t += (masked - t + step - 1) / step * step;
      rounds = max(rounds, (full - (t - masked) + step - 1) / step);
    }
    const bool active = r0 + wq0 < rows;
    if (!active) {                                         // loads and barriers only
      tile = split * kKW + kw;
      if (tile < masked) tile += (masked - tile + step - 1) / step * step;
      tile -= masked;
    }
    u32x4 kr[2][kPart], vr[2][kPart];
    auto fetch = [&](int t, u32x4 (&k)[kPart], u32x4 (&v)[kPart]) {
#pragma unroll
      for (int j = 0; j < kPart; ++j) k[j] = load(p.k, t, kPart * qw + j);
#pragma unroll
      for (int j = 0; j < kPart; ++j) v[j] = load(p.v, t, kPart * qw + j);
    };
    auto round = [&](int it, int buf, u32x4 (&kx)[kPart], u32x4 (&vx)[kPart]) {
      char* lk = smem + (buf * kKW + kw) * kKeys * 512;
      char* lv = lk + kKeys * 256;
      const int t = tile + it * step;
#pragma unroll
      for (int j = 0; j < kPart; ++j) {
        put_k(lk, kPart * qw + j, kx[j]);
        *reinterpret_cast<u32x4*>(lv + (4 * (kPart * qw + j) + g) * 256 + 16 * c) = vx[j];
      }
      fetch(t + 2 * step, kx, vx);
      __syncthreads();
      if (active && t < full) {
        u32x4 k[8], v[8];
        f32x4 st[kQ][2];
        f16x8 pb[kQ];
        get_k(lk, k);
        scores(k, st);
        weights(st, pb);
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            v[4 * a + i] = *reinterpret_cast<const u32x4*>(lv + (16 * a + 4 * g + i) * 256 + 16 * c);
        products(v, pb);
      }
    };
    fetch(tile, kr[0], vr[0]);
    fetch(tile + step, kr[1], vr[1]);
    for (int it = 0; it < rounds; it += 2) {               // an odd count's last round finds no tile
      round(it, 0, kr[0], vr[0]);
      round(it + 1, 1, kr[1], vr[1]);
    }
  }
  __syncthreads();                                         // LDS is taken over by the fold

  // Fold the waves.
  float (*fold_o)[kRows][kFoldRow] = reinterpret_cast<float (*)[kRows][kFoldRow]>(smem);
  float (*fold_m)[kRows] = reinterpret_cast<float (*)[kRows]>(smem + (size_t)kKW * kRows * kFoldRow * 4);
  float (*fold_l)[kRows] = fold_m + kKW;
#pragma unroll
  for (int u = 0; u < kQ; ++u) {
    float* dst = &fold_o[kw][wq0 + 16 * u + c][32 * g];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      *reinterpret_cast<f32x4*>(dst + 8 * i) = f32x4{o[u][0][i], o[u][1][i], o[u][2][i], o[u][3][i]};
      *reinterpret_cast<f32x4*>(dst + 8 * i + 4) = f32x4{o[u][4][i], o[u][5][i], o[u][6][i], o[u][7][i]};
    }
    if (g == 0) {
      fold_m[kw][wq0 + 16 * u + c] = m[u];
      fold_l[kw][wq0 + 16 * u + c] = ls[u][0];
    }
  }
  __syncthreads();
  // 16 threads per query row, 8 dims each.
  for (int i = threadIdx.x; i < kRows * 16; i += kThreads) {
    const int q = i >> 4, d = 8 * (i & 15), r = r0 + q;
    if (r >= rows) continue;
    float mx = kNone, l = 0.0f, acc[8];
#pragma unroll
    for (int w = 0; w < kKW; ++w) mx = fmaxf(mx, fold_m[w][q]);
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] = 0.0f;
#pragma unroll
    for (int w = 0; w < kKW; ++w) {
      const float mw = fold_m[w][q];
      if (mw == kNone && fold_l[w][q] == 0.0f) continue;   // saw no row
      const float a = mw == mx ? 1.0f : __builtin_amdgcn_exp2f(mw - mx);
      l += a * fold_l[w][q];
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] += a * fold_o[w][q][d + e];
    }
    if (p.splits == 1) {
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      f16x8 y;
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = (_Float16)(l == 0.0f ? 0.0f : acc[e] * inv);
      *reinterpret_cast<f16x8*>(p.out + (r / group) * p.out_stride + (kh * group + r % group) * 128 + d) = y;
    } else {
      const long long slot = ((long long)kh * rows + r) * p.splits + split;
      float* dst = p.part_o + slot * 128 + d;
      *reinterpret_cast<f32x4*>(dst) = f32x4{acc[0], acc[1], acc[2], acc[3]};
      *reinterpret_cast<f32x4*>(dst + 4) = f32x4{acc[4], acc[5], acc[6], acc[7]};
      if (d == 0) p.part_ml[slot] = float2{mx, l};
    }
  }
}

// Folds the splits of one query row of one cache head: a wave, whose halves take every other
// split, four dims per lane; eight splits' loads are in flight per half.
__global__ __launch_bounds__(256) void tree_attention_merge_kernel(TreeAttnParams p) {
  constexpr int kBatch = 8;
  const int lane = threadIdx.x & 63, half = lane >> 5, d = 4 * (lane & 31);
  const int group = p.heads / p.kv_heads, rows = p.nodes * group;
  const int i = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  if (i >= rows * p.kv_heads) return;
  const float2* ml = p.part_ml + (long long)i * p.splits;
  const float* po = p.part_o + (long long)i * p.splits * 128 + d;
  float mx = kNone, l = 0.0f;
  f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int s0 = half; s0 < p.splits; s0 += 2 * kBatch) {
    float2 w[kBatch];
    f32x4 x[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const int s = min(s0 + 2 * j, p.splits - 1);
      w[j] = ml[s];
      x[j] = *reinterpret_cast<const f32x4*>(po + (long long)s * 128);
      if (s0 + 2 * j >= p.splits) w[j] = float2{kNone, 0.0f};
    }
    float mn = mx;
#pragma unroll
    for (int j = 0; j < kBatch; ++j) mn = fmaxf(mn, w[j].x);
    const float keep = mn == mx ? 1.0f : __builtin_amdgcn_exp2f(mx - mn);
    l *= keep;
    acc *= keep;
    mx = mn;
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      if (w[j].x == kNone && w[j].y == 0.0f) continue;     // saw no row
      const float a = w[j].x == mx ? 1.0f : __builtin_amdgcn_exp2f(w[j].x - mx);
      l += a * w[j].y;
      acc += a * x[j];
    }
  }
  const float mo = __shfl_xor(mx, 32), mn = fmaxf(mx, mo);
  const float a = mx == mn ? 1.0f : __builtin_amdgcn_exp2f(mx - mn), b = mo == mn ? 1.0f : __builtin_amdgcn_exp2f(mo - mn);
  l = a * l + b * __shfl_xor(l, 32);
  typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
  f16x4 y;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float sum = a * acc[e] + b * __shfl_xor(acc[e], 32);
    y[e] = (_Float16)(l == 0.0f ? 0.0f : sum / l);
  }
  const int kh = i / rows, r = i % rows;
  if (half == 0) *reinterpret_cast<f16x4*>(p.out + (r / group) * p.out_stride + (kh * group + r % group) * 128 + d) = y;
}

template <int kQ, int kQW, int kKW>
hipError_t launch(const TreeAttnParams& p, int blocks, hipStream_t stream) {
  hipLaunchKernelGGL((tree_attention_kernel<kQ, kQW, kKW>), dim3(blocks * p.kv_heads * p.splits), dim3(kQW * kKW * 64), 0,
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
  const int rows = p.nodes * p.heads;
  hipLaunchKernelGGL(tree_attention_merge_kernel, dim3((rows + 3) / 4), dim3(256), 0, stream, p);
  return hipGetLastError();
}

}  // namespace qd
