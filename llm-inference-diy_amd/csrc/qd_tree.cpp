// C ABI of the drafted-token trees: argument checks, workspaces and launches.
// Declared in include/qdiy/decode.h.
#include <algorithm>
#include <cmath>
#include <initializer_list>

#include "qd_internal.h"
#include "qd_tree.h"
#include "qdiy/decode.h"

namespace {

using qd::aligned16;
using qd::aligned2;
using qd::aligned8;
using qd::fail;
using qd::hip_fail;
using qd::overlaps;

bool aligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }

// Strides beyond this are refused, so that no product of strides and counts
// that the checks and kernels form can overflow 64 bits.
constexpr long long kMaxStride = 1LL << 40;
bool stride_ok(long long s, long long least) { return s >= least && s % 8 == 0 && s <= kMaxStride; }

// The attention addresses 32 rows by 32-bit byte offsets from the first of them.
constexpr long long kMaxTreeRow = 1LL << 25;

int check_device(const qd_ctx* ctx) {
  int dev = -1;
  if (hipGetDevice(&dev) != hipSuccess || dev != ctx->device)
    return fail(QD_EINVAL, "current device %d is not the context's device %d", dev, ctx->device);
  return QD_OK;
}

int check_shape(const qd_ctx* ctx, int prefix, int nodes) {
  if (!ctx) return fail(QD_EINVAL, "ctx is NULL");
  if (nodes < 1 || nodes > QD_TREE_MAX_NODES)
    return fail(QD_EINVAL, "nodes %d outside [1, %d]", nodes, QD_TREE_MAX_NODES);
  if (prefix < 0 || prefix > ctx->cfg.max_seqlen)
    return fail(QD_EINVAL, "prefix %d outside [0, %d]", prefix, ctx->cfg.max_seqlen);
  return QD_OK;
}

int check_heads(const qd_ctx* ctx, int num_heads, int head_dim) {
  if (head_dim != QD_HEAD_DIM || head_dim != ctx->cfg.head_dim)
    return fail(QD_EINVAL, "head_dim %d unsupported (must be %d)", head_dim, QD_HEAD_DIM);
  if (num_heads < 1 || num_heads > 4096 || num_heads % ctx->cfg.num_heads != 0)
    return fail(QD_EINVAL, "num_heads %d is not a multiple (at most 4096) of the context's %d", num_heads,
                ctx->cfg.num_heads);
  return QD_OK;
}

// Bytes from the first to past the last element of `rows` rows of the cache's
// heads at the given strides.
size_t row_span(long long rows, long long row_stride, int heads, long long head_stride) {
  if (rows < 1) return 0;
  return ((size_t)(rows - 1) * row_stride + (size_t)(heads - 1) * head_stride + QD_HEAD_DIM) * 2;
}

// Whether rows of 128 halves that are written at these strides keep apart: every dimension steps
// past what the dimensions of smaller strides reach.  (All layouts that nest do; others are
// refused, also where their rows happen to miss each other.)
struct Dim {
  long long n, stride;
};
template <int kDims>
bool rows_apart(Dim (&d)[kDims]) {
  std::sort(d, d + kDims, [](const Dim& a, const Dim& b) { return a.stride < b.stride; });
  long long reach = QD_HEAD_DIM;
  for (const Dim& x : d) {
    if (x.n < 2) continue;
    if (x.stride < reach) return false;
    reach += (x.n - 1) * x.stride;
  }
  return true;
}
// K and V rows of the same strides are two of a kind, this far apart.
Dim k_and_v(const uint16_t* k, const uint16_t* v) { return {2, (long long)(k < v ? v - k : k - v)}; }

struct Span {
  const void* p;
  size_t n;
};
bool any_overlap(Span a, std::initializer_list<Span> others) {
  for (const Span& b : others)
    if (overlaps(a.p, a.n, b.p, b.n)) return true;
  return false;
}

bool verify_args_ok(int nodes, int vocab, int max_children) {
  return nodes >= 1 && nodes <= QD_TREE_MAX_NODES && vocab >= 1 && vocab <= (1 << 24) && max_children >= 0 &&
         max_children <= 64;
}

size_t round16(size_t n) { return (n + 15) & ~(size_t)15; }

}  // namespace

extern "C" {

int qd_tree_layout(const int* parents, int nodes, uint64_t* mask, int* depth) {
  if (!parents) return fail(QD_EINVAL, "parents is NULL");
  if (nodes < 1 || nodes > QD_TREE_MAX_NODES)
    return fail(QD_EINVAL, "nodes %d outside [1, %d]", nodes, QD_TREE_MAX_NODES);
  for (int t = 0; t < nodes; ++t)
    if (t == 0 ? parents[0] >= 0 : parents[t] < 0 || parents[t] >= t)
      return fail(QD_EINVAL, "parents[%d] = %d: node 0 has none (negative), node t one in [0, t)", t, parents[t]);
  const int words = (nodes + 63) / 64;
  for (int t = 0; t < nodes; ++t) {
    if (depth) depth[t] = t ? depth[parents[t]] + 1 : 0;
    if (mask) {
      uint64_t* row = mask + (size_t)t * words;
      for (int w = 0; w < words; ++w) row[w] = t ? mask[(size_t)parents[t] * words + w] : 0;
      row[t / 64] |= 1ull << (t % 64);
    }
  }
  return QD_OK;
}

int qd_tree_qkv_rope(qd_ctx* ctx, const uint16_t* qkv, long long qkv_stride, const uint16_t* bias, const int* depth,
                     uint16_t* q_out, long long q_stride, uint16_t* k_tree, uint16_t* v_tree,
                     long long tree_row_stride, long long tree_head_stride, int prefix, int nodes, int num_heads,
                     int head_dim, hipStream_t stream) {
  int rc = check_shape(ctx, prefix, nodes);
  if (rc == QD_OK) rc = check_heads(ctx, num_heads, head_dim);
  if (rc != QD_OK) return rc;
  if (!qkv || !depth || !q_out || !k_tree || !v_tree)
    return fail(QD_EINVAL, "qkv, depth, q_out, k_tree and v_tree must be non-NULL");
  if (!aligned16(qkv) || !aligned16(bias) || !aligned16(q_out) || !aligned16(k_tree) || !aligned16(v_tree))
    return fail(QD_EINVAL, "qkv, bias, q_out, k_tree and v_tree must be 16-byte aligned");
  if (!aligned4(depth)) return fail(QD_EINVAL, "depth must be 4-byte aligned");
  const int kvh = ctx->cfg.num_heads;
  const long long q_row = (long long)num_heads * QD_HEAD_DIM, row = q_row + 2LL * kvh * QD_HEAD_DIM;
  if (!stride_ok(qkv_stride, row) || !stride_ok(q_stride, q_row))
    return fail(QD_EINVAL, "qkv_stride and q_stride must be multiples of 8, at least %lld and %lld", row, q_row);
  if (!stride_ok(tree_row_stride, 8) || !stride_ok(tree_head_stride, 8))
    return fail(QD_EINVAL, "tree strides must be positive multiples of 8 elements");
  const Span in{qkv, ((size_t)(nodes - 1) * qkv_stride + row) * 2}, b{bias, (size_t)row * 2};
  const Span d{depth, (size_t)nodes * 4}, q{q_out, ((size_t)(nodes - 1) * q_stride + q_row) * 2};
  const size_t span = row_span(nodes, tree_row_stride, kvh, tree_head_stride);
  const Span k{k_tree, span}, v{v_tree, span};
  if (any_overlap(k, {in, b, d, q}) || any_overlap(v, {in, b, d, q}))
    return fail(QD_EINVAL, "k_tree or v_tree overlaps qkv, bias, depth or q_out");
  Dim dims[3] = {{nodes, tree_row_stride}, {kvh, tree_head_stride}, k_and_v(k_tree, v_tree)};
  if (!rows_apart(dims)) return fail(QD_EINVAL, "k_tree's and v_tree's rows overlap each other or themselves");
  const bool in_place = q_out == qkv && q_stride == qkv_stride;
  if (any_overlap(q, {b, d}) || (!in_place && overlaps(q.p, q.n, in.p, in.n)))
    return fail(QD_EINVAL, "q_out overlaps bias, depth or (other than in place) qkv");
  rc = check_device(ctx);
  if (rc != QD_OK) return rc;
  const qd::TreeRopeParams p{qkv, bias, depth, q_out, k_tree, v_tree, ctx->rope_cs, qkv_stride, q_stride,
                             tree_row_stride, tree_head_stride, prefix, nodes, num_heads, kvh, ctx->cfg.max_seqlen};
  const hipError_t e = qd::launch_tree_rope(p, stream);
  return e == hipSuccess ? QD_OK : hip_fail(e, "tree RoPE launch");
}

size_t qd_tree_attention_workspace_bytes(const qd_ctx* ctx, int nodes, int num_heads) {
  if (check_shape(ctx, 0, nodes) != QD_OK || check_heads(ctx, num_heads, QD_HEAD_DIM) != QD_OK) return 0;
  int splits = 1;
  const qd::TreeAttnPlan plan = qd::tree_attn_plan(nodes, num_heads, ctx->cfg.num_heads, 0, ctx->num_cus, &splits);
  return (size_t)plan.blocks * ctx->cfg.num_heads * splits * plan.block_rows * (128 + 2) * sizeof(float);
}

int qd_tree_attention(qd_ctx* ctx, const uint16_t* q, long long q_stride, const uint16_t* k_layer,
                      const uint16_t* v_layer, const uint16_t* k_tree, const uint16_t* v_tree,
                      long long tree_row_stride, long long tree_head_stride, const uint64_t* mask, uint16_t* out,
                      long long out_stride, int prefix, int nodes, int num_heads, int head_dim, void* workspace,
                      size_t workspace_bytes, hipStream_t stream) {
  int rc = check_shape(ctx, prefix, nodes);
  if (rc == QD_OK) rc = check_heads(ctx, num_heads, head_dim);
  if (rc != QD_OK) return rc;
  if (!q || !k_layer || !v_layer || !k_tree || !v_tree || !mask || !out || !workspace)
    return fail(QD_EINVAL, "q, k_layer, v_layer, k_tree, v_tree, mask, out and workspace must be non-NULL");
  if (!aligned16(q) || !aligned16(k_layer) || !aligned16(v_layer) || !aligned16(k_tree) || !aligned16(v_tree) ||
      !aligned16(out) || !aligned16(workspace))
    return fail(QD_EINVAL, "q, k_layer, v_layer, k_tree, v_tree, out and workspace must be 16-byte aligned");
  if (!aligned8(mask)) return fail(QD_EINVAL, "mask must be 8-byte aligned");
  const int kvh = ctx->cfg.num_heads;
  const long long row = (long long)num_heads * QD_HEAD_DIM;
  if (!stride_ok(q_stride, row) || !stride_ok(out_stride, row))
    return fail(QD_EINVAL, "q_stride and out_stride must be multiples of 8 and >= %lld", row);
  if (!stride_ok(tree_row_stride, 8) || !stride_ok(tree_head_stride, 8) || tree_row_stride > kMaxTreeRow)
    return fail(QD_EINVAL, "tree strides must be positive multiples of 8 elements, rows at most 2^25 apart");
  if (ctx->cfg.kv_row_stride > kMaxTreeRow)
    return fail(QD_EINVAL, "the context's kv_row_stride %lld exceeds 2^25", ctx->cfg.kv_row_stride);
  const size_t need = qd_tree_attention_workspace_bytes(ctx, nodes, num_heads);
  if (workspace_bytes < need)
    return fail(QD_EINVAL, "workspace of %zu bytes is smaller than the %zu needed", workspace_bytes, need);
  const Span o{out, ((size_t)(nodes - 1) * out_stride + row) * 2}, ws{workspace, need};
  const Span qs{q, ((size_t)(nodes - 1) * q_stride + row) * 2}, ms{mask, (size_t)nodes * ((nodes + 63) / 64) * 8};
  const size_t cache = row_span(prefix, ctx->cfg.kv_row_stride, kvh, ctx->cfg.kv_head_stride);
  const size_t span = row_span(nodes, tree_row_stride, kvh, tree_head_stride);
  const std::initializer_list<Span> read = {qs, ms, {k_layer, cache}, {v_layer, cache}, {k_tree, span}, {v_tree, span}};
  if (any_overlap(o, read) || any_overlap(ws, read) || overlaps(o.p, o.n, ws.p, ws.n))
    return fail(QD_EINVAL, "out or workspace overlaps the other, q, mask or the rows being read");
  rc = check_device(ctx);
  if (rc != QD_OK) return rc;
  int max_splits = 1;
  const qd::TreeAttnPlan plan = qd::tree_attn_plan(nodes, num_heads, kvh, prefix, ctx->num_cus, &max_splits);
  float* part_o = static_cast<float*>(workspace);
  float2* part_ml = reinterpret_cast<float2*>(part_o + (size_t)plan.blocks * kvh * max_splits * plan.block_rows * 128);
  const qd::TreeAttnParams p{q, k_layer, v_layer, k_tree, v_tree, mask, out, q_stride, out_stride,
                             ctx->cfg.kv_row_stride, ctx->cfg.kv_head_stride, tree_row_stride, tree_head_stride,
                             prefix, nodes, kvh, num_heads / kvh, (float)(1.4426950408889634 / std::sqrt(128.0)),
                             plan.splits, plan.rounds, plan.block_rows, reinterpret_cast<decltype(qd::TreeAttnParams::part_o)>(part_o), part_ml};
  const hipError_t e = qd::launch_tree_attention(p, plan, stream);
  return e == hipSuccess ? QD_OK : hip_fail(e, "tree attention launch");
}

size_t qd_tree_verify_workspace_bytes(int nodes, int vocab, int max_children) {
  if (!verify_args_ok(nodes, vocab, max_children)) return 0;
  const size_t chunks = (vocab + qd::kVerifyChunk - 1) / qd::kVerifyChunk, runs = qd::verify_runs(nodes, (int)chunks);
  const size_t rows = (size_t)nodes * chunks, groups = (size_t)nodes * ((chunks + runs - 1) / runs);
  return round16(2 * rows * sizeof(double)) + round16(2 * groups * sizeof(double)) +
         round16((size_t)max_children * rows * sizeof(double)) + round16(2 * groups * sizeof(float)) +
         round16(groups * sizeof(int));
}

int qd_tree_verify(const uint16_t* target_logits, long long ldt, const uint16_t* draft_logits, long long ldd,
                   const int* tokens, const int* parents, const float* accept_u, const float* sample_u,
                   float temperature, int nodes, int vocab, int max_children, void* workspace, size_t workspace_bytes,
                   int* path, int* emitted, int* count, hipStream_t stream) {
  if (nodes < 1 || nodes > QD_TREE_MAX_NODES)
    return fail(QD_EINVAL, "nodes %d outside [1, %d]", nodes, QD_TREE_MAX_NODES);
  if (vocab < 1 || vocab > (1 << 24)) return fail(QD_EINVAL, "vocab %d outside [1, 2^24]", vocab);
  if (!(temperature >= 0.0f) || temperature > 1e30f)
    return fail(QD_EINVAL, "temperature must be 0 (greedy) or a positive number");
  if (temperature > 0.0f && temperature < 1e-6f)
    return fail(QD_EINVAL, "temperature %g is below 1e-6 (0 is greedy)", (double)temperature);
  const bool greedy = temperature == 0.0f, drawn = !greedy && draft_logits;
  const int most = drawn && nodes > 1 ? max_children : 0;   // rounds of rejected siblings
  if (drawn && nodes > 1 && (most < 1 || most > 64))
    return fail(QD_EINVAL, "max_children %d outside [1, 64]", max_children);
  if (!target_logits || !tokens || !parents || !path || !emitted || !count || !workspace)
    return fail(QD_EINVAL, "target_logits, tokens, parents, path, emitted, count and workspace must be non-NULL");
  if (!greedy && (!accept_u || !sample_u))
    return fail(QD_EINVAL, "accept_u and sample_u must be non-NULL unless temperature is 0");
  if (!aligned2(target_logits) || (drawn && !aligned2(draft_logits)))
    return fail(QD_EINVAL, "logits must be 2-byte aligned");
  if (!aligned4(tokens) || !aligned4(parents) || !aligned4(path) || !aligned4(emitted) || !aligned4(count) ||
      (!greedy && (!aligned4(accept_u) || !aligned4(sample_u))))
    return fail(QD_EINVAL, "tokens, parents, accept_u, sample_u, path, emitted and count must be 4-byte aligned");
  if (!aligned16(workspace)) return fail(QD_EINVAL, "workspace must be 16-byte aligned");
  if (ldt < vocab || ldt > kMaxStride || (drawn && (ldd < vocab || ldd > kMaxStride)))
    return fail(QD_EINVAL, "ldt and ldd must be at least vocab %d", vocab);
  const size_t need = qd_tree_verify_workspace_bytes(nodes, vocab, most);
  if (workspace_bytes < need)
    return fail(QD_EINVAL, "workspace of %zu bytes is smaller than the %zu needed", workspace_bytes, need);
  const size_t n4 = (size_t)nodes * 4;
  const Span t{target_logits, ((size_t)(nodes - 1) * ldt + vocab) * 2};
  // Which draft rows are read only the device knows; those of leaves may be the outputs' memory.
  const Span d{drawn ? draft_logits : nullptr, drawn && nodes > 1 ? (size_t)vocab * 2 : 0};
  const Span au{greedy ? nullptr : accept_u, n4}, su{greedy ? nullptr : sample_u, 4};
  const Span out[4] = {{workspace, need}, {path, n4}, {emitted, n4}, {count, 4}};
  for (int i = 0; i < 4; ++i) {
    if (any_overlap(out[i], {t, d, {tokens, n4}, {parents, n4}, au, su}))
      return fail(QD_EINVAL, "workspace, path, emitted or count overlaps an input");
    for (int j = 0; j < i; ++j)
      if (overlaps(out[i].p, out[i].n, out[j].p, out[j].n))
        return fail(QD_EINVAL, "workspace, path, emitted and count must not overlap");
  }
  qd::TreeVerifyParams p;
  p.target = target_logits;
  p.draft = drawn ? draft_logits : nullptr;
  p.tokens = tokens;
  p.parents = parents;
  p.accept_u = accept_u;
  p.sample_u = sample_u;
  p.path = path;
  p.emitted = emitted;
  p.count = count;
  p.ldt = ldt;
  p.ldd = drawn ? ldd : 0;
  p.scale_log2 = greedy ? 0.0 : 32.0 * 1.4426950408889634 / (double)temperature;
  p.nodes = nodes;
  p.vocab = vocab;
  p.chunks = (vocab + qd::kVerifyChunk - 1) / qd::kVerifyChunk;
  p.runs = qd::verify_runs(nodes, p.chunks);
  p.groups = (p.chunks + p.runs - 1) / p.runs;
  p.max_children = most;
  p.greedy = greedy;
  const size_t rows = (size_t)nodes * p.chunks, groups = (size_t)nodes * p.groups;
  char* ws = static_cast<char*>(workspace);
  auto take = [&ws](size_t bytes) {
    char* at = ws;
    ws += round16(bytes);
    return at;
  };
  p.sums = reinterpret_cast<double*>(take(2 * rows * sizeof(double)));
  p.group_sums = reinterpret_cast<double*>(take(2 * groups * sizeof(double)));
  p.rounds = reinterpret_cast<double*>(take((size_t)most * rows * sizeof(double)));
  p.maxes = reinterpret_cast<float*>(take(2 * groups * sizeof(float)));
  p.args = reinterpret_cast<int*>(take(groups * sizeof(int)));
  const hipError_t e = qd::launch_tree_verify(p, stream);
  return e == hipSuccess ? QD_OK : hip_fail(e, "tree verification launch");
}

int qd_tree_commit(qd_ctx* ctx, const uint16_t* k_tree, const uint16_t* v_tree, long long tree_layer_stride,
                   long long tree_row_stride, long long tree_head_stride, uint16_t* k_cache, uint16_t* v_cache,
                   long long cache_layer_stride, const int* path, const int* count, int prefix, int nodes, int layers,
                   hipStream_t stream) {
  int rc = check_shape(ctx, prefix, nodes);
  if (rc != QD_OK) return rc;
  if (layers < 1 || layers > 4096) return fail(QD_EINVAL, "layers %d outside [1, 4096]", layers);
  if (!k_tree || !v_tree || !k_cache || !v_cache || !path || !count)
    return fail(QD_EINVAL, "k_tree, v_tree, k_cache, v_cache, path and count must be non-NULL");
  if (!aligned16(k_tree) || !aligned16(v_tree) || !aligned16(k_cache) || !aligned16(v_cache))
    return fail(QD_EINVAL, "k_tree, v_tree, k_cache and v_cache must be 16-byte aligned");
  if (!aligned4(path) || !aligned4(count)) return fail(QD_EINVAL, "path and count must be 4-byte aligned");
  if (!stride_ok(tree_row_stride, 8) || !stride_ok(tree_head_stride, 8))
    return fail(QD_EINVAL, "tree strides must be positive multiples of 8 elements");
  if (!stride_ok(tree_layer_stride, 0) || !stride_ok(cache_layer_stride, 0) ||
      (layers > 1 && (tree_layer_stride == 0 || cache_layer_stride == 0)))
    return fail(QD_EINVAL, "layer strides must be positive multiples of 8 elements");
  const qd_cfg& c = ctx->cfg;
  const int kvh = c.num_heads;
  const size_t tree = (size_t)(layers - 1) * tree_layer_stride * 2 + row_span(nodes, tree_row_stride, kvh, tree_head_stride);
  const size_t cache = (size_t)(layers - 1) * cache_layer_stride * 2 + row_span(std::min(prefix + nodes, c.max_seqlen), c.kv_row_stride, kvh, c.kv_head_stride);
  const long long at = (long long)prefix * c.kv_row_stride;
  const bool in_place = k_tree == k_cache + at && v_tree == v_cache + at && tree_row_stride == c.kv_row_stride &&
                        tree_head_stride == c.kv_head_stride && (layers == 1 || tree_layer_stride == cache_layer_stride);
  Dim dims[4] = {{std::min(nodes, c.max_seqlen - prefix), c.kv_row_stride},
                 {kvh, c.kv_head_stride},
                 {layers, cache_layer_stride},
                 k_and_v(k_cache, v_cache)};
  if (!rows_apart(dims)) return fail(QD_EINVAL, "the caches' rows overlap each other or themselves");
  const Span kc{k_cache, cache}, vc{v_cache, cache};
  if (any_overlap(kc, {{path, (size_t)nodes * 4}, {count, 4}}) || any_overlap(vc, {{path, (size_t)nodes * 4}, {count, 4}}))
    return fail(QD_EINVAL, "path or count overlaps the caches");
  if (!in_place && (any_overlap(kc, {{k_tree, tree}, {v_tree, tree}}) || any_overlap(vc, {{k_tree, tree}, {v_tree, tree}})))
    return fail(QD_EINVAL, "k_tree or v_tree overlaps the caches other than as their rows from prefix on");
  if (in_place && prefix + nodes > c.max_seqlen)
    return fail(QD_EINVAL, "node rows [%d, %d) in the cache end past its %d rows", prefix, prefix + nodes, c.max_seqlen);
  rc = check_device(ctx);
  if (rc != QD_OK) return rc;
  const qd::TreeCommitParams p{{k_tree, v_tree}, {k_cache, v_cache}, tree_layer_stride, tree_row_stride,
                               tree_head_stride, cache_layer_stride, c.kv_row_stride, c.kv_head_stride, path, count,
                               prefix, nodes, layers, kvh, c.max_seqlen, in_place ? 1 : 0};
  const hipError_t e = qd::launch_tree_commit(p, stream);
  return e == hipSuccess ? QD_OK : hip_fail(e, "tree commit launch");
}

}  // extern "C"
