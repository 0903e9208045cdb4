/*
 * qdiy/decode.h -- C ABI of the rest of one decode step on MI355X (gfx950):
 * the launches of the reference engine's QwenEngine::step around attention
 * (SeaTheDestiny/LLM-inference-DIY, framework_src/qwen_infer.cu:700-731).
 *
 *   gemm(d_attn_proj, d_qkv_out, attn_proj_w, 1, H, H)        (:701)
 *   add_bias_kernel(d_x, d_attn_proj, H)                      (:704)
 *       -> qd_proj_residual(d_qkv_out, attn_proj_w, d_x, d_x, H, H)
 *   rmsnorm_kernel(d_norm_x, d_x, ln_2, H, eps)               (:708)
 *   gemm(d_ffn_w1, ...) ; gemm(d_ffn_w2, ...)                 (:711-712)
 *   swiglu_kernel(d_ffn_act, d_ffn_w1, d_ffn_w2, IM)          (:715)
 *       -> qd_ffn_up_swiglu(d_x, ln_2, eps, ffn_w1, ffn_w2, d_ffn_act, H, IM)
 *   gemm(d_ffn_proj, d_ffn_act, ffn_proj_w, 1, H, IM)         (:718)
 *   add_bias_kernel(d_x, d_ffn_proj, H)                       (:721)
 *       -> qd_proj_residual(d_ffn_act, ffn_proj_w, d_x, d_x, H, IM)
 *   rmsnorm_kernel(d_norm_x, d_x, ln_f, H, eps)               (:725)
 *   gemm(d_logits, d_norm_x, lm_head, 1, V, H)                (:728)
 *   argmax_kernel(d_next_token, d_logits, V)                  (:731)
 *       -> qd_lm_head_argmax(d_x, ln_f, eps, lm_head, d_logits, V, H, ws, ...)
 *
 * Conventions are those of qdiy/attn.h: fp16 as uint16_t bit patterns in
 * device memory, asynchronous on `stream`, status codes, no host sync.
 * Weight matrices stay in the .bin file's [out][in] layout
 * (model_weights/convert_weights.py:135-172); the reference engine transposes
 * them at load (qwen_infer.cu:230-241) for its hgemv_kernel, this library
 * reads them as stored.
 *
 * Numerics: every GEMV output is the fp32 sum of exact fp16 x fp16 products in
 * one fixed order -- lane l of a 64-lane wave owns elements
 * k = 512*j + 8*l + e and adds them sequentially (j, then e ascending), then
 * the 64 lane sums are added in a fixed tree -- rounded once to fp16 where the
 * reference stores a half.  RMSNorm uses the same order for its sum of
 * squares.  Results are therefore bit-for-bit reproducible on the host.
 */
#ifndef QDIY_DECODE_H
#define QDIY_DECODE_H

#include <stddef.h>
#include <stdint.h>

#include "qdiy/attn.h"
#include <hip/hip_runtime_api.h>

#ifdef __cplusplus
extern "C" {
#endif

/* out[n] = half(residual[n] + half(sum_k W[n][k] * x[k])) for n < n_out.
 * W is [n_out][k_in] fp16; k_in a multiple of 8, at most 8192; x, w 16-byte
 * aligned.
 * residual and out may be the same buffer (the reference adds in place into
 * d_x); otherwise they must not overlap, and out must not overlap x or w
 * (QD_EINVAL).  Replaces hgemv_kernel + add_bias_kernel (hgemm_final.cuh:274-295,
 * bias.cuh:6-11; qwen_infer.cu:701-704 and :718-721). */
int qd_proj_residual(const uint16_t* x, const uint16_t* w, const uint16_t* residual,
                     uint16_t* out, int n_out, int k_in, hipStream_t stream);

/* act[i] = half(g_i * (u_i / (1 + exp(-u_i)))), g_i = half(W1[i] . xn),
 * u_i = half(W2[i] . xn), xn = half(x * (1/sqrt(mean(x^2) + eps)) * norm_w),
 * for i < inter.  W1 (gate, ffn_w1) and W2 (up, ffn_w2) are [inter][hidden];
 * hidden a multiple of 512, at most 4096.  exp(-u) is computed as
 * 2^(-u * log2 e) by a polynomial the host can repeat exactly.  act must
 * not overlap x, norm_w, w1 or w2 (QD_EINVAL).  Replaces
 * rmsnorm_kernel + 2 x hgemv_kernel + swiglu_kernel (rmsnorm.cuh:6-57,
 * swiglu.cuh:6-15; qwen_infer.cu:708-715). */
int qd_ffn_up_swiglu(const uint16_t* x, const uint16_t* norm_w, float eps, const uint16_t* w1,
                     const uint16_t* w2, uint16_t* act, int hidden, int inter,
                     hipStream_t stream);

/* Batched projection of m rows (prompt tokens at once):
 *   y[i][j] = half(sum_k x[i][k] * w[j][k])                        residual == NULL
 *   y[i][j] = half(float(residual[i][j]) + float(half(sum)))       otherwise
 * for i < m, j < n.  x rows are ldx elements apart, y and residual rows ldy
 * apart; w is [n][k], the .bin file's layout (the reference transposes its
 * weights at load and multiplies [k][n]).  Replaces QwenEngine::gemm for m > 1
 * (qwen_infer.cu:359-367: hgemm_swizzle_nn) in prefill (:462, :542, :573-574,
 * :593).
 *   mode QD_GEMM_EXACT: every output is the decode step's sum for that row --
 *     lane l of a wave adds k = 512j + 8l + e in order, then the fixed wave64
 *     tree -- so a prompt's rows are bit-identical to qd_proj_residual and the
 *     decode GEMVs token by token.  k a multiple of 8, at most 8192.
 *   mode QD_GEMM_MFMA: the matrix cores (v_mfma_f32_16x16x32_f16); products
 *     are exact and summed in fp32 in the hardware's order, so results are not
 *     reproducible on the host.  k a multiple of 64.
 * x and w 16-byte aligned, ldx a multiple of 8 and >= k, ldy >= n; y and
 * residual 2-byte aligned.  residual may be y (in place); y must not overlap x
 * or w (QD_EINVAL). */
#define QD_GEMM_EXACT 0
#define QD_GEMM_MFMA 1
int qd_gemm_nt(const uint16_t* x, long long ldx, const uint16_t* w, const uint16_t* residual,
               uint16_t* y, long long ldy, int m, int n, int k, int mode, hipStream_t stream);

/* Batched FFN up-projection of m prompt rows on the matrix cores, gate and up
 * GEMMs in one pass with the SwiGLU in the epilogue:
 *   act[i][j] = half(g * (u / (1 + exp(-u)))),  g = half(x[i] . w1[j]),
 *                                              u = half(x[i] . w2[j])
 * for i < m, j < n (x rows ldx apart, act rows ldy apart; w1 and w2 [n][k]).
 * Replaces the prompt's w1 and w2 gemms and swiglu_kernel
 * (qwen_infer.cu:573-586).  exp(-u) is this library's exp2 of -u * log2(e)
 * (as qd_ffn_up_swiglu); the sums are fp32 in the hardware's order, as in
 * QD_GEMM_MFMA.  k a positive multiple of 64; x, w1 and w2 16-byte aligned,
 * ldx a multiple of 8 and >= k, ldy >= n, act 2-byte aligned and not
 * overlapping x, w1 or w2. */
int qd_gemm_swiglu(const uint16_t* x, long long ldx, const uint16_t* w1, const uint16_t* w2,
                   uint16_t* act, long long ldy, int m, int n, int k, hipStream_t stream);

/* Causal attention of `tokens` prompt queries at positions pos0 .. pos0 +
 * tokens - 1 of one layer, all heads: query t attends over cache rows
 * [0, pos0 + t] (rows written beforehand, K rotated).  Query t's row is
 * q + t*q_stride (head h at + h*128: the rotated Q third of the prefill's QKV
 * rows); its output row is out + t*out_stride.  Replaces the reference's
 * prompt attention, qwen_infer.cu:484-527 (gather_q_from_qkv and
 * gather_kv_from_cache into per-head buffers, flash_attn_tuned_A_kernel with
 * the causal mask of flash_attn_causal.cuh once per head, then
 * scatter_interleaved_kernel), reading Q and the cache in place.
 *   mode QD_GEMM_EXACT: every query with the arithmetic qd_decode_attention
 *     uses at its length, batched (one fused launch for the queries of up to
 *     224 rows; one split launch per run of queries with one tile shape and
 *     one merge per 256 queries for the others): outputs are bit-identical
 *     to decoding the prompt token by token.  The first call with queries
 *     beyond 224 rows allocates the context's prefill scratch.
 *   mode QD_GEMM_MFMA: one causal FlashAttention launch on the matrix cores
 *     (v_mfma_f32_16x16x32_f16, softmax weights rounded to fp16 for the
 *     product, hardware exp2): within 2e-3 of the exact outputs for
 *     N(0,1)-scale inputs, not reproducible on the host.
 * Requires tokens >= 1, 0 <= pos0, pos0 + tokens <= max_seqlen; q, out,
 * k_layer and v_layer 16-byte aligned; q_stride and out_stride multiples of 8
 * and >= num_heads*128; out must not overlap q or the cache rows read. */
int qd_prefill_attention(qd_ctx* ctx, const uint16_t* q, long long q_stride, const uint16_t* k_layer,
                         const uint16_t* v_layer, uint16_t* out, long long out_stride, int pos0,
                         int tokens, int num_heads, int head_dim, int mode, hipStream_t stream);

/* Device workspace (bytes) qd_lm_head_argmax needs for a vocabulary size. */
size_t qd_lm_head_workspace_bytes(int vocab);

/* logits[v] = half(W[v] . xn) for v < vocab with xn the RMSNorm of x by
 * norm_w (as above), then *token (device int) = the index of the largest
 * logit.  Ties go to the lowest index; -0 equals +0; NaN never wins.  (The
 * reference's argmax_kernel breaks ties by its thread and lane order,
 * argmax.cuh:19-66.)  W is [vocab][hidden].  workspace: device memory of
 * qd_lm_head_workspace_bytes(vocab) bytes, 8-byte aligned.  logits,
 * workspace and token must not overlap each other or x, norm_w, w
 * (QD_EINVAL).  Replaces
 * rmsnorm_kernel + hgemv_kernel + argmax_kernel (qwen_infer.cu:725-731). */
int qd_lm_head_argmax(const uint16_t* x, const uint16_t* norm_w, float eps, const uint16_t* w,
                      uint16_t* logits, int vocab, int hidden, void* workspace,
                      size_t workspace_bytes, int* token, hipStream_t stream);

/* ---- Trees of drafted tokens ------------------------------------------------
 *
 * Speculative decoding over the KV cache; no counterpart in the reference,
 * whose engine decodes one token per step.  A drafter proposes `nodes` tokens
 * that form a tree: node 0 is the last emitted token (its K/V row is not in the
 * cache yet), node t > 0 a drafted token that follows parents[t] < t.  One
 * target step then checks all of them:
 *
 *   qd_tree_layout          (host, once per tree shape) masks and depths
 *   per layer: projections of the nodes' rows (qd_gemm_nt), then
 *     qd_tree_qkv_rope      bias, RoPE at prefix + depth, K/V rows of the nodes
 *     qd_tree_attention     every node over the prefix and its ancestors
 *   qd_tree_verify          which path stands, and the token after it
 *   qd_tree_commit          that path's K/V rows into the caches of all layers
 *
 * The nodes' K/V rows lie apart from the cache, row t at base + t*tree_row_stride
 * + head*tree_head_stride (elements), so a tree needs no cache rows of its own
 * and the cache changes only when a path is committed.  The context's num_heads
 * is the cache's head count; num_heads here is the number of query heads, a
 * multiple of it: query head h reads cache head h / (num_heads / ctx heads).
 * At most QD_TREE_MAX_NODES nodes, 4096 query heads, strides of 2^40 elements.
 * Depths, paths and counts are device int32, so the calls of one step follow each
 * other without the host.  prefix is the host's: the next step's is prefix +
 * count, which the host has to read first, and a captured graph of a step holds
 * for the prefix that it was captured with, no other.
 * These calls take only the context's sizes and its cos/sin table: calls with
 * distinct workspaces and outputs may run at the same time on several streams,
 * also of one context.  A workspace belongs to one call at a time (two captured
 * graphs that share one must not run together). */
#define QD_TREE_MAX_NODES 1024

/* Host only: masks and depths of a tree.  mask[t * ceil(nodes / 64) + w] bit b
 * says whether node t sees node 64 w + b (itself and its ancestors); depth[0] is
 * 0, depth[t] = depth[parents[t]] + 1.  parents[0] must be negative and
 * 0 <= parents[t] < t otherwise (QD_EINVAL).  Either output may be NULL.  All
 * three are host memory; copy the outputs to the device. */
int qd_tree_layout(const int* parents, int nodes, uint64_t* mask, int* depth);

/* QKV bias + rotate-half RoPE of a tree's nodes: for node t, with the
 * arithmetic and the bits of qd_qkv_bias_rope_cache at position
 * prefix + depth[t],
 *   b = half(qkv[t] + bias)            (bias == NULL: b = qkv[t])
 *   q_out[t] = rotated Q part, K row t of k_tree = rotated K part, V row t of
 *   v_tree = V part of b.
 * qkv rows are [num_heads + 2 * ctx heads][128] (Q, K, V), qkv_stride elements
 * apart; q_out rows are [num_heads][128], q_stride apart.  qkv is not changed,
 * unless q_out is qkv itself with the same stride (the Q part is then rotated in
 * place).  depth is device memory, depth[t] >= 0; a node whose position lies
 * outside [0, max_seqlen) gets NaN in all three rows, so that the mistake shows.
 * All fp16 buffers 16-byte aligned, strides multiples of 8; depth 4-byte
 * aligned; k_tree, v_tree and q_out must not overlap the inputs otherwise, nor
 * q_out the node rows, nor K and V rows each other or themselves: of rows, heads
 * and the step from k_tree to v_tree each is at least what those of smaller steps
 * reach (QD_EINVAL). */
int qd_tree_qkv_rope(qd_ctx* ctx, const uint16_t* qkv, long long qkv_stride, const uint16_t* bias,
                     const int* depth, uint16_t* q_out, long long q_stride, uint16_t* k_tree,
                     uint16_t* v_tree, long long tree_row_stride, long long tree_head_stride,
                     int prefix, int nodes, int num_heads, int head_dim, hipStream_t stream);

/* Attention of a tree's nodes, all heads:
 *   out[t][h] = half( sum_j w_j V_j ),  w = softmax_j( q[t][h] . K_j / sqrt(128) )
 * over the cache rows j < prefix and the node rows j whose bit is set in row t
 * of mask (ceil(nodes / 64) words a row, device memory; any mask, not only
 * qd_tree_layout's; bits past `nodes` are ignored).  A node that sees no row
 * (prefix 0, no bit) gets zeros.  What K and V hold in rows that a node does not
 * see, infinities and NaN too, does not reach its output; infinities and NaN in
 * V rows that it sees do, however small their weight.  fp32 accumulation on
 * the matrix cores, softmax weights rounded to fp16 for the second product: not
 * reproducible on the host, but the same bits from call to call.
 * q and out rows are [num_heads][128], q_stride and out_stride elements apart.
 * workspace: qd_tree_attention_workspace_bytes(ctx, nodes, num_heads) bytes of
 * device memory, 16-byte aligned; its contents need not survive between calls.
 * Requires 0 <= prefix <= max_seqlen; fp16 pointers 16-byte aligned, strides
 * multiples of 8, tree_row_stride (and the context's
 * kv_row_stride) at most 2^25; mask 8-byte aligned; out and workspace overlap neither each
 * other nor anything that is read (QD_EINVAL). */
int qd_tree_attention(qd_ctx* ctx, const uint16_t* q, long long q_stride, const uint16_t* k_layer,
                      const uint16_t* v_layer, const uint16_t* k_tree, const uint16_t* v_tree,
                      long long tree_row_stride, long long tree_head_stride, const uint64_t* mask,
                      uint16_t* out, long long out_stride, int prefix, int nodes, int num_heads,
                      int head_dim, void* workspace, size_t workspace_bytes, hipStream_t stream);

/* Workspace bytes of qd_tree_attention, at any prefix; 0 for arguments it
 * refuses. */
size_t qd_tree_attention_workspace_bytes(const qd_ctx* ctx, int nodes, int num_heads);

/* Which drafted tokens stand.  target_logits row t (vocab halves, ldt elements
 * apart) is the target's after node t, tokens[t] the node's token (tokens[0] is
 * not read), parents as in qd_tree_layout.  From node 0 on, the current node's
 * children are tested in index order; the first accepted one becomes the current
 * node; when none is left one more token is taken and the walk ends:
 *   temperature == 0 (greedy; the pointers u and draft_logits are not read):
 *     child c stands if tokens[c] is the argmax of the current row; the last
 *     token is the argmax.  Ties go to the lowest index, -0 equals +0, NaN
 *     never wins (as qd_lm_head_argmax).
 *   temperature > 0, draft_logits == NULL: with p = softmax(row / temperature),
 *     child c stands if accept_u[c] * (sum of p) < p(tokens[c]); otherwise
 *     p(tokens[c]) becomes 0.  (Drafts that are given tokens, e.g. the most
 *     likely ones or copies from the prompt.)
 *   temperature > 0 and draft_logits (row t: the drafter's logits after node t,
 *     ldd apart; rows of nodes without children are not read: the buffer may end
 *     before them, or hold something else there), the children drawn
 *     independently from q = softmax(draft row / temperature): child c stands if
 *     accept_u[c] * q(tokens[c]) < p(tokens[c]); otherwise p becomes
 *     max(p - q, 0), normalised.  Only the first max_children children of a
 *     node are tested (1 <= max_children <= 64; not read in the other modes,
 *     nor for one node).
 *   The last token of the two sampled modes is the first index whose cumulative
 *   p exceeds sample_u[0] times its total.
 * In both sampled modes the emitted tokens are distributed as the target's when
 * accept_u and sample_u are independent uniforms of [0, 1).  Weights are 64-bit
 * numbers good to a relative 2e-12, and summed in 64 bits; what rejected given
 * drafts leave for their siblings is 1 less their shares, good to some 1e-11 of
 * the whole.  (Random numbers nearer to a decision than that may fall to its other
 * side.)  temperature is 0 or in [1e-6, 1e30], vocab at most 2^24.  A NaN logit counts as -inf; +inf logits share the
 * whole probability; a row of -inf alone is uniform.  A token outside
 * [0, vocab) is never accepted, a node whose parent is not in [0, t) never
 * reached.  If max(p - q, 0) is zero everywhere, p is kept as it was; if nothing
 * is left of given drafts' p (numbers of 1 and more can do that), the last token is
 * 0.
 *   path[nodes]:    the accepted nodes from node 0 on, then -1
 *   emitted[nodes]: the tokens of path[1..], then the last token, then -1
 *   count[0]:       the number of entries of both (1 + accepted drafts)
 * tokens, parents, u and the outputs are device memory, 4-byte aligned; logits
 * 2-byte aligned, ldt and ldd >= vocab.  workspace: device memory, 16-byte
 * aligned, of qd_tree_verify_workspace_bytes(nodes, vocab, max_children) bytes
 * (enough with a max_children of 0 where it is not read).
 * Outputs and workspace overlap neither each other nor anything that is read
 * (QD_EINVAL; of the draft rows only row 0 is known to the host, the others are
 * the caller's to keep apart). */
int qd_tree_verify(const uint16_t* target_logits, long long ldt, const uint16_t* draft_logits,
                   long long ldd, const int* tokens, const int* parents, const float* accept_u,
                   const float* sample_u, float temperature, int nodes, int vocab,
                   int max_children, void* workspace, size_t workspace_bytes, int* path,
                   int* emitted, int* count, hipStream_t stream);

/* Workspace bytes of qd_tree_verify in any mode; 0 for arguments it refuses. */
size_t qd_tree_verify_workspace_bytes(int nodes, int vocab, int max_children);

/* Copies the K/V rows of an accepted path into the caches of all layers: for
 * every layer l and i < count[0], cache row prefix + i = node row path[i].
 * Layer l of the node rows starts at k_tree + l*tree_layer_stride, of the caches
 * at k_cache + l*cache_layer_stride (elements; v alike).  path and count are
 * device memory (qd_tree_verify's); entries outside [0, nodes), rows at or past
 * max_seqlen and entries from `nodes` on are skipped; other rows are left as they
 * were (a cache need not reach past row prefix + nodes).  The node rows may be the cache's own rows from prefix on, in every layer
 * (k_tree == k_cache + prefix*kv_row_stride, v alike, all strides the caches'),
 * with path strictly ascending, as qd_tree_verify's is: the path's rows are then
 * moved up in place.  Otherwise
 * they must not overlap the caches, nor the caches' rows each other (as in
 * qd_tree_qkv_rope; with layers) (QD_EINVAL).  fp16 pointers 16-byte aligned,
 * strides multiples of 8. */
int qd_tree_commit(qd_ctx* ctx, const uint16_t* k_tree, const uint16_t* v_tree,
                   long long tree_layer_stride, long long tree_row_stride,
                   long long tree_head_stride, uint16_t* k_cache, uint16_t* v_cache,
                   long long cache_layer_stride, const int* path, const int* count, int prefix,
                   int nodes, int layers, hipStream_t stream);

#ifdef __cplusplus
}
#endif
#endif /* QDIY_DECODE_H */
