/*
 * purin_train.h -- C ABI of the operators around a projection layer in a
 * network of experts (libpurin_cp.so, beside purin_cp.h).
 *
 * A projection onto a routing polytope gives every token its weights over the
 * experts, most of them exactly zero.  These entry points take such weights to
 * the tokens' experts, the tokens' rows to the experts and back, multiply the
 * rows of each expert by its weight matrix, and scale the gradients of a step
 * to a largest norm.  No counterpart in the reference, which ends at the layer.
 *
 * Conventions are purin_cp.h's: device pointers as void*, sizes as int64_t,
 * hipStream_t as void*, error codes PURIN_CP_*, purin_cp_last_error() for the
 * message.  Every kernel is enqueued on the given stream; no entry point
 * synchronises, allocates device memory or records memory operations, so each
 * may run on a stream under capture.  Calls keep no state: they may run on any
 * streams and threads at once, each with its own workspace and outputs.
 * Matrices are row-major with a row pitch in elements (``ld``); no pointer
 * needs more than its element's alignment (workspaces: 256 bytes).
 * The results do not depend on the launch's order: no floating-point atomics.
 */
#ifndef PURIN_TRAIN_H
#define PURIN_TRAIN_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Element types (PURIN_CP_F32 and PURIN_CP_F64, and the 16-bit ones). */
enum purin_train_dtype {
  PURIN_TRAIN_F32 = 0,
  PURIN_TRAIN_F64 = 1,
  PURIN_TRAIN_BF16 = 2,
  PURIN_TRAIN_F16 = 3
};

#define PURIN_TRAIN_MAX_EXPERTS 1024

/* Workspace bytes of route and sort for tokens * slots pairs (negative: invalid). */
int64_t purin_train_route_workspace_bytes(int64_t tokens, int64_t experts, int64_t slots);

/*
 * From weights (tokens, experts) to the tokens' experts and the order of rows.
 *   ids      (tokens, slots) int32: the experts of a token's ``slots`` largest
 *            positive weights, largest first, ties to the lowest expert; -1
 *            where fewer are positive.  Zero, negative weights and -infinity
 *            choose nothing; NaN counts as larger than any number, so that it
 *            shows in the results.
 *   chosen   (tokens, slots): those weights, 0 beside -1.
 *   offsets  (experts + 1) int32: an expert's first row; the rows' count last.
 *   place    (tokens, slots) int32: a pair's row among the rows sorted by
 *            expert, in the order of pairs (token * slots + slot) within each;
 *            -1 beside -1.
 *   source   (tokens * slots) int32: the pair of each row; -1 from
 *            offsets[experts] on.
 * experts <= PURIN_TRAIN_MAX_EXPERTS, slots <= experts, tokens * slots < 2^31.
 */
int purin_train_route(void* stream, int32_t dtype, int64_t tokens, int64_t experts, int64_t slots,
                      const void* weights, int64_t ld, void* workspace, int64_t workspace_bytes,
                      int32_t* ids, void* chosen, int32_t* offsets, int32_t* place,
                      int32_t* source);

/* offsets, place and source for experts given per pair (int32, or int64 with
 * ``wide``); ``ids`` gets them with -1 for every value outside [0, experts),
 * which sends the pair nowhere.  A token may name an expert more than once. */
int purin_train_sort(void* stream, int32_t wide, int64_t tokens, int64_t experts, int64_t slots,
                     const void* given, void* workspace, int64_t workspace_bytes, int32_t* ids,
                     int32_t* offsets, int32_t* place, int32_t* source);

/* The gradient of route's chosen weights: g_weights (tokens, experts), zero but
 * at the chosen experts. */
int purin_train_route_vjp(void* stream, int32_t dtype, int64_t tokens, int64_t experts,
                          int64_t slots, const int32_t* ids, const void* g_chosen,
                          void* g_weights);

/* rows (tokens * slots, width): rows[place(t, j)] = x(t); zero from
 * offsets[experts] on. */
int purin_train_dispatch(void* stream, int32_t dtype, int64_t tokens, int64_t experts,
                         int64_t slots, int64_t width, const void* x, int64_t ldx,
                         const int32_t* offsets, const int32_t* place, void* rows);

/* out(t) = sum over slots, in their order, of weight(t, j) rows[place(t, j)];
 * a token without experts gets zero.  weights (tokens, slots) of ``wdtype``, or
 * NULL for ones (then this is dispatch's gradient).  Sums are held in 32 bits
 * (64 for F64 rows) and rounded once; F64 weights beside narrower rows are
 * rounded to 32 bits first, and beyond that range are infinite. */
int purin_train_combine(void* stream, int32_t dtype, int32_t wdtype, int64_t tokens,
                        int64_t slots, int64_t width, const void* rows, int64_t ldr,
                        const int32_t* place, const void* weights, void* out);

/* combine's gradients: g_rows[place(t, j)] = weight(t, j) g_out(t), zero from
 * offsets[experts] on; g_weights(t, j) = <g_out(t), rows[place(t, j)]>, zero
 * beside -1.  Either output may be NULL.  Sums and weights as combine's: with
 * rows narrower than F64 an F64 g_weights holds sums of 32 bits. */
int purin_train_combine_vjp(void* stream, int32_t dtype, int32_t wdtype, int64_t tokens,
                            int64_t experts, int64_t slots, int64_t width, const void* g_out,
                            int64_t ldg, const void* rows, int64_t ldr, const int32_t* offsets,
                            const int32_t* place, const void* weights, void* g_rows,
                            void* g_weights);

/* Workspace bytes of expert_product (0 where none is used). */
int64_t purin_train_expert_product_workspace_bytes(int32_t dtype, int64_t rows, int64_t inner,
                                                   int64_t outer, int64_t experts);

/*
 * out (rows, outer): a(p) weight[e] for the rows offsets[e] <= p < offsets[e+1]
 * of each expert (offsets[0] is taken as 0); zero from offsets[experts] on.
 * Offsets ascend; a value outside [0, rows] is read as the nearer end.
 * Element (e, i, o) of weight sits at e * we + i * wi + o * wo, with wi or wo 1.
 * Sums are held in 32 bits (64 for F64) and rounded once.
 */
int purin_train_expert_product(void* stream, int32_t dtype, int64_t rows, int64_t inner,
                               int64_t outer, int64_t experts, const void* a, int64_t lda,
                               const void* weight, int64_t we, int64_t wi, int64_t wo,
                               const int32_t* offsets, void* workspace, int64_t workspace_bytes,
                               void* out, int64_t ldo);

/* Workspace bytes of expert_weights_vjp (0 where none is used). */
int64_t purin_train_expert_weights_vjp_workspace_bytes(int32_t dtype, int64_t rows, int64_t inner,
                                                       int64_t outer, int64_t experts);

/* g_weight (experts, inner, outer), contiguous: the sum over an expert's rows p
 * of a(p)^T g(p); zero for an expert without rows. */
int purin_train_expert_weights_vjp(void* stream, int32_t dtype, int64_t rows, int64_t inner,
                                   int64_t outer, int64_t experts, const void* a, int64_t lda,
                                   const void* g, int64_t ldg, const int32_t* offsets,
                                   void* workspace, int64_t workspace_bytes, void* g_weight);

/* One gradient of a list: ``count`` elements at ``in``, written to ``out``
 * (the same address for in place, or memory that overlaps no gradient). */
typedef struct {
  const void* in;
  void* out;
  int64_t count;
  int32_t dtype;
  int32_t reserved;
} purin_train_tensor;

/* Workspace bytes of clip for a list of ``tensors`` gradients (negative: invalid). */
int64_t purin_train_clip_workspace_bytes(int64_t tensors);

/*
 * norm = the 2-norm of all gradients together (F32 or F64 by norm_dtype; its
 * squares are summed in 64 bits, in an order that the sizes alone decide).
 * largest >= 0: out = in * largest / norm where norm > largest, out = in
 * elsewhere (written only where out is not in).  A NaN norm makes every output
 * NaN, an infinite one makes finite elements zero and infinite ones NaN.
 * largest < 0: the norm alone.  Squares of F64 elements leave the 64-bit range
 * beyond about 1e154 (the norm is infinite) and below 1e-162 (they count as
 * zero).  ``tensors`` is host memory, read before the call returns.  Outputs
 * that overlap each other or another's input are refused.
 */
int purin_train_clip(void* stream, int64_t count, const purin_train_tensor* tensors,
                     double largest, void* workspace, int64_t workspace_bytes,
                     int32_t norm_dtype, void* norm);

/* The gradient of clip's norm: out = in * g_norm / norm for each tensor, zero
 * where the norm is.  norm and g_norm are device scalars of norm_dtype; the
 * list's rules are clip's. */
int purin_train_norm_vjp(void* stream, int64_t count, const purin_train_tensor* tensors,
                         int32_t norm_dtype, const void* norm, const void* g_norm);

#ifdef __cplusplus
}
#endif

#endif /* PURIN_TRAIN_H */
