/*
 * flash-train for MI355X -- convenience C API.
 *
 * Drop-in for the reference's include/flash_train/flash_train.h:46-48.
 */
#ifndef FTRAIN_FLASH_TRAIN_H_
#define FTRAIN_FLASH_TRAIN_H_

#include <flash_train/common.h>

#ifdef __cplusplus
extern "C" {
#endif

/*
 * d = alpha * (a @ b) + beta * c with the recommended Primitive (index 0).
 *
 * Equivalent to building the Gemm Pattern, creating Ops and Args, creating a
 * Plan and executing its Primitive 0 (reference src/api/gemm_api.cpp:54-83);
 * the Ops is built once per process and Plan creation is a selection-cache
 * hit after the first call for a given problem description.  a, b, c, d are
 * rank-two device views (c may have null memory, which drops the beta term);
 * alpha and beta are host fp32 scalars.  Asynchronous on `stream`.  On
 * failure the thread's last message is the failing step's message.
 * Under stream capture a problem not yet seen on this thread and stream runs
 * the first Primitive that needs no more than `workspace_bytes` (nothing is
 * allocated during the capture); FTRAIN_STATUS_UNSUPPORTED when none does.
 * A graph that captured a call keeps its Plan alive until the graph and its
 * executable graphs are destroyed.
 */
FTRAIN_API FTrainStatus ftrainGemm(FTrainStorageView a, FTrainStorageView b, FTrainStorageView c, FTrainStorageView d,
                                   FTrainStorageView alpha, FTrainStorageView beta, FTrainNumericType compute_type,
                                   void* workspace, uint64_t workspace_bytes, FTrainStream stream);

/*
 * ftrainGemm without device allocation.  No counterpart in the reference: it
 * is for callers that cannot allocate device memory -- code under HIP graph
 * capture, tight serving loops, harnesses that forbid hipMalloc.
 *
 * Same operands, result and errors as ftrainGemm, minus the workspace: a
 * split-k Primitive keeps its partial tiles in the library's fixed device
 * scratch array (64 MiB per GPU, held from library load until the process
 * ends) and no call allocates or frees device memory.  The Primitive run is
 * the first in the Plan's rank order whose partial tiles fit the array
 * (Primitive 0 whenever it fits); UNSUPPORTED when none fits.  Every call on
 * one GPU shares that GPU's array: calls that may overlap on one GPU (other
 * streams, other threads) race and must be serialised by the caller.
 * Nothing in the array needs to start at zero.
 */
FTRAIN_API FTrainStatus ftrainGemmNoAlloc(FTrainStorageView a, FTrainStorageView b, FTrainStorageView c,
                                          FTrainStorageView d, FTrainStorageView alpha, FTrainStorageView beta,
                                          FTrainNumericType compute_type, FTrainStream stream);

/* ---- operators around a training step's products (no counterpart in the reference) ----
 *
 * Views are device memory.  A matrix may be FTRAIN_INDEX_TYPE_CONTINUOUS or,
 * with FTRAIN_INDEX_TYPE_INVALID, have contiguous rows at any row stride that
 * covers them; other arrays are dense.  Element types T are FP32, BF16 and
 * FP16; sums and exponentials are in FP32 or wider.  Each call is kernel
 * launches on `stream` only (nothing is allocated, copied or synchronised, so
 * it may be captured into a graph), and gives the same bits for the same
 * inputs.  `workspace` is device memory of at least the bytes that the
 * operator's ...WorkspaceBytes call names for the same views (their strides
 * and alignment matter), aligned to 256 bytes, with any contents; calls that
 * may overlap need one each.  Errors: INVALID_ARGUMENT
 * (null, shapes, host memory, workspace), UNSUPPORTED (types, strides,
 * limits), INTERNAL_ERROR (a launch failed).
 */

/*
 * Softmax cross entropy of an output head, without its logits in memory.
 * hidden (tokens x h, T), weight (classes x h, T), target (tokens, INT32 or
 * INT64) give, for every token,
 *   lse = log sum_v exp(hidden . weight_v),  loss = lse - hidden . weight_target
 * (tokens, FP32), both 0 where the target is `ignore_index`.  An ignored
 * token's hidden state is not read into any sum.  Any other target outside
 * the classes gives a loss of NaN.  At most 2^31 - 1024 tokens and classes,
 * 2^20 hidden values and row stride of the weight.
 */
FTRAIN_API FTrainStatus ftrainLinearCrossEntropyWorkspaceBytes(FTrainStorageView hidden, FTrainStorageView weight,
                                                               bool backward, uint64_t* workspace_bytes);
FTRAIN_API FTrainStatus ftrainLinearCrossEntropy(FTrainStorageView hidden, FTrainStorageView weight,
                                                 FTrainStorageView target, FTrainStorageView loss,
                                                 FTrainStorageView lse, int64_t ignore_index, void* workspace,
                                                 uint64_t workspace_bytes, FTrainStream stream);
/*
 * Its gradients for grad_loss (tokens, FP32), with the lse of the forward
 * call: grad_hidden and grad_weight, shaped and typed as hidden and weight and
 * overwritten.  With 16-bit T the logits' gradient is rounded to T before its
 * two products (FP16: times a power of two that keeps small probabilities).
 * A target outside the classes makes its token's and the weight's gradient NaN.
 */
FTRAIN_API FTrainStatus ftrainLinearCrossEntropyBackward(FTrainStorageView grad_loss, FTrainStorageView hidden,
                                                         FTrainStorageView weight, FTrainStorageView target,
                                                         FTrainStorageView lse, FTrainStorageView grad_hidden,
                                                         FTrainStorageView grad_weight, int64_t ignore_index,
                                                         void* workspace, uint64_t workspace_bytes,
                                                         FTrainStream stream);

/*
 * The router of a mixture of experts.  From logits (tokens x n, T) and an
 * optional mask (tokens, UINT8; null memory: none), with k the columns of
 * `experts` (at most n and 32; n at most 1024):
 *   p = softmax of each row of the logits;
 *   experts (tokens x k, INT32): the k largest logits, largest first, ties to
 *     the lowest index; never minus infinity or NaN, -1 when none is left;
 *   gates (tokens x k, FP32): p of the chosen, over their sum if `normalize`;
 *   slots (tokens x k, INT32): each choice's row when the choices are packed
 *     by expert and, within an expert, in token order; -1 with expert -1;
 *   counts (n, INT32): each expert's choices, the rows of its group;
 *   routed (1, INT32): N, the rows that take part;
 *   balance_loss (1, FP32): n sum_e f_e P_e, f_e = counts_e / sum of counts,
 *     P_e = mean of p_e over the routed rows.
 * A row with mask 0, or with every logit minus infinity, takes no part:
 * experts and slots -1, gates 0.
 */
FTRAIN_API FTrainStatus ftrainMoeRouteWorkspaceBytes(FTrainStorageView logits, uint64_t* workspace_bytes);
FTRAIN_API FTrainStatus ftrainMoeRoute(FTrainStorageView logits, FTrainStorageView mask, FTrainStorageView experts,
                                       FTrainStorageView gates, FTrainStorageView slots, FTrainStorageView counts,
                                       FTrainStorageView routed, FTrainStorageView balance_loss, bool normalize,
                                       void* workspace, uint64_t workspace_bytes, FTrainStream stream);
/*
 * The logits' gradient (shaped and typed as the logits, overwritten; zero in
 * rows that take no part) for grad_gates (tokens x k, FP32) and grad_loss (1,
 * FP32), with the forward call's experts, counts and routed.  The choice, and
 * with it the counts, is a constant of the differentiation.
 */
FTRAIN_API FTrainStatus ftrainMoeRouteBackward(FTrainStorageView grad_gates, FTrainStorageView grad_loss,
                                               FTrainStorageView logits, FTrainStorageView mask,
                                               FTrainStorageView experts, FTrainStorageView counts,
                                               FTrainStorageView routed, FTrainStorageView grad_logits, bool normalize,
                                               FTrainStream stream);

/*
 * norm (1, FP32) = sqrt of the sum of squares over all of `grads` (any rank,
 * CONTINUOUS, T each its own), and
 *   outputs[i] = grads[i] * min(1, max_norm / (norm + eps)).
 * outputs null: in place (no gradient is written when the factor is 1).  An
 * infinite or NaN gradient makes the norm infinite or NaN and, by the
 * formula, gradients zero or NaN.
 */
FTRAIN_API FTrainStatus ftrainClipGradNormWorkspaceBytes(uint64_t* workspace_bytes);
FTRAIN_API FTrainStatus ftrainClipGradNorm(const FTrainStorageView grads[], const FTrainStorageView outputs[],
                                           uint32_t num_grads, FTrainStorageView norm, float max_norm, float eps,
                                           void* workspace, uint64_t workspace_bytes, FTrainStream stream);

#ifdef __cplusplus
}
#endif

#endif
