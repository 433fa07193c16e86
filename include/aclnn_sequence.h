/*
 * aclnn_sequence.h - operators on sequences of tokens: the norm of a residual sum, rotary positions and attention over a sliding
 * window. They serve the blocks that take the resampled images, position tables and features of aclnn_resample.h as their tokens.
 *
 * The protocol is that of aclnn_resample.h: aclnnXxxGetWorkspaceSize validates, plans and returns the workspace's size and an
 * executor (no GPU work), aclnnXxx enqueues the kernels on `stream` and consumes the executor. Workspace is 256-byte aligned
 * device memory that one call uses at a time; calls that may overlap (other streams, captured graphs that run side by side) need
 * one each. Nothing is kept from one call for the next, so calls can be captured into a CUDA graph and replayed.
 *
 * Storage types are ACL_FLOAT, ACL_FLOAT16 and ACL_BF16, the same for all floating tensors of a call where nothing else is said;
 * sums, statistics and exponentials are fp32, and each output is rounded once (WindowAttention says what else it rounds). Views with
 * any strides are taken: the kernels read and write views whose last dimension is contiguous directly, other views go through copies
 * in the workspace (as long as they have at most four dimensions that do not merge). An output's elements must not overlap one
 * another. An output may lie exactly over an input of its type and strides where the operator says so; other overlaps of an output
 * with an input or another output give undefined values.
 */
#ifndef ACLNN_SEQUENCE_H
#define ACLNN_SEQUENCE_H

#include "opscv_acl.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- ResidualRmsNorm -------------------------------------------------------------------------------------------------------
 * sum = x + residual, rounded to the tensors' type; rstd = 1 / sqrt(mean(sum^2) + eps) over the last dimension;
 * y = sum * rstd * weight.
 * x, residual, y, sum: the same shape [..., width], 1 <= width < 2^30. residual may be null (sum is then x; `sum` may be null, and is a
 * copy of x where it is given). weight: [width] of the tensors' type or ACL_FLOAT, or null (ones). eps: taken in fp32, where it has to
 * be finite, and >= 0.
 * sum, rstd ([...], ACL_FLOAT, contiguous): null where they are not wanted; the backward reads both.
 * y may lie over x or residual, and sum over x or residual (each over another one). */
ACLNN_API aclnnStatus aclnnResidualRmsNormGetWorkspaceSize(const aclTensor* x, const aclTensor* residual,
                                                           const aclTensor* weight, double eps, aclTensor* y,
                                                           aclTensor* sum, aclTensor* rstd, uint64_t* workspaceSize,
                                                           aclOpExecutor** executor);
ACLNN_API aclnnStatus aclnnResidualRmsNorm(void* workspace, uint64_t workspaceSize, aclOpExecutor* executor,
                                           aclrtStream stream);

/* The gradients of y = norm(sum) * weight and of sum itself: with u = sum * rstd and g = gradY * weight
 *   gradX = gradSum + rstd * (g - u * mean(g * u)),  gradWeight = the sum over all rows of gradY * u.
 * gradX is the gradient of x and of residual alike. gradSum (the gradient that reaches `sum` by its other use) and weight may be
 * null; gradWeight has weight's type and is null exactly where weight is null or its gradient is not wanted. The sums are formed
 * in a fixed order: equal inputs give equal bits. gradX may lie over gradY, gradSum or sum. */
ACLNN_API aclnnStatus aclnnResidualRmsNormBackwardGetWorkspaceSize(const aclTensor* gradY, const aclTensor* sum,
                                                                   const aclTensor* rstd, const aclTensor* weight,
                                                                   const aclTensor* gradSum, aclTensor* gradX,
                                                                   aclTensor* gradWeight, uint64_t* workspaceSize,
                                                                   aclOpExecutor** executor);
ACLNN_API aclnnStatus aclnnResidualRmsNormBackward(void* workspace, uint64_t workspaceSize, aclOpExecutor* executor,
                                                   aclrtStream stream);

/* The same norm with y in 8 bits: each row (group = 0) or each `group` columns of a row (a multiple of 32; the last group may be
 * shorter) are divided by a scale of their own, max|y| / 448 for out of type ACL_FLOAT8_E4M3FN and max|y| / 127 for ACL_INT8, and
 * rounded to nearest even; y is about out * scale. The division is of the fp32 values, before any rounding of y. A group of zeros
 * (or of magnitudes below 1e-35) has scale 0 and zeros; one that holds a NaN or an infinity has a NaN or infinity as its scale,
 * and its values say nothing.
 * out: x's shape, contiguous. scales: [..., groups], ACL_FLOAT, contiguous, at most 10240 groups. sum: as above, may be null. */
ACLNN_API aclnnStatus aclnnResidualRmsNormQuantGetWorkspaceSize(const aclTensor* x, const aclTensor* residual,
                                                                const aclTensor* weight, double eps, int64_t group,
                                                                aclTensor* out, aclTensor* scales, aclTensor* sum,
                                                                uint64_t* workspaceSize, aclOpExecutor** executor);
ACLNN_API aclnnStatus aclnnResidualRmsNormQuant(void* workspace, uint64_t workspaceSize, aclOpExecutor* executor,
                                                aclrtStream stream);

/* ---- RotaryEmbedding ---------------------------------------------------------------------------------------------------------
 * q: [..., heads, dim], k: [..., kvHeads, dim] with the same leading dimensions, or null. The first rotary = 2 * half values of a
 * head are turned by the angles position * frequencies[i], i < half, and multiplied by `scale` (taken in fp32, where it has to be
 * finite); the others are copied. A token of more than 2^24 values, of q and k together, is refused, and so are more than 2^20 heads
 * or values of a head.
 * Pair i is values (i, half + i), or (2i, 2i + 1) where `interleaved`.
 * frequencies: [half] of ACL_DOUBLE or ACL_FLOAT, contiguous, 1 <= half <= dim / 2 and half <= 2048. The angle is formed in
 * 64 bits.
 * positions: q's leading dimensions, ACL_INT32 or ACL_INT64. Any of these may have stride 0, where one position serves several tokens;
 * the others have any strides, as long as they merge to at most two dimensions (neighbours merge where the outer one's stride is the
 * inner one's times its extent), and to at most four with those of stride 0 between and behind them. With `sections` (at most 4 whole numbers >= 0 that add up to half): [axes, ...], axis a turning the
 * a-th section of the frequencies.
 * qOut may lie over q and kOut over k. */
ACLNN_API aclnnStatus aclnnRotaryEmbeddingGetWorkspaceSize(const aclTensor* q, const aclTensor* k, const aclTensor* positions,
                                                           const aclTensor* frequencies, const aclIntArray* sections,
                                                           bool interleaved, double scale, aclTensor* qOut,
                                                           aclTensor* kOut, uint64_t* workspaceSize,
                                                           aclOpExecutor** executor);
ACLNN_API aclnnStatus aclnnRotaryEmbedding(void* workspace, uint64_t workspaceSize, aclOpExecutor* executor,
                                           aclrtStream stream);

/* The gradient: the same with the negative angles, from the gradients of qOut and kOut to those of q and k. */
ACLNN_API aclnnStatus aclnnRotaryEmbeddingBackwardGetWorkspaceSize(const aclTensor* gradQOut, const aclTensor* gradKOut,
                                                                   const aclTensor* positions,
                                                                   const aclTensor* frequencies,
                                                                   const aclIntArray* sections, bool interleaved,
                                                                   double scale, aclTensor* gradQ, aclTensor* gradK,
                                                                   uint64_t* workspaceSize, aclOpExecutor** executor);
ACLNN_API aclnnStatus aclnnRotaryEmbeddingBackward(void* workspace, uint64_t workspaceSize, aclOpExecutor* executor,
                                                   aclrtStream stream);

/* The frequencies base^(-i / half), i < half, in out ([half], ACL_DOUBLE or ACL_FLOAT, contiguous), computed in 64 bits and scaled
 * for contexts `factor` times as long as the trained one (base > 1, factor >= 1). scaling:
 *   0 none;
 *   1 linear: all divided by factor;
 *   2 base: the base times factor^(half / (half - 1)), which leaves the first frequency and divides the last by factor;
 *   3 wavelength: frequencies that turn `high` times or more within originalLength tokens stay, those that turn `low` times or
 *     less are divided by factor, the ones between are blended by their turns (0 <= low < high);
 *   4 ramp: the same, blended linearly over i between the (real-valued) indices that turn `high` and `low` times, rounded
 *     outwards and cut to [0, 2 half - 1] (0 < low < high).
 * originalLength > 0, low and high are read for scaling 3 and 4 only. */
ACLNN_API aclnnStatus aclnnRotaryFrequenciesGetWorkspaceSize(double base, int64_t scaling, double factor,
                                                             double originalLength, double low, double high,
                                                             aclTensor* out, uint64_t* workspaceSize,
                                                             aclOpExecutor** executor);
ACLNN_API aclnnStatus aclnnRotaryFrequencies(void* workspace, uint64_t workspaceSize, aclOpExecutor* executor,
                                             aclrtStream stream);

/* ---- WindowAttention ---------------------------------------------------------------------------------------------------------
 * Causal attention over a sliding window with a few first tokens ("sinks") that stay visible, for prompts, chunks of new tokens
 * over a cache, single tokens and training.
 * q, out: [batch, queries, heads, dim]; k, v: [batch, keys, kvHeads, dim]; heads a multiple of kvHeads (head h reads key head
 * h / (heads / kvHeads)), at most 2^24 to a key head; 1 <= dim <= 256; batch, queries, keys, heads and batch * heads at most 2^30.
 * kvLengths, qLengths: [batch], ACL_INT32 or ACL_INT64, contiguous, or null (all keys, all queries): how many keys and queries of
 * each sequence count; values outside [0, keys] and [0, queries] are cut to it. Query i of a sequence sits at position
 * p = kvLength - qLength + i, so that the last query sits at the last key; it sees the keys j <= p with j > p - window
 * (window >= 1) or j < sinks (sinks >= 0; both are cut to 2^30). scale multiplies the scores; it is taken in fp32,
 * where it has to be finite.
 * out = softmax(scale q.k over the keys seen) v; lse: [batch, heads, queries], ACL_FLOAT, contiguous, the natural logarithm of the
 * softmax's sum, or null. A query behind its sequence's length, or that sees no key, has out 0 and lse -infinity.
 * What lies in keys that a query does not see, NaN and infinities included, does not reach its result.
 * 16-bit tensors with heads of at most 128 values, whose rows are 16-byte aligned, are multiplied on the tensor cores: each weight is
 * rounded to the tensors' type before its product with v (the softmax's sum is of the weights before that), but for few queries, whose
 * weights are taken in two 16-bit parts. Other tensors keep fp32 throughout. */
ACLNN_API aclnnStatus aclnnWindowAttentionGetWorkspaceSize(const aclTensor* q, const aclTensor* k, const aclTensor* v,
                                                           const aclTensor* qLengths, const aclTensor* kvLengths,
                                                           int64_t window, int64_t sinks, double scale, aclTensor* out,
                                                           aclTensor* lse, uint64_t* workspaceSize,
                                                           aclOpExecutor** executor);
ACLNN_API aclnnStatus aclnnWindowAttention(void* workspace, uint64_t workspaceSize, aclOpExecutor* executor,
                                           aclrtStream stream);

/* The gradients of q, k and v, each of its tensor's shape, from out's, with the out and lse that the forward returned for the
 * same arguments. gradOut . out is formed from `out` as it is stored; on the tensor cores, weights and gradients of the scores are
 * rounded to the tensors' type once each before their products, for few queries too. The gradients of queries behind their sequence's
 * length and of keys that no query sees are 0. The sums are formed in a fixed order: equal inputs give equal bits. No output may lie
 * over an input. */
ACLNN_API aclnnStatus aclnnWindowAttentionBackwardGetWorkspaceSize(const aclTensor* gradOut, const aclTensor* q,
                                                                   const aclTensor* k, const aclTensor* v,
                                                                   const aclTensor* out, const aclTensor* lse,
                                                                   const aclTensor* qLengths, const aclTensor* kvLengths,
                                                                   int64_t window, int64_t sinks, double scale,
                                                                   aclTensor* gradQ, aclTensor* gradK, aclTensor* gradV,
                                                                   uint64_t* workspaceSize, aclOpExecutor** executor);
ACLNN_API aclnnStatus aclnnWindowAttentionBackward(void* workspace, uint64_t workspaceSize, aclOpExecutor* executor,
                                                   aclrtStream stream);

#ifdef __cplusplus
}
#endif
#endif /* ACLNN_SEQUENCE_H */
