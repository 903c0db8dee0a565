/* C ABI of libfyodor_hip.so, fourth part: what a program answers with, or
 * scores a text by, beside the tokens that nya_hip_greedy or a sampler chose.
 * The conventions are those of fyodor_hip.h.
 *
 * The reference has no counterpart beside its sampler
 * (backend/core/llm_cpu.c:896-904). */
#ifndef FYODOR_HIP_LOGPROBS_H
#define FYODOR_HIP_LOGPROBS_H
#include "fyodor_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

#define NYA_HIP_LOGPROBS_TOP 64   /* the most alternatives */

/* Of each of `count` rows of n fp32 logits x (logits + i stride floats), with
 * p_j = e^(scale x_j) / sum_k e^(scale x_k) (scale: 1 / temperature, from
 * 2^-20 to 2^20) over the entries j whose bit in `mask` is clear (uint32 words as
 * nya_hip_greedy's, 0: none masked):
 *   tokens      (or 0) int32 ids: logprobs[i] = ln p of tokens[i], and
 *               ranks[i] (ranks may be 0) how many tokens come before it;
 *   entropies   (or 0) entropies[i] = -sum_j p_j ln p_j;
 *   top         (or 0, at most NYA_HIP_LOGPROBS_TOP) the tokens that come
 *               first, top_ids[i top + k] (int32) with ln p in
 *               top_logprobs[i top + k].
 * Tokens come in the order of their logits, of equal ones the lower id first
 * (so rank 0 is nya_hip_greedy's choice). A token that is masked, or whose logit
 * is minus infinity, is in no order: ln p is minus infinity, its rank -1, and
 * if fewer than `top` others are left the rest of top_ids is -1 with minus
 * infinity. An id outside [0, n) is no token (a padded batch, a prompt's
 * first position): 0 and rank -1, whatever the row holds. A row with a NaN or
 * plus infinity among the entries that are not masked, or with no entry above
 * minus infinity, has no probabilities: NaN, ranks and ids -1.
 *
 * Logits enter as they are; exponentials and their sums are fp32, the
 * logarithm's argument and what follows 64 bits, rounded once. The same
 * call gives the same bits.
 *
 * n <= 2^24, count <= 2^22. Outputs overlap neither each other nor an input.
 * `workspace` (16-byte aligned) is scratch for rows that are split over several
 * workgroups (nothing in it is kept, nor has to be cleared): with less than
 * nya_hip_logprobs_bytes says, or none, the call may run with fewer of them, and
 * slower. What it says is enough for every call of up to `count` rows of n with up
 * to `top` alternatives (few rows are split and many are not, so it is not what a
 * call of `count` rows takes). Calls that may overlap in time need workspaces of
 * their own. */
NYA_HIP_EXPORT int nya_hip_logprobs_bytes(size_t n, size_t count, size_t top, size_t *bytes);
NYA_HIP_EXPORT int nya_hip_logprobs(uintptr_t logits, size_t stride, size_t n, size_t count, uintptr_t mask, float scale,
    uintptr_t tokens, uintptr_t logprobs, uintptr_t ranks, uintptr_t entropies, size_t top, uintptr_t top_ids,
    uintptr_t top_logprobs, uintptr_t workspace, size_t workspace_bytes, uintptr_t stream);

#ifdef __cplusplus
}
#endif
#endif
