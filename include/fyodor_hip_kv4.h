/* C ABI of libfyodor_hip.so, third part: the paged KV cache of
 * fyodor_hip_serving.h in 4 bits per value, for a program that serves more or
 * longer requests than 8 bits have memory for. Page tables, slots and rotary
 * angles are those of nya_hip_page_step and nya_hip_rope_angles; of a step's
 * calls nya_hip_kv4_store and nya_hip_kv4_attention take the place of the 8-bit
 * ones. Conventions, limits of sizes and what is declined are as there.
 *
 * The reference has no counterpart: its providers keep one sequence per plan,
 * in fp32 (CUDA/resident.inc:466-578). */
#ifndef FYODOR_HIP_KV4_H
#define FYODOR_HIP_KV4_H
#include "fyodor_hip_serving.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Each position has the blocks of 32 elements that GGUF's Q4_0 has: 4-bit codes
 * n and a step d, value = (n - 8) d. The step is that of the block's element m
 * of the largest magnitude (of -m and m: -m), d = m / -8, rounded to 8 bits
 * (ties to even), its magnitude at most 8160, then to fp16;
 * n = round(x / d) + 8 (ties to even) within 0 .. 15, and 8 where d is 0. So
 * an element is off by up to half a step, a sixteenth of |m|, and on m's other
 * side, where 7 |d| is the most there is, by up to 33/32 of one, an eighth of |m|.
 * Magnitudes from 65280 on are held as that on m's side, as 57120 on the other.
 * In blocks below 2^-14 the step is an fp16 number of fewer bits, which adds up to
 * 2^-22 to both; those whose m is no more than 2^-22 (in 8 bits) are zeros.
 * With 8 bits in the step (n - 8) d is an fp16 number: what attention multiplies
 * is exactly what is held. No position changes when another one is stored, so rows
 * may come in any order.
 *
 * Heads of 64, 128, 256 or 512. The codes of a page and head, page_tokens *
 * width / 2 bytes at (page * kv_heads + head) times that, are laid out for the
 * attention's loads. Element d of position t is 4 bits (the low half of a byte
 * first):
 *     of a key,   nibble d % 2 * 4 + d % 8 / 2 of the 4-byte word
 *                 (d / 32 * page_tokens + t) * 4 + d % 32 / 8,
 *     of a value, nibble d % 4 of the 2-byte word
 *                 (t / 8 * (width / 4) + d / 4) * 8 + t % 8.
 * Steps: fp16, page_tokens * width / 32 of a page and head, block b of
 * position t
 *     of a key   at (t / 16 * (width / 32) + b) * 16 + t % 4 * 4 + t % 16 / 4,
 *     of a value at b * page_tokens + t.
 * Codes and steps 16-byte aligned. Nothing needs to be cleared: only positions
 * that were stored are read. */
typedef struct nya_hip_kv4 {
    uintptr_t keys, values;             /* nya_hip_kv4_bytes' *codes each */
    uintptr_t key_steps, value_steps;   /* *steps each */
    size_t pages, page_tokens, kv_heads, width;
} nya_hip_kv4;

/* Bytes of one of the code arrays and of one of the step arrays; 1 for
 * geometries that the cache does not have (nya_hip_kv8_bytes'). The addresses
 * in `cache` are not looked at. */
NYA_HIP_EXPORT int nya_hip_kv4_bytes(const nya_hip_kv4 *cache, size_t *codes, size_t *steps);

/* `count` rows of k and v (kv_heads heads of width, strides in floats) into
 * the cache slots slots[i] (outside the cache: the row is left out), k rotated
 * by angles as nya_hip_rope does (angles = 0: as it is); with q, the q rows are
 * rotated into q_out as well (all `count` of them; q_out may be q with the same
 * stride, and does not overlap k or v), one launch for both; q without
 * angles is declined. Rows in any order, no slot twice. What is held is formed from
 * fp32 values (rotated ones rounded once). If a head's k or v of a row has an
 * infinite or NaN element, that head's position reads as NaN, k and v, until
 * its slot is stored anew (a NaN step of the keys marks it). */
NYA_HIP_EXPORT int nya_hip_kv4_store(const nya_hip_kv4 *cache, uintptr_t slots, size_t count, uintptr_t k,
    size_t k_stride, uintptr_t v, size_t v_stride, uintptr_t angles, size_t rotated, unsigned layout, uintptr_t q,
    size_t q_stride, uintptr_t q_out, size_t q_out_stride, size_t heads, uintptr_t stream);

/* The rows of `count` slots back as fp32, exactly what is held; rows of slots
 * outside the cache are left as they are. */
NYA_HIP_EXPORT int nya_hip_kv4_load(const nya_hip_kv4 *cache, uintptr_t slots, size_t count, uintptr_t k,
    size_t k_stride, uintptr_t v, size_t v_stride, uintptr_t stream);

/* Causal attention of the step's rows over their requests' pages: the
 * arguments, the rows, the positions they see and what is left alone are
 * nya_hip_kv8_attention's, and so is the workspace. q (and the softmax's
 * weights) enter the matrix cores as two fp16 pieces, 22 bits each, keys and
 * values exactly; all sums are fp32. A row that sees a position that reads as
 * NaN is NaN. A score above 2^128 / log2(e) (2.3e38), or nothing but scores
 * below minus that, gives NaN. The same call gives the same bits. */
NYA_HIP_EXPORT int nya_hip_kv4_attention_bytes(const nya_hip_kv4 *cache, size_t count, size_t requests,
    size_t max_tokens, size_t max_length, size_t heads, size_t window, size_t *bytes);
NYA_HIP_EXPORT int nya_hip_kv4_attention(const nya_hip_kv4 *cache, uintptr_t q, size_t q_stride, uintptr_t out,
    size_t out_stride, size_t count, uintptr_t starts, uintptr_t lengths, uintptr_t table, size_t table_stride,
    size_t requests, size_t max_tokens, size_t max_length, size_t heads, size_t window, float scale,
    uintptr_t workspace, size_t workspace_bytes, uintptr_t stream);

#ifdef __cplusplus
}
#endif
#endif
