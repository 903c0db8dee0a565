/* C ABI of libfyodor_hip.so, second part: what a program needs that serves
 * many requests at once over one KV cache. The cache is in pages and holds 8
 * bits per value; a step brings new tokens of some of the requests.
 *
 * One step, everything on the device and on one stream, so that the whole
 * step can be captured into a graph and replayed:
 *     nya_hip_page_step      pages, rows, positions and cache slots of the
 *                            step's tokens from the requests' lengths;
 *     nya_hip_rope_angles    (cos, sin) of those positions, once per step;
 *   and for every layer
 *     nya_hip_kv8_store      q and k rotated, k and v into the cache;
 *     nya_hip_kv8_attention  every row over its request's pages.
 *
 * The conventions are those of fyodor_hip.h: device addresses and the stream
 * as uintptr_t, owned by the caller; nothing is allocated, freed or waited
 * for; 0 enqueued (or answered), 1 declined before anything was enqueued, <0
 * a HIP failure. Vectors are fp32 device arrays, 4-byte aligned; 16-byte
 * aligned rows whose strides are multiples of 4 load and store faster.
 * Integers on the device (lengths, counts, tables, slots, positions) are
 * int32. A step has at most 2^22 rows (tokens), a row at most 2^22 floats;
 * count * kv_heads <= 2^25 where rows are stored or loaded; in attention
 * count * heads <= 2^27, requests <= 65535 and requests * kv_heads <= 2^21.
 * The integers are data of the step that no call can check beforehand:
 * an entry outside its range is taken as "nothing there", never followed.
 *
 * The reference has no counterpart: its providers keep one sequence per
 * plan, its cache one row per position ([capacity][kv_heads * width],
 * CUDA/resident.inc:466-578). */
#ifndef FYODOR_HIP_SERVING_H
#define FYODOR_HIP_SERVING_H
#include "fyodor_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- pages ---------------------------------------------------------------
 *
 * A page holds page_tokens positions of one request (16, 32, 64 or 128).
 * table[r * table_stride + j] is the page of positions [j page_tokens,
 * (j + 1) page_tokens) of request r, -1 where it has none; held[r] counts
 * its pages. free_pages[0 .. free_count[0]) is the stack of pages that no
 * request holds (room for `pages`, the cache's).
 *
 * lengths[r]: the positions that request r shall hold after this step;
 * counts[r]: how many of them are new, the last ones (0: the request brings
 * nothing). The step
 *   1. puts the pages past ceil(lengths[r] / page_tokens) back on the stack
 *      (a finished request: length 0; rejected drafts: a shorter one), in
 *      the order of the requests and of their pages, their entries -1;
 *   2. gives the requests that need more pages theirs from the stack's top,
 *      in the order of the requests. A request is served if what it and all
 *      before it need is there, else it keeps the pages it has;
 *      free_count[1] says how many were not served (lengths beyond
 *      table_stride pages among them, which count as needing none);
 *   3. numbers the step's rows: request r has rows starts[r] .. starts[r + 1)
 *      (starts: requests + 1 of them), row starts[r] + j is position
 *      p = lengths[r] - counts[r] + j, in slot
 *      table[r][p / page_tokens] * page_tokens + p % page_tokens of the
 *      cache, or -1 where the request holds no such page. Rows from
 *      starts[requests] to max_tokens: position -1, slot -1 (a batch padded
 *      for a captured graph). Rows past max_tokens are cut off, a request's
 *      last ones: they have a place in `starts` (starts[requests] >
 *      max_tokens says so; it ends at INT_MAX) but no position and slot, and
 *      the others keep theirs, here and in attention.
 * Negative lengths and counts are taken as 0. Run again with the same
 * lengths it changes nothing. requests <= 65536, and
 * requests * table_stride, table_stride * page_tokens and
 * pages * page_tokens <= INT_MAX. */
NYA_HIP_EXPORT int nya_hip_page_step(uintptr_t lengths, uintptr_t counts, size_t requests, size_t page_tokens,
    uintptr_t table, size_t table_stride, uintptr_t held, uintptr_t free_pages, size_t pages, uintptr_t free_count,
    uintptr_t starts, uintptr_t positions, uintptr_t slots, size_t max_tokens, uintptr_t stream);

/* ---- rotary positions ----------------------------------------------------
 *
 * Of a head of `width` the first `rotated` elements (even) turn in pairs:
 * pair j by the angle p * f_j, as INTERLEAVED pairs (2j, 2j + 1) or as
 * HALVES (j, j + rotated / 2); the others stay. */
enum { NYA_HIP_ROPE_INTERLEAVED = 0, NYA_HIP_ROPE_HALVES = 1 };

/* How frequencies are changed for contexts longer than `original` positions,
 * the ones a model was trained on, by `factor` (>= 1):
 *   NONE    f_j = base^(-2j / rotated);
 *   LINEAR  f_j / factor;
 *   BANDS   g f_j + (1 - g) f_j / factor, with g from 0 to 1 as pair j's
 *           turns within `original`, original * f_j / 2 pi, go from `low` to
 *           `high` (0 <= low < high);
 *   RAMP    the same with g going linearly in j instead, from 1 at the
 *           (rounded down) pair that turns `high` times to 0 at the (rounded
 *           up) one that turns `low` (> 0) times, and *magnitude =
 *           1 + 0.1 ln(factor).
 * *magnitude, which multiplies (cos, sin), is 1 otherwise. factors (or
 * null): rotated / 2 floats, finite and not 0, that divide the base
 * frequencies first, a model's own rope factors. On the host: `out` receives rotated / 2 floats,
 * each the 64-bit result rounded once. */
enum { NYA_HIP_ROPE_NONE = 0, NYA_HIP_ROPE_LINEAR = 1, NYA_HIP_ROPE_BANDS = 2, NYA_HIP_ROPE_RAMP = 3 };
NYA_HIP_EXPORT int nya_hip_rope_frequencies(float *out, size_t rotated, double base, const float *factors,
    unsigned scaling, double factor, double original, double low, double high, float *magnitude);

/* angles[i][j] = (cos, sin)(positions[i] * frequencies[j]) * magnitude for
 * `count` positions and rotated / 2 (at most 512) frequencies: the
 * table (8-byte aligned) that every layer of a step reads. Formed in 64 bits
 * and rounded once; the phase is right to p f 2^-51 (2^-27 at position 2^24,
 * 2^-20 at the last one). */
NYA_HIP_EXPORT int nya_hip_rope_angles(uintptr_t positions, size_t count, uintptr_t frequencies, size_t rotated,
    float magnitude, uintptr_t angles, uintptr_t stream);

/* The rotary step of `count` rows of q (`heads` heads of `width`) and of k
 * (kv_heads heads; k = 0: none) by angles ([count][rotated / 2] pairs as
 * above): q_out and k_out receive the whole rows, and may be q and k
 * themselves with the same stride, but not overlap them or each other
 * otherwise. Strides in floats. */
NYA_HIP_EXPORT int nya_hip_rope(uintptr_t q, size_t q_stride, uintptr_t q_out, size_t q_out_stride, size_t heads,
    uintptr_t k, size_t k_stride, uintptr_t k_out, size_t k_out_stride, size_t kv_heads, size_t width, size_t count,
    uintptr_t angles, size_t rotated, unsigned layout, uintptr_t stream);

/* ---- the 8-bit cache -----------------------------------------------------
 *
 * Keys and values as int8 codes in [-127, 127] with one fp32 scale per page
 * and head, K and V apart: value = code * scale. For heads of 64, 128, 256
 * or 512. Codes of a page and head, page_tokens * width bytes at
 * (page * kv_heads + head) * page_tokens * width, are laid out for the
 * attention's loads: element d of position t
 *     of a key at    (d / 16 * page_tokens + t) * 16 + d % 16,
 *     of a value at  (t / 16 * width + d) * 16 + t % 16.
 * Scales at page * kv_heads + head; a page's, once its first position is
 * stored, is from 2^-100 to FLT_MAX / 127, infinite or NaN. Codes 16-byte
 * aligned. Nothing needs to be cleared: a page's scale begins with its first
 * position. */
typedef struct nya_hip_kv8 {
    uintptr_t keys, values;               /* nya_hip_kv8_bytes' *codes each */
    uintptr_t key_scales, value_scales;   /* *scales each */
    size_t pages, page_tokens, kv_heads, width;
} nya_hip_kv8;

/* Bytes of one of the code arrays and of one of the scale arrays; 1 for
 * geometries that the cache does not have (widths and page sizes as above,
 * kv_heads <= 16384, pages * page_tokens and pages * kv_heads <= INT_MAX). The
 * addresses in `cache` are not looked at. */
NYA_HIP_EXPORT int nya_hip_kv8_bytes(const nya_hip_kv8 *cache, size_t *codes, size_t *scales);

/* `count` rows of k and v (kv_heads heads of width, strides in floats) into
 * the cache slots slots[i] (as nya_hip_page_step numbers them; outside the
 * cache: the row is left out), k rotated by angles as nya_hip_rope does
 * (angles = 0: as it is); with q, the q rows are rotated into q_out as well
 * (all `count` of them; q_out may be q with the same stride, and does not
 * overlap k or v), one launch for both; q without angles is declined.
 *
 * Rows of one page stand together, in the order of their positions, and no
 * slot twice; between two of them fewer than 128 rows may stand that are left
 * out. Positions that follow each other in rows that do are a run; a page's
 * runs are taken in their order. A run takes wanted = max|x| * (1 / 127) (in
 * fp32, at least 2^-100) of its rows in a head. A run from the page's first slot sets the
 * scale to that; a later one raises it to that if it is lower, and the
 * page's codes are rounded again to the new step, code = round(code * old /
 * new). Codes are round(x / scale), exactly (ties to even), of fp32 values
 * (rotated ones rounded once). Infinite or NaN elements make the scale so,
 * and the page's head reads as NaN until its first slot is stored anew. */
NYA_HIP_EXPORT int nya_hip_kv8_store(const nya_hip_kv8 *cache, uintptr_t slots, size_t count, uintptr_t k,
    size_t k_stride, uintptr_t v, size_t v_stride, uintptr_t angles, size_t rotated, unsigned layout, uintptr_t q,
    size_t q_stride, uintptr_t q_out, size_t q_out_stride, size_t heads, uintptr_t stream);

/* The rows of `count` slots back as fp32, code * scale; rows of slots outside
 * the cache are left as they are. The counterpart of the plan's reading of
 * its cache (backend/include/compute.h:37-51), for checks, for handing a
 * prefix on, and for paths that take fp32 rows. */
NYA_HIP_EXPORT int nya_hip_kv8_load(const nya_hip_kv8 *cache, uintptr_t slots, size_t count, uintptr_t k,
    size_t k_stride, uintptr_t v, size_t v_stride, uintptr_t stream);

/* Causal attention of the step's rows over their requests' pages: row
 * starts[r] + j of request r, at position p = lengths[r] - (starts[r + 1] -
 * starts[r]) + j, attends positions 0 .. p (window > 0: the last `window` of
 * them) that have a page, head h of `heads` over KV head h / (heads /
 * kv_heads): scores q.k * scale, a softmax, out = sum_t p_t v_t. A row that
 * sees nothing gives zeros; rows outside [starts[0], starts[requests]) stay
 * as they are. `count` rows of q and out there are (starts past it are cut
 * off), at most max_tokens of one request, the rest of whose rows stay as
 * they are. Requests may bring one token, a
 * few (drafts to check) or a prompt, in any mixture. max_length, the longest
 * request the caller expects, only says how finely to split the work; any
 * lengths[r] is attended in full.
 *
 * q (and the softmax's weights) enter the matrix cores as two fp16 pieces,
 * 22 bits each, the codes exactly; all sums are fp32. A score above
 * 2^128 / log2(e) (2.3e38), or nothing but scores below minus that, gives NaN.
 * Positions whose value scale is below 2^-116 of the largest one that a row
 * sees may be missing from its sum of weights. Which kernel and split
 * runs goes by the arguments alone: the same call gives the same bits.
 *
 * `workspace` (16-byte aligned) is scratch for work split over several
 * workgroups (nothing in it is kept, nor has to be cleared): with less than
 * nya_hip_kv8_attention_bytes says, or none, the call runs with fewer of
 * them, and slower; both calls with the same arguments. Calls that may overlap in time
 * need workspaces of their own. out must not overlap q. */
NYA_HIP_EXPORT int nya_hip_kv8_attention_bytes(const nya_hip_kv8 *cache, size_t count, size_t requests,
    size_t max_tokens, size_t max_length, size_t heads, size_t window, size_t *bytes);
NYA_HIP_EXPORT int nya_hip_kv8_attention(const nya_hip_kv8 *cache, uintptr_t q, size_t q_stride, uintptr_t out,
    size_t out_stride, size_t count, uintptr_t starts, uintptr_t lengths, uintptr_t table, size_t table_stride,
    size_t requests, size_t max_tokens, size_t max_length, size_t heads, size_t window, float scale,
    uintptr_t workspace, size_t workspace_bytes, uintptr_t stream);

#ifdef __cplusplus
}
#endif
#endif
