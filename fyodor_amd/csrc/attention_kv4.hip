// Causal attention over a paged 4-bit cache (include/fyodor_hip_kv4.h).
//
// For a KV head, its group's heads and the request's new tokens make the rows
// of one product: row i is token i / group, head i % group of the group,
//     s_it = q_i . K_t scale,   out_i = sum_t e^(s_it) V_t / sum_t e^(s_it).
// One pass over the positions, 64 a step: S^T = K Q^T and O^T = V^T P^T on the
// fp16 matrix cores, with the softmax's running maximum and sum (fp32, like S
// and O) per column, so that a column of S^T is already laid out as the operand
// P^T. A code times its step of 8 bits is an fp16 number, so keys and values
// enter exactly; q and P go in as two fp16 pieces each (22 bits, the error of
// fp32 sums of this length; one piece would be 2^-11), which makes two matrix
// instructions of one: half the fp16 rate is this kernel's ceiling. The maximum
// is rounded up to a whole power of two: rescaling by it is exact, and rare.
// From 2^22 on (kFar) the scores are rounded first, and their distances from the
// maximum taken after.
//
// A call of few rows reads each position once, 1.125 W bytes per KV head and
// position, and is bound by that and by the conversion: 13 instructions for a
// word of 8 codes, against 8 for 8 bytes of the 8-bit cache. One of many rows is
// bound by the matrix cores and by the softmax beside them. Hence two kernels, a
// workgroup of 16 rows that converts straight into the operands' lanes (kv4_rows),
// and one of 128 rows that convert each code once, in LDS (kv4_wide). What is
// too few tiles for the chip is split over the positions and joined by a second
// launch (kv4_join), by the rules of the 8-bit cache: the count of shares was
// measured again here (64 requests of 500 to 8192 positions, shares for 1536 to
// 4096 workgroups: 51 to 56 us, least with the 2048 of there).
//
// Measured, 32 heads over 8 of 128 unless said: one token of 65536 positions 19.9 us
// and 3.9 for the join (75 MB, 3.8 TB/s), 64 requests as above 50.8 and 6.0 (186 MB,
// 3.7 TB/s; the loads alone take 45, the arithmetic alone 48), eight requests of 5
// tokens, 32 heads over 4 of 64, 9.6 and 4.8; prompts of 16 heads over 8 of 256 85
// (kv4_wide). A prompt of 1024 tokens at the end of 8192 positions goes by the clock
// that the card's power leaves it, 1.6 to 1.9 GHz: 231 us in a few passes among
// others', 241 to 251 in 200 in a row, 269 to 284 in 20; 905 to 1116 TFLOP/s as issued,
// a library product of 8192^3 in such runs 1080 to 1320.
#include "paged_attention.h"

namespace fy {
namespace {

constexpr int kBlock = 32;   // elements that share a step

// Nibbles of a word's halves as codes from -8 to 7: under the exponent of 1024 the
// low nibble of a half, under that of 64 the high one, is that plus n. (The
// constants are opaque: as literals they would make two instructions of one.)
struct Codes {
    uint32_t low = 0x000F000Fu, high = 0x00F000F0u, low_one = 0x64006400u, high_one = 0x54005400u;
    __device__ __forceinline__ Codes() { asm("" : "+s"(low), "+s"(high), "+v"(low_one), "+v"(high_one)); }
    __device__ __forceinline__ half2 lows(uint32_t w) const
    {
        return __builtin_bit_cast(half2, (w & low) | low_one) - (half2){(_Float16)1032.f, (_Float16)1032.f};
    }
    __device__ __forceinline__ half2 highs(uint32_t w) const
    {
        return __builtin_bit_cast(half2, (w & high) | high_one) - (half2){(_Float16)72.f, (_Float16)72.f};
    }
};

// 8 positions of an element, or 8 elements of a position, by pairs.
union Pairs {
    half8 v;
    half2 p[4];
};

// 8 elements of a key.
__device__ __forceinline__ half8 key_word(const Codes &c, uint32_t w, _Float16 step)
{
    const half2 s = {step, step};
    Pairs u;
    u.p[0] = c.lows(w) * s;
    u.p[1] = c.highs(w) * s;
    u.p[2] = c.lows(w >> 8) * s;
    u.p[3] = c.highs(w >> 8) * s;
    return u.v;
}

// 8 positions of 4 elements of the values: a word of codes, and of steps, has two positions.
__device__ __forceinline__ void value_words(const Codes &c, const uint4 &w, const uint4 &steps, half8 *x)
{
    Pairs u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t n = word_of(w, i);
        const half2 s = __builtin_bit_cast(half2, word_of(steps, i));
        u[0].p[i] = c.lows(n) * s;
        u[1].p[i] = c.highs(n) * s;
        u[2].p[i] = c.lows(n >> 8) * s;
        u[3].p[i] = c.highs(n >> 8) * s;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = u[e].v;
}

// One of x's two pieces: hi (second 0), or lo (-1).
__device__ __forceinline__ half8 piece_f16(const float *x, float second)
{
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    union { half8 v; half2 p[4]; } u;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const f32x2 v = {x[2 * i], x[2 * i + 1]};
        const half2 h = __builtin_convertvector(v, half2);
        const f32x2 r = {__builtin_fmaf((float)h.x, second, v.x), __builtin_fmaf((float)h.y, second, v.y)};
        u.p[i] = __builtin_convertvector(r, half2);
    }
    return u.v;
}

// The value of the lane eight on (of eight back) in a row of 16, part of the addition that uses it.
__device__ __forceinline__ float eight_on(float v)
{
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x128, 0xF, 0xF, true));
}

// Steps of positions from .. limit - 1 of 8, 0 for the others (no row's, past the last or before
// every window): what memory holds there may be NaN, and a weight of 0 would not hide it.
__device__ __forceinline__ uint4 some_steps(const uint4 &s, int from, int limit)
{
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        w[i] = word_of(s, i) & ((from <= 2 * i && limit > 2 * i ? 0xFFFFu : 0u) |
                                (from <= 2 * i + 1 && limit > 2 * i + 1 ? 0xFFFF0000u : 0u));
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// Requests of a few rows: 16 rows per workgroup, whose wavefronts take every
// fourth step of its share of the positions and meet in LDS at the end. Keys
// and values go from memory straight into the operands' lanes: K and V of a
// step are requested as soon as the last step's are used up, pages a step
// before that (two steps ahead: 62 us for the 64 requests' 51). Steps [from, until) of the
// tile's; a `shared` tile's rows go to `to`, `stride` places apart.
//
// kPair, where a tile has at most eight rows: the two pieces of q and of the
// weights are columns of their own, eight apart, so a product is one matrix
// instruction, and half the registers of q let a third wavefront onto a SIMD
// (with conversions free of literals the 64 requests went from 68 to 51 us; four
// wavefronts, which leave no registers for a step ahead, 70).
template <int W, bool kPair>
__device__ __forceinline__ void few_rows(const Kv4Attention &a, int r, const Request &rq, const Range &g, int kvh, int tile,
    int from, int until, bool shared, const Share &to, int stride, float (*ml)[kWaves][kRows], float (*po)[kRows][64 + 4])
{
    // A lane has, of 16 positions of a step, 4 elements x U of the values, and of 4 positions B blocks of
    // the keys (half a block of heads of 64) in J words.
    constexpr int U = W / 64, D = W / 16, B = W < 128 ? 1 : W / 128, J = W / 32, kBlocks = W / kBlock;
    constexpr bool kAhead = W <= 256;   // room for a step's K and V in registers
    const Kv4 &c = a.cache;
    const Codes codes;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, part = lane >> 4;
    const float second = kPair && col & 8 ? -1.f : 0.f;
    const int group = a.heads / c.kv_heads;

    // Rows past the request's last repeat it and are not written.
    const int row = min(kRows * tile + (kPair ? col & 7 : col), rq.rows - 1), token = row / group, head = kvh * group + row % group;
    const int64_t p = rq.first + token;
    const int last = (int)(p < g.highest ? p : g.highest);
    const int first = (int)(a.window && p >= a.window ? (p - a.window < g.highest ? p - a.window + 1 : g.highest + 1) : 0);
    // Positions that all rows see: up to the first row's last, from the last row's first.
    const int64_t p0 = rq.first + kRows * tile / group, p1 = rq.first + min(kRows * tile + kRows - 1, rq.rows - 1) / group;
    const int all_to = (int)(p0 < g.highest ? p0 : g.highest);
    const int all_from = (int)(a.window && p1 >= a.window ? (p1 - a.window < g.highest ? p1 - a.window + 1 : g.highest + 1) : 0);

    const int *table = a.table + (size_t)r * a.table_stride;
    const int shift = 31 - __builtin_clz(c.page_tokens), within = c.page_tokens - 1;
    const int begin = from + wave, stop = until;
    // Lane l reads keys of the granule of 16 positions (l % 16) / 4 of a step and
    // holds scores and values of granule l / 16. Everything is read
    // unconditionally (positions past these steps' lead to page 0).
    const int most = min(g.highest, kStep * stop - 1);
    auto entry_of = [&](int at) {
        const int entry = table[min(at >> shift, a.table_stride - 1)];
        return at <= most ? entry : -1;
    };
    // A page's codes and steps of this head: whole pages of 32 bits of bytes from the first one's.
    const unsigned plane = c.page_tokens * (W / 2), steps = c.page_tokens * kBlocks;
    const unsigned page_codes = c.kv_heads * plane, page_steps = 2 * c.kv_heads * steps;
    const uint8_t *keys = c.keys + (size_t)kvh * plane, *values = c.values + (size_t)kvh * plane;
    const uint8_t *key_steps = (const uint8_t *)(c.key_steps + (size_t)kvh * steps),
                  *value_step = (const uint8_t *)(c.value_steps + (size_t)kvh * steps);
    auto page_of = [&](int page) { return (unsigned)page < (unsigned)c.pages ? (unsigned)page : 0u; };
    // (Half a block each of two lanes in heads of 64.)
    const int block = W == 64 ? part >> 1 : part;
    typedef uint32_t words __attribute__((ext_vector_type(W == 64 ? 2 : 4)));
    typedef _Float16 half4 __attribute__((ext_vector_type(4)));
    words kr[4][B];
    half4 ks[B];
    uint4 vr[2][U], vs[2][U];
    int kpage, vpage;
    bool there;
    const uint8_t *vb;
    const uint16_t *wb;
    auto look = [&](int step) {
        kpage = entry_of(kStep * step + 16 * (col >> 2));
        vpage = entry_of(kStep * step + 16 * part);
    };
    auto fetch_k = [&](int step) {
        const int at = kStep * step + 16 * (col >> 2);
        const unsigned page = page_of(kpage);
        const uint8_t *kb = keys + (uint64_t)page * page_codes + (block * c.page_tokens + (at & within) + (col & 3)) * 16 +
                            (W == 64 ? 8 * (part & 1) : 0);
        const uint16_t *sb = (const uint16_t *)(key_steps + (uint64_t)page * page_steps) +
                             (((at & within) >> 4) * kBlocks + block) * 16 + 4 * (col & 3);
#pragma unroll
        for (int b = 0; b < B; ++b) {
            ks[b] = *(const half4 *)(sb + 64 * b);
#pragma unroll
            for (int t = 0; t < 4; ++t) kr[t][b] = *(const words *)(kb + (size_t)64 * c.page_tokens * b + 64 * t);
        }
    };
    auto value_codes = [&](int n, int u) { return *(const uint4 *)(vb + ((W / 4) * n + 16 * u) * 16); };
    auto value_steps = [&](int n, int u) { return *(const uint4 *)(wb + 2 * u * c.page_tokens + 8 * n); };
    auto fetch_v = [&](int step) {
        const int at = kStep * step + 16 * part;
        const unsigned page = page_of(vpage);
        vb = values + (uint64_t)page * page_codes + (((at & within) >> 3) * (W / 4) + col) * 16;
        wb = (const uint16_t *)(value_step + (uint64_t)page * page_steps) + (col >> 3) * c.page_tokens + (at & within);
        there = (unsigned)vpage < (unsigned)c.pages;
        if constexpr (kAhead) {
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    vr[n][u] = value_codes(n, u);
                    vs[n][u] = value_steps(n, u);
                }
        }
    };
    look(begin);

    // The row's q in two pieces, scaled by a power of two; the scale's sign goes with it. Word j's
    // elements are 8 j.. of a lane's block (of its half block).
    half8 qh[J], ql[kPair ? 1 : J];
    float qscale;
    {
        const float *q = a.q + (rq.begin + token) * a.q_stride + (int64_t)head * W + (W == 64 ? 16 : kBlock) * part;
        auto place_in = [](int i) { return W == 64 ? 4 * i : 128 * (i / 8) + 4 * (i % 8); };
        float v[8 * J];
        if (((uintptr_t)a.q & 15) == 0 && a.q_stride % 4 == 0) {
#pragma unroll
            for (int i = 0; i < 2 * J; ++i) *(float4 *)(v + 4 * i) = *(const float4 *)(q + place_in(i));
        } else {
#pragma unroll
            for (int i = 0; i < 2 * J; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) v[4 * i + e] = q[place_in(i) + e];
        }
        if constexpr (kAhead) {
            fetch_k(begin);
            fetch_v(begin);
            look(begin + kWaves);
        }
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < 8 * J; ++i) top = fmaxf(top, fabsf(v[i]));
        const int e = 14 - __builtin_amdgcn_frexp_expf(column_max(top));
#pragma unroll
        for (int i = 0; i < 8 * J; ++i) v[i] = ldexpf(a.scale < 0.f ? -v[i] : v[i], e);
#pragma unroll
        for (int j = 0; j < J; ++j) {
            if constexpr (kPair) qh[j] = piece_f16(v + 8 * j, second);
            else split_f16(v + 8 * j, qh[j], ql[j]);
        }
        // exp(s) = exp2(s log2 e), q back to its size; above 0, so that it keeps minus infinity.
        qscale = fmaxf(ldexpf(fabsf(a.scale) * 1.44269504f, -e), 0x1p-126f);
    }

    f32x4 O[D];
#pragma unroll
    for (int d = 0; d < D; ++d) O[d] = (f32x4){0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;
    bool far = false;
    uint64_t saw = 0;   // lanes that had a score
    for (int step = begin; step < stop; step += kWaves) {
        if constexpr (!kAhead) {
            fetch_k(step);
            fetch_v(step);
            look(step + kWaves);
        }
        f32x4 S[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) S[t] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < J; ++j) {
            half8 k[4];
#pragma unroll
            for (int t = 0; t < 4; ++t) k[t] = key_word(codes, kr[t][j / 4][j % 4], ks[j / 4][t]);
#pragma unroll
            for (int t = 0; t < 4; ++t) S[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[t], qh[j], S[t], 0, 0, 0);
            if constexpr (!kPair) {
#pragma unroll
                for (int t = 0; t < 4; ++t) S[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[t], ql[j], S[t], 0, 0, 0);
            }
        }
        if constexpr (kPair) {
            // The other piece's score is eight columns on.
#pragma unroll
            for (int i = 0; i < 16; ++i) S[i >> 2][i & 3] += eight_on(S[i >> 2][i & 3]);
        }
        if constexpr (kAhead) fetch_k(step + kWaves);
        const int at = kStep * step, pos = at + 16 * part;
        int low = 0, limit = 16;   // the tile's positions of these 16
        if (all_from > at || all_to < at + kStep - 1 || __builtin_amdgcn_ballot_w64(!there)) {
            const int from = there ? max(first - pos, 0) : 16, to = min(last - pos, 15);
#pragma unroll
            for (int i = 0; i < 16; ++i) S[i >> 2][i & 3] = i >= from && i <= to ? S[i >> 2][i & 3] : -INFINITY;
            low = g.lowest - pos;
            limit = there ? min(g.highest - pos + 1, 16) : 0;
            if constexpr (kAhead) {
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int u = 0; u < U; ++u) vs[n][u] = some_steps(vs[n][u], low - 8 * n, limit - 8 * n);
            }
        }
        float best = S[0][0];
#pragma unroll
        for (int i = 1; i < 16; ++i) best = fmaxf(best, S[i >> 2][i & 3]);
        saw |= __builtin_amdgcn_ballot_w64(best > -INFINITY);
        const float top = best * qscale;
        if (__builtin_amdgcn_ballot_w64(top > m)) {
            const float next = fmaxf(m, ceilf(column_max(top)));
            const float alpha = __builtin_amdgcn_exp2f(m - (next == -INFINITY ? 0.f : next));
            m = next;
            l *= alpha;
#pragma unroll
            for (int d = 0; d < D; ++d) O[d] *= alpha;
            far = __builtin_amdgcn_ballot_w64(is_far(m));
        }
        const float base = m == -INFINITY ? 0.f : m;
        float scale = qscale, add = 15.f - base;
        if (far) {
#pragma clang fp contract(off)
#pragma unroll
            for (int i = 0; i < 16; ++i) S[i >> 2][i & 3] = S[i >> 2][i & 3] * qscale - base;
            scale = 1.f;
            add = 15.f;
        }
        half8 ph[2], pl[kPair ? 1 : 2];
        float sum[2] = {0.f, 0.f};
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            float w[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                w[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(S[2 * n + (i >> 2)][i & 3], scale, add));
                sum[i & 1] += w[i];
            }
            if constexpr (kPair) ph[n] = piece_f16(w, second);
            else split_f16(w, ph[n], pl[n]);
        }
        l += sum[0] + sum[1];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                half8 v[4];
                if constexpr (kAhead) value_words(codes, vr[n][u], vs[n][u], v);
                else value_words(codes, value_codes(n, u), some_steps(value_steps(n, u), low - 8 * n, limit - 8 * n), v);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    O[4 * u + e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[e], ph[n], O[4 * u + e], 0, 0, 0);
                if constexpr (!kPair) {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        O[4 * u + e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[e], pl[n], O[4 * u + e], 0, 0, 0);
                }
            }
        if constexpr (kAhead) {
            fetch_v(step + kWaves);
            look(step + 2 * kWaves);
        }
    }
    l = column_sum(l);
    if (m == -INFINITY && (saw >> col & 0x0001000100010001u)) m = -FLT_MAX;   // scores, none in fp32

    // The wavefronts' partial softmaxes meet in LDS, 64 columns at a time. (The thread's number is opaque: what
    // follows from it would be formed before the loops and live through them.)
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));
    const int my_wave = tid >> 6, my_col = tid & 15, my_part = tid >> 4 & 3;
    if (my_part == 0) {
        ml[0][my_wave][my_col] = m;
        ml[1][my_wave][my_col] = l;
    }
    const int mrow = tid >> 4, mcol = 4 * my_col;   // this thread's output: 4 columns of a row
    const int out_row = kRows * tile + mrow;
    const bool aligned = ((uintptr_t)a.out & 15) == 0 && a.out_stride % 4 == 0;
#pragma unroll
    for (int i = 0; i < U; ++i) {
        if (i) __syncthreads();
        // Row 4 part + k of tile 4 i + e is element 64 i + 16 part + 4 k + e.
#pragma unroll
        for (int k = 0; k < 4; ++k)
            *(f32x4 *)&po[my_wave][my_col][16 * my_part + 4 * k] =
                (f32x4){O[4 * i][k], O[4 * i + 1][k], O[4 * i + 2][k], O[4 * i + 3][k]};
        __syncthreads();
        float top = -INFINITY, total = 0.f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) top = fmaxf(top, ml[0][w][mrow]);
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
        const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float f = __builtin_amdgcn_exp2f(ml[0][w][mrow] - base);
            total += ml[1][w][mrow] * f;
            o += *(const f32x4 *)&po[w][mrow][mcol] * f;
            if constexpr (kPair) o += *(const f32x4 *)&po[w][mrow ^ 8][mcol] * f;
        }
        if (out_row < rq.rows && (!kPair || mrow < 8)) {
            if (shared) {
                *(f32x4 *)(to.o + (size_t)mrow * stride * W + 64 * i + mcol) = o;
                if (i == 0 && mcol == 0) to.ml[mrow * stride] = make_float2(top, total);
            } else {
                float *out = a.out + (rq.begin + out_row / group) * a.out_stride +
                             (int64_t)(kvh * group + out_row % group) * W + 64 * i + mcol;
                const float inverse = inverse_of(total, top);
                o = o * inverse;
                if (aligned) {
                    *(f32x4 *)out = o;
                } else {
#pragma unroll
                    for (int k = 0; k < 4; ++k) out[k] = o[k];
                }
            }
        }
    }
}

// Wavefronts of few rows on a SIMD, and so their workgroups on a CU: what their registers leave.
constexpr int waves_of(int width, bool pair)
{
    return width == 64 ? (pair ? 4 : 3) : width == 128 ? (pair ? 3 : 2) : 1;
}

template <int W, bool kPair>
__global__ __launch_bounds__(64 * kWaves, waves_of(W, kPair)) void kv4_rows(Kv4Attention a, Split split, int most_rows)
{
    __shared__ float ml[2][kWaves][kRows];
    __shared__ __align__(16) float po[kWaves][kRows][64 + 4];
    const int kv_heads = a.cache.kv_heads, kvh = blockIdx.x % kv_heads;
    TileOf at = {(int)blockIdx.y, (int)(blockIdx.x / kv_heads)};
    int place = at.request, sp = split.most - 1 - (int)blockIdx.z;
    if (split.packed) {
        const ItemOf it = item_of(a, split, most_rows, at.tile);
        if (it.request < 0) return;
        at = {it.request, it.item.tile};
        place = it.request;
        sp = it.item.share;
    }
    if constexpr (W > 256) {   // every request runs here, prompts too
        if (split.listed) {
            place = at.tile;
            at = tile_of<kRows>(a, 0, place);
            if (at.request < 0) return;
        }
    }
    const Request rq = request_of(a, at.request);
    if (kRows * at.tile >= rq.rows || rq.rows > most_rows) return;
    const Range g = range_of(a, rq, at.tile, kRows, split.most, split.least);
    if (sp >= g.active) return;
    const Share to = split.share(kv_heads, place, kvh, split.listed ? 0 : kRows * at.tile, sp, W);
    few_rows<W, kPair>(a, at.request, rq, g, kvh, at.tile, g.from(sp), g.until(sp), g.active > 1, to, split.most, ml, po);
}

// Many rows of one request: 32 per wavefront, 128 per group of four
// wavefronts, which share every step's keys and values, converted to fp16 in
// LDS once. KS groups take every KS-th step of the same rows and meet at the
// end. Two groups run half a step apart: while one is in its MFMAs (last
// step's outputs, this step's scores) the other does its softmax and stages
// its next codes, so that the matrix cores of a SIMD always have one of its two
// wavefronts. Heads of 256 fill the registers with one group (q and the outputs are
// 256 of them; 16 rows per wavefront and two groups read LDS twice as often, 136 us
// for 110), which runs its conversions and weights under its own MFMAs: prompts of up
// to 700 tokens, 16 heads over 8, 85 us (110 with everything in turn; operands
// requested a tile ahead 104, the codes under the scores 100, the weights under the
// outputs 94, rows out whole 85). Of the 85 tables take 3, q 5 (32 MB that all CUs
// read at once), 18 steps 68, their last outputs and the rows 6. A step is 7900
// cycles: the scores 2930 and the outputs 2190, whose MFMAs are 2050 each, codes that
// are waited for and masked 630, the next ones' addresses 580, the maximum 730,
// rescaling 510, sums and the barrier 310.
template <int W, int KS>
__global__ __launch_bounds__(256 * KS) __attribute__((amdgpu_waves_per_eu(KS, KS)))
void kv4_wide(Kv4Attention a, Split split, int most_rows)
{
    constexpr int M = W / 16;       // MFMA steps of a score
    constexpr int D = W / 32;       // output tiles
    constexpr int N = W < 128 ? 1 : W / 128;   // 16-byte pieces of K, and of V, per thread and step
    constexpr int kBlocks = W / kBlock, kBytes = 2 * kStep * W;
    constexpr int kQuads = W / 4;   // pieces of V per 8 positions
    constexpr int kBuffers = KS == 1 ? 2 : 1;
    __shared__ __align__(16) uint8_t smem[KS][2 * kBuffers][kBytes];   // [group][K's, V's]
    __shared__ int theres[KS][2][4];                        // whether 16 positions have a page
    __shared__ float2 smem_ml[4][32];
    const Kv4 &c = a.cache;
    const Codes codes;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((threadIdx.x >> 6) & 3);
    const int ks = KS == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 8), tid = threadIdx.x & 255;
    const int col = lane & 31, h = lane >> 5;
    const int group = a.heads / c.kv_heads;
    int x = blockIdx.x;
    const int kvh = x % c.kv_heads;
    x /= c.kv_heads;
    const int tiles = gridDim.x / (c.kv_heads * split.most), sp = split.most - 1 - x / tiles;
    const TileOf at_tile = tile_of<kWideRows>(a, most_rows, x % tiles);
    const int r = at_tile.request, tile = at_tile.tile;
    if (r < 0) return;
    const Request rq = request_of(a, r);
    const Range g = range_of(a, rq, tile, kWideRows, split.most, split.least);
    if (sp >= g.active) return;

    const int row = kWideRows * tile + 32 * wave + col, row_in = min(row, rq.rows - 1), token = row_in / group;
    const int head = kvh * group + row_in % group;
    const int64_t p = rq.first + token;
    // (Rows past the request's last repeat it and are not written.)
    const int last = (int)(p < g.highest ? p : g.highest);
    const int first = (int)(a.window && p >= a.window ? (p - a.window < g.highest ? p - a.window + 1 : g.highest + 1) : 0);
    // Positions that all of the wavefront's rows see.
    int all_from = first, all_to = last;
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        all_from = max(all_from, __shfl_xor(all_from, o, 64));
        all_to = min(all_to, __shfl_xor(all_to, o, 64));
    }
    all_from = __builtin_amdgcn_readfirstlane(all_from);
    all_to = __builtin_amdgcn_readfirstlane(all_to);

    const int *table = a.table + (size_t)r * a.table_stride;
    const int shift = 31 - __builtin_clz(c.page_tokens), within = c.page_tokens - 1;
    // This group's steps: begin, begin + KS, ...
    const int begin = g.from(sp) + ks, stop = g.until(sp);
    const int rounds = (stop - (begin - ks) + KS - 1) / KS;   // the same for every group
    // Table entries are read a round before the codes they lead to, and
    // everything unconditionally (positions past the last one lead to page 0):
    // loads under a condition would be waited for where it ends.
    const int until = min(g.highest, kStep * stop - 1);   // this workgroup's last position
    // (What is past `until` is told where an entry is used: where it is read, the select would wait for it.)
    auto entry_of = [&](int at) { return table[min(at >> shift, a.table_stride - 1)]; };
    auto page_at = [&](int at, int entry) { return at <= until ? entry : -1; };
    // A page's codes and steps of this head: whole pages of 32 bits of bytes from the first one's.
    auto page_of = [&](int page) { return (unsigned)page < (unsigned)c.pages ? (unsigned)page : 0u; };
    const unsigned plane = c.page_tokens * (W / 2), steps = c.page_tokens * kBlocks;
    const unsigned page_codes = c.kv_heads * plane, page_steps = 2 * c.kv_heads * steps;
    const uint8_t *keys = c.keys + (size_t)kvh * plane, *values = c.values + (size_t)kvh * plane;
    const uint8_t *key_steps = (const uint8_t *)(c.key_steps + (size_t)kvh * steps),
                  *value_steps = (const uint8_t *)(c.value_steps + (size_t)kvh * steps);
    int kpage, vpage[N], spage;
    // This thread's piece i of K is block wave + 4 i of position `lane` of the
    // step, of V the elements 4 quad.. of 8 positions. Heads of 64 have half as many:
    // two of the wavefronts stage those of K, two of V.
    const int kblock = W < 128 ? wave & 1 : wave, vpiece = W < 128 ? tid & 127 : tid;
    auto look_k = [&](int step) {
        kpage = entry_of(kStep * step + (lane & 48));
        spage = entry_of(kStep * step + 16 * (tid & 3));
    };
    auto look_v = [&](int step) {
#pragma unroll
        for (int i = 0; i < N; ++i) vpage[i] = entry_of(kStep * step + 8 * ((vpiece + 256 * i) / kQuads));
    };
    uint4 kreg[N], vreg[N], vstep[N];
    _Float16 kstep[N];
    int vpage_at[N];   // the pages that vreg is of
    bool sthere;
    auto fetch_k = [&](int step) {
        const int t = (kStep * step + lane) & within;
        const unsigned page = page_of(page_at(kStep * step + (lane & 48), kpage));
        const uint8_t *kb = keys + (uint64_t)page * page_codes + (kblock * c.page_tokens + t) * 16;
        const uint16_t *sb = (const uint16_t *)(key_steps + (uint64_t)page * page_steps) +
                             (((t >> 4) * kBlocks + kblock) * 16 + (t & 3) * 4 + (t >> 2 & 3));
#pragma unroll
        for (int i = 0; i < N; ++i) {
            kreg[i] = *(const uint4 *)(kb + (size_t)64 * c.page_tokens * i);
            kstep[i] = __builtin_bit_cast(_Float16, sb[64 * i]);
        }
        sthere = (unsigned)page_at(kStep * step + 16 * (tid & 3), spage) < (unsigned)c.pages;
    };
    auto fetch_v = [&](int step) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int piece = vpiece + 256 * i, quad = piece % kQuads, vat = kStep * step + 8 * (piece / kQuads);
            vpage_at[i] = page_at(vat, vpage[i]);
            const unsigned page = page_of(vpage_at[i]);
            const int t = vat & within;
            vreg[i] = *(const uint4 *)(values + (uint64_t)page * page_codes + ((t >> 3) * kQuads + quad) * 16);
            vstep[i] = *(const uint4 *)(value_steps + (uint64_t)page * page_steps + 2 * ((quad >> 3) * c.page_tokens + t));
        }
    };
    auto ktile = [&](int buffer) { return smem[ks][buffer & (kBuffers - 1)]; };
    auto vtile = [&](int buffer) { return smem[ks][kBuffers + (buffer & (kBuffers - 1))]; };
    auto k_place = [&](int buffer, int i) {
        const int t = lane & 31, rho = 8 * ((t & 15) >> 2) + 4 * (t >> 4) + (t & 3);
        return ktile(buffer) + (((lane >> 5) * M + 2 * (kblock + 4 * i)) * 64 + rho) * 16;
    };
    auto stage_k = [&](int buffer) {
        if (W < 128 && wave >= 2) return;
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                *(half8 *)(k_place(buffer, i) + 512 * j) = key_word(codes, word_of(kreg[i], j), kstep[i]);
    };
    auto stage_there = [&](int buffer) {
        if (tid < 4) theres[ks][buffer & 1][tid] = sthere;
    };
    // The steps of V's piece i, of what this workgroup's rows see.
    auto v_limit = [&](int step, int i) {
        const int vat = kStep * step + 8 * ((vpiece + 256 * i) / kQuads);
        return (unsigned)vpage_at[i] < (unsigned)c.pages ? until - vat + 1 : 0;
    };
    auto v_low = [&](int step, int i) { return g.lowest - (kStep * step + 8 * ((vpiece + 256 * i) / kQuads)); };
    // Element 4 q + e of 32 is row 8 e + q of its tile, so that the threads of a wavefront write side by side.
    auto v_place = [&](int buffer, int i) {
        const int piece = vpiece + 256 * i, quad = piece % kQuads, eighth = piece / kQuads;
        return vtile(buffer) + ((((eighth >> 2) * D + (quad >> 3)) * 2 + (eighth & 1)) * 64 + 32 * (eighth >> 1 & 1) +
                                (quad & 7)) * 16;
    };
    auto stage_v = [&](int step, int buffer) {
        if (W < 128 && wave < 2) return;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int low = v_low(step, i), limit = v_limit(step, i);
            if (__builtin_amdgcn_ballot_w64(limit < 8 || low > 0)) vstep[i] = some_steps(vstep[i], low, limit);
            half8 x[4];
            value_words(codes, vreg[i], vstep[i], x);
#pragma unroll
            for (int e = 0; e < 4; ++e) *(half8 *)(v_place(buffer, i) + 128 * e) = x[e];
        }
    };
    look_k(begin);
    fetch_k(begin);
    look_v(begin);
    look_k(begin + KS);

    half8 qh[M], ql[M];
    float qscale;
    {
        const float *q = a.q + (rq.begin + token) * a.q_stride + (int64_t)head * W + 8 * h;
        const bool aligned = ((uintptr_t)a.q & 15) == 0 && a.q_stride % 4 == 0;
        float v[8 * M];
#pragma unroll
        for (int i = 0; i < M; ++i) {
            if (aligned) {
                *(float4 *)(v + 8 * i) = *(const float4 *)(q + 16 * i);
                *(float4 *)(v + 8 * i + 4) = *(const float4 *)(q + 16 * i + 4);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) v[8 * i + e] = q[16 * i + e];
            }
        }
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < 8 * M; ++i) top = fmaxf(top, fabsf(v[i]));
        const int e = 14 - __builtin_amdgcn_frexp_expf(halves_max(top));
#pragma unroll
        for (int i = 0; i < 8 * M; ++i) v[i] = ldexpf(a.scale < 0.f ? -v[i] : v[i], e);
#pragma unroll
        for (int i = 0; i < M; ++i) split_f16(v + 8 * i, qh[i], ql[i]);
        if constexpr (KS == 1) {
            // q in the accumulation registers, where MFMAs read it: left to the compiler it was copied from there.
#pragma unroll
            for (int i = 0; i < M; ++i) asm("" : "+a"(qh[i]), "+a"(ql[i]));
        }
        // Above 0, so that it keeps minus infinity.
        qscale = fmaxf(ldexpf(fabsf(a.scale) * 1.44269504f, -e), 0x1p-126f);
    }
    f32x16 O[D], S[2];
#pragma unroll
    for (int d = 0; d < D; ++d) O[d] = (f32x16){};
    half8 ph[2][2], pl[2][2];
    float m = -INFINITY, l = 0.f;
    bool far = false;
    uint64_t saw = 0;   // lanes that had a score
    // Each tile's operands are requested a tile ahead (the groups keep the compiler from moving the
    // reads to where they are used): a wavefront would wait for every one of them.
    constexpr int kMfma = 0x008, kRead = 0x100;
    auto outputs = [&](int buffer, auto beside) {
        const uint8_t *vs = vtile(buffer) + 16 * lane;
        auto tile = [&](int n, int d) { return *(const half8 *)(vs + ((n >> 1) * (2 * D) + 2 * d + (n & 1)) * 1024); };
        constexpr int kAhead = 4;   // (pairs of tiles are two apart)
        half8 v[kAhead];
#pragma unroll
        for (int d = 0; d < kAhead; ++d) v[d] = tile(d / D, d % D);
        if constexpr (KS == 2) __builtin_amdgcn_sched_group_barrier(kRead, kAhead, 0);
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
            for (int d = 0; d < D; d += 2) {
#pragma unroll
                for (int part = 0; part < 4; ++part) {
                    const int e = d + (part & 1);
                    if constexpr (KS == 1) __builtin_amdgcn_sched_barrier(0);
                    O[e] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[(n * D + e) % kAhead],
                                                                  part < 2 ? ph[n >> 1][n & 1] : pl[n >> 1][n & 1], O[e], 0, 0, 0);
                    if constexpr (KS == 1) __builtin_amdgcn_sched_barrier(0);
                    beside(n, d, part);
                }
                if constexpr (KS == 1) __builtin_amdgcn_sched_barrier(0);
                else __builtin_amdgcn_sched_group_barrier(kMfma, 4, 0);
                if (n * D + d + kAhead >= 4 * D) continue;
#pragma unroll
                for (int e = d; e < d + 2; ++e) v[(n * D + e) % kAhead] = tile((n * D + e + kAhead) / D, (n * D + e + kAhead) % D);
                if constexpr (KS == 2) __builtin_amdgcn_sched_group_barrier(kRead, 2, 0);
            }
    };
    auto scores = [&](int buffer, auto beside) {
        const uint8_t *kp = ktile(buffer) + 16 * lane;
#pragma unroll
        for (int t = 0; t < 2; ++t) S[t] = (f32x16){};
        constexpr int kAhead = KS == 1 ? 2 : 1;
        half8 k[kAhead + 1][2];
#pragma unroll
        for (int j = 0; j < kAhead; ++j)
#pragma unroll
            for (int t = 0; t < 2; ++t) k[j][t] = *(const half8 *)(kp + (t * M + j) * 1024);
        if constexpr (KS == 2) __builtin_amdgcn_sched_group_barrier(kRead, 2, 0);
#pragma unroll
        for (int j = 0; j < M; ++j) {
            if (j + kAhead < M) {
#pragma unroll
                for (int t = 0; t < 2; ++t) k[(j + kAhead) % (kAhead + 1)][t] = *(const half8 *)(kp + (t * M + j + kAhead) * 1024);
                if constexpr (KS == 2) __builtin_amdgcn_sched_group_barrier(kRead, 2, 0);
            }
#pragma unroll
            for (int part = 0; part < 4; ++part) {
                const int t = part & 1;
                if constexpr (KS == 1) __builtin_amdgcn_sched_barrier(0);
                S[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k[j % (kAhead + 1)][t], part < 2 ? qh[j] : ql[j], S[t], 0, 0, 0);
                if constexpr (KS == 1) __builtin_amdgcn_sched_barrier(0);
                beside(j, part);
            }
            if constexpr (KS == 1) __builtin_amdgcn_sched_barrier(0);
            else __builtin_amdgcn_sched_group_barrier(kMfma, 4, 0);
        }
    };
    // A step's softmax: its maximum (`grew`: alpha is what the sums so far are worth less) ...
    float alpha = 1.f, scale = 0.f, add = 0.f;
    bool grew = false;
    auto peak = [&](int step, int buffer) {
        const int at = kStep * step;
        const bool whole = all_from <= at && all_to >= at + kStep - 1;
        bool there[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) there[t] = theres[ks][buffer][2 * t + h];
        if (!whole || __builtin_amdgcn_ballot_w64(!there[0] || !there[1])) {
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const int from = max(first - (at + 32 * t + 16 * h), 0), to = min(last - (at + 32 * t + 16 * h), 15);
                const uint32_t seen = there[t] && from <= to ? (0xFFFFu >> (15 - to)) & (0xFFFFu << from) : 0;
#pragma unroll
                for (int n = 0; n < 16; ++n) S[t][n] = seen >> n & 1 ? S[t][n] : -INFINITY;
            }
        }
        float best = S[0][0];
#pragma unroll
        for (int n = 1; n < 32; ++n) best = fmaxf(best, S[n >> 4][n & 15]);
        saw |= __builtin_amdgcn_ballot_w64(best > -INFINITY);
        const float top = best * qscale;
        grew = __builtin_amdgcn_ballot_w64(top > m);
        if (grew) {
            const float next = fmaxf(m, ceilf(halves_max(top)));
            alpha = __builtin_amdgcn_exp2f(m - (next == -INFINITY ? 0.f : next));
            m = next;
            l *= alpha;
            far = __builtin_amdgcn_ballot_w64(is_far(m));
        }
        const float base = m == -INFINITY ? 0.f : m;
        scale = qscale;
        add = 15.f - base;
        if (far) {
#pragma clang fp contract(off)
#pragma unroll
            for (int n = 0; n < 32; ++n) S[n >> 4][n & 15] = S[n >> 4][n & 15] * qscale - base;
            scale = 1.f;
            add = 15.f;
        }
    };
    // ... what it makes of the outputs ...
    auto rescale = [&]() {
        if (!grew) return;
#pragma unroll
        for (int d = 0; d < D; ++d) O[d] *= alpha;
    };
    // ... and its weights.
    float sum[2];
    auto weight = [&](int n) {
        const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(S[n >> 4][n & 15], scale, add));
        sum[n & 1] += w;
        return w;
    };
    // A round past the group's last step is one of positions that are not there.
    if (KS == 2 && rounds > 0) {
        // The next codes set out before the MFMAs and are there after them, and go into
        // LDS between the MFMAs with the softmax.
        auto ahead = [&](int step) {
            fetch_k(step + KS);
            fetch_v(step);
            look_v(step + KS);
            look_k(step + 2 * KS);
        };
        auto between = [&](int i) {
            stage_v(begin + KS * i, 0);
            stage_k(0);
            stage_there(i + 1);
            peak(begin + KS * i, i & 1);
            rescale();
            sum[0] = sum[1] = 0.f;
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                float w[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) w[k] = weight(8 * n + k);
                split_f16(w, ph[n >> 1][n & 1], pl[n >> 1][n & 1]);
            }
            l += sum[0] + sum[1];
        };
        auto none = [](auto...) {};
        stage_k(0);
        stage_there(0);
        lds_barrier();
        if (ks) lds_barrier();   // half a step behind
        ahead(begin);
        __builtin_amdgcn_s_setprio(1);
        scores(0, none);
        __builtin_amdgcn_s_setprio(0);
        lds_barrier();
        between(0);
        lds_barrier();
        for (int i = 1; i < rounds; ++i) {
            ahead(begin + KS * i);
            __builtin_amdgcn_s_setprio(1);
            outputs(0, none);
            scores(0, none);
            __builtin_amdgcn_s_setprio(0);
            lds_barrier();   // this group's tiles are read
            between(i);
            lds_barrier();   // the next ones are there
        }
        outputs(0, none);
        if (!ks) lds_barrier();
        __syncthreads();
    }
    if constexpr (KS == 1) {
        // One wavefront per SIMD, so what is not an MFMA goes under those of the same wavefront, a few
        // instructions behind each: the next codes under the scores, into tiles of their own (a step
        // has one wait), the weights under the last step's outputs.
        static_assert(KS == 2 || (8 * N == M && D == 8), "as much as the MFMAs cover");
        Pairs u[4], key, high[4], low[4];
        // Behind MFMA `part` of four of part j of the scores: two elements of K's word j, or of V's word j - 4 N.
        auto stage = [&](int i, int j, int part) {
            const int piece = j / 4 % N, w = j % 4;
            const uint32_t n = (j < 4 * N ? word_of(kreg[piece], w) : word_of(vreg[piece], w)) >> (part & 2 ? 8 : 0);
            const half2 code = part & 1 ? codes.highs(n) : codes.lows(n);
            if (j < 4 * N) {
                key.p[part] = code * (half2){kstep[piece], kstep[piece]};
                if (part == 3) *(half8 *)(k_place(i + 1, piece) + 512 * w) = key.v;
            } else {
                u[part].p[w] = code * __builtin_bit_cast(half2, word_of(vstep[piece], w));
                if (w == 3) *(half8 *)(v_place(i, piece) + 128 * part) = u[part].v;
            }
        };
        // Behind MFMA `part` of four of the outputs' tiles d and d + 1: weights d and d + 1 of eight n, and their pieces.
        float minus = -1.f, w[2];
        asm("" : "+s"(minus));   // as in split_f16
        auto weigh = [&](int n, int d, int part) {
            if (part < 2) {
                w[part] = weight(8 * n + d + part);
            } else if (part == 2) {
                typedef float f32x2 __attribute__((ext_vector_type(2)));
                half2 hi = __builtin_convertvector((f32x2){w[0], w[1]}, half2);
                const f32x2 r = {__builtin_fmaf((float)hi.x, minus, w[0]), __builtin_fmaf((float)hi.y, minus, w[1])};
                half2 lo = __builtin_convertvector(r, half2);
                asm volatile("" : "+v"(hi), "+v"(lo), "+v"(sum[0]), "+v"(sum[1]));   // here, not where they are used
                high[n].p[d / 2] = hi;
                low[n].p[d / 2] = lo;
            }
        };
        // Codes wait for their turn in accumulation registers, as q does: loads reach them.
        auto wait_there = [](uint4 &x) {
            typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
            u32x4 v = __builtin_bit_cast(u32x4, x);
            asm volatile("" : "+a"(v));
            x = __builtin_bit_cast(uint4, v);
        };
        auto scored = [&](int i) {
            const int step = begin + i;
#pragma unroll
            for (int p = 0; p < N; ++p) {
                wait_there(kreg[p]);
                wait_there(vreg[p]);
                wait_there(vstep[p]);
            }
#pragma unroll
            for (int p = 0; p < N; ++p) {
                const int below = v_low(step, p), limit = v_limit(step, p);
                if (__builtin_amdgcn_ballot_w64(limit < 8 || below > 0)) vstep[p] = some_steps(vstep[p], below, limit);
            }
            scores(i, [&](int j, int part) { stage(i, j, part); });
            stage_there(i + 1);
            fetch_k(step + 2);
            fetch_v(step + 1);
            look_v(step + 2);
            look_k(step + 3);
            peak(step, i & 1);
            sum[0] = sum[1] = 0.f;
        };
        auto weighed = [&]() {
            l += sum[0] + sum[1];
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                ph[n >> 1][n & 1] = high[n].v;
                pl[n >> 1][n & 1] = low[n].v;
            }
            lds_barrier();   // this step's tiles are read, the next ones are there
        };
        stage_k(0);
        stage_there(0);
        fetch_k(begin + 1);
        fetch_v(begin);
        look_v(begin + 1);
        look_k(begin + 2);
        lds_barrier();
        if (rounds > 0) {
            scored(0);
#pragma unroll
            for (int n = 0; n < 4; ++n)
#pragma unroll
                for (int d = 0; d < D; d += 2)
#pragma unroll
                    for (int part = 0; part < 3; ++part) weigh(n, d, part);
            weighed();
        }
        for (int i = 1; i < rounds; ++i) {
            scored(i);
            outputs(i - 1, weigh);
            rescale();
            weighed();
        }
        if (rounds > 0) outputs(rounds - 1, [](auto...) {});
    }
    l = halves_sum(l);
    if (m == -INFINITY && (saw >> col & 0x0000000100000001u)) m = -FLT_MAX;   // scores, none in fp32
    if constexpr (KS == 2) {
        // The second group's rows through LDS, as they lie in its registers.
        float *po = (float *)&smem[0][0][0] + wave * (16 * D * 64) + lane;
        static_assert(sizeof(smem) >= 4 * 16 * D * 64 * sizeof(float), "the second group's outputs fit");
        if (ks) {
#pragma unroll
            for (int d = 0; d < D; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) po[(16 * d + i) * 64] = O[d][i];
            if (h == 0) smem_ml[wave][col] = make_float2(m, l);
        }
        __syncthreads();
        if (ks) return;
        const float2 other = smem_ml[wave][col];
        const float top = fmaxf(m, other.x), base = top == -INFINITY ? 0.f : top;
        const float f0 = __builtin_amdgcn_exp2f(m - base), f1 = __builtin_amdgcn_exp2f(other.x - base);
        m = top;
        l = l * f0 + other.y * f1;
#pragma unroll
        for (int d = 0; d < D; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) O[d][i] = O[d][i] * f0 + po[(16 * d + i) * 64] * f1;
        lds_wave();   // rows go where other lanes read
    }
    // Rows go out whole, through LDS: as they lie in registers a store would touch 32 rows (16 heads over 8 of
    // 256: 13 us at the kernel's end). Register 4 e + i of tile d is element 32 d + 16 h + 4 i + e. A row's
    // pieces of 16 bytes are turned by its number, so that neither side meets in a bank.
    if (KS == 1) __syncthreads();   // the last tiles are read
    constexpr int kPieces = W / 4, kTurn = (kPieces < 32 ? kPieces : 32) - 1, kAtOnce = 64 / (kPieces < 64 ? kPieces : 64);
    uint8_t *const rows = &smem[0][0][0] + wave * (32 * 4 * W);
    static_assert(sizeof(smem) >= 4 * 32 * 4 * W, "the rows fit");
    const bool shared = g.active > 1, aligned = shared || (((uintptr_t)a.out & 15) == 0 && a.out_stride % 4 == 0);
    const Share to = split.share(c.kv_heads, x % tiles, kvh, row - kWideRows * tile, sp, W);
    float *const mine = shared ? to.o : a.out + (rq.begin + token) * a.out_stride + (int64_t)head * W;
    if (shared && h == 0 && row < rq.rows) *to.ml = make_float2(m, l);
    const float inverse = shared ? 1.f : inverse_of(l, m);
#pragma unroll
    for (int d = 0; d < D; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            *(float4 *)(rows + (col * kPieces + ((8 * d + 4 * h + i) ^ (col & kTurn))) * 16) =
                make_float4(O[d][i] * inverse, O[d][4 + i] * inverse, O[d][8 + i] * inverse, O[d][12 + i] * inverse);
    lds_wave();   // a row is read by other lanes than wrote it
#pragma unroll 8
    for (int p = 0; p < 32; p += kAtOnce) {
        const int r = p + lane / kPieces, piece = lane % kPieces;
        const float4 o = *(const float4 *)(rows + (r * kPieces + (piece ^ (r & kTurn))) * 16);
        const uintptr_t at = (uintptr_t)mine;
        float *const out = (float *)((uint64_t)(uint32_t)__shfl((int)(at >> 32), r, 64) << 32 | (uint32_t)__shfl((int)at, r, 64)) +
                           4 * piece;
        if (kWideRows * tile + 32 * wave + r >= rq.rows) continue;
        if (aligned) {
            *(float4 *)out = o;
        } else {
            out[0] = o.x;
            out[1] = o.y;
            out[2] = o.z;
            out[3] = o.w;
        }
    }
}

// Both in one launch: `wide_blocks` workgroups of wide tiles, then those of few rows.
template <int W>
__global__ __launch_bounds__(256) void kv4_join(Kv4Attention a, Split few, Split wide, int most_rows, int wide_blocks)
{
    const int index = blockIdx.x;
    if (index >= wide_blocks) join_row<W>(a, few, most_rows, index - wide_blocks);
    else join_wide<W>(a, wide, most_rows, index);
}

template <int W>
hipError_t launch_width(const Kv4Attention &a, const Plan &p, hipStream_t s)
{
    const unsigned requests = a.requests, kv_heads = a.cache.kv_heads;
    if (p.any_few) {
        const bool listed = p.few.listed;
        const unsigned tiles = listed ? (unsigned)p.few.places : (unsigned)((p.few.tile + kRows - 1) / kRows);
        const unsigned most = p.few.most, packed = p.few.packed ? tiles * requests * most : 0;
        const dim3 grid = packed ? dim3(packed * kv_heads) : dim3(tiles * kv_heads, listed ? 1 : requests, most);
        // No request of few rows has more than eight: a column for each piece.
        if (p.few.tile <= 8) hipLaunchKernelGGL((kv4_rows<W, true>), grid, dim3(64 * kWaves), 0, s, a, p.few, p.most_rows);
        else hipLaunchKernelGGL((kv4_rows<W, false>), grid, dim3(64 * kWaves), 0, s, a, p.few, p.most_rows);
    }
    int64_t wide_blocks = 0;
    if constexpr (W <= 256) {
        if (p.any_wide) {
            constexpr int KS = W <= 128 ? 2 : 1;
            const int64_t tiles = p.wide.places;
            hipLaunchKernelGGL((kv4_wide<W, KS>), dim3((unsigned)(tiles * p.wide.most * kv_heads)), dim3(256 * KS), 0, s, a,
                               p.wide, p.most_rows);
            if (p.wide.most > 1) wide_blocks = tiles * kJoinParts * kv_heads;
        }
    }
    const int64_t blocks = wide_blocks + (p.any_few && p.few.most > 1 ? (int64_t)p.few.tile * kv_heads * p.few.places : 0);
    if (blocks)
        hipLaunchKernelGGL((kv4_join<W>), dim3((unsigned)blocks), dim3(256), 0, s, a, p.few, p.wide, p.most_rows,
                           (int)wide_blocks);
    return hipGetLastError();
}

}  // namespace

size_t kv4_attention_workspace(const Kv4Attention &a)
{
    const Plan p = plan_of(a, nullptr, SIZE_MAX);
    return (p.few.most > 1 ? p.few.most * share_bytes(a, p.few) : 0) +
           (p.wide.most > 1 ? p.wide.most * share_bytes(a, p.wide) : 0);
}

hipError_t launch_kv4_attention(const Kv4Attention &a, void *workspace, size_t workspace_bytes, hipStream_t s)
{
    const Plan p = plan_of(a, (float *)workspace, workspace ? workspace_bytes : 0);
    switch (a.cache.width) {
    case 64: return launch_width<64>(a, p, s);
    case 128: return launch_width<128>(a, p, s);
    case 256: return launch_width<256>(a, p, s);
    default: return launch_width<512>(a, p, s);
    }
}

}  // namespace fy
