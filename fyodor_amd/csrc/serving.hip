// The steps around attention over a paged 8-bit cache
// (include/fyodor_hip_serving.h): page tables from request lengths, rotary
// positions, and the cache's store and load. None of them does arithmetic worth
// counting: in a decode step they are bound by launches and by the chains of
// waits inside (the angles of 16 tokens take 2 us), for prompts by the
// bytes of the rows at a copy's rate.
#include <math.h>

#include "device.h"

#pragma clang fp contract(off)

#include "rotary.h"

namespace fy {
namespace {

// ---- pages ----------------------------------------------------------------

constexpr int kPageThreads = 1024;

constexpr uint32_t kMost = INT_MAX;   // where sums saturate: two such values add up within 32 bits

// Exclusive prefix sums over the workgroup's threads; *total over all of them.
// `parts`: one word per wavefront.
__device__ __forceinline__ uint32_t block_prefix(uint32_t v, uint32_t *parts, uint32_t *total)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t s = v;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const uint32_t o = (uint32_t)__shfl_up((int)s, d, 64);
        if (lane >= d) s = min(s + o, kMost);
    }
    __syncthreads();   // the last call's parts are read
    if (lane == 63) parts[wave] = s;
    __syncthreads();
    uint32_t before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kPageThreads / 64; ++w) {
        if (w == wave) before = all;
        all = min(all + parts[w], kMost);
    }
    *total = all;
    const uint32_t own = (uint32_t)__shfl_up((int)s, 1, 64);
    return min(before + (lane ? own : 0), kMost);
}

__device__ __forceinline__ int clamped(int v, int most) { return v < 0 ? 0 : v > most ? most : v; }

// The largest i < n with first[i] <= at (first[0] = 0 <= at), first ascending.
__device__ __forceinline__ int last_from(const uint32_t *first, int n, uint32_t at)
{
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (first[mid] <= at) lo = mid;
        else hi = mid;
    }
    return lo;
}

// One workgroup: the page stack is one thing. Requests go 1024 at a time, a
// thread each; the moved pages of such a chunk are spread over all threads.
__global__ __launch_bounds__(kPageThreads) void page_tables(PageStep p)
{
    __shared__ uint32_t parts[kPageThreads / 64], first[kPageThreads];
    __shared__ int base[kPageThreads];
    const int tid = threadIdx.x;
    const int chunks = (p.requests + kPageThreads - 1) / kPageThreads;
    uint32_t top = (uint32_t)clamped(p.free_count[0], p.pages);
    auto need_of = [&](int r, bool *beyond) {
        const int length = max(p.lengths[r], 0), need = (int)(((uint32_t)length + p.page_tokens - 1) / p.page_tokens);
        *beyond = need > p.table_stride;
        return need;
    };
    // 1. Pages past the need, back on the stack.
    for (int c = 0; c < chunks; ++c) {
        const int r = c * kPageThreads + tid;
        uint32_t back = 0;
        int need = 0;
        if (r < p.requests) {
            bool beyond;
            need = need_of(r, &beyond);
            const int held = clamped(p.held[r], p.table_stride);
            if (!beyond && held > need) {
                back = (uint32_t)(held - need);
                p.held[r] = need;
            }
        }
        uint32_t total;
        first[tid] = block_prefix(back, parts, &total);
        base[tid] = need;
        __syncthreads();
        for (uint32_t i = tid; i < total; i += kPageThreads) {
            const int k = last_from(first, kPageThreads, i);
            int *entry = p.table + (size_t)(c * kPageThreads + k) * p.table_stride + base[k] + (i - first[k]);
            if (top + i < (uint32_t)p.pages) p.free_pages[top + i] = *entry;
            *entry = -1;
        }
        top = min(top + total, (uint32_t)p.pages);
        __syncthreads();
    }
    // 2. Pages for the requests that grow, from the top.
    uint32_t asked = 0, given = 0, refused = 0;
    for (int c = 0; c < chunks; ++c) {
        const int r = c * kPageThreads + tid;
        uint32_t grow = 0;
        int held = 0;
        bool beyond = false;
        if (r < p.requests) {
            const int need = need_of(r, &beyond);
            held = clamped(p.held[r], p.table_stride);
            if (!beyond && need > held) grow = (uint32_t)(need - held);
        }
        uint32_t total, served;
        const uint32_t before = min(asked + block_prefix(grow, parts, &total), kMost);
        const bool fits = before + grow <= top;
        const uint32_t mine = fits ? grow : 0;
        // A request that is not served, and with it every later one that
        // needs pages, takes nothing: those served are a prefix.
        first[tid] = block_prefix(mine, parts, &served);
        base[tid] = held;
        if (mine) p.held[r] = held + (int)mine;
        __syncthreads();
        for (uint32_t i = tid; i < served; i += kPageThreads) {
            const int k = last_from(first, kPageThreads, i);
            p.table[(size_t)(c * kPageThreads + k) * p.table_stride + base[k] + (i - first[k])] =
                p.free_pages[top - 1 - given - i];
        }
        asked = min(asked + total, kMost);
        given += served;
        uint32_t left;
        block_prefix(beyond || (grow && !fits) ? 1 : 0, parts, &left);
        refused += left;
    }
    // 3. The rows' starts, those past max_tokens too: attention takes a
    // request's positions from them.
    uint32_t rows = 0;
    for (int c = 0; c < chunks; ++c) {
        const int r = c * kPageThreads + tid;
        const uint32_t n = r < p.requests ? (uint32_t)max(p.counts[r], 0) : 0;
        uint32_t total;
        const uint32_t before = block_prefix(n, parts, &total);
        if (r < p.requests) p.starts[r] = (int)min(rows + before, kMost);
        rows = min(rows + total, kMost);
    }
    if (tid == 0) {
        p.starts[p.requests] = (int)rows;
        p.free_count[0] = (int)(top - given);
        p.free_count[1] = (int)refused;
    }
}

// The row's position and slot.
__device__ __forceinline__ void place_row(const PageStep &p, int row, bool live, int r, int start, int length, int count,
    int held)
{
    int position = -1, slot = -1;
    if (live) {
        // 64 bits: the lengths are the caller's.
        const int64_t at = (int64_t)length - count + (row - start);
        position = (int)at;
        if (at >= 0) {
            const int64_t j = at / p.page_tokens;
            if (j < held) {
                const int page = p.table[(size_t)r * p.table_stride + j];
                if ((unsigned)page < (unsigned)p.pages) slot = page * p.page_tokens + (int)(at % p.page_tokens);
            }
        }
    }
    p.positions[row] = position;
    p.slots[row] = slot;
}

// The whole step of up to 1024 requests and 8192 rows in one launch: a request
// per thread, the three prefix sums together, rows from LDS. Bound by its chain
// of waits (lengths, stack and table, rows): 64 requests of a token each take 4.8 us
// (page_tables and page_rows 7.0 and 3.1), 8192 rows of theirs 10.5, by when the
// two are as fast; more rows want more than one CU.
__global__ __launch_bounds__(kPageThreads) void page_small(PageStep p)
{
    constexpr int kWavesHere = kPageThreads / 64;
    __shared__ uint32_t parts[3][kWavesHere], first[kPageThreads], starts[kPageThreads];
    __shared__ int lengths[kPageThreads], counts[kPageThreads], helds[kPageThreads];
    __shared__ uint32_t served, refused;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const bool mine = tid < p.requests;
    const int length = mine ? max(p.lengths[tid], 0) : 0;
    const uint32_t n = mine ? (uint32_t)max(p.counts[tid], 0) : 0;
    int held = mine ? clamped(p.held[tid], p.table_stride) : 0;
    uint32_t top = (uint32_t)clamped(p.free_count[0], p.pages);
    const int need = (int)(((uint32_t)length + p.page_tokens - 1) / p.page_tokens);
    const bool beyond = need > p.table_stride;
    const uint32_t back = !beyond && held > need ? (uint32_t)(held - need) : 0;
    const uint32_t grow = !beyond && need > held ? (uint32_t)(need - held) : 0;
    uint32_t sums[3] = {back, grow, n};
#pragma unroll
    for (int d = 1; d < 64; d *= 2)
#pragma unroll
        for (int k = 0; k < 3; ++k) {
            const uint32_t o = (uint32_t)__shfl_up((int)sums[k], d, 64);
            if (lane >= d) sums[k] = min(sums[k] + o, kMost);
        }
    if (lane == 63)
#pragma unroll
        for (int k = 0; k < 3; ++k) parts[k][wave] = sums[k];
    if (tid == 0) served = refused = 0;
    __syncthreads();
    uint32_t before[3], total[3];
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        uint32_t all = 0, here = 0;
#pragma unroll
        for (int w = 0; w < kWavesHere; ++w) {
            if (w == wave) here = all;
            all = min(all + parts[k][w], kMost);
        }
        const uint32_t own = (uint32_t)__shfl_up((int)sums[k], 1, 64);
        before[k] = min(here + (lane ? own : 0), kMost);
        total[k] = all;
    }
    // 1. Pages past the need, back on the stack.
    if (total[0]) {
        first[tid] = before[0];
        helds[tid] = need;
        __syncthreads();
        for (uint32_t i = tid; i < total[0]; i += kPageThreads) {
            const int k = last_from(first, kPageThreads, i);
            int *entry = p.table + (size_t)k * p.table_stride + helds[k] + (i - first[k]);
            if (top + i < (uint32_t)p.pages) p.free_pages[top + i] = *entry;
            *entry = -1;
        }
        top = min(top + total[0], (uint32_t)p.pages);
        __syncthreads();
    }
    if (back) held = need;
    // 2. Pages for the requests that grow; those served are a prefix of them.
    const bool fits = before[1] + grow <= top;
    first[tid] = before[1];
    helds[tid] = held;
    lengths[tid] = length;
    counts[tid] = (int)n;
    starts[tid] = before[2];
    if (grow && fits) atomicMax(&served, before[1] + grow);
    if (beyond || (grow && !fits)) atomicAdd(&refused, 1u);
    if (grow && fits) held += (int)grow;
    __syncthreads();
    for (uint32_t i = tid; i < served; i += kPageThreads) {
        const int k = last_from(first, kPageThreads, i);
        p.table[(size_t)k * p.table_stride + helds[k] + (i - first[k])] = p.free_pages[top - 1 - i];
    }
    if (mine) {
        if (back || grow) p.held[tid] = held;
        p.starts[tid] = (int)before[2];
    }
    if (tid == 0) {
        p.starts[p.requests] = (int)total[2];
        p.free_count[0] = (int)(top - served);
        p.free_count[1] = (int)refused;
    }
    __syncthreads();
    helds[tid] = held;
    __syncthreads();
    // 3. The rows.
    for (int row = tid; row < p.max_tokens; row += kPageThreads) {
        const int r = last_from(starts, p.requests, (uint32_t)row);
        place_row(p, row, row < (int)total[2], r, (int)starts[r], lengths[r], counts[r], helds[r]);
    }
}

__global__ __launch_bounds__(256) void page_rows(PageStep p)
{
    const int row = blockIdx.x * 256 + threadIdx.x;
    if (row >= p.max_tokens) return;
    const bool live = row < p.starts[p.requests];
    const int r = last_from((const uint32_t *)p.starts, p.requests, (uint32_t)row);
    place_row(p, row, live, r, p.starts[r], max(p.lengths[r], 0), max(p.counts[r], 0),
              clamped(p.held[r], p.table_stride));
}

// ---- rotary positions -----------------------------------------------------

__global__ __launch_bounds__(256) void rope_angles(const int *__restrict__ positions, int64_t n,
    const float *__restrict__ frequencies, int pairs, float magnitude, float2 *__restrict__ angles)
{
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    const double turns = (double)positions[i / pairs] * (double)frequencies[i % pairs] * (1 / M_PI);
    double s, c;
    sincospi(turns, &s, &c);
    angles[i] = make_float2((float)(c * magnitude), (float)(s * magnitude));
}

// Workgroup (row, part of its heads). Rows of 24 heads of 256, a quarter of
// each rotated: 2049 of them 24.5 us, 4.1 TB/s (a grid through the parts of a
// row first: 6 us more). Angles in 64 bits per step, not per layer: 4 us for
// 2049 x 32.
__global__ __launch_bounds__(256) void rope_rows(Rows q, Rows k, int width, const float2 *__restrict__ angles,
    int rotated, bool halves, int q_parts, int each, bool quads)
{
    const int row = blockIdx.x, part = blockIdx.y;
    if (part < q_parts)
        rotate_heads(q, row, part * each, min(part * each + each, q.heads), width, angles, rotated, halves, quads);
    else
        rotate_heads(k, row, (part - q_parts) * each, min((part - q_parts) * each + each, k.heads), width, angles,
                     rotated, halves, quads);
}

// ---- the 8-bit cache ------------------------------------------------------

constexpr float kScaleFloor = 0x1p-100f;

__device__ __forceinline__ int key_at(int t, int d, int page_tokens) { return ((d >> 4) * page_tokens + t) * 16 + (d & 15); }
__device__ __forceinline__ int value_at(int t, int d, int width) { return ((t >> 4) * width + d) * 16 + (t & 15); }

// round(x / scale), ties to even: the remainder x - n scale of the nearest
// guess is exact (a multiple of scale's last bit, below scale), so comparing it
// with half a step settles the guesses next to a border.
__device__ __forceinline__ int8_t code_of(float x, float scale, float inverse)
{
    float n = rintf(x * inverse);
    const float r = __builtin_fmaf(-n, scale, x), half = 0.5f * scale;
    const bool odd = (int)n & 1;
    if (r > half || (r == half && odd)) n += 1.f;
    else if (r < -half || (r == -half && odd)) n -= 1.f;
    return (int8_t)(int)fminf(fmaxf(n, -127.f), 127.f);
}

// The largest magnitude by its bits: NaN above infinity above the rest.
__device__ __forceinline__ uint32_t magnitude(float x) { return __builtin_bit_cast(uint32_t, x) & 0x7FFFFFFFu; }

struct Store {
    Kv8 c;
    const int *slots;
    int count;
    const float *k, *v;
    int64_t k_stride, v_stride;
    const float2 *angles;
    int rotated;
    bool halves, quads_k, quads_q;
    Rows q;
    int each;    // q heads per workgroup
    int parts;   // workgroups per row of q
    int rows;    // rows of a workgroup that stores
    int apart;   // groups of rows that follow in the grid are this far apart ..
    int lines;   // .. and `lines` of them go before the next ones
    int stores;  // workgroups that store
};

// 16 elements of a key from element 16 chunk, rotated; rows and angles in 16 bytes.
template <int W>
__device__ __forceinline__ void key_chunk(const Store &s, int row, int head, int chunk, float (&x)[16])
{
    const int d = 16 * chunk, half = s.rotated / 2;
    const float *k = s.k + row * s.k_stride + head * W;
    const float2 *angles = s.angles + (size_t)row * half;
#pragma unroll
    for (int i = 0; i < 4; ++i) *(float4 *)(x + 4 * i) = *(const float4 *)(k + d + 4 * i);
    if (d >= s.rotated) return;
    if (!s.halves) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float4 a = *(const float4 *)(angles + d / 2 + 2 * i);
            rotate_pair(x[4 * i], x[4 * i + 1], a.x, a.y);
            rotate_pair(x[4 * i + 2], x[4 * i + 3], a.z, a.w);
        }
        return;
    }
    const bool second = d >= half;
    const int j = second ? d - half : d;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float4 o = *(const float4 *)(k + (second ? j : d + half) + 4 * i);
        const float4 a0 = *(const float4 *)(angles + j + 4 * i), a1 = *(const float4 *)(angles + j + 4 * i + 2);
        const float ov[4] = {o.x, o.y, o.z, o.w}, cv[4] = {a0.x, a0.z, a1.x, a1.z}, sv[4] = {a0.y, a0.w, a1.y, a1.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float u = second ? ov[e] : x[4 * i + e], w = second ? x[4 * i + e] : ov[e];
            rotate_pair(u, w, cv[e], sv[e]);
            x[4 * i + e] = second ? w : u;
        }
    }
}

// Element d of the run's values of granule g (positions 16 g.. of the page);
// those outside the run are 0. g is the same in a wavefront: rows by scalar addresses.
template <int W>
__device__ __forceinline__ void value_granule(const Store &s, int row, int at, int n, int head, int g, int d,
    float (&x)[16])
{
    g = __builtin_amdgcn_readfirstlane(g);
    const float *v = s.v + row * s.v_stride + head * W;
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = (v + min(max(16 * g + i - at, 0), n - 1) * s.v_stride)[d];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        // All loads set out first: moved under the condition each would be waited for by itself.
        asm volatile("" : "+v"(x[i]));
        const int t = 16 * g + i - at;
        x[i] = t >= 0 && t < n ? x[i] : 0.f;
    }
}

__device__ __forceinline__ uint4 codes_of(const float (&x)[16], float scale, float inverse)
{
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        w[i] = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            w[i] |= (uint32_t)(uint8_t)code_of(x[4 * i + e], scale, inverse) << (8 * e);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// The nearest row in the cache of the 128 from `row` on (step 1) or back (-1): it
// if it is of this page, else -1.
__device__ __forceinline__ int page_goes_on(const Store &s, int row, int step, int page, int shift)
{
    const int lane = threadIdx.x & 63;
    for (int k = 0; k < 128; k += 64) {
        const int at = row + step * (k + lane), slot = s.slots[min(max(at, 0), s.count - 1)];
        const uint64_t live = __builtin_amdgcn_ballot_w64(at >= 0 && at < s.count &&
                                                          (unsigned)slot < (unsigned)(s.c.pages * s.c.page_tokens));
        if (live) {
            const int first = __builtin_ctzll(live);
            return __builtin_amdgcn_readlane(slot, first) >> shift == page ? row + step * (k + first) : -1;
        }
    }
    return -1;
}

// The run of rows that begins at `row`: its head's keys (kind 0) or values. In
// a long run a thread forms 16 codes that lie together: of one position's key, or
// of 16 positions of one element of the values; in a short one (decoding) single
// codes. Bound by its chain of waits (slots, rows and the old scale, codes) for a
// few rows, by the rows' bytes for many.
//
// Returns the row where the page's next run begins, -1 where there is none: runs of
// one page share its scale, so one workgroup takes them in turn.
template <int W>
__device__ __forceinline__ int store_run(const Store &args, int row, int head, int kind, uint32_t *top)
{
    constexpr int kChunks = W / 16, kShort = 4;   // elements per thread of a short run
    Store s = args;
    // Opaque: what follows from them is formed for each run instead of living
    // in registers over the loop of runs.
    asm volatile("" : "+s"(s.k_stride), "+s"(s.v_stride), "+s"(s.c.page_tokens), "+s"(s.rotated), "+s"(head));
    const Kv8 &c = s.c;
    const int tid = threadIdx.x, lane = tid & 63, page_tokens = c.page_tokens;
    const int slot = s.slots[row], shift = 31 - __builtin_clz(page_tokens), page = slot >> shift,
              at = slot & (page_tokens - 1);
    const int next0 = s.slots[min(row + lane, s.count - 1)], next1 = s.slots[min(row + lane + 64, s.count - 1)];
    // The run's length: up to the first row that does not follow on, or the page's end.
    int n = min(page_tokens - at, s.count - row);
    {
        const uint64_t off0 = __builtin_amdgcn_ballot_w64(lane >= n || next0 != slot + lane);
        const uint64_t off1 = __builtin_amdgcn_ballot_w64(lane + 64 >= n || next1 != slot + lane + 64);
        if (off0) n = __builtin_ctzll(off0);
        else if (off1) n = 64 + __builtin_ctzll(off1);
    }
    // The next run's row: mostly the slot after this run says that there is none;
    // else it is looked for when the stores have set out.
    bool last = at + n == page_tokens || row + n == s.count;
    if (!last) {
        const unsigned then = __builtin_amdgcn_readlane(n < 64 ? next0 : next1, n & 63);
        last = then < (unsigned)(c.pages * page_tokens) && (int)then >> shift != page;
    }
    auto next_run = [&]() { return last ? -1 : page_goes_on(s, row + n, 1, page, shift); };
    const size_t place = (size_t)page * c.kv_heads + head;
    uint4 *codes = (uint4 *)((kind ? c.values : c.keys) + place * page_tokens * W);
    int8_t *bytes = (int8_t *)codes;
    float *scale_at = (kind ? c.value_scales : c.key_scales) + place;
    const float old = at ? *scale_at : 0.f;
    // Single codes, too, of keys whose rows or angles do not come in 16 bytes.
    const bool brief = n * W <= 256 * kShort || (!kind && !s.quads_k);
    auto element = [&](int i) {
        const int r = row + i / W, d = i % W;
        return kind ? s.v[r * s.v_stride + head * W + d]
                    : rotated_at(s.k + r * s.k_stride + head * W, d, s.angles + (size_t)r * (s.rotated / 2), s.rotated,
                                 s.halves);
    };
    // Pieces: (position, 16 elements) of the keys, 16 positions together; or
    // (granule, element) of the values.
    const int g0 = at / 16;
    const int pieces = kind ? ((at + n - 1) / 16 - g0 + 1) * W : (n + 15) / 16 * 16 * kChunks;
    auto piece_at = [&](int i, float (&x)[16]) {
        if (kind) {
            value_granule<W>(s, row, at, n, head, g0 + i / W, i % W, x);
        } else {
            const int t = i / (16 * kChunks) * 16 + i % 16, chunk = i / 16 % kChunks;
            if (t < n) {
                key_chunk<W>(s, row + t, head, chunk, x);
            } else {
#pragma unroll
                for (int e = 0; e < 16; ++e) x[e] = 0.f;
            }
        }
    };
    uint32_t big = 0;
    float few[kShort], kept[2][16];   // this thread's elements, or first pieces (more are read again)
    if (brief) {
#pragma unroll
        for (int p = 0; p < kShort; ++p)
            if (tid + 256 * p < n * W) {
                few[p] = element(tid + 256 * p);
                big = max(big, magnitude(few[p]));
            }
#pragma unroll 1
        for (int i = tid + 256 * kShort; i < n * W; i += 256) big = max(big, magnitude(element(i)));
    } else {
#pragma unroll
        for (int p = 0; p < 2; ++p)
            if (tid + 256 * p < pieces) {
                piece_at(tid + 256 * p, kept[p]);
#pragma unroll
                for (int e = 0; e < 16; ++e) big = max(big, magnitude(kept[p][e]));
            }
#pragma unroll 1
        for (int i = tid + 512; i < pieces; i += 256) {
            float x[16];
            piece_at(i, x);
#pragma unroll
            for (int e = 0; e < 16; ++e) big = max(big, magnitude(x[e]));
        }
    }
#pragma unroll
    for (int o = 32; o; o >>= 1) big = max(big, (uint32_t)__shfl_xor((int)big, o, 64));
    if (lane == 0) top[tid >> 6] = big;
    __syncthreads();
    big = max(max(top[0], top[1]), max(top[2], top[3]));
    float scale = __builtin_bit_cast(float, big) * (1.f / 127.f);
    if (scale < kScaleFloor) scale = kScaleFloor;
    if (at) {
        if (scale <= old || old != old) {
            scale = old;
        } else {
            // The page's codes to the new step.
#pragma unroll 1
            for (int i = tid; i < page_tokens * W; i += 256)
                bytes[i] = (int8_t)(int)fmin(fmax(rint((double)bytes[i] * old / scale), -127.0), 127.0);
            __syncthreads();
        }
    }
    const float inverse = 1.f / scale;
    // Under an infinite scale every code is 0, so that code * scale is NaN.
    const uint32_t keep = __builtin_isfinite(scale) ? ~0u : 0u;
    if (tid == 0) *scale_at = scale;
    if (brief) {
#pragma unroll
        for (int p = 0; p < kShort; ++p) {
            const int i = tid + 256 * p, t = at + i / W, d = i % W;
            if (i < n * W)
                bytes[kind ? value_at(t, d, W) : key_at(t, d, page_tokens)] = (int8_t)(code_of(few[p], scale, inverse) & keep);
        }
#pragma unroll 1
        for (int i = tid + 256 * kShort; i < n * W; i += 256)
            bytes[key_at(at + i / W, i % W, page_tokens)] = (int8_t)(code_of(element(i), scale, inverse) & keep);
        return next_run();
    }
    auto put = [&](int i, const float (&x)[16]) {
        uint4 w = codes_of(x, scale, inverse);
        w = make_uint4(w.x & keep, w.y & keep, w.z & keep, w.w & keep);
        if (kind) {
            // Positions of the granule outside the run keep their codes.
            const int g = g0 + i / W, from = at - 16 * g, to = at + n - 16 * g;
            uint4 *there = codes + g * W + i % W;
            if (from <= 0 && to >= 16) {
                *there = w;
            } else {
                int8_t *b = (int8_t *)there;
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    if (e >= from && e < to) b[e] = (int8_t)(word_of(w, e >> 2) >> (8 * (e & 3)));
            }
        } else {
            const int t = i / (16 * kChunks) * 16 + i % 16, chunk = i / 16 % kChunks;
            if (t < n) codes[chunk * page_tokens + at + t] = w;
        }
    };
#pragma unroll
    for (int p = 0; p < 2; ++p)
        if (tid + 256 * p < pieces) put(tid + 256 * p, kept[p]);
#pragma unroll 1
    for (int i = tid + 512; i < pieces; i += 256) {
        float x[16];
        piece_at(i, x);
        put(i, x);
    }
    return next_run();
}

// Workgroup (group of rows, 2 head + kind): the runs that begin in its rows;
// from number `stores` on, (row, part): a part of a row's q. A group's
// workgroups stand together: with the rows' first head before all second ones, strides
// that are multiples of 4 KB sent everything in flight to the same few channels
// (4096 rows, 8 heads of 128, no q: 331 us, so 46). Most rows of a prompt begin
// no run, and a workgroup that finds none costs 0.35 ns of the chip: rows go in
// groups where there are many (those 46 us -> 27). Groups a page apart follow each other in the
// grid: in the rows' order the ones with a run, one in page_tokens / rows, were
// dealt to a part of the CUs only (27 us -> 17; the bytes alone take 8).
template <int W>
__global__ __launch_bounds__(256, 3) void kv8_store(Store s)
{
    __shared__ uint32_t top[4];
    const int pairs = 2 * s.c.kv_heads;
    if ((int)blockIdx.x >= s.stores) {
        const int i = blockIdx.x - s.stores, first = i % s.parts * s.each;
        rotate_heads(s.q, i / s.parts, first, min(first + s.each, s.q.heads), W, s.angles, s.rotated, s.halves,
                     s.quads_q);
        return;
    }
    const int at = blockIdx.x / pairs, part = blockIdx.x % pairs;
    const int first_row = (at % s.lines * s.apart + at / s.lines) * s.rows;
    const int lane = threadIdx.x & 63, rows = min(s.rows, s.count - first_row);
    if (rows <= 0) return;
    const int row = first_row + min(lane, rows - 1), slot = s.slots[row], before = row ? s.slots[row - 1] : -2;
    // The rows that are the first of their page: the row before is of another one. (If that
    // is not in the cache, the nearest one before it says.)
    const unsigned slots = (unsigned)(s.c.pages * s.c.page_tokens);
    const int shift = 31 - __builtin_clz(s.c.page_tokens), page = slot >> shift;
    const bool here = lane < rows && (unsigned)slot < slots, begins = row == 0 || (slot & (s.c.page_tokens - 1)) == 0;
    uint64_t mask = __builtin_amdgcn_ballot_w64(here && (begins || ((unsigned)before < slots && before >> shift != page)));
    for (uint64_t look = __builtin_amdgcn_ballot_w64(here && !begins && (unsigned)before >= slots); look; look &= look - 1) {
        const int at = __builtin_ctzll(look);
        if (page_goes_on(s, first_row + at - 1, -1, __builtin_amdgcn_readlane(page, at), shift) < 0) mask |= 1ull << at;
    }
    for (; mask; mask &= mask - 1)
        for (int run = first_row + __builtin_ctzll(mask); run >= 0;) {
            run = store_run<W>(s, run, part >> 1, part & 1, top);
            __syncthreads();   // `top` is read, the page's codes and scale are written
        }
}

// Workgroup (rows, 1024 columns of heads x width): a thread 4 columns of each
// row. The 4 x 16 codes of a granule's values stay for the rows that follow in it.
__global__ __launch_bounds__(256) void kv8_load(Kv8 c, const int *__restrict__ slots, int count, int rows,
    float *__restrict__ k, int64_t k_stride, float *__restrict__ v, int64_t v_stride, bool quads)
{
    const int i = 4 * (blockIdx.y * 256 + threadIdx.x), head = i / c.width, d = i % c.width;
    if (head >= c.kv_heads) return;
    const int end = min((int)(blockIdx.x + 1) * rows, count);
    int held = -1;
    uint4 w[4];
    float ks = 0.f, vs = 0.f;
    for (int row = blockIdx.x * rows; row < end; ++row) {
        const int slot = slots[row];
        if (slot < 0 || slot >= c.pages * c.page_tokens) continue;
        const int t = slot % c.page_tokens;
        const size_t place = (size_t)(slot / c.page_tokens) * c.kv_heads + head, codes = place * c.page_tokens * c.width;
        if (slot / 16 != held) {
            held = slot / 16;
            const uint4 *there = (const uint4 *)(c.values + codes + value_at(t & ~15, d, c.width));
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = there[e];
            ks = c.key_scales[place];
            vs = c.value_scales[place];
        }
        const uint32_t kw = *(const uint32_t *)(c.keys + codes + key_at(t, d, c.page_tokens));
        float x[4], y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t q = (t & 8) ? ((t & 4) ? w[e].w : w[e].z) : ((t & 4) ? w[e].y : w[e].x);
            x[e] = (float)(int8_t)(kw >> (8 * e)) * ks;
            y[e] = (float)(int8_t)(q >> (8 * (t & 3))) * vs;
        }
        float *to_k = k + row * k_stride + i, *to_v = v + row * v_stride + i;
        if (quads) {
            *(float4 *)to_k = make_float4(x[0], x[1], x[2], x[3]);
            *(float4 *)to_v = make_float4(y[0], y[1], y[2], y[3]);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                to_k[e] = x[e];
                to_v[e] = y[e];
            }
        }
    }
}

}  // namespace

hipError_t launch_page_step(const PageStep &p, hipStream_t s)
{
    if (p.requests <= kPageThreads && p.max_tokens <= 8 * kPageThreads) {
        hipLaunchKernelGGL(page_small, dim3(1), dim3(kPageThreads), 0, s, p);
        return hipGetLastError();
    }
    hipLaunchKernelGGL(page_tables, dim3(1), dim3(kPageThreads), 0, s, p);
    hipLaunchKernelGGL(page_rows, dim3((unsigned)((p.max_tokens + 255ll) / 256)), dim3(256), 0, s, p);
    return hipGetLastError();
}

hipError_t launch_rope_angles(const int *positions, int count, const float *frequencies, int pairs, float magnitude,
    float2 *angles, hipStream_t s)
{
    const int64_t n = (int64_t)count * pairs;
    hipLaunchKernelGGL(rope_angles, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, positions, n, frequencies,
                       pairs, magnitude, angles);
    return hipGetLastError();
}

hipError_t launch_rope(const Rows &q, const Rows &k, int width, int count, const float2 *angles, int rotated,
    bool halves, hipStream_t s)
{
    const bool quads = quads_ok(q, width, rotated, halves, angles) && quads_ok(k, width, rotated, halves, angles);
    const int each = heads_each(count, q.heads + k.heads, width);
    const int q_parts = (q.heads + each - 1) / each, k_parts = (k.heads + each - 1) / each;
    hipLaunchKernelGGL(rope_rows, dim3((unsigned)count, (unsigned)(q_parts + k_parts)), dim3(256), 0, s, q, k, width,
                       angles, rotated, halves, q_parts, each, quads);
    return hipGetLastError();
}

hipError_t launch_kv8_store(const Kv8 &cache, const int *slots, int count, const float *k, int64_t k_stride,
    const float *v, int64_t v_stride, const float2 *angles, int rotated, bool halves, const Rows &q, hipStream_t s)
{
    const uintptr_t all = (uintptr_t)k | (uintptr_t)angles;
    const bool quads_k = (all & 15) == 0 && k_stride % 4 == 0 && rotated % (halves ? 32 : 16) == 0;
    const bool quads_q = quads_ok(q, cache.width, rotated, halves, angles);
    const int each = q.heads ? heads_each(count, q.heads, cache.width) : 1, parts = (q.heads + each - 1) / each;
    const int64_t work = (int64_t)count * cache.kv_heads;
    const int rows = work <= 2048 ? 1 : work <= 8192 ? 4 : 8;
    const int groups = (count + rows - 1) / rows, page = cache.page_tokens / rows;
    const int apart = page < groups ? page : groups, lines = (groups + apart - 1) / apart;
    const int64_t stores = (int64_t)lines * apart * 2 * cache.kv_heads;
    const Store args = {cache, slots, count, k, v, k_stride, v_stride, angles, rotated, halves, quads_k, quads_q, q, each,
                        parts, rows, apart, lines, (int)stores};
    const dim3 grid((unsigned)(stores + (int64_t)count * parts));
    switch (cache.width) {
    case 64: hipLaunchKernelGGL(kv8_store<64>, grid, dim3(256), 0, s, args); break;
    case 128: hipLaunchKernelGGL(kv8_store<128>, grid, dim3(256), 0, s, args); break;
    case 256: hipLaunchKernelGGL(kv8_store<256>, grid, dim3(256), 0, s, args); break;
    default: hipLaunchKernelGGL(kv8_store<512>, grid, dim3(256), 0, s, args); break;
    }
    return hipGetLastError();
}

hipError_t launch_kv8_load(const Kv8 &cache, const int *slots, int count, float *k, int64_t k_stride, float *v,
    int64_t v_stride, hipStream_t s)
{
    const bool quads = (((uintptr_t)k | (uintptr_t)v) & 15) == 0 && k_stride % 4 == 0 && v_stride % 4 == 0;
    const int64_t parts = ((int64_t)cache.kv_heads * cache.width + 1023) / 1024;
    const int rows = count * parts >= 8192 ? 16 : 4;
    hipLaunchKernelGGL(kv8_load, dim3((unsigned)((count + rows - 1) / rows), (unsigned)parts), dim3(256), 0, s, cache,
                       slots, count, rows, k, k_stride, v, v_stride, quads);
    return hipGetLastError();
}

}  // namespace fy
