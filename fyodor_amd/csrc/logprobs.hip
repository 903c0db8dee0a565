// Log probabilities of given tokens, entropies and the most likely tokens of
// rows of logits, and their entry points (include/fyodor_hip_logprobs.h).
//
// With M the largest logit that is not masked, z_j = scale (x_j - M) and
// S = sum e^z_j: ln p_j = z_j - ln S, and the entropy is ln S - sum z_j e^z_j / S.
#include <limits.h>
#include <math.h>

#include "../../include/fyodor_hip_logprobs.h"
#include "device.h"
#include "kernels.h"

namespace fy {
namespace {

// Workgroup: a row, read once for each of its results.
__global__ __launch_bounds__(256) void logprobs_simple(Logprobs a)
{
    const int row = blockIdx.x, tid = threadIdx.x;
    const float *x = a.logits + row * a.stride;
    __shared__ float sf[256];
    __shared__ double sd[256], se[256];
    __shared__ int si[256];
    auto at = [&](int i) { return a.mask && (a.mask[i >> 5] >> (i & 31) & 1u) ? -INFINITY : x[i]; };
    auto before = [](float x, int i, float y, int j) { return x > y || (x == y && i < j); };
    float m = -INFINITY;
    bool bad = false;
    for (int i = tid; i < a.n; i += 256) {
        const float v = at(i);
        bad |= !(v < INFINITY);
        m = fmaxf(m, v);
    }
    bad = __syncthreads_or(bad);
    sf[tid] = m;
    __syncthreads();
    for (int i = 0; i < 256; ++i) m = fmaxf(m, sf[i]);
    bad |= m == -INFINITY;
    const int token = a.tokens ? a.tokens[row] : -1;
    const bool given = (unsigned)token < (unsigned)a.n;
    const float xt = given ? at(token) : 0.f;
    double s = 0, t = 0;
    int rank = 0;
    for (int i = tid; i < a.n; i += 256) {
        const float v = at(i), z = (v - m) * a.scale, e = expf(z);
        s += e;
        if (e > 0.f) t += (double)z * e;
        rank += before(v, i, xt, token);
    }
    sd[tid] = s;
    se[tid] = t;
    si[tid] = rank;
    __syncthreads();
    s = t = rank = 0;
    for (int i = 0; i < 256; ++i) {
        s += sd[i];
        t += se[i];
        rank += si[i];
    }
    const double lse = log(s);
    const bool none = !given || xt == -INFINITY;
    if (tid == 0) {
        if (a.tokens) {
            a.logprobs[row] = !given ? 0.f : bad ? NAN : (float)(((double)xt - m) * a.scale - lse);
            if (a.ranks) a.ranks[row] = bad || none ? -1 : rank;
        }
        if (a.entropies) a.entropies[row] = bad ? NAN : (float)(lse - t / s);
    }
    float lv = INFINITY;
    int li = -1;
    for (int k = 0; k < a.top; ++k) {
        float best = -INFINITY;
        int bi = INT_MAX;
        for (int i = tid; i < a.n; i += 256) {
            const float v = at(i);
            if (before(lv, li, v, i) && before(v, i, best, bi)) {
                best = v;
                bi = i;
            }
        }
        __syncthreads();
        sf[tid] = best;
        si[tid] = bi;
        __syncthreads();
        for (int i = 0; i < 256; ++i)
            if (before(sf[i], si[i], best, bi)) {
                best = sf[i];
                bi = si[i];
            }
        if (tid == 0) {
            a.top_ids[(size_t)row * a.top + k] = bad || best == -INFINITY ? -1 : bi;
            a.top_logprobs[(size_t)row * a.top + k] = bad ? NAN : (float)(((double)best - m) * a.scale - lse);
        }
        lv = best;
        li = bi;
    }
}

}  // namespace

size_t logprobs_workspace(int, int, int)
{
    return 0;
}

hipError_t launch_logprobs(const Logprobs &a, void *, size_t, hipStream_t s)
{
    hipLaunchKernelGGL(logprobs_simple, dim3(a.count), dim3(256), 0, s, a);
    return hipGetLastError();
}

}  // namespace fy

namespace {

using namespace fy;

bool sizes_ok(size_t n, size_t count, size_t top)
{
    return n && n <= (size_t)1 << 24 && count && count <= (size_t)1 << 22 && top <= NYA_HIP_LOGPROBS_TOP;
}

// Arrays of 4-byte elements (0: none): a start and an end.
struct Array {
    uintptr_t from;
    size_t n;
    bool ok() const { return !(from & 3u); }
    bool apart(const Array &o) const { return !from || !o.from || from + 4 * n <= o.from || o.from + 4 * o.n <= from; }
};

}  // namespace

extern "C" {

NYA_HIP_EXPORT int nya_hip_logprobs_bytes(size_t n, size_t count, size_t top, size_t *bytes)
{
    if (!bytes || !sizes_ok(n, count, top)) return 1;
    *bytes = logprobs_workspace((int)n, (int)count, (int)top);
    return 0;
}

NYA_HIP_EXPORT int nya_hip_logprobs(uintptr_t logits, size_t stride, size_t n, size_t count, uintptr_t mask, float scale,
    uintptr_t tokens, uintptr_t logprobs, uintptr_t ranks, uintptr_t entropies, size_t top, uintptr_t top_ids,
    uintptr_t top_logprobs, uintptr_t workspace, size_t workspace_bytes, uintptr_t stream)
{
    if (!sizes_ok(n, count, top) || !logits || stride < n || stride > (size_t)INT_MAX || !(scale > 0) ||
        !isfinite(scale) || (workspace & 15u) || (!tokens && !entropies && !top) || (tokens && !logprobs) ||
        (top && (!top_ids || !top_logprobs)))
        return 1;
    const Array in[] = {{logits, (count - 1) * stride + n}, {mask, (n + 31) / 32}, {tokens, count}};
    const Array out[] = {{tokens ? logprobs : 0, count}, {tokens ? ranks : 0, count}, {entropies, count},
                         {top ? top_ids : 0, count * top}, {top ? top_logprobs : 0, count * top}};
    for (const Array &o : out) {
        if (!o.ok()) return 1;
        for (const Array &i : in)
            if (!i.ok() || !o.apart(i)) return 1;
        for (const Array &p : out)
            if (&p != &o && !o.apart(p)) return 1;
    }
    const Logprobs a = {(const float *)logits, (int64_t)stride, (int)n, (int)count, (const uint32_t *)mask, scale,
                        (const int *)tokens, (float *)logprobs, tokens ? (int *)ranks : nullptr, (float *)entropies,
                        (int)top, (int *)top_ids, (float *)top_logprobs};
    const hipError_t e = launch_logprobs(a, (void *)workspace, workspace ? workspace_bytes : 0, (hipStream_t)stream);
    return e == hipSuccess ? 0 : -(int)(e > 0 ? e : 1);
}

}  // extern "C"
