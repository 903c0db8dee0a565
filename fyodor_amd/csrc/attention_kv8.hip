// Causal attention over a paged 8-bit cache (include/fyodor_hip_serving.h).
#include <math.h>

#include "device.h"
#include "serving.h"

namespace fy {
namespace {

// Row j of request r and the positions [first, last] it attends (last < first:
// none).
struct Seen {
    int row, first, last;
};

__device__ __forceinline__ Seen seen_by(const Kv8Attention &a, int r, int j)
{
    const int begin = max(a.starts[r], 0), end = min(a.starts[r + 1], a.count);
    Seen s = {-1, 0, -1};
    if (j >= end - begin) return s;
    s.row = begin + j;
    const int64_t most = (int64_t)a.table_stride * a.cache.page_tokens;
    const int64_t p = (int64_t)a.lengths[r] - (a.starts[r + 1] - (int64_t)begin) + j;
    s.last = (int)(p < 0 ? -1 : p < most ? p : most - 1);
    s.first = a.window && p >= a.window ? (int)(p - a.window + 1) : 0;
    return s;
}

// One wavefront per (row, head): 64 positions at a time, a lane each.
template <int W>
__global__ __launch_bounds__(64) void kv8_attention(Kv8Attention a)
{
    __shared__ float qs[W];
    const int lane = threadIdx.x, head = blockIdx.x % a.heads, j = blockIdx.x / a.heads, r = blockIdx.y;
    const Seen seen = seen_by(a, r, j);
    if (seen.row < 0) return;
    const Kv8 &c = a.cache;
    const int kvh = head / (a.heads / c.kv_heads);
    const int *table = a.table + (size_t)r * a.table_stride;
    for (int d = lane; d < W; d += 64) qs[d] = a.q[seen.row * a.q_stride + (int64_t)head * W + d];
    __syncthreads();
    float m = -INFINITY, l = 0.f, o[W / 64] = {};
    for (int t0 = seen.first; t0 <= seen.last; t0 += 64) {
        const int t = t0 + lane;
        int page = -1;
        if (t <= seen.last) page = table[t / c.page_tokens];
        const bool there = (unsigned)page < (unsigned)c.pages;
        const size_t place = there ? (size_t)page * c.kv_heads + kvh : 0;
        float s = -INFINITY;
        if (there) {
            const int8_t *codes = c.keys + place * c.page_tokens * W + (size_t)(t % c.page_tokens) * 16;
            float dot = 0.f;
            for (int d = 0; d < W; ++d) dot += qs[d] * (float)codes[(size_t)(d >> 4) * c.page_tokens * 16 + (d & 15)];
            s = dot * (c.key_scales[place] * a.scale);
        }
        const uint64_t any = __builtin_amdgcn_ballot_w64(there);
        if (!any) continue;
        const float next = fmaxf(m, wave_reduce<true>(s)), base = next == -INFINITY ? 0.f : next;
        const float p = there ? expf(s - base) : 0.f, alpha = expf(m - base);
        l = l * alpha + wave_sum(p);
        m = next;
        for (int e = 0; e < W / 64; ++e) o[e] *= alpha;
        const float weight = there ? p * c.value_scales[place] : 0.f;
        for (int i = 0; i < 64; ++i) {
            if (!(any >> i & 1)) continue;
            const float w = lane_value(weight, i);
            const size_t pl = (size_t)__builtin_amdgcn_readlane(page, i) * c.kv_heads + kvh;
            const int tt = (t0 + i) % c.page_tokens;
            const int8_t *codes = c.values + pl * c.page_tokens * W + (size_t)(tt >> 4) * W * 16 + (tt & 15);
            for (int e = 0; e < W / 64; ++e) o[e] += w * (float)codes[(size_t)(lane + 64 * e) * 16];
        }
    }
    for (int e = 0; e < W / 64; ++e)
        a.out[seen.row * a.out_stride + (int64_t)head * W + lane + 64 * e] = l == 0.f ? 0.f : o[e] / l;
}

}  // namespace

size_t kv8_attention_workspace(int requests, int max_tokens, int max_length, int heads, int kv_heads, int width,
    int window)
{
    return 0;
}

hipError_t launch_kv8_attention(const Kv8Attention &a, void *workspace, size_t workspace_bytes, hipStream_t s)
{
    const dim3 grid((unsigned)(a.max_tokens * a.heads), (unsigned)a.requests);
    switch (a.cache.width) {
    case 64: hipLaunchKernelGGL(kv8_attention<64>, grid, dim3(64), 0, s, a); break;
    case 128: hipLaunchKernelGGL(kv8_attention<128>, grid, dim3(64), 0, s, a); break;
    case 256: hipLaunchKernelGGL(kv8_attention<256>, grid, dim3(64), 0, s, a); break;
    default: hipLaunchKernelGGL(kv8_attention<512>, grid, dim3(64), 0, s, a); break;
    }
    return hipGetLastError();
}

}  // namespace fy
