// Causal attention over a paged 4-bit cache (include/fyodor_hip_kv4.h).
#include "paged_attention.h"

namespace fy {
namespace {

// Workgroup (token and head, request) of one wavefront: a lane scores every
// 64th position and has every 64th element of the output.
template <int W>
__global__ __launch_bounds__(64) void kv4_simple(Kv4Attention a)
{
    const Kv4 &c = a.cache;
    const int r = blockIdx.y, token = blockIdx.x / a.heads, head = blockIdx.x % a.heads, lane = threadIdx.x;
    const int group = a.heads / c.kv_heads, kvh = head / group;
    const Request rq = request_of(a, r);
    if (token >= rq.rows / group) return;
    __shared__ float q[W];
    for (int d = lane; d < W; d += 64) q[d] = a.q[(rq.begin + token) * a.q_stride + (int64_t)head * W + d];
    __syncthreads();
    const int64_t p = rq.first + token, limit = min((int64_t)a.table_stride * c.page_tokens - 1, (int64_t)INT32_MAX - 128);
    const int last = (int)(p < 0 ? -1 : min(p, limit));
    const int first = (int)(a.window && p >= a.window ? min(p - a.window + 1, limit + 1) : 0);
    float m = -INFINITY, l = 0.f, o[W / 64] = {};
    bool saw = false;
    for (int at = first; at <= last; at += 64) {
        const int pos = at + lane, page = pos <= last ? a.table[(size_t)r * a.table_stride + pos / c.page_tokens] : -1;
        const bool there = (unsigned)page < (unsigned)c.pages;
        const int t = pos & (c.page_tokens - 1);
        const size_t place = (size_t)(there ? page : 0) * c.kv_heads + kvh;
        const uint8_t *keys = c.keys + place * (c.page_tokens * (W / 2));
        const uint16_t *steps = c.key_steps + place * (c.page_tokens * (W / 32));
        float s = 0.f;
        for (int b = 0; b < W / 32; ++b) {
            float sum = 0.f;
            for (int w = 0; w < 4; ++w) {
                const uint32_t word = *(const uint32_t *)(keys + (b * c.page_tokens + t) * 16 + 4 * w);
                for (int e = 0; e < 8; ++e)
                    sum += q[32 * b + 8 * w + e] * (float)((int)(word >> (e % 2 * 16 + e / 2 * 4) & 15u) - 8);
            }
            s += sum * f16_to_f32(steps[(t / 16 * (W / 32) + b) * 16 + t % 4 * 4 + t % 16 / 4]);
        }
        saw |= there;
        s = there ? s * a.scale : -INFINITY;
        const float top = fmaxf(m, wave_reduce<true>(s)), base = top == -INFINITY ? 0.f : top;
        const float alpha = expf(m - base), e = expf(s - base);
        m = top;
        l = l * alpha + e;
        for (int i = 0; i < W / 64; ++i) o[i] *= alpha;
        for (int j = 0; j < 64 && at + j <= last; ++j) {
            const int pg = __builtin_amdgcn_readlane(page, j);
            if ((unsigned)pg >= (unsigned)c.pages) continue;
            const float w = lane_value(e, j);
            const int tj = (at + j) & (c.page_tokens - 1);
            const size_t pl = (size_t)pg * c.kv_heads + kvh;
            for (int i = 0; i < W / 64; ++i) {
                const int d = 64 * i + lane;
                const uint32_t n = *(const uint16_t *)(c.values + pl * (c.page_tokens * (W / 2)) + ((tj / 8 * (W / 4) + d / 4) * 8 + tj % 8) * 2);
                o[i] += w * (float)((int)(n >> (4 * (d % 4)) & 15u) - 8) *
                        f16_to_f32(c.value_steps[pl * (c.page_tokens * (W / 32)) + d / 32 * c.page_tokens + tj]);
            }
        }
    }
    l = wave_sum(l);
    if (m == -INFINITY && __builtin_amdgcn_ballot_w64(saw)) m = -FLT_MAX;
    float *out = a.out + (rq.begin + token) * a.out_stride + (int64_t)head * W + lane;
    for (int i = 0; i < W / 64; ++i) out[64 * i] = o[i] * inverse_of(l, m);
}

}  // namespace

size_t kv4_attention_workspace(const Kv4Attention &)
{
    return 0;
}

hipError_t launch_kv4_attention(const Kv4Attention &a, void *, size_t, hipStream_t s)
{
    const dim3 grid((unsigned)((int64_t)a.max_tokens * a.heads), a.requests);
    switch (a.cache.width) {
    case 64: hipLaunchKernelGGL((kv4_simple<64>), grid, dim3(64), 0, s, a); break;
    case 128: hipLaunchKernelGGL((kv4_simple<128>), grid, dim3(64), 0, s, a); break;
    case 256: hipLaunchKernelGGL((kv4_simple<256>), grid, dim3(64), 0, s, a); break;
    default: hipLaunchKernelGGL((kv4_simple<512>), grid, dim3(64), 0, s, a); break;
    }
    return hipGetLastError();
}

}  // namespace fy
