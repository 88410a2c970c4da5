// paged_attn.hip -- attention of each request's new tokens over its pages of the cache.
//
// For a token at position i and a query head h over KV head h / group:
//     s_j = scale * q . k_j;  with a cap s_j = cap * tanh(s_j / cap);  with slopes s_j -= slope_h * |i - j|
//     o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m)   over the positions j that i sees (paged_sees), m their greatest s_j
// A token that sees nothing gets zeros.
#include "device_util.h"
#include "paged.h"

namespace mg {

// 4 ints a request: first row, rows, length, prefix -- clamped, so that no later read depends on what the caller's arrays held
__global__ __launch_bounds__(256) void paged_plan_kernel(PagedPlan p) {
    const int r = blockIdx.x * 256 + threadIdx.x;
    if (r >= p.nReqs) return;
    const int first = max(0, min(p.rowStart[r], p.rows)), last = max(first, min(p.rowStart[r + 1], p.rows));
    const int len = max(0, min(p.lens[r], p.maxLen));
    reinterpret_cast<int4*>(p.reqs)[r] = make_int4(first, last - first, len, p.prefixLens ? max(0, min(p.prefixLens[r], len)) : 0);
}
hipError_t launch_paged_plan(const PagedPlan& p, hipStream_t s) {
    if (p.nReqs == 0) return hipSuccess;
    hipLaunchKernelGGL(paged_plan_kernel, dim3((p.nReqs + 255) / 256), dim3(256), 0, s, p);
    return hipGetLastError();
}

// A workgroup a row and query head; its four waves take every fourth position.
template <typename KVT, int HD>
__global__ __launch_bounds__(WG) void paged_attn_kernel(PagedAttention p) {
    constexpr int E = HD / 64;
    __shared__ float sm[4], sl[4], so[4][HD];
    const int row = blockIdx.x, head = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int4 rq = make_int4(0, 0, 0, 0);
    int r = 0;
    for (; r < p.nReqs; r++) {
        rq = reinterpret_cast<const int4*>(p.reqs)[r];
        if (row >= rq.x && row < rq.x + rq.y) break;
    }
    if (r == p.nReqs) return;                      // a row behind the last request's
    const int pos = rq.z - rq.y + row - rq.x;
    const int kvh = head / p.g.group;
    float q[E], o[E];
    for (int e = 0; e < E; e++) { q[e] = p.q[(size_t)row * p.ldq + (size_t)head * HD + e * 64 + lane]; o[e] = 0.f; }
    const float slope = p.slopes ? p.slopes[head] : 0.f;
    float m = -INFINITY, l = 0.f;
    for (int j = wave; j < rq.z; j += 4) {
        if (!paged_sees(pos, j, rq.z, p.window, rq.w)) continue;
        const int page = p.table[(size_t)r * p.g.width + (j >> p.g.pageShift)];
        if (page < 0 || page >= p.g.nPages) continue;
        const size_t at = ((size_t)page * p.g.pageSize + (j & (p.g.pageSize - 1))) * p.g.kvDim + (size_t)kvh * HD + lane;
        float s = 0.f;
        for (int e = 0; e < E; e++) s = fmaf(q[e], (float)static_cast<const KVT*>(p.K)[at + e * 64], s);
        s = wave_sum(s) * p.scale;
        if (p.softcap > 0.f) s = p.softcap * tanhf(s / p.softcap);
        if (p.slopes) s -= slope * (float)abs(pos - j);
        const float mNew = fmaxf(m, s);
        const float base = mNew == -INFINITY ? 0.f : mNew;       // (a NaN among the scores stays one)
        const float corr = expf(m - base), w = expf(s - base);
        l = l * corr + w;
        for (int e = 0; e < E; e++) o[e] = fmaf(w, (float)static_cast<const KVT*>(p.V)[at + e * 64], o[e] * corr);
        m = mNew;
    }
    if (lane == 0) { sm[wave] = m; sl[wave] = l; }
    for (int e = 0; e < E; e++) so[wave][e * 64 + lane] = o[e];
    __syncthreads();
    if (tid >= HD) return;
    const float M = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
    float num = 0.f, den = 0.f;
    for (int w = 0; w < 4; w++) {
        const float f = expf(sm[w] - (M == -INFINITY ? 0.f : M));
        num = fmaf(f, so[w][tid], num);
        den = fmaf(f, sl[w], den);
    }
    p.out[(size_t)row * p.ldo + (size_t)head * HD + tid] = den == 0.f ? num : num / den;
}
hipError_t launch_paged_attention(const PagedAttention& p0, hipStream_t s) {
    PagedAttention p = p0;
    if (p.scale == 0.f) p.scale = 1.0f / sqrtf((float)p.g.headDim);
    const dim3 grid((unsigned)p.rows, (unsigned)p.g.nHeads);
    if (p.g.kvHalf) {
        if (p.g.headDim == 64) hipLaunchKernelGGL((paged_attn_kernel<_Float16, 64>), grid, dim3(WG), 0, s, p);
        else hipLaunchKernelGGL((paged_attn_kernel<_Float16, 128>), grid, dim3(WG), 0, s, p);
    } else {
        if (p.g.headDim == 64) hipLaunchKernelGGL((paged_attn_kernel<float, 64>), grid, dim3(WG), 0, s, p);
        else hipLaunchKernelGGL((paged_attn_kernel<float, 128>), grid, dim3(WG), 0, s, p);
    }
    return hipGetLastError();
}

}  // namespace mg
