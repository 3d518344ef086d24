// paged_attention.hip -- attention of the new tokens of many requests over a
// KV cache in pages.
//
// Row i of request s (n rows, kv_len keys) has position kv_len - n + i and
// sees the keys (position - window, position]:
//   out = sum_j softmax_j(scale q . k_j) v_j,
// zeros where it sees none.  Key j of the request is row j % page of page
// table[s][j / page].
//
// One wave per (row, head): lane l holds values l, l + 64, .. of q and of the
// accumulator, and takes the keys one by one with an online softmax.
#include "rt_common.hpp"
#include "rt_launch.hpp"

namespace rt_hip {
namespace {

constexpr float kLog2e = 1.44269504088896341f;

template <class Q, class T, int HD>
__global__ __launch_bounds__(64) void k_paged_attn(PagedAttn p) {
    constexpr int N = HD / 64;
    const int t = blockIdx.x, h = blockIdx.y, lane = threadIdx.x;
    int s = 0;
    while (s < p.n_seq && p.q_start[s + 1] <= t) ++s;
    if (s == p.n_seq || t < p.q_start[s]) return;
    const int cap = static_cast<int>(p.cols << p.kv.page_shift);
    const int len = min(max(p.kv_len[s], 0), cap);
    const int pos = len - (p.q_start[s + 1] - t);
    const int from = p.window ? max(0, pos - p.window + 1) : 0;
    const int kvh = h / (p.n_q / p.kv.n_kv);
    const int64_t row = static_cast<int64_t>(p.kv.n_kv) * HD;
    float q[N], o[N], m = -__builtin_inff(), l = 0.0f;
#pragma unroll
    for (int e = 0; e < N; ++e) {
        q[e] = static_cast<float>(static_cast<const Q*>(p.q)[t * p.q_stride + h * HD + e * 64 + lane]) * (p.scale * kLog2e);
        o[e] = 0.0f;
    }
    for (int j = from; j <= pos; ++j) {
        const int page = p.table[s * p.cols + (j >> p.kv.page_shift)];
        const bool ok = static_cast<uint32_t>(page) < static_cast<uint32_t>(p.kv.n_pages);
        const int64_t at = (ok ? page : 0) * p.kv.page_stride + (j & ((1 << p.kv.page_shift) - 1)) * row + kvh * HD + lane;
        float d = 0.0f, v[N];
#pragma unroll
        for (int e = 0; e < N; ++e) {
            d += q[e] * (ok ? static_cast<float>(static_cast<const T*>(p.kv.k)[at + e * 64]) : 0.0f);
            v[e] = ok ? static_cast<float>(static_cast<const T*>(p.kv.v)[at + e * 64]) : 0.0f;
        }
        d = segment_sum<64>(d);
        const float mn = fmaxf(m, d), mu = mn == -__builtin_inff() ? 0.0f : mn;
        const float a = __builtin_amdgcn_exp2f(m - mu), b = __builtin_amdgcn_exp2f(d - mu);
        l = l * a + b;
#pragma unroll
        for (int e = 0; e < N; ++e) o[e] = o[e] * a + b * v[e];
        m = mn;
    }
#pragma unroll
    for (int e = 0; e < N; ++e)
        static_cast<Q*>(p.out)[t * p.out_stride + h * HD + e * 64 + lane] = static_cast<Q>(l == 0.0f ? 0.0f : o[e] / l);
}

template <class Q, class T>
hipError_t run(const PagedAttn& p, hipStream_t s) {
    const dim3 grid(static_cast<unsigned>(p.n_tokens), static_cast<unsigned>(p.n_q));
    switch (p.kv.head_dim) {
        case 64: hipLaunchKernelGGL((k_paged_attn<Q, T, 64>), grid, dim3(64), 0, s, p); break;
        case 128: hipLaunchKernelGGL((k_paged_attn<Q, T, 128>), grid, dim3(64), 0, s, p); break;
        default: hipLaunchKernelGGL((k_paged_attn<Q, T, 256>), grid, dim3(64), 0, s, p); break;
    }
    return hipGetLastError();
}

}  // namespace

size_t paged_attention_workspace(const PagedAttn&) { return 0; }

hipError_t launch_paged_attention(const PagedAttn& p, void*, uint32_t*, hipStream_t s) {
    if (p.dtype == RT_HIP_BF16) return run<__bf16, __bf16>(p, s);
    if (p.dtype == RT_HIP_F16) return run<_Float16, _Float16>(p, s);
    switch (p.kv.dtype) {
        case RT_HIP_F32: return run<float, float>(p, s);
        case RT_HIP_F16: return run<float, _Float16>(p, s);
        default: return run<float, __bf16>(p, s);
    }
}

}  // namespace rt_hip
