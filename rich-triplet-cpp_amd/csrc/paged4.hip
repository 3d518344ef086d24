// paged4.hip -- rows of keys and values into a 4-bit cache, and rows of any
// paged cache back out of it.
#include "paged4.hpp"
#include "paged_rows.hpp"
#include "rt_launch.hpp"

namespace rt_hip {
namespace {

// v of the lanes 1 and 2 away, in turn, within four.
template <class F>
__device__ __forceinline__ float of_four(float v, F op) {
    v = op(v, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0xb1, 0xf, 0xf, true)));
    return op(v, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x4e, 0xf, 0xf, true)));
}

// An f32 result rounded to f16.  (Opaque: the compiler would otherwise make one
// instruction of the product or sum and this, v_fma_mixlo_f16, which rounds once.)
__device__ __forceinline__ _Float16 to_f16(float x) {
    asm volatile("" : "+v"(x));
    return static_cast<_Float16>(x);
}

// Units of 8 values, four lanes to a group: (token, head, eight of the row), keys
// in blockIdx.y 0, values in 1.  Bound by the bytes.
template <class S, int HD>
__global__ __launch_bounds__(256) void k_paged4_append(const S* __restrict__ k, const S* __restrict__ v, PagedKv kv,
                                                       const int32_t* __restrict__ slots, uint32_t n_tokens,
                                                       int64_t src_stride) {
    using P = Page4<HD>;
    const uint32_t row_units = static_cast<uint32_t>(kv.n_kv) * (HD / 8);
    const uint32_t u = blockIdx.x * 256 + threadIdx.x;  // (the host keeps units below 2^31)
    const uint32_t t = u / row_units;
    if (t >= n_tokens) return;  // (row_units is a multiple of four: whole groups)
    const uint32_t c = u - t * row_units, head = c / (HD / 8), w = c % (HD / 8);
    const uint32_t slot = static_cast<uint32_t>(slots[t]);
    if (slot >= static_cast<uint32_t>(kv.n_pages) << kv.page_shift) return;  // no slot (-1), or none of this cache
    float x[8];
    load8((blockIdx.y ? v : k) + static_cast<int64_t>(t) * src_stride + c * 8, x);
    float lo = x[0], hi = x[0], far = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        lo = fminf(lo, x[e]);
        hi = fmaxf(hi, x[e]);
        far = fabsf(x[e]) <= 16384.0f ? far : 1.0f;  // (NaN too)
    }
    lo = of_four(lo, [](float a, float b) { return fminf(a, b); });
    hi = of_four(hi, [](float a, float b) { return fmaxf(a, b); });
    far = of_four(far, [](float a, float b) { return fmaxf(a, b); });
    // Every step rounded as it stands here: what the codes are does not depend on
    // who computes them.
    const _Float16 a = to_f16((hi - lo) * static_cast<float>(16.0 / 15.0));
    const _Float16 b = to_f16(lo - static_cast<float>(a));
    const float af = static_cast<float>(a), bf = static_cast<float>(b);
    const float steps = af > 0.0f ? 16.0f / af : 0.0f;
    uint32_t word = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float y = rintf((x[e] - bf) * steps) - 16.0f;
        const uint32_t code = static_cast<uint32_t>(fminf(fmaxf(y, 0.0f), 15.0f));
        word |= code_at(code, e);
    }
    uint32_t ab = static_cast<uint32_t>(__builtin_bit_cast(uint16_t, a)) | static_cast<uint32_t>(__builtin_bit_cast(uint16_t, b)) << 16;
    if (far != 0.0f) {
        ab = 0x7e007e00u;
        word = 0;
    }
    const uint32_t in_page = slot & ((1u << kv.page_shift) - 1);
    uint8_t* const base = static_cast<uint8_t*>(blockIdx.y ? kv.v : kv.k) +
                          static_cast<uint64_t>(slot >> kv.page_shift) * static_cast<uint64_t>(kv.page_stride) +
                          (static_cast<uint32_t>(P::kSlotAll) << kv.page_shift) * head;
    uint8_t* const codes = base + P::codes(in_page);
    uint8_t* const numbers = base + P::numbers(in_page, kv.page_shift);
    if (blockIdx.y == 0) {
        *reinterpret_cast<uint32_t*>(codes + P::key_word(in_page & 7, w)) = word;
        if (w % 4 == 0) *reinterpret_cast<uint32_t*>(numbers + P::key_number(in_page & 7, w / 4)) = ab;
    } else {
        *reinterpret_cast<uint32_t*>(codes + P::value_word(in_page & 7, w)) = word;
        uint16_t* const num = reinterpret_cast<uint16_t*>(numbers + P::value_number(in_page & 7, w / 4));
        if (w % 4 == 0) num[0] = static_cast<uint16_t>(ab);
        if (w % 4 == 1) num[8] = static_cast<uint16_t>(ab >> 16);
    }
}

// Units of 8 values as above: rows at `slots` to dense ones, zeros for a slot
// that is none of the cache's.  HD 0: a cache of D.
template <class S, class D, int HD>
__global__ __launch_bounds__(256) void k_paged_read(PagedKv kv, const int32_t* __restrict__ slots, uint32_t n_tokens,
                                                    uint32_t row_units, S* __restrict__ k, S* __restrict__ v,
                                                    int64_t dst_stride) {
    const uint32_t u = blockIdx.x * 256 + threadIdx.x;
    const uint32_t t = u / row_units;
    if (t >= n_tokens) return;
    const uint32_t c = u - t * row_units;
    const uint32_t slot = static_cast<uint32_t>(slots[t]);
    const uint32_t in_page = slot & ((1u << kv.page_shift) - 1);
    const uint8_t* const pages = static_cast<const uint8_t*>(blockIdx.y ? kv.v : kv.k);
    float x[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    if (slot < static_cast<uint32_t>(kv.n_pages) << kv.page_shift) {
        if constexpr (HD > 0) {
            using P = Page4<HD>;
            const uint32_t head = c / (HD / 8), w = c % (HD / 8);
            const uint8_t* const base = pages + static_cast<uint64_t>(slot >> kv.page_shift) * static_cast<uint64_t>(kv.page_stride) +
                                        (static_cast<uint32_t>(P::kSlotAll) << kv.page_shift) * head;
            const uint8_t* const codes = base + P::codes(in_page);
            const uint8_t* const numbers = base + P::numbers(in_page, kv.page_shift);
            uint32_t word, ab;
            if (blockIdx.y == 0) {
                word = *reinterpret_cast<const uint32_t*>(codes + P::key_word(in_page & 7, w));
                ab = *reinterpret_cast<const uint32_t*>(numbers + P::key_number(in_page & 7, w / 4));
            } else {
                word = *reinterpret_cast<const uint32_t*>(codes + P::value_word(in_page & 7, w));
                const uint16_t* const num = reinterpret_cast<const uint16_t*>(numbers + P::value_number(in_page & 7, w / 4));
                ab = num[0] | static_cast<uint32_t>(num[8]) << 16;
            }
            const u32x4 y = Codes().word(word, ab);
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = f16_bits_to_f32(y[e >> 1] >> (16 * (e & 1)) & 0xffffu);
        } else {
            load8(reinterpret_cast<const D*>(pages) + static_cast<int64_t>(slot >> kv.page_shift) * kv.page_stride +
                      (static_cast<int64_t>(in_page) * row_units + c) * 8, x);
        }
    }
    store8((blockIdx.y ? v : k) + static_cast<int64_t>(t) * dst_stride + c * 8, x);
}

unsigned blocks_of(int n_tokens, int units) {
    return static_cast<unsigned>((static_cast<int64_t>(n_tokens) * units + 255) / 256);
}

template <class S>
hipError_t run_append(const void* k, const void* v, int64_t stride, const PagedKv& kv, const int32_t* slots, int n,
                      hipStream_t s) {
    const auto kernel = kv.head_dim == 64 ? k_paged4_append<S, 64> : kv.head_dim == 128 ? k_paged4_append<S, 128> : k_paged4_append<S, 256>;
    hipLaunchKernelGGL(kernel, dim3(blocks_of(n, kv.n_kv * kv.head_dim / 8), 2), dim3(256), 0, s, static_cast<const S*>(k),
                       static_cast<const S*>(v), kv, slots, static_cast<uint32_t>(n), stride);
    return hipGetLastError();
}

template <class S>
hipError_t run_read(const PagedKv& kv, const int32_t* slots, int n, void* k, void* v, int64_t stride, hipStream_t s) {
    const int units = kv.n_kv * kv.head_dim / 8;
    const auto four = kv.head_dim == 64 ? k_paged_read<S, float, 64> : kv.head_dim == 128 ? k_paged_read<S, float, 128> : k_paged_read<S, float, 256>;
    const auto kernel = kv.dtype == RT_HIP_Q4KV ? four : kv.dtype == RT_HIP_F32 ? k_paged_read<S, float, 0>
                        : kv.dtype == RT_HIP_F16 ? k_paged_read<S, _Float16, 0> : k_paged_read<S, __bf16, 0>;
    hipLaunchKernelGGL(kernel, dim3(blocks_of(n, units), 2), dim3(256), 0, s, kv, slots, static_cast<uint32_t>(n),
                       static_cast<uint32_t>(units), static_cast<S*>(k), static_cast<S*>(v), stride);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_paged4_append(int src_dtype, const void* k, const void* v, int64_t src_stride, const PagedKv& kv,
                                const int32_t* slots, int n_tokens, hipStream_t s) {
    switch (src_dtype) {
        case RT_HIP_F32: return run_append<float>(k, v, src_stride, kv, slots, n_tokens, s);
        case RT_HIP_F16: return run_append<_Float16>(k, v, src_stride, kv, slots, n_tokens, s);
        default: return run_append<__bf16>(k, v, src_stride, kv, slots, n_tokens, s);
    }
}

hipError_t launch_paged_read(const PagedKv& kv, const int32_t* slots, int n_tokens, int dst_dtype, void* k, void* v,
                             int64_t dst_stride, hipStream_t s) {
    switch (dst_dtype) {
        case RT_HIP_F32: return run_read<float>(kv, slots, n_tokens, k, v, dst_stride, s);
        case RT_HIP_F16: return run_read<_Float16>(kv, slots, n_tokens, k, v, dst_stride, s);
        default: return run_read<__bf16>(kv, slots, n_tokens, k, v, dst_stride, s);
    }
}

}  // namespace rt_hip
