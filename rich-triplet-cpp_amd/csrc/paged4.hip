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

// A 4 x 4 square of words turned over in four neighbouring lanes: word i of lane
// j becomes word j of lane i.
__device__ __forceinline__ u32x4 turned(u32x4 x) {
    const bool odd = threadIdx.x & 1, upper = threadIdx.x & 2;
    auto swap = [](uint32_t& a, uint32_t& b, bool second, auto from) {
        const uint32_t got = from(second ? a : b);
        (second ? a : b) = got;
    };
    uint32_t a = x[0], b = x[1], c = x[2], d = x[3];
    auto one = [](uint32_t y) { return static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(y), 0xb1, 0xf, 0xf, true)); };
    auto two = [](uint32_t y) { return static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(y), 0x4e, 0xf, 0xf, true)); };
    swap(a, b, odd, one);
    swap(c, d, odd, one);
    swap(a, c, upper, two);
    swap(b, d, upper, two);
    return u32x4{a, b, c, d};
}

// Eight values as a word of codes, and the two numbers (a low, b high) of the
// group that four neighbouring lanes hold.
__device__ __forceinline__ void encode(const float (&x)[8], uint32_t* word, uint32_t* ab) {
    float lo = x[0], hi = x[0];  // (NaN if one is)
#pragma unroll
    for (int e = 1; e < 8; ++e) {
        lo = __builtin_elementwise_minimum(lo, x[e]);
        hi = __builtin_elementwise_maximum(hi, x[e]);
    }
    lo = of_four(lo, [](float a, float b) { return __builtin_elementwise_minimum(a, b); });
    hi = of_four(hi, [](float a, float b) { return __builtin_elementwise_maximum(a, b); });
    // Every step rounded as it stands here: what the codes are does not depend on
    // who computes them.
    const _Float16 a = to_f16((hi - lo) * static_cast<float>(16.0 / 15.0));
    const _Float16 b = to_f16(lo - static_cast<float>(a));
    const float af = static_cast<float>(a), bf = static_cast<float>(b);
    const float steps = af > 0.0f ? 16.0f / af : 0.0f;
    // rint(t) - 16 as the low bits of t + 2^23 - 16, t in 16..31: that sum is rounded
    // to whole numbers, ties to even.  (What the shifts bring along is above bit 23.)
    uint32_t half[2] = {0, 0};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float t = __builtin_amdgcn_fmed3f((x[e] - bf) * steps, 16.0f, 31.0f);
        half[e & 1] |= __float_as_uint(t + 8388592.0f) << (4 * (e >> 1));
    }
    *word = turned_codes(__builtin_amdgcn_perm(half[1], half[0], 0x05040100u));
    *ab = static_cast<uint32_t>(__builtin_bit_cast(uint16_t, a)) | static_cast<uint32_t>(__builtin_bit_cast(uint16_t, b)) << 16;
    if (!(hi <= 16384.0f) || !(lo >= -16384.0f)) {
        *ab = 0x7e007e00u;
        *word = 0;
    }
}

// Four tokens whose slots are four in a row of those whose words lie together.
template <int U>
__device__ __forceinline__ bool in_a_row(const uint32_t (&slot)[U], uint32_t n_slots) {
    bool yes = U == 4 && slot[0] % 4 == 0 && slot[0] < n_slots;
#pragma unroll
    for (int i = 1; i < U; ++i) yes &= slot[i] == slot[0] + i;
    return yes;
}

// A thread has one word of eight values in U tokens, four lanes a group: (U
// tokens, head, word); keys in blockIdx.y 0, values in 1.  All it reads is asked
// for at once.  Four tokens in a row of slots are written in 16 bytes a lane, any
// others word by word.  Bound by the bytes: 32768 tokens of 8 heads of 128 in
// bf16 are 176 MB in 31 us, 5.7 TB/s; few tokens by the start of a launch.
template <class S, int HD, int U>
__global__ __launch_bounds__(256) void k_paged4_append(const S* __restrict__ k, const S* __restrict__ v, PagedKv kv,
                                                       const int32_t* __restrict__ slots, uint32_t n_tokens,
                                                       int64_t src_stride) {
    using P = Page4<HD>;
    const uint32_t row_units = static_cast<uint32_t>(kv.n_kv) * (HD / 8);
    const uint32_t u = blockIdx.x * 256 + threadIdx.x;  // (the host keeps units below 2^31)
    const uint32_t t0 = u / row_units * U;
    if (t0 >= n_tokens) return;  // (row_units is a multiple of four: whole groups)
    const uint32_t c = u % row_units, head = c / (HD / 8), w = c % (HD / 8);
    const uint32_t n_slots = static_cast<uint32_t>(kv.n_pages) << kv.page_shift;
    uint32_t slot[U];
    float x[U][8];
#pragma unroll
    for (int i = 0; i < U; ++i) {
        const uint32_t t = min(t0 + i, n_tokens - 1);
        slot[i] = static_cast<uint32_t>(slots[t]);
        load8((blockIdx.y ? v : k) + static_cast<int64_t>(t) * src_stride + c * 8, x[i]);
        if (t0 + i >= n_tokens) slot[i] = ~0u;
    }
    uint32_t word[U], ab[U];
#pragma unroll
    for (int i = 0; i < U; ++i) encode(x[i], &word[i], &ab[i]);
    auto base = [&](uint32_t slot) {
        return static_cast<uint8_t*>(blockIdx.y ? kv.v : kv.k) +
               static_cast<uint64_t>(slot >> kv.page_shift) * static_cast<uint64_t>(kv.page_stride) +
               (static_cast<uint32_t>(P::kSlotAll) << kv.page_shift) * head;
    };
    if (in_a_row(slot, n_slots)) {
        const uint32_t in_page = slot[0] & ((1u << kv.page_shift) - 1), four = in_page & 7;
        uint8_t* const codes = base(slot[0]) + P::codes(in_page);
        uint8_t* const numbers = base(slot[0]) + P::numbers(in_page, kv.page_shift);
        const u32x4 words = {word[0], word[U > 1], word[U > 2 ? 2 : 0], word[U > 3 ? 3 : 0]};
        const u32x4 all = {ab[0], ab[U > 1], ab[U > 2 ? 2 : 0], ab[U > 3 ? 3 : 0]};
        if (blockIdx.y == 0) {
            *reinterpret_cast<u32x4*>(codes + P::key_word(four + w % 4, w & ~3u)) = turned(words);
            if (w % 4 == 0) *reinterpret_cast<u32x4*>(numbers + P::key_number(four, w / 4)) = all;
        } else {
            *reinterpret_cast<u32x4*>(codes + P::value_word(four, w)) = words;
            u32x2* const num = reinterpret_cast<u32x2*>(numbers + P::value_number(four, w / 4));
            if (w % 4 == 0) num[0] = u32x2{(all[0] & 0xffffu) | all[1] << 16, (all[2] & 0xffffu) | all[3] << 16};
            if (w % 4 == 1) num[2] = u32x2{all[0] >> 16 | (all[1] & 0xffff0000u), all[2] >> 16 | (all[3] & 0xffff0000u)};
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
        if (slot[i] >= n_slots) continue;  // no slot (-1), or none of this cache
        const uint32_t in_page = slot[i] & ((1u << kv.page_shift) - 1);
        uint8_t* const codes = base(slot[i]) + P::codes(in_page);
        uint8_t* const numbers = base(slot[i]) + P::numbers(in_page, kv.page_shift);
        if (blockIdx.y == 0) {
            *reinterpret_cast<uint32_t*>(codes + P::key_word(in_page & 7, w)) = word[i];
            if (w % 4 == 0) *reinterpret_cast<uint32_t*>(numbers + P::key_number(in_page & 7, w / 4)) = ab[i];
        } else {
            *reinterpret_cast<uint32_t*>(codes + P::value_word(in_page & 7, w)) = word[i];
            uint16_t* const num = reinterpret_cast<uint16_t*>(numbers + P::value_number(in_page & 7, w / 4));
            if (w % 4 == 0) num[0] = static_cast<uint16_t>(ab[i]);
            if (w % 4 == 1) num[8] = static_cast<uint16_t>(ab[i] >> 16);
        }
    }
}

// The same units: rows at `slots` to dense ones, zeros for a slot that is none of
// the cache's.  HD 0: a cache of D.  Those tokens back into bf16 rows: 28 us, 6.2 TB/s.
template <class S, class D, int HD, int U>
__global__ __launch_bounds__(256) void k_paged_read(PagedKv kv, const int32_t* __restrict__ slots, uint32_t n_tokens,
                                                    uint32_t row_units, S* __restrict__ k, S* __restrict__ v,
                                                    int64_t dst_stride) {
    const uint32_t u = blockIdx.x * 256 + threadIdx.x;
    const uint32_t t0 = u / row_units * U;
    if (t0 >= n_tokens) return;
    const uint32_t c = u % row_units;
    const uint32_t n_slots = static_cast<uint32_t>(kv.n_pages) << kv.page_shift;
    const uint8_t* const pages = static_cast<const uint8_t*>(blockIdx.y ? kv.v : kv.k);
    uint32_t slot[U];
#pragma unroll
    for (int i = 0; i < U; ++i) slot[i] = static_cast<uint32_t>(slots[min(t0 + i, n_tokens - 1)]);
    float x[U][8] = {};
    if constexpr (HD > 0) {
        using P = Page4<HD>;
        const uint32_t head = c / (HD / 8), w = c % (HD / 8);
        auto base = [&](uint32_t slot) {
            return pages + static_cast<uint64_t>(slot >> kv.page_shift) * static_cast<uint64_t>(kv.page_stride) +
                   (static_cast<uint32_t>(P::kSlotAll) << kv.page_shift) * head;
        };
        uint32_t word[U] = {}, ab[U] = {};
        if (in_a_row(slot, n_slots)) {
            const uint32_t in_page = slot[0] & ((1u << kv.page_shift) - 1), four = in_page & 7;
            const uint8_t* const codes = base(slot[0]) + P::codes(in_page);
            const uint8_t* const numbers = base(slot[0]) + P::numbers(in_page, kv.page_shift);
            u32x4 words, all;
            if (blockIdx.y == 0) {
                words = turned(*reinterpret_cast<const u32x4*>(codes + P::key_word(four + w % 4, w & ~3u)));
                all = *reinterpret_cast<const u32x4*>(numbers + P::key_number(four, w / 4));
            } else {
                words = *reinterpret_cast<const u32x4*>(codes + P::value_word(four, w));
                const u32x2* const num = reinterpret_cast<const u32x2*>(numbers + P::value_number(four, w / 4));
                const u32x2 a = num[0], b = num[2];
                all = u32x4{(a[0] & 0xffffu) | b[0] << 16, a[0] >> 16 | (b[0] & 0xffff0000u), (a[1] & 0xffffu) | b[1] << 16,
                            a[1] >> 16 | (b[1] & 0xffff0000u)};
            }
#pragma unroll
            for (int i = 0; i < U; ++i) {
                word[i] = words[i];
                ab[i] = all[i];
            }
        } else {
#pragma unroll
            for (int i = 0; i < U; ++i) {
                if (slot[i] >= n_slots) continue;  // (codes and numbers of 0: zeros)
                const uint32_t in_page = slot[i] & ((1u << kv.page_shift) - 1);
                const uint8_t* const codes = base(slot[i]) + P::codes(in_page);
                const uint8_t* const numbers = base(slot[i]) + P::numbers(in_page, kv.page_shift);
                if (blockIdx.y == 0) {
                    word[i] = *reinterpret_cast<const uint32_t*>(codes + P::key_word(in_page & 7, w));
                    ab[i] = *reinterpret_cast<const uint32_t*>(numbers + P::key_number(in_page & 7, w / 4));
                } else {
                    word[i] = *reinterpret_cast<const uint32_t*>(codes + P::value_word(in_page & 7, w));
                    const uint16_t* const num = reinterpret_cast<const uint16_t*>(numbers + P::value_number(in_page & 7, w / 4));
                    ab[i] = num[0] | static_cast<uint32_t>(num[8]) << 16;
                }
            }
        }
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const u32x4 y = Codes().word(word[i], ab[i]);
#pragma unroll
            for (int e = 0; e < 8; ++e) x[i][e] = f16_bits_to_f32(y[e >> 1] >> (16 * (e & 1)) & 0xffffu);
        }
    } else {
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const uint32_t in_page = slot[i] & ((1u << kv.page_shift) - 1);
            if (slot[i] < n_slots)
                load8(reinterpret_cast<const D*>(pages) + static_cast<int64_t>(slot[i] >> kv.page_shift) * kv.page_stride +
                          (static_cast<int64_t>(in_page) * row_units + c) * 8, x[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < U; ++i)
        if (t0 + i < n_tokens) store8((blockIdx.y ? v : k) + static_cast<int64_t>(t0 + i) * dst_stride + c * 8, x[i]);
}

// Four tokens to a thread once that leaves every SIMD a wave: launching waves is
// what costs then (rows of 8 heads of 128, bf16, append and read back: 8192 tokens
// 9.6 and 9.5 us, by single tokens 12.7 and 12.1; 1024 tokens 3.3 and 3.2, 3.6 and
// 3.1).  Fewer tokens are over in the time of a few loads (64: 3.0 and 2.7, by
// single ones 2.5 and 2.4).
bool by_four(int n_tokens, int units) { return static_cast<int64_t>(n_tokens) * units >= 512ll * device_info().cus; }
unsigned blocks_of(int n_tokens, int units, int per) {
    return static_cast<unsigned>(((static_cast<int64_t>(n_tokens) + per - 1) / per * units + 255) / 256);
}

template <class S, int U>
hipError_t run_append(const void* k, const void* v, int64_t stride, const PagedKv& kv, const int32_t* slots, int n,
                      hipStream_t s) {
    const auto kernel = kv.head_dim == 64 ? k_paged4_append<S, 64, U> : kv.head_dim == 128 ? k_paged4_append<S, 128, U> : k_paged4_append<S, 256, U>;
    hipLaunchKernelGGL(kernel, dim3(blocks_of(n, kv.n_kv * kv.head_dim / 8, U), 2), dim3(256), 0, s, static_cast<const S*>(k),
                       static_cast<const S*>(v), kv, slots, static_cast<uint32_t>(n), stride);
    return hipGetLastError();
}

template <class S>
hipError_t run_append_by(const void* k, const void* v, int64_t stride, const PagedKv& kv, const int32_t* slots, int n,
                         hipStream_t s) {
    return by_four(n, kv.n_kv * kv.head_dim / 8) ? run_append<S, 4>(k, v, stride, kv, slots, n, s)
                                                 : run_append<S, 1>(k, v, stride, kv, slots, n, s);
}

template <class S, int U>
hipError_t run_read(const PagedKv& kv, const int32_t* slots, int n, void* k, void* v, int64_t stride, hipStream_t s) {
    const int units = kv.n_kv * kv.head_dim / 8;
    const auto four = kv.head_dim == 64 ? k_paged_read<S, float, 64, U> : kv.head_dim == 128 ? k_paged_read<S, float, 128, U>
                                                                                              : k_paged_read<S, float, 256, U>;
    const auto kernel = kv.dtype == RT_HIP_Q4KV ? four : kv.dtype == RT_HIP_F32 ? k_paged_read<S, float, 0, U>
                        : kv.dtype == RT_HIP_F16 ? k_paged_read<S, _Float16, 0, U> : k_paged_read<S, __bf16, 0, U>;
    hipLaunchKernelGGL(kernel, dim3(blocks_of(n, units, U), 2), dim3(256), 0, s, kv, slots, static_cast<uint32_t>(n),
                       static_cast<uint32_t>(units), static_cast<S*>(k), static_cast<S*>(v), stride);
    return hipGetLastError();
}

template <class S>
hipError_t run_read_by(const PagedKv& kv, const int32_t* slots, int n, void* k, void* v, int64_t stride, hipStream_t s) {
    return by_four(n, kv.n_kv * kv.head_dim / 8) ? run_read<S, 4>(kv, slots, n, k, v, stride, s)
                                                 : run_read<S, 1>(kv, slots, n, k, v, stride, s);
}

}  // namespace

hipError_t launch_paged4_append(int src_dtype, const void* k, const void* v, int64_t src_stride, const PagedKv& kv,
                                const int32_t* slots, int n_tokens, hipStream_t s) {
    switch (src_dtype) {
        case RT_HIP_F32: return run_append_by<float>(k, v, src_stride, kv, slots, n_tokens, s);
        case RT_HIP_F16: return run_append_by<_Float16>(k, v, src_stride, kv, slots, n_tokens, s);
        default: return run_append_by<__bf16>(k, v, src_stride, kv, slots, n_tokens, s);
    }
}

hipError_t launch_paged_read(const PagedKv& kv, const int32_t* slots, int n_tokens, int dst_dtype, void* k, void* v,
                             int64_t dst_stride, hipStream_t s) {
    switch (dst_dtype) {
        case RT_HIP_F32: return run_read_by<float>(kv, slots, n_tokens, k, v, dst_stride, s);
        case RT_HIP_F16: return run_read_by<_Float16>(kv, slots, n_tokens, k, v, dst_stride, s);
        default: return run_read_by<__bf16>(kv, slots, n_tokens, k, v, dst_stride, s);
    }
}

}  // namespace rt_hip
