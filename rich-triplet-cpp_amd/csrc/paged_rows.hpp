// paged_rows.hpp -- eight values of a row, in f32, from and to memory of each type.
#pragma once

#include "rt_common.hpp"

namespace rt_hip {
namespace {

__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
    const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        v[e] = a[e];
        v[4 + e] = b[e];
    }
}
__device__ __forceinline__ void load8(const __bf16* p, float (&v)[8]) {
    const u32x4 a = ld16(p);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        v[2 * e] = bf16_lo_to_f32(a[e]);
        v[2 * e + 1] = bf16_hi_to_f32(a[e]);
    }
}
__device__ __forceinline__ void load8(const _Float16* p, float (&v)[8]) {
    const u32x4 a = ld16(p);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        v[2 * e] = f16_bits_to_f32(a[e] & 0xffffu);
        v[2 * e + 1] = f16_bits_to_f32(a[e] >> 16);
    }
}
__device__ __forceinline__ void store8(float* p, const float (&v)[8]) {
    *reinterpret_cast<f32x4*>(p) = f32x4{v[0], v[1], v[2], v[3]};
    *reinterpret_cast<f32x4*>(p + 4) = f32x4{v[4], v[5], v[6], v[7]};
}
__device__ __forceinline__ void store8(__bf16* p, const float (&v)[8]) {
    *reinterpret_cast<u32x4*>(p) = u32x4{bf16_pair(v[0], v[1]), bf16_pair(v[2], v[3]), bf16_pair(v[4], v[5]),
                                         bf16_pair(v[6], v[7])};
}
__device__ __forceinline__ void store8(_Float16* p, const float (&v)[8]) {
    typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
    f16x8 o;
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = static_cast<_Float16>(v[e]);  // round to nearest even; past the range: infinity
    *reinterpret_cast<f16x8*>(p) = o;
}

}  // namespace
}  // namespace rt_hip
