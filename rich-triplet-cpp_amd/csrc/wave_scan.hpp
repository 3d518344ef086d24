// Scans and reductions over the 64 lanes of a wave whose steps are moves between
// lanes inside VALU instructions (DPP): a step takes a few cycles, where a
// shuffle takes the way through LDS, 60 and more.  All lanes have to be active.
#pragma once

#include "rt_common.hpp"

namespace rt_hip {

// Lane i's value in a lane ahead of it, `old` in lanes without one: rows of 16
// shifted by 1, 2, 4, 8, then the last lane of a row or half to the rows behind
// it.  Running an operation over these six leaves lane i with lanes 0 .. i.
template <int CTRL, int ROWS>
__device__ __forceinline__ int from_before(int old, int v) {
    return __builtin_amdgcn_update_dpp(old, v, CTRL, ROWS, 0xf, false);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ float from_before(float old, float v) {
    return __int_as_float(from_before<CTRL, ROWS>(__float_as_int(old), __float_as_int(v)));
}
template <int CTRL, int ROWS, class V>
__device__ __forceinline__ V from_before(V old, V v) {
    static_assert(sizeof(V) == 8, "two registers");
    const uint64_t o = __builtin_bit_cast(uint64_t, old), b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = from_before<CTRL, ROWS>(static_cast<int>(o), static_cast<int>(b));
    const uint32_t hi = from_before<CTRL, ROWS>(static_cast<int>(o >> 32), static_cast<int>(b >> 32));
    return __builtin_bit_cast(V, static_cast<uint64_t>(hi) << 32 | lo);
}
// op over lanes 0 .. i; none: what op(., none) leaves alone.
template <class V, class F>
__device__ __forceinline__ V running(V v, V none, F op) {
    v = op(v, from_before<0x111, 0xf>(none, v));
    v = op(v, from_before<0x112, 0xf>(none, v));
    v = op(v, from_before<0x114, 0xf>(none, v));
    v = op(v, from_before<0x118, 0xf>(none, v));
    v = op(v, from_before<0x142, 0xa>(none, v));
    return op(v, from_before<0x143, 0xc>(none, v));
}
// One lane's value in all of them.  (Every lane that is read must be active where v is computed.)
__device__ __forceinline__ int of_lane(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }
__device__ __forceinline__ float of_lane(float v, int lane) { return __int_as_float(of_lane(__float_as_int(v), lane)); }
template <class V>
__device__ __forceinline__ V of_lane(V v, int lane) {
    static_assert(sizeof(V) == 8, "two registers");
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = of_lane(static_cast<int>(b), lane), hi = of_lane(static_cast<int>(b >> 32), lane);
    return __builtin_bit_cast(V, static_cast<uint64_t>(hi) << 32 | lo);
}
// Sum over lanes 0 .. i.
template <class V>
__device__ __forceinline__ V running_sum(V v) {
    return running(v, V(0), [](V a, V b) { return a + b; });
}

}  // namespace rt_hip
