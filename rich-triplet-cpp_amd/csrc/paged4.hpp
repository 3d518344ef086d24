// paged4.hpp -- the 4-bit KV cache: where its bytes are and what they stand for.
//
// 32 neighbouring values of a head's row are a group: two f16 numbers a, b and
// 32 codes c of 0 .. 15, five bits a value.  A code stands for the f16 number
//   f16(a * (1 + c / 16) + b),     rounded once.
// 1 + c / 16 is the f16 number whose top four bits of mantissa are c, so one
// instruction (and, or) makes two of them out of the codes and one more
// (v_pk_fma_f16) their values: 1.4 to 1.6 instructions a value with the shifts,
// against HBM that brings a value in 0.7 of the time that three take.
//
// A page (page_size slots, n_kv heads) holds head after head; of a head first
// the codes of its slots, then their groups' numbers:
//   keys    codes [slot][hd / 8] words; numbers [slot][hd / 32] of a, b
//   values  codes [slot / 8][hd / 8][slot % 8] words;
//           numbers [slot / 8][hd / 32] of a [slot % 8], then b [slot % 8]
// A word has eight neighbouring values' codes, value 2 i at bits 4 i, value
// 2 i + 1 at bits 16 + 4 i.  The matrix steps take keys along their dims and
// values along 8 keys: either way a lane's operands are 16 and 32 neighbouring
// bytes, and a token's codes are whole words, so that no two tokens share one.
#pragma once

#include "rt_common.hpp"

namespace rt_hip {
namespace {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));

template <int HD>
struct Page4 {
    static constexpr int kSlot = HD / 2;                // bytes of a slot's codes
    static constexpr int kGroups = HD / 32;
    static constexpr int kSlotAll = HD / 2 + HD / 8;    // ... and of its numbers
    // (bytes from the head's first)
    __device__ __forceinline__ static uint32_t key_codes(uint32_t slot) { return slot * kSlot; }
    __device__ __forceinline__ static uint32_t key_numbers(uint32_t slot, int page_shift) {
        return (static_cast<uint32_t>(kSlot) << page_shift) + slot * (kGroups * 4);
    }
    // The 8 slots that `slot` is of: word w of slot i at 32 w + 4 i, numbers of group g at 32 g + 2 i (b: 16 on).
    __device__ __forceinline__ static uint32_t value_codes(uint32_t slot) { return (slot >> 3) * (8 * kSlot); }
    __device__ __forceinline__ static uint32_t value_numbers(uint32_t slot, int page_shift) {
        return (static_cast<uint32_t>(kSlot) << page_shift) + (slot >> 3) * (kGroups * 32);
    }
};

// (By value: the cast of a vector's element would read the vector's first.)
__device__ __forceinline__ h2 halves(uint32_t w) { return __builtin_bit_cast(h2, w); }

// 1 + c / 16 for the codes at bits 4 I and 16 + 4 I of w.
template <int I>
__device__ __forceinline__ h2 code_pair(uint32_t w) {
    const uint32_t at = I == 0 ? w << 6 : I == 1 ? w << 2 : I == 2 ? w >> 2 : w >> 6;
    return __builtin_bit_cast(h2, (at & 0x03c003c0u) | 0x3c003c00u);
}
template <int I>
__device__ __forceinline__ uint32_t value_pair(uint32_t w, h2 a, h2 b) {
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(code_pair<I>(w), a, b));
}
// The eight values of a word, in order, for one a and b (a in the low half of ab).
__device__ __forceinline__ u32x4 values_of(uint32_t w, h2 a, h2 b) {
    return u32x4{value_pair<0>(w, a, b), value_pair<1>(w, a, b), value_pair<2>(w, a, b), value_pair<3>(w, a, b)};
}
__device__ __forceinline__ u32x4 values_of(uint32_t w, uint32_t ab) {
    const h2 x = halves(ab);
    return values_of(w, h2{x[0], x[0]}, h2{x[1], x[1]});
}
// Whether a or b (16 bits each) is an infinity or a NaN.
__device__ __forceinline__ bool no_number(uint32_t a, uint32_t b) {
    return (a & 0x7c00u) == 0x7c00u || (b & 0x7c00u) == 0x7c00u;
}

}  // namespace
}  // namespace rt_hip
