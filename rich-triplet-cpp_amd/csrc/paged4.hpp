// paged4.hpp -- the 4-bit KV cache: where its bytes are and what they stand for.
//
// 32 neighbouring values of a head's row are a group: two f16 numbers a, b and
// 32 codes c of 0 .. 15, five bits a value.  A code stands for the f16 number
//   f16(a * (1 + c / 16) + b),     rounded once.
// 1 + c / 16 is the f16 number whose top four bits of mantissa are c, so one
// instruction (and, or) makes two of them out of the codes and one more
// (v_pk_fma_f16) their values: with the shifts 1.4 to 1.5 instructions a value, in
// less than half of the time that HBM takes to bring it.
//
// A page (page_size slots, n_kv heads) holds head after head; of a head first
// the codes of its slots, 8 slots after 8, then their groups' numbers.  Of 8 slots:
//   keys    codes [hd / 32][slot % 8] of the group's four words; numbers
//           [hd / 32][slot % 8] of a, b
//   values  codes [slot / 4 % 2][hd / 8][slot % 4] words; numbers [hd / 32] of
//           a [slot % 8], then b [slot % 8]
// A word has eight neighbouring values' codes, 2 i in its low and 2 i + 1 in its
// high half at bits 4 i + 2 (mod 16), so that of a half's four codes one is where
// f16's top bits of mantissa are, two are a shift and one is an exchange of bytes away.
// The matrix steps take keys along their dims and
// values along 8 keys.  Either way four neighbouring lanes' operands are 64
// neighbouring bytes (with a key's words together they were four accesses of the
// cache), and a token's codes are whole words, so that no two tokens share one.
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
    // The codes, and the numbers, of the 8 slots that `slot` is of: bytes from the head's first.
    __host__ __device__ __forceinline__ static constexpr uint32_t codes(uint32_t slot) { return (slot >> 3) * (8 * kSlot); }
    __host__ __device__ __forceinline__ static constexpr uint32_t numbers(uint32_t slot, int page_shift) {
        return (static_cast<uint32_t>(kSlot) << page_shift) + (slot >> 3) * (kGroups * 32);
    }
    // Word w and the numbers of group g of slot i of 8, from those; of a value a's (b: 16 on).
    __host__ __device__ __forceinline__ static constexpr uint32_t key_word(uint32_t i, uint32_t w) {
        return (w >> 2) * 128 + i * 16 + (w & 3) * 4;
    }
    __host__ __device__ __forceinline__ static constexpr uint32_t key_number(uint32_t i, uint32_t g) { return g * 32 + i * 4; }
    __host__ __device__ __forceinline__ static constexpr uint32_t value_word(uint32_t i, uint32_t w) {
        return (i >> 2) * (4 * kSlot) + w * 16 + (i & 3) * 4;
    }
    __host__ __device__ __forceinline__ static constexpr uint32_t value_number(uint32_t i, uint32_t g) { return g * 32 + i * 2; }
};

// (By value: the cast of a vector's element would read the vector's first.)
__device__ __forceinline__ h2 halves(uint32_t w) { return __builtin_bit_cast(h2, w); }

// The constants of the two instructions.  (Opaque, one in a scalar and one in a
// vector register: an instruction takes one constant besides.)
struct Codes {
    uint32_t top, one;  // the top four bits of mantissa; 1.0
    __device__ __forceinline__ Codes() {
        asm("s_mov_b32 %0, 0x3c003c0" : "=s"(top));
        asm("v_mov_b32 %0, 0x3c003c00" : "=v"(one));
    }
    // 1 + c / 16 of two codes, from a word that has them at bits 6 and 22 on.
    __device__ __forceinline__ h2 pair(uint32_t w) const { return halves((w & top) | one); }
    // Code I of each half of w as a word for pair (I = 3: of w with the bytes of its halves exchanged).
    template <int I>
    __device__ __forceinline__ static uint32_t place(uint32_t w) {
        return I == 0 ? w << 4 : I == 2 ? w >> 4 : w;
    }
    __device__ __forceinline__ static uint32_t swapped(uint32_t w) { return __builtin_amdgcn_perm(w, w, 0x02030001u); }
    template <int I>
    __device__ __forceinline__ uint32_t values(uint32_t w, h2 a, h2 b) const {
        return __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(pair(place<I>(w)), a, b));
    }
    // The eight values of a word, in order, for one a and b (a in the low half of ab).
    __device__ __forceinline__ u32x4 word(uint32_t w, uint32_t ab) const {
        const h2 x = halves(ab), a = {x[0], x[0]}, b = {x[1], x[1]};
        return u32x4{values<0>(w, a, b), values<1>(w, a, b), values<2>(w, a, b), values<3>(swapped(w), a, b)};
    }
};
// A word of eight codes from its halves' plain ones (code e at bits 4 (e / 2) of half e % 2): each half turned by two bits.
__device__ __forceinline__ uint32_t turned_codes(uint32_t w) { return (w << 2 & 0xfffcfffcu) | (w >> 14 & 0x00030003u); }
// Whether a or b (16 bits each) is an infinity or a NaN.
__device__ __forceinline__ bool no_number(uint32_t a, uint32_t b) {
    return (a & 0x7c00u) == 0x7c00u || (b & 0x7c00u) == 0x7c00u;
}

}  // namespace
}  // namespace rt_hip
