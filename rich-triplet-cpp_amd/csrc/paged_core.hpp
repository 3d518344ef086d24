// paged_core.hpp -- what the kernels of attention over a paged cache share
// (paged_attention.hip, paged4_attention.hip): the walk over the items, the
// products and the weighing of a tile in LDS, the states of cut items.  How the
// work is cut and what the arithmetic is: at the top of paged_attention.hip.
#pragma once

#include <utility>

#include "rt_common.hpp"
#include "rt_launch.hpp"
#include "wave_scan.hpp"

namespace rt_hip {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.44269504088896341f;
constexpr float kInf = __builtin_inff();

#define LDS_AS __attribute__((address_space(3)))
#define GLOBAL_AS __attribute__((address_space(1)))
#define CONST_AS __attribute__((address_space(4)))

// A page of the cache that is none: its keys and values (at most one row of
// 256 f32 is read, every row from the same place; of a 4-bit page 8 slots' codes or
// numbers, 1024 bytes too).
__device__ const __attribute__((aligned(16))) float kZeros[256] = {};

template <class T> struct KindOf;
template <> struct KindOf<float> { static constexpr bool f32 = true, f16 = false; };
template <> struct KindOf<_Float16> { static constexpr bool f32 = false, f16 = true; };
template <> struct KindOf<__bf16> { static constexpr bool f32 = false, f16 = false; };

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ __forceinline__ void st_dev(float* p, float v) {
    __hip_atomic_store((GLOBAL_AS float*)p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float ld_dev(const float* p) {
    return __hip_atomic_load((const GLOBAL_AS float*)p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Two f32 to 16 bits each (nearest even), and back.
template <class T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (KindOf<T>::f16) return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), f16x2));
    else return bf16_pair(a, b);
}
template <class T>
__device__ __forceinline__ f32x2 unpack2(uint32_t w) {
    if constexpr (KindOf<T>::f16) return __builtin_convertvector(__builtin_bit_cast(f16x2, w), f32x2);
    else return f32x2{bf16_lo_to_f32(w), bf16_hi_to_f32(w)};
}

// N steps that each read a fragment from LDS and use it, B reads ahead of the
// uses; the scheduling barriers keep the compiler from moving all the reads to
// the front, into registers that the accumulators need.
// (A fold instead of a loop, which the compiler leaves rolled past some length.)
template <class F, int N, int B, class R, class U, int... X>
__device__ __forceinline__ void read_ahead_steps(R read, U use, std::integer_sequence<int, X...>) {
    F f[B];
    auto first = [&](int x) {
        if (x < B) f[x] = read(x);
    };
    auto step = [&](int x) {
        use(x, f[x % B]);
        if (x + B < N) f[x % B] = read(x + B);
        if (x % 2 == 1) __builtin_amdgcn_sched_barrier(0);
    };
    (first(X), ...);
    __builtin_amdgcn_sched_barrier(0);
    (step(X), ...);
    __builtin_amdgcn_sched_barrier(0);
}
template <class F, int N, int B, class R, class U>
__device__ __forceinline__ void read_ahead(R read, U use) {
    read_ahead_steps<F, N, B>(read, use, std::make_integer_sequence<int, N>());
}

// A value that every lane of the wave holds, in a scalar register.
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ int64_t uniform(int64_t v) {
    const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v));
    const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v >> 32));
    return static_cast<int64_t>(static_cast<uint64_t>(hi) << 32 | lo);
}

// 16 bytes a lane from memory to LDS at dst + 16 lane.  (In assembly, without a
// result: after the builtin the compiler waits for all such copies before it
// reads anything transposed from LDS.  The kernels wait themselves.  M0 holds the
// place in LDS, as an operand, so that the compiler knows who writes it; it needs
// a wait state before the copy.)
__device__ __forceinline__ void copy_to_lds(const uint8_t* src, uint32_t offset, uint32_t dst) {
    src = reinterpret_cast<const uint8_t*>(uniform(static_cast<int64_t>(reinterpret_cast<uintptr_t>(src))));
    dst = static_cast<uint32_t>(uniform(static_cast<int>(dst)));
    asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"{m0}"(dst), "v"(offset), "s"(src) : "memory");
}
// 4 bytes a lane to LDS at dst + 4 lane.
__device__ __forceinline__ void copy_words_to_lds(const void* src, uint32_t offset, uint32_t dst) {
    src = reinterpret_cast<const void*>(uniform(static_cast<int64_t>(reinterpret_cast<uintptr_t>(src))));
    dst = static_cast<uint32_t>(uniform(static_cast<int>(dst)));
    asm volatile("s_nop 0\n\tglobal_load_lds_dword %1, %2" ::"{m0}"(dst), "v"(offset), "s"(src) : "memory");
}
template <int N>
__device__ __forceinline__ void wait_copies() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }
__device__ __forceinline__ uint32_t lds_address(const void* p) {
    return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((const LDS_AS void*)p));
}

template <class V>
__device__ __forceinline__ V lds_read(uint32_t at) {
    return *(const LDS_AS V*)(static_cast<uintptr_t>(at));
}
// A lane's number that the compiler must take as new here: what is derived from
// it (addresses of fragments) is then derived again for every tile, instead of
// being kept in registers that the accumulators need.
__device__ __forceinline__ uint32_t anew(uint32_t x) {
    asm volatile("" : "+v"(x));
    return x;
}

// The core of both kernels: DB rows of queries per block, RBLK blocks a wave,
// DB x DB matrix steps (DB = 32 or 16), tiles of BK keys.
template <class Q, class T, int HD, int DB, int RBLK, int BK>
struct Core {
    static constexpr bool F32 = KindOf<T>::f32, F16 = KindOf<T>::f16;
    static constexpr int NL = F32 || sizeof(Q) == 2 ? 1 : (F16 ? 2 : 3);  // limbs of q and of the weights
    // bf16 rows over f16 values: one limb holds their 8 bits, times a power of two as f32 rows.
    static constexpr bool kScaled = F16 && !KindOf<Q>::f16;
    static constexpr int RB = HD * static_cast<int>(sizeof(T));           // bytes of a key
    static constexpr int CPR = RB / 16, RPI = 64 / CPR;  // 16-byte chunks of a key, keys a wave's copy takes
    static constexpr int KG = 64 / DB, EL = 16 / static_cast<int>(sizeof(T));  // lane groups of a step, values of a chunk
    static constexpr int STEPS = CPR / KG, NC = HD / DB, KB = BK / DB, ACC = DB == 32 ? 16 : 4;
    static constexpr int KS = DB == 32 ? 16 : 32;  // keys of a 16-bit step of P V
    static constexpr int TB = BK * RB;             // bytes of a tile of K or V
    // The forms whose limbs of q leave few registers: f32 rows over f16 in two blocks
    // of 16, over bf16 in blocks of 32 at head_dim 256.  They derive the places of
    // their copies anew for every tile, and the first reads less ahead: without that
    // 20 registers went to memory at head_dim 256 (24 requests of 27 rows 150 us,
    // now 142), 3 at 128 (73.4, now 72.1).
    static constexpr bool kTight = NL == 2 ? RBLK == 2 && HD >= 128 : NL == 3 && DB == 32 && HD == 256;
    static constexpr int kAhead = kTight && NL == 2 ? 6 : 8;  // fragments read ahead of the matrix steps
    // Weights are kept times 2^kBias, and the running maximum may lag by 2^kLag.
    static constexpr int kBias = F16 ? 6 : 0;
    static constexpr float kLag = 8.0f;
    using Acc = typename std::conditional<DB == 32, f32x16, f32x4>::type;

    u32x4 q[RBLK][NL][STEPS];
    Acc o[RBLK][NC], s[RBLK][KB];
    u32x4 w[RBLK][F32 ? 1 : BK / KS][NL];  // weights as matrix operands (an f32 cache's stay in s)
    float m[RBLK], l[RBLK], c[RBLK];  // maximum of scores, sum of weights (this lane's keys), scale log2(e)
    int last[RBLK], first[RBLK];      // the keys the row sees
    int n, kg;                        // this lane's row of the block, its group

    __device__ __forceinline__ static Acc mma(u32x4 a, u32x4 b, Acc x) {
        if constexpr (F32) {
            const f32x4 fa = __builtin_bit_cast(f32x4, a), fb = __builtin_bit_cast(f32x4, b);
#pragma unroll
            for (int e = 0; e < 4; ++e) x = mma1(fa[e], fb[e], x);
            return x;
        } else if constexpr (F16) {
            if constexpr (DB == 32)
                return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), x, 0, 0, 0);
            else
                return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), x, 0, 0, 0);
        } else {
            if constexpr (DB == 32)
                return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), x, 0, 0, 0);
            else
                return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), x, 0, 0, 0);
        }
    }
    __device__ __forceinline__ static Acc mma1(float a, float b, Acc x) {
        if constexpr (DB == 32) return __builtin_amdgcn_mfma_f32_32x32x2f32(a, b, x, 0, 0, 0);
        else return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, x, 0, 0, 0);
    }

    // Granules of 16 bytes of a key's row are exchanged by these (xor), so that
    // the lanes that LDS serves together, 256 bytes' worth of them, read
    // different banks: 16 keys' granules of K, 4 keys' 64 bytes (DB = 32) or 8
    // keys' 32 bytes (16) of V, for f32 the keys 4 apart of the lane groups.
    // (Rows of 128 bytes lie two to 256.)  swz_v is the same 8 keys on.
    __device__ __forceinline__ static int swz_k(int row) { return CPR >= 16 ? row & 15 : (row >> 1) & 7; }
    __device__ __forceinline__ static int swz_v(int row) {
        if constexpr (F32) return DB == 32 ? 8 * ((row >> 2) & 1) : 4 * ((row >> 2) & 3);
        else if constexpr (DB == 32) return CPR >= 16 ? 4 * (row & 3) : 4 * ((row >> 1) & 1);
        else return CPR >= 16 ? 2 * (row & 7) : 2 * ((row >> 1) & 3);
    }

    // Copies of keys [8 j, 8 j + 8) of a tile, those from `off` (a multiple of
    // RPI) on that one instruction takes, to LDS at `dst`; base: key 8 j's (and
    // head's) bytes, or zeros with row_bytes 0; at most `most` keys further.
    template <bool V>
    __device__ __forceinline__ static void copy_rows(const uint8_t* base, uint32_t row_bytes, int most, int j, int off,
                                                     uint32_t dst) {
        const int lane = kTight ? static_cast<int>(anew(threadIdx.x & 63)) : threadIdx.x & 63;
        const int r = off + lane / CPR, row = 8 * j + r;
        const uint32_t at = static_cast<uint32_t>(min(r, most)) * row_bytes +
                            16u * static_cast<uint32_t>((lane % CPR) ^ (V ? swz_v(row) : swz_k(row)));
        copy_to_lds(base, at, dst);
    }

    __device__ __forceinline__ void setup() {
#pragma unroll
        for (int b = 0; b < RBLK; ++b)
#pragma unroll
            for (int t = 0; t < (F32 ? 1 : BK / KS); ++t)
#pragma unroll
                for (int k = 0; k < NL; ++k) w[b][t][k] = u32x4{0, 0, 0, 0};
        n = threadIdx.x & (DB - 1);
        kg = (threadIdx.x & 63) / DB;
    }

    // Queries of block b: `row` points at the row's head, null where there is none.
    __device__ __forceinline__ void load_q(int b, const Q* row, float c1) {
        m[b] = -kInf;
        l[b] = 0.0f;
#pragma unroll
        for (int i = 0; i < NC; ++i) o[b][i] = Acc{};
        c[b] = c1;
        if constexpr (NL == 1 && !kScaled) {
#pragma unroll
            for (int t = 0; t < STEPS; ++t) q[b][0][t] = row ? ld16(row + (t * KG + kg) * EL) : u32x4{0, 0, 0, 0};
        } else {
            f32x4 x[STEPS][2];
#pragma unroll
            for (int t = 0; t < STEPS; ++t)
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    x[t][i] = row ? four(row + (t * KG + kg) * EL + 4 * i) : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            float up = 1.0f;
            if constexpr (F16) {
                float big = 0.0f;
#pragma unroll
                for (int t = 0; t < STEPS; ++t)
#pragma unroll
                    for (int i = 0; i < 2; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e) big = fmaxf(big, fabsf(x[t][i][e]));
                c[b] = scaled(across_max(big), c1, &up);
            }
#pragma unroll
            for (int t = 0; t < STEPS; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    uint32_t w[NL];
                    limbs(x[t][i >> 1][2 * (i & 1)] * up, x[t][i >> 1][2 * (i & 1) + 1] * up, w);
#pragma unroll
                    for (int k = 0; k < NL; ++k) q[b][k][t][i] = w[k];
                }
        }
    }

    // *up: 2^(14 - exponent) of a row's largest value, which it puts into [2^14,
    // 2^15); returned: c1 times its inverse.  (Exponents that leave f32's range on
    // either side are cut: values below 2^-112 count less, above 2^126 too.)
    __device__ __forceinline__ static float scaled(float big, float c1, float* up) {
        int ex = static_cast<int>(__float_as_uint(big) >> 23);
        ex = big > 0.0f && ex < 255 ? min(max(14 + 127 - ex + 127, 1), 253) : 127;
        *up = __uint_as_float(static_cast<uint32_t>(ex) << 23);
        // (Not 0, which would make a NaN of the maximum of no scores; times 2^-126 all scores vanish.)
        return fmaxf(c1 * __uint_as_float(static_cast<uint32_t>(254 - ex) << 23), 0x1p-126f);
    }

    // Four values of a row of q.
    __device__ __forceinline__ static f32x4 four(const Q* row) {
        if constexpr (sizeof(Q) == 4) {
            return *reinterpret_cast<const f32x4*>(row);
        } else {
            const u32x2 w = *reinterpret_cast<const u32x2*>(row);
            const f32x2 lo = unpack2<Q>(w[0]), hi = unpack2<Q>(w[1]);
            return f32x4{lo[0], lo[1], hi[0], hi[1]};
        }
    }

    // A pair of f32 as NL limbs, packed.
    __device__ __forceinline__ static void limbs(float a, float b, uint32_t (&w)[NL]) {
#pragma unroll
        for (int k = 0; k < NL; ++k) {
            w[k] = pack2<T>(a, b);
            if (k + 1 < NL) {
                const f32x2 h = unpack2<T>(w[k]);
                a -= h[0];
                b -= h[1];
            }
        }
    }

    // Maximum and sum over the lanes that hold one row (a swap of a register
    // with itself leaves a lane's own value in one half and its partner's in
    // the other).
    __device__ __forceinline__ static float across_max(float v) {
        if constexpr (DB == 16) {
            const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
            v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
        }
        const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    }
    __device__ __forceinline__ static float across_sum(float v) {
        if constexpr (DB == 16) {
            const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
            v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
        }
        const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        return __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }

    // K's fragments, from the lane's first address.  (Tiles start at multiples of
    // a key's bytes, so the granule's exchange is an xor of the address.)
    __device__ __forceinline__ uint32_t k_first(uint32_t k) const { return k + n * RB + ((kg ^ swz_k(n)) << 4); }
    __device__ __forceinline__ static u32x4 k_frag(uint32_t at, int x) {
        return lds_read<u32x4>((at ^ (x / KB * KG * 16)) + x % KB * DB * RB);
    }
    __device__ __forceinline__ void score(int x, u32x4 a) {
#pragma unroll
        for (int i = NL - 1; i >= 0; --i)
#pragma unroll
            for (int b = 0; b < RBLK; ++b) s[b][x % KB] = mma(a, q[b][i][x / KB], s[b][x % KB]);
    }
    __device__ __forceinline__ void no_values() {
#pragma unroll
        for (int b = 0; b < RBLK; ++b)
#pragma unroll
            for (int i = 0; i < NC; ++i) o[b][i] = Acc{};
    }
    __device__ __forceinline__ void no_scores() {
#pragma unroll
        for (int b = 0; b < RBLK; ++b)
#pragma unroll
            for (int j = 0; j < KB; ++j) s[b][j] = Acc{};
    }
    // Scores of the tile whose keys lie at `k`.
    __device__ __forceinline__ void scores(uint32_t k) {
        no_scores();
        const uint32_t at = anew(k_first(k));
        read_ahead<u32x4, KB * STEPS, F32 ? 2 : kAhead>([&](int x) { return k_frag(at, x); },
                                                   [&](int x, u32x4 a) { score(x, a); });
    }

    // Weights in place of the scores; the running state moved to a new maximum
    // where one grew by more than 2^kLag.  key: the tile's first; edge: some
    // row does not see some of its keys.
    __device__ __forceinline__ void softmax(int key, bool edge) {
#pragma unroll
        for (int b = 0; b < RBLK; ++b) {
            if (edge) {
#pragma unroll
                for (int j = 0; j < KB; ++j)
#pragma unroll
                    for (int e = 0; e < ACC; ++e) {
                        // (what the row sees from key + 4 kg on)
                        const int at = j * DB + 8 * (e >> 2) + (e & 3);
                        s[b][j][e] = at > last[b] - key - 4 * kg || at < first[b] - key - 4 * kg ? -kInf : s[b][j][e];
                        if (e % 4 == 3) __builtin_amdgcn_sched_barrier(0);
                    }
            }
            // (four chains: one would wait for each of its steps)
            float top[4] = {-kInf, -kInf, -kInf, -kInf};
#pragma unroll
            for (int j = 0; j < KB; ++j)
#pragma unroll
                for (int e = 0; e < ACC; ++e) top[e & 3] = fmaxf(top[e & 3], s[b][j][e]);
            const float mx = across_max(fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])));
            // (a row of nothing but -inf so far: m stays -inf, weights are 0)
            if (__builtin_amdgcn_ballot_w64(mx * c[b] > m[b] * c[b] + kLag) != 0) {
                const float mn = fmaxf(m[b], mx);
                const float a = mn == -kInf ? 1.0f : exp2_fast((m[b] - mn) * c[b]);
                m[b] = mn;
                l[b] *= a;
#pragma unroll
                for (int i = 0; i < NC; ++i) o[b][i] *= a;
            }
            const float base = static_cast<float>(kBias) - (m[b] == -kInf ? 0.0f : m[b]) * c[b];
            float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int j = 0; j < KB; ++j)
#pragma unroll
                for (int e = 0; e < ACC; ++e) {
                    s[b][j][e] = exp2_fast(__builtin_fmaf(s[b][j][e], c[b], base));
                    if constexpr (F32 || NL > 1) sum[e & 3] += s[b][j][e];
                }
            if constexpr (!F32) {
#pragma unroll
                for (int t = 0; t < BK / KS; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int e = 8 * t + 2 * i;
                        uint32_t x[NL];
                        limbs(s[b][e / ACC][e % ACC], s[b][(e + 1) / ACC][(e + 1) % ACC], x);
#pragma unroll
                        for (int k = 0; k < NL; ++k) w[b][t][k][i] = x[k];
                        // (the sum of the weights as they multiply v, two to an instruction)
                        if constexpr (NL == 1) sum[i] = sum2(x[0], sum[i]);
                    }
            }
            l[b] += (sum[0] + sum[1]) + (sum[2] + sum[3]);
            // (opaque: the compiler would compute them where they are used, among the products)
            if constexpr (F32) {
#pragma unroll
                for (int j = 0; j < KB; ++j) asm volatile("" : "+v"(s[b][j]));
            } else {
#pragma unroll
                for (int t = 0; t < BK / KS; ++t)
#pragma unroll
                    for (int k = 0; k < NL; ++k) asm volatile("" : "+v"(w[b][t][k]));
            }
        }
    }
    __device__ __forceinline__ static float sum2(uint32_t x, float sum) {
        if constexpr (F16) {
            typedef _Float16 h2 __attribute__((ext_vector_type(2)));
            return __builtin_amdgcn_fdot2(__builtin_bit_cast(h2, x), h2{1.0f, 1.0f}, sum, false);
        } else {
            const uint32_t one = 0x3f803f80u;
            return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, x), __builtin_bit_cast(bf16x2, one), sum, false);
        }
    }

    // V's fragments.  16-bit step t, dims DB c ..: keys t KS + (KS / 2) a + 4 kg
    // + {0..3}, a = 0, 1, from the lane's first address.
    __device__ __forceinline__ uint32_t v_first(uint32_t v) const {
        const int lane = threadIdx.x & 63;
        if constexpr (F32) {  // the value for a register's key and this lane's dim
            return v + 4 * kg * RB + (((n >> 2) ^ swz_v(4 * kg)) << 4) + 4 * (n & 3);
        } else {
            const int row = 4 * kg + ((lane & 15) >> 2);
            const int chunk = (DB == 32 ? 2 * ((lane >> 4) & 1) : 0) + ((lane & 3) >> 1);
            return v + row * RB + ((chunk ^ swz_v(row)) << 4) + 8 * (lane & 1);
        }
    }
    __device__ __forceinline__ static u32x4 v_frag(uint32_t at, int t, int c) {
        u32x4 f;
#pragma unroll
        for (int a = 0; a < 2; ++a) {
            const uint32_t x = (at ^ (c * DB * 2)) + (t * KS + a * (KS / 2)) * RB;
            const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_AS s16x4*)static_cast<uintptr_t>(x));
            const u32x2 w = __builtin_bit_cast(u32x2, y);
            f[2 * a] = w[0];
            f[2 * a + 1] = w[1];
        }
        return f;
    }
    // f32: register e of block j, dims DB c ..
    __device__ __forceinline__ static float v_val(uint32_t at, int j, int e, int c) {
        return lds_read<float>((at ^ (c * DB * 4)) + (j * DB + 8 * (e >> 2) + (e & 3)) * RB);
    }

    // o += P V of the tile whose values lie at `v`.
    __device__ __forceinline__ void pv(uint32_t v) {
        const uint32_t at = anew(v_first(v));
        if constexpr (F32) {
            read_ahead<float, KB * ACC * NC, 8>(
                [&](int x) { return v_val(at, x / NC / ACC, x / NC % ACC, x % NC); },
                [&](int x, float a) {
#pragma unroll
                    for (int b = 0; b < RBLK; ++b)
                        o[b][x % NC] = mma1(a, s[b][x / NC / ACC][x / NC % ACC], o[b][x % NC]);
                });
        } else {
            read_ahead<u32x4, BK / KS * NC, kAhead>([&](int x) { return v_frag(at, x / NC, x % NC); },
                                                             [&](int x, u32x4 a) { add_value(x, a); });
        }
    }
    __device__ __forceinline__ void add_value(int x, u32x4 a) {
#pragma unroll
        for (int k = NL - 1; k >= 0; --k)
#pragma unroll
            for (int b = 0; b < RBLK; ++b) o[b][x % NC] = mma(a, w[b][x / NC][k], o[b][x % NC]);
    }
    // pv(v), then scores(k), the reads of the second running ahead into the
    // first; between(i), i < N, at even distances.
    template <int N, class F>
    __device__ __forceinline__ void products(uint32_t k, uint32_t v, F between) {
        if constexpr (F32) {
#pragma unroll
            for (int i = 0; i < N; ++i) between(i);
            pv(v);
            scores(k);
        } else {
            constexpr int NV = BK / KS * NC, NK = KB * STEPS;
            const uint32_t at_v = anew(v_first(v)), at_k = anew(k_first(k));
            no_scores();
            read_ahead<u32x4, NV + NK, kAhead>([&](int x) { return x < NV ? v_frag(at_v, x / NC, x % NC) : k_frag(at_k, x - NV); },
                                          [&](int x, u32x4 a) {
#pragma unroll
                                              for (int i = 0; i < N; ++i)
                                                  if (x == (i + 1) * ((NV + NK) / (N + 1))) between(i);
                                              if (x < NV) add_value(x, a);
                                              else score(x - NV, a);
                                          });
        }
    }

    // Infinities and NaN in 16 bytes of v made 0; whether there were any.
    __device__ __forceinline__ static bool clean(u32x4& x) {
        bool any = false;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t was = x[i];
            if constexpr (F32) {
                if ((x[i] & 0x7f800000u) == 0x7f800000u) x[i] = 0;
            } else {
                constexpr uint32_t kTop = F16 ? 0x7c00u : 0x7f80u;
                if ((x[i] & kTop) == kTop) x[i] &= 0xffff0000u;
                if ((x[i] >> 16 & kTop) == kTop) x[i] &= 0xffffu;
            }
            any |= x[i] != was;
        }
        return any;
    }
    // The same for this lane's granule at LDS address `at`.
    __device__ __forceinline__ static bool clean_at(uint32_t at) {
        u32x4 x = lds_read<u32x4>(at);
        const bool any = clean(x);
        if (any) *(LDS_AS u32x4*)static_cast<uintptr_t>(at) = x;
        return any;
    }
    // What was made 0 of key's values, whose head's bytes are at v, added to the
    // rows that see the key.
    __device__ __forceinline__ void add_special(int key, const uint8_t* v) {
#pragma unroll
        for (int i = 0; i < NC; ++i)
#pragma unroll
            for (int e = 0; e < ACC; e += 4) {
                f32x4 x;
                const T* const at = reinterpret_cast<const T*>(v) + dim_of(i, e);
                if constexpr (F32) {
                    x = *reinterpret_cast<const f32x4*>(at);
                } else {
                    const u32x2 w = *reinterpret_cast<const u32x2*>(at);
                    const f32x2 lo = unpack2<T>(w[0]), hi = unpack2<T>(w[1]);
                    x = f32x4{lo[0], lo[1], hi[0], hi[1]};
                }
#pragma unroll
                for (int b = 0; b < RBLK; ++b)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (key <= last[b] && key >= first[b] && !(fabsf(x[r]) < kInf)) o[b][i][e + r] += x[r];
                __builtin_amdgcn_sched_barrier(0);
            }
    }

    // Whether some o of the wave's is an infinity or a NaN (0 times it is a NaN).
    __device__ __forceinline__ bool not_finite() const {
        float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int b = 0; b < RBLK; ++b)
#pragma unroll
            for (int i = 0; i < NC; ++i)
#pragma unroll
                for (int e = 0; e < ACC; ++e) x[e & 3] = __builtin_fmaf(o[b][i][e], 0.0f, x[e & 3]);
        const float any = (x[0] + x[1]) + (x[2] + x[3]);
        return __builtin_amdgcn_ballot_w64(any != any) != 0;
    }

    // Dim of register e of block i of o.
    __device__ __forceinline__ int dim_of(int i, int e) const { return i * DB + 8 * (e >> 2) + 4 * kg + (e & 3); }
};

// ---- the walk over the items ---------------------------------------------------

// Which requests a launch takes, its blocks, and where states go.
struct Launch {
    float* part;         // [workgroups][2] states
    uint32_t* counters;  // per workgroup: arrivals of the item cut at its end
    int group;               // query heads of a KV head
    uint32_t group_mul;      // x / group = x * group_mul >> group_shift for x < 2^31
    int group_shift;
    int min_rows, max_rows;  // requests with rows (tokens x group) in (min_rows, max_rows]
};

// An item is EXTRA units, what its start and end cost, and then a unit for each
// of its tiles.
template <int BM, int BN, int EXTRA>
struct Walk {
    const PagedAttn& p;
    const Launch& la;
    int group, cap;
    // the request
    int s = 0, row0 = 0, n = 0, len = 0, blocks = 0;
    // the item: KV head, block, its first tile (a multiple of BN keys) and number of tiles
    int kvh = 0, blk = 0, tile0 = 0, tiles = 0;

    __device__ __forceinline__ Walk(const PagedAttn& p_, const Launch& la_) : p(p_), la(la_) {
        group = la.group;
        cap = static_cast<int>(p.cols << p.kv.page_shift);
    }
    __device__ __forceinline__ int rows() const { return n * group; }
    // Row's token; its head in the group.
    __device__ __forceinline__ int token(int row) const {
        return static_cast<int>(static_cast<uint64_t>(static_cast<uint32_t>(row)) * la.group_mul >> la.group_shift);
    }
    __device__ __forceinline__ int head(int row, int token) const { return row - token * group; }
    __device__ __forceinline__ void request(int s_) {
        s = s_;
        const CONST_AS int* qs = (const CONST_AS int*)p.q_start;
        const CONST_AS int* kl = (const CONST_AS int*)p.kv_len;
        row0 = min(max(qs[s], 0), p.n_tokens);
        n = min(max(qs[s + 1], row0), p.n_tokens) - row0;
        len = min(max(kl[s], 0), cap);
        if (rows() <= la.min_rows || rows() > la.max_rows) n = 0;
        blocks = (rows() + BM - 1) / BM;
    }
    // Keys [lo, hi) that block b's rows see.
    __device__ __forceinline__ void span(int b, int* lo, int* hi) const {
        const int i0 = token(b * BM), i1 = min(n - 1, token(b * BM + BM - 1));
        *hi = len - n + i1 + 1;
        *lo = first_seen(len - n + i0);
    }
    // The first key that a row at position `at` (below 0: it sees none) sees.  (The
    // longest windows reach further back than 32 bits from a position below 0.)
    __device__ __forceinline__ int first_seen(int at) const { return p.window && at >= p.window ? at - p.window + 1 : 0; }
    __device__ __forceinline__ int count(int b, int* first) const {
        int lo, hi;
        span(b, &lo, &hi);
        *first = hi > lo ? lo / BN : 0;
        return hi > lo ? (hi - 1) / BN + 1 - *first : 1;  // (none visible: one tile, to write zeros)
    }
    // Units of block b, and of the request for one KV head.
    __device__ __forceinline__ int units(int b) const {
        int first;
        return count(b, &first) + EXTRA;
    }
    __device__ __forceinline__ int64_t total() const {
        int64_t t = 0;
        for (int b = 0; b < blocks; ++b) t += units(b);
        return t;
    }
    __device__ __forceinline__ void block(int b) {
        blk = b;
        tiles = count(b, &tile0);
    }
    // The walk is the same in every lane: its numbers in scalar registers.
    __device__ __forceinline__ void pin() {
        s = uniform(s), row0 = uniform(row0), n = uniform(n), len = uniform(len), blocks = uniform(blocks);
        kvh = uniform(kvh), blk = uniform(blk), tile0 = uniform(tile0), tiles = uniform(tiles);
    }
    // The item behind this one; false where there is none.
    __device__ __forceinline__ bool next() {
        if (blk + 1 < blocks) {
            block(blk + 1);
            return true;
        }
        if (++kvh == p.kv.n_kv) {
            kvh = 0;
            n = 0;
            while (n == 0 && s + 1 < p.n_seq) request(s + 1);
        }
        block(0);
        return n > 0;
    }
};

// a / b, of numbers that rarely need 64 bits.
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
    if (((a | b) >> 32) == 0) return static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
    return a / b;
}

// Units of the walk's request for one KV head, its blocks counted by the wave's
// lanes (the walk is the same in all of them).
template <class W>
__device__ __forceinline__ int64_t wave_total(const W& walk) {
    int64_t t = 0;
    for (int b = threadIdx.x & 63; b < walk.blocks; b += 64) t += walk.units(b);
    return of_lane(running_sum(t), 63);
}

// Positions the walk at workgroup w's range of the sequence of all units (of
// nw equal ones) and returns how many units it takes (0: none); *skip: how many
// of the first item's lie before them; *per: units of a range.  Up to 64
// requests every wave sums for itself, one to a lane; otherwise the workgroup's
// threads do, several to a thread.  A request of many blocks is counted by its
// wave's lanes together.
template <int NT, class W>
__device__ __forceinline__ int64_t find_range(W& walk, int w, int nw, int64_t* skip, int64_t* per) {
    const int tid = threadIdx.x, lane = tid & 63, n_seq = walk.p.n_seq, n_kv = walk.p.kv.n_kv;
    __shared__ int64_t sums[NT / 64];
    __shared__ int found_s;
    __shared__ int64_t found_before;
    const bool small = n_seq <= 64;
    const int each = small ? 1 : (n_seq + NT - 1) / NT, base = small ? lane : tid * each;
    W scan(walk.p, walk.la);  // at the lane's request
    // units of this lane's i-th request, for one KV head
    auto units_of = [&](int i) -> int64_t {
        scan.n = scan.blocks = 0;
        if (base + i < n_seq) scan.request(base + i);
        int64_t t = scan.blocks <= 2 ? scan.total() : 0;
        for (uint64_t many = __builtin_amdgcn_ballot_w64(scan.blocks > 2); many; many &= many - 1) {
            const int src = __builtin_ctzll(many);
            W one(walk.p, walk.la);
            one.n = __builtin_amdgcn_readlane(scan.n, src);
            one.len = __builtin_amdgcn_readlane(scan.len, src);
            one.blocks = __builtin_amdgcn_readlane(scan.blocks, src);
            const int64_t sum = wave_total(one);
            if (lane == src) t = sum;
        }
        return t;
    };
    int64_t mine = 0, last = 0;
    for (int i = 0; i < each; ++i) {
        last = units_of(i);
        mine += last * n_kv;
    }
    int64_t incl = running_sum(mine);
    int64_t all = of_lane(incl, 63);
    if (!small) {
        if (lane == 63) sums[tid >> 6] = incl;
        __syncthreads();
        int64_t before = 0;
        all = 0;
#pragma unroll
        for (int i = 0; i < NT / 64; ++i) {
            if (i == (tid >> 6)) before = all;
            all += sums[i];
        }
        incl += before;
    }
    all = uniform(all);
    *per = max(quotient(all + nw - 1, nw), int64_t{1});
    const int64_t u = w * *per;
    if (u >= all) return 0;
    const bool here = u < incl && u >= incl - mine;
    int64_t at = incl - mine, t;  // units before the request, and of it for one KV head
    if (small) {
        // (the lane has the request: it is not read again)
        const int s = __builtin_ctzll(__builtin_amdgcn_ballot_w64(here));
        at = of_lane(at, s);
        t = of_lane(last, s);
        walk.s = s;
        walk.row0 = of_lane(scan.row0, s), walk.n = of_lane(scan.n, s);
        walk.len = of_lane(scan.len, s), walk.blocks = of_lane(scan.blocks, s);
    } else {
        if (__builtin_amdgcn_ballot_w64(here) != 0) {  // (whole waves, as units_of counts)
            for (int i = 0; i < each; ++i) {
                const int64_t t = units_of(i) * n_kv;
                if (here && u >= at && u < at + t) {
                    found_s = base + i;
                    found_before = at;
                }
                at += t;
            }
        }
        __syncthreads();
        walk.request(uniform(found_s));
        at = uniform(found_before);
        t = wave_total(walk);
    }
    int64_t off = u - at;
    walk.kvh = static_cast<int>(quotient(off, t));
    off -= walk.kvh * t;
    if (walk.blocks == 1) walk.block(0);
    else for (int b0 = 0;; b0 += 64) {
        const int c = b0 + lane < walk.blocks ? walk.units(b0 + lane) : 0;
        const int64_t sum = running_sum(static_cast<int64_t>(c));
        const uint64_t behind = __builtin_amdgcn_ballot_w64(off < sum);
        if (behind || b0 + 64 >= walk.blocks) {
            const int l = behind ? __builtin_ctzll(behind) : 0;
            walk.block(b0 + l);
            off -= of_lane(sum - c, l);
            break;
        }
        off -= of_lane(sum, 63);
    }
    *skip = off;
    return min(*per, all - u);
}

// A state of the few-row form: o [bm][hd], maxima [bm], sums [bm]; of the
// many-row form: a lane's values, maximum and sum, two lanes to a row.
constexpr int part_floats(int bm, int hd) { return bm * hd + 2 * bm; }
constexpr int wide_part_floats(int bm, int hd) { return bm * hd + 4 * bm; }
// Keys of a tile of the many-row form.  (Three limbs at head_dim 256 leave no room
// for the scores and weights of 64: 2048 tokens over 4000 keys 920 us, with 32 761;
// 64 over 500 57 and 49.  12 registers of q still go to memory there.)
template <class Q, class T>
constexpr int wide_keys(int hd) {
    return KindOf<T>::f32 || (hd == 256 && sizeof(Q) == 4 && !KindOf<T>::f16) ? 32 : 64;
}
// Tiles of K, and of V, that the many-row form keeps in LDS: three where they
// fit, so that copies run a step further ahead.
constexpr int wide_slots(int tile_bytes) { return 6 * tile_bytes <= 147456 ? 3 : 2; }

// The store of four values of a row (zeros where its sum of weights is 0).
template <class Q>
__device__ __forceinline__ void store_out(Q* dst, f32x4 o, float l) {
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    o *= inv;
    if (l == 0.0f) o = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    if constexpr (sizeof(Q) == 4) *reinterpret_cast<f32x4*>(dst) = o;
    else *reinterpret_cast<u32x2*>(dst) = u32x2{pack2<Q>(o[0], o[1]), pack2<Q>(o[2], o[3])};
}

// The weight of a state whose maximum lies x below the one it is joined under.
// Never 0, so that an infinity in the state's o stays one; the 2^-126 that the
// exponential would round to 0 change a sum by no more than that of its values.
__device__ __forceinline__ float state_weight(float x) { return fmaxf(exp2_fast(x), 0x1p-126f); }

// Four values of a row with the row's maximum (in powers of two) and sum.
struct State {
    float m, l;
    f32x4 o;
};
__device__ __forceinline__ void join_state(State& a, const State& b) {
    const float m = fmaxf(a.m, b.m);
    const float fa = m == -kInf ? 0.0f : state_weight(a.m - m), fb = m == -kInf ? 0.0f : state_weight(b.m - m);
    a.l = a.l * fa + b.l * fb;
    a.o = a.o * fa + b.o * fb;
    a.m = m;
}

// States of an item cut between workgroups first_wg .. last_wg, joined into
// out.  Part of workgroup w: its second slot for first_wg (whose range ends
// inside the item), the first for the others.  A thread takes four values of a
// row; where there are fewer of those than threads, several share the parts,
// each in order, and their results are joined through LDS (`tmp`, NT states).
template <class Q, int BM, int HD, int NT, class W>
__device__ __forceinline__ void join_parts(const W& walk, int first_wg, int last_wg, int rows, State* tmp) {
    const PagedAttn& p = walk.p;
    const Launch& la = walk.la;
    constexpr int kPart = part_floats(BM, HD), kAhead = 8;
    const int quads = rows * (HD / 4), share = quads >= NT ? 1 : NT / quads;
    for (int i0 = 0; i0 < quads; i0 += NT) {
        const int i = share == 1 ? i0 + static_cast<int>(threadIdx.x) : static_cast<int>(threadIdx.x) % quads;
        const int g = share == 1 ? 0 : static_cast<int>(threadIdx.x) / quads;
        const bool in = i < quads && g < share;
        const int r = in ? i / (HD / 4) : 0, d = in ? (i % (HD / 4)) * 4 : 0;
        State s = {-kInf, 0.0f, {0.0f, 0.0f, 0.0f, 0.0f}};
        for (int w = first_wg + g; in && w <= last_wg; w += share * kAhead) {
            State x[kAhead];  // all loads in flight together
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                const int at = w + k * share;
                if (at > last_wg) continue;
                const float* const src = la.part + (static_cast<int64_t>(at) * 2 + (at == first_wg)) * kPart;
                x[k].m = ld_dev(src + BM * HD + r);
                x[k].l = ld_dev(src + BM * HD + BM + r);
#pragma unroll
                for (int e = 0; e < 4; ++e) x[k].o[e] = ld_dev(src + r * HD + d + e);
            }
#pragma unroll
            for (int k = 0; k < kAhead; ++k)
                if (w + k * share <= last_wg) join_state(s, x[k]);
        }
        if (share > 1) {
            __syncthreads();
            tmp[threadIdx.x] = s;
            __syncthreads();
            if (in && g == 0)
                for (int k = 1; k < share; ++k) join_state(s, tmp[threadIdx.x + k * quads]);
        }
        if (in && g == 0) {
            const int row = walk.blk * BM + r, t = walk.token(row);
            store_out(static_cast<Q*>(p.out) + (walk.row0 + t) * p.out_stride +
                          (walk.kvh * walk.group + walk.head(row, t)) * HD + d, s.o, s.l);
        }
    }
}

// A request's pages, for one KV head.
struct Pages {
    const CONST_AS int* table;  // its row
    const uint8_t* k;           // the head's first key in page 0
    int64_t v;                  // from keys to values
    uint32_t page_bytes, row_bytes;
    int shift, n_pages, end;    // end: the last key that is read
};
template <class T>
__device__ __forceinline__ Pages pages_of(const PagedAttn& p, int s, int kvh, int end) {
    constexpr int64_t B = sizeof(T);
    Pages g;
    g.table = (const CONST_AS int*)p.table + static_cast<int64_t>(s) * p.cols;
    g.k = static_cast<const uint8_t*>(p.kv.k) + kvh * p.kv.head_dim * B;
    g.v = static_cast<const uint8_t*>(p.kv.v) - static_cast<const uint8_t*>(p.kv.k);
    g.page_bytes = static_cast<uint32_t>(p.kv.page_stride * B);  // (the host keeps it below 2^32)
    g.row_bytes = static_cast<uint32_t>(p.kv.n_kv * p.kv.head_dim * B);
    g.shift = p.kv.page_shift;
    g.n_pages = p.kv.n_pages;
    g.end = end;
    return g;
}
// A group of 8 keys: where they are.
struct Group {
    const uint8_t* k;
    int64_t v;           // from keys to values
    uint32_t row_bytes;
    int most;            // the last key that may be read, from the group's first
};
// The group's place in the request: that of `key` (a multiple of 8), behind the
// last key the one that holds it.  (Tiles copied ahead may start past 2^31.)
__device__ __forceinline__ int group_at(const Pages& g, uint32_t key) {
    return static_cast<int>(min(key, static_cast<uint32_t>(g.end & ~7)));
}
// The group at `at` on page `id`.
__device__ __forceinline__ Group group_on(const Pages& g, int at, int id) {
    const bool real = static_cast<uint32_t>(id) < static_cast<uint32_t>(g.n_pages);
    const uint8_t* const k = g.k + static_cast<uint64_t>(static_cast<uint32_t>(id)) * g.page_bytes +
                             static_cast<uint32_t>(at & ((1 << g.shift) - 1)) * g.row_bytes;
    Group x;
    x.k = real ? k : reinterpret_cast<const uint8_t*>(kZeros);
    x.v = real ? g.v : 0;
    x.row_bytes = real ? g.row_bytes : 0u;
    x.most = g.end - at;
    return x;
}
__device__ __forceinline__ Group group_of(const Pages& g, uint32_t key) {
    const int at = group_at(g, key);
    return group_on(g, at, g.table[at >> g.shift]);
}
// Where the values of one key are (key <= end).
__device__ __forceinline__ const uint8_t* value_of(const Pages& g, int key) {
    const Group x = group_of(g, key & ~7);
    return x.k + x.v + static_cast<uint32_t>(key & 7) * x.row_bytes;
}

// Page numbers of a walk along a request's keys: a wave's ring of 128 table
// entries in LDS, filled 64 at a time by copies that its waits for keys and
// values cover.  Entry `col` is word col % 128.
struct PageWindow {
    uint32_t ring;
    int base;  // entries base .. base + 127 are there or on their way
    __device__ __forceinline__ void fill(const Pages& g, int col) const {
        const int at = min(col + (static_cast<int>(threadIdx.x) & 63), g.end >> g.shift);
        copy_words_to_lds((const void*)g.table, static_cast<uint32_t>(at) * 4u, ring + (col & 127) * 4);
    }
    __device__ __forceinline__ void start(const Pages& g, int col) {
        base = col & ~63;
        fill(g, base);
        fill(g, base + 64);
    }
    // Entry `col`, no smaller than those asked for before and at most 64 from
    // the last of them; the copies that were on their way at that one are there.
    __device__ __forceinline__ int at(const Pages& g, int col) {
        if (col - base >= 64) {
            base += 64;
            fill(g, base + 64);
        }
        return uniform(lds_read<int>(ring + (col & 127) * 4));
    }
};

// Counts this workgroup's state of an item in; true in the one that is last.
// Relaxed: the states went out in agent-scope stores that every wave waits for
// here, and are read with agent-scope loads once the count is known.
__device__ __forceinline__ bool arrive(uint32_t* counter, int parts, int* flag) {
    wait_vmcnt<0>();
    __syncthreads();
    if (threadIdx.x == 0) {
        const uint32_t before = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        const bool is_last = before == static_cast<uint32_t>(parts) - 1;
        if (is_last) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        *flag = is_last;
    }
    __syncthreads();
    return *flag != 0;
}

// Workgroup blockIdx.x's place in the sequence: neighbours share an XCD (block
// b runs on XCD b % 8), whose L2 then serves the blocks of one KV head.
__device__ __forceinline__ int place_of(int b, int nw) {
    const int q = nw / 8, r = nw % 8, x = b % 8;
    return x * q + min(x, r) + b / 8;
}

// ---- host side -------------------------------------------------------------------

inline int slots() { return static_cast<int>(device_info().cus); }

// The most rows a request can have.
inline int64_t most_rows(const PagedAttn& p) {
    const int fresh = p.max_fresh > 0 && p.max_fresh < p.n_tokens ? p.max_fresh : p.n_tokens;
    return static_cast<int64_t>(fresh) * (p.n_q / p.kv.n_kv);
}

inline Launch launch_of(const PagedAttn& p, float* part, uint32_t* counters) {
    Launch la;
    la.part = part;
    la.counters = counters;
    la.group = p.n_q / p.kv.n_kv;
    int log = 0;
    while (1 << log < la.group) ++log;
    la.group_shift = 31 + log;  // (group_mul <= 2^31, over the quotient by less than x / 2^31)
    la.group_mul = static_cast<uint32_t>(((uint64_t{1} << la.group_shift) + la.group - 1) / la.group);
    la.min_rows = 0;
    la.max_rows = 0x7fffffff;
    return la;
}

}  // namespace
}  // namespace rt_hip
