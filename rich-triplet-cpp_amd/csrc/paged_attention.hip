// paged_attention.hip -- attention of the new tokens of many requests over a
// KV cache in pages.
//
// Row i of request s (n rows, len keys) has position len - n + i and sees the
// keys (position - window, position]:
//   out = sum_j softmax_j(scale q . k_j) v_j,
// zeros where it sees none.  Key j of the request is row j % page of page
// table[s][j / page].
//
// Work.  The rows of one request that share a KV head, (token, head of the
// group) in that order, are taken in blocks; an item is (request, KV head,
// block) and its tiles are the spans of keys the block's rows can see.  The
// sequence of all tiles of all items is cut into equal ranges, one per
// workgroup: the lengths are read on the device, so nothing is known of them
// when the launch is made, and a batch of very unequal requests still ends
// everywhere at once.  A workgroup finds its range by summing the requests'
// tiles itself.  An item cut between workgroups leaves its states (o, m, l) in
// the workspace; the last to arrive joins them in order, so results do not
// depend on who that is.
//
// Arithmetic.  Products on the matrix cores, online softmax per row:
//  * S^T = K Q^T, so that a lane holds one row's scores against several keys:
//    the row's maximum and sum are the lane's own and its partners' in the
//    other halves (32x32) or quarters (16x16) of the wave.
//  * O^T += V^T P^T: the lane that has a row's weights supplies them as they
//    are, for the keys its registers hold; V's fragments are read from LDS
//    transposed (ds_read_b64_tr_b16) for the same keys.
//  * 16-bit rows of q: products of 16-bit values, weights rounded to the type.
//    f16 weights are kept times 2^6, so that a weight of 2^-20 of the largest
//    still has all its bits.
//  * f32 rows over a 16-bit cache: q and the weights as limbs of the cache's
//    type, two of f16 (22 bits; q's row times a power of two that puts its
//    largest value at 2^14) or three of bf16 (24 bits), each multiplied with
//    the exact values of the cache.
//  * an f32 cache: f32 matrix steps.
//
// Bounds and times: at each of the two kernels.
//
// Infinities and NaN in v.  Keys a row does not see get weight 0, but 0 times an
// infinity or a NaN of their v would reach the row: in tiles with such pairs
// those values of v are made 0 in LDS, and added at the end to the rows that see
// them.  In the other tiles every row sees every key, but a product with a
// weight that has vanished, or with a limb that is 0 or negative, would turn an
// infinity into a NaN: a workgroup whose o has come out as something not finite
// walks its tiles again and does the same in all of them.  So whatever the tile,
// the limbs and the weight, such a value reaches the rows that see it as it is.
// (To look costs 0.1 to 0.3 us an item; to clean every tile from the start would
// cost each of them the reads and compares of all its values.)
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
// 256 f32 is read, every row from the same place).
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
        if constexpr (NL == 1) {
#pragma unroll
            for (int t = 0; t < STEPS; ++t) q[b][0][t] = row ? ld16(row + (t * KG + kg) * EL) : u32x4{0, 0, 0, 0};
        } else {
            f32x4 x[STEPS][2];
#pragma unroll
            for (int t = 0; t < STEPS; ++t)
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    x[t][i] = row ? *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(row) + (t * KG + kg) * EL + 4 * i)
                                  : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            float up = 1.0f;
            if constexpr (F16) {
                float big = 0.0f;
#pragma unroll
                for (int t = 0; t < STEPS; ++t)
#pragma unroll
                    for (int i = 0; i < 2; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e) big = fmaxf(big, fabsf(x[t][i][e]));
                big = across_max(big);
                // 2^(14 - exponent): the largest value in [2^14, 2^15); c has the inverse.  (Exponents that
                // leave f32's range on either side are cut: values below 2^-112 count less, above 2^126 too.)
                int ex = static_cast<int>(__float_as_uint(big) >> 23);
                ex = big > 0.0f && ex < 255 ? min(max(14 + 127 - ex + 127, 1), 253) : 127;
                up = __uint_as_float(static_cast<uint32_t>(ex) << 23);
                // (Not 0, which would make a NaN of the maximum of no scores; times 2^-126 all scores vanish.)
                c[b] = fmaxf(c1 * __uint_as_float(static_cast<uint32_t>(254 - ex) << 23), 0x1p-126f);
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

constexpr int narrow_ring(int hd) { return hd == 256 ? 32768 : 16384; }

// ---- few rows: the waves split the keys ------------------------------------------
// Single tokens and drafts, bound by the bytes of keys and values.  A wave
// streams tiles of its own through its own LDS ring, no barrier between them,
// and the four waves' states are joined at the item's end.
// 64 requests of 100 to 16000 keys, 8 KV heads of 128 in bf16: 151 us for 782 MB
// (5.2 TB/s; a plain read of as much reaches 5.9).  16 requests of 5 tokens, a
// window of 1024, head_dim 256: 23 us for 48 MB.  One token over 777 keys: 11.2
// us, a chain of latencies: lengths, pages, keys, the waves' states, the join of
// the workgroups'.
template <class Q, class T, int HD, int RBLK>
__global__ __launch_bounds__(256, HD < 256 ? 2 : 1) void k_paged_narrow(PagedAttn p, Launch la) {
    constexpr int NW = 4, DB = 16, BM = DB * RBLK, BK = KindOf<T>::f32 ? 16 : 32, BN = NW * BK;
    using C = Core<Q, T, HD, DB, RBLK, BK>;
    constexpr int kRing = narrow_ring(HD);  // bytes of a wave's ring
    constexpr int D = kRing / 2 / C::TB;    // tiles of K, and of V, in the ring
    constexpr int H = BK / C::RPI;      // copies of a tile of K, or of V
    constexpr int G = BK / 8, PER = 8 / C::RPI;
    constexpr int kPart = part_floats(BM, HD);
    static_assert(BM * HD * 4 <= kRing && D >= 1, "a tile and a wave's state fit its ring");
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    __shared__ float sm[NW][BM], sl[NW][BM];
    __shared__ int flag;
    __shared__ int dirty;  // the last of this workgroup's items whose o came out as something not finite
    if (threadIdx.x == 0) dirty = -1;
    int item = 0;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    uint8_t* const ring = lds + wave * kRing;
    const int nw = gridDim.x, w = place_of(blockIdx.x, nw);
    // Tiles that take as long as an item's start and end, 6 us.  (0: 47 us where 2
    // takes 36 for 128 requests of 50 to 2000 keys, 380 where it takes 331 for 200
    // of up to 4000 at head_dim 256, 12 where it takes 14 for 16 of up to 900.)
    constexpr int EXTRA = 2;
    Walk<BM, BN, EXTRA> walk(p, la);
    int64_t skip = 0, per = 0;
    int64_t left = find_range<256>(walk, w, nw, &skip, &per);
    int64_t item_at = w * per - skip + EXTRA;  // of the item's first tile in the sequence
    const uint32_t ring_at = uniform(static_cast<int>(lds_address(ring)));
    const float c1 = p.scale * kLog2e;
    C core;
    core.setup();
    bool all = false;  // the item once more, every tile of it as an edge tile
    while ((left = uniform(left)) > 0) {
        walk.pin();
        const int from = uniform(static_cast<int>(skip));
        const int to = uniform(static_cast<int>(min(static_cast<int64_t>(walk.tiles + EXTRA), skip + left)));
        skip = 0;
        left -= to - from;
        const int a = max(from - EXTRA, 0), b = max(to - EXTRA, 0);  // tiles
        if (a >= b) break;  // (the range ends before the item's first tile)
        int lo, hi;
        walk.span(walk.blk, &lo, &hi);
        const int rows = min(BM, walk.rows() - walk.blk * BM), row_first = walk.blk * BM;
        const int pos0 = walk.len - walk.n;
        // position of the block's first row (below every key: all tiles are edge tiles)
        const int low_pos = all ? -1 : pos0 + walk.token(row_first);
        const Pages pages = pages_of<T>(p, walk.s, walk.kvh, hi - 1);
        const int key0 = (walk.tile0 + a) * BN + wave * BK;
        int nt = b - a;
        if (key0 + (nt - 1) * BN >= hi) --nt;  // (the last tile's keys may end before this wave's)
        auto copy_k = [&](int i, const Group (&g)[G]) {
#pragma unroll
            for (int j = 0; j < H; ++j)
                C::template copy_rows<false>(g[j / PER].k, g[j / PER].row_bytes, g[j / PER].most, j / PER,
                                             j % PER * C::RPI, ring_at + (i % D) * C::TB + j * 1024);
        };
        auto copy_v = [&](int i, const Group (&g)[G]) {
#pragma unroll
            for (int j = 0; j < H; ++j)
                C::template copy_rows<true>(g[j / PER].k + g[j / PER].v, g[j / PER].row_bytes, g[j / PER].most, j / PER,
                                            j % PER * C::RPI, ring_at + (D + i % D) * C::TB + j * 1024);
        };
        auto groups = [&](int i, Group (&g)[G]) {
#pragma unroll
            for (int j = 0; j < G; ++j) g[j] = group_of(pages, key0 + i * BN + 8 * j);
        };
        for (int i = 0; i < D; ++i)
            if (i < nt) {
                Group g[G];
                groups(i, g);
                copy_k(i, g);
                copy_v(i, g);
            }
#pragma unroll
        for (int i = 0; i < RBLK; ++i) {
            const int r = i * DB + core.n, row = row_first + r;
            const bool real = r < rows;
            const int t = walk.token(row);
            core.load_q(i, real ? static_cast<const Q*>(p.q) + (walk.row0 + t) * p.q_stride +
                                      (walk.kvh * walk.group + walk.head(row, t)) * HD
                                : nullptr, c1);
            core.last[i] = real ? pos0 + t : -1;
            core.first[i] = walk.first_seen(core.last[i]);
        }
        // q is here: from now on only copies are in flight.  (The builtin, which the
        // compiler understands: it would wait for q's loads in every tile otherwise,
        // and with them for the copies.)
        wait_vmcnt<0>();
        auto is_edge = [&](int key) { return key + BK - 1 > low_pos || (p.window && hi - 1 - key >= p.window); };
        bool special = false;
        for (int i = 0; i < nt; ++i) {
            const int key = key0 + i * BN;
            const bool more = i + D < nt;
            const bool edge = is_edge(key);
            Group g[G];
            if (more) groups(i + D, g);
            // (what is in flight behind this tile's K: its V, and the later tiles in the ring)
            if (nt - i >= D) wait_copies<(2 * D - 1) * H>();
            else wait_copies<0>();
            core.scores(ring_at + (i % D) * C::TB);
            wait_lds();
            if (more) copy_k(i + D, g);
            core.softmax(key, edge);
            if (more) wait_copies<(2 * D - 1) * H>();
            else wait_copies<0>();
            const uint32_t v = ring_at + (D + i % D) * C::TB;
            if (edge) {
                bool any = false;
#pragma unroll
                for (int j = 0; j < C::TB / 1024; ++j) any |= C::clean_at(v + j * 1024 + anew((tid & 63) * 16));
                special |= __builtin_amdgcn_ballot_w64(any) != 0;
                wait_lds();
            }
            core.pv(v);
            wait_lds();
            if (more) copy_v(i + D, g);
        }
        if (special) {
            for (int i = 0; i < nt; ++i)
                if (const int key = key0 + i * BN; is_edge(key))
                    for (int j = 0; j < min(BK, hi - key); ++j)
                        core.add_special(key + j, value_of(pages, key + j));
        }
        // The waves' states, joined in order.
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        float* const mine = reinterpret_cast<float*>(ring);
#pragma unroll
        for (int i = 0; i < RBLK; ++i) {
            const int r = i * DB + core.n;
            const float l = C::across_sum(core.l[i]);
            if (core.kg == 0) {
                sm[wave][r] = core.m[i] * core.c[i];
                sl[wave][r] = l;
            }
#pragma unroll
            for (int j = 0; j < C::NC; ++j)
                *reinterpret_cast<f32x4*>(mine + r * HD + ((j * DB + 4 * core.kg) ^ (4 * (core.n & 7)))) = core.o[i][j];
        }
        __syncthreads();
        const int first_wg = static_cast<int>(item_at / per), last_wg = static_cast<int>((item_at + walk.tiles - 1) / per);
        const bool cut = first_wg != last_wg;
        float* const part = la.part + (static_cast<int64_t>(w) * 2 + (w == first_wg)) * kPart;
        for (int i = tid; i < rows * (HD / 4); i += 256) {
            const int r = i / (HD / 4), d = (i % (HD / 4)) * 4;
            float M = -kInf, L = 0.0f;
#pragma unroll
            for (int x = 0; x < NW; ++x) M = fmaxf(M, sm[x][r]);
            f32x4 O = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int x = 0; x < NW; ++x) {
                const float f = M == -kInf ? 1.0f : state_weight(sm[x][r] - M);
                L += sl[x][r] * f;
                O += *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(lds + x * kRing) + r * HD + (d ^ (4 * (r & 7)))) * f;
            }
            if (const f32x4 z = O * 0.0f; (z[0] + z[1]) + (z[2] + z[3]) != 0.0f) dirty = item;
            if (!cut) {
                const int row = row_first + r, t = walk.token(row);
                store_out(static_cast<Q*>(p.out) + (walk.row0 + t) * p.out_stride +
                              (walk.kvh * walk.group + walk.head(row, t)) * HD + d, O, L);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) st_dev(part + r * HD + d + e, O[e]);
                if (d == 0) {
                    st_dev(part + BM * HD + r, M);
                    st_dev(part + BM * HD + BM + r, L);
                }
            }
        }
        if (!all) {
            lds_barrier();
            if (uniform(dirty) == item) {
                all = true;
                skip = from, left += to - from;
                continue;
            }
        }
        ++item;
        if (cut) {
            if (arrive(la.counters + first_wg, last_wg - first_wg + 1, &flag))
                join_parts<Q, BM, HD, 256>(walk, first_wg, last_wg, rows, reinterpret_cast<State*>(lds));
        }
        __syncthreads();  // the rings are free again
        all = false;
        item_at += walk.tiles + EXTRA;
        if (left > 0 && !walk.next()) break;
    }
}

// ---- many rows: the waves split the rows -------------------------------------------
// Chunks of prompts, bound by the matrix cores: every wave has 32 rows of its
// own, and K and V tiles are read from memory once for all of them.  Four waves
// or eight: enough_rows.
// 4096 tokens over 8192 keys before them, 24 heads of 128 in bf16: 490 to 535 us,
// 960 to 1050 TFLOP/s, by the clock that the card's power limit leaves (a library
// product of 8192^3: 1212); the matrix cores are busy half of the time, the VALU
// the other half.  900-token chunks of head_dim 64: 88 us for 43 GFLOP, the VALU
// busy 40% of it, the matrix cores 20%.  517 tokens over 1100 keys in f32: 106
// us, 81 TFLOP/s, the matrix cores busy 54% of it.
template <class Q, class T, int HD, int NW>
__global__ __launch_bounds__(NW * 64) void k_paged_wide(PagedAttn p, Launch la) {
    constexpr int DB = 32, BM = DB * NW, BK = wide_keys<Q, T>(HD), BN = BK, NT = NW * 64;
    using C = Core<Q, T, HD, DB, 1, BK>;
    constexpr int PER = 8 / C::RPI;               // copies of a group of 8 keys
    constexpr int COPIES = BK / C::RPI / NW;      // copies of a tile of K, or of V, by each wave
    constexpr int GROUPS = COPIES < PER ? 1 : COPIES / PER;  // groups they are of
    constexpr int SLOTS = wide_slots(C::TB), L = SLOTS - 2;  // tiles of K, and of V, in LDS; copies run L steps further ahead
    constexpr int kPart = wide_part_floats(BM, HD);
    static_assert(COPIES >= 1 && COPIES * NW * C::RPI == BK && (COPIES < PER ? PER % COPIES : COPIES % PER) == 0,
                  "every wave copies alike, whole groups or part of one");
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];  // SLOTS tiles of K, SLOTS of V
    __shared__ int page_ring[NW][128];
    __shared__ int special;  // the last of this workgroup's items whose v held what was made 0
    __shared__ int dirty;    // the last whose o came out as something not finite
    __shared__ int flag;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int nw = gridDim.x, w = place_of(blockIdx.x, nw);
    // Tiles that take as long as an item's start and end, 5 us.  (35 requests, three
    // of them chunks of 800 to 900, head_dim 64 in bf16: 157 us with 0, 118 with
    // 6, 126 with 12; in f32 over f16, eight waves, 182 with 1, 144 with 6; one
    // chunk of 517 in f32, four waves: 120 with 1, 129 with 12.)
    constexpr int EXTRA = KindOf<T>::f32 ? (NW == 8 ? 3 : 1) : (NW == 8 ? 6 : 3);
    Walk<BM, BN, EXTRA> walk(p, la);
    int64_t skip = 0, per = 0;
    int64_t left = find_range<NT>(walk, w, nw, &skip, &per);
    int64_t item_at = w * per - skip + EXTRA;  // of the item's first tile in the sequence
    const uint32_t lds_at = uniform(static_cast<int>(lds_address(lds)));
    const float c1 = p.scale * kLog2e;
    if (tid == 0) special = dirty = -1;
    int item = 0;
    C core;
    core.setup();
    bool all = false;  // the item once more, every tile of it as an edge tile
    while ((left = uniform(left)) > 0) {
        walk.pin();
        const int from = uniform(static_cast<int>(skip));
        const int to = uniform(static_cast<int>(min(static_cast<int64_t>(walk.tiles + EXTRA), skip + left)));
        skip = 0;
        left -= to - from;
        const int a = max(from - EXTRA, 0), b = max(to - EXTRA, 0);  // tiles
        if (a >= b) break;  // (the range ends before the item's first tile)
        int lo, hi;
        walk.span(walk.blk, &lo, &hi);
        const int rows = min(BM, walk.rows() - walk.blk * BM), row_first = walk.blk * BM;
        const int pos0 = walk.len - walk.n;
        const int low_pos = all ? -1 : pos0 + walk.token(row_first);  // (as above)
        const int r = wave * DB + core.n, row = row_first + r;
        const bool real = r < rows;
        const int t = walk.token(row);
        const int64_t head = (walk.kvh * walk.group + walk.head(row, t)) * HD;
        // the wave's rows see keys from wave_lo to wave_hi
        const int wave_low = pos0 + walk.token(row_first + min(wave * DB, rows - 1));
        const int wave_hi = pos0 + walk.token(row_first + min(wave * DB + DB, rows) - 1);
        const Pages pages = pages_of<T>(p, walk.s, walk.kvh, hi - 1);
        const int key0 = (walk.tile0 + a) * BN;
        const int nt = hi > 0 ? b - a : 0;
        // This wave's groups of the tiles whose K and whose V are copied next.
        PageWindow window;
        window.ring = uniform(static_cast<int>(lds_address(page_ring[wave])));
        Group grp_k[GROUPS], grp_v[GROUPS];
        const int group0 = wave * COPIES / PER;  // (the wave's copies start in it, at part0)
        const int part0 = COPIES < PER ? wave * COPIES % PER : 0;
        auto find_groups = [&](int i) {
#pragma unroll
            for (int x = 0; x < GROUPS; ++x) {
                const int at = group_at(pages, static_cast<uint32_t>(key0) + i * BN + 8 * (group0 + x));
                grp_k[x] = group_on(pages, at, window.at(pages, at >> pages.shift));
            }
        };
        // Copy x of this wave's of a tile of K, or V, into a slot.
        auto copy_k = [&](int slot, int x) {
            const Group& g = grp_k[x / PER];
            C::template copy_rows<false>(g.k, g.row_bytes, g.most, group0 + x / PER, (part0 + x % PER) * C::RPI,
                                         lds_at + slot * C::TB + (wave * COPIES + x) * 1024);
        };
        auto copy_v = [&](int slot, int x) {
            const Group& g = grp_v[x / PER];
            C::template copy_rows<true>(g.k + g.v, g.row_bytes, g.most, group0 + x / PER, (part0 + x % PER) * C::RPI,
                                        lds_at + (SLOTS + slot) * C::TB + (wave * COPIES + x) * 1024);
        };
        auto is_edge = [&](int key) { return key + BK - 1 > low_pos || (p.window && hi - 1 - key >= p.window); };
        int ahead = 0;  // the tile grp_k is of
        auto advance = [&] {
#pragma unroll
            for (int x = 0; x < GROUPS; ++x) grp_v[x] = grp_k[x];
            find_groups(++ahead);
        };
        lds_barrier();  // (every wave is done with the item before)
        if (nt > 0) {
            window.start(pages, group_at(pages, key0 + 8 * group0) >> pages.shift);
            wait_copies<0>();
            find_groups(0);
#pragma unroll
            for (int x = 0; x < COPIES; ++x) copy_k(0, x);
            advance();
            if constexpr (L == 1) {
#pragma unroll
                for (int x = 0; x < COPIES; ++x) copy_v(0, x);
#pragma unroll
                for (int x = 0; x < COPIES; ++x) copy_k(1, x);
                advance();
            }
        }
        core.load_q(0, real ? static_cast<const Q*>(p.q) + (walk.row0 + t) * p.q_stride + head : nullptr, c1);
        core.last[0] = real ? pos0 + t : -1;
        core.first[0] = walk.first_seen(core.last[0]);
        wait_vmcnt<0>();  // (the builtin: so that the compiler, too, knows that q is there)
        lds_barrier();
        // Step i in two halves: the products, O += P V of tile i - 1 and the
        // scores of tile i, and the weighing of tile i.  With eight waves, w and
        // w + 4 share a SIMD: the second four run a half behind the first, so
        // that one wave of a SIMD has the matrix cores while the other has the
        // VALU, a barrier between the halves.
        // Among its products a wave sends the copies of V of tile i + L and K of
        // tile i + 1 + L, into the slots of V of tile i - 2 and K of tile i - 1,
        // which every wave has read by then; it waits for them in step i + L,
        // before the barrier that step i + L + 1 lies behind.  (Past the last
        // tile they bring its last keys again, for no one.)
        constexpr bool kTwo = NW == 8;
        static_assert(!kTwo || L == 1, "the second four send their copies a half late");
        const bool second = kTwo && wave >= 4;
        // This wave's copies of V of tile i are there; of an edge tile's, cleaned.
        auto settle = [&](int i, int slot) {
            wait_copies<2 * COPIES * L>();
            if (is_edge(key0 + i * BN)) {
                bool any = false;
#pragma unroll
                for (int x = 0; x < COPIES; ++x)
                    any |= C::clean_at(lds_at + (SLOTS + slot) * C::TB + (wave * COPIES + x) * 1024 + anew((tid & 63) * 16));
                if (__builtin_amdgcn_ballot_w64(any) != 0) special = item;
            }
        };
        if (nt > 0) {
            if (second) lds_barrier();
            int now = 0;  // slot of tile i
            for (int i = 0; i <= nt; ++i) {
                const int before = now == 0 ? SLOTS - 1 : now - 1, behind = now + 1 == SLOTS ? 0 : now + 1;
                // (no branch around the products of what is not there or not seen: the
                // weights of a tile that no row of the wave sees are 0 and its V is
                // clean, being an edge tile; in step 0 the accumulator is cleared
                // after; scores of no tile are not used)
                __builtin_amdgcn_s_setprio(1);
                core.template products<2 * COPIES>(lds_at + now * C::TB, lds_at + (SLOTS + before) * C::TB, [&](int x) {
                    if (x < COPIES) copy_v(L ? behind : now, x);
                    else copy_k(before, x - COPIES);
                });
                __builtin_amdgcn_s_setprio(0);
                if (i == 0) core.no_values();
                if (second && i < nt) settle(i, now);
                if (kTwo) lds_barrier();
                // (behind the last tile: from hi on, keys that no row sees, which change nothing)
                const int key = i < nt ? key0 + i * BN : hi;
                core.softmax(key, i == nt || key + BK - 1 > wave_low || (p.window && wave_hi - key >= p.window));
                advance();
                if (!second && i < nt) settle(i, now);
                lds_barrier();
                now = behind;
            }
            if (kTwo && !second) lds_barrier();
            wait_copies<0>();
        }
        if (uniform(special) == item) {
            for (int i = 0; i < nt; ++i)
                if (const int key = key0 + i * BN; is_edge(key))
                    for (int j = 0; j < min(BK, hi - key); ++j)
                        core.add_special(key + j, value_of(pages, key + j));
        }
        float l = C::across_sum(core.l[0]);
        const int first_wg = static_cast<int>(item_at / per), last_wg = static_cast<int>((item_at + walk.tiles - 1) / per);
        bool whole = first_wg == last_wg;
        auto part = [&](int wg) { return la.part + (static_cast<int64_t>(wg) * 2 + (wg == first_wg)) * kPart + tid; };
        if (!whole) {
            // States as the registers are, a lane's values NT apart.
            float* const mine = part(w);
#pragma unroll
            for (int i = 0; i < C::NC; ++i)
#pragma unroll
                for (int e = 0; e < C::ACC; ++e) st_dev(mine + (i * C::ACC + e) * NT, core.o[0][i][e]);
            st_dev(mine + BM * HD, core.m[0] * core.c[0]);
            st_dev(mine + BM * HD + NT, l);
        }
        if (!all) {
            if (core.not_finite()) dirty = item;
            lds_barrier();
            if (uniform(dirty) == item) {
                all = true;
                skip = from, left += to - from;
                continue;
            }
        }
        ++item;
        if (!whole) {
            whole = arrive(la.counters + first_wg, last_wg - first_wg + 1, &flag);
            if (whole) {
                float M = -kInf;
                l = 0.0f;
                core.no_values();
                for (int x = first_wg; x <= last_wg; ++x) {
                    // (all loads before the first use: they are served one latency after
                    // the other otherwise)
                    const float* const src = part(x);
                    const float m = ld_dev(src + BM * HD), sum = ld_dev(src + BM * HD + NT);
                    float o[C::NC * C::ACC];
#pragma unroll
                    for (int i = 0; i < C::NC * C::ACC; ++i) o[i] = ld_dev(src + i * NT);
                    __builtin_amdgcn_sched_barrier(0);
                    const float top = fmaxf(M, m);
                    const float fa = top == -kInf ? 0.0f : state_weight(M - top), fb = top == -kInf ? 0.0f : state_weight(m - top);
                    l = l * fa + sum * fb;
#pragma unroll
                    for (int i = 0; i < C::NC; ++i)
#pragma unroll
                        for (int e = 0; e < C::ACC; ++e)
                            core.o[0][i][e] = core.o[0][i][e] * fa + o[i * C::ACC + e] * fb;
                    M = top;
                }
            }
        }
        if (whole && real) {
            Q* const dst = static_cast<Q*>(p.out) + (walk.row0 + t) * p.out_stride + head;
#pragma unroll
            for (int i = 0; i < C::NC; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    store_out(dst + core.dim_of(i, 4 * e),
                              f32x4{core.o[0][i][4 * e], core.o[0][i][4 * e + 1], core.o[0][i][4 * e + 2], core.o[0][i][4 * e + 3]}, l);
        }
        all = false;
        item_at += walk.tiles + EXTRA;
        if (left > 0 && !walk.next()) break;
    }
}

// Rows (tokens x group) of a request up to which its keys are split over the
// waves.  24 requests of 1500 to 5000 keys at head_dim 128, bf16, few-row form
// against many-row form: 16 rows 64 us; 32 rows 75 and 100; 48 rows 114 and 97;
// 64 rows 118 and 99.  (At head_dim 64 the two meet at 64 rows, with f32 rows
// over a bf16 cache at 40.)
constexpr int kNarrowRows = 32;
// Whether eight waves of 32 rows, two to a SIMD, have registers enough.  (Three
// limbs of q at head_dim 128 have not: 2048 tokens over 4000 keys take 367 us with
// eight, 372 with four, 64 over 500 45 and 28.)
template <class Q, class T>
constexpr bool eight_fit(int hd) {
    return hd == 64 || (hd == 128 && !(sizeof(Q) == 4 && !KindOf<T>::f32 && !KindOf<T>::f16));
}

// Blocks of 16 rows that a wave of the few-row form takes together where there
// are more than one: two, but for f32 rows over bf16, whose three limbs of two
// blocks do not fit the registers (24 requests of 32 rows, head_dim 128: 116 us
// with two, 102 with one, keys and values read twice; 294 and 205 at 256).
template <class Q, class T>
constexpr int narrow_blocks(int hd) {
    return hd > 64 && sizeof(Q) == 4 && !KindOf<T>::f32 && !KindOf<T>::f16 ? 1 : 2;
}

int slots() { return static_cast<int>(device_info().cus); }

// Workgroups of the narrow form: those the CUs hold at once.  (With one to a CU
// 64 decoding requests take 166 us instead of 157, a mixed step 127 instead of 118.)
int narrow_slots(int hd) { return slots() * (hd == 256 ? 1 : 2); }

// The most rows a request can have.
int64_t most_rows(const PagedAttn& p) {
    const int fresh = p.max_fresh > 0 && p.max_fresh < p.n_tokens ? p.max_fresh : p.n_tokens;
    return static_cast<int64_t>(fresh) * (p.n_q / p.kv.n_kv);
}

// Whether the many-row form takes blocks of 256 rows, eight waves, or of 128,
// four: where a request's rows fill more than one of the smaller, and all rows
// together are 40 to a CU (80 with an f32 cache), so that keys are read fewer
// times and one wave of a SIMD can work while the other waits.  Four and eight
// waves, us, head_dim 128, 24 heads, 3 to a KV head:
//   tokens over keys      bf16        f32 over f16   f32
//   64 over 500           25    31    27    36       36    56
//   256 over 1000         27    37    32    42       63    72
//   512 over 9000        108    86   150   131      509   478
//   1024 over 3000        88    70   119   108      397   374
//   2048 over 4000       209   148   296   241     1080   999
// 40 requests, 32 heads, 4 to a KV head: of 30 tokens (120 rows) 47 and 53, of
// 100 (400 rows) 164 and 115.  (The rule does not know the keys, so that 512 over
// 9000 in f32, 48 rows to a CU, takes four waves and loses 6%; and it counts the
// rows there is room for.)
bool enough_rows(const PagedAttn& p, int64_t rows) {
    const int64_t each = p.kv.dtype == RT_HIP_F32 ? 80 : 40;
    return rows > 128 && static_cast<int64_t>(p.n_tokens) * p.n_q >= slots() * each;
}

template <class Q, class T, int HD>
hipError_t run(const PagedAttn& p, float* part, uint32_t* counters, hipStream_t s) {
    Launch la;
    la.part = part;
    la.counters = counters;
    la.group = p.n_q / p.kv.n_kv;
    int log = 0;
    while (1 << log < la.group) ++log;
    la.group_shift = 31 + log;  // (group_mul <= 2^31, over the quotient by less than x / 2^31)
    la.group_mul = static_cast<uint32_t>(((uint64_t{1} << la.group_shift) + la.group - 1) / la.group);
    const int64_t rows = most_rows(p);
    const bool wide = rows > kNarrowRows, narrow = !wide || p.n_seq > 1;
    // (one workgroup to a CU, LDS holds no more; ranges of a single tile are worth
    // it: with 8 at least, 64 tokens over 500 keys took 65 us in f32 instead of 37)
    const unsigned grid = static_cast<unsigned>(slots());
    if (wide) {
        constexpr int BK = wide_keys<Q, T>(HD), LDS = 2 * wide_slots(BK * HD * sizeof(T)) * BK * HD * sizeof(T);
        constexpr int MOST = eight_fit<Q, T>(HD) ? 8 : 4;
        la.min_rows = narrow ? kNarrowRows : 0;
        la.max_rows = 0x7fffffff;
        const bool eight = MOST == 8 && enough_rows(p, rows);
        hipLaunchKernelGGL((eight ? k_paged_wide<Q, T, HD, MOST> : k_paged_wide<Q, T, HD, 4>), dim3(grid),
                           dim3(eight ? 512 : 256), LDS, s, p, la);
    }
    if (narrow) {
        la.min_rows = 0;
        la.max_rows = wide ? kNarrowRows : 0x7fffffff;
        const unsigned many = static_cast<unsigned>(narrow_slots(HD));
        const auto kernel = rows <= 16 ? k_paged_narrow<Q, T, HD, 1> : k_paged_narrow<Q, T, HD, narrow_blocks<Q, T>(HD)>;
        hipLaunchKernelGGL(kernel, dim3(many), dim3(256), 4 * narrow_ring(HD), s, p, la);
    }
    return hipGetLastError();
}

template <class Q, class T>
hipError_t run_hd(const PagedAttn& p, float* part, uint32_t* counters, hipStream_t s) {
    switch (p.kv.head_dim) {
        case 64: return run<Q, T, 64>(p, part, counters, s);
        case 128: return run<Q, T, 128>(p, part, counters, s);
        default: return run<Q, T, 256>(p, part, counters, s);
    }
}

}  // namespace

size_t paged_attention_workspace(const PagedAttn& p) {
    const int64_t rows = most_rows(p);
    const int hd = p.kv.head_dim, waves = hd < 256 ? 8 : 4;
    const size_t narrow = static_cast<size_t>(narrow_slots(hd)) * 2 * part_floats(rows <= 16 ? 16 : 32, hd);
    const size_t wide = rows > kNarrowRows ? static_cast<size_t>(slots()) * 2 * wide_part_floats(waves * 32, hd) : 0;
    return (narrow > wide ? narrow : wide) * sizeof(float);
}

hipError_t launch_paged_attention(const PagedAttn& p, void* part, uint32_t* counters, hipStream_t s) {
    if (static_cast<size_t>(narrow_slots(64)) > kArrivalCounters) return hipErrorInvalidValue;
    float* const f = static_cast<float*>(part);
    if (p.dtype == RT_HIP_BF16) return run_hd<__bf16, __bf16>(p, f, counters, s);
    if (p.dtype == RT_HIP_F16) return run_hd<_Float16, _Float16>(p, f, counters, s);
    switch (p.kv.dtype) {
        case RT_HIP_F32: return run_hd<float, float>(p, f, counters, s);
        case RT_HIP_F16: return run_hd<float, _Float16>(p, f, counters, s);
        default: return run_hd<float, __bf16>(p, f, counters, s);
    }
}

}  // namespace rt_hip
