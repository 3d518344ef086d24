// paged4_attention.hip -- attention over a KV cache in 4 bits (paged4.hpp).
//
// The cache stands for f16 numbers, and what is computed of them is what
// paged_attention.hip computes over an f16 cache, work cut and states joined in
// the same way: S^T = K Q^T, online softmax per row, O^T += V^T P^T on the
// matrix cores, sums in f32, f16 weights times 2^6; f32 rows as two limbs of
// f16, bf16 rows as one, both times a power of two that puts the row's largest
// value at 2^14.  K and V become f16 in registers.
//
// A group of values that is no number (a or b an infinity or a NaN: what append
// makes of values that are not finite) is NaN in every value.  Weights of keys
// that a row does not see are 0, and 0 times NaN would reach the row: in tiles
// with such pairs the group's a and b are made 0, and NaN is added at the end to
// the rows that see it.  In the other tiles every row sees every key, and a NaN
// times any weight is the NaN that the row is to have.
// Keys that no row sees, behind the last one and in front of the first, may never
// have been written.  Their a and b are made 0 whatever they are: finite ones may
// still stand for infinities (a = b = 61280, say), which a weight of 0 makes NaN.
#include "paged4.hpp"
#include "paged_core.hpp"

namespace rt_hip {
namespace {

// A request's pages, for one KV head.
struct Pages4 {
    const GLOBAL_AS int* table;  // its row
    const uint8_t* k;            // the head's first byte in page 0
    const uint8_t* v;
    uint32_t page_bytes;         // (the host keeps it below 2^32)
    int shift, n_pages, end;     // end: the last key that is read
};
template <int HD>
__device__ __forceinline__ Pages4 pages4_of(const PagedAttn& p, int s, int kvh, int end) {
    Pages4 g;
    g.table = (const GLOBAL_AS int*)p.table + static_cast<int64_t>(s) * p.cols;
    const uint32_t head = (static_cast<uint32_t>(Page4<HD>::kSlotAll) << p.kv.page_shift) * static_cast<uint32_t>(kvh);
    g.k = static_cast<const uint8_t*>(p.kv.k) + head;
    g.v = static_cast<const uint8_t*>(p.kv.v) + head;
    g.page_bytes = static_cast<uint32_t>(p.kv.page_stride);
    g.shift = p.kv.page_shift;
    g.n_pages = p.kv.n_pages;
    g.end = end;
    return g;
}
// The page that holds `key`, behind the last key the last one's.
__device__ __forceinline__ int page4_at(const Pages4& g, uint32_t key) {
    return g.table[min(key, static_cast<uint32_t>(g.end)) >> g.shift];
}
__device__ __forceinline__ bool real_page(const Pages4& g, int id) {
    return static_cast<uint32_t>(id) < static_cast<uint32_t>(g.n_pages);
}
// a and b of group `grp` of a key's values (key <= end); 0 on a page that is none.
template <int HD>
__device__ __forceinline__ uint32_t value_numbers_of(const Pages4& g, int key, int grp) {
    const int id = page4_at(g, key);
    if (!real_page(g, id)) return 0;
    const uint32_t slot = key & ((1 << g.shift) - 1);
    const uint16_t* const at = reinterpret_cast<const uint16_t*>(
        g.v + static_cast<uint64_t>(static_cast<uint32_t>(id)) * g.page_bytes + Page4<HD>::numbers(slot, g.shift) +
        Page4<HD>::value_number(slot & 7, grp));
    return at[0] | static_cast<uint32_t>(at[8]) << 16;
}

// ---- few rows: the waves split the keys ------------------------------------------

// A wave's tile of 32 keys against RBLK blocks of 16 rows.  Key 8 a + i of the
// tile: row 4 a + i of the first matrix step for i < 4, of the second behind,
// so that a lane (row n of a block, quarter kg) has the scores of the eight keys
// 8 kg .. 8 kg + 7, and as many weights as a step of P V takes of it.
template <class Q, int HD, int RBLK>
struct Few {
    static constexpr int NL = sizeof(Q) == 4 ? 2 : 1;  // limbs of q and of the weights
    static constexpr int SETS = HD == 256 ? 2 : 1;     // of 128 dims
    static constexpr int W = HD == 64 ? 16 : 32;       // dims of a set that one lane multiplies keys along
    static constexpr int WORDS = W / 8, STEPS = HD / 32, NT = HD / 16;
    static constexpr bool kScaled = !KindOf<Q>::f16;
    static constexpr int kBias = 6;
    static constexpr float kLag = 8.0f;
    using Limb = Core<Q, _Float16, 64, 16, 1, 32>;  // (its limbs and its moves across lanes)

    u32x4 q[RBLK][NL][STEPS];
    f32x4 o[RBLK][NT], s[RBLK][2];
    u32x4 w[RBLK][NL];
    float m[RBLK], l[RBLK], c[RBLK];
    int last[RBLK], first[RBLK];
    int n, kg;
    // A tile's codes and numbers, as they come from memory.
    struct Tile {
        uint32_t kc[2][SETS][WORDS], kn[2][SETS];
        u32x4 vc[SETS][2], va[SETS], vb[SETS];
        bool no_keys, no_values;  // this lane's group of 8 is on a page that is none
    };
    Codes codes;

    __device__ __forceinline__ void setup() {
        n = threadIdx.x & 15;
        kg = (threadIdx.x & 63) >> 4;
    }
    // Dims of q's step t: 8 from here.
    __device__ __forceinline__ int dim_q(int t) const { return t / WORDS * 128 + kg * W + t % WORDS * 8; }
    // Dim of value e of tile t of o.  (A lane has 32 neighbouring dims of a set, at head_dim 64 16 in all.)
    __device__ __forceinline__ int dim_o(int t, int e) const {
        if constexpr (HD == 64) return 8 * (2 * kg + (e >> 1)) + 2 * t + (e & 1);
        else return t / 8 * 128 + 8 * (4 * kg + e) + 2 * (t & 3) + (t >> 2 & 1);
    }

    // A row of q as it is in memory, this lane's dims of it; zeros for null.
    struct Row {
        u32x4 x[STEPS][sizeof(Q) / 2];
    };
    __device__ __forceinline__ Row load_row(const Q* row) const {
        Row r;
#pragma unroll
        for (int t = 0; t < STEPS; ++t)
#pragma unroll
            for (int i = 0; i < static_cast<int>(sizeof(Q)) / 2; ++i)
                r.x[t][i] = row ? ld16(row + dim_q(t) + 4 * i) : u32x4{0, 0, 0, 0};
        return r;
    }
    __device__ __forceinline__ void set_q(int b, const Row& row, float c1) {
        m[b] = -kInf;
        l[b] = 0.0f;
#pragma unroll
        for (int i = 0; i < NT; ++i) o[b][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        c[b] = c1;
        if constexpr (!kScaled) {
#pragma unroll
            for (int t = 0; t < STEPS; ++t) q[b][0][t] = row.x[t][0];
        } else {
            auto two = [&](int t, int i) {
                if constexpr (sizeof(Q) == 4) {
                    const u32x4 w = row.x[t][i >> 1];
                    return f32x2{__uint_as_float(w[2 * (i & 1)]), __uint_as_float(w[2 * (i & 1) + 1])};
                } else {
                    const uint32_t w = row.x[t][0][i];
                    return f32x2{bf16_lo_to_f32(w), bf16_hi_to_f32(w)};
                }
            };
            float big = 0.0f;
#pragma unroll
            for (int t = 0; t < STEPS; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) big = fmaxf(big, fmaxf(fabsf(two(t, i)[0]), fabsf(two(t, i)[1])));
            float up;
            c[b] = Limb::scaled(Limb::across_max(big), c1, &up);
#pragma unroll
            for (int t = 0; t < STEPS; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    uint32_t y[NL];
                    Limb::limbs(two(t, i)[0] * up, two(t, i)[1] * up, y);
#pragma unroll
                    for (int k = 0; k < NL; ++k) q[b][k][t][i] = y[k];
                }
        }
    }

    // Loads of a tile's keys from key0 on; id: the page of this lane's group of
    // 8, key0 + 8 (n / 4), behind the last key that one's.  (What is read there then
    // is some of that page, and for a page that is none some of page 0.)
    __device__ __forceinline__ void load_keys(Tile& x, const Pages4& g, uint32_t key0, int id) const {
        x.no_keys = !real_page(g, id);
        const uint8_t* const page = g.k + static_cast<uint64_t>(x.no_keys ? 0u : static_cast<uint32_t>(id)) * g.page_bytes;
        const uint32_t slot = (key0 + 8u * (static_cast<uint32_t>(n) >> 2)) & ((1u << g.shift) - 1);
        const uint32_t i0 = static_cast<uint32_t>(n) & 3u;  // the lane's slots of the eight: this and 4 on
        const uint8_t* const at = page + (Page4<HD>::codes(slot) + Page4<HD>::key_word(i0, kg * WORDS));
        const uint8_t* const num = page + (Page4<HD>::numbers(slot, g.shift) + Page4<HD>::key_number(i0, HD == 64 ? kg >> 1 : kg));
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int u = 0; u < SETS; ++u) {
                const uint8_t* const codes_at = at + Page4<HD>::key_word(4 * j, 16 * u);
                if constexpr (WORDS == 4) {
                    const u32x4 y = *(const GLOBAL_AS u32x4*)codes_at;
#pragma unroll
                    for (int i = 0; i < 4; ++i) x.kc[j][u][i] = y[i];
                } else {
                    const u32x2 y = *(const GLOBAL_AS u32x2*)codes_at;
#pragma unroll
                    for (int i = 0; i < 2; ++i) x.kc[j][u][i] = y[i];
                }
                x.kn[j][u] = *(const GLOBAL_AS uint32_t*)(num + Page4<HD>::key_number(4 * j, 4 * u));
            }
    }
    // Loads of the values; id: the page of this lane's group of 8, key0 + 8 kg.
    __device__ __forceinline__ void load_values(Tile& x, const Pages4& g, uint32_t key0, int id) const {
        x.no_values = !real_page(g, id);
        const uint8_t* const page = g.v + static_cast<uint64_t>(x.no_values ? 0u : static_cast<uint32_t>(id)) * g.page_bytes;
        const uint32_t slot = (key0 + 8u * kg) & ((1u << g.shift) - 1);
        const int word = HD == 64 ? n >> 1 : n;
        const uint8_t* const at = page + (Page4<HD>::codes(slot) + Page4<HD>::value_word(0, word));
        const uint8_t* const num = page + (Page4<HD>::numbers(slot, g.shift) + Page4<HD>::value_number(0, word >> 2));
#pragma unroll
        for (int u = 0; u < SETS; ++u) {
#pragma unroll
            for (int i = 0; i < 2; ++i) x.vc[u][i] = *(const GLOBAL_AS u32x4*)(at + Page4<HD>::value_word(4 * i, 16 * u));
            x.va[u] = *(const GLOBAL_AS u32x4*)(num + Page4<HD>::value_number(0, 4 * u));
            x.vb[u] = *(const GLOBAL_AS u32x4*)(num + Page4<HD>::value_number(0, 4 * u) + 16);
        }
    }

    __device__ __forceinline__ static f32x4 mma(u32x4 a, u32x4 b, f32x4 x) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), x, 0, 0, 0);
    }
    __device__ __forceinline__ void scores(Tile& x) {
        if (__builtin_amdgcn_ballot_w64(x.no_keys) != 0) {
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int u = 0; u < SETS; ++u) x.kn[j][u] = x.no_keys ? 0u : x.kn[j][u];
        }
#pragma unroll
        for (int b = 0; b < RBLK; ++b)
#pragma unroll
            for (int j = 0; j < 2; ++j) s[b][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int t = 0; t < STEPS; ++t)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const u32x4 a = codes.word(x.kc[j][t / WORDS][t % WORDS], x.kn[j][t / WORDS]);
#pragma unroll
                for (int k = NL - 1; k >= 0; --k)
#pragma unroll
                    for (int b = 0; b < RBLK; ++b) s[b][j] = mma(a, q[b][k][t], s[b][j]);
            }
    }
    // Weights of the scores of the keys from `key` on; edge: some row does not see some of them.
    __device__ __forceinline__ void softmax(int key, bool edge) {
#pragma unroll
        for (int b = 0; b < RBLK; ++b) {
            if (edge) {
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int at = 4 * j + e;  // (from key + 8 kg on)
                        s[b][j][e] = at > last[b] - key - 8 * kg || at < first[b] - key - 8 * kg ? -kInf : s[b][j][e];
                    }
            }
            float top = fmaxf(fmaxf(fmaxf(s[b][0][0], s[b][0][1]), fmaxf(s[b][0][2], s[b][0][3])),
                              fmaxf(fmaxf(s[b][1][0], s[b][1][1]), fmaxf(s[b][1][2], s[b][1][3])));
            const float mx = Limb::across_max(top);
            // (a row of nothing but -inf so far: m stays -inf, weights are 0)
            if (__builtin_amdgcn_ballot_w64(mx * c[b] > m[b] * c[b] + kLag) != 0) {
                const float mn = fmaxf(m[b], mx);
                const float a = mn == -kInf ? 1.0f : exp2_fast((m[b] - mn) * c[b]);
                m[b] = mn;
                l[b] *= a;
#pragma unroll
                for (int i = 0; i < NT; ++i) o[b][i] *= a;
            }
            const float base = static_cast<float>(kBias) - (m[b] == -kInf ? 0.0f : m[b]) * c[b];
            float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    s[b][j][e] = exp2_fast(__builtin_fmaf(s[b][j][e], c[b], base));
                    if constexpr (NL > 1) sum[e] += s[b][j][e];
                }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint32_t x[NL];
                Limb::limbs(s[b][i >> 1][2 * (i & 1)], s[b][i >> 1][2 * (i & 1) + 1], x);
#pragma unroll
                for (int k = 0; k < NL; ++k) w[b][k][i] = x[k];
                // (the sum of the weights as they multiply v)
                if constexpr (NL == 1) sum[i] = Limb::sum2(x[0], sum[i]);
            }
            l[b] += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        }
    }
    // a and b made 0 for values that are no numbers and for keys before `begin` and
    // behind `end` (no row sees those); whether some of the first were met.
    __device__ __forceinline__ bool clean(Tile& x, int key, int begin, int end) const {
        bool any = false;
#pragma unroll
        for (int u = 0; u < SETS; ++u)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int sh = 16 * (i & 1);
                const int at = key + 8 * kg + i;
                const bool unseen = at < begin || at > end;
                const bool bad = no_number(x.va[u][i >> 1] >> sh, x.vb[u][i >> 1] >> sh);
                any |= bad && !unseen;
                const uint32_t keep = bad || unseen ? ~(0xffffu << sh) : ~0u;
                x.va[u][i >> 1] &= keep;
                x.vb[u][i >> 1] &= keep;
            }
        return any;
    }
    // o += P V.  Two keys' words are exchanged by halves, so that each has the
    // same four values of both.
    __device__ __forceinline__ void pv(Tile& tile) {
        if (__builtin_amdgcn_ballot_w64(tile.no_values) != 0) {
#pragma unroll
            for (int u = 0; u < SETS; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    tile.va[u][i] = tile.no_values ? 0u : tile.va[u][i];
                    tile.vb[u][i] = tile.no_values ? 0u : tile.vb[u][i];
                }
        }
#pragma unroll
        for (int u = 0; u < SETS; ++u)
#pragma unroll
            for (int h = 0; h < (HD == 64 ? 1 : 2); ++h) {
                const bool high = HD == 64 ? (n & 1) != 0 : h != 0;
                const uint32_t sel = high ? 0x07060302u : 0x05040100u, swapped = high ? 0x06070203u : 0x04050001u;
                uint32_t x[4];
                auto exchange = [&](uint32_t by) {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        x[i] = __builtin_amdgcn_perm(tile.vc[u][i >> 1][2 * (i & 1) + 1], tile.vc[u][i >> 1][2 * (i & 1)], by);
                };
                auto step = [&](int t, auto values) {
                    u32x4 a;
#pragma unroll
                    for (int i = 0; i < 4; ++i) a[i] = values(x[i], halves(tile.va[u][i]), halves(tile.vb[u][i]));
#pragma unroll
                    for (int k = NL - 1; k >= 0; --k)
#pragma unroll
                        for (int b = 0; b < RBLK; ++b) o[b][t] = mma(a, w[b][k], o[b][t]);
                };
                const int t = u * 8 + h * 4;
                exchange(sel);
                step(t, [&](uint32_t y, h2 a, h2 b) { return codes.template values<0>(y, a, b); });
                step(t + 1, [&](uint32_t y, h2 a, h2 b) { return codes.template values<1>(y, a, b); });
                step(t + 2, [&](uint32_t y, h2 a, h2 b) { return codes.template values<2>(y, a, b); });
                exchange(swapped);
                step(t + 3, [&](uint32_t y, h2 a, h2 b) { return codes.template values<3>(y, a, b); });
            }
    }
    // NaN to the rows that see `key` where its group of this lane's dims is no number.
    __device__ __forceinline__ void add_special(const Pages4& g, int key) {
#pragma unroll
        for (int u = 0; u < SETS; ++u) {
            const uint32_t ab = value_numbers_of<HD>(g, key, HD == 64 ? kg >> 1 : kg + 4 * u);
            if (!no_number(ab, ab >> 16)) continue;
#pragma unroll
            for (int b = 0; b < RBLK; ++b)
                if (key <= last[b] && key >= first[b])
#pragma unroll
                    for (int t = 0; t < NT / SETS; ++t) o[b][u * 8 + t] = f32x4{NAN, NAN, NAN, NAN};
        }
    }
};

// LDS of it: the waves' states, and at least the join's.
constexpr int few_lds(int waves, int bm, int hd) {
    const int join = waves * 64 * static_cast<int>(sizeof(State));
    return waves * bm * hd * 4 > join ? waves * bm * hd * 4 : join;
}

// A wave's priority goes down as its range is done, a step each quarter: a SIMD
// serves its oldest wave first, and of as many ranges of one length some would end
// at two thirds of the time and leave the others alone, with their latencies.
struct Progress {
    int quarter, until, level = 3;
    __device__ __forceinline__ explicit Progress(int steps) : quarter(max(steps / 4, 1)), until(quarter) {
        __builtin_amdgcn_s_setprio(3);
    }
    __device__ __forceinline__ void step() {
        if (--until != 0) return;
        until = quarter;
        if (level == 3) __builtin_amdgcn_s_setprio(2);
        else if (level == 2) __builtin_amdgcn_s_setprio(1);
        else __builtin_amdgcn_s_setprio(0);
        --level;
    }
};

// Workgroups of it that a CU holds: by the registers.
constexpr int few_per_cu(int waves, int bm, int hd) { return waves > 4 ? 1 : bm == 16 && hd < 256 ? 3 : 2; }

// (f32 rows' second limbs do not all fit the registers: 16 bytes of a lane go to memory
// in blocks of 32 rows at head_dim 128, 20 at 256.  64 requests decoding, whose form has
// none there, 56.5 us, bf16 rows 53.4; 16 requests of 5 tokens 28.3 and 24.3; a window
// of 1024 at head_dim 256 19.8, f16 rows 16.5.)
template <class Q, int HD, int RBLK, int NW>
__global__ __launch_bounds__(NW * 64, few_per_cu(NW, 16 * RBLK, HD)) void k_paged4_narrow(PagedAttn p, Launch la) {
    constexpr int DB = 16, BM = DB * RBLK, BK = 32, BN = NW * BK, NT = NW * 64;
    using C = Few<Q, HD, RBLK>;
    constexpr int kPart = part_floats(BM, HD);
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];  // the waves' states; a join's results
    float* const states = reinterpret_cast<float*>(lds);
    __shared__ float sm[NW][BM], sl[NW][BM];
    __shared__ int flag;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int nw = gridDim.x, w = place_of(blockIdx.x, nw);
    // Tiles that take as long as an item's start and end.  (us with 0, 1, 2, 3, 4, head_dim
    // 128: 64 requests decoding in four waves 77.7, 54.3, 54.3, 55.0, 55.2, 128 of up to 3000
    // keys 53.4, 40.7, 39.7, 42.0, 42.4; 16 requests of 5 tokens in eight waves 33.7, 27.5,
    // 26.4, 24.3, 24.5, 24 of 9 tokens 47.0, 31.9, 28.3, 28.1, 27.5.)
    constexpr int EXTRA = NW == 4 ? 2 : 3;
    Walk<BM, BN, EXTRA> walk(p, la);
    int64_t skip = 0, per = 0;
    int64_t left = find_range<NT>(walk, w, nw, &skip, &per);
    int64_t item_at = w * per - skip + EXTRA;  // of the item's first tile in the sequence
    const float c1 = p.scale * kLog2e;
    C core;
    core.setup();
    Progress progress(static_cast<int>(min(left, int64_t{0x7fffffff})));
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
        const int low_pos = pos0 + walk.token(row_first);
        const Pages4 pages = pages4_of<HD>(p, walk.s, walk.kvh, hi - 1);
        const uint32_t key0 = static_cast<uint32_t>(walk.tile0 + a) * BN + wave * BK;  // (below 2^31 + 2^10)
        int nt = b - a;
        if (static_cast<int64_t>(key0) + static_cast<int64_t>(nt - 1) * BN >= hi) --nt;  // (the last tile's keys may end before this wave's)
        const uint32_t my_k = 8u * (core.n >> 2), my_v = 8u * core.kg;
        int id_k = 0, id_v = 0;  // pages of the tile that is loaded next
        typename C::Tile tile;
        auto find = [&](int i) {
            id_k = page4_at(pages, key0 + i * BN + my_k);
            id_v = page4_at(pages, key0 + i * BN + my_v);
        };
        if (nt > 0) find(0);
        // (q is asked for before the first tile, so that it can be made limbs of while that is on its way)
        typename C::Row row_q[RBLK];
#pragma unroll
        for (int i = 0; i < RBLK; ++i) {
            const int r = i * DB + core.n, row = row_first + r;
            const bool real = r < rows;
            const int t = walk.token(row);
            row_q[i] = core.load_row(real ? static_cast<const Q*>(p.q) + (walk.row0 + t) * p.q_stride +
                                                (walk.kvh * walk.group + walk.head(row, t)) * HD
                                          : nullptr);
            core.last[i] = real ? pos0 + t : -1;
            core.first[i] = walk.first_seen(core.last[i]);
        }
        if (nt > 0) {
            core.load_keys(tile, pages, key0, id_k);
            core.load_values(tile, pages, key0, id_v);
            find(1);
        }
#pragma unroll
        for (int i = 0; i < RBLK; ++i) core.set_q(i, row_q[i], c1);
        auto is_edge = [&](int key) { return key + BK - 1 > low_pos || (p.window && hi - 1 - key >= p.window); };
        bool special = false;
        // (The loads of a tile go into the registers that the products before it have
        // left.  With a second set, sent a whole tile ahead, 64 requests decoding took as long.)
        for (int i = 0; i < nt; ++i) {
            const uint32_t at = key0 + i * BN;
            const int key = static_cast<int>(at);
            const bool edge = is_edge(key), more = i + 1 < nt;
            progress.step();
            core.scores(tile);
            if (more) core.load_keys(tile, pages, at + BN, id_k);
            core.softmax(key, edge);
            if (edge) special |= __builtin_amdgcn_ballot_w64(core.clean(tile, key, lo, hi - 1)) != 0;
            core.pv(tile);
            if (more) {
                core.load_values(tile, pages, at + BN, id_v);
                find(i + 2);
            }
        }
        if (special) {
            for (int i = 0; i < nt; ++i)
                if (const int key = static_cast<int>(key0) + i * BN; is_edge(key))
                    for (int j = 0; j < min(BK, hi - key); ++j) core.add_special(pages, key + j);
        }
        // The waves' states, joined in order.
        float* const mine = states + wave * (BM * HD);
#pragma unroll
        for (int i = 0; i < RBLK; ++i) {
            const int r = i * DB + core.n;
            const float l = C::Limb::across_sum(core.l[i]);
            if (core.kg == 0) {
                sm[wave][r] = core.m[i] * core.c[i];
                sl[wave][r] = l;
            }
#pragma unroll
            for (int u = 0; u < C::SETS; ++u)
#pragma unroll
                for (int e = 0; e < (HD == 64 ? 2 : 4); ++e)
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        // four neighbouring dims: a word's 4 x ..
                        f32x4 y;
                        if constexpr (HD == 64)
                            y = f32x4{core.o[i][2 * x][2 * e], core.o[i][2 * x][2 * e + 1], core.o[i][2 * x + 1][2 * e],
                                      core.o[i][2 * x + 1][2 * e + 1]};
                        else
                            y = f32x4{core.o[i][8 * u + 2 * x][e], core.o[i][8 * u + 4 + 2 * x][e], core.o[i][8 * u + 2 * x + 1][e],
                                      core.o[i][8 * u + 4 + 2 * x + 1][e]};
                        const int d = 128 * u + C::W * core.kg + 8 * e + 4 * x;
                        *reinterpret_cast<f32x4*>(mine + r * HD + (d ^ (4 * (core.n & 7)))) = y;
                    }
        }
        __syncthreads();
        const int first_wg = static_cast<int>(item_at / per), last_wg = static_cast<int>((item_at + walk.tiles - 1) / per);
        const bool cut = first_wg != last_wg;
        float* const part = la.part + (static_cast<int64_t>(w) * 2 + (w == first_wg)) * kPart;
        for (int i = tid; i < rows * (HD / 4); i += NT) {
            const int r = i / (HD / 4), d = (i % (HD / 4)) * 4;
            float M = -kInf, L = 0.0f;
#pragma unroll
            for (int x = 0; x < NW; ++x) M = fmaxf(M, sm[x][r]);
            f32x4 O = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int x = 0; x < NW; ++x) {
                const float f = M == -kInf ? 1.0f : state_weight(sm[x][r] - M);
                L += sl[x][r] * f;
                O += *reinterpret_cast<const f32x4*>(states + x * (BM * HD) + r * HD + (d ^ (4 * (r & 7)))) * f;
            }
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
        if (cut) {
            if (arrive(la.counters + first_wg, last_wg - first_wg + 1, &flag))
                join_parts<Q, BM, HD, NT>(walk, first_wg, last_wg, rows, reinterpret_cast<State*>(lds));
        }
        __syncthreads();  // the states are read
        item_at += walk.tiles + EXTRA;
        if (left > 0 && !walk.next()) break;
    }
}

// ---- many rows: the waves split the rows -------------------------------------------
// As paged_attention.hip's, but for how tiles reach LDS: a lane's word of codes
// and its numbers are loaded a step ahead into registers, and become 16 bytes of
// the tile among the products.  LDS holds two tiles of K and two of V.
// Keys of its tiles.  (At head_dim 256 the words on their way to 64 do not fit the
// registers beside the rest.  Nor do all of f32 rows' limbs: 56 bytes of a lane go to
// memory in eight waves at head_dim 128, 100 at 256.  2048 tokens over 8048 keys 431 us,
// bf16 rows 271, of half as many products; 512 over 4512 at head_dim 256 109 and 93.)
constexpr int wide4_keys(int hd) { return hd == 256 ? 32 : 64; }

template <class Q, int HD, int NW>
__global__ __launch_bounds__(NW * 64) void k_paged4_wide(PagedAttn p, Launch la) {
    constexpr int DB = 32, BM = DB * NW, BK = wide4_keys(HD), BN = BK, NT = NW * 64;
    using C = Core<Q, _Float16, HD, DB, 1, BK>;
    constexpr int COPIES = BK / C::RPI / NW;  // pieces of a tile of K, or of V, by each wave: RPI keys
    constexpr int GROUPS = (COPIES * C::RPI + 7) / 8;
    constexpr int kPart = wide_part_floats(BM, HD);
    static_assert(COPIES >= 1 && COPIES * NW * C::RPI == BK && (COPIES * C::RPI) % 8 == 0, "every wave has as many pieces, of whole groups");
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];  // two tiles of K, two of V
    __shared__ int special;  // the last of this workgroup's items whose v held what was made 0
    __shared__ int flag;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int nw = gridDim.x, w = place_of(blockIdx.x, nw);
    constexpr int EXTRA = NW == 8 ? 6 : 3;  // tiles that take as long as an item's start and end
    Walk<BM, BN, EXTRA> walk(p, la);
    int64_t skip = 0, per = 0;
    int64_t left = find_range<NT>(walk, w, nw, &skip, &per);
    int64_t item_at = w * per - skip + EXTRA;  // of the item's first tile in the sequence
    const uint32_t lds_at = uniform(static_cast<int>(lds_address(lds)));
    const float c1 = p.scale * kLog2e;
    if (tid == 0) special = -1;
    int item = 0;
    const Codes codes;
    C core;
    core.setup();
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
        const int low_pos = pos0 + walk.token(row_first);
        const int r = wave * DB + core.n, row = row_first + r;
        const bool real = r < rows;
        const int t = walk.token(row);
        const int64_t head = (walk.kvh * walk.group + walk.head(row, t)) * HD;
        // the wave's rows see keys from wave_lo to wave_hi
        const int wave_low = pos0 + walk.token(row_first + min(wave * DB, rows - 1));
        const int wave_hi = pos0 + walk.token(row_first + min(wave * DB + DB, rows) - 1);
        const Pages4 pages = pages4_of<HD>(p, walk.s, walk.kvh, hi - 1);
        const uint32_t key0 = static_cast<uint32_t>(walk.tile0 + a) * BN;
        const int nt = hi > 0 ? b - a : 0;
        auto is_edge = [&](int key) { return key + BK - 1 > low_pos || (p.window && hi - 1 - key >= p.window); };
        // A wave's pieces of a tile are of GROUPS groups of 8 keys.  Where a group is, from
        // the pages' first bytes, for the keys that are loaded next and for the
        // values, a tile behind them; behind the last key its group.
        struct Place {
            int64_t codes, numbers;  // the first slot's; below 0: on a page that is none
        };
        uint32_t kc[COPIES], kn[COPIES], vc[COPIES], va[COPIES], vb[COPIES];
        int id[GROUPS];  // pages of the groups a tile further on
        Place at_k[GROUPS], at_v[GROUPS];
        auto group_of = [&](int i, int x) {
            return min(key0 + static_cast<uint32_t>(i * BN + wave * COPIES * C::RPI + 8 * x), static_cast<uint32_t>(pages.end)) & ~7u;
        };
        auto find_pages = [&](int i) {
#pragma unroll
            for (int x = 0; x < GROUPS; ++x) id[x] = pages.table[group_of(i, x) >> pages.shift];
        };
        auto find_places = [&](int i) {
#pragma unroll
            for (int x = 0; x < GROUPS; ++x) {
                const int page = uniform(id[x]);
                const uint32_t slot = static_cast<uint32_t>(uniform(static_cast<int>(group_of(i, x)))) & ((1u << pages.shift) - 1);
                const int64_t first = static_cast<int64_t>(static_cast<uint64_t>(static_cast<uint32_t>(page)) * pages.page_bytes);
                at_v[x] = at_k[x];
                at_k[x].codes = real_page(pages, page) ? first + Page4<HD>::codes(slot) : -1;
                at_k[x].numbers = first + Page4<HD>::numbers(slot, pages.shift);
            }
        };
        const uint8_t* const none = reinterpret_cast<const uint8_t*>(kZeros);
        // This lane's slot of a piece's group, and its word: as tiles lie in LDS.
        auto slot_of = [&](int x) { return static_cast<uint32_t>((wave * COPIES + x) * C::RPI & 7) + static_cast<uint32_t>(lane / C::CPR); };
        auto word_of = [&](int x, bool v) {
            const int row = (wave * COPIES + x) * C::RPI + lane / C::CPR;
            return static_cast<uint32_t>((lane % C::CPR) ^ (v ? C::swz_v(row) : C::swz_k(row)));
        };
        auto fetch_k = [&](int x) {
            const Place& g = at_k[x * C::RPI / 8];
            const uint8_t* const codes_at = g.codes < 0 ? none : pages.k + g.codes;
            const uint8_t* const numbers_at = g.codes < 0 ? none : pages.k + g.numbers;
            const uint32_t c = word_of(x, false);
            kc[x] = *(const GLOBAL_AS uint32_t*)(codes_at + Page4<HD>::key_word(slot_of(x), c));
            kn[x] = *(const GLOBAL_AS uint32_t*)(numbers_at + Page4<HD>::key_number(slot_of(x), c >> 2));
        };
        auto fetch_v = [&](int x) {
            const Place& g = at_v[x * C::RPI / 8];
            const uint8_t* const codes_at = g.codes < 0 ? none : pages.v + g.codes;
            const uint8_t* const numbers_at = g.codes < 0 ? none : pages.v + g.numbers;
            const uint32_t c = word_of(x, true);
            vc[x] = *(const GLOBAL_AS uint32_t*)(codes_at + Page4<HD>::value_word(slot_of(x), c));
            const uint32_t number = Page4<HD>::value_number(slot_of(x), c >> 2);
            va[x] = *(const GLOBAL_AS uint16_t*)(numbers_at + number);
            vb[x] = *(const GLOBAL_AS uint16_t*)(numbers_at + number + 16);
        };
        auto put = [&](uint32_t tile, int x, u32x4 y) {
            *(LDS_AS u32x4*)(static_cast<uintptr_t>(tile + (wave * COPIES + x) * 1024 + lane * 16)) = y;
        };
        auto put_k = [&](int slot, int x) { put(lds_at + slot * C::TB, x, codes.word(kc[x], kn[x])); };
        auto put_v = [&](int slot, int x, int key, bool edge) {
            uint32_t ab = va[x] | vb[x] << 16;
            if (edge) {
                const int at = key + (wave * COPIES + x) * C::RPI + lane / C::CPR;
                const bool unseen = at < lo || at > pages.end, bad = no_number(ab, ab >> 16);
                if (__builtin_amdgcn_ballot_w64(bad && !unseen) != 0) special = item;
                ab = bad || unseen ? 0u : ab;
            }
            put(lds_at + (2 + slot) * C::TB, x, codes.word(vc[x], ab));
        };
        lds_barrier();  // (every wave is done with the item before)
        if (nt > 0) {
            find_pages(0);
            find_places(0);
            find_pages(1);
#pragma unroll
            for (int x = 0; x < COPIES; ++x) fetch_k(x);
#pragma unroll
            for (int x = 0; x < COPIES; ++x) put_k(0, x);
            find_places(1);
            find_pages(2);
#pragma unroll
            for (int x = 0; x < COPIES; ++x) fetch_v(x);
#pragma unroll
            for (int x = 0; x < COPIES; ++x) fetch_k(x);
        }
        core.load_q(0, real ? static_cast<const Q*>(p.q) + (walk.row0 + t) * p.q_stride + head : nullptr, c1);
        core.last[0] = real ? pos0 + t : -1;
        core.first[0] = walk.first_seen(core.last[0]);
        lds_barrier();
        // Step i: the products, O += P V of tile i - 1 and the scores of tile i, and
        // the weighing of tile i; a wave among its products goes before one that weighs.
        // (2048 tokens over 8048 keys, us, f16 and bf16 rows: 267 and 273.  The second
        // four waves a half step behind the first, with a barrier between the halves:
        // 275 and 274, there without priorities 283 and 284; on a slower card 293 and
        // 293 where this takes 286 and 288.)
        // Among its products a wave puts V of tile i and K of tile i + 1 where V of
        // tile i - 2 and K of tile i - 1 were, whose products every wave has behind
        // it, and sends the loads of the tiles behind them.
        if (nt > 0) {
            for (int i = 0; i <= nt; ++i) {
                const int now = i & 1;
                const bool edge_v = is_edge(static_cast<int>(key0 + i * BN));
                // (no branch around the products of what is not there or not seen: the
                // weights of a tile that no row of the wave sees are 0 and its V is
                // clean, being an edge tile; in step 0 the accumulator is cleared
                // after; scores of no tile are not used)
                __builtin_amdgcn_s_setprio(1);
                core.template products<2 * COPIES>(lds_at + now * C::TB, lds_at + (2 + (now ^ 1)) * C::TB, [&](int x) {
                    if (x == 0) {
                        find_places(i + 2);
                        find_pages(i + 3);
                    }
                    if (x < COPIES) {
                        put_v(now, x, static_cast<int>(key0 + i * BN), edge_v);
                        fetch_v(x);
                    } else {
                        put_k(now ^ 1, x - COPIES);
                        fetch_k(x - COPIES);
                    }
                });
                __builtin_amdgcn_s_setprio(0);
                if (i == 0) core.no_values();
                // (behind the last tile: from hi on, keys that no row sees, which change nothing)
                const int key = i < nt ? static_cast<int>(key0) + i * BN : hi;
                core.softmax(key, i == nt || key + BK - 1 > wave_low || (p.window && wave_hi - key >= p.window));
                lds_barrier();
            }
        }
        if (uniform(special) == item) {
            for (int i = 0; i < nt; ++i)
                if (const int key = static_cast<int>(key0) + i * BN; is_edge(key))
                    for (int j = 0; j < min(BK, hi - key); ++j)
                        if (key + j <= core.last[0] && key + j >= core.first[0])
#pragma unroll
                            for (int g = 0; g < C::NC; ++g)  // (a block of o is a group's 32 dims)
                                if (const uint32_t ab = value_numbers_of<HD>(pages, key + j, g); no_number(ab, ab >> 16))
                                    for (int e = 0; e < C::ACC; ++e) core.o[0][g][e] = NAN;
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
        ++item;
        if (!whole) {
            whole = arrive(la.counters + first_wg, last_wg - first_wg + 1, &flag);
            if (whole) {
                float M = -kInf;
                l = 0.0f;
                core.no_values();
                for (int x = first_wg; x <= last_wg; ++x) {
                    const float* const src = part(x);
                    const float m = ld_dev(src + BM * HD), sum = ld_dev(src + BM * HD + NT);
                    float o[C::NC * C::ACC];
#pragma unroll
                    for (int i = 0; i < C::NC * C::ACC; ++i) o[i] = ld_dev(src + i * NT);
                    __builtin_amdgcn_sched_barrier(0);  // (all loads before the first use)
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
        item_at += walk.tiles + EXTRA;
        if (left > 0 && !walk.next()) break;
    }
}

// Rows of a request up to which its keys are split over the waves.
constexpr int kFewRows = 32;

// Rows of a block of the few-row form; the waves of a workgroup; its workgroups,
// those the CUs hold at once.  Where two waves to a SIMD are all that the
// registers allow, they are one workgroup of eight or two of four: one has fewer
// states to join across workgroups, two work on while one of them ends an item.
// us, four and eight waves: blocks of 32 rows at head_dim 128, 16 requests of 5
// tokens 35.5 and 24.3, 24 of 9 tokens 35.7 and 28.2.  head_dim 256: 64 and 128 items
// 21.1 and 16.8, 34.3 and 27.0; 512 items, 64 requests decoding, 52.3 and 56.5.
int few_block(int64_t rows, int hd) { return rows <= 16 || hd == 256 ? 16 : 32; }
int few_waves(const PagedAttn& p, int64_t rows) {
    if (p.kv.head_dim < 256) return few_block(rows, p.kv.head_dim) == 16 ? 4 : 8;
    return static_cast<int64_t>(p.n_seq) * p.kv.n_kv > slots() ? 4 : 8;
}
int few_slots(const PagedAttn& p, int64_t rows) {
    return slots() * few_per_cu(few_waves(p, rows), few_block(rows, p.kv.head_dim), p.kv.head_dim);
}

// Whether blocks of 256 rows, eight waves, or of 128, four (as over 16-bit caches).
bool eight_waves(const PagedAttn& p, int64_t rows) {
    return p.kv.head_dim < 256 && rows > 128 && static_cast<int64_t>(p.n_tokens) * p.n_q >= slots() * int64_t{40};
}

template <class Q, int HD>
hipError_t run(const PagedAttn& p, float* part, uint32_t* counters, hipStream_t s) {
    Launch la = launch_of(p, part, counters);
    const int64_t rows = most_rows(p);
    const bool wide = rows > kFewRows, narrow = !wide || p.n_seq > 1;
    if (wide) {
        constexpr int MOST = HD == 256 ? 4 : 8;
        la.min_rows = narrow ? kFewRows : 0;
        const bool eight = MOST == 8 && eight_waves(p, rows);
        hipLaunchKernelGGL((eight ? k_paged4_wide<Q, HD, MOST> : k_paged4_wide<Q, HD, 4>), dim3(static_cast<unsigned>(slots())),
                           dim3(eight ? 512 : 256), 4 * wide4_keys(HD) * HD * 2, s, p, la);
    }
    if (narrow) {
        la.min_rows = 0;
        la.max_rows = wide ? kFewRows : 0x7fffffff;
        const unsigned grid = static_cast<unsigned>(few_slots(p, rows));
        auto launch = [&](auto blocks, auto waves) {
            constexpr int B = decltype(blocks)::value, NW = decltype(waves)::value;
            hipLaunchKernelGGL((k_paged4_narrow<Q, HD, B, NW>), dim3(grid), dim3(NW * 64), few_lds(NW, 16 * B, HD), s, p, la);
        };
        using std::integral_constant;
        if constexpr (HD < 256) {
            if (few_block(rows, HD) == 16) launch(integral_constant<int, 1>(), integral_constant<int, 4>());
            else launch(integral_constant<int, 2>(), integral_constant<int, 8>());
        } else {
            if (few_waves(p, rows) == 4) launch(integral_constant<int, 1>(), integral_constant<int, 4>());
            else launch(integral_constant<int, 1>(), integral_constant<int, 8>());
        }
    }
    return hipGetLastError();
}

template <class Q>
hipError_t run_hd(const PagedAttn& p, float* part, uint32_t* counters, hipStream_t s) {
    switch (p.kv.head_dim) {
        case 64: return run<Q, 64>(p, part, counters, s);
        case 128: return run<Q, 128>(p, part, counters, s);
        default: return run<Q, 256>(p, part, counters, s);
    }
}

}  // namespace

size_t paged4_attention_workspace(const PagedAttn& p) {
    const int64_t rows = most_rows(p);
    const int hd = p.kv.head_dim, waves = hd < 256 ? 8 : 4;
    const auto few = [&](int64_t rows) { return static_cast<size_t>(few_slots(p, rows)) * 2 * part_floats(few_block(rows, hd), hd); };
    // (enough for steps of fewer rows too: blocks of 16 take more than ones of 32)
    const size_t narrow = few(1) > few(rows) ? few(1) : few(rows);
    const size_t wide = rows > kFewRows ? static_cast<size_t>(slots()) * 2 * wide_part_floats(waves * 32, hd) : 0;
    return (narrow > wide ? narrow : wide) * sizeof(float);
}

hipError_t launch_paged4_attention(const PagedAttn& p, void* part, uint32_t* counters, hipStream_t s) {
    if (static_cast<size_t>(few_slots(p, most_rows(p))) > kArrivalCounters) return hipErrorInvalidValue;
    float* const f = static_cast<float*>(part);
    if (p.dtype == RT_HIP_BF16) return run_hd<__bf16>(p, f, counters, s);
    if (p.dtype == RT_HIP_F16) return run_hd<_Float16>(p, f, counters, s);
    return run_hd<float>(p, f, counters, s);
}

}  // namespace rt_hip
