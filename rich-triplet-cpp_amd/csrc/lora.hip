// lora.hip -- low-rank adapters of many requests beside a shared projection:
//   y[row] += scale[i] * B_i (A_i x[row]),   i the adapter of the row's request.
//
// Two launches.  The first, t = A x, takes 16 rows of one request and a slice of
// k; the second adds B t, 16 rows and a part of n.  The lengths of the requests
// are on the device: a launch has a workgroup for every block that there could
// be, and each finds its own among the requests.  Slices of k leave their sums in
// the workspace and the second launch adds them in order, so results do not
// depend on who was first.  (One call behind another one token takes 7.1 us, 64
// decoding requests 16.0.  In one launch, each workgroup of the second computing t for
// itself, 8.2 and 18.1 where the two took 7.4 and 15.7, 32 of 5 rows 12.9 and 10.6.)
//
// Products on the bf16 matrix cores with f32's accuracy: x and t as three bf16
// values that add up to the f32 one, bf16 weights as they are, f16 ones as two
// (the product of the two last is below 2^-24 of the whole and left out).
// An infinity has zeros for its other parts, whose products with one are NaN, and
// what f32 holds past bf16's largest number becomes one: a sum that is no number is
// computed again from the factors themselves.
#include "paged_rows.hpp"
#include "rt_common.hpp"
#include "rt_launch.hpp"
#include "wave_scan.hpp"

namespace rt_hip {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// Eight f32 values as three bf16 each.
struct Limbs {
    u32x4 h, m, l;
};
__device__ __forceinline__ Limbs limbs_of(f32x4 a, f32x4 b) {
    u32x2 h0, m0, l0, h1, m1, l1;
    bf16_limbs4(a, h0, m0, l0);
    bf16_limbs4(b, h1, m1, l1);
    return {u32x4{h0[0], h0[1], h1[0], h1[1]}, u32x4{m0[0], m0[1], m1[0], m1[1]}, u32x4{l0[0], l0[1], l1[0], l1[1]}};
}

// Eight weights a lane: bf16 as they are in memory, f16 as two bf16 each.
template <class W> struct Weights;
template <> struct Weights<__bf16> {
    u32x4 w;
    __device__ __forceinline__ explicit Weights(u32x4 raw) : w(raw) {}
    // c + w x, weights along the rows; along the columns.
    __device__ __forceinline__ f32x4 times(const Limbs& x, f32x4 c) const {
        c = mma(w, x.l, c);
        c = mma(w, x.m, c);
        return mma(w, x.h, c);
    }
    __device__ __forceinline__ f32x4 under(const Limbs& x, f32x4 c) const {
        c = mma(x.l, w, c);
        c = mma(x.m, w, c);
        return mma(x.h, w, c);
    }
};
template <> struct Weights<_Float16> {
    u32x4 hi, lo;
    __device__ __forceinline__ explicit Weights(u32x4 raw) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t u = raw[i];
            const float a = f16_bits_to_f32(u & 0xffffu), b = f16_bits_to_f32(u >> 16);
            const uint32_t top = bf16_pair(a, b);
            hi[i] = top;
            // (11 bits: what 8 leave fits the next 8.  An infinity stays alone.)
            const float ra = fabsf(a) < 65520.0f ? a - bf16_lo_to_f32(top) : 0.0f;
            const float rb = fabsf(b) < 65520.0f ? b - bf16_hi_to_f32(top) : 0.0f;
            lo[i] = bf16_pair(ra, rb);
        }
    }
    __device__ __forceinline__ f32x4 times(const Limbs& x, f32x4 c) const {
        c = mma(hi, x.l, c);
        c = mma(lo, x.m, c);
        c = mma(hi, x.m, c);
        c = mma(lo, x.h, c);
        return mma(hi, x.h, c);
    }
    __device__ __forceinline__ f32x4 under(const Limbs& x, f32x4 c) const {
        c = mma(x.l, hi, c);
        c = mma(x.m, lo, c);
        c = mma(x.m, hi, c);
        c = mma(x.h, lo, c);
        return mma(x.h, hi, c);
    }
};

// Eight values of x, as they are in memory, as limbs.
template <class X>
__device__ __forceinline__ Limbs limbs_at(const uint8_t* p) {
    const u32x4 a = ld16(p);
    if constexpr (sizeof(X) == 4) {
        return limbs_of(__builtin_bit_cast(f32x4, a), *reinterpret_cast<const f32x4*>(p + 16));
    } else if constexpr (__is_same(X, __bf16)) {
        return {a, u32x4{0, 0, 0, 0}, u32x4{0, 0, 0, 0}};
    } else {
        f32x4 x, y;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t u = a[i], v = a[i + 2];
            x[2 * i] = f16_bits_to_f32(u & 0xffffu);
            x[2 * i + 1] = f16_bits_to_f32(u >> 16);
            y[2 * i] = f16_bits_to_f32(v & 0xffffu);
            y[2 * i + 1] = f16_bits_to_f32(v >> 16);
        }
        return limbs_of(x, y);
    }
}

// Whether some of four values is an infinity or a NaN.
__device__ __forceinline__ bool no_numbers(f32x4 v) {
    float any = 0.0f;
#pragma unroll
    for (int e = 0; e < 4; ++e) any = __builtin_fmaf(v[e], 0.0f, any);
    return any != any;
}

// What a wave has stored to its part of LDS is there for all of its lanes (they
// are served in order; this is for the compiler).
__device__ __forceinline__ void wave_fence() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); __builtin_amdgcn_wave_barrier(); }

// Block `index` of the rows that have an adapter: its rows and that adapter.
struct Block {
    int row, rows, adapter;
};
template <int kRows>
__device__ __forceinline__ bool find_block(const LoraAdd& p, int index, Block* out) {
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int s0 = 0; s0 < p.n_seq; s0 += 64) {
        const int s = s0 + lane;
        int row = 0, rows = 0, adapter = -1;
        if (s < p.n_seq) {
            row = min(max(p.row_start[s], 0), p.n_rows);
            rows = min(max(p.row_start[s + 1], row), p.n_rows) - row;
            adapter = p.adapter[s];
            if (static_cast<uint32_t>(adapter) >= static_cast<uint32_t>(p.n_adapters)) rows = 0;
        }
        const int blocks = (rows + kRows - 1) / kRows, sum = running_sum(blocks), all = of_lane(sum, 63);
        if (index < before + all) {
            const int l = __builtin_ctzll(__builtin_amdgcn_ballot_w64(index < before + sum));
            const int b = index - before - of_lane(sum - blocks, l);
            out->row = of_lane(row, l) + b * kRows;
            out->rows = min(of_lane(rows, l) - b * kRows, kRows);
            out->adapter = of_lane(adapter, l);
            return true;
        }
        before += all;
    }
    return false;
}

// Operands take one row to a lane, 16 lanes at 16 rows: loaded so, every lane's 16
// bytes are an access of their own for the cache.  So waves load rows 64 bytes and
// more at a time and turn them in LDS, each in a part of its own, its rows 16 bytes
// apart for the banks.

// t = A x of a block of 16 RB rows over a slice of k: RT tiles of 16 ranks.  The
// four waves take 32 values of k in turn, and their sums are added in LDS.
// (Waves to a SIMD: as many as the products' registers leave, which the code for
// sums that are no numbers would otherwise lower by one.  The same in the second
// launch: 2700 rows in both 38 us, without the bounds 44.)
template <class X, class W, int RT, int RB>
__global__ __launch_bounds__(256, RT < 4 ? 1 : sizeof(X) == 4 && RT * RB >= 8 ? 2 : 3) void k_lora_shrink(LoraAdd p) {
    constexpr int kAhead = RT * RB >= 8 ? 2 : 4;  // steps whose loads are in flight together
    constexpr int XB = 32 * sizeof(X), XC = XB / 16, XL = 16 * RB * XC / 64;  // bytes of a row of x in a step, chunks, loads
    constexpr int XS = XB + 16, WS = 64 + 16;  // bytes between rows in LDS
    constexpr int kWave = 16 * RB * XS + 16 * RT * WS, kSums = 3 * RB * RT * 64 * 16;
    __shared__ __attribute__((aligned(16))) uint8_t lds[4 * kWave > kSums ? 4 * kWave : kSums];
    Block blk;
    if (!find_block<16 * RB>(p, blockIdx.x, &blk)) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 15, kg = lane >> 4;
    const int k0 = blockIdx.y * p.k_slice, k1 = min(p.k, k0 + p.k_slice);
    uint8_t* const xs = lds + wave * kWave;
    uint8_t* const ws = xs + 16 * RB * XS;
    // This lane's chunks: of row lane / XC (+ 64 / XC for each further load) of x, of rank lane / 4 (+ 16) of a.
    const X* x[XL];
    const W* a[RT];
    bool there[XL];
#pragma unroll
    for (int i = 0; i < XL; ++i) {
        const int row = i * (64 / XC) + lane / XC;
        there[i] = row < blk.rows;
        x[i] = static_cast<const X*>(p.x) + static_cast<int64_t>(blk.row + (there[i] ? row : 0)) * p.x_stride;
    }
    // (ranks past the last repeat that: no one reads their sums)
#pragma unroll
    for (int t = 0; t < RT; ++t)
        a[t] = static_cast<const W*>(p.a) + (static_cast<int64_t>(blk.adapter) * p.rank + min(t * 16 + lane / 4, p.rank - 1)) * p.k;
    f32x4 c[RB][RT];
#pragma unroll
    for (int b = 0; b < RB; ++b)
#pragma unroll
        for (int t = 0; t < RT; ++t) c[b][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    for (int kk = k0 + wave * 32; kk < k1; kk += 128 * kAhead) {
        u32x4 w[kAhead][RT], v[kAhead][XL];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int at_x = kk + u * 128 + lane % XC * (16 / static_cast<int>(sizeof(X))), at_w = kk + u * 128 + lane % 4 * 8;
#pragma unroll
            for (int t = 0; t < RT; ++t) w[u][t] = at_w < k1 ? ld16(a[t] + at_w) : u32x4{0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < XL; ++i) v[u][i] = there[i] && at_x < k1 ? ld16(x[i] + at_x) : u32x4{0, 0, 0, 0};
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            if (u > 0 && kk + u * 128 >= k1) break;
            wave_fence();  // (the step before is read)
#pragma unroll
            for (int i = 0; i < XL; ++i)
                *reinterpret_cast<u32x4*>(xs + (i * (64 / XC) + lane / XC) * XS + lane % XC * 16) = v[u][i];
#pragma unroll
            for (int t = 0; t < RT; ++t) *reinterpret_cast<u32x4*>(ws + (t * 16 + lane / 4) * WS + lane % 4 * 16) = w[u][t];
            wave_fence();
            Limbs l[RB];
#pragma unroll
            for (int b = 0; b < RB; ++b) l[b] = limbs_at<X>(xs + (b * 16 + n) * XS + kg * (8 * sizeof(X)));
#pragma unroll
            for (int t = 0; t < RT; ++t) {
                const Weights<W> m(ld16(ws + (t * 16 + n) * WS + kg * 16));
#pragma unroll
                for (int b = 0; b < RB; ++b) c[b][t] = m.times(l[b], c[b][t]);
            }
        }
    }
    __syncthreads();
    f32x4(*const sums)[RB][RT][64] = reinterpret_cast<f32x4(*)[RB][RT][64]>(lds);
    if (wave > 0) {
#pragma unroll
        for (int b = 0; b < RB; ++b)
#pragma unroll
            for (int t = 0; t < RT; ++t) sums[wave - 1][b][t][lane] = c[b][t];
    }
    __syncthreads();
    if (wave > 0) return;
    float* const out = p.part + (static_cast<int64_t>(blockIdx.y) * p.n_rows + blk.row) * p.rank;
    uint32_t again = 0;  // tiles of this lane's with sums that are no numbers
#pragma unroll
    for (int b = 0; b < RB; ++b) {
        if (b * 16 + n >= blk.rows) continue;
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            const int r = t * 16 + kg * 4;  // (the rank is a multiple of 8)
            if (r >= p.rank) continue;
            const f32x4 sum = ((c[b][t] + sums[0][b][t][lane]) + sums[1][b][t][lane]) + sums[2][b][t][lane];
            *reinterpret_cast<f32x4*>(out + (b * 16 + n) * p.rank + r) = sum;
            if (no_numbers(sum)) again |= 1u << (b * RT + t);
            if (t % 4 == 3) __builtin_amdgcn_sched_barrier(0);  // (not all tiles' sums in registers at once)
        }
    }
#pragma unroll 1
    for (; again != 0; again &= again - 1) {
        const int i = __builtin_ctz(again), row = i / RT * 16 + n, r = i % RT * 16 + kg * 4;
        const X* const xr = static_cast<const X*>(p.x) + static_cast<int64_t>(blk.row + row) * p.x_stride;
        const W* const ar = static_cast<const W*>(p.a) + (static_cast<int64_t>(blk.adapter) * p.rank + r) * p.k;
        f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 1
        for (int kk = k0; kk < k1; kk += 8) {
            float xv[8], av[8];
            load8(xr + kk, xv);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                load8(ar + q * p.k + kk, av);
#pragma unroll
                for (int e = 0; e < 8; ++e) sum[q] = __builtin_fmaf(xv[e], av[e], sum[q]);
            }
            if (sum[0] != sum[0] && sum[1] != sum[1] && sum[2] != sum[2] && sum[3] != sum[3]) break;  // (NaN they stay)
        }
        *reinterpret_cast<f32x4*>(out + row * p.rank + r) = sum;
    }
}

// y += B t of a block over p.cols columns: RS steps of 32 ranks.  Rows of t along
// the rows of the product, so that a lane has one column of four rows and 16
// lanes 64 bytes of a row of y.
template <class W, int RS, int RB>
__global__ __launch_bounds__(256, RS * RB == 8 ? 2 : RS * RB == 4 ? 4 : RS * RB == 2 ? 5 : 8) void k_lora_expand(LoraAdd p) {
    constexpr int kAhead = 2;  // tiles of 16 columns whose loads are in flight together
    constexpr int TS = RS * 64 + 16, kT = 16 * RB * TS;  // bytes between rows of t, and of weights; of a limb of t
    constexpr int kTile = 16 * TS, kWaves = 4 * kAhead * kTile;
    __shared__ __attribute__((aligned(16))) uint8_t lds[3 * kT > kWaves ? 3 * kT : kWaves];
    __shared__ __attribute__((aligned(16))) float whole[16 * RB][RS * 32];  // t as it is
    Block blk;
    if (!find_block<16 * RB>(p, blockIdx.x, &blk)) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 15, kg = lane >> 4;
    const float scale = p.scale[blk.adapter];
    // t of the block, the slices' sums added in order, as limbs in LDS; then in registers.
    const int quads = p.rank / 4;
    for (int i = threadIdx.x; i < 16 * RB * quads; i += 256) {
        const int row = i / quads, r = (i - row * quads) * 4;
        f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
        if (row < blk.rows) {
            const float* at = p.part + (static_cast<int64_t>(blk.row) + row) * p.rank + r;
#pragma unroll 4
            for (int s = 0; s < p.slices; ++s, at += static_cast<int64_t>(p.n_rows) * p.rank) sum += *reinterpret_cast<const f32x4*>(at);
        }
        sum *= scale;
        *reinterpret_cast<f32x4*>(&whole[row][r]) = sum;
        u32x2 h, m, l;
        bf16_limbs4(sum, h, m, l);
        uint8_t* const to = lds + row * TS + r * 2;
        *reinterpret_cast<u32x2*>(to) = h;
        *reinterpret_cast<u32x2*>(to + kT) = m;
        *reinterpret_cast<u32x2*>(to + 2 * kT) = l;
    }
    __syncthreads();
    Limbs t[RB][RS];
#pragma unroll
    for (int b = 0; b < RB; ++b)
#pragma unroll
        for (int q = 0; q < RS; ++q) {
            const uint8_t* const at = lds + (b * 16 + n) * TS + q * 64 + kg * 16;
            const bool in = q * 32 + kg * 8 < p.rank;
            t[b][q].h = in ? ld16(at) : u32x4{0, 0, 0, 0};
            t[b][q].m = in ? ld16(at + kT) : u32x4{0, 0, 0, 0};
            t[b][q].l = in ? ld16(at + 2 * kT) : u32x4{0, 0, 0, 0};
        }
    __syncthreads();
    // The weights of 16 columns are neighbours in memory: chunk i of them is column i / (rank / 8)'s.
    const int chunks = p.rank / 8;
    int col_of[RS], to_of[RS];  // of this lane's chunks: the column, the place in LDS
#pragma unroll
    for (int q = 0; q < RS; ++q) {
        const int i = q * 64 + lane;
        col_of[q] = i / chunks;
        to_of[q] = col_of[q] * TS + (i - col_of[q] * chunks) * 16;
    }
    uint8_t* const ws = lds + wave * (kAhead * kTile);
    const W* const b0 = static_cast<const W*>(p.b) + static_cast<int64_t>(blk.adapter) * p.n * p.rank;
    float* const y = p.y + static_cast<int64_t>(blk.row) * p.y_stride;
    const int c1 = min(p.n, (static_cast<int>(blockIdx.y) + 1) * p.cols);
    int c0 = blockIdx.y * p.cols + wave * (16 * kAhead);
    for (; c0 < c1; c0 += 64 * kAhead) {
        u32x4 w[kAhead][RS];
        f32x4 old[kAhead][RB];
        // Values of this lane in block b, tile u: rows 16 b + 4 kg + e.  (No row of the
        // wave from the first past the block's on, as for single tokens 15 of 16.)
        auto each = [&](auto f) {
#pragma unroll
            for (int b = 0; b < RB; ++b)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (b * 16 + e >= blk.rows) continue;
                    const int row = b * 16 + 4 * kg + e;
#pragma unroll
                    for (int u = 0; u < kAhead; ++u)
                        if (const int col = c0 + u * 16 + n; row < blk.rows && col < c1) f(u, b, e, y + row * p.y_stride + col);
                }
        };
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
#pragma unroll
            for (int q = 0; q < RS; ++q) {
                const bool in = col_of[q] < 16 && c0 + u * 16 + col_of[q] < c1;
                w[u][q] = in ? ld16(b0 + static_cast<int64_t>(c0 + u * 16) * p.rank + (q * 64 + lane) * 8) : u32x4{0, 0, 0, 0};
            }
        each([&](int u, int b, int e, const float* at) { old[u][b][e] = *at; });
        wave_fence();  // (the tiles before are read)
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
#pragma unroll
            for (int q = 0; q < RS; ++q)
                if (col_of[q] < 16) *reinterpret_cast<u32x4*>(ws + u * kTile + to_of[q]) = w[u][q];
        wave_fence();
        f32x4 c[kAhead][RB];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
#pragma unroll
            for (int b = 0; b < RB; ++b) c[u][b] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int q = 0; q < RS; ++q) {
                const bool in = q * 32 + kg * 8 < p.rank;
                const Weights<W> m(in ? ld16(ws + u * kTile + n * TS + q * 64 + kg * 16) : u32x4{0, 0, 0, 0});
#pragma unroll
                for (int b = 0; b < RB; ++b) c[u][b] = m.under(t[b][q], c[u][b]);
            }
        }
        bool again = false;  // some sum of this lane's is no number
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
#pragma unroll
            for (int b = 0; b < RB; ++b) again |= no_numbers(c[u][b]);
        if (__builtin_amdgcn_ballot_w64(again) != 0) break;
        each([&](int u, int b, int e, float* at) { *at = old[u][b][e] + c[u][b][e]; });
    }
    // From the first such sum on: the same products tile by tile, where they are numbers.
#pragma unroll 1
    for (; c0 < c1; c0 += 64 * kAhead)
#pragma unroll 1
        for (int u = 0; u < kAhead; ++u) {
            const int col = c0 + u * 16 + n;
            const W* const w = b0 + static_cast<int64_t>(col) * p.rank;
            f32x4 c[RB];
#pragma unroll
            for (int b = 0; b < RB; ++b) c[b] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int q = 0; q < RS; ++q) {
                const bool in = col < c1 && q * 32 + kg * 8 < p.rank;
                const Weights<W> m(in ? ld16(w + q * 32 + kg * 8) : u32x4{0, 0, 0, 0});
#pragma unroll
                for (int b = 0; b < RB; ++b) c[b] = m.under(t[b][q], c[b]);
            }
            uint32_t which = 0;
#pragma unroll
            for (int b = 0; b < RB; ++b)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int row = b * 16 + 4 * kg + e;
                    if (row >= blk.rows || col >= c1) continue;
                    if (fabsf(c[b][e]) < __builtin_inff()) y[row * p.y_stride + col] += c[b][e];
                    else which |= 1u << (b * 4 + e);
                }
#pragma unroll 1
            for (; which != 0; which &= which - 1) {
                const int i = __builtin_ctz(which), row = i / 4 * 16 + 4 * kg + i % 4;
                float sum = 0.0f;
#pragma unroll 1
                for (int r = 0; r < p.rank && sum == sum; r += 8) {
                    float wv[8];
                    load8(w + r, wv);
#pragma unroll
                    for (int e = 0; e < 8; ++e) sum = __builtin_fmaf(whole[row][r + e], wv[e], sum);
                }
                y[row * p.y_stride + col] += sum;
            }
        }
}

// Blocks of 16 rows that a workgroup takes together, in each launch: two where
// requests have as many rows on average, so that weights are read, and f16 ones
// split, half as often.  (One in the first launch past rank 64, whose sums leave no
// registers: 4000 rows at rank 128 61 us, with two 75.  Four in the second: 2700
// rows at rank 64 62 us, with two 54.)
int tall(int n_seq, int n_rows, int most) { return most == 2 && n_rows / n_seq >= 32 ? 2 : 1; }
int tall_shrink(int rank, int n_seq, int n_rows) { return tall(n_seq, n_rows, rank > 64 ? 1 : 2); }
int tall_expand(int n_seq, int n_rows) { return tall(n_seq, n_rows, 2); }
// Blocks that there can be: every request's last may be partly empty.
int64_t most_blocks(int n_seq, int n_rows, int tall) {
    const int64_t b = (static_cast<int64_t>(n_rows) + 16 * tall - 1) / (16 * tall) + n_seq - 1;
    return b < n_rows ? b : n_rows;
}
// Slices of k: so that there are two workgroups to a CU, of 512 values each at least.
// (Every workgroup of the second launch reads all slices' sums of its rows: with
// as many slices again 2048 rows at rank 16 are no faster, 4000 at rank 128 slower.)
int slices_of(int rank, int n_seq, int n_rows, int k) {
    const int64_t blocks = most_blocks(n_seq, n_rows, tall_shrink(rank, n_seq, n_rows));
    const int64_t want = (2 * static_cast<int64_t>(device_info().cus) + blocks - 1) / blocks, most = (static_cast<int64_t>(k) + 511) / 512;
    return static_cast<int>(want < most ? want : most);
}

template <class X, class W, int RB>
void shrink(const LoraAdd& p, dim3 grid, hipStream_t s) {
    auto kernel = p.rank <= 16 ? k_lora_shrink<X, W, 1, RB> : p.rank <= 32 ? k_lora_shrink<X, W, 2, RB> : k_lora_shrink<X, W, 4, RB>;
    if constexpr (RB == 1)  // (two blocks go up to rank 64)
        if (p.rank > 64) kernel = k_lora_shrink<X, W, 8, RB>;
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, p);
}
template <class X, class W>
void shrink_rows(const LoraAdd& p, dim3 grid, hipStream_t s) {
    if (tall_shrink(p.rank, p.n_seq, p.n_rows) == 2) shrink<X, W, 2>(p, grid, s);
    else shrink<X, W, 1>(p, grid, s);
}
template <class W, int RB>
void expand(const LoraAdd& p, dim3 grid, hipStream_t s) {
    const auto kernel = p.rank <= 32 ? k_lora_expand<W, 1, RB> : p.rank <= 64 ? k_lora_expand<W, 2, RB> : k_lora_expand<W, 4, RB>;
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, p);
}

template <class W>
void run(LoraAdd p, hipStream_t s) {
    const dim3 slices(static_cast<unsigned>(most_blocks(p.n_seq, p.n_rows, tall_shrink(p.rank, p.n_seq, p.n_rows))), static_cast<unsigned>(p.slices));
    switch (p.x_dtype) {
        case RT_HIP_F32: shrink_rows<float, W>(p, slices, s); break;
        case RT_HIP_F16: shrink_rows<_Float16, W>(p, slices, s); break;
        default: shrink_rows<__bf16, W>(p, slices, s);
    }
    // Columns of a workgroup of the second launch: a multiple of its 128 of a step, so
    // that there are at most four workgroups to a CU.  (With eight 2048 rows at rank 16
    // take 27.4 us instead of 24.7, 64 decoding requests 15.8 instead of 15.3.)
    const int rows = tall_expand(p.n_seq, p.n_rows);
    const int64_t blocks = most_blocks(p.n_seq, p.n_rows, rows), steps = (static_cast<int64_t>(p.n) + 127) / 128;
    const int64_t most = 4 * static_cast<int64_t>(device_info().cus), want = (blocks * steps + most - 1) / most;
    p.cols = static_cast<int>(128 * (want < steps ? want : steps));
    const dim3 parts(static_cast<unsigned>(blocks), (static_cast<unsigned>(p.n) + static_cast<unsigned>(p.cols) - 1) / static_cast<unsigned>(p.cols));
    if (rows == 2) expand<W, 2>(p, parts, s);
    else expand<W, 1>(p, parts, s);
}

}  // namespace

// Enough for as many rows and fewer, of however many requests, though fewer blocks take
// more slices: b blocks of at most 16 t rows take below 2 CUs / b + 1.
size_t lora_workspace(int rank, int k, int n_rows) {
    const int64_t rows = n_rows, most = (static_cast<int64_t>(k) + 511) / 512 * rows;
    const int64_t some = 2 * static_cast<int64_t>(device_info().cus) * 16 * (rank > 64 ? 1 : 2) + rows;
    return static_cast<size_t>(most < some ? most : some) * rank * sizeof(float);
}

hipError_t launch_lora_add(LoraAdd p, hipStream_t s) {
    p.slices = slices_of(p.rank, p.n_seq, p.n_rows, p.k);
    p.k_slice = ((p.k + p.slices - 1) / p.slices + 127) / 128 * 128;
    if (p.w_dtype == RT_HIP_BF16) run<__bf16>(p, s);
    else run<_Float16>(p, s);
    return hipGetLastError();
}

}  // namespace rt_hip
