// lora.hip -- low-rank adapters of many requests beside a shared projection:
//   y[row] += scale[i] * B_i (A_i x[row]),   i the adapter of the row's request.
//
// Two launches.  The first, t = A x, takes 16 rows of one request and a slice of
// k; the second adds B t, 16 rows and a part of n.  The lengths of the requests
// are on the device: a launch has a workgroup for every block that there could
// be, and each finds its own among the requests.  Slices of k leave their sums in
// the workspace and the second launch adds them in order, so results do not
// depend on who was first.
//
// Products on the bf16 matrix cores with f32's accuracy: x and t as three bf16
// values that add up to the f32 one, bf16 weights as they are, f16 ones as two
// (the product of the two last is below 2^-24 of the whole and left out).
#include "rt_common.hpp"
#include "rt_launch.hpp"
#include "wave_scan.hpp"

namespace rt_hip {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr int kRows = 16;  // of a block

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

// c + w x for eight weights a lane, as they are in memory.
template <class W>
__device__ __forceinline__ f32x4 add_product(u32x4 w, const Limbs& x, f32x4 c) {
    if constexpr (__is_same(W, __bf16)) {
        c = mma(w, x.l, c);
        c = mma(w, x.m, c);
        return mma(w, x.h, c);
    } else {
        u32x4 hi, lo;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t u = w[i];
            const float a = f16_bits_to_f32(u & 0xffffu), b = f16_bits_to_f32(u >> 16);
            const uint32_t top = bf16_pair(a, b);
            hi[i] = top;
            // (11 bits: what 8 leave fits the next 8.  An infinity stays alone.)
            const float ra = fabsf(a) < 65520.0f ? a - bf16_lo_to_f32(top) : 0.0f;
            const float rb = fabsf(b) < 65520.0f ? b - bf16_hi_to_f32(top) : 0.0f;
            lo[i] = bf16_pair(ra, rb);
        }
        c = mma(hi, x.l, c);
        c = mma(lo, x.m, c);
        c = mma(hi, x.m, c);
        c = mma(lo, x.h, c);
        return mma(hi, x.h, c);
    }
}

// Eight values of a row of x.
__device__ __forceinline__ Limbs load_x(const float* p) {
    return limbs_of(*reinterpret_cast<const f32x4*>(p), *reinterpret_cast<const f32x4*>(p + 4));
}
__device__ __forceinline__ Limbs load_x(const __bf16* p) {
    return {ld16(p), u32x4{0, 0, 0, 0}, u32x4{0, 0, 0, 0}};
}
__device__ __forceinline__ Limbs load_x(const _Float16* p) {
    const u32x4 u = ld16(p);
    f32x4 a, b;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        a[2 * i] = f16_bits_to_f32(u[i] & 0xffffu);
        a[2 * i + 1] = f16_bits_to_f32(u[i] >> 16);
        b[2 * i] = f16_bits_to_f32(u[i + 2] & 0xffffu);
        b[2 * i + 1] = f16_bits_to_f32(u[i + 2] >> 16);
    }
    return limbs_of(a, b);
}

// Block `index` of the rows that have an adapter: its rows and that adapter.
struct Block {
    int row, rows, adapter;
};
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

// t = A x of a block over a slice of k: RT tiles of 16 ranks.  The four waves
// take 32 values of k in turn, and their sums are added in LDS.
template <class X, class W, int RT>
__global__ __launch_bounds__(256) void k_lora_shrink(LoraAdd p) {
    __shared__ __attribute__((aligned(16))) f32x4 sums[3][RT][64];
    Block blk;
    if (!find_block(p, blockIdx.x, &blk)) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 15, kg = lane >> 4;
    const int k0 = blockIdx.y * p.k_slice, k1 = min(p.k, k0 + p.k_slice);
    const X* const x = static_cast<const X*>(p.x) + static_cast<int64_t>(blk.row + min(n, blk.rows - 1)) * p.x_stride;
    const W* const a = static_cast<const W*>(p.a) + static_cast<int64_t>(blk.adapter) * p.rank * p.k;
    f32x4 c[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) c[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    // (rows past the block's repeat its last, ranks past the last repeat that: no one reads their sums)
    for (int kk = k0 + wave * 32; kk < k1; kk += 128) {
        const int at = kk + kg * 8;
        const bool in = at < k1;
        u32x4 w[RT];
#pragma unroll
        for (int t = 0; t < RT; ++t)
            w[t] = in ? ld16(a + static_cast<int64_t>(min(t * 16 + n, p.rank - 1)) * p.k + at) : u32x4{0, 0, 0, 0};
        const Limbs v = in ? load_x(x + at) : Limbs{u32x4{0, 0, 0, 0}, u32x4{0, 0, 0, 0}, u32x4{0, 0, 0, 0}};
#pragma unroll
        for (int t = 0; t < RT; ++t) c[t] = add_product<W>(w[t], v, c[t]);
    }
    if (wave > 0) {
#pragma unroll
        for (int t = 0; t < RT; ++t) sums[wave - 1][t][lane] = c[t];
    }
    __syncthreads();
    if (wave > 0 || n >= blk.rows) return;
    float* const out = p.part + (static_cast<int64_t>(blockIdx.y) * p.n_rows + blk.row + n) * p.rank;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        const int r = t * 16 + kg * 4;  // (the rank is a multiple of 8)
        if (r < p.rank) *reinterpret_cast<f32x4*>(out + r) = ((c[t] + sums[0][t][lane]) + sums[1][t][lane]) + sums[2][t][lane];
    }
}

// y += B t of a block over kCols columns: RS steps of 32 ranks.
constexpr int kCols = 256;
template <class W, int RS>
__global__ __launch_bounds__(256) void k_lora_expand(LoraAdd p) {
    Block blk;
    if (!find_block(p, blockIdx.x, &blk)) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 15, kg = lane >> 4;
    const bool mine = n < blk.rows;
    const float scale = p.scale[blk.adapter];
    Limbs t[RS];
#pragma unroll
    for (int q = 0; q < RS; ++q) {
        const int r = q * 32 + kg * 8;
        f32x4 lo = {0.0f, 0.0f, 0.0f, 0.0f}, hi = lo;
        if (mine && r < p.rank)
            for (int s = 0; s < p.slices; ++s) {
                const float* const at = p.part + (static_cast<int64_t>(s) * p.n_rows + blk.row + n) * p.rank + r;
                lo += *reinterpret_cast<const f32x4*>(at);
                hi += *reinterpret_cast<const f32x4*>(at + 4);
            }
        t[q] = limbs_of(lo * scale, hi * scale);
    }
    const W* const b = static_cast<const W*>(p.b) + static_cast<int64_t>(blk.adapter) * p.n * p.rank;
    float* const y = p.y + static_cast<int64_t>(blk.row + (mine ? n : 0)) * p.y_stride;
    const int c1 = min(p.n, (static_cast<int>(blockIdx.y) + 1) * kCols);
    for (int c0 = blockIdx.y * kCols + wave * 16; c0 < c1; c0 += 64) {
        f32x4 c = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int q = 0; q < RS; ++q) {
            const int r = q * 32 + kg * 8;
            const u32x4 w = r < p.rank ? ld16(b + static_cast<int64_t>(min(c0 + n, p.n - 1)) * p.rank + r) : u32x4{0, 0, 0, 0};
            c = add_product<W>(w, t[q], c);
        }
        const int col = c0 + kg * 4;
        if (!mine || col >= c1) continue;
        if (p.y_wide) {
            f32x4* const at = reinterpret_cast<f32x4*>(y + col);
            *at += c;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (col + e < p.n) y[col + e] += c[e];
        }
    }
}

template <class X, class W>
void shrink(const LoraAdd& p, dim3 grid, hipStream_t s) {
    const auto kernel = p.rank <= 16 ? k_lora_shrink<X, W, 1> : p.rank <= 32 ? k_lora_shrink<X, W, 2>
                        : p.rank <= 64 ? k_lora_shrink<X, W, 4> : k_lora_shrink<X, W, 8>;
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, p);
}
template <class W>
void run(const LoraAdd& p, unsigned blocks, hipStream_t s) {
    const dim3 slices(blocks, static_cast<unsigned>(p.slices));
    switch (p.x_dtype) {
        case RT_HIP_F32: shrink<float, W>(p, slices, s); break;
        case RT_HIP_F16: shrink<_Float16, W>(p, slices, s); break;
        default: shrink<__bf16, W>(p, slices, s);
    }
    const dim3 parts(blocks, (static_cast<unsigned>(p.n) + kCols - 1) / kCols);
    const auto kernel = p.rank <= 32 ? k_lora_expand<W, 1> : p.rank <= 64 ? k_lora_expand<W, 2> : k_lora_expand<W, 4>;
    hipLaunchKernelGGL(kernel, parts, dim3(256), 0, s, p);
}

// Blocks that there can be: every request's last may be partly empty.
int64_t most_blocks(int n_seq, int n_rows) {
    const int64_t b = (static_cast<int64_t>(n_rows) + kRows - 1) / kRows + n_seq - 1;
    return b < n_rows ? b : n_rows;
}
// Slices of k: as many workgroups as twice the CUs, of 512 values each at least.
int slices_of(int n_seq, int n_rows, int k) {
    const int64_t want = (2 * static_cast<int64_t>(device_info().cus) + most_blocks(n_seq, n_rows) - 1) / most_blocks(n_seq, n_rows);
    const int64_t most = (static_cast<int64_t>(k) + 511) / 512;
    return static_cast<int>(want < most ? want : most);
}

}  // namespace

size_t lora_workspace(int rank, int k, int n_seq, int n_rows) {
    return static_cast<size_t>(slices_of(n_seq, n_rows, k)) * n_rows * rank * sizeof(float);
}

hipError_t launch_lora_add(LoraAdd p, hipStream_t s) {
    p.slices = slices_of(p.n_seq, p.n_rows, p.k);
    p.k_slice = ((p.k + p.slices - 1) / p.slices + 127) / 128 * 128;
    const unsigned blocks = static_cast<unsigned>(most_blocks(p.n_seq, p.n_rows));
    if (p.w_dtype == RT_HIP_BF16) run<__bf16>(p, blocks, s);
    else run<_Float16>(p, blocks, s);
    return hipGetLastError();
}

}  // namespace rt_hip
