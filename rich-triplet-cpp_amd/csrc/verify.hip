// verify.hip -- drafted tokens accepted or replaced by the target model's
// distributions, from given random numbers.
//
// Row r of the logits predicts token r + 1 of its request, so row r judges
// the draft d = tokens[r + 1].  With p and q the target's and the draft
// model's softmax(x / T) (q certain of d without draft logits; T = 0: certain
// of the first largest token), drafts are accepted in order while
//   u_r q(d) < p(d),
// and the token after the accepted ones is the first v whose running sum of w
// exceeds u_s sum(w), where w = max(0, p - q) at the first refused row (p if
// that is zero everywhere) and w = p after the last draft.  The tokens are
// then distributed as if drawn from p alone.
//
// Which token is chosen depends on sums over the vocabulary next to a border,
// so weights and sums are in 64 bits: a token of probability 1e-5 then changes
// hands with odds below 1e-10, with 32-bit sums 1e-3.
//
// Two launches: k_verify_stats reads every row once, in chunks, and leaves
// each chunk's maximum and sum of exp((x - maximum) / T); k_verify_pick joins
// them (every workgroup of a request for itself), decides on the drafts, sums
// w of the deciding row by chunks and, in the request's last workgroup to
// arrive, finds the chunk that holds the border and the token in it.  Rows of
// a request whose T is 0 need no sums.
//
// Bound: the bytes of the logits.  A 64-bit exponential is about 20
// instructions at the rate of 32-bit ones, 21 us of the card for 320 rows of
// 128256 values, which take 30 us to read.
#include "rt_common.hpp"
#include "rt_launch.hpp"

namespace rt_hip {
namespace {

constexpr int kT = 256;
constexpr int kQuads = 4;                  // groups of 4 values a thread holds
constexpr int kChunk = kT * 4 * kQuads;    // values of a row per workgroup
constexpr float kInf = __builtin_inff();

struct Stat {
    double sum;   // of exp((x - top) / T) over the chunk
    float top;    // its maximum, NaN aside (-inf: nothing above)
    int32_t idx;  // where that first stands
};

// exp(x) for x <= 0 (zero below -745): 2^n times the Taylor polynomial of
// degree 12 in |r| <= ln(2) / 2, whose remainder is below 2e-16.
__device__ __forceinline__ double exp64(double x) {
    x = fmax(x, -800.0);
    const double n = __builtin_rint(x * 1.4426950408889634074);
    double r = __builtin_fma(n, -6.93147180369123816490e-01, x);
    r = __builtin_fma(n, -1.90821492927058770002e-10, r);
    double y = 1.0 / 479001600.0;
    y = __builtin_fma(y, r, 1.0 / 39916800.0);
    y = __builtin_fma(y, r, 1.0 / 3628800.0);
    y = __builtin_fma(y, r, 1.0 / 362880.0);
    y = __builtin_fma(y, r, 1.0 / 40320.0);
    y = __builtin_fma(y, r, 1.0 / 5040.0);
    y = __builtin_fma(y, r, 1.0 / 720.0);
    y = __builtin_fma(y, r, 1.0 / 120.0);
    y = __builtin_fma(y, r, 1.0 / 24.0);
    y = __builtin_fma(y, r, 1.0 / 6.0);
    y = __builtin_fma(y, r, 0.5);
    y = __builtin_fma(y, r, 1.0);
    y = __builtin_fma(y, r, 1.0);
    return __builtin_ldexp(y, static_cast<int>(n));
}

// Weight of x in a row whose maximum is top > -inf (the rule for infinities:
// what equals the maximum weighs 1).
__device__ __forceinline__ double weight(float x, float top, double inv_t) {
    if (x == top) return 1.0;
    if (!(x > -kInf)) return 0.0;
    return exp64((static_cast<double>(x) - static_cast<double>(top)) * inv_t);
}

typedef float f32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint16_t u16x4_a2 __attribute__((ext_vector_type(4), aligned(2)));

// Four values at p (any alignment); past the row's end -inf.
__device__ __forceinline__ void load4(const float* row, int at, int n, float (&x)[4]) {
    if (at + 4 <= n) {
        const f32x4_a4 v = *reinterpret_cast<const f32x4_a4*>(row + at);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = v[e];
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = at + e < n ? row[at + e] : -kInf;
    }
}
__device__ __forceinline__ void load4(const uint16_t* row, int at, int n, float (&x)[4]) {
    if (at + 4 <= n) {
        const u16x4_a2 v = *reinterpret_cast<const u16x4_a2*>(row + at);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = __uint_as_float(static_cast<uint32_t>(v[e]) << 16);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = at + e < n ? __uint_as_float(static_cast<uint32_t>(row[at + e]) << 16) : -kInf;
    }
}
__device__ __forceinline__ float load1(const float* row, int at) { return row[at]; }
__device__ __forceinline__ float load1(const uint16_t* row, int at) {
    return __uint_as_float(static_cast<uint32_t>(row[at]) << 16);
}

// The request's temperature, 0 or above (NaN and negative ones: 0).
__device__ __forceinline__ float temperature_of(const VerifyDrafts& p, int s) {
    const float t = p.temperature ? p.temperature[s] : 1.0f;
    return t > 0.0f ? t : 0.0f;
}
// First row and number of drafts of request s, inside the arrays.
__device__ __forceinline__ int rows_of(const VerifyDrafts& p, int s, int* first) {
    const int a = min(max(p.row_start[s], 0), p.n_rows), b = min(max(p.row_start[s + 1], a), p.n_rows);
    *first = a;
    return min(b - a, p.max_draft + 1);  // rows; drafts are one fewer
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) v += __shfl_xor(v, off, kWave);
    return v;
}
__device__ __forceinline__ uint64_t wave_max(uint64_t v) {
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) {
        const uint64_t o = __shfl_xor(v, off, kWave);
        v = o > v ? o : v;
    }
    return v;
}
// Sum over the workgroup, the same bits in every thread.
__device__ __forceinline__ double block_sum(double v, double* tmp) {
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) tmp[threadIdx.x >> 6] = v;
    __syncthreads();
    return (tmp[0] + tmp[1]) + (tmp[2] + tmp[3]);
}
// Sum over the threads before this one; *total: over all of them.
__device__ __forceinline__ double block_before(double v, double* tmp, double* total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    double sum = v;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const double o = __shfl_up(sum, off, kWave);
        if (lane >= off) sum += o;
    }
    double before = __shfl_up(sum, 1, kWave);
    if (lane == 0) before = 0.0;
    __syncthreads();
    if (lane == 63) tmp[wave] = sum;
    __syncthreads();
    double all = 0.0, base = 0.0;
#pragma unroll
    for (int w = 0; w < kT / 64; ++w) {
        if (w == wave) base = all;
        all += tmp[w];
    }
    *total = all;
    return base + before;
}
// Of the weights in thread order (thread t's first[0 .. N) lie `before` it):
// the place of the first with which the running sum exceeds target, else of
// the last weight above 0, else -1.  place(e): where weight e stands, below 2^31.
template <int N, class F>
__device__ __forceinline__ int find_border(const double (&w)[N], double before, double target, F place, int* tmp2) {
    if (threadIdx.x == 0) {
        tmp2[0] = 0x7fffffff;
        tmp2[1] = -1;
    }
    __syncthreads();
    int hit = 0x7fffffff, heavy = -1;
#pragma unroll
    for (int e = 0; e < N; ++e) {
        before += w[e];
        if (w[e] > 0.0) {
            heavy = place(e);
            if (before > target && hit == 0x7fffffff) hit = heavy;
        }
    }
    if (hit != 0x7fffffff) atomicMin(tmp2, hit);
    if (heavy >= 0) atomicMax(tmp2 + 1, heavy);
    __syncthreads();
    return tmp2[0] != 0x7fffffff ? tmp2[0] : tmp2[1];
}

// Statistics [which][row][chunk]; grid (chunks, n_seq * (max_draft + 1), 1 or 2).
template <class X>
__global__ __launch_bounds__(kT) void k_verify_stats(VerifyDrafts p, Stat* __restrict__ stats) {
    __shared__ double tmp[4];
    __shared__ uint64_t tmp_key[4];
    const int s = blockIdx.y / (p.max_draft + 1), j = blockIdx.y % (p.max_draft + 1);
    const bool draft = blockIdx.z != 0;
    int first;
    const int rows = rows_of(p, s, &first);
    if (j >= rows || (draft && j + 1 >= rows)) return;
    const float temp = temperature_of(p, s);
    if (draft && temp == 0.0f) return;  // (greedy requests decide by the target alone)
    const int row = first + j, tid = threadIdx.x;
    const X* const x = static_cast<const X*>(draft ? p.draft_logits : p.logits) +
                       row * (draft ? p.draft_stride : p.logit_stride);
    const int c0 = blockIdx.x * kChunk;
    float v[kQuads][4];
#pragma unroll
    for (int i = 0; i < kQuads; ++i) load4(x, c0 + (i * kT + tid) * 4, p.vocab, v[i]);
    // first place of the maximum: larger values, then lower indices, have larger keys
    uint64_t key = 0;
#pragma unroll
    for (int i = 0; i < kQuads; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int at = c0 + (i * kT + tid) * 4 + e;
            const uint64_t k = v[i][e] == v[i][e] && at < p.vocab ? argmax_key(v[i][e], at) : 0;
            key = k > key ? k : key;
        }
    key = wave_max(key);
    if ((tid & 63) == 0) tmp_key[tid >> 6] = key;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kT / 64; ++w) key = tmp_key[w] > key ? tmp_key[w] : key;
    const uint32_t u = static_cast<uint32_t>(key >> 32);
    const float top = key == 0 ? -kInf : __uint_as_float((u & 0x80000000u) ? u & 0x7fffffffu : ~u);
    double sum = 0.0;
    if (temp > 0.0f && top > -kInf) {
        const double inv_t = 1.0 / static_cast<double>(temp);
#pragma unroll
        for (int i = 0; i < kQuads; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) sum += weight(v[i][e], top, inv_t);
        sum = block_sum(sum, tmp);
    }
    if (tid == 0) {
        Stat& o = stats[(static_cast<int64_t>(draft ? p.n_rows : 0) + row) * gridDim.x + blockIdx.x];
        o.sum = sum;
        o.top = top;
        o.idx = static_cast<int32_t>(0xffffffffu - static_cast<uint32_t>(key));
    }
}

// The row's maximum (-inf: nothing above), its first place and the sum, from
// its chunks; one wave, every lane ends with them.
struct RowStat {
    double inv_sum;
    float top;
    int idx;
};
__device__ __forceinline__ RowStat join_row(const Stat* st, int chunks, double inv_t) {
    const int lane = threadIdx.x & 63;
    uint64_t key = 0;
    for (int c = lane; c < chunks; c += 64) {
        const uint64_t k = st[c].top > -kInf ? argmax_key(st[c].top, static_cast<uint32_t>(st[c].idx)) : 0;
        key = k > key ? k : key;
    }
    key = wave_max(key);
    RowStat r;
    const uint32_t u = static_cast<uint32_t>(key >> 32);
    r.top = key == 0 ? -kInf : __uint_as_float((u & 0x80000000u) ? u & 0x7fffffffu : ~u);
    r.idx = key == 0 ? 0 : static_cast<int>(0xffffffffu - static_cast<uint32_t>(key));
    double sum = 0.0;
    for (int c = lane; c < chunks; c += 64) sum += st[c].sum * (key == 0 ? 0.0 : weight(st[c].top, r.top, inv_t));
    r.inv_sum = 1.0 / wave_sum(sum);
    return r;
}

// Probability from a row's joined statistics (nothing above -inf: certain of token 0).
__device__ __forceinline__ double prob(float x, int at, const RowStat& r, double inv_t) {
    if (r.top == -kInf) return at == 0 ? 1.0 : 0.0;
    return weight(x, r.top, inv_t) * r.inv_sum;
}

__device__ __forceinline__ void st_dev(double* p, double v) {
    __hip_atomic_store((__attribute__((address_space(1))) double*)p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ double ld_dev(const double* p) {
    return __hip_atomic_load((const __attribute__((address_space(1))) double*)p, __ATOMIC_RELAXED,
                             __HIP_MEMORY_SCOPE_AGENT);
}

// grid (chunks, n_seq); sums [n_seq][chunks].
template <class X>
__global__ __launch_bounds__(kT) void k_verify_pick(VerifyDrafts p, const Stat* __restrict__ stats,
                                                    double* __restrict__ sums, uint32_t* __restrict__ arrivals) {
    constexpr int kWaves = kT / 64;
    __shared__ RowStat best[kWaves][2];   // statistics of the row each wave saw first refused
    __shared__ int stop[kWaves];
    __shared__ double tmp[kWaves];
    __shared__ int last, tmp2[2];
    const int s = blockIdx.y, chunks = gridDim.x, tid = threadIdx.x, wave = tid >> 6;
    int first;
    const int rows = rows_of(p, s, &first);
    int32_t* const out = p.out_tokens + static_cast<int64_t>(s) * (p.max_draft + 1);
    if (rows == 0) {  // no rows, no tokens
        if (blockIdx.x == 0) {
            for (int i = tid; i <= p.max_draft; i += kT) out[i] = -1;
            if (tid == 0) p.out_count[s] = 0;
        }
        return;
    }
    const float temp = temperature_of(p, s);
    const double inv_t = temp > 0.0f ? 1.0 / static_cast<double>(temp) : 1.0;
    const Stat* const draft_stats = stats + static_cast<int64_t>(p.n_rows) * chunks;

    // Wave w takes rows w, w + 4, ..: the first that stops the request (a
    // refused draft, or the row behind the last draft).
    if ((tid & 63) == 0) stop[wave] = rows;
    for (int j = wave; j < rows; j += kWaves) {
        const int row = first + j;
        const RowStat rp = join_row(stats + static_cast<int64_t>(row) * chunks, chunks, inv_t);
        RowStat rq = rp;
        bool stops = j + 1 == rows;
        if (!stops) {
            const int d = p.tokens[row + 1];
            const bool real = static_cast<uint32_t>(d) < static_cast<uint32_t>(p.vocab);
            if (temp == 0.0f) {
                stops = d != rp.idx;
            } else {
                double pd = 0.0, qd = real ? 1.0 : 0.0;
                if (real) pd = prob(load1(static_cast<const X*>(p.logits) + row * p.logit_stride, d), d, rp, inv_t);
                if (p.draft_logits) {
                    rq = join_row(draft_stats + static_cast<int64_t>(row) * chunks, chunks, inv_t);
                    if (real) qd = prob(load1(static_cast<const X*>(p.draft_logits) + row * p.draft_stride, d), d, rq, inv_t);
                }
                stops = !(static_cast<double>(p.accept_u[row]) * qd < pd);
            }
        }
        if (stops) {
            if ((tid & 63) == 0) {
                stop[wave] = j;
                best[wave][0] = rp;
                best[wave][1] = rq;
            }
            break;
        }
    }
    __syncthreads();
    int j = rows, who = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w)
        if (stop[w] < j) {
            j = stop[w];
            who = w;
        }
    const RowStat rp = best[who][0], rq = best[who][1];
    const int row = first + j;
    const bool refused = j + 1 < rows;
    const int d = refused ? p.tokens[row + 1] : -1;
    if (blockIdx.x == 0) {
        for (int i = tid; i <= p.max_draft; i += kT)
            if (i != j) out[i] = i < j ? p.tokens[first + 1 + i] : -1;
        if (tid == 0) p.out_count[s] = j + 1;
    }
    if (temp == 0.0f || rp.top == -kInf) {  // a certain row
        if (blockIdx.x == 0 && tid == 0) out[j] = rp.idx;
        return;
    }
    const X* const x = static_cast<const X*>(p.logits) + row * p.logit_stride;
    const X* const y = p.draft_logits ? static_cast<const X*>(p.draft_logits) + row * p.draft_stride : nullptr;
    const Stat* const st = stats + static_cast<int64_t>(row) * chunks;

    // Weights of four values from `at` on.
    auto weights4 = [&](int at, bool rest, double (&w)[4]) {
        float xv[4], yv[4];
        load4(x, at, p.vocab, xv);
        if (rest && y) load4(y, at, p.vocab, yv);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            w[e] = at + e < p.vocab ? weight(xv[e], rp.top, inv_t) * rp.inv_sum : 0.0;
            if (rest) {
                const double q = y ? (at + e < p.vocab ? prob(yv[e], at + e, rq, inv_t) : 0.0) : (at + e == d ? 1.0 : 0.0);
                w[e] = fmax(w[e] - q, 0.0);
            }
        }
    };

    __shared__ double left;
    bool rest = refused;
    double* const mine = sums + static_cast<int64_t>(s) * chunks;
    if (refused) {
        double sum = 0.0;
#pragma unroll
        for (int i = 0; i < kQuads; ++i) {
            double w[4];
            weights4(blockIdx.x * kChunk + (i * kT + tid) * 4, true, w);
            sum += (w[0] + w[1]) + (w[2] + w[3]);
        }
        sum = block_sum(sum, tmp);
        if (tid == 0) {
            st_dev(mine + blockIdx.x, sum);
            wait_vmcnt<0>();
            last = __hip_atomic_fetch_add(arrivals + s, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
                   static_cast<uint32_t>(chunks) - 1;
        }
        __syncthreads();
        if (!last) return;
        if (tid == 0) __hip_atomic_store(arrivals + s, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    } else if (blockIdx.x != 0) {
        return;  // (the chunk sums of p are there: one workgroup finds the token)
    }

    // The chunk with the border: thread c holds chunk c's sum.
    double w1[1] = {0.0}, total;
    if (tid < chunks)
        w1[0] = rest ? ld_dev(mine + tid) : (st[tid].top > -kInf ? st[tid].sum * weight(st[tid].top, rp.top, inv_t) * rp.inv_sum : 0.0);
    double before = block_before(w1[0], tmp, &total);
    if (rest && !(total > 0.0)) {  // (p is nowhere above q: from p after all)
        rest = false;
        if (tid < chunks) w1[0] = st[tid].top > -kInf ? st[tid].sum * weight(st[tid].top, rp.top, inv_t) * rp.inv_sum : 0.0;
        before = block_before(w1[0], tmp, &total);
    }
    const double target = static_cast<double>(p.sample_u[s]) * total;
    const int border = find_border(w1, before, target, [&](int) { return tid; }, tmp2);
    if (tid == border) left = target - before;
    __syncthreads();
    // The token in it: thread t takes values [16 t, 16 t + 16) of the chunk,
    // the vocabulary's order.
    constexpr int kOwn = kChunk / kT;
    const int c0 = border * kChunk + tid * kOwn;
    double own = 0.0, w[kOwn];
#pragma unroll
    for (int i = 0; i < kOwn / 4; ++i) {
        double q[4];
        weights4(c0 + 4 * i, rest, q);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            w[4 * i + e] = q[e];
            own += q[e];
        }
    }
    before = block_before(own, tmp, &total);
    const int token = find_border(w, before, left, [&](int e) { return c0 + e; }, tmp2);
    if (tid == 0) out[j] = token;
}

int chunks_of(int vocab) { return (vocab + kChunk - 1) / kChunk; }

size_t stats_bytes(const VerifyDrafts& p) {
    return static_cast<size_t>(p.n_rows) * (p.draft_logits ? 2 : 1) * chunks_of(p.vocab) * sizeof(Stat);
}

template <class X>
hipError_t run(const VerifyDrafts& p, void* work, uint32_t* counters, hipStream_t s) {
    Stat* const stats = static_cast<Stat*>(work);
    double* const sums = reinterpret_cast<double*>(static_cast<uint8_t*>(work) + stats_bytes(p));
    const unsigned chunks = static_cast<unsigned>(chunks_of(p.vocab));
    const unsigned rows = static_cast<unsigned>(p.n_seq) * static_cast<unsigned>(p.max_draft + 1);
    hipLaunchKernelGGL(k_verify_stats<X>, dim3(chunks, rows, p.draft_logits ? 2 : 1), dim3(kT), 0, s, p, stats);
    hipLaunchKernelGGL(k_verify_pick<X>, dim3(chunks, static_cast<unsigned>(p.n_seq)), dim3(kT), 0, s, p, stats, sums,
                       counters);
    return hipGetLastError();
}

}  // namespace

size_t verify_drafts_workspace(const VerifyDrafts& p) {
    return stats_bytes(p) + static_cast<size_t>(p.n_seq) * chunks_of(p.vocab) * sizeof(double);
}

hipError_t launch_verify_drafts(const VerifyDrafts& p, void* work, uint32_t* counters, hipStream_t s) {
    return p.dtype == RT_HIP_F32 ? run<float>(p, work, counters, s) : run<uint16_t>(p, work, counters, s);
}

}  // namespace rt_hip
