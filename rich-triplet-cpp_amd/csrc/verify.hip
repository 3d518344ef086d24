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
// Three launches.  k_verify_stats reads every row once, in chunks, and leaves
// each chunk's maximum and sum of exp((x - maximum) / T); k_verify_decide joins
// a request's rows and decides on its drafts; k_verify_pick sums w of the row
// behind a refused draft by chunks and, in the request's last workgroup to
// arrive, finds the chunk that holds the border and the token in it (behind the
// last draft the chunks' sums are there already).  Rows of a request whose T is
// 0 need no sums.
//
// Bound: the bytes of the logits, and as much the exponentials, 18 64-bit
// instructions each at the rate of 32-bit ones.  64 requests of up to 4 drafts,
// 128256 values in f32, 173 MB: 30 to 34 us for the sums (5.1 to 5.8 TB/s), 5 to
// decide, 21 to pick, for which the rows behind refused drafts are read once more.
// One request of 7 drafts: 4.7 + 4.5 + 11, chains of dependent loads.  (Decisions
// in every workgroup of the pick: 66 us and 25; in the sums' last workgroup to
// arrive: 125 and 40, an arrival costs each of 10000 workgroups 2 us.)
#include "rt_common.hpp"
#include "rt_launch.hpp"
#include "wave_scan.hpp"

namespace rt_hip {
namespace {

constexpr int kT = 256;
constexpr int kQuads = 4;                  // groups of 4 values a thread holds
constexpr int kChunk = kT * 4 * kQuads;    // values of a row per workgroup
constexpr int kPickT = 512;                // (k_verify_pick, 64 requests: 22 us; 1024 threads 31, 256 25)
constexpr int kPickQuads = kChunk / 4 / kPickT;
constexpr float kInf = __builtin_inff();

struct Stat {
    double sum;   // of exp((x - top) / T) over the chunk
    float top;    // its maximum, NaN aside (-inf: nothing above)
    int32_t idx;  // where that first stands (T = 0)
};

// 2^x for x <= 0, exactly 1 for 0, and 0 for -inf and NaN.  Adding 1.5 2^52
// leaves the whole part of x in the low bits; 2^r of the rest, |r| <= 1/2, is
// 1 + r P(r), where P takes the values of (2^r - 1) / r at the nine Chebyshev
// nodes (relative error below 4e-14).
__device__ __forceinline__ double exp2_64(double x) {
    constexpr double kMagic = 6755399441055744.0;
    x = __builtin_fmax(x, -2000.0);
    const double t = x + kMagic;
    const double r = x - (t - kMagic);
    double y = 1.0203121063391729e-07;
    y = __builtin_fma(y, r, 1.3255224878668817e-06);
    y = __builtin_fma(y, r, 1.525268684626772e-05);
    y = __builtin_fma(y, r, 0.00015403455852453838);
    y = __builtin_fma(y, r, 0.0013333558179043112);
    y = __builtin_fma(y, r, 0.009618129159402558);
    y = __builtin_fma(y, r, 0.055504108664760424);
    y = __builtin_fma(y, r, 0.2402265069581299);
    y = __builtin_fma(y, r, 0.6931471805599453);
    y = __builtin_fma(y, r, 1.0);
    return __builtin_ldexp(y, static_cast<int>(__builtin_bit_cast(uint64_t, t)));
}

// Weights of a row's values against its maximum, top > -inf: exp((x - top) / T),
// 1 for what equals the maximum (infinities share the weight), 0 for -inf and NaN.
struct Weigh {
    double scale;  // log2(e) / T
    float top;
    __device__ __forceinline__ double finite(float x) const {  // top < inf
        return exp2_64((static_cast<double>(x) - static_cast<double>(top)) * scale);
    }
    __device__ __forceinline__ double operator()(float x) const {
        const double w = finite(x);  // (a select, no branch)
        return x == top ? 1.0 : w;
    }
};

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
__device__ __forceinline__ double scale_of(float t) { return t > 0.0f ? 1.4426950408889634074 / static_cast<double>(t) : 1.0; }
// First row and number of drafts of request s, inside the arrays.
__device__ __forceinline__ int rows_of(const VerifyDrafts& p, int s, int* first) {
    const int a = min(max(p.row_start[s], 0), p.n_rows), b = min(max(p.row_start[s + 1], a), p.n_rows);
    *first = a;
    return min(b - a, p.max_draft + 1);  // rows; drafts are one fewer
}

__device__ __forceinline__ double wave_sum(double v) { return of_lane(running_sum(v), 63); }
__device__ __forceinline__ float wave_max(float v) {
    return of_lane(running(v, -kInf, [](float a, float b) { return fmaxf(a, b); }), 63);
}
__device__ __forceinline__ int wave_min(int v) {
    return of_lane(running(v, 0x7fffffff, [](int a, int b) { return min(a, b); }), 63);
}

// Sum over a workgroup of W waves, the same bits in every thread.
template <int W>
__device__ __forceinline__ double block_sum(double v, double* tmp) {
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) tmp[threadIdx.x >> 6] = v;
    __syncthreads();
    double sum = tmp[0];
#pragma unroll
    for (int w = 1; w < W; ++w) sum += tmp[w];
    return sum;
}
// Sum over the threads before this one; *total: over all of them.
template <int W>
__device__ __forceinline__ double block_before(double v, double* tmp, double* total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const double sum = running_sum(v);
    const double before = from_before<0x138, 0xf>(0.0, sum);  // (one lane on)
    __syncthreads();
    if (lane == 63) tmp[wave] = sum;
    __syncthreads();
    double all = 0.0, base = 0.0;
#pragma unroll
    for (int w = 0; w < W; ++w) {
        base = w == wave ? all : base;
        all += tmp[w];
    }
    *total = all;
    return base + before;
}
// Of the weights in thread order (thread t's first[0 .. N) lie `before` it):
// the place of the first with which the running sum exceeds target, else of
// the last weight above 0, else -1.  place(e): where weight e stands, below 2^31.
template <int W, int N, class F>
__device__ __forceinline__ int find_border(const double (&w)[N], double before, double target, F place, int* tmp2) {
    const int wave = threadIdx.x >> 6;
    int hit = -1, heavy = -1;
#pragma unroll
    for (int e = 0; e < N; ++e) {
        before += w[e];
        if (w[e] > 0.0) {
            heavy = place(e);
            if (before > target && hit < 0) hit = heavy;
        }
    }
    const uint64_t hits = __ballot(hit >= 0), heavies = __ballot(heavy >= 0);
    hit = hits ? of_lane(hit, __builtin_ctzll(hits)) : -1;  // (by all lanes, which hold them)
    heavy = heavies ? of_lane(heavy, 63 - __builtin_clzll(heavies)) : -1;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) {
        tmp2[wave] = hit;
        tmp2[W + wave] = heavy;
    }
    __syncthreads();
    int first = -1, last = -1;
#pragma unroll
    for (int i = 0; i < W; ++i) {
        if (first < 0) first = tmp2[i];
        last = max(last, tmp2[W + i]);
    }
    return first >= 0 ? first : last;
}

__device__ __forceinline__ void st_dev(double* p, double v) {
    __hip_atomic_store((__attribute__((address_space(1))) double*)p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ double ld_dev(const double* p) {
    return __hip_atomic_load((const __attribute__((address_space(1))) double*)p, __ATOMIC_RELAXED,
                             __HIP_MEMORY_SCOPE_AGENT);
}

// A row's maximum (-inf: nothing above), its first place, and the inverse of its
// sum, from its chunks (up to 256, four to a lane); one wave, all lanes end with
// them.
struct RowStat {
    double inv_sum;
    float top;
    int idx;
};
__device__ __forceinline__ RowStat join_row(const Stat* st, int chunks, double scale) {
    const int lane = threadIdx.x & 63;
    Stat x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[i] = st[min(lane + 64 * i, chunks - 1)];
        if (lane + 64 * i >= chunks) x[i] = Stat{0.0, -kInf, 0};
    }
    RowStat r;
    r.top = wave_max(fmaxf(fmaxf(x[0].top, x[1].top), fmaxf(x[2].top, x[3].top)));
    int idx = 0x7fffffff;
    double sum = 0.0;
    const Weigh weigh{scale, r.top};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        idx = x[i].top == r.top ? min(idx, x[i].idx) : idx;
        sum += x[i].sum * weigh(x[i].top);
    }
    idx = wave_min(idx);
    r.idx = r.top > -kInf ? idx : 0;
    r.inv_sum = 1.0 / wave_sum(sum);
    return r;
}

// Probability from a row's joined statistics (nothing above -inf: certain of token 0).
__device__ __forceinline__ double prob(float x, int at, const RowStat& r, double scale) {
    const double w = Weigh{scale, r.top}(x) * r.inv_sum;
    return r.top == -kInf ? (at == 0 ? 1.0 : 0.0) : w;
}

// Statistics [which][row][chunk]; grid (chunks, n_seq * (max_draft + 1), 1 or 2).
template <class X>
__global__ __launch_bounds__(kT) void k_verify_stats(VerifyDrafts p, Stat* __restrict__ stats) {
    __shared__ double tmp[4];
    __shared__ float tmp_top[4];
    __shared__ int tmp_idx[4];
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
    float top = -kInf;  // (the maximum passes NaN over)
#pragma unroll
    for (int i = 0; i < kQuads; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) top = fmaxf(top, v[i][e]);
    top = wave_max(top);
    if ((tid & 63) == 0) tmp_top[tid >> 6] = top;
    __syncthreads();
    top = fmaxf(fmaxf(tmp_top[0], tmp_top[1]), fmaxf(tmp_top[2], tmp_top[3]));
    Stat o{0.0, top, 0};
    if (temp == 0.0f) {
        int idx = 0x7fffffff;
#pragma unroll
        for (int i = 0; i < kQuads; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (v[i][e] == top) idx = min(idx, c0 + (i * kT + tid) * 4 + e);
        idx = wave_min(idx);
        if ((tid & 63) == 0) tmp_idx[tid >> 6] = idx;
        __syncthreads();
        o.idx = min(min(tmp_idx[0], tmp_idx[1]), min(tmp_idx[2], tmp_idx[3]));
    } else if (top > -kInf) {
        const Weigh weigh{scale_of(temp), top};
        double sum[4] = {0.0, 0.0, 0.0, 0.0};
        if (top < kInf) {
#pragma unroll
            for (int i = 0; i < kQuads; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) sum[e] += weigh.finite(v[i][e]);
        } else {
#pragma unroll
            for (int i = 0; i < kQuads; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) sum[e] += v[i][e] == top ? 1.0 : 0.0;
        }
        o.sum = block_sum<kT / 64>((sum[0] + sum[1]) + (sum[2] + sum[3]), tmp);
    }
    if (tid == 0) stats[(static_cast<int64_t>(draft ? p.n_rows : 0) + row) * gridDim.x + blockIdx.x] = o;
}

// What is left to do for a request: w of `row` chooses the token out[at].
struct Choice {
    RowStat p, q;
    int32_t row, at, draft;
    int32_t kind;  // 0: nothing is; 1: w = max(0, p - q), q certain of `draft` where no logits are given; 2: w = p
};

// Accepted drafts, their count, and the choice that is left; grid n_seq.  Wave w
// takes rows w, w + 8, ..: the first that stops the request, a refused draft or
// the row behind the last one.
template <class X>
__global__ __launch_bounds__(kPickT) void k_verify_decide(VerifyDrafts p, const Stat* __restrict__ stats, int chunks,
                                                          Choice* __restrict__ choices) {
    constexpr int kWaves = kPickT / 64;
    __shared__ RowStat best[kWaves][2];
    __shared__ int stop[kWaves];
    const int s = blockIdx.x, tid = threadIdx.x, wave = tid >> 6;
    int first;
    const int rows = rows_of(p, s, &first);
    int32_t* const out = p.out_tokens + static_cast<int64_t>(s) * (p.max_draft + 1);
    if (rows == 0) {  // no rows, no tokens
        for (int i = tid; i <= p.max_draft; i += kPickT) out[i] = -1;
        if (tid == 0) {
            p.out_count[s] = 0;
            choices[s].kind = 0;
        }
        return;
    }
    const float temp = temperature_of(p, s);
    const double scale = scale_of(temp);
    const Stat* const draft_stats = stats + static_cast<int64_t>(p.n_rows) * chunks;
    if ((tid & 63) == 0) stop[wave] = rows;
    for (int j = wave; j < rows; j += kWaves) {
        const int row = first + j;
        const bool behind = j + 1 == rows;
        // (loads that depend on each other first)
        const int d = behind ? -1 : p.tokens[row + 1];
        const float u = behind ? 0.0f : p.accept_u[row];
        const bool real = static_cast<uint32_t>(d) < static_cast<uint32_t>(p.vocab);
        const float xd = real ? load1(static_cast<const X*>(p.logits) + row * p.logit_stride, d) : 0.0f;
        const float yd = real && p.draft_logits
                             ? load1(static_cast<const X*>(p.draft_logits) + row * p.draft_stride, d) : 0.0f;
        const RowStat rp = join_row(stats + static_cast<int64_t>(row) * chunks, chunks, scale);
        RowStat rq = rp;
        bool stops = behind;
        if (!behind && temp == 0.0f) {
            stops = d != rp.idx;
        } else if (!behind) {
            double qd = real ? 1.0 : 0.0;
            if (p.draft_logits) {
                rq = join_row(draft_stats + static_cast<int64_t>(row) * chunks, chunks, scale);
                if (real) qd = prob(yd, d, rq, scale);
            }
            stops = !(static_cast<double>(u) * qd < (real ? prob(xd, d, rp, scale) : 0.0));
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
    const RowStat rp = best[who][0];
    const bool refused = j + 1 < rows, certain = temp == 0.0f || rp.top == -kInf;
    for (int i = tid; i <= p.max_draft; i += kPickT)
        if (i != j || certain) out[i] = i < j ? p.tokens[first + 1 + i] : (i == j ? rp.idx : -1);
    if (tid == 0) {
        p.out_count[s] = j + 1;
        choices[s] = Choice{rp, best[who][1], first + j, j, refused ? p.tokens[first + j + 1] : -1,
                            certain ? 0 : (refused ? 1 : 2)};
    }
}

// grid (chunks, n_seq); sums [n_seq][chunks].
template <class X>
__global__ __launch_bounds__(kPickT) void k_verify_pick(VerifyDrafts p, const Stat* __restrict__ stats,
                                                        const Choice* __restrict__ choices, double* __restrict__ sums,
                                                        uint32_t* __restrict__ arrivals) {
    constexpr int kWaves = kPickT / 64;
    __shared__ double tmp[kWaves], left;
    __shared__ int last, tmp2[2 * kWaves];
    const int s = blockIdx.y, chunks = gridDim.x, tid = threadIdx.x;
    const Choice c = choices[s];
    if (c.kind == 0 || (c.kind == 2 && blockIdx.x != 0)) return;  // (sums of p are there: one workgroup is enough)
    const double scale = scale_of(temperature_of(p, s));
    const X* const x = static_cast<const X*>(p.logits) + c.row * p.logit_stride;
    const X* const y = p.draft_logits ? static_cast<const X*>(p.draft_logits) + c.row * p.draft_stride : nullptr;
    const Weigh weigh_p{scale, c.p.top};

    // Weights of four values from `at` on.
    auto weights4 = [&](int at, bool rest, double* w) {
        float xv[4], yv[4];
        load4(x, at, p.vocab, xv);
        if (rest && y) load4(y, at, p.vocab, yv);
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = at + e < p.vocab ? weigh_p(xv[e]) * c.p.inv_sum : 0.0;
        if (rest) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const double q = y ? (at + e < p.vocab ? prob(yv[e], at + e, c.q, scale) : 0.0)
                                   : (at + e == c.draft ? 1.0 : 0.0);
                w[e] = fmax(w[e] - q, 0.0);
            }
        }
    };
    auto of_p = [&](int chunk) {
        const Stat st = stats[static_cast<int64_t>(c.row) * chunks + chunk];
        return st.top > -kInf ? st.sum * weigh_p(st.top) * c.p.inv_sum : 0.0;
    };

    bool rest = c.kind == 1;
    double* const mine = sums + static_cast<int64_t>(s) * chunks;
    if (rest) {
        double sum = 0.0;
#pragma unroll
        for (int i = 0; i < kPickQuads; ++i) {
            double w[4];
            weights4(blockIdx.x * kChunk + (i * kPickT + tid) * 4, true, w);
            sum += (w[0] + w[1]) + (w[2] + w[3]);
        }
        sum = block_sum<kWaves>(sum, tmp);
        // Relaxed: the sum goes out in an agent-scope store that is waited for.
        if (tid == 0) {
            st_dev(mine + blockIdx.x, sum);
            wait_vmcnt<0>();
            last = __hip_atomic_fetch_add(arrivals + s, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
                   static_cast<uint32_t>(chunks) - 1;
        }
        __syncthreads();
        if (!last) return;
        if (tid == 0) __hip_atomic_store(arrivals + s, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }

    // The chunk with the border: thread i holds chunk i's sum.
    double w1[1] = {0.0}, total;
    if (tid < chunks) w1[0] = rest ? ld_dev(mine + tid) : of_p(tid);
    double before = block_before<kWaves>(w1[0], tmp, &total);
    if (rest && !(total > 0.0)) {  // (p is nowhere above q: from p after all)
        rest = false;
        if (tid < chunks) w1[0] = of_p(tid);
        before = block_before<kWaves>(w1[0], tmp, &total);
    }
    const double target = static_cast<double>(p.sample_u[s]) * total;
    const int border = find_border<kWaves>(w1, before, target, [&](int) { return tid; }, tmp2);
    if (tid == border) left = target - before;
    __syncthreads();
    // The token in it: a thread's values lie next to each other, the vocabulary's order.
    const int c0 = border * kChunk + tid * (4 * kPickQuads);
    double w[4 * kPickQuads], own = 0.0;
#pragma unroll
    for (int i = 0; i < kPickQuads; ++i) {
        weights4(c0 + 4 * i, rest, w + 4 * i);
        own += (w[4 * i] + w[4 * i + 1]) + (w[4 * i + 2] + w[4 * i + 3]);
    }
    before = block_before<kWaves>(own, tmp, &total);
    const int token = find_border<kWaves>(w, before, left, [&](int e) { return c0 + e; }, tmp2);
    if (tid == 0) p.out_tokens[static_cast<int64_t>(s) * (p.max_draft + 1) + c.at] = token;
}

int chunks_of(int vocab) { return (vocab + kChunk - 1) / kChunk; }

size_t stats_bytes(const VerifyDrafts& p) {
    return static_cast<size_t>(p.n_rows) * (p.draft_logits ? 2 : 1) * chunks_of(p.vocab) * sizeof(Stat);
}

template <class X>
hipError_t run(const VerifyDrafts& p, void* work, uint32_t* counters, hipStream_t s) {
    Stat* const stats = static_cast<Stat*>(work);
    Choice* const choices = reinterpret_cast<Choice*>(static_cast<uint8_t*>(work) + stats_bytes(p));
    double* const sums = reinterpret_cast<double*>(choices + p.n_seq);
    const unsigned chunks = static_cast<unsigned>(chunks_of(p.vocab));
    const unsigned rows = static_cast<unsigned>(p.n_seq) * static_cast<unsigned>(p.max_draft + 1);
    hipLaunchKernelGGL(k_verify_stats<X>, dim3(chunks, rows, p.draft_logits ? 2 : 1), dim3(kT), 0, s, p, stats);
    hipLaunchKernelGGL(k_verify_decide<X>, dim3(static_cast<unsigned>(p.n_seq)), dim3(kPickT), 0, s, p, stats,
                       static_cast<int>(chunks), choices);
    hipLaunchKernelGGL(k_verify_pick<X>, dim3(chunks, static_cast<unsigned>(p.n_seq)), dim3(kPickT), 0, s, p, stats, choices,
                       sums, counters);
    return hipGetLastError();
}

}  // namespace

size_t verify_drafts_workspace(const VerifyDrafts& p) {
    return stats_bytes(p) + static_cast<size_t>(p.n_seq) * (sizeof(Choice) + chunks_of(p.vocab) * sizeof(double));
}

hipError_t launch_verify_drafts(const VerifyDrafts& p, void* work, uint32_t* counters, hipStream_t s) {
    return p.dtype == RT_HIP_F32 ? run<float>(p, work, counters, s) : run<uint16_t>(p, work, counters, s);
}

}  // namespace rt_hip
