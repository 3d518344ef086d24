// paged.hip -- the pages of a KV cache shared by many requests: their
// bookkeeping for one step (block table, slots, positions, from the requests'
// lengths) and the append of the step's keys and values.
//
// Plan.  Request s has cached[s] tokens in held[s] pages of P tokens and gets
// fresh[s] new ones (-1: it has ended).  With want_s = max(0, ceil((cached +
// fresh) / P) - held) where that fits the table's row and rows are left, a
// request is served if want_s = 0 or want_0 + .. + want_s <= free pages, and
// takes pages [sum of want before s, + want_s) of the queue's front.  An ended
// request's pages go to the queue's end, in request order.  Token t of request
// s has position cached[s] + t - q_start[s] and slot page * P + position % P.
//
// Bound: latency, 6 us for 64 decoding requests, 12 for a thousand with 47754
// new tokens (0.5 MB).  The sums over requests are scans; every workgroup does
// them for itself (the requests' lengths are a few KB in L2), so nothing
// has to be handed from one launch to the next, then takes its share of the
// pages and tokens.  A token's page is read from the table where the request
// held it before and from the queue otherwise, never from what this launch
// writes.  held and the queue's state may be updated in place: the last
// workgroup to have read them stores them.
//
// Append.  One thread converts and stores 8 values of a row; bound by the
// bytes read and written: 8192 rows of 1024 bf16 keys and values, 67 MB, in 11 us
// (6 TB/s, part of them in the last-level cache), 40 rows of f32 in 2.4.
#include "rt_common.hpp"
#include "rt_launch.hpp"
#include "wave_scan.hpp"

namespace rt_hip {
namespace {

constexpr int kPlanTokens = 4;  // consecutive tokens a thread takes at a time

// Inclusive sum over the workgroup of NT threads in thread order; *total: over all.
template <int NT, class T>
__device__ __forceinline__ T block_scan(T v, T* tmp, T* total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    v = running_sum(v);
    __syncthreads();  // (tmp's readers of the call before)
    if (lane == 63) tmp[wave] = v;
    __syncthreads();
    T before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) {
        if (w == wave) before = all;
        all += tmp[w];
    }
    *total = all;
    return v + before;
}

// Largest i in [0, n) with a[i] <= x; a is non-decreasing and a[0] <= x.
__device__ __forceinline__ int last_not_above(const int* a, int n, int x) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

template <int NT>
__global__ __launch_bounds__(NT) void k_paged_plan(PagedPlan p, uint32_t* __restrict__ arrivals) {
    // per request: first row, first page of the queue's front, pages put back
    // before it; cached (-1: not served), pages held
    extern __shared__ int lds[];
    __shared__ int64_t tmp64[NT / 64];
    __shared__ int tmp32[NT / 64];
    __shared__ int last;
    const int n = p.n_seq, tid = threadIdx.x;
    int* const start = lds;             // [n + 1]
    int* const first = start + n + 1;   // [n + 1]
    int* const behind = first + n + 1;  // [n + 1]
    int* const base = behind + n + 1;   // [n]
    int* const had = base + n;          // [n]
    const int cap = p.n_pages, shift = p.page_shift, page_size = 1 << shift;
    const int cols = static_cast<int>(p.cols);
    int head = p.queue_state[0] % cap;
    if (head < 0) head += cap;
    const int free_pages = min(max(p.queue_state[1], 0), cap);
    const bool lead = blockIdx.x == 0;

    int64_t row0 = 0;      // rows before this chunk of requests
    int want0 = 0, take0 = 0, gone0 = 0;
    for (int s0 = 0; s0 < n; s0 += NT) {
        const int s = s0 + tid;
        const bool in = s < n;
        const int cached = in ? p.cached[s] : 0, fresh = in ? p.fresh[s] : 0;
        const int raw_held = in ? p.held[s] : 0, held = min(max(raw_held, 0), cols);
        const int rows = max(fresh, 0);
        int64_t all_rows;
        const int64_t end = row0 + block_scan<NT, int64_t>(rows, tmp64, &all_rows);
        row0 += all_rows;
        // pages of the request after this step; not served: past the rows or the table
        const int64_t pages = (static_cast<int64_t>(cached) + rows + page_size - 1) >> shift;
        const bool fits = fresh >= 0 && cached >= 0 && raw_held == held && end <= p.n_tokens &&
                          pages <= cols;
        const int want = fits && pages > held ? static_cast<int>(pages) - held : 0;
        int all_want;
        const int upto = want0 + block_scan<NT, int>(want, tmp32, &all_want);
        want0 += all_want;
        const bool served = fits && (want == 0 || upto <= free_pages);
        const int take = served ? want : 0, gone = fresh < 0 ? held : 0;
        // (requests are served up to the first whose pages run out, so what is
        // taken before a served request is what is wanted before it)
        int all_take, all_gone;
        const int taken = take0 + block_scan<NT, int>(take, tmp32, &all_take);
        const int back = gone0 + block_scan<NT, int>(gone, tmp32, &all_gone);
        take0 += all_take;
        gone0 += all_gone;
        if (in) {
            const int from = static_cast<int>(min(end - rows, static_cast<int64_t>(p.n_tokens)));
            start[s] = from;
            first[s] = taken - take;
            behind[s] = back - gone;
            base[s] = served ? cached : -1;
            had[s] = held;
            if (lead) {
                p.q_start[s] = from;
                p.kv_len[s] = served ? cached + rows : 0;
            }
        }
    }
    if (tid == 0) {
        const int end = static_cast<int>(min(row0, static_cast<int64_t>(p.n_tokens)));
        start[n] = end;
        first[n] = take0;
        behind[n] = gone0;
        if (lead) p.q_start[n] = end;
    }
    __syncthreads();

    const int gid = blockIdx.x * NT + tid, gsize = gridDim.x * NT;
    for (int t = gid; t < take0; t += gsize) {
        const int s = last_not_above(first, n, t);
        p.table[s * p.cols + had[s] + t - first[s]] = p.queue[(static_cast<int64_t>(head) + t) % cap];
    }
    for (int t = gid; t < gone0; t += gsize) {
        const int s = last_not_above(behind, n, t);
        p.queue[(static_cast<int64_t>(head) + free_pages + t) % cap] = p.table[s * p.cols + t - behind[s]];
    }
    for (int64_t t0 = static_cast<int64_t>(gid) * kPlanTokens; t0 < p.n_tokens;
         t0 += static_cast<int64_t>(gsize) * kPlanTokens) {
        int slot[kPlanTokens], pos[kPlanTokens];
        int s = last_not_above(start, n, static_cast<int>(min(t0, static_cast<int64_t>(start[n]))));
#pragma unroll
        for (int e = 0; e < kPlanTokens; ++e) {
            const int t = static_cast<int>(min(t0 + e, static_cast<int64_t>(p.n_tokens) - 1));
            while (s + 1 < n && start[s + 1] <= t) ++s;
            slot[e] = pos[e] = -1;
            if (t < start[n] && base[s] >= 0) {
                pos[e] = base[s] + t - start[s];
                const int col = pos[e] >> shift;
                // (col < cols: the request fits its row)
                const int id = col < had[s] ? p.table[s * p.cols + col]
                                            : p.queue[(static_cast<int64_t>(head) + first[s] + col - had[s]) % cap];
                if (static_cast<uint32_t>(id) < static_cast<uint32_t>(cap)) slot[e] = (id << shift) + (pos[e] & (page_size - 1));
            }
        }
#pragma unroll
        for (int e = 0; e < kPlanTokens; ++e)
            if (t0 + e < p.n_tokens) {
                p.slots[t0 + e] = slot[e];
                p.positions[t0 + e] = pos[e];
            }
    }

    // held and the queue's state, once every workgroup has read them
    if (gridDim.x > 1) {
        __syncthreads();  // (waits for this workgroup's loads: their values are in LDS or registers)
        if (tid == 0)
            last = __hip_atomic_fetch_add(arrivals, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == gridDim.x - 1;
        __syncthreads();
        if (!last) return;
        if (tid == 0) __hip_atomic_store(arrivals, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    for (int s = tid; s < n; s += NT) {
        const int took = first[s + 1] - first[s], gone = behind[s + 1] - behind[s];
        // (a request that is neither served nor ended keeps what it said it holds)
        p.held_out[s] = gone ? 0 : (took ? had[s] + took : (p.fresh[s] < 0 ? 0 : p.held[s]));
    }
    if (tid == 0) {
        p.queue_state_out[0] = static_cast<int>((static_cast<int64_t>(head) + take0) % cap);
        p.queue_state_out[1] = min(free_pages - take0 + gone0, cap);
    }
}

__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
    const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        v[e] = a[e];
        v[4 + e] = b[e];
    }
}
__device__ __forceinline__ void load8(const __bf16* p, float (&v)[8]) {
    const u32x4 a = ld16(p);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        v[2 * e] = bf16_lo_to_f32(a[e]);
        v[2 * e + 1] = bf16_hi_to_f32(a[e]);
    }
}
__device__ __forceinline__ void load8(const _Float16* p, float (&v)[8]) {
    const u32x4 a = ld16(p);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        v[2 * e] = f16_bits_to_f32(a[e] & 0xffffu);
        v[2 * e + 1] = f16_bits_to_f32(a[e] >> 16);
    }
}
__device__ __forceinline__ void store8(float* p, const float (&v)[8]) {
    *reinterpret_cast<f32x4*>(p) = f32x4{v[0], v[1], v[2], v[3]};
    *reinterpret_cast<f32x4*>(p + 4) = f32x4{v[4], v[5], v[6], v[7]};
}
__device__ __forceinline__ void store8(__bf16* p, const float (&v)[8]) {
    *reinterpret_cast<u32x4*>(p) = u32x4{bf16_pair(v[0], v[1]), bf16_pair(v[2], v[3]), bf16_pair(v[4], v[5]),
                                         bf16_pair(v[6], v[7])};
}
__device__ __forceinline__ void store8(_Float16* p, const float (&v)[8]) {
    typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
    f16x8 o;
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = static_cast<_Float16>(v[e]);  // round to nearest even; past the range: infinity
    *reinterpret_cast<f16x8*>(p) = o;
}

// Units of 8 values: (token, unit of the row), keys in blockIdx.y 0, values in 1.
template <class S, class D>
__global__ __launch_bounds__(256) void k_paged_append(const S* __restrict__ k, const S* __restrict__ v, D* __restrict__ kp,
                                                      D* __restrict__ vp, const int32_t* __restrict__ slots, uint32_t n_tokens,
                                                      uint32_t row_units, int64_t src_stride, int64_t page_stride,
                                                      uint32_t n_slots, int page_shift) {
    const uint32_t u = blockIdx.x * 256 + threadIdx.x;  // (the host keeps units below 2^31)
    const uint32_t t = u / row_units;
    if (t >= n_tokens) return;
    const uint32_t c = (u - t * row_units) * 8;
    const uint32_t slot = static_cast<uint32_t>(slots[t]);
    if (slot >= n_slots) return;  // no slot (-1), or none of this cache
    const S* const src = (blockIdx.y ? v : k) + static_cast<int64_t>(t) * src_stride + c;
    D* const dst = (blockIdx.y ? vp : kp) + (slot >> page_shift) * page_stride +
                   static_cast<int64_t>((slot & ((1u << page_shift) - 1)) * row_units) * 8 + c;
    float x[8];
    load8(src, x);
    store8(dst, x);
}

template <class S, class D>
hipError_t run_append(const void* k, const void* v, int64_t src_stride, const PagedKv& kv, const int32_t* slots,
                      int n_tokens, hipStream_t s) {
    const int units = kv.n_kv * kv.head_dim / 8;
    const int64_t blocks = (static_cast<int64_t>(n_tokens) * units + 255) / 256;
    hipLaunchKernelGGL((k_paged_append<S, D>), dim3(static_cast<unsigned>(blocks), 2), dim3(256), 0, s,
                       static_cast<const S*>(k), static_cast<const S*>(v), static_cast<D*>(kv.k), static_cast<D*>(kv.v),
                       slots, static_cast<uint32_t>(n_tokens), static_cast<uint32_t>(units), src_stride, kv.page_stride,
                       static_cast<uint32_t>(kv.n_pages) << kv.page_shift, kv.page_shift);
    return hipGetLastError();
}

template <class S>
hipError_t run_append_from(const void* k, const void* v, int64_t src_stride, const PagedKv& kv, const int32_t* slots,
                           int n_tokens, hipStream_t s) {
    switch (kv.dtype) {
        case RT_HIP_F32: return run_append<S, float>(k, v, src_stride, kv, slots, n_tokens, s);
        case RT_HIP_F16: return run_append<S, _Float16>(k, v, src_stride, kv, slots, n_tokens, s);
        default: return run_append<S, __bf16>(k, v, src_stride, kv, slots, n_tokens, s);
    }
}

}  // namespace

hipError_t launch_paged_plan(const PagedPlan& p, uint32_t* arrivals, hipStream_t s) {
    const size_t lds = (3 * (static_cast<size_t>(p.n_seq) + 1) + 2 * static_cast<size_t>(p.n_seq)) * sizeof(int);
    // One workgroup up to 4096 tokens; beyond, one per 4096, at most one per CU
    // (1000 requests, 47754 tokens: 12.0 us, with one per 16384 25.0, with one per
    // 1024 11.8).  Up to 256 requests in one workgroup 256 threads: 6.0 us, with
    // 1024 7.6.
    const int64_t blocks = (static_cast<int64_t>(p.n_tokens) + 4095) / 4096;
    const unsigned grid = static_cast<unsigned>(blocks < 1 ? 1 : (blocks > device_info().cus ? device_info().cus : blocks));
    if (p.n_seq <= 256 && grid == 1)
        hipLaunchKernelGGL(k_paged_plan<256>, dim3(1), dim3(256), lds, s, p, arrivals);
    else
        hipLaunchKernelGGL(k_paged_plan<1024>, dim3(grid), dim3(1024), lds, s, p, arrivals);
    return hipGetLastError();
}

hipError_t launch_paged_append(int src_dtype, const void* k, const void* v, int64_t src_stride, const PagedKv& kv,
                               const int32_t* slots, int n_tokens, hipStream_t s) {
    switch (src_dtype) {
        case RT_HIP_F32: return run_append_from<float>(k, v, src_stride, kv, slots, n_tokens, s);
        case RT_HIP_F16: return run_append_from<_Float16>(k, v, src_stride, kv, slots, n_tokens, s);
        default: return run_append_from<__bf16>(k, v, src_stride, kv, slots, n_tokens, s);
    }
}

}  // namespace rt_hip
