// logits.hip -- logits under penalties for repeated tokens, biases and masks.
//
// Row i of request s (rows row_start[s] .. row_start[s + 1]), token v with
// logit x; T is the request's history and behind it its drafts of rows 1 .. i:
//   v in T:                       x = x > 0 ? x / repetition : x * repetition
//   c times behind the prompt:    x = (x - frequency c) - presence      (c > 0)
//   in the request's biases:      x = x + its last entry
//   mask bit 0:                   x = -inf
// In place: only what changes is read and written, so a step without masks costs
// its histories, and a masked row the store of its -inf.
//
// A workgroup has a request and up to kChunk tokens of the vocabulary.  It counts
// the whole history's tokens that fall there in LDS (integers: the order of the
// additions does not matter), puts the biases into a small table, and lists the
// tokens it met; then it goes through the request's rows with that list alone.  A
// mask closes whole quads of tokens by one store and the rest one by one, so it
// reads no logits, and list and mask never meet at a token.
// 64 requests under penalties and biases take 13 us, of which 3 are the start and
// the rest one after another a request's numbers, its history, LDS and the logits
// met; 40 requests' drafts, 159 bf16 rows of 262144 tokens, all under masks 29 us, with
// masks alone 22.  There 84 MB go to memory for 71 that masks close, 99% of it in whole
// lines, and waves wait 57% of their time: what is left is the workgroups' own chains,
// 2640 of them over places for 1792.
#include "rt_common.hpp"
#include "rt_launch.hpp"

namespace rt_hip {
namespace {

// (A CU holds seven workgroups: LDS and vector registers have room for eight, the
// scalar registers, which the rules' pointers fill, for seven waves a SIMD.  64 requests,
// half of them masked, 15.5 us; in an earlier form with a list as long as the chunk and
// an array for the biases, four to a CU, 17.2, and with three 20.3.)
constexpr int kChunk = 4032;
// Of a token of the chunk: that it is listed, that the request's biases or the rows'
// drafts have it; below, twice the count behind the prompt and 1 if in the prompt.
constexpr uint32_t kListed = 1u << 31, kBiased = 1u << 30, kDrafted = 1u << 29, kCount = kDrafted - 1;
constexpr int kListedMost = 1504, kFew = 32;  // tokens of a list; drafts of one
constexpr int kPlaces = 128, kBiases = 96;    // places of biases' tokens, and the biases they take
constexpr uint32_t kNone = ~0u;

__device__ __forceinline__ float load(const float* p) { return *p; }
__device__ __forceinline__ float load(const __bf16* p) { return __uint_as_float(static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(p)) << 16); }
__device__ __forceinline__ void store(float* p, float x) { *p = x; }
__device__ __forceinline__ void store(__bf16* p, float x) { *reinterpret_cast<uint16_t*>(p) = f32_to_bf16_rne(x); }
// -inf; four of them, at an address aligned to them.
__device__ __forceinline__ void close(float* p) { *p = -__builtin_inff(); }
__device__ __forceinline__ void close(__bf16* p) { *reinterpret_cast<uint16_t*>(p) = 0xff80u; }
__device__ __forceinline__ void close4(float* p) {
    *reinterpret_cast<u32x4*>(p) = u32x4{0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u};
}
__device__ __forceinline__ void close4(__bf16* p) { *reinterpret_cast<u32x2*>(p) = u32x2{0xff80ff80u, 0xff80ff80u}; }

template <class T, int kThreads>
__global__ __launch_bounds__(kThreads) void k_adjust_logits(AdjustLogits p) {
    constexpr int kQuads = (kChunk / 4 + kThreads - 1) / kThreads;  // of a thread: four tokens each, kThreads * 4 apart
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    uint32_t* const seen = reinterpret_cast<uint32_t*>(lds);
    uint16_t* const list = reinterpret_cast<uint16_t*>(seen + kChunk);   // the tokens met
    __shared__ int listed, n_drafts, n_entries;
    __shared__ int draft_row[kFew], draft_at[kFew];  // the rows' drafts that fall into the chunk
    __shared__ uint32_t entry_at[kPlaces], entry_of[kPlaces];  // the request's biases that do: a token, 1 + its last entry
    const int s = blockIdx.y, tid = threadIdx.x;
    // (everything of the request at once: what is not there is read from row_start and not used)
    const float* const some = reinterpret_cast<const float*>(p.row_start);
    const int start = p.row_start[s], stop = p.row_start[s + 1];
    const float rep0 = (p.repetition ? p.repetition : some)[s], pres0 = (p.presence ? p.presence : some)[s],
                freq0 = (p.frequency ? p.frequency : some)[s];
    const int32_t* const starts = p.bias ? p.bias_start : p.row_start;
    const int bias0 = starts[s], bias1 = starts[s + 1];
    const int len0 = (p.history ? p.history_len : p.row_start)[s], prompt0 = (p.prompt_len ? p.prompt_len : p.row_start)[s];
    const int row0 = min(max(start, 0), p.n_rows);
    const int rows = min(max(stop, row0), p.n_rows) - row0;
    if (rows == 0) return;
    const int base = static_cast<int>(blockIdx.x) * p.chunk, here = min(p.chunk, p.vocab - base);
    const float rep = p.repetition && rep0 > 0.0f ? rep0 : 1.0f;
    const float pres = p.presence ? pres0 : 0.0f, freq = p.frequency ? freq0 : 0.0f;
    const int len = p.history ? static_cast<int>(min(static_cast<int64_t>(max(len0, 0)), p.history_cols)) : 0;
    const int prompt = p.prompt_len ? prompt0 : 0;
    const bool counts = rep != 1.0f || pres != 0.0f || freq != 0.0f;
    const int b0 = p.bias ? min(max(bias0, 0), p.n_bias) : 0, b1 = p.bias ? min(max(bias1, b0), p.n_bias) : 0;
    const bool biased = b1 > b0;
    T* const logits = static_cast<T*>(p.logits) + static_cast<int64_t>(row0) * p.stride + base;
    auto mask_of = [&](int i) -> const uint32_t* {
        const int m = !p.mask ? -1 : p.mask_row ? p.mask_row[row0 + i] : row0 + i;
        return static_cast<uint32_t>(m) < static_cast<uint32_t>(p.n_masks) ? p.mask + m * p.mask_stride + base / 32 : nullptr;
    };
    const int32_t* const text = p.history + s * p.history_cols;
    constexpr int kAhead = 4;  // loads in flight together
    int x[kAhead];
    auto ask = [&](int i) {
#pragma unroll
        for (int k = 0; k < kAhead; ++k) x[k] = i + k * kThreads < len ? text[i + k * kThreads] : -1;
    };
    auto clear = [&] {
        for (int i = tid * 4; i < p.chunk; i += kThreads * 4) *reinterpret_cast<u32x4*>(seen + i) = u32x4{0, 0, 0, 0};
        if (tid < kPlaces) entry_at[tid] = kNone, entry_of[tid] = 0;
        if (tid == 0) listed = n_drafts = n_entries = 0;
    };
    int first_bias = -1, first_draft = -1;
    if (counts || biased) {
        if (counts) ask(tid);
        if (b0 + tid < b1) first_bias = p.bias_token[b0 + tid];
        if (counts && p.tokens && 1 + tid < rows) first_draft = p.tokens[row0 + 1 + tid];
        clear();
    }
    // The masks, while the history is on its way.  (Four rows' words asked for
    // together: one row 3.2 us instead of 2.4, drafts' rows no faster.)
    if (p.mask) {
        for (int i = 0; i < rows; ++i) {
            const uint32_t* const mask = mask_of(i);
            if (!mask) continue;
            T* const row = logits + i * p.stride;
            const bool aligned = (reinterpret_cast<uintptr_t>(row) & (4 * sizeof(T) - 1)) == 0;
            uint32_t word[kQuads];
#pragma unroll
            for (int q = 0; q < kQuads; ++q) {
                const int v = (q * kThreads + tid) * 4;
                word[q] = v < here ? mask[v / 32] : ~0u;
            }
#pragma unroll
            for (int q = 0; q < kQuads; ++q) {
                const int v = (q * kThreads + tid) * 4;
                const uint32_t open = word[q] >> (v % 32) & 15u;
                if (open == 15u) continue;
                if (open == 0 && aligned && v + 4 <= here) {
                    close4(row + v);
                } else {
                    // (Masks of 160 bf16 rows: 22.2 us.  Where many of a wave's quads have holes,
                    // quads read and written back whole 23.9, tokens stored 64 after 64 23.7.)
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        if (!(open >> k & 1) && v + k < here) close(row + v + k);
                }
            }
        }
    }
    if (!counts && !biased) return;
    __syncthreads();
    // The chunk's tokens from `from` on, `size` of them: all, or where more biases meet
    // them than are collected one half and then the other, whose last entries take the
    // place of the other's counts.
    uint32_t* const last = seen + p.chunk / 2;  // 1 + a token's last entry
    bool halves = false;
    int from = 0, size = here;
    auto in_part = [&](int token, uint32_t* at) {
        *at = static_cast<uint32_t>(token) - static_cast<uint32_t>(base + from);  // (tokens below 0 too)
        return *at < static_cast<uint32_t>(size);
    };
    // A token is met: `as` is what it counts.
    auto meet = [&](uint32_t at, uint32_t as, uint32_t flags) {
        if (!(atomicOr(seen + at, flags | (as & 1u)) & kListed)) {
            const int i = atomicAdd(&listed, 1);
            if (i < kListedMost) list[i] = static_cast<uint16_t>(at);
        }
        if (as > 1) atomicAdd(seen + at, as);
    };
    auto place_of = [](uint32_t at) { return at * 2654435761u >> 25; };
    for (bool again = false;;) {
        uint32_t at;
        if (counts) {
            for (int i = tid; i < len; i += kAhead * kThreads) {
                if (i != tid || again) ask(i);
#pragma unroll
                for (int k = 0; k < kAhead; ++k)
                    if (in_part(x[k], &at)) meet(at, i + k * kThreads < prompt ? 1u : 2u, kListed);
            }
            if (p.tokens)
                for (int i = 1 + tid; i < rows; i += kThreads)
                    if (in_part(i == 1 + tid ? first_draft : p.tokens[row0 + i], &at)) {
                        meet(at, 0, kListed | kDrafted);
                        const int d = atomicAdd(&n_drafts, 1);
                        if (d < kFew) draft_row[d] = i, draft_at[d] = static_cast<int>(at);
                    }
        }
        for (int i = b0 + tid; i < b1; i += kThreads)
            if (in_part(i == b0 + tid ? first_bias : p.bias_token[i], &at)) {
                meet(at, 0, kListed | kBiased);
                const uint32_t entry = static_cast<uint32_t>(i - b0 + 1);
                if (halves) {
                    atomicMax(last + at, entry);
                } else if (atomicAdd(&n_entries, 1) < kBiases) {
                    uint32_t place = place_of(at);
                    for (uint32_t was; (was = atomicCAS(entry_at + place, kNone, at)) != kNone && was != at;) place = (place + 1) % kPlaces;
                    atomicMax(entry_of + place, entry);
                }
            }
        __syncthreads();
        // (more tokens than the list holds: every token of the part)
        const bool all = listed > kListedMost;
        const uint32_t n = static_cast<uint32_t>(all ? size : listed);
        const int drafts = n_drafts, entries = n_entries;
        if (entries <= kBiases) {
            // A thread has a token of the list in a row; its mask and its logit are asked for together.
            const uint32_t each = (n + 63) / 64 * 64;  // (a wave has one row)
            for (uint64_t job = tid; job < static_cast<uint64_t>(each) * static_cast<uint32_t>(rows); job += kThreads) {
                const int i = __builtin_amdgcn_readfirstlane(static_cast<int>(job / each));
                const uint32_t at_list = static_cast<uint32_t>(job - static_cast<uint64_t>(i) * each);
                if (at_list >= n) continue;
                const uint32_t mine = all ? at_list : list[at_list], v = static_cast<uint32_t>(from) + mine;
                T* const where = logits + i * p.stride + v;
                const uint32_t* const mask = mask_of(i);
                const uint32_t bits = mask ? mask[v / 32] : ~0u;
                const float old = load(where);
                const uint32_t what = seen[mine];
                int e = -1;  // the token's last entry
                if (what & kBiased) {
                    uint32_t entry;
                    if (halves) {
                        entry = last[mine];
                    } else {
                        uint32_t place = place_of(mine);
                        while (entry_at[place] != mine) place = (place + 1) % kPlaces;
                        entry = entry_of[place];
                    }
                    e = b0 - 1 + static_cast<int>(entry);
                }
                const float bias = e >= 0 ? p.bias[e] : 0.0f;
                uint32_t t = what & kCount;
                if (what & kDrafted) {
                    if (drafts <= kFew) {
                        for (int d = 0; d < drafts; ++d) t += draft_row[d] <= i && draft_at[d] == static_cast<int>(mine) ? 2u : 0u;
                    } else {
                        for (int k = 1; k <= i; ++k) t += in_part(p.tokens[row0 + k], &at) && at == mine ? 2u : 0u;
                    }
                }
                if (!(bits >> (v % 32) & 1) || (t == 0 && e < 0)) continue;
                float y = old;
                if (t) y = y > 0.0f ? y / rep : y * rep;
                if (t > 1) y = (y - freq * static_cast<float>(t >> 1)) - pres;
                if (e >= 0) y += bias;
                store(where, y);
            }
            from += size;
            if (from >= here) break;
        }
        halves = true;
        size = min(p.chunk / 2, here - from);
        again = true;
        __syncthreads();  // (the part's numbers are read)
        clear();
        __syncthreads();
    }
}

}  // namespace

hipError_t launch_adjust_logits(AdjustLogits p, hipStream_t s) {
    // As many tokens to a workgroup as leave each CU one, up to kChunk, and twice the
    // waves where a CU has two at most (3 requests' 2 rows of 4042 tokens, histories of
    // 3000: 7 us, with kChunk tokens and 256 threads 27; one row of 128256 after 400 tokens
    // 4.5 and 5.1; 52 requests' 5 rows of 9309 tokens 20 and 40, with 1024 threads 16, but
    // there 44 requests' rows of 3026 after 94 tokens 6.5 instead of 5.7).
    const int64_t cus = device_info().cus, parts = cus > p.n_seq ? cus / p.n_seq : 1, even = (p.vocab + parts - 1) / parts;
    p.chunk = static_cast<int>(even < 128 ? 128 : even < kChunk ? (even + 31) / 32 * 32 : kChunk);
    const dim3 grid((static_cast<unsigned>(p.vocab) + p.chunk - 1) / p.chunk, static_cast<unsigned>(p.n_seq));
    const int64_t groups = static_cast<int64_t>(grid.x) * grid.y;
    const bool few = groups <= 2 * cus;
    const auto kernel = p.dtype == RT_HIP_F32 ? (few ? k_adjust_logits<float, 512> : k_adjust_logits<float, 256>)
                                              : (few ? k_adjust_logits<__bf16, 512> : k_adjust_logits<__bf16, 256>);
    hipLaunchKernelGGL(kernel, grid, dim3(few ? 512 : 256), kChunk * sizeof(uint32_t) + kListedMost * sizeof(uint16_t), s, p);
    return hipGetLastError();
}

}  // namespace rt_hip
