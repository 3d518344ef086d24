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
// A workgroup has a request and kChunk tokens of the vocabulary: it counts the
// whole history's tokens that fall into the chunk in LDS (integers: the order of
// the additions does not matter), takes the last bias of each, and walks the
// request's rows, a draft more counted for each.
#include "rt_common.hpp"
#include "rt_launch.hpp"

namespace rt_hip {
namespace {

constexpr int kChunk = 4096, kThreads = 256;
constexpr float kNone = -__builtin_inff();

__device__ __forceinline__ float load(const float* p) { return *p; }
__device__ __forceinline__ float load(const __bf16* p) { return static_cast<float>(*p); }
__device__ __forceinline__ void store(float* p, float x) { *p = x; }
__device__ __forceinline__ void store(__bf16* p, float x) {
    *reinterpret_cast<uint16_t*>(p) = f32_to_bf16_rne(x);
}
// Four -inf, `p` aligned to them.
__device__ __forceinline__ void close4(float* p) { *reinterpret_cast<f32x4*>(p) = f32x4{kNone, kNone, kNone, kNone}; }
__device__ __forceinline__ void close4(__bf16* p) { *reinterpret_cast<u32x2*>(p) = u32x2{0xff80ff80u, 0xff80ff80u}; }

template <class T>
__global__ __launch_bounds__(kThreads) void k_adjust_logits(AdjustLogits p) {
    __shared__ __attribute__((aligned(16))) uint32_t seen[kChunk];  // twice the count behind the prompt, 1: in the prompt
    __shared__ __attribute__((aligned(16))) int entry[kChunk];      // 1 + the last bias entry, 0: none
    const int s = blockIdx.y, tid = threadIdx.x;
    const int row0 = min(max(p.row_start[s], 0), p.n_rows);
    const int rows = min(max(p.row_start[s + 1], row0), p.n_rows) - row0;
    if (rows == 0) return;
    const int base = static_cast<int>(blockIdx.x) * kChunk, here = min(kChunk, p.vocab - base);
    float rep = p.repetition ? p.repetition[s] : 1.0f;
    rep = rep > 0.0f ? rep : 1.0f;
    const float pres = p.presence ? p.presence[s] : 0.0f, freq = p.frequency ? p.frequency[s] : 0.0f;
    const bool counts = rep != 1.0f || pres != 0.0f || freq != 0.0f;
    int b0 = 0, b1 = 0;
    if (p.bias) {
        b0 = min(max(p.bias_start[s], 0), p.n_bias);
        b1 = min(max(p.bias_start[s + 1], b0), p.n_bias);
    }
    const bool biased = b1 > b0;
    if (counts || biased) {
        for (int i = tid * 4; i < kChunk; i += kThreads * 4) {
            *reinterpret_cast<u32x4*>(seen + i) = u32x4{0, 0, 0, 0};
            if (biased) *reinterpret_cast<u32x4*>(entry + i) = u32x4{0, 0, 0, 0};
        }
        __syncthreads();
        if (counts && p.history) {
            const int len = static_cast<int>(min(static_cast<int64_t>(max(p.history_len[s], 0)), p.history_cols));
            const int prompt = p.prompt_len ? p.prompt_len[s] : 0;
            const int32_t* const text = p.history + s * p.history_cols;
            auto count = [&](int i, int token) {
                const uint32_t at = static_cast<uint32_t>(token) - static_cast<uint32_t>(base);
                if (at >= static_cast<uint32_t>(here)) return;  // (tokens below 0 too)
                if (i < prompt) atomicOr(seen + at, 1u);
                else atomicAdd(seen + at, 2u);
            };
            constexpr int kAhead = 8;  // loads in flight together
            int i = tid;
            for (; i + (kAhead - 1) * kThreads < len; i += kAhead * kThreads) {
                int x[kAhead];
#pragma unroll
                for (int k = 0; k < kAhead; ++k) x[k] = text[i + k * kThreads];
#pragma unroll
                for (int k = 0; k < kAhead; ++k) count(i + k * kThreads, x[k]);
            }
            for (; i < len; i += kThreads) count(i, text[i]);
        }
        for (int i = b0 + tid; i < b1; i += kThreads) {
            const uint32_t at = static_cast<uint32_t>(p.bias_token[i]) - static_cast<uint32_t>(base);
            if (at < static_cast<uint32_t>(here)) atomicMax(entry + at, i - b0 + 1);
        }
        __syncthreads();
    }
    T* const logits = static_cast<T*>(p.logits) + base;
    for (int r = row0; r < row0 + rows; ++r) {
        if (r > row0 && counts && p.tokens) {
            __syncthreads();  // (every thread is done with the row before)
            const uint32_t at = static_cast<uint32_t>(p.tokens[r]) - static_cast<uint32_t>(base);
            if (tid == 0 && at < static_cast<uint32_t>(here)) seen[at] += 2;
            __syncthreads();
        }
        T* const row = logits + static_cast<int64_t>(r) * p.stride;
        const uint32_t* mask = nullptr;
        if (p.mask) {
            const int m = p.mask_row ? p.mask_row[r] : r;
            if (static_cast<uint32_t>(m) < static_cast<uint32_t>(p.n_masks)) mask = p.mask + m * p.mask_stride + base / 32;
        }
        if (!mask && !counts && !biased) continue;
        const bool whole = (reinterpret_cast<uintptr_t>(row) & (4 * sizeof(T) - 1)) == 0;
        for (int i = tid * 4; i < here; i += kThreads * 4) {
            uint32_t open = mask ? mask[i / 32] >> (i % 32) & 15u : 15u;
            const int n = min(4, here - i);
            if (open == 0 && whole && n == 4) {
                close4(row + i);
                continue;
            }
            u32x4 t = {0, 0, 0, 0}, e = {0, 0, 0, 0};
            if (counts) t = *reinterpret_cast<const u32x4*>(seen + i);
            if (biased) e = *reinterpret_cast<const u32x4*>(entry + i);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if (k >= n) break;
                if (!(open >> k & 1)) {
                    store(row + i + k, kNone);
                } else if (t[k] | e[k]) {
                    float x = load(row + i + k);
                    if (t[k]) x = x > 0.0f ? x / rep : x * rep;
                    if (t[k] > 1) x = (x - freq * static_cast<float>(t[k] >> 1)) - pres;
                    if (e[k]) x += p.bias[b0 + static_cast<int>(e[k]) - 1];
                    store(row + i + k, x);
                }
            }
        }
    }
}

}  // namespace

hipError_t launch_adjust_logits(const AdjustLogits& p, hipStream_t s) {
    const dim3 grid((static_cast<unsigned>(p.vocab) + kChunk - 1) / kChunk, static_cast<unsigned>(p.n_seq));
    if (p.dtype == RT_HIP_F32) hipLaunchKernelGGL(k_adjust_logits<float>, grid, dim3(kThreads), 0, s, p);
    else hipLaunchKernelGGL(k_adjust_logits<__bf16>, grid, dim3(kThreads), 0, s, p);
    return hipGetLastError();
}

}  // namespace rt_hip
