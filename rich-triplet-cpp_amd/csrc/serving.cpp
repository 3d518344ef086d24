// serving.cpp -- the C ABI of batched serving over a paged KV cache
// (include/rt_hip.h): argument checks, workspace and dispatch.
#include <hip/hip_runtime.h>

#include <string>

#include "rt_hip.h"
#include "rt_launch.hpp"

using namespace rt_hip;

namespace {

int fail(const char* fn, int code, const std::string& what) { return set_error(code, std::string(fn) + ": " + what); }

int launched(const char* fn, hipError_t e) {
    if (e == hipErrorStreamCaptureUnsupported)
        return fail(fn, RT_HIP_E_HIP,
                    "the workspace must grow, which cannot happen while the stream is captured (call "
                    "rt_hip_reserve_workspace / rt_hip_init before capture)");
    return e == hipSuccess ? RT_HIP_OK : fail(fn, RT_HIP_E_HIP, hipGetErrorString(e));
}

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

struct Range {
    const void* p;
    int64_t bytes;
};
bool overlap(const Range& a, const Range& b) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a.p), y = reinterpret_cast<uintptr_t>(b.p);
    return a.bytes > 0 && b.bytes > 0 && x < y + static_cast<uintptr_t>(b.bytes) && y < x + static_cast<uintptr_t>(a.bytes);
}

int value_bytes(int32_t dtype) { return dtype == RT_HIP_F32 ? 4 : (dtype == RT_HIP_F16 || dtype == RT_HIP_BF16 ? 2 : 0); }

// log2 of a page size the kernels take, -1 otherwise.
int page_shift(int32_t page_size) {
    for (int s = 3; s <= 10; ++s)
        if (page_size == 1 << s) return s;
    return -1;
}

// The caller's description of a cache, checked, as the kernels take it.
int cache_args(const char* fn, const rt_hip_paged_kv* kv, PagedKv* out) {
    if (!kv || !kv->k || !kv->v) return fail(fn, RT_HIP_E_ARG, "null cache");
    if (!value_bytes(kv->dtype)) return fail(fn, RT_HIP_E_UNSUPPORTED, "the cache must be F32, F16 or BF16");
    const int shift = page_shift(kv->page_size);
    if (shift < 0) return fail(fn, RT_HIP_E_SHAPE, "page_size must be a power of two from 8 to 1024");
    if (kv->head_dim != 64 && kv->head_dim != 128 && kv->head_dim != 256)
        return fail(fn, RT_HIP_E_SHAPE, "head_dim must be 64, 128 or 256");
    if (kv->n_kv_heads < 1 || kv->n_kv_heads > 256) return fail(fn, RT_HIP_E_SHAPE, "n_kv_heads must be in [1, 256]");
    if (kv->n_pages < 1 || (static_cast<int64_t>(kv->n_pages) << shift) > 0x7fffffffLL)
        return fail(fn, RT_HIP_E_SHAPE, "n_pages must be >= 1 and n_pages * page_size below 2^31");
    const int64_t dense = (static_cast<int64_t>(kv->n_kv_heads) * kv->head_dim) << shift;
    const int64_t stride = kv->page_stride ? kv->page_stride : dense;
    if (stride < dense) return fail(fn, RT_HIP_E_ARG, "page_stride below a page's values");
    if (stride > 0xffffffffLL / value_bytes(kv->dtype)) return fail(fn, RT_HIP_E_SHAPE, "page_stride must be below 2^32 bytes");
    if (!aligned(kv->k, 16) || !aligned(kv->v, 16) || stride * value_bytes(kv->dtype) % 16)
        return fail(fn, RT_HIP_E_ALIGN, "pages must be 16-byte aligned");
    out->k = kv->k;
    out->v = kv->v;
    out->dtype = kv->dtype;
    out->n_pages = kv->n_pages;
    out->page_shift = shift;
    out->n_kv = kv->n_kv_heads;
    out->head_dim = kv->head_dim;
    out->page_stride = stride;
    return RT_HIP_OK;
}

Range pages_of(const PagedKv& c, const void* p) {
    const int64_t page = (static_cast<int64_t>(c.n_kv) * c.head_dim) << c.page_shift;
    return {p, ((c.n_pages - 1) * c.page_stride + page) * value_bytes(c.dtype)};
}

// Whether a page of keys and one of values share memory (pages of the two may lie in turn).
bool keys_over_values(const PagedKv& c) {
    const uintptr_t k = reinterpret_cast<uintptr_t>(c.k), v = reinterpret_cast<uintptr_t>(c.v), apart = k < v ? v - k : k - v;
    const uintptr_t stride = c.page_stride * value_bytes(c.dtype);
    const uintptr_t page = ((static_cast<uintptr_t>(c.n_kv) * c.head_dim) << c.page_shift) * value_bytes(c.dtype);
    if (apart >= (c.n_pages - 1) * stride + page) return false;
    // (a page's nearest of the other kind starts apart % stride before it, or what is left of a stride behind it)
    return apart % stride < page || stride - apart % stride < page;
}

int table_args(const char* fn, const int32_t* table, int64_t cols, int n_seq, int shift) {
    if (!table && n_seq > 0) return fail(fn, RT_HIP_E_ARG, "null block table");
    if (cols < 1) return fail(fn, RT_HIP_E_ARG, "table_cols must be >= 1");
    if ((cols << shift) > 0x7fffffffLL || cols > 0x7fffffffLL / (n_seq > 0 ? n_seq : 1))
        return fail(fn, RT_HIP_E_SHAPE, "table_cols * page_size and n_seq * table_cols must be below 2^31");
    return RT_HIP_OK;
}

}  // namespace

extern "C" {

int rt_hip_paged_plan(const int32_t* cached, const int32_t* fresh, const int32_t* held, int32_t* held_out,
                      int32_t* table, int64_t table_cols, int32_t* queue, const int32_t* queue_state,
                      int32_t* queue_state_out, int32_t n_pages, int32_t page_size, int32_t n_seq, int32_t n_tokens,
                      int32_t* q_start, int32_t* kv_len, int32_t* slots, int32_t* positions, rt_hip_stream stream) {
    const char* fn = "rt_hip_paged_plan";
    if (n_seq < 0 || n_tokens < 0) return fail(fn, RT_HIP_E_ARG, "negative size");
    if (n_seq > kPlanMaxSeq) return fail(fn, RT_HIP_E_SHAPE, "n_seq must be at most " + std::to_string(kPlanMaxSeq));
    if (n_seq > 0 && (!cached || !fresh || !held || !held_out || !kv_len)) return fail(fn, RT_HIP_E_ARG, "null pointer");
    if (!queue || !queue_state || !queue_state_out || !q_start || (n_tokens > 0 && (!slots || !positions)))
        return fail(fn, RT_HIP_E_ARG, "null pointer");
    const int shift = page_shift(page_size);
    if (shift < 0) return fail(fn, RT_HIP_E_SHAPE, "page_size must be a power of two from 8 to 1024");
    if (n_pages < 1 || (static_cast<int64_t>(n_pages) << shift) > 0x7fffffffLL)
        return fail(fn, RT_HIP_E_SHAPE, "n_pages must be >= 1 and n_pages * page_size below 2^31");
    if (const int rc = table_args(fn, table, table_cols, n_seq, shift)) return rc;
    const int64_t n = n_seq, t = n_tokens;
    const Range written[] = {{held_out, 4 * n}, {table, 4 * n * table_cols}, {queue, 4LL * n_pages}, {queue_state_out, 8},
                             {q_start, 4 * (n + 1)}, {kv_len, 4 * n}, {slots, 4 * t}, {positions, 4 * t}};
    const Range read[] = {{cached, 4 * n}, {fresh, 4 * n}, {held, 4 * n}, {queue_state, 8}};
    for (size_t i = 0; i < sizeof written / sizeof *written; ++i) {
        for (size_t j = 0; j < i; ++j)
            if (overlap(written[i], written[j])) return fail(fn, RT_HIP_E_ARG, "outputs overlap");
        for (const Range& r : read) {
            const bool in_place = (written[i].p == held_out && r.p == held && held_out == held) ||
                                  (written[i].p == queue_state_out && r.p == queue_state && queue_state_out == queue_state);
            if (!in_place && overlap(written[i], r)) return fail(fn, RT_HIP_E_ARG, "an output overlaps an input");
        }
    }
    PagedPlan p;
    p.cached = cached;
    p.fresh = fresh;
    p.held = held;
    p.held_out = held_out;
    p.table = table;
    p.cols = table_cols;
    p.queue = queue;
    p.queue_state = queue_state;
    p.queue_state_out = queue_state_out;
    p.q_start = q_start;
    p.kv_len = kv_len;
    p.slots = slots;
    p.positions = positions;
    p.n_pages = n_pages;
    p.page_shift = shift;
    p.n_seq = n_seq;
    p.n_tokens = n_tokens;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    hipError_t e;
    uint32_t* const counters = arrival_counters(s, &e);
    if (!counters) return launched(fn, e);
    return launched(fn, launch_paged_plan(p, counters, s));
}

int rt_hip_paged_append(const rt_hip_paged_kv* kv, const void* k, const void* v, int32_t dtype, int64_t row_stride,
                        const int32_t* slots, int32_t n_tokens, rt_hip_stream stream) {
    const char* fn = "rt_hip_paged_append";
    PagedKv c;
    if (const int rc = cache_args(fn, kv, &c)) return rc;
    if (keys_over_values(c)) return fail(fn, RT_HIP_E_ARG, "the cache's keys and values overlap");
    if (n_tokens < 0) return fail(fn, RT_HIP_E_ARG, "n_tokens must be >= 0");
    if (!value_bytes(dtype)) return fail(fn, RT_HIP_E_UNSUPPORTED, "k and v must be F32, F16 or BF16");
    if (n_tokens == 0) return RT_HIP_OK;
    if (!k || !v || !slots) return fail(fn, RT_HIP_E_ARG, "null pointer");
    const int64_t row = static_cast<int64_t>(c.n_kv) * c.head_dim;
    if (row_stride < row) return fail(fn, RT_HIP_E_ARG, "row_stride below a row's values");
    if (!aligned(k, 16) || !aligned(v, 16) || row_stride * value_bytes(dtype) % 16)
        return fail(fn, RT_HIP_E_ALIGN, "rows must be 16-byte aligned");
    if (row / 8 * n_tokens > 0x7fffffffLL - 256)
        return fail(fn, RT_HIP_E_SHAPE, "n_tokens * n_kv_heads * head_dim must be below 2^34");
    const int64_t bytes = ((n_tokens - 1) * row_stride + row) * value_bytes(dtype);
    for (const void* src : {k, v})
        for (const void* dst : {static_cast<const void*>(c.k), static_cast<const void*>(c.v)})
            if (overlap({src, bytes}, pages_of(c, dst))) return fail(fn, RT_HIP_E_ARG, "k or v overlaps the cache");
    return launched(fn, launch_paged_append(dtype, k, v, row_stride, c, slots, n_tokens, static_cast<hipStream_t>(stream)));
}

}  // extern "C"

namespace {

int attention_args(const char* fn, const rt_hip_paged_kv* kv, int32_t dtype, int32_t n_q_heads, int32_t n_seq,
                   int32_t n_tokens, int32_t max_fresh, PagedAttn* p) {
    if (const int rc = cache_args(fn, kv, &p->kv)) return rc;
    if (!value_bytes(dtype) || (dtype != RT_HIP_F32 && dtype != p->kv.dtype))
        return fail(fn, RT_HIP_E_UNSUPPORTED, "q must be F32 or of the cache's type");
    if (n_q_heads < p->kv.n_kv || n_q_heads % p->kv.n_kv || n_q_heads > 1024)
        return fail(fn, RT_HIP_E_SHAPE, "n_q_heads must be a multiple of n_kv_heads, at most 1024");
    if (n_seq < 0 || n_tokens < 0 || max_fresh < 0) return fail(fn, RT_HIP_E_ARG, "negative size");
    if (n_seq > kPlanMaxSeq) return fail(fn, RT_HIP_E_SHAPE, "n_seq must be at most " + std::to_string(kPlanMaxSeq));
    if (static_cast<int64_t>(n_tokens) * n_q_heads > 0x7fffffffLL)
        return fail(fn, RT_HIP_E_SHAPE, "n_tokens * n_q_heads must be below 2^31");
    p->dtype = dtype;
    p->n_q = n_q_heads;
    p->n_seq = n_seq;
    p->n_tokens = n_tokens;
    p->max_fresh = max_fresh;
    return RT_HIP_OK;
}

}  // namespace

extern "C" {

int rt_hip_paged_attention(const void* q, int32_t dtype, int64_t q_stride, int32_t n_q_heads, const rt_hip_paged_kv* kv,
                           const int32_t* table, int64_t table_cols, const int32_t* q_start, const int32_t* kv_len,
                           int32_t n_seq, int32_t n_tokens, int32_t max_fresh, float scale, int32_t window, void* out,
                           int64_t out_stride, rt_hip_stream stream) {
    const char* fn = "rt_hip_paged_attention";
    PagedAttn p;
    if (const int rc = attention_args(fn, kv, dtype, n_q_heads, n_seq, n_tokens, max_fresh, &p)) return rc;
    if (!(scale > 0.0f) || scale > 0x1p127f)  // (scores are weighed as powers of two: times log2(e))
        return fail(fn, RT_HIP_E_ARG, "scale must be positive and at most 2^127");
    if (window < 0) return fail(fn, RT_HIP_E_ARG, "window must be >= 0");
    if (n_seq == 0 || n_tokens == 0) return RT_HIP_OK;
    if (!q || !out || !q_start || !kv_len) return fail(fn, RT_HIP_E_ARG, "null pointer");
    if (const int rc = table_args(fn, table, table_cols, n_seq, p.kv.page_shift)) return rc;
    const int64_t row = static_cast<int64_t>(n_q_heads) * p.kv.head_dim, bytes = value_bytes(dtype);
    if (q_stride < row || out_stride < row) return fail(fn, RT_HIP_E_ARG, "q_stride or out_stride below a row's values");
    if (!aligned(q, 16) || !aligned(out, 16) || q_stride * bytes % 16 || out_stride * bytes % 16)
        return fail(fn, RT_HIP_E_ALIGN, "rows of q and out must be 16-byte aligned");
    const Range dst = {out, ((n_tokens - 1) * out_stride + row) * bytes};
    const Range read[] = {{q, ((n_tokens - 1) * q_stride + row) * bytes}, pages_of(p.kv, p.kv.k), pages_of(p.kv, p.kv.v),
                          {table, 4 * n_seq * table_cols}, {q_start, 4 * (static_cast<int64_t>(n_seq) + 1)},
                          {kv_len, 4 * static_cast<int64_t>(n_seq)}};
    for (const Range& r : read)
        if (overlap(dst, r)) return fail(fn, RT_HIP_E_ARG, "out overlaps an input");
    p.q = q;
    p.out = out;
    p.q_stride = q_stride;
    p.out_stride = out_stride;
    p.table = table;
    p.cols = table_cols;
    p.q_start = q_start;
    p.kv_len = kv_len;
    p.window = window;
    p.scale = scale;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    hipError_t e;
    uint32_t* const counters = arrival_counters(s, &e);
    if (!counters) return launched(fn, e);
    void* part = nullptr;
    if (const size_t need = paged_attention_workspace(p))
        if (!(part = workspace(need, s, &e))) return launched(fn, e);
    return launched(fn, launch_paged_attention(p, part, counters, s));
}

int64_t rt_hip_paged_attention_workspace_bytes(const rt_hip_paged_kv* kv, int32_t dtype, int32_t n_q_heads,
                                               int32_t n_seq, int32_t n_tokens, int32_t max_fresh) {
    PagedAttn p;
    if (attention_args("rt_hip_paged_attention_workspace_bytes", kv, dtype, n_q_heads, n_seq, n_tokens, max_fresh, &p))
        return -1;
    return n_seq == 0 || n_tokens == 0 ? 0 : static_cast<int64_t>(paged_attention_workspace(p));
}

}  // extern "C"

namespace {

constexpr int kMaxVocab = 1 << 20;

int verify_args(const char* fn, int32_t dtype, int32_t vocab, int32_t n_seq, int32_t n_rows, int32_t max_draft) {
    if (dtype != RT_HIP_F32 && dtype != RT_HIP_BF16) return fail(fn, RT_HIP_E_UNSUPPORTED, "logits must be F32 or BF16");
    if (vocab < 1 || n_seq < 0 || n_rows < 0 || max_draft < 0) return fail(fn, RT_HIP_E_ARG, "negative size or no vocabulary");
    if (vocab > kMaxVocab) return fail(fn, RT_HIP_E_SHAPE, "vocab must be at most 2^20");
    if (max_draft > 255 || static_cast<int64_t>(n_seq) * (max_draft + 1) > 65535)
        return fail(fn, RT_HIP_E_SHAPE, "max_draft must be at most 255 and n_seq * (max_draft + 1) at most 65535");
    if (n_seq > kPlanMaxSeq) return fail(fn, RT_HIP_E_SHAPE, "n_seq must be at most " + std::to_string(kPlanMaxSeq));
    return RT_HIP_OK;
}

}  // namespace

extern "C" {

int rt_hip_verify_drafts(const void* logits, int64_t logit_stride, const void* draft_logits, int64_t draft_stride,
                         int32_t dtype, int32_t vocab, const int32_t* tokens, const int32_t* row_start,
                         const float* accept_u, const float* sample_u, const float* temperature, int32_t n_seq,
                         int32_t n_rows, int32_t max_draft, int32_t* out_tokens, int32_t* out_count,
                         rt_hip_stream stream) {
    const char* fn = "rt_hip_verify_drafts";
    if (const int rc = verify_args(fn, dtype, vocab, n_seq, n_rows, max_draft)) return rc;
    if (n_seq == 0) return RT_HIP_OK;
    if (!row_start || !out_tokens || !out_count || !sample_u || (n_rows > 0 && (!logits || !tokens || !accept_u)))
        return fail(fn, RT_HIP_E_ARG, "null pointer");
    if (logit_stride < vocab || (draft_logits && draft_stride < vocab)) return fail(fn, RT_HIP_E_ARG, "row stride below vocab");
    const int64_t b = value_bytes(dtype), rows = n_rows, n = n_seq;
    if (!aligned(logits, static_cast<uintptr_t>(b)) || !aligned(draft_logits, static_cast<uintptr_t>(b)))
        return fail(fn, RT_HIP_E_ALIGN, "logits must be aligned to their type");
    const Range written[] = {{out_tokens, 4 * n * (max_draft + 1)}, {out_count, 4 * n}};
    const int64_t span = rows > 0 ? rows - 1 : 0;
    const Range read[] = {{logits, rows ? (span * logit_stride + vocab) * b : 0},
                          {draft_logits, draft_logits && rows ? (span * draft_stride + vocab) * b : 0},
                          {tokens, 4 * rows}, {row_start, 4 * (n + 1)}, {accept_u, 4 * rows}, {sample_u, 4 * n},
                          {temperature, temperature ? 4 * n : 0}};
    for (const Range& w : written)
        for (const Range& r : read)
            if (overlap(w, r)) return fail(fn, RT_HIP_E_ARG, "an output overlaps an input");
    if (overlap(written[0], written[1])) return fail(fn, RT_HIP_E_ARG, "outputs overlap");
    VerifyDrafts p;
    p.logits = logits;
    p.draft_logits = draft_logits;
    p.dtype = dtype;
    p.logit_stride = logit_stride;
    p.draft_stride = draft_stride;
    p.tokens = tokens;
    p.row_start = row_start;
    p.accept_u = accept_u;
    p.sample_u = sample_u;
    p.temperature = temperature;
    p.out_tokens = out_tokens;
    p.out_count = out_count;
    p.vocab = vocab;
    p.n_seq = n_seq;
    p.n_rows = n_rows;
    p.max_draft = max_draft;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    hipError_t e;
    uint32_t* const counters = arrival_counters(s, &e);
    if (!counters) return launched(fn, e);
    void* const work = workspace(verify_drafts_workspace(p), s, &e);
    if (!work) return launched(fn, e);
    return launched(fn, launch_verify_drafts(p, work, counters, s));
}

int64_t rt_hip_verify_drafts_workspace_bytes(int32_t vocab, int32_t n_seq, int32_t n_rows, int32_t max_draft,
                                             int32_t with_draft_logits) {
    if (verify_args("rt_hip_verify_drafts_workspace_bytes", RT_HIP_F32, vocab, n_seq, n_rows, max_draft)) return -1;
    VerifyDrafts p;
    p.vocab = vocab;
    p.n_seq = n_seq;
    p.n_rows = n_rows;
    p.max_draft = max_draft;
    p.draft_logits = with_draft_logits ? &p : nullptr;  // (only whether there are any counts)
    return n_seq == 0 ? 0 : static_cast<int64_t>(verify_drafts_workspace(p));
}

}  // extern "C"
