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

bool cache_type(int32_t dtype) { return value_bytes(dtype) != 0 || dtype == RT_HIP_Q4KV; }
// Bytes of `values` of a cache's; of its page_stride.
int64_t cache_bytes(int32_t dtype, int64_t values) { return dtype == RT_HIP_Q4KV ? values / 8 * 5 : values * value_bytes(dtype); }
int64_t stride_bytes(const PagedKv& c) { return c.dtype == RT_HIP_Q4KV ? c.page_stride : c.page_stride * value_bytes(c.dtype); }
int64_t page_bytes(const PagedKv& c) {
    return cache_bytes(c.dtype, (static_cast<int64_t>(c.n_kv) * c.head_dim) << c.page_shift);
}

// log2 of a page size the kernels take, -1 otherwise.
int page_shift(int32_t page_size) {
    for (int s = 3; s <= 10; ++s)
        if (page_size == 1 << s) return s;
    return -1;
}

// The caller's description of a cache, checked, as the kernels take it.
int cache_args(const char* fn, const rt_hip_paged_kv* kv, PagedKv* out) {
    if (!kv || !kv->k || !kv->v) return fail(fn, RT_HIP_E_ARG, "null cache");
    if (!cache_type(kv->dtype)) return fail(fn, RT_HIP_E_UNSUPPORTED, "the cache must be F32, F16, BF16 or Q4KV");
    const int shift = page_shift(kv->page_size);
    if (shift < 0) return fail(fn, RT_HIP_E_SHAPE, "page_size must be a power of two from 8 to 1024");
    if (kv->head_dim != 64 && kv->head_dim != 128 && kv->head_dim != 256)
        return fail(fn, RT_HIP_E_SHAPE, "head_dim must be 64, 128 or 256");
    if (kv->n_kv_heads < 1 || kv->n_kv_heads > 256) return fail(fn, RT_HIP_E_SHAPE, "n_kv_heads must be in [1, 256]");
    if (kv->n_pages < 1 || (static_cast<int64_t>(kv->n_pages) << shift) > 0x7fffffffLL)
        return fail(fn, RT_HIP_E_SHAPE, "n_pages must be >= 1 and n_pages * page_size below 2^31");
    const bool four = kv->dtype == RT_HIP_Q4KV;  // (its page_stride counts bytes)
    const int64_t values = (static_cast<int64_t>(kv->n_kv_heads) * kv->head_dim) << shift;
    const int64_t dense = four ? cache_bytes(kv->dtype, values) : values, unit = four ? 1 : value_bytes(kv->dtype);
    const int64_t stride = kv->page_stride ? kv->page_stride : dense;
    if (stride < dense) return fail(fn, RT_HIP_E_ARG, "page_stride below a page's values");
    if (stride > 0xffffffffLL / unit) return fail(fn, RT_HIP_E_SHAPE, "page_stride must be below 2^32 bytes");
    if (!aligned(kv->k, 16) || !aligned(kv->v, 16) || stride * unit % 16)
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
    return {p, (c.n_pages - 1) * stride_bytes(c) + page_bytes(c)};
}

// Whether a page of keys and one of values share memory (pages of the two may lie in turn).
bool keys_over_values(const PagedKv& c) {
    const uintptr_t k = reinterpret_cast<uintptr_t>(c.k), v = reinterpret_cast<uintptr_t>(c.v), apart = k < v ? v - k : k - v;
    const uintptr_t stride = stride_bytes(c), page = page_bytes(c);
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

int64_t rt_hip_paged_page_bytes(int32_t dtype, int32_t page_size, int32_t n_kv_heads, int32_t head_dim) {
    void* const some = reinterpret_cast<void*>(uintptr_t{16});  // (only the sizes are looked at)
    const rt_hip_paged_kv kv = {some, some, dtype, 1, page_size, n_kv_heads, head_dim, 0};
    PagedKv c;
    return cache_args("rt_hip_paged_page_bytes", &kv, &c) ? -1 : page_bytes(c);
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
    const auto launch = c.dtype == RT_HIP_Q4KV ? launch_paged4_append : launch_paged_append;
    return launched(fn, launch(dtype, k, v, row_stride, c, slots, n_tokens, static_cast<hipStream_t>(stream)));
}

int rt_hip_paged_read(const rt_hip_paged_kv* kv, const int32_t* slots, int32_t n_tokens, void* k, void* v, int32_t dtype,
                      int64_t row_stride, rt_hip_stream stream) {
    const char* fn = "rt_hip_paged_read";
    PagedKv c;
    if (const int rc = cache_args(fn, kv, &c)) return rc;
    if (n_tokens < 0) return fail(fn, RT_HIP_E_ARG, "n_tokens must be >= 0");
    if (!value_bytes(dtype)) return fail(fn, RT_HIP_E_UNSUPPORTED, "k and v must be F32, F16 or BF16");
    if (n_tokens == 0) return RT_HIP_OK;
    if (!k || !v || !slots) return fail(fn, RT_HIP_E_ARG, "null pointer");
    const int64_t row = static_cast<int64_t>(c.n_kv) * c.head_dim;
    if (row_stride < row) return fail(fn, RT_HIP_E_ARG, "row_stride below a row's values");
    if (row_stride > 0x7fffffffffffLL / n_tokens) return fail(fn, RT_HIP_E_SHAPE, "n_tokens * row_stride must be below 2^47");
    if (!aligned(k, 16) || !aligned(v, 16) || row_stride * value_bytes(dtype) % 16)
        return fail(fn, RT_HIP_E_ALIGN, "rows must be 16-byte aligned");
    if (row / 8 * n_tokens > 0x7fffffffLL - 256)
        return fail(fn, RT_HIP_E_SHAPE, "n_tokens * n_kv_heads * head_dim must be below 2^34");
    const int64_t bytes = ((n_tokens - 1) * row_stride + row) * value_bytes(dtype);
    const Range slot_range = {slots, 4 * static_cast<int64_t>(n_tokens)};
    for (const void* dst : {k, v}) {
        if (overlap({dst, bytes}, pages_of(c, c.k)) || overlap({dst, bytes}, pages_of(c, c.v)))
            return fail(fn, RT_HIP_E_ARG, "k or v overlaps the cache");
        if (overlap({dst, bytes}, slot_range)) return fail(fn, RT_HIP_E_ARG, "k or v overlaps slots");
    }
    // (rows of the two may lie in turn, as halves of one tensor)
    const uintptr_t a = reinterpret_cast<uintptr_t>(k), b = reinterpret_cast<uintptr_t>(v);
    const uintptr_t apart = a < b ? b - a : a - b, stride = row_stride * value_bytes(dtype), dense = row * value_bytes(dtype);
    if (apart < static_cast<uintptr_t>(bytes) && (apart % stride < dense || stride - apart % stride < dense))
        return fail(fn, RT_HIP_E_ARG, "k and v overlap");
    return launched(fn, launch_paged_read(c, slots, n_tokens, dtype, k, v, row_stride, static_cast<hipStream_t>(stream)));
}

}  // extern "C"

namespace {

int attention_args(const char* fn, const rt_hip_paged_kv* kv, int32_t dtype, int32_t n_q_heads, int32_t n_seq,
                   int32_t n_tokens, int32_t max_fresh, PagedAttn* p) {
    if (const int rc = cache_args(fn, kv, &p->kv)) return rc;
    if (!value_bytes(dtype) || (dtype != RT_HIP_F32 && dtype != p->kv.dtype && p->kv.dtype != RT_HIP_Q4KV))
        return fail(fn, RT_HIP_E_UNSUPPORTED, "q must be F32 or of the cache's type (any over Q4KV)");
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
    const bool four = p.kv.dtype == RT_HIP_Q4KV;
    if (const size_t need = four ? paged4_attention_workspace(p) : paged_attention_workspace(p))
        if (!(part = workspace(need, s, &e))) return launched(fn, e);
    return launched(fn, (four ? launch_paged4_attention : launch_paged_attention)(p, part, counters, s));
}

int64_t rt_hip_paged_attention_workspace_bytes(const rt_hip_paged_kv* kv, int32_t dtype, int32_t n_q_heads,
                                               int32_t n_seq, int32_t n_tokens, int32_t max_fresh) {
    PagedAttn p;
    if (attention_args("rt_hip_paged_attention_workspace_bytes", kv, dtype, n_q_heads, n_seq, n_tokens, max_fresh, &p))
        return -1;
    if (n_seq == 0 || n_tokens == 0) return 0;
    return static_cast<int64_t>(p.kv.dtype == RT_HIP_Q4KV ? paged4_attention_workspace(p) : paged_attention_workspace(p));
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

extern "C" {

int rt_hip_adjust_logits(void* logits, int64_t stride, int32_t dtype, int32_t vocab, const int32_t* row_start,
                         int32_t n_seq, int32_t n_rows, const int32_t* tokens, const rt_hip_logit_rules* rules,
                         rt_hip_stream stream) {
    const char* fn = "rt_hip_adjust_logits";
    if (dtype != RT_HIP_F32 && dtype != RT_HIP_BF16) return fail(fn, RT_HIP_E_UNSUPPORTED, "logits must be F32 or BF16");
    if (!rules) return fail(fn, RT_HIP_E_ARG, "null rules");
    const rt_hip_logit_rules& u = *rules;
    if (vocab < 1 || n_seq < 0 || n_rows < 0 || u.n_bias < 0 || u.n_masks < 0)
        return fail(fn, RT_HIP_E_ARG, "negative size or no vocabulary");
    if (vocab > kMaxVocab) return fail(fn, RT_HIP_E_SHAPE, "vocab must be at most 2^20");
    if (n_seq > kPlanMaxSeq) return fail(fn, RT_HIP_E_SHAPE, "n_seq must be at most " + std::to_string(kPlanMaxSeq));
    if (u.history && (!u.history_len || u.history_cols < 1)) return fail(fn, RT_HIP_E_ARG, "a history needs history_len and history_cols");
    if (u.history && u.history_cols > 0x0fffffff) return fail(fn, RT_HIP_E_SHAPE, "history_cols must be below 2^28");
    if (u.bias && (!u.bias_start || (u.n_bias > 0 && !u.bias_token))) return fail(fn, RT_HIP_E_ARG, "biases need bias_start and bias_token");
    const int64_t words = (static_cast<int64_t>(vocab) + 31) / 32;
    if (u.mask && u.mask_stride < words) return fail(fn, RT_HIP_E_ARG, "mask_stride below a row's words");
    if (u.mask && !u.mask_row && u.n_masks < n_rows) return fail(fn, RT_HIP_E_ARG, "fewer masks than rows, and no mask_row");
    if (n_seq == 0 || n_rows == 0) return RT_HIP_OK;
    if (!logits || !row_start) return fail(fn, RT_HIP_E_ARG, "null pointer");
    if (stride < vocab) return fail(fn, RT_HIP_E_ARG, "row stride below vocab");
    const int64_t b = value_bytes(dtype), rows = n_rows, n = n_seq;
    if (stride > 0x7fffffffffffLL / rows || (u.mask && u.n_masks > 0 && u.mask_stride > 0x7fffffffffffLL / u.n_masks))
        return fail(fn, RT_HIP_E_SHAPE, "rows * stride must be below 2^47");
    if (!aligned(logits, static_cast<uintptr_t>(b))) return fail(fn, RT_HIP_E_ALIGN, "logits must be aligned to their type");
    const Range written = {logits, ((rows - 1) * stride + vocab) * b};
    const Range read[] = {{row_start, 4 * (n + 1)}, {tokens, tokens ? 4 * rows : 0},
                          {u.history, u.history ? 4 * n * u.history_cols : 0}, {u.history_len, u.history_len ? 4 * n : 0},
                          {u.prompt_len, u.prompt_len ? 4 * n : 0}, {u.repetition, u.repetition ? 4 * n : 0},
                          {u.presence, u.presence ? 4 * n : 0}, {u.frequency, u.frequency ? 4 * n : 0},
                          {u.bias_start, u.bias ? 4 * (n + 1) : 0}, {u.bias_token, u.bias ? 4LL * u.n_bias : 0},
                          {u.bias, u.bias ? 4LL * u.n_bias : 0},
                          {u.mask, u.mask && u.n_masks > 0 ? 4 * ((u.n_masks - 1) * u.mask_stride + words) : 0},
                          {u.mask_row, u.mask_row ? 4 * rows : 0}};
    for (const Range& r : read)
        if (overlap(written, r)) return fail(fn, RT_HIP_E_ARG, "logits overlap an input");
    AdjustLogits p;
    p.logits = logits;
    p.stride = stride;
    p.dtype = dtype;
    p.vocab = vocab;
    p.n_seq = n_seq;
    p.n_rows = n_rows;
    p.row_start = row_start;
    p.tokens = tokens;
    p.history = u.history;
    p.history_cols = u.history_cols;
    p.history_len = u.history_len;
    p.prompt_len = u.prompt_len;
    p.repetition = u.repetition;
    p.presence = u.presence;
    p.frequency = u.frequency;
    p.bias_start = u.bias_start;
    p.bias_token = u.bias_token;
    p.bias = u.bias;
    p.mask = u.mask;
    p.mask_stride = u.mask_stride;
    p.mask_row = u.mask_row;
    p.n_bias = u.n_bias;
    p.n_masks = u.n_masks;
    return launched(fn, launch_adjust_logits(p, static_cast<hipStream_t>(stream)));
}

}  // extern "C"

namespace {

int lora_args(const char* fn, const rt_hip_lora* l, int32_t n_seq, int32_t n_rows) {
    if (!l) return fail(fn, RT_HIP_E_ARG, "null adapters");
    if (l->dtype != RT_HIP_BF16 && l->dtype != RT_HIP_F16) return fail(fn, RT_HIP_E_UNSUPPORTED, "adapters must be BF16 or F16");
    if (l->n_adapters < 0 || n_seq < 0 || n_rows < 0) return fail(fn, RT_HIP_E_ARG, "negative size");
    if (l->k < 1 || l->n < 1 || l->k > (1 << 20) || l->n > (1 << 20)) return fail(fn, RT_HIP_E_SHAPE, "k and n must be in [1, 2^20]");
    if (l->rank < 8 || l->rank > 128) return fail(fn, RT_HIP_E_SHAPE, "rank must be in [8, 128]");
    if (l->rank % 8 || l->k % 8) return fail(fn, RT_HIP_E_ALIGN, "rank and k must be multiples of 8");
    if (n_seq > kPlanMaxSeq) return fail(fn, RT_HIP_E_SHAPE, "n_seq must be at most " + std::to_string(kPlanMaxSeq));
    if (n_rows > (1 << 24)) return fail(fn, RT_HIP_E_SHAPE, "n_rows must be at most 2^24");
    return RT_HIP_OK;
}

}  // namespace

extern "C" {

int rt_hip_lora_add(float* y, int64_t y_stride, const void* x, int32_t x_dtype, int64_t x_stride, const rt_hip_lora* lora,
                    const int32_t* row_start, const int32_t* adapter, int32_t n_seq, int32_t n_rows, rt_hip_stream stream) {
    const char* fn = "rt_hip_lora_add";
    if (const int rc = lora_args(fn, lora, n_seq, n_rows)) return rc;
    const rt_hip_lora& l = *lora;
    if (!value_bytes(x_dtype)) return fail(fn, RT_HIP_E_UNSUPPORTED, "x must be F32, F16 or BF16");
    if (n_seq == 0 || n_rows == 0 || l.n_adapters == 0) return RT_HIP_OK;
    if (!y || !x || !row_start || !adapter || !l.a || !l.b || !l.scale) return fail(fn, RT_HIP_E_ARG, "null pointer");
    if (y_stride < l.n || x_stride < l.k) return fail(fn, RT_HIP_E_ARG, "y_stride or x_stride below a row's values");
    const int64_t rows = n_rows, xb = value_bytes(x_dtype), m = l.n_adapters;
    if (y_stride > 0x7fffffffffffLL / rows || x_stride > 0x7fffffffffffLL / rows)
        return fail(fn, RT_HIP_E_SHAPE, "n_rows * stride must be below 2^47");
    if (!aligned(x, 16) || x_stride * xb % 16 || !aligned(l.a, 16) || !aligned(l.b, 16))
        return fail(fn, RT_HIP_E_ALIGN, "rows of x, and a and b, must be 16-byte aligned");
    if (!aligned(y, 4)) return fail(fn, RT_HIP_E_ALIGN, "y must be 4-byte aligned");
    const Range written = {y, 4 * ((rows - 1) * y_stride + l.n)};
    const Range read[] = {{x, ((rows - 1) * x_stride + l.k) * xb}, {l.a, 2 * m * l.rank * l.k}, {l.b, 2 * m * l.rank * l.n},
                          {l.scale, 4 * m}, {row_start, 4 * (static_cast<int64_t>(n_seq) + 1)}, {adapter, 4 * static_cast<int64_t>(n_seq)}};
    for (const Range& r : read)
        if (overlap(written, r)) return fail(fn, RT_HIP_E_ARG, "y overlaps an input");
    LoraAdd p;
    p.y = y;
    p.x = x;
    p.y_stride = y_stride;
    p.x_stride = x_stride;
    p.x_dtype = x_dtype;
    p.w_dtype = l.dtype;
    p.a = l.a;
    p.b = l.b;
    p.scale = l.scale;
    p.n_adapters = l.n_adapters;
    p.rank = l.rank;
    p.k = l.k;
    p.n = l.n;
    p.row_start = row_start;
    p.adapter = adapter;
    p.n_seq = n_seq;
    p.n_rows = n_rows;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    hipError_t e;
    p.part = static_cast<float*>(workspace(lora_workspace(l.rank, l.k, n_rows), s, &e));
    if (!p.part) return launched(fn, e);
    return launched(fn, launch_lora_add(p, s));
}

int64_t rt_hip_lora_workspace_bytes(const rt_hip_lora* lora, int32_t n_seq, int32_t n_rows) {
    if (lora_args("rt_hip_lora_workspace_bytes", lora, n_seq, n_rows)) return -1;
    return n_seq == 0 || n_rows == 0 ? 0 : static_cast<int64_t>(lora_workspace(lora->rank, lora->k, n_rows));
}

}  // extern "C"
