// Host side of the cache's operators (include/q8_cache.h): argument checks and
// launches.
#include "cache_internal.hpp"
#include "q8_host.hpp"

namespace {

using namespace q8;

// Row numbers and the 8-bit data's offsets stay below these.
constexpr uint64_t kMostPageBytes = 1ull << 31, kMostCacheBytes = 1ull << 48;

uint32_t pitch_of(uint32_t dim) { return (dim + 15) / 16 * 16; }

// Kernels count a few tokens' heads and their pieces in 31 bits.
int check_columns(uint64_t heads, uint64_t dim) {
    if (heads * dim >= (1u << 24)) return fail(SGEMM_E_SHAPE, "%llu values a token: 2^24 and more are not served", (unsigned long long)(heads * dim));
    return SGEMM_OK;
}

int check_cache(const q8_cache* c) {
    if (!c) return fail(SGEMM_E_INVALID, "cache is null");
    if (!c->dim || c->dim > Q8_MAX_DIM) return fail(SGEMM_E_SHAPE, "cache: heads of %u values: 1 to %u are served", c->dim, Q8_MAX_DIM);
    if (!c->heads || !c->page_tokens) return fail(SGEMM_E_SHAPE, "cache: no heads, or pages of no tokens");
    CHECK(check_columns(c->heads, c->dim));
    if (c->pages >= (1u << 31)) return fail(SGEMM_E_SHAPE, "cache: %u pages: page numbers have 31 bits", c->pages);
    const uint64_t rows = (uint64_t)c->heads * c->page_tokens, bytes = rows * pitch_of(c->dim);
    // rows below 2^31 first: their product with the pitch may not pass 64 bits
    if (rows >= kMostPageBytes || bytes >= kMostPageBytes) return fail(SGEMM_E_SHAPE, "cache: a page of 2^31 bytes or more");
    if (bytes * c->pages > kMostCacheBytes) return fail(SGEMM_E_SHAPE, "cache: more than 2^48 bytes");
    return SGEMM_OK;
}

int check_batch(const q8_batch* b, const q8_cache* c) {
    if (!b) return fail(SGEMM_E_INVALID, "batch is null");
    if (b->tokens >= (1u << 31) || b->seqs >= (1u << 31)) return fail(SGEMM_E_SHAPE, "batch: tokens and sequences have 31 bits");
    // kernels look some steps past a sequence's end, still in 31 bits
    if ((uint64_t)b->width * c->page_tokens >= (1ull << 31) - (1u << 16))
        return fail(SGEMM_E_SHAPE, "batch: %u pages of %u tokens: positions end at 2^31 - 2^16", b->width, c->page_tokens);
    return SGEMM_OK;
}

// The tensors of a cache and a batch, checked; `outs` of them are written (the cache's, for q8_cache_write).
struct Tensors {
    Span cache[4], batch[3];
};
int check_tensors(const q8_cache& c, const q8_batch& b, Tensors& t) {
    const uint64_t rows = (uint64_t)c.pages * c.heads * c.page_tokens, pitch = pitch_of(c.dim);
    // as one row each: rows of whole pitches have nothing between them
    t.cache[0] = vec("cache k", c.k, rows * pitch, 1);
    t.cache[1] = vec("cache v", c.v, rows * pitch, 1);
    t.cache[2] = vec("cache k_scale", c.k_scale, rows, 4);
    t.cache[3] = vec("cache v_scale", c.v_scale, rows, 4);
    t.batch[0] = vec("starts", b.starts, (uint64_t)b.seqs + 1, 4);
    t.batch[1] = vec("lengths", b.lengths, b.seqs, 4);
    t.batch[2] = Span{"table", b.table, b.seqs, b.width, b.table_ld, 4};
    for (const Span& s : t.cache) CHECK(check(s));
    for (const Span& s : t.batch) CHECK(check(s));
    for (int i = 0; i < 2; ++i)
        if (rows && (uintptr_t)t.cache[i].p % 16) return fail(SGEMM_E_INVALID, "%s is not aligned to 16 bytes", t.cache[i].name);
    return SGEMM_OK;
}

Paged paged(const q8_cache& c, const q8_batch& b) {
    return Paged{c.k, c.v, c.k_scale, c.v_scale, c.pages, c.page_tokens, c.heads, c.dim, pitch_of(c.dim),
                 b.starts, b.lengths, b.table, b.seqs, b.tokens, b.width, b.table_ld, divisor(c.page_tokens)};
}

int cache_rows(q8_handle* h, int dtype, const q8_cache* cache, const q8_batch* batch, void* k, uint32_t ldk, void* v, uint32_t ldv,
               bool write) {
    CHECK(check_handle(h));
    CHECK(check_type(dtype));
    CHECK(check_cache(cache));
    CHECK(check_batch(batch, cache));
    if (!batch->tokens || !batch->seqs) return SGEMM_OK;
    Tensors t;
    CHECK(check_tensors(*cache, *batch, t));
    const uint64_t cols = (uint64_t)cache->heads * cache->dim;
    const uint32_t size = type_bytes(dtype);
    const Span rows[] = {{"k", k, batch->tokens, cols, ldk, size}, {"v", v, batch->tokens, cols, ldv, size}};
    for (const Span& s : rows) CHECK(check(s));
    if (write) {
        for (int i = 0; i < 4; ++i) {
            for (const Span& s : rows) CHECK(check_apart(t.cache[i], s));
            for (const Span& s : t.batch) CHECK(check_apart(t.cache[i], s));
            for (int j = 0; j < i; ++j) CHECK(check_apart(t.cache[i], t.cache[j]));
        }
    } else {
        for (const Span& s : rows) {
            for (const Span& o : t.cache) CHECK(check_apart(s, o));
            for (const Span& o : t.batch) CHECK(check_apart(s, o));
        }
        CHECK(check_apart(rows[1], rows[0]));
    }
    OnDevice on(h->device);
    HIP_TRY(on.status());
    const CacheRows p = {paged(*cache, *batch), k, v, ldk, ldv};
    return write ? launched(launch_cache_write(dtype, p, h->stream), "launch of the cache's writing failed")
                 : launched(launch_cache_read(dtype, p, h->stream), "launch of the cache's reading failed");
}

int plan(int dtype, const q8_cache& c, const q8_batch& b, uint32_t heads, AttentionPlan& p) {
    if (!heads || heads % c.heads) return fail(SGEMM_E_SHAPE, "%u heads are no multiple of the cache's %u", heads, c.heads);
    CHECK(check_columns(heads, c.dim));
    if ((uint64_t)b.tokens * heads >= (1ull << 31)) return fail(SGEMM_E_SHAPE, "%u tokens of %u heads: rows have 31 bits", b.tokens, heads);
    p = plan_attention(dtype == Q8_F32, b.tokens, b.seqs, (uint64_t)b.width * c.page_tokens, b.longest, heads, c.heads, c.dim);
    for (const AttentionLaunch* l : {&p.few, &p.many})
        if ((uint64_t)l->slots * c.heads * l->pieces > l->most_groups)
            return fail(SGEMM_E_SHAPE, "%u tokens of %u heads are more tiles than a grid holds", b.tokens, heads);
    return SGEMM_OK;
}

}  // namespace

extern "C" {

int q8_rotary(q8_handle* h, int dtype, const q8_rotation* form, const void* x, uint32_t ldx, const int32_t* positions,
              uint32_t ldp, const float* freq, void* y, uint32_t ldy, uint32_t tokens, uint32_t heads, int inverse) {
    CHECK(check_handle(h));
    CHECK(check_type(dtype));
    if (!form) return fail(SGEMM_E_INVALID, "form is null");
    if (!form->dim || form->dim > Q8_MAX_DIM) return fail(SGEMM_E_SHAPE, "heads of %u values: 1 to %u are served", form->dim, Q8_MAX_DIM);
    if (form->pairs > form->dim / 2) return fail(SGEMM_E_SHAPE, "%u pairs in heads of %u values", form->pairs, form->dim);
    if (!form->axes || form->axes > Q8_MAX_AXES) return fail(SGEMM_E_SHAPE, "%u axes: 1 to %u are served", form->axes, Q8_MAX_AXES);
    for (uint32_t j = 0; j < form->pairs; ++j)
        if (form->axis[j] >= form->axes) return fail(SGEMM_E_INVALID, "pair %u is on axis %u of %u", j, form->axis[j], form->axes);
    const uint64_t cols = (uint64_t)heads * form->dim;
    CHECK(check_columns(heads, form->dim));
    if (tokens >= (1u << 31)) return fail(SGEMM_E_SHAPE, "%u tokens: 31 bits are served", tokens);
    if (!tokens || !heads) return SGEMM_OK;
    const uint32_t size = type_bytes(dtype);
    const Span in[] = {{"x", x, tokens, cols, ldx, size}, {"positions", positions, form->pairs ? form->axes : 0u, tokens, ldp, 4},
                       vec("freq", freq, form->pairs, 4)};
    const Span out{"y", y, tokens, cols, ldy, size};
    for (const Span& s : in) CHECK(check(s));
    CHECK(check(out));
    for (int i = 0; i < 3; ++i) CHECK(check_apart(out, in[i], i == 0));
    OnDevice on(h->device);
    HIP_TRY(on.status());
    const Rotary p = {x, positions, freq, y, ldx, ldp, ldy, tokens, heads, inverse != 0, *form};
    return launched(launch_rotary(dtype, p, h->stream), "launch of the rotation failed");
}

int q8_cache_write(q8_handle* h, int dtype, const q8_cache* cache, const q8_batch* batch, const void* k, uint32_t ldk,
                   const void* v, uint32_t ldv) {
    return cache_rows(h, dtype, cache, batch, const_cast<void*>(k), ldk, const_cast<void*>(v), ldv, true);
}

int q8_cache_read(q8_handle* h, int dtype, const q8_cache* cache, const q8_batch* batch, void* k, uint32_t ldk, void* v,
                  uint32_t ldv) {
    return cache_rows(h, dtype, cache, batch, k, ldk, v, ldv, false);
}

int q8_attention(q8_handle* h, int dtype, const q8_cache* cache, const q8_batch* batch, uint32_t heads, const void* q,
                 uint32_t ldq, float scale, uint32_t window, void* out, uint32_t ldo, float* lse) {
    CHECK(check_handle(h));
    CHECK(check_type(dtype));
    CHECK(check_cache(cache));
    CHECK(check_batch(batch, cache));
    AttentionPlan p;
    CHECK(plan(dtype, *cache, *batch, heads, p));
    // times the exponential's base and a key's scale it stays a number
    if (!(scale >= -0x1p100f && scale <= 0x1p100f)) return fail(SGEMM_E_INVALID, "scale is not in -2^100 .. 2^100");
    if (!batch->tokens || !batch->seqs) return SGEMM_OK;
    Tensors t;
    CHECK(check_tensors(*cache, *batch, t));
    const uint64_t cols = (uint64_t)heads * cache->dim;
    const uint32_t size = type_bytes(dtype);
    const Span in{"q", q, batch->tokens, cols, ldq, size};
    const Span outs[] = {{"out", out, batch->tokens, cols, ldo, size},
                         vec("lse", lse, lse ? (uint64_t)batch->tokens * heads : 0u, 4)};
    CHECK(check(in));
    for (const Span& s : outs) {
        CHECK(check(s));
        CHECK(check_apart(s, in));
        for (const Span& o : t.cache) CHECK(check_apart(s, o));
        for (const Span& o : t.batch) CHECK(check_apart(s, o));
    }
    CHECK(check_apart(outs[1], outs[0]));
    OnDevice on(h->device);
    HIP_TRY(on.status());
    const Attention a = {paged(*cache, *batch), q, out, lse, ldq, ldo, heads, heads / cache->heads, window, scale};
    CHECK(take_workspace(h, p.bytes));
    for (const AttentionLaunch* l : {&p.few, &p.many}) {
        if (!l->slots) continue;
        const uint64_t rows = (uint64_t)l->pieces * batch->tokens * heads;
        float* sums = l->pieces > 1 ? reinterpret_cast<float*>(h->workspace + p.image_bytes) : nullptr;
        const AttentionArgs g = {a, divisor(a.group), l->slots, l->least, l->most, l->piece,
                                 sums, sums ? sums + rows * held_dim(cache->dim) : nullptr, h->tickets,
                                 l == &p.many && p.images ? h->workspace : nullptr, p.images};
        CHECK(launched((l == &p.few ? launch_few : p.images ? launch_prompt : launch_many)(dtype, g, l->pieces, h->stream), "launch of the attention failed"));
    }
    return SGEMM_OK;
}

int q8_attention_workspace(int dtype, const q8_cache* cache, const q8_batch* batch, uint32_t heads, size_t* bytes) {
    if (!bytes) return fail(SGEMM_E_INVALID, "bytes is null");
    *bytes = 0;
    CHECK(check_type(dtype));
    CHECK(check_cache(cache));
    CHECK(check_batch(batch, cache));
    AttentionPlan p;
    CHECK(plan(dtype, *cache, *batch, heads, p));
    *bytes = p.bytes;
    return SGEMM_OK;
}

}  // extern "C"
