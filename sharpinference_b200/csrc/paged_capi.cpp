// C ABI of the paged 4-bit cache and of the logits processing: shape checks
// (SI_ERR_ADAPTATION as an instruction's Generate raises them), pointer checks
// against the device allocations, then the kernels.
#include <cmath>
#include <cstdint>
#include <initializer_list>

#include "si_internal.h"

using namespace si;

namespace {

si_status adapt(const char *op, const char *msg) { return fail(SI_ERR_ADAPTATION, "%s: %s", op, msg); }

struct Port {
    const char *name;
    const void *ptr;
    uint64_t bytes;
    uint32_t align;
};

si_status ports(std::initializer_list<Port> list) {
    for (const Port &p : list) {
        if (reinterpret_cast<uintptr_t>(p.ptr) % p.align)
            return fail(SI_ERR_INVALID_ARGUMENT, "port '%s': not aligned to %u bytes", p.name, p.align);
        if (si_status st = device_range(p.name, p.ptr, p.bytes)) return st;
    }
    return SI_OK;
}

// What a call writes may not lie in what its other blocks still read.
si_status apart(const Port &written, std::initializer_list<Port> read) {
    for (const Port &p : read)
        if (p.ptr && p.bytes && ranges_overlap(written.ptr, written.bytes, p.ptr, p.bytes))
            return fail(SI_ERR_INVALID_ARGUMENT, "port '%s': overlaps port '%s'", written.name, p.name);
    return SI_OK;
}

si_status tensor_type(const char *op, uint32_t type, uint32_t *size) {
    if (type != SI_TYPE_F32 && type != SI_TYPE_F16)
        return fail(SI_ERR_ADAPTATION, "%s: tensors must be F32 or F16.", op);
    *size = type == SI_TYPE_F32 ? 4 : 2;
    return SI_OK;
}

si_status cache_geometry(const char *op, int64_t page_count, int32_t page_size, int32_t kv_heads, int32_t head_size) {
    if (page_count <= 0 || kv_heads <= 0) return adapt(op, "dimensions must be positive.");
    if (page_size < 16 || page_size > 256 || (page_size & (page_size - 1)))
        return fail(SI_ERR_UNSUPPORTED, "%s: page sizes 16, 32, 64, 128 and 256 are supported, not %d.", op, page_size);
    if (head_size != 64 && head_size != 128 && head_size != 192 && head_size != 256)
        return fail(SI_ERR_UNSUPPORTED, "%s: head sizes 64, 128, 192 and 256 are supported, not %d.", op, head_size);
    if (page_count > INT32_MAX || kv_heads > 4096) return adapt(op, "cache too large.");
    return SI_OK;
}

uint64_t page_bytes(int32_t page_size, int32_t kv_heads, int32_t head_size) {
    return uint64_t(kv_heads) * uint64_t(page_size / 16) * 18u * uint64_t(head_size);
}

// Bytes that `rows` rows of `width` elements `stride` apart span.
uint64_t span(int64_t rows, int64_t stride, int64_t width, uint32_t size) {
    return (uint64_t(rows - 1) * uint64_t(stride) + uint64_t(width)) * size;
}

si_status cache_args(const char *op, const si_paged_cache *c, const int32_t *row_starts, const int32_t *lengths,
                     int64_t rows, PagedArgs *out) {
    if (!c) return fail(SI_ERR_INVALID_ARGUMENT, "%s: null cache", op);
    if (si_status st = cache_geometry(op, c->page_count, c->page_size, c->kv_heads, c->head_size)) return st;
    if (c->streams <= 0 || c->table_width <= 0 || rows <= 0) return adapt(op, "dimensions must be positive.");
    if (int64_t(c->table_width) * c->page_size > INT32_MAX || rows > INT32_MAX)
        return adapt(op, "more than 2^31 - 1 tokens.");
    int shift = 4;
    while ((16 << (shift - 4)) < c->page_size) ++shift;
    *out = PagedArgs{static_cast<uint8_t *>(c->pages), c->page_table, row_starts, lengths, c->page_count, rows,
                     c->streams, c->table_width, shift, c->kv_heads, c->head_size};
    return SI_OK;
}

si_status rows_of_streams(const char *op, const PagedArgs &a) {
    if (!a.row_starts && a.rows != a.streams) return adapt(op, "without row_starts there is one row per stream.");
    return SI_OK;
}

si_status cache_ports(const si_paged_cache *c, const PagedArgs &a) {
    if (a.row_starts)
        if (si_status st = ports({{"row_starts", a.row_starts, uint64_t(a.streams + 1) * 4, 4}})) return st;
    return ports({{"pages", a.pages, page_bytes(c->page_size, a.kv_heads, a.head_size) * uint64_t(a.page_count), 16},
                  {"page_table", a.page_table, uint64_t(a.streams) * uint64_t(a.table_width) * 4, 4},
                  {"lengths", a.lengths, uint64_t(a.streams) * 4, 4}});
}

// A written tensor against the cache and the row descriptors.
si_status apart_from_cache(const Port &written, const si_paged_cache *c, const PagedArgs &a) {
    return apart(written,
                 {{"pages", a.pages, page_bytes(c->page_size, a.kv_heads, a.head_size) * uint64_t(a.page_count), 16},
                  {"page_table", a.page_table, uint64_t(a.streams) * uint64_t(a.table_width) * 4, 4},
                  {"row_starts", a.row_starts, uint64_t(a.streams + 1) * 4, 4},
                  {"lengths", a.lengths, uint64_t(a.streams) * 4, 4}});
}

si_status attention_shape(const char *op, const PagedArgs &a, int32_t max_rows, int32_t query_heads) {
    if (query_heads <= 0 || max_rows <= 0) return adapt(op, "dimensions must be positive.");
    if (query_heads % a.kv_heads) return adapt(op, "Query heads must be divisible by key/value heads.");
    if (a.rows * query_heads > INT32_MAX / 2) return fail(SI_ERR_UNSUPPORTED, "%s: too many rows.", op);
    return SI_OK;
}

}  // namespace

extern "C" {

si_status si_paged_cache_bytes(int64_t page_count, int32_t page_size, int32_t kv_heads, int32_t head_size,
                               uint64_t *bytes) {
    if (!bytes) return fail(SI_ERR_INVALID_ARGUMENT, "null argument");
    if (si_status st = cache_geometry("paged-cache", page_count, page_size, kv_heads, head_size)) return st;
    *bytes = page_bytes(page_size, kv_heads, head_size) * uint64_t(page_count);
    return SI_OK;
}

si_status si_paged_rope_kv_append(const si_paged_cache *cache, uint32_t type, const void *qkv, int64_t qkv_stride,
                                  const int32_t *row_starts, const int32_t *lengths, const float *frequencies,
                                  void *query, int64_t query_stride, int64_t rows, int32_t query_heads,
                                  int32_t rotary_size, float rope_scale, void *stream) {
    const char *op = "paged-rope-kv-append";
    uint32_t size = 0;
    PagedArgs a;
    if (si_status st = tensor_type(op, type, &size)) return st;
    if (si_status st = cache_args(op, cache, row_starts, lengths, rows, &a)) return st;
    if (si_status st = rows_of_streams(op, a)) return st;
    if (si_status st = attention_shape(op, a, 1, query_heads)) return st;
    if (rotary_size < 0 || rotary_size > a.head_size || rotary_size % 2)
        return adapt(op, "Invalid query, cache, head, or rotary dimensions.");
    if (!std::isfinite(rope_scale) || rope_scale <= 0.0f)
        return adapt(op, "Attribute 'rope_scale' must be finite and positive.");
    const int64_t q = int64_t(query_heads) * a.head_size, width = q + 2 * int64_t(a.kv_heads) * a.head_size;
    if (qkv_stride < width || query_stride < q) return adapt(op, "a row stride is shorter than its row.");
    if (qkv_stride > INT32_MAX || query_stride > INT32_MAX) return adapt(op, "a row stride is too large.");
    const uint64_t in = span(rows, qkv_stride, width, size), out = span(rows, query_stride, q, size);
    if (ranges_overlap(query, out, qkv, in)) return fail(SI_ERR_UNSUPPORTED, "%s: output aliases an input.", op);
    if (si_status st = apart_from_cache({"query", query, out, size}, cache, a)) return st;
    if (si_status st = apart({"query", query, out, size}, {{"frequencies", frequencies, uint64_t(rotary_size / 2) * 4, 4}}))
        return st;
    if (si_status st = apart({"pages", a.pages, page_bytes(cache->page_size, a.kv_heads, a.head_size) * uint64_t(a.page_count), 16},
                             {{"qkv", qkv, in, size}}))
        return st;
    if (si_status st = cache_ports(cache, a)) return st;
    if (si_status st = ports({{"qkv", qkv, in, size}, {"query", query, out, size}})) return st;
    if (rotary_size)
        if (si_status st = ports({{"frequencies", frequencies, uint64_t(rotary_size / 2) * 4, 4}})) return st;
    return kernels::paged_append(a, type, qkv, qkv_stride, frequencies, query, query_stride, query_heads, rotary_size,
                                 rope_scale, stream);
}

si_status si_paged_kv_gather(const si_paged_cache *cache, uint32_t type, const int32_t *row_starts,
                             const int32_t *lengths, void *keys, void *values, int64_t rows, void *stream) {
    const char *op = "paged-kv-gather";
    uint32_t size = 0;
    PagedArgs a;
    if (si_status st = tensor_type(op, type, &size)) return st;
    if (si_status st = cache_args(op, cache, row_starts, lengths, rows, &a)) return st;
    if (si_status st = rows_of_streams(op, a)) return st;
    const uint64_t bytes = uint64_t(rows) * a.kv_heads * a.head_size * size;
    if (ranges_overlap(keys, bytes, values, bytes)) return fail(SI_ERR_UNSUPPORTED, "%s: outputs overlap.", op);
    if (si_status st = apart_from_cache({"keys", keys, bytes, size}, cache, a)) return st;
    if (si_status st = apart_from_cache({"values", values, bytes, size}, cache, a)) return st;
    if (si_status st = cache_ports(cache, a)) return st;
    if (si_status st = ports({{"keys", keys, bytes, size}, {"values", values, bytes, size}})) return st;
    return kernels::paged_gather(a, type, keys, values, stream);
}

si_status si_paged_attention_workspace_bytes(const si_paged_cache *cache, int64_t rows, int32_t max_rows,
                                             int32_t query_heads, uint64_t *bytes) {
    const char *op = "paged-attention";
    if (!bytes) return fail(SI_ERR_INVALID_ARGUMENT, "null argument");
    PagedArgs a;
    if (si_status st = cache_args(op, cache, nullptr, nullptr, rows, &a)) return st;
    if (si_status st = attention_shape(op, a, max_rows, query_heads)) return st;
    *bytes = kernels::paged_attention_workspace(a, rows, max_rows, query_heads);
    return SI_OK;
}

si_status si_paged_attention(const si_paged_cache *cache, uint32_t type, const void *query, int64_t query_stride,
                             const int32_t *row_starts, const int32_t *lengths, void *output, int64_t output_stride,
                             int64_t rows, int32_t max_rows, int32_t query_heads, float scale, int32_t window,
                             void *workspace, uint64_t workspace_bytes, void *stream) {
    const char *op = "paged-attention";
    uint32_t size = 0;
    PagedArgs a;
    if (si_status st = tensor_type(op, type, &size)) return st;
    if (si_status st = cache_args(op, cache, row_starts, lengths, rows, &a)) return st;
    if (si_status st = rows_of_streams(op, a)) return st;
    if (si_status st = attention_shape(op, a, max_rows, query_heads)) return st;
    if (!std::isfinite(scale) || scale <= 0.0f) return adapt(op, "Attribute 'scale' must be finite and positive.");
    if (window < 0) return adapt(op, "Attribute 'window' must be non-negative.");
    const int64_t width = int64_t(query_heads) * a.head_size;
    if (query_stride < width || output_stride < width) return adapt(op, "a row stride is shorter than its row.");
    if (query_stride > INT32_MAX || output_stride > INT32_MAX) return adapt(op, "a row stride is too large.");
    const uint64_t need = kernels::paged_attention_workspace(a, rows, max_rows, query_heads);
    if (workspace_bytes < need)
        return fail(SI_ERR_INVALID_ARGUMENT, "%s: workspace of %llu bytes, %llu required", op,
                    (unsigned long long)workspace_bytes, (unsigned long long)need);
    const uint64_t in = span(rows, query_stride, width, size), out = span(rows, output_stride, width, size);
    if (ranges_overlap(output, out, query, in) || (need && ranges_overlap(output, out, workspace, need)))
        return fail(SI_ERR_UNSUPPORTED, "%s: output aliases an input.", op);
    if (si_status st = apart_from_cache({"output", output, out, size}, cache, a)) return st;
    if (si_status st = apart_from_cache({"workspace", workspace, need, 16}, cache, a)) return st;
    if (si_status st = apart({"workspace", workspace, need, 16}, {{"query", query, in, size}})) return st;
    if (si_status st = cache_ports(cache, a)) return st;
    if (si_status st = ports({{"query", query, in, size}, {"output", output, out, size}})) return st;
    if (need)
        if (si_status st = ports({{"workspace", workspace, need, 16}})) return st;
    const kernels::PagedAttention q{query,       output,   query_stride, output_stride, query_heads,
                                    max_rows,    window,   scale,        workspace};
    return kernels::paged_attention(a, type, q, stream);
}

si_status si_process_logits(uint32_t type, const void *logits, int64_t logits_stride, const si_logit_controls *controls,
                            void *output, int64_t output_stride, int32_t *next_token, int64_t rows, int64_t vocab,
                            void *stream) {
    const char *op = "process-logits";
    uint32_t size = 0;
    if (si_status st = tensor_type(op, type, &size)) return st;
    if (rows <= 0 || vocab <= 0) return adapt(op, "dimensions must be positive.");
    if (vocab > INT32_MAX / 2 || rows > INT32_MAX / 64) return fail(SI_ERR_UNSUPPORTED, "%s: too many logits.", op);
    if (!controls) return fail(SI_ERR_INVALID_ARGUMENT, "%s: null controls", op);
    if (!output && !next_token) return fail(SI_ERR_INVALID_ARGUMENT, "%s: neither output nor next_token", op);
    if (logits_stride < vocab || (output && output_stride < vocab))
        return adapt(op, "a row stride is shorter than its row.");
    if (logits_stride > INT32_MAX || output_stride > INT32_MAX) return adapt(op, "a row stride is too large.");
    si_logit_controls c = *controls;
    // an empty list is an absent one: the kernel takes a list's starts where its tokens are given, and only those of
    // a list that is not empty are checked below
    if (!c.history_count) c.history = c.history_starts = nullptr;
    if (!c.bias_count) c.bias_tokens = c.bias_starts = nullptr;
    const uint64_t in = span(rows, logits_stride, vocab, size);
    if (si_status st = ports({{"logits", logits, in, size}})) return st;
    if (output) {
        const uint64_t out = span(rows, output_stride, vocab, size);
        if (!(output == logits && output_stride == logits_stride) && ranges_overlap(output, out, logits, in))
            return fail(SI_ERR_UNSUPPORTED, "%s: output aliases an input.", op);
        if (si_status st = ports({{"output", output, out, size}})) return st;
    }
    const uint64_t starts = uint64_t(rows + 1) * 4, per_row = uint64_t(rows) * 4;
    if (next_token)
        if (si_status st = ports({{"next_token", next_token, per_row, 4}})) return st;
    if (c.history_count < 0 || c.bias_count < 0 || c.history_count > INT32_MAX || c.bias_count > INT32_MAX)
        return adapt(op, "list lengths must be 0 .. 2^31 - 1.");
    if (c.history)
        if (si_status st = ports({{"history", c.history, uint64_t(c.history_count) * 4, 4},
                                  {"history_starts", c.history_starts, starts, 4}}))
            return st;
    if (c.repetition)
        if (si_status st = ports({{"repetition", c.repetition, per_row, 4}})) return st;
    if (c.frequency)
        if (si_status st = ports({{"frequency", c.frequency, per_row, 4}})) return st;
    if (c.presence)
        if (si_status st = ports({{"presence", c.presence, per_row, 4}})) return st;
    if (c.bias_tokens)
        if (si_status st = ports({{"bias_tokens", c.bias_tokens, uint64_t(c.bias_count) * 4, 4},
                                  {"bias_values", c.bias_values, uint64_t(c.bias_count) * 4, 4},
                                  {"bias_starts", c.bias_starts, starts, 4}}))
            return st;
    if (c.allowed) {
        if (c.allowed_rows <= 0 || c.allowed_stride < (vocab + 31) / 32 || c.allowed_stride > INT32_MAX)
            return adapt(op, "the token mask has fewer words than the vocabulary.");
        if (!c.allowed_index && c.allowed_rows < rows) return adapt(op, "the token mask has fewer rows than the logits.");
        if (si_status st = ports({{"allowed", c.allowed,
                                   span(c.allowed_rows, c.allowed_stride, (vocab + 31) / 32, 4), 4}}))
            return st;
        if (c.allowed_index)
            if (si_status st = ports({{"allowed_index", c.allowed_index, per_row, 4}})) return st;
    }
    return kernels::process_logits(type, logits, logits_stride, c, output, output_stride, next_token, rows, vocab,
                                   stream);
}

}  // extern "C"
