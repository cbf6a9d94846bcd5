// Whether strided tensors share memory, or repeat themselves: host only.
//
// Results that a launch writes may not be read or written by another of its threads.  Slices of one projection's output, or keys and values side by side
// in a page, lie between each other without meeting, so first and last bytes do not tell; the strides do.
#pragma once

#include <algorithm>
#include <initializer_list>
#include <stdint.h>

#include "hfrk_gfx950.h"

namespace hfrk {

// Runs of `run` bytes, one for each index of up to four dimensions of more than one element, the largest stride first.
struct Extent {
    struct Dim {
        int64_t size, stride;  // bytes
    };
    int64_t at = 0, run = 0;   // (run 0: nothing)
    int dims = 0;
    Dim dim[4];

    Extent(const void* p, int64_t run_bytes, std::initializer_list<Dim> of) : at((int64_t)reinterpret_cast<uintptr_t>(p)), run(run_bytes) {
        for (Dim d : of) {
            if (d.size < 1) run = 0;
            if (d.size <= 1) continue;
            if (d.stride < 0) {
                at += (d.size - 1) * d.stride;
                d.stride = -d.stride;
            }
            dim[dims++] = d;
        }
        std::sort(dim, dim + dims, [](const Dim& a, const Dim& b) { return a.stride > b.stride; });
    }
};

inline int64_t span(const Extent::Dim* d, int dims, int64_t run) {
    for (int i = 0; i < dims; ++i) run += (d[i].size - 1) * d[i].stride;
    return run;
}

// Whether two indices may name one byte: a stride smaller than what the smaller ones span.  (True for some that do not, whose strides interleave.)
inline bool repeats(const Extent& e) {
    int64_t inside = e.run;
    for (int i = e.dims; i-- > 0;) {
        if (e.dim[i].stride < inside) return e.run > 0;
        inside += (e.dim[i].size - 1) * e.dim[i].stride;
    }
    return false;
}

inline int64_t floor_div(int64_t a, int64_t b) { return a / b - (a % b < 0); }  // b > 0

// The same for a and b, which begins `ahead` bytes behind a.  The largest stride of either is taken out: by how many of its steps b's index is ahead of a's, for
// all steps that bring the rests together.  (True where these are too many to look at, which strides that lie within each other do not have.)
inline bool meets(const Extent::Dim* a, int a_dims, int64_t a_run, const Extent::Dim* b, int b_dims, int64_t b_run, int64_t ahead) {
    if (a_dims && a->stride == 0) a_dims = 0;  // (repeats its runs)
    if (b_dims && b->stride == 0) b_dims = 0;
    const int64_t a_span = span(a, a_dims, a_run), b_span = span(b, b_dims, b_run);
    if (ahead >= a_span || -ahead >= b_span) return false;
    if (!a_dims && !b_dims) return true;
    const int64_t stride = std::max(a_dims ? a->stride : 0, b_dims ? b->stride : 0);
    const bool of_a = a_dims && a->stride == stride, of_b = b_dims && b->stride == stride;
    const int64_t a_rest = a_span - (of_a ? (a->size - 1) * stride : 0), b_rest = b_span - (of_b ? (b->size - 1) * stride : 0);
    const int64_t first = std::max(of_a ? 1 - a->size : 0, -floor_div(b_rest + ahead - 1, stride));
    const int64_t last = std::min(of_b ? b->size - 1 : 0, floor_div(a_rest - ahead - 1, stride));
    if (last - first >= 16) return true;
    for (int64_t steps = first; steps <= last; ++steps)
        if (meets(a + of_a, a_dims - of_a, a_run, b + of_b, b_dims - of_b, b_run, ahead + steps * stride)) return true;
    return false;
}

inline bool meets(const Extent& a, const Extent& b) {
    return a.run > 0 && b.run > 0 && meets(a.dim, a.dims, a.run, b.dim, b.dims, b.run, b.at - a.at);
}

inline bool same(const Extent& a, const Extent& b) {
    return a.at == b.at && a.run == b.run && a.dims == b.dims &&
           std::equal(a.dim, a.dim + a.dims, b.dim, [](const Extent::Dim& x, const Extent::Dim& y) { return x.size == y.size && x.stride == y.stride; });
}

// What is wrong with the memory of an append's (or a rotation's) tensors, or nullptr.
inline const char* append_overlap(const hfrk_append_args& a) {
    const int64_t run = 2 * a.head_dim;
    auto heads = [&](const void* p, int64_t token_stride, int64_t head_stride, int n) {
        return Extent(p, n > 0 ? run : 0, {{a.tokens, 2 * token_stride}, {n, 2 * head_stride}});
    };
    const Extent query = heads(a.query, a.query_token_stride, a.query_head_stride, a.heads);
    const Extent output = heads(a.query_output, a.output_token_stride, a.output_head_stride, a.heads);
    if (repeats(output) || (!same(query, output) && meets(query, output))) return "the rotated heads' output must be the input itself or lie apart from it";
    if (a.kv_heads < 1) return nullptr;
    const Extent key = heads(a.key, a.key_token_stride, a.key_head_stride, a.kv_heads), value = heads(a.value, a.value_token_stride, a.value_head_stride, a.kv_heads);
    if (meets(output, key) || meets(output, value)) return "query_output must lie apart from key and value";
    const int64_t size = a.cache_dtype == HFRK_FP8_E4M3FN ? 1 : 2;
    auto cache = [&](const void* p, int64_t page, int64_t place, int64_t head) {
        return Extent(p, size * a.head_dim, {{a.pages, size * page}, {a.page_size, size * place}, {a.kv_heads, size * head}});
    };
    const Extent keys = cache(a.key_cache, a.key_page_stride, a.key_place_stride, a.key_cache_head_stride);
    const Extent values = cache(a.value_cache, a.value_page_stride, a.value_place_stride, a.value_cache_head_stride);
    for (const Extent* c : {&keys, &values})
        if (repeats(*c) || meets(*c, key) || meets(*c, value) || meets(*c, query) || meets(*c, output))
            return "the caches must lie apart from the step's tensors and not overlap themselves";
    return meets(keys, values) ? "key_cache and value_cache must not share the same memory" : nullptr;
}

}  // namespace hfrk
