// A cache in pages: where a request's tokens stand.
#pragma once
#include "mam_types.h"

namespace mam {

// Pages of `S` tokens, a multiple of 16: keys (P, Hkv, S, 2, d), values (P, Hkv, S, dv), contiguous, so that a head's tokens of a page follow each other.
struct Pages {
    void *k, *v;
    const int32_t *table, *lengths, *counts;
    int P, S, Hkv, d, dv, B, slots;
};

int fill_pages(const mam_pages_t *a, Pages &p);

// What a table, its lengths and counts say is taken with care: none of it leads out of the pages.
__device__ __forceinline__ int length_of(const Pages &p, int b)
{
    const int n = p.lengths[b];
    const int64_t most = (int64_t)p.slots * p.S;
    return n < 0 ? 0 : n < most ? n : (int)most;
}

// Tokens of `n` new ones that request b has.
__device__ __forceinline__ int count_of(const Pages &p, int b, int n)
{
    if (!p.counts) return n;
    const int c = p.counts[b];
    return c < 0 ? 0 : c < n ? c : n;
}

// Row (page * Hkv) * S + token of the page of token `at` in the first key head's pages; a head is S rows on.  -1: the request has no page there.
__device__ __forceinline__ int64_t row_of(const Pages &p, int b, uint32_t at)
{
    const uint32_t slot = at / (uint32_t)p.S;
    if (slot >= (uint32_t)p.slots) return -1;
    const int page = p.table[(int64_t)b * p.slots + slot];
    return page < 0 || page >= p.P ? -1 : (int64_t)page * p.Hkv * p.S + (int64_t)(at - slot * (uint32_t)p.S);
}

}  // namespace mam
