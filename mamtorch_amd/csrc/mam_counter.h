// Random words from counters: Philox4x32-10 (J. K. Salmon, M. A. Moraes, R. O. Dror, D. E. Shaw, "Parallel random numbers: as easy as
// 1, 2, 3", SC 2011).  Element i of a tensor takes word i % 4 of counter (i / 4, offset) under key seed and is kept where
// that word is at least p * 2^32, so that a mask is a function of (seed, offset, i) alone: it is never stored, and forward and
// backward form it again at whatever split of the tensor suits them.
#pragma once
#include "mam_common.h"

namespace mam {

struct Dropout {
    uint64_t seed, offset;      // key; high half of the counter
    const int64_t *step;        // device word added to offset, or NULL
    uint32_t least;             // smallest word that is kept
    float scale;                // what a kept element is multiplied by
    int none;                   // nothing is kept (p == 1, whose threshold does not fit a word)
};

// Checks `d` and fills `out`; MAM_OK or a negative code.
inline int make_dropout(const mam_dropout_t *d, Dropout &out)
{
    if (!d) return fail(MAM_ERR_INVALID_ARGUMENT, "null pointer");
    if (!(d->p >= 0.0 && d->p <= 1.0)) return fail(MAM_ERR_INVALID_ARGUMENT, "p must be between 0 and 1");
    const uint64_t least = (uint64_t)llrint(d->p * 4294967296.0);
    out.seed = d->seed;
    out.offset = d->offset;
    out.step = d->step;
    out.none = least > 0xffffffffull;
    out.least = out.none ? 0 : (uint32_t)least;
    out.scale = d->scale;
    return MAM_OK;
}

__device__ __forceinline__ uint64_t dropout_offset(const Dropout &d)
{
    return d.offset + (d.step ? (uint64_t)*d.step : 0);
}

// The four words of counter (group, offset).  Where `group_high` and `offset` are uniform, half of the first two rounds' products are
// the scalar unit's.
__device__ __forceinline__ void random_words(uint32_t group_low, uint32_t group_high, uint64_t offset, uint64_t seed, uint32_t (&w)[4])
{
    uint32_t c0 = group_low, c1 = group_high, c2 = (uint32_t)offset, c3 = (uint32_t)(offset >> 32);
    uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
        c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
        c1 = (uint32_t)b;
        c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
        c3 = (uint32_t)a;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    w[0] = c0; w[1] = c1; w[2] = c2; w[3] = c3;
}

// Factors of elements i .. i+N-1 (scale where kept, else 0).  Any i: the groups that the elements touch are formed once and turned
// to the first one in two steps.
template <int N>
__device__ __forceinline__ void keep_factors(const Dropout &d, uint64_t offset, uint64_t i, bool whole_groups, float (&f)[N])
{
    static_assert(N % 4 == 0, "whole groups");
    if (d.least == 0 && !d.none) {          // nothing is dropped: no words
#pragma unroll
        for (int u = 0; u < N; ++u) f[u] = d.scale;
        return;
    }
    uint32_t w[N + 4];
    const uint64_t g = i >> 2;
#pragma unroll
    for (int q = 0; q < N / 4; ++q) {
        uint32_t t[4];
        random_words((uint32_t)(g + q), (uint32_t)((g + q) >> 32), offset, d.seed, t);
#pragma unroll
        for (int u = 0; u < 4; ++u) w[4 * q + u] = t[u];
    }
    if (!whole_groups) {        // i % 4 may differ from 0
        uint32_t t[4];
        const uint64_t last = g + N / 4;
        random_words((uint32_t)last, (uint32_t)(last >> 32), offset, d.seed, t);
#pragma unroll
        for (int u = 0; u < 4; ++u) w[N + u] = t[u];
        const bool by2 = i & 2, by1 = i & 1;
#pragma unroll
        for (int u = 0; u < N + 2; ++u) w[u] = by2 ? w[u + 2] : w[u];
#pragma unroll
        for (int u = 0; u < N; ++u) w[u] = by1 ? w[u + 1] : w[u];
    }
#pragma unroll
    for (int u = 0; u < N; ++u) f[u] = (w[u] >= d.least && !d.none) ? d.scale : 0.0f;
}

// x * factor, where a dropped element is 0 whatever it holds.
__device__ __forceinline__ float keep_value(float x, float factor) { return factor == 0.0f ? 0.0f : x * factor; }

}  // namespace mam
