// Differential attention over the pages of a cache: single tokens, trees of drafted tokens, chunks of a prompt behind what a request has.
//
// Few rows are bound by reading K and V once.  A wave takes 16 rows (queries times the heads that share a key head) and a range of the keys, 32 at a time, straight from
// the pages as the fragments of both products (as mam_attention_split.hip does from dense keys); no wave waits for another.  A page's size is a multiple of 16 tokens, so the
// 16 keys of a fragment stand in one page, and what a tile of 32 needs of the table is two numbers that all its lanes share: a wave keeps 64 entries of the table in a
// register, an entry a lane.
//
// All tokens of the cache are seen by every row; of the new ones a row sees those that its mask names, or those up to itself.  So only the last tiles are limited.
#include "mam_attention.h"
#include "mam_pages.h"

namespace mam {
namespace attention {

constexpr int ROWS = 16;                // rows of a wave
#ifndef FEWROWS
#define FEWROWS 16
#endif
constexpr int FEW = FEWROWS;

// A request's table, walked in steps of 16 tokens.
struct Walk {
    const int32_t *row;
    int slots, P, S, Hkv, hk;
    int base, ids;                      // 64 entries from `base` on, one a lane
    int slot, off;

    __device__ __forceinline__ Walk(const Pages &p, int b, int head, int key)
        : row(p.table + (int64_t)b * p.slots), slots(p.slots), P(p.P), S(p.S), Hkv(p.Hkv), hk(head), base(0), ids(-1)
    {
        slot = key / S;
        off = key - slot * S;
        read();
    }
    __device__ __forceinline__ void read()
    {
        base = slot;
        const int mine = slot + (threadIdx.x & 63);
        ids = mine < slots ? row[mine] : -1;
    }
    // Row of the pages where the next 16 tokens begin, -1 where the request has none.
    __device__ __forceinline__ int64_t next()
    {
        if (slot - base >= 64) read();
        const int page = __builtin_amdgcn_readlane(ids, slot - base);
        const int64_t r = page < 0 || page >= P ? -1 : ((int64_t)page * Hkv + hk) * S + off;
        off += 16;
        if (off == S) {
            off = 0;
            ++slot;
        }
        return r;
    }
};

// Bits of the keys key .. key + 31 that a row sees: all of the cache's `length`, then those that `mask` names.
__device__ __forceinline__ uint32_t seen_word(int key, int length, uint64_t mask)
{
    const int behind = key - length;
    if (behind >= 64) return 0;
    if (behind >= 0) return (uint32_t)(mask >> behind);
    if (behind <= -32) return 0xffffffffu;
    return ((1u << -behind) - 1) | (uint32_t)(mask << -behind);
}

template <class T, int PE, bool FAST>
__device__ __forceinline__ void page_piece(const T *base, uint32_t offset, bool in, int left, uint32_t *w)
{
    constexpr int BYTES = PE * (int)sizeof(T);
    if constexpr (FAST) {
        const auto rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<T *>(base), 0, 0x7fffffff, 0x00027000);
        const int at = (int)(in ? offset * (uint32_t)sizeof(T) : NOWHERE);
        if constexpr (BYTES == 16) {
            typedef uint32_t words __attribute__((ext_vector_type(4)));
            const words t = __builtin_amdgcn_raw_buffer_load_b128(rsrc, at, 0, 0);
#pragma unroll
            for (int u = 0; u < 4; ++u) w[u] = t[u];
        } else {
            typedef uint32_t words __attribute__((ext_vector_type(2)));
            const words t = __builtin_amdgcn_raw_buffer_load_b64(rsrc, at, 0, 0);
#pragma unroll
            for (int u = 0; u < 2; ++u) w[u] = t[u];
        }
    } else {
        T e[PE];
#pragma unroll
        for (int u = 0; u < PE; ++u) e[u] = in && u < left ? base[offset + u] : (T)0.0f;
        __builtin_memcpy(w, e, BYTES);
    }
}

template <class T, int D, int DV, bool FAST>
__global__ __launch_bounds__(256, D > 64 || (sizeof(T) == 4 && DV > 64) ? 1 : 2) void pages_kernel(const Call a, const Pages p, const int64_t *__restrict__ masks,
                                                                                                  void *out, float *partial, int splits, int row_tiles)
{
    constexpr int TR = ROWS, NK = D / KS<T, TR>, E = DV / 16;           // E: elements of a lane's values
    constexpr int PE = E < FE<T> ? E : FE<T>, PIECES = E / PE, WORDS = E * (int)sizeof(T) / 4, PW = PE * (int)sizeof(T) / 4;
    constexpr int PARTS = sizeof(T) == 2 ? 2 : 1;
    // Values are asked for at the head of a turn and the next keys before the softmax, where both fit the registers beside the products.
    constexpr bool EARLY = sizeof(T) == 2 || D <= 64;
    __shared__ float joined[2][ROWS][DV + 4];
    __shared__ float tops[2][4][ROWS], sums[2][4][ROWS];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), heads = a.B * a.Hkv;
    const int bh = blockIdx.x % heads, rest_id = blockIdx.x / heads, tile = rest_id % row_tiles, split = rest_id / row_tiles;
    const int b = bh / a.Hkv, hk = bh % a.Hkv;
    const int length = length_of(p, b), count = count_of(p, b, a.Lq), room = p.slots * p.S;
    const int row = tile * ROWS + lane_row<TR>();
    const int query = row < a.R ? row / a.G : 0;
    const bool there = row < a.R && query < count;
    const uint64_t mask = masks && there ? (uint64_t)masks[(int64_t)b * a.Lq + query] : 0;
    const int limit = there ? length + (masks ? count : query + 1) : 0;
    const int last_row = tile * ROWS + ROWS - 1 < a.R ? tile * ROWS + ROWS - 1 : a.R - 1, last = last_row / a.G;
    int any = length + (masks || last + 1 > count ? count : last + 1);
    if (any > room) any = room;
    if (tile * ROWS / a.G >= count) any = 0;
    // this wave's keys: whole tiles of 32, as even as they come
    const int per = ((any + 31) / 32 + 4 * splits - 1) / (4 * splits) * 32;
    const int64_t begin64 = (int64_t)per * (split * 4 + wave);
    const int begin = begin64 < any ? (int)begin64 : any, end = begin64 + per < any ? (int)(begin64 + per) : any;

    const Source<T> qs{static_cast<const T *>(a.q) + b * a.qb + (int64_t)hk * a.G * a.qh, a.ql, a.qh, a.qm, a.G, a.d, a.inverse};
    const T *keys = static_cast<const T *>(p.k), *values = static_cast<const T *>(p.v);
    const int lane = lane_row<TR>(), group = lane_group<TR>();
    Frag<T> q[2][NK];
#pragma unroll
    for (int m = 0; m < 2; ++m) load_rows<T, TR, D>(qs, row, there, m, q[m]);
    const float c = a.scale * LOG2E;

    Walk walk(p, b, hk, begin);
    int64_t rows[2], next_rows[2];
    Frag<T> k[2][BLOCKS<TR>][NK];
    const auto load_keys = [&](int first, const int64_t (&r)[2]) {
#pragma unroll
        for (int blk = 0; blk < BLOCKS<TR>; ++blk) {
            const T *base = keys + (r[blk] < 0 ? 0 : r[blk]) * (2 * a.d);
            const bool ok = r[blk] >= 0 && first + blk * TR + lane < end;
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int kk = 0; kk < NK; ++kk) {
                    const int col = kk * KS<T, TR> + FE<T> * group;
                    const uint32_t off = (uint32_t)lane * (uint32_t)(2 * a.d) + (uint32_t)(m * a.d + col);
                    if constexpr (FAST) {
                        k[m][blk][kk] = buffer_frag<T>(base, ok && col < a.d ? off * (uint32_t)sizeof(T) : NOWHERE);
                    } else {
#pragma unroll
                        for (int u = 0; u < FE<T>; ++u) k[m][blk][kk][u] = (T)0.0f;
                        if (ok && col < a.d) k[m][blk][kk] = load_frag<T>(base + off, a.d - col);
                    }
                }
        }
    };
    uint32_t v[REGS<TR>][WORDS];
    const auto load_values = [&](int first, const int64_t (&r)[2]) {
#pragma unroll
        for (int f = 0; f < REGS<TR>; ++f) {
            const T *base = values + (r[f / 4] < 0 ? 0 : r[f / 4]) * a.dv;
            const int at = 4 * group + f % 4;
            const bool ok = r[f / 4] >= 0 && first + index_of<TR>(f) < end;
#pragma unroll
            for (int n = 0; n < PIECES; ++n) {
                const int col = E * lane + n * PE;
                page_piece<T, PE, FAST>(base, (uint32_t)at * (uint32_t)a.dv + (uint32_t)col, ok && col < a.dv, a.dv - col, &v[f][n * PW]);
            }
        }
    };

    Acc<TR> o[2][E];
    float top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.0f, 0.0f};
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int j = 0; j < E; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[m][j][i] = 0.0f;
    if (begin < end) {
        rows[0] = walk.next();
        rows[1] = walk.next();
        load_keys(begin, rows);
    }
    for (int key = begin; key < end; key += 32) {
        if (EARLY) load_values(key, rows);
        Acc<TR> s[2][BLOCKS<TR>];
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int blk = 0; blk < BLOCKS<TR>; ++blk) {
#pragma unroll
                for (int i = 0; i < 4; ++i) s[m][blk][i] = 0.0f;
#pragma unroll
                for (int kk = 0; kk < NK; ++kk) mma<TR>(k[m][blk][kk], q[m][kk], s[m][blk]);
            }
        const bool pages = rows[0] >= 0 && rows[1] >= 0;
        if (key + 32 < end) {
            next_rows[0] = walk.next();
            next_rows[1] = walk.next();
        } else {                // past the range: nothing
            next_rows[0] = next_rows[1] = -1;
        }
        if (EARLY) load_keys(key + 32, next_rows);
        else load_values(key, rows);
        const bool limited = key + 32 > length || key + 32 > end || !pages;
        uint32_t word = 0xffffffffu;
        if (limited) word = (masks ? seen_word(key, length, mask) : 0xffffffffu) & ((rows[0] < 0 ? 0u : 0xffffu) | (rows[1] < 0 ? 0u : 0xffff0000u));
        const int most_keys = (limit < end ? limit : end) - key;
        Frag<T> frag[2][FRAGS<T, TR>], rest[FRAGS<T, TR>];
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            float x[REGS<TR>], most = -INFINITY;
#pragma unroll
            for (int f = 0; f < REGS<TR>; ++f) {
                x[f] = s[m][f / 4][f % 4];
                if (limited) {
                    const int at = index_of<TR>(f);
                    x[f] = at < most_keys && (word >> at & 1) ? x[f] : -INFINITY;
                }
                most = fmaxf(most, x[f]);
            }
            most = groups_max<TR>(most) * c;
            if (__any(most > top[m] + SLACK)) {
                asm volatile("; a new maximum");
                const float rise = fmaxf(top[m], most), factor = rise == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(top[m] - rise);
                top[m] = rise;
                sum[m] *= factor;
#pragma unroll
                for (int j = 0; j < E; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[m][j][i] *= factor;
            }
            const float base = top[m] == -INFINITY ? 0.0f : top[m];
#pragma unroll
            for (int f = 0; f < REGS<TR>; ++f) {
                x[f] = __builtin_amdgcn_exp2f(fmaf(x[f], c, -base));
                sum[m] += x[f];
            }
            to_frags<T, TR>(x, frag[m]);
            // what 16 bits leave of the first map's probabilities, as a product of its own (see mam_attention_split.hip)
            if (PARTS == 2 && m == 0) {
#pragma unroll
                for (int f = 0; f < REGS<TR>; ++f) x[f] -= element(frag[0][f / FE<T>], f % FE<T>);
                to_frags<T, TR>(x, rest);
            }
        }
#pragma unroll
        for (int j = 0; j < E; ++j) {
            if constexpr (PARTS == 2) {
                typedef uint32_t words __attribute__((ext_vector_type(4)));
                words w;
#pragma unroll
                for (int u = 0; u < 4; ++u) w[u] = __builtin_amdgcn_perm(v[2 * u + 1][j / 2], v[2 * u][j / 2], j % 2 ? 0x07060302u : 0x05040100u);
                const Frag<T> value = __builtin_bit_cast(Frag<T>, w);
                mma<TR>(value, frag[0][0], o[0][j]);
                mma<TR>(value, frag[1][0], o[1][j]);
                mma<TR>(value, rest[0], o[0][j]);
            } else {
#pragma unroll
                for (int n = 0; n < FRAGS<T, TR>; ++n) {
                    Frag<T> value;
#pragma unroll
                    for (int u = 0; u < FE<T>; ++u) value[u] = __builtin_bit_cast(float, v[n * FE<T> + u][j]);
                    mma<TR>(value, frag[0][n], o[0][j]);
                    mma<TR>(value, frag[1][n], o[1][j]);
                }
            }
        }
        if (!EARLY) load_keys(key + 32, next_rows);
        rows[0] = next_rows[0];
        rows[1] = next_rows[1];
    }

    // the four waves' ranges; a row that is no query's has seen nothing
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        sum[m] = there ? groups_sum<TR>(sum[m]) : 0.0f;
        if (!there) top[m] = -INFINITY;
        if (group == 0) {
            tops[m][wave][lane] = top[m];
            sums[m][wave][lane] = sum[m];
        }
    }
    __syncthreads();
    // A range of which a row sees nothing has a sum of 0, and its products do not count whatever the values there hold.  Scores that are all NaN leave
    // the maximum at -inf too, but not the sum: they go on as NaN.
    float most[2];
#pragma unroll
    for (int m = 0; m < 2; ++m) most[m] = fmaxf(fmaxf(tops[m][0][lane], tops[m][1][lane]), fmaxf(tops[m][2][lane], tops[m][3][lane]));
    for (int w = 0; w < 4; ++w) {
        if (w == wave) {
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                const float factor = __builtin_amdgcn_exp2f(top[m] - most[m]);
#pragma unroll
                for (int j = 0; j < E; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float &cell = joined[m][lane][E * (4 * group + i) + j];
                        const float part = sum[m] == 0.0f ? 0.0f : o[m][j][i] * factor;
                        cell = w ? cell + part : part;
                    }
            }
        }
        __syncthreads();
    }
    // 16 threads a row write it
    const int mine = threadIdx.x / 16, place = threadIdx.x % 16, out_row = tile * ROWS + mine;
    if (out_row >= a.R) return;
    float m_top[2], m_sum[2];
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        m_top[m] = fmaxf(fmaxf(tops[m][0][mine], tops[m][1][mine]), fmaxf(tops[m][2][mine], tops[m][3][mine]));
        m_sum[m] = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) m_sum[m] += sums[m][w][mine] == 0.0f ? 0.0f : sums[m][w][mine] * __builtin_amdgcn_exp2f(tops[m][w][mine] - m_top[m]);
    }
    if (splits == 1) {
        const int i = out_row / a.G, h = hk * a.G + out_row - i * a.G;
        const float lam = lambda_of(a, h, static_cast<const T *>(nullptr));
        const float inv[2] = {m_sum[0] > 0.0f ? 1.0f / m_sum[0] : 0.0f, m_sum[1] > 0.0f ? 1.0f / m_sum[1] : 0.0f};
        T *to = static_cast<T *>(out) + (((int64_t)b * a.Lq + i) * a.H + h) * a.dv;
        for (int col = 4 * place; col < a.dv; col += 64) {
            float r[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) r[u] = fmaf(-lam, joined[1][mine][col + u] * inv[1], joined[0][mine][col + u] * inv[0]);
            store_pack<T, 4>(to + col, a.dv - col, r);
        }
    } else {
        float *to = partial + (((int64_t)split * a.B * a.Hkv + bh) * a.R + out_row) * (2 * (int64_t)a.dv + 4);
        for (int m = 0; m < 2; ++m)
            for (int col = place; col < a.dv; col += 16) to[m * a.dv + col] = joined[m][mine][col];
        if (place < 2) {
            to[2 * a.dv + 2 * place] = m_top[place];
            to[2 * a.dv + 2 * place + 1] = m_sum[place];
        }
    }
}

// ---- more rows: tiles of keys in LDS ----
// Where a key head has more rows than a wave takes, every wave for itself reads K and V again from the L2: 128 rows a key head (trees of 32 tokens, four heads each) 99 us.  Here eight waves
// share them: four row groups of TR rows, and two halves of the workgroup's keys, each with a tile of 32 keys in LDS for its four waves.  The halves meet in LDS, the workgroups
// that share a row's keys in the workspace.
//
// ROWS16 rounded once: what 16 bits leave of the first map's probabilities is not kept here, as in mam_attention.hip's kernels for many rows; a product more for 0.0019 against 0.0024.

// 32 rows of MAPS segments of W elements between the pages and LDS by 256 threads (Stage, with 16 rows in a page each).
template <class T, int MAPS, int W, bool FAST>
struct PageStage {
    typedef Stage<T, 256, KT, MAPS, W, FAST> Dense;
    static constexpr int PITCH = Dense::PITCH, N = Dense::N, SEGMENT = Dense::SEGMENT, PER = Dense::PER;
    static_assert(64 / PER <= 16, "the rows of a wave's pieces stand in one page");
    Frag<T> piece[N];

    static __device__ __forceinline__ int thread() { return threadIdx.x & 255; }
    static __device__ __forceinline__ uint32_t first_of(int i) { return (i * 256 + (__builtin_amdgcn_readfirstlane(threadIdx.x >> 6) & 3) * 64u); }
    static __device__ __forceinline__ int map_of(int i) { return MAPS == 1 ? 0 : (int)(first_of(i) / SEGMENT); }
    static __device__ __forceinline__ int block_of(int i) { return (int)(first_of(i) % SEGMENT / PER / 16); }
    static __device__ __forceinline__ int row_of(int i) { return (int)((i * 256 + thread()) % SEGMENT / PER); }
    static __device__ __forceinline__ int column_of(int i) { return (int)((i * 256 + thread()) % SEGMENT % PER * FE<T>); }

    // row0, row1: where the two halves of 16 begin, -1: nowhere; left: how many of the 32 there are.  Others are zeros.
    __device__ __forceinline__ void load(const T *pool, int64_t row0, int64_t row1, int width, int left)
    {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int64_t begin = block_of(i) ? row1 : row0;
            const T *base = pool + (begin < 0 ? 0 : begin) * (MAPS * width) + map_of(i) * width;
            const bool ok = begin >= 0 && row_of(i) < left && column_of(i) < width;
            const uint32_t off = (uint32_t)(row_of(i) & 15) * (uint32_t)(MAPS * width) + (uint32_t)column_of(i);
            if constexpr (FAST) {
                piece[i] = buffer_frag<T>(base, ok ? off * (uint32_t)sizeof(T) : NOWHERE);
            } else {
#pragma unroll
                for (int u = 0; u < FE<T>; ++u) piece[i][u] = (T)0.0f;
                if (ok) piece[i] = load_frag<T>(base + off, width - column_of(i));
            }
        }
    }
    __device__ __forceinline__ void store(T *tile) const
    {
#pragma unroll
        for (int i = 0; i < N; ++i) *reinterpret_cast<Frag<T> *>(tile + place_of<T>(row_of(i)) * PITCH + map_of(i) * W + column_of(i)) = piece[i];
    }
};

constexpr int LDS_BYTES = 160 * 1024;
template <class T, int D, int DV>
constexpr int TILE_BYTES = KT * (2 * D + DV + 2 * FE<T>) * (int)sizeof(T);
// Tiles of a half of the workgroup: one is written while the other is read, where both fit.
template <class T, int D, int DV>
constexpr int PAGE_TILES = 4 * TILE_BYTES<T, D, DV> <= LDS_BYTES - 1024 ? 2 : 1;

template <class T, int TR, int D, int DV, bool FAST>
__global__ __launch_bounds__(512, 2) void page_tiles_kernel(const Call a, const Pages p, const int64_t *__restrict__ masks, void *out, float *partial,
                                                            int splits, int row_tiles)
{
    constexpr int BUFFERS = PAGE_TILES<T, D, DV>, AR = TR * TR / 64, ACC = DV / TR * AR;
    typedef PageStage<T, 2, D, FAST> StageK;
    typedef PageStage<T, 1, DV, FAST> StageV;
    constexpr int TILES_AT = 2 * BUFFERS * TILE_BYTES<T, D, DV>, JOIN_AT = 4 * 64 * ACC * 4;
    __shared__ __attribute__((aligned(16))) unsigned char lds[TILES_AT > JOIN_AT ? TILES_AT : JOIN_AT];
    __shared__ float tops[2][4][TR], sums[2][4][TR];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = wave >> 2, heads = a.B * a.Hkv;
    const int bh = blockIdx.x % heads, rest_id = blockIdx.x / heads, tile = row_tiles - 1 - rest_id % row_tiles, split = rest_id / row_tiles;
    const int b = bh / a.Hkv, hk = bh % a.Hkv;
    const int length = length_of(p, b), count = count_of(p, b, a.Lq), room = p.slots * p.S;
    const int first = tile * 4 * TR + (wave & 3) * TR, row = first + lane_row<TR>();
    const int query = row < a.R ? row / a.G : 0;
    const bool there = row < a.R && query < count;
    const uint64_t mask = masks && there ? (uint64_t)masks[(int64_t)b * a.Lq + query] : 0;
    const int limit = there ? length + (masks ? count : query + 1) : 0;
    // keys that rows up to `last` see at most: none where the first of them is no query
    const auto reach = [&](int from, int last) {
        const int q = (last < a.R ? last : a.R - 1) / a.G;
        const int n = length + (masks || q + 1 > count ? count : q + 1);
        return from >= a.R || from / a.G >= count ? 0 : n < room ? n : room;
    };
    const int wave_any = reach(first, first + TR - 1), any = reach(tile * 4 * TR, tile * 4 * TR + 4 * TR - 1);
    // and those that every row of the wave sees (rows that are none see what they like)
    const int wave_all = masks || wave_any == 0 ? length : length + first / a.G + 1;
    // the workgroup's tiles, and this half's
    const int tiles = (any + KT - 1) / KT, per = (tiles + splits - 1) / splits, from = split * per < tiles ? split * per : tiles;
    const int mine = from + per < tiles ? per : tiles - from, part = (mine + 1) / 2;
    const int begin = from + half * part, number = half ? mine - part : part;

    const Source<T> qs{static_cast<const T *>(a.q) + b * a.qb + (int64_t)hk * a.G * a.qh, a.ql, a.qh, a.qm, a.G, a.d, a.inverse};
    Frag<T> q[2][D / KS<T, TR>];
#pragma unroll
    for (int m = 0; m < 2; ++m) load_rows<T, TR, D>(qs, row, there, m, q[m]);
    const float c = a.scale * LOG2E;
    State<T, TR, D, DV, true> state;
    state.clear();

    T *k_tile = reinterpret_cast<T *>(lds + half * BUFFERS * TILE_BYTES<T, D, DV>), *v_tile = k_tile + KT * StageK::PITCH;
    constexpr int NEXT = TILE_BYTES<T, D, DV> / (int)sizeof(T);
    StageK k_stage;
    StageV v_stage;
    Walk walk(p, b, hk, begin * KT);
    uint32_t pages = 0, next_pages = 0;         // which halves of the tile have a page
    const auto load = [&](int t) {
        const int64_t row0 = walk.next(), row1 = walk.next();
        next_pages = (row0 < 0 ? 0u : 0xffffu) | (row1 < 0 ? 0u : 0xffff0000u);
        k_stage.load(static_cast<const T *>(p.k), row0, row1, a.d, any - t * KT);
        v_stage.load(static_cast<const T *>(p.v), row0, row1, a.dv, any - t * KT);
    };
    if (number > 0) {
        load(begin);
        if (BUFFERS == 2) {
            k_stage.store(k_tile);
            v_stage.store(v_tile);
        }
    }
    // A tile's part of the loop, with `use` what a wave does that sees some of its keys.  The first half has as many tiles as the second, or one more; waves that are past their
    // keys go on loading for the others, in a loop of its own (a condition around the products has the accumulators copied in every tile).
    int now = 0, i = 0;
    const auto tile_of = [&](const auto &use) {
        const bool more = i + 1 < number;
        if (BUFFERS == 1) {
            __syncthreads();
            if (i < number) {
                k_stage.store(k_tile);
                v_stage.store(v_tile);
            }
        }
        pages = next_pages;
        if (more) load(begin + i + 1);
        __syncthreads();
        use((begin + i) * KT, k_tile + now * NEXT, v_tile + now * NEXT);
        if (BUFFERS == 2) {
            now ^= 1;
            if (more) {         // the other tile: every wave is past it
                k_stage.store(k_tile + now * NEXT);
                v_stage.store(v_tile + now * NEXT);
            }
        }
        ++i;
    };
    const int open = (wave_all < wave_any ? wave_all : wave_any) / KT - begin, seen = (wave_any + KT - 1) / KT - begin;
    while (i < number && i < open && next_pages == 0xffffffffu)
        tile_of([&](int, const T *k, const T *v) { state.template keys<false, false>(q, k, StageK::PITCH, v, StageV::PITCH, c, 0, 0); });
    while (i < number && i < seen)
        tile_of([&](int key, const T *k, const T *v) {
            const uint32_t word = (masks ? seen_word(key, length, mask) : 0xffffffffu) & pages;
            state.template keys<true, false>(q, k, StageK::PITCH, v, StageV::PITCH, c, limit - key, word);
        });
    while (i < part) tile_of([](int, const T *, const T *) {});

    // the halves: the second one's sums, then its products map by map; a row that is no query's has seen nothing
    float factor[2], total[2];
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        total[m] = there ? groups_sum<TR>(state.sum[m]) : 0.0f;
        if (!there) state.top[m] = -INFINITY;
    }
    __syncthreads();
    if (half && lane_group<TR>() == 0) {
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            tops[m][wave & 3][lane_row<TR>()] = state.top[m];
            sums[m][wave & 3][lane_row<TR>()] = total[m];
        }
    }
    float *cells = reinterpret_cast<float *>(lds) + (wave & 3) * 64 * ACC + (threadIdx.x & 63);
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        if (m) __syncthreads();
        if (half) {
#pragma unroll
            for (int blk = 0; blk < DV / TR; ++blk)
#pragma unroll
                for (int f = 0; f < AR; ++f) cells[(blk * AR + f) * 64] = state.o[m][blk][f];
        }
        __syncthreads();
        if (!half) {
            // a range of which a row sees nothing has a sum of 0, and its products do not count whatever the values there hold
            const float top = tops[m][wave & 3][lane_row<TR>()], sum = sums[m][wave & 3][lane_row<TR>()], most = fmaxf(top, state.top[m]);
            const float old = total[m] == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(state.top[m] - most), more = sum == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(top - most);
#pragma unroll
            for (int blk = 0; blk < DV / TR; ++blk)
#pragma unroll
                for (int f = 0; f < AR; ++f) {
                    const float x = total[m] == 0.0f ? 0.0f : state.o[m][blk][f] * old, y = sum == 0.0f ? 0.0f : cells[(blk * AR + f) * 64] * more;
                    state.o[m][blk][f] = x + y;
                }
            total[m] = (total[m] == 0.0f ? 0.0f : total[m] * old) + (sum == 0.0f ? 0.0f : sum * more);
            state.top[m] = most;
        }
    }
    if (half || row >= a.R) return;
    if (splits == 1) {
        const int head = hk * a.G + row - query * a.G;
        const float lam = lambda_of(a, head, static_cast<const T *>(nullptr));
#pragma unroll
        for (int m = 0; m < 2; ++m) factor[m] = total[m] > 0.0f ? 1.0f / total[m] : 0.0f;
        T *to = static_cast<T *>(out) + (((int64_t)b * a.Lq + query) * a.H + head) * a.dv;
#pragma unroll
        for (int blk = 0; blk < DV / TR; ++blk)
#pragma unroll
            for (int f = 0; f < AR; f += 4) {
                const int col = blk * TR + (f / 4) * 4 * GROUPS<TR> + 4 * lane_group<TR>();
                if (col >= a.dv) continue;
                float r[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) r[u] = fmaf(-lam, state.o[1][blk][f + u] * factor[1], state.o[0][blk][f + u] * factor[0]);
                store_pack<T, 4>(to + col, a.dv - col, r);
            }
    } else {
        float *to = partial + (((int64_t)split * a.B * a.Hkv + bh) * a.R + row) * (2 * (int64_t)a.dv + 4);
#pragma unroll
        for (int m = 0; m < 2; ++m) {
#pragma unroll
            for (int blk = 0; blk < DV / TR; ++blk)
#pragma unroll
                for (int f = 0; f < AR; f += 4) {
                    const int col = blk * TR + (f / 4) * 4 * GROUPS<TR> + 4 * lane_group<TR>();
                    if (col >= a.dv) continue;
                    float r[4];
#pragma unroll
                    for (int u = 0; u < 4; ++u) r[u] = state.o[m][blk][f + u];
                    store_pack<float, 4>(to + m * a.dv + col, a.dv - col, r);
                }
            if (lane_group<TR>() == 0) {
                to[2 * a.dv + 2 * m] = state.top[m];
                to[2 * a.dv + 2 * m + 1] = total[m];
            }
        }
    }
}

// How a call runs: rows of a wave in tiles (0: streamed, 16 rows), workgroups that share a row's keys.
struct Plan { int tr, splits; };

// Rows of a wave's tile in LDS; streamed rows where a key head has few.
inline int tile_rows(const Call &a, int type)
{
    if (a.R <= FEW) return 0;
    return type == MAM_F32 || a.d > 64 || a.dv > 128 || a.R <= 64 ? 16 : 32;
}

// Workgroups that share a row's keys: two a CU over the whole call, but 64 keys a wave at least of what a request has room for; of the tiles' eight waves one a CU.
inline Plan plan_of(const Call &a, int type)
{
    Plan p{tile_rows(a, type), 1};
    const int64_t rows = (int64_t)a.B * a.Hkv * ceil_div(a.R, p.tr ? 4 * p.tr : ROWS), most = ceil_div(a.Lk, 4 * 64);
    int64_t n = p.tr ? kNumCU / (rows > 0 ? rows : 1) : ceil_div(2 * (int64_t)kNumCU, rows);
    if (n > 64) n = 64;
    if (n > most) n = most;
    p.splits = n < 1 ? 1 : (int)n;
    return p;
}

inline size_t pages_workspace(const Call &a, int type)
{
    const int n = plan_of(a, type).splits;
    return n > 1 ? (size_t)n * a.B * a.Hkv * a.R * partial_size(a) * sizeof(float) : 0;
}

template <class T>
struct PagesRun {
    const Call &a;
    const Pages &p;
    const int64_t *masks;
    void *out;
    float *partial;
    Plan plan;
    hipStream_t st;
    template <int D, int DV, int TR, bool FAST>
    void tiles(dim3 grid, int row_tiles) const
    {
        hipLaunchKernelGGL((page_tiles_kernel<T, TR, D, DV, FAST>), grid, dim3(512), 0, st, a, p, masks, out, partial, plan.splits, row_tiles);
    }
    template <int D, int DV>
    int operator()() const
    {
        const int64_t row_tiles = ceil_div(a.R, plan.tr ? 4 * plan.tr : ROWS), blocks = row_tiles * a.B * a.Hkv * plan.splits;
        if (blocks > INT32_MAX) return fail(MAM_ERR_UNSUPPORTED, "too many tiles");
        const dim3 grid((unsigned)blocks);
        if (plan.tr == 32) {
            if constexpr (sizeof(T) == 2 && D <= 64) {
                if (a.fast) tiles<D, DV, 32, true>(grid, (int)row_tiles);
                else tiles<D, DV, 32, false>(grid, (int)row_tiles);
            }
            return check_launch("attention::page_tiles_kernel");
        }
        if (plan.tr) {
            if (a.fast) tiles<D, DV, 16, true>(grid, (int)row_tiles);
            else tiles<D, DV, 16, false>(grid, (int)row_tiles);
            return check_launch("attention::page_tiles_kernel");
        }
        if (a.fast) hipLaunchKernelGGL((pages_kernel<T, D, DV, true>), grid, dim3(256), 0, st, a, p, masks, out, partial, plan.splits, (int)row_tiles);
        else hipLaunchKernelGGL((pages_kernel<T, D, DV, false>), grid, dim3(256), 0, st, a, p, masks, out, partial, plan.splits, (int)row_tiles);
        return check_launch("attention::pages_kernel");
    }
};

int fill_pages_call(const mam_diff_attention_pages_t *x, Call &c, Pages &p)
{
    if (!x) return fail(MAM_ERR_INVALID_ARGUMENT, "null pointer");
    const mam_pages_t &g = x->pages;
    int rc = fill_pages(&g, p);
    if (rc != MAM_OK) return rc;
    mam_diff_attention_t a{};
    a.q = x->q;
    a.lam = x->lam;
    for (int i = 0; i < 4; ++i) a.q_stride[i] = x->q_stride[i];
    a.B = g.B; a.Lq = x->N; a.Lk = g.slots * g.S; a.H = x->H; a.Hkv = g.Hkv; a.D = g.D; a.Dv = g.Dv;
    a.scale = x->scale;
    a.type = g.type;
    a.lam_type = x->lam_type;
    rc = fill_call(&a, c);
    if (rc != MAM_OK) return rc;
    if (x->masks && x->N > 64) return fail(MAM_ERR_UNSUPPORTED, "a tree has 64 tokens at most, got %lld", (long long)x->N);
    const int64_t pack = 16 / type_size(g.type);
    c.fast = g.D % pack == 0 && g.Dv % pack == 0;
    return MAM_OK;
}

}  // namespace attention
}  // namespace mam

extern "C" size_t mam_diff_attention_pages_workspace(const mam_diff_attention_pages_t *args)
{
    using namespace mam;
    attention::Call a;
    Pages p;
    if (attention::fill_pages_call(args, a, p) != MAM_OK || a.B == 0 || a.R == 0) return 0;
    return attention::pages_workspace(a, args->pages.type);
}

extern "C" int mam_diff_attention_pages(const mam_diff_attention_pages_t *args, void *out, void *workspace, size_t workspace_bytes, void *stream)
{
    using namespace mam;
    attention::Call a;
    Pages p;
    int rc = attention::fill_pages_call(args, a, p);
    if (rc != MAM_OK || a.B == 0 || a.R == 0) return rc;
    if (!a.q || !a.lam || !out || (p.P > 0 && (!p.k || !p.v))) return fail(MAM_ERR_INVALID_ARGUMENT, "null pointer");
    const size_t need = attention::pages_workspace(a, args->pages.type);
    if (need > 0 && (!workspace || workspace_bytes < need))
        return fail(MAM_ERR_WORKSPACE, "the attention needs %zu workspace bytes, got %zu", need, workspace ? workspace_bytes : (size_t)0);
    hipStream_t st = static_cast<hipStream_t>(stream);
    float *partial = need > 0 ? static_cast<float *>(workspace) : nullptr;
    const attention::Plan plan = attention::plan_of(a, args->pages.type);
    if (args->pages.type == MAM_F32) rc = attention::with_head_sizes(a.d, a.dv, attention::PagesRun<float>{a, p, args->masks, out, partial, plan, st});
    else if (args->pages.type == MAM_BF16) rc = attention::with_head_sizes(a.d, a.dv, attention::PagesRun<bf16>{a, p, args->masks, out, partial, plan, st});
    else rc = attention::with_head_sizes(a.d, a.dv, attention::PagesRun<f16>{a, p, args->masks, out, partial, plan, st});
    if (rc != MAM_OK || need == 0) return rc;
    return attention::join_parts(a, args->pages.type, out, partial, plan.splits, st);
}
