// Differential attention over the pages of a cache: single tokens, trees of drafted tokens, chunks of a prompt behind what a request has.
//
// Few rows are bound by reading K and V once.  A wave takes 16 rows (queries times the heads that share a key head) and a range of the keys, 32 at a time, straight from
// the pages as the fragments of both products (as mam_attention_split.hip does from dense keys); no wave waits for another.  A page's size is a multiple of 16 tokens, so the
// 16 keys of a fragment stand in one page, and what a tile of 32 needs of the table is two numbers that all its lanes share: a wave keeps where 64 steps of 16 tokens stand in a
// register, a step a lane.
//
// Measured: 16 requests of up to 16384 tokens, 4 key heads of 64/128 for 16, bf16, one token each: 87 us with the join's 7, 4.7 TB/s (a copy reaches 5.4).
//
// All tokens of the cache are seen by every row; of the new ones a row sees those that its mask names, or those up to itself.  So only the last tiles are limited.
#include "mam_attention.h"
#include "mam_pages.h"

namespace mam {
namespace attention {
namespace {         // names of mam_attention_split.hip's own parts, for the paged ones

constexpr int ROWS = 16;                // rows of a wave

// A partial row: both maps' products relative to their maxima, then maximum and sum of each.
inline int64_t partial_size(const Call &a) { return 2 * (int64_t)a.dv + 4; }
// Rows of a key head that are streamed; more share tiles of keys.  Eight requests with 4 key heads of 64/128 behind 16384 tokens, 32 rows: bf16 55 us by tiles, 72 streamed (four requests 43
// and 45, one 41 and 37); fp32, which the matrix cores bound, 232 by tiles, 178 streamed (64 rows: 239 by tiles, 303 streamed).
constexpr int FEW(int type) { return type == MAM_F32 ? 32 : 16; }

// A value that all lanes share, where the compiler does not see it: loops over it are branches of the wave, not of lanes.
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// Quotients of whole numbers below 2^31 by one that the host knows: a multiplication, where a division is 25 instructions in the way of the first load.
struct Divider {
    uint32_t factor;
    int shift;

    explicit Divider(int64_t d) : shift(0)
    {
        while (((int64_t)1 << shift) < d) ++shift;
        factor = (uint32_t)((((uint64_t)1 << (31 + shift)) + d - 1) / d);       // too large by less than 1, so that a quotient is by less than n / 2^(31 + shift) < 1 / d
    }
    __device__ __forceinline__ int operator()(int n) const { return (int)(__umulhi((uint32_t)n << 1, factor) >> shift); }
};
struct Grid {
    int slots, row_tiles;
    Divider heads, group, page;         // of Hkv, of G, of the steps of 16 tokens of a page
};

// A request's table as steps of 16 tokens, 64 of them from `first` on, one a lane: which step of the pages each is, those that there are, and those that are below `end` tokens as a whole.
struct Steps {
    const int32_t *row;
    int slots, P, per, heads, head;
    int first, at;
    uint64_t there, whole;

    __device__ __forceinline__ Steps(const Pages &p, int b, int head) : row(p.table + (int64_t)b * p.slots), slots(p.slots), P(p.P), per(p.S / 16), heads(p.Hkv), head(head) {}
    __device__ __forceinline__ void read(int from, int end, const Divider &page)
    {
        first = from;
        const int step = from + (threadIdx.x & 63), slot = page(step), id = slot < slots ? row[slot] : -1;
        const bool ok = id >= 0 && id < P;
        at = ok ? (id * heads + head) * per + step - slot * per : 0;
        there = __ballot(ok);
        whole = __ballot(ok && (step + 1) * 16 <= end);
        asm volatile("" : "+v"(at));        // waited for here: behind the branch around this call every use would wait for all loads on their way
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

// A workgroup's share of a call: a request, and which part of its keys.  The slots go to the requests by their lengths: one each, the others in proportion, as far as a part keeps
// LEAST_TILES tiles, of which each of a workgroup's waves has one then.  Every wave works them out for itself from the lengths, a request a lane.  (Eight requests behind 1000 tokens, 4 key
// heads of 64/128, fp32, 4 rows each: 28 us; with 8 tiles at least 32, with 2 37 us.  Parts of equal tiles, found by trying, balance no better: trees of 32 tokens 47.7 us, so 46.6,
// both before probabilities had two parts there.)
constexpr int LEAST_TILES = 4;
struct Share { int b, part, parts, slot, length, count; };

__device__ __forceinline__ Share share_of(const Call &a, const Pages &p, int slot, int slots, int32_t *spans)
{
    if (slots == a.B) return {slot, 0, 1, slot, uniform(length_of(p, slot)), uniform(count_of(p, slot, a.Lq))};
    const int lane = threadIdx.x & 63, width = a.B < 64 ? a.B : 64;        // lanes that have requests
    int length = 0, count = 0;
    const auto tiles_of = [&](int b) {
        length = b < a.B ? length_of(p, b) : 0;
        count = b < a.B ? count_of(p, b, a.Lq) : 0;
        const int most = p.slots * p.S, n = length + count;
        return count == 0 ? 0 : ((n < most ? n : most) + KT - 1) / KT;
    };
    float all = 0.0f;
    for (int b = lane; b - lane < a.B; b += 64) all += (float)tiles_of(b);
    for (int x = 1; x < width; x <<= 1) all += __shfl_xor(all, x);
    all = __builtin_bit_cast(float, uniform(__builtin_bit_cast(int, all)));
    // a little less than the proportion, so that rounding gives out no slot too many
    const float each = all > 0.0f ? (float)(slots - a.B) / all * (1.0f - 0x1p-18f) : 0.0f;
    int before = 0;
    Share s{-1, 0, 0, slot, 0, 0};
    for (int b = lane; b - lane < a.B; b += 64) {
        const int tiles = tiles_of(b), most = tiles / LEAST_TILES < 64 ? tiles / LEAST_TILES : 64;
        int n = 1 + (int)((float)tiles * each);
        if (n > most) n = most > 1 ? most : 1;
        if (b >= a.B) n = 0;
        int until = n;
        for (int x = 1; x < width; x <<= 1) {
            const int t = __shfl_up(until, x);
            if (lane >= x) until += t;
        }
        until += before;
        const uint64_t mine = __ballot(slot < until && slot >= until - n);
        if (mine) {
            const int l = __ffsll((unsigned long long)mine) - 1;
            s.b = uniform(b - lane + l);
            s.parts = uniform(__shfl(n, l));
            s.part = uniform(slot - (__shfl(until, l) - s.parts));
            s.length = uniform(__shfl(length, l));
            s.count = uniform(__shfl(count, l));
        }
        before = __shfl(until, 63);
    }
    s.b = uniform(s.b);
    s.part = uniform(s.part);
    s.parts = uniform(s.parts);
    s.length = uniform(s.length);
    s.count = uniform(s.count);
    if (s.b >= 0 && s.part == 0 && threadIdx.x == 0) {
        spans[2 * s.b] = slot;
        spans[2 * s.b + 1] = s.parts;
    }
    return s;
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
        for (int u = 0; u < PE; ++u) e[u] = (T)0.0f;
        if (in && left >= PE) {
            const typename Pack<T, PE>::type t = *reinterpret_cast<const typename Pack<T, PE>::type *>(base + offset);
#pragma unroll
            for (int u = 0; u < PE; ++u) e[u] = t[u];
        } else if (in) {
#pragma unroll
            for (int u = 0; u < PE; ++u)
                if (u < left) e[u] = base[offset + u];
        }
        __builtin_memcpy(w, e, BYTES);
    }
}

// Workgroups of a CU that the registers leave room for.  More than fit at once are a second round: eight requests behind 4000 tokens, 4 key heads of 128/256, 4 rows each: bf16 48 us,
// with two a CU 70; fp32, 128 rows, 331 and 519 us.
constexpr int STREAMS(int size, int d, int dv, bool fast) { return d > 64 || dv > 128 || ((size == 4 || !fast) && dv > 64) ? 1 : 2; }

template <class T, int D, int DV, bool FAST>
__global__ __launch_bounds__(256, STREAMS(sizeof(T), D, DV, FAST)) void pages_kernel(const Call a, const Pages p, const int64_t *__restrict__ masks,
                                                                                                            void *out, float *partial, int32_t *spans, Grid grid)
{
    constexpr int TR = ROWS, NK = D / KS<T, TR>, E = DV / 16;           // E: elements of a lane's values
    constexpr int PE = E < FE<T> ? E : FE<T>, PIECES = E / PE, WORDS = E * (int)sizeof(T) / 4, PW = PE * (int)sizeof(T) / 4;
    constexpr int PARTS = sizeof(T) == 2 ? 2 : 1;
    // Values are asked for at the head of a turn and the next keys before the softmax, where both fit the registers beside the products; in the widest
    // fp32 heads, and where pieces are put together element by element, they come where they are used, one operand after the other: no kernel here may spill a register.  Spilled inside a
    // branch of lanes it came back for those lanes alone.
    constexpr bool AHEAD = FAST && !(sizeof(T) == 4 && DV > 128), EARLY = AHEAD && (sizeof(T) == 2 || D <= 64);
    __shared__ float joined[2][ROWS][DV + 4];
    __shared__ float tops[2][4][ROWS], sums[2][4][ROWS];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), slot = uniform(grid.heads(blockIdx.x)), hk = blockIdx.x - slot * a.Hkv, tile = blockIdx.y;
    // (the slot is the wave's: held a lane each it was kept elsewhere inside a branch of lanes, and came back for those lanes alone)
    const Share share = share_of(a, p, slot, grid.slots, spans);
    if (share.b < 0) return;            // a slot that no request has
    const int b = share.b, split = share.part, splits = share.parts;
    const int length = share.length, count = share.count, room = p.slots * p.S;
    const int row = tile * ROWS + lane_row<TR>();
    const int query = row < a.R ? grid.group(row) : 0;
    const bool there = row < a.R && query < count;
    const uint64_t mask = masks && there ? (uint64_t)masks[(int64_t)b * a.Lq + query] : 0;
    const int limit = there ? length + (masks ? count : query + 1) : 0;
    const int last_row = tile * ROWS + ROWS - 1 < a.R ? tile * ROWS + ROWS - 1 : a.R - 1, last = grid.group(last_row);
    int any = length + (masks || last + 1 > count ? count : last + 1);
    if (any > room) any = room;
    if (grid.group(tile * ROWS) >= count) any = 0;
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

    Steps steps(p, b, hk);
    steps.read(begin / 16, room, grid.page);
    // rows of the pages where the 16 keys from key and from key + 16 on begin, -1 where the request has none
    const auto rows_of = [&](int key, int64_t (&r)[2]) {
        int j = key / 16 - steps.first;
        if (j >= 64) {
            steps.read(key / 16, room, grid.page);
            j = 0;
        }
#pragma unroll
        for (int n = 0; n < 2; ++n) r[n] = steps.there >> (j + n) & 1 ? (int64_t)__builtin_amdgcn_readlane(steps.at, j + n) * 16 : -1;
    };
    int64_t rows[2], next_rows[2];
    Frag<T> k[2][BLOCKS<TR>][NK];
    // addresses of single elements are formed where they are used, not kept for the loop
    const auto here = [](int v) {
        if (!FAST) asm volatile("" : "+v"(v));
        return v;
    };
    const auto load_keys = [&](int first, const int64_t (&r)[2]) {
        const int lane = here(lane_row<TR>()), group = here(lane_group<TR>());
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
        const int lane = here(lane_row<TR>()), group = here(lane_group<TR>());
#pragma unroll
        for (int f = 0; f < REGS<TR>; ++f) {
            const T *base = values + (r[f / 4] < 0 ? 0 : r[f / 4]) * a.dv;
            const int at = 4 * group + f % 4;
            const bool ok = r[f / 4] >= 0 && first + f / 4 * 16 + at < end;
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
        rows_of(begin, rows);
        if (AHEAD) load_keys(begin, rows);
    }
    for (int key = begin; key < end; key += 32) {
        if (!AHEAD) load_keys(key, rows);
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
            rows_of(key + 32, next_rows);
        } else {                // past the range: nothing
            next_rows[0] = next_rows[1] = -1;
        }
        if (EARLY) load_keys(key + 32, next_rows);
        else if (AHEAD) load_values(key, rows);
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
        if (!AHEAD) load_values(key, rows);
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
        if (AHEAD && !EARLY) load_keys(key + 32, next_rows);
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
    if (!partial) {
        const int i = grid.group(out_row), h = hk * a.G + out_row - i * a.G;
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
        float *to = partial + (((int64_t)share.slot * a.Hkv + hk) * a.R + out_row) * (2 * (int64_t)a.dv + 4);
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
// of 16 rows each share tiles of 32 keys: RG of them the same tile, and the workgroup's keys are cut in 8 / RG parts, so that few rows keep eight waves busy too.  The parts meet in
// LDS, the workgroups that share a row's keys in the workspace.
//
// Tiles go from memory to LDS past the registers, several ahead of the one that is used: what a CU has on its way is what hides the memory's latency, and registers for as much there are
// none (one tile ahead in registers: 73 us for the trees above).  A load puts 64 pieces of 16 bytes one behind the other, so rows cannot be padded; instead piece c of row r stands at place
// c ^ turn(r) of its row, and the lanes fetch the pieces in that order.  What a tile has past the last key, or on a page that is not there, is a copy of another of its rows, which
// no score counts; heads smaller than the kernel's have zeros behind them that no load touches.
//
// In 16-bit types what 16 bits leave of the first map's probabilities is a product of its own, as where rows are streamed: a drafted token more or less does not change how exact the others
// are.  Without it 47 us for the trees below and 82 for the chunks; their errors against 64 bits 0.0025 and 0.00032, with it 0.0019 and 0.00024 (results rounded once from 64 bits: 0.0017 and
// 0.00021).
//
// Measured: 8 trees of 32 tokens behind up to 8192, 4 key heads of 64/128 for 16, bf16: 51 us, of which this kernel 46 and the join 9 (overlapped by 4): 5 us to the first tile, 25 tiles of 1.6 us,
// 2 us to store 34 MB of parts.  By counters the kernel's 90000 cycles, 3600 a tile, hold for each tile 1020 of products and 1600 of vector instructions of a SIMD's two waves, which hide each
// other only in part, and 530 of reads of the CU's LDS, without conflicts.  Two chunks of 509 behind up to 4099, 2 key heads of 128/256 for 8, fp16: 94 us, 511 TFLOP/s.  Tried before the probabilities had two parts, beside 47 us:
// scores of the next tile under the exponentials of this one 47.0; six and eight tiles of LDS instead of four 50.5 and 51.1 (49.4 at the time); 64 rows and two parts of the keys in a workgroup, which
// halves the parts' bytes and reads every key twice, 72.

// Places of a tile's pieces: W elements a row, so that 16 rows' pieces of a column (keys), and the 8 rows of 32 bytes (16-bit types) or 4 rows of 64 (fp32) that a read of columns
// takes at a time (values), are in all banks.
template <class T, int W, bool VALUES>
struct Swizzled {
    static constexpr int CHUNKS = W / FE<T>, BYTES = KT * W * (int)sizeof(T), LOADS = BYTES / 1024;
    static __device__ __forceinline__ int turn(int row)
    {
        if (!VALUES) return CHUNKS == 8 ? row >> 1 & 7 : row & 15;
        if (sizeof(T) == 4) return 4 * (row >> 2 & 3);
        return CHUNKS == 8 ? 2 * (row >> 1 & 3) : 2 * (row & 7);
    }
    static __device__ __forceinline__ const unsigned char *piece(const unsigned char *tile, int row, int chunk)
    {
        return tile + row * (W * (int)sizeof(T)) + (chunk ^ turn(row)) * 16;
    }
};

typedef __attribute__((address_space(3))) void *lds_pointer;
typedef const __attribute__((address_space(1))) void *global_pointer;

constexpr int WAVES = 8, LDS_BYTES = 156 * 1024;
template <class T, int D, int DV>
constexpr int PAGE_TILE = KT * (2 * D + DV) * (int)sizeof(T);
// Tiles of a part of the workgroup's keys: one in use, the others on their way.
template <class T, int D, int DV, int RG>
constexpr int RING = LDS_BYTES / (WAVES / RG * PAGE_TILE<T, D, DV>) < 4 ? LDS_BYTES / (WAVES / RG * PAGE_TILE<T, D, DV>) : 4;

// Waits until at most N of the wave's loads are on their way and all of its reads of LDS are done, then for the other waves.
template <int N>
__device__ __forceinline__ void wait_and_meet()
{
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt((N & 15) | N >> 4 << 14 | 7 << 4);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

__device__ __forceinline__ uint32_t lds_offset(const unsigned char *p)
{
    return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const unsigned char *)p;
}

// Fragments of 16 columns each of 32 rows by the transposing read (column_frag): 16 lanes give the addresses of 4 rows x 16 columns and get a column's 4 rows each; the second read's rows
// stand HIGH bytes on.  Four fragments and their wait in one block: before the builtin the compiler waits for every load from memory to LDS that is on its way.
template <int HIGH, class F>
__device__ __forceinline__ void columns_of(const uint32_t (&from)[4], F *v)
{
    typedef uint32_t quad __attribute__((ext_vector_type(2)));
    typedef uint32_t octet __attribute__((ext_vector_type(4)));
    quad lo[4], hi[4];
    asm volatile("ds_read_b64_tr_b16 %0, %8\n\t"
                 "ds_read_b64_tr_b16 %4, %8 offset:%12\n\t"
                 "ds_read_b64_tr_b16 %1, %9\n\t"
                 "ds_read_b64_tr_b16 %5, %9 offset:%12\n\t"
                 "ds_read_b64_tr_b16 %2, %10\n\t"
                 "ds_read_b64_tr_b16 %6, %10 offset:%12\n\t"
                 "ds_read_b64_tr_b16 %3, %11\n\t"
                 "ds_read_b64_tr_b16 %7, %11 offset:%12\n\t"
                 "s_waitcnt lgkmcnt(0)"
                 : "=&v"(lo[0]), "=&v"(lo[1]), "=&v"(lo[2]), "=&v"(lo[3]), "=&v"(hi[0]), "=&v"(hi[1]), "=&v"(hi[2]), "=&v"(hi[3])
                 : "v"(from[0]), "v"(from[1]), "v"(from[2]), "v"(from[3]), "n"(HIGH)
                 : "memory");
#pragma unroll
    for (int n = 0; n < 4; ++n) {
        const octet all = __builtin_shufflevector(lo[n], hi[n], 0, 1, 2, 3);
        v[n] = __builtin_bit_cast(F, all);
    }
}

// A wave's running products and sums; exponentials are relative to `base`, the maximum in powers of two or 0 before there is one.
template <int DV>
struct Running {
    Acc<ROWS> o[2][DV / ROWS];
    float top[2], base[2], sum[2];

    __device__ __forceinline__ void clear()
    {
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            top[m] = -INFINITY;
            base[m] = sum[m] = 0.0f;
#pragma unroll
            for (int b = 0; b < DV / ROWS; ++b)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[m][b][i] = 0.0f;
        }
    }
};

// 32 keys of a tile: their scores, probabilities, and the products with their values.  The vector units are what bounds it (16 exponentials a lane), so nothing else is done for a tile that
// need not be: whether a maximum rises is asked of both maps at once and of each lane's own scores; the rows' maxima are formed across lanes where one does.  Values are read behind the
// products of the scores, which run meanwhile.
template <bool LIMITED, class T, int D, int DV>
__device__ __forceinline__ void page_keys(Running<DV> &state, const Frag<T> (&q)[2][D / KS<T, ROWS>], const unsigned char *tile, float c, int limit, uint32_t word)
{
    constexpr int TR = ROWS, NK = D / KS<T, TR>, BLK = DV / TR, WIDE = sizeof(T) == 2, FIRST = WIDE && BLK <= 8 ? BLK : 0;
    typedef Swizzled<T, 2 * D, false> KeyTile;
    typedef Swizzled<T, DV, true> ValueTile;
    const unsigned char *values = tile + KeyTile::BYTES;
    const int lane = threadIdx.x & 63, row = lane_row<TR>(), group = lane_group<TR>();
    Acc<TR> s[2][BLOCKS<TR>];
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int blk = 0; blk < BLOCKS<TR>; ++blk)
#pragma unroll
            for (int n = 0; n < 4; ++n) s[m][blk][n] = 0.0f;
#pragma unroll
    for (int n = 0; n < 2 * BLOCKS<TR> * NK; ++n) {
        // sums that do not wait for each other in turn; one after the other where there are no registers for their keys
        const int sum = DV > 128 ? n / NK : n % (2 * BLOCKS<TR>), kk = DV > 128 ? n % NK : n / (2 * BLOCKS<TR>), m = sum / BLOCKS<TR>, blk = sum % BLOCKS<TR>;
        mma<TR>(*reinterpret_cast<const Frag<T> *>(KeyTile::piece(tile, blk * TR + row, m * (D / FE<T>) + kk * GROUPS<TR> + group)), q[m][kk], s[m][blk]);
    }
    // column fragments of 16-bit values
    const int r = 4 * group + lane % 16 / 4, half = lane % 4 / 2;
    const uint32_t at = lds_offset(values) + r * (DV * 2) + lane % 2 * 8;
    const auto columns = [&](int blk, Frag<T> *v) __attribute__((always_inline)) {
        uint32_t from[4];
#pragma unroll
        for (int n = 0; n < 4; ++n) from[n] = at + ((2 * (blk + n) + half) ^ ValueTile::turn(r)) * 16;
        columns_of<16 * DV * 2>(from, v);
    };
    Frag<T> v[FIRST ? FIRST : 1];
#pragma unroll
    for (int blk = 0; blk < FIRST; blk += 4) columns(blk, v + blk);

    float high[2];
#pragma unroll
    for (int m = 0; m < 2; ++m) {
#pragma unroll
        for (int f = 0; f < REGS<TR>; ++f)
            if constexpr (LIMITED) {
                const int key = index_of<TR>(f);
                s[m][f / 4][f % 4] = key < limit && (word >> key & 1) ? s[m][f / 4][f % 4] : -INFINITY;
            }
        float x = s[m][0][0];
#pragma unroll
        for (int f = 1; f < REGS<TR>; ++f) x = fmaxf(x, s[m][f / 4][f % 4]);
        high[m] = x * c;
    }
    if (__any(high[0] > state.top[0] + SLACK || high[1] > state.top[1] + SLACK)) {
        asm volatile("; a new maximum");        // kept a branch
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            const float rise = fmaxf(state.top[m], groups_max<TR>(high[m])), factor = rise == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(state.top[m] - rise);
            state.top[m] = rise;
            state.base[m] = rise == -INFINITY ? 0.0f : rise;
            state.sum[m] *= factor;
#pragma unroll
            for (int b = 0; b < BLK; ++b)
#pragma unroll
                for (int i = 0; i < 4; ++i) state.o[m][b][i] *= factor;
        }
    }
    Frag<T> frag[2][FRAGS<T, TR>], rest[FRAGS<T, TR>];
    const auto exponentials = [&](int m) __attribute__((always_inline)) {
        float x[REGS<TR>];
#pragma unroll
        for (int f = 0; f < REGS<TR>; ++f) x[f] = __builtin_amdgcn_exp2f(fmaf(s[m][f / 4][f % 4], c, -state.base[m]));
        state.sum[m] += ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
        to_frags<T, TR>(x, frag[m]);
        if (WIDE && m == 0) {           // what 16 bits leave of the first map's
#pragma unroll
            for (int f = 0; f < REGS<TR>; ++f) x[f] -= element(frag[0][f / FE<T>], f % FE<T>);
            to_frags<T, TR>(x, rest);
        }
    };
    exponentials(0);
    if constexpr (WIDE) {
#pragma unroll
        for (int blk = 0; blk < FIRST; ++blk) mma<TR>(v[blk], frag[0][0], state.o[0][blk]);
#pragma unroll
        for (int blk = 0; blk < FIRST; ++blk) mma<TR>(v[blk], rest[0], state.o[0][blk]);
        exponentials(1);
#pragma unroll
        for (int blk = 0; blk < FIRST; ++blk) mma<TR>(v[blk], frag[1][0], state.o[1][blk]);
#pragma unroll
        for (int blk = FIRST; blk < BLK; blk += 4) {
            Frag<T> more[4];
            columns(blk, more);
#pragma unroll
            for (int n = 0; n < 4; ++n)
#pragma unroll
                for (int m = 0; m < 2; ++m) mma<TR>(more[n], frag[m][0], state.o[m][blk + n]);
#pragma unroll
            for (int n = 0; n < 4; ++n) mma<TR>(more[n], rest[0], state.o[0][blk + n]);
        }
    } else {
        exponentials(1);
#pragma unroll
        for (int blk = 0; blk < BLK; ++blk)
#pragma unroll
            for (int j = 0; j < FRAGS<T, TR>; ++j) {
                Frag<T> x;
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    x[u] = *reinterpret_cast<const float *>(ValueTile::piece(values, 16 * j + 4 * group + u, 4 * blk + lane % 16 / 4) + lane % 4 * 4);
#pragma unroll
                for (int m = 0; m < 2; ++m) mma<TR>(x, frag[m][j], state.o[m][blk]);
            }
    }
}

template <class T, int D, int DV, int RG>
__global__ __launch_bounds__(WAVES * 64) __attribute__((amdgpu_waves_per_eu(2, 2))) void page_tiles_kernel(const Call a, const Pages p, const int64_t *__restrict__ masks, void *out, float *partial,
                                                                   int32_t *spans, Grid grid)
{
    constexpr int TR = ROWS, PARTS = WAVES / RG, NB = RING<T, D, DV, RG>, AHEAD = NB - 1, TILE = PAGE_TILE<T, D, DV>, AR = 4, ACC = DV / TR * AR, NK = D / KS<T, TR>;
    typedef Swizzled<T, 2 * D, false> KeyTile;
    typedef Swizzled<T, DV, true> ValueTile;
    constexpr int LOADS = (KeyTile::LOADS + ValueTile::LOADS + RG - 1) / RG;            // of a wave, for a tile
    static_assert(NB >= 2 && AHEAD * LOADS < 64, "a tile on its way, and all of them counted");
    constexpr int TILES_AT = PARTS * NB * TILE, JOIN_AT = (PARTS - 1) * RG * 2 * 64 * ACC * 4;
    __shared__ __attribute__((aligned(1024))) unsigned char lds[TILES_AT > JOIN_AT ? TILES_AT : JOIN_AT];
    __shared__ float tops[PARTS][2][RG][TR], sums[PARTS][2][RG][TR];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), part = wave / RG, group = wave % RG, lane = threadIdx.x & 63;
    const int slot = uniform(grid.heads(blockIdx.x)), hk = blockIdx.x - slot * a.Hkv, tile = grid.row_tiles - 1 - blockIdx.y;
    const Share share = share_of(a, p, slot, grid.slots, spans);
    if (share.b < 0) return;            // a slot that no request has
    const int b = share.b, split = share.part, splits = share.parts;
    const int length = share.length, count = share.count, room = p.slots * p.S;
    const int first = (tile * RG + group) * TR, row = first + lane_row<TR>();
    const int query = row < a.R ? grid.group(row) : 0;
    const bool there = row < a.R && query < count;
    const uint64_t mask = masks && there ? (uint64_t)masks[(int64_t)b * a.Lq + query] : 0;
    const int limit = there ? length + (masks ? count : query + 1) : 0;
    // keys that rows from .. last see at most: none where the first of them is no query
    const auto reach = [&](int from, int last) {
        const int q = grid.group(last < a.R ? last : a.R - 1);
        const int n = length + (masks || q + 1 > count ? count : q + 1);
        return from >= a.R || grid.group(from) >= count ? 0 : n < room ? n : room;
    };
    const int wave_any = reach(first, first + TR - 1), any = reach(tile * RG * TR, (tile + 1) * RG * TR - 1);
    // and those that every row of the wave sees (rows that are none see what they like)
    const int wave_all = masks || wave_any == 0 ? length : length + grid.group(first) + 1;
    // the workgroup's tiles, and this part's; parts differ by one tile at most, the first ones having more
    const int tiles = (any + KT - 1) / KT, per = (tiles + splits - 1) / splits, from = split * per < tiles ? split * per : tiles;
    const int mine = from + per < tiles ? per : tiles - from, most = (mine + PARTS - 1) / PARTS;
    const int begin = from + (part * mine + PARTS - 1) / PARTS, number = from + ((part + 1) * mine + PARTS - 1) / PARTS - begin;

    const Source<T> qs{static_cast<const T *>(a.q) + b * a.qb + (int64_t)hk * a.G * a.qh, a.ql, a.qh, a.qm, a.G, a.d, a.inverse};
    Frag<T> q[2][NK];
#pragma unroll
    for (int m = 0; m < 2; ++m) load_rows<T, TR, D>(qs, row, there, m, q[m]);
    Steps steps(p, b, hk);
    steps.read(2 * begin, any, grid.page);
    // the queries come with the table: waited for in the loop they would have every tile waited for
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int kk = 0; kk < NK; ++kk) {
            typedef uint32_t words __attribute__((ext_vector_type(4)));
            words w = __builtin_bit_cast(words, q[m][kk]);
            asm volatile("" : "+v"(w));
            q[m][kk] = __builtin_bit_cast(Frag<T>, w);
        }
    const float c = a.scale * LOG2E;
    Running<DV> state;
    state.clear();
    if (a.d < D || a.dv < DV) {
        typedef uint32_t words __attribute__((ext_vector_type(4)));
        for (int i = threadIdx.x * 16; i < TILES_AT; i += WAVES * 64 * 16) *reinterpret_cast<words *>(lds + i) = words{0, 0, 0, 0};
        __syncthreads();
    }

    // A tile on its way.
    unsigned char *const ring = lds + part * NB * TILE;
    const unsigned char *const keys = static_cast<const unsigned char *>(p.k), *const values = static_cast<const unsigned char *>(p.v);
    const uint32_t key_step = 16 * 2 * (uint32_t)(a.d * (int)sizeof(T)), value_step = 16 * (uint32_t)(a.dv * (int)sizeof(T));
    constexpr int ALL = KeyTile::LOADS + ValueTile::LOADS;
    uint32_t offset[LOADS];                     // bytes from a half's rows to a lane's piece of a whole tile
    bool mine_there[LOADS];
    const auto number_of = [&](int i) __attribute__((always_inline)) { return (i * RG + group) % ALL; };       // a wave that has none left loads another one's again
    const auto is_value = [&](int i) __attribute__((always_inline)) { return KeyTile::LOADS % RG == 0 && ALL % RG == 0 ? i >= KeyTile::LOADS / RG : number_of(i) >= KeyTile::LOADS; };
    const auto second_of = [&](int i) __attribute__((always_inline)) {
        const bool value = is_value(i);
        return (value ? number_of(i) - KeyTile::LOADS : number_of(i)) >= (value ? ValueTile::LOADS : KeyTile::LOADS) / 2;
    };
    const auto place = [&](int i, int lane, int &r, int &column) __attribute__((always_inline)) {
        const bool value = is_value(i);
        const int at = (value ? number_of(i) - KeyTile::LOADS : number_of(i)) * 1024 + lane * 16, bytes = (value ? DV : 2 * D) * (int)sizeof(T);   // of a row of LDS
        const int chunk = at % bytes / 16 ^ (value ? ValueTile::turn(at / bytes) : KeyTile::turn(at / bytes));
        const int map = value ? 0 : chunk / (D / FE<T>), col = (value ? chunk : chunk % (D / FE<T>)) * FE<T>;
        r = at / bytes & 15;
        column = map * a.d + col;
        return col < (value ? a.dv : a.d);
    };
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
        int r, column;
        mine_there[i] = place(i, lane, r, column);
        offset[i] = (uint32_t)(r * (is_value(i) ? a.dv : 2 * a.d) + column) * (uint32_t)sizeof(T);
    }
    uint32_t ways = 0;                          // of the tiles from the one in use on, two bits each: which halves of them there are
    int from_ring = 0, to_ring = 0;             // where the tile in use and the next one to load stand
    const auto fetch = [&](const unsigned char *base, uint32_t off, unsigned char *to) __attribute__((always_inline)) {
        const auto rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char *>(base), 0, 0x7fffffff, 0x00027000);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_pointer)to, 16, (int)off, 0, 0, 0);
    };
    const auto load = [&](int t, int ahead) __attribute__((always_inline)) {
        int j = 2 * t - steps.first;
        if (j >= 64) {
            steps.read(2 * t, any, grid.page);
            j = 0;
        }
        // Whole tiles take every row as it is; of another one, rows past the last key are the last key's, and a half that is not there is the other one's rows.
        const int left = any - t * KT;          // keys of the tile
        const bool all = (steps.whole >> j & 3) == 3;
        const uint32_t halves = all ? 3 : (uint32_t)(steps.there >> j) & (left > 16 ? 3 : 1);
        ways |= halves << 2 * ahead;
        uint32_t half[2] = {(uint32_t)__builtin_amdgcn_readlane(steps.at, j), (uint32_t)__builtin_amdgcn_readlane(steps.at, j + 1)};
        if (halves == 2) half[0] = half[1];
        if (!(halves & 2)) half[1] = half[0];
        uint32_t off[LOADS];
#pragma unroll
        for (int i = 0; i < LOADS; ++i) off[i] = offset[i];
        if (!all) {
            int here = lane;                    // rows are formed here, not kept for the loop
            asm volatile("" : "+v"(here));
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {
                int r, column;
                place(i, here, r, column);
                const int past = r + 1 - ((second_of(i) ? halves & 2 : halves == 2) ? left - 16 : left);
                if (past > 0) off[i] -= (uint32_t)(past * (is_value(i) ? a.dv : 2 * a.d)) * (uint32_t)sizeof(T);
            }
        }
        const unsigned char *const k[2] = {keys + (uint64_t)half[0] * key_step, keys + (uint64_t)half[1] * key_step};
        const unsigned char *const v[2] = {values + (uint64_t)half[0] * value_step, values + (uint64_t)half[1] * value_step};
        unsigned char *const to = ring + to_ring;
        to_ring = to_ring + TILE < NB * TILE ? to_ring + TILE : 0;
        // (a load covers rows as a whole, so that some of its lanes are always there, and it counts)
#pragma unroll
        for (int i = 0; i < LOADS; ++i)
            if (mine_there[i]) fetch(is_value(i) ? v[second_of(i)] : k[second_of(i)], off[i], to + number_of(i) * 1024);
    };
    for (int i = 0; i < AHEAD && i < number; ++i) load(begin + i, i);

    int i = 0;
    const auto next_tile = [&](const auto &use) __attribute__((always_inline)) {
        const uint32_t halves = ways & 3;
        ways >>= 2;
        if (i + AHEAD < number) load(begin + i + AHEAD, AHEAD - 1);         // where the last tile stood: every wave is past it
        use((begin + i) * KT, halves, ring + from_ring);
        from_ring = from_ring + TILE < NB * TILE ? from_ring + TILE : 0;
        ++i;
    };
    const int open = (wave_all < wave_any ? wave_all : wave_any) / KT - begin, seen = (wave_any + KT - 1) / KT - begin;
    // as long as there is a tile to load for each that is used, and every row sees all of it
    const int many = open < number - AHEAD ? open : number - AHEAD;
    while (i < many && (ways & 3) == 3) {
        wait_and_meet<(AHEAD - 1) * LOADS>();
        next_tile([&](int, uint32_t, const unsigned char *t) { page_keys<false, T, D, DV>(state, q, t, c, 0, 0); });
    }
    // then the others.  Waves that are past their keys go on loading for those that are not, in a loop of its own (a condition around the products has the accumulators copied in every tile).
    const auto wait = [&]() __attribute__((always_inline)) {
        if (i + AHEAD <= number) wait_and_meet<(AHEAD - 1) * LOADS>();
        else wait_and_meet<0>();
    };
    while (i < number && i < seen) {
        wait();
        next_tile([&](int key, uint32_t halves, const unsigned char *t) {
            const uint32_t word = (masks ? seen_word(key, length, mask) : 0xffffffffu) & ((halves & 1 ? 0xffffu : 0u) | (halves & 2 ? 0xffff0000u : 0u));
            if (halves) page_keys<true, T, D, DV>(state, q, t, c, limit - key, word);
        });
    }
    while (i < most) {
        wait();
        next_tile([](int, uint32_t, const unsigned char *) {});
    }

    // the parts: every row's maxima, sums and products but the first part's go to LDS; a row that is no query's has seen nothing
    float total[2];
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        total[m] = there ? groups_sum<TR>(state.sum[m]) : 0.0f;
        if (!there) state.top[m] = -INFINITY;
    }
    if constexpr (PARTS > 1) {
        __syncthreads();
        float *cells = reinterpret_cast<float *>(lds) + lane;
        constexpr int SIZE = 2 * 64 * ACC;
        if (part) {
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                if (lane_group<TR>() == 0) {
                    tops[part][m][group][lane_row<TR>()] = state.top[m];
                    sums[part][m][group][lane_row<TR>()] = total[m];
                }
#pragma unroll
                for (int n = 0; n < ACC; ++n) cells[((part - 1) * RG + group) * SIZE + (m * ACC + n) * 64] = state.o[m][n / AR][n % AR];
            }
        }
        __syncthreads();
        if (part) return;
#pragma unroll 1
        for (int other = 1; other < PARTS; ++other)
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                // a range of which a row sees nothing has a sum of 0, and its products do not count whatever the values there hold
                const float top = tops[other][m][group][lane_row<TR>()], sum = sums[other][m][group][lane_row<TR>()], rise = fmaxf(top, state.top[m]);
                const float old = total[m] == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(state.top[m] - rise), more = sum == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(top - rise);
#pragma unroll
                for (int n = 0; n < ACC; ++n) {
                    const float x = total[m] == 0.0f ? 0.0f : state.o[m][n / AR][n % AR] * old;
                    const float y = sum == 0.0f ? 0.0f : cells[((other - 1) * RG + group) * SIZE + (m * ACC + n) * 64] * more;
                    state.o[m][n / AR][n % AR] = x + y;
                }
                total[m] = (total[m] == 0.0f ? 0.0f : total[m] * old) + (sum == 0.0f ? 0.0f : sum * more);
                state.top[m] = rise;
            }
    } else {
#pragma unroll
        for (int m = 0; m < 2; ++m)
            if (total[m] == 0.0f)
#pragma unroll
                for (int n = 0; n < ACC; ++n) state.o[m][n / AR][n % AR] = 0.0f;
    }
    int late = lane_row<TR>();          // the row and its query once more, not kept for the loop
    asm volatile("" : "+v"(late));
    const int out_row = first + late, out_query = grid.group(out_row);
    if (out_row >= a.R) return;
    if (!partial) {
        const int head = hk * a.G + out_row - out_query * a.G;
        const float lam = lambda_of(a, head, static_cast<const T *>(nullptr));
        float factor[2];
#pragma unroll
        for (int m = 0; m < 2; ++m) factor[m] = total[m] > 0.0f ? 1.0f / total[m] : 0.0f;
        T *to = static_cast<T *>(out) + (((int64_t)b * a.Lq + out_query) * a.H + head) * a.dv;
#pragma unroll
        for (int blk = 0; blk < DV / TR; ++blk) {
            const int col = blk * TR + 4 * lane_group<TR>();
            if (col >= a.dv) continue;
            float r[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) r[u] = fmaf(-lam, state.o[1][blk][u] * factor[1], state.o[0][blk][u] * factor[0]);
            store_pack<T, 4>(to + col, a.dv - col, r);
        }
    } else {
        float *to = partial + (((int64_t)share.slot * a.Hkv + hk) * a.R + out_row) * (2 * (int64_t)a.dv + 4);
#pragma unroll
        for (int m = 0; m < 2; ++m) {
#pragma unroll
            for (int blk = 0; blk < DV / TR; ++blk) {
                const int col = blk * TR + 4 * lane_group<TR>();
                if (col >= a.dv) continue;
                float r[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) r[u] = state.o[m][blk][u];
                store_pack<float, 4>(to + m * a.dv + col, a.dv - col, r);
            }
            if (lane_group<TR>() == 0) {
                to[2 * a.dv + 2 * m] = state.top[m];
                to[2 * a.dv + 2 * m + 1] = total[m];
            }
        }
    }
}

// The slots' parts of a row, a wave a row, in the slots' order.
template <class T>
__global__ __launch_bounds__(256) void join_pages_kernel(const Call a, void *out, const float *__restrict__ partial, const int32_t *__restrict__ spans)
{
    const int64_t id = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (id >= (int64_t)a.B * a.Hkv * a.R) return;
    const int lane = threadIdx.x & 63, row = (int)(id % a.R), bh = (int)(id / a.R), b = bh / a.Hkv, hk = bh - b * a.Hkv;
    const int query = row / a.G, head = hk * a.G + row - query * a.G;
    const int first = uniform(spans[2 * b]), parts = uniform(spans[2 * b + 1]);
    const int64_t size = 2 * (int64_t)a.dv + 4, step = (int64_t)a.Hkv * a.R * size;
    const float *p = partial + (((int64_t)first * a.Hkv + hk) * a.R + row) * size;
    // lane s holds part s's maxima and sums (parts <= 64)
    float factor[2];
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        float top = -INFINITY, sum = 0.0f;
        if (lane < parts) {
            top = p[lane * step + 2 * a.dv + 2 * m];
            sum = p[lane * step + 2 * a.dv + 2 * m + 1];
        }
        float most = top;
#pragma unroll
        for (int x = 1; x < 64; x <<= 1) most = fmaxf(most, __shfl_xor(most, x));
        const float mine = most == -INFINITY ? sum == 0.0f ? 0.0f : 1.0f : __builtin_amdgcn_exp2f(top - most);
        float total = sum == 0.0f ? 0.0f : sum * mine;
#pragma unroll
        for (int x = 1; x < 64; x <<= 1) total += __shfl_xor(total, x);
        factor[m] = total != 0.0f ? sum == 0.0f ? 0.0f : mine / total : 0.0f;
    }
    const float lam = lambda_of(a, head, static_cast<const T *>(nullptr));
    const int left = a.dv - 4 * lane;
    float r[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    constexpr int AHEAD = 8;            // parts on their way at once
    for (int s0 = 0; s0 < parts; s0 += AHEAD) {         // every lane stays to the end: each has a part's factors
        float p1[AHEAD][4], p2[AHEAD][4];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const float *t = p + (s0 + u < parts ? s0 + u : parts - 1) * step + 4 * lane;
            load_pack<float, 4>(t, left, p1[u]);
            load_pack<float, 4>(t + a.dv, left, p2[u]);
        }
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const int s = s0 + u;
            const float f0 = s < parts ? __shfl(factor[0], s) : 0.0f, f1 = s < parts ? -lam * __shfl(factor[1], s) : 0.0f;
#pragma unroll
            for (int e = 0; e < 4; ++e) r[e] = fmaf(f1, p2[u][e], fmaf(f0, p1[u][e], r[e]));
        }
    }
    if (left > 0) store_pack<T, 4>(static_cast<T *>(out) + (((int64_t)b * a.Lq + query) * a.H + head) * a.dv + 4 * lane, left, r);
}

// Row groups of a workgroup's tiles for `rows` rows of a key head, as few as hold them and as the ring leaves room for; 0: rows are streamed.  The widest heads have no registers for more
// than one part (16 bits) and for any (fp32).
template <class T, int D, int DV>
constexpr bool FITS(int groups)
{
    if (DV > 128) return sizeof(T) == 2 && groups == 8;
    if (groups == 2 && sizeof(T) == 4) return false;            // as few rows are streamed
    return (groups == 2 ? RING<T, D, DV, 2> : groups == 4 ? RING<T, D, DV, 4> : RING<T, D, DV, 8>) >= 2;
}
template <class T>
struct GroupsOf {
    int rows;
    template <int D, int DV>
    int operator()() const
    {
        if (rows <= 2 * ROWS && FITS<T, D, DV>(2)) return 2;
        if (rows <= 4 * ROWS && FITS<T, D, DV>(4)) return 4;
        return FITS<T, D, DV>(8) ? 8 : 0;
    }
};

// How a call runs: row groups, and slots: workgroups that share the keys of a key head's tile of rows over all requests.
struct Plan {
    int groups, slots;
    int64_t row_tiles;
};
Plan plan_of(const Call &a, const Pages &p, int type)
{
    Plan plan{};
    if (a.R > FEW(type) && a.fast && p.P > 0)         // heads that end inside 16 bytes are streamed
        plan.groups = type == MAM_F32 ? with_head_sizes(a.d, a.dv, GroupsOf<float>{a.R}) : with_head_sizes(a.d, a.dv, GroupsOf<bf16>{a.R});
    plan.row_tiles = ceil_div(a.R, plan.groups ? plan.groups * ROWS : ROWS);
    // as many workgroups as there is room for at once
    const int64_t rows = a.Hkv * plan.row_tiles, want = (plan.groups ? 1 : STREAMS((int)type_size(type), a.d, a.dv, a.fast)) * kNumCU / (rows > 0 ? rows : 1), most = ceil_div(a.Lk, LEAST_TILES * KT) * a.B;
    int64_t n = want < most ? want : most;
    if (n > 64 * (int64_t)a.B) n = 64 * (int64_t)a.B;
    plan.slots = n > a.B ? (int)n : a.B;
    return plan;
}
inline bool parted(const Call &a, const Plan &plan) { return plan.slots > a.B; }

// Partial rows of every slot, and each request's first slot and their number.
size_t pages_workspace(const Call &a, const Plan &plan)
{
    return parted(a, plan) ? (size_t)plan.slots * a.Hkv * a.R * partial_size(a) * sizeof(float) + 2 * (size_t)a.B * sizeof(int32_t) : 0;
}

template <class T>
struct PagesRun {
    const Call &a;
    const Pages &p;
    const int64_t *masks;
    void *out;
    Plan plan;
    float *partial;
    int32_t *spans;
    hipStream_t st;
    template <int D, int DV, int RG>
    void tiles(dim3 blocks, const Grid &grid) const
    {
        if constexpr (FITS<T, D, DV>(RG))
            hipLaunchKernelGGL((page_tiles_kernel<T, D, DV, RG>), blocks, dim3(WAVES * 64), 0, st, a, p, masks, out, partial, spans, grid);
    }
    template <int D, int DV>
    int operator()() const
    {
        if ((int64_t)a.Hkv * plan.slots > UINT32_MAX / (WAVES * 64) || plan.row_tiles > 65535) return fail(MAM_ERR_UNSUPPORTED, "too many requests or rows for a launch");
        const dim3 blocks((unsigned)(a.Hkv * plan.slots), (unsigned)plan.row_tiles);
        const Grid grid{plan.slots, (int)plan.row_tiles, Divider(a.Hkv), Divider(a.G), Divider(p.S / 16)};
        if (plan.groups == 8) tiles<D, DV, 8>(blocks, grid);
        else if (plan.groups == 4) tiles<D, DV, 4>(blocks, grid);
        else if (plan.groups == 2) tiles<D, DV, 2>(blocks, grid);
        else if (a.fast) hipLaunchKernelGGL((pages_kernel<T, D, DV, true>), blocks, dim3(256), 0, st, a, p, masks, out, partial, spans, grid);
        else hipLaunchKernelGGL((pages_kernel<T, D, DV, false>), blocks, dim3(256), 0, st, a, p, masks, out, partial, spans, grid);
        int rc = check_launch("attention over pages");
        if (rc != MAM_OK || !partial) return rc;
        hipLaunchKernelGGL((join_pages_kernel<T>), dim3((unsigned)ceil_div((int64_t)a.B * a.Hkv * a.R, 4)), dim3(256), 0, st, a, out, partial, spans);
        return check_launch("attention::join_pages_kernel");
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
    if (g.P * g.Hkv > INT32_MAX / (g.S / 16 > 0 ? g.S / 16 : 1)) return fail(MAM_ERR_UNSUPPORTED, "too many pages");      // their steps of 16 tokens are counted in 32 bits
    if (x->masks && x->N > 64) return fail(MAM_ERR_UNSUPPORTED, "a tree has 64 tokens at most, got %lld", (long long)x->N);
    const int64_t pack = 16 / type_size(g.type);
    c.fast = g.D % pack == 0 && g.Dv % pack == 0;
    return MAM_OK;
}

}  // namespace
}  // namespace attention
}  // namespace mam

extern "C" size_t mam_diff_attention_pages_workspace(const mam_diff_attention_pages_t *args)
{
    using namespace mam;
    attention::Call a;
    Pages p;
    if (attention::fill_pages_call(args, a, p) != MAM_OK || a.B == 0 || a.R == 0) return 0;
    return attention::pages_workspace(a, attention::plan_of(a, p, args->pages.type));
}

extern "C" int mam_diff_attention_pages(const mam_diff_attention_pages_t *args, void *out, void *workspace, size_t workspace_bytes, void *stream)
{
    using namespace mam;
    attention::Call a;
    Pages p;
    int rc = attention::fill_pages_call(args, a, p);
    if (rc != MAM_OK || a.B == 0 || a.R == 0) return rc;
    if (!a.q || !a.lam || !out || (p.P > 0 && (!p.k || !p.v))) return fail(MAM_ERR_INVALID_ARGUMENT, "null pointer");
    const attention::Plan plan = attention::plan_of(a, p, args->pages.type);
    const size_t need = attention::pages_workspace(a, plan);
    if (need > 0 && (!workspace || workspace_bytes < need))
        return fail(MAM_ERR_WORKSPACE, "the attention needs %zu workspace bytes, got %zu", need, workspace ? workspace_bytes : (size_t)0);
    hipStream_t st = static_cast<hipStream_t>(stream);
    float *partial = need > 0 ? static_cast<float *>(workspace) : nullptr;
    int32_t *spans = need > 0 ? reinterpret_cast<int32_t *>(static_cast<char *>(workspace) + need) - 2 * (int64_t)a.B : nullptr;
    if (args->pages.type == MAM_F32) return attention::with_head_sizes(a.d, a.dv, attention::PagesRun<float>{a, p, args->masks, out, plan, partial, spans, st});
    if (args->pages.type == MAM_BF16) return attention::with_head_sizes(a.d, a.dv, attention::PagesRun<bf16>{a, p, args->masks, out, plan, partial, spans, st});
    return attention::with_head_sizes(a.d, a.dv, attention::PagesRun<f16>{a, p, args->masks, out, plan, partial, spans, st});
}
