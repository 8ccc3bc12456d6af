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

// A value that all lanes share, where the compiler does not see it: loops over it are branches of the wave, not of lanes.
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

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
        asm volatile("" : "+v"(ids));       // waited for here: behind the branch around this call every use would wait for all loads on their way
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

template <class T, int D, int DV, bool FAST>
__global__ __launch_bounds__(256, D > 64 || ((sizeof(T) == 4 || !FAST) && DV > 64) ? 1 : 2) void pages_kernel(const Call a, const Pages p, const int64_t *__restrict__ masks,
                                                                                                  void *out, float *partial, int splits, int row_tiles)
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
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), heads = a.B * a.Hkv;
    const int bh = blockIdx.x % heads, rest_id = blockIdx.x / heads, tile = rest_id % row_tiles, split = rest_id / row_tiles;
    const int b = bh / a.Hkv, hk = bh % a.Hkv;
    const int length = uniform(length_of(p, b)), count = uniform(count_of(p, b, a.Lq)), room = p.slots * p.S;
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
        rows[0] = walk.next();
        rows[1] = walk.next();
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
            next_rows[0] = walk.next();
            next_rows[1] = walk.next();
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
// of 16 rows each share tiles of 32 keys: RG of them the same tile, and the workgroup's keys are cut in 8 / RG parts, so that few rows keep eight waves busy too.  The parts meet in
// LDS, the workgroups that share a row's keys in the workspace.
//
// Tiles go from memory to LDS past the registers, several ahead of the one that is used: what a CU has on its way is what hides the memory's latency, and registers for as much there are
// none (one tile ahead in registers: 73 us for the trees above).  A load puts 64 pieces of 16 bytes one behind the other, so rows cannot be padded; instead piece c of row r stands at place
// c ^ turn(r) of its row, and the lanes fetch the pieces in that order.  What a tile has past the last key, or on a page that is not there, is a copy of another of its rows, which
// no score counts; heads smaller than the kernel's have zeros behind them that no load touches.
//
// In 16-bit types the probabilities are rounded once: what 16 bits leave of the first map's is not kept here, as in mam_attention.hip's kernels for many rows (a third product of the values).

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

constexpr int LDS_BYTES = 156 * 1024;
template <class T, int D, int DV>
constexpr int PAGE_TILE = KT * (2 * D + DV) * (int)sizeof(T);
// Tiles of a part of the workgroup's keys: one in use, the others on their way.
template <class T, int D, int DV, int RG>
constexpr int RING = LDS_BYTES / (8 / RG * PAGE_TILE<T, D, DV>) < 4 ? LDS_BYTES / (8 / RG * PAGE_TILE<T, D, DV>) : 4;

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
__device__ __forceinline__ void columns_of(const uint32_t (&from)[4], F (&v)[4])
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

// 32 keys of a tile: their scores, probabilities, and the products with their values.
template <bool LIMITED, class T, int D, int DV>
__device__ __forceinline__ void page_keys(State<T, ROWS, D, DV, true> &state, const Frag<T> (&q)[2][D / KS<T, ROWS>], const unsigned char *tile, float c, int limit,
                                          uint32_t word)
{
    constexpr int TR = ROWS, NK = D / KS<T, TR>;
    typedef Swizzled<T, 2 * D, false> KeyTile;
    typedef Swizzled<T, DV, true> ValueTile;
    const unsigned char *values = tile + KeyTile::BYTES;
    const int lane = threadIdx.x & 63, row = lane_row<TR>(), group = lane_group<TR>();
    Frag<T> frag[2][FRAGS<T, TR>];
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        Acc<TR> s[BLOCKS<TR>];
#pragma unroll
        for (int blk = 0; blk < BLOCKS<TR>; ++blk) {
#pragma unroll
            for (int n = 0; n < 4; ++n) s[blk][n] = 0.0f;
#pragma unroll
            for (int kk = 0; kk < NK; ++kk)
                mma<TR>(*reinterpret_cast<const Frag<T> *>(KeyTile::piece(tile, blk * TR + row, m * (D / FE<T>) + kk * GROUPS<TR> + group)), q[m][kk], s[blk]);
        }
        float x[REGS<TR>];
        state.template softmax<LIMITED, REGS<TR>>(m, s, c, limit, word, x);
        to_frags<T, TR>(x, frag[m]);
    }
    if constexpr (sizeof(T) == 2) {
        const int r = 4 * group + lane % 16 / 4, half = lane % 4 / 2;
        const uint32_t at = lds_offset(values) + r * (DV * 2) + lane % 2 * 8;
#pragma unroll
        for (int blk = 0; blk < DV / TR; blk += 4) {
            Frag<T> v[4];
            uint32_t from[4];
#pragma unroll
            for (int n = 0; n < 4; ++n) from[n] = at + ((2 * (blk + n) + half) ^ ValueTile::turn(r)) * 16;
            columns_of<16 * DV * 2>(from, v);
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                mma<TR>(v[n], frag[0][0], state.o[0][blk + n]);
                mma<TR>(v[n], frag[1][0], state.o[1][blk + n]);
            }
        }
    } else {
#pragma unroll
        for (int blk = 0; blk < DV / TR; ++blk)
#pragma unroll
            for (int j = 0; j < FRAGS<T, TR>; ++j) {
                Frag<T> v;
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    v[u] = *reinterpret_cast<const float *>(ValueTile::piece(values, 16 * j + 4 * group + u, 4 * blk + lane % 16 / 4) + lane % 4 * 4);
                mma<TR>(v, frag[0][j], state.o[0][blk]);
                mma<TR>(v, frag[1][j], state.o[1][blk]);
            }
    }
}

template <class T, int D, int DV, int RG>
__global__ __launch_bounds__(512, 2) void page_tiles_kernel(const Call a, const Pages p, const int64_t *__restrict__ masks, void *out, float *partial,
                                                            int splits, int row_tiles)
{
    constexpr int TR = ROWS, PARTS = 8 / RG, NB = RING<T, D, DV, RG>, AHEAD = NB - 1, TILE = PAGE_TILE<T, D, DV>, AR = 4, ACC = DV / TR * AR, NK = D / KS<T, TR>;
    typedef Swizzled<T, 2 * D, false> KeyTile;
    typedef Swizzled<T, DV, true> ValueTile;
    constexpr int LOADS = (KeyTile::LOADS + ValueTile::LOADS + RG - 1) / RG;            // of a wave, for a tile
    static_assert(NB >= 2 && AHEAD * LOADS < 64, "a tile on its way, and all of them counted");
    constexpr int TILES_AT = PARTS * NB * TILE, JOIN_AT = (PARTS - 1) * RG * 2 * 64 * ACC * 4;
    __shared__ __attribute__((aligned(1024))) unsigned char lds[TILES_AT > JOIN_AT ? TILES_AT : JOIN_AT];
    __shared__ float tops[PARTS][2][RG][TR], sums[PARTS][2][RG][TR];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), part = wave / RG, group = wave % RG, lane = threadIdx.x & 63, heads = a.B * a.Hkv;
    const int bh = blockIdx.x % heads, rest_id = blockIdx.x / heads, tile = row_tiles - 1 - rest_id % row_tiles, split = rest_id / row_tiles;
    const int b = bh / a.Hkv, hk = bh % a.Hkv;
    const int length = uniform(length_of(p, b)), count = uniform(count_of(p, b, a.Lq)), room = p.slots * p.S;
    const int first = (tile * RG + group) * TR, row = first + lane_row<TR>();
    const int query = row < a.R ? row / a.G : 0;
    const bool there = row < a.R && query < count;
    const uint64_t mask = masks && there ? (uint64_t)masks[(int64_t)b * a.Lq + query] : 0;
    const int limit = there ? length + (masks ? count : query + 1) : 0;
    // keys that rows from .. last see at most: none where the first of them is no query
    const auto reach = [&](int from, int last) {
        const int q = (last < a.R ? last : a.R - 1) / a.G;
        const int n = length + (masks || q + 1 > count ? count : q + 1);
        return from >= a.R || from / a.G >= count ? 0 : n < room ? n : room;
    };
    const int wave_any = reach(first, first + TR - 1), any = reach(tile * RG * TR, (tile + 1) * RG * TR - 1);
    // and those that every row of the wave sees (rows that are none see what they like)
    const int wave_all = masks || wave_any == 0 ? length : length + first / a.G + 1;
    // the workgroup's tiles, and this part's; parts differ by one tile at most, the first ones having more
    const int tiles = (any + KT - 1) / KT, per = (tiles + splits - 1) / splits, from = split * per < tiles ? split * per : tiles;
    const int mine = from + per < tiles ? per : tiles - from, most = (mine + PARTS - 1) / PARTS;
    const int begin = from + (part * mine + PARTS - 1) / PARTS, number = from + ((part + 1) * mine + PARTS - 1) / PARTS - begin;

    const Source<T> qs{static_cast<const T *>(a.q) + b * a.qb + (int64_t)hk * a.G * a.qh, a.ql, a.qh, a.qm, a.G, a.d, a.inverse};
    Frag<T> q[2][NK];
#pragma unroll
    for (int m = 0; m < 2; ++m) load_rows<T, TR, D>(qs, row, there, m, q[m]);
    const float c = a.scale * LOG2E;
    State<T, TR, D, DV, true> state;
    state.clear();
    if (a.d < D || a.dv < DV) {
        typedef uint32_t words __attribute__((ext_vector_type(4)));
        for (int i = threadIdx.x * 16; i < TILES_AT; i += 512 * 16) *reinterpret_cast<words *>(lds + i) = words{0, 0, 0, 0};
        __syncthreads();
    }

    // A tile on its way.  Whole ones take every row as it is; of another one, rows past the last key are the last key's, and a half that is not there is the other one's rows.
    unsigned char *const ring = lds + part * NB * TILE;
    Walk walk(p, b, hk, begin * KT);
    uint32_t offset[LOADS];                     // of a lane's piece of a whole tile, in its half's rows
    bool mine_there[LOADS];
    const auto place = [&](int i, bool &value, int &second, int &r, int &column) __attribute__((always_inline)) {
        const int n = (i * RG + group) % (KeyTile::LOADS + ValueTile::LOADS);           // a wave that has none left loads another one's again
        value = n >= KeyTile::LOADS;
        const int at = (value ? n - KeyTile::LOADS : n) * 1024, bytes = (value ? DV : 2 * D) * (int)sizeof(T);          // of a row of LDS
        const int row_of_tile = (at + lane * 16) / bytes, spot = (at + lane * 16) % bytes / 16;
        const int chunk = spot ^ (value ? ValueTile::turn(row_of_tile) : KeyTile::turn(row_of_tile));
        const int map = value ? 0 : chunk / (D / FE<T>), col = (value ? chunk : chunk % (D / FE<T>)) * FE<T>;
        second = at / bytes / 16;
        r = row_of_tile & 15;
        column = map * a.d + col;
        return col < (value ? a.dv : a.d);
    };
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
        bool value;
        int second, r, column;
        mine_there[i] = place(i, value, second, r, column);
        offset[i] = (uint32_t)(r * (value ? a.dv : 2 * a.d) + column);
    }
    uint32_t ways = 0;                          // of the tiles from the one in use on, two bits each: which halves of them there are
    int from_ring = 0, to_ring = 0;             // where the tile in use and the next one to load stand
    const auto load = [&](int t, int ahead) __attribute__((always_inline)) {
        const int64_t row0 = walk.next(), row1 = walk.next();
        const int left = any - t * KT;          // keys of the tile
        const uint32_t halves = (row0 < 0 ? 0u : 1u) | (row1 < 0 || left <= 16 ? 0u : 2u);
        ways |= halves << 2 * ahead;
        unsigned char *const to = ring + to_ring * TILE;
        to_ring = to_ring + 1 < NB ? to_ring + 1 : 0;
        if (halves == 3 && left >= KT) {
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {
                const int n = (i * RG + group) % (KeyTile::LOADS + ValueTile::LOADS);
                const bool value = n >= KeyTile::LOADS;
                const int second = (value ? n - KeyTile::LOADS : n) * 1024 / ((value ? DV : 2 * D) * (int)sizeof(T)) / 16;
                const T *base = static_cast<const T *>(value ? p.v : p.k) + (second ? row1 : row0) * (value ? a.dv : 2 * a.d);
                if (mine_there[i]) __builtin_amdgcn_global_load_lds((global_pointer)(base + offset[i]), (lds_pointer)(to + n * 1024), 16, 0, 0);
            }
        } else {
            const int64_t rows0 = halves & 1 ? row0 : halves ? row1 : 0, rows1 = halves & 2 ? row1 : rows0;
            const int end0 = halves == 2 ? left - 16 : left, end1 = halves & 2 ? left - 16 : left;
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {
                bool value;
                int second, r, column;
                const bool there_too = place(i, value, second, r, column);
                const int n = (i * RG + group) % (KeyTile::LOADS + ValueTile::LOADS), end = second ? end1 : end0;
                const T *base = static_cast<const T *>(value ? p.v : p.k) + (second ? rows1 : rows0) * (value ? a.dv : 2 * a.d);
                const uint32_t off = (uint32_t)((r < end ? r : end - 1) * (value ? a.dv : 2 * a.d) + column);
                if (there_too) __builtin_amdgcn_global_load_lds((global_pointer)(base + off), (lds_pointer)(to + n * 1024), 16, 0, 0);
            }
        }
    };
    for (int i = 0; i < AHEAD && i < number; ++i) load(begin + i, i);

    // A tile's part of the loop, with `use` what a wave does that sees some of its keys.  Waves that are past their keys go on loading for the others, in a loop of its own
    // (a condition around the products has the accumulators copied in every tile).
    int i = 0;
    const auto tile_of = [&](const auto &use) __attribute__((always_inline)) {
        if (i + AHEAD <= number) wait_and_meet<(AHEAD - 1) * LOADS>();
        else wait_and_meet<0>();
        const uint32_t halves = ways & 3;
        ways >>= 2;
        if (i + AHEAD < number) load(begin + i + AHEAD, AHEAD - 1);         // where the last tile stood: every wave is past it
        use((begin + i) * KT, halves, ring + from_ring * TILE);
        from_ring = from_ring + 1 < NB ? from_ring + 1 : 0;
        ++i;
    };
    const int open = (wave_all < wave_any ? wave_all : wave_any) / KT - begin, seen = (wave_any + KT - 1) / KT - begin;
    while (i < number && i < open && (ways & 3) == 3)
        tile_of([&](int, uint32_t, const unsigned char *t) { page_keys<false, T, D, DV>(state, q, t, c, 0, 0); });
    while (i < number && i < seen)
        tile_of([&](int key, uint32_t halves, const unsigned char *t) {
            const uint32_t word = (masks ? seen_word(key, length, mask) : 0xffffffffu) & ((halves & 1 ? 0xffffu : 0u) | (halves & 2 ? 0xffff0000u : 0u));
            if (halves) page_keys<true, T, D, DV>(state, q, t, c, limit - key, word);
        });
    while (i < most) tile_of([](int, uint32_t, const unsigned char *) {});

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
        constexpr int WAVE = 2 * 64 * ACC;
        if (part) {
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                if (lane_group<TR>() == 0) {
                    tops[part][m][group][lane_row<TR>()] = state.top[m];
                    sums[part][m][group][lane_row<TR>()] = total[m];
                }
#pragma unroll
                for (int n = 0; n < ACC; ++n) cells[((part - 1) * RG + group) * WAVE + (m * ACC + n) * 64] = state.o[m][n / AR][n % AR];
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
                    const float y = sum == 0.0f ? 0.0f : cells[((other - 1) * RG + group) * WAVE + (m * ACC + n) * 64] * more;
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
    if (row >= a.R) return;
    if (splits == 1) {
        const int head = hk * a.G + row - query * a.G;
        const float lam = lambda_of(a, head, static_cast<const T *>(nullptr));
        float factor[2];
#pragma unroll
        for (int m = 0; m < 2; ++m) factor[m] = total[m] > 0.0f ? 1.0f / total[m] : 0.0f;
        T *to = static_cast<T *>(out) + (((int64_t)b * a.Lq + query) * a.H + head) * a.dv;
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
        float *to = partial + (((int64_t)split * a.B * a.Hkv + bh) * a.R + row) * (2 * (int64_t)a.dv + 4);
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

// How a call runs: row groups of a workgroup's tiles (0: rows are streamed), workgroups that share a row's keys.
struct Plan { int groups, splits; };

// The fewest row groups whose rings have room, and registers for the widest heads (16 bits: 8 groups; fp32: none, 0).
template <class T, int D, int DV>
constexpr int FEWEST_GROUPS = DV > 128 ? sizeof(T) == 2 ? 8 : 0 : RING<T, D, DV, 2> >= 2 ? 2 : RING<T, D, DV, 4> >= 2 ? 4 : 8;

template <class T>
struct Fewest {
    template <int D, int DV>
    int operator()() const { return FEWEST_GROUPS<T, D, DV>; }
};

// Tiles where a key head has more rows than a wave streams: as few row groups as hold them and as the ring's tiles leave room for.  Heads that end inside 16 bytes are streamed.
inline int row_groups(const Call &a, const Pages &p, int type)
{
    if (a.R <= FEW || !a.fast || p.P == 0) return 0;
    const int fewest = type == MAM_F32 ? with_head_sizes(a.d, a.dv, Fewest<float>()) : with_head_sizes(a.d, a.dv, Fewest<bf16>());
    const int want = a.R <= 2 * ROWS ? 2 : a.R <= 4 * ROWS ? 4 : 8;
    return fewest == 0 ? 0 : want < fewest ? fewest : want;
}

// Workgroups that share a row's keys: two a CU over the whole call, but 64 keys a wave at least of what a request has room for; of the tiles' eight waves one a CU.
inline Plan plan_of(const Call &a, const Pages &pages, int type)
{
    Plan p{row_groups(a, pages, type), 1};
    const int64_t rows = (int64_t)a.B * a.Hkv * ceil_div(a.R, p.groups ? p.groups * ROWS : ROWS), most = ceil_div(a.Lk, 4 * 64);
    int64_t n = p.groups ? kNumCU / (rows > 0 ? rows : 1) : ceil_div(2 * (int64_t)kNumCU, rows);
    if (n > 64) n = 64;
    if (n > most) n = most;
    p.splits = n < 1 ? 1 : (int)n;
    return p;
}

inline size_t pages_workspace(const Call &a, const Pages &p, int type)
{
    const int n = plan_of(a, p, type).splits;
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
    template <int D, int DV, int RG>
    int tiles(dim3 grid, int row_tiles) const
    {
        if constexpr (FEWEST_GROUPS<T, D, DV> > 0 && RG >= FEWEST_GROUPS<T, D, DV>)
            hipLaunchKernelGGL((page_tiles_kernel<T, D, DV, RG>), grid, dim3(512), 0, st, a, p, masks, out, partial, plan.splits, row_tiles);
        return check_launch("attention::page_tiles_kernel");
    }
    template <int D, int DV>
    int operator()() const
    {
        const int64_t row_tiles = ceil_div(a.R, plan.groups ? plan.groups * ROWS : ROWS), blocks = row_tiles * a.B * a.Hkv * plan.splits;
        if (blocks > INT32_MAX) return fail(MAM_ERR_UNSUPPORTED, "too many tiles");
        const dim3 grid((unsigned)blocks);
        if (plan.groups == 8) return tiles<D, DV, 8>(grid, (int)row_tiles);
        if (plan.groups == 4) return tiles<D, DV, 4>(grid, (int)row_tiles);
        if (plan.groups == 2) return tiles<D, DV, 2>(grid, (int)row_tiles);
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
    return attention::pages_workspace(a, p, args->pages.type);
}

extern "C" int mam_diff_attention_pages(const mam_diff_attention_pages_t *args, void *out, void *workspace, size_t workspace_bytes, void *stream)
{
    using namespace mam;
    attention::Call a;
    Pages p;
    int rc = attention::fill_pages_call(args, a, p);
    if (rc != MAM_OK || a.B == 0 || a.R == 0) return rc;
    if (!a.q || !a.lam || !out || (p.P > 0 && (!p.k || !p.v))) return fail(MAM_ERR_INVALID_ARGUMENT, "null pointer");
    const size_t need = attention::pages_workspace(a, p, args->pages.type);
    if (need > 0 && (!workspace || workspace_bytes < need))
        return fail(MAM_ERR_WORKSPACE, "the attention needs %zu workspace bytes, got %zu", need, workspace ? workspace_bytes : (size_t)0);
    hipStream_t st = static_cast<hipStream_t>(stream);
    float *partial = need > 0 ? static_cast<float *>(workspace) : nullptr;
    const attention::Plan plan = attention::plan_of(a, p, args->pages.type);
    if (args->pages.type == MAM_F32) rc = attention::with_head_sizes(a.d, a.dv, attention::PagesRun<float>{a, p, args->masks, out, partial, plan, st});
    else if (args->pages.type == MAM_BF16) rc = attention::with_head_sizes(a.d, a.dv, attention::PagesRun<bf16>{a, p, args->masks, out, partial, plan, st});
    else rc = attention::with_head_sizes(a.d, a.dv, attention::PagesRun<f16>{a, p, args->masks, out, partial, plan, st});
    if (rc != MAM_OK || need == 0) return rc;
    return attention::join_parts(a, args->pages.type, out, partial, plan.splits, st);
}
