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
constexpr float SLACK = 8.0f;           // see mam_attention.hip

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

// Workgroups that share a row's keys: two a CU over the whole call, but 64 keys a wave at least of what a request has room for.
inline int pages_split_count(const Call &a)
{
    const int64_t rows = (int64_t)a.B * a.Hkv * ceil_div(a.R, ROWS), most = ceil_div(a.Lk, 4 * 64);
    int64_t n = ceil_div(2 * (int64_t)kNumCU, rows);
    if (n > 64) n = 64;
    if (n > most) n = most;
    return n < 1 ? 1 : (int)n;
}

inline size_t pages_workspace(const Call &a)
{
    const int n = pages_split_count(a);
    return n > 1 ? (size_t)n * a.B * a.Hkv * a.R * partial_size(a) * sizeof(float) : 0;
}

template <class T>
struct PagesRun {
    const Call &a;
    const Pages &p;
    const int64_t *masks;
    void *out;
    float *partial;
    hipStream_t st;
    template <int D, int DV>
    int operator()() const
    {
        const int splits = pages_split_count(a);
        const int64_t row_tiles = ceil_div(a.R, ROWS), blocks = row_tiles * a.B * a.Hkv * splits;
        if (blocks > INT32_MAX) return fail(MAM_ERR_UNSUPPORTED, "too many tiles");
        const dim3 grid((unsigned)blocks);
        if (a.fast) hipLaunchKernelGGL((pages_kernel<T, D, DV, true>), grid, dim3(256), 0, st, a, p, masks, out, partial, splits, (int)row_tiles);
        else hipLaunchKernelGGL((pages_kernel<T, D, DV, false>), grid, dim3(256), 0, st, a, p, masks, out, partial, splits, (int)row_tiles);
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
    return attention::pages_workspace(a);
}

extern "C" int mam_diff_attention_pages(const mam_diff_attention_pages_t *args, void *out, void *workspace, size_t workspace_bytes, void *stream)
{
    using namespace mam;
    attention::Call a;
    Pages p;
    int rc = attention::fill_pages_call(args, a, p);
    if (rc != MAM_OK || a.B == 0 || a.R == 0) return rc;
    if (!a.q || !a.lam || !out || (p.P > 0 && (!p.k || !p.v))) return fail(MAM_ERR_INVALID_ARGUMENT, "null pointer");
    const size_t need = attention::pages_workspace(a);
    if (need > 0 && (!workspace || workspace_bytes < need))
        return fail(MAM_ERR_WORKSPACE, "the attention needs %zu workspace bytes, got %zu", need, workspace ? workspace_bytes : (size_t)0);
    hipStream_t st = static_cast<hipStream_t>(stream);
    float *partial = need > 0 ? static_cast<float *>(workspace) : nullptr;
    if (args->pages.type == MAM_F32) rc = attention::with_head_sizes(a.d, a.dv, attention::PagesRun<float>{a, p, args->masks, out, partial, st});
    else if (args->pages.type == MAM_BF16) rc = attention::with_head_sizes(a.d, a.dv, attention::PagesRun<bf16>{a, p, args->masks, out, partial, st});
    else rc = attention::with_head_sizes(a.d, a.dv, attention::PagesRun<f16>{a, p, args->masks, out, partial, st});
    if (rc != MAM_OK || need == 0) return rc;
    return attention::join_parts(a, args->pages.type, out, partial, attention::pages_split_count(a), st);
}
