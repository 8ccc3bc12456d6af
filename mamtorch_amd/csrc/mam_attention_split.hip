// Differential attention for few queries over many keys: single tokens over a cache, short prompts behind a long one.
//
// Bound by reading K and V once.  A wave takes 16 rows (queries times the heads that share a key head) and a range of the keys; nothing of the loop
// goes through LDS and no wave waits for another, so eight waves a CU keep 128 KiB on their way.  Keys are read as the fragments of
// the first product: 16 keys of 64 bytes a load.  Values are read by rows as well, a lane DV / 16 elements of 8 keys, and the second
// product's rows are taken in the order that this gives: row r of product j is element DV / 16 * r + j, so that its fragment is element j of
// the lane's 8 keys, put together by one byte permutation for two of them (16-bit types) or as it is (fp32).
//
// The ranges of a row meet in two steps, both in a fixed order: the four waves of a workgroup through LDS, and the workgroups through
// the workspace and a second kernel where one workgroup a row would leave CUs without work.
//
// Measured: one token of 16 requests over caches of up to 16384 (200704 keys in all, 4 key heads of 64/128, 4 query heads each, bf16, 411 MB) 95 us, 4.3 TB/s, and 6 us
// for the join; a large copy reaches 5.2 TB/s.  16 queries, 8 heads, over 8192 keys 13 and 11 us.
#include "mam_attention.h"

namespace mam {
namespace attention {

constexpr int ROWS = 16;                // rows of a wave
constexpr float SLACK = 8.0f;           // see mam_attention.hip

// Workgroups that share a row's keys: two a CU over the whole call, but 64 keys a wave at least.
inline int split_count(const Call &a)
{
    const int64_t rows = (int64_t)a.B * a.Hkv * ceil_div(a.R, ROWS), most = ceil_div(a.Lk, 4 * 64);
    int64_t n = ceil_div(2 * (int64_t)kNumCU, rows);
    if (n > 64) n = 64;
    if (n > most) n = most;
    return n < 1 ? 1 : (int)n;
}

// Rows of one tile always; more where the call's tiles of 16 rows are two a CU at most, one in 16-bit types of heads past 64: there the tiles' kernels,
// which pass over all keys in every workgroup, leave CUs and their waves idle, and here every tile reads the keys for itself.  Both measured, tiles' -> here:
// bf16 64/128 over 4096 keys 512 tiles 185..197 -> 84..122 us, 1024 tiles 191 -> 160 to 225 -> 369; 128/256 256 tiles 243 -> 156, 384 tiles 121 -> 154 (2048
// keys), 512 tiles 243 -> 245; fp32 64/128 over 1024 keys 512 tiles 120 -> 97, 1024 tiles 131 -> 205; 128/256 512 tiles 945 -> 714 (causal).  Few keys
// leave a wave too few of them: fp32, 312 tiles over 197 keys 30 -> 39 us.  16 queries of 2048 (request, head) pairs over 512 keys, bf16: 152 -> 111 us.
bool use_split(const Call &a, int type, bool keep)
{
    if (keep || a.Lk < 1) return false;
    const int64_t tiles = (int64_t)a.B * a.Hkv * ceil_div(a.R, ROWS);
    return a.R <= ROWS || (a.Lk >= 512 && tiles <= (type == MAM_F32 || (a.d <= 64 && a.dv <= 128) ? 2 : 1) * kNumCU);
}

// A partial row: both maps' products relative to their maxima, then maximum and sum of each.
inline int64_t partial_size(const Call &a) { return 2 * (int64_t)a.dv + 4; }

size_t split_workspace(const Call &a)
{
    const int n = split_count(a);
    return n > 1 ? (size_t)n * a.B * a.Hkv * a.R * partial_size(a) * sizeof(float) : 0;
}

// Elements PE of a lane's values of a key, as words.
template <class T, int PE>
__device__ __forceinline__ void value_piece(const T *base, uint32_t offset, bool fast, const T *slow, int left, uint32_t *w)
{
    constexpr int BYTES = PE * (int)sizeof(T);
    if (fast) {
        const auto rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<T *>(base), 0, 0x7fffffff, 0x00027000);
        if constexpr (BYTES == 16) {
            typedef uint32_t words __attribute__((ext_vector_type(4)));
            const words t = __builtin_amdgcn_raw_buffer_load_b128(rsrc, (int)offset, 0, 0);
#pragma unroll
            for (int u = 0; u < 4; ++u) w[u] = t[u];
        } else {
            typedef uint32_t words __attribute__((ext_vector_type(2)));
            const words t = __builtin_amdgcn_raw_buffer_load_b64(rsrc, (int)offset, 0, 0);
#pragma unroll
            for (int u = 0; u < 2; ++u) w[u] = t[u];
        }
    } else {
        T e[PE];
#pragma unroll
        for (int u = 0; u < PE; ++u) e[u] = (T)0.0f;
        if (left >= PE) {
            const typename Pack<T, PE>::type t = *reinterpret_cast<const typename Pack<T, PE>::type *>(slow);
#pragma unroll
            for (int u = 0; u < PE; ++u) e[u] = t[u];
        } else {
#pragma unroll
            for (int u = 0; u < PE; ++u)
                if (u < left) e[u] = slow[u];
        }
        __builtin_memcpy(w, e, BYTES);
    }
}

template <class T, int D, int DV, bool FAST>
__global__ __launch_bounds__(256, D > 64 || (sizeof(T) == 4 && DV > 64) ? 1 : 2) void split_kernel(const Call a, void *out, float *partial, int splits, int row_tiles)
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
    const Reach reach = reach_of(a, b);
    const int row = tile * ROWS + lane_row<TR>();
    const bool there = row < a.R;
    const int query = there ? row / a.G : 0;
    const int limit = there ? reach.of_query(query) : 0;
    const int first_row = tile * ROWS, last_row = first_row + ROWS - 1 < a.R ? first_row + ROWS - 1 : a.R - 1;
    const int all = reach.of_query(first_row / a.G), any = reach.of_query(last_row / a.G);
    // this wave's keys: whole tiles of 32, as even as they come
    const int per = ((any + 31) / 32 + 4 * splits - 1) / (4 * splits) * 32;
    const int64_t begin64 = (int64_t)per * (split * 4 + wave);
    const int begin = begin64 < any ? (int)begin64 : any, end = begin64 + per < any ? (int)(begin64 + per) : any;

    const Source<T> qs{static_cast<const T *>(a.q) + b * a.qb + (int64_t)hk * a.G * a.qh, a.ql, a.qh, a.qm, a.G, a.d, a.inverse};
    const T *keys = static_cast<const T *>(a.k) + b * a.kb + hk * a.kh, *values = static_cast<const T *>(a.v) + b * a.vb + hk * a.vh;
    const int lane = lane_row<TR>(), group = lane_group<TR>();
    Frag<T> q[2][NK];
#pragma unroll
    for (int m = 0; m < 2; ++m) load_rows<T, TR, D>(qs, row, there, m, q[m]);
    const float c = a.scale * LOG2E;
    const auto seen = [&](int key) { return key < end && (FAST || !a.mask || a.mask[b * a.mask_b + key] != 0); };

    Frag<T> k[2][BLOCKS<TR>][NK];
    const auto load_keys = [&](int first) {
        const T *base = keys + (int64_t)first * a.kl;
#pragma unroll
        for (int blk = 0; blk < BLOCKS<TR>; ++blk) {
            const int at = blk * TR + lane;
            const bool ok = seen(first + at);
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int kk = 0; kk < NK; ++kk) {
                    const int col = kk * KS<T, TR> + FE<T> * group;
                    if constexpr (FAST) {
                        const uint32_t off = ((uint32_t)at * (uint32_t)a.kl + (uint32_t)col) * (uint32_t)sizeof(T);
                        k[m][blk][kk] = buffer_frag<T>(base + m * a.km, ok && col < a.d ? off : NOWHERE);
                    } else {
#pragma unroll
                        for (int u = 0; u < FE<T>; ++u) k[m][blk][kk][u] = (T)0.0f;
                        if (ok && col < a.d) k[m][blk][kk] = load_frag<T>(base + m * a.km + (int64_t)at * a.kl + col, a.d - col);
                    }
                }
        }
    };
    uint32_t v[REGS<TR>][WORDS];
    const auto load_values = [&](int first) {
        const T *base = values + (int64_t)first * a.vl;
#pragma unroll
        for (int f = 0; f < REGS<TR>; ++f) {
            const int at = index_of<TR>(f);
            const bool ok = seen(first + at);
#pragma unroll
            for (int p = 0; p < PIECES; ++p) {
                const int col = E * lane + p * PE;
                const bool in = ok && col < a.dv;
                const uint32_t off = ((uint32_t)at * (uint32_t)a.vl + (uint32_t)col) * (uint32_t)sizeof(T);
                value_piece<T, PE>(base, in ? off : NOWHERE, FAST, base + (int64_t)at * a.vl + col, in ? a.dv - col : 0, &v[f][p * PW]);
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
    if (begin < end) load_keys(begin);
    for (int key = begin; key < end; key += 32) {
        if (EARLY) load_values(key);
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
        const int next = key + 32 < end ? key + 32 : key;       // past the range: the last keys again, not used
        if (EARLY) load_keys(next);
        else load_values(key);
        const bool limited = key + 32 > all || key + 32 > end || (!FAST && a.mask);
        const uint32_t word = !FAST && a.mask ? mask_word(a, b, key) : 0xffffffffu;
        const int most_keys = (limit < end ? limit : end) - key;
        Frag<T> frag[2][FRAGS<T, TR>], rest[FRAGS<T, TR>];
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            float p[REGS<TR>], most = -INFINITY;
#pragma unroll
            for (int f = 0; f < REGS<TR>; ++f) {
                p[f] = s[m][f / 4][f % 4];
                if (limited) {
                    const int at = index_of<TR>(f);
                    p[f] = at < most_keys && (word >> at & 1) ? p[f] : -INFINITY;
                }
                most = fmaxf(most, p[f]);
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
                p[f] = __builtin_amdgcn_exp2f(fmaf(p[f], c, -base));
                sum[m] += p[f];
            }
            to_frags<T, TR>(p, frag[m]);
            // What 16 bits leave of the first map's probabilities, as a product of its own.  The second map, which lambda weighs down, goes without: 0.0019 against
            // 64 bits in bf16 where fp32 probabilities give 0.0017.
            if (PARTS == 2 && m == 0) {
#pragma unroll
                for (int f = 0; f < REGS<TR>; ++f) p[f] -= element(frag[0][f / FE<T>], f % FE<T>);
                to_frags<T, TR>(p, rest);
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
        if (!EARLY) load_keys(next);
    }

    // the four waves' ranges
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        sum[m] = groups_sum<TR>(sum[m]);
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
        T *p = static_cast<T *>(out) + (((int64_t)b * a.Lq + i) * a.H + h) * a.dv;
        for (int col = 4 * place; col < a.dv; col += 64) {
            float r[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) r[u] = fmaf(-lam, joined[1][mine][col + u] * inv[1], joined[0][mine][col + u] * inv[0]);
            store_pack<T, 4>(p + col, a.dv - col, r);
        }
    } else {
        float *p = partial + (((int64_t)split * a.B * a.Hkv + bh) * a.R + out_row) * (2 * (int64_t)a.dv + 4);
        for (int m = 0; m < 2; ++m)
            for (int col = place; col < a.dv; col += 16) p[m * a.dv + col] = joined[m][mine][col];
        if (place < 2) {
            p[2 * a.dv + 2 * place] = m_top[place];
            p[2 * a.dv + 2 * place + 1] = m_sum[place];
        }
    }
}

// The workgroups' parts of a row, a wave a row.
template <class T>
__global__ __launch_bounds__(256) void join_kernel(const Call a, void *out, const float *__restrict__ partial, int splits)
{
    const int64_t rows = (int64_t)a.B * a.Hkv * a.R, id = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (id >= rows) return;
    const int lane = threadIdx.x & 63, row = (int)(id % a.R), bh = (int)(id / a.R), b = bh / a.Hkv;
    const int query = row / a.G, head = bh % a.Hkv * a.G + row - query * a.G;
    const int64_t size = 2 * (int64_t)a.dv + 4, step = rows * size;
    const float *p = partial + id * size;
    // lane s holds split s's maxima and sums (splits <= 64)
    float factor[2];
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        float top = -INFINITY, sum = 0.0f;
        if (lane < splits) {
            top = p[lane * step + 2 * a.dv + 2 * m];
            sum = p[lane * step + 2 * a.dv + 2 * m + 1];
        }
        float most = top;
#pragma unroll
        for (int x = 1; x < 64; x <<= 1) most = fmaxf(most, __shfl_xor(most, x));
        const float mine = most == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(top - most);
        float total = sum * mine;
#pragma unroll
        for (int x = 1; x < 64; x <<= 1) total += __shfl_xor(total, x);
        factor[m] = total > 0.0f ? mine / total : 0.0f;
    }
    const float lam = lambda_of(a, head, static_cast<const T *>(nullptr));
    const int left = a.dv - 4 * lane;
    float r[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    constexpr int AHEAD = 8;            // parts on their way at once
    for (int s0 = 0; s0 < splits; s0 += AHEAD) {        // every lane stays to the end: each has a split's factors
        float p1[AHEAD][4], p2[AHEAD][4];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const float *t = p + (s0 + u < splits ? s0 + u : splits - 1) * step + 4 * lane;
            load_pack<float, 4>(t, left, p1[u]);
            load_pack<float, 4>(t + a.dv, left, p2[u]);
        }
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const int s = s0 + u;
            const float f0 = s < splits ? __shfl(factor[0], s) : 0.0f, f1 = s < splits ? -lam * __shfl(factor[1], s) : 0.0f;
#pragma unroll
            for (int e = 0; e < 4; ++e) r[e] = fmaf(f1, p2[u][e], fmaf(f0, p1[u][e], r[e]));
        }
    }
    if (left > 0)
        store_pack<T, 4>(static_cast<T *>(out) + (((int64_t)b * a.Lq + query) * a.H + head) * a.dv + 4 * lane, left, r);
}

template <class T>
struct Split {
    const Call &a;
    void *out;
    float *partial;
    int splits;
    hipStream_t st;
    template <int D, int DV>
    int operator()() const
    {
        const int64_t row_tiles = ceil_div(a.R, ROWS), blocks = row_tiles * a.B * a.Hkv * splits;
        if (blocks > INT32_MAX) return fail(MAM_ERR_UNSUPPORTED, "too many tiles");
        const dim3 grid((unsigned)blocks);
        if (a.fast) hipLaunchKernelGGL((split_kernel<T, D, DV, true>), grid, dim3(256), 0, st, a, out, partial, splits, (int)row_tiles);
        else hipLaunchKernelGGL((split_kernel<T, D, DV, false>), grid, dim3(256), 0, st, a, out, partial, splits, (int)row_tiles);
        int rc = check_launch("attention::split_kernel");
        if (rc != MAM_OK || splits == 1) return rc;
        hipLaunchKernelGGL((join_kernel<T>), dim3((unsigned)ceil_div((int64_t)a.B * a.Hkv * a.R, 4)), dim3(256), 0, st, a, out, partial, splits);
        return check_launch("attention::join_kernel");
    }
};

int run_split(const Call &a, int type, void *out, void *workspace, size_t workspace_bytes, hipStream_t st)
{
    const size_t need = split_workspace(a);
    if (need > 0 && (!workspace || workspace_bytes < need))
        return fail(MAM_ERR_WORKSPACE, "the attention needs %zu workspace bytes, got %zu", need, workspace ? workspace_bytes : (size_t)0);
    const int splits = split_count(a);
    float *partial = static_cast<float *>(workspace);
    if (type == MAM_F32) return with_head_sizes(a.d, a.dv, Split<float>{a, out, partial, splits, st});
    if (type == MAM_BF16) return with_head_sizes(a.d, a.dv, Split<bf16>{a, out, partial, splits, st});
    return with_head_sizes(a.d, a.dv, Split<f16>{a, out, partial, splits, st});
}

}  // namespace attention
}  // namespace mam
