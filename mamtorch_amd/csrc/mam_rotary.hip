// Norms of queries and keys for each head with the position rotation in the same pass, their gradients, and their serving form, which puts keys and values
// into the pages of a cache (mam_pages.h).
//
// y = R(p) (x / sqrt(mean(x^2) + eps) * w) for each row of D elements, R(p) turning pair i of the first 2 `pairs` by p * frequency[i].  The
// gradient turns back first, g = R(-p) dy, then dw = sum g xh and dx = rstd (g w - xh mean(g w xh)) with xh = x rstd, which is formed again: x is read anyway.
//
// Bound by memory, so that nothing else may take its time: a token's angles are the same for all of its rows, and a workgroup forms them once, in LDS.  They are formed in
// fp64 and reduced in whole turns before fp32 takes over: an fp32 angle at place 500000 would be off by up to 0.03.
//
// A row is held by `lanes` lanes (a power of 2), each with V pairs: elements s and s + pairs where pairs are halves of the turned part, 2 s and 2 s + 1 where they are
// neighbours and behind the turned part.  So both elements of a pair are in one lane, and a lane loads and stores 16 bytes at a time but where a part ends inside its V.
#include "mam_pages.h"
#include "mam_types.h"

namespace mam {
namespace rotary {

constexpr int MOST_TOKENS = 16, MOST_PAIRS = 64, THREADS = 256;

struct Side {
    const void *x, *weight, *dy;
    void *out;
    int64_t b, l, h, m, db, dl, dh, dm;     // strides of x and of dy
    int heads, tokens, groups;              // tokens of a workgroup's turn, workgroups
};

struct Call {
    Side side[2];                           // queries, keys
    const double *frequencies;
    const int32_t *positions;
    int64_t pb, pl;
    int L, M, D, pairs, norm, interleaved, same, lanes;             // lanes of a row
    int64_t all;                            // tokens of the call
    float eps, inverse;                     // inverse: 1 / D
};

// Where a call's keys and values go; the values have workgroups of their own.
struct Append {
    Pages to;
    const void *v;
    int64_t vb, vl, vh;
    int tokens, groups;
};

template <class T>
constexpr int V = kPack<T>;

// A lane's pairs of a row, first elements in a, second ones in b.  Behind the turned part it does not matter which elements are a pair: where pairs are halves, a lane there has
// its elements in two pieces as well, so that only neighbours (MIXED) are sorted in registers.
template <class T, bool MIXED>
struct Slots {
    enum Kind { WHOLE, SINGLE, NONE };
    int first, pairs, D, at, next;          // at, next: a lane's two pieces where both are whole
    Kind kind;

    __device__ __forceinline__ Slots(const Call &c, int lane) : first(lane * V<T>), pairs(MIXED ? 0 : c.pairs), D(c.D)
    {
        const bool halves = first + V<T> <= pairs, behind = first >= pairs && 2 * (first + V<T>) <= D;
        kind = halves || behind ? WHOLE : 2 * first < D || first < pairs ? SINGLE : NONE;
        at = halves ? first : 2 * first;
        next = halves ? first + pairs : 2 * first + V<T>;
    }
    // elements of the lane's pair u, and of place u of its pieces; D and beyond: none
    __device__ __forceinline__ int one(int u) const
    {
        if (kind == WHOLE) return MIXED ? at + 2 * u : at + u;
        return kind == NONE ? D : single(first, u, 0);
    }
    __device__ __forceinline__ int other(int u) const
    {
        if (kind == WHOLE) return MIXED ? at + 2 * u + 1 : next + u;
        return kind == NONE ? D : single(first, u, 1);
    }
    __device__ __forceinline__ int single(int from, int u, int second) const
    {
        return from + u < pairs ? from + u + second * pairs : 2 * (from + u) + second;
    }
    __device__ __forceinline__ int place(int from, int u, int second) const { return MIXED ? 2 * from + second * V<T> + u : single(from, u, second); }
    // Where a row ends inside a lane's pieces: addresses are formed where they are used, not kept for the loop in registers that all lanes would need.
    __device__ __forceinline__ int here() const
    {
        int f = first;
        asm volatile("" : "+v"(f));
        return f;
    }

    // As they stand in memory: whole pieces where they are; else in that order too, one by one.
    __device__ __forceinline__ void load(const T *p, Raw<T> &x, Raw<T> &y) const
    {
        if (kind == WHOLE) {
            x = *reinterpret_cast<const Raw<T> *>(p + at);
            y = *reinterpret_cast<const Raw<T> *>(p + next);
        } else if (kind == SINGLE) {
            const int f = here();
#pragma unroll
            for (int u = 0; u < V<T>; ++u) {
                const int i = place(f, u, 0), j = place(f, u, 1);
                x[u] = i < D ? p[i] : (T)0.0f;
                y[u] = j < D ? p[j] : (T)0.0f;
            }
        } else {
#pragma unroll
            for (int u = 0; u < V<T>; ++u) x[u] = y[u] = (T)0.0f;
        }
    }
    __device__ __forceinline__ void spread(const Raw<T> &x, const Raw<T> &y, float (&a)[V<T>], float (&b)[V<T>]) const
    {
        constexpr int H = V<T> / 2;
#pragma unroll
        for (int u = 0; u < V<T>; ++u) {
            a[u] = !MIXED ? (float)x[u] : u < H ? (float)x[2 * u] : (float)y[2 * (u - H)];
            b[u] = !MIXED ? (float)y[u] : u < H ? (float)x[2 * u + 1] : (float)y[2 * (u - H) + 1];
        }
    }
    __device__ __forceinline__ void store(T *p, const float (&a)[V<T>], const float (&b)[V<T>]) const
    {
        constexpr int H = V<T> / 2;
        Raw<T> x, y;
#pragma unroll
        for (int u = 0; u < V<T>; ++u) {
            x[u] = (T)(!MIXED ? a[u] : u % 2 ? b[u / 2] : a[u / 2]);
            y[u] = (T)(!MIXED ? b[u] : u % 2 ? b[H + u / 2] : a[H + u / 2]);
        }
        if (kind == WHOLE) {
            *reinterpret_cast<Raw<T> *>(p + at) = x;
            *reinterpret_cast<Raw<T> *>(p + next) = y;
        } else if (kind == SINGLE) {
            const int f = here();
#pragma unroll
            for (int u = 0; u < V<T>; ++u) {
                const int i = place(f, u, 0), j = place(f, u, 1);
                if (i < D) p[i] = x[u];
                if (j < D) p[j] = y[u];
            }
        }
    }
    __device__ __forceinline__ void weights(const float *w, float (&a)[V<T>], float (&b)[V<T>]) const
    {
#pragma unroll
        for (int u = 0; u < V<T>; ++u) {
            a[u] = one(u) < D ? w[one(u)] : 0.0f;
            b[u] = other(u) < D ? w[other(u)] : 0.0f;
        }
    }
};

// What a workgroup knows of its tokens: where their rows begin in x and in dy, cos and sin of each pair's angle, and where they go in the pages.
struct Shared {
    float2 turn[MOST_TOKENS * MOST_PAIRS];
    int64_t x[MOST_TOKENS], dy[MOST_TOKENS], v[MOST_TOKENS];
    int64_t to[MOST_TOKENS];                // row of the first key head in the pages, -1: nowhere
    double place[MOST_TOKENS];
    float weight[2 * MOST_PAIRS];           // 1 where there is none
};

template <class T>
__device__ __forceinline__ void load_weight(const Call &c, const Side &side, Shared &s)
{
    const int e = threadIdx.x;
    if (e < c.D) s.weight[e] = !side.weight ? 1.0f : c.same ? (float)static_cast<const T *>(side.weight)[e] : static_cast<const float *>(side.weight)[e];
}

template <bool APPEND>
__device__ __forceinline__ void place_tokens(const Call &c, const Side &side, const Append &to, int64_t first, int count, Shared &s)
{
    const int t = threadIdx.x;
    if (t < count) {
        const int b = (int)((uint32_t)(first + t) / (uint32_t)c.L), i = (int)(first + t - (int64_t)b * c.L);
        s.x[t] = b * side.b + i * side.l;
        s.dy[t] = b * side.db + i * side.dl;
        if (c.positions) s.place[t] = (double)c.positions[b * c.pb + i * c.pl];
        else s.place[t] = APPEND ? (double)length_of(to.to, b) + i : (double)i;
        if (APPEND) {
            s.v[t] = b * to.vb + i * to.vl;
            s.to[t] = i < count_of(to.to, b, c.L) ? row_of(to.to, b, (uint32_t)length_of(to.to, b) + (uint32_t)i) : -1;
        }
    }
    __syncthreads();
}

__device__ __forceinline__ void form_angles(const Call &c, int count, Shared &s)
{
    for (int e = threadIdx.x; e < count * c.pairs; e += THREADS) {
        const int t = e / c.pairs, n = e - t * c.pairs;
        constexpr double TURN = 0.15915494309189533577;     // 1 / (2 pi)
        double turns = s.place[t] * c.frequencies[n] * TURN;
        turns -= rint(turns);
        const float halves = (float)(2.0 * turns);
        s.turn[e] = make_float2(cospif(halves), sinpif(halves));
    }
    __syncthreads();
}

// Sum over the 1 to 16 lanes of a row, by vector instructions alone: within pairs, within fours, of two fours (mirrored in 8), of two eights (mirrored in 16).
template <int CONTROL>
__device__ __forceinline__ float moved(float v)
{
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CONTROL, 0xf, 0xf, true));
}
__device__ __forceinline__ float row_sum(float v, int lanes)
{
    if (lanes > 1) v += moved<0xb1>(v);
    if (lanes > 2) v += moved<0x4e>(v);
    if (lanes > 4) v += moved<0x141>(v);
    if (lanes > 8) v += moved<0x140>(v);
    return v;
}

// a and b, turned by a token's angles (back: sign -1)
template <class T>
__device__ __forceinline__ void turn(const Call &c, const float2 *cs, int first, float sign, float (&a)[V<T>], float (&b)[V<T>])
{
#pragma unroll
    for (int u = 0; u < V<T>; ++u)
        if (first + u < c.pairs) {
            const float2 t = cs[first + u];
            const float x = a[u], y = b[u], sn = sign * t.y;
            a[u] = fmaf(x, t.x, -(y * sn));
            b[u] = fmaf(x, sn, y * t.x);
        }
}

template <class T>
__device__ __forceinline__ float scale_of(const Call &c, const float (&a)[V<T>], const float (&b)[V<T>])
{
    float sum = 0.0f;
#pragma unroll
    for (int u = 0; u < V<T>; ++u) sum = fmaf(a[u], a[u], fmaf(b[u], b[u], sum));
    return 1.0f / sqrtf(row_sum(sum, c.lanes) * c.inverse + c.eps);
}

// The rows of a workgroup's tokens: which token, and which head and map of it.
struct Rows {
    int per, rows, maps;
    float inv_per, inv_m;
    __device__ __forceinline__ Rows(const Call &c, const Side &side, int count)
        : per(side.heads * c.M), rows(count * side.heads * c.M), maps(c.M), inv_per(1.0f / (float)per), inv_m(1.0f / (float)c.M) {}
    // (rows are fewer than 2^22, so the quotients are exact)
    __device__ __forceinline__ void find(int row, int &t, int &place, int &head, int &map) const
    {
        t = (int)(((float)row + 0.5f) * inv_per);
        place = row - t * per;
        head = (int)(((float)place + 0.5f) * inv_m);
        map = place - head * maps;
    }
};

// Values as they are, to their pages.
template <class T>
__device__ void append_values(const Call &c, const Append &to, int group, Shared &s)
{
    const int64_t first = (int64_t)group * to.tokens;
    const int count = (int)(c.all - first < to.tokens ? c.all - first : to.tokens);
    place_tokens<true>(c, c.side[1], to, first, count, s);
    const int dv = to.to.dv, pieces = (dv + V<T> - 1) / V<T>, token = c.side[1].heads * pieces;
    for (int e = threadIdx.x; e < count * token; e += THREADS) {
        const int t = e / token, head = (e - t * token) / pieces, col = (e - t * token - head * pieces) * V<T>;
        if (s.to[t] < 0) continue;
        float v[V<T>];
        load_pack<T>(static_cast<const T *>(to.v) + s.v[t] + head * to.vh + col, dv - col, v);
        store_pack<T>(static_cast<T *>(to.to.v) + (s.to[t] + (int64_t)head * to.to.S) * dv + col, dv - col, v);
    }
}

// Measured: 64 x 197 tokens, 6 heads of 2 x 64 and as many key heads, fp32 28 us, 5.5 TB/s; 2 x 8192 tokens, 16 heads of 2 x 128 on 4, fp16 63 us, 5.3 TB/s.
template <class T, bool MIXED, bool APPEND>
__global__ __launch_bounds__(THREADS) void forward_kernel(const Call c, const Append to)
{
    __shared__ Shared s;
    if (APPEND && (int)blockIdx.x >= c.side[0].groups + c.side[1].groups)
        return append_values<T>(c, to, blockIdx.x - c.side[0].groups - c.side[1].groups, s);
    const int key = (int)blockIdx.x >= c.side[0].groups;
    const Side &side = c.side[key];
    const int64_t first = (int64_t)(blockIdx.x - (key ? c.side[0].groups : 0)) * side.tokens;
    const int count = (int)(c.all - first < side.tokens ? c.all - first : side.tokens);
    load_weight<T>(c, side, s);
    place_tokens<APPEND>(c, side, to, first, count, s);
    const int lane = threadIdx.x % c.lanes, groups = THREADS / c.lanes, mine = threadIdx.x / c.lanes;
    const Slots<T, MIXED> slots(c, lane);
    const Rows rows(c, side, count);
    const int turns = (rows.rows + groups - 1) / groups;
    const auto load = [&](int row, Raw<T> &x, Raw<T> &y) {
        int t, place, head, map;
        rows.find(row < rows.rows ? row : rows.rows - 1, t, place, head, map);
        slots.load(static_cast<const T *>(side.x) + s.x[t] + head * side.h + map * side.m, x, y);
    };
    // a row is on its way while the angles are formed, and then while the last one is used
    Raw<T> x, y, next_x, next_y;
    if (turns > 0) load(mine, x, y);
    float wa[V<T>], wb[V<T>];
    slots.weights(s.weight, wa, wb);
    form_angles(c, count, s);
    // every lane of a wave takes part in the rows' sums to the end
    for (int n = 0; n < turns; ++n) {
        const int row = n * groups + mine;
        if (n + 1 < turns) load(row + groups, next_x, next_y);
        int t, place, head, map;
        rows.find(row < rows.rows ? row : rows.rows - 1, t, place, head, map);
        float a[V<T>], b[V<T>];
        slots.spread(x, y, a, b);
        if (c.norm) {
            const float r = scale_of<T>(c, a, b);
#pragma unroll
            for (int u = 0; u < V<T>; ++u) {
                a[u] = a[u] * r * wa[u];
                b[u] = b[u] * r * wb[u];
            }
        }
        turn<T>(c, s.turn + t * c.pairs, slots.first, 1.0f, a, b);
        if (row < rows.rows) {
            T *out = static_cast<T *>(side.out);
            if (APPEND && key) {
                if (s.to[t] >= 0) slots.store(out + ((s.to[t] + (int64_t)head * to.to.S) * c.M + map) * c.D, a, b);
            } else {
                slots.store(out + ((first + t) * rows.per + place) * c.D, a, b);
            }
        }
        x = next_x;
        y = next_y;
    }
}

// A backward call's workgroups: each takes tokens in turn and keeps its share of dw in registers until the end.  Measured, a step with 1024 and 2048 workgroups:
// 64 x 197 tokens as above 100.1 and 97.7 us, 2 x 8192 as above 197 and 190 us.
constexpr int MOST_GROUPS = 2048;

template <class T, bool MIXED>
__global__ __launch_bounds__(THREADS, 4) void backward_kernel(const Call c, float *__restrict__ partial)
{
    __shared__ Shared s;
    __shared__ float joined[4][2 * MOST_PAIRS];
    const int key = (int)blockIdx.x >= c.side[0].groups;
    const Side &side = c.side[key];
    const int group = blockIdx.x - (key ? c.side[0].groups : 0);
    const int lane = threadIdx.x % c.lanes, groups = THREADS / c.lanes, mine = threadIdx.x / c.lanes;
    const Slots<T, MIXED> slots(c, lane);
    float da[V<T>], db[V<T>], wa[V<T>], wb[V<T>];
#pragma unroll
    for (int u = 0; u < V<T>; ++u) da[u] = db[u] = 0.0f;
    load_weight<T>(c, side, s);
    __syncthreads();
    slots.weights(s.weight, wa, wb);
    for (int64_t first = (int64_t)group * side.tokens; first < c.all; first += (int64_t)side.groups * side.tokens) {
        const int count = (int)(c.all - first < side.tokens ? c.all - first : side.tokens);
        __syncthreads();
        place_tokens<false>(c, side, Append(), first, count, s);
        const Rows rows(c, side, count);
        const int turns = (rows.rows + groups - 1) / groups;
        const auto load = [&](int row, Raw<T> &x, Raw<T> &y, Raw<T> &gx, Raw<T> &gy) {
            int t, place, head, map;
            rows.find(row < rows.rows ? row : rows.rows - 1, t, place, head, map);
            slots.load(static_cast<const T *>(side.dy) + s.dy[t] + head * side.dh + map * side.dm, gx, gy);
            if (c.norm) slots.load(static_cast<const T *>(side.x) + s.x[t] + head * side.h + map * side.m, x, y);
        };
        Raw<T> x, y, gx, gy, next_x, next_y, next_gx, next_gy;
        load(mine, x, y, gx, gy);
        form_angles(c, count, s);
        for (int n = 0; n < turns; ++n) {
            const int row = n * groups + mine;
            if (n + 1 < turns) load(row + groups, next_x, next_y, next_gx, next_gy);
            int t, place, head, map;
            rows.find(row < rows.rows ? row : rows.rows - 1, t, place, head, map);
            float ga[V<T>], gb[V<T>];
            slots.spread(gx, gy, ga, gb);
            turn<T>(c, s.turn + t * c.pairs, slots.first, -1.0f, ga, gb);
            if (c.norm) {
                float a[V<T>], b[V<T>], dot = 0.0f;
                slots.spread(x, y, a, b);
                const float r = scale_of<T>(c, a, b);
#pragma unroll
                for (int u = 0; u < V<T>; ++u) {
                    a[u] *= r;
                    b[u] *= r;
                    if (row < rows.rows) {
                        da[u] = fmaf(ga[u], a[u], da[u]);
                        db[u] = fmaf(gb[u], b[u], db[u]);
                    }
                    ga[u] *= wa[u];
                    gb[u] *= wb[u];
                    dot = fmaf(ga[u], a[u], fmaf(gb[u], b[u], dot));
                }
                const float mean = row_sum(dot, c.lanes) * c.inverse;
#pragma unroll
                for (int u = 0; u < V<T>; ++u) {
                    ga[u] = r * fmaf(-a[u], mean, ga[u]);
                    gb[u] = r * fmaf(-b[u], mean, gb[u]);
                }
            }
            if (row < rows.rows && side.out) slots.store(static_cast<T *>(side.out) + ((first + t) * rows.per + place) * c.D, ga, gb);
            x = next_x;
            y = next_y;
            gx = next_gx;
            gy = next_gy;
        }
    }
    if (!partial) return;
    const int wave = threadIdx.x >> 6;
#pragma unroll
    for (int u = 0; u < V<T>; ++u) {
        for (int k = c.lanes; k < 64; k <<= 1) {
            da[u] += __shfl_xor(da[u], k);
            db[u] += __shfl_xor(db[u], k);
        }
        if ((int)(threadIdx.x & 63) < c.lanes) {
            if (slots.one(u) < c.D) joined[wave][slots.one(u)] = da[u];
            if (slots.other(u) < c.D) joined[wave][slots.other(u)] = db[u];
        }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < c.D; e += THREADS)
        partial[(int64_t)blockIdx.x * c.D + e] = (joined[0][e] + joined[1][e]) + (joined[2][e] + joined[3][e]);
}

// The workgroups' sums of dw, 16 columns a workgroup: 64 threads a column, four of a thread's loads at a time, then the threads' sums, each in a fixed order.
constexpr int JOIN = 1024;
template <class W>
__global__ __launch_bounds__(JOIN) void weights_kernel(const float *__restrict__ partial, int q_groups, int k_groups, int D, W *dwq, W *dwk)
{
    __shared__ float part[64][17];
    const int column = threadIdx.x % 16, col = blockIdx.x * 16 + column, turn = threadIdx.x / 16, key = blockIdx.y;
    W *out = key ? dwk : dwq;
    if (!out) return;
    const int groups = key ? k_groups : q_groups;
    const float *from = partial + (key ? (int64_t)q_groups * D : 0);
    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (col < D)
        for (int g = turn; g < groups; g += 256)
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (g + 64 * u < groups) sum[u] += from[(int64_t)(g + 64 * u) * D + col];
    part[turn][column] = (sum[0] + sum[1]) + (sum[2] + sum[3]);
    __syncthreads();
    for (int half = 32; half > 0; half /= 2) {
        if (turn < half) part[turn][column] += part[turn + half][column];
        __syncthreads();
    }
    if (turn == 0 && col < D) out[col] = (W)part[0][column];
}

int fill(const mam_norm_rotate_t *a, Call &c)
{
    if (!a) return fail(MAM_ERR_INVALID_ARGUMENT, "null pointer");
    if (!is_type(a->type)) return fail(MAM_ERR_INVALID_ARGUMENT, "unknown element type %d", a->type);
    if (a->weight_type != a->type && a->weight_type != MAM_F32)
        return fail(MAM_ERR_INVALID_ARGUMENT, "weights are of the operands' type or fp32, got type %d", a->weight_type);
    if (a->B < 0 || a->L < 0 || a->H < 0 || a->Hkv < 0 || a->M < 0) return fail(MAM_ERR_INVALID_ARGUMENT, "negative size");
    if (a->D < 1 || a->D > 2 * MOST_PAIRS) return fail(MAM_ERR_UNSUPPORTED, "head sizes are 1 to %d", 2 * MOST_PAIRS);
    if (a->pairs < 0 || 2 * a->pairs > a->D) return fail(MAM_ERR_INVALID_ARGUMENT, "a head of %lld has no %lld pairs", (long long)a->D, (long long)a->pairs);
    if (a->pairs > 0 && !a->frequencies) return fail(MAM_ERR_INVALID_ARGUMENT, "null pointer");
    if (a->norm && !(a->eps >= 0.0 && a->eps <= 1e30)) return fail(MAM_ERR_INVALID_ARGUMENT, "eps must not be negative, and finite");
    const int64_t most = (int64_t)1 << 20;      // rows of a token: their number within a workgroup is divided in fp32
    if (a->H > most || a->Hkv > most || a->M > 64 || MOST_TOKENS * (a->H + a->Hkv) * a->M >= (int64_t)1 << 22)
        return fail(MAM_ERR_UNSUPPORTED, "a token has too many heads");
    if (a->B > INT32_MAX || a->L > INT32_MAX || (a->L > 0 && a->B > INT32_MAX / a->L)) return fail(MAM_ERR_UNSUPPORTED, "more than 2^31 tokens");
    c = Call();
    for (int k = 0; k < 2; ++k) {
        const int64_t *st = k ? a->k_stride : a->q_stride;
        Side &s = c.side[k];
        s.x = k ? a->k : a->q;
        s.weight = k ? a->k_weight : a->q_weight;
        s.b = st[0]; s.l = st[1]; s.h = st[2]; s.m = st[3];
        s.heads = (int)(k ? a->Hkv : a->H);
        if (s.heads > 0 && a->M > 0 && a->B > 0 && a->L > 0 && !s.x) return fail(MAM_ERR_INVALID_ARGUMENT, "null pointer");
    }
    c.frequencies = a->frequencies;
    c.positions = a->positions;
    c.pb = a->position_stride[0]; c.pl = a->position_stride[1];
    c.L = (int)a->L; c.M = (int)a->M; c.D = (int)a->D; c.pairs = (int)a->pairs;
    c.norm = a->norm != 0; c.interleaved = a->interleaved != 0; c.same = a->weight_type == a->type;
    c.eps = (float)a->eps;
    c.inverse = 1.0f / (float)c.D;
    c.all = a->B * a->L;
    const int slots = (c.D + 1) / 2, v = (int)(16 / type_size(a->type));
    c.lanes = 1;
    while (c.lanes * v < slots) c.lanes *= 2;
    return MAM_OK;
}

// Tokens of a turn of a side's workgroups: enough rows that each of a workgroup's groups of lanes has `turns` of them, fewer where less than `want` turns would be left over the
// call, but one row for each group.
void tokens_of(const Call &c, Side &s, int turns, int64_t want)
{
    const int rows = s.heads * c.M, groups = THREADS / c.lanes;
    int n = rows > 0 ? (int)ceil_div((int64_t)turns * groups, rows) : 1;
    if (n > MOST_TOKENS) n = MOST_TOKENS;
    while (n > 1 && ceil_div(c.all, n) < want && n / 2 * rows >= groups) n /= 2;
    s.tokens = n;
    s.groups = rows > 0 ? (int)ceil_div(c.all, n) : 0;
}

template <class T>
int launch_forward(const Call &c, const Append *to, hipStream_t st)
{
    const dim3 grid((unsigned)(c.side[0].groups + c.side[1].groups + (to ? to->groups : 0)));
    const Append none{};
    if (to && c.interleaved) hipLaunchKernelGGL((forward_kernel<T, true, true>), grid, dim3(THREADS), 0, st, c, *to);
    else if (to) hipLaunchKernelGGL((forward_kernel<T, false, true>), grid, dim3(THREADS), 0, st, c, *to);
    else if (c.interleaved) hipLaunchKernelGGL((forward_kernel<T, true, false>), grid, dim3(THREADS), 0, st, c, none);
    else hipLaunchKernelGGL((forward_kernel<T, false, false>), grid, dim3(THREADS), 0, st, c, none);
    return check_launch("rotary::forward_kernel");
}

int run_forward(Call &c, int type, Append *to, hipStream_t st)
{
    for (Side &s : c.side) tokens_of(c, s, 4, 2 * kNumCU);
    int64_t groups = (int64_t)c.side[0].groups + c.side[1].groups;
    if (to) {
        const int64_t pieces = c.side[1].heads * ceil_div(to->to.dv, 16 / type_size(type));
        int n = pieces > 0 ? (int)ceil_div(4 * THREADS, pieces) : 1;
        if (n > MOST_TOKENS) n = MOST_TOKENS;
        while (n > 1 && ceil_div(c.all, n) < 2 * kNumCU) n /= 2;
        to->tokens = n;
        to->groups = pieces > 0 ? (int)ceil_div(c.all, n) : 0;
        groups += to->groups;
    }
    if (groups > INT32_MAX) return fail(MAM_ERR_UNSUPPORTED, "too many tokens");
    if (groups == 0) return MAM_OK;
    if (type == MAM_F32) return launch_forward<float>(c, to, st);
    if (type == MAM_BF16) return launch_forward<bf16>(c, to, st);
    return launch_forward<f16>(c, to, st);
}

template <class T>
int launch_backward(const Call &c, float *partial, hipStream_t st)
{
    const dim3 grid((unsigned)(c.side[0].groups + c.side[1].groups));
    if (grid.x == 0) return MAM_OK;
    if (c.interleaved) hipLaunchKernelGGL((backward_kernel<T, true>), grid, dim3(THREADS), 0, st, c, partial);
    else hipLaunchKernelGGL((backward_kernel<T, false>), grid, dim3(THREADS), 0, st, c, partial);
    return check_launch("rotary::backward_kernel");
}

// The workgroups of a backward call are shared out by the sides' rows.
void backward_groups(Call &c)
{
    const int heads = c.side[0].heads + c.side[1].heads;
    for (Side &s : c.side) {
        const int most = heads > 0 ? (int)ceil_div((int64_t)MOST_GROUPS * s.heads, heads) : 0;
        tokens_of(c, s, 4, most);
        if (s.groups > most) s.groups = most;
    }
}

size_t backward_workspace(const Call &c) { return (size_t)(c.side[0].groups + c.side[1].groups) * c.D * sizeof(float); }

}  // namespace rotary
}  // namespace mam

extern "C" int mam_norm_rotate(const mam_norm_rotate_t *args, void *q_out, void *k_out, void *stream)
{
    using namespace mam;
    rotary::Call c;
    const int rc = rotary::fill(args, c);
    if (rc != MAM_OK || c.all == 0 || c.M == 0) return rc;
    if ((c.side[0].heads && !q_out) || (c.side[1].heads && !k_out)) return fail(MAM_ERR_INVALID_ARGUMENT, "null pointer");
    c.side[0].out = q_out;
    c.side[1].out = k_out;
    return rotary::run_forward(c, args->type, nullptr, static_cast<hipStream_t>(stream));
}

extern "C" int mam_norm_rotate_append(const mam_norm_rotate_t *args, const void *v, const int64_t *v_stride, const mam_pages_t *pages, void *q_out,
                                      void *stream)
{
    using namespace mam;
    rotary::Call c;
    rotary::Append to;
    int rc = rotary::fill(args, c);
    if (rc == MAM_OK) rc = fill_pages(pages, to.to);
    if (rc != MAM_OK) return rc;
    if (pages->type != args->type || pages->B != args->B || pages->Hkv != args->Hkv || pages->D != args->D || args->M != 2)
        return fail(MAM_ERR_INVALID_ARGUMENT, "the pages are for other keys");
    if (c.all == 0) return MAM_OK;
    if ((c.side[0].heads && !q_out) || (c.side[1].heads && (!v || !v_stride || (to.to.P > 0 && (!to.to.k || !to.to.v))))) return fail(MAM_ERR_INVALID_ARGUMENT, "null pointer");
    to.v = v;
    if (v_stride) {
        to.vb = v_stride[0]; to.vl = v_stride[1]; to.vh = v_stride[2];
    }
    c.side[0].out = q_out;
    c.side[1].out = to.to.k;
    return rotary::run_forward(c, args->type, &to, static_cast<hipStream_t>(stream));
}

extern "C" size_t mam_norm_rotate_backward_workspace(const mam_norm_rotate_t *args)
{
    using namespace mam;
    rotary::Call c;
    if (rotary::fill(args, c) != MAM_OK || c.all == 0 || c.M == 0 || !c.norm) return 0;
    rotary::backward_groups(c);
    return rotary::backward_workspace(c);
}

extern "C" int mam_norm_rotate_backward(const mam_norm_rotate_t *args, const void *q_grad, const int64_t *q_grad_stride, const void *k_grad,
                                        const int64_t *k_grad_stride, void *dq, void *dk, void *dq_weight, void *dk_weight, void *workspace,
                                        size_t workspace_bytes, void *stream)
{
    using namespace mam;
    rotary::Call c;
    const int rc = rotary::fill(args, c);
    if (rc != MAM_OK) return rc;
    if ((dq_weight || dk_weight) && !c.norm) return fail(MAM_ERR_INVALID_ARGUMENT, "there is no norm whose weights have gradients");
    if ((q_grad && !q_grad_stride) || (k_grad && !k_grad_stride)) return fail(MAM_ERR_INVALID_ARGUMENT, "null pointer");
    if ((dq || dq_weight) && !q_grad && c.side[0].heads && c.all && c.M) return fail(MAM_ERR_INVALID_ARGUMENT, "null pointer");
    if ((dk || dk_weight) && !k_grad && c.side[1].heads && c.all && c.M) return fail(MAM_ERR_INVALID_ARGUMENT, "null pointer");
    for (int k = 0; k < 2; ++k) {
        rotary::Side &s = c.side[k];
        const int64_t *st = k ? k_grad_stride : q_grad_stride;
        s.dy = (k ? dk || dk_weight : dq || dq_weight) ? (k ? k_grad : q_grad) : nullptr;
        s.out = k ? dk : dq;
        if (s.dy) {
            s.db = st[0]; s.dl = st[1]; s.dh = st[2]; s.dm = st[3];
        }
    }
    hipStream_t st = static_cast<hipStream_t>(stream);
    const bool weights = dq_weight || dk_weight;
    float *partial = nullptr;
    if (c.all > 0 && c.M > 0) {
        rotary::backward_groups(c);
        const size_t need = weights ? rotary::backward_workspace(c) : 0;
        if (need > 0 && (!workspace || workspace_bytes < need))
            return fail(MAM_ERR_WORKSPACE, "the gradient needs %zu workspace bytes, got %zu", need, workspace ? workspace_bytes : (size_t)0);
        partial = weights ? static_cast<float *>(workspace) : nullptr;
        for (rotary::Side &s : c.side)
            if (!s.dy) s.groups = 0;
        const int launched = args->type == MAM_F32    ? rotary::launch_backward<float>(c, partial, st)
                             : args->type == MAM_BF16 ? rotary::launch_backward<bf16>(c, partial, st)
                                                      : rotary::launch_backward<f16>(c, partial, st);
        if (launched != MAM_OK) return launched;
    }
    if (!weights) return MAM_OK;
    const dim3 grid((unsigned)ceil_div(c.D, 16), 2);
    if (args->weight_type == MAM_F32)
        hipLaunchKernelGGL((rotary::weights_kernel<float>), grid, dim3(rotary::JOIN), 0, st, partial, c.side[0].groups, c.side[1].groups, c.D, static_cast<float *>(dq_weight),
                           static_cast<float *>(dk_weight));
    else if (args->weight_type == MAM_BF16)
        hipLaunchKernelGGL((rotary::weights_kernel<bf16>), grid, dim3(rotary::JOIN), 0, st, partial, c.side[0].groups, c.side[1].groups, c.D, static_cast<bf16 *>(dq_weight),
                           static_cast<bf16 *>(dk_weight));
    else
        hipLaunchKernelGGL((rotary::weights_kernel<f16>), grid, dim3(rotary::JOIN), 0, st, partial, c.side[0].groups, c.side[1].groups, c.D, static_cast<f16 *>(dq_weight),
                           static_cast<f16 *>(dk_weight));
    return check_launch("rotary::weights_kernel");
}
