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
    int heads;
};

struct Call {
    Side side[2];                           // queries, keys
    const double *frequencies;
    const int32_t *positions;
    int64_t pb, pl;
    int L, M, D, pairs, norm, interleaved, same, lanes, tokens;     // lanes of a row, tokens of a workgroup
    int64_t all;                            // tokens of the call
    float eps, inverse;                     // inverse: 1 / D
};

// Where a call's keys and values go.
struct Append {
    Pages to;
    const void *v;
    int64_t vb, vl, vh;
};

template <class T>
constexpr int V = kPack<T>;

// A lane's pairs of a row, first elements in a, second ones in b.
template <class T>
struct Slots {
    enum Kind { HALVES, NEIGHBOURS, SINGLE, NONE };
    int first, pairs, D;
    Kind kind;

    __device__ __forceinline__ Slots(const Call &c, int lane) : first(lane * V<T>), pairs(c.interleaved ? 0 : c.pairs), D(c.D)
    {
        kind = first + V<T> <= pairs ? HALVES : first >= pairs && 2 * (first + V<T>) <= D ? NEIGHBOURS
               : 2 * first < D || first < pairs                 ? SINGLE
                                                                : NONE;
    }
    // elements of pair `first + u`; D and beyond: none
    __device__ __forceinline__ int one(int u) const { return first + u < pairs ? first + u : 2 * (first + u); }
    __device__ __forceinline__ int other(int u) const { return first + u < pairs ? first + u + pairs : 2 * (first + u) + 1; }

    template <class E>
    __device__ __forceinline__ void load(const E *p, float (&a)[V<T>], float (&b)[V<T>]) const
    {
        if (kind == HALVES) {
            load_pack<E, V<T>>(p + first, V<T>, a);
            load_pack<E, V<T>>(p + first + pairs, V<T>, b);
        } else if (kind == NEIGHBOURS) {
            float x[V<T>], y[V<T>];
            load_pack<E, V<T>>(p + 2 * first, V<T>, x);
            load_pack<E, V<T>>(p + 2 * first + V<T>, V<T>, y);
#pragma unroll
            for (int u = 0; u < V<T> / 2; ++u) {
                a[u] = x[2 * u];
                b[u] = x[2 * u + 1];
                a[V<T> / 2 + u] = y[2 * u];
                b[V<T> / 2 + u] = y[2 * u + 1];
            }
        } else {
#pragma unroll
            for (int u = 0; u < V<T>; ++u) {
                a[u] = kind == SINGLE && one(u) < D ? (float)p[one(u)] : 0.0f;
                b[u] = kind == SINGLE && other(u) < D ? (float)p[other(u)] : 0.0f;
            }
        }
    }
    __device__ __forceinline__ void store(T *p, const float (&a)[V<T>], const float (&b)[V<T>]) const
    {
        if (kind == HALVES) {
            store_pack<T, V<T>>(p + first, V<T>, a);
            store_pack<T, V<T>>(p + first + pairs, V<T>, b);
        } else if (kind == NEIGHBOURS) {
            float x[V<T>], y[V<T>];
#pragma unroll
            for (int u = 0; u < V<T> / 2; ++u) {
                x[2 * u] = a[u];
                x[2 * u + 1] = b[u];
                y[2 * u] = a[V<T> / 2 + u];
                y[2 * u + 1] = b[V<T> / 2 + u];
            }
            store_pack<T, V<T>>(p + 2 * first, V<T>, x);
            store_pack<T, V<T>>(p + 2 * first + V<T>, V<T>, y);
        } else if (kind == SINGLE) {
#pragma unroll
            for (int u = 0; u < V<T>; ++u) {
                if (one(u) < D) p[one(u)] = (T)a[u];
                if (other(u) < D) p[other(u)] = (T)b[u];
            }
        }
    }
    // weights, of T or fp32; 1 where there are none
    __device__ __forceinline__ void weights(const Call &c, const void *w, float (&a)[V<T>], float (&b)[V<T>]) const
    {
        if (!w) {
#pragma unroll
            for (int u = 0; u < V<T>; ++u) a[u] = b[u] = 1.0f;
        } else if (c.same) {
            load(static_cast<const T *>(w), a, b);
        } else {
            load(static_cast<const float *>(w), a, b);
        }
    }
};

// What a workgroup knows of its tokens: batch and number, cos and sin of each pair's angle, and where they go in the pages.
struct Shared {
    float2 turn[MOST_TOKENS * MOST_PAIRS];
    int b[MOST_TOKENS], i[MOST_TOKENS];
    int64_t to[MOST_TOKENS];                // row of the first key head in the pages, -1: nowhere
};

template <bool APPEND>
__device__ __forceinline__ void prepare(const Call &c, const Append &to, int64_t first, int count, Shared &s)
{
    for (int t = threadIdx.x; t < count; t += THREADS) {
        const int b = (int)((uint32_t)(first + t) / (uint32_t)c.L), i = (int)(first + t - (int64_t)b * c.L);
        s.b[t] = b;
        s.i[t] = i;
        if (APPEND) s.to[t] = i < count_of(to.to, b, c.L) ? row_of(to.to, b, (uint32_t)length_of(to.to, b) + (uint32_t)i) : -1;
    }
    for (int e = threadIdx.x; e < count * c.pairs; e += THREADS) {
        const int t = e / c.pairs, n = e - t * c.pairs;
        const int b = (int)((uint32_t)(first + t) / (uint32_t)c.L), i = (int)(first + t - (int64_t)b * c.L);
        double place;
        if (c.positions) place = (double)c.positions[b * c.pb + i * c.pl];
        else place = APPEND ? (double)length_of(to.to, b) + i : (double)i;
        constexpr double TURN = 0.15915494309189533577;     // 1 / (2 pi)
        double turns = place * c.frequencies[n] * TURN;
        turns -= rint(turns);
        float2 cs;
        sincospif((float)(2.0 * turns), &cs.y, &cs.x);
        s.turn[e] = cs;
    }
    __syncthreads();
}

// Sum over the lanes of a row.
__device__ __forceinline__ float row_sum(float v, int lanes)
{
    for (int x = 1; x < lanes; x <<= 1) v += __shfl_xor(v, x);
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
    const float mean = row_sum(sum, c.lanes) * c.inverse;
    return 1.0f / sqrtf(mean + c.eps);
}

template <class T, bool APPEND>
__global__ __launch_bounds__(THREADS) void forward_kernel(const Call c, const Append to)
{
    __shared__ Shared s;
    const int64_t first = (int64_t)blockIdx.x * c.tokens;
    const int count = (int)(c.all - first < c.tokens ? c.all - first : c.tokens);
    prepare<APPEND>(c, to, first, count, s);
    const int lane = threadIdx.x % c.lanes, groups = THREADS / c.lanes;
    const Slots<T> slots(c, lane);
    const int q_rows = c.side[0].heads * c.M, per = q_rows + c.side[1].heads * c.M, rows = count * per;
    const float inv_per = 1.0f / (float)per, inv_m = 1.0f / (float)c.M;
    // every lane of a wave takes part in the rows' sums to the end
    const int turns = (rows + groups - 1) / groups;
    for (int n = 0; n < turns; ++n) {
        const int row = n * groups + threadIdx.x / c.lanes;
        const bool there = row < rows;
        const int t = there ? (int)(((float)row + 0.5f) * inv_per) : 0, rest = there ? row - t * per : 0, key = rest >= q_rows;
        const int place = key ? rest - q_rows : rest, head = (int)(((float)place + 0.5f) * inv_m), map = place - head * c.M;
        const Side &q = c.side[0], &k = c.side[1];
        float a[V<T>], b[V<T>];
        slots.load(static_cast<const T *>(key ? k.x : q.x) + s.b[t] * (key ? k.b : q.b) + s.i[t] * (key ? k.l : q.l) + head * (key ? k.h : q.h) +
                       map * (key ? k.m : q.m), a, b);
        if (c.norm) {
            const float r = scale_of<T>(c, a, b);
            float wa[V<T>], wb[V<T>];
            slots.weights(c, key ? k.weight : q.weight, wa, wb);
#pragma unroll
            for (int u = 0; u < V<T>; ++u) {
                a[u] = a[u] * r * wa[u];
                b[u] = b[u] * r * wb[u];
            }
        }
        turn<T>(c, s.turn + t * c.pairs, slots.first, 1.0f, a, b);
        if (!there) continue;
        T *out = static_cast<T *>(key ? k.out : q.out);
        if (APPEND && key) {
            if (s.to[t] >= 0) slots.store(out + ((s.to[t] + (int64_t)head * to.to.S) * c.M + map) * c.D, a, b);
        } else {
            slots.store(out + ((first + t) * (key ? per - q_rows : q_rows) + place) * c.D, a, b);
        }
    }
    if (APPEND) {
        const int dv = to.to.dv, pieces = (dv + V<T> - 1) / V<T>, token = c.side[1].heads * pieces;
        for (int e = threadIdx.x; e < count * token; e += THREADS) {
            const int t = e / token, head = (e - t * token) / pieces, col = (e - t * token - head * pieces) * V<T>;
            if (s.to[t] < 0) continue;
            float x[V<T>];
            load_pack<T>(static_cast<const T *>(to.v) + s.b[t] * to.vb + s.i[t] * to.vl + head * to.vh + col, dv - col, x);
            store_pack<T>(static_cast<T *>(to.to.v) + (s.to[t] + (int64_t)head * to.to.S) * dv + col, dv - col, x);
        }
    }
}

// Workgroups of a backward call: each takes tokens in turn and keeps its share of dw in registers until the end.
constexpr int MOST_GROUPS = 1024;

template <class T>
__global__ __launch_bounds__(THREADS) void backward_kernel(const Call c, float *__restrict__ partial)
{
    __shared__ Shared s;
    __shared__ float joined[4][2 * MOST_PAIRS];
    const int lane = threadIdx.x % c.lanes, groups = THREADS / c.lanes;
    const Slots<T> slots(c, lane);
    const float inv_m = 1.0f / (float)c.M;
    float da[2][V<T>], db[2][V<T>];
#pragma unroll
    for (int u = 0; u < V<T>; ++u) da[0][u] = da[1][u] = db[0][u] = db[1][u] = 0.0f;
    for (int64_t first = (int64_t)blockIdx.x * c.tokens; first < c.all; first += (int64_t)gridDim.x * c.tokens) {
        const int count = (int)(c.all - first < c.tokens ? c.all - first : c.tokens);
        __syncthreads();
        prepare<false>(c, Append(), first, count, s);
#pragma unroll
        for (int key = 0; key < 2; ++key) {
            const Side &side = c.side[key];
            const int per = side.heads * c.M, rows = count * per, turns = (rows + groups - 1) / groups;
            if (!side.dy) continue;
            const float inv_per = 1.0f / (float)per;
            for (int n = 0; n < turns; ++n) {
                const int row = n * groups + threadIdx.x / c.lanes;
                const bool there = row < rows;
                const int t = there ? (int)(((float)row + 0.5f) * inv_per) : 0, place = there ? row - t * per : 0;
                const int head = (int)(((float)place + 0.5f) * inv_m), map = place - head * c.M;
                float a[V<T>], b[V<T>], ga[V<T>], gb[V<T>];
                slots.load(static_cast<const T *>(side.dy) + s.b[t] * side.db + s.i[t] * side.dl + head * side.dh + map * side.dm, ga, gb);
                if (c.norm)
                    slots.load(static_cast<const T *>(side.x) + s.b[t] * side.b + s.i[t] * side.l + head * side.h + map * side.m, a, b);
                turn<T>(c, s.turn + t * c.pairs, slots.first, -1.0f, ga, gb);
                if (c.norm) {
                    const float r = scale_of<T>(c, a, b);
                    float wa[V<T>], wb[V<T>], dot = 0.0f;
                    slots.weights(c, side.weight, wa, wb);
#pragma unroll
                    for (int u = 0; u < V<T>; ++u) {
                        a[u] *= r;
                        b[u] *= r;
                        if (there) {
                            da[key][u] = fmaf(ga[u], a[u], da[key][u]);
                            db[key][u] = fmaf(gb[u], b[u], db[key][u]);
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
                if (there && side.out) slots.store(static_cast<T *>(side.out) + ((first + t) * side.heads * c.M + place) * c.D, ga, gb);
            }
        }
    }
    if (!partial) return;
    const int wave = threadIdx.x >> 6;
#pragma unroll
    for (int key = 0; key < 2; ++key) {
        __syncthreads();
#pragma unroll
        for (int u = 0; u < V<T>; ++u) {
            float x = da[key][u], y = db[key][u];
            for (int k = c.lanes; k < 64; k <<= 1) {
                x += __shfl_xor(x, k);
                y += __shfl_xor(y, k);
            }
            if ((int)(threadIdx.x & 63) < c.lanes) {
                if (slots.one(u) < c.D) joined[wave][slots.one(u)] = x;
                if (slots.other(u) < c.D) joined[wave][slots.other(u)] = y;
            }
        }
        __syncthreads();
        for (int e = threadIdx.x; e < c.D; e += THREADS)
            partial[((int64_t)blockIdx.x * 2 + key) * c.D + e] = (joined[0][e] + joined[1][e]) + (joined[2][e] + joined[3][e]);
    }
}

// The workgroups' sums of dw, 16 columns a workgroup: 16 threads a column, then those, each in a fixed order.
template <class W>
__global__ __launch_bounds__(THREADS) void weights_kernel(const float *__restrict__ partial, int groups, int D, W *dwq, W *dwk)
{
    __shared__ float part[16][17];
    const int col = blockIdx.x * 16 + threadIdx.x % 16, turn = threadIdx.x / 16, key = blockIdx.y;
    float sum = 0.0f;
    if (col < D)
        for (int g = turn; g < groups; g += 16) sum += partial[((int64_t)g * 2 + key) * D + col];
    part[turn][threadIdx.x % 16] = sum;
    __syncthreads();
    if (turn == 0 && col < D) {
        float total = 0.0f;
#pragma unroll
        for (int t = 0; t < 16; ++t) total += part[t][threadIdx.x % 16];
        W *out = key ? dwk : dwq;
        if (out) out[col] = (W)total;
    }
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

// Tokens of a workgroup: enough rows that each of its groups of lanes has `turns` of them, while `want` workgroups are left.
void tokens_of(Call &c, int rows, int turns, int64_t want)
{
    const int groups = THREADS / c.lanes;
    int n = rows > 0 ? (int)ceil_div((int64_t)turns * groups, rows) : 1;
    if (n > MOST_TOKENS) n = MOST_TOKENS;
    while (n > 1 && ceil_div(c.all, n) < want) n /= 2;
    c.tokens = n;
}

template <class T>
int launch_forward(const Call &c, const Append *to, hipStream_t st)
{
    const dim3 grid((unsigned)ceil_div(c.all, c.tokens));
    if (to) hipLaunchKernelGGL((forward_kernel<T, true>), grid, dim3(THREADS), 0, st, c, *to);
    else hipLaunchKernelGGL((forward_kernel<T, false>), grid, dim3(THREADS), 0, st, c, Append());
    return check_launch("rotary::forward_kernel");
}

int run_forward(Call &c, int type, const Append *to, hipStream_t st)
{
    tokens_of(c, (c.side[0].heads + c.side[1].heads) * c.M, 4, 4 * kNumCU);
    if (type == MAM_F32) return launch_forward<float>(c, to, st);
    if (type == MAM_BF16) return launch_forward<bf16>(c, to, st);
    return launch_forward<f16>(c, to, st);
}

int backward_groups(const Call &c)
{
    const int64_t n = ceil_div(c.all, c.tokens);
    return (int)(n < MOST_GROUPS ? n : MOST_GROUPS);
}

void backward_tokens(Call &c) { tokens_of(c, (c.side[0].heads + c.side[1].heads) * c.M, 4, MOST_GROUPS); }

size_t backward_workspace(const Call &c) { return (size_t)backward_groups(c) * 2 * c.D * sizeof(float); }

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
    if ((c.side[0].heads && !q_out) || (c.side[1].heads && (!v || !v_stride || !to.to.k || !to.to.v))) return fail(MAM_ERR_INVALID_ARGUMENT, "null pointer");
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
    rotary::backward_tokens(c);
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
        if (s.heads == 0) s.dy = nullptr;
    }
    hipStream_t st = static_cast<hipStream_t>(stream);
    const bool weights = dq_weight || dk_weight;
    int groups = 0;
    float *partial = nullptr;
    if (c.all > 0 && c.M > 0) {
        rotary::backward_tokens(c);
        groups = rotary::backward_groups(c);
        const size_t need = weights ? rotary::backward_workspace(c) : 0;
        if (need > 0 && (!workspace || workspace_bytes < need))
            return fail(MAM_ERR_WORKSPACE, "the gradient needs %zu workspace bytes, got %zu", need, workspace ? workspace_bytes : (size_t)0);
        partial = weights ? static_cast<float *>(workspace) : nullptr;
        const dim3 grid((unsigned)groups);
        if (args->type == MAM_F32) hipLaunchKernelGGL((rotary::backward_kernel<float>), grid, dim3(rotary::THREADS), 0, st, c, partial);
        else if (args->type == MAM_BF16) hipLaunchKernelGGL((rotary::backward_kernel<bf16>), grid, dim3(rotary::THREADS), 0, st, c, partial);
        else hipLaunchKernelGGL((rotary::backward_kernel<f16>), grid, dim3(rotary::THREADS), 0, st, c, partial);
        const int launched = check_launch("rotary::backward_kernel");
        if (launched != MAM_OK) return launched;
    }
    if (!weights) return MAM_OK;
    const dim3 grid((unsigned)ceil_div(c.D, 16), 2);
    if (args->weight_type == MAM_F32)
        hipLaunchKernelGGL((rotary::weights_kernel<float>), grid, dim3(rotary::THREADS), 0, st, partial, groups, c.D, static_cast<float *>(dq_weight),
                           static_cast<float *>(dk_weight));
    else if (args->weight_type == MAM_BF16)
        hipLaunchKernelGGL((rotary::weights_kernel<bf16>), grid, dim3(rotary::THREADS), 0, st, partial, groups, c.D, static_cast<bf16 *>(dq_weight),
                           static_cast<bf16 *>(dk_weight));
    else
        hipLaunchKernelGGL((rotary::weights_kernel<f16>), grid, dim3(rotary::THREADS), 0, st, partial, groups, c.D, static_cast<f16 *>(dq_weight),
                           static_cast<f16 *>(dk_weight));
    return check_launch("rotary::weights_kernel");
}
