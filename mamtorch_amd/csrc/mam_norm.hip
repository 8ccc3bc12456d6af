// Layer norm over the rows of a matrix, forward and backward with the reduction of the weight's and bias's gradient, and the join of an
// encoder layer's halves: s = residual + dropout(x), y = norm(s).
//
//   mu = mean_c x, r = 1 / sqrt(mean_c (x - mu)^2 + eps), xh = (x - mu) r, y = xh w + b
//   g = dy w, dx = r (g - mean_c g - xh mean_c (g xh)), dw = sum_n dy xh, db = sum_n dy
//
// Bound by memory: a row is read once into the registers of the LANES lanes that own it (16 lanes of a wave, a wave, or a workgroup of 128
// to 1024, so that a lane holds at most 16 elements, 24 where that keeps a row in one wave), its mean is taken first and then the squares of
// what is left, all in fp32.  The backward's workgroups take rows in turn, the next one's loads on their way while this one is worked on, keep
// their sums of dw and db in registers over all of them and write them once; a second kernel adds the workgroups' sums in a fixed order, so
// two calls give the same bits.  Rows beyond 16384 elements are read again for each pass.
//
// Measured (forward, backward; a large copy reaches 5.2 TB/s): norm of 12608 x 768 fp32 17.2 and 22.2 us, 4.5 and 5.2 TB/s; of 16384 x 4096 fp16 62 and 89 us,
// 4.3 and 4.5 TB/s; join of 12608 x 768 fp32 37.4 and 47 us, 4.1 TB/s both.  Ragged rows in 16 bits are further off: 8191 x 1030 fp16 joined take 38 and
// 47 us, 1.8 TB/s: a wave's third piece is nearly empty, the generator forms a group more a piece, and one batch of waves holds all rows. 197 x 768: 4.5 us, the launch.
#include "mam_counter.h"
#include "mam_types.h"

namespace mam {
namespace norm {

constexpr int HELD = 16;                    // elements of a lane
constexpr int HELD_BY_WAVE = 24;            // the same where a wave has the row
constexpr int MOST_HELD = 1024 * HELD;      // longest row that is held in registers

// Threads of a workgroup: a row's lanes, or 256 for several rows.
template <int LANES>
constexpr int THREADS_OF = LANES > 64 ? LANES : 256;

// The row of a workgroup's that a thread belongs to; the same for a wave where rows are no less than that.
template <int LANES>
__device__ __forceinline__ int group_of()
{
    if constexpr (LANES >= 64) return __builtin_amdgcn_readfirstlane(threadIdx.x / LANES);
    return threadIdx.x / LANES;
}

struct Args {
    const void *x, *residual, *weight, *bias;   // residual: joins only
    void *s, *y;                                // s: joins only
    float *mean, *rstd;                         // may be NULL
    int64_t ldx, ldr, N;
    int C, w_same;                              // w_same: weight and bias are of x's type, else fp32
    float eps;
    Dropout drop;
};

struct BackwardArgs {
    const void *dy, *ds, *x, *weight;           // ds: joins only, may be NULL
    const float *mean, *rstd;
    void *dx, *dropped;                         // dropped: the gradient behind the dropout, joins only
    float *partial;                             // (workgroups, 2, C), or NULL
    int64_t lddy, lddsum, ldx, N;
    int C, w_same;
    Dropout drop;
};

// Sum over the LANES lanes that own a row, in every one of them; `scratch` holds two words for each wave of a workgroup-wide row.
template <int LANES>
__device__ __forceinline__ float row_sum(float v, float *scratch)
{
#pragma unroll
    for (int m = 1; m < (LANES < 64 ? LANES : 64); m <<= 1) v += __shfl_xor(v, m);
    if constexpr (LANES > 64) {
        __syncthreads();
        if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = v;
        __syncthreads();
        v = 0.0f;
#pragma unroll
        for (int w = 0; w < LANES / 64; ++w) v += scratch[w];
    }
    return v;
}

template <int LANES>
__device__ __forceinline__ void row_sums(float &a, float &b, float *scratch)
{
#pragma unroll
    for (int m = 1; m < (LANES < 64 ? LANES : 64); m <<= 1) {
        a += __shfl_xor(a, m);
        b += __shfl_xor(b, m);
    }
    if constexpr (LANES > 64) {
        __syncthreads();
        if ((threadIdx.x & 63) == 0) {
            scratch[2 * (threadIdx.x >> 6)] = a;
            scratch[2 * (threadIdx.x >> 6) + 1] = b;
        }
        __syncthreads();
        a = b = 0.0f;
#pragma unroll
        for (int w = 0; w < LANES / 64; ++w) {
            a += scratch[2 * w];
            b += scratch[2 * w + 1];
        }
    }
}

// A lane's piece of a join's sum, rounded to the type that it is handed on in: the norm is that of what is returned.
template <class T>
__device__ __forceinline__ void join_piece(const Args &a, int64_t row, int c, uint64_t offset, const Raw<T> &residual, const Raw<T> &x,
                                           float (&v)[kPack<T>])
{
    constexpr int N = kPack<T>;
    float f[N];
    keep_factors<N>(a.drop, offset, (uint64_t)row * (uint64_t)a.C + (uint64_t)c, ((uint32_t)row * (uint32_t)a.C & 3) == 0, f);
#pragma unroll
    for (int u = 0; u < N; ++u) v[u] = (float)(T)((float)residual[u] + keep_value((float)x[u], f[u]));
    store_pack<T>(static_cast<T *>(a.s) + row * a.C + c, a.C - c, v);
}

template <class T, int LANES, int PACKS, bool JOIN>
__global__ __launch_bounds__(THREADS_OF<LANES>) void norm_kernel(const Args a)
{
    constexpr int N = kPack<T>, THREADS = THREADS_OF<LANES>;
    __shared__ float scratch[LANES > 64 ? LANES / 64 : 1];
    const int lane = threadIdx.x % LANES;
    const int64_t row = (int64_t)blockIdx.x * (THREADS / LANES) + group_of<LANES>();
    if (row >= a.N) return;                     // rows of more than a wave: a workgroup's, which leaves as a whole
    const uint64_t offset = JOIN ? dropout_offset(a.drop) : 0;
    float v[PACKS][N];
    Raw<T> residual[PACKS], x[PACKS];
    if (JOIN) {         // all of them before the first store of s, which could be one of them for all that the compiler knows
#pragma unroll
        for (int i = 0; i < PACKS; ++i) {
            const int c = (lane + i * LANES) * N;
            residual[i] = load_raw<T>(static_cast<const T *>(a.residual) + row * a.ldr + c, a.C - c);
            x[i] = load_raw<T>(static_cast<const T *>(a.x) + row * a.ldx + c, a.C - c);
        }
    }
#pragma unroll
    for (int i = 0; i < PACKS; ++i) {
        const int c = (lane + i * LANES) * N;
        if (JOIN) {
            if (c < a.C) {
                join_piece<T>(a, row, c, offset, residual[i], x[i], v[i]);
            } else {
#pragma unroll
                for (int u = 0; u < N; ++u) v[i][u] = 0.0f;
            }
        } else {
            load_pack<T>(static_cast<const T *>(a.x) + row * a.ldx + c, a.C - c, v[i]);
        }
    }
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < PACKS; ++i)
#pragma unroll
        for (int u = 0; u < N; ++u) sum += v[i][u];
    const float inv = 1.0f / (float)a.C;
    const float mean = row_sum<LANES>(sum, scratch) * inv;
    float squares = 0.0f;
#pragma unroll
    for (int i = 0; i < PACKS; ++i)
#pragma unroll
        for (int u = 0; u < N; ++u) {
            v[i][u] -= mean;
            const float t = (lane + i * LANES) * N + u < a.C ? v[i][u] : 0.0f;
            squares = fmaf(t, t, squares);
        }
    const float rstd = 1.0f / sqrtf(row_sum<LANES>(squares, scratch) * inv + a.eps);
    if (lane == 0) {
        if (a.mean) a.mean[row] = mean;
        if (a.rstd) a.rstd[row] = rstd;
    }
#pragma unroll
    for (int i = 0; i < PACKS; ++i) {
        const int c = (lane + i * LANES) * N;
        if (c >= a.C) continue;
        float w[N], b[N];
        if (a.weight) {
            load_pack_of<T>(a.weight, a.w_same, c, a.C - c, w);
#pragma unroll
            for (int u = 0; u < N; ++u) w[u] *= rstd;
        } else {
#pragma unroll
            for (int u = 0; u < N; ++u) w[u] = rstd;
        }
        if (a.bias) {
            load_pack_of<T>(a.bias, a.w_same, c, a.C - c, b);
        } else {
#pragma unroll
            for (int u = 0; u < N; ++u) b[u] = 0.0f;
        }
#pragma unroll
        for (int u = 0; u < N; ++u) v[i][u] = fmaf(v[i][u], w[u], b[u]);
        store_pack<T>(static_cast<T *>(a.y) + row * a.C + c, a.C - c, v[i]);
    }
}

// Rows too long for the registers: a workgroup of 1024 reads its row three times.
template <class T, bool JOIN>
__global__ __launch_bounds__(1024) void norm_long_kernel(const Args a)
{
    constexpr int N = kPack<T>;
    __shared__ float scratch[16];
    const int64_t row = blockIdx.x;
    const uint64_t offset = JOIN ? dropout_offset(a.drop) : 0;
    const T *src = JOIN ? static_cast<const T *>(a.s) + row * a.C : static_cast<const T *>(a.x) + row * a.ldx;
    float sum = 0.0f;
    for (int c = threadIdx.x * N; c < a.C; c += 1024 * N) {
        float v[N];
        if (JOIN)
            join_piece<T>(a, row, c, offset, load_raw<T>(static_cast<const T *>(a.residual) + row * a.ldr + c, a.C - c),
                          load_raw<T>(static_cast<const T *>(a.x) + row * a.ldx + c, a.C - c), v);
        else load_pack<T>(src + c, a.C - c, v);
#pragma unroll
        for (int u = 0; u < N; ++u) sum += c + u < a.C ? v[u] : 0.0f;
    }
    const float inv = 1.0f / (float)a.C;
    const float mean = row_sum<1024>(sum, scratch) * inv;
    float squares = 0.0f;
    for (int c = threadIdx.x * N; c < a.C; c += 1024 * N) {     // a thread reads what it wrote itself
        float v[N];
        load_pack<T>(src + c, a.C - c, v);
#pragma unroll
        for (int u = 0; u < N; ++u) {
            const float t = c + u < a.C ? v[u] - mean : 0.0f;
            squares = fmaf(t, t, squares);
        }
    }
    const float rstd = 1.0f / sqrtf(row_sum<1024>(squares, scratch) * inv + a.eps);
    if (threadIdx.x == 0) {
        if (a.mean) a.mean[row] = mean;
        if (a.rstd) a.rstd[row] = rstd;
    }
    for (int c = threadIdx.x * N; c < a.C; c += 1024 * N) {
        float v[N], w[N], b[N];
        load_pack<T>(src + c, a.C - c, v);
        if (a.weight) load_pack_of<T>(a.weight, a.w_same, c, a.C - c, w);
        if (a.bias) load_pack_of<T>(a.bias, a.w_same, c, a.C - c, b);
#pragma unroll
        for (int u = 0; u < N; ++u) v[u] = fmaf(v[u] - mean, a.weight ? w[u] * rstd : rstd, a.bias ? b[u] : 0.0f);
        store_pack<T>(static_cast<T *>(a.y) + row * a.C + c, a.C - c, v);
    }
}

// A piece of the sum's own gradient, zeros where it has none.
template <class T>
__device__ __forceinline__ Raw<T> load_ds(const BackwardArgs &a, int64_t row, int c)
{
    return load_raw<T>(static_cast<const T *>(a.ds) + row * a.lddsum + c, a.ds ? a.C - c : 0);
}

// What leaves a join's backward for elements c .. of a row: the gradient of the sum, and behind the dropout.
template <class T>
__device__ __forceinline__ void join_out(const BackwardArgs &a, int64_t row, int c, uint64_t offset, const Raw<T> &ds, float (&g)[kPack<T>])
{
    constexpr int N = kPack<T>;
#pragma unroll
    for (int u = 0; u < N; ++u) g[u] += (float)ds[u];
    if (a.dx) store_pack<T>(static_cast<T *>(a.dx) + row * a.C + c, a.C - c, g);
    if (a.dropped) {
        float f[N];
        keep_factors<N>(a.drop, offset, (uint64_t)row * (uint64_t)a.C + (uint64_t)c, ((uint32_t)row * (uint32_t)a.C & 3) == 0, f);
#pragma unroll
        for (int u = 0; u < N; ++u) f[u] = keep_value(g[u], f[u]);
        store_pack<T>(static_cast<T *>(a.dropped) + row * a.C + c, a.C - c, f);
    }
}

// Workgroups take rows in turn.  A lane's columns are the same in every row, so its sums of dw and db stay in registers; the rows of
// a workgroup that are a wave's or a part of one are joined in LDS at the end.
template <class T, int LANES, int PACKS, bool JOIN>
__global__ __launch_bounds__(THREADS_OF<LANES>) void norm_backward_kernel(const BackwardArgs a)
{
    constexpr int N = kPack<T>, THREADS = THREADS_OF<LANES>, ROWS = THREADS / LANES;
    __shared__ float scratch[LANES > 64 ? 2 * (LANES / 64) : 1];
    __shared__ float joined[ROWS > 1 ? ROWS * LANES * PACKS * N : 1];
    const int lane = threadIdx.x % LANES, which = group_of<LANES>();
    const uint64_t offset = JOIN ? dropout_offset(a.drop) : 0;
    const float inv = 1.0f / (float)a.C;
    float w[PACKS][N], dw[PACKS][N], db[PACKS][N];
#pragma unroll
    for (int i = 0; i < PACKS; ++i) {
        const int c = (lane + i * LANES) * N;
        if (a.weight) {
            load_pack_of<T>(a.weight, a.w_same, c, a.C - c, w[i]);
        } else {
#pragma unroll
            for (int u = 0; u < N; ++u) w[i][u] = 1.0f;
        }
#pragma unroll
        for (int u = 0; u < N; ++u) dw[i][u] = db[i][u] = 0.0f;
    }
    Raw<T> next_dy[PACKS], next_x[PACKS];
    float next_mean = 0.0f, next_rstd = 0.0f;
    const auto load_row = [&](int64_t row) {
#pragma unroll
        for (int i = 0; i < PACKS; ++i) {
            const int c = (lane + i * LANES) * N;
            next_dy[i] = load_raw<T>(static_cast<const T *>(a.dy) + row * a.lddy + c, a.C - c);
            next_x[i] = load_raw<T>(static_cast<const T *>(a.x) + row * a.ldx + c, a.C - c);
        }
        next_mean = a.mean[row];
        next_rstd = a.rstd[row];
    };
    constexpr bool AHEAD = LANES < 1024;        // 16 waves have no registers for a second row
    const int64_t first = (int64_t)blockIdx.x * ROWS + which, step = (int64_t)gridDim.x * ROWS;
    if (AHEAD && first < a.N) load_row(first);
    for (int64_t row = first; row < a.N; row += step) {
        float dy[PACKS][N], xh[PACKS][N];
        if (!AHEAD) load_row(row);
        const float mean = next_mean, rstd = next_rstd;
#pragma unroll
        for (int i = 0; i < PACKS; ++i)
#pragma unroll
            for (int u = 0; u < N; ++u) {
                dy[i][u] = (float)next_dy[i][u];
                xh[i][u] = (float)next_x[i][u];
            }
        Raw<T> ds[JOIN ? PACKS : 1];
        if (JOIN) {
#pragma unroll
            for (int i = 0; i < PACKS; ++i) ds[i] = load_ds<T>(a, row, (lane + i * LANES) * N);
        }
        if (AHEAD && row + step < a.N) load_row(row + step);
        float sum = 0.0f, dot = 0.0f;
#pragma unroll
        for (int i = 0; i < PACKS; ++i)
#pragma unroll
            for (int u = 0; u < N; ++u) {       // past the end of the row dy is 0
                xh[i][u] = (xh[i][u] - mean) * rstd;
                dw[i][u] = fmaf(dy[i][u], xh[i][u], dw[i][u]);
                db[i][u] += dy[i][u];
                dy[i][u] *= w[i][u];
                sum += dy[i][u];
                dot = fmaf(dy[i][u], xh[i][u], dot);
            }
        row_sums<LANES>(sum, dot, scratch);
        sum *= inv;
        dot *= inv;
#pragma unroll
        for (int i = 0; i < PACKS; ++i) {
            const int c = (lane + i * LANES) * N;
            if (c >= a.C) continue;
#pragma unroll
            for (int u = 0; u < N; ++u) dy[i][u] = rstd * (dy[i][u] - sum - xh[i][u] * dot);
            if (JOIN) join_out<T>(a, row, c, offset, ds[i], dy[i]);
            else if (a.dx) store_pack<T>(static_cast<T *>(a.dx) + row * a.C + c, a.C - c, dy[i]);
        }
    }
    if (!a.partial) return;
    float *out = a.partial + (int64_t)blockIdx.x * 2 * a.C;
#pragma unroll
    for (int part = 0; part < 2; ++part) {
        if constexpr (ROWS > 1) {
            if (part) __syncthreads();
#pragma unroll
            for (int i = 0; i < PACKS; ++i)
#pragma unroll
                for (int u = 0; u < N; ++u) joined[which * (LANES * PACKS * N) + (lane + i * LANES) * N + u] = part ? db[i][u] : dw[i][u];
            __syncthreads();
            for (int c = threadIdx.x; c < a.C; c += THREADS) {
                float t = 0.0f;
#pragma unroll
                for (int r = 0; r < ROWS; ++r) t += joined[r * (LANES * PACKS * N) + c];
                out[part * a.C + c] = t;
            }
        } else {
#pragma unroll
            for (int i = 0; i < PACKS; ++i) {
                const int c = (lane + i * LANES) * N;
                store_pack<float, N>(out + part * a.C + c, a.C - c, part ? db[i] : dw[i]);
            }
        }
    }
}

// Rows too long for the registers: dx by a workgroup a row, in two passes.
template <class T, bool JOIN>
__global__ __launch_bounds__(1024) void norm_backward_long_kernel(const BackwardArgs a)
{
    constexpr int N = kPack<T>;
    __shared__ float scratch[32];
    const int64_t row = blockIdx.x;
    const uint64_t offset = JOIN ? dropout_offset(a.drop) : 0;
    const float mean = a.mean[row], rstd = a.rstd[row], inv = 1.0f / (float)a.C;
    float sum = 0.0f, dot = 0.0f;
    for (int pass = 0; pass < 2; ++pass) {
        for (int c = threadIdx.x * N; c < a.C; c += 1024 * N) {
            float g[N], xh[N], w[N];
            load_pack<T>(static_cast<const T *>(a.dy) + row * a.lddy + c, a.C - c, g);
            load_pack<T>(static_cast<const T *>(a.x) + row * a.ldx + c, a.C - c, xh);
            if (a.weight) {
                load_pack_of<T>(a.weight, a.w_same, c, a.C - c, w);
#pragma unroll
                for (int u = 0; u < N; ++u) g[u] *= w[u];
            }
#pragma unroll
            for (int u = 0; u < N; ++u) {
                xh[u] = (xh[u] - mean) * rstd;
                if (pass) {
                    g[u] = rstd * (g[u] - sum - xh[u] * dot);
                } else {
                    sum += g[u];
                    dot = fmaf(g[u], xh[u], dot);
                }
            }
            if (!pass) continue;
            if (JOIN) join_out<T>(a, row, c, offset, load_ds<T>(a, row, c), g);
            else if (a.dx) store_pack<T>(static_cast<T *>(a.dx) + row * a.C + c, a.C - c, g);
        }
        if (!pass) {
            row_sums<1024>(sum, dot, scratch);
            sum *= inv;
            dot *= inv;
        }
    }
}

// The sums of dw and db for them: a workgroup takes 256 packs of columns and a share of the rows.
template <class T>
__global__ __launch_bounds__(256) void norm_columns_kernel(const BackwardArgs a, int64_t rows_per_share)
{
    constexpr int N = kPack<T>;
    const int c = (blockIdx.x * 256 + threadIdx.x) * N;
    if (c >= a.C) return;
    const int64_t first = (int64_t)blockIdx.y * rows_per_share, end = first + rows_per_share < a.N ? first + rows_per_share : a.N;
    float dw[N], db[N];
#pragma unroll
    for (int u = 0; u < N; ++u) dw[u] = db[u] = 0.0f;
    for (int64_t row = first; row < end; ++row) {
        float dy[N], x[N];
        load_pack<T>(static_cast<const T *>(a.dy) + row * a.lddy + c, a.C - c, dy);
        load_pack<T>(static_cast<const T *>(a.x) + row * a.ldx + c, a.C - c, x);
        const float mean = a.mean[row], rstd = a.rstd[row];
#pragma unroll
        for (int u = 0; u < N; ++u) {
            dw[u] = fmaf(dy[u], (x[u] - mean) * rstd, dw[u]);
            db[u] += dy[u];
        }
    }
    float *out = a.partial + (int64_t)blockIdx.y * 2 * a.C;
    store_pack<float, N>(out + c, a.C - c, dw);
    store_pack<float, N>(out + a.C + c, a.C - c, db);
}

// dw and db from the workgroups' sums: a thread adds every 16th of them, the sixteen threads of a column join in LDS.
template <class W>
__global__ __launch_bounds__(1024) void norm_join_kernel(const float *__restrict__ partial, W *__restrict__ dw, W *__restrict__ db,
                                                         int C, int shares)
{
    __shared__ float part[16][64];
    const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6;
    const int column = blockIdx.x * 64 + tx;        // of 2 * C
    float sum = 0.0f;
    if (column < 2 * C) {
        const float *p = partial + column;
        int s = ty;
        for (; s + 7 * 16 < shares; s += 8 * 16) {
            float v[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) v[u] = p[(int64_t)(s + 16 * u) * 2 * C];
            sum += ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
        }
        for (; s < shares; s += 16) sum += p[(int64_t)s * 2 * C];
    }
    part[ty][tx] = sum;
    __syncthreads();
    if (ty == 0 && column < 2 * C) {
#pragma unroll
        for (int r = 1; r < 16; ++r) sum += part[r][tx];
        if (column < C) {
            if (dw) dw[column] = (W)sum;
        } else if (db) {
            db[column - C] = (W)sum;
        }
    }
}

// Lanes of a row: 16 while they hold it in two 16-byte pieces each, a wave up to HELD_BY_WAVE elements a lane, else the fewest of 128 to 1024
// that hold it with HELD each.
inline int lanes_of(int64_t C, int type)
{
    const int64_t pack = type == MAM_F32 ? 4 : 8;
    if (C <= 2 * 16 * pack) return 16;
    if (C <= 64 * HELD_BY_WAVE) return 64;
    int lanes = 128;
    while (C > lanes * HELD) lanes *= 2;
    return lanes;
}

// Workgroups of the backward: 16 waves for each CU, which have several rows each where there are many.
inline int64_t backward_shares(int64_t N, int64_t C, int type)
{
    if (C > MOST_HELD) {
        const int64_t s = ceil_div(N, 32);
        return s < 64 ? s : 64;
    }
    const int lanes = lanes_of(C, type), threads = lanes > 64 ? lanes : 256;
    const int64_t groups = ceil_div(N, threads / lanes), most = (int64_t)kNumCU * 1024 / threads;
    return groups < most ? groups : most;
}

template <class T, int LANES, int PACKS>
void launch_forward(const Args &a, bool join, hipStream_t st)
{
    constexpr int THREADS = THREADS_OF<LANES>;
    const dim3 grid((unsigned)ceil_div(a.N, THREADS / LANES));
    if (join) hipLaunchKernelGGL((norm_kernel<T, LANES, PACKS, true>), grid, dim3(THREADS), 0, st, a);
    else hipLaunchKernelGGL((norm_kernel<T, LANES, PACKS, false>), grid, dim3(THREADS), 0, st, a);
}

template <class T, int LANES, int PACKS>
void launch_backward(const BackwardArgs &a, bool join, int64_t shares, hipStream_t st)
{
    constexpr int THREADS = THREADS_OF<LANES>;
    if (join) hipLaunchKernelGGL((norm_backward_kernel<T, LANES, PACKS, true>), dim3((unsigned)shares), dim3(THREADS), 0, st, a);
    else hipLaunchKernelGGL((norm_backward_kernel<T, LANES, PACKS, false>), dim3((unsigned)shares), dim3(THREADS), 0, st, a);
}

// Calls f.operator()<LANES, PACKS>() with the lanes of a row and the pieces that each holds of it.
template <class T, class F>
void with_shape(int C, const F &f)
{
    constexpr int N = kPack<T>, MOST = HELD / N;
    const int lanes = lanes_of(C, N == 4 ? MAM_F32 : MAM_BF16);
    const int packs = (int)ceil_div(C, (int64_t)lanes * N);
    if (lanes == 16) {
        if (packs == 1) f.template operator()<16, 1>();
        else f.template operator()<16, 2>();
    } else if (lanes == 64) {
        if (packs <= 1) f.template operator()<64, 1>();
        else if (packs == 2) f.template operator()<64, 2>();
        else if (packs == 3) f.template operator()<64, 3>();
        else if constexpr (N == 4) {
            if (packs == 4) f.template operator()<64, 4>();
            else f.template operator()<64, 6>();
        }
    } else if (lanes == 128) {
        f.template operator()<128, MOST>();
    } else if (lanes == 256) {
        if constexpr (N == 4)
            if (packs == 3) return f.template operator()<256, 3>();
        f.template operator()<256, MOST>();
    } else if (lanes == 512) {
        if constexpr (N == 4)
            if (packs == 3) return f.template operator()<512, 3>();
        f.template operator()<512, MOST>();
    } else {
        if constexpr (N == 4)
            if (packs == 3) return f.template operator()<1024, 3>();
        f.template operator()<1024, MOST>();
    }
}

template <class T>
struct Forward {
    const Args &a;
    bool join;
    hipStream_t st;
    template <int LANES, int PACKS>
    void operator()() const { launch_forward<T, LANES, PACKS>(a, join, st); }
};

template <class T>
struct Backward {
    const BackwardArgs &a;
    bool join;
    int64_t shares;
    hipStream_t st;
    template <int LANES, int PACKS>
    void operator()() const { launch_backward<T, LANES, PACKS>(a, join, shares, st); }
};

template <class T>
int forward(const Args &a, bool join, hipStream_t st)
{
    if (a.C <= MOST_HELD) {
        with_shape<T>(a.C, Forward<T>{a, join, st});
        return check_launch("norm_kernel");
    }
    if (join) hipLaunchKernelGGL((norm_long_kernel<T, true>), dim3((unsigned)a.N), dim3(1024), 0, st, a);
    else hipLaunchKernelGGL((norm_long_kernel<T, false>), dim3((unsigned)a.N), dim3(1024), 0, st, a);
    return check_launch("norm_long_kernel");
}

template <class T>
int backward(const BackwardArgs &a, bool join, void *dw, void *db, int64_t shares, hipStream_t st)
{
    int rc;
    if (a.C <= MOST_HELD) {
        with_shape<T>(a.C, Backward<T>{a, join, shares, st});
        rc = check_launch("norm_backward_kernel");
    } else {
        if (join) hipLaunchKernelGGL((norm_backward_long_kernel<T, true>), dim3((unsigned)a.N), dim3(1024), 0, st, a);
        else hipLaunchKernelGGL((norm_backward_long_kernel<T, false>), dim3((unsigned)a.N), dim3(1024), 0, st, a);
        rc = check_launch("norm_backward_long_kernel");
        if (rc == MAM_OK && a.partial) {
            hipLaunchKernelGGL((norm_columns_kernel<T>), dim3((unsigned)ceil_div(a.C, 256 * kPack<T>), (unsigned)shares), dim3(256), 0, st, a,
                               ceil_div(a.N, shares));
            rc = check_launch("norm_columns_kernel");
        }
    }
    if (rc != MAM_OK || !a.partial) return rc;
    const dim3 grid((unsigned)ceil_div(2 * (int64_t)a.C, 64));
    if (a.w_same)
        hipLaunchKernelGGL((norm_join_kernel<T>), grid, dim3(1024), 0, st, a.partial, static_cast<T *>(dw), static_cast<T *>(db), a.C, (int)shares);
    else
        hipLaunchKernelGGL((norm_join_kernel<float>), grid, dim3(1024), 0, st, a.partial, static_cast<float *>(dw), static_cast<float *>(db), a.C,
                           (int)shares);
    return check_launch("norm_join_kernel");
}

int check_sizes(int64_t N, int64_t C, int type, int weight_type)
{
    if (N < 0 || C < 0) return fail(MAM_ERR_INVALID_ARGUMENT, "negative size");
    if (!is_type(type)) return fail(MAM_ERR_INVALID_ARGUMENT, "unknown element type %d", type);
    if (weight_type != type && weight_type != MAM_F32)
        return fail(MAM_ERR_INVALID_ARGUMENT, "weight and bias are of the operand's type or fp32, got type %d", weight_type);
    if (N > INT32_MAX / 2 || C > INT32_MAX / 2) return fail(MAM_ERR_UNSUPPORTED, "a dimension exceeds 2^30");
    return MAM_OK;
}

int run_forward(const Args &a, int type, bool join, void *stream)
{
    hipStream_t st = static_cast<hipStream_t>(stream);
    return type == MAM_F32 ? forward<float>(a, join, st) : type == MAM_BF16 ? forward<bf16>(a, join, st) : forward<f16>(a, join, st);
}

int run_backward(BackwardArgs &a, int type, bool join, void *dw, void *db, void *workspace, size_t workspace_bytes, void *stream)
{
    hipStream_t st = static_cast<hipStream_t>(stream);
    int64_t shares = backward_shares(a.N, a.C, type);
    a.partial = nullptr;
    if (dw || db) {
        const size_t need = mam_layer_norm_backward_workspace(a.N, a.C, type);
        if (!workspace || workspace_bytes < need)
            return fail(MAM_ERR_WORKSPACE, "the norm's backward needs %zu workspace bytes, got %zu", need, workspace ? workspace_bytes : (size_t)0);
        a.partial = static_cast<float *>(workspace);
    }
    return type == MAM_F32    ? backward<float>(a, join, dw, db, shares, st)
           : type == MAM_BF16 ? backward<bf16>(a, join, dw, db, shares, st)
                              : backward<f16>(a, join, dw, db, shares, st);
}

// No rows: the sums of nothing (the join of no shares).
int zero_weights(void *dw, void *db, int64_t C, int weight_type, hipStream_t st)
{
    if (!dw && !db) return MAM_OK;
    const dim3 grid((unsigned)ceil_div(2 * C, 64));
    const float *none = nullptr;
    if (weight_type == MAM_F32)
        hipLaunchKernelGGL((norm_join_kernel<float>), grid, dim3(1024), 0, st, none, static_cast<float *>(dw), static_cast<float *>(db), (int)C, 0);
    else        // zeros of both 16-bit types have the same bits
        hipLaunchKernelGGL((norm_join_kernel<f16>), grid, dim3(1024), 0, st, none, static_cast<f16 *>(dw), static_cast<f16 *>(db), (int)C, 0);
    return check_launch("norm_join_kernel");
}

}  // namespace norm
}  // namespace mam

extern "C" int mam_layer_norm(const void *x, int64_t ldx, const void *weight, const void *bias, double eps, void *y, float *mean, float *rstd,
                              int64_t N, int64_t C, int type, int weight_type, void *stream)
{
    using namespace mam;
    const int rc = norm::check_sizes(N, C, type, weight_type);
    if (rc != MAM_OK || N == 0 || C == 0) return rc;
    if (!x || !y) return fail(MAM_ERR_INVALID_ARGUMENT, "null pointer");
    if (ldx < C) return fail(MAM_ERR_INVALID_ARGUMENT, "leading dimension smaller than the row length");
    norm::Args a{};
    a.x = x; a.weight = weight; a.bias = bias; a.y = y; a.mean = mean; a.rstd = rstd;
    a.ldx = ldx; a.N = N; a.C = (int)C; a.w_same = weight_type == type; a.eps = (float)eps;
    return norm::run_forward(a, type, false, stream);
}

extern "C" size_t mam_layer_norm_backward_workspace(int64_t N, int64_t C, int type)
{
    if (N <= 0 || C <= 0 || !mam::is_type(type)) return 0;
    return (size_t)mam::norm::backward_shares(N, C, type) * 2 * (size_t)C * sizeof(float);
}

extern "C" int mam_layer_norm_backward(const void *dy, int64_t lddy, const void *x, int64_t ldx, const void *weight, const float *mean,
                                       const float *rstd, void *dx, void *dw, void *db, int64_t N, int64_t C, int type, int weight_type,
                                       void *workspace, size_t workspace_bytes, void *stream)
{
    using namespace mam;
    const int rc = norm::check_sizes(N, C, type, weight_type);
    if (rc != MAM_OK || C == 0) return rc;
    if (N == 0) return norm::zero_weights(dw, db, C, weight_type, static_cast<hipStream_t>(stream));
    if (!dy || !x || !mean || !rstd) return fail(MAM_ERR_INVALID_ARGUMENT, "null pointer");
    if (ldx < C || lddy < C) return fail(MAM_ERR_INVALID_ARGUMENT, "leading dimension smaller than the row length");
    norm::BackwardArgs a{};
    a.dy = dy; a.x = x; a.weight = weight; a.mean = mean; a.rstd = rstd; a.dx = dx;
    a.lddy = lddy; a.ldx = ldx; a.N = N; a.C = (int)C; a.w_same = weight_type == type;
    return norm::run_backward(a, type, false, dw, db, workspace, workspace_bytes, stream);
}

extern "C" int mam_add_dropout_layer_norm(const void *x, int64_t ldx, const void *residual, int64_t ldr, const mam_dropout_t *drop,
                                          const void *weight, const void *bias, double eps, void *y, void *s, float *mean, float *rstd,
                                          int64_t N, int64_t C, int type, int weight_type, void *stream)
{
    using namespace mam;
    int rc = norm::check_sizes(N, C, type, weight_type);
    if (rc != MAM_OK) return rc;
    norm::Args a{};
    rc = make_dropout(drop, a.drop);
    if (rc != MAM_OK || N == 0 || C == 0) return rc;
    if (!x || !residual || !y || !s) return fail(MAM_ERR_INVALID_ARGUMENT, "null pointer");
    if (ldx < C || ldr < C) return fail(MAM_ERR_INVALID_ARGUMENT, "leading dimension smaller than the row length");
    a.x = x; a.residual = residual; a.weight = weight; a.bias = bias; a.y = y; a.s = s; a.mean = mean; a.rstd = rstd;
    a.ldx = ldx; a.ldr = ldr; a.N = N; a.C = (int)C; a.w_same = weight_type == type; a.eps = (float)eps;
    return norm::run_forward(a, type, true, stream);
}

extern "C" int mam_add_dropout_layer_norm_backward(const void *dy, int64_t lddy, const void *ds, int64_t ldds, const void *s,
                                                   const void *weight, const float *mean, const float *rstd, const mam_dropout_t *drop,
                                                   void *d_residual, void *dx, void *dw, void *db, int64_t N, int64_t C, int type,
                                                   int weight_type, void *workspace, size_t workspace_bytes, void *stream)
{
    using namespace mam;
    int rc = norm::check_sizes(N, C, type, weight_type);
    if (rc != MAM_OK) return rc;
    norm::BackwardArgs a{};
    rc = make_dropout(drop, a.drop);
    if (rc != MAM_OK || C == 0) return rc;
    if (N == 0) return norm::zero_weights(dw, db, C, weight_type, static_cast<hipStream_t>(stream));
    if (!dy || !s || !mean || !rstd) return fail(MAM_ERR_INVALID_ARGUMENT, "null pointer");
    if (lddy < C || (ds && ldds < C)) return fail(MAM_ERR_INVALID_ARGUMENT, "leading dimension smaller than the row length");
    a.dy = dy; a.ds = ds; a.x = s; a.weight = weight; a.mean = mean; a.rstd = rstd; a.dx = d_residual; a.dropped = dx;
    a.lddy = lddy; a.lddsum = ldds; a.ldx = C; a.N = N; a.C = (int)C; a.w_same = weight_type == type;
    return norm::run_backward(a, type, true, dw, db, workspace, workspace_bytes, stream);
}
