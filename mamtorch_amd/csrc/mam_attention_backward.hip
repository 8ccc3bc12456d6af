// Differential attention, backward. With A = P1 - lambda P2 (Pm formed again from the scores and the forward's sums):
//
//   dV = A^T dO,  dA = dO V^T,  d1 = rowsum(dO O1),  d2 = rowsum(dO O2)
//   dS1 = P1 (dA - d1),  dS2 = -lambda P2 (dA - d2),  dQm = scale dSm Km,  dKm = scale dSm^T Qm,  dlambda = -sum d2
//
// Four kernels: what the rows need beside the scores (sums, d1, d2, lambda), dQ and the rows' d2 for dlambda by workgroups that own rows and pass over the keys, dK and dV
// by workgroups that own keys and pass over the rows of all heads that share them, and dlambda.  Scores and dA are formed in both of the
// middle ones, 7 parts of work instead of 5, and nothing is added to memory by more than one workgroup: no atomics, the same bits on every call.
//
// In 16-bit types A and dSm are rounded to the type where they enter a product; with the forward's rounding of A the step's results are 0.0025 from 64 bits in bf16 (2 x 4096
// causal), 0.0018 with fp32 throughout.  A second part of each would be one more product for each.
//
// Bound by the matrix cores in fp32 and by them and the vector units in turn in 16-bit types.  Measured, fp32 64 images of 197 tokens, 6 heads of 64/128: dQ
// 152 us (75 TFLOP/s, matrix cores busy in 60 % of the cycles), dK and dV 213 us (72 TFLOP/s, 59 %), both with the waits of short workgroups that the forward
// has.  bf16 2 x 4096 causal, 8 heads of 64/128: dQ 160 us (644 TFLOP/s), dK and dV 253 us (544); 2 x 2048 causal of 128/256: 102 us (506), 157 us (438).
#include "mam_attention.h"

#include <type_traits>

namespace mam {
namespace attention {

constexpr int STEP = KT;        // keys (dQ) or rows (dK, dV) of a tile

// What a row brings beside its query: five planes of B * Hkv * R floats, in fp16 a sixth, its gradient's size (below).  The queries' kernel, which is the last to read d2, puts it back as formed from the
// probabilities before they are rounded to the operands' type, for dlambda: rounded ones put an error of their type's last place into every row's d2, and
// their sum was over 1.5 times as far off as one that is rounded once.
enum { MINUS_SUM1, MINUS_SUM2, DOT1, DOT2, LAMBDA, PLANES, SIZE = PLANES };

// fp16 holds gradients of scores, dSm, as normal numbers from 2^-14 to 2^16 only: those of 4096 keys and a dO of 1e-4 are 2e-7, those of a dO behind a loss
// scaler can leave it at the top where dQ and dK do not.  So they are formed times 2^shift, a row's own for dQ and the workgroup's for dK, from the size of dO:
// its rows' sums of absolute values.  Ordinary gradients, of 2^3 to 2^9, are left as they are; smaller ones are brought up to 2^3, larger ones down to 2^9.
// P (dA - d) is at most a quarter of dA's range, half of size max |V|: it stays below 2^16 while values are below
// 2^13 beside small gradients that were brought up, and below 2^8 beside the largest.
// Measured, steps with and without: 4 x 1024 causal, 16 heads on 4, 352 and 349 us; 64 x 197, 6 heads, 192 and 188 us (the workgroup's size before its first tile).
template <class T>
constexpr bool SHIFTED = std::is_same<T, f16>::value;
__device__ __forceinline__ int shift_of(float size)
{
    const int e = __builtin_amdgcn_frexp_expf(size);        // size = m 2^e, m from 1/2 to 1
    return size > 0.0f ? (e < 4 ? 4 - e : e > 9 ? 9 - e : 0) : 0;
}

struct BackwardCall {
    Call a;
    const void *dout, *out;             // dout strided, out contiguous (B, Lq, H, dv)
    int64_t gb, gl, gh;
    const float *kept, *lse;            // KEPT<T> planes like out
    bool fast;                          // dout may be read by Stage<..., FAST> like the operands
    void *dq, *dk, *dv, *dlam;
    float *rows;                        // PLANES planes, one more in fp16
};

// A row's planes: 16 lanes a row.  Bound by memory: 116 MB (fp32, 64 x 197 tokens of 6 x 128) in 21 us, 5.5 TB/s.
template <class T>
__global__ __launch_bounds__(256) void rows_kernel(const BackwardCall g)
{
    const Call &a = g.a;
    const int64_t count = (int64_t)a.B * a.Hkv * a.R, id = (int64_t)blockIdx.x * 16 + threadIdx.x / 16;
    if (id >= count) return;
    const int lane = threadIdx.x & 15, row = (int)(id % a.R), bh = (int)(id / a.R), b = bh / a.Hkv;
    const int query = row / a.G, head = bh % a.Hkv * a.G + row % a.G;
    const T *grad = static_cast<const T *>(g.dout) + b * g.gb + query * g.gl + head * g.gh;
    const int64_t at = (((int64_t)b * a.Lq + query) * a.H + head) * a.dv;
    const int64_t plane = (int64_t)a.B * a.Lq * a.H * a.dv;
    float dot = 0.0f, dot2 = 0.0f, size = 0.0f;
    for (int c = lane * kPack<T>; c < a.dv; c += 16 * kPack<T>) {
        float v[kPack<T>], o[kPack<T>], o2[kPack<T>];
        load_pack<T>(grad + c, a.dv - c, v);
        if (KEPT<T> == 2) load_pack<float, kPack<T>>(g.kept + plane + at + c, a.dv - c, o);
        else load_pack<T>(static_cast<const T *>(g.out) + at + c, a.dv - c, o);
        load_pack<float, kPack<T>>(g.kept + at + c, a.dv - c, o2);
#pragma unroll
        for (int u = 0; u < kPack<T>; ++u) {
            dot = fmaf(v[u], o[u], dot);
            dot2 = fmaf(v[u], o2[u], dot2);
            size += fabsf(v[u]);
        }
    }
#pragma unroll
    for (int m = 1; m < 16; m <<= 1) {
        dot += __shfl_xor(dot, m);
        dot2 += __shfl_xor(dot2, m);
        if (SHIFTED<T>) size += __shfl_xor(size, m);
    }
    if (lane) return;
    const float lam = lambda_of(a, head, static_cast<const T *>(nullptr));
    const int64_t sums = ((int64_t)b * a.H + head) * a.Lq + query;
    g.rows[MINUS_SUM1 * count + id] = -g.lse[sums];
    g.rows[MINUS_SUM2 * count + id] = -g.lse[(int64_t)a.B * a.H * a.Lq + sums];
    g.rows[DOT1 * count + id] = KEPT<T> == 2 ? dot : fmaf(lam, dot2, dot);      // O1 = out + lambda O2
    g.rows[DOT2 * count + id] = dot2;
    g.rows[LAMBDA * count + id] = lam;
    if (SHIFTED<T>) g.rows[SIZE * count + id] = size * fmaxf(fabsf(lam), 1.0f);       // the second map's gradients come with lambda
}

// dlambda of a head, a workgroup each: its waves share the requests, or some waves a request where there are fewer.  Five loads after each other and
// the launch: 5 us.
template <class T>
__global__ __launch_bounds__(1024) void lambda_kernel(const BackwardCall g)
{
    __shared__ float part[16];
    const Call &a = g.a;
    const int head = blockIdx.x, hk = head / a.G, which = head % a.G;
    const float *dots = g.rows + DOT2 * (int64_t)a.B * a.Hkv * a.R;
    int groups = 1;
    while (groups < 16 && groups < a.B) groups *= 2;
    const int threads = 1024 / groups, group = threadIdx.x / threads;
    float sum = 0.0f;
    for (int b = group; b < a.B; b += groups) {
        const float *p = dots + ((int64_t)b * a.Hkv + hk) * a.R + which;
        for (int i = threadIdx.x % threads; i < a.Lq; i += 4 * threads) {
            float v[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) v[u] = i + u * threads < a.Lq ? p[(int64_t)(i + u * threads) * a.G] : 0.0f;
            sum -= (v[0] + v[1]) + (v[2] + v[3]);
        }
    }
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) sum += __shfl_xor(sum, m);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x) return;
    sum = 0.0f;
    for (int w = 0; w < 16; ++w) sum += part[w];
    if (a.lam_same) static_cast<T *>(g.dlam)[head] = (T)sum;
    else static_cast<float *>(g.dlam)[head] = sum;
}

// Waves of a SIMD that the registers are shared between: a lane holds its wave's operands and gradients, and 48 of scores.
template <class T, int TR, int D, int DV>
constexpr int OPERANDS = (2 * D + DV) * TR * (int)sizeof(T) / 256;
template <class T, int TR, int D, int DV>
constexpr int QUERIES_WAVES = OPERANDS<T, TR, D, DV> + D * TR / 32 <= 128 ? 2 : 1;
template <class T, int TR, int D, int DV>
constexpr int KEYS_WAVES = OPERANDS<T, TR, D, DV> + D * TR / 32 + DV * TR / 64 <= 128 ? 2 : 1;

template <int TR>
__device__ __forceinline__ void clear(Acc<TR> &c)
{
#pragma unroll
    for (int i = 0; i < TR * TR / 64; ++i) c[i] = 0.0f;
}

// A wave's accumulators (columns col .. of its lanes' rows) to memory, times `scale`.
template <class T, int TR>
__device__ __forceinline__ void store_columns(T *p, int left, const Acc<TR> &c, float scale)
{
#pragma unroll
    for (int f = 0; f < TR * TR / 64; f += 4) {
        const int col = (f / 4) * 4 * GROUPS<TR> + 4 * lane_group<TR>();
        float v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) v[u] = c[f + u] * scale;
        if (col < left) store_pack<T, 4>(p + col, left - col, v);
    }
}

template <class T, int TR, int D, int DV, bool FAST>
__global__ __launch_bounds__(256, (QUERIES_WAVES<T, TR, D, DV>)) void queries_kernel(const BackwardCall g, int row_tiles)
{
    constexpr int BUFFERS = TILES<T, D, DV>;
    typedef Stage<T, 256, STEP, 2, D, FAST> StageK;
    typedef Stage<T, 256, STEP, 1, DV, FAST> StageV;
    __shared__ __attribute__((aligned(16))) T k_tile[BUFFERS][STEP * StageK::PITCH];
    __shared__ __attribute__((aligned(16))) T v_tile[BUFFERS][STEP * StageV::PITCH];
    const Call &a = g.a;
    const Place<TR> at(a, row_tiles);

    const Source<T> qs{static_cast<const T *>(a.q) + at.b * a.qb + (int64_t)at.hk * a.G * a.qh, a.ql, a.qh, a.qm, a.G, a.d, a.inverse};
    const Source<T> gs{static_cast<const T *>(g.dout) + at.b * g.gb + (int64_t)at.hk * a.G * g.gh, g.gl, g.gh, 0, a.G, a.dv, a.inverse};
    const Source<T> ks{static_cast<const T *>(a.k) + at.b * a.kb + at.hk * a.kh, a.kl, 0, a.km, 1, a.d, 1.0f};
    const Source<T> vs{static_cast<const T *>(a.v) + at.b * a.vb + at.hk * a.vh, a.vl, 0, 0, 1, a.dv, 1.0f};
    Frag<T> q[2][D / KS<T, TR>], grad[DV / KS<T, TR>];
#pragma unroll
    for (int m = 0; m < 2; ++m) load_rows<T, TR, D>(qs, at.row, at.there, m, q[m]);
    load_rows<T, TR, DV>(gs, at.row, at.there, 0, grad);
    const int64_t count = (int64_t)a.B * a.Hkv * a.R;
    const float *plane = g.rows + ((int64_t)at.b * a.Hkv + at.hk) * a.R + at.row;
    const auto brought = [&](int p) { return at.there ? plane[p * count] : 0.0f; };      // a wave reads the planes of its own rows only
    const float shift = SHIFTED<T> ? (float)shift_of(brought(SIZE) / fmaxf(fabsf(brought(LAMBDA)), 1.0f)) : 0.0f, back = SHIFTED<T> ? __builtin_amdgcn_exp2f(-shift) : 1.0f;
    const float minus_sum[2] = {brought(MINUS_SUM1) + shift, brought(MINUS_SUM2) + shift}, dot[2] = {brought(DOT1), brought(DOT2)}, weight[2] = {1.0f, -brought(LAMBDA)};
    const float c = a.scale * LOG2E;
    float exact = 0.0f;         // this lane's share of sum_j P2 (dA - d2) with the d2 that was brought: the rest of the exact one

    Acc<TR> dq[2][D / TR];
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int blk = 0; blk < D / TR; ++blk) clear<TR>(dq[m][blk]);
    const auto seen = [&](int key) { return !a.mask || a.mask[at.b * a.mask_b + key] != 0; };
    StageK k_stage;
    StageV v_stage;
    k_stage.load(ks, 0, at.end, seen);
    v_stage.load(vs, 0, at.end, seen);
    if (BUFFERS == 2) {
        k_stage.store(k_tile[0]);
        v_stage.store(v_tile[0]);
    }
    // a tile's part of the loop, and a wave that is past its keys in a loop of its own, as in the forward
    int now = 0;
    const auto tile_of = [&](int key, const auto &use) {
        const bool more = key + STEP < at.end;
        if (BUFFERS == 1) {
            __syncthreads();
            k_stage.store(k_tile[0]);
            v_stage.store(v_tile[0]);
        }
        if (more) {
            k_stage.load(ks, key + STEP, at.end, seen);
            v_stage.load(vs, key + STEP, at.end, seen);
        }
        __syncthreads();
        use();
        if (BUFFERS == 2) {
            now ^= 1;
            if (more) {
                k_stage.store(k_tile[now]);
                v_stage.store(v_tile[now]);
            }
        }
    };
    int key = 0;
    const auto use = [&](auto limited, auto half, uint32_t word) {
        constexpr int PART = decltype(half)::value ? 2 : 1;
        Acc<TR> da[BLOCKS<TR>];
#pragma unroll
        for (int blk = 0; blk < BLOCKS<TR> / PART; ++blk) {
            clear<TR>(da[blk]);
#pragma unroll
            for (int kk = 0; kk < DV / KS<T, TR>; ++kk)
                mma<TR>(row_frag<T, TR>(v_tile[now], StageV::PITCH, blk * TR + lane_row<TR>(), kk), grad[kk], da[blk]);
        }
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            float ds[REGS<TR>];
#pragma unroll
            for (int blk = 0; blk < BLOCKS<TR> / PART; ++blk) {
                Acc<TR> s;
                clear<TR>(s);
#pragma unroll
                for (int kk = 0; kk < D / KS<T, TR>; ++kk)
                    mma<TR>(row_frag<T, TR>(k_tile[now] + m * D, StageK::PITCH, blk * TR + lane_row<TR>(), kk), q[m][kk], s);
#pragma unroll
                for (int i = 0; i < TR * TR / 64; ++i) {
                    const int f = blk * (TR * TR / 64) + i, n = index_of<TR>(f);
                    float p = __builtin_amdgcn_exp2f(fmaf(s[i], c, minus_sum[m]));
                    if (decltype(limited)::value && !(n < at.limit - key && (FAST || (word >> n & 1)))) p = 0.0f;
                    ds[f] = p * (da[blk][i] - dot[m]);          // the second map's factor -lambda is a row's: it comes at the end
                    if (m) exact += ds[f];
                }
            }
            Frag<T> frag[FRAGS<T, TR>];
            to_frags<T, TR>(ds, frag, FRAGS<T, TR> / PART);
#pragma unroll
            for (int blk = 0; blk < D / TR; ++blk)
#pragma unroll
                for (int j = 0; j < FRAGS<T, TR> / PART; ++j)
                    mma<TR>(column_frag<TR>(k_tile[now] + m * D, StageK::PITCH, blk * TR, j), frag[j], dq[m][blk]);
        }
    };
    if (FAST || !a.mask)
        for (; key + STEP <= at.wave_all; key += STEP) tile_of(key, [&] { use(std::false_type(), std::false_type(), 0); });
    const auto word_of = [&] { return !FAST && a.mask ? mask_word(a, at.b, key) : 0xffffffffu; };
    constexpr int SHORT = HALVES<T, TR> ? STEP / 2 : 0;
    for (; key + SHORT < at.wave_any; key += STEP) tile_of(key, [&] { use(std::true_type(), std::false_type(), word_of()); });
    if constexpr (SHORT > 0)
        if (key < at.wave_any) {
            tile_of(key, [&] { use(std::true_type(), std::true_type(), word_of()); });
            key += STEP;
        }
    for (; key < at.end; key += STEP) tile_of(key, [] {});
    exact = groups_sum<TR>(exact) * back;
    if (!at.there) return;
    if (lane_group<TR>() == 0) g.rows[DOT2 * count + ((int64_t)at.b * a.Hkv + at.hk) * a.R + at.row] = dot[1] + exact;
    if (!g.dq) return;
    T *out = static_cast<T *>(g.dq) + (((int64_t)at.b * a.Lq + at.query) * a.H + at.head) * 2 * a.d;
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int blk = 0; blk < D / TR; ++blk) store_columns<T, TR>(out + m * a.d + blk * TR, a.d - blk * TR, dq[m][blk], a.scale * weight[m] * back);
}

template <class T, int TR, int D, int DV, bool FAST>
__global__ __launch_bounds__(256, (KEYS_WAVES<T, TR, D, DV>)) void keys_kernel(const BackwardCall g, int key_tiles)
{
    constexpr int ROW_KEYS = 4 * TR, BUFFERS = TILES<T, D, DV>;
    typedef Stage<T, 256, STEP, 2, D, FAST> StageQ;
    typedef Stage<T, 256, STEP, 1, DV, FAST> StageG;
    __shared__ __attribute__((aligned(16))) T q_tile[BUFFERS][STEP * StageQ::PITCH];
    __shared__ __attribute__((aligned(16))) T g_tile[BUFFERS][STEP * StageG::PITCH];
    __shared__ __attribute__((aligned(16))) float planes[BUFFERS][PLANES][STEP];
    __shared__ float sizes[4];
    const Call &a = g.a;
    const int workgroups = KEYS_WAVES<T, TR, D, DV> == 2 ? gridDim.x : 2 * gridDim.x;       // as if two fit a CU
    const int heads = a.B * a.Hkv, bh = blockIdx.x % heads, tile = tile_of_turn(blockIdx.x / heads, key_tiles, false, workgroups);
    const int b = bh / a.Hkv, hk = bh % a.Hkv;
    const Reach reach = reach_of(a, b);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int first = tile * ROW_KEYS + wave * TR, key = first + lane_row<TR>();
    // rows that see a key begin at (key - reach.first) * G; past every row where none does
    const auto from = [&](int k) {
        const int64_t i = (int64_t)k - reach.first;
        return i <= 0 ? 0 : i >= a.Lq ? a.R : (int)(i * a.G);
    };
    const bool seen = key < reach.keys && from(key) < a.R && (!a.mask || a.mask[b * a.mask_b + key] != 0);
    const int lane_from = seen ? from(key) : a.R;
    const bool wave_seen = first < reach.keys;
    const int wave_any = wave_seen ? from(first) : a.R;
    const int wave_all = first + TR <= reach.keys && !a.mask ? from(first + TR - 1) : a.R;    // from here on every lane's key is seen
    const int begin = tile * ROW_KEYS < reach.keys ? from(tile * ROW_KEYS) / STEP * STEP : a.R;

    const Source<T> qs{static_cast<const T *>(a.q) + b * a.qb + (int64_t)hk * a.G * a.qh, a.ql, a.qh, a.qm, a.G, a.d, a.inverse};
    const Source<T> gs{static_cast<const T *>(g.dout) + b * g.gb + (int64_t)hk * a.G * g.gh, g.gl, g.gh, 0, a.G, a.dv, a.inverse};
    const Source<T> ks{static_cast<const T *>(a.k) + b * a.kb + hk * a.kh, a.kl, 0, a.km, 1, a.d, 1.0f};
    const Source<T> vs{static_cast<const T *>(a.v) + b * a.vb + hk * a.vh, a.vl, 0, 0, 1, a.dv, 1.0f};
    Frag<T> k[2][D / KS<T, TR>], v[DV / KS<T, TR>];
#pragma unroll
    for (int m = 0; m < 2; ++m) load_rows<T, TR, D>(ks, key, seen, m, k[m]);
    load_rows<T, TR, DV>(vs, key, seen, 0, v);
    const int64_t count = (int64_t)a.B * a.Hkv * a.R;
    const float *rows = g.rows + (int64_t)bh * a.R;
    const float c = a.scale * LOG2E;

    Acc<TR> dk[2][D / TR], dv[DV / TR];
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int blk = 0; blk < D / TR; ++blk) clear<TR>(dk[m][blk]);
#pragma unroll
    for (int blk = 0; blk < DV / TR; ++blk) clear<TR>(dv[blk]);
    const auto in = [](int) { return true; };
    StageQ q_stage;
    StageG g_stage;
    float plane = 0.0f;
    // a row past the last has a sum of +inf: its probabilities are 0
    const auto load_planes = [&](int row0) {
        const int p = threadIdx.x / STEP, row = row0 + threadIdx.x % STEP;
        if (p < PLANES) plane = row < a.R ? rows[p * count + row] : p <= MINUS_SUM2 ? -INFINITY : 0.0f;
    };
    if (begin < a.R) {
        q_stage.load(qs, begin, a.R, in);
        g_stage.load(gs, begin, a.R, in);
        load_planes(begin);
    }
    float up = 1.0f;            // 2^shift of the largest row that the workgroup's keys are seen by
    if (SHIFTED<T>) {           // behind the first tile's loads
        float size = 0.0f;
        for (int r = begin + threadIdx.x; r < a.R; r += 8 * 256) {       // eight loads on their way; past the end the last row again
            float v[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) v[u] = rows[SIZE * count + (r + 256 * u < a.R ? r + 256 * u : a.R - 1)];
#pragma unroll
            for (int u = 0; u < 8; ++u) size = fmaxf(size, v[u]);
        }
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) size = fmaxf(size, __shfl_xor(size, m));
        if ((threadIdx.x & 63) == 0) sizes[wave] = size;
        __syncthreads();
        size = fmaxf(fmaxf(sizes[0], sizes[1]), fmaxf(sizes[2], sizes[3]));
        up = __builtin_amdgcn_exp2f((float)__builtin_amdgcn_readfirstlane(shift_of(size)));
    }
    const float plane_up = threadIdx.x / STEP == DOT1 || threadIdx.x / STEP == DOT2 ? up : 1.0f;
    const auto store = [&](int to) {
        q_stage.store(q_tile[to]);
        g_stage.store(g_tile[to]);
        // scaled here and not where it is asked for, which would wait for it
        if (threadIdx.x < PLANES * STEP) planes[to][threadIdx.x / STEP][threadIdx.x % STEP] = SHIFTED<T> ? plane * plane_up : plane;
    };
    if (BUFFERS == 2 && begin < a.R) store(0);
    int at = 0;
    const auto tile_of = [&](int row, const auto &use) {
        const bool more = row + STEP < a.R;
        if (BUFFERS == 1) {
            __syncthreads();
            store(0);
        }
        if (more) {
            q_stage.load(qs, row + STEP, a.R, in);
            g_stage.load(gs, row + STEP, a.R, in);
            load_planes(row + STEP);
        }
        __syncthreads();
        use();
        if (BUFFERS == 2) {
            at ^= 1;
            if (more) store(at);
        }
    };
    int row = begin;
    for (; row + STEP <= wave_any && row < a.R; row += STEP) tile_of(row, [] {});        // rows that see none of the wave's keys
    const auto scores = [&](int m, int blk, auto limited, float (&p)[REGS<TR>]) {      // probabilities of one map
        Acc<TR> s;
        clear<TR>(s);
#pragma unroll
        for (int kk = 0; kk < D / KS<T, TR>; ++kk)
            mma<TR>(row_frag<T, TR>(q_tile[at] + m * D, StageQ::PITCH, blk * TR + lane_row<TR>(), kk), k[m][kk], s);
#pragma unroll
        for (int i = 0; i < TR * TR / 64; ++i) {
            const int f = blk * (TR * TR / 64) + i, n = index_of<TR>(f);
            p[f] = __builtin_amdgcn_exp2f(fmaf(s[i], c, planes[at][m ? MINUS_SUM2 : MINUS_SUM1][n]));
            if (decltype(limited)::value && row + n < lane_from) p[f] = 0.0f;
            if (m) p[f] *= planes[at][LAMBDA][n];       // the second map's with lambda
        }
    };
    const auto use = [&](auto limited, auto half) {
        constexpr int PART = decltype(half)::value ? 2 : 1;
        Acc<TR> da[BLOCKS<TR>];
        float p[2][REGS<TR>];
#pragma unroll
        for (int blk = 0; blk < BLOCKS<TR> / PART; ++blk) {
            clear<TR>(da[blk]);
#pragma unroll
            for (int kk = 0; kk < DV / KS<T, TR>; ++kk)
                mma<TR>(row_frag<T, TR>(g_tile[at], StageG::PITCH, blk * TR + lane_row<TR>(), kk), v[kk], da[blk]);
        }
        const auto add_keys = [&](int m) {
            Frag<T> frag[FRAGS<T, TR>];
#pragma unroll
            for (int f = 0; f < REGS<TR> / PART; ++f) {
                const float all = da[f / (TR * TR / 64)][f % (TR * TR / 64)], own = planes[at][m ? DOT2 : DOT1][index_of<TR>(f)];
                const float d = SHIFTED<T> ? fmaf(all, up, -own) : all - own;
                p[m][f] = (m ? -p[m][f] : p[m][f]) * d;
            }
            to_frags<T, TR>(p[m], frag, FRAGS<T, TR> / PART);
#pragma unroll
            for (int blk = 0; blk < D / TR; ++blk)
#pragma unroll
                for (int j = 0; j < FRAGS<T, TR> / PART; ++j)
                    mma<TR>(column_frag<TR>(q_tile[at] + m * D, StageQ::PITCH, blk * TR, j), frag[j], dk[m][blk]);
        };
#pragma unroll
        for (int m = 0; m < 2; ++m) {
#pragma unroll
            for (int blk = 0; blk < BLOCKS<TR> / PART; ++blk) scores(m, blk, limited, p[m]);
        }
        {
            float diff[REGS<TR>];
            Frag<T> frag[FRAGS<T, TR>];
#pragma unroll
            for (int f = 0; f < REGS<TR> / PART; ++f) diff[f] = p[0][f] - p[1][f];
            to_frags<T, TR>(diff, frag, FRAGS<T, TR> / PART);
#pragma unroll
            for (int blk = 0; blk < DV / TR; ++blk)
#pragma unroll
                for (int j = 0; j < FRAGS<T, TR> / PART; ++j) mma<TR>(column_frag<TR>(g_tile[at], StageG::PITCH, blk * TR, j), frag[j], dv[blk]);
        }
        add_keys(0);
        add_keys(1);
    };
    // Dividing the two gradients between two passes of fewer registers costs the scores twice: 228 + 151 us where one pass takes 252.
    // Rows that a limit cuts and rows that it does not have loops of their own, and so have the rows before them: a condition in the loop has
    // the accumulators copied in every turn (2 x 4096 causal bf16: 348 us with conditions, 252 in loops).
    for (; row < wave_all && row < a.R; row += STEP) tile_of(row, [&] { use(std::true_type(), std::false_type()); });
    constexpr int SHORT = HALVES<T, TR> ? STEP / 2 : 0;
    for (; row + SHORT < a.R; row += STEP) tile_of(row, [&] { use(std::false_type(), std::false_type()); });
    if constexpr (SHORT > 0)
        if (row < a.R) tile_of(row, [&] { use(std::false_type(), std::true_type()); });
    if (key >= a.Lk) return;
    const int64_t place = ((int64_t)b * a.Lk + key) * a.Hkv + hk;
    if (g.dk) {
        T *out = static_cast<T *>(g.dk) + place * 2 * a.d;
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int blk = 0; blk < D / TR; ++blk) store_columns<T, TR>(out + m * a.d + blk * TR, a.d - blk * TR, dk[m][blk], a.scale * (1.0f / up));
    }
    if (g.dv) {
        T *out = static_cast<T *>(g.dv) + place * a.dv;
#pragma unroll
        for (int blk = 0; blk < DV / TR; ++blk) store_columns<T, TR>(out + blk * TR, a.dv - blk * TR, dv[blk], 1.0f);
    }
}

template <class T>
struct Backward {
    const BackwardCall &g;
    hipStream_t st;
    template <int D, int DV>
    int operator()() const
    {
        constexpr int TR = TILE_ROWS<T, D>;
        const Call &a = g.a;
        const int64_t rows = (int64_t)a.B * a.Hkv * a.R, row_tiles = ceil_div(a.R, 4 * TR), key_tiles = ceil_div(a.Lk, 4 * TR);
        if (ceil_div(rows, 16) > INT32_MAX || key_tiles * a.B * a.Hkv > INT32_MAX) return fail(MAM_ERR_UNSUPPORTED, "too many tiles");
        int rc = MAM_OK;
        if (rows > 0) {
            hipLaunchKernelGGL((rows_kernel<T>), dim3((unsigned)ceil_div(rows, 16)), dim3(256), 0, st, g);
            rc = check_launch("attention::rows_kernel");
        }
        // before the queries' kernel, which changes d2
        if (rc == MAM_OK && (g.dk || g.dv) && key_tiles * a.B * a.Hkv > 0) {
            const dim3 grid((unsigned)(key_tiles * a.B * a.Hkv));
            if (a.fast && g.fast) hipLaunchKernelGGL((keys_kernel<T, TR, D, DV, true>), grid, dim3(256), 0, st, g, (int)key_tiles);
            else hipLaunchKernelGGL((keys_kernel<T, TR, D, DV, false>), grid, dim3(256), 0, st, g, (int)key_tiles);
            rc = check_launch("attention::keys_kernel");
        }
        if (rc == MAM_OK && (g.dq || g.dlam) && rows > 0) {
            const dim3 grid((unsigned)(row_tiles * a.B * a.Hkv));
            if (a.fast) hipLaunchKernelGGL((queries_kernel<T, TR, D, DV, true>), grid, dim3(256), 0, st, g, (int)row_tiles);
            else hipLaunchKernelGGL((queries_kernel<T, TR, D, DV, false>), grid, dim3(256), 0, st, g, (int)row_tiles);
            rc = check_launch("attention::queries_kernel");
        }
        if (rc == MAM_OK && g.dlam && a.H > 0) {
            hipLaunchKernelGGL((lambda_kernel<T>), dim3((unsigned)a.H), dim3(1024), 0, st, g);
            rc = check_launch("attention::lambda_kernel");
        }
        return rc;
    }
};

}  // namespace attention
}  // namespace mam

extern "C" size_t mam_diff_attention_backward_workspace(const mam_diff_attention_t *args)
{
    if (!args || args->B <= 0 || args->Lq <= 0 || args->H <= 0) return 0;
    return (size_t)(mam::attention::PLANES + (args->type == MAM_F16 ? 1 : 0)) * (size_t)args->B * (size_t)args->Lq * (size_t)args->H * sizeof(float);
}

extern "C" int mam_diff_attention_backward(const mam_diff_attention_t *args, const void *dout, const int64_t *dout_stride, const void *out,
                                           const float *kept, const float *lse, void *dq, void *dk, void *dv, void *dlam, void *workspace,
                                           size_t workspace_bytes, void *stream)
{
    using namespace mam;
    attention::BackwardCall g{};
    const int rc = attention::fill_call(args, g.a);
    if (rc != MAM_OK) return rc;
    const attention::Call &a = g.a;
    const bool rows = a.B > 0 && a.R > 0;
    if (rows && (!a.q || !a.lam || !dout || !dout_stride || !out || !kept || !lse)) return fail(MAM_ERR_INVALID_ARGUMENT, "null pointer");
    if (a.B > 0 && a.Lk > 0 && a.H > 0 && (!a.k || !a.v)) return fail(MAM_ERR_INVALID_ARGUMENT, "null pointer");
    const size_t need = mam_diff_attention_backward_workspace(args);
    if (need > 0 && (!workspace || workspace_bytes < need))
        return fail(MAM_ERR_WORKSPACE, "the attention's backward needs %zu workspace bytes, got %zu", need, workspace ? workspace_bytes : (size_t)0);
    g.dout = dout; g.out = out; g.kept = kept; g.lse = lse;
    if (dout_stride) { g.gb = dout_stride[0]; g.gl = dout_stride[1]; g.gh = dout_stride[2]; }
    g.fast = attention::fast_operand(dout, type_size(args->type), a.dv, g.gb, g.gl, g.gh, 0, a.G);
    g.dq = dq; g.dk = dk; g.dv = dv; g.dlam = dlam;
    g.rows = static_cast<float *>(workspace);
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (args->type == MAM_F32) return attention::with_head_sizes(a.d, a.dv, attention::Backward<float>{g, st});
    if (args->type == MAM_BF16) return attention::with_head_sizes(a.d, a.dv, attention::Backward<bf16>{g, st});
    return attention::with_head_sizes(a.d, a.dv, attention::Backward<f16>{g, st});
}
