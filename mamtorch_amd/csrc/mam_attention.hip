// Differential attention, forward: out = softmax(scale Q1 K1^T) V - lambda softmax(scale Q2 K2^T) V for each head, with a
// running maximum and sum for each of the two softmaxes and each row, so that no score leaves the registers.
//
// A workgroup of four waves shares tiles of 32 keys in LDS, each wave with TR rows of its own (16 or 32, mam_attention.h).  The next tile's loads are
// in flight while this one is used.  fp32 passes over the keys once (tiles_kernel), 16-bit types twice (twice_kernel, below).
//
// fp32 is bound by the matrix cores: 64 images of 197 tokens, 6 heads of 64/128, 11.4 GFLOP in 159 us, 72 TFLOP/s where a large library product
// reaches 151.  They are busy in 58 % of its cycles; a workgroup has 7 tiles only, and the rest is the loads before its first tile, which all
// workgroups that begin together wait for at once, and its last stores.  Three waves a SIMD over one tile buffer instead of two over two: 166 -> 201 us.
#include "mam_attention.h"

#include <type_traits>

namespace mam {
namespace attention {

struct ForwardOut {
    void *out;                  // (B, Lq, H, dv) contiguous
    float *kept;                // KEPT<T> planes like it: the second map's product, in 16-bit types the first's as well; or NULL
    float *lse;                 // (2, B, H, Lq): log2 of the sums of exponentials, or NULL
};

// A wave's running state of TR rows.
template <class T, int TR, int D, int DV, bool MASKED>
struct State {
    Acc<TR> o[2][DV / TR];
    float top[2], sum[2];       // maximum (powers of two) that the exponentials are relative to; this lane's share of their sum

    __device__ __forceinline__ void clear()
    {
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            top[m] = -INFINITY;
            sum[m] = 0.0f;
#pragma unroll
            for (int b = 0; b < DV / TR; ++b)
#pragma unroll
                for (int i = 0; i < TR * TR / 64; ++i) o[m][b][i] = 0.0f;
        }
    }

    // Scores of one map (32 keys x TR rows) to probabilities relative to `top`, which rises first where it has to.
    template <bool LIMITED, int USED>
    __device__ __forceinline__ void softmax(int m, const Acc<TR> (&s)[BLOCKS<TR>], float c, int limit, uint32_t word, float (&p)[REGS<TR>])
    {
        float most = -INFINITY;
#pragma unroll
        for (int f = 0; f < USED; ++f) {
            float v = s[f / (TR * TR / 64)][f % (TR * TR / 64)];
            if constexpr (LIMITED) {
                const int key = index_of<TR>(f);
                v = key < limit && (!MASKED || (word >> key & 1)) ? v : -INFINITY;
            }
            p[f] = v;
            most = fmaxf(most, v);
        }
        most = groups_max<TR>(most) * c;
        if (__any(most > top[m] + SLACK)) {
            asm volatile("; a new maximum");       // kept a branch: as selects it is two operations for each accumulator and tile
            const float rise = fmaxf(top[m], most), factor = rise == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(top[m] - rise);
            top[m] = rise;
            sum[m] *= factor;
#pragma unroll
            for (int b = 0; b < DV / TR; ++b)
#pragma unroll
                for (int i = 0; i < TR * TR / 64; ++i) o[m][b][i] *= factor;
        }
        const float base = top[m] == -INFINITY ? 0.0f : top[m];
        float add = 0.0f;
#pragma unroll
        for (int f = 0; f < USED; ++f) {
            p[f] = __builtin_amdgcn_exp2f(fmaf(p[f], c, -base));
            add += p[f];
        }
        sum[m] += add;
    }

    // 32 keys (the first 16: HALF): their scores, probabilities, and the products with their values.
    template <bool LIMITED, bool HALF>
    __device__ __forceinline__ void keys(const Frag<T> (&q)[2][D / KS<T, TR>], const T *k_tile, int k_pitch, const T *v_tile, int v_pitch,
                                         float c, int limit, uint32_t word)
    {
        constexpr int PART = HALF ? 2 : 1, USED = REGS<TR> / PART;
        Frag<T> frag[2][FRAGS<T, TR>];
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            Acc<TR> s[BLOCKS<TR>];
#pragma unroll
            for (int b = 0; b < BLOCKS<TR> / PART; ++b) {
#pragma unroll
                for (int i = 0; i < TR * TR / 64; ++i) s[b][i] = 0.0f;
#pragma unroll
                for (int kk = 0; kk < D / KS<T, TR>; ++kk)
                    mma<TR>(row_frag<T, TR>(k_tile + m * D, k_pitch, b * TR + lane_row<TR>(), kk), q[m][kk], s[b]);
            }
            float p[REGS<TR>];
            softmax<LIMITED, USED>(m, s, c, limit, word, p);
            to_frags<T, TR>(p, frag[m], FRAGS<T, TR> / PART);
        }
#pragma unroll
        for (int b = 0; b < DV / TR; ++b) {
#pragma unroll
            for (int j = 0; j < FRAGS<T, TR> / PART; ++j) {
                const Frag<T> v = column_frag<TR>(v_tile, v_pitch, b * TR, j);
                mma<TR>(v, frag[0][j], o[0][b]);
                mma<TR>(v, frag[1][j], o[1][b]);
            }
        }
    }
};

// Waves of a SIMD that the registers are shared between: accumulators take DV * TR / 32 of a lane's, queries D * TR * size / 128.
template <class T, int TR, int D, int DV>
constexpr int WAVES = DV * TR / 32 + D * TR * (int)sizeof(T) / 128 <= 160 ? 2 : 1;

template <class T, int TR, int D, int DV, bool FAST>
__global__ __launch_bounds__(256, (WAVES<T, TR, D, DV>)) void tiles_kernel(const Call a, const ForwardOut out, int row_tiles)
{
    constexpr int BUFFERS = TILES<T, D, DV>;
    typedef Stage<T, 256, KT, 2, D, FAST> StageK;
    typedef Stage<T, 256, KT, 1, DV, FAST> StageV;
    __shared__ __attribute__((aligned(16))) T k_tile[BUFFERS][KT * StageK::PITCH];
    __shared__ __attribute__((aligned(16))) T v_tile[BUFFERS][KT * StageV::PITCH];
    const Place<TR> at(a, row_tiles);

    const Source<T> qs{static_cast<const T *>(a.q) + at.b * a.qb + (int64_t)at.hk * a.G * a.qh, a.ql, a.qh, a.qm, a.G, a.d, a.inverse};
    const Source<T> ks{static_cast<const T *>(a.k) + at.b * a.kb + at.hk * a.kh, a.kl, 0, a.km, 1, a.d, 1.0f};
    const Source<T> vs{static_cast<const T *>(a.v) + at.b * a.vb + at.hk * a.vh, a.vl, 0, 0, 1, a.dv, 1.0f};
    Frag<T> q[2][D / KS<T, TR>];
#pragma unroll
    for (int m = 0; m < 2; ++m) load_rows<T, TR, D>(qs, at.row, at.there, m, q[m]);
    const float c = a.scale * LOG2E;

    State<T, TR, D, DV, !FAST> state;
    state.clear();
    // a key that nobody sees is zeros in LDS, whatever its memory holds
    const auto seen = [&](int key) { return !a.mask || a.mask[at.b * a.mask_b + key] != 0; };
    StageK k_stage;
    StageV v_stage;
    k_stage.load(ks, 0, at.end, seen);
    v_stage.load(vs, 0, at.end, seen);
    if (BUFFERS == 2) {
        k_stage.store(k_tile[0]);
        v_stage.store(v_tile[0]);
    }
    // A tile's part of the loop: `use` is what a wave that sees some of its keys does.  Waves that are past their keys go on loading for the others, in a
    // loop of its own (a condition around the products has the accumulators copied in every tile).
    int now = 0;
    const auto tile_of = [&](int key, const auto &use) {
        const bool more = key + KT < at.end;
        if (BUFFERS == 1) {
            __syncthreads();
            k_stage.store(k_tile[0]);
            v_stage.store(v_tile[0]);
        }
        if (more) {
            k_stage.load(ks, key + KT, at.end, seen);
            v_stage.load(vs, key + KT, at.end, seen);
        }
        __syncthreads();
        use();
        if (BUFFERS == 2) {
            now ^= 1;
            if (more) {         // the other tile: every wave is past it
                k_stage.store(k_tile[now]);
                v_stage.store(v_tile[now]);
            }
        }
    };
    int key = 0;
    if (FAST || !a.mask)
        for (; key + KT <= at.wave_all; key += KT)
            tile_of(key, [&] { state.template keys<false, false>(q, k_tile[now], StageK::PITCH, v_tile[now], StageV::PITCH, c, 0, 0); });
    const auto limited = [&](auto half) {
        const uint32_t word = !FAST && a.mask ? mask_word(a, at.b, key) : 0xffffffffu;
        state.template keys<true, decltype(half)::value>(q, k_tile[now], StageK::PITCH, v_tile[now], StageV::PITCH, c, at.limit - key, word);
    };
    constexpr int SHORT = HALVES<T, TR> ? KT / 2 : 0;
    for (; key + SHORT < at.wave_any; key += KT) tile_of(key, [&] { limited(std::false_type()); });
    if constexpr (SHORT > 0)
        if (key < at.wave_any) {
            tile_of(key, [&] { limited(std::true_type()); });
            key += KT;
        }
    for (; key < at.end; key += KT) tile_of(key, [] {});
    if (!at.there) return;
    const float lam = lambda_of(a, at.head, static_cast<const T *>(nullptr));
    float inv[2], total[2];
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        total[m] = groups_sum<TR>(state.sum[m]);
        inv[m] = total[m] > 0.0f ? 1.0f / total[m] : 0.0f;         // a row that sees nothing is zeros
    }
    const int64_t place = (((int64_t)at.b * a.Lq + at.query) * a.H + at.head) * a.dv;
#pragma unroll
    for (int blk = 0; blk < DV / TR; ++blk)
#pragma unroll
        for (int f = 0; f < TR * TR / 64; f += 4) {
            const int col = blk * TR + (f / 4) * 4 * GROUPS<TR> + 4 * lane_group<TR>();
            if (col >= a.dv) continue;
            float o[4], o2[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                o2[u] = state.o[1][blk][f + u] * inv[1];
                o[u] = fmaf(-lam, o2[u], state.o[0][blk][f + u] * inv[0]);
            }
            store_pack<T, 4>(static_cast<T *>(out.out) + place + col, a.dv - col, o);
            if (out.kept) store_pack<float, 4>(out.kept + place + col, a.dv - col, o2);
        }
    if (out.lse && lane_group<TR>() == 0) {
#pragma unroll
        for (int m = 0; m < 2; ++m)
            out.lse[(((int64_t)m * a.B + at.b) * a.H + at.head) * a.Lq + at.query] = total[m] > 0.0f ? state.top[m] + log2f(total[m]) : INFINITY;
    }
}

// ---- 16-bit types: the keys twice ----
// A probability rounded to 16 bits is as far off as the rounded result, and of two maps both errors come to it; with a second part of
// each (as fp32 keeps them) products grow by half.  Instead a first pass over the keys finds each row's two sums, and the second forms
// A = P1 - lambda P2 in fp32 and rounds it once, for ONE product with the values: 2 (4 D + Dv) flops a (query, key) against 2 (2 D + 2 Dv), half the
// accumulators, nothing to scale when a maximum rises, and less work for the vector units beside the exponentials, of which there are twice
// as many.  A training forward brings P2's product with the values as well, which the backward reads.
//
// Bound by the vector units and the matrix cores in turn: two exponentials a (query, key) and pass stand beside products of 16 bits.  Measured: 8 x 2048 all keys,
// 8 heads of 64/128, bf16 356 us (206 GFLOP done, 579 TFLOP/s; a large library product reaches 1079); 2 x 4096 causal with what training keeps
// 244 us (137 GFLOP, 564 TFLOP/s; matrix cores busy in 27 % of the cycles, vector units in about 36 %).  Deeper pipelines of the scores and queries kept in
// LDS measured the same or slower (340 to 435 us where the first is 356).
//
// Both products are scaled so that fp16 holds the probabilities of long rows as normal numbers: P2 by g2 = min(the larger sum, 2^12), A by
// g = min(g2, 2^12 / |lambda|), which keeps both of its terms below 2^13 whatever lambda is.

// Both maps' scores of 32 keys.
template <class T, int TR, int D>
__device__ __forceinline__ void scores_of(const Frag<T> (&q)[2][D / KS<T, TR>], const T *k_tile, int pitch, Acc<TR> (&s)[2][BLOCKS<TR>])
{
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int b = 0; b < BLOCKS<TR>; ++b) {
#pragma unroll
            for (int i = 0; i < TR * TR / 64; ++i) s[m][b][i] = 0.0f;
#pragma unroll
            for (int kk = 0; kk < D / KS<T, TR>; ++kk)
                mma<TR>(row_frag<T, TR>(k_tile + m * D, pitch, b * TR + lane_row<TR>(), kk), q[m][kk], s[m][b]);
        }
}

template <bool MASKED, int TR>
__device__ __forceinline__ void hide(Acc<TR> (&s)[2][BLOCKS<TR>], int limit, uint32_t word)
{
    constexpr int AR = TR * TR / 64;
#pragma unroll
    for (int f = 0; f < REGS<TR>; ++f) {
        const int key = index_of<TR>(f);
        const bool seen = key < limit && (!MASKED || (word >> key & 1));
#pragma unroll
        for (int m = 0; m < 2; ++m) s[m][f / AR][f % AR] = seen ? s[m][f / AR][f % AR] : -INFINITY;
    }
}

template <class T, int TR, int D, int DV, bool FAST, bool KEEP>
__global__ __launch_bounds__(256, 2) void twice_kernel(const Call a, const ForwardOut out, int row_tiles)
{
    // TURN: two tiles between barriers measured 366 -> 354 us (8 x 2048, 64/128); of 128 elements a key they leave one workgroup a CU: 138 -> 171 us
    constexpr int AR = TR * TR / 64, MAPS = KEEP ? 2 : 1, TURN = D <= 64 ? 2 : 1;
    typedef Stage<T, 256, KT, 2, D, FAST> StageK;
    typedef Stage<T, 256, KT, 1, DV, FAST> StageV;
    __shared__ __attribute__((aligned(16))) T k_tile[2][TURN * KT * StageK::PITCH];
    __shared__ __attribute__((aligned(16))) T v_tile[2][KT * StageV::PITCH];
    const Place<TR> at(a, row_tiles);
    const Source<T> qs{static_cast<const T *>(a.q) + at.b * a.qb + (int64_t)at.hk * a.G * a.qh, a.ql, a.qh, a.qm, a.G, a.d, a.inverse};
    const Source<T> ks{static_cast<const T *>(a.k) + at.b * a.kb + at.hk * a.kh, a.kl, 0, a.km, 1, a.d, 1.0f};
    const Source<T> vs{static_cast<const T *>(a.v) + at.b * a.vb + at.hk * a.vh, a.vl, 0, 0, 1, a.dv, 1.0f};
    Frag<T> q[2][D / KS<T, TR>];
#pragma unroll
    for (int m = 0; m < 2; ++m) load_rows<T, TR, D>(qs, at.row, at.there, m, q[m]);
    const float c = a.scale * LOG2E;
    // a key that nobody sees is zeros in LDS, whatever its memory holds
    const auto seen = [&](int key) { return !a.mask || a.mask[at.b * a.mask_b + key] != 0; };
    const int tiles = (at.end + KT - 1) / KT, mine = (at.wave_any + KT - 1) / KT, whole = FAST || !a.mask ? at.wave_all / KT : 0;
    const auto word_of = [&](int t) { return !FAST && a.mask ? mask_word(a, at.b, t * KT) : 0xffffffffu; };

    // first pass: maximum (powers of two) and sum of exponentials of each map, TURN tiles between two barriers
    float top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.0f, 0.0f};
    {
        Stage<T, 256, TURN * KT, 2, D, FAST> stage;
        stage.load(ks, 0, at.end, seen);
        stage.store(k_tile[0]);
        const auto turn = [&](int t, const auto &use) {
            if (t + TURN < tiles) stage.load(ks, (t + TURN) * KT, at.end, seen);
            __syncthreads();
            use(k_tile[t / TURN & 1]);
            if (t + TURN < tiles) stage.store(k_tile[(t / TURN + 1) & 1]);        // every wave is past that tile
        };
        const auto add = [&](Acc<TR> (&s)[2][BLOCKS<TR>]) {
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                float most = -INFINITY;
#pragma unroll
                for (int f = 0; f < REGS<TR>; ++f) most = fmaxf(most, s[m][f / AR][f % AR]);
                most = fmaxf(top[m], groups_max<TR>(most) * c);
                const float base = most == -INFINITY ? 0.0f : most;
                float part[2] = {sum[m] * __builtin_amdgcn_exp2f(top[m] - base), 0.0f};
#pragma unroll
                for (int f = 0; f < REGS<TR>; ++f) part[f & 1] += __builtin_amdgcn_exp2f(fmaf(s[m][f / AR][f % AR], c, -base));
                sum[m] = part[0] + part[1];
                top[m] = most;
            }
        };
        int t = 0;
        for (; t + TURN <= whole; t += TURN)
            turn(t, [&](const T *tile) {
#pragma unroll
                for (int n = 0; n < TURN; ++n) {
                    Acc<TR> s[2][BLOCKS<TR>];
                    scores_of<T, TR, D>(q, tile + n * KT * StageK::PITCH, StageK::PITCH, s);
                    add(s);
                }
            });
        for (; t < mine; t += TURN)
            turn(t, [&](const T *tile) {
                for (int n = 0; n < TURN && t + n < mine; ++n) {
                    Acc<TR> s[2][BLOCKS<TR>];
                    scores_of<T, TR, D>(q, tile + n * KT * StageK::PITCH, StageK::PITCH, s);
                    hide<!FAST, TR>(s, at.limit - (t + n) * KT, word_of(t + n));
                    add(s);
                }
            });
        for (; t < tiles; t += TURN) turn(t, [](const T *) {});
    }
    // base[m]: what the second pass subtracts, so that exp2(score - base) is g P1 and g2 P2; +inf where a row sees nothing
    float lse[2], base[2];
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        sum[m] = groups_sum<TR>(sum[m]);
        lse[m] = sum[m] > 0.0f ? top[m] + log2f(sum[m]) : INFINITY;
    }
    const float lam = lambda_of(a, at.head, static_cast<const T *>(nullptr));
    const float g2 = fminf(fmaxf(fmaxf(sum[0], sum[1]), 1.0f), 4096.0f), g = fminf(g2, 4096.0f / fmaxf(fabsf(lam), 1.0f));
    const float back = 1.0f / g, weight = lam * (g / g2);
    base[0] = lse[0] - log2f(g);
    base[1] = lse[1] - log2f(g2);

    // second pass
    Acc<TR> o[MAPS][DV / TR];
#pragma unroll
    for (int m = 0; m < MAPS; ++m)
#pragma unroll
        for (int blk = 0; blk < DV / TR; ++blk)
#pragma unroll
            for (int i = 0; i < AR; ++i) o[m][blk][i] = 0.0f;
    {
        StageK k_stage;
        StageV v_stage;
        k_stage.load(ks, 0, at.end, seen);
        v_stage.load(vs, 0, at.end, seen);
        __syncthreads();
        k_stage.store(k_tile[0]);
        v_stage.store(v_tile[0]);
        const auto turn = [&](int t, const auto &use) {
            if (t + 1 < tiles) {
                k_stage.load(ks, (t + 1) * KT, at.end, seen);
                v_stage.load(vs, (t + 1) * KT, at.end, seen);
            }
            __syncthreads();
            use(k_tile[t & 1], v_tile[t & 1]);
            if (t + 1 < tiles) {
                k_stage.store(k_tile[(t + 1) & 1]);
                v_stage.store(v_tile[(t + 1) & 1]);
            }
        };
        const auto add = [&](Acc<TR> (&s)[2][BLOCKS<TR>], const T *tile) {
            float p[MAPS][REGS<TR>];
            Frag<T> frag[MAPS][FRAGS<T, TR>];
#pragma unroll
            for (int f = 0; f < REGS<TR>; ++f) {
                const float p1 = __builtin_amdgcn_exp2f(fmaf(s[0][f / AR][f % AR], c, -base[0]));
                const float p2 = __builtin_amdgcn_exp2f(fmaf(s[1][f / AR][f % AR], c, -base[1]));
                p[0][f] = fmaf(-weight, p2, p1);
                if (KEEP) p[MAPS - 1][f] = p2;
            }
#pragma unroll
            for (int m = 0; m < MAPS; ++m) to_frags<T, TR>(p[m], frag[m]);
#pragma unroll
            for (int blk = 0; blk < DV / TR; ++blk)
#pragma unroll
                for (int j = 0; j < FRAGS<T, TR>; ++j) {
                    const Frag<T> v = column_frag<TR>(tile, StageV::PITCH, blk * TR, j);
#pragma unroll
                    for (int m = 0; m < MAPS; ++m) mma<TR>(v, frag[m][j], o[m][blk]);
                }
        };
        int t = 0;
        for (; t < whole; ++t)
            turn(t, [&](const T *k, const T *v) {
                Acc<TR> s[2][BLOCKS<TR>];
                scores_of<T, TR, D>(q, k, StageK::PITCH, s);
                add(s, v);
            });
        for (; t < mine; ++t)
            turn(t, [&](const T *k, const T *v) {
                Acc<TR> s[2][BLOCKS<TR>];
                scores_of<T, TR, D>(q, k, StageK::PITCH, s);
                hide<!FAST, TR>(s, at.limit - t * KT, word_of(t));
                add(s, v);
            });
        for (; t < tiles; ++t) turn(t, [](const T *, const T *) {});
    }
    if (!at.there) return;
    const int64_t place = (((int64_t)at.b * a.Lq + at.query) * a.H + at.head) * a.dv, plane = (int64_t)a.B * a.Lq * a.H * a.dv;
#pragma unroll
    for (int blk = 0; blk < DV / TR; ++blk)
#pragma unroll
        for (int f = 0; f < AR; f += 4) {
            const int col = blk * TR + (f / 4) * 4 * GROUPS<TR> + 4 * lane_group<TR>();
            if (col >= a.dv) continue;
            float r[4], o1[4], o2[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                r[u] = o[0][blk][f + u] * back;
                if (KEEP) {
                    o2[u] = o[MAPS - 1][blk][f + u] * (1.0f / g2);
                    o1[u] = fmaf(lam, o2[u], r[u]);
                }
            }
            store_pack<T, 4>(static_cast<T *>(out.out) + place + col, a.dv - col, r);
            if (KEEP) {
                store_pack<float, 4>(out.kept + place + col, a.dv - col, o2);
                store_pack<float, 4>(out.kept + plane + place + col, a.dv - col, o1);
            }
        }
    if (KEEP && lane_group<TR>() == 0) {
#pragma unroll
        for (int m = 0; m < 2; ++m) out.lse[(((int64_t)m * a.B + at.b) * a.H + at.head) * a.Lq + at.query] = lse[m];
    }
}

template <class T>
struct Forward {
    const Call &a;
    const ForwardOut &out;
    hipStream_t st;
    template <int D, int DV>
    int operator()() const
    {
        constexpr int TR = TILE_ROWS<T, D>;
        const int64_t row_tiles = ceil_div(a.R, 4 * TR), blocks = row_tiles * a.B * a.Hkv;
        if (blocks > INT32_MAX) return fail(MAM_ERR_UNSUPPORTED, "too many tiles");
        const dim3 grid((unsigned)blocks);
        if constexpr (sizeof(T) == 4) {
            if (a.fast) hipLaunchKernelGGL((tiles_kernel<T, TR, D, DV, true>), grid, dim3(256), 0, st, a, out, (int)row_tiles);
            else hipLaunchKernelGGL((tiles_kernel<T, TR, D, DV, false>), grid, dim3(256), 0, st, a, out, (int)row_tiles);
            return check_launch("attention::tiles_kernel");
        } else {
            if (out.kept && a.fast) hipLaunchKernelGGL((twice_kernel<T, TR, D, DV, true, true>), grid, dim3(256), 0, st, a, out, (int)row_tiles);
            else if (out.kept) hipLaunchKernelGGL((twice_kernel<T, TR, D, DV, false, true>), grid, dim3(256), 0, st, a, out, (int)row_tiles);
            else if (a.fast) hipLaunchKernelGGL((twice_kernel<T, TR, D, DV, true, false>), grid, dim3(256), 0, st, a, out, (int)row_tiles);
            else hipLaunchKernelGGL((twice_kernel<T, TR, D, DV, false, false>), grid, dim3(256), 0, st, a, out, (int)row_tiles);
            return check_launch("attention::twice_kernel");
        }
    }
};

int fill_call(const mam_diff_attention_t *a, Call &c)
{
    if (!a) return fail(MAM_ERR_INVALID_ARGUMENT, "null pointer");
    if (!is_type(a->type)) return fail(MAM_ERR_INVALID_ARGUMENT, "unknown element type %d", a->type);
    if (a->lam_type != a->type && a->lam_type != MAM_F32)
        return fail(MAM_ERR_INVALID_ARGUMENT, "lam is of the operands' type or fp32, got type %d", a->lam_type);
    if (a->B < 0 || a->Lq < 0 || a->Lk < 0 || a->H < 0 || a->Hkv < 0) return fail(MAM_ERR_INVALID_ARGUMENT, "negative size");
    if (a->H > 0 && (a->Hkv < 1 || a->H % a->Hkv)) return fail(MAM_ERR_INVALID_ARGUMENT, "the key heads must divide the query heads");
    if (!head_sizes_fit(a->D, a->Dv)) return fail(MAM_ERR_UNSUPPORTED, "head sizes are 1 to 128 (queries, keys) and 1 to 256 (values)");
    if (!((float)a->scale > 0.0f) || !(a->scale <= 1e30)) return fail(MAM_ERR_INVALID_ARGUMENT, "scale must be positive and finite");
    const int64_t most = INT32_MAX / 4;
    if (a->B > most || a->Lq > most || a->Lk > most || a->H > most || a->Lq * (a->H > 0 ? a->H : 1) > most)
        return fail(MAM_ERR_UNSUPPORTED, "a dimension exceeds 2^29");
    c.q = a->q; c.k = a->k; c.v = a->v; c.lam = a->lam;
    c.qb = a->q_stride[0]; c.ql = a->q_stride[1]; c.qh = a->q_stride[2]; c.qm = a->q_stride[3];
    c.kb = a->k_stride[0]; c.kl = a->k_stride[1]; c.kh = a->k_stride[2]; c.km = a->k_stride[3];
    c.vb = a->v_stride[0]; c.vl = a->v_stride[1]; c.vh = a->v_stride[2];
    c.lengths = a->lengths; c.starts = a->starts; c.mask = a->key_mask; c.mask_b = a->mask_stride;
    c.B = (int)a->B; c.Lq = (int)a->Lq; c.Lk = (int)a->Lk; c.H = (int)a->H; c.Hkv = (int)a->Hkv;
    c.G = a->Hkv ? (int)(a->H / a->Hkv) : 1;
    c.d = (int)a->D; c.dv = (int)a->Dv; c.causal = a->causal != 0; c.lam_same = a->lam_type == a->type;
    c.R = c.Hkv ? c.Lq * c.G : 0;
    c.scale = (float)a->scale;
    c.inverse = 1.0f / (float)(c.G ? c.G : 1);
    const int64_t size = type_size(a->type);
    c.fast = !c.mask && fast_operand(c.q, size, c.d, c.qb, c.ql, c.qh, c.qm, c.G) && fast_operand(c.k, size, c.d, c.kb, c.kl, c.kh, c.km, 1) &&
             fast_operand(c.v, size, c.dv, c.vb, c.vl, c.vh, 0, 1);
    return MAM_OK;
}

}  // namespace attention
}  // namespace mam

extern "C" int mam_diff_attention(const mam_diff_attention_t *args, void *out, float *kept, float *lse, void *workspace,
                                  size_t workspace_bytes, void *stream)
{
    using namespace mam;
    attention::Call a;
    const int rc = attention::fill_call(args, a);
    if (rc != MAM_OK || a.B == 0 || a.R == 0) return rc;
    if (!a.q || !a.lam || !out || (a.Lk > 0 && (!a.k || !a.v))) return fail(MAM_ERR_INVALID_ARGUMENT, "null pointer");
    if (!kept != !lse) return fail(MAM_ERR_INVALID_ARGUMENT, "kept and lse are wanted together");
    if (attention::use_split(a, args->type, kept != nullptr)) return attention::run_split(a, args->type, out, workspace, workspace_bytes, static_cast<hipStream_t>(stream));
    hipStream_t st = static_cast<hipStream_t>(stream);
    const attention::ForwardOut o{out, kept, lse};
    if (args->type == MAM_F32) return attention::with_head_sizes(a.d, a.dv, attention::Forward<float>{a, o, st});
    if (args->type == MAM_BF16) return attention::with_head_sizes(a.d, a.dv, attention::Forward<bf16>{a, o, st});
    return attention::with_head_sizes(a.d, a.dv, attention::Forward<f16>{a, o, st});
}

extern "C" size_t mam_diff_attention_workspace(const mam_diff_attention_t *args)
{
    using namespace mam;
    attention::Call a;
    if (attention::fill_call(args, a) != MAM_OK || a.B == 0 || a.R == 0) return 0;
    return attention::use_split(a, args->type, false) ? attention::split_workspace(a) : 0;
}
