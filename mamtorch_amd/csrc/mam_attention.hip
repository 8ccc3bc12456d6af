// Differential attention, forward: out = softmax(scale Q1 K1^T) V - lambda softmax(scale Q2 K2^T) V for each head, with a
// running maximum and sum for each of the two softmaxes and each row, so that no score leaves the registers.
//
// tiles: a workgroup of four waves shares tiles of 32 keys in LDS, each wave with TR rows of its own (16 or 32, mam_attention.h).
// The next tile's loads are in flight while this one is used.  Bound by the matrix cores and, in 16-bit types, as much by the exponentials:
// two for each (query, key), 16 cycles of a wave for 64 of them.
#include "mam_attention.h"

namespace mam {
namespace attention {

constexpr int KT = 32;          // keys of a tile

// A new maximum moves the accumulators only where it is more than this (in powers of two) above the last one: what is left in the exponent
// is exact in fp32 either way, and 2^8 is within every type's range.
constexpr float SLACK = 8.0f;

struct ForwardOut {
    void *out, *out2;           // (B, Lq, H, dv) contiguous; out2: the second map's, or NULL
    float *lse;                 // (2, B, H, Lq): log2 of the sums of exponentials, or NULL
};

// A wave's running state of TR rows.
template <class T, int TR, int D, int DV>
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
    __device__ __forceinline__ void softmax(int m, const Acc<TR> (&s)[BLOCKS<TR>], float c, bool limited, int limit, uint32_t word,
                                            float (&p)[REGS<TR>])
    {
        float most = -INFINITY;
#pragma unroll
        for (int f = 0; f < REGS<TR>; ++f) {
            float v = s[f / (TR * TR / 64)][f % (TR * TR / 64)];
            if (limited) {
                const int key = index_of<TR>(f);
                v = key < limit && (word >> key & 1) ? v : -INFINITY;
            }
            p[f] = v;
            most = fmaxf(most, v);
        }
        most = groups_max<TR>(most) * c;
        if (__any(most > top[m] + SLACK)) {
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
        for (int f = 0; f < REGS<TR>; ++f) {
            p[f] = __builtin_amdgcn_exp2f(fmaf(p[f], c, -base));
            add += p[f];
        }
        sum[m] += add;
    }

    // 32 keys: their scores, probabilities, and the products with their values.
    __device__ __forceinline__ void keys(const Frag<T> (&q)[2][D / KS<T, TR>], const T *k_tile, int k_pitch, const T *v_tile, int v_pitch,
                                         float c, bool limited, int limit, uint32_t word)
    {
        Frag<T> frag[2][FRAGS<T, TR>];
        Acc<TR> s[2][BLOCKS<TR>];
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int b = 0; b < BLOCKS<TR>; ++b) {
#pragma unroll
                for (int i = 0; i < TR * TR / 64; ++i) s[m][b][i] = 0.0f;
#pragma unroll
                for (int kk = 0; kk < D / KS<T, TR>; ++kk)
                    mma<TR>(row_frag<T, TR>(k_tile + m * D, k_pitch, b * TR + lane_row<TR>(), kk), q[m][kk], s[m][b]);
            }
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            float p[REGS<TR>];
            softmax(m, s[m], c, limited, limit, word, p);
            to_frags<T, TR>(p, frag[m]);
        }
#pragma unroll
        for (int b = 0; b < DV / TR; ++b)
#pragma unroll
            for (int j = 0; j < FRAGS<T, TR>; ++j) {
                const Frag<T> v = column_frag<TR>(v_tile, v_pitch, b * TR, j);
                mma<TR>(v, frag[0][j], o[0][b]);
                mma<TR>(v, frag[1][j], o[1][b]);
            }
    }
};

// Four elements of a row's result at column c.
template <class T>
__device__ __forceinline__ void store_quad(T *p, int left, float v0, float v1, float v2, float v3)
{
    const float v[4] = {v0, v1, v2, v3};
    store_pack<T, 4>(p, left, v);
}

// Waves of a SIMD that the registers are shared between: accumulators and queries take DV * TR / 32 and D * TR * size / 128 of a lane's.
template <class T, int TR, int D, int DV>
constexpr int WAVES = DV * TR / 32 + D * TR * (int)sizeof(T) / 128 <= 128 ? 2 : 1;

template <class T, int TR, int D, int DV>
__global__ __launch_bounds__(256, (WAVES<T, TR, D, DV>)) void tiles_kernel(const Call a, const ForwardOut out, int row_tiles)
{
    constexpr int ROWS = 4 * TR;
    typedef Stage<T, 256, KT, 2, D> StageK;
    typedef Stage<T, 256, KT, 1, DV> StageV;
    __shared__ __attribute__((aligned(16))) T k_tile[KT * StageK::PITCH];
    __shared__ __attribute__((aligned(16))) T v_tile[KT * StageV::PITCH];
    // tiles of rows that share keys run on one XCD; the last rows, which see the most keys of a causal call, begin first
    const int id = xcd_remap(blockIdx.x, gridDim.x);
    const int bh = id / row_tiles, tile = row_tiles - 1 - id % row_tiles;
    const int b = bh / a.Hkv, hk = bh % a.Hkv;
    const Reach reach = reach_of(a, b);
    const int wave = threadIdx.x >> 6;
    const int first = tile * ROWS + wave * TR, row = first + lane_row<TR>();
    const bool there = row < a.R;
    const int query = there ? row / a.G : 0, head = hk * a.G + (there ? row - query * a.G : 0);
    const int limit = there ? reach.of_query(query) : 0;
    // the keys that every row of the wave sees, and that some row of it and of the workgroup sees
    const int wave_last = first + TR - 1 < a.R ? first + TR - 1 : a.R - 1;
    const int wave_all = first < a.R ? reach.of_query(first / a.G) : 0, wave_any = first < a.R ? reach.of_query(wave_last / a.G) : 0;
    const int last = tile * ROWS + ROWS - 1 < a.R ? tile * ROWS + ROWS - 1 : a.R - 1;
    const int end = reach.of_query(last / a.G);

    const Source<T> qs{static_cast<const T *>(a.q) + b * a.qb + (int64_t)hk * a.G * a.qh, a.ql, a.qh, a.qm, a.G, a.d};
    const Source<T> ks{static_cast<const T *>(a.k) + b * a.kb + hk * a.kh, a.kl, 0, a.km, 1, a.d};
    const Source<T> vs{static_cast<const T *>(a.v) + b * a.vb + hk * a.vh, a.vl, 0, 0, 1, a.dv};
    Frag<T> q[2][D / KS<T, TR>];
#pragma unroll
    for (int m = 0; m < 2; ++m) load_rows<T, TR, D>(qs, row, there, m, q[m]);
    const float c = a.scale * LOG2E;

    State<T, TR, D, DV> state;
    state.clear();
    // a key that nobody sees is zeros in LDS, whatever its memory holds
    const auto seen = [&](int key) { return key < end && (!a.mask || a.mask[b * a.mask_b + key] != 0); };
    StageK k_stage;
    StageV v_stage;
    k_stage.load(ks, 0, seen);
    v_stage.load(vs, 0, seen);
    for (int key = 0; key < end; key += KT) {
        __syncthreads();
        k_stage.store(k_tile);
        v_stage.store(v_tile);
        __syncthreads();
        if (key + KT < end) {
            k_stage.load(ks, key + KT, seen);
            v_stage.load(vs, key + KT, seen);
        }
        if (key >= wave_any) continue;
        const bool limited = key + KT > wave_all || a.mask;
        const uint32_t word = a.mask ? mask_word(a, b, key) : 0xffffffffu;
        state.keys(q, k_tile, StageK::PITCH, v_tile, StageV::PITCH, c, limited, limit - key, word);
    }
    if (!there) return;
    const float lam = lambda_of(a, head, static_cast<const T *>(nullptr));
    float inv[2], total[2];
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        total[m] = groups_sum<TR>(state.sum[m]);
        inv[m] = total[m] > 0.0f ? 1.0f / total[m] : 0.0f;         // a row that sees nothing is zeros
    }
    const int64_t at = (((int64_t)b * a.Lq + query) * a.H + head) * a.dv;
#pragma unroll
    for (int blk = 0; blk < DV / TR; ++blk)
#pragma unroll
        for (int f = 0; f < TR * TR / 64; f += 4) {
            const int col = blk * TR + (f / 4) * 4 * GROUPS<TR> + 4 * lane_group<TR>();
            if (col >= a.dv) continue;
            float o1[4], o2[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                o2[u] = state.o[1][blk][f + u] * inv[1];
                o1[u] = fmaf(-lam, o2[u], state.o[0][blk][f + u] * inv[0]);
            }
            store_pack<T, 4>(static_cast<T *>(out.out) + at + col, a.dv - col, o1);
            if (out.out2) store_pack<T, 4>(static_cast<T *>(out.out2) + at + col, a.dv - col, o2);
        }
    if (out.lse && lane_group<TR>() == 0) {
#pragma unroll
        for (int m = 0; m < 2; ++m)
            out.lse[(((int64_t)m * a.B + b) * a.H + head) * a.Lq + query] = total[m] > 0.0f ? state.top[m] + log2f(total[m]) : INFINITY;
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
        constexpr int TR = TILE_ROWS<D, DV>;
        const int64_t row_tiles = ceil_div(a.R, 4 * TR), blocks = row_tiles * a.B * a.Hkv;
        if (blocks > INT32_MAX) return fail(MAM_ERR_UNSUPPORTED, "too many tiles");
        hipLaunchKernelGGL((tiles_kernel<T, TR, D, DV>), dim3((unsigned)blocks), dim3(256), 0, st, a, out, (int)row_tiles);
        return check_launch("attention::tiles_kernel");
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
    if (!(a->scale > 0.0) || !(a->scale <= 1e30)) return fail(MAM_ERR_INVALID_ARGUMENT, "scale must be positive and finite");
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
    return MAM_OK;
}

}  // namespace attention
}  // namespace mam

extern "C" int mam_diff_attention(const mam_diff_attention_t *args, void *out, void *out2, float *lse, void *workspace,
                                  size_t workspace_bytes, void *stream)
{
    using namespace mam;
    attention::Call a;
    const int rc = attention::fill_call(args, a);
    if (rc != MAM_OK || a.B == 0 || a.R == 0) return rc;
    if (!a.q || !a.lam || !out || (a.Lk > 0 && (!a.k || !a.v))) return fail(MAM_ERR_INVALID_ARGUMENT, "null pointer");
    hipStream_t st = static_cast<hipStream_t>(stream);
    const attention::ForwardOut o{out, out2, lse};
    if (args->type == MAM_F32) return attention::with_head_sizes(a.d, a.dv, attention::Forward<float>{a, o, st});
    if (args->type == MAM_BF16) return attention::with_head_sizes(a.d, a.dv, attention::Forward<bf16>{a, o, st});
    return attention::with_head_sizes(a.d, a.dv, attention::Forward<f16>{a, o, st});
}

extern "C" size_t mam_diff_attention_workspace(const mam_diff_attention_t *) { return 0; }
