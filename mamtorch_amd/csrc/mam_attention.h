// Shared parts of the differential attention kernels: operands, matrix-core tiles and the staging of rows in LDS.
//
// A query head's rows and the heads that share its keys are one axis of rows, r = query * group + head of the group, so a causal
// limit ascends with r and a few rows fill a tile where many heads share a key head.
//
// Products are formed "transposed": a wave owns TR rows as the COLUMNS of its accumulators (lane % TR), and a product's other index
// runs over the registers.  Scores come out as S^T (keys x rows), so a row's softmax is a lane's own registers plus one or two
// exchanges, and a probability is already where the next product wants it: in the accumulator of 32 x 32 (16 x 16) tiles, lane
// group h holds other-index 4 * groups * (f / 4) + 4 h + f % 4 in register f, and a contraction may take its terms in any order that both
// operands agree on.  So P^T goes from the accumulators into the second product's operand with no exchange at all; the operand
// beside it is read in that order: rows of LDS by the transposing read for 16-bit types, word by word for fp32.
#pragma once
#include "mam_types.h"

namespace mam {
namespace attention {

constexpr float LOG2E = 1.44269504088896340736f;

// The call's operands.  Strides in elements.
struct Call {
    const void *q, *k, *v, *lam;
    int64_t qb, ql, qh, qm, kb, kl, kh, km, vb, vl, vh;
    const int32_t *lengths, *starts;
    const unsigned char *mask;
    int64_t mask_b;
    int B, Lq, Lk, H, Hkv, G, d, dv, causal, lam_same;
    int R;              // rows of a key head: Lq * G
    float scale;
};

// What rows of batch b see: keys below `keys`, and with a causal limit those up to query + first.
struct Reach {
    int keys;
    int64_t first;      // key that query 0 sees last; beyond all keys where nothing limits
    __device__ __forceinline__ int of_query(int i) const
    {
        const int64_t e = first + i + 1;
        return e < 0 ? 0 : e < keys ? (int)e : keys;
    }
};

__device__ __forceinline__ Reach reach_of(const Call &a, int b)
{
    Reach r;
    r.keys = a.Lk;
    if (a.lengths) {
        const int n = a.lengths[b];
        r.keys = n < 0 ? 0 : n < a.Lk ? n : a.Lk;
    }
    r.first = a.causal ? (a.starts ? (int64_t)a.starts[b] : (int64_t)a.Lk - a.Lq) : (int64_t)a.Lk;
    return r;
}

__device__ __forceinline__ float lambda_of(const Call &a, int head, const float *) { return static_cast<const float *>(a.lam)[head]; }
template <class T>
__device__ __forceinline__ float lambda_of(const Call &a, int head, const T *)
{
    return a.lam_same ? (float)static_cast<const T *>(a.lam)[head] : static_cast<const float *>(a.lam)[head];
}

// ---- matrix-core tiles ----
template <class T>
constexpr int FE = 16 / (int)sizeof(T);     // elements of a fragment: 16 bytes a lane
template <class T>
struct FragOf { typedef T type __attribute__((ext_vector_type(16 / sizeof(T)))); };
template <class T>
using Frag = typename FragOf<T>::type;

template <int TR>
struct AccOf { typedef float type __attribute__((ext_vector_type(TR * TR / 64))); };
template <int TR>
using Acc = typename AccOf<TR>::type;
template <int TR>
constexpr int GROUPS = 64 / TR;             // lane groups, each with its own terms of a contraction
template <int TR>
constexpr int BLOCKS = 32 / TR;             // accumulators of 32 other-index values
template <int TR>
constexpr int REGS = TR / 2;                // registers of 32 x TR values
template <class T, int TR>
constexpr int KS = FE<T> * GROUPS<TR>;      // contraction length of a fragment pair
template <class T, int TR>
constexpr int FRAGS = REGS<TR> / FE<T>;     // fragments that 32 contraction terms fill

// acc += A B over KS terms
template <int TR>
__device__ __forceinline__ void mma(const Frag<bf16> &a, const Frag<bf16> &b, Acc<TR> &c)
{
    if constexpr (TR == 32) c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    else c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
template <int TR>
__device__ __forceinline__ void mma(const Frag<f16> &a, const Frag<f16> &b, Acc<TR> &c)
{
    if constexpr (TR == 32) c = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    else c = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
template <int TR>
__device__ __forceinline__ void mma(const Frag<float> &a, const Frag<float> &b, Acc<TR> &c)
{
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        if constexpr (TR == 32) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[u], b[u], c, 0, 0, 0);
        else c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[u], b[u], c, 0, 0, 0);
    }
}

template <int TR>
__device__ __forceinline__ int lane_row() { return (threadIdx.x & 63) % TR; }
template <int TR>
__device__ __forceinline__ int lane_group() { return (threadIdx.x & 63) / TR; }

// Other-index (0 .. 31) of register f of a lane's 32 x TR values.
template <int TR>
__device__ __forceinline__ int index_of(int f) { return (f / 4) * 4 * GROUPS<TR> + 4 * lane_group<TR>() + f % 4; }

// Fragment of a row of LDS: terms kk * KS .. of row `row`.
template <class T, int TR>
__device__ __forceinline__ Frag<T> row_frag(const T *tile, int pitch, int row, int kk)
{
    return *reinterpret_cast<const Frag<T> *>(tile + row * pitch + kk * KS<T, TR> + FE<T> * lane_group<TR>());
}

// Fragment j of the columns col .. col + TR - 1 of 32 rows of LDS, taken as the contraction's terms in the accumulators' order.
template <int TR, class T>
__device__ __forceinline__ Frag<T> column_frag(const T *tile, int pitch, int col, int j)
{
    const int lane = threadIdx.x & 63;
    if constexpr (sizeof(T) == 2) {
        // the transposing read: 16 lanes give the addresses of 4 rows x 16 columns and get a column's 4 rows each
        typedef short quad __attribute__((ext_vector_type(4)));
        typedef short octet __attribute__((ext_vector_type(8)));
        typedef __attribute__((address_space(3))) quad *lds_quad;
        const T *p = tile + (8 * GROUPS<TR> * j + 4 * lane_group<TR>() + (lane % 16) / 4) * pitch + col + 16 * ((lane % TR) / 16) + 4 * (lane % 4);
        const quad lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_quad)p);
        const quad hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_quad)(p + 4 * GROUPS<TR> * pitch));
        const octet all = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        return __builtin_bit_cast(Frag<T>, all);
    } else {
        const T *p = tile + (4 * GROUPS<TR> * j + 4 * lane_group<TR>()) * pitch + col + lane % TR;
        Frag<T> r;
#pragma unroll
        for (int u = 0; u < 4; ++u) r[u] = p[u * pitch];
        return r;
    }
}

// 32 x TR values as the fragments of a contraction over the 32.
template <class T, int TR>
__device__ __forceinline__ void to_frags(const float (&p)[REGS<TR>], Frag<T> (&f)[FRAGS<T, TR>])
{
#pragma unroll
    for (int j = 0; j < FRAGS<T, TR>; ++j)
#pragma unroll
        for (int u = 0; u < FE<T>; ++u) f[j][u] = (T)p[j * FE<T> + u];
}

// Maximum and sum over the lane groups that hold a row's values.
template <int TR>
__device__ __forceinline__ float groups_max(float v)
{
    v = fmaxf(v, __shfl_xor(v, 32));
    if constexpr (TR == 16) v = fmaxf(v, __shfl_xor(v, 16));
    return v;
}
template <int TR>
__device__ __forceinline__ float groups_sum(float v)
{
    v += __shfl_xor(v, 32);
    if constexpr (TR == 16) v += __shfl_xor(v, 16);
    return v;
}

// ---- operands in LDS ----
// Rows of `maps` segments of W elements, of which `width` are there, the rest being zeros in LDS.
template <class T>
struct Source {
    const T *base;
    int64_t row, head, map;     // strides; a row's head is its number modulo G
    int G, width;
    __device__ __forceinline__ const T *at(int r, int m) const
    {
        const int64_t off = G == 1 ? (int64_t)r * row : (int64_t)(r / G) * row + (int64_t)(r % G) * head;
        return base + off + (int64_t)m * map;
    }
};

template <class T>
__device__ __forceinline__ Frag<T> load_frag(const T *p, int left)
{
    typedef typename Pack<T, FE<T>>::type pack;
    Frag<T> r;
    if (left >= FE<T>) {
        const pack t = *reinterpret_cast<const pack *>(p);
#pragma unroll
        for (int u = 0; u < FE<T>; ++u) r[u] = t[u];
    } else {
#pragma unroll
        for (int u = 0; u < FE<T>; ++u) r[u] = u < left ? p[u] : (T)0.0f;
    }
    return r;
}

// ROWS rows of MAPS segments of W elements between global memory and LDS by THREADS threads, in 16-byte pieces that stay in
// registers between load() and store().
template <class T, int THREADS, int ROWS, int MAPS, int W>
struct Stage {
    static constexpr int PER = MAPS * W / FE<T>, PIECES = ROWS * PER, N = (PIECES + THREADS - 1) / THREADS;
    static constexpr int PITCH = MAPS * W + FE<T>;
    Frag<T> piece[N];

    // `there(row)`: whether a row is read or taken as zeros
    template <class There>
    __device__ __forceinline__ void load(const Source<T> &src, int first, const There &there)
    {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int id = i * THREADS + threadIdx.x, row = id / PER, col = id % PER * FE<T>, c = col % W;
            const bool ok = (PIECES % THREADS == 0 || id < PIECES) && c < src.width && there(first + row);
#pragma unroll
            for (int u = 0; u < FE<T>; ++u) piece[i][u] = (T)0.0f;
            if (ok) piece[i] = load_frag<T>(src.at(first + row, col / W) + c, src.width - c);
        }
    }
    __device__ __forceinline__ void store(T *tile) const
    {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int id = i * THREADS + threadIdx.x, row = id / PER, col = id % PER * FE<T>;
            if (PIECES % THREADS == 0 || id < PIECES) *reinterpret_cast<Frag<T> *>(tile + row * PITCH + col) = piece[i];
        }
    }
};

// A wave's own TR rows as the fragments of a contraction over their W elements.
template <class T, int TR, int W>
__device__ __forceinline__ void load_rows(const Source<T> &src, int row, bool there, int map, Frag<T> (&f)[W / KS<T, TR>])
{
    const T *p = src.at(there ? row : 0, map);
#pragma unroll
    for (int kk = 0; kk < W / KS<T, TR>; ++kk) {
        const int c = kk * KS<T, TR> + FE<T> * lane_group<TR>();
#pragma unroll
        for (int u = 0; u < FE<T>; ++u) f[kk][u] = (T)0.0f;
        if (there && c < src.width) f[kk] = load_frag<T>(p + c, src.width - c);
    }
}

// Which of keys first .. first + 31 the mask leaves, one bit each.
__device__ __forceinline__ uint32_t mask_word(const Call &a, int b, int first)
{
    const int key = first + (threadIdx.x & 31);
    return (uint32_t)__ballot(key < a.Lk && a.mask[b * a.mask_b + key] != 0);
}

// Head sizes that kernels are built for: the smallest of them that holds a call's runs it, on zeros past its own.
//   (32, 64), (64, 64), (64, 128), (128, 128), (128, 256)
inline bool head_sizes_fit(int64_t d, int64_t dv) { return d >= 1 && dv >= 1 && d <= 128 && dv <= 256; }

template <class F>
int with_head_sizes(int d, int dv, const F &f)
{
    if (d <= 32 && dv <= 64) return f.template operator()<32, 64>();
    if (d <= 64 && dv <= 64) return f.template operator()<64, 64>();
    if (d <= 64 && dv <= 128) return f.template operator()<64, 128>();
    if (dv <= 128) return f.template operator()<128, 128>();
    return f.template operator()<128, 256>();
}

// Rows of a wave's tile.
template <int D, int DV>
constexpr int TILE_ROWS = D > 64 ? 16 : 32;

int fill_call(const mam_diff_attention_t *a, Call &c);

}  // namespace attention
}  // namespace mam
