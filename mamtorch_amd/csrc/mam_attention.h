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
    float scale, inverse;
    bool fast;          // k and v may be read by Stage<..., FAST>, and q too; no mask
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

// The tile that a workgroup takes: workgroups of one turn are those of all (request, key head) pairs, which follow each other on the XCDs, so that where there are a
// multiple of 8 of them a head's workgroups meet in one L2.  A causal call's tiles differ in length, from the last rows (the first keys) on;
// the longest begin first.  Where the device holds all workgroups at once, two a CU, the second half takes the shortest first, so that a CU has a long and a short one.
__device__ __forceinline__ int tile_of_turn(int turn, int tiles, bool last_first, int workgroups)
{
    const int half = (tiles + 1) / 2;
    const int order = workgroups <= 2 * kNumCU && turn >= half ? tiles - 1 - (turn - half) : turn;
    return last_first ? tiles - 1 - order : order;
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

// Where 16 values of a contraction are whole fragments (fp32) a last tile of 16 keys or rows or less is half a tile's work: 197 keys are 13 of 14 halves.
template <class T, int TR>
constexpr bool HALVES = BLOCKS<TR> == 2 && FRAGS<T, TR> % 2 == 0;

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
    static_assert(TR == 16, "fp32 tiles are of 16 rows (TILE_ROWS)");
#pragma unroll
    for (int u = 0; u < 4; ++u) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[u], b[u], c, 0, 0, 0);
}

template <int TR>
__device__ __forceinline__ int lane_row() { return (threadIdx.x & 63) % TR; }
template <int TR>
__device__ __forceinline__ int lane_group() { return (threadIdx.x & 63) / TR; }

// Other-index (0 .. 31) of register f of a lane's 32 x TR values.
template <int TR>
__device__ __forceinline__ int index_of(int f) { return (f / 4) * 4 * GROUPS<TR> + 4 * lane_group<TR>() + f % 4; }

// Where row `row` of a tile stands in LDS.  A pitch is 4 words more than a multiple of 32, so rows that follow each other are 4 banks apart: right for
// the 16-byte reads of 16 rows.  The transposing read takes 4 rows of 16 words at a time: 4 consecutive ones stand 4 rows, 16 banks, apart.  fp32 columns
// are read a row a lane group and have their rows in order.  Counted: no conflicts in 16-bit types; in fp32, where the 16-byte reads of four lane groups meet,
// 19 to 27 % of the LDS's cycles, which are a fifth of the kernels'.
template <class T>
__device__ __forceinline__ int place_of(int row)
{
    return sizeof(T) == 2 ? (row & ~15) | (row & 3) << 2 | (row >> 2 & 3) : row;
}

// Fragment of a row of LDS: terms kk * KS .. of row `row`.
template <class T, int TR>
__device__ __forceinline__ Frag<T> row_frag(const T *tile, int pitch, int row, int kk)
{
    return *reinterpret_cast<const Frag<T> *>(tile + place_of<T>(row) * pitch + kk * KS<T, TR> + FE<T> * lane_group<TR>());
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
        const T *p = tile + place_of<T>(8 * GROUPS<TR> * j + 4 * lane_group<TR>() + (lane % 16) / 4) * pitch + col + 16 * ((lane % TR) / 16) + 4 * (lane % 4);
        const quad lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_quad)p);
        // 4 * GROUPS rows on: 8 rows (two lane groups of 4) stand 2 rows on, 16 stand 16 rows on
        const quad hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_quad)(p + (TR == 32 ? 2 : 16) * pitch));
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
__device__ __forceinline__ void to_frags(const float (&p)[REGS<TR>], Frag<T> (&f)[FRAGS<T, TR>], int count = FRAGS<T, TR>)
{
#pragma unroll
    for (int j = 0; j < count; ++j)
#pragma unroll
        for (int u = 0; u < FE<T>; ++u) f[j][u] = (T)p[j * FE<T> + u];
}

// Has elements u and u + 1 of a fragment made here and not where they are used, behind a later branch.
template <class F>
__device__ __forceinline__ void keep_here(F &f, int u)
{
    constexpr int SIZE = sizeof(f[0]);
    typedef uint32_t words __attribute__((ext_vector_type(4)));
    words w = __builtin_bit_cast(words, f);
#pragma unroll
    for (int i = u * SIZE / 4; i < (u + 2) * SIZE / 4; ++i) {
        uint32_t t = w[i];
        asm volatile("" : "+v"(t));
        w[i] = t;
    }
    f = __builtin_bit_cast(F, w);
}

// Element u of a fragment in fp32, from the words that hold it.
__device__ __forceinline__ float element(const Frag<bf16> &f, int u)
{
    typedef uint32_t words __attribute__((ext_vector_type(4)));
    const words w = __builtin_bit_cast(words, f);
    return __uint_as_float(u & 1 ? w[u / 2] & 0xffff0000u : w[u / 2] << 16);
}
__device__ __forceinline__ float element(const Frag<f16> &f, int u) { return (float)f[u]; }
__device__ __forceinline__ float element(const Frag<float> &f, int u) { return f[u]; }

// Maximum and sum over the lane groups that hold a row's values: the halves (quarters) of a wave meet by vector instructions that
// swap them, not through LDS.  Of a value swapped with itself the two results are one half's and the other's.
typedef uint32_t Halves __attribute__((ext_vector_type(2)));
__device__ __forceinline__ Halves halves(float v)
{
    return __builtin_bit_cast(Halves, __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false));
}
__device__ __forceinline__ Halves quarters(float v)
{
    return __builtin_bit_cast(Halves, __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false));
}
template <int TR>
__device__ __forceinline__ float groups_max(float v)
{
    Halves t = halves(v);
    v = fmaxf(__uint_as_float(t[0]), __uint_as_float(t[1]));
    if constexpr (TR == 16) {
        t = quarters(v);
        v = fmaxf(__uint_as_float(t[0]), __uint_as_float(t[1]));
    }
    return v;
}
template <int TR>
__device__ __forceinline__ float groups_sum(float v)
{
    Halves t = halves(v);
    v = __uint_as_float(t[0]) + __uint_as_float(t[1]);
    if constexpr (TR == 16) {
        t = quarters(v);
        v = __uint_as_float(t[0]) + __uint_as_float(t[1]);
    }
    return v;
}

// ---- operands in LDS ----
// Rows of `maps` segments of W elements, of which `width` are there, the rest being zeros in LDS.
template <class T>
struct Source {
    const T *base;
    int64_t row, head, map;     // strides; a row's head is its number modulo G
    int G, width;
    float inverse;              // 1 / G
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

// 16 bytes at a 32-bit offset from a uniform base; an offset of NOWHERE reads nothing and gives zeros (the buffer's own bounds check).
constexpr uint32_t NOWHERE = 0x80000000u;
template <class T>
__device__ __forceinline__ Frag<T> buffer_frag(const T *base, uint32_t offset)
{
    typedef uint32_t words __attribute__((ext_vector_type(4)));
    const auto rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<T *>(base), 0, 0x7fffffff, 0x00027000);
    const words w = __builtin_amdgcn_raw_buffer_load_b128(rsrc, (int)offset, 0, 0);
    return __builtin_bit_cast(Frag<T>, w);
}

// ROWS rows of MAPS segments of W elements between global memory and LDS by THREADS threads, in 16-byte pieces that stay in
// registers between load() and store().  FAST: widths are whole pieces, addresses and strides multiples of 16 bytes, a tile's rows
// within 2^30 bytes and all rows below an end are there, so that a piece is one buffer load whatever of it is there; else element by element
// where a row ends inside a piece, and rows that are there by a test of each.
template <class T, int THREADS, int ROWS, int MAPS, int W, bool FAST>
struct Stage {
    static constexpr int PER = W / FE<T>, SEGMENT = ROWS * PER, PIECES = MAPS * SEGMENT, N = PIECES / THREADS;
    static constexpr int PITCH = MAPS * W + FE<T>;
    static_assert(PIECES % THREADS == 0 && SEGMENT % 64 == 0, "whole pieces a thread, a segment a wave");
    Frag<T> piece[N];

    static __device__ __forceinline__ uint32_t map_of(int i)
    {
        return MAPS == 1 ? 0 : (i * THREADS + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * 64u) / SEGMENT;
    }
    static __device__ __forceinline__ int row_of(int i) { return (int)((i * THREADS + threadIdx.x) % SEGMENT / PER); }
    static __device__ __forceinline__ int column_of(int i) { return (int)((i * THREADS + threadIdx.x) % SEGMENT % PER * FE<T>); }

    // Rows first .. of the source; those from `end` on, and those that `there` denies (slow loads only), are zeros.
    template <class There>
    __device__ __forceinline__ void load(const Source<T> &src, int first, int end, const There &there)
    {
        if constexpr (FAST) {
            const int left = end - first;
            if (src.G == 1) {
                const T *base = src.base + (int64_t)first * src.row;
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const uint32_t off = ((uint32_t)row_of(i) * (uint32_t)src.row + (uint32_t)column_of(i)) * (uint32_t)sizeof(T);
                    piece[i] = buffer_frag<T>(base + map_of(i) * src.map, row_of(i) < left && column_of(i) < src.width ? off : NOWHERE);
                }
            } else {            // heads of a shared key head: rows of a token are its heads
                const int token = first / src.G, turn = first - token * src.G;
                const T *base = src.base + (int64_t)token * src.row;
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const int t = turn + row_of(i), more = (int)(((float)t + 0.5f) * src.inverse);
                    const uint32_t off = (uint32_t)more * (uint32_t)src.row + (uint32_t)(t - more * src.G) * (uint32_t)src.head + (uint32_t)column_of(i);
                    piece[i] = buffer_frag<T>(base + map_of(i) * src.map,
                                              row_of(i) < left && column_of(i) < src.width ? off * (uint32_t)sizeof(T) : NOWHERE);
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int row = first + row_of(i), c = column_of(i);
#pragma unroll
                for (int u = 0; u < FE<T>; ++u) piece[i][u] = (T)0.0f;
                if (row < end && c < src.width && there(row)) piece[i] = load_frag<T>(src.at(row, map_of(i)) + c, src.width - c);
            }
        }
    }
    __device__ __forceinline__ void clear()
    {
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int u = 0; u < FE<T>; ++u) piece[i][u] = (T)0.0f;
    }
    __device__ __forceinline__ void store(T *tile) const
    {
#pragma unroll
        for (int i = 0; i < N; ++i) *reinterpret_cast<Frag<T> *>(tile + place_of<T>(row_of(i)) * PITCH + map_of(i) * W + column_of(i)) = piece[i];
    }
};

constexpr int KT = 32;          // rows of a tile in LDS

// Tiles in LDS: two where two workgroups still fit a CU, so that a tile is written while the last one is read.
template <class T, int D, int DV>
constexpr int TILES = 2 * KT * (2 * D + DV + 2 * FE<T>) * (int)sizeof(T) + 2 * 5 * KT * 4 <= 80 * 1024 ? 2 : 1;

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

// What a workgroup of four waves with TR rows each knows of its rows and of the keys that they see.
template <int TR>
struct Place {
    int b, hk, wave, row, query, head, limit, wave_all, wave_any, end;
    bool there;

    __device__ __forceinline__ Place(const Call &a, int row_tiles)
    {
        const int heads = a.B * a.Hkv, bh = blockIdx.x % heads, tile = tile_of_turn(blockIdx.x / heads, row_tiles, true, gridDim.x);
        b = bh / a.Hkv;
        hk = bh % a.Hkv;
        const Reach reach = reach_of(a, b);
        wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const int first = tile * 4 * TR + wave * TR;
        row = first + lane_row<TR>();
        there = row < a.R;
        query = there ? row / a.G : 0;
        head = hk * a.G + (there ? row - query * a.G : 0);
        limit = there ? reach.of_query(query) : 0;
        // the keys that every row of the wave sees, and that some row of it and of the workgroup sees
        const int wave_last = first + TR - 1 < a.R ? first + TR - 1 : a.R - 1;
        wave_all = first < a.R ? reach.of_query(first / a.G) : 0;
        wave_any = first < a.R ? reach.of_query(wave_last / a.G) : 0;
        const int last = tile * 4 * TR + 4 * TR - 1 < a.R ? tile * 4 * TR + 4 * TR - 1 : a.R - 1;
        end = reach.of_query(last / a.G);
    }
};

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

// Rows of a wave's tile.  fp32 products take 8 times as long for the bytes that they read of LDS, so tiles of 16 rows keep the matrix cores as busy
// and take half the registers; in 16-bit types 32 rows halve the reads, while the accumulators fit two waves a SIMD.
template <class T, int D>
constexpr int TILE_ROWS = sizeof(T) == 4 || D > 64 ? 16 : 32;

// Whether every operand can be read in whole 16-byte pieces at 32-bit offsets from its tiles (Stage).
inline bool fast_operand(const void *p, int64_t size, int width, int64_t batch, int64_t row, int64_t head, int64_t map, int64_t heads)
{
    const int64_t pack = 16 / size;
    return (uintptr_t)p % 16 == 0 && width % pack == 0 && batch % pack == 0 && row % pack == 0 && head % pack == 0 && map % pack == 0 && row >= 0 &&
           head >= 0 && map >= 0 && row <= (int64_t)1 << 22 && head * heads <= (int64_t)1 << 26;
}

// Planes of fp32 that the backward reads of the forward's products: the second map's, from which and the result the first's follows in fp32; in
// 16-bit types the first's too, since the result's rounding would enter every score gradient of its row.
template <class T>
constexpr int KEPT = sizeof(T) == 2 ? 2 : 1;

int fill_call(const mam_diff_attention_t *a, Call &c);

// Few queries over many keys (mam_attention_split.hip): whether a call runs there, its workspace, and the call.
bool use_split(const Call &a, int type, bool keep);
size_t split_workspace(const Call &a);
int run_split(const Call &a, int type, void *out, void *workspace, size_t workspace_bytes, hipStream_t st);

}  // namespace attention
}  // namespace mam
