// Element types of the encoder operators (fp32, bf16, fp16) and rows of them read and written in 16-byte pieces.
#pragma once
#include "mam_common.h"

namespace mam {

typedef __bf16 bf16;
typedef _Float16 f16;

inline bool is_type(int t) { return t == MAM_F32 || t == MAM_BF16 || t == MAM_F16; }
inline int64_t type_size(int t) { return t == MAM_F32 ? 4 : 2; }

// N elements of T as one load or store of at least T's own alignment: rows of odd lengths and offsets take the same path.
template <class T, int N>
struct Pack { typedef T type __attribute__((ext_vector_type(N), aligned(sizeof(T)))); };
template <class T>
constexpr int kPack = 16 / (int)sizeof(T);      // elements of a 16-byte piece

// Elements 0 .. N-1 of p in fp32, those from `left` on as 0 (and not read).
template <class T, int N = kPack<T>>
__device__ __forceinline__ void load_pack(const T *p, int left, float (&v)[N])
{
    if (left >= N) {
        const typename Pack<T, N>::type t = *reinterpret_cast<const typename Pack<T, N>::type *>(p);
#pragma unroll
        for (int u = 0; u < N; ++u) v[u] = (float)t[u];
    } else {
#pragma unroll
        for (int u = 0; u < N; ++u) v[u] = u < left ? (float)p[u] : 0.0f;
    }
}

template <class T, int N = kPack<T>>
__device__ __forceinline__ void store_pack(T *p, int left, const float (&v)[N])
{
    if (left >= N) {
        typename Pack<T, N>::type t;
#pragma unroll
        for (int u = 0; u < N; ++u) t[u] = (T)v[u];
        *reinterpret_cast<typename Pack<T, N>::type *>(p) = t;
    } else {
#pragma unroll
        for (int u = 0; u < N; ++u)
            if (u < left) p[u] = (T)v[u];
    }
}

// A piece as it is, to be loaded before it is used: half the registers of its elements in fp32.
template <class T>
using Raw = typename Pack<T, kPack<T>>::type;
template <class T>
__device__ __forceinline__ Raw<T> load_raw(const T *p, int left)
{
    if (left >= kPack<T>) return *reinterpret_cast<const Raw<T> *>(p);
    Raw<T> t;
#pragma unroll
    for (int u = 0; u < kPack<T>; ++u) t[u] = u < left ? p[u] : (T)0.0f;
    return t;
}

// The same of a vector whose type is known at run time only: `same` says that it is T, else fp32.
template <class T, int N = kPack<T>>
__device__ __forceinline__ void load_pack_of(const void *p, bool same, int64_t at, int left, float (&v)[N])
{
    if (same)
        load_pack<T, N>(static_cast<const T *>(p) + at, left, v);
    else
        load_pack<float, N>(static_cast<const float *>(p) + at, left, v);
}

}  // namespace mam
