// Dropout whose mask is never stored (mam_counter.h): y = keep ? x * scale : 0, plus a residual where there is one.  Its gradient
// is the same call on the incoming gradient.
//
// Reads and writes each element once; beside the memory the bound is the generator, 20 32 x 32 -> 64 bit products for 4 elements on
// the vector units.  Measured: 12608 x 3072 bf16 32 us, 4.8 TB/s, where a large copy reaches 5.2; 256 x 4096 fp32 3.5 us, mostly the launch.  The
// generator's rounds as a loop (a quarter of the code) are no better: 31.7 and 4.0 us.
#include "mam_counter.h"
#include "mam_types.h"

namespace mam {
namespace dropout {

constexpr int UNROLL = 2;      // 16-byte pieces of a thread, loaded before the first is used

// A workgroup takes 256 * UNROLL pieces that follow each other; their number of groups is a power of two, so that the low word of a
// group's number does not wrap within the workgroup and the high word is uniform.
template <class T, bool RESIDUAL>
__global__ __launch_bounds__(256) void dropout_kernel(const T *__restrict__ x, const T *__restrict__ residual, T *__restrict__ y,
                                                      int64_t n, const Dropout d)
{
    constexpr int N = kPack<T>;
    const int64_t first = (int64_t)blockIdx.x * (256 * UNROLL * N);
    const uint64_t offset = dropout_offset(d);
    const uint32_t group_low = (uint32_t)((uint64_t)first >> 2), group_high = (uint32_t)((uint64_t)first >> 34);
    const int left_all = n - first < 256 * UNROLL * N ? (int)(n - first) : 256 * UNROLL * N;
    float v[UNROLL][N], r[UNROLL][N];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
        const int at = (u * 256 + threadIdx.x) * N;
        load_pack<T>(x + first + at, left_all - at, v[u]);
        if (RESIDUAL) load_pack<T>(residual + first + at, left_all - at, r[u]);
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
        const int at = (u * 256 + threadIdx.x) * N;
        if (at >= left_all) continue;
#pragma unroll
        for (int q = 0; q < N / 4; ++q) {
            uint32_t w[4];
            random_words(group_low + (uint32_t)(at / 4 + q), group_high, offset, d.seed, w);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const bool keep = w[e] >= d.least && !d.none;
                const float kept = keep ? v[u][4 * q + e] * d.scale : 0.0f;
                v[u][4 * q + e] = RESIDUAL ? r[u][4 * q + e] + kept : kept;
            }
        }
        store_pack<T>(y + first + at, left_all - at, v[u]);
    }
}

template <class T>
int launch(const void *x, const void *residual, void *y, int64_t n, const Dropout &d, hipStream_t st)
{
    const int64_t blocks = ceil_div(n, 256 * UNROLL * kPack<T>);
    if (blocks > INT32_MAX) return fail(MAM_ERR_UNSUPPORTED, "too many elements");
    if (residual)
        hipLaunchKernelGGL((dropout_kernel<T, true>), dim3((unsigned)blocks), dim3(256), 0, st, static_cast<const T *>(x),
                           static_cast<const T *>(residual), static_cast<T *>(y), n, d);
    else
        hipLaunchKernelGGL((dropout_kernel<T, false>), dim3((unsigned)blocks), dim3(256), 0, st, static_cast<const T *>(x),
                           static_cast<const T *>(nullptr), static_cast<T *>(y), n, d);
    return check_launch("dropout_kernel");
}

}  // namespace dropout
}  // namespace mam

extern "C" int mam_dropout(const void *x, const void *residual, void *y, int64_t n, int type, const mam_dropout_t *drop, void *stream)
{
    using namespace mam;
    if (n < 0) return fail(MAM_ERR_INVALID_ARGUMENT, "negative size");
    if (!is_type(type)) return fail(MAM_ERR_INVALID_ARGUMENT, "unknown element type %d", type);
    Dropout d;
    const int rc = make_dropout(drop, d);
    if (rc != MAM_OK || n == 0) return rc;
    if (!x || !y) return fail(MAM_ERR_INVALID_ARGUMENT, "null pointer");
    hipStream_t st = static_cast<hipStream_t>(stream);
    return type == MAM_F32 ? dropout::launch<float>(x, residual, y, n, d, st)
           : type == MAM_BF16 ? dropout::launch<bf16>(x, residual, y, n, d, st)
                              : dropout::launch<f16>(x, residual, y, n, d, st);
}
