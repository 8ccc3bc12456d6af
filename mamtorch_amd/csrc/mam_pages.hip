// The pages of a cache: room for new tokens, forks, release, copies and compaction, and what drafted tokens see of each other.
//
// The bookkeeping is on the device, so that a step of a server that drafts, appends, attends and takes over is enqueued, or captured, as a whole: which pages a
// request holds (table), how many requests hold a page (refs; a free page has 0), how many tokens a request has (lengths).  All of it is whole numbers, and every sum
// and choice has a fixed result whatever order the GPU works in: reference counts are changed by integer atomics, whose order does not change them, and pages are given out
// by rank, the free pages of lowest number in the requests' order.
//
// Each of these calls is a few microseconds of latency: none reads more than the table, the counts and, until enough pages are found, the free ones among refs.
#include "mam_pages.h"

namespace mam {

int fill_pages(const mam_pages_t *a, Pages &p)
{
    if (!a) return fail(MAM_ERR_INVALID_ARGUMENT, "null pointer");
    if (!is_type(a->type)) return fail(MAM_ERR_INVALID_ARGUMENT, "unknown element type %d", a->type);
    if (a->P < 0 || a->S < 0 || a->Hkv < 0 || a->B < 0 || a->slots < 0) return fail(MAM_ERR_INVALID_ARGUMENT, "negative size");
    if (a->D < 1 || a->D > 128 || a->Dv < 1 || a->Dv > 256) return fail(MAM_ERR_UNSUPPORTED, "head sizes are 1 to 128 (keys) and 1 to 256 (values)");
    if (a->S < 16 || a->S % 16) return fail(MAM_ERR_UNSUPPORTED, "a page holds a multiple of 16 tokens, got %lld", (long long)a->S);
    const int64_t most = INT32_MAX / 4;
    if (a->P > most || a->S > 1 << 20 || a->Hkv > 1 << 16 || a->B > most || a->slots > most || a->slots * a->S > most)
        return fail(MAM_ERR_UNSUPPORTED, "a dimension is too large");
    if (a->S * a->Hkv > most) return fail(MAM_ERR_UNSUPPORTED, "a page has too many rows");
    if (a->B > 0 && ((!a->table && a->slots > 0) || !a->lengths)) return fail(MAM_ERR_INVALID_ARGUMENT, "null pointer");
    if ((uintptr_t)a->k % 16 || (uintptr_t)a->v % 16) return fail(MAM_ERR_INVALID_ARGUMENT, "pages must begin at a multiple of 16 bytes");
    p.k = a->k; p.v = a->v;
    p.table = a->table; p.lengths = a->lengths; p.counts = a->counts;
    p.P = (int)a->P; p.S = (int)a->S; p.Hkv = (int)a->Hkv; p.d = (int)a->D; p.dv = (int)a->Dv; p.B = (int)a->B; p.slots = (int)a->slots;
    return MAM_OK;
}

namespace pages {

constexpr int MOST_REQUESTS = 4096;

// Requests, slots, pages and tokens of a page, as the calls of the bookkeeping have them.
struct Book {
    int32_t *table, *lengths, *refs;
    int B, slots, P, S;
};

int fill(int32_t *table, const int32_t *lengths, int32_t *refs, int64_t B, int64_t slots, int64_t P, int64_t S, Book &k)
{
    if (B < 0 || slots < 0 || P < 0) return fail(MAM_ERR_INVALID_ARGUMENT, "negative size");
    if (S < 16 || S % 16 || S > 1 << 20) return fail(MAM_ERR_UNSUPPORTED, "a page holds a multiple of 16 tokens, got %lld", (long long)S);
    if (B > MOST_REQUESTS) return fail(MAM_ERR_UNSUPPORTED, "a table is for %d requests at most, got %lld", MOST_REQUESTS, (long long)B);
    const int64_t most = INT32_MAX / 4;
    if (slots > most || P > most || slots * S > most || B * slots > most) return fail(MAM_ERR_UNSUPPORTED, "a dimension is too large");
    if (B > 0 && (!lengths || (slots > 0 && !table) || (P > 0 && !refs))) return fail(MAM_ERR_INVALID_ARGUMENT, "null pointer");
    k = {table, const_cast<int32_t *>(lengths), refs, (int)B, (int)slots, (int)P, (int)S};
    return MAM_OK;
}

__device__ __forceinline__ bool is_page(const Book &k, int page) { return page >= 0 && page < k.P; }
__device__ __forceinline__ int length_at(const Book &k, int n)
{
    const int most = k.slots * k.S;
    return n < 0 ? 0 : n < most ? n : most;
}

// Sum of the threads' values before this one's, and of all; THREADS / 64 words of LDS.
template <int THREADS>
__device__ __forceinline__ int before(int v, int *waves, int &total)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int sum = v;
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) {
        const int t = __shfl_up(sum, x);
        if (lane >= x) sum += t;
    }
    __syncthreads();
    if (lane == 63) waves[wave] = sum;
    __syncthreads();
    int base = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) {
        if (w < wave) base += waves[w];
        total += waves[w];
    }
    return base + sum - v;
}

// Room for counts[b] tokens behind each request's, by one workgroup.  What a request takes: pages for slots that have none, and one for a begun last page that others
// hold too, unless they all come before it and take one themselves.  The requests' needs are added up, the free pages are ranked, and rank r goes to the request
// whose needs reach past r.  A request whose needs go beyond what is free gets nothing, and so do those behind it that need any, or that could have gone without if it had been served.
//
// Bound by latency: a request a thread (four where there are more than 1024), its few loads side by side, those of the first 16384 pages' counts before all.  Measured:
// 256 requests of up to 1021 tokens, all of them beams of four that write to pages in common, 1507 pages, 10 us (four requests a thread from the start on: 24 us).
constexpr int EXTEND = 1024, PER = MOST_REQUESTS / EXTEND, SCAN = 16;

// Which of pages at .. at + 15 are free, a bit each.
__device__ __forceinline__ uint32_t free_of(const Book &k, int at)
{
    uint32_t free = 0;
    if (at + SCAN <= k.P) {
        typedef int32_t words __attribute__((ext_vector_type(4), aligned(4)));
        words w[SCAN / 4];
#pragma unroll
        for (int i = 0; i < SCAN / 4; ++i) w[i] = *reinterpret_cast<const words *>(k.refs + at + 4 * i);
#pragma unroll
        for (int i = 0; i < SCAN; ++i) free |= (uint32_t)(w[i / 4][i % 4] == 0) << i;
    } else {
        for (int i = 0; i < SCAN && at + i < k.P; ++i) free |= (uint32_t)(k.refs[at + i] == 0) << i;
    }
    return free;
}

__global__ __launch_bounds__(EXTEND) void extend_kernel(const Book k, const int32_t *__restrict__ counts, int32_t *__restrict__ granted,
                                                        int32_t *__restrict__ copies, int32_t *__restrict__ found)
{
    __shared__ int until[MOST_REQUESTS];                                        // needs of the requests up to this one
    __shared__ __attribute__((aligned(16))) int last[MOST_REQUESTS];           // begun last page that others hold too, or -1
    __shared__ int waves[EXTEND / 64];
    const int t = threadIdx.x;
    uint32_t free = free_of(k, t * SCAN);
    int held[PER], want[PER], n_of[PER], c_of[PER], copy[PER], first[PER];
    bool shared = false;
#pragma unroll
    for (int u = 0; u < PER; ++u) {
        const int b = u * EXTEND + t;
        held[u] = want[u] = n_of[u] = c_of[u] = first[u] = 0;
        copy[u] = -1;
        if (b < k.B) {
            const int n = length_at(k, k.lengths[b]), c = counts[b];
            const int32_t *row = k.table + (int64_t)b * k.slots;
            const int64_t end = (int64_t)n + (c > 0 ? c : 0);
            const bool fits = c > 0 && end <= (int64_t)k.slots * k.S;
            const int slots = fits ? (int)((end + k.S - 1) / k.S) : 0;
            int h = (n + k.S - 1) / k.S, page = -1;
            int behind = h < slots ? row[h] : -1;
            if (fits && n % k.S) {
                page = row[n / k.S];
                if (!is_page(k, page) || k.refs[page] < 2) page = -1;
            }
            while (behind >= 0) {
                ++h;
                behind = h < slots ? row[h] : -1;
            }
            held[u] = h;
            want[u] = h < slots ? slots - h : 0;
            n_of[u] = n;
            c_of[u] = fits ? c : 0;
            last[b] = page;
            shared = shared || page >= 0;
        } else if (b < MOST_REQUESTS) {
            last[b] = -1;
        }
    }
    // of the requests that write to a page, the earlier ones give it up first
    if (__syncthreads_or(shared)) {
        typedef int quad __attribute__((ext_vector_type(4)));
#pragma unroll
        for (int u = 0; u < PER; ++u) {
            const int b = u * EXTEND + t, page = b < k.B ? last[b] : -1;
            if (page < 0) continue;
            int earlier = 0, i = 0;
            for (; i + 4 <= b; i += 4) {
                const quad w = *reinterpret_cast<const quad *>(last + i);
                earlier += (w[0] == page) + (w[1] == page) + (w[2] == page) + (w[3] == page);
            }
            for (; i < b; ++i) earlier += last[i] == page;
            if (k.refs[page] - earlier > 1) copy[u] = page;
        }
    }
    int total = 0;
#pragma unroll
    for (int u = 0; u < PER; ++u) {
        if (u * EXTEND >= k.B) break;
        const int take = want[u] + (copy[u] >= 0);
        int all;
        first[u] = total + before<EXTEND>(take, waves, all);
        if (u * EXTEND + t < k.B) until[u * EXTEND + t] = first[u] + take;
        total += all;
    }
    // the free pages of lowest number, as many as are needed, by rank
    int have = 0;
    for (int base = 0; base < k.P && have < total; base += EXTEND * SCAN) {
        const int at = base + t * SCAN;
        if (base > 0) free = free_of(k, at);
        int all;
        int rank = have + before<EXTEND>(__popc(free), waves, all);
        for (; free && rank < total; free &= free - 1) found[rank++] = at + __ffs(free) - 1;
        have += all;
    }
    __threadfence_block();
    __syncthreads();
    // Where pages run out, an earlier request that was to give up a page keeps it: the one that counted on that needs a copy, for which there is no page either.  All
    // that write to the page before it were to give it up, and needs are met up to some request, so the last of them tells.
    if (total > have) {
#pragma unroll
        for (int u = 0; u < PER; ++u) {
            const int b = u * EXTEND + t, page = b < k.B && copy[u] < 0 && want[u] == 0 ? last[b] : -1;
            if (page < 0) continue;
            int i = b - 1;
            while (i >= 0 && last[i] != page) --i;
            if (i >= 0 && until[i] > have) c_of[u] = 0;
        }
        __syncthreads();
    }
    // requests whose needs are met are the first ones, and of those behind them the ones without needs
#pragma unroll
    for (int u = 0; u < PER; ++u) {
        const int b = u * EXTEND + t, take = want[u] + (copy[u] >= 0);
        if (b >= k.B) continue;
        const bool served = c_of[u] > 0 && (take == 0 || first[u] + take <= have), moved = served && copy[u] >= 0;
        const int to = moved ? found[first[u]] : -1;
        granted[b] = served ? c_of[u] : 0;
        copies[2 * b] = moved ? copy[u] : -1;
        copies[2 * b + 1] = to;
        if (moved) {
            atomicSub(&k.refs[copy[u]], 1);
            k.refs[to] = 1;
            k.table[(int64_t)b * k.slots + n_of[u] / k.S] = to;
        }
        // what the ranks below need of it: whether its first page is a copy's, and the slot of the next one
        last[b] = served && want[u] > 0 ? 2 * held[u] + (copy[u] >= 0) : -1;
    }
    __syncthreads();
    const int ranks = total < have ? total : have;
    for (int r = t; r < ranks; r += EXTEND) {
        int lo = 0, hi = k.B - 1;               // the first request with until > r
        while (lo < hi) {
            const int mid = (lo + hi) / 2;
            if (until[mid] > r) hi = mid;
            else lo = mid + 1;
        }
        const int what = last[lo], at = r - (lo ? until[lo - 1] : 0) - (what & 1);
        if (what < 0 || at < 0) continue;
        const int slot = what / 2 + at, page = found[r];
        k.table[(int64_t)lo * k.slots + slot] = page;
        k.refs[page] = 1;
    }
}

// Requests end at `ends`, or at the end of the pages that they hold; pages behind are given back.  A workgroup a request.
constexpr int TRIM = 256;
__global__ __launch_bounds__(TRIM) void trim_kernel(const Book k, const int32_t *__restrict__ ends)
{
    __shared__ int held;
    const int b = blockIdx.x;
    int32_t *row = k.table + (int64_t)b * k.slots;
    if (threadIdx.x == 0) held = k.slots;
    __syncthreads();
    for (int s = threadIdx.x; s < k.slots; s += TRIM)
        if (row[s] < 0) {
            atomicMin(&held, s);
            break;
        }
    __syncthreads();
    int n = ends[b];
    n = n < 0 ? 0 : (int64_t)n < (int64_t)held * k.S ? n : held * k.S;
    const int keep = (n + k.S - 1) / k.S;
    for (int s = keep + threadIdx.x; s < k.slots; s += TRIM) {
        const int page = row[s];
        if (page == -1) continue;
        if (is_page(k, page)) atomicSub(&k.refs[page], 1);
        row[s] = -1;
    }
    if (threadIdx.x == 0) k.lengths[b] = n;
}

// Request b goes on from request sources[b]: its table becomes that one's, up to the page of its last token; a source that is no request leaves it empty.  A workgroup has
// some columns of the table for itself, all requests of them in LDS, so that the table is changed in place.  Every workgroup reads the lengths: where one has the whole
// table it changes them at its end, else a launch of their own does.  Measured: 256 requests of 16 pages 6.5 us (17 and 4 us by 256 threads and a launch for the lengths).
constexpr int FORK = 1024, FORK_CELLS = 8192;
__device__ __forceinline__ void fork_lengths(const Book &k, const int32_t *sources, int32_t *old)
{
    for (int b = threadIdx.x; b < k.B; b += FORK) old[b] = length_at(k, k.lengths[b]);
    __syncthreads();
    for (int b = threadIdx.x; b < k.B; b += FORK) {
        const int source = sources[b];
        k.lengths[b] = source >= 0 && source < k.B ? old[source] : 0;
    }
}

__global__ __launch_bounds__(FORK) void fork_kernel(const Book k, const int32_t *__restrict__ sources, int columns, int whole)
{
    __shared__ int32_t old[FORK_CELLS];
    const int first = blockIdx.x * columns, width = k.slots - first < columns ? k.slots - first : columns, cells = k.B * width;
    for (int e = threadIdx.x; e < cells; e += FORK) {
        const int b = e / width, c = e - b * width;
        old[e] = k.table[(int64_t)b * k.slots + first + c];
    }
    __syncthreads();
    for (int e = threadIdx.x; e < cells; e += FORK) {
        const int b = e / width, c = e - b * width, source = sources[b];
        int page = -1;
        if (source >= 0 && source < k.B && first + c < (length_at(k, k.lengths[source]) + k.S - 1) / k.S) page = old[source * width + c];
        const int was = old[e];
        if (page == was) continue;
        k.table[(int64_t)b * k.slots + first + c] = page;
        if (is_page(k, page)) atomicAdd(&k.refs[page], 1);
        if (is_page(k, was)) atomicSub(&k.refs[was], 1);
    }
    if (whole) {
        __syncthreads();
        fork_lengths(k, sources, old);
    }
}

__global__ __launch_bounds__(FORK) void fork_lengths_kernel(const Book k, const int32_t *__restrict__ sources)
{
    __shared__ int32_t old[MOST_REQUESTS];
    fork_lengths(k, sources, old);
}

typedef uint32_t Words __attribute__((ext_vector_type(4)));

// Whole pieces of 16 bytes (a page's sizes are multiples of it) between places that do not overlap.
__device__ __forceinline__ void copy_pieces(Words *to, const Words *from, int64_t n, int64_t first, int64_t step)
{
    constexpr int AHEAD = 4;
    int64_t i = first;
    for (; i + (AHEAD - 1) * step < n; i += AHEAD * step) {
        Words w[AHEAD];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) w[u] = from[i + u * step];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) to[i + u * step] = w[u];
    }
    for (; i < n; i += step) to[i] = from[i];
}

// Whole pages, `parts` workgroups each.
constexpr int COPY = 256;
__global__ __launch_bounds__(COPY) void copy_kernel(const Pages p, const int32_t *__restrict__ copies, int parts, int size)
{
    const int pair = blockIdx.x / parts, part = blockIdx.x - pair * parts;
    const int from = copies[2 * pair], to = copies[2 * pair + 1];
    if (from < 0 || from >= p.P || to < 0 || to >= p.P || from == to) return;
    const int64_t rows = (int64_t)p.Hkv * p.S, k = rows * 2 * p.d * size / 16, v = rows * p.dv * size / 16;
    Words *kp = static_cast<Words *>(p.k), *vp = static_cast<Words *>(p.v);
    const int64_t first = (int64_t)part * COPY + threadIdx.x, step = (int64_t)parts * COPY;
    copy_pieces(kp + to * k, kp + from * k, k, first, step);
    copy_pieces(vp + to * v, vp + from * v, v, first, step);
}

// Token path[i] behind the cache becomes the i-th.  A thread has its piece of every token, so that a token is read before it is overwritten: the path ascends, path[i] >= i, and
// what step i writes no later step reads.  Eight tokens are read before the first of them is written.
constexpr int COMPACT = 64, MOVED = 8;
template <class E>
__global__ __launch_bounds__(COMPACT) void compact_kernel(const Pages p, const int32_t *__restrict__ path, int n, int parts, int row_k, int row_v)
{
    const int b = blockIdx.x / parts, piece = (blockIdx.x - b * parts) * COMPACT + threadIdx.x;
    const int per = row_k + row_v, head = piece / per, e = piece - head * per;     // pieces of E of a head's keys and values
    if (head >= p.Hkv) return;
    const bool value = e >= row_k;
    E *base = static_cast<E *>(value ? p.v : p.k) + (int64_t)head * p.S * (value ? row_v : row_k) + (value ? e - row_k : e);
    const int row = value ? row_v : row_k, length = length_of(p, b), count = count_of(p, b, n);
    const int32_t *steps = path + (int64_t)b * n;
    int above = -1;                     // the last place that was taken over: the path ascends, and ends where it does not
    bool on = true;
    for (int i = 0; i < count && on; i += MOVED) {
        E w[MOVED];
        int64_t to[MOVED];
#pragma unroll
        for (int u = 0; u < MOVED; ++u) {
            to[u] = -1;
            if (i + u < count && on) {
                const int step = steps[i + u];
                on = step > above;
                above = step;
                if (on && step != i + u) {
                    const int64_t from = row_of(p, b, (uint32_t)length + (uint32_t)step);
                    to[u] = row_of(p, b, (uint32_t)length + (uint32_t)(i + u));
                    if (from < 0) to[u] = -1;
                    if (to[u] >= 0) w[u] = base[from * row];
                }
            }
        }
#pragma unroll
        for (int u = 0; u < MOVED; ++u)
            if (to[u] >= 0) base[to[u] * row] = w[u];
    }
}

// What drafted tokens see, a wave a request: ancestors by doubling, six times for up to 64.
__global__ __launch_bounds__(64) void tree_kernel(const int32_t *__restrict__ parents, const int32_t *__restrict__ lengths, int64_t *__restrict__ masks,
                                                  int32_t *__restrict__ positions, int n)
{
    const int b = blockIdx.x, i = threadIdx.x;
    int parent = i < n ? parents[(int64_t)b * n + i] : -1;
    if (parent >= i) parent = -1;
    uint64_t seen = (uint64_t)1 << i;
#pragma unroll
    for (int x = 0; x < 6; ++x) {
        const int at = parent < 0 ? i : parent;
        const uint64_t more = (uint64_t)__shfl((unsigned long long)seen, at);
        const int next = __shfl(parent, at);
        if (parent >= 0) {
            seen |= more;
            parent = next;
        }
    }
    if (i < n) {
        masks[(int64_t)b * n + i] = (int64_t)seen;
        positions[(int64_t)b * n + i] = (lengths ? lengths[b] : 0) + __popcll(seen) - 1;
    }
}

}  // namespace pages
}  // namespace mam

extern "C" size_t mam_pages_extend_workspace(int64_t B, int64_t slots, int64_t P)
{
    if (B <= 0 || slots <= 0 || P <= 0) return 0;
    // ranks that are looked for: every free page at most, and what all requests can need
    const int64_t need = B * (slots + 1);
    return (size_t)(need < P ? need : P) * sizeof(int32_t);
}

extern "C" int mam_pages_extend(int32_t *table, const int32_t *lengths, int32_t *refs, const int32_t *counts, int32_t *granted, int32_t *copies, int64_t B,
                                int64_t slots, int64_t P, int64_t S, void *workspace, size_t workspace_bytes, void *stream)
{
    using namespace mam;
    pages::Book k;
    const int rc = pages::fill(table, lengths, refs, B, slots, P, S, k);
    if (rc != MAM_OK || k.B == 0) return rc;
    if (!counts || !granted || !copies) return fail(MAM_ERR_INVALID_ARGUMENT, "null pointer");
    const size_t need = mam_pages_extend_workspace(B, slots, P);
    if (need > 0 && (!workspace || workspace_bytes < need))
        return fail(MAM_ERR_WORKSPACE, "the search for pages needs %zu workspace bytes, got %zu", need, workspace ? workspace_bytes : (size_t)0);
    hipLaunchKernelGGL(pages::extend_kernel, dim3(1), dim3(pages::EXTEND), 0, static_cast<hipStream_t>(stream), k, counts, granted, copies,
                       static_cast<int32_t *>(workspace));
    return check_launch("pages::extend_kernel");
}

extern "C" int mam_pages_trim(int32_t *table, int32_t *lengths, int32_t *refs, const int32_t *ends, int64_t B, int64_t slots, int64_t P, int64_t S, void *stream)
{
    using namespace mam;
    pages::Book k;
    const int rc = pages::fill(table, lengths, refs, B, slots, P, S, k);
    if (rc != MAM_OK || k.B == 0) return rc;
    if (!ends) return fail(MAM_ERR_INVALID_ARGUMENT, "null pointer");
    hipLaunchKernelGGL(pages::trim_kernel, dim3((unsigned)k.B), dim3(pages::TRIM), 0, static_cast<hipStream_t>(stream), k, ends);
    return check_launch("pages::trim_kernel");
}

extern "C" int mam_pages_fork(int32_t *table, int32_t *lengths, int32_t *refs, const int32_t *sources, int64_t B, int64_t slots, int64_t P, int64_t S, void *stream)
{
    using namespace mam;
    pages::Book k;
    int rc = pages::fill(table, lengths, refs, B, slots, P, S, k);
    if (rc != MAM_OK || k.B == 0) return rc;
    if (!sources) return fail(MAM_ERR_INVALID_ARGUMENT, "null pointer");
    hipStream_t st = static_cast<hipStream_t>(stream);
    const int64_t cells = (int64_t)k.B * k.slots;
    const bool whole = cells > 0 && cells <= pages::FORK_CELLS;
    if (cells > 0) {
        int columns = whole ? k.slots : (int)ceil_div(k.slots, kNumCU);         // as many workgroups as CUs, of 2 columns at most where there are 4096 requests
        if (columns > pages::FORK_CELLS / k.B) columns = pages::FORK_CELLS / k.B;
        hipLaunchKernelGGL(pages::fork_kernel, dim3((unsigned)ceil_div(k.slots, columns)), dim3(pages::FORK), 0, st, k, sources, columns, (int)whole);
        rc = check_launch("pages::fork_kernel");
        if (rc != MAM_OK || whole) return rc;
    }
    hipLaunchKernelGGL(pages::fork_lengths_kernel, dim3(1), dim3(pages::FORK), 0, st, k, sources);
    return check_launch("pages::fork_lengths_kernel");
}

extern "C" int mam_pages_copy(const mam_pages_t *args, const int32_t *copies, int64_t n, void *stream)
{
    using namespace mam;
    Pages p;
    const int rc = fill_pages(args, p);
    if (rc != MAM_OK) return rc;
    if (n < 0) return fail(MAM_ERR_INVALID_ARGUMENT, "negative size");
    if (n == 0 || p.P == 0 || p.Hkv == 0) return MAM_OK;
    if (!copies || !p.k || !p.v) return fail(MAM_ERR_INVALID_ARGUMENT, "null pointer");
    const int size = (int)type_size(args->type);
    const int64_t bytes = (int64_t)p.Hkv * p.S * (2 * p.d + p.dv) * size;
    int64_t parts = ceil_div(bytes, 16 * 4 * pages::COPY);      // four pieces a thread
    if (parts > 64) parts = 64;
    if (n > INT32_MAX / parts) return fail(MAM_ERR_UNSUPPORTED, "too many pages");
    hipLaunchKernelGGL(pages::copy_kernel, dim3((unsigned)(n * parts)), dim3(pages::COPY), 0, static_cast<hipStream_t>(stream), p, copies, (int)parts, size);
    return check_launch("pages::copy_kernel");
}

extern "C" int mam_pages_compact(const mam_pages_t *args, const int32_t *path, int64_t n, void *stream)
{
    using namespace mam;
    Pages p;
    const int rc = fill_pages(args, p);
    if (rc != MAM_OK) return rc;
    if (n < 0) return fail(MAM_ERR_INVALID_ARGUMENT, "negative size");
    if (n > INT32_MAX / 4) return fail(MAM_ERR_UNSUPPORTED, "the path is too long");
    if (n == 0 || p.B == 0 || p.P == 0 || p.Hkv == 0) return MAM_OK;
    if (!path || !p.k || !p.v) return fail(MAM_ERR_INVALID_ARGUMENT, "null pointer");
    const int64_t size = type_size(args->type), k = 2 * p.d * size, v = p.dv * size;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const auto launch = [&](auto kernel, int64_t piece) {
        const int64_t parts = ceil_div(p.Hkv * (k + v) / piece, pages::COMPACT);
        if (parts > INT32_MAX / p.B) return fail(MAM_ERR_UNSUPPORTED, "too many rows");
        hipLaunchKernelGGL(kernel, dim3((unsigned)(p.B * parts)), dim3(pages::COMPACT), 0, st, p, path, (int)n, (int)parts, (int)(k / piece), (int)(v / piece));
        return check_launch("pages::compact_kernel");
    };
    if (k % 16 == 0 && v % 16 == 0) return launch(pages::compact_kernel<pages::Words>, 16);
    if (size == 2) return launch(pages::compact_kernel<uint16_t>, 2);
    return launch(pages::compact_kernel<uint32_t>, 4);
}

extern "C" int mam_draft_tree(const int32_t *parents, const int32_t *lengths, int64_t *masks, int32_t *positions, int64_t B, int64_t n, void *stream)
{
    using namespace mam;
    if (B < 0 || n < 0) return fail(MAM_ERR_INVALID_ARGUMENT, "negative size");
    if (n > 64 || B > INT32_MAX) return fail(MAM_ERR_UNSUPPORTED, "a tree has 64 tokens at most, got %lld", (long long)n);
    if (B == 0 || n == 0) return MAM_OK;
    if (!parents || !masks || !positions) return fail(MAM_ERR_INVALID_ARGUMENT, "null pointer");
    hipLaunchKernelGGL(pages::tree_kernel, dim3((unsigned)B), dim3(64), 0, static_cast<hipStream_t>(stream), parents, lengths, masks, positions, (int)n);
    return check_launch("pages::tree_kernel");
}
