// Host-only check of the row stride that the encoder operators hand to their kernels (mamtorch_amd/csrc/mam_rows.h): every tensor of up to four
// dimensions of 1 to 3 elements over a set of strides.  Prints one line per failure and returns 1 if there is one.
#include <stdio.h>

#include "../mamtorch_amd/csrc/mam_rows.h"

static const int64_t STRIDES[] = {0, 1, 2, 3, 4, 6, 9, 12};
static int bad = 0, taken = 0;

static void check(const int64_t *size, const int64_t *stride, int64_t dims)
{
    const int64_t ld = mam::row_stride(size, stride, dims), c = size[dims - 1];
    int64_t rows = 1, dense = 1;
    for (int64_t i = 0; i < dims - 1; ++i) rows *= size[i];
    bool same = ld >= c && (c == 1 || stride[dims - 1] == 1), contiguous = true;
    for (int64_t i = dims - 1; i >= 0; --i) {
        contiguous = contiguous && (size[i] == 1 || stride[i] == dense);
        dense *= size[i];
    }
    for (int64_t r = 0; r < rows; ++r) {        // where row r stands, and where a kernel looks for it
        int64_t at = 0, rest = r;
        for (int64_t i = dims - 2; i >= 0; --i) {
            at += rest % size[i] * stride[i];
            rest /= size[i];
        }
        same = same && at == r * ld;
    }
    taken += ld >= 0;
    if ((ld >= 0 && !same) || (ld < 0 && contiguous)) {
        printf("sizes");
        for (int64_t i = 0; i < dims; ++i) printf(" %lld", (long long)size[i]);
        printf(" strides");
        for (int64_t i = 0; i < dims; ++i) printf(" %lld", (long long)stride[i]);
        printf(": row stride %lld\n", (long long)ld);
        bad = 1;
    }
}

static void strides(const int64_t *size, int64_t *stride, int64_t dims, int64_t at)
{
    if (at == dims) return check(size, stride, dims);
    for (int64_t s : STRIDES) {
        stride[at] = s;
        strides(size, stride, dims, at + 1);
    }
}

static void sizes(int64_t *size, int64_t dims, int64_t at)
{
    int64_t stride[4];
    if (at == dims) return strides(size, stride, dims, 0);
    for (size[at] = 1; size[at] <= 3; ++size[at]) sizes(size, dims, at + 1);
}

int main()
{
    int64_t size[4];
    for (int64_t dims = 1; dims <= 4; ++dims) sizes(size, dims, 0);
    if (!taken) printf("no tensor is rows\n");
    return bad || !taken;
}
