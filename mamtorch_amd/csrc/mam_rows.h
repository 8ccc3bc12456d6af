// Rows of a tensor's last dimension, from its sizes and strides alone (host).
#pragma once
#include <stdint.h>

namespace mam {

// Elements between rows that follow each other in the order of the outer dimensions, where those are one stride of at least a row's length
// apart; -1 where they are not.  A dimension of more than one row may have stride 0 (a broadcast operand, the gradient of a sum), which is no stride
// that all rows have: such a tensor is not rows.
inline int64_t row_stride(const int64_t *size, const int64_t *stride, int64_t dims)
{
    const int64_t c = size[dims - 1];
    if (c != 1 && stride[dims - 1] != 1) return -1;
    int64_t ld = c, next = 0;       // next: what the stride of the next outer dimension must be
    bool rows = false;
    for (int64_t i = dims - 2; i >= 0; --i) {
        if (size[i] == 1) continue;
        if (!rows) ld = stride[i];
        else if (stride[i] != next) return -1;
        rows = true;
        next = stride[i] * size[i];
    }
    return ld >= c ? ld : -1;
}

}  // namespace mam
