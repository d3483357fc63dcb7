// Feed::set_length on the CPU, cut out of the kernels' source (slabs.inc): the slabs of contractions of up to 2^31 - 513 elements.
#include <algorithm>
#include <cstdint>
#include <cstdio>

#define __device__
#define __forceinline__ inline
using std::max;

#include "slabs.inc"

template <bool PX, bool QX>
struct Feed {
    int n_slabs, full, len_p, len_q;
#include "set_length.inc"
};

template <bool PX, bool QX>
int check(int64_t elements, int bytes_per) {
    Feed<PX, QX> f;
    f.set_length((int)elements, bytes_per);
    const int64_t bytes = elements * bytes_per, whole = bytes / kSlab, all = std::max<int64_t>((bytes + kSlab - 1) / kSlab, 2);
    if (f.full == whole && f.n_slabs == all && f.len_p == (PX ? elements : bytes) && f.len_q == (QX ? elements : bytes)) return 0;
    std::fprintf(stderr, "%lld elements of %d bytes: %d whole slabs of %d, lengths %d and %d\n", (long long)elements, bytes_per, f.full,
                 f.n_slabs, f.len_p, f.len_q);
    return 1;
}

int main() {
    int bad = 0;
    for (int64_t rows : {0ll, 1ll, 63ll, 64ll, 65ll, 127ll, 128ll, 129ll, 1ll << 29, (1ll << 30) - 1, 1ll << 30, (1ll << 30) + 65, (1ll << 31) - 513})
        bad += check<true, true>(rows, 2);  // a group's rows, in the gradient of the weights
    for (int64_t depth : {0ll, 8ll, 16ll, 64ll, 72ll, 128ll, 136ll, 131056ll, 1ll << 28}) {
        bad += check<false, false>(depth, 2) + check<false, true>(depth, 2);
        if (depth % 16 == 0) bad += check<false, false>(depth, 1);
    }
    return bad > 0;
}
