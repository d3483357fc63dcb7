// Limits that the entry points of the ragged expert products share.
#pragma once
#include <initializer_list>

#include "pmoe_common.h"

namespace pmoe {
namespace gmm {

constexpr int64_t kMaxRows = INT32_MAX - 512;  // row numbers, and those of a tile's end, are 32-bit
constexpr int kMaxSide = 1 << 28;              // columns, contraction
constexpr int64_t kMaxStride = 4 << 20;        // 16-bit elements: 256 rows stay inside 32-bit byte offsets

// Tiles a launch can have at most, -1 if they cannot be counted in 32 bits.
int64_t most_tiles(int64_t rows, int cols, int n_groups);
int grid_of(int64_t tiles);
// Whether even tiles of 128 rows are more than one round of workgroups.
bool fills(int64_t rows, int cols);

}  // namespace gmm
}  // namespace pmoe

#define PMOE_REQUIRE_STRIDE(what, stride, width, unit, most)                                                                      \
    PMOE_REQUIRE((stride) >= (width) && (stride) % (unit) == 0 && (stride) <= (most),                                             \
                 "%s: rows %lld elements apart (supported: %lld .. %lld, multiples of %d)", what, (long long)(stride),            \
                 (long long)(width), (long long)(most), (int)(unit))

#define PMOE_REQUIRE_ALIGNED(what, ...)                                                                                           \
    for (const void *p : std::initializer_list<const void *>{__VA_ARGS__})                                                        \
        PMOE_REQUIRE(reinterpret_cast<uintptr_t>(p) % 16 == 0, "%s: operands and outputs must be 16-byte aligned", what)
