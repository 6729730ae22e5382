// lrn_grid.h — how rows are dealt out to workgroups, for the host and the kernels (plain C++: it compiles without a GPU).
#pragma once
#include <cstdint>

#if defined(__HIP__)
#define LRN_BOTH __host__ __device__ __forceinline__
#else
#define LRN_BOTH inline
#endif

namespace lrn {

// Workgroups are numbered over two dimensions of the grid, of at most 2^20 in each line: one dimension holds fewer than 2^32 lanes.
// The lines are equally long, so that fewer workgroups are launched in excess than there are lines.
struct RowGrid { int64_t x, y; };
LRN_BOTH RowGrid row_grid(int64_t blocks) {
    const int64_t lines = (blocks + ((int64_t)1 << 20) - 1) >> 20, y = lines > 0 ? lines : 1;
    return RowGrid{(blocks + y - 1) / y, y};
}

// Rows of the workgroup that begins at row `first`, of `each` rows; 0 behind the last one, however far: what a kernel moves is
// counted from this and from nothing else.
LRN_BOTH int rows_here(int64_t rows, int64_t first, int each) {
    const int64_t left = rows - first;
    return left <= 0 ? 0 : left < each ? (int)left : each;
}

}  // namespace lrn
