// Lists of blocks as attention's workgroups hold them in LDS, and the union of
// several: steps of one lane of 64, in host code too (a check of them runs
// without a GPU).
#pragma once

#if defined(__HIPCC__)
#define MLXVS_LANE __host__ __device__ __forceinline__
#else
#define MLXVS_LANE inline
#endif

namespace mlxvs::kern {

constexpr int kNoBlock = 0x7FFFFFFF;  // after a list's last entry
constexpr int kWindow = 2048;         // blocks whose union is made at a time

// Whether block b of a table of `cols` columns shows anything to a token whose
// own block is `own`.
MLXVS_LANE bool block_shows(int b, int cols, int own) { return b >= 0 && b < cols && b <= own; }

// Ends a list of `count` entries in `stride` places: in every place after them,
// since the lanes that read a list each start at a place of their own, and LDS
// holds what other workgroups left there.
MLXVS_LANE void end_list(int* list, int count, int stride, int lane) {
  for (int e = count + lane; e < stride; e += 64) list[e] = kNoBlock;
}

// A list's blocks within the window from `base` on: add(block - base) for each.
// (None past the table, whatever the list holds: blocks are looked up there.)
template <typename Add>
MLXVS_LANE void blocks_in_window(const int* list, int stride, int lane, int base, int cols,
                                 Add add) {
  const int end = cols - base < kWindow ? cols : base + kWindow;
  for (int e = lane; e < stride; e += 64) {
    const int b = list[e];
    if (b >= base && b < end) add(b - base);
  }
}

}  // namespace mlxvs::kern
