// Index arithmetic of the paged key/value cache, shared by its kernels and compiled by
// any C++ compiler (it holds no CUDA code), so that it is checked on the host as well.
//
// A pool is [pages, kv_heads, page_size, head_dim]; row s of the page table names the pages
// of sequence s in order: position p lives in row p % page_size of page table[s][p / page_size].
#pragma once

#include <stdint.h>

#ifdef __CUDACC__
#define Q3T_HD __host__ __device__ __forceinline__
#else
#define Q3T_HD inline
#endif

namespace q3t {

struct PageTable {
  const int32_t* table;  // [sequences][columns], row stride `stride`
  int64_t stride, sequences, columns;
  int64_t pages;         // pages of the pool: a valid entry is 0 .. pages - 1
  int page_size;         // positions per page, a multiple of 16

  // The table column that holds `position` >= 0 (32-bit division where that is enough: a third of the instructions).
  Q3T_HD int64_t column_of(int64_t position) const {
    if (position <= 0xffffffffll) return uint32_t(position) / uint32_t(page_size);
    return position / page_size;
  }
  // The page that holds `position` of `sequence`, and the position's row there; -1 where the table has none.
  Q3T_HD int64_t lookup(int64_t sequence, int64_t position, int& row) const {
    row = 0;
    if (sequence < 0 || sequence >= sequences || position < 0) return -1;
    const int64_t column = column_of(position);
    if (column >= columns) return -1;
    row = int(position - column * page_size);
    const int64_t page = table[sequence * stride + column];
    return page >= 0 && page < pages ? page : -1;
  }
};

// Where a packed sequence starts, kept far from the ends of 64 bits: its i-th row (i < 2^31) is at the result + i, which
// is negative or past every table where the given position + i is, or would not be a number.
Q3T_HD int64_t clamped_start(int64_t start) {
  const int64_t most = int64_t(1) << 40;
  return start > most ? most : start < -most ? -most : start;
}

// Decode attention streams keys in steps of 16, which never cross a page.
constexpr int kStepKeys = 16;

// Steps of a row at `position` (the row sees keys 0 .. position; -1: none).
Q3T_HD int64_t steps_of(int64_t position) { return position < 0 ? 0 : position / kStepKeys + 1; }

// The ranges that `total` steps are split into where at most `parts` can work: none of them is empty.
Q3T_HD int64_t split_parts(int64_t total, int64_t parts) { return total < parts ? total : parts; }
// `total` steps in `parts` even contiguous ranges: part i holds [split_begin(i), split_begin(i + 1)).
// total * parts stays below 2^63: a pool holds fewer than 2^47 steps and parts are at most 2^14.
Q3T_HD int64_t split_begin(int64_t i, int64_t total, int64_t parts) { return i * total / parts; }
// The part that holds step `at` (0 <= at < total): the largest i with split_begin(i) <= at.
Q3T_HD int64_t split_owner(int64_t at, int64_t total, int64_t parts) { return ((at + 1) * parts - 1) / total; }

// The row whose steps hold flattened step `at`: prefix[r] <= at / units < prefix[r + 1], where row r
// has (prefix[r + 1] - prefix[r]) * units steps (`units`: key/value heads, times the passes over wide groups).
Q3T_HD int row_of(const int32_t* prefix, int rows, int64_t at, int64_t units) {
  int lo = 0, hi = rows;  // the answer is in [lo, hi)
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (int64_t(prefix[mid]) * units <= at) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Groups of 2^shift neighbours that `count` are in, and the least shift with which they are no more than `most`.
Q3T_HD int groups_of(int64_t count, int shift) { return int((count + (int64_t(1) << shift) - 1) >> shift); }
Q3T_HD int group_shift(int64_t count, int most) {
  int shift = 0;
  while (groups_of(count, shift) > most) ++shift;
  return shift;
}

}  // namespace q3t
