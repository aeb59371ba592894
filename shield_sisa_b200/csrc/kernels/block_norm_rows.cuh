// Where rows of any pitch lie in groups of eight values, and which of those groups may be read whole.
#pragma once

namespace sb {

// Where a row starts in its group: rows of class `cls` (of P, see block_norm.cu) all at the same place.
__host__ __device__ inline int row_shift(int cls, long long ld) { return int(cls * (ld & 7) & 7); }

// The values [lo, hi) of a group that belong to a row of D; c: the row's column that the group's first value is (before the row: negative).
__host__ __device__ inline int group_lo(int c) { return c < 0 ? (-c < 8 ? -c : 8) : 0; }
__host__ __device__ inline int group_hi(int c, int D) { return D - c < 8 ? (D - c > 0 ? D - c : 0) : 8; }

// The first rows of an array, in which a group that reaches over the row's end (by seven values at most) may be read whole: those that as
// many rows follow as hold seven values.  (The last row's end is the array's, and the rows in front of it may be shorter than seven.)
__host__ __device__ inline int whole_rows(int rows, long long ld) { return ld >= 7 ? rows - 1 : ld > 0 ? rows - (6 + int(ld)) / int(ld) : 0; }
// ... and any group that ends inside its row's `width` values: `end`, the column behind the group's last value.
__host__ __device__ inline bool reads_whole(int end, int width, int row, int whole) { return end <= width || row < whole; }

}  // namespace sb
