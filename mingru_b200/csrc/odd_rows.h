// odd_rows.h -- which 16-byte vectors of rows that do not start on 16 bytes are
// loaded whole (norm.cu; host and device, no CUDA needed).
#pragma once

namespace mgs {
namespace odd {

// How many of the last rows have nothing behind them that their last vector could
// still be part of: a row's end rounded up to v elements passes it by v - 1 at most,
// and row r has (rows - 1 - r) * ld elements of later rows behind it. (With ld = 0 rows
// are whole vectors: way_of.)
constexpr int tail_rows(long long ld, int v) { return ld <= 0 || ld >= v - 1 ? 1 : (int)((v - 2 + ld) / ld); }

// Whether the vector at `pos` of a group that ends at `end` (both from the group's
// first vector on) is loaded whole: its elements past the end are another group's or
// row's, or the row is not one of the tail.
constexpr bool whole(int pos, int end, int v, bool tail) { return !tail || pos + v <= end; }

}  // namespace odd
}  // namespace mgs
