// odd_rows.h -- which 16-byte vectors of rows that do not start on 16 bytes are
// loaded whole (norm.cu; host and device, no CUDA needed).
#pragma once

namespace mgs {
namespace odd {

// Whether rows ld elements apart may be read by the vectors of v elements that they lie
// in: a row's end rounded up to v elements passes it by v - 1 at most, which has to be
// memory of the row after it. Shorter steps (rows shorter than a vector, overlapping
// rows) would let vectors before the last row pass the tensor's end. With ld = 0 rows
// are whole vectors (norm.cu's way_of wants ld and the row alike modulo v).
constexpr bool steps_far_enough(long long ld, int v) { return ld == 0 || ld >= v - 1; }

// Whether the vector at `pos` of a group that ends at `end` (both from the group's
// first vector on) is loaded whole: its elements past the end are another group's or
// row's, or the row is not the last.
constexpr bool whole(int pos, int end, int v, bool last) { return !last || pos + v <= end; }

}  // namespace odd
}  // namespace mgs
