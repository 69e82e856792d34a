// Which row of w a row of a tile's LDS holds (fp8_linear.hip).  Plain constexpr, for the kernels and for a host program.
#pragma once

namespace itts {

// The 64 rows of a wave's four fragments are dealt as 16 (r / 4) + 4 j + r % 4 (fragment j, row r of it)
constexpr int dealt_row(int i) { return (i & ~63) + 16 * (i >> 2 & 3) + 4 * (i >> 4 & 3) + (i & 3); }
// the row of the tile that is fetched for LDS row i: behind the matrix' last row (`last`, within the tile) the last again
constexpr int fetched_row(int i, int last) { return dealt_row(i) < last ? dealt_row(i) : last; }

}  // namespace itts
