// Which bytes of a table of scales a tile reads (host and device; nothing of HIP, so that it is tested without a GPU).
#pragma once
#include <cstdint>

namespace ocrhip {

// A tile of `tile` rows from `first` on (first < rows) reads the scale bytes of its rows in loads of 4.  The window holds the
// rows that exist, rounded up to whole loads: rows beyond are not the table's where it lies between other columns of a wider
// buffer.  The rounding stays inside: a table starts on 16 bytes and its rows are a multiple of 16 apart.
constexpr int64_t scale_window(int64_t tile, int64_t rows, int64_t first) {
    const int64_t left = (rows - first + 3) / 4 * 4;
    return left < tile ? left : tile;
}

}  // namespace ocrhip
