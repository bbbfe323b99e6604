// Windowed tree attention at head sizes up to 128.
#include "tv_window.h"

namespace tv {

// Blocks of fewer rows than 128 gain nothing, although waves have no rows: the keys' way bounds them.  8 KV heads: 128
// single tokens over 4096 / 512 keys 374 / 60 us, 64 trees of 8 nodes over 4096 / 512 193 / 30, 64 of 16 nodes 197 / 35
// (with 32 and 64 rows 370 / 60, 195 / 34, 203 / 36).
// From 129 rows on 256: 32 requests of 33 / 40 / 56 nodes and 4 heads a group over 4096 keys 150 / 151 / 172 us, 8 of them
// 54 / 55 / 60 (with 128: 173 / 172 / 188 and 59 / 60 / 63).
WindowShape window_shape_d128(int64_t average_rows) {
    if (average_rows <= 128) return {128, 256, 2, 32};
    return {256, 512, 1, 64};
}

void launch_window_d128(const WindowParams& p, const WindowShape& shape, bool bf16, hipStream_t s) {
    if (shape.rows == 128) win_launch<128, 4, 1, 32, 4>(p, bf16, s);
    else win_launch<128, 8, 1, 64, 4>(p, bf16, s);
}

}  // namespace tv
