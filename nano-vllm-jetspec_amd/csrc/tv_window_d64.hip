// Windowed tree attention at head sizes up to 64.
#include "tv_window.h"

namespace tv {

// Up to 32 rows: four workgroups of two waves a compute unit; 128 single tokens over 512 keys 34 us, 64 over 4096 118 us
// (one of four waves with three buffers of 128 keys: 66 and 124).  From 129 rows on 256: 32 requests of 33 / 40 / 56
// nodes and 4 heads a group over 4096 keys 112 / 114 / 128 us (with 128: 134 / 136 / 128).
WindowShape window_shape_d64(int64_t average_rows) {
    if (average_rows <= 32) return {32, 128, 4, 64};
    if (average_rows <= 64) return {64, 256, 2, 64};
    if (average_rows <= 128) return {128, 256, 2, 32};
    return {256, 512, 1, 64};
}

void launch_window_d64(const WindowParams& p, const WindowShape& shape, bool bf16, hipStream_t s) {
    switch (shape.rows) {
        case 32: return win_launch<64, 1, 2, 64, 2>(p, bf16, s);
        case 64: return win_launch<64, 2, 2, 64, 3>(p, bf16, s);
        case 128: return win_launch<64, 4, 1, 32, 4>(p, bf16, s);
        default: return win_launch<64, 8, 1, 64, 4>(p, bf16, s);
    }
}

}  // namespace tv
