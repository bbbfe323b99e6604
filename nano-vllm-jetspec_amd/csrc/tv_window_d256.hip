// Windowed tree attention at head sizes up to 256.
#include "tv_window.h"

namespace tv {

// Up to 32 rows: two workgroups of two waves and one buffer a compute unit; 44 single tokens over 5 keys, 128 over 512,
// 48 and 16 over 4096: 16 / 132 / 317 / 115 us (64 rows, four waves, two buffers: 27 / 148 / 338 / 103).
WindowShape window_shape_d256(int64_t average_rows) {
    if (average_rows <= 32) return {32, 128, 2, 64};
    if (average_rows <= 64) return {64, 256, 1, 64};
    return {128, 256, 1, 32};
}

void launch_window_d256(const WindowParams& p, const WindowShape& shape, bool bf16, hipStream_t s) {
    switch (shape.rows) {
        case 32: return win_launch<256, 1, 2, 64, 1>(p, bf16, s);
        case 64: return win_launch<256, 2, 2, 64, 2>(p, bf16, s);
        default: return win_launch<256, 4, 1, 32, 4>(p, bf16, s);
    }
}

}  // namespace tv
