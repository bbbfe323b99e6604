// Windowed tree attention at head sizes up to 64.
#include "tv_window.h"

namespace tv {

WindowShape window_shape_d64(int64_t average_rows) {
    if (average_rows <= 32) return {32, 256, 1, 128};
    if (average_rows <= 64) return {64, 256, 2, 64};
    if (average_rows <= 192) return {128, 256, 2, 32};
    return {256, 512, 1, 64};
}

void launch_window_d64(const WindowParams& p, const WindowShape& shape, bool bf16, hipStream_t s) {
    switch (shape.rows) {
        case 32: return win_launch<64, 1, 4, 128, 3>(p, bf16, s);
        case 64: return win_launch<64, 2, 2, 64, 3>(p, bf16, s);
        case 128: return win_launch<64, 4, 1, 32, 4>(p, bf16, s);
        default: return win_launch<64, 8, 1, 64, 4>(p, bf16, s);
    }
}

}  // namespace tv
