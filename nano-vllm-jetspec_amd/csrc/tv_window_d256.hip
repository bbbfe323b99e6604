// Windowed tree attention at head sizes up to 256.
#include "tv_window.h"

namespace tv {

WindowShape window_shape_d256(int64_t average_rows) {
    if (average_rows <= 64) return {64, 256, 1, 64};
    return {128, 256, 1, 32};
}

void launch_window_d256(const WindowParams& p, const WindowShape& shape, bool bf16, hipStream_t s) {
    switch (shape.rows) {
        case 64: return win_launch<256, 2, 2, 64, 2>(p, bf16, s);
        default: return win_launch<256, 4, 1, 32, 4>(p, bf16, s);
    }
}

}  // namespace tv
