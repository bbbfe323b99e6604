// Windowed tree attention at head sizes up to 64.
#include "tv_window.h"

namespace tv {

// Up to 32 rows: four workgroups of two waves a compute unit where there are as many, else larger ones, which have more
// keys on their way.  128 single tokens over 512 keys and 8 KV heads 31 us, 200 trees of 4 nodes over 1024 111 (with 64
// rows 40 and 120); 64 single tokens over 512 20, 64 trees of 8 nodes over 4096 114 (with 32 rows 26 and 149).
// Up to 64: 64 trees of 16 nodes over 4096 117 (with 128 rows 124).
// From 129 on 256: 32 requests of 33 / 40 / 56 nodes and 4 heads a group over 4096 103 / 104 / 114 us (with 128:
// 126 / 125 / 129).
WindowShape window_shape_d64(int64_t average_rows, int64_t per_cu) {
    if (average_rows <= 32 && per_cu >= 4) return {32, 128, 4, 64};
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
