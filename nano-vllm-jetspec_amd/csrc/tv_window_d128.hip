// Windowed tree attention at head sizes up to 128.
#include "tv_window.h"

namespace tv {

// Up to 32 rows: two workgroups of two waves a compute unit, one of which loads while the other looks up and joins.
// 128 single tokens over 4096 / 512 keys, 44 over 5, 300 over 1024: 385 / 64 / 13 / 252 us; one workgroup of four waves
// with steps of 128 keys 403 / 91 / 22 / 295, four workgroups of one buffer 388 / 55 / 18 / 240.
// From 129 rows on 256: 32 requests of 33 / 40 / 56 nodes and 4 heads a group over 4096 keys 167 / 169 / 192 us, 8 of them
// 57 / 60 / 66 (with 128: 193 / 195 / 192 and 64 / 67 / 66).
WindowShape window_shape_d128(int64_t average_rows) {
    if (average_rows <= 32) return {32, 128, 2, 64};
    if (average_rows <= 64) return {64, 256, 2, 64};
    if (average_rows <= 128) return {128, 256, 2, 32};
    return {256, 512, 1, 64};
}

void launch_window_d128(const WindowParams& p, const WindowShape& shape, bool bf16, hipStream_t s) {
    switch (shape.rows) {
        case 32: return win_launch<128, 1, 2, 64, 2>(p, bf16, s);
        case 64: return win_launch<128, 2, 2, 64, 2>(p, bf16, s);
        case 128: return win_launch<128, 4, 1, 32, 4>(p, bf16, s);
        default: return win_launch<128, 8, 1, 64, 4>(p, bf16, s);
    }
}

}  // namespace tv
