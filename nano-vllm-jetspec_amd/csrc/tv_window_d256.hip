// Windowed tree attention at head sizes up to 256.
#include "tv_window.h"

namespace tv {

// Up to 32 rows: two workgroups of two waves and one buffer a compute unit where there are as many, else larger ones.
// 100 trees of 4 nodes over 1024 keys and 8 KV heads 190 us, 64 single tokens over 512 58 (with 64 rows 213 and 66); 32
// trees of 8 nodes over 4096 182, 32 single tokens over 512 33 (with 32 rows 264 and 44).
// Up to 64 rows in blocks of 64, more in blocks of 128: 4 heads a group over 4096 keys, 8 requests of 9 / 16 nodes 60 / 63
// us, 32 of them 195 / 196 (with 128 rows 72 / 73 and 221 / 222); 8 of 24 / 64 nodes 79 / 139, 32 of 32 254 (with 64 rows 91 /
// 154 and 320).
WindowShape window_shape_d256(int64_t average_rows, int64_t per_cu) {
    if (average_rows <= 32 && per_cu >= 2) return {32, 128, 2, 64};
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
