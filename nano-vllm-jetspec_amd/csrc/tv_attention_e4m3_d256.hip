// Tree attention over an e4m3 cache at head size 256.
#include "tv_attention_e4m3.h"

namespace tv {

// A wave's 32 rows take 128 accumulator and 64 query registers, so one wave a SIMD; steps are half
// as long, so the staged keys take the same LDS.  64 requests of 8192 to 32768 keys (uniform) and 8 KV heads, blocks
// of 32 / 64 / 128: 4 rows 1777 / 2076 / 2750 us, 60 rows 3559 / 2107 / 2804, 120 rows 7018 / 4457 / 2830; 64
// rows with two waves on the rows alone, two workgroups a CU: 60 rows 2339.
E4m3Shape e4m3_shape_d256(int64_t average_rows) {
    if (average_rows <= 32) return {32, 128, 2};
    if (average_rows <= 64) return {64, 256, 1};
    return {128, 256, 1};
}

void launch_e4m3_d256(const E4m3Params& p, const E4m3Shape& shape, bool bf16, hipStream_t s) {
    switch (shape.rows) {
        case 32: return e4_launch<256, 1, 2, 1>(p, bf16, s);
        case 64: return e4_launch<256, 2, 2, 1>(p, bf16, s);
        default: return e4_launch<256, 4, 1, 1>(p, bf16, s);
    }
}

}  // namespace tv
