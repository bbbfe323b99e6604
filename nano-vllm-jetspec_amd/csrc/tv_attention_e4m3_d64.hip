// Tree attention over an e4m3 cache at head size 64.
#include "tv_attention_e4m3.h"

namespace tv {

// Few rows put the four waves side by side on the keys, many rows on the rows.  Where row blocks of 256
// would be well filled, eight waves share each key that is moved and converted, with two buffers in place
// of a second workgroup.  64 requests of 8192 to 32768 keys (uniform) and 8 KV heads, blocks of 32 / 64 / 128 / 256:
// 64 rows 1132 / 597 / 627 / 896 us, 120 rows 2113 / 1186 / 761 / 925, 250 rows 4130 / 2224 / 1483 / 1292; of
// 256 to 4096 keys, 4 rows 66 / 73 / 81 / 131, 160 rows 285 / 218 / 180 / 182.  4 rows over the long ones 556 / 567.
// The rule sees the batch's average: requests of unlike rows share one block size.
E4m3Shape e4m3_shape_d64(int64_t average_rows) {
    if (average_rows <= 32) return {32, 256, 2};
    if (average_rows <= 64) return {64, 256, 2};
    if (average_rows <= 192) return {128, 256, 2};
    return {256, 512, 1};
}

void launch_e4m3_d64(const E4m3Params& p, const E4m3Shape& shape, bool bf16, hipStream_t s) {
    switch (shape.rows) {
        case 32: return e4_launch<64, 1, 4, 1>(p, bf16, s);
        case 64: return e4_launch<64, 2, 2, 1>(p, bf16, s);
        case 128: return e4_launch<64, 4, 1, 1>(p, bf16, s);
        default: return e4_launch<64, 8, 1, 2>(p, bf16, s);
    }
}

}  // namespace tv
