// Windowed tree attention: entry checks, launch shape and the merge of row blocks that several
// workgroups share (the kernel and its mathematics are in tv_window.h).
#include "tv_window.h"

namespace tv {
namespace {

constexpr int kMergeThreads = 256;
constexpr int kLongRun = 1024;       // keys of a block, from which on 256 rows pay
constexpr int kFewPieces = 8, kManyRows = 1024;
constexpr int kMergeGroups = 2048;   // workgroups of the merge, about
constexpr int kLeastKeys = 128, kFewKeys = 2048;   // that a part of a block's keys is cut to; of short blocks
// Scores are in units of log2: scale * log2(e) is an fp32 number, which it is up to 2.358e38.
constexpr float kMaxScale = 2.3e38f;

// Joins the pieces of a row block: o = sum_i w_i O_i / sum_i w_i l_i, w_i = 2^(m_i - max m).
template <int D, int ROWS, int SK, class T>
__global__ void __launch_bounds__(kMergeThreads)
window_merge_kernel(const WindowParams p) {
    constexpr int CH = D / 4, kSlots = kMergeThreads / CH;
    __shared__ win_f32x4 part[2][kMergeThreads];
    __shared__ float2 part_ml[2][kSlots];
    __shared__ int32_t find[3 + kMergeThreads / 64];
    const int tid = threadIdx.x, ch = tid % CH, slot = tid / CH;
    const int id = blockIdx.x / p.num_kv_heads, head = blockIdx.x - id * p.num_kv_heads;
    WinBlock block;
    if (!win_find<ROWS, SK, kMergeThreads, false>(p, find, block, id) || block.parts == 1) return;
    const int b = block.b;
    const WinRequest req = block.req;
    const int row0 = b * ROWS, left = req.nodes * p.groups - row0, rows = left < ROWS ? left : ROWS;
    const int64_t piece0 = static_cast<int64_t>(block.first) * p.num_kv_heads + head * block.parts;
    const int splits = block.parts;
    float best, sum;
    win_f32x4 v;
    // Pieces i0, i0 + step, ... of a row.
    auto join = [&](int row, int i0, int step) {
        best = -INFINITY;
        sum = 0.0f;
        v = win_f32x4{0, 0, 0, 0};
        for (; i0 < splits; i0 += 4 * step) {
            float2 ml[4];
            win_f32x4 o[4];
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                const int i = i0 + n * step < splits ? i0 + n * step : i0;
                const int64_t of = (piece0 + i) * ROWS + row;
                ml[n] = p.ws_ml[of];
                o[n] = *reinterpret_cast<const win_f32x4*>(p.ws_o + of * D + 4 * ch);
            }
            float top = best;
#pragma unroll
            for (int n = 0; n < 4; ++n) top = fmaxf(top, ml[n].x);
            const float keep = best == top ? 1.0f : __builtin_amdgcn_exp2f(best - top);   // -inf twice: 1
            sum *= keep;
            v *= keep;
            best = top;
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                // A piece without steps has written no sums.
                if (i0 + n * step >= splits || ml[n].y == 0.0f) continue;
                const float f = win_weight(ml[n], best);
                sum += f * ml[n].y;
                v += f * o[n];
            }
        }
    };
    auto store = [&](int row) {
        const float scale = sum == 0.0f ? 0.0f : 1.0f / sum;
        const int of = row0 + row, node = of / p.groups;
        win_store4<T>(p, req.first_row + node, head * p.groups + of - node * p.groups, 4 * ch, v * scale);
    };
    if (p.row_slots) {
        for (int row = blockIdx.y * kSlots + slot; row < rows; row += gridDim.y * kSlots) {
            join(row, 0, 1);
            store(row);
        }
        return;
    }
    int buffer = 0;
    for (int row = blockIdx.y; row < rows; row += gridDim.y, buffer ^= 1) {
        join(row, slot, kSlots);
        part[buffer][tid] = v;
        if (ch == 0) part_ml[buffer][slot] = make_float2(best, sum);
        __syncthreads();   // the next row's parts go to the other buffer
        if (slot != 0) continue;
#pragma unroll
        for (int n = 1; n < kSlots; ++n) best = fmaxf(best, part_ml[buffer][n].x);
        sum = 0.0f;
        v = win_f32x4{0, 0, 0, 0};
#pragma unroll
        for (int n = 0; n < kSlots; ++n) {
            const float2 ml = part_ml[buffer][n];
            const float f = win_weight(ml, best);
            sum += f * ml.y;
            v += f * part[buffer][n * CH + ch];
        }
        store(row);
    }
}

template <int D, int ROWS, int SK>
void launch_merge(const WindowParams& p, bool bf16, hipStream_t s) {
    constexpr int kSlots = kMergeThreads / (D / 4);
    const int64_t blocks = static_cast<int64_t>(p.block_ids) * p.num_kv_heads;
    const int64_t most = p.row_slots ? (ROWS + kSlots - 1) / kSlots : ROWS;
    int64_t parts = (kMergeGroups + blocks - 1) / blocks;
    parts = parts < most ? parts : most;
    const dim3 grid(static_cast<uint32_t>(blocks), static_cast<uint32_t>(parts));
    if (bf16) hipLaunchKernelGGL((window_merge_kernel<D, ROWS, SK, __bf16>), grid, dim3(kMergeThreads), 0, s, p);
    else hipLaunchKernelGGL((window_merge_kernel<D, ROWS, SK, _Float16>), grid, dim3(kMergeThreads), 0, s, p);
}

template <int D>
void launch_merge_d(const WindowParams& p, int rows, bool bf16, hipStream_t s) {
    if constexpr (D != 128) {   // shapes of up to 32 rows are for more blocks than are cut
        if (rows == 64) return launch_merge<D, 64, 64>(p, bf16, s);
    }
    if constexpr (D != 256) {
        if (rows == 256) return launch_merge<D, 256, 64>(p, bf16, s);
    }
    launch_merge<D, 128, 32>(p, bf16, s);
}

struct Launch {
    WindowShape shape;
    int32_t width;     // of the head-size template
    int64_t block_ids;
    int64_t units;     // workgroups of a KV head
    int32_t splits, least_steps;
    int64_t bytes;     // of the workspace
};

// The launch of a batch of this shape: row blocks by the rows an average request has, and the
// keys of a block cut where the blocks alone would leave compute units idle.
Launch launch_of(const tv_window_attention_args* a) {
    const int64_t groups = a->num_q_heads / a->num_kv_heads, rows = a->total_queries * groups;
    int64_t average = (rows + a->num_requests - 1) / a->num_requests;
    const int64_t reach = static_cast<int64_t>(a->block_table_width) * a->block_size;
    // Keys of a block, about: what its window spans and its own nodes, or all that there are.
    const int64_t nodes = average / groups;
    int64_t keys = static_cast<int64_t>(a->window) + a->sinks + (average < 256 ? average : 256) / groups;
    keys = keys < reach + nodes ? keys : reach + nodes;
    // Blocks have at most 128 nodes.  256 rows read their keys once for twice the rows, 128 are two workgroups a compute
    // unit, one of which fills the other's start and end: 32 query heads over 8 KV heads of 128, 4 chains of 1024 nodes,
    // window 128 / 512 / 1024 / 4096: 128 rows 52 / 91 / 136 / 355 us, 256 rows 67 / 102 / 138 / 328; 64 trees of 64 nodes,
    // 512 / 1024 / 4096: 79 / 131 / 393 and 88 / 131 / 365.
    // One chunk among single tokens runs in the blocks of the average: 63 tokens and a chunk of 512 / 2048 nodes, window
    // 4096, 277 / 394 us, the tokens alone 205 and the chunk 73 / 199; at head size 64 155 / 285, alone 118 and 54 / 145.
    if (average > 128 && (groups == 1 || keys < kLongRun)) average = 128;
    Launch n;
    n.width = a->head_dim <= 64 ? 64 : a->head_dim <= 128 ? 128 : 256;
    const int64_t per_cu = static_cast<int64_t>(a->num_requests) * a->num_kv_heads / a->compute_units;
    n.shape = n.width == 64    ? window_shape_d64(average, per_cu)
              : n.width == 128 ? window_shape_d128(average)
                               : window_shape_d256(average, per_cu);
    n.block_ids = rows / n.shape.rows + a->num_requests;
    int64_t blocks = (rows + n.shape.rows - 1) / n.shape.rows;
    blocks = (blocks > a->num_requests ? blocks : a->num_requests) * a->num_kv_heads;
    // Few rows have small pieces, and their keys' latency is what they wait for: one request of 1 / 16 nodes over 1024 keys
    // 13.1 / 15.7 us (with parts of 128 14.6 / 16.9), over 200 keys 12.5 (16.4), but 4 of 16 nodes over 1000 18.4 with 128
    // (23.3).  Two parts do not pay for the merge: one token and a window of 100 11.8 in one (12.6), 32 and of 200 15.4
    // (19.4).
    const bool few = static_cast<int64_t>(a->total_queries) * a->num_q_heads < kManyRows && keys <= kFewKeys;
    const int64_t least = few ? kLeastKeys / 2 : kLeastKeys;
    const int64_t most = (keys + least - 1) / least;
    const int64_t room = static_cast<int64_t>(a->compute_units) * n.shape.per_cu;
    int64_t splits = room / blocks;
    splits = splits < most ? splits : most;
    splits = splits < kMostSplits ? splits : kMostSplits;
    n.splits = static_cast<int32_t>(splits > 1 && most > 2 ? splits : 1);
    n.least_steps = static_cast<int32_t>(least / n.shape.step);
    // The parts are dealt out on the device, by the lengths there; a block takes one at least, and as many as its keys
    // allow at most.  32 query heads over 8 KV heads of 128, as many parts for every block in brackets: 8 requests of 1 to
    // 64 nodes over 100 to 16384 keys 91 us (109), 16 of 1 to 16 over 10 to 8192 61 (72), 4 of 8 to 60 over 100 to 8192 51
    // (55); where the lengths are alike it gains nothing (8 of 40 over 4096 keys 57 (57), one token 13.0 (11.7)).
    n.units = n.block_ids * n.splits;
    if (n.splits > 1 && a->num_requests <= 64) {
        n.units = n.block_ids * (most < kMostSplits ? most : kMostSplits);
        n.units = n.units < room / a->num_kv_heads ? n.units : room / a->num_kv_heads;
        n.units = n.units > n.block_ids ? n.units : n.block_ids;
    }
    n.bytes = n.splits == 1 ? 0 : n.units * a->num_kv_heads * n.shape.rows * (n.width * 4ll + 8);
    return n;
}

int check(const tv_window_attention_args* a) {
    const char* what = "window_attention";
    if (!a) return fail(TV_ERR_INVALID, "%s: null args", what);
    if (a->num_requests < 0 || a->total_queries < 0) return fail(TV_ERR_INVALID, "%s: negative batch size", what);
    if (a->num_kv_heads < 1 || a->num_q_heads < 1 || a->num_q_heads % a->num_kv_heads) {
        return fail(TV_ERR_INVALID, "%s: %d query heads over %d KV heads", what, a->num_q_heads, a->num_kv_heads);
    }
    if (a->head_dim < 8 || a->head_dim > 256 || a->head_dim % 8) {
        return fail(TV_ERR_UNSUPPORTED, "%s: head_dim %d (multiples of 8 up to 256 are built)", what, a->head_dim);
    }
    if (a->in_dtype != TV_BF16 && a->in_dtype != TV_F16) return fail(TV_ERR_UNSUPPORTED, "%s: operands must be bf16 or f16", what);
    if (a->out_dtype != a->in_dtype && a->out_dtype != TV_F32) {
        return fail(TV_ERR_UNSUPPORTED, "%s: output must be fp32 or of the queries' type", what);
    }
    if (!(fabsf(a->scale) <= kMaxScale)) {
        return fail(TV_ERR_INVALID, "%s: scale must be finite, and its product with log2(e) in fp32", what);
    }
    if (a->window < 1 || a->sinks < 0) return fail(TV_ERR_INVALID, "%s: window %d, sinks %d", what, a->window, a->sinks);
    if (a->num_blocks < 1 || a->block_size < 1 || a->block_table_width < 0 || a->block_table_stride < 0 ||
        a->qq_bias_elems < 0 || a->compute_units < 1) {
        return fail(TV_ERR_INVALID, "%s: invalid pool, table or bias size", what);
    }
    if (a->num_blocks > 0x7fffffff / a->block_size) return fail(TV_ERR_UNSUPPORTED, "%s: pools of 2^31 slots or more", what);
    if (static_cast<int64_t>(a->total_queries) * a->num_q_heads > 0x7fffffff - 512) {
        return fail(TV_ERR_UNSUPPORTED, "%s: 2^31 query rows and heads or more", what);
    }
    if (a->num_requests > 0 && a->total_queries > 0) {
        const Launch n = launch_of(a);
        // A launch has fewer than 2^32 threads.
        if (n.units > 0xffffffffll / n.shape.threads / a->num_kv_heads) {
            return fail(TV_ERR_UNSUPPORTED, "%s: too many row blocks", what);
        }
    }
    return TV_OK;
}

}  // namespace
}  // namespace tv

using namespace tv;

extern "C" int64_t tv_sizeof_window_attention_args(void) { return static_cast<int64_t>(sizeof(tv_window_attention_args)); }

extern "C" int64_t tv_window_attention_workspace_bytes(const tv_window_attention_args* a) {
    clear_error();
    const int code = check(a);
    if (code != TV_OK) return code;
    return a->num_requests == 0 || a->total_queries == 0 ? 0 : launch_of(a).bytes;
}

extern "C" int tv_window_attention(const tv_window_attention_args* a, void* workspace, int64_t workspace_bytes, void* stream) {
    clear_error();
    const int code = check(a);
    if (code != TV_OK) return code;
    const char* what = "window_attention";
    if (a->num_requests == 0 || a->total_queries == 0) return TV_OK;
    if (!a->q || !a->k_pool || !a->v_pool || !a->out || !a->cu_seqlens_q || !a->prefix_lens || !a->node_counts ||
        !a->block_tables || !a->tree_slots || !a->qq_bias || !a->qq_bias_offsets || !a->positions) {
        return fail(TV_ERR_INVALID, "%s: null pointer", what);
    }
    bool ok = aligned(a->q, 16) && a->q_stride_row % 8 == 0 && a->q_stride_head % 8 == 0 && aligned(a->k_pool, 16) &&
              aligned(a->v_pool, 16) && a->k_stride[3] == 1 && a->v_stride[3] == 1;
    for (int i = 0; i < 3; ++i) ok = ok && a->k_stride[i] % 8 == 0 && a->v_stride[i] % 8 == 0;
    const int64_t piece = 16 / (a->out_dtype == TV_F32 ? 4 : 2);
    ok = ok && aligned(a->out, 16) && a->out_stride_row % piece == 0 && a->out_stride_head % piece == 0;
    if (!ok) return fail(TV_ERR_UNSUPPORTED, "%s: query, pool and output rows must start at 16 bytes, head dim contiguous", what);
    for (int i = 0; i < 3; ++i) {
        if (a->k_stride[i] < 0 || a->v_stride[i] < 0) return fail(TV_ERR_INVALID, "%s: negative pool strides", what);
        if (i < 2 && (a->k_stride[i] > 0x7fffffff || a->v_stride[i] > 0x7fffffff)) {
            return fail(TV_ERR_UNSUPPORTED, "%s: page and slot strides must be below 2^31", what);
        }
    }
    const Launch n = launch_of(a);
    if (n.bytes && (!workspace || !aligned(workspace, 16))) return fail(TV_ERR_INVALID, "%s: null or unaligned workspace", what);
    if (workspace_bytes < n.bytes) {
        return fail(TV_ERR_CAPACITY, "%s: workspace of %lld bytes, %lld needed", what, static_cast<long long>(workspace_bytes),
                    static_cast<long long>(n.bytes));
    }
    WindowParams p = {};
    p.q = a->q;
    p.q_s0 = a->q_stride_row;
    p.q_s1 = a->q_stride_head;
    p.k = static_cast<const char*>(a->k_pool);
    p.v = static_cast<const char*>(a->v_pool);
    p.k_s0 = static_cast<uint32_t>(2 * a->k_stride[0]);
    p.k_s1 = static_cast<uint32_t>(2 * a->k_stride[1]);
    p.k_s2 = 2 * a->k_stride[2];
    p.v_s0 = static_cast<uint32_t>(2 * a->v_stride[0]);
    p.v_s1 = static_cast<uint32_t>(2 * a->v_stride[1]);
    p.v_s2 = 2 * a->v_stride[2];
    p.same = p.k_s0 == p.v_s0 && p.k_s1 == p.v_s1;
    p.num_blocks = static_cast<int32_t>(a->num_blocks);
    p.block_size = a->block_size;
    uint32_t shift = 0;
    while ((1ull << shift) < static_cast<uint64_t>(a->block_size)) ++shift;
    p.div_shift = shift;
    p.div_mul = static_cast<uint32_t>(((1ull << 32) * ((1ull << shift) - a->block_size)) / a->block_size + 1);
    p.out = a->out;
    p.o_s0 = a->out_stride_row;
    p.o_s1 = a->out_stride_head;
    p.out_f32 = a->out_dtype == TV_F32;
    p.cu = a->cu_seqlens_q;
    p.plen = a->prefix_lens;
    p.cnt = a->node_counts;
    p.tables = a->block_tables;
    p.t_s0 = a->block_table_stride;
    const int64_t reach = static_cast<int64_t>(a->block_table_width) * a->block_size;
    p.max_prefix = reach < kWinMaxKeys ? reach : kWinMaxKeys;
    p.tree_slots = a->tree_slots;
    p.bias = a->qq_bias;
    p.bias_off = a->qq_bias_offsets;
    p.bias_elems = a->qq_bias_elems;
    p.positions = static_cast<const int32_t*>(a->positions);
    p.pos_step = a->positions_is_int64 ? 2 : 1;
    p.num_requests = a->num_requests;
    p.total_queries = a->total_queries;
    p.num_kv_heads = a->num_kv_heads;
    p.groups = a->num_q_heads / a->num_kv_heads;
    p.dim = a->head_dim;
    p.window = a->window;
    p.sinks = a->sinks;
    p.c = a->scale * 1.44269504088896340736f;
    p.block_ids = static_cast<int32_t>(n.block_ids);
    p.units = static_cast<int32_t>(n.units);
    p.splits = n.splits;
    p.least_steps = n.least_steps;
    // A group of lanes joins a row where there are rows for all, or few pieces; else a workgroup does.  One request of 1 /
    // 16 nodes over 8192 keys 18 / 27 us (with groups of lanes 28 / 36), 4 of 64 68 (with workgroups 80), 8 of 40 over 4096
    // keys 55 (65), 32 of 8 over 777 keys and one KV head 18.3 (19.8).
    p.row_slots = n.splits <= kFewPieces || static_cast<int64_t>(a->total_queries) * a->num_q_heads >= kManyRows;
    if (n.bytes) {
        const int64_t pieces = n.units * a->num_kv_heads * n.shape.rows;
        p.ws_o = static_cast<float*>(workspace);
        p.ws_ml = reinterpret_cast<float2*>(p.ws_o + pieces * n.width);
    }
    p.status = a->status;
    const bool bf16 = a->in_dtype == TV_BF16;
    const hipStream_t s = as_stream(stream);
    if (n.width == 64) launch_window_d64(p, n.shape, bf16, s);
    else if (n.width == 128) launch_window_d128(p, n.shape, bf16, s);
    else launch_window_d256(p, n.shape, bf16, s);
    const int launched = check_launch(what);
    if (launched != TV_OK || n.splits == 1) return launched;
    if (n.width == 64) launch_merge_d<64>(p, n.shape.rows, bf16, s);
    else if (n.width == 128) launch_merge_d<128>(p, n.shape.rows, bf16, s);
    else launch_merge_d<256>(p, n.shape.rows, bf16, s);
    return check_launch("window_attention merge");
}
