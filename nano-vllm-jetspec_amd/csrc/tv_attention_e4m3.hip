// Tree attention over an e4m3 cache: entry checks, launch shape and the merge of row blocks that
// several workgroups share (the kernel and its mathematics are in tv_attention_e4m3.h).
#include "tv_attention_e4m3.h"

namespace tv {
namespace {

constexpr int kMergeThreads = 256;
constexpr int kMaxShares = 1024;     // workgroups of the attention
constexpr int kMergeGroups = 1024;   // workgroups of the merge: four a compute unit
// Up to here the merge launches a workgroup per share and eighth of its rows, most of which find
// no job; above, the search for the work costs less.  One request of 777 keys, 64 shares: 13.1 us against
// 14.1 with the search; one of 16384 keys, 512 shares: 33.6 us with it, 64.1 without.
constexpr int kFewShares = 128;
// A row of up to so many pieces is joined by one group of lanes, others by a whole workgroup.  Four requests
// of 12288 keys and 250 rows, 17 pieces: 92 us so, 101 with a limit of 4; a limit above 64 costs a request
// of 16384 keys and 64 rows 39.8 us in place of 33.6.
constexpr int kFewPieces = 16;
// Scores are in units of log2: scale * log2(e) is an fp32 number, which it is up to 2.358e38.
constexpr float kMaxScale = 2.3e38f;

template <int CTRL, int ROW_MASK>
__device__ __forceinline__ int32_t add_from(int32_t x) {
    return x + __builtin_amdgcn_update_dpp(0, x, CTRL, ROW_MASK, 0xf, false);
}

// Sum over the lanes up to this one: inside the rows of 16, then each row's last lane to the rows behind.
__device__ __forceinline__ int32_t running_sum(int32_t x) {
    x = add_from<0x111, 0xf>(x);   // row_shr 1, 2, 4, 8
    x = add_from<0x112, 0xf>(x);
    x = add_from<0x114, 0xf>(x);
    x = add_from<0x118, 0xf>(x);
    x = add_from<0x142, 0xa>(x);   // row_bcast 15 to rows 1 and 3
    x = add_from<0x143, 0xc>(x);   // row_bcast 31 to rows 2 and 3
    return x;
}

// Joins the pieces of the row blocks that several workgroups share: o = sum_i w_i O_i / sum_i w_i l_i,
// w_i = 2^(m_i - max m).  Which blocks these are only the attention's workgroups know (their jobs), so each
// workgroup here adds up all jobs' work, a row's pieces, and takes an equal part of the rows.  The pieces
// come from memory and their latency bounds it, so a thread keeps four in flight.
template <int D, int ROWS, class T>
__global__ void __launch_bounds__(kMergeThreads)
e4m3_merge_kernel(const E4m3Params p) {
    constexpr int CH = D / 4, kSlots = kMergeThreads / CH;
    __shared__ e4_f32x4 part[2][kMergeThreads];
    __shared__ float2 part_ml[2][kSlots];
    __shared__ int32_t work[kMaxShares + 64];   // a wave looks at 64 shares from any of them on
    __shared__ int32_t wave_work[kMergeThreads / 64], start[2];
    const int tid = threadIdx.x, lane = tid & 63;
    const int ch = tid % CH, slot = tid / CH;
    int share = blockIdx.x, buffer = 0;
    E4m3Job job;
    float best, sum;
    e4_f32x4 v;
    // Pieces i0, i0 + step, ... of a row.
    auto join = [&](int row, int i0, int step) {
        best = -INFINITY;
        sum = 0.0f;
        v = e4_f32x4{0, 0, 0, 0};
        for (; i0 < job.pieces; i0 += 4 * step) {
            float2 ml[4];
            e4_f32x4 o[4];
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                const int i = i0 + n * step < job.pieces ? i0 + n * step : i0;
                // The first piece is its share's second, the following shares begin with theirs.
                const int64_t of = static_cast<int64_t>(2 * (share + i) + (i == 0 ? 1 : 0)) * ROWS + row;
                ml[n] = p.ws_ml[of];
                o[n] = *reinterpret_cast<const e4_f32x4*>(p.ws_o + of * D + 4 * ch);
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
                if (i0 + n * step >= job.pieces) break;
                const float f = e4_weight(ml[n], best);
                sum += f * ml[n].y;
                v += f * o[n];
            }
        }
    };
    auto store = [&](int row) {
        const float scale = sum == 0.0f ? 0.0f : 1.0f / sum;
        const int of = job.row0 + row, node = of / p.groups;
        e4_store4<T>(p, job.first_row + node, job.head0 + of - node * p.groups, 4 * ch, v * scale);
    };
    // Rows [row0, row1) of the job that `share` left.
    auto join_rows = [&](int row0, int row1) {
        if (job.pieces <= kFewPieces) {
            for (int row = row0 + slot; row < row1; row += kSlots) {
                join(row, 0, 1);
                store(row);
            }
            return;
        }
        for (int row = row0; row < row1; ++row, buffer ^= 1) {
            join(row, slot, kSlots);
            part[buffer][tid] = v;
            if (ch == 0) part_ml[buffer][slot] = make_float2(best, sum);
            __syncthreads();   // the next row's parts go to the other buffer
            if (slot != 0) continue;
#pragma unroll
            for (int n = 1; n < kSlots; ++n) best = fmaxf(best, part_ml[buffer][n].x);
            sum = 0.0f;
            v = e4_f32x4{0, 0, 0, 0};
#pragma unroll
            for (int n = 0; n < kSlots; ++n) {
                const float2 ml = part_ml[buffer][n];
                const float f = e4_weight(ml, best);
                sum += f * ml.y;
                v += f * part[buffer][n * CH + ch];
            }
            store(row);
        }
    };
    if (gridDim.y > 1) {
        job = p.jobs[share];
        if (job.pieces == 0) return;
        const int rows = (job.rows + gridDim.y - 1) / gridDim.y, row0 = blockIdx.y * rows;
        join_rows(row0, min(row0 + rows, static_cast<int>(job.rows)));
        return;
    }
    const int per = (p.workgroups + kMergeThreads - 1) / kMergeThreads;
    int32_t mine = 0;
    for (int k = 0; k < per; ++k) {
        const int j = tid * per + k;
        const int32_t w = j < p.workgroups ? p.jobs[j].pieces * p.jobs[j].rows : 0;
        work[j] = w;
        mine += w;
    }
    int32_t upto = running_sum(mine);   // of the threads up to this one
    if (lane == 63) wave_work[tid >> 6] = upto;
    __syncthreads();
    int32_t total = 0;
#pragma unroll
    for (int w = 0; w < kMergeThreads / 64; ++w) {
        if (w < (tid >> 6)) upto += wave_work[w];
        total += wave_work[w];
    }
    const int32_t each = (total + static_cast<int32_t>(gridDim.x) - 1) / static_cast<int32_t>(gridDim.x);
    const int32_t lo = blockIdx.x * each, hi = lo + each < total ? lo + each : total;
    if (lo >= hi) return;
    if (upto - mine <= lo && lo < upto) {
        int32_t before = upto - mine;
        int j = tid * per;
        while (before + work[j] <= lo) before += work[j++];
        start[0] = j;
        start[1] = before;
    }
    __syncthreads();
    share = __builtin_amdgcn_readfirstlane(start[0]);
    for (int32_t before = __builtin_amdgcn_readfirstlane(start[1]); before < hi; before += work[share++]) {
        // The next share that left a job: there is one, since `before` is below the total.
        for (;;) {
            const uint64_t any = __ballot(work[share + lane] != 0);
            if (any) {
                share += __ffsll(static_cast<unsigned long long>(any)) - 1;
                break;
            }
            share += 64;
        }
        job = p.jobs[share];
        const int32_t from = lo - before, to = hi - before;
        join_rows(from <= 0 ? 0 : (from + job.pieces - 1) / job.pieces,
                  to >= work[share] ? job.rows : (to + job.pieces - 1) / job.pieces);
    }
}

template <int D, int ROWS>
void launch_merge(const E4m3Params& p, bool bf16, hipStream_t s) {
    const int32_t heads = p.num_kv_heads * p.groups;
    const int64_t most = static_cast<int64_t>(p.total_queries) * heads;   // a row is the least part
    const dim3 grid = p.workgroups <= kFewShares ? dim3(p.workgroups, 8)
                                                 : dim3(static_cast<uint32_t>(most < kMergeGroups ? most : kMergeGroups));
    if (bf16) hipLaunchKernelGGL((e4m3_merge_kernel<D, ROWS, __bf16>), grid, dim3(kMergeThreads), 0, s, p);
    else hipLaunchKernelGGL((e4m3_merge_kernel<D, ROWS, _Float16>), grid, dim3(kMergeThreads), 0, s, p);
}

template <int D>
void launch_merge_d(const E4m3Params& p, int rows, bool bf16, hipStream_t s) {
    if (rows == 32) launch_merge<D, 32>(p, bf16, s);
    else if (rows == 64) launch_merge<D, 64>(p, bf16, s);
    else if (rows == 128) launch_merge<D, 128>(p, bf16, s);
    else launch_merge<D, 256>(p, bf16, s);
}

struct Launch {
    E4m3Shape shape;
    int32_t workgroups;
    int64_t bytes;     // of the workspace
};

// The launch of a batch of this shape: row blocks by the rows an average request has, and as many
// workgroups as the chip holds, or the steps a batch of this shape can have where that is fewer.
Launch launch_of(const tv_tree_attention_e4m3_args* a) {
    const int64_t groups = a->num_q_heads / a->num_kv_heads, rows = a->total_queries * groups;
    const int64_t average = (rows + a->num_requests - 1) / a->num_requests;
    Launch n;
    n.shape = a->head_dim == 64 ? e4m3_shape_d64(average) : a->head_dim == 128 ? e4m3_shape_d128(average)
                                                                               : e4m3_shape_d256(average);
    const int64_t keys = e4_step_keys(a->head_dim);
    const int64_t reach = static_cast<int64_t>(a->block_table_width) * a->block_size;
    const int64_t blocks = (rows / n.shape.rows + a->num_requests) * a->num_kv_heads;
    const int64_t most = blocks * ((reach + keys - 1) / keys + (a->total_queries + keys - 1) / keys);
    int64_t full = static_cast<int64_t>(a->compute_units) * n.shape.per_cu;
    full = full < kMaxShares ? full : kMaxShares;
    n.workgroups = static_cast<int32_t>(((most < full ? most : full) + 7) / 8 * 8);
    n.bytes = 2ll * n.workgroups * n.shape.rows * (a->head_dim * 4 + 8) + n.workgroups * static_cast<int64_t>(sizeof(E4m3Job));
    return n;
}

int check(const tv_tree_attention_e4m3_args* a) {
    const char* what = "tree_attention_e4m3";
    if (!a) return fail(TV_ERR_INVALID, "%s: null args", what);
    if (a->num_requests < 0 || a->total_queries < 0) return fail(TV_ERR_INVALID, "%s: negative batch size", what);
    if (a->num_kv_heads < 1 || a->num_q_heads < 1 || a->num_q_heads % a->num_kv_heads) {
        return fail(TV_ERR_INVALID, "%s: %d query heads over %d KV heads", what, a->num_q_heads, a->num_kv_heads);
    }
    if (a->head_dim != 64 && a->head_dim != 128 && a->head_dim != 256) {
        return fail(TV_ERR_UNSUPPORTED, "%s: head_dim %d (64, 128 and 256 are built)", what, a->head_dim);
    }
    if (a->in_dtype != TV_BF16 && a->in_dtype != TV_F16) return fail(TV_ERR_UNSUPPORTED, "%s: queries must be bf16 or f16", what);
    if (a->out_dtype != a->in_dtype && a->out_dtype != TV_F32) {
        return fail(TV_ERR_UNSUPPORTED, "%s: output must be fp32 or of the queries' type", what);
    }
    if (!(fabsf(a->scale) <= kMaxScale)) {
        return fail(TV_ERR_INVALID, "%s: scale must be finite, and its product with log2(e) in fp32", what);
    }
    if (a->num_blocks < 1 || a->block_size < 1 || a->block_table_width < 0 || a->block_table_stride < 0 ||
        a->qq_bias_elems < 0 || a->compute_units < 1) {
        return fail(TV_ERR_INVALID, "%s: invalid pool, table or bias size", what);
    }
    if (a->num_blocks > 0x7fffffff / a->block_size) return fail(TV_ERR_UNSUPPORTED, "%s: pools of 2^31 slots or more", what);
    if (static_cast<int64_t>(a->total_queries) * a->num_q_heads > 0x7fffffff - 512) {
        return fail(TV_ERR_UNSUPPORTED, "%s: 2^31 query rows and heads or more", what);
    }
    return TV_OK;
}

}  // namespace
}  // namespace tv

using namespace tv;

extern "C" int64_t tv_sizeof_tree_attention_e4m3_args(void) {
    return static_cast<int64_t>(sizeof(tv_tree_attention_e4m3_args));
}

extern "C" int64_t tv_tree_attention_e4m3_workspace_bytes(const tv_tree_attention_e4m3_args* a) {
    clear_error();
    const int code = check(a);
    if (code != TV_OK) return code;
    return a->num_requests == 0 || a->total_queries == 0 ? 0 : launch_of(a).bytes;
}

extern "C" int tv_tree_attention_e4m3(const tv_tree_attention_e4m3_args* a, void* workspace, int64_t workspace_bytes,
                                      void* stream) {
    clear_error();
    const int code = check(a);
    if (code != TV_OK) return code;
    const char* what = "tree_attention_e4m3";
    if (a->num_requests == 0 || a->total_queries == 0) return TV_OK;
    if (!a->q || !a->k_pool || !a->v_pool || !a->k_scale || !a->v_scale || !a->out || !a->cu_seqlens_q || !a->prefix_lens ||
        !a->node_counts || !a->block_tables || !a->tree_slots || !a->qq_bias || !a->qq_bias_offsets) {
        return fail(TV_ERR_INVALID, "%s: null pointer", what);
    }
    bool ok = aligned(a->q, 16) && a->q_stride_row % 8 == 0 && a->q_stride_head % 8 == 0 && aligned(a->k_pool, 16) &&
              aligned(a->v_pool, 16) && a->k_stride[3] == 1 && a->v_stride[3] == 1;
    for (int i = 0; i < 3; ++i) ok = ok && a->k_stride[i] % 16 == 0 && a->v_stride[i] % 16 == 0;
    const int64_t piece = 16 / (a->out_dtype == TV_F32 ? 4 : 2);
    ok = ok && aligned(a->out, 16) && a->out_stride_row % piece == 0 && a->out_stride_head % piece == 0;
    if (!ok) return fail(TV_ERR_UNSUPPORTED, "%s: query, pool and output rows must start at 16 bytes, head dim contiguous", what);
    const int64_t* strides[] = {a->k_stride, a->v_stride, a->k_scale_stride, a->v_scale_stride};
    for (const int64_t* stride : strides) {
        if (stride[0] < 0 || stride[1] < 0 || stride[2] < 0 || stride[1] > 0x7fffffff || stride[2] > 0x7fffffff) {
            return fail(TV_ERR_UNSUPPORTED, "%s: slot and head strides must be below 2^31, none negative", what);
        }
    }
    const Launch n = launch_of(a);
    if (!workspace || !aligned(workspace, 16)) return fail(TV_ERR_INVALID, "%s: null or unaligned workspace", what);
    if (workspace_bytes < n.bytes) {
        return fail(TV_ERR_CAPACITY, "%s: workspace of %lld bytes, %lld needed", what, static_cast<long long>(workspace_bytes),
                    static_cast<long long>(n.bytes));
    }
    E4m3Params p = {};
    p.q = a->q;
    p.q_s0 = a->q_stride_row;
    p.q_s1 = a->q_stride_head;
    p.k = static_cast<const uint8_t*>(a->k_pool);
    p.v = static_cast<const uint8_t*>(a->v_pool);
    p.k_s0 = a->k_stride[0];
    p.v_s0 = a->v_stride[0];
    p.kc_s0 = a->k_scale_stride[0];
    p.vc_s0 = a->v_scale_stride[0];
    p.k_s1 = static_cast<int32_t>(a->k_stride[1]);
    p.k_s2 = static_cast<int32_t>(a->k_stride[2]);
    p.v_s1 = static_cast<int32_t>(a->v_stride[1]);
    p.v_s2 = static_cast<int32_t>(a->v_stride[2]);
    p.kc_s1 = static_cast<int32_t>(a->k_scale_stride[1]);
    p.kc_s2 = static_cast<int32_t>(a->k_scale_stride[2]);
    p.vc_s1 = static_cast<int32_t>(a->v_scale_stride[1]);
    p.vc_s2 = static_cast<int32_t>(a->v_scale_stride[2]);
    p.ks = a->k_scale;
    p.vs = a->v_scale;
    p.num_blocks = static_cast<int32_t>(a->num_blocks);
    p.block_size = a->block_size;
    const int64_t keys = e4_step_keys(a->head_dim);
    bool same = a->block_size % keys == 0;
    for (int i = 0; i < 3; ++i) {
        same = same && a->k_stride[i] == a->v_stride[i] && a->k_scale_stride[i] == a->v_scale_stride[i];
    }
    const int64_t reach_of[] = {a->block_size * a->k_stride[1], 4 * a->block_size * a->k_scale_stride[1]};
    p.page_steps = same && a->k_stride[0] <= 0xffffffffll && a->k_scale_stride[0] <= 0x3fffffffll &&
                   reach_of[0] <= 0x7fffffff && reach_of[1] <= 0x7fffffff;
    if (p.page_steps) {
        p.f_s0 = static_cast<uint32_t>(a->k_stride[0]);
        p.f_s1 = static_cast<uint32_t>(a->k_stride[1]);
        p.f_c0 = static_cast<uint32_t>(4 * a->k_scale_stride[0]);
        p.f_c1 = static_cast<uint32_t>(4 * a->k_scale_stride[1]);
    }
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
    p.max_prefix = reach < 0x7fffff00 ? reach : 0x7fffff00;
    p.tree_slots = a->tree_slots;
    p.bias = a->qq_bias;
    p.bias_off = a->qq_bias_offsets;
    p.bias_elems = a->qq_bias_elems;
    p.num_requests = a->num_requests;
    p.total_queries = a->total_queries;
    p.num_kv_heads = a->num_kv_heads;
    p.groups = a->num_q_heads / a->num_kv_heads;
    p.c = a->scale * 1.44269504088896340736f;
    p.workgroups = n.workgroups;
    p.ws_o = static_cast<float*>(workspace);
    p.ws_ml = reinterpret_cast<float2*>(p.ws_o + 2ll * n.workgroups * n.shape.rows * a->head_dim);
    p.jobs = reinterpret_cast<E4m3Job*>(p.ws_ml + 2ll * n.workgroups * n.shape.rows);
    p.status = a->status;
    const bool bf16 = a->in_dtype == TV_BF16;
    const hipStream_t s = as_stream(stream);
    if (a->head_dim == 64) launch_e4m3_d64(p, n.shape, bf16, s);
    else if (a->head_dim == 128) launch_e4m3_d128(p, n.shape, bf16, s);
    else launch_e4m3_d256(p, n.shape, bf16, s);
    const int launched = check_launch(what);
    if (launched != TV_OK) return launched;
    if (a->head_dim == 64) launch_merge_d<64>(p, n.shape.rows, bf16, s);
    else if (a->head_dim == 128) launch_merge_d<128>(p, n.shape.rows, bf16, s);
    else launch_merge_d<256>(p, n.shape.rows, bf16, s);
    return check_launch("tree_attention_e4m3 merge");
}
