// Tree attention with a sliding window and first tokens that stay visible: the kernel template and what
// its translation units share (tv_window_d<D>.hip instantiate it per head size; tv_window.hip holds the
// entry and the merge).
//
// Row (node i, query head) of a request at position P_i, over the keys of its KV head:
//     o_i = sum_j p_ij V_j / sum_j p_ij,     p_ij = 2^((scale * q_i . K_j + bias_ij - m_i) log2 e),
// prefix key j (position j) if P_i - j < window or j < sinks, tree node j <= i if its bias is not -inf and
// P_i - P_j < window or P_j < sinks.  A key at position x is seen by rows up to position x + window - 1, or
// by all; that `reach` is stored beside the key, and a row's test is one comparison.  Positions are the
// prefix length plus a depth of at most the node's index, so a row block at positions lo.. sees, without
// looking at the others, the first tokens, the prefix from lo - window + 1 on, and the nodes from index
// lo - window + 1 - prefix on (all nodes where the first tokens reach into the tree): these N keys, in
// this order, are its work, in steps of SK.  Pages outside are never looked up.
//
// A workgroup takes one row block (ROWS score rows of one request and KV head), or an equal part of its
// steps where the batch has too few blocks for the chip; a second launch joins the parts.  The request of
// a block is found from the live lengths: its blocks have the numbers from cu[r] * G / ROWS + r on, of
// which there are always enough, so a search in cu finds it and no plan or scan is needed.
//
// A step: every wave moves its share of the keys from memory to registers one step ahead (page numbers
// and slots two ahead) and from there to LDS, K and V as [key][dim] with the 16-byte chunks swizzled per
// key.  Wave (wm, wk) takes rows 32*wm.. and every WK-th 32-key tile: few rows put the waves side by side
// on the keys, many rows on the rows.  S^T = K . Q^T by 32x32x16 MFMAs leaves a row's scores in one lane
// pair, and the S^T registers are the P^T operand as they stand: product slot t of lane half g is key
// 16*kk + 8*(t/4) + 4*g + t%4, which the transposing reads of V deliver.
//
// A probability is rounded to the operands' type once where the result is of that type, and kept in
// more terms for fp32 results (bf16: 3, to 2^-26; f16: 2, to 2^-23).  f16 probabilities are held times
// 2^7, which keeps those down to 2^-21 of a row's largest normal, and 2^8 above the reference finite.
#pragma once

#include <float.h>
#include <math.h>
#include <stdint.h>

#include "tv_internal.h"

namespace tv {

struct WindowParams {
    const void* q;
    int64_t q_s0, q_s1;
    const char* k;
    const char* v;
    int64_t k_s0, k_s1, k_s2, v_s0, v_s1, v_s2;   // page, slot and head strides in bytes
    int32_t num_blocks, block_size;
    uint32_t div_mul, div_shift;                  // pos / block_size by multiplication (win_page_of)
    void* out;
    int64_t o_s0, o_s1;
    int32_t out_f32;
    const int32_t* cu;
    const int32_t* plen;
    const int32_t* cnt;
    const int32_t* tables;
    int64_t t_s0;
    int64_t max_prefix;            // keys a table row can address
    const int64_t* tree_slots;
    const float* bias;
    const int64_t* bias_off;
    int64_t bias_elems;
    const int32_t* positions;      // low words
    int32_t pos_step;              // words from one to the next: 1 or 2
    int32_t num_requests, total_queries, num_kv_heads, groups;
    int32_t dim;                   // head size, a multiple of 8 up to the template's
    int32_t window, sinks;
    float c;                       // scale * log2(e)
    int32_t block_ids;             // numbers that row blocks can have
    int32_t splits;                // workgroups a row block
    float* ws_o;
    float2* ws_ml;
    int32_t* status;
};

// How a launch of average `rows` score rows per request and KV head is shaped.
struct WindowShape {
    int32_t rows;          // score rows of a row block
    int32_t threads;
    int32_t per_cu;        // workgroups a compute unit holds
    int32_t step;          // keys of a step
};

WindowShape window_shape_d64(int64_t average_rows);
WindowShape window_shape_d128(int64_t average_rows);
WindowShape window_shape_d256(int64_t average_rows);
void launch_window_d64(const WindowParams& p, const WindowShape& shape, bool bf16, hipStream_t s);
void launch_window_d128(const WindowParams& p, const WindowShape& shape, bool bf16, hipStream_t s);
void launch_window_d256(const WindowParams& p, const WindowShape& shape, bool bf16, hipStream_t s);

namespace {

typedef __bf16 win_bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 win_f16x8 __attribute__((ext_vector_type(8)));
typedef float win_f32x16 __attribute__((ext_vector_type(16)));
typedef float win_f32x4 __attribute__((ext_vector_type(4)));
typedef int32_t win_i32x4 __attribute__((ext_vector_type(4)));
typedef short win_i16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) win_i16x4 win_lds_i16x4;

constexpr int kWinTile = 32;          // keys of an MFMA tile
constexpr int64_t kWinMaxKeys = 0x7fffff00;

// Quotient by the block size, exact below 2^31: multiplication by a rounded-up reciprocal
// (Granlund and Montgomery, "Division by invariant integers using multiplication", 1994).
__device__ __forceinline__ int32_t win_page_of(uint32_t mul, uint32_t shift, int32_t pos) {
    const uint32_t n = static_cast<uint32_t>(pos);
    return static_cast<int32_t>((__umulhi(mul, n) + n) >> shift);
}

// One request's live lengths; blocks 0: nothing to compute.
struct WinRequest {
    int32_t prefix, nodes, first_row, blocks;
    int64_t bias;
};

template <int ROWS>
__device__ __forceinline__ WinRequest win_request(const WindowParams& p, int r, bool& bad) {
    WinRequest q;
    q.prefix = p.plen[r];
    q.nodes = p.cnt[r];
    q.first_row = p.cu[r];
    q.bias = p.bias_off[r];
    q.blocks = 0;
    bad = false;
    const int32_t next = p.cu[r + 1];
    if (q.nodes == 0) return q;
    // The rows, the bias and the table row have to hold what the lengths say.
    const int64_t square = static_cast<int64_t>(q.nodes) * q.nodes;
    bad = q.prefix < 0 || q.prefix > p.max_prefix || q.nodes < 0 || q.first_row < 0 || next > p.total_queries ||
          q.first_row > next - q.nodes || q.bias < 0 || q.bias > p.bias_elems - square ||
          static_cast<int64_t>(q.prefix) + q.nodes > kWinMaxKeys;
    if (!bad) q.blocks = (q.nodes * p.groups + ROWS - 1) / ROWS;   // nodes * groups <= Q * heads < 2^31
    return q;
}

// The request that block number `id` belongs to (the last whose numbers begin at or below it), by a search
// of 64 places at a time; whether it has such a block, the caller asks.
template <int ROWS>
__device__ __forceinline__ int win_first_id(const WindowParams& p, int r) {
    const int64_t rows = static_cast<int64_t>(p.cu[r]) * p.groups;
    const int64_t id = (rows < 0 ? 0 : rows / ROWS) + r;
    return id < 0x7fffffff ? static_cast<int>(id) : 0x7fffffff;
}

template <int ROWS>
__device__ __forceinline__ int win_find(const WindowParams& p, int id) {
    const int lane = threadIdx.x & 63;
    int lo = 0, n = p.num_requests;
    while (n > 1) {
        const int step = (n + 63) / 64;
        const int64_t at = static_cast<int64_t>(lane) * step;
        const bool below = at < n && win_first_id<ROWS>(p, lo + static_cast<int>(at < n ? at : 0)) <= id;
        const int found = __popcll(__ballot(below));
        const int skip = (found > 0 ? found - 1 : 0) * step;
        lo += skip;
        n = n - skip < step ? n - skip : step;
    }
    return __builtin_amdgcn_readfirstlane(lo);
}

// A node's position: the prefix length plus a depth that its index bounds.
__device__ __forceinline__ int32_t win_position(const WinRequest& q, int node, int32_t given) {
    const int32_t most = q.prefix + node;
    return given < q.prefix ? q.prefix : given > most ? most : given;
}

template <class T>
struct WinType;
template <>
struct WinType<__bf16> {
    typedef win_bf16x8 vec;
    static constexpr uint32_t kExponent = 0x7f807f80u, kStep = 0x00800080u;
    static constexpr float kShift = 0.0f;
    static __device__ __forceinline__ win_f32x16 run(vec a, vec b, win_f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
};
template <>
struct WinType<_Float16> {
    typedef win_f16x8 vec;
    static constexpr uint32_t kExponent = 0x7c007c00u, kStep = 0x04000400u;
    static constexpr float kShift = 7.0f;
    static __device__ __forceinline__ win_f32x16 run(vec a, vec b, win_f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    }
};

// Swizzles of the 16-byte chunks of a [key][dim] row: a b128 read of one chunk column by 16 keys
// (K), and a transposing read of 4 keys x 4 chunks (V), each spread over all banks.
template <int D>
__device__ __forceinline__ int win_k_chunk(int key, int chunk) {
    return D == 64 ? chunk ^ ((key >> 1) & 7) : chunk ^ (key & 15);
}
template <int D>
__device__ __forceinline__ int win_v_chunk(int key, int chunk) {
    return D == 64 ? chunk ^ (4 * ((key >> 1) & 1)) : chunk ^ (4 * (key & 3));
}

// Maximum / sum over a lane pair (c, c + 32): the swap leaves the lower half's value in one register
// and the upper half's in the other, in every lane.
__device__ __forceinline__ float win_pair_max(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float win_pair_sum(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Weight of a partial result (m, l) against the joined maximum.  One that saw nothing has l = 0 and
// adds nothing; one whose scores are all NaN has m = -inf and a NaN l, which stays.
__device__ __forceinline__ float win_weight(float2 ml, float best) {
    return ml.x == -INFINITY ? (ml.y == 0.0f ? 0.0f : 1.0f) : __builtin_amdgcn_exp2f(ml.x - best);
}

// Writes four consecutive output dims of a row.
template <class T>
__device__ __forceinline__ void win_store4(const WindowParams& p, int64_t row, int head, int dim, win_f32x4 v) {
    if (dim >= p.dim) return;   // the head size is a multiple of 8
    if (p.out_f32) {
        float* o = static_cast<float*>(p.out) + row * p.o_s0 + head * p.o_s1 + dim;
        *reinterpret_cast<win_f32x4*>(o) = v;
    } else {
        T* o = static_cast<T*>(p.out) + row * p.o_s0 + head * p.o_s1 + dim;
        T h[4] = {static_cast<T>(v[0]), static_cast<T>(v[1]), static_cast<T>(v[2]), static_cast<T>(v[3])};
        *reinterpret_cast<u32x2*>(o) = __builtin_bit_cast(u32x2, h);
    }
}

template <int D, int WM, int WK, int SK, int NBUF, class T, int TERMS>
__global__ void __launch_bounds__(64 * WM * WK, D == 256 ? 1 : 2)
window_attention_kernel(const WindowParams p) {
    constexpr int THREADS = 64 * WM * WK, ROWS = 32 * WM;
    constexpr int LPR = D / 8;                     // lanes that move one key's row
    constexpr int KPP = THREADS / LPR;             // keys a pass of the workgroup moves
    constexpr int PASSES = SK / KPP;
    constexpr int KB = SK * D * 2;                 // bytes of a step's K (or V) in LDS
    constexpr int TILES = SK / kWinTile / WK;      // tiles a wave takes of a step
    constexpr int NK = D / 16, NB = D / 32;        // MFMAs of a tile's scores; output blocks
    constexpr float kShift = WinType<T>::kShift;
    const float kOver = __builtin_amdgcn_exp2f(8.0f + kShift);
    static_assert(PASSES <= LPR, "a lane of its row for each pass's reach");
    static_assert(SK % KPP == 0 && SK % (kWinTile * WK) == 0, "a step is whole passes and tiles");
    static_assert(KPP % 16 == 0 || (KPP % 4 == 0 && D != 64), "the swizzle's period");
    static_assert(WK == 1 || WK * 32 * D * 4 <= NBUF * 2 * KB, "the waves' results share the staging memory");
    typedef typename WinType<T>::vec V8;

    __shared__ __attribute__((aligned(1024))) char lds[NBUF * 2 * KB];
    __shared__ __attribute__((aligned(16))) int32_t lds_reach[NBUF][SK];
    __shared__ float2 lds_ml[WM * WK][32];
    __shared__ int lds_bad[NBUF];

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave % WM, wk = wave / WM;
    const int c = lane & 31, half = lane >> 5;

    // --- the row block and its keys -------------------------------------------------------------
    const int unit = blockIdx.x / p.num_kv_heads, head = blockIdx.x - unit * p.num_kv_heads;
    const int id = unit / p.splits, split = unit - id * p.splits;
    const int r = win_find<ROWS>(p, id);
    bool bad_request;
    const WinRequest req = win_request<ROWS>(p, r, bad_request);
    const int b = id - win_first_id<ROWS>(p, r);
    // The last number mostly names no block: its workgroup looks over all requests.
    if (blockIdx.x + 1 == gridDim.x) {
        for (int i = tid; i < p.num_requests; i += THREADS) {
            bool bad;
            win_request<ROWS>(p, i, bad);
            if (bad) set_status(p.status, TV_STATUS_BAD_REQUEST);
        }
    }
    if (b < 0 || b >= req.blocks) return;
    const int rows_all = req.nodes * p.groups;
    const int node0 = b * ROWS / p.groups;
    const int node1 = (b * ROWS + ROWS < rows_all ? b * ROWS + ROWS - 1 : rows_all - 1) / p.groups;   // the last
    const int32_t* positions = p.positions + static_cast<int64_t>(req.first_row) * p.pos_step;
    int32_t lowest = 0x7fffffff, highest = 0;
    for (int n = node0 + lane; n <= node1; n += 64) {
        const int32_t given = positions[static_cast<int64_t>(n) * p.pos_step];
        const int32_t at = win_position(req, n, given);
        bool wrong = at != given;
        if (p.pos_step == 2) wrong |= positions[static_cast<int64_t>(n) * 2 + 1] != 0;
        if (wrong) set_status(p.status, TV_STATUS_BAD_POSITION);
        lowest = at < lowest ? at : lowest;
        highest = at > highest ? at : highest;
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        lowest = min(lowest, __shfl_xor(lowest, o));
        highest = max(highest, __shfl_xor(highest, o));
    }
    lowest = __builtin_amdgcn_readfirstlane(lowest);
    highest = __builtin_amdgcn_readfirstlane(highest);
    const int32_t from_low = lowest >= p.window ? lowest - p.window + 1 : 0;     // seen by some row
    const int32_t from_high = highest >= p.window ? highest - p.window + 1 : 0;  // seen by all
    const int32_t n_first = p.sinks < req.prefix ? p.sinks : req.prefix;         // first tokens
    const int32_t w0 = from_low < n_first ? n_first : from_low < req.prefix ? from_low : req.prefix;
    const int32_t n_prefix = n_first + (req.prefix - w0);
    const int32_t t0 = req.prefix < p.sinks || from_low <= req.prefix ? 0 : from_low - req.prefix;
    const int32_t n_keys = n_prefix + (node1 + 1 - t0);
    const int steps = (n_keys + SK - 1) / SK;
    const int run0 = static_cast<int>(static_cast<int64_t>(steps) * split / p.splits);
    const int run1 = static_cast<int>(static_cast<int64_t>(steps) * (split + 1) / p.splits);
    const int64_t piece = (static_cast<int64_t>(id) * p.num_kv_heads + head) * p.splits + split;
    if (run0 >= run1) {   // fewer steps than workgroups
        for (int i = tid; i < ROWS; i += THREADS) p.ws_ml[piece * ROWS + i] = make_float2(-INFINITY, 0.0f);
        return;
    }
    const int32_t* table = p.tables + r * p.t_s0;
    const int64_t* slots = p.tree_slots + req.first_row;
    const char* k_head = p.k + head * p.k_s2;
    const char* v_head = p.v + head * p.v_s2;

    // The position of the v-th key of the prefix part.
    auto position_of = [&](int v) { return v < n_first ? v : v - n_first + w0; };
    // Keys [v, v + n) are all there, in the prefix, and seen by every row.
    auto clear_run = [&](int v, int n) {
        return v + n <= n_prefix && (v + n <= n_first || (v >= n_first && v - n_first + w0 >= from_high));
    };

    // --- moving a step's keys -------------------------------------------------------------------
    const int my_key = tid / LPR, my_chunk = tid % LPR;
    const bool my_dims = my_chunk * 8 < p.dim;
    int32_t entry[PASSES], entry_high[PASSES];   // page numbers, or tree slots in two halves
    u32x4 kreg[PASSES], vreg[PASSES];
    int32_t node_at = 0;            // position of the tree key of pass my_chunk
    uint32_t good = 0, wrong = 0;   // passes whose key is live and found / live and not found

    const int k_put = my_key * 2 * D + 16 * win_k_chunk<D>(my_key, my_chunk);
    const int v_put = my_key * 2 * D + 16 * win_v_chunk<D>(my_key, my_chunk);
    const int k_get = c * 2 * D + 16 * win_k_chunk<D>(c, half);
    const int v_key = 4 * half + ((lane & 15) >> 2), v_dim = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
    const int v_get = v_key * 2 * D + 16 * win_v_chunk<D>(v_key, v_dim >> 3) + 2 * (v_dim & 7);

    // Loads the page numbers (tree slots: both halves) of a step; nothing looks at them before fetch_keys().
    auto fetch_entries = [&](int i) {
#pragma unroll
        for (int n = 0; n < PASSES; ++n) {
            const int v = i * SK + n * KPP + my_key, of = v < n_keys ? v : n_keys - 1;
            const bool tree = of >= n_prefix;
            const int32_t* from = tree ? reinterpret_cast<const int32_t*>(slots + (of - n_prefix + t0))
                                       : table + win_page_of(p.div_mul, p.div_shift, position_of(of));
            entry[n] = from[0];
            entry_high[n] = from[tree ? 1 : 0];
        }
    };
    constexpr uint32_t kAll = (1u << PASSES) - 1;
    auto fetch_keys = [&](int i) {
        good = wrong = 0;
        int64_t k_of[PASSES], v_of[PASSES];
        int of_mine = 0;
#pragma unroll
        for (int n = 0; n < PASSES; ++n) {
            const int v = i * SK + n * KPP + my_key;
            const bool live = v < n_keys, tree = v >= n_prefix;
            const int32_t pos = tree ? entry[n] : position_of(v);   // a slot or a position
            const int32_t quotient = win_page_of(p.div_mul, p.div_shift, pos < 0 ? 0 : pos);
            const int32_t page = !tree ? entry[n] : entry[n] < 0 || entry_high[n] != 0 ? -1 : quotient;
            const bool found = live && page >= 0 && page < p.num_blocks;
            if (found) good |= 1u << n;
            if (live && !found) wrong |= 1u << n;
            // Every lane loads, one whose key is past the end or not found from the pool's first row.
            const int64_t at = found ? page : 0, offset = found ? pos - quotient * p.block_size : 0;
            const int64_t chunk = my_dims ? 16 * my_chunk : 0;
            k_of[n] = at * p.k_s0 + offset * p.k_s1 + chunk;
            v_of[n] = at * p.v_s0 + offset * p.v_s1 + chunk;
            if (my_chunk == n && live && tree) of_mine = v - n_prefix + t0;
        }
#pragma unroll
        for (int n = 0; n < PASSES; ++n) {
            kreg[n] = *reinterpret_cast<const u32x4*>(k_head + k_of[n]);
            vreg[n] = *reinterpret_cast<const u32x4*>(v_head + v_of[n]);
        }
        if ((i + 1) * SK > n_prefix) node_at = positions[static_cast<int64_t>(of_mine) * p.pos_step];
    };
    auto stage = [&](int step, int buf, int mark) {
        char* kb = lds + buf * 2 * KB;
        char* vb = kb + KB;
        const bool clear = clear_run(step * SK, SK) && p.dim == D;
        if (!clear || __any(good != kAll)) {
#pragma unroll
            for (int i = 0; i < PASSES; ++i) {
                const uint32_t keep = my_dims && ((good >> i) & 1) ? 0xffffffffu : 0u;
                kreg[i] &= keep;
                vreg[i] &= keep;
                // Rows that do not see a key have to get zero from its V row, and zero times NaN or infinity is
                // not.  So such elements become zeros, and the key's scores NaN instead, which hidden scores never show.
                uint32_t odd = 0;
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const uint32_t high = ((vreg[i][w] & WinType<T>::kExponent) + WinType<T>::kStep) & 0x80008000u;
                    vreg[i][w] &= ~((high >> 15) * 0xffffu);
                    odd |= high;
                }
                const uint64_t lanes = __ballot(odd != 0);
                if ((lanes >> (lane & ~(LPR - 1))) & ((1ull << LPR) - 1)) kreg[i] = u32x4{0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu};
            }
        }
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
            const int at = i * KPP * 2 * D;
            // Passes that are no multiple of 16 keys apart: the swizzle of this pass's key, an exclusive or away.
            const int kx = KPP % 16 ? k_put ^ (16 * ((win_k_chunk<D>(my_key + i * KPP, 0) ^ win_k_chunk<D>(my_key, 0)))) : k_put;
            *reinterpret_cast<u32x4*>(kb + at + kx) = kreg[i];
            *reinterpret_cast<u32x4*>(vb + at + v_put) = vreg[i];
            if (my_chunk == i) {
                const int v = step * SK + i * KPP + my_key;
                const int32_t pos = v < n_prefix ? position_of(v) : win_position(req, v - n_prefix + t0, node_at);
                const int64_t until = pos < p.sinks ? 0x7fffffff : static_cast<int64_t>(pos) + p.window - 1;
                lds_reach[buf][i * KPP + my_key] = !((good >> i) & 1) ? -1 : until < 0x7fffffff ? static_cast<int32_t>(until) : 0x7fffffff;
            }
        }
        if (wrong) {
            lds_bad[buf] = mark;
            set_status(p.status, TV_STATUS_BAD_PAGE);
        }
    };

    // --- the rows -------------------------------------------------------------------------------
    const int row = b * ROWS + 32 * wm + c;
    const bool wave_rows = b * ROWS + 32 * wm < rows_all;   // any row of this wave
    const int node = row < rows_all ? row / p.groups : -1;  // -1: no row
    const int qhead = head * p.groups + row - (node < 0 ? 0 : node) * p.groups;
    const int32_t my_pos = node < 0 ? 0 : win_position(req, node, positions[static_cast<int64_t>(node) * p.pos_step]);
    const float* bias = p.bias + req.bias + static_cast<int64_t>(node < 0 ? 0 : node) * req.nodes;
    V8 qb[NK];
    {
        const T* src = static_cast<const T*>(p.q) + static_cast<int64_t>(req.first_row + (node < 0 ? 0 : node)) * p.q_s0 +
                       (node < 0 ? 0 : qhead) * p.q_s1 + 8 * half;
#pragma unroll
        for (int i = 0; i < NK; ++i) {
            u32x4 x = {0, 0, 0, 0};
            if (node >= 0 && 16 * i + 8 * half < p.dim) x = *reinterpret_cast<const u32x4*>(src + 16 * i);
            qb[i] = __builtin_bit_cast(V8, x);
        }
    }
    win_f32x16 acc[NB];
#pragma unroll
    for (int i = 0; i < NB; ++i) acc[i] = win_f32x16{};
    float m = -INFINITY, l = 0.0f;

    // K . Q^T of a tile (LDS at `kb`): element i is key 8*(i/4) + 4*half + i%4 of the tile.
    auto products = [&](const char* kb) {
        win_f32x16 x = {};
#pragma unroll
        for (int i = 0; i < NK; ++i) {
            const u32x4 a = *reinterpret_cast<const u32x4*>(kb + (k_get ^ (32 * i)));
            x = WinType<T>::run(__builtin_bit_cast(V8, a), qb[i], x);
        }
        return x;
    };
    // Products to scores in units of log2, with the biases; those that the row does not see become -inf,
    // whatever they are.  v0: the tile's first key.
    auto mask = [&](int v0, int buf, int key0, win_f32x16& x) {
        const bool tree = v0 + kWinTile > n_prefix;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float add[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) add[i] = 0.0f;
            if (tree) {
                const int of0 = v0 - n_prefix + t0 + 16 * h + 4 * half;
                const int last = node < 0 ? 0 : node;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int of = of0 + 8 * (i >> 2) + (i & 3);
                    add[i] = bias[of < 0 ? 0 : of < last ? of : last];
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int of = of0 + 8 * (i >> 2) + (i & 3);
                    float b2 = add[i] * 1.44269504088896340736f;   // a finite bias stays finite
                    if (fabsf(b2) == INFINITY) b2 = copysignf(FLT_MAX, b2);
                    add[i] = of < t0 ? 0.0f : of <= last && add[i] != -INFINITY ? b2 : -INFINITY;
                }
            }
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                const win_i32x4 reach = *reinterpret_cast<const win_i32x4*>(&lds_reach[buf][key0 + 16 * h + 8 * g + 4 * half]);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int i = 8 * h + 4 * g + e;
                    const bool seen = my_pos <= reach[e] && add[4 * g + e] != -INFINITY;
                    x[i] = seen ? fmaf(x[i], p.c, add[4 * g + e]) : -INFINITY;
                }
            }
            __builtin_amdgcn_sched_barrier(0);   // eight biases in registers at a time
        }
    };
    auto tiles_of = [&](int step, int buf, bool bad) {
        const char* kb = lds + buf * 2 * KB + wk * kWinTile * 2 * D;
        const char* vb = kb + KB;
        const int left = n_keys - step * SK;
        const int tiles = (left < SK ? left + kWinTile - 1 : SK) / kWinTile;
        win_f32x16 x = products(kb);
#pragma unroll
        for (int n = 0; n < TILES; ++n) {
            const int t = n * WK + wk;
            if (t >= tiles) break;
            const int key = n * WK * kWinTile;   // of the tile, from the wave's first
            const int v0 = step * SK + t * kWinTile;
            float cs = p.c;
            if (bad || !clear_run(v0, kWinTile)) {
                mask(v0, buf, t * kWinTile, x);
                cs = 1.0f;
            }
            // Probabilities against the row's reference, which is near the largest score seen: it is
            // raised only when a tile's would pass 2^8, until when they cost no precision.
            float negative = m == -INFINITY ? 0.0f : kShift - m;
            win_f32x16 pr;
            // Both times in one order: a row whose neighbours raise their reference is summed a second time.
            auto exponentials = [&]() {
                float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    pr[i] = __builtin_amdgcn_exp2f(fmaf(x[i], cs, negative));
                    sum[i & 3] += pr[i];
                }
                return (sum[0] + sum[1]) + (sum[2] + sum[3]);
            };
            float tile_sum = exponentials();
            const bool over = !(tile_sum <= kOver) || m == -INFINITY;
            if (__any(over)) {   // other rows of the wave keep their reference: no row depends on another
                float top = x[0] * cs;
#pragma unroll
                for (int i = 1; i < 16; ++i) top = fmaxf(top, x[i] * cs);
                const float raised = win_pair_max(over ? 1.0f : 0.0f) != 0.0f ? fmaxf(m, win_pair_max(top)) : m;
                const float factor = raised == m ? 1.0f : __builtin_amdgcn_exp2f(m - raised);
                m = raised;
                l *= factor;
#pragma unroll
                for (int i = 0; i < NB; ++i) acc[i] *= factor;
                negative = m == -INFINITY ? 0.0f : kShift - m;
                tile_sum = exponentials();
            }
            l += tile_sum;
            V8 pb[TERMS][2];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                float pv = pr[i];
#pragma unroll
                for (int q = 0; q < TERMS; ++q) {
                    pb[q][i >> 3][i & 7] = static_cast<T>(pv);
                    if (q + 1 < TERMS) pv -= static_cast<float>(pb[q][i >> 3][i & 7]);
                }
            }
            win_i16x4 va[NB][2];
            auto read_values = [&](int kk) {
#pragma unroll
                for (int db = 0; db < NB; ++db) {
                    const char* lo = vb + (key + 16 * kk) * 2 * D + (v_get ^ (64 * db));
                    va[db][0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((win_lds_i16x4*)lo);
                    va[db][1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((win_lds_i16x4*)(lo + 8 * 2 * D));
                }
            };
            read_values(0);
            if (n + 1 < TILES) x = products(kb + (key + WK * kWinTile) * 2 * D);
#pragma unroll
            for (int kk = 0; kk < 2; ++kk) {
                if (kk) read_values(kk);
#pragma unroll
                for (int db = 0; db < NB; ++db) {
                    const V8 v8 = __builtin_bit_cast(V8, __builtin_shufflevector(va[db][0], va[db][1], 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
                    for (int q = 0; q < TERMS; ++q) acc[db] = WinType<T>::run(v8, pb[q][kk], acc[db]);
                }
            }
        }
    };

    // --- the steps ------------------------------------------------------------------------------
    if (tid < NBUF) lds_bad[tid] = 0;
    __syncthreads();
    int count = 1;   // steps begun, the mark of a buffer with a missing page
    auto compute = [&](int i, int buf) {
        if (wave_rows) tiles_of(i, buf, lds_bad[buf] == count);
    };
    fetch_entries(run0);
    fetch_keys(run0);
    if (run0 + 1 < run1) fetch_entries(run0 + 1);
    if constexpr (NBUF == 1) {
        for (int i = run0; i < run1; ++i, ++count) {
            __syncthreads();   // the last step's reads of the buffer are done
            stage(i, 0, count);
            if (i + 1 < run1) fetch_keys(i + 1);
            if (i + 2 < run1) fetch_entries(i + 2);
            __syncthreads();
            compute(i, 0);
        }
    } else {
        // Two buffers: a step is staged while the one before it is computed, by half of the waves before
        // their tiles and by the others after, so that a SIMD's matrix unit has work while the other wave moves.
        static_assert(WK == 1, "the waves would join over buffers in use");
        const bool late = wave >= WM / 2;
        auto prepare = [&](int i, int buf, int mark) {
            if (i >= run1) return;
            stage(i, buf, mark);
            if (i + 1 < run1) fetch_keys(i + 1);
            if (i + 2 < run1) fetch_entries(i + 2);
        };
        prepare(run0, 0, count);
        __syncthreads();
        int buf = 0;
        for (int i = run0; i < run1; ++i, ++count, buf ^= 1) {
            if (!late) prepare(i + 1, buf ^ 1, count + 1);
            compute(i, buf);
            if (late) prepare(i + 1, buf ^ 1, count + 1);
            __syncthreads();
        }
    }

    // --- the result: the row's output, or its unnormalised sum with (m, l) for the merge ---------
    const bool whole = p.splits == 1;
    auto put = [&](int row_in_block, int row_node, int row_head, int dim, win_f32x4 v, float row_l) {
        if (whole) {
            const float scale = row_l == 0.0f ? 0.0f : 1.0f / row_l;   // a row that sees nothing is zero
            win_store4<T>(p, req.first_row + row_node, row_head, dim, v * scale);
        } else {
            *reinterpret_cast<win_f32x4*>(p.ws_o + (piece * ROWS + row_in_block) * D + dim) = v;
        }
    };
    l = win_pair_sum(l);
    if constexpr (WK == 1) {
        if (node >= 0) {
#pragma unroll
            for (int db = 0; db < NB; ++db) {
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const win_f32x4 v = {acc[db][4 * g], acc[db][4 * g + 1], acc[db][4 * g + 2], acc[db][4 * g + 3]};
                    put(32 * wm + c, node, qhead, 32 * db + 8 * g + 4 * half, v, l);
                }
            }
            if (!whole && half == 0) p.ws_ml[piece * ROWS + 32 * wm + c] = make_float2(m, l);
        }
    } else {
        // The waves of one row group join their keys through LDS, one row group at a time.
        __syncthreads();
        if (half == 0) lds_ml[wave][c] = make_float2(m, l);
        win_f32x4* all = reinterpret_cast<win_f32x4*>(lds);
        constexpr int CH = D / 4, XM = CH < 32 ? CH - 1 : 31;
        for (int g0 = 0; g0 < WM; ++g0) {
            if (wm == g0) {
#pragma unroll
                for (int db = 0; db < NB; ++db) {
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        const win_f32x4 v = {acc[db][4 * g], acc[db][4 * g + 1], acc[db][4 * g + 2], acc[db][4 * g + 3]};
                        const int ch = (32 * db + 8 * g + 4 * half) / 4;
                        all[(wk * 32 + c) * CH + (ch ^ (c & XM))] = v;
                    }
                }
            }
            __syncthreads();
            for (int e = tid; e < 32 * CH; e += THREADS) {
                const int of_row = e / CH, ch = e % CH;
                const int in_block = 32 * g0 + of_row, of = b * ROWS + in_block;
                if (of >= rows_all) continue;
                const int n = of / p.groups;
                float best = -INFINITY;
#pragma unroll
                for (int w = 0; w < WK; ++w) best = fmaxf(best, lds_ml[w * WM + g0][of_row].x);
                float sum = 0.0f;
                win_f32x4 v = {0, 0, 0, 0};
#pragma unroll
                for (int w = 0; w < WK; ++w) {
                    const float2 ml = lds_ml[w * WM + g0][of_row];
                    const float f = win_weight(ml, best);
                    sum += f * ml.y;
                    v += f * all[(w * 32 + of_row) * CH + (ch ^ (of_row & XM))];
                }
                put(in_block, n, head * p.groups + of - n * p.groups, 4 * ch, v, sum);
                if (!whole && ch == 0) p.ws_ml[piece * ROWS + in_block] = make_float2(best, sum);
            }
            __syncthreads();
        }
    }
}

template <int D, int WM, int WK, int SK, int NBUF>
void win_launch(const WindowParams& p, bool bf16, hipStream_t s) {
    const dim3 grid(static_cast<uint32_t>(p.block_ids) * p.splits * p.num_kv_heads), block(64 * WM * WK);
    if (bf16 && !p.out_f32) hipLaunchKernelGGL((window_attention_kernel<D, WM, WK, SK, NBUF, __bf16, 1>), grid, block, 0, s, p);
    else if (bf16) hipLaunchKernelGGL((window_attention_kernel<D, WM, WK, SK, NBUF, __bf16, 3>), grid, block, 0, s, p);
    else if (!p.out_f32) hipLaunchKernelGGL((window_attention_kernel<D, WM, WK, SK, NBUF, _Float16, 1>), grid, block, 0, s, p);
    else hipLaunchKernelGGL((window_attention_kernel<D, WM, WK, SK, NBUF, _Float16, 2>), grid, block, 0, s, p);
}

}  // namespace
}  // namespace tv
