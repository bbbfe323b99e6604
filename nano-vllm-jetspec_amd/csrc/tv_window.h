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
// steps where the batch has too few blocks for the chip (win_parts); a second launch joins the parts.  Every
// workgroup finds its block from the live lengths by a sum over the requests' blocks, so no plan is needed;
// blocks that are not there come last in the launch, since they are what balances it when they lie between others
// (every second one missing kept half of the shader engines idle, at twice the time).
//
// A key's page, place and reach are looked up once, a thread a key, into tables of 256 or 512 keys in LDS,
// made one step before their first use.  Tiles of 32 keys that every node of the block sees are found with
// them by one vote; of the others a table holds a bit a node and key, from the reaches and the biases,
// which are read there once, coalesced, instead of by every row of every step.  Between the tables a step
// has no other loads than the DMA of K and V rows to LDS ([key][dim], 16-byte chunks swizzled per key),
// which stays under way over barriers, up to three steps ahead.
// Wave (wm, wk) takes rows 32*wm.. and every WK-th 32-key tile: few rows put the waves side by side
// on the keys, many rows on the rows.  S^T = K . Q^T by 32x32x16 MFMAs leaves a row's scores in one lane
// pair, and the S^T registers are the P^T operand as they stand: product slot t of lane half g is key
// 16*kk + 8*(t/4) + 4*g + t%4, which the transposing reads of V deliver.  With the waves on the rows the scores of
// the next tile are multiplied in turn with the values of this one, each operand read kAhead products before.
// A row's reference is raised only when a tile's probabilities would pass 2^8, so most tiles rescale nothing.
//
// 32 query heads over 8 KV heads of 128, bf16: 64 trees of 64 nodes over 8192 keys each take 666 to 705 us by the box,
// 0.78 to 0.82 PFLOP/s, the matrix and the vector units busy 40 and 38 % of the time, hardly at once, since a tile's exponentials stand
// before its step's products (keys through registers, and a reach test and a bias read for every score, took 1302);
// 128 single tokens over 4096 keys are bound by memory, 376 us at 5.7 TB/s (484).
//
// A probability is rounded to the operands' type once where the result is of that type, since the matrix unit takes both
// operands in one type and each further term is as many products of P . V again.  The sum is of the rounded ones, so an
// error common to all cancels; against 64 bits results of N(0, 1) inputs in bf16 are off by 0.0021 to 0.0023 of their size
// where the last rounding alone is 0.0017.  For fp32 results it is kept in more terms (bf16: 3, to 2^-26; f16: 2, to
// 2^-23).  f16 probabilities are held times 2^7, which keeps those down to 2^-21 of a row's largest normal, and 2^8 above
// the reference finite.
#pragma once

#include <float.h>
#include <math.h>
#include <stdint.h>

#include <type_traits>

#include "tv_internal.h"

namespace tv {

struct WindowParams {
    const void* q;
    int64_t q_s0, q_s1;
    const char* k;
    const char* v;
    uint32_t k_s0, k_s1, v_s0, v_s1;              // page and slot strides in bytes
    int64_t k_s2, v_s2;                           // head strides
    int32_t num_blocks, block_size;
    uint32_t div_mul, div_shift;                  // pos / block_size by multiplication (win_page_of)
    int32_t same;                                 // K and V have the same page and slot strides
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
    const int32_t* positions;      // int32, or int64 as its words
    int32_t pos_step;              // words from one to the next: 1 or 2
    int32_t num_requests, total_queries, num_kv_heads, groups;
    int32_t dim;                   // head size, a multiple of 8 up to the template's
    int32_t window, sinks;
    float c;                       // scale * log2(e)
    int32_t block_ids;             // numbers that row blocks can have
    int32_t units;                 // workgroups of a KV head
    int32_t splits;                // of a row block, if each has as many
    int32_t least_steps;           // of a part
    int32_t row_slots;             // the merge gives a row a group of lanes, not a workgroup
    float* ws_o;
    float2* ws_ml;
    int32_t* status;
};

// How a launch is shaped: by the score rows of an average request and KV head, and by how many of these there are a
// compute unit.
struct WindowShape {
    int32_t rows;          // score rows of a row block
    int32_t threads;
    int32_t per_cu;        // workgroups a compute unit holds
    int32_t step;          // keys of a step
};

WindowShape window_shape_d64(int64_t average_rows, int64_t per_cu);
WindowShape window_shape_d128(int64_t average_rows);
WindowShape window_shape_d256(int64_t average_rows, int64_t per_cu);
void launch_window_d64(const WindowParams& p, const WindowShape& shape, bool bf16, hipStream_t s);
void launch_window_d128(const WindowParams& p, const WindowShape& shape, bool bf16, hipStream_t s);
void launch_window_d256(const WindowParams& p, const WindowShape& shape, bool bf16, hipStream_t s);

namespace {

typedef __bf16 win_bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 win_f16x8 __attribute__((ext_vector_type(8)));
typedef float win_f32x16 __attribute__((ext_vector_type(16)));
typedef float win_f32x4 __attribute__((ext_vector_type(4)));
typedef int32_t win_i32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t win_u32x4u __attribute__((ext_vector_type(4), aligned(4)));   // at any element
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
          static_cast<int64_t>(q.first_row) + q.nodes > next || q.bias < 0 || q.bias > p.bias_elems - square ||
          static_cast<int64_t>(q.prefix) + q.nodes > kWinMaxKeys;
    if (!bad) q.blocks = (q.nodes * p.groups + ROWS - 1) / ROWS;   // nodes * groups <= Q * heads < 2^31
    return q;
}

// A row block: its request, its place among the request's blocks, the parts that its keys are cut into, the first
// part's number among those of all blocks, and the part that was asked for.
struct WinBlock {
    int32_t r, b, parts, first, split;
    WinRequest req;
};

// Sum over the wave's lanes, in all of them.
__device__ __forceinline__ int32_t win_wave_sum(int32_t v) {
    v += __builtin_amdgcn_mov_dpp(v, 0xB1, 0xf, 0xf, false);    // quad_perm [1, 0, 3, 2]
    v += __builtin_amdgcn_mov_dpp(v, 0x4E, 0xf, 0xf, false);    // quad_perm [2, 3, 0, 1]
    v += __builtin_amdgcn_mov_dpp(v, 0x141, 0xf, 0xf, false);   // half row mirrored
    v += __builtin_amdgcn_mov_dpp(v, 0x140, 0xf, 0xf, false);   // row mirrored
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = static_cast<int32_t>(r[0] + r[1]);
    const auto h = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return static_cast<int32_t>(h[0] + h[1]);
}

// Inclusive sums over the wave's lanes: within rows of 16, then from row to row.
template <int CTRL, int ROW_MASK>
__device__ __forceinline__ int32_t win_shifted(int32_t v) {
    return __builtin_amdgcn_update_dpp(0, v, CTRL, ROW_MASK, 0xf, false);
}
__device__ __forceinline__ int32_t win_wave_scan(int32_t v) {
    v += win_shifted<0x111, 0xf>(v);   // row_shr by 1, 2, 4, 8
    v += win_shifted<0x112, 0xf>(v);
    v += win_shifted<0x114, 0xf>(v);
    v += win_shifted<0x118, 0xf>(v);
    v += win_shifted<0x142, 0xa>(v);   // lane 15 of the row before to rows 1 and 3
    v += win_shifted<0x143, 0xc>(v);   // lane 31 to rows 2 and 3
    return v;
}

// Parts that a request's row blocks are cut into, a lane per request: one each, and the workgroups that are left
// over by their keys, but no part shorter than the least.  All in integers: the merge has to find the same.
constexpr int32_t kMostSplits = 64;
template <int ROWS, int SK>
__device__ __forceinline__ int32_t win_parts(const WindowParams& p, const WinRequest& q) {
    if (p.splits == 1) return 1;
    // Keys of a block, about: all that there are, or what its window spans and its own nodes.
    const int64_t own = q.nodes < ROWS ? q.nodes : ROWS, all = static_cast<int64_t>(q.prefix) + q.nodes;
    const int64_t most = static_cast<int64_t>(p.window) + p.sinks + own, keys = all < most ? all : most;
    const int32_t steps = keys < (SK << 14) ? static_cast<int32_t>(keys + SK - 1) / SK : 1 << 14;   // sums stay below 2^31
    const int32_t total = win_wave_sum(q.blocks * steps), left = p.units - win_wave_sum(q.blocks);
    int32_t parts = total > 0 && left > 0 ? static_cast<int32_t>(static_cast<uint32_t>(steps) * left / total) + 1 : 1;
    const int32_t limit = p.least_steps == 1 ? steps : steps / p.least_steps;
    parts = parts < limit ? parts : limit;
    parts = parts < kMostSplits ? parts : kMostSplits;
    return parts > 1 ? parts : 1;
}

// Finds part `unit` (BY_PART) of the batch's row blocks, or their block number `unit`: blocks of a request and requests
// follow each other; false if there is none.  All threads of the workgroup call it; `scratch` is LDS of its own, 3 +
// a word a wave.
template <int ROWS, int SK, int THREADS, bool BY_PART>
__device__ __forceinline__ bool win_find(const WindowParams& p, int32_t* scratch, WinBlock& block, int unit) {
    constexpr int WAVES = THREADS / 64;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    // The last workgroup of a launch reports what is wrong with the requests.
    const bool report = blockIdx.x + 1 == gridDim.x;
    bool bad;
    if (p.num_requests <= 64) {
        // A lane per request, in every wave by itself.
        WinRequest q = {};
        if (lane < p.num_requests) {
            q = win_request<ROWS>(p, lane, bad);
            if (bad && report) set_status(p.status, TV_STATUS_BAD_REQUEST);
        }
        const int32_t parts = win_parts<ROWS, SK>(p, q), mine = q.blocks * parts, end = win_wave_scan(mine);
        const int32_t found = BY_PART || p.splits == 1 ? end : win_wave_scan(q.blocks);
        const uint64_t behind = __ballot(found > unit);
        if (behind == 0) return false;
        const int r = __ffsll(static_cast<unsigned long long>(behind)) - 1;
        block.r = r;
        block.parts = __builtin_amdgcn_readlane(parts, r);
        const int32_t first = __builtin_amdgcn_readlane(end - mine, r);
        if constexpr (BY_PART) {
            block.b = (unit - first) / block.parts;
            block.split = unit - first - block.b * block.parts;
        } else {
            block.b = unit - __builtin_amdgcn_readlane(found - q.blocks, r);
            block.split = 0;
        }
        block.first = first + block.b * block.parts;
        // Requests that overlap can have more blocks than rows have.
        if (block.first + block.parts > p.units) return false;
        block.req.prefix = __builtin_amdgcn_readlane(q.prefix, r);
        block.req.nodes = __builtin_amdgcn_readlane(q.nodes, r);
        block.req.first_row = __builtin_amdgcn_readlane(q.first_row, r);
        block.req.blocks = __builtin_amdgcn_readlane(q.blocks, r);
        block.req.bias = static_cast<int64_t>(__builtin_amdgcn_readlane(static_cast<int32_t>(q.bias >> 32), r)) << 32 |
                         static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int32_t>(q.bias), r));
        return true;
    }
    const int per = (p.num_requests + THREADS - 1) / THREADS;
    const int r0 = tid * per, r1 = r0 + per < p.num_requests ? r0 + per : p.num_requests;
    int32_t mine = 0;   // the sum is at most block_ids
    for (int i = r0; i < r1; ++i) {
        mine += win_request<ROWS>(p, i, bad).blocks;
        if (bad && report) set_status(p.status, TV_STATUS_BAD_REQUEST);
    }
    int32_t end = win_wave_scan(mine);
    if (lane == 63) scratch[3 + wave] = end;
    if (tid == 0) scratch[0] = -1;
    __syncthreads();
    int32_t total = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        if (w < wave) end += scratch[3 + w];
        total += scratch[3 + w];
    }
    const int id = BY_PART ? unit / p.splits : unit;
    if (id >= __builtin_amdgcn_readfirstlane(total)) return false;   // the same in every thread
    if (end - mine <= id && id < end) {   // this thread's requests hold it
        int32_t first = end - mine;
        for (int i = r0; i < r1; ++i) {
            const int32_t next = first + win_request<ROWS>(p, i, bad).blocks;
            if (id < next) {
                scratch[0] = i;
                scratch[1] = id - first;
                break;
            }
            first = next;
        }
    }
    __syncthreads();
    block.r = __builtin_amdgcn_readfirstlane(scratch[0]);
    if (block.r < 0) return false;   // requests that overlap can have more blocks than are counted
    block.b = __builtin_amdgcn_readfirstlane(scratch[1]);
    block.req = win_request<ROWS>(p, block.r, bad);
    block.parts = p.splits;
    block.first = id * p.splits;
    block.split = unit - (BY_PART ? block.first : unit);
    // Requests that overlap by the ten thousands wrap the sums, and two threads can have found a block, one of which wrote
    // the request and the other the number.
    return static_cast<uint32_t>(block.b) < static_cast<uint32_t>(block.req.blocks);
}

// Position i as it is given, in 32 bits: one that they do not hold is as far outside as they say.
__device__ __forceinline__ int32_t win_given(const int32_t* positions, int32_t step, int64_t i) {
    const int32_t low = positions[i * step], high = positions[i * step + step - 1];   // step 1: the same word
    if (step == 1 || high == low >> 31) return low;
    return high < 0 ? -0x7fffffff - 1 : 0x7fffffff;
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
    typedef __bf16 pair __attribute__((ext_vector_type(2)));
    static __device__ __forceinline__ float add_pair(__bf16 a, __bf16 b, float sum) {
        const pair x = {a, b}, one = {static_cast<__bf16>(1.0f), static_cast<__bf16>(1.0f)};
        return __builtin_amdgcn_fdot2_f32_bf16(x, one, sum, false);
    }
    static __device__ __forceinline__ win_f32x16 run(vec a, vec b, win_f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
};
template <>
struct WinType<_Float16> {
    typedef win_f16x8 vec;
    static constexpr uint32_t kExponent = 0x7c007c00u, kStep = 0x04000400u;
    static constexpr float kShift = 7.0f;
    typedef _Float16 pair __attribute__((ext_vector_type(2)));
    static __device__ __forceinline__ float add_pair(_Float16 a, _Float16 b, float sum) {
        const pair x = {a, b}, one = {static_cast<_Float16>(1.0f), static_cast<_Float16>(1.0f)};
        return __builtin_amdgcn_fdot2(x, one, sum, false);
    }
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

// f(0), f(1), ... with the numbers as types.
template <int FROM, int TO, class F>
__device__ __forceinline__ void win_each(F& f) {
    if constexpr (FROM < TO) {
        f(std::integral_constant<int, FROM>());
        win_each<FROM + 1, TO>(f);
    }
}

constexpr int kAhead = 4;      // products between an operand's read and its use

// s_waitcnt immediates: vector memory operations down to n with nothing else, LDS operations down to none.
template <int N>
__device__ __forceinline__ void win_wait_loads() {
    static_assert(N >= 0 && N < 64, "vmcnt range");
    __builtin_amdgcn_s_waitcnt((N & 0xF) | ((N >> 4) << 14) | (0x7 << 4) | (0xF << 8));
}
// A workgroup barrier behind the wave's own LDS operations that leaves its loads under way.
__device__ __forceinline__ void win_barrier() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}
// 16 bytes a lane from memory to LDS at `lds_addr` + 16 * lane.  Issued from inline asm so that the compiler does not
// wait for it before every later LDS read; win_wait_loads and a barrier order it.  M0 has no other use in these
// kernels, which build.py checks in their assembly.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void win_dma(const void* src, uint32_t lds_addr) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
                 :
                 : "s"(lds_addr), "v"(src)
                 : "memory", "m0");
}
#pragma clang diagnostic pop

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
    constexpr int AHEAD = WK == 1 ? 3 : NBUF;      // steps between a step's loads and its products
    constexpr int KT = WM == 8 ? 512 : 256;   // keys of a table
    constexpr int TSTEPS = KT / SK;                // steps of a table
    constexpr int KBYTES = KT / 8, KTILES = KT / kWinTile;
    constexpr int NODES = ROWS < 128 ? ROWS : 128;       // at most, of a block: 256 rows have two heads a node or more
    static_assert(SK % KPP == 0 && SK % (kWinTile * WK) == 0, "a step is whole passes and tiles");
    static_assert(TSTEPS > AHEAD, "a table is read no longer when the next but one is made");
    static_assert(WK == 1 || WK * 32 * D * 4 <= NBUF * 2 * KB, "the waves' results share the staging memory");
    typedef typename WinType<T>::vec V8;

    __shared__ __attribute__((aligned(1024))) char lds[NBUF * 2 * KB];
    // Of the keys of two tables, page and place in it; of those of the last one made, the last position that sees
    // the key, -1 if it is not there.
    __shared__ __attribute__((aligned(16))) u32x2 tab_at[2][KT];
    __shared__ __attribute__((aligned(16))) int32_t tab_reach[KT];
    // Which keys a node sees, a bit each; of a tile whether some node does not see all of it (kHides; kWhole: by
    // looking, 0: without), and whether there is a bias that is neither zero nor -inf.
    __shared__ __attribute__((aligned(16))) uint8_t tab_bits[2][NODES][KBYTES];
    __shared__ __attribute__((aligned(4))) uint8_t tab_hides[2][KTILES], tab_other[2][KTILES];
    __shared__ int32_t node_pos[NODES];
    constexpr uint8_t kHides = 1, kWhole = 2;
    __shared__ float2 lds_ml[WK > 1 ? WM * WK : 1][32];
    __shared__ int32_t lds_find[3 + THREADS / 64];

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave % WM, wk = wave / WM;
    const int c = lane & 31, half = lane >> 5;

    // --- the row block and its keys -------------------------------------------------------------
    // Heads fastest: workgroups are dealt to the 8 XCDs in turn, so of 8 KV heads each has one, whose row blocks share its L2.  Runs of
    // whole requests on an XCD gained nothing (64 trees over windows of 8192: 881 us and 889), and lose balance (8 ragged
    // requests: 116 us and 75).
    WinBlock block;
    const int unit = blockIdx.x / p.num_kv_heads, head = blockIdx.x - unit * p.num_kv_heads;
    if (!win_find<ROWS, SK, THREADS, true>(p, lds_find, block, unit)) return;
    const int r = block.r, b = block.b;
    const WinRequest req = block.req;
    const int rows_all = req.nodes * p.groups;
    const int node0 = b * ROWS / p.groups;
    const int node1 = (b * ROWS + ROWS < rows_all ? b * ROWS + ROWS - 1 : rows_all - 1) / p.groups;   // the last
    const int32_t* positions = p.positions + static_cast<int64_t>(req.first_row) * p.pos_step;
    int32_t lowest = 0x7fffffff, highest = 0;
    for (int n = node0 + lane; n <= node1; n += 64) {
        const int32_t given = win_given(positions, p.pos_step, n);
        const int32_t at = win_position(req, n, given);
        if (at != given) set_status(p.status, TV_STATUS_BAD_POSITION);
        node_pos[n - node0] = at;   // by every wave, the same
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
    const int split = block.split, part = steps / block.parts, longer = steps - part * block.parts;   // the first have a step more
    const int run0 = split * part + (split < longer ? split : longer);
    const int run1 = run0 + part + (split < longer ? 1 : 0);
    const int64_t piece = static_cast<int64_t>(block.first) * p.num_kv_heads + head * block.parts + split;
    if (run0 >= run1) {   // fewer steps than workgroups
        for (int i = tid; i < ROWS; i += THREADS) p.ws_ml[piece * ROWS + i] = make_float2(-INFINITY, 0.0f);
        return;
    }
    const int32_t* table = p.tables + r * p.t_s0;
    const int64_t* slots = p.tree_slots + req.first_row;
    const char* k_head = p.k + head * p.k_s2;
    const char* v_head = p.v + head * p.v_s2;

    // Parameters that the steps do not need are read where they are used: held over the loop, with the others,
    // they would not fit the scalar registers.
    typedef const __attribute__((address_space(4))) WindowParams* Params;
    auto cold = [&]() {
        Params a = (Params)__builtin_amdgcn_kernarg_segment_ptr();
        asm volatile("" : "+s"(a));
        return a;
    };

    // --- the tables: keys [run0 * SK + t * KT, ...), a thread a key -------------------------------
    auto table_keys = [&](int t) {
        const int keys = (run1 - run0) * SK - t * KT;
        return keys < KT ? keys : KT;
    };
    auto make_keys = [&](int t) {
        const Params a = cold();
        const int keys = table_keys(t);
#pragma unroll 1
        for (int kk = tid; kk < keys; kk += THREADS) {
            const int v = run0 * SK + t * KT + kk;
            const bool live = v < n_keys, tree = v >= n_prefix;
            const int of = live ? v : n_keys - 1, t_of = of - n_prefix + t0;   // a key that is there
            const bool slot = of >= n_prefix;
            const int32_t pos = of < n_first ? of : of - n_first + w0;
            int32_t page = win_page_of(a->div_mul, a->div_shift, slot ? 0 : pos);
            const int32_t* from = slot ? reinterpret_cast<const int32_t*>(slots + t_of) : table + page;
            const int32_t entry = from[0], entry_high = from[slot ? 1 : 0];
            const int32_t given = win_given(positions, a->pos_step, slot ? t_of : 0);
            uint32_t offset = static_cast<uint32_t>(pos - page * a->block_size);
            if (slot) {
                page = win_page_of(a->div_mul, a->div_shift, entry < 0 ? 0 : entry);
                offset = static_cast<uint32_t>(entry - page * a->block_size);
                if (entry < 0 || entry_high != 0) page = -1;
            } else {
                page = entry;
            }
            const bool there = page >= 0 && page < a->num_blocks, found = live && there;
            if (live && !there) set_status(a->status, TV_STATUS_BAD_PAGE);
            // Every lane loads: a key that is not there from the pool's first row.
            tab_at[t & 1][kk] = found ? u32x2{static_cast<uint32_t>(page), offset} : u32x2{0, 0};
            const int32_t at = tree ? win_position(req, t_of, given) : pos;
            const int64_t until = at < a->sinks ? 0x7fffffff : static_cast<int64_t>(at) + a->window - 1;
            tab_reach[kk] = !found ? -1 : until < 0x7fffffff ? static_cast<int32_t>(until) : 0x7fffffff;
            const uint64_t clear = __ballot(found && !tree && (pos < a->sinks || pos >= from_high));
            if ((lane & 31) == 0) {
                tab_hides[t & 1][kk / kWinTile] = static_cast<uint32_t>(clear >> lane) == 0xffffffffu ? 0 : kWhole;
                tab_other[t & 1][kk / kWinTile] = 0;
            }
        }
        win_wait_loads<0>();   // said here, or the compiler says it in every step, for registers that could be loaded yet
    };
    // Behind a barrier: the bits of the tiles that are not clear, eight keys of a node a thread.  A chain's tiles below the
    // diagonal turn out whole.  The biases are read once here, coalesced, and not by every row in the steps, where
    // waiting for them would wait for the keys under way too.
    auto make_bits = [&](int t, auto at_once) {
        const Params a = cold();
        const int bytes = table_keys(t) / 8, nodes = node1 - node0 + 1;
        const int my_tile = lane < bytes / (kWinTile / 8) ? lane : 0;
        if (!__any(tab_hides[t & 1][my_tile] != 0)) return;   // all clear, as most tables of a long window
        const int v_table = run0 * SK + t * KT;
        const bool trees = v_table + 8 * bytes > n_prefix, few = a->bias_elems < 8;
        const float* biases = a->bias + req.bias + static_cast<int64_t>(node0) * req.nodes + (v_table - n_prefix + t0);
        const float* last = a->bias + a->bias_elems - 8;   // eight can be read from here
        constexpr int AT_ONCE = decltype(at_once)::value;   // places whose loads are under way
#pragma unroll 1
        for (int e0 = tid; e0 < nodes * KBYTES; e0 += AT_ONCE * THREADS) {
            win_u32x4u b[AT_ONCE][2];
            if (trees) {
#pragma unroll
                for (int q = 0; q < AT_ONCE; ++q) {
                    const int e = e0 + q * THREADS, n = e / KBYTES, byte = e % KBYTES;
                    const float* from = biases + (static_cast<int64_t>(n) * req.nodes + 8 * byte);
                    const bool inside = n < nodes && byte < bytes && from >= a->bias && from <= last;
                    from = few ? biases : inside ? from : a->bias;
                    if (!few) {
                        b[q][0] = *reinterpret_cast<const win_u32x4u*>(from);
                        b[q][1] = *reinterpret_cast<const win_u32x4u*>(from + 4);
                    }
                }
            }
#pragma unroll
            for (int q = 0; q < AT_ONCE; ++q) {
                const int e = e0 + q * THREADS, n = e / KBYTES, byte = e % KBYTES, tile = byte / (kWinTile / 8);
                if (n >= nodes || byte >= bytes || tab_hides[t & 1][tile] == 0) continue;
                const win_i32x4 *reach = reinterpret_cast<const win_i32x4*>(&tab_reach[8 * byte]), low = reach[0], high = reach[1];
                const int32_t pos = node_pos[n];
                uint32_t near = 0, other = 0;
#pragma unroll
                for (int i = 0; i < 8; ++i) near |= pos <= (i < 4 ? low[i % 4] : high[i % 4]) ? 1u << i : 0u;
                const int first = v_table + 8 * byte - n_prefix, node = node0 + n;   // below 0: prefix keys
                if (first + 8 > 0) {
                    const float* from = biases + (static_cast<int64_t>(n) * req.nodes + 8 * byte);
                    const bool inside = !few && from >= a->bias && from <= last;
                    if (!inside) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const int of = first + t0 + i;
                            b[q][i / 4][i % 4] = __float_as_uint(from[of < t0 ? i + t0 - of : of < node ? i : i + node - of]);
                        }
                    }
                    uint32_t hidden = 0;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const uint32_t bias = b[q][i / 4][i % 4], tree = first + i >= 0 ? 1u << i : 0u;
                        hidden |= first + t0 + i > node || bias == 0xff800000u ? tree : 0u;
                        other |= bias << 1 ? tree : 0u;
                    }
                    near &= ~hidden;
                    other &= near;
                }
                tab_bits[t & 1][n][byte] = static_cast<uint8_t>(near);
                if (near != 0xff || other) tab_hides[t & 1][tile] = kHides;
                if (other) tab_other[t & 1][tile] = 1;
            }
        }
        win_wait_loads<0>();
    };
    // Which tiles of step j some node does not see all of, a byte a tile.
    auto hiding_tiles = [&](int j) {
        const uint8_t* at = &tab_hides[j / TSTEPS & 1][j % TSTEPS * (SK / kWinTile)];
        uint32_t flags;
        if constexpr (SK / kWinTile == 1) flags = *at;
        else if constexpr (SK / kWinTile == 2) flags = *reinterpret_cast<const uint16_t*>(at);
        else flags = *reinterpret_cast<const uint32_t*>(at);
        return static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(flags)) & 0x01010101u * kHides;
    };

    // --- moving a step's keys -------------------------------------------------------------------
    // Lane l of a load fills place l % LPR of a row, which holds the chunk that the swizzle puts there.
    const int my_key = tid / LPR, my_place = tid % LPR;
    const uint32_t lds_base = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(reinterpret_cast<uintptr_t>(lds))) + wave * (64 / LPR) * 2 * D;
    auto k_chunk = [&](int n) { return win_k_chunk<D>(my_key + n * KPP, my_place); };
    auto v_chunk = [&](int n) { return win_v_chunk<D>(my_key + n * KPP, my_place); };
    auto issue = [&](int j) {
        const uint32_t to = lds_base + j % NBUF * (2 * KB);
        const u32x2* at = &tab_at[j / TSTEPS & 1][j % TSTEPS * SK + my_key];
#pragma unroll
        for (int n = 0; n < PASSES; ++n) {
            const u32x2 e = at[n * KPP];
            int kc = k_chunk(n), vc = v_chunk(n);
            if (p.dim != D) {   // places behind the head's end: the first chunk, which mend() drops
                kc = kc * 8 < p.dim ? kc : 0;
                vc = vc * 8 < p.dim ? vc : 0;
            }
            const uint64_t row = static_cast<uint64_t>(e[0]) * p.k_s0 + static_cast<uint64_t>(e[1]) * p.k_s1;
            uint64_t v_row = row;
            if (!p.same) {
                const Params a = cold();
                v_row = static_cast<uint64_t>(e[0]) * a->v_s0 + static_cast<uint64_t>(e[1]) * a->v_s1;
            }
            win_dma(k_head + row + 16 * kc, to + n * KPP * 2 * D);
            win_dma(v_head + v_row + 16 * vc, to + KB + n * KPP * 2 * D);
        }
    };
    // Rows that do not see a key have to get zero from its V row, and zero times NaN or infinity is not.  So where some
    // node does not see all of a step, each thread, behind its own loads, makes zeros of such elements, and the key's
    // scores NaN instead, which hidden scores never show.  It also clears what lies behind a head's end, in every step of a
    // head size between the templates': 64 trees of 8 nodes over 4096 keys and 8 KV heads of 64 / 72 / 96 / 120 / 128 / 136 /
    // 192 / 248 / 256 take 114 / 192 / 199 / 229 / 200 / 456 / 483 / 508 / 389 us.
    auto mend = [&](int j) {
        const bool whole = p.dim == D;
        if (hiding_tiles(j) == 0 && whole) return;
        char* kb = lds + j % NBUF * (2 * KB) + my_key * 2 * D + 16 * my_place;
        char* vb = kb + KB;
#pragma unroll
        for (int n = 0; n < PASSES; ++n) {
            const int at = n * KPP * 2 * D;
            u32x4 x = *reinterpret_cast<const u32x4*>(vb + at);
            uint32_t odd = 0;
#pragma unroll
            for (int w = 0; w < 4; ++w) odd |= ((x[w] & WinType<T>::kExponent) + WinType<T>::kStep) & 0x80008000u;
            const bool behind = !whole && v_chunk(n) * 8 >= p.dim;
            const uint64_t lanes = __ballot(odd != 0 && !behind);
            if (odd != 0 || behind) {
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const uint32_t high = ((x[w] & WinType<T>::kExponent) + WinType<T>::kStep) & 0x80008000u;
                    x[w] = behind ? 0 : x[w] & ~((high >> 15) * 0xffffu);
                }
                *reinterpret_cast<u32x4*>(vb + at) = x;
            }
            const bool poison = (lanes >> (lane & ~(LPR - 1))) & ((1ull << LPR) - 1);
            if (poison || (!whole && k_chunk(n) * 8 >= p.dim)) {
                const uint32_t word = poison ? 0x7fff7fffu : 0;
                *reinterpret_cast<u32x4*>(kb + at) = u32x4{word, word, word, word};
            }
        }
    };
    const int k_get = c * 2 * D + 16 * win_k_chunk<D>(c, half);
    const int v_key = 4 * half + ((lane & 15) >> 2), v_dim = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
    const int v_get = v_key * 2 * D + 16 * win_v_chunk<D>(v_key, v_dim >> 3) + 2 * (v_dim & 7);

    // --- the rows -------------------------------------------------------------------------------
    const int row = b * ROWS + 32 * wm + c;
    const bool wave_rows = b * ROWS + 32 * wm < rows_all;   // any row of this wave
    const int node = row < rows_all ? row / p.groups : -1;  // -1: no row
    const int qhead = head * p.groups + row - (node < 0 ? 0 : node) * p.groups;
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

    // Products of tile t of step j to scores in units of log2; those that the row does not see become -inf,
    // whatever they are.
    const int my_node = node < 0 ? 0 : node - node0;
    auto mask = [&](int j, int t, win_f32x16& x) {
        const int tile = j % TSTEPS * (SK / kWinTile) + t;
        const uint32_t bits = *reinterpret_cast<const uint32_t*>(&tab_bits[j / TSTEPS & 1][my_node][4 * tile]) >> (4 * half);
        if (!__builtin_amdgcn_readfirstlane(tab_other[j / TSTEPS & 1][tile])) {
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = bits & (1u << (8 * (i >> 2) + (i & 3))) ? x[i] * p.c : -INFINITY;
            return;
        }
        const Params a = cold();
        const float* bias = a->bias + req.bias + static_cast<int64_t>(node < 0 ? 0 : node) * req.nodes;
        const int of0 = (run0 + j) * SK + t * kWinTile - n_prefix + t0 + 4 * half;   // the node of element 0
        const int last = node < 0 ? 0 : node;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            __builtin_amdgcn_sched_barrier(0);   // four biases in registers at a time
            float b[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int of = of0 + 8 * g + e;
                b[e] = bias[of < 0 ? 0 : of < last ? of : last];
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int i = 4 * g + e;
                float add = b[e] * 1.44269504088896340736f;   // a finite bias stays finite
                if (fabsf(add) == INFINITY) add = copysignf(FLT_MAX, add);
                x[i] = bits & (1u << (8 * g + e)) ? fmaf(x[i], a->c, of0 + 8 * g + e < t0 ? 0.0f : add) : -INFINITY;
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        win_wait_loads<0>();
    };
    // The factor that is left to the scores.
    auto hide = [&](uint32_t hiding, int j, int t, win_f32x16& x) {
        if (!((hiding >> (8 * t)) & kHides)) return p.c;
        mask(j, t, x);
        return 1.0f;
    };
    V8 pb[TERMS][2];
    // The sum is of the probabilities as they are multiplied.
    auto exponentials = [&](const win_f32x16& x, float cs, float negative) {
        float sum[2] = {0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
            float a = __builtin_amdgcn_exp2f(fmaf(x[i], cs, negative)), b = __builtin_amdgcn_exp2f(fmaf(x[i + 1], cs, negative));
            if constexpr (TERMS > 1) sum[(i >> 1) & 1] += a + b;
#pragma unroll
            for (int q = 0; q < TERMS; ++q) {
                const T a1 = static_cast<T>(a), b1 = static_cast<T>(b);
                pb[q][i >> 3][i & 7] = a1;
                pb[q][i >> 3][(i & 7) + 1] = b1;
                if constexpr (TERMS == 1) sum[(i >> 1) & 1] = WinType<T>::add_pair(a1, b1, sum[(i >> 1) & 1]);
                if (q + 1 < TERMS) {
                    a -= static_cast<float>(a1);
                    b -= static_cast<float>(b1);
                }
            }
        }
        return sum[0] + sum[1];
    };
    // Probabilities against the row's reference, which is near the largest score seen: it is raised only when
    // a tile's would pass 2^8, until when they cost no precision.
    auto reference = [&]() { return m == -INFINITY ? 0.0f : kShift - m; };
    auto raise = [&](const win_f32x16& x, float cs, float& tile_sum) {
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
            // In the same order as before: a row whose neighbours raise their reference is summed a second time.
            tile_sum = exponentials(x, cs, reference());
        }
        l += tile_sum;
    };
    // The matrix products of a tile step in a fixed order: K . Q^T of a tile (LDS at `kb`) into x, of which element i is
    // key 8*(i/4) + 4*half + i%4, and V^T . P^T of another (at `vb`), in turn, each with its operands read from LDS
    // kAhead products before.  `first` runs while the first operands are read.
    auto multiply = [&](auto with_keys, const char* kb, win_f32x16& x, auto with_values, const char* vb, auto first) {
        constexpr bool KEYS = decltype(with_keys)::value, VALUES = decltype(with_values)::value;
        constexpr int NV = 2 * NB, SLOTS = (KEYS ? NK : 0) + (VALUES ? NV : 0);
        static_assert(NK == NV, "as many products of either kind");
        u32x4 operand[SLOTS];
        auto read = [&](auto slot) {
            constexpr int S = decltype(slot)::value;
            if constexpr (S < SLOTS) {
                constexpr bool KEY = KEYS && (!VALUES || S % 2 == 0);
                constexpr int N = KEYS && VALUES ? S / 2 : S;
                if constexpr (KEY) {
                    operand[S] = *reinterpret_cast<const u32x4*>(kb + (k_get ^ (32 * N)));
                } else {
                    const char* lo = vb + 16 * (N / NB) * 2 * D + (v_get ^ (64 * (N % NB)));
                    const win_i16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((win_lds_i16x4*)lo);
                    const win_i16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((win_lds_i16x4*)(lo + 8 * 2 * D));
                    operand[S] = __builtin_bit_cast(u32x4, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
                }
            }
        };
        auto product = [&](auto slot) {
            constexpr int S = decltype(slot)::value;
            constexpr bool KEY = KEYS && (!VALUES || S % 2 == 0);
            constexpr int N = KEYS && VALUES ? S / 2 : S;
            read(std::integral_constant<int, S + kAhead>());
            const V8 a = __builtin_bit_cast(V8, operand[S]);
            if constexpr (KEY) {
                x = WinType<T>::run(a, qb[N], x);
            } else {
#pragma unroll
                for (int q = 0; q < TERMS; ++q) acc[N % NB] = WinType<T>::run(a, pb[q][N / NB], acc[N % NB]);
            }
            __builtin_amdgcn_sched_barrier(0);
        };
        win_each<0, kAhead>(read);
        __builtin_amdgcn_sched_barrier(0);
        first();
        if constexpr (KEYS) x = win_f32x16{};
        __builtin_amdgcn_sched_barrier(0);
        win_each<0, SLOTS>(product);
    };
    constexpr std::true_type yes;
    constexpr std::false_type no;
    auto nothing = []() {};

    // --- the steps ------------------------------------------------------------------------------
    const int todo = run1 - run0;
    make_keys(0);
    win_barrier();
    // The table of the steps that are loaded from the next one on, and a step later its bits.
    auto next_table = [&](int j) {
        const int of = j + AHEAD;
        if ((of + 1) % TSTEPS == 0 && of + 1 < todo) make_keys((of + 1) / TSTEPS);
        if (of % TSTEPS == 0 && of < todo) make_bits(of / TSTEPS, std::integral_constant<int, 2>());   // beside the results' registers
    };
    // Biases of the first table are waited for with the first step's keys.
    issue(0);
    make_bits(0, std::integral_constant<int, 8>());
    if constexpr (WK > 1) {
#pragma unroll
        for (int j = 1; j < NBUF; ++j) {
            if (j < todo) issue(j);
        }
        win_barrier();
#pragma unroll 1
        for (int j = 0; j < todo; ++j) {
            if (j + NBUF <= todo) win_wait_loads<(NBUF - 1) * 2 * PASSES>();
            else win_wait_loads<0>();
            mend(j);
            win_barrier();
            if (wave_rows) {
                const uint32_t hiding = hiding_tiles(j);
                const char* kb = lds + j % NBUF * (2 * KB) + wk * kWinTile * 2 * D;
                const int left = n_keys - (run0 + j) * SK, tiles = (left < SK ? left + kWinTile - 1 : SK) / kWinTile;
#pragma unroll
                for (int n = 0; n < TILES; ++n) {
                    const int t = n * WK + wk;
                    if (t >= tiles) break;
                    const char* at = kb + n * WK * kWinTile * 2 * D;
                    win_f32x16 x;
                    multiply(yes, at, x, no, nullptr, nothing);
                    const float cs = hide(hiding, j, t, x);
                    multiply(no, nullptr, x, yes, at + KB, [&]() {
                        float tile_sum = exponentials(x, cs, reference());
                        raise(x, cs, tile_sum);
                    });
                }
            }
            next_table(j);
            win_barrier();   // the step's reads of its buffer are done
            if (j + NBUF < todo) issue(j + NBUF);
        }
    } else {
        // Four buffers: this step's, the next one's, whose first scores are multiplied with this one's last values, and
        // two on their way.
        static_assert(NBUF == 4, "a step is loaded into the buffer of the one before");
        const int total = ((run1 * SK < n_keys ? run1 * SK : n_keys) - run0 * SK + kWinTile - 1) / kWinTile;   // tiles
        if (1 < todo) issue(1);
        if (2 < todo) issue(2);
        win_barrier();
        if (2 < todo) win_wait_loads<2 * PASSES>();
        else win_wait_loads<0>();
        mend(0);
        if (1 < todo) mend(1);
        win_barrier();
        win_f32x16 x;
        if (wave_rows) multiply(yes, lds, x, no, nullptr, nothing);
#pragma unroll 1
        for (int j = 0; j < todo; ++j) {
            const uint32_t hiding = hiding_tiles(j);
            if (j + 3 < todo) issue(j + 3);
            if (wave_rows) {
                const char* at = lds + j % NBUF * (2 * KB);
                const char* next = lds + (j + 1) % NBUF * (2 * KB);
#pragma unroll
                for (int t = 0; t < TILES; ++t) {
                    if (j * TILES + t >= total) break;
                    const float cs = hide(hiding, j, t, x);
                    // Past the last tile the scores are of what the buffer holds, and not used.
                    multiply(yes, t + 1 < TILES ? at + (t + 1) * kWinTile * 2 * D : next, x, yes, at + t * kWinTile * 2 * D + KB, [&]() {
                        float tile_sum = exponentials(x, cs, reference());
                        raise(x, cs, tile_sum);
                    });
                }
            }
            if (j + 3 < todo) win_wait_loads<2 * PASSES>();
            else win_wait_loads<0>();
            if (j + 2 < todo) mend(j + 2);
            next_table(j);
            win_barrier();
        }
    }

    // --- the result: the row's output, or its unnormalised sum with (m, l) for the merge ---------
    const bool whole = block.parts == 1;
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
    const dim3 grid(static_cast<uint32_t>(p.units) * p.num_kv_heads), block(64 * WM * WK);
    if (bf16 && !p.out_f32) hipLaunchKernelGGL((window_attention_kernel<D, WM, WK, SK, NBUF, __bf16, 1>), grid, block, 0, s, p);
    else if (bf16) hipLaunchKernelGGL((window_attention_kernel<D, WM, WK, SK, NBUF, __bf16, 3>), grid, block, 0, s, p);
    else if (!p.out_f32) hipLaunchKernelGGL((window_attention_kernel<D, WM, WK, SK, NBUF, _Float16, 1>), grid, block, 0, s, p);
    else hipLaunchKernelGGL((window_attention_kernel<D, WM, WK, SK, NBUF, _Float16, 2>), grid, block, 0, s, p);
}

}  // namespace
}  // namespace tv
