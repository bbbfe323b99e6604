// Tree attention over an e4m3 cache: the kernel template and what its translation units share
// (tv_attention_e4m3_d<D>.hip instantiate it per head size; tv_attention_e4m3.hip holds the entry
// and the merge).
//
// Row r = (node, query head) of a request, key k, codes K8, V8 with scales ks, vs per key and head:
//     s_rk = scale * ks_k * (q_r . K8_k) + bias_rk,     o_r = sum_k p_rk vs_k V8_k / sum_k p_rk,
//     p_rk = 2^((s_rk - m_r) log2 e)
// over the request's prefix keys (through its block table) and the tree nodes its bias shows it.
// An e4m3 code is a bf16 and an f16 value exactly, so both products run on the matrix cores at
// operand precision with fp32 sums: 32x32x16 MFMAs, K . Q^T in the queries' type and V^T . P^T in
// bf16, where p * vs is rounded once or kept in TERMS bf16 terms (2: to 2^-17, 3: to 2^-26).  The scales never touch
// the codes: ks multiplies a score, vs a probability, one multiplication each.
//
// Work.  A step is SK keys of one row block (ROWS score rows of one request and KV head), prefix
// keys and tree nodes in separate steps; a block's steps are contiguous, blocks of a head, heads of
// a request and requests follow each other.  The launch has a fixed number of workgroups, each of
// which takes an equal, contiguous share of all steps, computed from the live lengths: no plan, no
// host copies, the same launch for every batch of a shape, and no tail.  A block that one workgroup
// covers is written at once; the pieces of the others go to the workspace and a second launch joins
// them (at most two pieces a workgroup).
//
// A step.  Every wave moves its share of the keys' codes from memory to registers one step ahead
// (and the page numbers two ahead), turns them into bf16/f16 and writes them to LDS, K and V as
// [key][dim] with the 16-byte chunks swizzled per key: converting once per workgroup costs an eighth
// of what every wave converting its own operands would.  Wave (wm, wk) then takes rows 32*wm.. and
// every WK-th 32-key tile: few rows (decode) put the waves side by side on the keys, many rows
// on the rows.  S^T = K . Q^T leaves a row's scores in one lane pair, so the softmax needs one
// exchange per tile and the row's factors none, and the S^T registers are the P^T operand as they
// stand: product slot t of lane half g is key 16*kk + 8*(t/4) + 4*g + t%4, which the transposing
// reads of V deliver.
//
// What bounds it.  Few rows: memory; single tokens of 32 requests over 16384 keys of 8 heads of 128 read 4.3 TB/s,
// 5.2 where the slots of a head are contiguous.  At head size 64 two heads share a 128-byte line and are read at
// different times: 64 requests over 8192 to 32768 keys, 557 us against 316 with a head's slots contiguous.  Many
// rows: the matrix unit (36 % busy), the vector unit (39 %: exponentials, scales, rounding, conversion) and LDS
// (37 %), which the two waves of a SIMD hardly overlap; 64 trees of 64 nodes and 4 query heads a KV head over 8192
// to 32768 keys (uniform) take 1.85 ms, 0.80 PFLOP/s.  Whole steps with one of these parts left out take 7 to 12 %
// less.
#pragma once

#include <float.h>
#include <math.h>
#include <stdint.h>

#include "tv_internal.h"

namespace tv {

// A row block whose pieces the merge joins, written by the workgroup whose share its first step ends.
struct alignas(16) E4m3Job {
    uint16_t pieces;       // 0: none
    uint16_t rows;         // live rows of the block
    int32_t first_row;     // packed row of the request's first node
    int32_t head0;         // first query head of the KV head
    int32_t row0;          // the block's first row, counted as node * group + head over the request
};

struct E4m3Params {
    const void* q;
    int64_t q_s0, q_s1;
    const uint8_t* k;
    const uint8_t* v;
    int64_t k_s0, v_s0, kc_s0, vc_s0;   // page strides of the codes and the scales
    int32_t k_s1, k_s2, v_s1, v_s2;     // slot and head strides
    int32_t kc_s1, kc_s2, vc_s1, vc_s2;
    const float* ks;
    const float* vs;
    int32_t num_blocks, block_size;
    // A whole prefix step lies in one page, K and V (and their scales) have the same strides, and a page's
    // offsets are below 2^31; strides in bytes.
    int32_t page_steps;
    uint32_t f_s0, f_s1, f_c0, f_c1;
    uint32_t div_mul, div_shift;   // pos / block_size by multiplication (e4_page_of)
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
    int32_t num_requests, total_queries, num_kv_heads, groups;
    float c;                       // scale * log2(e)
    float* ws_o;
    float2* ws_ml;
    struct E4m3Job* jobs;          // one a workgroup of the attention launch
    int32_t workgroups;            // of the attention launch
    int32_t* status;
};

// How a launch of average `rows` score rows per request and KV head is shaped.
struct E4m3Shape {
    int32_t rows;          // score rows of a row block
    int32_t threads;
    int32_t per_cu;        // workgroups a compute unit holds
};

E4m3Shape e4m3_shape_d64(int64_t average_rows);
E4m3Shape e4m3_shape_d128(int64_t average_rows);
E4m3Shape e4m3_shape_d256(int64_t average_rows);
// Enqueue the attention (and nothing else).  A probability is rounded to one bf16 term for bf16
// output, whose own step is as coarse, and kept in two for f16 output and three for fp32.
void launch_e4m3_d64(const E4m3Params& p, const E4m3Shape& shape, bool bf16, hipStream_t s);
void launch_e4m3_d128(const E4m3Params& p, const E4m3Shape& shape, bool bf16, hipStream_t s);
void launch_e4m3_d256(const E4m3Params& p, const E4m3Shape& shape, bool bf16, hipStream_t s);

namespace {

typedef __bf16 e4_bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 e4_f16x8 __attribute__((ext_vector_type(8)));
typedef float e4_f32x16 __attribute__((ext_vector_type(16)));
typedef float e4_f32x4 __attribute__((ext_vector_type(4)));
typedef float e4_f32x4u __attribute__((ext_vector_type(4), aligned(4)));   // at any element
typedef short e4_i16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) e4_i16x4 e4_lds_i16x4;

// Quotient by the block size, exact below 2^31: multiplication by a rounded-up reciprocal
// (Granlund and Montgomery, "Division by invariant integers using multiplication", 1994).
__device__ __forceinline__ int32_t e4_page_of(uint32_t mul, uint32_t shift, int32_t pos) {
    const uint32_t n = static_cast<uint32_t>(pos);
    return static_cast<int32_t>((__umulhi(mul, n) + n) >> shift);
}

constexpr int kE4Tile = 32;                        // keys of an MFMA tile
// Keys of a step: 32 KiB of codes at head size 128 are in flight per workgroup, and K and V take
// 64 KiB of LDS (two workgroups a CU).
constexpr int e4_step_keys(int d) { return d == 256 ? 64 : 128; }

__device__ __forceinline__ int64_t e4_uniform(int64_t x) {
    return (static_cast<int64_t>(__builtin_amdgcn_readfirstlane(static_cast<int32_t>(x >> 32))) << 32) |
           static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int32_t>(x)));
}

// One request's live lengths, and the steps of its row blocks.
struct E4Request {
    int32_t prefix, nodes, first_row;
    int64_t bias;
    int32_t prefix_steps, blocks;   // blocks 0: nothing to compute
};

template <int ROWS, int SK>
__device__ __forceinline__ E4Request e4_request(const E4m3Params& p, int r, bool report) {
    E4Request q;
    q.prefix = p.plen[r];
    q.nodes = p.cnt[r];
    q.first_row = p.cu[r];
    q.bias = p.bias_off[r];
    q.prefix_steps = q.blocks = 0;
    if (q.nodes == 0) return q;
    // The rows, the bias and the table row have to hold what the lengths say.
    const int64_t square = static_cast<int64_t>(q.nodes) * q.nodes;
    if (q.prefix < 0 || q.prefix > p.max_prefix || q.nodes < 0 || q.nodes > p.total_queries || q.first_row < 0 ||
        q.first_row > p.total_queries - q.nodes || q.bias < 0 || q.bias > p.bias_elems - square) {
        if (report) set_status(p.status, TV_STATUS_BAD_REQUEST);
        return q;
    }
    q.prefix_steps = (q.prefix + SK - 1) / SK;
    q.blocks = (q.nodes * p.groups + ROWS - 1) / ROWS;   // nodes * groups <= rows of Q * heads < 2^31
    return q;
}

// Tree nodes that some row of block b may see (nodes up to the block's last one).
template <int ROWS>
__device__ __forceinline__ int32_t e4_tree_keys(const E4m3Params& p, const E4Request& q, int b) {
    if (b + 1 == q.blocks) return q.nodes;
    return (b * ROWS + ROWS - 1) / p.groups + 1;   // at most nodes: the block ends before the last row
}

template <int ROWS, int SK>
__device__ __forceinline__ int32_t e4_block_steps(const E4m3Params& p, const E4Request& q, int b) {
    return q.prefix_steps + (e4_tree_keys<ROWS>(p, q, b) + SK - 1) / SK;
}

template <int ROWS, int SK>
__device__ __forceinline__ int64_t e4_head_steps(const E4m3Params& p, const E4Request& q) {
    int64_t n = 0;
    for (int b = 0; b < q.blocks; ++b) n += e4_block_steps<ROWS, SK>(p, q, b);
    return n;
}

// A place in the order of all steps.
struct E4Place {
    int32_t r, h, b;
    int32_t step;    // step within the block
    int32_t steps;   // of the block
};

// Unsigned quotient; 64-bit division only where it has to be.
__device__ __forceinline__ int64_t e4_divide(int64_t a, int64_t b) {
    if (((a | b) >> 32) == 0) return static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
    return a / b;
}

// First step of workgroup w: equal shares of all.  With fewer steps than workgroups the first `total` take
// one each.
__device__ __forceinline__ int64_t e4_first_step(int64_t total, int32_t workgroups, int32_t w) {
    if (total <= workgroups) return w < total ? w : total;
    const int64_t each = e4_divide(total, workgroups);
    const uint32_t rest = static_cast<uint32_t>(total - each * workgroups);   // below the workgroups: 32-bit products
    return each * w + rest * static_cast<uint32_t>(w) / static_cast<uint32_t>(workgroups);
}

// Counts every step of the launch into `total`, then finds step `pick(total)`; false if that is no step.
// All threads of the workgroup call it; `scratch` is LDS of its own.
template <int ROWS, int SK, int THREADS, class PICK>
__device__ __forceinline__ bool e4_find(const E4m3Params& p, int64_t* scratch, int64_t& total, E4Place& place, E4Request& request,
                                        PICK pick) {
    constexpr int WAVES = THREADS / 64;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const bool report = blockIdx.x == 0;
    int64_t at, target;    // first step of request r, the step to find
    int r;
    if (p.num_requests <= 64) {
        // A lane per request, in every wave by itself.
        E4Request q = {};
        int64_t mine = 0;
        if (lane < p.num_requests) {
            q = e4_request<ROWS, SK>(p, lane, report && wave == 0);
            mine = e4_head_steps<ROWS, SK>(p, q) * p.num_kv_heads;
        }
        int64_t end = mine;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int64_t y = __shfl_up(end, o);
            if (lane >= o) end += y;
        }
        total = e4_uniform(__shfl(end, 63));
        target = e4_uniform(pick(total));
        if (target < 0 || target >= total) return false;
        r = __builtin_amdgcn_readfirstlane(__ffsll(static_cast<long long>(__ballot(end > target))) - 1);
        at = e4_uniform(__shfl(end - mine, r));
        request.prefix = __builtin_amdgcn_readlane(q.prefix, r);
        request.nodes = __builtin_amdgcn_readlane(q.nodes, r);
        request.first_row = __builtin_amdgcn_readlane(q.first_row, r);
        request.bias = e4_uniform(__shfl(q.bias, r));
        request.prefix_steps = __builtin_amdgcn_readlane(q.prefix_steps, r);
        request.blocks = __builtin_amdgcn_readlane(q.blocks, r);
    } else {
        const int per = (p.num_requests + THREADS - 1) / THREADS;
        const int r0 = tid * per, r1 = r0 + per < p.num_requests ? r0 + per : p.num_requests;
        int64_t mine = 0;
        for (int i = r0; i < r1; ++i) {
            const E4Request q = e4_request<ROWS, SK>(p, i, report);
            mine += e4_head_steps<ROWS, SK>(p, q) * p.num_kv_heads;
        }
        int64_t end = mine;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int64_t y = __shfl_up(end, o);
            if (lane >= o) end += y;
        }
        if (lane == 63) scratch[wave] = end;
        __syncthreads();
        total = 0;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            if (w < wave) end += scratch[w];
            total += scratch[w];
        }
        __syncthreads();
        total = e4_uniform(total);
        target = e4_uniform(pick(total));
        if (target < 0 || target >= total) return false;   // the same in every thread
        if (end - mine <= target && target < end) {        // this thread's requests hold it
            int64_t first = end - mine;
            for (int i = r0; i < r1; ++i) {
                const E4Request q = e4_request<ROWS, SK>(p, i, false);
                const int64_t next = first + e4_head_steps<ROWS, SK>(p, q) * p.num_kv_heads;
                if (target < next) {
                    scratch[0] = i;
                    scratch[1] = first;
                    break;
                }
                first = next;
            }
        }
        __syncthreads();
        r = __builtin_amdgcn_readfirstlane(static_cast<int>(scratch[0]));
        at = e4_uniform(scratch[1]);
        __syncthreads();
        request = e4_request<ROWS, SK>(p, r, false);
    }
    place.r = r;
    const int64_t head = e4_head_steps<ROWS, SK>(p, request);
    place.h = static_cast<int32_t>(e4_divide(target - at, head));
    at += place.h * head;
    place.b = 0;
    place.steps = e4_block_steps<ROWS, SK>(p, request, 0);
    while (target >= at + place.steps) {
        at += place.steps;
        place.steps = e4_block_steps<ROWS, SK>(p, request, ++place.b);
    }
    place.step = static_cast<int32_t>(target - at);
    return true;
}

template <class T>
struct E4Type;
template <>
struct E4Type<__bf16> {
    typedef e4_bf16x8 vec;
    static __device__ __forceinline__ e4_f32x16 run(vec a, vec b, e4_f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
    // Two codes of a word (the low or the high pair) as two values; a scale of 1 leaves them exact.
    template <bool HI>
    static __device__ __forceinline__ uint32_t two(uint32_t codes) {
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, 1.0f, HI));
    }
};
template <>
struct E4Type<_Float16> {
    typedef e4_f16x8 vec;
    static __device__ __forceinline__ e4_f32x16 run(vec a, vec b, e4_f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    }
    template <bool HI>
    static __device__ __forceinline__ uint32_t two(uint32_t codes) {
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, 1.0f, HI));
    }
};

// Swizzles of the 16-byte chunks of a [key][dim] row: a b128 read of one chunk column by 16 keys
// (K), and a transposing read of 4 keys x 4 chunks (V), each spread over all banks.
template <int D>
__device__ __forceinline__ int e4_k_chunk(int key, int chunk) {
    return D == 64 ? chunk ^ ((key >> 1) & 7) : chunk ^ (key & 15);
}
template <int D>
__device__ __forceinline__ int e4_v_chunk(int key, int chunk) {
    return D == 64 ? chunk ^ (4 * ((key >> 1) & 1)) : chunk ^ (4 * (key & 3));
}

// Maximum / sum over a lane pair (c, c + 32): the swap leaves the lower half's value in one register
// and the upper half's in the other, in every lane.
__device__ __forceinline__ float e4_pair_max(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float e4_pair_sum(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Weight of a partial result (m, l) against the joined maximum.  One that saw nothing has l = 0 and
// adds nothing; one whose scores are all NaN has m = -inf and a NaN l, which stays.
__device__ __forceinline__ float e4_weight(float2 ml, float best) {
    return ml.x == -INFINITY ? (ml.y == 0.0f ? 0.0f : 1.0f) : __builtin_amdgcn_exp2f(ml.x - best);
}

// Writes four consecutive output dims of a row.
template <class T>
__device__ __forceinline__ void e4_store4(const E4m3Params& p, int64_t row, int head, int dim, e4_f32x4 v) {
    if (p.out_f32) {
        float* o = static_cast<float*>(p.out) + row * p.o_s0 + head * p.o_s1 + dim;
        *reinterpret_cast<e4_f32x4*>(o) = v;
    } else {
        T* o = static_cast<T*>(p.out) + row * p.o_s0 + head * p.o_s1 + dim;
        T h[4] = {static_cast<T>(v[0]), static_cast<T>(v[1]), static_cast<T>(v[2]), static_cast<T>(v[3])};
        *reinterpret_cast<u32x2*>(o) = __builtin_bit_cast(u32x2, h);
    }
}

template <int D, int WM, int WK, int NBUF, class T, int TERMS>
__global__ void __launch_bounds__(64 * WM * WK, D == 256 ? 1 : 2)
e4m3_attention_kernel(const E4m3Params p) {
    constexpr int THREADS = 64 * WM * WK, ROWS = 32 * WM, SK = e4_step_keys(D);
    constexpr int LPR = D / 16;                    // lanes that move one key's row
    constexpr int KPP = THREADS / LPR;             // keys a pass of the workgroup moves
    constexpr int PASSES = SK / KPP;
    constexpr int KB = SK * D * 2;                 // bytes of a step's K (or V) in LDS
    constexpr int TILES = SK / kE4Tile / WK;       // tiles a wave takes of a step
    constexpr int NK = D / 16, NB = D / 32;        // MFMAs of a tile's scores; output blocks
    static_assert(PASSES <= LPR, "a lane of its row for each pass's scales");
    static_assert(SK % KPP == 0 && SK % (kE4Tile * WK) == 0, "a step is whole passes and tiles");
    static_assert(KPP % 16 == 0 || (KPP == 8 && D != 64), "the swizzle's period");
    static_assert(WK == 1 || WK * 32 * D * 4 <= NBUF * 2 * KB, "the waves' results share the staging memory");
    typedef typename E4Type<T>::vec V8;

    __shared__ __attribute__((aligned(1024))) char lds[NBUF * 2 * KB];
    __shared__ __attribute__((aligned(16))) float lds_ks[NBUF][SK], lds_vs[NBUF][SK], lds_kb[NBUF][SK];
    __shared__ float2 lds_ml[WM * WK][32];
    __shared__ int lds_bad[NBUF];
    __shared__ int64_t lds_scan[THREADS / 64 < 3 ? 3 : THREADS / 64];

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave % WM, wk = wave / WM;
    const int c = lane & 31, half = lane >> 5;

    if (tid < NBUF) lds_bad[tid] = 0;   // ordered before the first mark by the barrier behind the search
    // Neighbouring shares go to one XCD (workgroups are dealt to the 8 in turn), whose L2 then
    // holds what they have in common: the scales of a key's heads, the keys of a head's blocks.
    const int W = p.workgroups;
    int64_t total = 0, s0 = 0, s1 = 0;   // all steps; this share's
    int share = 0;
    E4Place at;
    E4Request req;
    const bool any = e4_find<ROWS, SK, THREADS>(p, lds_scan, total, at, req, [&](int64_t all) -> int64_t {
        share = all < W ? static_cast<int>(blockIdx.x) : static_cast<int>(blockIdx.x % 8 * (W / 8) + blockIdx.x / 8);
        s0 = e4_first_step(all, W, share);
        s1 = e4_first_step(all, W, share + 1);
        return s0 < s1 ? s0 : -1;
    });
    if (tid == 0) p.jobs[share].pieces = 0;
    if (!any) return;
    // Two buffers stage the first step, and may mark it, without a barrier of their own (the search has none for up
    // to 64 requests); with one buffer every step begins with a barrier.
    if constexpr (NBUF == 2) __syncthreads();
    share = __builtin_amdgcn_readfirstlane(share);
    int todo = __builtin_amdgcn_readfirstlane(static_cast<int>(s1 - s0));   // steps not yet run

    // Parameters that the whole prefix steps do not need are read where they are used: held over the loop,
    // with the others, they would not fit the scalar registers.
    typedef const __attribute__((address_space(4))) E4m3Params* Params;
    auto cold = [&]() {
        Params a = (Params)__builtin_amdgcn_kernarg_segment_ptr();
        asm volatile("" : "+s"(a));
        return a;
    };

    // --- a run: steps [run0, run1) of one row block ---------------------------------------------
    int n_tree = 0;                        // nodes that the block may see
    int run0 = at.step, run1 = 0;
    const int32_t* table = nullptr;        // of the request
    const int64_t* slots = nullptr;
    const char *k_head = nullptr, *v_head = nullptr, *ks_head = nullptr, *vs_head = nullptr;   // of the KV head
    const uint32_t s0_ = p.f_s0, s1_ = p.f_s1, c0_ = p.f_c0, c1_ = p.f_c1;

    auto is_tree = [&](int i) { return i >= req.prefix_steps; };
    auto first_key = [&](int i) { return (is_tree(i) ? i - req.prefix_steps : i) * SK; };
    auto keys_left = [&](int i) { return (is_tree(i) ? n_tree : req.prefix) - first_key(i); };
    auto in_page = [&](int i) { return p.page_steps && !is_tree(i) && keys_left(i) >= SK; };

    // --- moving a step's keys -----------------------------------------------------------------
    const int my_key = tid / LPR, my_chunk = tid % LPR;
    int32_t entry[PASSES], entry_high[PASSES];   // page numbers, or tree slots in two halves
    u32x4 kreg[PASSES], vreg[PASSES];
    float ksr = 0.0f, vsr = 0.0f;   // scales of the key of pass my_chunk
    uint32_t good = 0, wrong = 0;   // passes whose key is live and found / live and not found

    auto here = [](int x) {   // the same value, which the compiler cannot compute with ahead of its use
        asm volatile("" : "+v"(x));
        return x;
    };
    // LDS offsets. Keys 16 apart share a swizzle, so what differs between passes, tiles and the halves of
    // a product is a constant; the chunks of a row are an exclusive or away from the first.
    const int k_put = my_key * 2 * D + 16 * e4_k_chunk<D>(my_key, 2 * my_chunk);
    const int v_put = my_key * 2 * D + 16 * e4_v_chunk<D>(my_key, 2 * my_chunk);
    const int k_get = c * 2 * D + 16 * e4_k_chunk<D>(c, half);
    const int v_key = 4 * half + ((lane & 15) >> 2), v_dim = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
    const int v_get = v_key * 2 * D + 16 * e4_v_chunk<D>(v_key, v_dim >> 3) + 2 * (v_dim & 7);

    // Loads the page numbers (tree slots: both halves) of a step; nothing looks at them before fetch_keys().
    auto fetch_entries = [&](int i) {
        const int key0 = first_key(i), last = keys_left(i) - 1;
        if (in_page(i)) {
            // One page number, the same in every lane: a vector load, which the waits on LDS do not wait for.
            entry[0] = table[e4_page_of(p.div_mul, p.div_shift, key0) + here(0)];
            return;
        }
        const Params a = cold();
        const int my_key = here(tid) / LPR;
        const bool tree = is_tree(i);
#pragma unroll
        for (int n = 0; n < PASSES; ++n) {
            const int kk = n * KPP + my_key, of = key0 + (kk < last ? kk : last);
            const int32_t* from = tree ? reinterpret_cast<const int32_t*>(slots + of)
                                       : table + e4_page_of(a->div_mul, a->div_shift, of);
            entry[n] = from[0];
            entry_high[n] = from[tree ? 1 : 0];
        }
    };
    constexpr uint32_t kAll = (1u << PASSES) - 1;
    const uint32_t code_of = my_key * s1_ + 16 * my_chunk, scale_of = (my_chunk * KPP + my_key) * c1_;
    auto fetch_keys = [&](int i) {
        const int key0 = first_key(i), left = keys_left(i);
        good = wrong = 0;
        // Every lane loads on every path, one whose key is past the end or not found from the pool's first
        // row, which stage() drops: a load in a branch would be waited for where the branch ends.
        int64_t k_of[PASSES], v_of[PASSES], ks_of = 0, vs_of = 0;
        if (in_page(i)) {
            const int32_t page = __builtin_amdgcn_readfirstlane(entry[0]);
            const uint32_t offset = key0 - e4_page_of(p.div_mul, p.div_shift, key0) * p.block_size;
            const bool found = page >= 0 && page < p.num_blocks;
            (found ? good : wrong) = kAll;
            const uint64_t from = found ? page : 0;
            const uint64_t code = from * s0_ + offset * s1_;
#pragma unroll
            for (int n = 0; n < PASSES; ++n) k_of[n] = v_of[n] = code + n * KPP * s1_ + code_of;
            ks_of = vs_of = from * c0_ + offset * c1_ + (my_chunk < PASSES ? scale_of : 0);
        } else {
            const Params a = cold();
            const int my_key = here(tid) / LPR, my_chunk = here(tid) % LPR;
            const bool tree = is_tree(i);
#pragma unroll
            for (int n = 0; n < PASSES; ++n) {
                const int kk = n * KPP + my_key;
                const int32_t pos = tree ? entry[n] : key0 + kk;   // a slot or a position
                const int32_t quotient = e4_page_of(a->div_mul, a->div_shift, pos < 0 ? 0 : pos);
                const int32_t page = !tree ? entry[n] : entry[n] < 0 || entry_high[n] != 0 ? -1 : quotient;
                const bool live = kk < left, found = live && page >= 0 && page < a->num_blocks;
                if (found) good |= 1u << n;
                if (live && !found) wrong |= 1u << n;
                const int64_t from = found ? page : 0, offset = found ? pos - quotient * a->block_size : 0;
                k_of[n] = from * a->k_s0 + offset * a->k_s1 + 16 * my_chunk;
                v_of[n] = from * a->v_s0 + offset * a->v_s1 + 16 * my_chunk;
                if (my_chunk == n) {
                    ks_of = 4 * (from * a->kc_s0 + offset * a->kc_s1);
                    vs_of = 4 * (from * a->vc_s0 + offset * a->vc_s1);
                }
            }
        }
#pragma unroll
        for (int n = 0; n < PASSES; ++n) {
            kreg[n] = *reinterpret_cast<const u32x4*>(k_head + k_of[n]);
            vreg[n] = *reinterpret_cast<const u32x4*>(v_head + v_of[n]);
        }
        ksr = *reinterpret_cast<const float*>(ks_head + ks_of);
        vsr = *reinterpret_cast<const float*>(vs_head + vs_of);
    };
    // Codes to LDS as bf16/f16 values, with the step's scales; `mark` tags the buffer if a key's
    // page was not found.
    auto stage = [&](int step, int buf, int mark) {
        const float scale = p.c;
        const bool tree = is_tree(step);
        char* kb = lds + buf * 2 * KB;
        char* vb = kb + KB;
        if (__any(good != kAll)) {
#pragma unroll
            for (int i = 0; i < PASSES; ++i) {
                const uint32_t keep = (good >> i) & 1 ? 0xffffffffu : 0u;
                kreg[i] &= keep;
                vreg[i] &= keep;
            }
            if (!((good >> my_chunk) & 1)) ksr = vsr = 0.0f;
        }
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
            const int kk = i * KPP + my_key;
            float kscale = ksr * scale, vscale = vsr;
            if (tree) {
                // Rows that do not see a node have to get zero from its V row, and zero times NaN is not.
                // So NaN codes become zeros, and they or a scale that is not finite make the node's score
                // NaN instead, which hidden scores never show.
                uint32_t nan = 0;
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const uint32_t high = ((vreg[i][w] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
                    vreg[i][w] &= ~((high >> 7) * 0xffu);
                    nan |= high;
                }
                const uint64_t lanes = __ballot(nan != 0);
                if (((lanes >> (lane & ~(LPR - 1))) & ((1ull << LPR) - 1)) || !(fabsf(vscale) < INFINITY)) {
                    kscale = NAN;
                    vscale = 0.0f;
                }
            }
            u32x4 a, b;
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                a[2 * w] = E4Type<T>::template two<false>(kreg[i][w]);
                a[2 * w + 1] = E4Type<T>::template two<true>(kreg[i][w]);
                b[2 * w] = E4Type<T>::template two<false>(kreg[i][w + 2]);
                b[2 * w + 1] = E4Type<T>::template two<true>(kreg[i][w + 2]);
            }
            constexpr bool kAlternate = KPP % 16 != 0;   // every second pass is 8 keys off the swizzle's period
            const int at = i * KPP * 2 * D;
            const int kx = kAlternate && (i & 1) ? k_put ^ (8 * 16) : k_put;
            *reinterpret_cast<u32x4*>(kb + at + kx) = a;
            *reinterpret_cast<u32x4*>(kb + at + (kx ^ 16)) = b;
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                a[2 * w] = E4Type<__bf16>::two<false>(vreg[i][w]);
                a[2 * w + 1] = E4Type<__bf16>::two<true>(vreg[i][w]);
                b[2 * w] = E4Type<__bf16>::two<false>(vreg[i][w + 2]);
                b[2 * w + 1] = E4Type<__bf16>::two<true>(vreg[i][w + 2]);
            }
            *reinterpret_cast<u32x4*>(vb + at + v_put) = a;
            *reinterpret_cast<u32x4*>(vb + at + (v_put ^ 16)) = b;
            if (my_chunk == i) {
                lds_ks[buf][kk] = kscale;
                lds_vs[buf][kk] = vscale;
                lds_kb[buf][kk] = (good >> i) & 1 ? 0.0f : -INFINITY;
            }
        }
        if (wrong) {
            lds_bad[buf] = mark;
            set_status(p.status, TV_STATUS_BAD_PAGE);
        }
    };

    // --- a row block's state ------------------------------------------------------------------
    V8 qb[NK];
    e4_f32x16 acc[NB];
    float m = -INFINITY, l = 0.0f;
    int node = -1, qhead = 0;      // of this lane's row; node -1: no row
    bool wave_rows = false;        // any row of this wave
    int nodes = 0, first_row = 0;  // of the request
    const float* bias = nullptr;   // of this lane's node

    // The block that `at` names, whose run begins at at.step.
    auto start_block = [&]() {
        const Params a = cold();
        nodes = req.nodes;
        first_row = req.first_row;
        n_tree = e4_tree_keys<ROWS>(p, req, at.b);
        run0 = at.step;
        run1 = at.steps - run0 < todo ? at.steps : run0 + todo;
        table = a->tables + at.r * a->t_s0;
        slots = a->tree_slots + req.first_row;
        k_head = reinterpret_cast<const char*>(a->k) + at.h * static_cast<int64_t>(a->k_s2);
        v_head = reinterpret_cast<const char*>(a->v) + at.h * static_cast<int64_t>(a->v_s2);
        ks_head = reinterpret_cast<const char*>(a->ks + at.h * static_cast<int64_t>(a->kc_s2));
        vs_head = reinterpret_cast<const char*>(a->vs + at.h * static_cast<int64_t>(a->vc_s2));
        const int groups = a->groups;
        const int row = at.b * ROWS + 32 * wm + c;
        wave_rows = at.b * ROWS + 32 * wm < nodes * groups;
        const int n = row / groups;
        node = n < nodes ? n : -1;
        qhead = at.h * groups + row - n * groups;
        bias = a->bias + req.bias + static_cast<int64_t>(node < 0 ? 0 : node) * nodes;
        const T* src = static_cast<const T*>(a->q) + static_cast<int64_t>(first_row + (node < 0 ? 0 : node)) * a->q_s0 +
                       qhead * a->q_s1 + 8 * half;
#pragma unroll
        for (int i = 0; i < NK; ++i) {
            u32x4 x = {0, 0, 0, 0};
            if (node >= 0) x = *reinterpret_cast<const u32x4*>(src + 16 * i);
            qb[i] = __builtin_bit_cast(V8, x);
        }
#pragma unroll
        for (int i = 0; i < NB; ++i) acc[i] = e4_f32x16{};
        m = -INFINITY;
        l = 0.0f;
    };

    // K . Q^T of a tile (LDS at `kb`): element i is key 8*(i/4) + 4*half + i%4 of the tile.
    auto products = [&](const char* kb) {
        e4_f32x16 x = {};
#pragma unroll
        for (int i = 0; i < NK; ++i) {
            const u32x4 a = *reinterpret_cast<const u32x4*>(kb + (k_get ^ (32 * i)));
            x = E4Type<T>::run(__builtin_bit_cast(V8, a), qb[i], x);
        }
        return x;
    };
    // Products to scores, with the biases; those that the row does not see become -inf, whatever they are.
    auto mask = [&](int step, int buf, int t, e4_f32x16& x, const e4_f32x16& ks) {
        const int key0 = t * kE4Tile + 4 * (here(lane) >> 5);
        const int last = node < n_tree ? node : n_tree - 1;   // the last node seen
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float b[8];
            if (is_tree(step)) {
                const int of0 = first_key(step) + key0 + 16 * h;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int of = of0 + 8 * (i >> 2) + (i & 3);
                    b[i] = bias[of <= last ? of : 0];
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int of = of0 + 8 * (i >> 2) + (i & 3);
                    // In score units; a finite bias stays finite.
                    float b2 = b[i] * 1.44269504088896340736f;
                    if (fabsf(b2) == INFINITY) b2 = copysignf(FLT_MAX, b2);
                    b[i] = of <= last && b[i] != -INFINITY ? b2 : -INFINITY;
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) b[i] = 0.0f;
            }
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                const e4_f32x4 kb = *reinterpret_cast<const e4_f32x4*>(&lds_kb[buf][key0 + 16 * h + 8 * g]);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int i = 8 * h + 4 * g + e;
                    const float add = kb[e] == 0.0f ? b[4 * g + e] : kb[e];
                    x[i] = add == -INFINITY ? -INFINITY : fmaf(x[i], ks[i], add);
                }
            }
            __builtin_amdgcn_sched_barrier(0);   // eight biases in registers at a time
        }
    };
    // The same for the largest shape, that of chunks: prefix tails apart, and four biases a load, of which those
    // behind the last node seen are dropped, unless they could lie behind all biases.  8 chunks of 512 nodes: 613 us
    // against 665.  The other shapes' trees are short, and their registers full (head size 256 would spill).
    auto mask_wide = [&](int step, int buf, int t, e4_f32x16& x, const e4_f32x16& ks) {
        const int key0 = t * kE4Tile + 4 * (here(lane) >> 5);
        if (!is_tree(step)) {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const e4_f32x4 kb = *reinterpret_cast<const e4_f32x4*>(&lds_kb[buf][key0 + 8 * g]);
#pragma unroll
                for (int e = 0; e < 4; ++e) x[4 * g + e] = kb[e] == 0.0f ? x[4 * g + e] * ks[4 * g + e] : -INFINITY;
            }
            return;
        }
        const int of0 = first_key(step) + key0;
        const int last = node < n_tree ? node : n_tree - 1;   // the last node seen
        const Params a = cold();
        const bool wide = __all(bias + first_key(step) + (t + 1) * kE4Tile <= a->bias + a->bias_elems);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float b[8];
            if (wide) {
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                    const e4_f32x4u four = *reinterpret_cast<const e4_f32x4u*>(bias + of0 + 16 * h + 8 * g);
#pragma unroll
                    for (int e = 0; e < 4; ++e) b[4 * g + e] = four[e];
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int of = of0 + 16 * h + 8 * (i >> 2) + (i & 3);
                    b[i] = bias[of <= last ? of : 0];
                }
            }
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                const e4_f32x4 kb = *reinterpret_cast<const e4_f32x4*>(&lds_kb[buf][key0 + 16 * h + 8 * g]);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int i = 8 * h + 4 * g + e;
                    const float bias_ = b[4 * g + e];
                    const bool seen = of0 + 16 * h + 8 * g + e <= last && bias_ != -INFINITY && kb[e] == 0.0f;
                    float add = bias_ * 1.44269504088896340736f;   // in score units; a finite bias stays finite
                    if (fabsf(add) == INFINITY) add = copysignf(FLT_MAX, add);
                    x[i] = seen ? fmaf(x[i], ks[i], add) : -INFINITY;
                }
            }
            __builtin_amdgcn_sched_barrier(0);   // eight biases in registers at a time
        }
    };
    // The wave's tiles of a step, in two phases each: the exponentials of a tile, while the next tile's K
    // operands arrive, and the matrix products of both, while this tile's V operands do.  At head size 256, with
    // one wave a SIMD, the next tile's scores run beside the exponentials instead: 64 requests of 4096 to
    // 16384 keys and 250 rows 2818 us against 2948; at 128, whose second wave fills the gaps, 1848 either way.
    constexpr bool kEarly = D == 256;
    auto tiles_of = [&](int step, int buf, bool masked) {
        const char* kb = lds + buf * 2 * KB + wk * kE4Tile * 2 * D;
        const char* vb = kb + KB;
        const float* ksb = &lds_ks[buf][wk * kE4Tile + 4 * half];
        const float* vsb = &lds_vs[buf][wk * kE4Tile + 4 * half];
        const int tiles = (keys_left(step) + kE4Tile - 1) / kE4Tile;   // at most TILES * WK count
        e4_f32x16 x = products(kb);
#pragma unroll
        for (int n = 0; n < TILES; ++n) {
            const int t = n * WK + wk;
            if (t >= tiles) break;
            const int key = n * WK * kE4Tile;   // of the tile, from the wave's first
            e4_f32x16 ks;
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const e4_f32x4 four = *reinterpret_cast<const e4_f32x4*>(ksb + key + 8 * g);
#pragma unroll
                for (int e = 0; e < 4; ++e) ks[4 * g + e] = four[e];
            }
            if (masked) {
                if constexpr (WM == 8) mask_wide(step, buf, t, x, ks);
                else mask(step, buf, t, x, ks);
#pragma unroll
                for (int i = 0; i < 16; ++i) ks[i] = 1.0f;
            }
            // Probabilities against the row's reference, which is near the largest score seen: it is
            // raised only when a tile's would pass 2^8, until when they cost no precision.
            float negative = m == -INFINITY ? 0.0f : -m;
            e4_f32x16 pr, next = {};
            if (kEarly && n + 1 < TILES) next = products(kb + (key + WK * kE4Tile) * 2 * D);
            // Both times in one order: a row whose neighbours raise their reference is summed a second time.
            auto exponentials = [&]() {
                float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    pr[i] = __builtin_amdgcn_exp2f(fmaf(x[i], ks[i], negative));
                    sum[i & 3] += pr[i];
                }
                return (sum[0] + sum[1]) + (sum[2] + sum[3]);
            };
            float tile_sum = exponentials();
            const bool over = !(tile_sum <= 256.0f) || m == -INFINITY;
            if (__any(over)) {   // other rows of the wave keep their reference: no row depends on another
                float top = x[0] * ks[0];
#pragma unroll
                for (int i = 1; i < 16; ++i) top = fmaxf(top, x[i] * ks[i]);
                const float raised = e4_pair_max(over ? 1.0f : 0.0f) != 0.0f ? fmaxf(m, e4_pair_max(top)) : m;
                const float factor = raised == m ? 1.0f : __builtin_amdgcn_exp2f(m - raised);
                m = raised;
                l *= factor;
#pragma unroll
                for (int i = 0; i < NB; ++i) acc[i] *= factor;
                negative = m == -INFINITY ? 0.0f : -m;
                tile_sum = exponentials();
            }
            l += tile_sum;
            e4_bf16x8 pb[TERMS][2];
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const e4_f32x4 vs = *reinterpret_cast<const e4_f32x4*>(vsb + key + 8 * g);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int i = 4 * g + e;
                    float pv = pr[i] * vs[e];
#pragma unroll
                    for (int q = 0; q < TERMS; ++q) {
                        pb[q][i >> 3][i & 7] = static_cast<__bf16>(pv);
                        if (q + 1 < TERMS) pv -= static_cast<float>(pb[q][i >> 3][i & 7]);
                    }
                }
            }
            e4_i16x4 va[NB][2];
            auto read_values = [&](int kk) {
#pragma unroll
                for (int db = 0; db < NB; ++db) {
                    const char* lo = vb + (key + 16 * kk) * 2 * D + (v_get ^ (64 * db));
                    va[db][0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((e4_lds_i16x4*)lo);
                    va[db][1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((e4_lds_i16x4*)(lo + 8 * 2 * D));
                }
            };
            read_values(0);
            if (!kEarly && n + 1 < TILES) x = products(kb + (key + WK * kE4Tile) * 2 * D);
#pragma unroll
            for (int kk = 0; kk < 2; ++kk) {
                if (kk) read_values(kk);
#pragma unroll
                for (int db = 0; db < NB; ++db) {
                    const e4_bf16x8 v8 = __builtin_bit_cast(
                        e4_bf16x8, __builtin_shufflevector(va[db][0], va[db][1], 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
                    for (int q = 0; q < TERMS; ++q) acc[db] = E4Type<__bf16>::run(v8, pb[q][kk], acc[db]);
                }
            }
            if (kEarly) x = next;
        }
    };

    // A finished run: the row's output, or its unnormalised sum with (m, l) for the merge, in the share's
    // second piece if the run begins its block.
    bool whole = false;
    int64_t piece = 0;
    auto put = [&](int row_in_block, int row_node, int head, int dim, e4_f32x4 v, float row_l) {
        if (whole) {
            const float scale = row_l == 0.0f ? 0.0f : 1.0f / row_l;   // a row that sees nothing is zero
            e4_store4<T>(p, first_row + row_node, head, dim, v * scale);
        } else {
            *reinterpret_cast<e4_f32x4*>(p.ws_o + (piece * ROWS + row_in_block) * D + dim) = v;
        }
    };
    auto finish = [&]() {
        // The lane's place, opaque: addresses made of it here would otherwise be kept over the whole share.
        const int c = here(lane) & 31, half = here(lane) >> 5, tid = here(threadIdx.x);
        l = e4_pair_sum(l);
        whole = run0 == 0 && run1 == at.steps;
        piece = 2 * static_cast<int64_t>(share) + (run0 == 0 ? 1 : 0);
        if (run0 == 0 && !whole && tid == 0) {
            // The share ends inside the block: the pieces go on to the share that holds the block's last
            // step, the first u with first_step(u) >= end (each share of `total` steps is total / n long).
            const int64_t n = total < W ? total : W, end = s1 + (at.steps - run1);
            E4m3Job job = {};
            job.pieces = static_cast<uint16_t>(static_cast<int32_t>(e4_divide(end * n + total - 1, total)) - share);
            const int32_t row0 = at.b * ROWS, live = nodes * p.groups - row0;
            job.rows = static_cast<uint16_t>(live < ROWS ? live : ROWS);
            job.first_row = first_row;
            job.head0 = at.h * p.groups;
            job.row0 = row0;
            p.jobs[share] = job;
        }
        if constexpr (WK == 1) {
            if (node >= 0) {
#pragma unroll
                for (int db = 0; db < NB; ++db) {
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        const e4_f32x4 v = {acc[db][4 * g], acc[db][4 * g + 1], acc[db][4 * g + 2], acc[db][4 * g + 3]};
                        put(32 * wm + c, node, qhead, 32 * db + 8 * g + 4 * half, v, l);
                    }
                }
                if (!whole && half == 0) p.ws_ml[piece * ROWS + 32 * wm + c] = make_float2(m, l);
            }
        } else {
            // The waves of one row group join their keys through LDS, one row group at a time.
            __syncthreads();
            if (half == 0) lds_ml[wave][c] = make_float2(m, l);
            e4_f32x4* all = reinterpret_cast<e4_f32x4*>(lds);
            constexpr int CH = D / 4;
            for (int g0 = 0; g0 < WM; ++g0) {
                if (wm == g0) {
#pragma unroll
                    for (int db = 0; db < NB; ++db) {
#pragma unroll
                        for (int g = 0; g < 4; ++g) {
                            const e4_f32x4 v = {acc[db][4 * g], acc[db][4 * g + 1], acc[db][4 * g + 2], acc[db][4 * g + 3]};
                            const int ch = (32 * db + 8 * g + 4 * half) / 4;
                            all[(wk * 32 + c) * CH + (ch ^ (c & (CH - 1 < 31 ? CH - 1 : 31)))] = v;
                        }
                    }
                }
                __syncthreads();
                for (int e = tid; e < 32 * CH; e += THREADS) {
                    const int row = e / CH, ch = e % CH;
                    const int in_block = 32 * g0 + row, of = at.b * ROWS + in_block;
                    const int n = of / p.groups;
                    if (n >= nodes) continue;
                    float best = -INFINITY;
#pragma unroll
                    for (int w = 0; w < WK; ++w) best = fmaxf(best, lds_ml[w * WM + g0][row].x);
                    float sum = 0.0f;
                    e4_f32x4 v = {0, 0, 0, 0};
#pragma unroll
                    for (int w = 0; w < WK; ++w) {
                        const float2 ml = lds_ml[w * WM + g0][row];
                        const float f = e4_weight(ml, best);
                        sum += f * ml.y;
                        v += f * all[(w * 32 + row) * CH + (ch ^ (row & (CH - 1 < 31 ? CH - 1 : 31)))];
                    }
                    put(in_block, n, at.h * p.groups + of - n * p.groups, 4 * ch, v, sum);
                    if (!whole && ch == 0) p.ws_ml[piece * ROWS + in_block] = make_float2(best, sum);
                }
                __syncthreads();
            }
        }
    };

    // --- the share, run by run ----------------------------------------------------------------
    int count = 1;   // steps begun, the mark of a buffer with a missing page
    auto compute = [&](int i, int buf) {
        if (wave_rows) tiles_of(i, buf, is_tree(i) || keys_left(i) < SK || lds_bad[buf] == count);
    };
    for (;;) {
        start_block();
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
            // Two buffers: a step is staged while the one before it is computed, by half of the waves (one
            // a SIMD) before their tiles and by the others after, so that each SIMD has one wave on its
            // matrix unit while the other converts.
            static_assert(WK == 1, "finish() would join over buffers in use");
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
        finish();
        todo -= run1 - run0;
        if (todo <= 0) break;
        at.step = 0;
        if (++at.b == req.blocks) {
            at.b = 0;
            if (++at.h == p.num_kv_heads) {
                at.h = 0;
                do {
                    ++at.r;
                    req = e4_request<ROWS, SK>(p, at.r, false);
                } while (req.blocks == 0);   // todo > 0: a later request has steps
            }
        }
        at.steps = e4_block_steps<ROWS, SK>(p, req, at.b);
    }
}

template <int D, int WM, int WK, int NBUF>
void e4_launch(const E4m3Params& p, bool bf16, hipStream_t s) {
    const dim3 grid(p.workgroups), block(64 * WM * WK);
    if (bf16 && !p.out_f32) hipLaunchKernelGGL((e4m3_attention_kernel<D, WM, WK, NBUF, __bf16, 1>), grid, block, 0, s, p);
    else if (bf16) hipLaunchKernelGGL((e4m3_attention_kernel<D, WM, WK, NBUF, __bf16, 3>), grid, block, 0, s, p);
    else if (!p.out_f32) hipLaunchKernelGGL((e4m3_attention_kernel<D, WM, WK, NBUF, _Float16, 2>), grid, block, 0, s, p);
    else hipLaunchKernelGGL((e4m3_attention_kernel<D, WM, WK, NBUF, _Float16, 3>), grid, block, 0, s, p);
}

}  // namespace
}  // namespace tv
