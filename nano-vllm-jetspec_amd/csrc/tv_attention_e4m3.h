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
// bf16, where p * vs is rounded once (or, TWO, kept to 2^-17 in two terms).  The scales never touch
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
#pragma once

#include <float.h>
#include <math.h>
#include <stdint.h>

#include "tv_internal.h"

namespace tv {

struct E4m3Params {
    const void* q;
    int64_t q_s0, q_s1;
    const uint8_t* k;
    const uint8_t* v;
    int64_t k_s0, k_s1, k_s2;
    int64_t v_s0, v_s1, v_s2;
    const float* ks;
    const float* vs;
    int64_t kc_s0, kc_s1, kc_s2;
    int64_t vc_s0, vc_s1, vc_s2;
    int32_t num_blocks, block_size;
    uint32_t div_mul, div_shift;   // pos / block_size by multiplication (E4m3Params::page_of)
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
    int32_t workgroups;            // of the attention launch
    int32_t* status;

    // Quotient by the block size, exact below 2^31: multiplication by a rounded-up reciprocal
    // (Granlund and Montgomery, "Division by invariant integers using multiplication", 1994).
    __device__ __forceinline__ int32_t page_of(int32_t pos) const {
        const uint32_t n = static_cast<uint32_t>(pos);
        return static_cast<int32_t>((__umulhi(div_mul, n) + n) >> div_shift);
    }
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
// Enqueue the attention (and nothing else); `two`: probabilities in two bf16 terms.
void launch_e4m3_d64(const E4m3Params& p, const E4m3Shape& shape, bool bf16, bool two, hipStream_t s);
void launch_e4m3_d128(const E4m3Params& p, const E4m3Shape& shape, bool bf16, bool two, hipStream_t s);
void launch_e4m3_d256(const E4m3Params& p, const E4m3Shape& shape, bool bf16, bool two, hipStream_t s);

namespace {

typedef __bf16 e4_bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 e4_f16x8 __attribute__((ext_vector_type(8)));
typedef float e4_f32x16 __attribute__((ext_vector_type(16)));
typedef float e4_f32x4 __attribute__((ext_vector_type(4)));
typedef short e4_i16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) e4_i16x4 e4_lds_i16x4;

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
    const int32_t last = (b * ROWS + ROWS - 1) / p.groups;
    return last + 1 < q.nodes ? last + 1 : q.nodes;
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
    int64_t begin;   // first step of the block, counted over the whole launch
    int32_t step;    // step within the block
    int32_t steps;   // of the block
};

// Counts every step of the launch into `total`, then finds step `pick(total)`.  All threads of the
// workgroup call it; `scratch` is LDS of its own.
template <int ROWS, int SK, int THREADS, class PICK>
__device__ __forceinline__ bool e4_find(const E4m3Params& p, int64_t* scratch, int64_t& total, E4Place& place, PICK pick) {
    constexpr int WAVES = THREADS / 64;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int per = (p.num_requests + THREADS - 1) / THREADS;
    const int r0 = tid * per, r1 = r0 + per < p.num_requests ? r0 + per : p.num_requests;
    int64_t mine = 0;
    for (int r = r0; r < r1; ++r) {
        const E4Request q = e4_request<ROWS, SK>(p, r, blockIdx.x == 0 && blockIdx.y == 0);
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
    const int64_t target = pick(total);
    if (target < 0 || target >= total) return false;   // the same in every thread
    const int64_t begin = end - mine;
    if (begin <= target && target < end) {
        // This thread's requests hold it.
        int64_t at = begin;
        for (int r = r0; r < r1; ++r) {
            const E4Request q = e4_request<ROWS, SK>(p, r, false);
            const int64_t head = e4_head_steps<ROWS, SK>(p, q);
            if (target >= at + head * p.num_kv_heads) {
                at += head * p.num_kv_heads;
                continue;
            }
            const int32_t h = static_cast<int32_t>((target - at) / head);
            at += h * head;
            int b = 0, steps = e4_block_steps<ROWS, SK>(p, q, 0);
            while (target >= at + steps) {
                at += steps;
                steps = e4_block_steps<ROWS, SK>(p, q, ++b);
            }
            scratch[0] = (static_cast<int64_t>(r) << 32) | static_cast<uint32_t>(h);
            scratch[1] = (static_cast<int64_t>(b) << 32) | static_cast<uint32_t>(steps);
            scratch[2] = at;
            break;
        }
    }
    __syncthreads();
    const int64_t a = scratch[0], c = scratch[1], at = scratch[2];
    __syncthreads();
    place.r = __builtin_amdgcn_readfirstlane(static_cast<int32_t>(a >> 32));
    place.h = __builtin_amdgcn_readfirstlane(static_cast<int32_t>(a));
    place.b = __builtin_amdgcn_readfirstlane(static_cast<int32_t>(c >> 32));
    place.steps = __builtin_amdgcn_readfirstlane(static_cast<int32_t>(c));
    place.begin = e4_uniform(at);
    place.step = __builtin_amdgcn_readfirstlane(static_cast<int32_t>(target - place.begin));
    return true;
}

// Steps [first, last) of workgroup w: an equal share of all.  With fewer steps than workgroups the
// first `total` take one each.
__device__ __forceinline__ int64_t e4_first_step(int64_t total, int64_t workgroups, int64_t w) {
    const int64_t n = total < workgroups ? total : workgroups;
    return w >= n ? total : total * w / n;
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

// What a step needs, the same in every lane.
struct E4Step {
    int32_t r, h, b;
    int32_t key0, count;      // first key of the step among the prefix keys or the nodes, live keys
    int32_t tree;
    int32_t prefix, nodes, first_row;
    int64_t bias;
    int32_t first, last;      // of this workgroup's run through the block
    int32_t whole;            // the run is the whole block
    int32_t second;           // which of the workgroup's two workspace pieces the run writes
};

template <int D, int WM, int WK, int NBUF, class T, bool TWO>
__global__ void __launch_bounds__(64 * WM * WK, D == 256 ? 1 : 2)
e4m3_attention_kernel(const E4m3Params p) {
    constexpr int THREADS = 64 * WM * WK, ROWS = 32 * WM, SK = e4_step_keys(D);
    constexpr int LPR = D / 16;                    // lanes that move one key's row
    constexpr int KPP = THREADS / LPR;             // keys a pass of the workgroup moves
    constexpr int PASSES = SK / KPP;
    constexpr int TILES = SK / kE4Tile / WK;       // tiles a wave takes of a step
    constexpr int KB = SK * D * 2;                 // bytes of a step's K (or V) in LDS
    constexpr int NK = D / 16, NB = D / 32;        // MFMAs of a tile's scores; output blocks
    static_assert(SK % KPP == 0 && SK % (kE4Tile * WK) == 0, "a step is whole passes and tiles");
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

    // Neighbouring shares go to one XCD (workgroups are dealt to the 8 in turn), whose L2 then
    // holds what they have in common: the scales of a key's heads, the keys of a head's blocks.
    if (tid < NBUF) lds_bad[tid] = 0;   // the search's barriers follow
    const int W = p.workgroups;
    int64_t total = 0, s0 = 0, s1 = 0;
    int share = 0;
    E4Place at;
    const bool any = e4_find<ROWS, SK, THREADS>(p, lds_scan, total, at, [&](int64_t all) -> int64_t {
        share = all < W ? static_cast<int>(blockIdx.x) : static_cast<int>(blockIdx.x % 8 * (W / 8) + blockIdx.x / 8);
        s0 = e4_first_step(all, W, share);
        s1 = e4_first_step(all, W, share + 1);
        return s0 < s1 ? s0 : -1;
    });
    if (!any) return;
    s0 = e4_uniform(s0);
    s1 = e4_uniform(s1);
    int64_t todo = s1 - s0;

    // --- the order of steps -------------------------------------------------------------------
    E4Request req = e4_request<ROWS, SK>(p, at.r, false);
    int n_tree = e4_tree_keys<ROWS>(p, req, at.b);
    int run_first = 1;
    auto describe = [&](E4Step& s) {
        s.r = at.r;
        s.h = at.h;
        s.b = at.b;
        s.tree = at.step >= req.prefix_steps;
        s.key0 = (s.tree ? at.step - req.prefix_steps : at.step) * SK;
        const int rest = (s.tree ? n_tree : req.prefix) - s.key0;
        s.count = rest < SK ? rest : SK;
        s.prefix = req.prefix;
        s.nodes = req.nodes;
        s.first_row = req.first_row;
        s.bias = req.bias;
        s.first = run_first;
        s.last = at.step + 1 == at.steps || todo == 1;
        s.whole = at.begin >= s0 && at.begin + at.steps <= s1;
        s.second = at.begin >= s0;
        run_first = s.last;
    };
    auto advance = [&]() {
        --todo;
        if (++at.step < at.steps || todo <= 0) return;
        at.begin += at.steps;
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
        n_tree = e4_tree_keys<ROWS>(p, req, at.b);
    };

    // --- moving a step's keys -----------------------------------------------------------------
    const int my_key = tid / LPR, my_chunk = tid % LPR;
    int32_t entry[PASSES];
    u32x4 kreg[PASSES], vreg[PASSES];
    float ksr[PASSES], vsr[PASSES];
    uint32_t good = 0, wrong = 0;   // passes whose key is live and found / live and not found
    const int64_t pool_slots = static_cast<int64_t>(p.num_blocks) * p.block_size;

    auto fetch_entries = [&](const E4Step& s) {
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
            const int kk = i * KPP + my_key;
            entry[i] = -1;
            if (kk < s.count) {
                if (s.tree) {
                    const int64_t slot = p.tree_slots[s.first_row + s.key0 + kk];
                    entry[i] = slot >= 0 && slot < pool_slots ? static_cast<int32_t>(slot) : -1;
                } else {
                    entry[i] = p.tables[s.r * p.t_s0 + p.page_of(s.key0 + kk)];
                }
            }
        }
    };
    auto fetch_keys = [&](const E4Step& s) {
        good = wrong = 0;
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
            const int kk = i * KPP + my_key;
            const int32_t pos = s.tree ? entry[i] : s.key0 + kk;   // a slot or a position
            const int32_t quotient = p.page_of(pos < 0 ? 0 : pos);
            const int32_t page = s.tree ? (entry[i] < 0 ? -1 : quotient) : entry[i];
            const int32_t offset = pos - quotient * p.block_size;
            const bool live = kk < s.count, found = live && page >= 0 && page < p.num_blocks;
            kreg[i] = u32x4{0, 0, 0, 0};
            vreg[i] = u32x4{0, 0, 0, 0};
            ksr[i] = vsr[i] = 0.0f;
            if (found) {
                good |= 1u << i;
                kreg[i] = *reinterpret_cast<const u32x4*>(p.k + page * p.k_s0 + offset * p.k_s1 + s.h * p.k_s2 + 16 * my_chunk);
                vreg[i] = *reinterpret_cast<const u32x4*>(p.v + page * p.v_s0 + offset * p.v_s1 + s.h * p.v_s2 + 16 * my_chunk);
                ksr[i] = p.ks[page * p.kc_s0 + offset * p.kc_s1 + s.h * p.kc_s2];
                vsr[i] = p.vs[page * p.vc_s0 + offset * p.vc_s1 + s.h * p.vc_s2];
            } else if (live) {
                wrong |= 1u << i;
            }
        }
    };
    // Codes to LDS as bf16/f16 values, with the step's scales; `mark` tags the buffer if a key's
    // page was not found.
    auto stage = [&](const E4Step& s, int buf, int mark) {
        char* kb = lds + buf * 2 * KB;
        char* vb = kb + KB;
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
            const int kk = i * KPP + my_key;
            float vscale = vsr[i];
            if (s.tree) {
                // A product with a zero probability has to be zero: NaN codes of a node's V row turn
                // into a NaN scale, which only rows that see the node multiply by.
                uint32_t nan = 0;
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const uint32_t high = ((vreg[i][w] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
                    vreg[i][w] &= ~((high >> 7) * 0xffu);
                    nan |= high;
                }
                const uint64_t lanes = __ballot(nan != 0);
                if ((lanes >> (lane & ~(LPR - 1))) & ((1ull << LPR) - 1)) vscale = NAN;
            }
            u32x4 a, b;
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                a[2 * w] = E4Type<T>::template two<false>(kreg[i][w]);
                a[2 * w + 1] = E4Type<T>::template two<true>(kreg[i][w]);
                b[2 * w] = E4Type<T>::template two<false>(kreg[i][w + 2]);
                b[2 * w + 1] = E4Type<T>::template two<true>(kreg[i][w + 2]);
            }
            char* row = kb + kk * (2 * D);
            *reinterpret_cast<u32x4*>(row + 16 * e4_k_chunk<D>(kk, 2 * my_chunk)) = a;
            *reinterpret_cast<u32x4*>(row + 16 * e4_k_chunk<D>(kk, 2 * my_chunk + 1)) = b;
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                a[2 * w] = E4Type<__bf16>::two<false>(vreg[i][w]);
                a[2 * w + 1] = E4Type<__bf16>::two<true>(vreg[i][w]);
                b[2 * w] = E4Type<__bf16>::two<false>(vreg[i][w + 2]);
                b[2 * w + 1] = E4Type<__bf16>::two<true>(vreg[i][w + 2]);
            }
            row = vb + kk * (2 * D);
            *reinterpret_cast<u32x4*>(row + 16 * e4_v_chunk<D>(kk, 2 * my_chunk)) = a;
            *reinterpret_cast<u32x4*>(row + 16 * e4_v_chunk<D>(kk, 2 * my_chunk + 1)) = b;
            if (my_chunk == 0) {
                lds_ks[buf][kk] = ksr[i] * p.c;
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

    auto start_block = [&](const E4Step& s) {
        const int row = s.b * ROWS + 32 * wm + c;
        wave_rows = s.b * ROWS + 32 * wm < s.nodes * p.groups;
        const int n = row / p.groups;
        node = n < s.nodes ? n : -1;
        qhead = s.h * p.groups + row - n * p.groups;
#pragma unroll
        for (int i = 0; i < NK; ++i) {
            u32x4 x = {0, 0, 0, 0};
            if (node >= 0) {
                const T* src = static_cast<const T*>(p.q) + static_cast<int64_t>(s.first_row + node) * p.q_s0 +
                               qhead * p.q_s1 + 16 * i + 8 * half;
                x = *reinterpret_cast<const u32x4*>(src);
            }
            qb[i] = __builtin_bit_cast(V8, x);
        }
#pragma unroll
        for (int i = 0; i < NB; ++i) acc[i] = e4_f32x16{};
        m = -INFINITY;
        l = 0.0f;
    };

    auto tile = [&](const E4Step& s, int buf, int t, bool masked) {
        const char* kb = lds + buf * 2 * KB + t * kE4Tile * 2 * D;
        const char* vb = kb + KB;
        e4_f32x16 x = {};
#pragma unroll
        for (int i = 0; i < NK; ++i) {
            const u32x4 a = *reinterpret_cast<const u32x4*>(kb + c * 2 * D + 16 * e4_k_chunk<D>(c, 2 * i + half));
            x = E4Type<T>::run(__builtin_bit_cast(V8, a), qb[i], x);
        }
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const e4_f32x4 ks = *reinterpret_cast<const e4_f32x4*>(&lds_ks[buf][t * kE4Tile + 8 * g + 4 * half]);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[4 * g + e] *= ks[e];
        }
        if (masked) {
            const float* bias = p.bias + s.bias + static_cast<int64_t>(node < 0 ? 0 : node) * s.nodes;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int kk = t * kE4Tile + 8 * (i >> 2) + 4 * half + (i & 3);
                float add = lds_kb[buf][kk];
                if (s.tree) {
                    const int of = s.key0 + kk;
                    const bool seen = kk < s.count && of <= node;
                    const float b = bias[seen ? of : 0];
                    // In score units; a finite bias stays finite.
                    float b2 = b * 1.44269504088896340736f;
                    if (fabsf(b2) == INFINITY && fabsf(b) != INFINITY) b2 = copysignf(FLT_MAX, b2);
                    add = seen && add == 0.0f ? b2 : -INFINITY;
                }
                x[i] = add == -INFINITY ? -INFINITY : x[i] + add;
            }
        }
        float top = x[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) top = fmaxf(top, x[i]);
        top = e4_pair_max(top);
        // The reference maximum is raised only when a tile passes it by 2^8: until then the
        // probabilities stay below 2^8, which costs no precision.
        if (__any(top > m + 8.0f)) {
            const float raised = fmaxf(m, top);
            const float factor = raised == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - raised);
            m = raised;
            l *= factor;
#pragma unroll
            for (int i = 0; i < NB; ++i) acc[i] *= factor;
        }
        const float ref = m == -INFINITY ? 0.0f : m;
        e4_bf16x8 pb[2], pl[2];
        float sum = 0.0f;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const e4_f32x4 vs = *reinterpret_cast<const e4_f32x4*>(&lds_vs[buf][t * kE4Tile + 8 * g + 4 * half]);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int i = 4 * g + e;
                const float pr = __builtin_amdgcn_exp2f(x[i] - ref);
                sum += pr;
                float pv = pr * vs[e];
                if (masked && x[i] == -INFINITY) pv = 0.0f;   // whatever the key's scale is
                const __bf16 hi = static_cast<__bf16>(pv);
                pb[i >> 3][i & 7] = hi;
                if constexpr (TWO) pl[i >> 3][i & 7] = static_cast<__bf16>(pv - static_cast<float>(hi));
            }
        }
        l += sum;
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
#pragma unroll
            for (int db = 0; db < NB; ++db) {
                const int s16 = lane & 15, group = lane >> 4;
                const int key = 16 * kk + 4 * half + (s16 >> 2);
                const int dim = 32 * db + 16 * (group & 1) + 4 * (s16 & 3);
                const char* lo = vb + key * 2 * D + 16 * e4_v_chunk<D>(key, dim >> 3) + 2 * (dim & 7);
                const char* hi = vb + (key + 8) * 2 * D + 16 * e4_v_chunk<D>(key + 8, dim >> 3) + 2 * (dim & 7);
                const e4_i16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((e4_lds_i16x4*)lo);
                const e4_i16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((e4_lds_i16x4*)hi);
                const e4_bf16x8 v8 = __builtin_bit_cast(e4_bf16x8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
                acc[db] = E4Type<__bf16>::run(v8, pb[kk], acc[db]);
                if constexpr (TWO) acc[db] = E4Type<__bf16>::run(v8, pl[kk], acc[db]);
            }
        }
    };

    // A finished run: the row's output, or its unnormalised sum with (m, l) for the merge.
    auto put = [&](const E4Step& s, int row_in_block, int row_node, int head, int dim, e4_f32x4 v, float row_l) {
        if (s.whole) {
            const float scale = row_l == 0.0f ? 0.0f : 1.0f / row_l;   // a row that sees nothing is zero
            e4_store4<T>(p, s.first_row + row_node, head, dim, v * scale);
        } else {
            const int64_t piece = 2 * static_cast<int64_t>(share) + s.second;
            *reinterpret_cast<e4_f32x4*>(p.ws_o + (piece * ROWS + row_in_block) * D + dim) = v;
        }
    };
    auto finish = [&](const E4Step& s) {
        l = e4_pair_sum(l);
        const int64_t piece = 2 * static_cast<int64_t>(share) + s.second;
        if constexpr (WK == 1) {
            if (node >= 0) {
#pragma unroll
                for (int db = 0; db < NB; ++db) {
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        const e4_f32x4 v = {acc[db][4 * g], acc[db][4 * g + 1], acc[db][4 * g + 2], acc[db][4 * g + 3]};
                        put(s, 32 * wm + c, node, qhead, 32 * db + 8 * g + 4 * half, v, l);
                    }
                }
                if (!s.whole && half == 0) p.ws_ml[piece * ROWS + 32 * wm + c] = make_float2(m, l);
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
                    const int in_block = 32 * g0 + row, of = s.b * ROWS + in_block;
                    const int n = of / p.groups;
                    if (n >= s.nodes) continue;
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
                    put(s, in_block, n, s.h * p.groups + of - n * p.groups, 4 * ch, v, sum);
                    if (!s.whole && ch == 0) p.ws_ml[piece * ROWS + in_block] = make_float2(best, sum);
                }
                __syncthreads();
            }
        }
    };

    // --- the run ------------------------------------------------------------------------------
    E4Step now, next, after;
    int count = 1;   // steps begun, the mark of a buffer with a missing page
    describe(now);
    fetch_entries(now);
    fetch_keys(now);
    advance();
    bool more = todo > 0;
    if (more) {
        describe(next);
        fetch_entries(next);
        advance();
    }
    for (int buf = 0;; buf = NBUF == 2 ? buf ^ 1 : 0, ++count) {
        if (NBUF == 1) __syncthreads();   // the last step's reads of the buffer are done
        stage(now, buf, count);
        if (more) {
            fetch_keys(next);
            if (todo > 0) {
                describe(after);
                fetch_entries(after);
            }
        }
        if (now.first) start_block(now);
        __syncthreads();
        if (wave_rows) {
            const bool masked = now.tree || now.count < SK || lds_bad[buf] == count;
            if (masked) {
                for (int t = wk; t * kE4Tile < now.count; t += WK) tile(now, buf, t, true);
            } else {
#pragma unroll 1
                for (int t = 0; t < TILES; ++t) tile(now, buf, t * WK + wk, false);
            }
        }
        if (now.last) finish(now);
        if (!more) break;
        more = todo > 0;
        now = next;
        if (more) {
            next = after;
            advance();
        }
    }
}

template <int D, int WM, int WK, int NBUF>
void e4_launch(const E4m3Params& p, bool bf16, bool two, hipStream_t s) {
    const dim3 grid(p.workgroups), block(64 * WM * WK);
    if (bf16 && !two) hipLaunchKernelGGL((e4m3_attention_kernel<D, WM, WK, NBUF, __bf16, false>), grid, block, 0, s, p);
    else if (bf16) hipLaunchKernelGGL((e4m3_attention_kernel<D, WM, WK, NBUF, __bf16, true>), grid, block, 0, s, p);
    else hipLaunchKernelGGL((e4m3_attention_kernel<D, WM, WK, NBUF, _Float16, true>), grid, block, 0, s, p);
}

}  // namespace
}  // namespace tv
