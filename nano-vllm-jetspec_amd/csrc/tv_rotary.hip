// Rotation of queries and keys from positions and frequencies, with the K/V scatter, for gfx950.
//
// Row i at position P, pair (a, b) = (x[p], x[n + p]) of a head, or (x[2p], x[2p + 1]) where pairs are
// interleaved, p < n:
//     t = P f_p / 2 pi,   (a, b) -> g (a cos 2 pi t - b sin 2 pi t,  b cos 2 pi t + a sin 2 pi t);
// dimensions from 2n on are copied, as V is.  The turns t are taken in 64 bits and reduced there to at most an
// eighth of a turn from a multiple of a quarter, which an fp32 number holds to 2^-28 turns (at positions near 2^31
// the 64-bit product's own rounding is 2^-24 turns); what follows is fp32, rounded once when it is stored.  No
// table: positions have no longest one, and the only memory an angle costs is the frequencies, which stay in the
// caches.
//
// GS lanes hold one head of one row, each VEC dimensions in either of two places: pairs stay in the lane.
// A wave passes over heads of one row, 64 / GS at a time, with its angles in registers; it computes them
// once, an angle a lane, and deals them out through LDS while the first heads are on their way.  A pass's
// elements are loaded while the one before it is computed.
//
// Memory bounds it: 4096 rows of 32 + 8 heads of 128 in bf16 with 64 dimensions turned, 101 MB, 18.0 us (5.6 TB/s) out
// of the Infinity Cache and 26.0 (3.9) out of memory, where a copy of as many bytes takes 15.6 and 21.0; 6001 fp32 rows
// of 10 + 5 heads of 80, 77 MB, 15.2 and 22.  16 rows 3.7 us: a launch and three dependent loads.
#include <math.h>
#include <stdint.h>

#include "tv_internal.h"

namespace tv {
namespace {

struct Bf16 {
    typedef uint16_t storage;
    static __device__ __forceinline__ float load(storage s) { return __uint_as_float(static_cast<uint32_t>(s) << 16); }
    static __device__ __forceinline__ storage store(float f) {
        return __builtin_bit_cast(uint16_t, static_cast<__bf16>(f));
    }
};

struct F16 {
    typedef uint16_t storage;
    static __device__ __forceinline__ float load(storage s) { return static_cast<float>(__builtin_bit_cast(_Float16, s)); }
    static __device__ __forceinline__ storage store(float f) {
        return __builtin_bit_cast(uint16_t, static_cast<_Float16>(f));
    }
};

struct F32 {
    typedef float storage;
    static __device__ __forceinline__ float load(storage s) { return s; }
    static __device__ __forceinline__ storage store(float f) { return f; }
};

// A tensor [rows, heads, dim] that is read (element strides).
struct Source {
    const void* data;
    int64_t s0, s1, s2;
};

// A tensor that is written: the output [rows, -, heads, dim] or a pool [pages, page_size, heads, dim].
struct Target {
    void* data;
    int64_t s0, s1, s2, s3;
};

struct RotaryParams {
    Source src[3];   // queries, keys, values
    Target dst[3];   // the output, the key pool, the value pool
    const void* positions;
    int64_t pos_s;
    int32_t pos64;
    const double* frequencies;
    int32_t pairs;   // n
    int32_t interleaved;
    float gain;
    int64_t pool_pages, page_size;
    const void* slots;
    int64_t slot_s;
    int32_t slot64;
    int64_t rows;
    int32_t q_heads, kv_heads, head_dim;
    int32_t passes_per_wave;
    int32_t* status;
};

constexpr int kMostPairs = 128;
constexpr int64_t kMostPosition = 0x7fffffff;

template <int BYTES>
struct Piece;
template <>
struct Piece<16> { typedef u32x4 type; };
template <>
struct Piece<8> { typedef u32x2 type; };
template <>
struct Piece<4> { typedef uint32_t type; };
template <>
struct Piece<2> { typedef uint16_t type; };

// VEC consecutive elements (the host takes VEC > 1 for unit strides and alignment).
template <typename S, int VEC>
__device__ __forceinline__ void load_elems(const S* p, S (&out)[VEC]) {
    typedef typename Piece<VEC * sizeof(S)>::type P;
    const P raw = *reinterpret_cast<const P*>(p);
    __builtin_memcpy(out, &raw, sizeof(P));
}

template <typename S, int VEC>
__device__ __forceinline__ void store_elems(S* p, const S (&in)[VEC]) {
    typedef typename Piece<VEC * sizeof(S)>::type P;
    P raw;
    __builtin_memcpy(&raw, in, sizeof(P));
    *reinterpret_cast<P*>(p) = raw;
}

// INTER: pairs are neighbours inside a lane's VEC dimensions; else a pair is one dimension from either
// place (VEC 1: of any layout).
template <class T, int VEC, int GS, int NP, bool INTER>
__global__ void __launch_bounds__(256)
rotary_kernel(const RotaryParams) {
    typedef typename T::storage S;
    // The arguments where they are: the tables of tensors are indexed.
    typedef const __attribute__((address_space(4))) RotaryParams* Params;
    const Params p = (Params)__builtin_amdgcn_kernarg_segment_ptr();
    __shared__ __attribute__((aligned(16))) float angles[4][2][kMostPairs];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + wave;
    if (row >= p->rows) return;
    const int part = blockIdx.y;
    const int pairs = p->pairs, half = p->head_dim >> 1;
    constexpr int kGroups = 64 / GS;
    const int lane = threadIdx.x & (GS - 1), group = (threadIdx.x & 63) / GS;

    // The lane's dimensions: VEC from `first` and VEC from `second`; whether they turn, and their first pair.
    int first[NP], second[NP], pair[NP];
    bool live[NP], turns[NP];
#pragma unroll
    for (int n = 0; n < NP; ++n) {
        const int j = (lane + n * GS) * VEC;   // pairs before it, counted over the whole head
        live[n] = j < half;
        turns[n] = j < pairs;
        pair[n] = turns[n] ? j : 0;
        if (!live[n]) first[n] = second[n] = 0;   // lanes without dimensions load others' and drop them
        else if (INTER || (VEC == 1 && p->interleaved)) first[n] = 2 * j, second[n] = 2 * j + VEC;
        else if (turns[n]) first[n] = j, second[n] = pairs + j;
        else first[n] = pairs + j, second[n] = half + j;   // 2 n + (j - n), and half of what is copied further
    }
    // Passes of the wave over the row's heads: queries, keys, values, a head per group of lanes.
    const int nq = (p->q_heads + kGroups - 1) / kGroups, nk = (p->kv_heads + kGroups - 1) / kGroups;
    const int pass0 = part * p->passes_per_wave;
    const int pass1 = min(pass0 + p->passes_per_wave, nq + 2 * nk);
    const int kind0 = pass0 < nq ? 0 : pass0 < nq + nk ? 1 : 2;
    const int done0 = (pass0 - (kind0 == 0 ? 0 : kind0 == 1 ? nq : nq + nk)) * kGroups;

    // What is loaded next: from `src` on, `src_left` heads of source `src_kind`.
    const S* src;
    int64_t src_step, src_group, src_a[NP], src_b[NP];
    int src_left, src_kind;
    auto enter_source = [&](int kind, int done) {
        src_kind = kind;
        src = static_cast<const S*>(p->src[kind].data) + row * p->src[kind].s0 + done * p->src[kind].s1;
        src_step = kGroups * p->src[kind].s1;
        src_group = group * p->src[kind].s1;
        src_left = (kind == 0 ? p->q_heads : p->kv_heads) - done;
#pragma unroll
        for (int n = 0; n < NP; ++n) {
            src_a[n] = src_group + first[n] * p->src[kind].s2;
            src_b[n] = src_group + second[n] * p->src[kind].s2;
        }
    };
    S a[NP][VEC], b[NP][VEC];   // a pass's elements
    auto load = [&]() {
        if (src_left <= 0) enter_source(src_kind + 1, 0);
        const int64_t back = group < src_left ? 0 : src_group;   // no such head: the first one's, dropped
#pragma unroll
        for (int n = 0; n < NP; ++n) {
            load_elems<S, VEC>(src + (src_a[n] - back), a[n]);
            load_elems<S, VEC>(src + (src_b[n] - back), b[n]);
        }
        src += src_step;
        src_left -= kGroups;
    };
    enter_source(kind0, done0);
    load();   // on its way while the slot and the position are read

    const int64_t slot = p->slot64 ? static_cast<const int64_t*>(p->slots)[row * p->slot_s]
                                   : static_cast<int64_t>(static_cast<const int32_t*>(p->slots)[row * p->slot_s]);
    const int64_t pos = p->pos64 ? static_cast<const int64_t*>(p->positions)[row * p->pos_s]
                                 : static_cast<int64_t>(static_cast<const int32_t*>(p->positions)[row * p->pos_s]);
    if (slot == -1) return;   // a padding row
    if (pos < 0 || pos > kMostPosition) {
        if (part == 0 && (threadIdx.x & 63) == 0) set_status(p->status, TV_STATUS_BAD_POSITION);
        return;
    }
    if (slot < 0 || slot >= p->pool_pages * p->page_size) {
        if (part == 0 && (threadIdx.x & 63) == 0) set_status(p->status, TV_STATUS_BAD_SLOT);
        return;
    }
    float cs[NP][VEC], sn[NP][VEC];
    if (kind0 < 2) {
        for (int i = threadIdx.x & 63; i < pairs; i += 64) {
            double turn = static_cast<double>(pos) * p->frequencies[i] * 0.15915494309189533577;
            turn -= rint(turn);
            const double quarter = rint(4.0 * turn);   // -2 to 2, and what is left at most an eighth
            float s, c;
            sincospif(2.0f * static_cast<float>(turn - 0.25 * quarter), &s, &c);
            const int q = static_cast<int>(quarter);
            const float cq = q & 1 ? s : c, sq = q & 1 ? c : s;
            angles[wave][0][i] = (q + 1) & 2 ? -cq * p->gain : cq * p->gain;
            angles[wave][1][i] = q & 2 ? -sq * p->gain : sq * p->gain;
        }
        // One wave's exchange: its LDS operations run in order, the compiler's must too.
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
        for (int n = 0; n < NP; ++n) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                cs[n][e] = angles[wave][0][pair[n] + e];
                sn[n][e] = angles[wave][1][pair[n] + e];
            }
        }
    }
    // A 64-bit division is some 120 dependent instructions; nearly every pool's slots fit 32 bits.
    const bool narrow = ((static_cast<uint64_t>(slot) | static_cast<uint64_t>(p->page_size)) >> 32) == 0;
    const int64_t page = narrow ? static_cast<uint32_t>(slot) / static_cast<uint32_t>(p->page_size) : slot / p->page_size;
    const int64_t offset = slot - page * p->page_size;

    // Where the pass under way goes, in the same manner: the output's row, or the slot's in a pool.
    S* dst;
    int64_t dst_step, dst_a[NP], dst_b[NP];
    int left, kind;
    auto enter_target = [&](int which, int done) {
        kind = which;
        const int64_t per_head = p->dst[kind].s2, per_dim = p->dst[kind].s3;
        const int64_t outer = kind == 0 ? row : page, inner = kind == 0 ? 0 : offset;
        dst = static_cast<S*>(p->dst[kind].data) + outer * p->dst[kind].s0 + inner * p->dst[kind].s1 + done * per_head;
        dst_step = kGroups * per_head;
        left = (kind == 0 ? p->q_heads : p->kv_heads) - done;
#pragma unroll
        for (int n = 0; n < NP; ++n) {
            dst_a[n] = group * per_head + first[n] * per_dim;
            dst_b[n] = group * per_head + second[n] * per_dim;
        }
    };
    enter_target(kind0, done0);
    for (int pass = pass0; pass < pass1; ++pass) {
        if (left <= 0) enter_target(kind + 1, 0);
        S y[NP][VEC], z[NP][VEC];
#pragma unroll
        for (int n = 0; n < NP; ++n) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                y[n][e] = a[n][e];
                z[n][e] = b[n][e];
            }
        }
        if (pass + 1 < pass1) load();
#pragma unroll
        for (int n = 0; n < NP; ++n) {
            if (kind < 2 && turns[n]) {   // what does not turn is copied, bit for bit
                if constexpr (INTER) {
#pragma unroll
                    for (int e = 0; e < VEC; e += 2) {
                        const float y1 = T::load(y[n][e]), y2 = T::load(y[n][e + 1]);
                        const float z1 = T::load(z[n][e]), z2 = T::load(z[n][e + 1]);
                        const float c1 = cs[n][e / 2], s1 = sn[n][e / 2], c2 = cs[n][(VEC + e) / 2], s2 = sn[n][(VEC + e) / 2];
                        y[n][e] = T::store(y1 * c1 - y2 * s1);
                        y[n][e + 1] = T::store(y2 * c1 + y1 * s1);
                        z[n][e] = T::store(z1 * c2 - z2 * s2);
                        z[n][e + 1] = T::store(z2 * c2 + z1 * s2);
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < VEC; ++e) {
                        const float x1 = T::load(y[n][e]), x2 = T::load(z[n][e]);
                        y[n][e] = T::store(x1 * cs[n][e] - x2 * sn[n][e]);
                        z[n][e] = T::store(x2 * cs[n][e] + x1 * sn[n][e]);
                    }
                }
            }
            if (group < left && live[n]) {
                store_elems<S, VEC>(dst + dst_a[n], y[n]);
                store_elems<S, VEC>(dst + dst_b[n], z[n]);
            }
        }
        dst += dst_step;
        left -= kGroups;
    }
}

// Waves that fill the chip's 1024 SIMDs: with fewer rows than that a row's heads are spread over
// several waves, since what counts there is the latency of one.  16 / 256 / 1024 / 2048 rows of 32 + 8 heads of 128 in
// bf16 3.7 / 4.2 / 6.3 / 9.9 us; with 2048 waves 3.7 / 4.2 / 6.5 / 10.6, with 8192 3.7 / 4.2 / 6.6 / 10.3, with a wave a
// row 5.9 / 6.2 / 7.3 / 10.6.
constexpr int64_t kFullWaves = 4096;

template <class T, int VEC, int GS, int NP, bool INTER>
int enqueue(RotaryParams& p, hipStream_t stream) {
    constexpr int kGroups = 64 / GS;
    const int passes = (p.q_heads + kGroups - 1) / kGroups + 2 * ((p.kv_heads + kGroups - 1) / kGroups);
    int64_t waves = (kFullWaves + p.rows - 1) / p.rows;
    waves = waves < passes ? waves : passes;
    p.passes_per_wave = static_cast<int>((passes + waves - 1) / waves);
    const dim3 grid(static_cast<uint32_t>((p.rows + 3) / 4), (passes + p.passes_per_wave - 1) / p.passes_per_wave);
    hipLaunchKernelGGL((rotary_kernel<T, VEC, GS, NP, INTER>), grid, dim3(256), 0, stream, p);
    return check_launch("rotary_scatter");
}

template <class T, int VEC, bool INTER>
int by_lanes(RotaryParams& p, hipStream_t stream) {
    const int lanes = (p.head_dim / 2 + VEC - 1) / VEC;   // at most 128 / VEC
    if (lanes <= 8) return enqueue<T, VEC, 8, 1, INTER>(p, stream);
    if (VEC == 8 || lanes <= 16) return enqueue<T, VEC, 16, 1, INTER>(p, stream);
    if constexpr (VEC < 8) {
        if (VEC == 4 || lanes <= 32) return enqueue<T, VEC, 32, 1, INTER>(p, stream);
    }
    if constexpr (VEC < 4) return enqueue<T, VEC, 64, 1, INTER>(p, stream);
    return TV_OK;
}

// VEC dimensions a lane in either place: both the pairs and what is copied have to be whole pieces, and
// every address a multiple of one.  Pieces of 16 and 8 bytes are built, and single elements for whatever else: 4096 rows
// of 32 + 8 heads of 80 in bf16 with 16 / 40 / 20 turned dimensions (8, 20, 10 pairs) 13.6 / 15.1 / 31.1 us.
template <class T>
int by_size(RotaryParams& p, int64_t vec, hipStream_t stream) {
    constexpr int kVec = 16 / sizeof(typename T::storage);
    if (p.pairs % vec || (p.head_dim / 2) % vec) vec /= 2;
    if (p.pairs % vec || (p.head_dim / 2) % vec) vec /= 2;
    if (p.pairs % vec || (p.head_dim / 2) % vec) vec = 1;
    if (vec == kVec) return p.interleaved ? by_lanes<T, kVec, true>(p, stream) : by_lanes<T, kVec, false>(p, stream);
    if (vec == kVec / 2) return p.interleaved ? by_lanes<T, kVec / 2, true>(p, stream) : by_lanes<T, kVec / 2, false>(p, stream);
    return enqueue<T, 1, 64, 2, false>(p, stream);
}

// The widest piece, of up to 16 bytes, whose multiples the rows and heads start at.
int64_t piece_of(const void* ptr, const int64_t* stride, int n, int64_t elem, int64_t most) {
    if (stride[n - 1] != 1) return 1;
    for (int64_t v = most; v > 1; v /= 2) {
        bool ok = aligned(ptr, v * elem);
        for (int i = 0; i < n - 1; ++i) ok = ok && stride[i] % v == 0;
        if (ok) return v;
    }
    return 1;
}

bool all_positive(const int64_t* stride, int n) {
    for (int i = 0; i < n; ++i) {
        if (stride[i] <= 0) return false;
    }
    return true;
}

}  // namespace
}  // namespace tv

using namespace tv;

extern "C" int64_t tv_sizeof_rotary_args(void) { return static_cast<int64_t>(sizeof(tv_rotary_args)); }

extern "C" int tv_rotary_scatter(const tv_rotary_args* args, void* stream) {
    clear_error();
    const char* what = "rotary_scatter";
    if (!args) return fail(TV_ERR_INVALID, "%s: null args", what);
    const tv_rope_scatter_args* a = &args->rope;
    if (a->rows < 0 || a->q_heads < 1 || a->kv_heads < 1 || a->q_heads % a->kv_heads) {
        return fail(TV_ERR_INVALID, "%s: invalid GQA geometry (%d query heads, %d KV heads)", what, a->q_heads, a->kv_heads);
    }
    if (a->head_dim < 2 || a->head_dim % 2 || a->head_dim > 256) {
        return fail(TV_ERR_INVALID, "%s: head_dim %d must be even and in [2, 256]", what, a->head_dim);
    }
    if (args->num_frequencies < 1 || args->num_frequencies > a->head_dim / 2) {
        return fail(TV_ERR_INVALID, "%s: %d frequencies for a head of %d", what, args->num_frequencies, a->head_dim);
    }
    if (a->dtype != TV_BF16 && a->dtype != TV_F16 && a->dtype != TV_F32) {
        return fail(TV_ERR_UNSUPPORTED, "%s: operands must be bf16, f16 or fp32", what);
    }
    if (!(fabsf(args->gain) <= 3.0e38f)) return fail(TV_ERR_INVALID, "%s: gain must be finite", what);
    if (a->rows == 0) return TV_OK;
    if (a->rows > 0x7fffffff) return fail(TV_ERR_UNSUPPORTED, "%s: too many rows", what);
    if (!a->q || !a->k || !a->v || !a->positions || !args->frequencies || !a->k_pool || !a->v_pool || !a->node_slots || !a->out) {
        return fail(TV_ERR_INVALID, "%s: null pointer", what);
    }
    if (!aligned(args->frequencies, 8)) return fail(TV_ERR_INVALID, "%s: unaligned frequencies", what);
    if (a->pool_pages < 1 || a->page_size < 1) return fail(TV_ERR_INVALID, "%s: empty KV pool", what);
    if (!all_positive(a->q_stride, 3) || !all_positive(a->k_stride, 3) || !all_positive(a->v_stride, 3) ||
        !all_positive(a->out_stride, 3) || !all_positive(a->k_pool_stride, 4) || !all_positive(a->v_pool_stride, 4) ||
        a->positions_stride <= 0 || a->slots_stride <= 0) {
        return fail(TV_ERR_INVALID, "%s: strides must be positive", what);
    }
    const int64_t elem = a->dtype == TV_F32 ? 4 : 2;
    int64_t vec = 16 / elem;
    vec = piece_of(a->q, a->q_stride, 3, elem, vec);
    vec = piece_of(a->k, a->k_stride, 3, elem, vec);
    vec = piece_of(a->v, a->v_stride, 3, elem, vec);
    vec = piece_of(a->out, a->out_stride, 3, elem, vec);
    vec = piece_of(a->k_pool, a->k_pool_stride, 4, elem, vec);
    vec = piece_of(a->v_pool, a->v_pool_stride, 4, elem, vec);
    RotaryParams p = {};
    p.src[0] = {a->q, a->q_stride[0], a->q_stride[1], a->q_stride[2]};
    p.src[1] = {a->k, a->k_stride[0], a->k_stride[1], a->k_stride[2]};
    p.src[2] = {a->v, a->v_stride[0], a->v_stride[1], a->v_stride[2]};
    p.dst[0] = {a->out, a->out_stride[0], 0, a->out_stride[1], a->out_stride[2]};
    p.dst[1] = {a->k_pool, a->k_pool_stride[0], a->k_pool_stride[1], a->k_pool_stride[2], a->k_pool_stride[3]};
    p.dst[2] = {a->v_pool, a->v_pool_stride[0], a->v_pool_stride[1], a->v_pool_stride[2], a->v_pool_stride[3]};
    p.positions = a->positions;
    p.pos_s = a->positions_stride;
    p.pos64 = a->positions_is_int64 != 0;
    p.frequencies = args->frequencies;
    p.pairs = args->num_frequencies;
    p.interleaved = args->interleaved != 0;
    p.gain = args->gain;
    p.pool_pages = a->pool_pages;
    p.page_size = a->page_size;
    p.slots = a->node_slots;
    p.slot_s = a->slots_stride;
    p.slot64 = a->slots_is_int64 != 0;
    p.rows = a->rows;
    p.q_heads = a->q_heads;
    p.kv_heads = a->kv_heads;
    p.head_dim = a->head_dim;
    p.status = a->status;
    if (a->dtype == TV_BF16) return by_size<Bf16>(p, vec, as_stream(stream));
    if (a->dtype == TV_F16) return by_size<F16>(p, vec, as_stream(stream));
    return by_size<F32>(p, vec, as_stream(stream));
}
