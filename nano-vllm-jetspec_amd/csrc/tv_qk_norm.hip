// Per-head RMS norm of the queries and keys with the HF-order rotation and the K/V scatter in one
// pass, and the append of K/V rows to an 8-bit cache, for gfx950.
//
// Row i, head h, x = q[i, h] or k[i, h]:
//     y = x * rsqrt(mean(x^2) + eps) * w,   z = [y1*cos - y2*sin | y2*cos + y1*sin]
// over the halves y1, y2 of the head, cos/sin from the cache row of the row's position.  Everything
// is fp32 and rounded once when it is stored: z(q) to `out`, z(k) and v to the slot's page.  An
// 8-bit (e4m3) pool takes a K or V row x of one head as
//     scale = max(amax|x| / 448, 2^-100),   code = rne(x * (1 / scale))
// with the scale beside the pool, so a read of code * scale is within half an e4m3 step of x.  A row
// that holds an infinity or a NaN gets a NaN scale and zero codes: it reads as NaN, and no code of
// the pool ever is one.
//
// GS lanes hold one head of one row, each VEC consecutive dimensions of the first half and the
// matching ones of the second, so the rotation stays in the lane and the norm is a sum over GS lanes
// (DPP, no LDS).  A wave passes over heads of one row, 64 / GS at a time: the position, the slot, and the
// weights times the angles are in registers for all of them, and a pass's elements are loaded while
// the one before it is computed.
//
// Memory bounds it.  4096 rows of 32 query and 8 KV heads of 128 in bf16 to an e4m3 pool are 95 MB in
// 19.4 us, 4.9 TB/s; a copy that moves as much takes 12.1.  To a bf16 pool 103 MB in 19.2 us (5.4 TB/s), fp32
// operands to an fp32 pool 203 MB in 33.0 (6.2), to an e4m3 pool 179 MB in 30.8 (5.8).  Without the arithmetic the
// first is 19.3 us, without the stores 12.9, without all loads but each wave's first 16.5.  Where the rows go
// does not matter: 19.3 us with the slots (and positions) in order.  What did not help: loads two and three
// passes ahead, non-temporal loads or stores, 16-byte stores of codes, and waves that begin at different heads.
// The append alone, 8192 rows of 8 heads of 128: 11.3 us in bf16 (4.5 TB/s, in order too), 15.0 in fp32 (5.6).
#include <math.h>
#include <stdint.h>

#include "tv_internal.h"

namespace tv {
namespace {

constexpr float kE4m3Max = 448.0f;
constexpr float kMinScale = 0x1p-100f;

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

// A tensor that is written: the output [rows, -, heads, dim], or a K/V pool [pages, page_size, heads, dim]
// (element strides) and, for e4m3 codes, its scales [pages, page_size, heads].
struct Target {
    void* data;
    int64_t s0, s1, s2, s3;
    float* scale;
    int64_t c0, c1, c2;
};

struct NormParams {
    Source src[3];   // queries, keys, values
    Target dst[3];   // the output, the key pool, the value pool
    const void* qw;
    const void* kw;
    int32_t weight_f32;
    const void* positions;
    int64_t pos_s;
    int32_t pos64;
    const void* cache;
    int64_t cache_rows, cache_s0, cache_s1;
    int32_t cache_f32, cache_vec;
    int64_t pool_pages, page_size;
    const void* slots;
    int64_t slot_s;
    int32_t slot64;
    int64_t rows;
    int32_t q_heads, kv_heads, head_dim;
    int32_t passes_per_wave;
    float eps, inverse_dim;
    int32_t* status;
};

template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
    return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), CTRL, 0xf, 0xf, true));
}

// Sum / maximum over aligned groups of GS lanes, the same bits in every lane: after a step over 2^k
// lanes they agree inside 2^k, so the mirrors exchange whole groups as an xor would.
template <int GS>
__device__ __forceinline__ float group_sum(float x) {
    if constexpr (GS >= 2) x += dpp<0xB1>(x);     // quad_perm [1,0,3,2]
    if constexpr (GS >= 4) x += dpp<0x4E>(x);     // quad_perm [2,3,0,1]
    if constexpr (GS >= 8) x += dpp<0x141>(x);    // row_half_mirror
    if constexpr (GS >= 16) x += dpp<0x140>(x);   // row_mirror
    if constexpr (GS >= 32) x += __shfl_xor(x, 16);
    if constexpr (GS >= 64) x += __shfl_xor(x, 32);
    return x;
}

template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t x) {
    return __builtin_amdgcn_update_dpp(0, x, CTRL, 0xf, 0xf, true);
}

template <int GS>
__device__ __forceinline__ uint32_t group_max(uint32_t x) {
    if constexpr (GS >= 2) x = max(x, dpp<0xB1>(x));
    if constexpr (GS >= 4) x = max(x, dpp<0x4E>(x));
    if constexpr (GS >= 8) x = max(x, dpp<0x141>(x));
    if constexpr (GS >= 16) x = max(x, dpp<0x140>(x));
    if constexpr (GS >= 32) x = max(x, static_cast<uint32_t>(__shfl_xor(static_cast<int>(x), 16)));
    if constexpr (GS >= 64) x = max(x, static_cast<uint32_t>(__shfl_xor(static_cast<int>(x), 32)));
    return x;
}

// VEC consecutive elements (16 bytes: the host takes this form for unit strides and alignment), or one.
template <typename S, int VEC>
__device__ __forceinline__ void load_elems(const S* p, S (&out)[VEC]) {
    if constexpr (VEC > 1) {
        static_assert(VEC * sizeof(S) == 16, "vector path moves 16 bytes");
        const u32x4 raw = *reinterpret_cast<const u32x4*>(p);
        __builtin_memcpy(out, &raw, 16);
    } else {
        out[0] = p[0];
    }
}

template <typename S, int VEC>
__device__ __forceinline__ void store_elems(S* p, const S (&in)[VEC]) {
    if constexpr (VEC > 1) {
        u32x4 raw;
        __builtin_memcpy(&raw, in, 16);
        *reinterpret_cast<u32x4*>(p) = raw;
    } else {
        p[0] = in[0];
    }
}

template <class T, int VEC>
__device__ __forceinline__ void load_weight(const void* w, int f32, int j, float (&out)[VEC]) {
    if (f32) {
        const float* s = static_cast<const float*>(w) + j;
#pragma unroll
        for (int e = 0; e < VEC; ++e) out[e] = s[e];
    } else {
        typename T::storage s[VEC];
        load_elems<typename T::storage, VEC>(static_cast<const typename T::storage*>(w) + j, s);
#pragma unroll
        for (int e = 0; e < VEC; ++e) out[e] = T::load(s[e]);
    }
}

// Angles from element j of a cache row on (bf16 or f32, any element stride).
template <int VEC>
__device__ __forceinline__ void load_angles(const __attribute__((address_space(4))) NormParams* p, const char* row, int j, float (&out)[VEC]) {
    if constexpr (VEC > 1) {
        if (p->cache_vec) {
            if (p->cache_f32) {
#pragma unroll
                for (int i = 0; i < VEC / 4; ++i) {
                    const float4 x = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(row) + j + 4 * i);
                    out[4 * i] = x.x;
                    out[4 * i + 1] = x.y;
                    out[4 * i + 2] = x.z;
                    out[4 * i + 3] = x.w;
                }
            } else {
                uint16_t x[VEC];
                __builtin_memcpy(x, __builtin_assume_aligned(reinterpret_cast<const uint16_t*>(row) + j, 2 * VEC), 2 * VEC);
#pragma unroll
                for (int i = 0; i < VEC; ++i) out[i] = Bf16::load(x[i]);
            }
            return;
        }
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
        const int64_t at = static_cast<int64_t>(j + i) * p->cache_s1;
        out[i] = p->cache_f32 ? reinterpret_cast<const float*>(row)[at] : Bf16::load(reinterpret_cast<const uint16_t*>(row)[at]);
    }
}

// VEC fp32 values as e4m3 codes, four to a word (a lone value in the low byte).
template <int VEC>
__device__ __forceinline__ void codes_of(const float (&x)[VEC], uint32_t (&words)[(VEC + 3) / 4]) {
    if constexpr (VEC > 1) {
#pragma unroll
        for (int i = 0; i < VEC / 4; ++i) {
            int w = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i], x[4 * i + 1], 0, false);
            w = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i + 2], x[4 * i + 3], w, true);
            words[i] = static_cast<uint32_t>(w);
        }
    } else {
        words[0] = static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[0], 0, false));
    }
}

// Stores a head's row, of which each lane holds NP pieces of VEC dimensions in either half: at[n] are
// their bytes from `base` on in the first half, `to_half` those between the halves.
template <class T, int VEC, int GS, int NP>
__device__ __forceinline__ void store_halves(char* base, const int64_t (&at)[NP], int64_t to_half, int lane, int half,
                                             const float (&x1)[NP][VEC], const float (&x2)[NP][VEC]) {
    typedef typename T::storage S;
#pragma unroll
    for (int n = 0; n < NP; ++n) {
        if ((lane + n * GS) * VEC >= half) continue;
        S y1[VEC], y2[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            y1[e] = T::store(x1[n][e]);
            y2[e] = T::store(x2[n][e]);
        }
        store_elems<S, VEC>(reinterpret_cast<S*>(base + at[n]), y1);
        store_elems<S, VEC>(reinterpret_cast<S*>(base + to_half + at[n]), y2);
    }
}

// The same as e4m3 codes, and the row's scale.
template <int VEC, int GS, int NP>
__device__ __forceinline__ void store_quantised(char* base, const int64_t (&at)[NP], int64_t to_half, float* scale, int lane,
                                                int half, float (&x1)[NP][VEC], float (&x2)[NP][VEC]) {
    // Without the sign, floats order as integers, with infinity and NaN above all finite values.
    uint32_t top = 0;
#pragma unroll
    for (int n = 0; n < NP; ++n) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const uint32_t u1 = __float_as_uint(x1[n][e]) & 0x7fffffffu, u2 = __float_as_uint(x2[n][e]) & 0x7fffffffu;
            top = max(top, max(u1, u2));
        }
    }
    top = group_max<GS>(top);
    const bool finite = top < 0x7f800000u;
    const float wide = fmaxf(__uint_as_float(finite ? top : 0u) / kE4m3Max, kMinScale);
    const float inverse = 1.0f / wide;
#pragma unroll
    for (int n = 0; n < NP; ++n) {
        if ((lane + n * GS) * VEC >= half) continue;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            x1[n][e] *= inverse;
            x2[n][e] *= inverse;
        }
        if (!finite) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) x1[n][e] = x2[n][e] = 0.0f;
        }
        uint32_t lo[(VEC + 3) / 4], hi[(VEC + 3) / 4];
        codes_of<VEC>(x1[n], lo);
        codes_of<VEC>(x2[n], hi);
        __builtin_memcpy(__builtin_assume_aligned(base + at[n], VEC), lo, VEC);
        __builtin_memcpy(__builtin_assume_aligned(base + to_half + at[n], VEC), hi, VEC);
    }
    if (lane == 0) *scale = finite ? wide : NAN;
}

// What a pool holds.
template <class T, bool E4M3>
struct PoolCode {
    typedef typename T::storage type;
};
template <class T>
struct PoolCode<T, true> {
    typedef uint8_t type;
};

// NORM: the whole operator (query heads, key heads, value heads).  Not NORM: the append (key heads, value
// heads, stored as they are).
template <class T, int VEC, int GS, int NP, bool E4M3, bool NORM>
__global__ void __launch_bounds__(256)
qk_norm_kernel(const NormParams) {
    typedef typename T::storage S;
    typedef typename PoolCode<T, E4M3>::type C;
    // The arguments where they are: the tables of tensors are indexed.
    typedef const __attribute__((address_space(4))) NormParams* Params;
    const Params p = (Params)__builtin_amdgcn_kernarg_segment_ptr();
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + wave;
    if (row >= p->rows) return;
    const int part = blockIdx.y;
    const int half = p->head_dim >> 1;
    constexpr int kGroups = 64 / GS;
    const int lane = threadIdx.x & (GS - 1), group = (threadIdx.x & 63) / GS;
    const bool whole = half == GS * VEC * NP;   // every lane has dimensions
    int64_t first[NP];
#pragma unroll
    for (int n = 0; n < NP; ++n) {
        const int j = (lane + n * GS) * VEC;
        first[n] = j < half ? j : 0;   // lanes without dimensions load others' and drop them
    }
    // Passes of the wave over the row's heads: queries, keys, values, a head per group of lanes.
    const int nq = NORM ? (p->q_heads + kGroups - 1) / kGroups : 0, nk = (p->kv_heads + kGroups - 1) / kGroups;
    const int pass0 = part * p->passes_per_wave;
    const int pass1 = min(pass0 + p->passes_per_wave, nq + 2 * nk);
    const int kind0 = pass0 < nq ? 0 : pass0 < nq + nk ? 1 : 2;
    const int done0 = (pass0 - (kind0 == 0 ? 0 : kind0 == 1 ? nq : nq + nk)) * kGroups;

    // What is loaded next: from `src` on, `src_left` heads of source `src_kind`.  Only the lane's place
    // from there differs between lanes; the rest stays in scalar registers.
    const S* src;
    int64_t src_step, src_half, src_group, src_at[NP];
    int src_left, src_kind;
    auto enter_source = [&](int kind, int done) {
        src_kind = kind;
        src = static_cast<const S*>(p->src[kind].data) + row * p->src[kind].s0 + done * p->src[kind].s1;
        src_step = kGroups * p->src[kind].s1;
        src_half = half * p->src[kind].s2;
        src_group = group * p->src[kind].s1;
        src_left = (kind == 0 ? p->q_heads : p->kv_heads) - done;
#pragma unroll
        for (int n = 0; n < NP; ++n) src_at[n] = src_group + first[n] * p->src[kind].s2;
    };
    S a[NP][VEC], b[NP][VEC];   // a pass's elements
    auto load = [&]() {
        if (src_left <= 0) enter_source(src_kind + 1, 0);
        const int64_t back = group < src_left ? 0 : src_group;   // no such head: the first one's, dropped
#pragma unroll
        for (int n = 0; n < NP; ++n) {
            load_elems<S, VEC>(src + (src_at[n] - back), a[n]);
            load_elems<S, VEC>(src + src_half + (src_at[n] - back), b[n]);
        }
        src += src_step;
        src_left -= kGroups;
    };
    enter_source(kind0, done0);
    load();   // on its way while the slot and the position are read

    const int64_t slot = p->slot64 ? static_cast<const int64_t*>(p->slots)[row * p->slot_s]
                                   : static_cast<int64_t>(static_cast<const int32_t*>(p->slots)[row * p->slot_s]);
    if (slot == -1) return;   // a padding row
    int64_t pos = 0;
    if constexpr (NORM) {
        pos = p->pos64 ? static_cast<const int64_t*>(p->positions)[row * p->pos_s]
                       : static_cast<int64_t>(static_cast<const int32_t*>(p->positions)[row * p->pos_s]);
        if (pos < 0 || pos >= p->cache_rows) {
            if (part == 0 && (threadIdx.x & 63) == 0) set_status(p->status, TV_STATUS_BAD_POSITION);
            return;
        }
    }
    if (slot < 0 || slot >= p->pool_pages * p->page_size) {
        if (part == 0 && (threadIdx.x & 63) == 0) set_status(p->status, TV_STATUS_BAD_SLOT);
        return;
    }
    // The rotation with the weights in it: z1 = x1 c1 - x2 s1, z2 = x2 c2 + x1 s2.
    float cs[NP][VEC], sn[NP][VEC], kw1[NP][VEC], kw2[NP][VEC];
    float c1[NP][VEC], c2[NP][VEC], s1[NP][VEC], s2[NP][VEC];
    if constexpr (NORM) {
        const char* cache_row = static_cast<const char*>(p->cache) + pos * p->cache_s0 * (p->cache_f32 ? 4 : 2);
#pragma unroll
        for (int n = 0; n < NP; ++n) {
            const int j = static_cast<int>(first[n]);
            float qw1[VEC], qw2[VEC];
            load_angles<VEC>(p, cache_row, j, cs[n]);
            load_angles<VEC>(p, cache_row, half + j, sn[n]);
            load_weight<T, VEC>(p->qw, p->weight_f32, j, qw1);
            load_weight<T, VEC>(p->qw, p->weight_f32, half + j, qw2);
            load_weight<T, VEC>(p->kw, p->weight_f32, j, kw1[n]);
            load_weight<T, VEC>(p->kw, p->weight_f32, half + j, kw2[n]);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                c1[n][e] = qw1[e] * cs[n][e];
                c2[n][e] = qw2[e] * cs[n][e];
                s1[n][e] = qw2[e] * sn[n][e];
                s2[n][e] = qw1[e] * sn[n][e];
            }
        }
    }
    // A 64-bit division is some 120 dependent instructions; nearly every pool's slots fit 32 bits.
    const bool narrow = ((static_cast<uint64_t>(slot) | static_cast<uint64_t>(p->page_size)) >> 32) == 0;
    const int64_t page = narrow ? static_cast<uint32_t>(slot) / static_cast<uint32_t>(p->page_size) : slot / p->page_size;
    const int64_t offset = slot - page * p->page_size;

    // Where the pass under way goes, in the same manner: the output's row, or the slot's in a pool.
    char* dst;
    float* scale;
    int64_t dst_step, dst_half, scale_step, scale_at, dst_at[NP];
    int left, kind;
    auto enter_target = [&](int which, int done) {
        kind = which;
        const int64_t per_head = p->dst[kind].s2, per_dim = p->dst[kind].s3;
        const int64_t bytes = NORM && kind == 0 ? sizeof(S) : sizeof(C);
        const int64_t outer = NORM && kind == 0 ? row : page, inner = NORM && kind == 0 ? 0 : offset;
        dst = static_cast<char*>(p->dst[kind].data) + (outer * p->dst[kind].s0 + inner * p->dst[kind].s1 + done * per_head) * bytes;
        dst_step = kGroups * per_head * bytes;
        dst_half = half * per_dim * bytes;
        left = (kind == 0 ? p->q_heads : p->kv_heads) - done;
#pragma unroll
        for (int n = 0; n < NP; ++n) dst_at[n] = (group * per_head + first[n] * per_dim) * bytes;
        if constexpr (E4M3) {
            scale = p->dst[kind].scale + outer * p->dst[kind].c0 + inner * p->dst[kind].c1 + done * p->dst[kind].c2;
            scale_step = kGroups * p->dst[kind].c2;
            scale_at = group * p->dst[kind].c2;
        }
        if constexpr (NORM) {
            if (kind == 1) {
#pragma unroll
                for (int n = 0; n < NP; ++n) {
#pragma unroll
                    for (int e = 0; e < VEC; ++e) {
                        c1[n][e] = kw1[n][e] * cs[n][e];
                        c2[n][e] = kw2[n][e] * cs[n][e];
                        s1[n][e] = kw2[n][e] * sn[n][e];
                        s2[n][e] = kw1[n][e] * sn[n][e];
                    }
                }
            }
        }
    };
    enter_target(kind0, done0);
    for (int pass = pass0; pass < pass1; ++pass) {
        if (left <= 0) enter_target(kind + 1, 0);
        float x1[NP][VEC], x2[NP][VEC];
#pragma unroll
        for (int n = 0; n < NP; ++n) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                x1[n][e] = T::load(a[n][e]);
                x2[n][e] = T::load(b[n][e]);
            }
            if (!whole && (lane + n * GS) * VEC >= half) {
#pragma unroll
                for (int e = 0; e < VEC; ++e) x1[n][e] = x2[n][e] = 0.0f;
            }
        }
        if (pass + 1 < pass1) load();
        if constexpr (NORM) {
            if (kind < 2) {
                float square = 0.0f;
#pragma unroll
                for (int n = 0; n < NP; ++n) {
#pragma unroll
                    for (int e = 0; e < VEC; ++e) square = fmaf(x1[n][e], x1[n][e], fmaf(x2[n][e], x2[n][e], square));
                }
                const float mean = group_sum<GS>(square) * p->inverse_dim + p->eps;
                // The reciprocal root instruction is good to one unit in the last place of normal numbers.
                const float r = mean >= 0x1p-100f ? __builtin_amdgcn_rsqf(mean) : 1.0f / sqrtf(mean);
#pragma unroll
                for (int n = 0; n < NP; ++n) {
#pragma unroll
                    for (int e = 0; e < VEC; ++e) {
                        const float y1 = x1[n][e] * r, y2 = x2[n][e] * r;
                        x1[n][e] = y1 * c1[n][e] - y2 * s1[n][e];
                        x2[n][e] = y2 * c2[n][e] + y1 * s2[n][e];
                    }
                }
            }
        }
        if (group < left) {   // whole groups: a head's maximum stays inside one
            if (NORM && kind == 0) {
                store_halves<T, VEC, GS, NP>(dst, dst_at, dst_half, lane, half, x1, x2);
            } else if constexpr (E4M3) {
                store_quantised<VEC, GS, NP>(dst, dst_at, dst_half, scale + scale_at, lane, half, x1, x2);
            } else {
                store_halves<T, VEC, GS, NP>(dst, dst_at, dst_half, lane, half, x1, x2);
            }
        }
        dst += dst_step;
        if constexpr (E4M3) scale += scale_step;
        left -= kGroups;
    }
}

// Waves that fill the chip's 1024 SIMDs: with fewer rows than that a row's heads are spread over
// several waves, since what counts there is the latency of one.  4096 rows of 32 and 8 heads: 19.6 us
// with one wave a row, 21.4 with two, 22.0 with four; the append of 64 rows of 8 heads: 3.3 us with two
// waves a row, 4.2 with one.
constexpr int64_t kFullWaves = 4096;

template <class T, int VEC, int GS, int NP, bool E4M3, bool NORM>
int enqueue(NormParams& p, hipStream_t stream) {
    constexpr int kGroups = 64 / GS;
    const int passes = (NORM ? (p.q_heads + kGroups - 1) / kGroups : 0) + 2 * ((p.kv_heads + kGroups - 1) / kGroups);
    int64_t waves = (kFullWaves + p.rows - 1) / p.rows;
    waves = waves < passes ? waves : passes;
    p.passes_per_wave = static_cast<int>((passes + waves - 1) / waves);
    const dim3 grid(static_cast<uint32_t>((p.rows + 3) / 4), (passes + p.passes_per_wave - 1) / p.passes_per_wave);
    p.inverse_dim = 1.0f / static_cast<float>(p.head_dim);
    hipLaunchKernelGGL((qk_norm_kernel<T, VEC, GS, NP, E4M3, NORM>), grid, dim3(256), 0, stream, p);
    return check_launch(NORM ? "qk_norm_rope_scatter" : "store_kvcache_e4m3");
}

template <class T, bool E4M3, bool NORM>
int by_size(NormParams& p, bool vec, hipStream_t stream) {
    constexpr int kVec = 16 / sizeof(typename T::storage);
    if (vec) {
        const int lanes = (p.head_dim / 2 + kVec - 1) / kVec;   // at most 16, fp32: 32
        if (lanes <= 4) return enqueue<T, kVec, 4, 1, E4M3, NORM>(p, stream);
        if (lanes <= 8) return enqueue<T, kVec, 8, 1, E4M3, NORM>(p, stream);
        if (lanes <= 16) return enqueue<T, kVec, 16, 1, E4M3, NORM>(p, stream);
        return enqueue<T, kVec, 32, 1, E4M3, NORM>(p, stream);
    }
    return enqueue<T, 1, 64, 2, E4M3, NORM>(p, stream);
}

template <bool NORM>
int by_type(NormParams& p, int dtype, bool e4m3, bool vec, hipStream_t stream) {
    if (!NORM || e4m3) {
        if (dtype == TV_BF16) return by_size<Bf16, true, NORM>(p, vec, stream);
        if (dtype == TV_F16) return by_size<F16, true, NORM>(p, vec, stream);
        return by_size<F32, true, NORM>(p, vec, stream);
    }
    if constexpr (NORM) {
        if (dtype == TV_BF16) return by_size<Bf16, false, NORM>(p, vec, stream);
        if (dtype == TV_F16) return by_size<F16, false, NORM>(p, vec, stream);
        return by_size<F32, false, NORM>(p, vec, stream);
    }
    return TV_OK;
}

bool unit_and_aligned(const void* ptr, const int64_t* stride, int n, int64_t elems, int64_t bytes) {
    bool ok = stride[n - 1] == 1 && aligned(ptr, bytes);
    for (int i = 0; i < n - 1; ++i) ok = ok && stride[i] % elems == 0;
    return ok;
}

bool all_positive(const int64_t* stride, int n) {
    for (int i = 0; i < n; ++i) {
        if (stride[i] <= 0) return false;
    }
    return true;
}

Source source_of(const void* data, const int64_t* stride) { return {data, stride[0], stride[1], stride[2]}; }

Target target_of(void* data, const int64_t* stride, float* scale, const int64_t* scale_stride) {
    Target p = {data, stride[0], stride[1], stride[2], stride[3], scale, 0, 0, 0};
    if (scale) {
        p.c0 = scale_stride[0];
        p.c1 = scale_stride[1];
        p.c2 = scale_stride[2];
    }
    return p;
}

}  // namespace
}  // namespace tv

using namespace tv;

extern "C" int64_t tv_sizeof_qk_norm_args(void) { return static_cast<int64_t>(sizeof(tv_qk_norm_args)); }

extern "C" int64_t tv_sizeof_store_e4m3_args(void) { return static_cast<int64_t>(sizeof(tv_store_e4m3_args)); }

extern "C" int tv_qk_norm_rope_scatter(const tv_qk_norm_args* args, void* stream) {
    clear_error();
    const char* what = "qk_norm_rope_scatter";
    if (!args) return fail(TV_ERR_INVALID, "%s: null args", what);
    const tv_rope_scatter_args* a = &args->rope;
    if (a->rows < 0 || a->q_heads < 1 || a->kv_heads < 1 || a->q_heads % a->kv_heads) {
        return fail(TV_ERR_INVALID, "%s: invalid GQA geometry (%d query heads, %d KV heads)", what, a->q_heads, a->kv_heads);
    }
    if (a->head_dim < 2 || a->head_dim % 2 || a->head_dim > 256) {
        return fail(TV_ERR_INVALID, "%s: head_dim %d must be even and in [2, 256]", what, a->head_dim);
    }
    if (a->dtype != TV_BF16 && a->dtype != TV_F16 && a->dtype != TV_F32) {
        return fail(TV_ERR_UNSUPPORTED, "%s: operands must be bf16, f16 or fp32", what);
    }
    if (a->cache_dtype != TV_BF16 && a->cache_dtype != TV_F32) {
        return fail(TV_ERR_UNSUPPORTED, "%s: cos/sin cache must be bf16 or fp32", what);
    }
    if (args->weight_dtype != a->dtype && args->weight_dtype != TV_F32) {
        return fail(TV_ERR_UNSUPPORTED, "%s: norm weights must be fp32 or of the operands' type", what);
    }
    if (!(args->eps >= 0.0f) || args->eps > 3.0e38f) return fail(TV_ERR_INVALID, "%s: eps must be finite and not negative", what);
    if (a->rows == 0) return TV_OK;
    if (a->rows > 0x7fffffff) return fail(TV_ERR_UNSUPPORTED, "%s: too many rows", what);
    if (!a->q || !a->k || !a->v || !a->positions || !a->cache || !a->k_pool || !a->v_pool || !a->node_slots || !a->out ||
        !args->q_weight || !args->k_weight) {
        return fail(TV_ERR_INVALID, "%s: null pointer", what);
    }
    if (args->pool_e4m3 && (!args->k_scale || !args->v_scale)) {
        return fail(TV_ERR_INVALID, "%s: e4m3 pools need their scales", what);
    }
    if (a->cache_rows < 1 || a->pool_pages < 1 || a->page_size < 1) {
        return fail(TV_ERR_INVALID, "%s: empty cos/sin cache or KV pool", what);
    }
    if (!all_positive(a->q_stride, 3) || !all_positive(a->k_stride, 3) || !all_positive(a->v_stride, 3) ||
        !all_positive(a->out_stride, 3) || !all_positive(a->k_pool_stride, 4) || !all_positive(a->v_pool_stride, 4) ||
        a->positions_stride <= 0 || a->slots_stride <= 0 || a->cache_stride_row <= 0 || a->cache_stride_elem <= 0 ||
        (args->pool_e4m3 && (!all_positive(args->k_scale_stride, 3) || !all_positive(args->v_scale_stride, 3)))) {
        return fail(TV_ERR_INVALID, "%s: strides must be positive", what);
    }
    const int64_t elem = a->dtype == TV_F32 ? 4 : 2, n = 16 / elem;
    const bool e4m3 = args->pool_e4m3 != 0;
    const int64_t pool_align = e4m3 ? n : 16;
    const bool vec = (a->head_dim / 2) % n == 0 && unit_and_aligned(a->q, a->q_stride, 3, n, 16) &&
                     unit_and_aligned(a->k, a->k_stride, 3, n, 16) && unit_and_aligned(a->v, a->v_stride, 3, n, 16) &&
                     unit_and_aligned(a->out, a->out_stride, 3, n, 16) &&
                     unit_and_aligned(a->k_pool, a->k_pool_stride, 4, n, pool_align) &&
                     unit_and_aligned(a->v_pool, a->v_pool_stride, 4, n, pool_align) && aligned(args->q_weight, 16) &&
                     aligned(args->k_weight, 16);
    NormParams p = {};
    p.src[0] = source_of(a->q, a->q_stride);
    p.src[1] = source_of(a->k, a->k_stride);
    p.src[2] = source_of(a->v, a->v_stride);
    p.qw = args->q_weight;
    p.kw = args->k_weight;
    p.weight_f32 = args->weight_dtype == TV_F32;
    p.positions = a->positions;
    p.pos_s = a->positions_stride;
    p.pos64 = a->positions_is_int64 != 0;
    p.cache = a->cache;
    p.cache_rows = a->cache_rows;
    p.cache_s0 = a->cache_stride_row;
    p.cache_s1 = a->cache_stride_elem;
    p.cache_f32 = a->cache_dtype == TV_F32;
    p.cache_vec = a->cache_stride_elem == 1 && aligned(a->cache, 16) &&
                  a->cache_stride_row * (p.cache_f32 ? 4 : 2) % 16 == 0;
    p.dst[1] = target_of(a->k_pool, a->k_pool_stride, e4m3 ? args->k_scale : nullptr, args->k_scale_stride);
    p.dst[2] = target_of(a->v_pool, a->v_pool_stride, e4m3 ? args->v_scale : nullptr, args->v_scale_stride);
    p.pool_pages = a->pool_pages;
    p.page_size = a->page_size;
    p.slots = a->node_slots;
    p.slot_s = a->slots_stride;
    p.slot64 = a->slots_is_int64 != 0;
    p.dst[0] = {a->out, a->out_stride[0], 0, a->out_stride[1], a->out_stride[2], nullptr, 0, 0, 0};
    p.rows = a->rows;
    p.q_heads = a->q_heads;
    p.kv_heads = a->kv_heads;
    p.head_dim = a->head_dim;
    p.eps = args->eps;
    p.status = a->status;
    return by_type<true>(p, a->dtype, e4m3, vec, as_stream(stream));
}

extern "C" int tv_store_kvcache_e4m3(const tv_store_e4m3_args* a, void* stream) {
    clear_error();
    const char* what = "store_kvcache_e4m3";
    if (!a) return fail(TV_ERR_INVALID, "%s: null args", what);
    if (a->rows < 0 || a->kv_heads < 1) return fail(TV_ERR_INVALID, "%s: invalid row or head count", what);
    if (a->head_dim < 2 || a->head_dim % 2 || a->head_dim > 256) {
        return fail(TV_ERR_INVALID, "%s: head_dim %d must be even and in [2, 256]", what, a->head_dim);
    }
    if (a->dtype != TV_BF16 && a->dtype != TV_F16 && a->dtype != TV_F32) {
        return fail(TV_ERR_UNSUPPORTED, "%s: rows must be bf16, f16 or fp32", what);
    }
    if (a->rows == 0) return TV_OK;
    if (a->rows > 0x7fffffff) return fail(TV_ERR_UNSUPPORTED, "%s: too many rows", what);
    if (!a->key || !a->value || !a->k_cache || !a->v_cache || !a->k_scale || !a->v_scale || !a->slots) {
        return fail(TV_ERR_INVALID, "%s: null pointer", what);
    }
    if (a->pool_pages < 1 || a->page_size < 1) return fail(TV_ERR_INVALID, "%s: empty KV pool", what);
    if (!all_positive(a->key_stride, 3) || !all_positive(a->value_stride, 3) || !all_positive(a->k_cache_stride, 4) ||
        !all_positive(a->v_cache_stride, 4) || !all_positive(a->k_scale_stride, 3) || !all_positive(a->v_scale_stride, 3) ||
        a->slots_stride <= 0) {
        return fail(TV_ERR_INVALID, "%s: strides must be positive", what);
    }
    const int64_t n = a->dtype == TV_F32 ? 4 : 8;
    const bool vec = (a->head_dim / 2) % n == 0 && unit_and_aligned(a->key, a->key_stride, 3, n, 16) &&
                     unit_and_aligned(a->value, a->value_stride, 3, n, 16) &&
                     unit_and_aligned(a->k_cache, a->k_cache_stride, 4, n, n) &&
                     unit_and_aligned(a->v_cache, a->v_cache_stride, 4, n, n);
    NormParams p = {};
    p.src[1] = source_of(a->key, a->key_stride);
    p.src[2] = source_of(a->value, a->value_stride);
    p.dst[1] = target_of(a->k_cache, a->k_cache_stride, a->k_scale, a->k_scale_stride);
    p.dst[2] = target_of(a->v_cache, a->v_cache_stride, a->v_scale, a->v_scale_stride);
    p.pool_pages = a->pool_pages;
    p.page_size = a->page_size;
    p.slots = a->slots;
    p.slot_s = a->slots_stride;
    p.slot64 = a->slots_is_int64 != 0;
    p.rows = a->rows;
    p.kv_heads = a->kv_heads;
    p.head_dim = a->head_dim;
    p.status = a->status;
    return by_type<false>(p, a->dtype, true, vec, as_stream(stream));
}
