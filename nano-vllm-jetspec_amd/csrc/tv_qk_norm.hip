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
// The work is 2 x 16 bytes a lane and some 60 VALU operations on them, so the bytes bound it.  A
// unit is one head of one row; GS lanes hold it, each VEC consecutive dimensions of the first half
// and the matching ones of the second, so the rotation stays in the lane and the norm is a sum
// over GS lanes (DPP, no LDS).  A wave takes the units of one row in turn: the position, the slot,
// the angles and the weights are loaded once and stay in registers for all of them.
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

// One K/V pool [pages, page_size, heads, dim] (element strides) and, for e4m3 codes, its scales
// [pages, page_size, heads].
struct Pool {
    void* data;
    int64_t s0, s1, s2, s3;
    float* scale;
    int64_t c0, c1, c2;
};

struct NormParams {
    const void* q;
    int64_t q_s0, q_s1, q_s2;
    const void* k;
    int64_t k_s0, k_s1, k_s2;
    const void* v;
    int64_t v_s0, v_s1, v_s2;
    const void* qw;
    const void* kw;
    int32_t weight_f32;
    const void* positions;
    int64_t pos_s;
    int32_t pos64;
    const void* cache;
    int64_t cache_rows, cache_s0, cache_s1;
    int32_t cache_f32, cache_vec;
    Pool kp, vp;
    int64_t pool_pages, page_size;
    const void* slots;
    int64_t slot_s;
    int32_t slot64;
    void* out;
    int64_t o_s0, o_s1, o_s2;
    int64_t rows;
    int32_t q_heads, kv_heads, head_dim;
    int32_t units_per_wave, waves_per_row;
    float eps;
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

template <int GS>
__device__ __forceinline__ float group_max(float x) {
    if constexpr (GS >= 2) x = fmaxf(x, dpp<0xB1>(x));
    if constexpr (GS >= 4) x = fmaxf(x, dpp<0x4E>(x));
    if constexpr (GS >= 8) x = fmaxf(x, dpp<0x141>(x));
    if constexpr (GS >= 16) x = fmaxf(x, dpp<0x140>(x));
    if constexpr (GS >= 32) x = fmaxf(x, __shfl_xor(x, 16));
    if constexpr (GS >= 64) x = fmaxf(x, __shfl_xor(x, 32));
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
__device__ __forceinline__ void load_angles(const NormParams& p, const char* row, int j, float (&out)[VEC]) {
    if constexpr (VEC > 1) {
        if (p.cache_vec) {
            if (p.cache_f32) {
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
        const int64_t at = static_cast<int64_t>(j + i) * p.cache_s1;
        out[i] = p.cache_f32 ? reinterpret_cast<const float*>(row)[at] : Bf16::load(reinterpret_cast<const uint16_t*>(row)[at]);
    }
}

// VEC fp32 values as e4m3 codes, four to a word (a lone value in the low byte).
template <int VEC>
__device__ __forceinline__ void store_codes(uint8_t* p, const float (&x)[VEC]) {
    if constexpr (VEC > 1) {
        uint32_t words[VEC / 4];
#pragma unroll
        for (int i = 0; i < VEC / 4; ++i) {
            int w = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i], x[4 * i + 1], 0, false);
            w = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i + 2], x[4 * i + 3], w, true);
            words[i] = static_cast<uint32_t>(w);
        }
        __builtin_memcpy(__builtin_assume_aligned(p, VEC), words, VEC);
    } else {
        *p = static_cast<uint8_t>(__builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[0], 0, false));
    }
}

// Stores a head's row (each lane NP pieces of VEC dimensions in either half) to its slot.
template <class T, int VEC, int GS, int NP, bool E4M3>
__device__ __forceinline__ void to_pool(const Pool& pool, int64_t page, int64_t offset, int h, int lane, int half,
                                        float (&x1)[NP][VEC], float (&x2)[NP][VEC]) {
    if constexpr (E4M3) {
        // x * 0 is NaN for an infinity and a NaN alone: one sum over the row finds either.
        float amax = 0.0f, probe = 0.0f;
#pragma unroll
        for (int n = 0; n < NP; ++n) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                amax = fmaxf(amax, fmaxf(fabsf(x1[n][e]), fabsf(x2[n][e])));
                probe += x1[n][e] * 0.0f + x2[n][e] * 0.0f;
            }
        }
        amax = group_max<GS>(amax);
        probe = group_sum<GS>(probe);
        const bool finite = probe == 0.0f;
        const float scale = fmaxf(amax / kE4m3Max, kMinScale);
        const float inverse = finite ? 1.0f / scale : 0.0f;
        uint8_t* row = static_cast<uint8_t*>(pool.data) + page * pool.s0 + offset * pool.s1 + h * pool.s2;
#pragma unroll
        for (int n = 0; n < NP; ++n) {
            const int j = (lane + n * GS) * VEC;
            if (j >= half) break;
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                x1[n][e] = finite ? x1[n][e] * inverse : 0.0f;
                x2[n][e] = finite ? x2[n][e] * inverse : 0.0f;
            }
            store_codes<VEC>(row + j * pool.s3, x1[n]);
            store_codes<VEC>(row + (half + j) * pool.s3, x2[n]);
        }
        if (lane == 0) pool.scale[page * pool.c0 + offset * pool.c1 + h * pool.c2] = finite ? scale : NAN;
    } else {
        typedef typename T::storage S;
        S* row = static_cast<S*>(pool.data) + page * pool.s0 + offset * pool.s1 + h * pool.s2;
#pragma unroll
        for (int n = 0; n < NP; ++n) {
            const int j = (lane + n * GS) * VEC;
            if (j >= half) break;
            S y1[VEC], y2[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                y1[e] = T::store(x1[n][e]);
                y2[e] = T::store(x2[n][e]);
            }
            store_elems<S, VEC>(row + j * pool.s3, y1);
            store_elems<S, VEC>(row + (half + j) * pool.s3, y2);
        }
    }
}

// NORM: the whole operator (units: query heads, key heads, value heads).  Not NORM: the append
// (units: key heads, value heads, stored as they are).
template <class T, int VEC, int GS, int NP, bool E4M3, bool NORM>
__global__ void __launch_bounds__(256)
qk_norm_kernel(const NormParams p) {
    typedef typename T::storage S;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t at = static_cast<int64_t>(blockIdx.x) * 4 + wave;
    const int64_t row = at / p.waves_per_row;
    if (row >= p.rows) return;
    const int part = static_cast<int>(at - row * p.waves_per_row);
    const int64_t slot = p.slot64 ? static_cast<const int64_t*>(p.slots)[row * p.slot_s]
                                  : static_cast<int64_t>(static_cast<const int32_t*>(p.slots)[row * p.slot_s]);
    if (slot == -1) return;   // a padding row
    int64_t pos = 0;
    if constexpr (NORM) {
        pos = p.pos64 ? static_cast<const int64_t*>(p.positions)[row * p.pos_s]
                      : static_cast<int64_t>(static_cast<const int32_t*>(p.positions)[row * p.pos_s]);
        if (pos < 0 || pos >= p.cache_rows) {
            if (part == 0 && (threadIdx.x & 63) == 0) set_status(p.status, TV_STATUS_BAD_POSITION);
            return;
        }
    }
    if (slot < 0 || slot >= p.pool_pages * p.page_size) {
        if (part == 0 && (threadIdx.x & 63) == 0) set_status(p.status, TV_STATUS_BAD_SLOT);
        return;
    }
    const int64_t page = slot / p.page_size, offset = slot - page * p.page_size;
    const int half = p.head_dim >> 1;
    constexpr int kGroups = 64 / GS;
    const int lane = threadIdx.x & (GS - 1), group = (threadIdx.x & 63) / GS;
    const int hq = NORM ? p.q_heads : 0;
    const int units = hq + 2 * p.kv_heads;
    const int unit0 = part * p.units_per_wave;
    const int unit1 = unit0 + p.units_per_wave < units ? unit0 + p.units_per_wave : units;

    float cs[NP][VEC], sn[NP][VEC], qw1[NP][VEC], qw2[NP][VEC], kw1[NP][VEC], kw2[NP][VEC];
    if constexpr (NORM) {
        const char* cache_row = static_cast<const char*>(p.cache) + pos * p.cache_s0 * (p.cache_f32 ? 4 : 2);
#pragma unroll
        for (int n = 0; n < NP; ++n) {
            const int j = (lane + n * GS) * VEC;
            if (j >= half) break;
            load_angles<VEC>(p, cache_row, j, cs[n]);
            load_angles<VEC>(p, cache_row, half + j, sn[n]);
            load_weight<T, VEC>(p.qw, p.weight_f32, j, qw1[n]);
            load_weight<T, VEC>(p.qw, p.weight_f32, half + j, qw2[n]);
            load_weight<T, VEC>(p.kw, p.weight_f32, j, kw1[n]);
            load_weight<T, VEC>(p.kw, p.weight_f32, half + j, kw2[n]);
        }
    }
    for (int u = unit0 + group; u < unit1; u += kGroups) {
        const bool is_q = u < hq, is_k = !is_q && u < hq + p.kv_heads;
        const int h = is_q ? u : is_k ? u - hq : u - hq - p.kv_heads;
        const S* src = is_q ? static_cast<const S*>(p.q) + row * p.q_s0 + h * p.q_s1
                            : is_k ? static_cast<const S*>(p.k) + row * p.k_s0 + h * p.k_s1
                                   : static_cast<const S*>(p.v) + row * p.v_s0 + h * p.v_s1;
        const int64_t s2 = is_q ? p.q_s2 : is_k ? p.k_s2 : p.v_s2;
        float x1[NP][VEC], x2[NP][VEC];
        float square = 0.0f;
#pragma unroll
        for (int n = 0; n < NP; ++n) {
            const int j = (lane + n * GS) * VEC;
            S a[VEC] = {}, b[VEC] = {};
            if (j < half) {
                load_elems<S, VEC>(src + j * s2, a);
                load_elems<S, VEC>(src + (half + j) * s2, b);
            }
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                x1[n][e] = T::load(a[e]);
                x2[n][e] = T::load(b[e]);
                square = fmaf(x1[n][e], x1[n][e], fmaf(x2[n][e], x2[n][e], square));
            }
        }
        if constexpr (NORM) {
            if (is_q || is_k) {
                const float r = 1.0f / sqrtf(group_sum<GS>(square) / static_cast<float>(p.head_dim) + p.eps);
#pragma unroll
                for (int n = 0; n < NP; ++n) {
                    if ((lane + n * GS) * VEC >= half) break;
#pragma unroll
                    for (int e = 0; e < VEC; ++e) {
                        const float y1 = x1[n][e] * r * (is_q ? qw1[n][e] : kw1[n][e]);
                        const float y2 = x2[n][e] * r * (is_q ? qw2[n][e] : kw2[n][e]);
                        x1[n][e] = y1 * cs[n][e] - y2 * sn[n][e];
                        x2[n][e] = y2 * cs[n][e] + y1 * sn[n][e];
                    }
                }
            }
            if (is_q) {
                S* dst = static_cast<S*>(p.out) + row * p.o_s0 + h * p.o_s1;
#pragma unroll
                for (int n = 0; n < NP; ++n) {
                    const int j = (lane + n * GS) * VEC;
                    if (j >= half) break;
                    S y1[VEC], y2[VEC];
#pragma unroll
                    for (int e = 0; e < VEC; ++e) {
                        y1[e] = T::store(x1[n][e]);
                        y2[e] = T::store(x2[n][e]);
                    }
                    store_elems<S, VEC>(dst + j * p.o_s2, y1);
                    store_elems<S, VEC>(dst + (half + j) * p.o_s2, y2);
                }
                continue;
            }
        }
        if (is_k) to_pool<T, VEC, GS, NP, E4M3>(p.kp, page, offset, h, lane, half, x1, x2);
        else to_pool<T, VEC, GS, NP, E4M3>(p.vp, page, offset, h, lane, half, x1, x2);
    }
}

// Waves that fill the chip's 1024 SIMDs a few times over: with fewer rows than that a row's heads
// are spread over several waves, since what counts there is the latency of one.
constexpr int64_t kFullWaves = 4096;

template <class T, int VEC, int GS, int NP, bool E4M3, bool NORM>
int enqueue(NormParams& p, hipStream_t stream) {
    constexpr int kGroups = 64 / GS;
    const int units = (NORM ? p.q_heads : 0) + 2 * p.kv_heads;
    const int steps = (units + kGroups - 1) / kGroups;
    int64_t waves = (kFullWaves + p.rows - 1) / p.rows;
    waves = waves < 1 ? 1 : waves < steps ? waves : steps;
    const int per = static_cast<int>((steps + waves - 1) / waves);
    p.units_per_wave = per * kGroups;
    p.waves_per_row = (steps + per - 1) / per;
    const int64_t groups = (p.rows * p.waves_per_row + 3) / 4;
    if (groups > 0x7fffffff) return fail(TV_ERR_UNSUPPORTED, "too many rows and heads for one launch");
    hipLaunchKernelGGL((qk_norm_kernel<T, VEC, GS, NP, E4M3, NORM>), dim3(static_cast<uint32_t>(groups)), dim3(256), 0,
                       stream, p);
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

Pool pool_of(void* data, const int64_t* stride, float* scale, const int64_t* scale_stride) {
    Pool p = {data, stride[0], stride[1], stride[2], stride[3], scale, 0, 0, 0};
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
    p.q = a->q;
    p.q_s0 = a->q_stride[0];
    p.q_s1 = a->q_stride[1];
    p.q_s2 = a->q_stride[2];
    p.k = a->k;
    p.k_s0 = a->k_stride[0];
    p.k_s1 = a->k_stride[1];
    p.k_s2 = a->k_stride[2];
    p.v = a->v;
    p.v_s0 = a->v_stride[0];
    p.v_s1 = a->v_stride[1];
    p.v_s2 = a->v_stride[2];
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
    p.kp = pool_of(a->k_pool, a->k_pool_stride, e4m3 ? args->k_scale : nullptr, args->k_scale_stride);
    p.vp = pool_of(a->v_pool, a->v_pool_stride, e4m3 ? args->v_scale : nullptr, args->v_scale_stride);
    p.pool_pages = a->pool_pages;
    p.page_size = a->page_size;
    p.slots = a->node_slots;
    p.slot_s = a->slots_stride;
    p.slot64 = a->slots_is_int64 != 0;
    p.out = a->out;
    p.o_s0 = a->out_stride[0];
    p.o_s1 = a->out_stride[1];
    p.o_s2 = a->out_stride[2];
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
    p.k = a->key;
    p.k_s0 = a->key_stride[0];
    p.k_s1 = a->key_stride[1];
    p.k_s2 = a->key_stride[2];
    p.v = a->value;
    p.v_s0 = a->value_stride[0];
    p.v_s1 = a->value_stride[1];
    p.v_s2 = a->value_stride[2];
    p.kp = pool_of(a->k_cache, a->k_cache_stride, a->k_scale, a->k_scale_stride);
    p.vp = pool_of(a->v_cache, a->v_cache_stride, a->v_scale, a->v_scale_stride);
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
