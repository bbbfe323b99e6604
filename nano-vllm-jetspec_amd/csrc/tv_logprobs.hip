// Log probabilities of given tokens, the entropy and the top alternatives of logits rows, for gfx950.
//
// Row x of V logits, in one pass:
//     Z = sum_j 2^(c x_j - R),  E = sum_j 2^(c x_j - R) (c x_j - R),  c = log2 e, R a reference near c max x,
//     log p_t = x_t - (R + log2 Z) / c,   entropy = (log2 Z - E / Z) / c,
// and the k largest logits by (value, lowest index).  A lane keeps its own R, Z and E; R is raised, and the
// sums scaled, only when a logit passes it by more than 8, so terms stay below 2^12.  A word at -inf adds
// nothing to either sum (its exponent is held at -200, whose power is zero).
//
// The top k: a wave keeps the 64 largest it has seen, sorted, a lane each, and a queue in LDS.  What does
// not pass the k-th of them, which per 16-byte unit is one comparison with the unit's maximum, is done with;
// other units are queued, and when there are 64 what still passes is sorted and merged (bitonic).  The first bound is
// the k-th largest of the lanes' maxima over the first units, and all waves of a row share theirs.  A wave's elements come in the order of their indices, so a
// later one of equal value never counts, and the waves' lists are joined by their order as 64-bit numbers,
// value before index: the result depends on no timing.
//
// Memory bounds it where no alternatives are asked for (4096 rows of 151936 bf16 logits, 1.25 GB: 197 us, 6.3 TB/s);
// the vector unit is as busy, ten instruction slots an element, of which the exponential takes four, and bounds it
// with 20 alternatives (207 us; 316 with every element of a unit looked at where one passes, exchanges through LDS
// and bounds of a wave's own).  8 rows with 5: 12.7 us, two launches' latencies.
#include <math.h>
#include <stdint.h>

#include "tv_internal.h"

namespace tv {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kUnroll = 4;      // units a lane loads at a time
constexpr int kMostTop = 64;
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kMargin = 8.0f;
// R is c x rounded to fp32, and c x - R has to stay near zero for the x it was made of: so up to 2^16.  Larger
// logits (masks of -1e9 or the type's lowest value) are summed against references of their own, below, to
// zero, and above all others.  A row left with such a one is summed again, by differences, and so is one whose largest
// logit is within 100 of the far ones below it (its reference under kNearLow), whose terms a lane has lost when it saw
// them before a near one.  Above that they are less than 2^-130 of the largest.
constexpr float kFar = 65536.0f, kFarLow = -9.0e4f, kFarHigh = 1.0e5f, kNearLow = -9.44e4f;

struct LogprobParams {
    const char* logits;
    int64_t stride;                 // elements
    int64_t held, vocab;
    const void* rows;
    int32_t rows64;
    const void* tokens;
    int32_t tokens64;
    int64_t num_rows;
    int32_t given, top, splits;
    float* logprobs;
    float* entropy;
    int64_t* top_ids;
    float* top_logprobs;
    float* ws_sums;                 // [rows * splits, 4]
    uint64_t* ws_top;               // [rows * splits, top]
    int32_t* status;
};

struct LogBf16 {
    typedef uint16_t storage;
    static constexpr uint32_t kNone = 0xff80ff80u;   // -inf in every element of a word
    static __device__ __forceinline__ float load(storage s) { return __uint_as_float(static_cast<uint32_t>(s) << 16); }
};
struct LogF16 {
    typedef uint16_t storage;
    static constexpr uint32_t kNone = 0xfc00fc00u;
    static __device__ __forceinline__ float load(storage s) { return static_cast<float>(__builtin_bit_cast(_Float16, s)); }
};
struct LogF32 {
    typedef float storage;
    static constexpr uint32_t kNone = 0xff800000u;
    static __device__ __forceinline__ float load(storage s) { return s; }
};

__device__ __forceinline__ int64_t load_int(const void* p, int is64, int64_t i) {
    return is64 ? static_cast<const int64_t*>(p)[i] : static_cast<int64_t>(static_cast<const int32_t*>(p)[i]);
}

// Order-preserving map of floats to integers: -0 equals +0, a NaN lies above everything; never 0.
__device__ __forceinline__ uint32_t order_of(float x) {
    if (x != x) return 0xffffffffu;
    const uint32_t u = __float_as_uint(x + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t order) {
    return __uint_as_float(order & 0x80000000u ? order & 0x7fffffffu : ~order);
}
// A value that whatever has a higher order than `order` is not at or below.
__device__ __forceinline__ float bound_of(uint32_t order) {
    if (order == 0xffffffffu) return INFINITY;
    return order == 0x7fffffffu ? -__uint_as_float(1u) : value_of(order);   // 0x7fffffff: -0, which no value has
}

__device__ __forceinline__ uint64_t entry_of(float x, int64_t index) {
    return static_cast<uint64_t>(order_of(x)) << 32 | static_cast<uint32_t>(~static_cast<uint32_t>(index));
}

// The value of lane ^ M: by a row's own permutations up to 8, and by swaps of half rows and rows above, which take a
// tenth of the latency of an exchange through LDS.  All lanes call it.
template <int CTRL>
__device__ __forceinline__ uint32_t row_moved(uint32_t v) {
    return static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), CTRL, 0xf, 0xf, false));
}
template <int M>
__device__ __forceinline__ uint32_t lane_xor(uint32_t v) {
    if constexpr (M == 1) return row_moved<0xB1>(v);                        // quad_perm [1, 0, 3, 2]
    else if constexpr (M == 2) return row_moved<0x4E>(v);                   // quad_perm [2, 3, 0, 1]
    else if constexpr (M == 4) return row_moved<0x1B>(row_moved<0x141>(v)); // half row mirrored, quad_perm [3, 2, 1, 0]
    else if constexpr (M == 8) return row_moved<0x128>(v);                  // row rotated by 8
    else if constexpr (M == 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        return threadIdx.x & 16 ? r[0] : r[1];
    } else {
        static_assert(M == 32, "a power of two below 64");
        const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        return threadIdx.x & 32 ? r[0] : r[1];
    }
}
template <int M>
__device__ __forceinline__ float lane_xor(float v) {
    return __uint_as_float(lane_xor<M>(__float_as_uint(v)));
}
template <int M>
__device__ __forceinline__ uint64_t lane_xor(uint64_t v) {
    return static_cast<uint64_t>(lane_xor<M>(static_cast<uint32_t>(v >> 32))) << 32 | lane_xor<M>(static_cast<uint32_t>(v));
}
// v, joined by `f` over the wave's lanes in a fixed order, in all of them.
template <class V, class F>
__device__ __forceinline__ V over_lanes(V v, F f) {
    v = f(v, lane_xor<1>(v));
    v = f(v, lane_xor<2>(v));
    v = f(v, lane_xor<4>(v));
    v = f(v, lane_xor<8>(v));
    v = f(v, lane_xor<16>(v));
    return f(v, lane_xor<32>(v));
}

// Bitonic steps over the wave's 64 lanes, largest first: halves of J lanes compared, in blocks of K.
template <int J, int K, class V>
__device__ __forceinline__ void merge_step(V& v) {
    if constexpr (J > 0) {
        const V o = lane_xor<J>(v);
        const int lane = threadIdx.x & 63;
        const bool larger = ((lane & J) == 0) == ((lane & K) == 0);
        v = larger == (v > o) ? v : o;
        merge_step<J / 2, K>(v);
    }
}
template <class V>
__device__ __forceinline__ V merged(V v) {
    merge_step<32, 64>(v);
    return v;
}
template <class V>
__device__ __forceinline__ V sorted(V v) {
    merge_step<1, 2>(v);
    merge_step<2, 4>(v);
    merge_step<4, 8>(v);
    merge_step<8, 16>(v);
    merge_step<16, 32>(v);
    return merged(v);
}
template <class V>
__device__ __forceinline__ V lane_reversed(V v) {
    v = lane_xor<32>(lane_xor<16>(v));
    return lane_xor<8>(lane_xor<4>(lane_xor<2>(lane_xor<1>(v))));
}
// A lane's value in all; the lane is the same for all.
__device__ __forceinline__ uint32_t of_lane(uint32_t v, int lane) {
    return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), lane));
}
__device__ __forceinline__ uint64_t of_lane(uint64_t v, int lane) {
    return static_cast<uint64_t>(of_lane(static_cast<uint32_t>(v >> 32), lane)) << 32 | of_lane(static_cast<uint32_t>(v), lane);
}

// How many of `lanes` lie before this one.
__device__ __forceinline__ int lanes_before(uint64_t lanes) {
    return __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(lanes >> 32), __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(lanes), 0));
}

// A wave's largest entries.  Entries are distinct, but for the empty one, 0.
struct WaveTop {
    uint64_t best = 0;     // sorted over the lanes
    uint64_t kth = 0;      // the top-th of them
    uint64_t* queue;       // LDS of the wave's own: fewer than 64, and a push of up to 64
    int queued = 0, top;
    bool held = false;     // anything in the list

    // One wave's exchange through LDS: its operations run in order, the compiler's must too.
    static __device__ __forceinline__ void settle() {
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
    // Merges the last 64 entries of the queue.
    __device__ __forceinline__ void flush() {
        if (queued == 0) return;
        const int lane = threadIdx.x & 63, from = queued > 64 ? queued - 64 : 0;
        settle();
        const uint64_t mine = from + lane < queued ? queue[from + lane] : 0;
        queued = from;
        merge(sorted(mine));
    }
    // Merges another sorted list.
    __device__ __forceinline__ void merge(uint64_t list) {
        if (held) {
            const uint64_t other = lane_reversed(list);
            list = merged(best > other ? best : other);
        }
        held = true;
        best = list;
        kth = of_lane(best, top - 1);
    }
    __device__ __forceinline__ void push(bool want, uint64_t entry) {
        const uint64_t lanes = __ballot(want);
        if (lanes == 0) return;
        if (want) queue[queued + lanes_before(lanes)] = entry;
        queued += __popcll(lanes);
    }
};

// Sums over one row or a part of it.
struct Sums {
    float r = -INFINITY, z = 0.0f, e = 0.0f;   // the reference times log2 e, and the sums against it

    // Against another reference, at or above this one's unless there is nothing to scale.
    __device__ __forceinline__ void rescale(float to) {
        if (r == to) return;
        const float f = __builtin_amdgcn_exp2f(r - to);
        const bool none = z == 0.0f || f == 0.0f;   // nothing yet, or nothing left
        e = none ? 0.0f : (e - (to - r) * z) * f;
        z = z != z ? z : none ? 0.0f : z * f;
        r = to;
    }
    __device__ __forceinline__ void add(Sums o) {
        const float top = fmaxf(r, o.r);
        rescale(top);
        o.rescale(top);
        z += o.z;
        e += o.e;
    }
};

// Joins the waves' sums and lists: all threads get the sums, the first wave the list.
struct Joined {
    float sums[kWaves][3];
    uint64_t all[kWaves][64];
};

template <bool TOP>
__device__ __forceinline__ Sums join(Joined& s, WaveTop& t, Sums mine) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    mine.rescale(over_lanes(mine.r, [](float a, float b) { return fmaxf(a, b); }));
    mine.z = over_lanes(mine.z, [](float a, float b) { return a + b; });
    mine.e = over_lanes(mine.e, [](float a, float b) { return a + b; });
    if (lane == 0) {
        s.sums[wave][0] = mine.r;
        s.sums[wave][1] = mine.z;
        s.sums[wave][2] = mine.e;
    }
    if constexpr (TOP) s.all[wave][lane] = t.best;
    __syncthreads();
    Sums row;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) row.add({s.sums[w][0], s.sums[w][1], s.sums[w][2]});
    if constexpr (TOP) {
        if (wave == 0) {
#pragma unroll
            for (int w = 1; w < kWaves; ++w) t.merge(s.all[w][lane]);
        }
    }
    return row;
}

// A row's sums against its own largest logit, which it returns, differences first.  All threads call it.
template <class T>
__device__ __forceinline__ float sum_far(const LogprobParams& p, const typename T::storage* x, Sums& sums) {
    __shared__ float parts[kWaves][2];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    float most = -INFINITY;
    for (int64_t j = threadIdx.x; j < p.vocab; j += kThreads) most = __builtin_elementwise_maximum(most, T::load(x[j]));
    most = over_lanes(most, [](float a, float b) { return __builtin_elementwise_maximum(a, b); });
    if (lane == 0) parts[wave][0] = most;
    __syncthreads();
    for (int w = 0; w < kWaves; ++w) most = __builtin_elementwise_maximum(most, parts[w][0]);
    __syncthreads();
    float z = 0.0f, e = 0.0f;
    for (int64_t j = threadIdx.x; j < p.vocab; j += kThreads) {
        const float d = fmaxf((T::load(x[j]) - most) * kLog2e, -200.0f), one = __builtin_amdgcn_exp2f(d);
        z += one;
        e = fmaf(one, d, e);
    }
    z = over_lanes(z, [](float a, float b) { return a + b; });
    e = over_lanes(e, [](float a, float b) { return a + b; });
    if (lane == 0) {
        parts[wave][0] = z;
        parts[wave][1] = e;
    }
    __syncthreads();
    sums.z = sums.e = 0.0f;
    for (int w = 0; w < kWaves; ++w) {
        sums.z += parts[w][0];
        sums.e += parts[w][1];
    }
    if (!(most < INFINITY)) sums.z = NAN;
    return most;
}

// What a row's sums and list say.  All threads call it; lane j of the first wave holds the list's j-th `entry`.
template <class T, bool TOP>
__device__ __forceinline__ void finish(const LogprobParams& p, int64_t i, int64_t row, Sums sums, uint64_t entry) {
    typedef typename T::storage S;
    const S* x = reinterpret_cast<const S*>(p.logits) + row * p.stride;
    double reference = static_cast<double>(sums.r) / static_cast<double>(kLog2e);
    if (sums.r == kFarLow || sums.r == kFarHigh || (sums.r < kNearLow && sums.r > -INFINITY)) reference = sum_far<T>(p, x, sums);
    const double log_sum = static_cast<double>(log2f(sums.z)) / static_cast<double>(kLog2e);
    // A sum over nothing but -inf has no distribution.
    const bool none = !(sums.z > 0.0f);
    // No logarithm of a probability is above zero, which the sum's rounding would make of a nearly certain word's.
    auto logprob = [&](float logit) {
        const float value = static_cast<float>(static_cast<double>(logit) - reference - log_sum);
        return none ? NAN : value > 0.0f ? 0.0f : value;
    };
    if (threadIdx.x == 0) {
        const float entropy = (log2f(sums.z) - sums.e / sums.z) / kLog2e;
        p.entropy[i] = none ? NAN : entropy < 0.0f ? 0.0f : entropy;
    }
    for (int j = threadIdx.x; j < p.given; j += kThreads) {
        const int64_t t = load_int(p.tokens, p.tokens64, i * p.given + j);
        float value = t == -1 ? 0.0f : NAN;
        if (t >= 0 && t < p.vocab) value = logprob(T::load(x[t]));
        else if (t != -1) set_status(p.status, TV_STATUS_BAD_REQUEST);
        p.logprobs[i * p.given + j] = value;
    }
    if constexpr (TOP) {
        const int j = threadIdx.x;
        if (j < p.top) {
            p.top_ids[i * p.top + j] = static_cast<int64_t>(~static_cast<uint32_t>(entry));
            p.top_logprobs[i * p.top + j] = logprob(value_of(static_cast<uint32_t>(entry >> 32)));
        }
    }
}

// The logits row of result row i; -1: none, and its results are written here.
__device__ __forceinline__ int64_t find_row(const LogprobParams& p, int64_t i, bool write) {
    const int64_t row = p.rows ? load_int(p.rows, p.rows64, i) : i;
    if (row >= 0 && row < p.held) return row;
    if (write) {
        const float value = row == -1 ? 0.0f : NAN;
        if (threadIdx.x == 0) {
            p.entropy[i] = value;
            if (row != -1) set_status(p.status, TV_STATUS_BAD_REQUEST);
        }
        for (int j = threadIdx.x; j < p.given; j += kThreads) p.logprobs[i * p.given + j] = value;
        for (int j = threadIdx.x; j < p.top; j += kThreads) {
            p.top_ids[i * p.top + j] = -1;
            p.top_logprobs[i * p.top + j] = value;
        }
    }
    return -1;
}

template <class T, bool TOP>
__global__ void __launch_bounds__(kThreads)
logprobs_kernel(const LogprobParams p) {
    typedef typename T::storage S;
    constexpr int VEC = 16 / sizeof(S);
    __shared__ Joined joined;
    __shared__ uint64_t queues[kWaves][TOP ? 128 : 1];
    // Units with a candidate in them: fewer than 64, and those of a step.
    __shared__ u32x4 unit_of[kWaves][TOP ? 128 : 1];
    __shared__ int32_t unit_at[kWaves][TOP ? 128 : 1];
    // A wave reads what others have written so far.  (Relaxed accesses: through volatile ones the compiler goes by flat
    // addresses, one at a time.)
    __shared__ uint32_t shared_full[kWaves], shared_quarter[kWaves];
    const int64_t i = blockIdx.x / p.splits;
    const int split = static_cast<int>(blockIdx.x - i * p.splits);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t row = find_row(p, i, p.splits == 1);
    if (row < 0) return;
    // A row has fewer than VEC elements before its first 16 bytes: those, the units, the rest.
    const S* base = reinterpret_cast<const S*>(p.logits) + row * p.stride;
    const uint32_t past = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(base)) & 15u;
    int64_t head = ((16u - past) & 15u) / sizeof(S);
    head = head < p.vocab ? head : p.vocab;
    const int64_t units = (p.vocab - head) / VEC;
    const S* body = base + head;
    const int64_t unit0 = units * split / p.splits, unit1 = units * (split + 1) / p.splits;

    Sums sums;
    float limit = -INFINITY;       // no logit seen passes it by much
    WaveTop tops;
    tops.queue = queues[wave];
    tops.top = p.top;
    uint32_t pass = 0;             // whatever has this order or a lower one is not among the row's largest
    float bound = __uint_as_float(0x7fc00000u);   // its value; NaN: everything is a candidate
    auto raise_pass = [&](uint32_t to) {
        if (to <= pass) return;
        pass = to;
        bound = bound_of(to);
    };
    // What a wave's sorted list says to all: its top-th entry has top elements from it on, and where every wave has a
    // quarter of them at some value, so have they all together.  Another wave's equal value can come first.
    auto publish = [&](auto list) {
        constexpr int kShift = sizeof(list) == 8 ? 32 : 0;
        const uint32_t full = static_cast<uint32_t>(of_lane(list, p.top - 1) >> kShift);
        const uint32_t quarter = static_cast<uint32_t>(of_lane(list, (p.top + kWaves - 1) / kWaves - 1) >> kShift);
        if (lane == 0) {
            __hip_atomic_store(&shared_full[wave], full, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
            __hip_atomic_store(&shared_quarter[wave], quarter, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
        }
    };
    auto look = [&]() {
        uint32_t most = 0, least = 0xffffffffu;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            most = max(most, __hip_atomic_load(&shared_full[w], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP));
            least = min(least, __hip_atomic_load(&shared_quarter[w], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP));
        }
        most = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(max(most, least))));
        if (most > 0) raise_pass(most - 1);
    };
    auto values = [&](u32x4 from, float (&x)[VEC]) {
        S s[VEC];
        __builtin_memcpy(s, &from, 16);
#pragma unroll
        for (int e = 0; e < VEC; ++e) x[e] = T::load(s[e]);
    };
    int units_queued = 0;
    auto merge_queue = [&]() {
        tops.flush();
        // This wave's elements to come have higher indices, so an equal value is not enough.
        raise_pass(static_cast<uint32_t>(tops.kth >> 32));
        publish(tops.best);
    };
    // The elements of all queued units that are candidates yet, to the list; the bound stays until all are through.
    auto expand = [&]() {
        WaveTop::settle();
        for (int u0 = 0; u0 < units_queued; u0 += 64) {
            const bool live = u0 + lane < units_queued;
            const int at = live ? u0 + lane : 0;
            const int64_t first = head + static_cast<int64_t>(unit_at[wave][at]) * VEC;
            float x[VEC];
            values(unit_of[wave][at], x);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                tops.push(live && !(x[e] <= bound), entry_of(x[e], first + e));
                if (tops.queued >= 64) tops.flush();
            }
        }
        units_queued = 0;
        merge_queue();
    };
    // A lane's elements x; `found` gets those of lanes that are `live` and can be among the largest.
    auto process = [&](const float (&x)[VEC], bool live, auto found) {
        float most = x[0];
#pragma unroll
        for (int e = 1; e < VEC; ++e) most = __builtin_elementwise_maximum(most, x[e]);   // NaN where one is
        const bool raise = !(most <= limit), candidate = TOP && !(most <= bound);
        if (__any(raise || candidate)) {
            if (raise) {
                if (!(most < INFINITY)) {
                    sums.z = NAN;
                    limit = INFINITY;
                } else {
                    sums.rescale(fabsf(most) < kFar ? most * kLog2e : most < 0.0f ? kFarLow : kFarHigh);
                    limit = most + kMargin;
                }
            }
            if constexpr (TOP) found(live && candidate);
        }
        float z[VEC], z_e[2] = {0.0f, 0.0f};
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const float d = fmaxf(fmaf(x[e], kLog2e, -sums.r), -200.0f);
            z[e] = __builtin_amdgcn_exp2f(d);
            z_e[e & 1] = fmaf(z[e], d, z_e[e & 1]);
        }
#pragma unroll
        for (int o = 1; o < VEC; o <<= 1) {
#pragma unroll
            for (int e = 0; e + o < VEC; e += 2 * o) z[e] += z[e + o];
        }
        sums.z += z[0];
        sums.e += z_e[0] + z_e[1];
    };
    auto lone = [&](int64_t index, bool live) {
        float x[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) x[e] = -INFINITY;
        if (live) x[0] = T::load(base[index]);
        process(x, live, [&](bool candidate) {
            tops.push(candidate, entry_of(x[0], index));
            if (tops.queued >= 64) merge_queue();
        });
    };
    constexpr int kStride = 64 * kWaves;    // units between a lane's
    u32x4 raw[kUnroll];
    auto load = [&](int64_t u0) {
#pragma unroll
        for (int k = 0; k < kUnroll; ++k) {
            const int64_t u = u0 + kStride * k + lane;
            raw[k] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(body + (u < unit1 ? u : unit1 - 1) * VEC));
        }
        if (u0 + kStride * (kUnroll - 1) + 64 > unit1) {
#pragma unroll
            for (int k = 0; k < kUnroll; ++k) {
                if (u0 + kStride * k + lane >= unit1) raw[k] = u32x4{T::kNone, T::kNone, T::kNone, T::kNone};
            }
        }
    };
    int64_t u0 = unit0 + 64 * wave;
    if (u0 < unit1) load(u0);
    if constexpr (TOP) {
        // The k-th largest of the lanes' maxima is at most the k-th largest element.
        uint32_t most = 0;
        if (u0 < unit1) {
#pragma unroll
            for (int k = 0; k < kUnroll; ++k) {
                float x[VEC];
                values(raw[k], x);
                float top = x[0];
#pragma unroll
                for (int e = 1; e < VEC; ++e) top = __builtin_elementwise_maximum(top, x[e]);
                if (u0 + kStride * k + lane < unit1) most = max(most, order_of(top));
            }
        }
        publish(sorted(most));
        __syncthreads();
    }
    if (split == 0 && wave == 0 && head > 0) lone(lane < head ? lane : 0, lane < head);
    while (u0 < unit1) {
        if constexpr (TOP) look();
#pragma unroll
        for (int k = 0; k < kUnroll; ++k) {
            const int64_t u = u0 + kStride * k + lane;
            float x[VEC];
            values(raw[k], x);
            process(x, u < unit1, [&](bool candidate) {
                const uint64_t lanes = __ballot(candidate);
                if (candidate) {
                    const int at = units_queued + lanes_before(lanes);
                    unit_of[wave][at] = raw[k];
                    unit_at[wave][at] = static_cast<int32_t>(u);
                }
                units_queued += __popcll(lanes);
                if (units_queued >= 64) expand();
            });
        }
        u0 += kStride * kUnroll;
        if (u0 < unit1) load(u0);
    }
    if constexpr (TOP) expand();
    const int64_t rest = head + units * VEC;
    if (split == p.splits - 1 && wave == kWaves - 1 && rest < p.vocab) {
        lone(rest + lane < p.vocab ? rest + lane : rest, rest + lane < p.vocab);
    }
    if constexpr (TOP) tops.flush();
    const Sums all = join<TOP>(joined, tops, sums);
    if (p.splits == 1) {
        finish<T, TOP>(p, i, row, all, tops.best);
        return;
    }
    if (threadIdx.x == 0) {
        float* to = p.ws_sums + 4 * static_cast<int64_t>(blockIdx.x);
        to[0] = all.r;
        to[1] = all.z;
        to[2] = all.e;
    }
    if constexpr (TOP) {
        if (threadIdx.x < p.top) p.ws_top[static_cast<int64_t>(blockIdx.x) * p.top + threadIdx.x] = tops.best;
    }
}

// Joins the parts of a row.
template <class T, bool TOP>
__global__ void __launch_bounds__(kThreads)
logprobs_join_kernel(const LogprobParams p) {
    __shared__ Joined joined;
    __shared__ uint64_t queues[kWaves][TOP ? 128 : 1];
    const int64_t i = blockIdx.x;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t row = find_row(p, i, true);
    if (row < 0) return;
    Sums sums;
    for (int s = threadIdx.x; s < p.splits; s += kThreads) {
        const float* from = p.ws_sums + 4 * (i * p.splits + s);
        sums.add({from[0], from[1], from[2]});
    }
    WaveTop tops;
    tops.queue = queues[wave];
    tops.top = p.top;
    if constexpr (TOP) {
        const int entries = p.splits * p.top;
        for (int at = 64 * wave; at < entries; at += kThreads) {
            const uint64_t entry = at + lane < entries ? p.ws_top[i * entries + at + lane] : 0;
            tops.push(entry > tops.kth, entry);
            if (tops.queued >= 64) tops.flush();
        }
        tops.flush();
    }
    const Sums all = join<TOP>(joined, tops, sums);
    finish<T, TOP>(p, i, row, all, tops.best);
}

// Parts of a row: three workgroups a compute unit where there are not two rows for each, since every part begins its
// bounds anew and the join is a launch; the shortest parts have 2 to 4 units a thread.  700 / 1000 rows with 20
// alternatives (151936 and 50257 words of bf16) whole 48 / 29 us, in two parts 54 / 36; 64 in 12 parts 17.5, in 16 20.2;
// 333 fp32 rows of 50257 in 3 parts 16.2, in 2 17.2, in 4 17.9.
int64_t splits_of(const tv_token_logprobs_args* a) {
    const int64_t vec = a->dtype == TV_F32 ? 4 : 8;
    const int64_t most = (a->vocab / vec + kThreads * kUnroll - 1) / (kThreads * kUnroll);
    const int64_t units = a->compute_units;
    int64_t splits = a->num_rows >= 2 * units ? 1 : (3 * units + a->num_rows - 1) / a->num_rows;
    splits = splits < most ? splits : most;
    return splits > 1 ? splits : 1;
}

template <class T, bool TOP>
int enqueue(const LogprobParams& p, hipStream_t s) {
    hipLaunchKernelGGL((logprobs_kernel<T, TOP>), dim3(static_cast<uint32_t>(p.num_rows * p.splits)), dim3(kThreads), 0, s, p);
    const int launched = check_launch("token_logprobs");
    if (launched != TV_OK || p.splits == 1) return launched;
    hipLaunchKernelGGL((logprobs_join_kernel<T, TOP>), dim3(static_cast<uint32_t>(p.num_rows)), dim3(kThreads), 0, s, p);
    return check_launch("token_logprobs join");
}

template <class T>
int by_top(const LogprobParams& p, hipStream_t s) {
    return p.top > 0 ? enqueue<T, true>(p, s) : enqueue<T, false>(p, s);
}

int check(const tv_token_logprobs_args* a) {
    const char* what = "token_logprobs";
    if (!a) return fail(TV_ERR_INVALID, "%s: null args", what);
    if (a->num_rows < 0 || a->num_logits < 0 || a->vocab < 1 || a->logits_stride < a->vocab || a->tokens < 0 || a->compute_units < 1) {
        return fail(TV_ERR_INVALID, "%s: invalid sizes", what);
    }
    if (a->dtype != TV_BF16 && a->dtype != TV_F16 && a->dtype != TV_F32) {
        return fail(TV_ERR_UNSUPPORTED, "%s: logits must be bf16, f16 or fp32", what);
    }
    if (a->vocab > 0x7fffffff) return fail(TV_ERR_UNSUPPORTED, "%s: vocabularies of 2^31 words or more", what);
    if (a->top < 0 || a->top > kMostTop || a->top > a->vocab) {
        return fail(TV_ERR_INVALID, "%s: %d alternatives (at most 64, and the vocabulary)", what, a->top);
    }
    if (!a->rows && a->num_rows > a->num_logits) return fail(TV_ERR_INVALID, "%s: more results than logits rows", what);
    // A launch has fewer than 2^32 threads.
    if (a->num_rows > 0 && (a->num_rows > 0xffffff || a->num_rows * splits_of(a) > 0xffffff)) {
        return fail(TV_ERR_UNSUPPORTED, "%s: too many rows", what);
    }
    return TV_OK;
}

}  // namespace
}  // namespace tv

using namespace tv;

extern "C" int64_t tv_sizeof_token_logprobs_args(void) { return static_cast<int64_t>(sizeof(tv_token_logprobs_args)); }

extern "C" int64_t tv_token_logprobs_workspace_bytes(const tv_token_logprobs_args* a) {
    clear_error();
    const int code = check(a);
    if (code != TV_OK) return code;
    if (a->num_rows == 0) return 0;
    const int64_t splits = splits_of(a);
    return splits == 1 ? 0 : a->num_rows * splits * (16 + 8ll * a->top);
}

extern "C" int tv_token_logprobs(const tv_token_logprobs_args* a, void* workspace, int64_t workspace_bytes, void* stream) {
    clear_error();
    const int code = check(a);
    if (code != TV_OK) return code;
    const char* what = "token_logprobs";
    if (a->num_rows == 0) return TV_OK;
    if ((!a->logits && a->num_logits > 0) || !a->entropy || (a->tokens > 0 && (!a->token_ids || !a->logprobs)) ||
        (a->top > 0 && (!a->top_ids || !a->top_logprobs))) {
        return fail(TV_ERR_INVALID, "%s: null pointer", what);
    }
    if (!aligned(a->logits, a->dtype == TV_F32 ? 4 : 2)) return fail(TV_ERR_INVALID, "%s: unaligned logits", what);
    const int64_t splits = splits_of(a), bytes = splits == 1 ? 0 : a->num_rows * splits * (16 + 8ll * a->top);
    if (bytes && (!workspace || !aligned(workspace, 16))) return fail(TV_ERR_INVALID, "%s: null or unaligned workspace", what);
    if (workspace_bytes < bytes) {
        return fail(TV_ERR_CAPACITY, "%s: workspace of %lld bytes, %lld needed", what, static_cast<long long>(workspace_bytes),
                    static_cast<long long>(bytes));
    }
    LogprobParams p = {};
    p.logits = static_cast<const char*>(a->logits);
    p.stride = a->logits_stride;
    p.held = a->num_logits;
    p.vocab = a->vocab;
    p.rows = a->rows;
    p.rows64 = a->rows_is_int64 != 0;
    p.tokens = a->token_ids;
    p.tokens64 = a->tokens_is_int64 != 0;
    p.num_rows = a->num_rows;
    p.given = a->tokens;
    p.top = a->top;
    p.splits = static_cast<int32_t>(splits);
    p.logprobs = a->logprobs;
    p.entropy = a->entropy;
    p.top_ids = a->top_ids;
    p.top_logprobs = a->top_logprobs;
    if (bytes) {
        p.ws_sums = static_cast<float*>(workspace);
        p.ws_top = reinterpret_cast<uint64_t*>(p.ws_sums + 4 * a->num_rows * splits);
    }
    p.status = a->status;
    const hipStream_t s = as_stream(stream);
    if (a->dtype == TV_BF16) return by_top<LogBf16>(p, s);
    if (a->dtype == TV_F16) return by_top<LogF16>(p, s);
    return by_top<LogF32>(p, s);
}
