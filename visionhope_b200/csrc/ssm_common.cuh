// Shared pieces of the selective state space kernels (ssm_scan.cu, ssm_scan_bwd.cu, short_conv.cu).
//
// Sequences are channels-last token rows.  `Seqs` says where each one lies: equally long ones
// follow a batch stride, packed ones start at seq_offsets[s].  Offsets come from the device, so
// the host cannot check them; every kernel clamps them to [0, length], which keeps each access
// inside the tensors whatever they hold.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "common.cuh"
#include "f32x2.cuh"

namespace vh {
namespace ssm {

struct Seqs {
    const int32_t* offsets;  // [count + 1] or null: `count` sequences of `length` tokens
    int64_t length;          // tokens per sequence, or of all packed sequences together
    int32_t count;
    int32_t reverse;         // read each sequence from its last token to its first
};

// One sequence: its first row counted over all tokens (batch-major) and its length.
struct Seq {
    int64_t row;
    int64_t len;
};

__device__ __forceinline__ Seq seq_at(const Seqs& q, int s) {
    if (!q.offsets) return {(int64_t)s * q.length, q.length};
    int64_t lo = q.offsets[s], hi = q.offsets[s + 1];
    lo = lo < 0 ? 0 : (lo > q.length ? q.length : lo);
    hi = hi < lo ? lo : (hi > q.length ? q.length : hi);
    return {lo, hi - lo};
}

// Packed rows of no sequence lie before the first offset and from the last one on (buffers may be
// longer than what they hold).  Outputs and gradients are zero there.
struct Outside {
    int64_t first, last;  // rows [first, last) belong to sequences
    int64_t length;
    __device__ __forceinline__ explicit Outside(const Seqs& q) : first(0), last(INT64_MAX), length(INT64_MAX) {
        if (!q.offsets) return;
        length = q.length;
        first = seq_at(q, 0).row;
        const Seq e = seq_at(q, q.count - 1);
        last = max(first, e.row + e.len);
    }
    __device__ __forceinline__ int64_t count() const { return first + length - last; }
    __device__ __forceinline__ int64_t row(int64_t i) const { return i < first ? i : last + i - first; }
    __device__ __forceinline__ bool has(int64_t row) const { return row < first || row >= last; }
};
// Zeros there in contiguous [rows][width] tensors (null: none); every thread of `blocks` takes part.
template <typename T>
__device__ __forceinline__ void zero_outside(const Seqs& q, int width, int64_t block, int64_t blocks, void* a, void* b = nullptr,
                                             void* c = nullptr) {
    if (!q.offsets) return;
    const Outside o(q);
    const int64_t n = o.count() * width;
    for (int64_t i = block * blockDim.x + threadIdx.x; i < n; i += blocks * blockDim.x) {
        const int64_t at = o.row(i / width) * width + i % width;
        for (void* t : {a, b, c})
            if (t) static_cast<T*>(t)[at] = from_f<T>(0.f);
    }
}

// Slots of `step` tokens: sequence s owns the slots from slot_base on, at least one and at least
// ceil(len / step).  Packed sequences: floor(lo / step) + s, because consecutive starts then
// differ by floor(hi / step) - floor(lo / step) + 1 >= ceil((hi - lo) / step); the total is at
// most floor(length / step) + count.
__host__ __device__ __forceinline__ int64_t slots_per_seq(int64_t len, int step) {
    return len > 0 ? (len + step - 1) / step : 1;
}
__host__ __device__ __forceinline__ int64_t slot_total(bool packed, int64_t length, int32_t count, int step) {
    return packed ? length / step + count : (int64_t)count * slots_per_seq(length, step);
}
__device__ __forceinline__ int64_t slot_base(const Seqs& q, int s, int64_t row, int step) {
    return q.offsets ? row / step + s : (int64_t)s * slots_per_seq(q.length, step);
}

// The sequence that owns slot `slot` (binary search over the monotone slot bases).
__device__ __forceinline__ int seq_of_slot(const Seqs& q, int64_t slot, int step) {
    if (!q.offsets) return (int)(slot / slots_per_seq(q.length, step));
    int lo = 0, hi = q.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        int64_t row = q.offsets[mid];
        row = row < 0 ? 0 : (row > q.length ? q.length : row);
        if (row / step + mid <= slot) lo = mid; else hi = mid - 1;
    }
    return lo;
}

// Token rows of one tensor: element (row r of sequence s, channel c).  Packed tensors ignore the
// batch stride.
struct Rows {
    int64_t batch, token;  // strides in elements
};
__device__ __forceinline__ int64_t first_row(const Seqs& q, const Seq& e, int s, const Rows& r) {
    const int64_t base = q.offsets ? e.row * r.token : (int64_t)s * r.batch;
    return q.reverse && e.len > 0 ? base + (e.len - 1) * r.token : base;
}
__device__ __forceinline__ int64_t row_step(const Seqs& q, const Rows& r) { return q.reverse ? -r.token : r.token; }

// Four consecutive values; `vec`: the address is aligned for one access.
template <typename T>
__device__ __forceinline__ void load_four(const T* p, bool vec, float (&v)[4]) {
    if (vec) {
        const float4 q = load4(p);
        v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = to_f(p[i]);
    }
}
// V consecutive channels from c on, none at or past `end`.  `vec`: the caller's rule says that V-wide
// accesses are aligned and never straddle `end`.
template <int V, typename T>
__device__ __forceinline__ void store_v(T* p, int c, int end, bool vec, const float (&v)[V]) {
    if (V > 1 && vec) {
        if (c < end) {
            if constexpr (V == 4) {
                store4(p, make_float4(v[0], v[1], v[2], v[3]));
            } else {
                struct alignas(sizeof(T) * V) Pack { T e[V]; };
                Pack q;
#pragma unroll
                for (int i = 0; i < V; ++i) q.e[i] = from_f<T>(v[i]);
                *reinterpret_cast<Pack*>(p) = q;
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (c + i < end) p[i] = from_f<T>(v[i]);
    }
}

// V elements as they lie in memory, in whole words (separate 16-bit values would take a register
// each).
__device__ __forceinline__ float2 halves(uint32_t w, __nv_bfloat16) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
__device__ __forceinline__ float2 halves(uint32_t w, __half) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
__device__ __forceinline__ uint32_t join(float a, float b, __nv_bfloat16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t join(float a, float b, __half) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename T, int V>
struct Pack {
    static constexpr int kBytes = sizeof(T) * V;
    using Word = std::conditional_t<kBytes == 2, uint16_t, std::conditional_t<kBytes == 4, uint32_t,
                 std::conditional_t<kBytes == 8, uint2, uint4>>>;
    static_assert(kBytes == 2 || kBytes == 4 || kBytes == 8 || kBytes == 16, "one access");
    Word w;
    __device__ __forceinline__ uint32_t word(int i) const {
        if constexpr (kBytes <= 4) return w;
        else if constexpr (kBytes == 8) return i == 0 ? w.x : w.y;
        else return i == 0 ? w.x : i == 1 ? w.y : i == 2 ? w.z : w.w;
    }
    __device__ __forceinline__ void set_word(int i, uint32_t v) {
        if constexpr (kBytes <= 4) w = (Word)v;
        else if constexpr (kBytes == 8) { if (i == 0) w.x = v; else w.y = v; }
        else { if (i == 0) w.x = v; else if (i == 1) w.y = v; else if (i == 2) w.z = v; else w.w = v; }
    }
    __device__ __forceinline__ void get(float (&v)[V]) const {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < V; ++i) v[i] = __uint_as_float(word(i));
        } else if constexpr (V == 1) {
            v[0] = halves(w, T{}).x;
        } else {
#pragma unroll
            for (int i = 0; i < V / 2; ++i) {
                const float2 f = halves(word(i), T{});
                v[2 * i] = f.x;
                v[2 * i + 1] = f.y;
            }
        }
    }
    __device__ __forceinline__ void set(const float (&v)[V]) {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < V; ++i) set_word(i, __float_as_uint(v[i]));
        } else if constexpr (V == 1) {
            set_word(0, join(v[0], 0.f, T{}));
        } else {
#pragma unroll
            for (int i = 0; i < V / 2; ++i) set_word(i, join(v[2 * i], v[2 * i + 1], T{}));
        }
    }
    // `left`: how many of them exist (vec: the pointer is aligned and all do); missing ones repeat
    // the last
    __device__ __forceinline__ void load(const T* p, int left, bool vec) {
        if (vec) {
            *this = *reinterpret_cast<const Pack*>(p);
        } else {
            float v[V];
#pragma unroll
            for (int i = 0; i < V; ++i) v[i] = to_f(p[max(min(i, left - 1), 0)]);
            set(v);  // exact: they came from T
        }
    }
};

// A Pack into shared memory, asynchronously where the copy is one of 4, 8 or 16 bytes.  Issued a
// group or two ahead of its use it takes no registers; plain loads ahead of their use do, and were
// moved next to it by the compiler (the forward then waited for memory in 4 of 10 cycles).
template <typename T, int V>
__device__ __forceinline__ void fetch(Pack<T, V>* dst, const T* p, int left, bool vec) {
    if constexpr (sizeof(T) * V >= 4) {
        if (vec) {
            cp_async<sizeof(T) * V>(dst, p);
            return;
        }
    }
    Pack<T, V> r;
    r.load(p, left, vec);
    *dst = r;
}

// V values as pairs for the packed arithmetic (V = 1: the second half repeats the first).
template <int V>
constexpr int kPairs = (V + 1) / 2;
template <int V>
__device__ __forceinline__ void to_pairs(const float (&f)[V], float2 (&v)[kPairs<V>]) {
#pragma unroll
    for (int i = 0; i < kPairs<V>; ++i) v[i] = make_float2(f[2 * i], f[V > 1 ? 2 * i + 1 : 0]);
}
template <int V>
__device__ __forceinline__ void from_pairs(const float2 (&v)[kPairs<V>], float (&f)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = i % 2 ? v[i / 2].y : v[i / 2].x;
}
template <typename T, int V>
__device__ __forceinline__ void unpack(const Pack<T, V>& q, float2 (&v)[kPairs<V>]) {
    float f[V];
    q.get(f);
    to_pairs<V>(f, v);
}

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// 2^(s a) on the FMA pipe.  s a = i + f with i the nearest integer (rounded to by adding 1.5 *
// 2^23, whose last mantissa bits then hold i) and |f| <= 1/2, f from one fused multiply-add; 2^f =
// 1 + f q(f), q of degree 5 fitted for the relative error of 2^f by Lawson's iteration (2.0e-9);
// 2^i goes into the exponent.  Evaluated in fp32 it is off by 2.7e-8 root mean square and 0.9e-9
// on average, against 3.8e-8 and -2e-8 for ex2.approx on [-0.1, 0] (one rounding: 1.8e-8): a
// state that remembers a thousand tokens multiplies by a thousand decays, and there an average
// error adds up.  Past |s a| = 126 (and for NaN) the hardware function: no scaling of the
// exponent there.
constexpr float kRound = 12582912.f;
constexpr int kExp2Terms = 6;
__device__ __forceinline__ float exp2_term(int i) {
    constexpr float kQ[kExp2Terms] = {0.6931471824645996f,  0.24022647738456726f,  0.055503323674201965f,
                                      0.00961843691766262f, 0.0013398873852565885f, 0.00015353361959569156f};
    return kQ[i];
}
__device__ __forceinline__ float exp2_fma(float s, float a) {
    const float t = __fmaf_rn(s, a, kRound), f = __fmaf_rn(s, a, __fsub_rn(kRound, t));
    float q = exp2_term(kExp2Terms - 1);
#pragma unroll
    for (int i = kExp2Terms - 2; i >= 0; --i) q = __fmaf_rn(q, f, exp2_term(i));
    const float y = __int_as_float(__float_as_int(__fmaf_rn(q, f, 1.f)) + (__float_as_int(t) << 23));
    const float x = s * a;
    return fabsf(x) <= 126.f ? y : ex2(x);
}

__device__ __forceinline__ float rcp(float x) {  // of a normal number or infinity
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float sigmoid(float x) { return rcp(1.f + ex2(-kLog2e * x)); }
// Each with a reciprocal of its own.  One reciprocal for both, 1 / a = b / (a b), is an operation of the
// special-function unit less, but a b has to be kept finite (the result then stays above a bound,
// and times a large negative x grows with it) and a result of 1 comes out as 1 + O(2^-23) by its
// neighbour, which x (1 - sigmoid(x)) in silu's derivative multiplies by x.
__device__ __forceinline__ float2 sigmoid2(float2 x) {
    const float2 m = fmul2(x, splat2(-kLog2e)), d = fadd2(make_float2(ex2(m.x), ex2(m.y)), splat2(1.f));
    return make_float2(rcp(d.x), rcp(d.y));
}

// log(1 + exp(x)) without cancellation on either side: max(x, 0) + log1p(e), e = exp(-|x|) in
// (0, 1], log1p(e) = e r(e) with r of degree 8 fitted for the relative error by Lawson's
// iteration (3.0e-8).  The rounding of |x| log2(e), which e would carry as a relative error of
// up to |x| 2^-24, is added back to first order.
constexpr int kLog1pTerms = 9;
__device__ __forceinline__ float log1p_term(int i) {
    constexpr float kR[kLog1pTerms] = {0.9999999403953552f,   -0.4999949336051941f, 0.3331909775733948f,
                                       -0.2484298199415207f,  0.19106006622314453f, -0.13663244247436523f,
                                       0.07822594046592712f, -0.029505232349038124f, 0.005232692696154118f};
    return kR[i];
}
__device__ __forceinline__ float max_nan(float a, float b) {  // NaN if either is
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 softplus2(float2 x) {
    // exp(-104) is 0 here: past it the result is max(x, 0)
    const float2 m = make_float2(fmaxf(-fabsf(x.x), -104.f), fmaxf(-fabsf(x.y), -104.f));
    const float2 hi = fmul2(m, splat2(kLog2e)), lo = ffma2(m, splat2(kLog2e), fmul2(hi, splat2(-1.f)));
    float2 e = make_float2(ex2(hi.x), ex2(hi.y));
    e = ffma2(e, fmul2(lo, splat2(kLn2)), e);
    float2 r = splat2(log1p_term(kLog1pTerms - 1));
#pragma unroll
    for (int i = kLog1pTerms - 2; i >= 0; --i) r = ffma2(r, e, splat2(log1p_term(i)));
    return ffma2(e, r, make_float2(max_nan(x.x, 0.f), max_nan(x.y, 0.f)));
}
__device__ __forceinline__ float softplus(float x) { return softplus2(make_float2(x, x)).x; }

// Two of them, without the range check: |s a| <= 126.  The same bits as exp2_fma.
__device__ __forceinline__ float2 exp2_fma2(float2 s, float2 a) {
    const float2 t = ffma2(s, a, splat2(kRound)), f = ffma2(s, a, fsub2(splat2(kRound), t));
    float2 q = splat2(exp2_term(kExp2Terms - 1));
#pragma unroll
    for (int i = kExp2Terms - 2; i >= 0; --i) q = ffma2(q, f, splat2(exp2_term(i)));
    q = ffma2(q, f, splat2(1.f));
    return make_float2(__int_as_float(__float_as_int(q.x) + (__float_as_int(t.x) << 23)),
                       __int_as_float(__float_as_int(q.y) + (__float_as_int(t.y) << 23)));
}

__device__ __forceinline__ float2 ex2_2(float2 x) { return make_float2(ex2(x.x), ex2(x.y)); }

// A in the exponential's base: log2(e) A, kept finite so that a step of zero leaves the state as
// it is (0 * inf would not).  NaN stays NaN.
__device__ __forceinline__ float to_log2(float a) {
    const float v = a * kLog2e;
    constexpr float kMax = 3.4028234e38f;
    return v < -kMax ? -kMax : (v > kMax ? kMax : v);
}

// Sum over lane groups with the values scattered: V values per lane enter, and after log2(LANES)
// exchanges over lane distances DIST, 2 DIST, ... (largest first) each lane holds the sums of
// V / LANES of them (one, summed over all lanes, when LANES > V).  The lane whose index among
// the LANES is j keeps the values from j * V / LANES on.
template <int V, int LANES, int DIST>
__device__ __forceinline__ void reduce_scatter(float (&v)[V], int lane) {
    if constexpr (LANES > 1) {
        constexpr int kMask = (LANES / 2) * DIST;
        if constexpr (V > 1) {
            const bool upper = lane & kMask;
            float keep[V / 2];
#pragma unroll
            for (int i = 0; i < V / 2; ++i) {
                const float send = upper ? v[i] : v[i + V / 2];
                keep[i] = (upper ? v[i + V / 2] : v[i]) + __shfl_xor_sync(0xffffffffu, send, kMask);
            }
            reduce_scatter<V / 2, LANES / 2, DIST>(keep, lane);
#pragma unroll
            for (int i = 0; i < V / 2; ++i) v[i] = keep[i];
        } else {
            v[0] += __shfl_xor_sync(0xffffffffu, v[0], kMask);
            reduce_scatter<1, LANES / 2, DIST>(v, lane);
        }
    }
}

}  // namespace ssm
}  // namespace vh
