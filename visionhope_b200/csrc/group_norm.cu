// Group norm over channels-last data with an activation and a gate, forward and backward.
//
// A sample has `pixels` rows of `channels`, and a group `per` = channels / groups of them.  Over the
// m = pixels * per values of a group:
//     x^ = (x - mean) rstd,   pre = weight x^ + bias,   y = act(pre) silu(gate)
// and back, with dn = dy silu(gate) act'(pre), a = weight dn:
//     dx = rstd (a - mean(a) - x^ mean(a x^)),  dgate = dy act(pre) silu'(gate),
//     dweight = sum dn x^,  dbias = sum dn.
// All of it is fp32 and bound by memory: x (and the gate) in, y out; back x, dy (and the gate) in, dx
// (and the gate's) out.  Three forms, by where a group's values fit:
//   rows      one pixel a sample: a group in the registers of 4 to 32 lanes
//   resident  a slab of whole groups in the shared memory of a cluster of 1 to 8 CTAs, each a slice of
//             the pixels: x is read once
//   split     larger ones: partial sums a slice, one kernel that joins them, a second pass over x
// The variance comes from differences to the mean (rows) or to a channel's first value in the slice, joined by
// Chan's formula, so that a large mean costs nothing.
//
// Measured (bf16, forward + backward): 50176 gated rows of 256 channels 23 + 28 us, 3.3 and 4.5 TB/s; 64 maps of
// 56 x 56 x 128 with SiLU 41 + 70 us (resident), 2.5 and 2.2 TB/s; two maps of 128 x 512 x 128 with GELU 36 us
// (split, forward).  Issue slots are 38 to 48 % busy, with 14 to 20 warps an SM: latency between the passes.
#include <algorithm>

#include "abi_util.h"
#include "activations.cuh"
#include "common.cuh"
#include "ssm_common.cuh"
#include "vhope.h"

namespace vh {
namespace gn {
namespace {

constexpr int kThreads = 128;  // of a block; half as many as 256 pay half as often for a channel's parameters
constexpr int kJoinThreads = 256;
constexpr int kMaxCluster = 8;

struct Norm {
    const void *x, *gate;
    int64_t xs, xp, gs, gp;  // sample and pixel strides of x and the gate
    const float *weight, *bias;
    void* y;                 // contiguous, as dy, dx and dgate
    float *mean, *rstd;      // [samples, groups]
    const void* dy;
    void *dx, *dgate;
    float* part;             // sums for the parameters [parts][2][channels], or the split form's
    int64_t samples, pixels;
    float eps;
    int channels, groups, per, act;
};

// ---- V consecutive values, as pairs for the packed arithmetic --------------------------------------
template <int V>
constexpr int kP = ssm::kPairs<V>;

template <int V, typename T>
__device__ __forceinline__ void unpack(const ssm::Pack<T, V>& q, float2 (&v)[kP<V>]) {
    ssm::unpack<T, V>(q, v);
}
template <int V, typename T>
__device__ __forceinline__ void get(const T* p, float2 (&v)[kP<V>]) {
    ssm::unpack<T, V>(*reinterpret_cast<const ssm::Pack<T, V>*>(p), v);
}
template <int V, typename T>
__device__ __forceinline__ void put(T* p, const float2 (&v)[kP<V>]) {
    float f[V];
    ssm::from_pairs<V>(v, f);
    ssm::Pack<T, V> q;
    q.set(f);
    *reinterpret_cast<ssm::Pack<T, V>*>(p) = q;
}
template <int V>
__device__ __forceinline__ void set_pair(float2 (&v)[kP<V>], int i, float f) {
    if (V == 1) v[0] = splat2(f);
    else if (i % 2) v[i / 2].y = f;
    else v[i / 2].x = f;
}
// The sum of V values.
template <int V>
__device__ __forceinline__ float total(const float2 (&v)[kP<V>]) {
    if constexpr (V == 1) return v[0].x;
    float2 s = v[0];
#pragma unroll
    for (int i = 1; i < kP<V>; ++i) s = fadd2(s, v[i]);
    return s.x + s.y;
}

// ---- activations --------------------------------------------------------------------------------
// Phi(x) and its density.  16-bit outputs take the approximation of gelu2 (absolute error 7.5e-8).
template <typename T>
__device__ __forceinline__ void normal_cdf(float2 x, float2* cdf, float2* density) {
    constexpr float kDensity = 0.3989422804014327f;
    if constexpr (sizeof(T) == 4) {
        *cdf = make_float2(0.5f * erfcf(-0.70710678118654752f * x.x), 0.5f * erfcf(-0.70710678118654752f * x.y));
        *density = make_float2(kDensity * expf(-0.5f * x.x * x.x), kDensity * expf(-0.5f * x.y * x.y));
    } else {
        const float2 ax = make_float2(fabsf(x.x), fabsf(x.y));
        const float2 d = ffma2(ax, splat2(0.3275911f * 0.70710678118654752f), splat2(1.f));
        const float2 t = make_float2(rcp_approx(d.x), rcp_approx(d.y));
        const float2 arg = fmul2(fmul2(x, x), splat2(-0.5f * 1.4426950408889634f));
        const float2 e = make_float2(ex2_approx(arg.x), ex2_approx(arg.y));
        float2 q = ffma2(t, splat2(0.5f * 1.061405429f), splat2(0.5f * -1.453152027f));
        q = ffma2(q, t, splat2(0.5f * 1.421413741f));
        q = ffma2(q, t, splat2(0.5f * -0.284496736f));
        q = ffma2(q, t, splat2(0.5f * 0.254829592f));
        q = fmul2(fmul2(q, t), e);
        const float2 r = fsub2(splat2(1.f), q);
        *cdf = make_float2(x.x >= 0.f ? r.x : (x.x < 0.f ? q.x : x.x), x.y >= 0.f ? r.y : (x.y < 0.f ? q.y : x.y));
        *density = fmul2(e, splat2(kDensity));
    }
}

// x sigmoid(x), and its derivative s + x s (1 - s).
__device__ __forceinline__ float2 silu2(float2 x, float2* slope) {
    const float2 s = ssm::sigmoid2(x), y = fmul2(x, s);
    *slope = ffma2(y, fsub2(splat2(1.f), s), s);
    return y;
}
__device__ __forceinline__ float2 silu2(float2 x) { return fmul2(x, ssm::sigmoid2(x)); }

// act(pre) in place of pre.
template <typename T, int V>
__device__ __forceinline__ void activate(int act, float2 (&pre)[kP<V>]) {
    if (act == 1) {
#pragma unroll
        for (int i = 0; i < kP<V>; ++i) pre[i] = silu2(pre[i]);
    } else if (act == 2) {
#pragma unroll
        for (int i = 0; i < kP<V>; ++i) {
            float2 cdf, density;
            normal_cdf<T>(pre[i], &cdf, &density);
            pre[i] = fmul2(pre[i], cdf);
        }
    }
}
// d act'(pre) in place of d; act(pre) in place of pre if WANT.
template <typename T, bool WANT, int V>
__device__ __forceinline__ void through(int act, float2 (&pre)[kP<V>], float2 (&d)[kP<V>]) {
    if (act == 1) {
#pragma unroll
        for (int i = 0; i < kP<V>; ++i) {
            float2 slope;
            const float2 y = silu2(pre[i], &slope);
            d[i] = fmul2(d[i], slope);
            if (WANT) pre[i] = y;
        }
    } else if (act == 2) {
#pragma unroll
        for (int i = 0; i < kP<V>; ++i) {
            float2 cdf, density;
            normal_cdf<T>(pre[i], &cdf, &density);
            d[i] = fmul2(d[i], ffma2(pre[i], density, cdf));
            if (WANT) pre[i] = fmul2(pre[i], cdf);
        }
    }
}

// ---- channels -----------------------------------------------------------------------------------
// f(i, g) for V channels from c on, i = 0..V-1, with g the group of channel c + i: one division for all of them
// (a thread has some fifty values, and one division a channel were a third of its instructions).
template <int V, typename F>
__device__ __forceinline__ void with_groups(int c, int per, F&& f) {
    int g = c / per, left = per - (c - g * per);
#pragma unroll
    for (int i = 0; i < V; ++i) {
        f(i, g);
        if (--left == 0) {
            ++g;
            left = per;
        }
    }
}
// Parameters and statistics of V channels from c on.
template <int V>
struct Channel {
    float2 w[kP<V>], b[kP<V>], mean[kP<V>], rstd[kP<V>];
    __device__ __forceinline__ void params(const Norm& p, int c) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            set_pair<V>(w, i, p.weight ? p.weight[c + i] : 1.f);
            set_pair<V>(b, i, p.bias ? p.bias[c + i] : 0.f);
        }
    }
    // `m`, `r`: of the groups from the one of channel c0 on
    __device__ __forceinline__ void stats(const float* m, const float* r, int per, int c, int c0) {
        with_groups<V>(c - c0, per, [&](int i, int g) {
            set_pair<V>(mean, i, m[g]);
            set_pair<V>(rstd, i, r[g]);
        });
    }
    __device__ __forceinline__ void stats(float m, float r) {
#pragma unroll
        for (int i = 0; i < kP<V>; ++i) {
            mean[i] = splat2(m);
            rstd[i] = splat2(r);
        }
    }
};

// y of V values.
template <typename T, int V>
__device__ __forceinline__ void forward(const Norm& p, const Channel<V>& k, float2 (&x)[kP<V>], bool gated, const ssm::Pack<T, V>& gate, T* y) {
#pragma unroll
    for (int i = 0; i < kP<V>; ++i) x[i] = ffma2(fmul2(fsub2(x[i], k.mean[i]), k.rstd[i]), k.w[i], k.b[i]);
    activate<T, V>(p.act, x);
    if (gated) {
        float2 z[kP<V>];
        unpack<V>(gate, z);
#pragma unroll
        for (int i = 0; i < kP<V>; ++i) x[i] = fmul2(x[i], silu2(z[i]));
    }
    put<V>(y, x);
}

// x^ in place of x and dn in place of dy; the gate's gradient if `dgate`.
template <typename T, int V>
__device__ __forceinline__ void backward(const Norm& p, const Channel<V>& k, float2 (&x)[kP<V>], float2 (&dy)[kP<V>], bool gated,
                                         const ssm::Pack<T, V>& gate, T* dgate) {
    float2 pre[kP<V>];
#pragma unroll
    for (int i = 0; i < kP<V>; ++i) {
        x[i] = fmul2(fsub2(x[i], k.mean[i]), k.rstd[i]);
        pre[i] = ffma2(x[i], k.w[i], k.b[i]);
    }
    if (gated) {
        float2 z[kP<V>], dz[kP<V>];
        unpack<V>(gate, z);
#pragma unroll
        for (int i = 0; i < kP<V>; ++i) {
            const float2 g = silu2(z[i], &z[i]);
            dz[i] = fmul2(dy[i], z[i]);
            dy[i] = fmul2(dy[i], g);
        }
        through<T, true, V>(p.act, pre, dy);
        if (dgate) {
#pragma unroll
            for (int i = 0; i < kP<V>; ++i) dz[i] = fmul2(dz[i], pre[i]);
            put<V>(dgate, dz);
        }
    } else {
        through<T, false, V>(p.act, pre, dy);
    }
}
// rstd (w dn - a - x^ b) from x^ and dn, with a and b times rstd already.
template <int V>
__device__ __forceinline__ void input_gradient(const Channel<V>& k, const float2 (&x)[kP<V>], float2 (&d)[kP<V>], const float2 (&ra)[kP<V>],
                                               const float2 (&rb)[kP<V>]) {
#pragma unroll
    for (int i = 0; i < kP<V>; ++i) d[i] = fsub2(fsub2(fmul2(fmul2(k.rstd[i], k.w[i]), d[i]), ra[i]), fmul2(x[i], rb[i]));
}

__device__ __forceinline__ float rstd_of(float m2, float count, float eps) { return 1.f / sqrtf(m2 / count + eps); }

// ---- rows ---------------------------------------------------------------------------------------
// SW lanes hold a group, NV vectors of V each; a block covers `gb` groups of several rows at a time and
// walks down the rows, so that a thread's channels, and their parameters and sums, stay in registers.
template <int SW>
__device__ __forceinline__ float lanes_sum(float v) {
    const unsigned mask = SW == 32 ? 0xffffffffu : ((1u << SW) - 1u) << (threadIdx.x & 31 & ~(SW - 1));
#pragma unroll
    for (int o = SW / 2; o > 0; o >>= 1) v += __shfl_xor_sync(mask, v, o, SW);
    return v;
}

template <typename T, int V, int SW, int NV, bool BACK>
__global__ void __launch_bounds__(kThreads) rows_kernel(Norm p, int gb) {
    constexpr int P = kP<V>;
    using Pack = ssm::Pack<T, V>;
    const int lane = threadIdx.x % SW, unit = threadIdx.x / SW, phases = kThreads / (gb * SW);
    const int g = blockIdx.y * gb + unit % gb, phase = unit / gb;
    const bool live = phase < phases && g < p.groups, gated = p.gate != nullptr;
    const int c0 = live ? g * p.per : 0;
    Channel<V> k[NV];
    bool has[NV];
    float2 aw[NV][P], ab[NV][P];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int c = (lane + j * SW) * V;
        has[j] = live && c < p.per;
        k[j].params(p, has[j] ? c0 + c : 0);
#pragma unroll
        for (int i = 0; i < P; ++i) aw[j][i] = ab[j][i] = splat2(0.f);
    }
    const float count = (float)p.per;
    // a row's values, fetched while the one before is worked on
    struct Row {
        Pack x[NV], z[NV], d[NV];
        float mean, rstd;
    };
    auto fetch = [&](Row& q, int64_t r) {
        const T* x = static_cast<const T*>(p.x) + r * p.xs + c0 + lane * V;
        const T* z = static_cast<const T*>(p.gate) + r * p.gs + c0 + lane * V;
        const T* d = static_cast<const T*>(p.dy) + r * p.channels + c0 + lane * V;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            if (has[j]) {
                q.x[j] = *reinterpret_cast<const Pack*>(x + j * SW * V);
                if (gated) q.z[j] = *reinterpret_cast<const Pack*>(z + j * SW * V);
                if (BACK) q.d[j] = *reinterpret_cast<const Pack*>(d + j * SW * V);
            }
        }
        if (BACK) {
            q.mean = p.mean[r * p.groups + g];
            q.rstd = p.rstd[r * p.groups + g];
        }
    };
    const int64_t step = (int64_t)gridDim.x * phases;
    int64_t r = (int64_t)blockIdx.x * phases + phase;
    if (live && r < p.samples) {
        Row next;
        fetch(next, r);
        for (; r < p.samples; r += step) {
            const Row q = next;
            if (r + step < p.samples) fetch(next, r + step);
            const int64_t at = r * p.channels + c0 + lane * V;
            float2 v[NV][P];
#pragma unroll
            for (int j = 0; j < NV; ++j) unpack<V>(q.x[j], v[j]);
            if constexpr (!BACK) {
                float s = 0.f;
#pragma unroll
                for (int j = 0; j < NV; ++j) s += has[j] ? total<V>(v[j]) : 0.f;
                const float mean = lanes_sum<SW>(s) / count;
                s = 0.f;
#pragma unroll
                for (int j = 0; j < NV; ++j) {
                    float2 d[P];
#pragma unroll
                    for (int i = 0; i < P; ++i) {
                        d[i] = fsub2(v[j][i], splat2(mean));
                        d[i] = fmul2(d[i], d[i]);
                    }
                    s += has[j] ? total<V>(d) : 0.f;
                }
                const float rstd = rstd_of(lanes_sum<SW>(s), count, p.eps);
                if (p.mean && lane == 0) {
                    p.mean[r * p.groups + g] = mean;
                    p.rstd[r * p.groups + g] = rstd;
                }
#pragma unroll
                for (int j = 0; j < NV; ++j)
                    if (has[j]) {
                        k[j].stats(mean, rstd);
                        forward<T, V>(p, k[j], v[j], gated, q.z[j], static_cast<T*>(p.y) + at + j * SW * V);
                    }
            } else {
                float2 d[NV][P];
                float s1 = 0.f, s2 = 0.f;
#pragma unroll
                for (int j = 0; j < NV; ++j)
                    if (has[j]) {
                        unpack<V>(q.d[j], d[j]);
                        k[j].stats(q.mean, q.rstd);
                        backward<T, V>(p, k[j], v[j], d[j], gated, q.z[j], p.dgate ? static_cast<T*>(p.dgate) + at + j * SW * V : nullptr);
                        float2 a[P], b[P];
#pragma unroll
                        for (int i = 0; i < P; ++i) {
                            ab[j][i] = fadd2(ab[j][i], d[j][i]);
                            aw[j][i] = ffma2(d[j][i], v[j][i], aw[j][i]);
                            a[i] = fmul2(d[j][i], k[j].w[i]);
                            b[i] = fmul2(a[i], v[j][i]);
                        }
                        s1 += total<V>(a);
                        s2 += total<V>(b);
                    }
                const float2 ra = splat2(lanes_sum<SW>(s1) / count * q.rstd), rb = splat2(lanes_sum<SW>(s2) / count * q.rstd);
#pragma unroll
                for (int j = 0; j < NV; ++j)
                    if (has[j]) {
                        float2 a[P], b[P];
#pragma unroll
                        for (int i = 0; i < P; ++i) {
                            a[i] = ra;
                            b[i] = rb;
                        }
                        input_gradient<V>(k[j], v[j], d[j], a, b);
                        put<V>(static_cast<T*>(p.dx) + at + j * SW * V, d[j]);
                    }
            }
        }
    }
    if constexpr (BACK) {
        // the row phases in order, each thread's channels
        extern __shared__ float red[];
        float* out = p.part + (int64_t)blockIdx.x * 2 * p.channels;
        for (int ph = 0; ph < phases; ++ph) {
            __syncthreads();
            if (live && phase == ph) {
#pragma unroll
                for (int j = 0; j < NV; ++j)
                    if (has[j]) {
                        const int c = (lane + j * SW) * V, at = (unit % gb) * p.per + c;
                        float fb[V], fw[V];
                        ssm::from_pairs<V>(ab[j], fb);
                        ssm::from_pairs<V>(aw[j], fw);
#pragma unroll
                        for (int i = 0; i < V; ++i) {
                            const float b = (ph ? red[2 * (at + i)] : 0.f) + fb[i];
                            const float w = (ph ? red[2 * (at + i) + 1] : 0.f) + fw[i];
                            if (ph + 1 < phases) {
                                red[2 * (at + i)] = b;
                                red[2 * (at + i) + 1] = w;
                            } else {
                                out[c0 + c + i] = b;
                                out[p.channels + c0 + c + i] = w;
                            }
                        }
                    }
            }
        }
    }
}

// Sums of `parts` rows of [2][channels] in a fixed order: bias, weight.
__global__ void __launch_bounds__(1024) params_kernel(const float* __restrict__ part, int64_t parts, int channels, float* dweight,
                                                      float* dbias) {
    __shared__ float red[32][33];
    const int i = blockIdx.x * 32 + threadIdx.x, n = 2 * channels;
    float s = 0.f;
    if (i < n)
        for (int64_t r = threadIdx.y; r < parts; r += 32) s += part[r * n + i];
    red[threadIdx.y][threadIdx.x] = s;
    __syncthreads();
    if (threadIdx.y == 0 && i < n) {
        s = 0.f;
        for (int r = 0; r < 32; ++r) s += red[r][threadIdx.x];
        float* out = i < channels ? dbias : dweight;
        if (out) out[i < channels ? i : i - channels] = s;
    }
}

// ---- pixels over a block ------------------------------------------------------------------------
// A block's threads over w channels: qn = w / V vectors side by side, kThreads / qn pixel phases.
// fetch(c, r) reads what work(c, r, .) takes for the vector at channel c of pixel r; U pixels are fetched
// before the first is worked on, as loads do not pass the stores of another pixel.  before(c) and
// after(...) stand around the pixels of each vector.
template <int V, int U, typename B, typename L, typename F, typename A>
__device__ __forceinline__ void each(int w, int rows, B&& before, L&& fetch, F&& work, A&& after) {
    const int q = w / V;
    for (int q0 = 0; q0 < q; q0 += kThreads) {
        const int qn = min(q - q0, kThreads), phases = kThreads / qn;
        const int qi = threadIdx.x % qn, ph = threadIdx.x / qn;
        {  // threads past the last phase have a vector and no pixel
            const int c = (q0 + qi) * V;
            before(c);
            int r = ph < phases ? ph : rows;
            for (; r + (U - 1) * phases < rows; r += U * phases) {
                decltype(fetch(c, r)) raw[U];
#pragma unroll
                for (int u = 0; u < U; ++u) raw[u] = fetch(c, r + u * phases);
#pragma unroll
                for (int u = 0; u < U; ++u) work(c, r + u * phases, raw[u]);
            }
            for (; r < rows; r += phases) work(c, r, fetch(c, r));
        }
        after(q0, qn, phases, qi, ph);
    }
}

// Adds V pairs of values of each thread over the pixel phases, into outa and outb [0..w), in a fixed order:
// the lanes of a warp with the same vector, then the warps; or, where the vectors are no power of two up to
// 32, runs of phases side by side, then the runs.  `red`: kThreads * V floats.
template <int V>
__device__ __forceinline__ void add_phases(const float2 (&pa)[kP<V>], const float2 (&pb)[kP<V>], int q0, int qn, int phases, int qi, int ph,
                                           float* red, float* outa, float* outb) {
    const int n = qn * V;
    float v[2][V];
    ssm::from_pairs<V>(pa, v[0]);
    ssm::from_pairs<V>(pb, v[1]);
    if (qn <= 4 && (qn & (qn - 1)) == 0) {
        for (int o = qn; o < 32; o *= 2)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                v[0][i] += __shfl_xor_sync(0xffffffffu, v[0][i], o);
                v[1][i] += __shfl_xor_sync(0xffffffffu, v[1][i], o);
            }
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;  // 2 n <= kThreads / 32 * V * 2: red holds all warps
        __syncthreads();
        if (lane < qn) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                red[warp * 2 * n + lane * V + i] = v[0][i];
                red[warp * 2 * n + n + lane * V + i] = v[1][i];
            }
        }
        __syncthreads();
        for (int c = threadIdx.x; c < 2 * n; c += kThreads) {
            float s = 0.f;
#pragma unroll
            for (int k = 0; k < kThreads / 32; ++k) s += red[k * 2 * n + c];
            (c < n ? outa : outb)[q0 * V + (c < n ? c : c - n)] = s;
        }
        __syncthreads();
        return;
    }
    for (int which = 0; which < 2; ++which) {
        float* out = which ? outb : outa;
        __syncthreads();
        if (ph < phases) {
#pragma unroll
            for (int i = 0; i < V; ++i) red[ph * n + qi * V + i] = which ? v[1][i] : v[0][i];
        }
        __syncthreads();
        const int runs = max(1, min(phases, kThreads / n)), len = (phases + runs - 1) / runs;
        float s = 0.f;
        if (runs > 1) {
            const int c = threadIdx.x % n, run = threadIdx.x / n;
            if (run < runs)
                for (int k = run * len; k < min(phases, (run + 1) * len); ++k) s += red[k * n + c];
            __syncthreads();
            if (run < runs) red[run * n + c] = s;
            __syncthreads();
        }
        const int left = runs > 1 ? runs : phases;
        for (int c = threadIdx.x; c < n; c += kThreads) {
            s = 0.f;
            for (int k = 0; k < left; ++k) s += red[k * n + c];
            out[q0 * V + c] = s;
        }
    }
    __syncthreads();
}

// Of values seen as differences to a pivot (`sum`, `square` over `rows` pixels): each channel's mean and sum of
// squares around it, in place.
template <typename Pivot>
__device__ __forceinline__ void center(float* sum, float* square, int w, int rows, Pivot&& pivot) {
    const float inv = rows ? 1.f / (float)rows : 0.f;
    for (int c = threadIdx.x; c < w; c += kThreads) {
        const float m = sum[c] * inv;
        const float q = square[c] - sum[c] * m;
        square[c] = q < 0.f ? 0.f : q;  // NaN stays
        sum[c] = rows ? pivot(c) + m : 0.f;
    }
    __syncthreads();
}

// Sums over each group's channels, a warp a group.
__device__ __forceinline__ void add_groups(const float* channel, int w, int per, float* out) {
    const int lane = threadIdx.x & 31;
    for (int g = threadIdx.x >> 5; g < w / per; g += kThreads / 32) {
        float s = 0.f;
        for (int c = lane; c < per; c += 32) s += channel[g * per + c];
        s = warp_sum(s);
        if (lane == 0) out[g] = s;
    }
    __syncthreads();
}

// A group's mean and squares from its channels', each over `rows` pixels: a warp a group.
__device__ __forceinline__ void join_groups(const float* mean, const float* square, int w, int per, int rows, float* gmean, float* gsquare) {
    const int lane = threadIdx.x & 31;
    for (int g = threadIdx.x >> 5; g < w / per; g += kThreads / 32) {
        float s = 0.f, q = 0.f;
        for (int c = lane; c < per; c += 32) s += mean[g * per + c];
        const float mu = warp_sum(s) / (float)per;
        for (int c = lane; c < per; c += 32) {
            const float d = mean[g * per + c] - mu;
            q += fmaf((float)rows * d, d, square[g * per + c]);
        }
        q = warp_sum(q);
        if (lane == 0) {
            gmean[g] = mu;
            gsquare[g] = q;
        }
    }
    __syncthreads();
}

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float ld_cluster(const float* local, uint32_t rank) {
    const uint32_t a = static_cast<uint32_t>(__cvta_generic_to_shared(local));
    uint32_t remote;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(a), "r"(rank));
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(remote) : "memory");
    return v;
}

// Pixels are cut into `parts` slices of one length, the last ones shorter or empty.
__host__ __device__ __forceinline__ int slice_len(int64_t pixels, int parts) { return (int)((pixels + parts - 1) / parts); }
__device__ __forceinline__ int slice_rows(int64_t pixels, int part, int parts) {
    const int len = slice_len(pixels, parts);
    const int64_t left = pixels - (int64_t)part * len;
    return (int)(left < 0 ? 0 : left < len ? left : len);
}

// A slab of w channels of a slice of pixels into shared memory, [rows][w].
template <typename T, int V>
__device__ __forceinline__ void load_slab(T* dst, const T* src, int64_t pixel, int rows, int w) {
    const int q = w / V;
    const unsigned total = (unsigned)rows * q;
    for (unsigned i = threadIdx.x; i < total; i += kThreads) {
        const int r = i / q, c = (i % q) * V;
        if constexpr (V * sizeof(T) == 16) cp_async<16>(dst + (int64_t)r * w + c, src + r * pixel + c);
        else dst[(int64_t)r * w + c] = src[r * pixel + c];
    }
}

// Floats ahead of the slab: two arrays of channels, the sums' scratch, four of groups, two of pairs.
__host__ __device__ inline size_t head_floats(int w, int per, int v) {
    return ((size_t)(2 * w + kThreads * v + 4 * (w / per)) + 3) / 4 * 4;
}

// ---- resident -----------------------------------------------------------------------------------
template <typename T, int V, bool BACK>
__global__ void __launch_bounds__(kThreads) resident_kernel(Norm p, int width, int slabs, int cluster) {
    extern __shared__ __align__(16) float head[];
    const uint32_t rank = cluster > 1 ? cluster_rank() : 0;
    const int64_t unit = blockIdx.x / cluster, n = unit / slabs;
    const int c0 = (int)(unit % slabs) * width, w = min(width, p.channels - c0), per = p.per, groups = w / per;
    float *ca = head, *cb = ca + width, *red = cb + width, *ga = red + kThreads * V, *gb = ga + width / per,
          *mean = gb + width / per, *rstd = mean + width / per;
    T* xs = reinterpret_cast<T*>(head + head_floats(width, per, V));
    const int len = slice_len(p.pixels, cluster), rows = slice_rows(p.pixels, rank, cluster);
    const int64_t s0 = (int64_t)rank * len;
    T* ds = xs + len * width;

    load_slab<T, V>(xs, static_cast<const T*>(p.x) + n * p.xs + s0 * p.xp + c0, p.xp, rows, w);
    const int64_t at = (n * p.pixels + s0) * p.channels + c0;  // in contiguous tensors
    const T* gate = p.gate ? static_cast<const T*>(p.gate) + n * p.gs + s0 * p.gp + c0 : nullptr;
    if constexpr (BACK) load_slab<T, V>(ds, static_cast<const T*>(p.dy) + at, p.channels, rows, w);
    cp_async_commit();
    cp_async_wait<0>();
    __syncthreads();

    Channel<V> k;
    constexpr int P = kP<V>;
    using Pack = ssm::Pack<T, V>;
    const bool gated = gate != nullptr;
    auto gate_at = [&](int c, int r) {
        Pack z = {};
        if (gated) z = *reinterpret_cast<const Pack*>(gate + r * p.gp + c);
        return z;
    };
    struct Two {
        Pack a, b;
    };
    struct Three {
        Pack a, b, c;
    };
    auto three = [&](int c, int r) {
        return Three{*reinterpret_cast<const Pack*>(xs + r * w + c), *reinterpret_cast<const Pack*>(ds + r * w + c), gate_at(c, r)};
    };
    if constexpr (!BACK) {
        // sums of differences to the slice's first pixel, a channel
        float2 sum[P], square[P], first[P];
        each<V, 1>(w, rows,
                   [&](int c) {
                       get<V>(xs + c, first);
#pragma unroll
                       for (int i = 0; i < P; ++i) sum[i] = square[i] = splat2(0.f);
                   },
                   [&](int c, int r) { return *reinterpret_cast<const Pack*>(xs + r * w + c); },
                   [&](int, int, const Pack& q) {
                       float2 v[P];
                       unpack<V>(q, v);
#pragma unroll
                       for (int i = 0; i < P; ++i) {
                           v[i] = fsub2(v[i], first[i]);
                           sum[i] = fadd2(sum[i], v[i]);
                           square[i] = ffma2(v[i], v[i], square[i]);
                       }
                   },
                   [&](int q0, int qn, int phases, int qi, int ph) { add_phases<V>(sum, square, q0, qn, phases, qi, ph, red, ca, cb); });
        center(ca, cb, w, rows, [&](int c) { return to_f(xs[c]); });
        join_groups(ca, cb, w, per, rows, ga, gb);
        if (cluster > 1) cluster_sync();
        const float m = (float)p.pixels * per;
        for (int g = threadIdx.x; g < groups; g += kThreads) {
            float part[kMaxCluster], more[kMaxCluster], mu = 0.f, m2 = 0.f;
#pragma unroll
            for (int j = 0; j < kMaxCluster; ++j) {
                part[j] = j < cluster ? (cluster > 1 ? ld_cluster(ga + g, j) : ga[g]) : 0.f;
                more[j] = j < cluster ? (cluster > 1 ? ld_cluster(gb + g, j) : gb[g]) : 0.f;
            }
#pragma unroll
            for (int j = 0; j < kMaxCluster; ++j) mu = fmaf((float)slice_rows(p.pixels, j, cluster) * per / m, part[j], mu);
#pragma unroll
            for (int j = 0; j < kMaxCluster; ++j) {
                const float d = part[j] - mu;
                if (j < cluster) m2 += fmaf((float)slice_rows(p.pixels, j, cluster) * per * d, d, more[j]);
            }
            mean[g] = mu;
            rstd[g] = rstd_of(m2, m, p.eps);
            if (rank == 0 && p.mean) {
                p.mean[n * p.groups + c0 / per + g] = mu;
                p.rstd[n * p.groups + c0 / per + g] = rstd[g];
            }
        }
        __syncthreads();
        each<V, 2>(w, rows,
                   [&](int c) {
                       k.params(p, c0 + c);
                       k.stats(mean, rstd, per, c, 0);
                   },
                   [&](int c, int r) { return Two{*reinterpret_cast<const Pack*>(xs + r * w + c), gate_at(c, r)}; },
                   [&](int c, int r, const Two& q) {
                       float2 v[P];
                       unpack<V>(q.a, v);
                       forward<T, V>(p, k, v, gated, q.b, static_cast<T*>(p.y) + at + (int64_t)r * p.channels + c);
                   },
                   [&](int, int, int, int, int) {});
        if (cluster > 1) cluster_sync();  // nobody leaves while its sums may still be read
    } else {
        for (int g = threadIdx.x; g < groups; g += kThreads) {
            mean[g] = p.mean[n * p.groups + c0 / per + g];
            rstd[g] = p.rstd[n * p.groups + c0 / per + g];
        }
        __syncthreads();
        float2 sb[P], sw[P];
        auto before = [&](int c) {
            k.params(p, c0 + c);
            k.stats(mean, rstd, per, c, 0);
        };
        each<V, 1>(w, rows,
                   [&](int c) {
                       before(c);
#pragma unroll
                       for (int i = 0; i < P; ++i) sb[i] = sw[i] = splat2(0.f);
                   },
                   three,
                   [&](int c, int r, const Three& q) {
                       float2 v[P], d[P];
                       unpack<V>(q.a, v);
                       unpack<V>(q.b, d);
                       backward<T, V>(p, k, v, d, gated, q.c, static_cast<T*>(nullptr));
#pragma unroll
                       for (int i = 0; i < P; ++i) {
                           sb[i] = fadd2(sb[i], d[i]);
                           sw[i] = ffma2(d[i], v[i], sw[i]);
                       }
                   },
                   [&](int q0, int qn, int phases, int qi, int ph) { add_phases<V>(sb, sw, q0, qn, phases, qi, ph, red, ca, cb); });
        if (cluster > 1) cluster_sync();
        // all slices' sums a channel (into the scratch, as others still read ca and cb), then a group's
        float *ta = red, *tb = red + w;
        const bool fits = 2 * w <= kThreads * V;
        for (int c = threadIdx.x; c < w; c += kThreads) {
            float fb[kMaxCluster], fw[kMaxCluster], b = 0.f, s = 0.f;
#pragma unroll
            for (int j = 0; j < kMaxCluster; ++j) {
                fb[j] = j < cluster ? (cluster > 1 ? ld_cluster(ca + c, j) : ca[c]) : 0.f;
                fw[j] = j < cluster ? (cluster > 1 ? ld_cluster(cb + c, j) : cb[c]) : 0.f;
            }
#pragma unroll
            for (int j = 0; j < kMaxCluster; ++j) {
                b += fb[j];
                s += fw[j];
            }
            if (rank == 0) {
                p.part[n * 2 * p.channels + c0 + c] = b;
                p.part[(n * 2 + 1) * p.channels + c0 + c] = s;
            }
            const float g = p.weight ? p.weight[c0 + c] : 1.f;
            if (fits) {
                ta[c] = g * b;
                tb[c] = g * s;
            } else {  // one CTA a slab: nobody else reads them
                ca[c] = g * b;
                cb[c] = g * s;
            }
        }
        __syncthreads();
        add_groups(fits ? ta : ca, w, per, ga);
        add_groups(fits ? tb : cb, w, per, gb);
        const float m = (float)p.pixels * per;
        for (int g = threadIdx.x; g < groups; g += kThreads) {
            ga[g] = ga[g] / m * rstd[g];
            gb[g] = gb[g] / m * rstd[g];
        }
        __syncthreads();
        float2 ra[P], rb[P];
        each<V, 1>(w, rows,
                   [&](int c) {
                       before(c);
                       with_groups<V>(c, per, [&](int i, int g) {
                           set_pair<V>(ra, i, ga[g]);
                           set_pair<V>(rb, i, gb[g]);
                       });
                   },
                   three,
                   [&](int c, int r, const Three& q) {
                       float2 v[P], d[P];
                       unpack<V>(q.a, v);
                       unpack<V>(q.b, d);
                       const int64_t to = at + (int64_t)r * p.channels + c;
                       backward<T, V>(p, k, v, d, gated, q.c, p.dgate ? static_cast<T*>(p.dgate) + to : nullptr);
                       input_gradient<V>(k, v, d, ra, rb);
                       put<V>(static_cast<T*>(p.dx) + to, d);
                   },
                   [&](int, int, int, int, int) {});
        if (cluster > 1) cluster_sync();
    }
}

// ---- split --------------------------------------------------------------------------------------
// Forward: mean and sum of squares around it, a slice and channel; backward: sums of dn and dn x^.
template <typename T, int V, bool BACK>
__global__ void __launch_bounds__(kThreads) part_kernel(Norm p, int splits, int width) {
    extern __shared__ __align__(16) float head[];
    float *red = head, *ca = red + kThreads * V, *cb = ca + width;
    const int split = blockIdx.x, c0 = blockIdx.y * width, w = min(width, p.channels - c0);
    const int rows = slice_rows(p.pixels, split, splits);
    const int64_t s0 = (int64_t)split * slice_len(p.pixels, splits);
    for (int64_t n = blockIdx.z; n < p.samples; n += gridDim.z) {
        const T* x = static_cast<const T*>(p.x) + n * p.xs + s0 * p.xp + c0;
        const int64_t at = (n * p.pixels + s0) * p.channels + c0;
        const T* gate = p.gate ? static_cast<const T*>(p.gate) + n * p.gs + s0 * p.gp + c0 : nullptr;
        constexpr int P = kP<V>;
        using Pack = ssm::Pack<T, V>;
        struct Raw {
            Pack x, d, z;
        };
        float2 sa[P], sq[P], first[P];
        Channel<V> k;
        each<V, BACK ? 2 : 4>(
            w, rows,
            [&](int c) {
#pragma unroll
                for (int i = 0; i < P; ++i) sa[i] = sq[i] = first[i] = splat2(0.f);
                if constexpr (BACK) {
                    const int g0 = (c0 + c) / p.per;
                    k.params(p, c0 + c);
                    k.stats(p.mean + n * p.groups + g0, p.rstd + n * p.groups + g0, p.per, c0 + c, g0 * p.per);
                } else if (rows > 0) {
                    get<V>(x + c, first);
                }
            },
            [&](int c, int r) {
                Raw q = {};
                q.x = *reinterpret_cast<const Pack*>(x + r * p.xp + c);
                if constexpr (BACK) {
                    q.d = *reinterpret_cast<const Pack*>(static_cast<const T*>(p.dy) + at + (int64_t)r * p.channels + c);
                    if (gate) q.z = *reinterpret_cast<const Pack*>(gate + r * p.gp + c);
                }
                return q;
            },
            [&](int, int, const Raw& q) {
                float2 v[P];
                unpack<V>(q.x, v);
                if constexpr (BACK) {
                    float2 d[P];
                    unpack<V>(q.d, d);
                    backward<T, V>(p, k, v, d, gate != nullptr, q.z, static_cast<T*>(nullptr));
#pragma unroll
                    for (int i = 0; i < P; ++i) {
                        sa[i] = fadd2(sa[i], d[i]);
                        sq[i] = ffma2(d[i], v[i], sq[i]);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < P; ++i) {
                        v[i] = fsub2(v[i], first[i]);
                        sa[i] = fadd2(sa[i], v[i]);
                        sq[i] = ffma2(v[i], v[i], sq[i]);
                    }
                }
            },
            [&](int q0, int qn, int phases, int qi, int ph) { add_phases<V>(sa, sq, q0, qn, phases, qi, ph, red, ca, cb); });
        if (!BACK) center(ca, cb, w, rows, [&](int c) { return to_f(x[c]); });
        float* out = p.part + ((n * splits + split) * 2) * p.channels + c0;
        for (int c = threadIdx.x; c < w; c += kThreads) {
            out[c] = ca[c];
            out[p.channels + c] = cb[c];
        }
        __syncthreads();
    }
}

// Joins the slices' means and squares of a group: a block per sample and group.
__global__ void __launch_bounds__(kJoinThreads) join_kernel(Norm p, int splits) {
    __shared__ float red[kJoinThreads / 32];
    const int g = blockIdx.x;
    const int64_t n = blockIdx.y + (int64_t)blockIdx.z * gridDim.y;
    if (n >= p.samples) return;
    const float* part = p.part + n * splits * 2 * p.channels + g * p.per;
    const int total = splits * p.per;
    auto block_sum = [&](float v) {
        v = warp_sum(v);
        __syncthreads();
        if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
        __syncthreads();
        v = 0.f;
        for (int i = 0; i < kJoinThreads / 32; ++i) v += red[i];
        return v;
    };
    const float m = (float)p.pixels * p.per;
    const int len = slice_len(p.pixels, splits);
    auto rows = [&](int s) { return (float)max((int64_t)0, min((int64_t)len, p.pixels - (int64_t)s * len)); };
    float mu = 0.f;
    for (int i = threadIdx.x; i < total; i += kJoinThreads) {
        const int s = i / p.per;
        mu = fmaf(rows(s) / m, part[(int64_t)s * 2 * p.channels + i % p.per], mu);
    }
    mu = block_sum(mu);
    float m2 = 0.f;
    for (int i = threadIdx.x; i < total; i += kJoinThreads) {
        const int s = i / p.per;
        const float* at = part + (int64_t)s * 2 * p.channels + i % p.per;
        const float d = at[0] - mu;
        m2 += fmaf(rows(s) * d, d, at[p.channels]);
    }
    m2 = block_sum(m2);
    if (threadIdx.x == 0) {
        p.mean[n * p.groups + g] = mu;
        p.rstd[n * p.groups + g] = rstd_of(m2, m, p.eps);
    }
}

// Sums the slices of a sample, in order: [samples][splits][2 channels] -> [samples][2 channels].
__global__ void __launch_bounds__(kJoinThreads) fold_kernel(const float* __restrict__ part, int splits, int64_t samples, int n, float* out) {
    const int64_t i = (int64_t)blockIdx.x * kJoinThreads + threadIdx.x;
    if (i >= samples * n) return;
    const float* at = part + i / n * splits * n + i % n;
    float s = 0.f;
#pragma unroll 8
    for (int k = 0; k < splits; ++k) s += at[(int64_t)k * n];
    out[i] = s;
}

template <typename T, int V, bool BACK>
__global__ void __launch_bounds__(kThreads) apply_kernel(Norm p, int splits, int width, const float* sums) {
    extern __shared__ __align__(16) float head[];
    const int split = blockIdx.x, c0 = blockIdx.y * width, w = min(width, p.channels - c0);
    const int rows = slice_rows(p.pixels, split, splits);
    const int64_t s0 = (int64_t)split * slice_len(p.pixels, splits);
    const float m = (float)p.pixels * p.per;
    for (int64_t n = blockIdx.z; n < p.samples; n += gridDim.z) {
        const T* x = static_cast<const T*>(p.x) + n * p.xs + s0 * p.xp + c0;
        const int64_t at = (n * p.pixels + s0) * p.channels + c0;
        const T* gate = p.gate ? static_cast<const T*>(p.gate) + n * p.gs + s0 * p.gp + c0 : nullptr;
        // sums over the groups that this block's channels touch
        const int g0 = c0 / p.per, g1 = (c0 + w - 1) / p.per + 1;
        float *ga = head, *gb = head + (width / p.per + 2);
        if constexpr (BACK) {
            const float* sb = sums + n * 2 * p.channels;
            const int lane = threadIdx.x & 31;
            __syncthreads();
            for (int g = g0 + (threadIdx.x >> 5); g < g1; g += kThreads / 32) {
                float a = 0.f, b = 0.f;
                for (int c = g * p.per + lane; c < (g + 1) * p.per; c += 32) {
                    const float wt = p.weight ? p.weight[c] : 1.f;
                    a = fmaf(wt, sb[c], a);
                    b = fmaf(wt, sb[p.channels + c], b);
                }
                a = warp_sum(a);
                b = warp_sum(b);
                if (lane == 0) {
                    const float rstd = p.rstd[n * p.groups + g] / m;
                    ga[g - g0] = a * rstd;
                    gb[g - g0] = b * rstd;
                }
            }
            __syncthreads();
        }
        constexpr int P = kP<V>;
        using Pack = ssm::Pack<T, V>;
        struct Raw {
            Pack x, d, z;
        };
        Channel<V> k;
        float2 ra[P], rb[P];
        each<V, BACK ? 2 : 4>(
            w, rows,
            [&](int c) {
                const int gc = (c0 + c) / p.per;
                k.params(p, c0 + c);
                k.stats(p.mean + n * p.groups + gc, p.rstd + n * p.groups + gc, p.per, c0 + c, gc * p.per);
                if constexpr (BACK) {
                    with_groups<V>(c0 + c, p.per, [&](int i, int g) {
                        set_pair<V>(ra, i, ga[g - g0]);
                        set_pair<V>(rb, i, gb[g - g0]);
                    });
                }
            },
            [&](int c, int r) {
                Raw q = {};
                q.x = *reinterpret_cast<const Pack*>(x + r * p.xp + c);
                if (gate) q.z = *reinterpret_cast<const Pack*>(gate + r * p.gp + c);
                if constexpr (BACK) q.d = *reinterpret_cast<const Pack*>(static_cast<const T*>(p.dy) + at + (int64_t)r * p.channels + c);
                return q;
            },
            [&](int c, int r, const Raw& q) {
                float2 v[P];
                unpack<V>(q.x, v);
                const int64_t to = at + (int64_t)r * p.channels + c;
                if constexpr (BACK) {
                    float2 d[P];
                    unpack<V>(q.d, d);
                    backward<T, V>(p, k, v, d, gate != nullptr, q.z, p.dgate ? static_cast<T*>(p.dgate) + to : nullptr);
                    input_gradient<V>(k, v, d, ra, rb);
                    put<V>(static_cast<T*>(p.dx) + to, d);
                } else {
                    forward<T, V>(p, k, v, gate != nullptr, q.z, static_cast<T*>(p.y) + to);
                }
            },
            [&](int, int, int, int, int) {});
    }
}

// ---- host ---------------------------------------------------------------------------------------
enum class Form { kRows, kResident, kSplit };

struct Plan {
    Form form;
    int v;                       // values an access
    int sw, nv, gb, blocks;      // rows
    int width, slabs, cluster;   // resident: channels a slab; split: channels a block
    int splits;
    size_t smem;
};

int vec_of(const vh_group_norm_args* a, const void* const* more, int count) {
    const int es = (int)dtype_size(a->dtype), v = 16 / es;
    bool ok = a->channels % v == 0 && aligned(a->x, 16) && a->x_sample_stride % v == 0 && a->x_pixel_stride % v == 0;
    if (a->gate) ok = ok && aligned(a->gate, 16) && a->gate_sample_stride % v == 0 && a->gate_pixel_stride % v == 0;
    if (a->y) ok = ok && aligned(a->y, 16);
    for (int i = 0; i < count; ++i) ok = ok && (!more[i] || aligned(more[i], 16));
    return ok ? v : 1;
}

// Which form, and its sizes.  Depends on sizes, type and the access width alone.
Plan plan_of(const vh_group_norm_args* a, int v, bool back) {
    Plan q{};
    const int per = a->channels / a->groups, es = (int)dtype_size(a->dtype);
    q.v = per % v == 0 ? v : 1;
    if (a->pixels == 1 && per <= (q.v > 1 ? 1024 : 256)) {
        q.form = Form::kRows;
        const int vectors = per / q.v;
        q.sw = q.v == 1 || vectors > 16 ? 32 : vectors > 8 ? 16 : vectors > 4 ? 8 : 4;
        q.nv = vectors <= q.sw ? 1 : vectors <= 2 * q.sw && q.v > 1 ? 2 : q.v > 1 ? 32 / q.v : 8;
        q.gb = std::min(a->groups, kThreads / q.sw);
        if (back) q.gb = std::max(1, std::min(q.gb, 6144 / per));  // 48 KB of sums
        const int phases = kThreads / (q.gb * q.sw), columns = (a->groups + q.gb - 1) / q.gb;
        // the rows' blocks fill the card: eight blocks an SM (backward: four, each leaves partial sums)
        const int64_t most = std::max<int64_t>(1, (int64_t)(back ? 4 : 8) * sm_count() / columns);
        q.blocks = (int)std::min<int64_t>((a->samples + phases - 1) / phases, most);
        q.smem = back ? (size_t)2 * q.gb * per * sizeof(float) : 0;
        return q;
    }
    q.v = v;
    // slabs of whole groups, at least 64 bytes wide where there are as many
    int gs = 1;
    while (gs < a->groups && (gs * per % v != 0 || gs * per * es < 64)) ++gs;
    auto slabs = [&](int s) { return (a->groups + s - 1) / s; };
    // small ones are joined while the card stays full
    while (2 * gs <= a->groups && 2 * gs * per % v == 0 && a->pixels * gs * per * es < 16384 &&
           a->samples * slabs(2 * gs) >= 4 * (int64_t)sm_count())
        gs *= 2;
    const int tensors = back ? 2 : 1;
    const int64_t bytes = a->pixels * gs * per * es * tensors;
    int k = 1;
    while (k < kMaxCluster && bytes > (int64_t)k * 64 * 1024) k *= 2;
    while (k < kMaxCluster && a->samples * slabs(gs) * k < sm_count() && bytes / k > 8192 && 2 * k <= a->pixels) k *= 2;
    const size_t head = head_floats(gs * per, per, v) * sizeof(float);
    const int64_t slice = (a->pixels + k - 1) / k * gs * per * es * tensors;
    if (slice + (int64_t)head <= 100 * 1024 && a->samples * slabs(gs) * k <= 0x7fffffff && (k == 1 || 2 * gs * per <= kThreads * v) && k <= a->pixels) {
        q.form = Form::kResident;
        q.width = gs * per;
        q.slabs = slabs(gs);
        q.cluster = k;
        q.smem = head + (size_t)slice;
        return q;
    }
    q.form = Form::kSplit;
    q.width = std::min(a->channels, kThreads * v);
    const int columns = (a->channels + q.width - 1) / q.width;
    const int64_t want = std::max<int64_t>(1, 4 * (int64_t)sm_count() / std::max<int64_t>(1, a->samples * columns));
    q.splits = (int)std::max<int64_t>(1, std::min<int64_t>({want, std::max<int64_t>(1, a->pixels / 8), 1024}));
    while (a->pixels / q.splits > (1 << 24)) q.splits *= 2;
    return q;
}

int64_t bytes_of(const vh_group_norm_args* a, const Plan& q, bool back) {
    const int64_t row = 2 * (int64_t)a->channels * sizeof(float);
    switch (q.form) {
        case Form::kRows: return back ? q.blocks * row : 0;
        case Form::kResident: return back ? a->samples * row : 0;
        default: return a->samples * q.splits * row + (back ? a->samples * row : 2 * a->samples * a->groups * (int64_t)sizeof(float));
    }
}
// The workspace is asked for before the pointers are known: whatever the access width turns out to be.
int64_t most_bytes(const vh_group_norm_args* a, bool back) {
    return std::max(bytes_of(a, plan_of(a, 1, back), back), bytes_of(a, plan_of(a, 16 / (int)dtype_size(a->dtype), back), back));
}

int check_sizes(const char* what, const vh_group_norm_args* a) {
    if (!a) return fail(VH_E_ARG, "%s: null argument struct", what);
    if (!dtype_ok(a->dtype)) return fail(VH_E_DTYPE, "%s: dtype must be VH_F32, VH_BF16 or VH_F16", what);
    if (a->samples <= 0 || a->pixels <= 0 || a->channels <= 0 || a->groups <= 0)
        return fail(VH_E_SHAPE, "%s: samples, pixels, channels and groups must be positive", what);
    if (a->channels % a->groups)
        return fail(VH_E_SHAPE, "%s: channels (%d) must be a multiple of groups (%d)", what, a->channels, a->groups);
    if (a->activation < 0 || a->activation > 2) return fail(VH_E_ARG, "%s: activation must be 0, 1 or 2", what);
    if (a->channels > (1 << 20)) return fail(VH_E_RANGE, "%s: at most 2^20 channels", what);
    if (a->pixels > 0x7fffffff || a->samples > 0x7fffffff) return fail(VH_E_RANGE, "%s: at most 2^31 - 1 samples and pixels", what);
    return 0;
}

int check_args(const char* what, const vh_group_norm_args* a) {
    if (!a) return fail(VH_E_ARG, "%s: null argument struct", what);
    if (!a->x) return fail(VH_E_ARG, "%s: null pointer argument", what);
    if (int rc = check_sizes(what, a)) return rc;
    const size_t es = dtype_size(a->dtype);
    for (const void* t : {a->x, a->gate, (const void*)a->y})
        if (t && !aligned(t, es)) return fail(VH_E_ALIGN, "%s: misaligned pointers", what);
    for (const void* t : {(const void*)a->weight, (const void*)a->bias, (const void*)a->mean, (const void*)a->rstd})
        if (t && !aligned(t, 4)) return fail(VH_E_ALIGN, "%s: misaligned pointers", what);
    if (!a->mean != !a->rstd) return fail(VH_E_ARG, "%s: mean and rstd come together", what);
    return 0;
}

Norm norm_of(const vh_group_norm_args* a) {
    Norm p{};
    p.x = a->x; p.gate = a->gate;
    p.xs = a->x_sample_stride; p.xp = a->x_pixel_stride;
    p.gs = a->gate_sample_stride; p.gp = a->gate_pixel_stride;
    p.weight = a->weight; p.bias = a->bias;
    p.y = a->y; p.mean = a->mean; p.rstd = a->rstd;
    p.samples = a->samples; p.pixels = a->pixels;
    p.eps = a->eps;
    p.channels = a->channels; p.groups = a->groups; p.per = a->channels / a->groups; p.act = a->activation;
    return p;
}

template <typename F>
int with_type(int dtype, int v, F&& f) {
    if (dtype == VH_F32) return v > 1 ? f(float{}, std::integral_constant<int, 4>{}) : f(float{}, std::integral_constant<int, 1>{});
    if (dtype == VH_BF16)
        return v > 1 ? f(__nv_bfloat16{}, std::integral_constant<int, 8>{}) : f(__nv_bfloat16{}, std::integral_constant<int, 1>{});
    return v > 1 ? f(__half{}, std::integral_constant<int, 8>{}) : f(__half{}, std::integral_constant<int, 1>{});
}

template <typename T, int V, int SW, int NV, bool BACK>
int launch_rows(const Norm& p, const Plan& q, cudaStream_t st) {
    const dim3 grid(q.blocks, (p.groups + q.gb - 1) / q.gb);
    rows_kernel<T, V, SW, NV, BACK><<<grid, kThreads, q.smem, st>>>(p, q.gb);
    return launch_status("group norm (rows)");
}

template <typename T, int V, bool BACK>
int run_rows(const Norm& p, const Plan& q, cudaStream_t st) {
    if constexpr (V == 1) {
        return q.nv == 1 ? launch_rows<T, V, 32, 1, BACK>(p, q, st) : launch_rows<T, V, 32, 8, BACK>(p, q, st);
    } else {
        if (q.sw == 4) return launch_rows<T, V, 4, 1, BACK>(p, q, st);
        if (q.sw == 8) return launch_rows<T, V, 8, 1, BACK>(p, q, st);
        if (q.sw == 16) return launch_rows<T, V, 16, 1, BACK>(p, q, st);
        if (q.nv == 1) return launch_rows<T, V, 32, 1, BACK>(p, q, st);
        if (q.nv == 2) return launch_rows<T, V, 32, 2, BACK>(p, q, st);
        return launch_rows<T, V, 32, 32 / V, BACK>(p, q, st);
    }
}

template <typename T, int V, bool BACK>
int run_resident(const Norm& p, const Plan& q, cudaStream_t st) {
    const void* fn = reinterpret_cast<const void*>(&resident_kernel<T, V, BACK>);
    if (!ensure_smem_attr(fn, q.smem)) return fail(VH_E_DEVICE, "group norm: shared memory");
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(p.samples * q.slabs * q.cluster));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = q.smem;
    cfg.stream = st;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = q.cluster;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = q.cluster > 1 ? 1 : 0;
    cudaLaunchKernelEx(&cfg, resident_kernel<T, V, BACK>, p, q.width, q.slabs, q.cluster);
    return launch_status("group norm (resident)");
}

template <typename T, int V, bool BACK>
int run_split(Norm p, const Plan& q, float* ws, cudaStream_t st) {
    const int columns = (p.channels + q.width - 1) / q.width, nz = (int)std::min<int64_t>(p.samples, 65535);
    const dim3 grid(q.splits, columns, nz);
    p.part = ws;
    const int64_t row = 2 * (int64_t)p.channels;
    float* after = ws + p.samples * q.splits * row;
    if (!BACK && !p.mean) {
        p.mean = after;
        p.rstd = after + p.samples * p.groups;
    }
    const size_t smem = (size_t)(kThreads * V + 2 * q.width) * sizeof(float);
    const void* fn = reinterpret_cast<const void*>(&part_kernel<T, V, BACK>);
    if (!ensure_smem_attr(fn, smem)) return fail(VH_E_DEVICE, "group norm: shared memory");
    part_kernel<T, V, BACK><<<grid, kThreads, smem, st>>>(p, q.splits, q.width);
    if (int rc = launch_status("group norm: slices")) return rc;
    if (!BACK) {
        join_kernel<<<dim3(p.groups, nz, (unsigned)((p.samples + nz - 1) / nz)), kJoinThreads, 0, st>>>(p, q.splits);
        if (int rc = launch_status("group norm: statistics")) return rc;
    } else {
        fold_kernel<<<(unsigned)((p.samples * row + kJoinThreads - 1) / kJoinThreads), kJoinThreads, 0, st>>>(ws, q.splits, p.samples, (int)row, after);
        if (int rc = launch_status("group norm: sums")) return rc;
    }
    const size_t more = BACK ? (size_t)2 * (q.width / p.per + 2) * sizeof(float) : 0;
    apply_kernel<T, V, BACK><<<grid, kThreads, more, st>>>(p, q.splits, q.width, after);
    return launch_status("group norm");
}

template <bool BACK>
int run(const vh_group_norm_args* a, const Norm& p, const Plan& q, void* ws, cudaStream_t st) {
    return with_type(a->dtype, q.v, [&](auto t, auto v) {
        using T = decltype(t);
        constexpr int V = decltype(v)::value;
        if (q.form == Form::kRows) return run_rows<T, V, BACK>(p, q, st);
        if (q.form == Form::kResident) return run_resident<T, V, BACK>(p, q, st);
        return run_split<T, V, BACK>(p, q, static_cast<float*>(ws), st);
    });
}

int check_workspace(const char* what, const void* ws, int64_t have, int64_t need) {
    if (need == 0) return 0;
    if (!ws || have < need) return fail(VH_E_ARG, "%s: workspace too small (%lld < %lld bytes)", what, (long long)have, (long long)need);
    if (!aligned(ws, 4)) return fail(VH_E_ALIGN, "%s: misaligned workspace", what);
    return 0;
}

}  // namespace
}  // namespace gn
}  // namespace vh

using namespace vh;
using namespace vh::gn;

extern "C" int64_t vh_group_norm_fwd_workspace_bytes(const vh_group_norm_args* a) {
    clear_error();
    return check_sizes("vh_group_norm_fwd_workspace_bytes", a) ? 0 : most_bytes(a, false);
}

extern "C" int vh_group_norm_fwd(const vh_group_norm_args* a, void* workspace, int64_t workspace_bytes, vh_stream_t stream) {
    clear_error();
    const char* what = "vh_group_norm_fwd";
    if (int rc = check_args(what, a)) return rc;
    if (!a->y) return fail(VH_E_ARG, "%s: null pointer argument", what);
    const Plan q = plan_of(a, vec_of(a, nullptr, 0), false);
    if (int rc = check_workspace(what, workspace, workspace_bytes, bytes_of(a, q, false))) return rc;
    return run<false>(a, norm_of(a), q, workspace, static_cast<cudaStream_t>(stream));
}

extern "C" int64_t vh_group_norm_bwd_workspace_bytes(const vh_group_norm_args* a) {
    clear_error();
    return check_sizes("vh_group_norm_bwd_workspace_bytes", a) ? 0 : most_bytes(a, true);
}

extern "C" int vh_group_norm_bwd(const vh_group_norm_args* a, const void* grad_y, void* grad_x, void* grad_gate,
                                 float* grad_weight, float* grad_bias, void* workspace, int64_t workspace_bytes,
                                 vh_stream_t stream) {
    clear_error();
    const char* what = "vh_group_norm_bwd";
    if (int rc = check_args(what, a)) return rc;
    if (!grad_y || !grad_x || !a->mean || (grad_gate && !a->gate)) return fail(VH_E_ARG, "%s: null pointer argument", what);
    const size_t es = dtype_size(a->dtype);
    for (const void* t : {grad_y, (const void*)grad_x, (const void*)grad_gate})
        if (t && !aligned(t, es)) return fail(VH_E_ALIGN, "%s: misaligned pointers", what);
    for (const void* t : {(const void*)grad_weight, (const void*)grad_bias})
        if (t && !aligned(t, 4)) return fail(VH_E_ALIGN, "%s: misaligned pointers", what);
    const void* more[] = {grad_y, grad_x, grad_gate};
    const Plan q = plan_of(a, vec_of(a, more, 3), true);
    if (int rc = check_workspace(what, workspace, workspace_bytes, bytes_of(a, q, true))) return rc;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    Norm p = norm_of(a);
    p.dy = grad_y; p.dx = grad_x; p.dgate = grad_gate;
    p.part = static_cast<float*>(workspace);
    if (int rc = run<true>(a, p, q, workspace, st)) return rc;
    if (!grad_weight && !grad_bias) return 0;
    const int64_t row = 2 * (int64_t)a->channels;
    const float* part = static_cast<const float*>(workspace) + (q.form == Form::kSplit ? a->samples * q.splits * row : 0);
    params_kernel<<<(unsigned)((row + 31) / 32), dim3(32, 32), 0, st>>>(part, q.form == Form::kRows ? q.blocks : a->samples,
                                                                       a->channels, grad_weight, grad_bias);
    return launch_status("group norm: parameters");
}
