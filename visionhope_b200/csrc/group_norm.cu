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
// The variance comes from differences to a mean (registers, shared memory) or to the first value of
// each channel that a thread sees (split), joined by Chan's formula, so that a large mean costs nothing.
#include <algorithm>

#include "abi_util.h"
#include "activations.cuh"
#include "common.cuh"
#include "ssm_common.cuh"
#include "vhope.h"

namespace vh {
namespace gn {
namespace {

constexpr int kThreads = 256;
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

// ---- activations --------------------------------------------------------------------------------
// Phi(x) and its density.  16-bit outputs take the approximation of gelu2 (absolute error 7.5e-8).
template <typename T>
__device__ __forceinline__ void normal_cdf(float x, float* cdf, float* density) {
    constexpr float kDensity = 0.3989422804014327f;
    if constexpr (sizeof(T) == 4) {
        *cdf = 0.5f * erfcf(-0.70710678118654752f * x);
        *density = kDensity * expf(-0.5f * x * x);
    } else {
        const float ax = fabsf(x), t = rcp_approx(fmaf(ax, 0.3275911f * 0.70710678118654752f, 1.f));
        const float e = ex2_approx(x * x * (-0.5f * 1.4426950408889634f));
        float q = fmaf(t, 0.5f * 1.061405429f, 0.5f * -1.453152027f);
        q = fmaf(q, t, 0.5f * 1.421413741f);
        q = fmaf(q, t, 0.5f * -0.284496736f);
        q = fmaf(q, t, 0.5f * 0.254829592f) * t * e;
        *cdf = x >= 0.f ? 1.f - q : (x < 0.f ? q : x);
        *density = kDensity * e;
    }
}

// act(pre) in place of pre, and act'(pre) in `slope` if SLOPE.
template <typename T, bool SLOPE, int V>
__device__ __forceinline__ void activate(int act, float (&pre)[V], float (&slope)[V]) {
    if (act == 1) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float x = pre[i], s = ssm::sigmoid(x);
            pre[i] = x * s;
            if (SLOPE) slope[i] = s * fmaf(x, 1.f - s, 1.f);
        }
    } else if (act == 2) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float x = pre[i];
            float cdf, density;
            normal_cdf<T>(x, &cdf, &density);
            pre[i] = x * cdf;
            if (SLOPE) slope[i] = fmaf(x, density, cdf);
        }
    } else if (SLOPE) {
#pragma unroll
        for (int i = 0; i < V; ++i) slope[i] = 1.f;
    }
}

// ---- V consecutive values -----------------------------------------------------------------------
template <int V, typename T>
__device__ __forceinline__ void get(const T* p, float (&v)[V]) {
    if constexpr (V == 8) {
        load8(p, v);
    } else if constexpr (V == 4) {
        const float4 f = load4(p);
        v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = to_f(p[i]);
    }
}
template <int V, typename T>
__device__ __forceinline__ void put(T* p, const float (&v)[V]) {
    if constexpr (V == 8) {
        store8(p, v);
    } else if constexpr (V == 4) {
        store4(p, make_float4(v[0], v[1], v[2], v[3]));
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) p[i] = from_f<T>(v[i]);
    }
}

// Parameters and statistics of V channels from c on.
template <int V>
struct Channel {
    float w[V], b[V], mean[V], rstd[V];
    __device__ __forceinline__ void params(const Norm& p, int c) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            w[i] = p.weight ? p.weight[c + i] : 1.f;
            b[i] = p.bias ? p.bias[c + i] : 0.f;
        }
    }
    // `m`, `r`: of the groups from the one of channel c0 on
    __device__ __forceinline__ void stats(const float* m, const float* r, int per, int c, int c0) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int g = (c + i - c0) / per;
            mean[i] = m[g];
            rstd[i] = r[g];
        }
    }
};

// y of V values.
template <typename T, int V>
__device__ __forceinline__ void forward(const Norm& p, const Channel<V>& k, float (&x)[V], const T* gate, T* y) {
    float unused[V];
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = fmaf((x[i] - k.mean[i]) * k.rstd[i], k.w[i], k.b[i]);
    activate<T, false, V>(p.act, x, unused);
    if (gate) {
        float z[V];
        get<V>(gate, z);
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] *= z[i] * ssm::sigmoid(z[i]);
    }
    put<V>(y, x);
}

// x^ in place of x and dn in place of dy; the gate's gradient if `dgate`.
template <typename T, int V>
__device__ __forceinline__ void backward(const Norm& p, const Channel<V>& k, float (&x)[V], float (&dy)[V], const T* gate, T* dgate) {
    float pre[V], slope[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        x[i] = (x[i] - k.mean[i]) * k.rstd[i];
        pre[i] = fmaf(x[i], k.w[i], k.b[i]);
    }
    activate<T, true, V>(p.act, pre, slope);
    if (gate) {
        float z[V], dz[V];
        get<V>(gate, z);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float s = ssm::sigmoid(z[i]);
            dz[i] = dy[i] * pre[i] * (s * fmaf(z[i], 1.f - s, 1.f));
            dy[i] *= z[i] * s;
        }
        if (dgate) put<V>(dgate, dz);
    }
#pragma unroll
    for (int i = 0; i < V; ++i) dy[i] *= slope[i];
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
    const int lane = threadIdx.x % SW, unit = threadIdx.x / SW, phases = kThreads / (gb * SW);
    const int g = blockIdx.y * gb + unit % gb, phase = unit / gb;
    const bool live = phase < phases && g < p.groups;
    const int c0 = live ? g * p.per : 0;
    Channel<V> k[NV];
    bool has[NV];
    float aw[NV][V], ab[NV][V];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int c = (lane + j * SW) * V;
        has[j] = live && c < p.per;
        k[j].params(p, has[j] ? c0 + c : 0);
#pragma unroll
        for (int i = 0; i < V; ++i) aw[j][i] = ab[j][i] = 0.f;
    }
    const float count = (float)p.per;
    if (live) {
        for (int64_t r = (int64_t)blockIdx.x * phases + phase; r < p.samples; r += (int64_t)gridDim.x * phases) {
            const T* x = static_cast<const T*>(p.x) + r * p.xs + c0 + lane * V;
            const T* z = p.gate ? static_cast<const T*>(p.gate) + r * p.gs + c0 + lane * V : nullptr;
            const int64_t at = r * p.channels + c0 + lane * V;
            float v[NV][V];
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                if (has[j]) get<V>(x + j * SW * V, v[j]);
            }
            if constexpr (!BACK) {
                float s = 0.f;
#pragma unroll
                for (int j = 0; j < NV; ++j)
#pragma unroll
                    for (int i = 0; i < V; ++i) s += has[j] ? v[j][i] : 0.f;
                const float mean = lanes_sum<SW>(s) / count;
                s = 0.f;
#pragma unroll
                for (int j = 0; j < NV; ++j)
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        const float d = v[j][i] - mean;
                        s += has[j] ? d * d : 0.f;
                    }
                const float rstd = rstd_of(lanes_sum<SW>(s), count, p.eps);
                if (p.mean && lane == 0) {
                    p.mean[r * p.groups + g] = mean;
                    p.rstd[r * p.groups + g] = rstd;
                }
#pragma unroll
                for (int j = 0; j < NV; ++j)
                    if (has[j]) {
#pragma unroll
                        for (int i = 0; i < V; ++i) {
                            k[j].mean[i] = mean;
                            k[j].rstd[i] = rstd;
                        }
                        forward<T, V>(p, k[j], v[j], z ? z + j * SW * V : nullptr, static_cast<T*>(p.y) + at + j * SW * V);
                    }
            } else {
                const float mean = p.mean[r * p.groups + g], rstd = p.rstd[r * p.groups + g];
                float d[NV][V], s1 = 0.f, s2 = 0.f;
#pragma unroll
                for (int j = 0; j < NV; ++j)
                    if (has[j]) {
                        get<V>(static_cast<const T*>(p.dy) + at + j * SW * V, d[j]);
#pragma unroll
                        for (int i = 0; i < V; ++i) {
                            k[j].mean[i] = mean;
                            k[j].rstd[i] = rstd;
                        }
                        backward<T, V>(p, k[j], v[j], d[j], z ? z + j * SW * V : nullptr,
                                       p.dgate ? static_cast<T*>(p.dgate) + at + j * SW * V : nullptr);
#pragma unroll
                        for (int i = 0; i < V; ++i) {
                            ab[j][i] += d[j][i];
                            aw[j][i] = fmaf(d[j][i], v[j][i], aw[j][i]);
                            d[j][i] *= k[j].w[i];
                            s1 += d[j][i];
                            s2 = fmaf(d[j][i], v[j][i], s2);
                        }
                    }
                s1 = lanes_sum<SW>(s1) / count;
                s2 = lanes_sum<SW>(s2) / count;
#pragma unroll
                for (int j = 0; j < NV; ++j)
                    if (has[j]) {
#pragma unroll
                        for (int i = 0; i < V; ++i) d[j][i] = rstd * (d[j][i] - s1 - v[j][i] * s2);
                        put<V>(static_cast<T*>(p.dx) + at + j * SW * V, d[j]);
                    }
            }
        }
    }
    if constexpr (BACK) {
        if (!p.part) return;
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
#pragma unroll
                        for (int i = 0; i < V; ++i) {
                            const float b = (ph ? red[2 * (at + i)] : 0.f) + ab[j][i];
                            const float w = (ph ? red[2 * (at + i) + 1] : 0.f) + aw[j][i];
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
// f(c, r) is called for the first channel of a vector and every pixel of this thread's phase;
// before(c) and after() around the pixels of each vector.
template <int V, typename B, typename F, typename A>
__device__ __forceinline__ void each(int w, int rows, B&& before, F&& f, A&& after) {
    const int q = w / V;
    for (int q0 = 0; q0 < q; q0 += kThreads) {
        const int qn = min(q - q0, kThreads), phases = kThreads / qn;
        const int qi = threadIdx.x % qn, ph = threadIdx.x / qn;
        if (ph < phases) {
            const int c = (q0 + qi) * V;
            before(c);
            for (int r = ph; r < rows; r += phases) f(c, r);
        }
        after(q0, qn, phases, qi, ph);
    }
}

// Adds the V values of each thread over the pixel phases, into out[0..w), in a fixed order: first runs
// of phases side by side, then the runs.
template <int V>
__device__ __forceinline__ void add_phases(const float (&v)[V], int q0, int qn, int phases, int qi, int ph, float* red, float* out) {
    const int n = qn * V;
    __syncthreads();
    if (ph < phases) {
#pragma unroll
        for (int i = 0; i < V; ++i) red[ph * n + qi * V + i] = v[i];
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
    const int64_t s0 = p.pixels * rank / cluster;
    const int rows = (int)(p.pixels * (rank + 1) / cluster - s0);
    T* ds = xs + (int64_t)((p.pixels + cluster - 1) / cluster) * width;

    load_slab<T, V>(xs, static_cast<const T*>(p.x) + n * p.xs + s0 * p.xp + c0, p.xp, rows, w);
    const int64_t at = (n * p.pixels + s0) * p.channels + c0;  // in contiguous tensors
    const T* gate = p.gate ? static_cast<const T*>(p.gate) + n * p.gs + s0 * p.gp + c0 : nullptr;
    if constexpr (BACK) load_slab<T, V>(ds, static_cast<const T*>(p.dy) + at, p.channels, rows, w);
    cp_async_commit();
    cp_async_wait<0>();
    __syncthreads();

    Channel<V> k;
    if constexpr (!BACK) {
        // the slice's mean, then its squares around it
        float acc[V];
        auto zero = [&] {
#pragma unroll
            for (int i = 0; i < V; ++i) acc[i] = 0.f;
        };
        zero();
        each<V>(w, rows, [&](int) {},
                [&](int c, int r) {
                    float v[V];
                    get<V>(xs + (int64_t)r * w + c, v);
#pragma unroll
                    for (int i = 0; i < V; ++i) acc[i] += v[i];
                },
                [&](int q0, int qn, int phases, int qi, int ph) { add_phases<V>(acc, q0, qn, phases, qi, ph, red, ca); zero(); });
        add_groups(ca, w, per, ga);
        const float count = (float)rows * per;
        for (int g = threadIdx.x; g < groups; g += kThreads) ga[g] = rows ? ga[g] / count : 0.f;
        __syncthreads();
        each<V>(w, rows,
                [&](int c) {
#pragma unroll
                    for (int i = 0; i < V; ++i) k.mean[i] = ga[(c + i) / per];
                },
                [&](int c, int r) {
                    float v[V];
                    get<V>(xs + (int64_t)r * w + c, v);
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        const float d = v[i] - k.mean[i];
                        acc[i] = fmaf(d, d, acc[i]);
                    }
                },
                [&](int q0, int qn, int phases, int qi, int ph) { add_phases<V>(acc, q0, qn, phases, qi, ph, red, cb); zero(); });
        add_groups(cb, w, per, gb);
        if (cluster > 1) cluster_sync();
        const float m = (float)p.pixels * per;
        for (int g = threadIdx.x; g < groups; g += kThreads) {
            float mu = 0.f, m2 = 0.f;
            for (int j = 0; j < cluster; ++j) {
                const float nk = (float)(p.pixels * (j + 1) / cluster - p.pixels * j / cluster) * per;
                mu = fmaf(nk / m, cluster > 1 ? ld_cluster(ga + g, j) : ga[g], mu);
            }
            for (int j = 0; j < cluster; ++j) {
                const float nk = (float)(p.pixels * (j + 1) / cluster - p.pixels * j / cluster) * per;
                const float d = (cluster > 1 ? ld_cluster(ga + g, j) : ga[g]) - mu;
                m2 += fmaf(nk * d, d, cluster > 1 ? ld_cluster(gb + g, j) : gb[g]);
            }
            mean[g] = mu;
            rstd[g] = rstd_of(m2, m, p.eps);
            if (rank == 0 && p.mean) {
                p.mean[n * p.groups + c0 / per + g] = mu;
                p.rstd[n * p.groups + c0 / per + g] = rstd[g];
            }
        }
        __syncthreads();
        each<V>(w, rows,
                [&](int c) {
                    k.params(p, c0 + c);
                    k.stats(mean, rstd, per, c, 0);
                },
                [&](int c, int r) {
                    float v[V];
                    get<V>(xs + (int64_t)r * w + c, v);
                    forward<T, V>(p, k, v, gate ? gate + r * p.gp + c : nullptr, static_cast<T*>(p.y) + at + (int64_t)r * p.channels + c);
                },
                [&](int, int, int, int, int) {});
        if (cluster > 1) cluster_sync();  // nobody leaves while its sums may still be read
    } else {
        for (int g = threadIdx.x; g < groups; g += kThreads) {
            mean[g] = p.mean[n * p.groups + c0 / per + g];
            rstd[g] = p.rstd[n * p.groups + c0 / per + g];
        }
        __syncthreads();
        float sb[V], sw[V];
        auto zero = [&] {
#pragma unroll
            for (int i = 0; i < V; ++i) sb[i] = sw[i] = 0.f;
        };
        auto before = [&](int c) {
            k.params(p, c0 + c);
            k.stats(mean, rstd, per, c, 0);
        };
        zero();
        each<V>(w, rows, before,
                [&](int c, int r) {
                    float v[V], d[V];
                    get<V>(xs + (int64_t)r * w + c, v);
                    get<V>(ds + (int64_t)r * w + c, d);
                    backward<T, V>(p, k, v, d, gate ? gate + r * p.gp + c : nullptr, nullptr);
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        sb[i] += d[i];
                        sw[i] = fmaf(d[i], v[i], sw[i]);
                    }
                },
                [&](int q0, int qn, int phases, int qi, int ph) {
                    add_phases<V>(sb, q0, qn, phases, qi, ph, red, ca);
                    add_phases<V>(sw, q0, qn, phases, qi, ph, red, cb);
                    zero();
                });
        if (cluster > 1) cluster_sync();
        // all slices' sums a channel (into the scratch, as others still read ca and cb), then a group's
        float *ta = red, *tb = red + w;
        const bool fits = 2 * w <= kThreads * V;
        for (int c = threadIdx.x; c < w; c += kThreads) {
            float b = 0.f, s = 0.f;
            for (int j = 0; j < cluster; ++j) {
                b += cluster > 1 ? ld_cluster(ca + c, j) : ca[c];
                s += cluster > 1 ? ld_cluster(cb + c, j) : cb[c];
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
        each<V>(w, rows, before,
                [&](int c, int r) {
                    float v[V], d[V];
                    get<V>(xs + (int64_t)r * w + c, v);
                    get<V>(ds + (int64_t)r * w + c, d);
                    const int64_t to = at + (int64_t)r * p.channels + c;
                    backward<T, V>(p, k, v, d, gate ? gate + r * p.gp + c : nullptr, p.dgate ? static_cast<T*>(p.dgate) + to : nullptr);
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        const int g = (c + i) / per;
                        d[i] = k.rstd[i] * (k.w[i] * d[i] - ga[g] / m - v[i] * (gb[g] / m));
                    }
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
    const int64_t s0 = p.pixels * split / splits;
    const int rows = (int)(p.pixels * (split + 1) / splits - s0);
    for (int64_t n = blockIdx.z; n < p.samples; n += gridDim.z) {
        const T* x = static_cast<const T*>(p.x) + n * p.xs + s0 * p.xp + c0;
        const int64_t at = (n * p.pixels + s0) * p.channels + c0;
        const T* gate = p.gate ? static_cast<const T*>(p.gate) + n * p.gs + s0 * p.gp + c0 : nullptr;
        float sa[V], sq[V], first[V];
        Channel<V> k;
        int mine = 0;
        auto zero = [&] {
#pragma unroll
            for (int i = 0; i < V; ++i) sa[i] = sq[i] = first[i] = 0.f;
            mine = 0;
        };
        zero();
        each<V>(w, rows,
                [&](int c) {
                    if constexpr (BACK) {
                        const int g0 = (c0 + c) / p.per;
                        k.params(p, c0 + c);
                        k.stats(p.mean + n * p.groups + g0, p.rstd + n * p.groups + g0, p.per, c0 + c, g0 * p.per);
                    }
                },
                [&](int c, int r) {
                    float v[V];
                    get<V>(x + r * p.xp + c, v);
                    if constexpr (BACK) {
                        float d[V];
                        get<V>(static_cast<const T*>(p.dy) + at + (int64_t)r * p.channels + c, d);
                        backward<T, V>(p, k, v, d, gate ? gate + r * p.gp + c : nullptr, nullptr);
#pragma unroll
                        for (int i = 0; i < V; ++i) {
                            sa[i] += d[i];
                            sq[i] = fmaf(d[i], v[i], sq[i]);
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < V; ++i) {
                            if (mine == 0) first[i] = v[i];
                            const float d = v[i] - first[i];
                            sa[i] += d;
                            sq[i] = fmaf(d, d, sq[i]);
                        }
                        ++mine;
                    }
                },
                [&](int q0, int qn, int phases, int qi, int ph) {
                    if constexpr (!BACK) {
                        // the slice's mean a channel, then this thread's squares around it
                        float sum[V];
#pragma unroll
                        for (int i = 0; i < V; ++i) sum[i] = fmaf((float)mine, first[i], sa[i]);
                        add_phases<V>(sum, q0, qn, phases, qi, ph, red, ca);
#pragma unroll
                        for (int i = 0; i < V; ++i) {
                            const float mu = rows && ph < phases ? ca[(q0 + qi) * V + i] / (float)rows : 0.f;
                            const float own = mine ? sa[i] / (float)mine : 0.f, d = first[i] + own - mu;
                            sq[i] = mine ? fmaf((float)mine * d, d, fmaxf(sq[i] - sa[i] * own, 0.f)) : 0.f;
                        }
                        add_phases<V>(sq, q0, qn, phases, qi, ph, red, cb);
                    } else {
                        add_phases<V>(sa, q0, qn, phases, qi, ph, red, ca);
                        add_phases<V>(sq, q0, qn, phases, qi, ph, red, cb);
                    }
                    zero();
                });
        float* out = p.part + ((n * splits + split) * 2) * p.channels + c0;
        for (int c = threadIdx.x; c < w; c += kThreads) {
            out[c] = BACK || rows == 0 ? ca[c] : ca[c] / (float)rows;
            out[p.channels + c] = cb[c];
        }
        __syncthreads();
    }
}

// Joins the slices' means and squares of a group: a block per sample and group.
__global__ void __launch_bounds__(kThreads) join_kernel(Norm p, int splits) {
    __shared__ float red[kThreads / 32];
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
        for (int i = 0; i < kThreads / 32; ++i) v += red[i];
        return v;
    };
    const float m = (float)p.pixels * p.per;
    auto rows = [&](int s) { return (float)(p.pixels * (s + 1) / splits - p.pixels * s / splits); };
    float mu = 0.f;
    for (int i = threadIdx.x; i < total; i += kThreads) {
        const int s = i / p.per;
        mu = fmaf(rows(s) / m, part[(int64_t)s * 2 * p.channels + i % p.per], mu);
    }
    mu = block_sum(mu);
    float m2 = 0.f;
    for (int i = threadIdx.x; i < total; i += kThreads) {
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
__global__ void __launch_bounds__(kThreads) fold_kernel(const float* __restrict__ part, int splits, int64_t samples, int n, float* out) {
    const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
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
    const int64_t s0 = p.pixels * split / splits;
    const int rows = (int)(p.pixels * (split + 1) / splits - s0);
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
                    ga[g - g0] = a / m;
                    gb[g - g0] = b / m;
                }
            }
            __syncthreads();
        }
        Channel<V> k;
        float ma[V], mb[V];
        each<V>(w, rows,
                [&](int c) {
                    const int gc = (c0 + c) / p.per;
                    k.params(p, c0 + c);
                    k.stats(p.mean + n * p.groups + gc, p.rstd + n * p.groups + gc, p.per, c0 + c, gc * p.per);
                    if constexpr (BACK) {
#pragma unroll
                        for (int i = 0; i < V; ++i) {
                            ma[i] = ga[(c0 + c + i) / p.per - g0];
                            mb[i] = gb[(c0 + c + i) / p.per - g0];
                        }
                    }
                },
                [&](int c, int r) {
                    float v[V];
                    get<V>(x + r * p.xp + c, v);
                    const T* z = gate ? gate + r * p.gp + c : nullptr;
                    const int64_t to = at + (int64_t)r * p.channels + c;
                    if constexpr (BACK) {
                        float d[V];
                        get<V>(static_cast<const T*>(p.dy) + to, d);
                        backward<T, V>(p, k, v, d, z, p.dgate ? static_cast<T*>(p.dgate) + to : nullptr);
#pragma unroll
                        for (int i = 0; i < V; ++i) d[i] = k.rstd[i] * (k.w[i] * d[i] - ma[i] - v[i] * mb[i]);
                        put<V>(static_cast<T*>(p.dx) + to, d);
                    } else {
                        forward<T, V>(p, k, v, z, static_cast<T*>(p.y) + to);
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
        join_kernel<<<dim3(p.groups, nz, (unsigned)((p.samples + nz - 1) / nz)), kThreads, 0, st>>>(p, q.splits);
        if (int rc = launch_status("group norm: statistics")) return rc;
    } else {
        fold_kernel<<<(unsigned)((p.samples * row + kThreads - 1) / kThreads), kThreads, 0, st>>>(ws, q.splits, p.samples, (int)row, after);
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
