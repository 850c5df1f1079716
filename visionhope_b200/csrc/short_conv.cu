// Short causal convolution over channels-last token rows: forward, backward and one-token step
// (vh_short_conv_fwd, vh_short_conv_bwd, vh_short_conv_step).
//
//   c_t = bias + sum_k w_k x_{t-K+1+k},   y_t = c_t or silu(c_t)
//
// A thread owns V neighbouring channels and walks a run of tokens of one sequence with the last K
// inputs in registers, so each input is read once, plus K - 1 rows of halo per run.  There is no
// reuse beyond the window and 2 K flops per element: the kernels are bounded by HBM.
#include <algorithm>
#include <type_traits>

#include "abi_util.h"
#include "ssm_common.cuh"

namespace vh {
namespace ssm {
namespace {

constexpr int kFwdRun = 16;   // tokens a thread walks in the forward
constexpr int kBwdRun = 32;   // and in the backward (its halo is K - 1 rows on both sides)
constexpr int kThreads = 256;

struct ConvParams {
    const void* x;
    Rows xr;
    const float *w, *bias;
    const void* initial;
    void* y;
    void* final_state;
    Seqs seqs;
    int32_t channels, silu, vec;
    // backward
    const void *dy, *dfinal;
    void *dx, *dinitial;
    float* partial;  // [blocks][K + 1][channels]
};

template <int V, int K>
struct Weights {
    float w[K][V], b[V];
    __device__ __forceinline__ void load(const ConvParams& p, int c) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
#pragma unroll
            for (int k = 0; k < K; ++k) w[k][v] = c + v < p.channels ? p.w[(int64_t)(c + v) * K + k] : 0.f;
            b[v] = p.bias && c + v < p.channels ? p.bias[c + v] : 0.f;
        }
    }
};

// Input j of a sequence, j >= -(K - 1): tokens, and before them the initial state.
template <typename T, int V, int K>
__device__ __forceinline__ void input_at(const ConvParams& p, const T* x, int64_t step, int s, int c, int64_t j,
                                         float (&v)[V]) {
    if (j >= 0) {
        load_v<V>(x + j * step, c, p.channels, p.vec, v);
    } else if (p.initial) {
        load_v<V>(static_cast<const T*>(p.initial) + ((int64_t)s * (K - 1) + (j + K - 1)) * p.channels + c, c,
                  p.channels, p.vec, v);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = 0.f;
    }
}

template <typename T, int V, int K>
__global__ void __launch_bounds__(kThreads) conv_fwd_kernel(const ConvParams p, int64_t items, int32_t cgroups) {
    const int64_t item = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (item >= items) return;
    const int64_t slot = item / cgroups;
    const int c = (int)(item % cgroups) * V;
    const int s = seq_of_slot(p.seqs, slot, kFwdRun);
    const Seq seq = seq_at(p.seqs, s);
    const int64_t j0 = (slot - slot_base(p.seqs, s, seq.row, kFwdRun)) * kFwdRun;
    if (j0 < 0 || (j0 > 0 && j0 >= seq.len)) return;  // a slot that no sequence, or not this one, needs
    const int64_t j1 = min(j0 + kFwdRun, seq.len);
    const T* x = static_cast<const T*>(p.x) + first_row(p.seqs, seq, s, p.xr) + c;
    const int64_t xs = row_step(p.seqs, p.xr);
    const Rows yr{p.seqs.length * p.channels, p.channels};
    T* y = static_cast<T*>(p.y) + first_row(p.seqs, seq, s, yr) + c;
    const int64_t ys = row_step(p.seqs, yr);
    Weights<V, K> wt;
    wt.load(p, c);
    float win[K][V];  // the last K inputs, newest last
#pragma unroll
    for (int k = 1; k < K; ++k) input_at<T, V, K>(p, x, xs, s, c, j0 - K + k, win[k]);
    for (int64_t j = j0; j < j1; ++j) {
#pragma unroll
        for (int k = 0; k + 1 < K; ++k)
#pragma unroll
            for (int v = 0; v < V; ++v) win[k][v] = win[k + 1][v];
        load_v<V>(x + j * xs, c, p.channels, p.vec, win[K - 1]);
        float out[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            float a = wt.b[v];
#pragma unroll
            for (int k = 0; k < K; ++k) a = fmaf(wt.w[k][v], win[k][v], a);
            out[v] = p.silu ? a * sigmoid(a) : a;
        }
        store_v<V>(y + j * ys, c, p.channels, p.vec, out);
    }
    if (p.final_state && j1 == seq.len) {
        // the last K - 1 inputs, which are the initial state's where the sequence is shorter
        T* f = static_cast<T*>(p.final_state) + (int64_t)s * (K - 1) * p.channels + c;
#pragma unroll
        for (int k = 1; k < K; ++k) store_v<V>(f + (k - 1) * p.channels, c, p.channels, p.vec, win[k]);
    }
}

// The backward.  With dc_t = dy_t act'(c_t) (zero outside the sequence):
//   dx_j = sum_k w_k dc_{j+K-1-k},   dw_k = sum_t dc_t x_{t-K+1+k},   db = sum_t dc_t.
// A run walks i from its first token to K - 1 tokens past its last: dc_i from the window of inputs
// (c_i is computed again), then dx_{i-K+1} from the last K values of dc.  A sequence's first run
// also emits the K - 1 values before it, the gradient of its initial state.  A final state's
// gradient belongs to the inputs that the state holds.  Threads of a block sum their dw and db over
// their runs in registers, the block in shared memory, and a second kernel over the blocks, all in
// a fixed order.
template <typename T, int V, int K>
__global__ void __launch_bounds__(kThreads) conv_bwd_kernel(const ConvParams p, int64_t slots, int32_t cblock) {
    // A block: `cblock` channel groups by kThreads / cblock runs.
    extern __shared__ float red[];
    const int lanes = kThreads / cblock;
    const int ci = threadIdx.x % cblock, ri = threadIdx.x / cblock;
    const int cg = blockIdx.x * cblock + ci;
    const int c = cg * V;
    const bool live = ri < lanes && c < p.channels;
    float dw[K][V], db[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        db[v] = 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k) dw[k][v] = 0.f;
    }
    if (live) {
        Weights<V, K> wt;
        wt.load(p, c);
        const Rows yr{p.seqs.length * p.channels, p.channels};
        for (int64_t slot = (int64_t)blockIdx.y * lanes + ri; slot < slots; slot += (int64_t)gridDim.y * lanes) {
            const int s = seq_of_slot(p.seqs, slot, kBwdRun);
            const Seq seq = seq_at(p.seqs, s);
            const int64_t j0 = (slot - slot_base(p.seqs, s, seq.row, kBwdRun)) * kBwdRun;
            if (j0 < 0 || (j0 > 0 && j0 >= seq.len)) continue;
            const int64_t j1 = min(j0 + kBwdRun, seq.len);
            const T* x = static_cast<const T*>(p.x) + first_row(p.seqs, seq, s, p.xr) + c;
            const int64_t xs = row_step(p.seqs, p.xr);
            const int64_t y0 = first_row(p.seqs, seq, s, yr), ys = row_step(p.seqs, yr);
            const T* dy = static_cast<const T*>(p.dy) + y0 + c;
            T* dx = static_cast<T*>(p.dx) + y0 + c;
            const T* df = p.dfinal ? static_cast<const T*>(p.dfinal) + (int64_t)s * (K - 1) * p.channels + c : nullptr;
            T* di = p.dinitial ? static_cast<T*>(p.dinitial) + (int64_t)s * (K - 1) * p.channels + c : nullptr;
            float win[K][V], dc[K][V];
#pragma unroll
            for (int k = 1; k < K; ++k) input_at<T, V, K>(p, x, xs, s, c, j0 - K + k, win[k]);
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int v = 0; v < V; ++v) dc[k][v] = 0.f;
            for (int64_t i = j0; i < j1 + K - 1; ++i) {
#pragma unroll
                for (int k = 0; k + 1 < K; ++k)
#pragma unroll
                    for (int v = 0; v < V; ++v) {
                        win[k][v] = win[k + 1][v];
                        dc[k][v] = dc[k + 1][v];
                    }
                if (i < seq.len) {
                    float g[V];
                    load_v<V>(x + i * xs, c, p.channels, p.vec, win[K - 1]);
                    load_v<V>(dy + i * ys, c, p.channels, p.vec, g);
#pragma unroll
                    for (int v = 0; v < V; ++v) {
                        if (p.silu) {
                            float a = wt.b[v];
#pragma unroll
                            for (int k = 0; k < K; ++k) a = fmaf(wt.w[k][v], win[k][v], a);
                            const float sg = sigmoid(a);
                            g[v] *= sg * (1.f + a * (1.f - sg));
                        }
                        dc[K - 1][v] = g[v];
                        if (i < j1) {
                            db[v] += g[v];
#pragma unroll
                            for (int k = 0; k < K; ++k) dw[k][v] = fmaf(g[v], win[k][v], dw[k][v]);
                        }
                    }
                } else {
#pragma unroll
                    for (int v = 0; v < V; ++v) dc[K - 1][v] = 0.f;
                }
                const int64_t j = i - (K - 1);
                if (j >= j0 || (j < 0 && di)) {
                    float out[V];
#pragma unroll
                    for (int v = 0; v < V; ++v) {
                        out[v] = 0.f;
                        // dc[m] is dc_{j+m}: tap K - 1 - m
#pragma unroll
                        for (int m = 0; m < K; ++m) out[v] = fmaf(wt.w[K - 1 - m][v], dc[m][v], out[v]);
                    }
                    const int64_t kept = j - (seq.len - (K - 1));  // place of input j in the final state
                    if (df && kept >= 0) {
                        float f[V];
                        load_v<V>(df + kept * p.channels, c, p.channels, p.vec, f);
#pragma unroll
                        for (int v = 0; v < V; ++v) out[v] += f[v];
                    }
                    if (j >= 0) store_v<V>(dx + j * ys, c, p.channels, p.vec, out);
                    else store_v<V>(di + (j + K - 1) * p.channels, c, p.channels, p.vec, out);
                }
            }
        }
    }
    // the block's sums: one value of every thread at a time, added over the runs in order
#pragma unroll
    for (int k = 0; k <= K; ++k)
#pragma unroll
        for (int v = 0; v < V; ++v) {
            red[threadIdx.x] = k < K ? dw[k < K ? k : 0][v] : db[v];
            __syncthreads();
            if (ri == 0 && live && c + v < p.channels) {
                float sum = 0.f;
                for (int r = 0; r < lanes; ++r) sum += red[r * cblock + ci];
                p.partial[((int64_t)blockIdx.y * (K + 1) + k) * p.channels + c + v] = sum;
            }
            __syncthreads();
        }
}

// Sums the blocks' partials: a warp per output, lanes over the blocks.
__global__ void __launch_bounds__(256) conv_bwd_reduce_kernel(const float* __restrict__ partial, int32_t blocks,
                                                              int32_t channels, int32_t taps, float* __restrict__ dw,
                                                              float* __restrict__ db) {
    const int i = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (i >= channels * (taps + 1)) return;
    const int k = i / channels, c = i % channels;
    float sum = 0.f;
    for (int b = lane; b < blocks; b += 32) sum += partial[((int64_t)b * (taps + 1) + k) * channels + c];
    sum = warp_sum(sum);
    if (lane == 0) {
        if (k < taps) dw[(int64_t)c * taps + k] = sum;
        else if (db) db[c] = sum;
    }
}

template <typename T, int V, int K>
__global__ void __launch_bounds__(kThreads) conv_step_kernel(const T* __restrict__ x, int64_t x_stride,
                                                             const float* __restrict__ w, const float* __restrict__ bias,
                                                             const T* state, T* state_out,
                                                             const int32_t* __restrict__ index, int32_t slots,
                                                             T* __restrict__ y, int64_t items, int32_t cgroups,
                                                             int32_t channels, int32_t silu, int32_t vec) {
    const int64_t item = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (item >= items) return;
    const int s = (int)(item / cgroups), c = (int)(item % cgroups) * V;
    const int slot = index ? index[s] : s;
    float out[V];
    if (slot < 0 || slot >= slots) {
#pragma unroll
        for (int v = 0; v < V; ++v) out[v] = 0.f;
        store_v<V>(y + (int64_t)s * channels + c, c, channels, vec, out);
        return;
    }
    float win[K][V];
    const int64_t at = (int64_t)slot * (K - 1) * channels + c;
#pragma unroll
    for (int k = 0; k + 1 < K; ++k) load_v<V>(state + at + (int64_t)k * channels, c, channels, vec, win[k]);
    load_v<V>(x + s * x_stride + c, c, channels, vec, win[K - 1]);
#pragma unroll
    for (int v = 0; v < V; ++v) {
        float a = bias && c + v < channels ? bias[c + v] : 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k) a = fmaf(c + v < channels ? w[(int64_t)(c + v) * K + k] : 0.f, win[k][v], a);
        out[v] = silu ? a * sigmoid(a) : a;
    }
    store_v<V>(y + (int64_t)s * channels + c, c, channels, vec, out);
#pragma unroll
    for (int k = 1; k < K; ++k) store_v<V>(state_out + at + (int64_t)(k - 1) * channels, c, channels, vec, win[k]);
}

template <typename F>
int with_dtype(int dtype, F&& f) {
    if (dtype == VH_F32) return f(float{});
    if (dtype == VH_BF16) return f(__nv_bfloat16{});
    return f(__half{});
}
template <typename F>
int with_taps(int taps, F&& f) {
    switch (taps) {
        case 2: return f(std::integral_constant<int, 2>{});
        case 3: return f(std::integral_constant<int, 3>{});
        case 4: return f(std::integral_constant<int, 4>{});
        case 5: return f(std::integral_constant<int, 5>{});
        case 6: return f(std::integral_constant<int, 6>{});
        case 7: return f(std::integral_constant<int, 7>{});
        default: return f(std::integral_constant<int, 8>{});
    }
}
template <typename F>
int with_width(bool vec, F&& f) {
    return vec ? f(std::integral_constant<int, 4>{}) : f(std::integral_constant<int, 1>{});
}

int check_conv(const char* what, const vh_short_conv_args* a) {
    if (!a) return fail(VH_E_ARG, "%s: null argument struct", what);
    if (!a->x || !a->weight || !a->y) return fail(VH_E_ARG, "%s: null pointer argument", what);
    if (!dtype_ok(a->dtype)) return fail(VH_E_DTYPE, "%s: dtype must be VH_F32, VH_BF16 or VH_F16", what);
    if (a->activation != 0 && a->activation != 1) return fail(VH_E_ARG, "%s: activation must be 0 (none) or 1 (silu)", what);
    if (a->taps < 2 || a->taps > 8) return fail(VH_E_SHAPE, "%s: taps must be 2 to 8 (got %d)", what, a->taps);
    if (a->batch <= 0 || a->channels <= 0) return fail(VH_E_SHAPE, "%s: batch and channels must be positive", what);
    if (a->length < 0) return fail(VH_E_SHAPE, "%s: negative length", what);
    if (a->length > 0x7fffffff) return fail(VH_E_RANGE, "%s: at most 2^31 - 1 tokens a sequence", what);
    const size_t es = dtype_size(a->dtype);
    for (const void* t : {a->x, a->initial_state, (const void*)a->y, (const void*)a->final_state})
        if (t && !aligned(t, es)) return fail(VH_E_ALIGN, "%s: misaligned pointers", what);
    if (!aligned(a->weight, 4) || (a->bias && !aligned(a->bias, 4)) || (a->seq_offsets && !aligned(a->seq_offsets, 4)))
        return fail(VH_E_ALIGN, "%s: misaligned pointers", what);
    return 0;
}

// Four channels at a time wherever every row starts on a boundary of four elements.
bool conv_vec(const vh_short_conv_args* a, std::initializer_list<const void*> more) {
    const size_t es = 4 * dtype_size(a->dtype);
    bool v = a->channels % 4 == 0 && a->x_batch_stride % 4 == 0 && a->x_token_stride % 4 == 0;
    for (const void* t : {a->x, a->initial_state}) v = v && (!t || aligned(t, es));
    for (const void* t : more) v = v && (!t || aligned(t, es));
    return v;
}

ConvParams conv_params(const vh_short_conv_args* a) {
    ConvParams p{};
    p.x = a->x; p.xr = {a->x_batch_stride, a->x_token_stride};
    p.w = a->weight; p.bias = a->bias; p.initial = a->initial_state; p.y = a->y; p.final_state = a->final_state;
    p.seqs = {a->seq_offsets, a->length, a->batch, a->reverse != 0};
    p.channels = a->channels; p.silu = a->activation;
    return p;
}

struct BwdPlan {
    int64_t slots;
    int cgroups, cblock, gx, gy;
};
BwdPlan bwd_plan(const vh_short_conv_args* a, int width) {
    BwdPlan b;
    b.slots = slot_total(a->seq_offsets != nullptr, a->length, a->batch, kBwdRun);
    b.cgroups = (a->channels + width - 1) / width;
    b.cblock = std::min(b.cgroups, 64);
    b.gx = (b.cgroups + b.cblock - 1) / b.cblock;
    const int lanes = kThreads / b.cblock;
    const int64_t want = (b.slots + lanes - 1) / lanes;
    b.gy = (int)std::max<int64_t>(1, std::min<int64_t>(want, (8 * 148 + b.gx - 1) / b.gx));
    return b;
}

}  // namespace
}  // namespace ssm
}  // namespace vh

using namespace vh;
using namespace vh::ssm;

extern "C" int vh_short_conv_fwd(const vh_short_conv_args* a, vh_stream_t stream) {
    clear_error();
    if (int rc = check_conv("vh_short_conv_fwd", a)) return rc;
    ConvParams p = conv_params(a);
    p.vec = conv_vec(a, {a->y, a->final_state});
    return with_dtype(a->dtype, [&](auto t) {
        using T = decltype(t);
        return with_width(p.vec, [&](auto width) {
            constexpr int V = decltype(width)::value;
            const int cgroups = (a->channels + V - 1) / V;
            const int64_t items = slot_total(a->seq_offsets != nullptr, a->length, a->batch, kFwdRun) * cgroups;
            const int64_t blocks = (items + kThreads - 1) / kThreads;
            if (blocks > 0x7fffffff) return fail(VH_E_RANGE, "vh_short_conv_fwd: too many elements");
            return with_taps(a->taps, [&](auto taps) {
                conv_fwd_kernel<T, V, decltype(taps)::value>
                    <<<(int)blocks, kThreads, 0, static_cast<cudaStream_t>(stream)>>>(p, items, cgroups);
                return launch_status("short convolution");
            });
        });
    });
}

extern "C" int64_t vh_short_conv_bwd_workspace_bytes(const vh_short_conv_args* a) {
    if (!a || a->batch <= 0 || a->channels <= 0 || a->length < 0 || a->taps < 2 || a->taps > 8) return 0;
    const int64_t rows = std::max(bwd_plan(a, 4).gy, bwd_plan(a, 1).gy);
    return rows * (a->taps + 1) * a->channels * 4;
}

extern "C" int vh_short_conv_bwd(const vh_short_conv_args* a, const void* grad_y, const void* grad_final, void* grad_x,
                                 float* grad_weight, float* grad_bias, void* grad_initial, void* workspace,
                                 int64_t workspace_bytes, vh_stream_t stream) {
    clear_error();
    vh_short_conv_args copy;
    if (a) {
        copy = *a;
        if (!copy.y) copy.y = grad_x;  // the backward does not read y
        copy.final_state = nullptr;
        a = &copy;
    }
    if (int rc = check_conv("vh_short_conv_bwd", a)) return rc;
    if (!grad_y || !grad_x || !grad_weight || !workspace) return fail(VH_E_ARG, "vh_short_conv_bwd: null pointer argument");
    const size_t es = dtype_size(a->dtype);
    for (const void* t : {grad_y, grad_final, (const void*)grad_x, (const void*)grad_initial})
        if (t && !aligned(t, es)) return fail(VH_E_ALIGN, "vh_short_conv_bwd: misaligned pointers");
    if (workspace_bytes < vh_short_conv_bwd_workspace_bytes(a) || !aligned(workspace, 4))
        return fail(VH_E_ARG, "vh_short_conv_bwd: workspace too small");
    ConvParams p = conv_params(a);
    p.vec = conv_vec(a, {grad_y, grad_final, grad_x, grad_initial});
    p.dy = grad_y; p.dfinal = grad_final; p.dx = grad_x; p.dinitial = grad_initial;
    p.partial = static_cast<float*>(workspace);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    int blocks = 0;
    const int rc = with_dtype(a->dtype, [&](auto t) {
        using T = decltype(t);
        return with_width(p.vec, [&](auto width) {
            constexpr int V = decltype(width)::value;
            const BwdPlan b = bwd_plan(a, V);
            blocks = b.gy;
            return with_taps(a->taps, [&](auto taps) {
                conv_bwd_kernel<T, V, decltype(taps)::value>
                    <<<dim3(b.gx, b.gy), kThreads, kThreads * sizeof(float), st>>>(p, b.slots, b.cblock);
                return launch_status("short convolution backward");
            });
        });
    });
    if (rc) return rc;
    conv_bwd_reduce_kernel<<<(a->channels * (a->taps + 1) + 7) / 8, 256, 0, st>>>(p.partial, blocks, a->channels, a->taps,
                                                                                  grad_weight, grad_bias);
    return launch_status("short convolution backward sums");
}

extern "C" int vh_short_conv_step(const void* x, int64_t x_batch_stride, int32_t dtype, const float* weight,
                                  const float* bias, int32_t activation, const void* state, void* state_out,
                                  const int32_t* slots_index, int32_t slots, void* y, int32_t batch, int32_t channels,
                                  int32_t taps, vh_stream_t stream) {
    clear_error();
    vh_short_conv_args a{};
    a.x = x; a.x_batch_stride = x_batch_stride; a.weight = weight; a.bias = bias; a.y = y;
    a.dtype = dtype; a.activation = activation; a.taps = taps; a.batch = batch; a.channels = channels;
    if (int rc = check_conv("vh_short_conv_step", &a)) return rc;
    if (!state || !state_out) return fail(VH_E_ARG, "vh_short_conv_step: null state");
    const size_t es = dtype_size(dtype);
    if (!aligned(state, es) || !aligned(state_out, es) || (slots_index && !aligned(slots_index, 4)))
        return fail(VH_E_ALIGN, "vh_short_conv_step: misaligned pointers");
    if (slots <= 0 || (!slots_index && slots < batch))
        return fail(VH_E_SHAPE, "vh_short_conv_step: %d slots for %d streams", slots, batch);
    const bool vec = conv_vec(&a, {state, (const void*)state_out, (const void*)y});
    return with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        return with_width(vec, [&](auto width) {
            constexpr int V = decltype(width)::value;
            const int cgroups = (channels + V - 1) / V;
            const int64_t items = (int64_t)batch * cgroups;
            const int64_t blocks = (items + kThreads - 1) / kThreads;
            if (blocks > 0x7fffffff) return fail(VH_E_RANGE, "vh_short_conv_step: too many elements");
            return with_taps(taps, [&](auto k) {
                conv_step_kernel<T, V, decltype(k)::value><<<(int)blocks, kThreads, 0, static_cast<cudaStream_t>(stream)>>>(
                    static_cast<const T*>(x), x_batch_stride, weight, bias, static_cast<const T*>(state),
                    static_cast<T*>(state_out), slots_index, slots, static_cast<T*>(y), items, cgroups, channels,
                    activation, vec);
                return launch_status("short convolution step");
            });
        });
    });
}
