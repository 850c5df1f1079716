// Short causal convolution over channels-last token rows: forward, backward and one-token step
// (vh_short_conv_fwd, vh_short_conv_bwd, vh_short_conv_step).
//
//   c_t = bias + sum_k w_k x_{t-K+1+k},   y_t = c_t or silu(c_t)
//
// A thread owns V neighbouring channels (8 bytes of them, or one) and walks runs of tokens with the
// last K inputs in registers, so each input is read once, plus K - 1 rows of halo per run.  There is
// no reuse beyond the window and 2 K flops per element, so what counts is bytes in flight and few
// instructions per element.  A thread therefore fetches its tokens into shared memory of its own two
// blocks of four ahead (asynchronous copies take no registers; forward and backward of the sizes
// below took 80 us with them and 95 with plain loads), and runs are as long as one
// wave of threads allows, so that weights, halo and the search for the sequence are paid once for
// many tokens (forward with runs of 8, 16 and 24 tokens: 42, 36 and 35 us against 31 at the time).
//
// 64 sequences of 3136 tokens, 128 channels, K = 4, silu, bf16: forward 24 us (103 MB, 4.2 TB/s),
// backward 48 us (154 MB, 3.2 TB/s), its sums over blocks 3.  No unit is at its limit: instruction issue
// at 42 %, the special-function unit at 57 and 27 %, DRAM at about 30 %, with 20 and 15 warps an SM
// waiting for memory.  Accesses of 16 bytes (eight channels a thread, half the threads) took 33
// against 31 us, blocks of eight tokens 42 against 39.  24 packed sequences of 16384 tokens, 1024
// channels: 20 us (67 MB, 3.4 TB/s).  The step of 256 streams of 2048 channels: 5.3 us, two dependent
// latencies.
#include <algorithm>
#include <type_traits>

#include "abi_util.h"
#include "ssm_common.cuh"

namespace vh {
namespace ssm {
namespace {

constexpr int kBlock = 4;     // tokens fetched at a time
constexpr int kRing = 3;      // blocks held: the one at hand and two ahead
constexpr int kThreads = 256;
constexpr int kFwdBlocks = 3, kBwdBlocks = 2;  // blocks an SM holds (three backward spill: 105 against 61 us)

struct ConvParams {
    const void* x;
    Rows xr;
    const float *w, *bias;
    const void* initial;
    void* y;
    void* final_state;
    Seqs seqs;
    int32_t channels, silu, run;  // run: tokens a thread walks
    // backward
    const void *dy, *dfinal;
    void *dx, *dinitial;
    float* partial;  // [blocks][K + 1][channels]
};

template <typename T, int V>
__device__ __forceinline__ void store(T* p, const float2 (&v)[kPairs<V>]) {
    Pack<T, V> q;
    float f[V];
    from_pairs<V>(v, f);
    q.set(f);
    *reinterpret_cast<Pack<T, V>*>(p) = q;
}
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> load(const T* p) { return *reinterpret_cast<const Pack<T, V>*>(p); }

template <int V, int K>
struct Weights {
    float2 w[K][kPairs<V>], b[kPairs<V>];
    __device__ __forceinline__ void load(const ConvParams& p, int c) {
        float v[V * K];
        const float* src = p.w + (int64_t)c * K;
        if (V % 4 == 0 && reinterpret_cast<uintptr_t>(p.w) % 16 == 0) {
#pragma unroll
            for (int i = 0; i < V * K / 4; ++i) {
                const float4 q = reinterpret_cast<const float4*>(src)[i];
                v[4 * i] = q.x; v[4 * i + 1] = q.y; v[4 * i + 2] = q.z; v[4 * i + 3] = q.w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < V * K; ++i) v[i] = src[i];
        }
#pragma unroll
        for (int i = 0; i < kPairs<V>; ++i) {
#pragma unroll
            for (int k = 0; k < K; ++k) w[k][i] = make_float2(v[2 * i * K + k], V > 1 ? v[(V > 1 ? 2 * i + 1 : 0) * K + k] : 0.f);
            b[i] = p.bias ? make_float2(p.bias[c + 2 * i], V > 1 ? p.bias[c + (V > 1 ? 2 * i + 1 : 0)] : 0.f)
                          : make_float2(0.f, 0.f);
        }
    }
    // c_t of the window whose newest input is win[K - 1]
    __device__ __forceinline__ float2 at(const float2 (&win)[K][kPairs<V>], int i) const {
        float2 a = b[i];
#pragma unroll
        for (int k = 0; k < K; ++k) a = ffma2(w[k][i], win[k][i], a);
        return a;
    }
};

template <int K, int P>
__device__ __forceinline__ void shift(float2 (&win)[K][P]) {
#pragma unroll
    for (int k = 0; k + 1 < K; ++k)
#pragma unroll
        for (int i = 0; i < P; ++i) win[k][i] = win[k + 1][i];
}

// The inputs before token j0 of a sequence into win[1 .. K - 1]: tokens, and before them the initial
// state.
template <typename T, int V, int K>
__device__ __forceinline__ void enter(const ConvParams& p, const T* x, int64_t step, int s, int c, int64_t j0,
                                      float2 (&win)[K][kPairs<V>]) {
#pragma unroll
    for (int k = 1; k < K; ++k) {
        const int64_t j = j0 - K + k;
        if (j >= 0) unpack<T, V>(load<T, V>(x + j * step), win[k]);
        else if (p.initial)
            unpack<T, V>(load<T, V>(static_cast<const T*>(p.initial) + ((int64_t)s * (K - 1) + (j + K - 1)) * p.channels + c),
                         win[k]);
        else
#pragma unroll
            for (int i = 0; i < kPairs<V>; ++i) win[k][i] = make_float2(0.f, 0.f);
    }
}

// A thread's ring of fetched rows: row i of block b lies kThreads apart from its neighbours, and the
// thread reads only what it fetched.
template <typename T, int V>
struct Ring {
    Pack<T, V>* own;
    __device__ __forceinline__ explicit Ring(void* smem) : own(static_cast<Pack<T, V>*>(smem) + threadIdx.x) {}
    __device__ __forceinline__ Pack<T, V>& at(int slot, int i) const { return own[(slot * kBlock + i) * kThreads]; }
    // rows from .. from + 3, none past `last`
    __device__ __forceinline__ void fill(int slot, const T* p, int64_t step, int from, int last) const {
        if (from + kBlock - 1 <= last) {
            const T* q = p + from * step;
#pragma unroll
            for (int i = 0; i < kBlock; ++i) fetch(&at(slot, i), q + i * step, V, true);
        } else {
#pragma unroll
            for (int i = 0; i < kBlock; ++i)
                if (from + i <= last) fetch(&at(slot, i), p + (from + i) * step, V, true);
        }
    }
};
__device__ __forceinline__ int next_slot(int slot) { return slot + 1 == kRing ? 0 : slot + 1; }

// Zeros in the thread's channels of packed rows of no sequence: every `step`-th row from the `at`-th.
template <typename T, int V>
__device__ __forceinline__ void zero_rows(const ConvParams& p, void* out, int c, int64_t at, int64_t step) {
    if (!p.seqs.offsets) return;
    const Outside o(p.seqs);
    float2 zero[kPairs<V>];
#pragma unroll
    for (int q = 0; q < kPairs<V>; ++q) zero[q] = make_float2(0.f, 0.f);
    for (; at < o.count(); at += step) store<T, V>(static_cast<T*>(out) + o.row(at) * p.channels + c, zero);
}

// A block: `cblock` channel groups by kThreads / cblock runs, over channels and slots.
template <typename T, int V, int K>
__global__ void __launch_bounds__(kThreads, kFwdBlocks)
    conv_fwd_kernel(const ConvParams p, int64_t slots, int32_t cblock) {
    constexpr int P = kPairs<V>;
    const int lanes = kThreads / cblock;
    const int ri = threadIdx.x / cblock;
    const int c = (blockIdx.x * cblock + threadIdx.x % cblock) * V;
    if (ri >= lanes || c >= p.channels) return;
    extern __shared__ __align__(16) unsigned char smem[];
    const Ring<T, V> ring(smem);
    Weights<V, K> wt;
    wt.load(p, c);
    const int64_t xs = row_step(p.seqs, p.xr);
    const Rows yr{p.seqs.length * p.channels, p.channels};
    const int64_t ys = row_step(p.seqs, yr);
    for (int64_t slot = (int64_t)blockIdx.y * lanes + ri; slot < slots; slot += (int64_t)gridDim.y * lanes) {
        const int s = seq_of_slot(p.seqs, slot, p.run);
        const Seq seq = seq_at(p.seqs, s);
        const int64_t j0 = (slot - slot_base(p.seqs, s, seq.row, p.run)) * p.run;
        if (j0 < 0 || (j0 > 0 && j0 >= seq.len)) continue;  // a slot that no sequence, or not this one, needs
        const int count = (int)min((int64_t)p.run, seq.len - j0);
        const T* x = static_cast<const T*>(p.x) + first_row(p.seqs, seq, s, p.xr) + c;
        T* y = static_cast<T*>(p.y) + first_row(p.seqs, seq, s, yr) + c + j0 * ys;
        const T* xj = x + j0 * xs;
        float2 win[K][P];
        auto step = [&](const Pack<T, V>& in) {
            shift(win);
            unpack<T, V>(in, win[K - 1]);
            float2 out[P];
#pragma unroll
            for (int q = 0; q < P; ++q) {
                const float2 a = wt.at(win, q);
                out[q] = p.silu ? fmul2(a, sigmoid2(a)) : a;
            }
            store<T, V>(y, out);
            y += ys;
        };
#pragma unroll
        for (int b = 0; b + 1 < kRing; ++b) {
            ring.fill(b, xj, xs, b * kBlock, count - 1);
            cp_async_commit();
        }
        enter<T, V, K>(p, x, xs, s, c, j0, win);
        for (int t = 0, slot = 0; t < count; t += kBlock, slot = next_slot(slot)) {
            cp_async_wait<kRing - 2>();
            Pack<T, V> in[kBlock];
#pragma unroll
            for (int i = 0; i < kBlock; ++i) in[i] = ring.at(slot, i);
            ring.fill(slot == 0 ? kRing - 1 : slot - 1, xj, xs, t + (kRing - 1) * kBlock, count - 1);
            cp_async_commit();
            if (t + kBlock <= count) {
#pragma unroll
                for (int i = 0; i < kBlock; ++i) step(in[i]);
            } else {
#pragma unroll
                for (int i = 0; i + 1 < kBlock; ++i)
                    if (t + i < count) step(in[i]);
            }
        }
        cp_async_wait<0>();
        if (p.final_state && j0 + count == seq.len) {
            // the last K - 1 inputs, which are the initial state's where the sequence is shorter
            T* f = static_cast<T*>(p.final_state) + (int64_t)s * (K - 1) * p.channels + c;
#pragma unroll
            for (int k = 1; k < K; ++k) store<T, V>(f + (k - 1) * p.channels, win[k]);
        }
    }
    zero_rows<T, V>(p, p.y, c, (int64_t)blockIdx.y * lanes + ri, (int64_t)gridDim.y * lanes);
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
__global__ void __launch_bounds__(kThreads, kBwdBlocks) conv_bwd_kernel(const ConvParams p, int64_t slots, int32_t cblock) {
    constexpr int P = kPairs<V>;
    extern __shared__ __align__(16) unsigned char smem[];
    const Ring<T, V> rx(smem), rg(static_cast<Pack<T, V>*>(static_cast<void*>(smem)) + kRing * kBlock * kThreads);
    const int lanes = kThreads / cblock;
    const int ci = threadIdx.x % cblock, ri = threadIdx.x / cblock;
    const int c = (blockIdx.x * cblock + ci) * V;
    const bool live = ri < lanes && c < p.channels;
    const float2 zero = make_float2(0.f, 0.f);
    float2 dw[K][P], db[P];
#pragma unroll
    for (int q = 0; q < P; ++q) {
        db[q] = zero;
#pragma unroll
        for (int k = 0; k < K; ++k) dw[k][q] = zero;
    }
    if (live) {
        Weights<V, K> wt;
        wt.load(p, c);
        const int64_t xs = row_step(p.seqs, p.xr);
        const Rows yr{p.seqs.length * p.channels, p.channels};
        const int64_t ys = row_step(p.seqs, yr);
        for (int64_t slot = (int64_t)blockIdx.y * lanes + ri; slot < slots; slot += (int64_t)gridDim.y * lanes) {
            const int s = seq_of_slot(p.seqs, slot, p.run);
            const Seq seq = seq_at(p.seqs, s);
            const int64_t j0 = (slot - slot_base(p.seqs, s, seq.row, p.run)) * p.run;
            if (j0 < 0 || (j0 > 0 && j0 >= seq.len)) continue;
            const T* x = static_cast<const T*>(p.x) + first_row(p.seqs, seq, s, p.xr) + c;
            const int64_t y0 = first_row(p.seqs, seq, s, yr);
            const T* dy = static_cast<const T*>(p.dy) + y0 + c + j0 * ys;
            T* dx = static_cast<T*>(p.dx) + y0 + c + j0 * ys;
            const T* df = p.dfinal ? static_cast<const T*>(p.dfinal) + (int64_t)s * (K - 1) * p.channels + c : nullptr;
            T* di = p.dinitial && j0 == 0 ? static_cast<T*>(p.dinitial) + (int64_t)s * (K - 1) * p.channels + c : nullptr;
            // tokens counted from j0: [0, count) are the run's, [count, ends) belong to the next one
            const int count = (int)min((int64_t)p.run, seq.len - j0);
            const int ends = (int)min((int64_t)(count + K - 1), seq.len - j0);
            const int64_t kept0 = j0 - (seq.len - (K - 1));  // place of token 0 in the final state
            const T* xj = x + j0 * xs;
            float2 win[K][P], dc[K][P];
            enter<T, V, K>(p, x, xs, s, c, j0, win);
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int q = 0; q < P; ++q) dc[k][q] = zero;
            // INNER: the token is the run's and so is the one that it completes
            auto step = [&](const Pack<T, V>& xin, const Pack<T, V>& gin, int t, auto inner) {
                constexpr bool kInner = decltype(inner)::value;
                shift(win);
                shift(dc);
                if (kInner || t < ends) {
                    float2 g[P];
                    unpack<T, V>(xin, win[K - 1]);
                    unpack<T, V>(gin, g);
#pragma unroll
                    for (int q = 0; q < P; ++q) {
                        if (p.silu) {
                            // silu'(a) = sg (1 + a (1 - sg))
                            const float2 a = wt.at(win, q), sg = sigmoid2(a);
                            const float2 r = ffma2(a, fsub2(splat2(1.f), sg), splat2(1.f));
                            g[q] = fmul2(g[q], fmul2(sg, r));
                        }
                        dc[K - 1][q] = g[q];
                    }
                    if (kInner || t < count)
#pragma unroll
                        for (int q = 0; q < P; ++q) {
                            db[q] = fadd2(db[q], g[q]);
#pragma unroll
                            for (int k = 0; k < K; ++k) dw[k][q] = ffma2(g[q], win[k][q], dw[k][q]);
                        }
                } else {
#pragma unroll
                    for (int q = 0; q < P; ++q) dc[K - 1][q] = zero;
                }
                const int j = t - (K - 1);
                if (kInner || j >= 0 || di) {
                    float2 out[P];
#pragma unroll
                    for (int q = 0; q < P; ++q) {
                        // dc[m] is dc_{j+m}: tap K - 1 - m
                        out[q] = fmul2(wt.w[K - 1][q], dc[0][q]);
#pragma unroll
                        for (int m = 1; m < K; ++m) out[q] = ffma2(wt.w[K - 1 - m][q], dc[m][q], out[q]);
                    }
                    if (!kInner && df && kept0 + j >= 0) {
                        float2 f[P];
                        unpack<T, V>(load<T, V>(df + (kept0 + j) * p.channels), f);
#pragma unroll
                        for (int q = 0; q < P; ++q) out[q] = fadd2(out[q], f[q]);
                    }
                    if (kInner || j >= 0) {
                        store<T, V>(dx, out);
                        dx += ys;
                    }
                    else store<T, V>(di + (j + K - 1) * p.channels, out);
                }
            };
            // token t's x and dy from block slot; past `ends` nothing was fetched, and nothing is used
            const int total = count + K - 1;
#pragma unroll
            for (int b = 0; b + 1 < kRing; ++b) {
                rx.fill(b, xj, xs, b * kBlock, ends - 1);
                rg.fill(b, dy, ys, b * kBlock, ends - 1);
                cp_async_commit();
            }
            for (int t = 0, slot = 0; t < total; t += kBlock, slot = next_slot(slot)) {
                cp_async_wait<kRing - 2>();
                Pack<T, V> xin[kBlock], gin[kBlock];
#pragma unroll
                for (int i = 0; i < kBlock; ++i) {
                    xin[i] = rx.at(slot, i);
                    gin[i] = rg.at(slot, i);
                }
                const int free = slot == 0 ? kRing - 1 : slot - 1;
                rx.fill(free, xj, xs, t + (kRing - 1) * kBlock, ends - 1);
                rg.fill(free, dy, ys, t + (kRing - 1) * kBlock, ends - 1);
                cp_async_commit();
                if (t >= K - 1 && t + kBlock <= count) {  // what these complete is the run's, and not in the final state
#pragma unroll
                    for (int i = 0; i < kBlock; ++i) step(xin[i], gin[i], t + i, std::true_type{});
                } else {
#pragma unroll
                    for (int i = 0; i < kBlock; ++i)
                        if (t + i < total) step(xin[i], gin[i], t + i, std::false_type{});
                }
            }
            cp_async_wait<0>();
        }
        zero_rows<T, V>(p, p.dx, c, (int64_t)blockIdx.y * lanes + ri, (int64_t)gridDim.y * lanes);
    }
    // the block's sums: one value of every thread at a time, added over the runs in order
    __syncthreads();  // the rings are no longer read
    float* red = reinterpret_cast<float*>(smem);
#pragma unroll
    for (int k = 0; k <= K; ++k)
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const float2 a = k < K ? dw[k < K ? k : 0][v / 2] : db[v / 2];
            red[threadIdx.x] = v % 2 ? a.y : a.x;
            __syncthreads();
            if (ri == 0 && live) {
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
                                                             int32_t channels, int32_t silu) {
    constexpr int P = kPairs<V>;
    const int64_t item = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (item >= items) return;
    const int s = (int)(item / cgroups), c = (int)(item % cgroups) * V;
    const int slot = index ? index[s] : s;
    float2 out[P];
    if (slot < 0 || slot >= slots) {
#pragma unroll
        for (int q = 0; q < P; ++q) out[q] = make_float2(0.f, 0.f);
        store<T, V>(y + (int64_t)s * channels + c, out);
        return;
    }
    ConvParams p{};
    p.w = w; p.bias = bias;
    Weights<V, K> wt;
    wt.load(p, c);
    const int64_t at = (int64_t)slot * (K - 1) * channels + c;
    float2 win[K][P];
#pragma unroll
    for (int k = 0; k + 1 < K; ++k) unpack<T, V>(load<T, V>(state + at + (int64_t)k * channels), win[k]);
    unpack<T, V>(load<T, V>(x + s * x_stride + c), win[K - 1]);
#pragma unroll
    for (int q = 0; q < P; ++q) {
        const float2 a = wt.at(win, q);
        out[q] = silu ? fmul2(a, sigmoid2(a)) : a;
    }
    store<T, V>(y + (int64_t)s * channels + c, out);
#pragma unroll
    for (int k = 1; k < K; ++k) store<T, V>(state_out + at + (int64_t)(k - 1) * channels, win[k]);
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
// V channels at a time: 8 bytes of them where `wide`, else one.
template <typename T, typename F>
int with_width(bool wide, F&& f) {
    if (wide) return f(std::integral_constant<int, 8 / (int)sizeof(T)>{});
    return f(std::integral_constant<int, 1>{});
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

// Whether every row's start and the channel count are multiples of 8 bytes.
bool conv_wide(const vh_short_conv_args* a, std::initializer_list<const void*> more) {
    const int64_t es = (int64_t)dtype_size(a->dtype);
    bool v = a->channels * es % 8 == 0 && a->x_token_stride * es % 8 == 0 &&
             (a->seq_offsets || a->x_batch_stride * es % 8 == 0);
    for (const void* t : {a->x, a->initial_state}) v = v && (!t || aligned(t, 8));
    for (const void* t : more) v = v && (!t || aligned(t, 8));
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

// A launch: blocks of `cblock` channel groups by runs; gy blocks share the slots.  A run
// is as long as one wave of per_sm blocks an SM needs to cover all tokens (8 at least).
struct Plan {
    int64_t slots;
    int cblock, gx, gy, run;
};
Plan plan(const vh_short_conv_args* a, int width, int per_sm) {
    Plan b;
    const bool packed = a->seq_offsets != nullptr;
    const int cgroups = (a->channels + width - 1) / width;
    b.cblock = std::min(cgroups, 16);  // 16 neighbouring groups fill the memory's lines
    b.gx = (cgroups + b.cblock - 1) / b.cblock;
    const int64_t lanes = kThreads / b.cblock;
    const int64_t fit = std::max<int64_t>(1, (int64_t)per_sm * sm_count() / b.gx);
    const int64_t tokens = packed ? a->length : a->length * a->batch;
    const int64_t want = (tokens + fit * lanes - 1) / (fit * lanes);
    b.run = (int)std::min<int64_t>(std::max<int64_t>((want + 3) / 4 * 4, 8), 1 << 20);
    if (!packed) {  // equal shares of every sequence
        const int64_t runs = slots_per_seq(a->length, b.run);
        b.run = (int)std::max<int64_t>(((a->length + runs - 1) / runs + 3) / 4 * 4, 8);
    }
    b.slots = slot_total(packed, a->length, a->batch, b.run);
    b.gy = (int)std::max<int64_t>(1, std::min<int64_t>((b.slots + lanes - 1) / lanes, 2 * fit));
    return b;
}
// The backward's sums over blocks hold as many rows as the largest of its launches has blocks.
int64_t bwd_rows(const vh_short_conv_args* a) {
    int64_t rows = 0;
    for (int width : {1, 2, 4}) rows = std::max<int64_t>(rows, plan(a, width, kBwdBlocks).gy);
    return rows;
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
    const bool wide = conv_wide(a, {a->y, a->final_state});
    return with_dtype(a->dtype, [&](auto t) {
        using T = decltype(t);
        return with_width<T>(wide, [&](auto width) {
            constexpr int V = decltype(width)::value;
            const Plan b = plan(a, V, kFwdBlocks);
            p.run = b.run;
            return with_taps(a->taps, [&](auto taps) {
                constexpr int K = decltype(taps)::value;
                constexpr size_t smem = sizeof(Pack<T, V>) * kRing * kBlock * kThreads;
                if (!ensure_smem_attr(reinterpret_cast<const void*>(&conv_fwd_kernel<T, V, K>), smem))
                    return fail(VH_E_DEVICE, "vh_short_conv_fwd: cannot reserve %zu bytes of shared memory", smem);
                conv_fwd_kernel<T, V, K><<<dim3(b.gx, b.gy), kThreads, smem, static_cast<cudaStream_t>(stream)>>>(
                    p, b.slots, b.cblock);
                return launch_status("short convolution");
            });
        });
    });
}

extern "C" int64_t vh_short_conv_bwd_workspace_bytes(const vh_short_conv_args* a) {
    if (!a || a->batch <= 0 || a->channels <= 0 || a->length < 0 || a->taps < 2 || a->taps > 8) return 0;
    return bwd_rows(a) * (a->taps + 1) * a->channels * 4;
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
    const bool wide = conv_wide(a, {grad_y, grad_final, grad_x, grad_initial});
    p.dy = grad_y; p.dfinal = grad_final; p.dx = grad_x; p.dinitial = grad_initial;
    p.partial = static_cast<float*>(workspace);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    int blocks = 0;
    const int rc = with_dtype(a->dtype, [&](auto t) {
        using T = decltype(t);
        return with_width<T>(wide, [&](auto width) {
            constexpr int V = decltype(width)::value;
            const Plan b = plan(a, V, kBwdBlocks);
            p.run = b.run;
            blocks = b.gy;
            return with_taps(a->taps, [&](auto taps) {
                constexpr int K = decltype(taps)::value;
                constexpr size_t smem = std::max(sizeof(Pack<T, V>) * 2 * kRing * kBlock, sizeof(float)) * kThreads;
                if (!ensure_smem_attr(reinterpret_cast<const void*>(&conv_bwd_kernel<T, V, K>), smem))
                    return fail(VH_E_DEVICE, "vh_short_conv_bwd: cannot reserve %zu bytes of shared memory", smem);
                conv_bwd_kernel<T, V, K><<<dim3(b.gx, b.gy), kThreads, smem, st>>>(p, b.slots, b.cblock);
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
    const bool wide = conv_wide(&a, {state, (const void*)state_out, (const void*)y});
    return with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        return with_width<T>(wide, [&](auto width) {
            constexpr int V = decltype(width)::value;
            const int cgroups = (channels + V - 1) / V;
            const int64_t items = (int64_t)batch * cgroups;
            const int64_t blocks = (items + kThreads - 1) / kThreads;
            if (blocks > 0x7fffffff) return fail(VH_E_RANGE, "vh_short_conv_step: too many elements");
            return with_taps(taps, [&](auto k) {
                conv_step_kernel<T, V, decltype(k)::value><<<(int)blocks, kThreads, 0, static_cast<cudaStream_t>(stream)>>>(
                    static_cast<const T*>(x), x_batch_stride, weight, bias, static_cast<const T*>(state),
                    static_cast<T*>(state_out), slots_index, slots, static_cast<T*>(y), items, cgroups, channels,
                    activation);
                return launch_status("short convolution step");
            });
        });
    });
}
