// The selective scan's kernel parameters and the per-warp machinery shared by its forward and
// backward kernels.
//
// Layout.  One warp owns a tile of channels of one sequence and walks its tokens.  A thread holds
// a 4 x 4 block of the state, four channels by four states: the warp's lanes are NL = N / 4 state
// lanes times CL = 32 / NL channel lanes, so a warp covers 4 CL channels (32 for N = 16).  A
// token's update needs four values of s and s u (its channels) and four of B and C (its states)
// per thread for sixteen state updates, against 2 + 2 N with one channel per thread; and sums
// over states (y) cross only the NL state lanes, sums over channels (the gradients of B and C)
// only the channel lanes after four are added in the thread.  State lane j holds the states j, j +
// NL, j + 2 NL and j + 3 NL, and a thread's values lie in the order [state][channel], so that the
// packed arithmetic (two channels an instruction) finds its pairs in one 16-byte load.
//
// Tokens go in groups of four.  The 4 x 4 CL elements of a group (tokens by channels) spread
// evenly over the lanes, 16 / NL each: a lane loads its own elements of u, delta and z, applies
// softplus once, and leaves s and s u in shared memory for the whole warp; y's sums over the
// state lanes come back scattered in the same way, so that the lane that holds an element's u
// and z finishes and stores its y.  The next group's loads are issued before a group is computed.
//
// Exponentials.  The decays are N exponentials per element, by far the largest part of the work:
// the special-function unit gives 16 a cycle and SM, one element of 16 states a cycle, when the
// bytes of an element (8 in bf16 with a gate) would allow three.  So a quarter of them, those of
// the states j (the lowest quarter), run on the FMA pipe as a polynomial (exp2_fma2).  It is also
// the more exact one (ex2.approx is off by -2e-8 on average near 0, which a state that remembers a
// thousand tokens multiplies up), and with decay rates that grow with the state's index, as they
// are initialised, it serves the longest memories.
#pragma once

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "abi_util.h"
#include "ssm_common.cuh"

namespace vh {
namespace ssm {

constexpr int kGroup = 4;        // tokens per group
constexpr int kCheckpoint = 32;  // tokens between saved states

template <int NL>
struct Tile {
    static constexpr int N = 4 * NL;          // states
    static constexpr int CL = 32 / NL;        // channel lanes
    static constexpr int CW = 4 * CL;         // channels of a warp
    static constexpr int E = 16 / NL;         // elements of a group per lane
    static constexpr int CE = E < 4 ? E : 4;  // ... as consecutive channels
    static constexpr int TE = E / CE;         // ... of this many tokens
    static constexpr int Q = NL >= 4 ? NL / 4 : 1;  // quads of B and C a lane stages per group
};

struct ScanParams {
    const void *u, *delta, *z, *b, *c;
    Rows ur, dr, zr, br, cr;
    int64_t bg, cg;  // group strides of b and c
    const float *a, *d_skip, *delta_bias, *initial;
    void* y;
    float* final_state;
    float* checkpoints;  // [slot][tile][512]: a warp's states in lane order, see store_lanes
    Seqs seqs;
    int32_t channels, groups, per_group, tiles_per_group, softplus;
    int32_t vec;     // channel loads of CE values are aligned and end with the group's channels
    int32_t vec_bc;  // loads of four states of b and c are aligned
};

// Which elements of a group a lane owns: tokens t0 .. t0 + TE - 1, channels c0 .. c0 + CE - 1 of
// the warp's tile (the layout reduce_scatter leaves over the state lanes).
template <int NL>
struct LaneElems {
    int t0, c0;
    __device__ __forceinline__ explicit LaneElems(int lane) {
        using K = Tile<NL>;
        const int j = lane / K::CL, k = lane % K::CL;
        const int at = j * K::E;  // first of the lane's values in [token][channel] order of its 4 x 4
        t0 = at / 4;
        c0 = 4 * k + at % 4;
    }
};

// V elements as they lie in memory, loaded ahead of their use.  `left`: how many of them exist
// (vec: the pointer is aligned and all do).
template <typename T, int V>
struct alignas(sizeof(T) * V) Pack {
    T e[V];
    __device__ __forceinline__ void load(const T* p, int left, bool vec) {
        if (vec) {
            *this = *reinterpret_cast<const Pack*>(p);
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) e[i] = i < left ? p[i] : from_f<T>(0.f);
        }
    }
    __device__ __forceinline__ void get(float (&v)[V]) const {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = to_f(e[i]);
    }
};

__device__ __forceinline__ void lds4(const float* p, float (&v)[4]) {
    const float4 q = *reinterpret_cast<const float4*>(p);
    v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
}
__device__ __forceinline__ void lds22(const float* p, float2 (&v)[2]) {
    const float4 q = *reinterpret_cast<const float4*>(p);
    v[0] = make_float2(q.x, q.y); v[1] = make_float2(q.z, q.w);
}
// four values that each fill both halves of a pair
__device__ __forceinline__ void lds_dup4(const float* p, float2 (&v)[4]) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    v[0] = make_float2(a.x, a.y); v[1] = make_float2(a.z, a.w);
    v[2] = make_float2(b.x, b.y); v[3] = make_float2(b.z, b.w);
}
template <int CE>
__device__ __forceinline__ void sts_v(float* p, const float (&v)[CE]) {
    if constexpr (CE == 4) *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    else if constexpr (CE == 2) *reinterpret_cast<float2*>(p) = make_float2(v[0], v[1]);
    else p[0] = v[0];
}
template <int CE>
__device__ __forceinline__ void lds_v(const float* p, float (&v)[CE]) {
    if constexpr (CE == 4) lds4(p, v);
    else if constexpr (CE == 2) { const float2 q = *reinterpret_cast<const float2*>(p); v[0] = q.x; v[1] = q.y; }
    else v[0] = p[0];
}

// A thread's 4 x 4 block of a [channels][N] matrix in the order [state][channel]; rows at or
// past `end` read as 0.
template <int NL>
__device__ __forceinline__ void load_block(const float* m, int c0, int end, int j, float (&v)[16]) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) v[4 * i + c] = c0 + c < end ? m[(int64_t)(c0 + c) * 4 * NL + j + NL * i] : 0.f;
}
template <int NL>
__device__ __forceinline__ void store_block(float* m, int c0, int end, int j, const float (&v)[16]) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c)
            if (c0 + c < end) m[(int64_t)(c0 + c) * 4 * NL + j + NL * i] = v[4 * i + c];
}

// A warp's 512 states in lane order: element (4 i + lane-major) -> float4 i of lane l at (32 i + l) * 4.
__device__ __forceinline__ void store_lanes(float* p, int lane, const float (&v)[16]) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
        reinterpret_cast<float4*>(p)[32 * i + lane] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
}
__device__ __forceinline__ void load_lanes(const float* p, int lane, float (&v)[16]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float4 q = reinterpret_cast<const float4*>(p)[32 * i + lane];
        v[4 * i] = q.x; v[4 * i + 1] = q.y; v[4 * i + 2] = q.z; v[4 * i + 3] = q.w;
    }
}

// The decays exp2(s a2) of one token: pairs of channels by four states.
// kHardware: all on the special-function unit.  kMixed: the first state's on the FMA pipe, for
// |s a2| <= 126 there; kChecked: the same values without that condition (the warp's choice between
// the two must not show in a channel's bits).
enum Decay { kHardware, kMixed, kChecked };
template <int MODE>
__device__ __forceinline__ void decays(const float2 (&s)[2], const float2 (&a2)[8], float2 (&e)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int p = 0; p < 2; ++p) {
            const float2 a = a2[2 * i + p];
            if (i > 0 || MODE == kHardware) e[2 * i + p] = ex2_2(fmul2(s[p], a));
            else if (MODE == kMixed) e[2 * i + p] = exp2_fma2(s[p], a);
            else e[2 * i + p] = make_float2(exp2_fma(s[p].x, a.x), exp2_fma(s[p].y, a.y));
        }
}

// ---- thread-block clusters -------------------------------------------------------------------
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
// p of this CTA's shared memory, in the CTA of `rank`
__device__ __forceinline__ float ld_cluster(const float* p, uint32_t rank) {
    const uint32_t here = static_cast<uint32_t>(__cvta_generic_to_shared(p));
    uint32_t there;
    float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(here), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(there) : "memory");
    return v;
}

// Shared memory of a group of tokens.  A row of B or C holds every value twice, for the packed
// arithmetic; its stride keeps the rows' stores in different banks.
template <int NL>
struct Stage {
    using K = Tile<NL>;
    static constexpr int kRow = 2 * K::N + 8;
    float step[kGroup * K::CW], su[kGroup * K::CW], bc[kGroup * 2 * kRow];
    // the four values of state lane j at token r
    __device__ __forceinline__ const float* b(int r, int j) const { return bc + 2 * r * kRow + 8 * j; }
    __device__ __forceinline__ const float* c(int r, int j) const { return bc + (2 * r + 1) * kRow + 8 * j; }
};

// Larger of the two, NaN if either is.
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
// ... over the warp, of values that are not negative
__device__ __forceinline__ float warp_max_nan(float v) {
    return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(v)));
}

// A warp's place in its chain: for each sequence the address of the lane's elements in the group
// at hand, moved from group to group.  A group that the run of tokens ends in reads its last
// token again in place of the missing ones, and channels past the tile's group read the last
// ones; both are then staged with the step 0 and s u = 0, which leave every state as it is and
// add nothing to a sum.
template <typename T, int NL>
struct Chain {
    using K = Tile<NL>;
    static constexpr int CE = K::CE, TE = K::TE, Q = K::Q;
    static constexpr int kQuads = kGroup * 2 * NL;
    const T *u, *dl, *z, *bc[Q];
    int64_t us, ds, zs, bcs;  // bcs: of the tensor (B or C) that the lane reads
    int cbase, cend, ec, lane, own_t, own_c, left;
    bool vec, vec_bc, softplus, gated;
    float bias[CE];

    __device__ __forceinline__ Chain(const ScanParams& p, const Seq& seq, int s, int tile, int lane_) {
        const LaneElems<NL> own(lane_);
        const int group = tile / p.tiles_per_group;
        lane = lane_; own_t = own.t0; own_c = own.c0;
        cbase = group * p.per_group + (tile % p.tiles_per_group) * K::CW;
        cend = (group + 1) * p.per_group;
        ec = cbase + own_c;
        left = cend - ec;
        vec = p.vec; vec_bc = p.vec_bc; softplus = p.softplus; gated = p.z != nullptr;
        const int at = left > 0 ? ec : cend - (vec ? CE : 1);
        us = row_step(p.seqs, p.ur); ds = row_step(p.seqs, p.dr); zs = row_step(p.seqs, p.zr);
        u = static_cast<const T*>(p.u) + first_row(p.seqs, seq, s, p.ur) + at + own_t * us;
        dl = static_cast<const T*>(p.delta) + first_row(p.seqs, seq, s, p.dr) + at + own_t * ds;
        z = gated ? static_cast<const T*>(p.z) + first_row(p.seqs, seq, s, p.zr) + at + own_t * zs : nullptr;
        // quad q of a group: token q / (2 NL), of it B's or C's states 4 (q % NL) on
        const bool is_b = lane % (2 * NL) < NL;  // 2 NL divides 32: all of a lane's quads are of one tensor
        bcs = row_step(p.seqs, is_b ? p.br : p.cr);
        const T* base = is_b ? static_cast<const T*>(p.b) + first_row(p.seqs, seq, s, p.br) + group * p.bg
                             : static_cast<const T*>(p.c) + first_row(p.seqs, seq, s, p.cr) + group * p.cg;
#pragma unroll
        for (int i = 0; i < Q; ++i) {
            const int q = min(lane + 32 * i, kQuads - 1);
            bc[i] = base + (q / (2 * NL)) * bcs + 4 * (q % NL);
        }
#pragma unroll
        for (int i = 0; i < CE; ++i) bias[i] = p.delta_bias && i < left ? p.delta_bias[ec + i] : 0.f;
    }
    // n tokens on (or back)
    __device__ __forceinline__ void move(int64_t n) {
        u += n * us;
        dl += n * ds;
        if (gated) z += n * zs;
#pragma unroll
        for (int i = 0; i < Q; ++i) bc[i] += n * bcs;
    }

    struct Raw {
        Pack<T, CE> u[TE], d[TE], z[TE];
        Pack<T, 4> bc[Q];
    };
    // The loads of the group at hand, of which the first `count` (or more) tokens exist.
    template <bool GATE>
    __device__ __forceinline__ void load(Raw& r, int64_t count) const {
        if (count >= kGroup) {
#pragma unroll
            for (int e = 0; e < TE; ++e) {
                r.u[e].load(u + e * us, left, vec);
                r.d[e].load(dl + e * ds, left, vec);
                if (GATE && gated) r.z[e].load(z + e * zs, left, vec);
            }
#pragma unroll
            for (int i = 0; i < Q; ++i) r.bc[i].load(bc[i], 4, vec_bc);
        } else {
            const int last = (int)count - 1;
#pragma unroll
            for (int e = 0; e < TE; ++e) {
                const int64_t by = min(e, last - own_t);
                r.u[e].load(u + by * us, left, vec);
                r.d[e].load(dl + by * ds, left, vec);
                if (GATE && gated) r.z[e].load(z + by * zs, left, vec);
            }
#pragma unroll
            for (int i = 0; i < Q; ++i) {
                const int t = min(lane + 32 * i, kQuads - 1) / (2 * NL);
                r.bc[i].load(bc[i] + min(0, last - t) * bcs, 4, vec_bc);
            }
        }
    }
    // s, s u, B and C of a loaded group into shared memory.  SUM: adds s to sum.  Returns the
    // largest |s| of the warp.
    template <bool SUM>
    __device__ __forceinline__ float stage(const Raw& r, int64_t count, Stage<NL>& st, float (&sum)[CE]) const {
        float top = 0.f;
#pragma unroll
        for (int e = 0; e < TE; ++e) {
            float uv[CE], sv[CE];
            r.u[e].get(uv);
            r.d[e].get(sv);
            const bool live = own_t + e < count;
#pragma unroll
            for (int i = 0; i < CE; ++i) sv[i] += bias[i];
            if (softplus) softplus_n<CE>(sv);
#pragma unroll
            for (int i = 0; i < CE; ++i) {
                const bool ok = live && (vec ? left > 0 : i < left);
                sv[i] = ok ? sv[i] : 0.f;
                uv[i] = ok ? sv[i] * uv[i] : 0.f;
                if (SUM) sum[i] += sv[i];
                top = max_nan(top, fabsf(sv[i]));
            }
            sts_v<CE>(st.step + (own_t + e) * K::CW + own_c, sv);
            sts_v<CE>(st.su + (own_t + e) * K::CW + own_c, uv);
        }
#pragma unroll
        for (int i = 0; i < Q; ++i) {
            const int at = lane + 32 * i;
            if (kQuads >= 32 || at < kQuads) {
                const int n = 4 * (at % NL);
                float* row = st.bc + (at / NL) * Stage<NL>::kRow;
                float v[4];
                r.bc[i].get(v);
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    *reinterpret_cast<float2*>(row + 2 * (((n + k) % NL) * 4 + (n + k) / NL)) = splat2(v[k]);
            }
        }
        return warp_max_nan(top);
    }
};

__device__ __forceinline__ void pair_up(const float (&v)[16], float2 (&p)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = make_float2(v[2 * i], v[2 * i + 1]);
}
__device__ __forceinline__ void pair_down(const float2 (&p)[8], float (&v)[16]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) { v[2 * i] = p[i].x; v[2 * i + 1] = p[i].y; }
}

// log2(e) A of the thread's block; returns the warp's largest of the states whose decays run on
// the FMA pipe (see decays).
template <int NL>
__device__ __forceinline__ float load_rates(const ScanParams& p, int c0, int cend, int j, float (&v)[16]) {
    load_block<NL>(p.a, c0, cend, j, v);
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = to_log2(v[i]);
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) top = max_nan(top, fabsf(v[i]));
    return warp_max_nan(top);
}

// ---- one chain over many warps ------------------------------------------------------------------
// The W warps of a CTA, and the CTAs of a cluster, take consecutive segments of one chain.  A
// segment maps the state that enters it to exp(a sum s) h + its own state, so what enters every
// segment follows from the own states and the step sums.  REV: entering from the right (the
// gradient's way).
template <int NL, int W>
struct SplitSmem {
    float sigma[W][Tile<NL>::CW];       // a segment's sum of steps per channel
    float a2[512];
    float total[512], total_sigma[Tile<NL>::CW];  // of all the CTA's segments
};

// The channel of the tile and the state of element x of the lane order.
template <int NL>
__device__ __forceinline__ void element(int x, int& c, int& n) {
    const int l = (x / 4) % 32;
    c = 4 * (l % Tile<NL>::CL) + x % 4;
    n = l / Tile<NL>::CL + NL * (x / 128);
}

// state(w): 512 floats of warp w, in: its segment's own state, out: what enters it.
// first: what enters the chain, [channels][N] of the sequence, or null.  Ends with a barrier of
// the CTA; with a cluster it leaves one cluster barrier to be waited for before the CTA ends
// (its totals are read until then).
template <int NL, int W, bool REV, typename State>
__device__ __forceinline__ void enter_segments(SplitSmem<NL, W>& sp, State&& state, const float* first, int cbase, int cend, int cluster,
                                               int rank) {
    constexpr int PER = 512 / (32 * W);
    constexpr int N = 4 * NL;
    __syncthreads();
    float dec[PER][W], add[PER][W], carry[PER];
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        const int x = threadIdx.x + 32 * W * k;
        int c, n;
        element<NL>(x, c, n);
        float run = 0.f, sig = 0.f;
#pragma unroll
        for (int i = 0; i < W; ++i) {
            const int w = REV ? W - 1 - i : i;
            const float sw = sp.sigma[w][c];
            dec[k][i] = exp2_fma(sw, sp.a2[x]);
            add[k][i] = state(w)[x];
            run = fmaf(dec[k][i], run, add[k][i]);
            sig += sw;
        }
        carry[k] = first && cbase + c < cend ? first[(int64_t)(cbase + c) * N + n] : 0.f;
        if (cluster > 1) {
            sp.total[x] = run;
            if (n == 0) sp.total_sigma[c] = sig;
        }
    }
    if (cluster > 1) {
        cluster_arrive();
        cluster_wait();
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            const int x = threadIdx.x + 32 * W * k;
            int c, n;
            element<NL>(x, c, n);
            const int steps = REV ? cluster - 1 - rank : rank;
            for (int i = 0; i < steps; ++i) {
                const int r = REV ? cluster - 1 - i : i;
                carry[k] = fmaf(exp2_fma(ld_cluster(&sp.total_sigma[c], r), sp.a2[x]), carry[k], ld_cluster(&sp.total[x], r));
            }
        }
        cluster_arrive();
    }
#pragma unroll
    for (int k = 0; k < PER; ++k)
#pragma unroll
        for (int i = 0; i < W; ++i) {
            state(REV ? W - 1 - i : i)[threadIdx.x + 32 * W * k] = carry[k];
            carry[k] = fmaf(dec[k][i], carry[k], add[k][i]);
        }
    __syncthreads();
}

// Sums v (per element channel) over the lanes that hold the same channels at other tokens, and
// leaves the tile's row of them at out.
template <int NL>
__device__ __forceinline__ void sum_tokens(float (&v)[Tile<NL>::CE], int lane, int own_c, float* out) {
    using K = Tile<NL>;
    constexpr int kLanesPerToken = NL <= 4 ? 1 : NL / 4;
#pragma unroll
    for (int o = 16; o >= K::CL * kLanesPerToken; o >>= 1)
#pragma unroll
        for (int i = 0; i < K::CE; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
    if (lane < K::CL * kLanesPerToken)
#pragma unroll
        for (int i = 0; i < K::CE; ++i) out[own_c + i] = v[i];
}

// Validates the arguments shared by the entry points; 0 or a status.  `one_token`: the step.
int check_scan_args(const char* what, const vh_ssm_scan_args* a, bool one_token);
void fill_scan_params(const vh_ssm_scan_args* a, ScanParams* p);
int64_t checkpoint_floats(const vh_ssm_scan_args* a);

// The largest cluster of split-kernel CTAs with which all `chains` run at once while a segment
// keeps `least` tokens (1: no cluster).  The occupancy of each cluster size is asked once per
// device and kept in known[device][size] (+ 1).
template <typename Kernel>
int pick_cluster(Kernel kernel, std::atomic<int> (&known)[64][9], int threads, size_t smem, int64_t chains,
                 int64_t length, int least) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 1;
    int best = 1;
    for (int size = 2; size <= 8; ++size) {
        if (chains * size > sm_count() || (int64_t)least * (threads / 32) * size > length) break;
        int n = known[dev][size].load(std::memory_order_relaxed);
        if (n == 0) {
            cudaLaunchAttribute at[1];
            at[0].id = cudaLaunchAttributeClusterDimension;
            at[0].val.clusterDim = {(unsigned)size, 1, 1};
            cudaLaunchConfig_t cfg{};
            cfg.gridDim = dim3(size);
            cfg.blockDim = dim3(threads);
            cfg.dynamicSmemBytes = smem;
            cfg.attrs = at;
            cfg.numAttrs = 1;
            int got = 0;
            if (cudaOccupancyMaxActiveClusters(&got, kernel, &cfg) != cudaSuccess) {
                cudaGetLastError();
                got = 0;
            }
            n = got + 1;
            known[dev][size].store(n, std::memory_order_relaxed);
        }
        if (n - 1 >= chains) best = size;
    }
    return best;
}

// Launches `kernel` with clusters of `cluster` CTAs.
template <typename... P, typename... A>
int launch_cluster(const char* what, void (*kernel)(P...), int64_t blocks, int threads, size_t smem, int cluster,
                   cudaStream_t st, A... args) {
    if (blocks > 0x7fffffff) return fail(VH_E_RANGE, "%s: too many channel tiles", what);
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim = {(unsigned)cluster, 1, 1};
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return fail((int)e, "%s: launch failed: %s", what, cudaGetErrorString(e));
    }
    return launch_status(what);
}

template <typename F>
int with_dtype(int dtype, F&& f) {
    if (dtype == VH_F32) return f(float{});
    if (dtype == VH_BF16) return f(__nv_bfloat16{});
    return f(__half{});
}
template <typename F>
int with_states(int n, F&& f) {
    switch (n) {
        case 4: return f(std::integral_constant<int, 1>{});
        case 8: return f(std::integral_constant<int, 2>{});
        case 16: return f(std::integral_constant<int, 4>{});
        case 32: return f(std::integral_constant<int, 8>{});
        default: return f(std::integral_constant<int, 16>{});
    }
}

}  // namespace ssm
}  // namespace vh
