// The selective scan's kernel parameters and the per-warp staging shared by its forward and
// backward kernels.
//
// One warp owns a tile of channels of one sequence and walks its tokens.  A thread holds a 4 x 4
// block of the state, four channels by four states: the warp's lanes are NL = N / 4 state lanes
// times 32 / NL channel lanes, so a warp covers 128 / NL channels (32 for N = 16).  A token's
// update needs four values of s and s u (its channels) and four of B and C (its states) per
// thread for sixteen state updates, against 2 + 2 N with one channel per thread; and sums over
// states (y) cross only the NL state lanes, sums over channels (the gradients of B and C) only
// the channel lanes after four are added in the thread.
//
// Tokens go in groups of four.  The 4 x 128 / NL elements of a group (tokens by channels) spread
// evenly over the lanes, 16 / NL each: a lane loads its own elements of u, delta and z, applies
// softplus once, and leaves s and s u in shared memory for the whole warp; y's sums over the
// state lanes come back scattered in the same way, so that the lane that holds an element's u
// and z finishes and stores its y.
#pragma once

#include "abi_util.h"
#include "ssm_common.cuh"

namespace vh {
namespace ssm {

constexpr int kGroup = 4;        // tokens per group
constexpr int kCheckpoint = 32;  // tokens between saved states
constexpr int kWarps = 4;        // warps per CTA: neighbouring channel tiles of one sequence

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
    float* checkpoints;
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

// Stages B and C of tokens [0, cnt) of a group into [token][2][N] (B, then C), zeros past cnt.
template <int NL, typename T>
__device__ __forceinline__ void stage_bc(const T* b, const T* c, int64_t bs, int64_t cs, int cnt, bool vec, int lane,
                                         float* sbc) {
    using K = Tile<NL>;
    constexpr int kQuads = kGroup * 2 * NL;
#pragma unroll
    for (int i = 0; i < K::Q; ++i) {
        const int q = lane + 32 * i;
        if (q < kQuads) {
            const int t = q / (2 * NL), r = q % (2 * NL), n = 4 * (r % NL);
            const T* p = (r < NL ? b + t * bs : c + t * cs) + n;
            float v[4] = {0.f, 0.f, 0.f, 0.f};
            if (t < cnt) load_v<4>(p, 0, 4, vec, v);
            *reinterpret_cast<float4*>(sbc + 4 * q) = make_float4(v[0], v[1], v[2], v[3]);
        }
    }
}

__device__ __forceinline__ void lds4(const float* p, float (&v)[4]) {
    const float4 q = *reinterpret_cast<const float4*>(p);
    v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
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

// A thread's 4 x 4 block of a [channels][N] matrix (row c0 + i, columns n0 ..): 0 past `end`.
template <int N>
__device__ __forceinline__ void load_block(const float* m, int c0, int end, int n0, float (&v)[16]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float4 q = make_float4(0.f, 0.f, 0.f, 0.f);
        if (c0 + i < end) q = *reinterpret_cast<const float4*>(m + (int64_t)(c0 + i) * N + n0);
        v[4 * i] = q.x; v[4 * i + 1] = q.y; v[4 * i + 2] = q.z; v[4 * i + 3] = q.w;
    }
}
template <int N>
__device__ __forceinline__ void store_block(float* m, int c0, int end, int n0, const float (&v)[16]) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (c0 + i < end)
            *reinterpret_cast<float4*>(m + (int64_t)(c0 + i) * N + n0) =
                make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
}

// Validates the arguments shared by the entry points; 0 or a status.  `one_token`: the step.
int check_scan_args(const char* what, const vh_ssm_scan_args* a, bool one_token);
void fill_scan_params(const vh_ssm_scan_args* a, ScanParams* p);

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
