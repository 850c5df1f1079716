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
// softplus once, and leaves s and s u in shared memory for the whole warp.  y's sums over the state
// lanes go through shared memory too: the lane that holds an element's u and z adds its parts, and
// finishes and stores its y.  Groups are fetched ahead, two in the forward and one in the backward.
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
// the warp's tile: of the 4 x 4 (tokens by channels) of a channel lane, state lane j has the j-th part.
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

__device__ __forceinline__ void lds4(const float* p, float (&v)[4]) {
    const float4 q = *reinterpret_cast<const float4*>(p);
    v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
}
__device__ __forceinline__ void lds22(const float* p, float2 (&v)[2]) {
    const float4 q = *reinterpret_cast<const float4*>(p);
    v[0] = make_float2(q.x, q.y); v[1] = make_float2(q.z, q.w);
}
// four values, each for both halves of a pair
__device__ __forceinline__ void lds_dup4(const float* p, float2 (&v)[4]) {
    const float4 a = *reinterpret_cast<const float4*>(p);
    v[0] = splat2(a.x); v[1] = splat2(a.y); v[2] = splat2(a.z); v[3] = splat2(a.w);
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
__device__ __forceinline__ void clear_lanes(float* p, int lane) {
#pragma unroll
    for (int i = 0; i < 4; ++i) reinterpret_cast<float4*>(p)[32 * i + lane] = make_float4(0.f, 0.f, 0.f, 0.f);
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
// LAST: the polynomials behind the others, whose latency is the longest (the forward is 2 % faster
// that way, the backward 7 % slower).
enum Decay { kHardware, kMixed, kChecked };
template <int MODE, bool LAST = false>
__device__ __forceinline__ void decays(const float2 (&s)[2], const float2 (&a2)[8], float2 (&e)[8]) {
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int p = 0; p < 2; ++p) {
            const int i = LAST ? 3 - k : k;
            const float2 a = a2[2 * i + p];
            if (i > 0 || MODE == kHardware) e[2 * i + p] = ex2_2(fmul2(s[p], a));
            else if (MODE == kMixed) e[2 * i + p] = exp2_fma2(s[p], a);
            else e[2 * i + p] = make_float2(exp2_fma(s[p].x, a.x), exp2_fma(s[p].y, a.y));
        }
}

// Shared memory of a group of tokens.  A row of B or C lies as [state lane][4 states]; its stride
// keeps the rows' stores in different banks.
template <int NL>
struct Stage {
    using K = Tile<NL>;
    static constexpr int kRow = K::N + 4;
    float step[kGroup * K::CW], su[kGroup * K::CW], bc[kGroup * 2 * kRow];
    // the four values of state lane j at token r
    __device__ __forceinline__ const float* b(int r, int j) const { return bc + 2 * r * kRow + 4 * j; }
    __device__ __forceinline__ const float* c(int r, int j) const { return bc + (2 * r + 1) * kRow + 4 * j; }
};

// The largest over the warp, of values that are not negative
__device__ __forceinline__ float warp_max_nan(float v) {
    return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(v)));
}

// Sums over the state lanes through shared memory: every lane leaves its four channels of token r,
// and the lane that owns an element adds the NL parts.  (Four stores and loads a group against 12
// shuffles, each with two selections and an addition.)  rows: 512 floats.
template <int NL>
__device__ __forceinline__ void put_part(float* rows, int j, int ct, const float2 (&v)[2]) {
    *reinterpret_cast<float4*>(rows + j * Tile<NL>::CW + ct) = make_float4(v[0].x, v[0].y, v[1].x, v[1].y);
}
// ... of one token: NL rows of CW
template <int NL>
__device__ __forceinline__ void sum_parts(const float* rows, int own_c, float2 (&v)[kPairs<Tile<NL>::CE>]) {
    using K = Tile<NL>;
    float f[K::CE];
    lds_v<K::CE>(rows + own_c, f);
    to_pairs<K::CE>(f, v);
#pragma unroll
    for (int k = 1; k < NL; ++k) {
        float2 w[kPairs<K::CE>];
        lds_v<K::CE>(rows + k * K::CW + own_c, f);
        to_pairs<K::CE>(f, w);
#pragma unroll
        for (int i = 0; i < kPairs<K::CE>; ++i) v[i] = fadd2(v[i], w[i]);
    }
}

// A warp's place in its chain: for each sequence the address of the lane's elements in the group
// at hand, moved from group to group.  A group that the run of tokens ends in reads its last
// token again in place of the missing ones, and channels past the tile's group read the last
// ones; both are then staged with the step 0 and s u = 0 (and missing tokens with B = C = 0), which
// leave every state as it is and add nothing to a sum.
template <typename T, int NL>
struct Chain {
    using K = Tile<NL>;
    static constexpr int CE = K::CE, TE = K::TE, Q = K::Q;
    static constexpr int kQuads = kGroup * 2 * NL;
    const T *u, *dl, *z, *bc[Q];
    int64_t us, ds, zs, bcs;  // bcs: of the tensor (B or C) that the lane reads
    int64_t ug, dg, zg, bcg;  // of a group
    int cbase, cend, ec, lane, own_t, own_c, left;
    bool vec, vec_bc, softplus, gated, whole;  // whole: every channel of the tile exists
    float2 bias[kPairs<CE>];

    __device__ __forceinline__ Chain(const ScanParams& p, const Seq& seq, int s, int tile, int lane_) {
        const LaneElems<NL> own(lane_);
        const int group = tile / p.tiles_per_group;
        lane = lane_; own_t = own.t0; own_c = own.c0;
        cbase = group * p.per_group + (tile % p.tiles_per_group) * K::CW;
        cend = (group + 1) * p.per_group;
        ec = cbase + own_c;
        left = cend - ec;
        vec = p.vec; vec_bc = p.vec_bc; softplus = p.softplus; gated = p.z != nullptr;
        whole = cbase + K::CW <= cend;
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
        load_params(p.delta_bias, bias);
        ug = kGroup * us; dg = kGroup * ds; zg = kGroup * zs; bcg = kGroup * bcs;
    }
    // one fp32 value per element channel; 0 for a null pointer and past the end
    __device__ __forceinline__ void load_params(const float* src, float2 (&v)[kPairs<CE>]) const {
        float f[CE];
#pragma unroll
        for (int i = 0; i < CE; ++i) f[i] = src && i < left ? src[ec + i] : 0.f;
        to_pairs<CE>(f, v);
    }
    // a group on
    __device__ __forceinline__ void advance() {
        u += ug;
        dl += dg;
        if (gated) z += zg;
#pragma unroll
        for (int i = 0; i < Q; ++i) bc[i] += bcg;
    }
    // n tokens on (or back)
    __device__ __forceinline__ void move(int64_t n) {
        u += n * us;
        dl += n * ds;
        if (gated) z += n * zs;
#pragma unroll
        for (int i = 0; i < Q; ++i) bc[i] += n * bcs;
    }

    // A group's values as loaded; every lane reads back only what it fetched.
    struct Raw {
        Pack<T, CE> u[TE][32], d[TE][32], z[TE][32];
        Pack<T, 4> bc[Q][32];
    };
    // Fetches the group at hand, of which the first `count` (or more) tokens exist.
    template <bool GATE>
    __device__ __forceinline__ void load(Raw& r, int count) const {
        if (count >= kGroup) {
#pragma unroll
            for (int e = 0; e < TE; ++e) {
                fetch(&r.u[e][lane], u + e * us, left, vec);
                fetch(&r.d[e][lane], dl + e * ds, left, vec);
                if (GATE && gated) fetch(&r.z[e][lane], z + e * zs, left, vec);
            }
#pragma unroll
            for (int i = 0; i < Q; ++i) fetch(&r.bc[i][lane], bc[i], 4, vec_bc);
            return;
        }
        const int last = count - 1;
#pragma unroll
        for (int e = 0; e < TE; ++e) {
            const int64_t by = min(e, last - own_t);
            fetch(&r.u[e][lane], u + by * us, left, vec);
            fetch(&r.d[e][lane], dl + by * ds, left, vec);
            if (GATE && gated) fetch(&r.z[e][lane], z + by * zs, left, vec);
        }
#pragma unroll
        for (int i = 0; i < Q; ++i) {
            const int t = min(lane + 32 * i, kQuads - 1) / (2 * NL);
            fetch(&r.bc[i][lane], bc[i] + min(0, last - t) * bcs, 4, vec_bc);
        }
    }
    // Zeros in place of values that do not exist: tokens from `count` on, channels past the end.
    __device__ __forceinline__ void keep_real(int e, int count, float2 (&v)[kPairs<CE>]) const {
        if (whole && count >= kGroup) return;  // the same for the whole warp
        const bool live = own_t + e < count;
#pragma unroll
        for (int i = 0; i < kPairs<CE>; ++i) {
            v[i].x = live && 2 * i < left ? v[i].x : 0.f;
            v[i].y = live && 2 * i + 1 < left ? v[i].y : 0.f;
        }
    }
    // s, s u, B and C of a loaded group into shared memory.  SUM: adds s to sum.  TOP: returns
    // whether every |s| of the warp is at most `most` (false with a NaN among them).
    template <bool SUM, bool TOP>
    __device__ __forceinline__ bool stage(const Raw& r, int count, Stage<NL>& st, float2 (&sum)[kPairs<CE>],
                                          float most = 0.f) const {
        constexpr int P = kPairs<CE>;
        float top = 0.f;
#pragma unroll
        for (int e = 0; e < TE; ++e) {
            float2 u2[P], s2[P];
            unpack<T, CE>(r.u[e][lane], u2);
            unpack<T, CE>(r.d[e][lane], s2);
#pragma unroll
            for (int i = 0; i < P; ++i) {
                s2[i] = fadd2(s2[i], bias[i]);
                if (softplus) s2[i] = softplus2(s2[i]);
                u2[i] = fmul2(u2[i], s2[i]);
            }
            keep_real(e, count, s2);
            keep_real(e, count, u2);
#pragma unroll
            for (int i = 0; i < P; ++i) {
                if (SUM) sum[i] = fadd2(sum[i], s2[i]);
                if (TOP) top = max_nan(top, max_nan(fabsf(s2[i].x), fabsf(s2[i].y)));
            }
            float f[CE];
            from_pairs<CE>(s2, f);
            sts_v<CE>(st.step + (own_t + e) * K::CW + own_c, f);
            from_pairs<CE>(u2, f);
            sts_v<CE>(st.su + (own_t + e) * K::CW + own_c, f);
        }
#pragma unroll
        for (int i = 0; i < Q; ++i) {
            const int at = lane + 32 * i;
            if (kQuads >= 32 || at < kQuads) {
                const int n = 4 * (at % NL);
                float* row = st.bc + (at / NL) * Stage<NL>::kRow;
                float v[4];
                r.bc[i][lane].get(v);
                if (count < kGroup && at / (2 * NL) >= count)  // 0 times an infinite value is no 0
                    v[0] = v[1] = v[2] = v[3] = 0.f;
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    row[((n + k) % NL) * 4 + (n + k) / NL] = v[k];
            }
        }
        return TOP && __all_sync(0xffffffffu, top <= most);
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

// log2(e) A of the thread's block; returns the warp's largest |.| of the states whose decays run on
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

// The largest |s| that kMixed takes with such a rate (none for NaN; an infinite one never).
__device__ __forceinline__ float mixed_limit(float top) { return top < 1e-30f ? 3e38f : 126.f / top; }

// ---- a chain in segments ----------------------------------------------------------------------
// With few chains, consecutive segments of `size` tokens of a chain go to warps of their own.  A
// segment maps the state that enters it to exp(a sum s) h + its own state (what leaves it when
// nothing enters), so a first kernel finds every segment's own state and sum of steps, a second one
// what enters each segment, and a third one runs the segments.  The gradient goes through the
// same, from the right.  Segment k of sequence s is slot slot_base(s) + k; a slot without tokens
// maps every state to itself.
struct Segments {
    float* state;  // [slot][tile][512]: own states, then what enters, in lane order; null: whole chains
    float* sigma;  // [slot][tile][CW]: sums of steps
    int64_t slots;
    int32_t size;
};

// The channel of the tile and the state of element x of the lane order.
template <int NL>
__device__ __forceinline__ void element(int x, int& c, int& n) {
    const int l = (x / 4) % 32;
    c = 4 * (l % Tile<NL>::CL) + x % 4;
    n = l / Tile<NL>::CL + NL * (x / 128);
}

// What a warp works on: tokens t0 .. t1 - 1 of a chain.
struct Unit {
    Seq seq;
    int64_t slot, t0, t1;
    int s, tile;
};
// Unit `item` of slots (or sequences) x tiles; false when its slot belongs to no sequence.
__device__ __forceinline__ bool unit_at(const ScanParams& p, const Segments& g, int64_t item, Unit& u) {
    const int tiles = p.groups * p.tiles_per_group;
    u.slot = item / tiles;
    u.tile = (int)(item % tiles);
    if (!g.state) {
        u.s = (int)u.slot;
        u.seq = seq_at(p.seqs, u.s);
        u.t0 = 0;
        u.t1 = u.seq.len;
        return true;
    }
    u.s = seq_of_slot(p.seqs, u.slot, g.size);
    u.seq = seq_at(p.seqs, u.s);
    const int64_t k = u.slot - slot_base(p.seqs, u.s, u.seq.row, g.size);
    u.t0 = min(u.seq.len, k * g.size);
    u.t1 = min(u.seq.len, u.t0 + g.size);
    return k == 0 || (k > 0 && u.t0 < u.t1);
}

// Programmatic dependent launch: the next kernel of the stream may start now / wait here for the
// previous one's results.
__device__ __forceinline__ void launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// Sums v (per element channel) over the lanes that hold the same channels at other tokens, and
// leaves the tile's row of them at out.
template <int NL>
__device__ __forceinline__ void sum_tokens(const float2 (&p)[kPairs<Tile<NL>::CE>], int lane, int own_c, float* out) {
    using K = Tile<NL>;
    constexpr int kLanesPerToken = NL <= 4 ? 1 : NL / 4;
    float v[K::CE];
    from_pairs<K::CE>(p, v);
#pragma unroll
    for (int o = 16; o >= K::CL * kLanesPerToken; o >>= 1)
#pragma unroll
        for (int i = 0; i < K::CE; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
    if (lane < K::CL * kLanesPerToken)
#pragma unroll
        for (int i = 0; i < K::CE; ++i) out[own_c + i] = v[i];
}

// Validates the arguments shared by the entry points; 0 or a status.  `one_token`: the step.
// The sizes alone are checked by the first, for queries that come before there are pointers.
int check_scan_sizes(const char* what, const vh_ssm_scan_args* a, bool one_token);
int check_scan_args(const char* what, const vh_ssm_scan_args* a, bool one_token);
void fill_scan_params(const vh_ssm_scan_args* a, ScanParams* p);
int64_t checkpoint_floats(const vh_ssm_scan_args* a);
int64_t tile_count(const vh_ssm_scan_args* a);

// The segment size that gives `warps` warps a segment each (0: whole chains, when there are
// `enough` of them or they are short): a multiple of `step` tokens.
int segment_size(const vh_ssm_scan_args* a, int64_t enough, int64_t warps, int step);
// Bytes of the segments' states and sums (0 without segments), and their places in a workspace.
int64_t segment_bytes(const vh_ssm_scan_args* a, int size);
void place_segments(const vh_ssm_scan_args* a, int size, void* workspace, Segments* g);
// What enters every segment, from their own states.  first: what enters each chain, [sequence]
// [channels][N], or null.  right: segments follow each other from the last to the first.
int enter_segments(const ScanParams& p, int states, const Segments& g, const float* first, bool right, cudaStream_t st);

// Launches `kernel` behind the previous kernel of the stream, which it may overlap up to its
// wait_for_previous().
template <typename... P, typename... A>
int launch_after(const char* what, void (*kernel)(P...), int64_t blocks, int threads, size_t smem, cudaStream_t st, A... args) {
    if (blocks > 0x7fffffff) return fail(VH_E_RANGE, "%s: too many channel tiles", what);
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
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
