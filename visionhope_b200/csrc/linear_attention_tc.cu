// Linear attention on tcgen05: bf16 rows whose addresses TMA takes, in chunks of 128 tokens.
//
// A CTA walks the chunks of one chain or segment (one head).  Per chunk, with the fp32
// state S in registers and its bf16 rounding in shared memory:
//     scores = Q K^T, O2 = Q S             -> TMEM   (operands as TMA brought them)
//     P = scores * lambda^(i-j), bf16      TMEM -> TMEM
//     O1 = P V                             -> TMEM   (P an operand in TMEM)
//     K~ = K * lambda^(n-1-j) in planes    shared -> shared, the first in place of K
//     U = K~^T V, one product a plane      -> TMEM
//     o = out_scale (O1 + lambda^(i+1) O2),  S = lambda^n S + U
// S never lives in TMEM: the matrix unit truncates its sums, and a state that stayed there for thousands
// of tokens would drift.  K~ has two planes (2^-17) where only outputs are asked for, three (exact)
// where the state is handed out.  The next chunks' tiles arrive meanwhile (two stages), and the next
// chunk's first products run while this chunk's outputs are written.
//
// A token and head of 128 keys and values takes 1 KB of memory (0.16 ns) and, with two planes, 2.2 times the
// recurrence's operations (0.12 ns at the tensor cores' rate); a CTA's steps depend on one another, which bounds
// it.  4 x 8192 tokens of 16 heads of 128: 184 us, 2.9 TB/s, tensor pipe 25 %; warp-level matrix instructions took
// 825.  64 x 784 tokens of 4 heads of 64, forward and backward: 135 us (577).
//
// Reversed sequences keep their rows in memory order and turn the mask and the weights around: local row
// r has position n-1-r.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <mutex>

#include "abi_util.h"
#include "linear_attention.cuh"
#include "tc_util.cuh"

namespace vh {
namespace lin {
namespace {

constexpr int kT = 128;         // tokens a chunk
constexpr int kCompute = 256;   // threads at the tiles
constexpr int kTileBytes = kT * 128;  // 128 rows of 64 bf16, 128-byte swizzle
constexpr uint64_t kWaitNs = 2000000000ull;

__device__ unsigned int g_status;  // non-zero once a bounded wait gave up

struct Maps {
    CUtensorMap q, k, v, o;
};

// ---- instructions that only this kernel uses ------------------------------------------------------
// Operands in 128-byte swizzle.  Rows of the contraction-contiguous kind: 8-row groups 1024 bytes apart.
// The other kind (64 contiguous elements of the outer axis a row, one row a step of the contraction):
// groups of 8 steps 1024 bytes apart, the next 64 outer elements `lead` bytes on.
__device__ __forceinline__ uint64_t desc(uint32_t addr, uint32_t lead) {
    return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)((lead >> 4) & 0x3FFFu) << 16) | ((uint64_t)(1024 >> 4) << 32) |
           (uint64_t(1) << 46) | (uint64_t(2) << 61);
}
// The operand `bytes` further on.  Descriptors come from one by additions of constants: a product that waits
// for its descriptor's arithmetic takes twice its 64 cycles to issue.
__device__ __forceinline__ uint64_t ahead(uint64_t d, uint32_t bytes) { return d + (bytes >> 4); }
constexpr uint32_t kMajorA = 1u << 15, kMajorB = 1u << 16;  // outer axis contiguous

// D (+)= A B with A in TMEM (32-bit columns of two consecutive contraction elements).
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %6, %7, %8}, p;\n\t}"
        ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(0u), "r"(0u), "r"(0u), "r"(0u)
        : "memory");
}
__device__ __forceinline__ void ld32(uint32_t addr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
        "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]),
          "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]),
          "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr));
}
__device__ __forceinline__ void st16(uint32_t addr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
// One thread of a converged warp.
__device__ __forceinline__ bool elect() {
    uint32_t p;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "elect.sync _|p, 0xffffffff;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(p));
    return p != 0;
}
// A value that all lanes have, in a form that the compiler knows to be one: what products are issued with then
// stays in uniform registers.
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return __shfl_sync(0xffffffffu, v, 0); }
// A tile from shared memory (rows of 64 columns in the same swizzle) to global memory.
__device__ __forceinline__ void tma_store_4d(const void* map, const void* src, int c0, int c1, int c2, int c3) {
    asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.bulk_group [%0, {%2, %3, %4, %5}], [%1];" ::"l"(
                     reinterpret_cast<uint64_t>(map)),
                 "r"(tcu::smem_u32(src)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
                 : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
__device__ __forceinline__ void stores_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// ---- shared memory ------------------------------------------------------------------------------
// Two stages of tiles [V | K | Q], each of blocks of 64 columns; then the state's operand, which is also
// where the third plane of K~ goes (the second goes where Q was).  A chunk's outputs leave from where its V
// was: Q and K of the chunk after next, which its scores wait for, are loaded at once, and V when they have left.
template <int DK, int DV, int KP>
struct Smem {
    static constexpr int kK = kTileBytes * (DK / 64), kV = kTileBytes * (DV / 64);
    static constexpr int kKeys = kV, kQueries = kV + kK, kStage = kV + 2 * kK;
    static constexpr int kState = KP == 3 && kK > DK * DV * 2 ? kK : DK * DV * 2;
    static constexpr bool kAhead = DK == 128 && DV == 64 && KP == 2;  // see tc_kernel
    static constexpr int kPlane = 2 * kStage + kState;             // the second plane, where it does not take Q's place
    static constexpr int kPower = kPlane + (kAhead ? kK : 0);      // lambda^n, n = 0..128, and times kv_scale
    static constexpr int kWeights = kPower + 2 * 132 * 4;          // of a score: by column, and on the diagonal
    static constexpr int kBars = kWeights + (32 + 64) * 4;         // 7 barriers, TMEM base, a flag
    static constexpr int kLaunch = kBars + 64 + 1024;              // the tiles start on 1024 bytes
    static_assert(kLaunch <= 232448, "shared memory of an SM");
};
// Without outputs: tiles [V | K], and the planes of K~ behind the first.  Where two CTAs share an SM, two stages
// and planes for two chunks, so that the keys of one are weighed while the other's product runs (64 x 256
// tokens of two images 14.6 us, against 19.8 in three stages); else three stages (two for three planes of
// 128 keys and values), as two leave too little time to load 64 KB (62 against 89 us for half of 4 x 8192
// tokens of 16 heads of 128).
template <int DK, int DV, int KP>
struct StatesSmem {
    static constexpr int kK = kTileBytes * (DK / 64), kV = kTileBytes * (DV / 64);
    static constexpr int kStage = kK + kV, kPlanes = (KP - 1) * kK;
    static constexpr int kBuffers = DK + DV == 128 ? 2 : 1;
    static constexpr int kStages = kBuffers == 1 && 3 * kStage + kPlanes + 2048 <= 226 * 1024 ? 3 : 2;
    static constexpr int kPower = kStages * kStage + kBuffers * kPlanes;
    static constexpr int kBars = kPower + 132 * 4;                 // a barrier a stage, the product's, TMEM base, a flag
    static constexpr int kLaunch = kBars + 64 + 1024;
    static_assert(kLaunch <= 232448, "shared memory of an SM");
};

// What both kernels know of their unit.
template <int DK, int DV>
struct Chain {
    static constexpr int NC = DK == 128 ? DV / 2 : DV / 4;  // state columns a thread
    const Params& p;
    const Unit& u;
    int col0, cols;  // the value columns of this CTA
    int a, b0;       // this thread's part of the state: key row a, NC of these columns from b0 on

    __device__ __forceinline__ Chain(const Params& params, const Unit& unit) : p(params), u(unit) {
        const int quad = threadIdx.x >> 5 & 3, half = threadIdx.x >> 7, lane = threadIdx.x & 31;
        col0 = blockIdx.z * DV;
        cols = min(DV, p.dv - col0);
        a = DK == 128 ? quad * 32 + lane : (quad & 1) * 32 + lane;
        b0 = DK == 128 ? half * NC : (half * 2 + (quad >> 1)) * NC;
    }
    __device__ __forceinline__ int chunks() const { return (int)((u.t1 - u.t0 + kT - 1) / kT); }
    __device__ __forceinline__ int tokens(int c) const { return (int)min((int64_t)kT, u.t1 - u.t0 - (int64_t)c * kT); }
    // a chunk's first row in memory, counted from the sequence's
    __device__ __forceinline__ int64_t first_row(int c) const {
        const int64_t t = u.t0 + (int64_t)c * kT;
        return p.seqs.reverse ? u.e.len - t - tokens(c) : t;
    }
    __device__ __forceinline__ int row_at(int c) const { return (int)(first_row(c) + (p.seqs.offsets ? u.e.row : 0)); }
    __device__ __forceinline__ int batch_at() const { return p.seqs.offsets ? 0 : u.s; }

    // The state from global memory, through shared memory (`tile`, rows of DV + 4), because a thread's columns
    // are far from its neighbour's.  `initial`: element (a, b) at a init_a + b init_b, or null; `adds`: what
    // `before` segments ahead of this one add, `stride` apart, or null, or (before 0) the state itself.  Ends
    // with everybody done reading.
    template <typename Sync>
    __device__ __forceinline__ void load_state(float (&s)[NC], const float* initial, const float* adds, int before, int64_t stride,
                                               float log_decay, float* tile, Sync sync) const {
        const float step = decay_power(log_decay, p.segment), first = decay_power(log_decay, p.segment - (p.entry ? 1 : 0));
        const bool across = !initial || p.init_b == 1;
        const int inner = across ? cols : p.dk, total = p.dk * cols;
        constexpr int kAhead = 8;
#pragma unroll 1
        for (int i0 = threadIdx.x; i0 < total; i0 += kAhead * kCompute) {
            float run[kAhead];
            int at[kAhead], to[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                const int i = min(i0 + k * kCompute, total - 1), o = i / inner, x = i - o * inner;
                const int ra = across ? o : x, cb = across ? x : o;
                to[k] = ra * (DV + 4) + cb;
                at[k] = ra * p.dv + col0 + cb;
                run[k] = initial ? initial[ra * p.init_a + (col0 + cb) * p.init_b] : adds && before == 0 ? adds[at[k]] : 0.f;
            }
            for (int j = 0; j < before; ++j) {
                const float w = j == 0 ? first : step;
#pragma unroll
                for (int k = 0; k < kAhead; ++k) run[k] = run[k] * w + adds[j * stride + at[k]];
            }
#pragma unroll
            for (int k = 0; k < kAhead; ++k) tile[to[k]] = run[k];
        }
        sync();
#pragma unroll
        for (int i = 0; i < NC; i += 4) {
            const float4 v = *reinterpret_cast<const float4*>(tile + a * (DV + 4) + b0 + i);
            const float f[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) s[i + e] = a < p.dk && b0 + i + e < cols ? f[e] : 0.f;
        }
        sync();
    }
    template <typename Sync>
    __device__ __forceinline__ void store_state(const float (&s)[NC], float* to, float scale, float* tile, Sync sync) const {
        sync();
#pragma unroll
        for (int i = 0; i < NC; i += 4)
            *reinterpret_cast<float4*>(tile + a * (DV + 4) + b0 + i) =
                make_float4(s[i] * scale, s[i + 1] * scale, s[i + 2] * scale, s[i + 3] * scale);
        sync();
        for (int i = threadIdx.x; i < p.dk * cols; i += kCompute) {
            const int r = i / cols, c = i - r * cols;
            to[r * p.dv + col0 + c] = tile[r * (DV + 4) + c];
        }
    }
    // S = w S + U
    __device__ __forceinline__ void update(float (&s)[NC], uint32_t at, float w) const {
#pragma unroll
        for (int i0 = 0; i0 < NC; i0 += 16) {
            float x[16];
            tcu::tmem_ld16(at + b0 + i0, x);
            tcu::tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i0 + i] = fmaf(s[i0 + i], w, x[i]);
        }
    }
};

// Planes of the weighted keys of n tokens, the first in place; rows past the sequence become zeros.
template <int DK, int KP>
__device__ __forceinline__ void weigh_keys(uint8_t* kt, uint8_t* plane1, uint8_t* plane2, const float* weight, int n, bool reverse) {
#pragma unroll 2
    for (int i = threadIdx.x; i < kT * DK / 8; i += kCompute) {
        const int j = i / 8 % kT;
        uint4 x = *reinterpret_cast<const uint4*>(kt + i * 16);
        if (j >= n) x = make_uint4(0, 0, 0, 0);
        const float2 w = splat2(weight[j < n ? (reverse ? j : n - 1 - j) : 0]);
        const uint32_t words[4] = {x.x, x.y, x.z, x.w};
        uint32_t out[3][4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float2 v = fmul2(make_float2(__uint_as_float(words[e] << 16), __uint_as_float(words[e] & 0xffff0000u)), w);
#pragma unroll
            for (int pl = 0; pl < KP; ++pl) {
                const uint32_t b = ssm::join(v.x, v.y, __nv_bfloat16{});
                out[pl][e] = b;
                if (pl + 1 < KP) v = fsub2(v, make_float2(__uint_as_float(b << 16), __uint_as_float(b & 0xffff0000u)));
            }
        }
        *reinterpret_cast<uint4*>(kt + i * 16) = make_uint4(out[0][0], out[0][1], out[0][2], out[0][3]);
        *reinterpret_cast<uint4*>(plane1 + i * 16) = make_uint4(out[1][0], out[1][1], out[1][2], out[1][3]);
        if constexpr (KP == 3) *reinterpret_cast<uint4*>(plane2 + i * 16) = make_uint4(out[2][0], out[2][1], out[2][2], out[2][3]);
    }
    tcu::fence_proxy_async_smem();
}

// Rows past the sequence are another's: their products with zeros must be zeros.
template <int DV>
__device__ __forceinline__ void clear_values(uint8_t* vt, int n) {
    for (int i = threadIdx.x; i < (kT - n) * (DV / 8); i += kCompute) {
        const int r = n + i / (DV / 8), ch = i % (DV / 8);
        *reinterpret_cast<uint4*>(vt + (ch / 8) * kTileBytes + r * 128 + (ch % 8) * 16) = make_uint4(0, 0, 0, 0);
    }
    tcu::fence_proxy_async_smem();
}

// U = K~^T V over n tokens, the smallest plane first.  64 keys: a lead of 0 puts them into both halves of
// the 128 rows, so that all four warps of a column half have a share of the state.
template <int DK, int DV, int KP>
__device__ __forceinline__ void issue_update(uint32_t d, uint32_t kt, uint32_t plane1, uint32_t plane2, uint32_t vt, int n) {
    constexpr uint32_t id = tcu::idesc_bf16_f32(128, DV) | kMajorA | kMajorB, lead = DK == 128 ? kTileBytes : 0;
    const uint64_t dv = desc(vt, kTileBytes), dk[3] = {desc(kt, lead), desc(plane1, lead), desc(plane2, lead)};
    if (n > kT - 16) {
#pragma unroll
        for (int pl = KP - 1; pl >= 0; --pl)
#pragma unroll
            for (int kk = 0; kk < kT / 16; ++kk)
                tcu::mma_bf16(d, ahead(dk[pl], kk * 2048), ahead(dv, kk * 2048), id, pl < KP - 1 || kk > 0);
    } else {
#pragma unroll
        for (int pl = KP - 1; pl >= 0; --pl)
#pragma unroll 1
            for (int kk = 0; kk * 16 < n; ++kk)
                tcu::mma_bf16(d, ahead(dk[pl], kk * 2048), ahead(dv, kk * 2048), id, pl < KP - 1 || kk > 0);
    }
}

struct Waits {
    uint64_t* bars;
    volatile uint32_t* dead;
    __device__ __forceinline__ void operator()(int bar, uint32_t parity) const {
        if (!tcu::mbar_wait(&bars[bar], parity, *dead ? 1000 : kWaitNs)) {
            *dead = 1;
            atomicOr(&g_status, 1u);
        }
    }
};
// After a wait gave up: no more copies are started, and those in flight get a millisecond to land.
__device__ __forceinline__ void settle(const Waits& wait) {
    if (!*wait.dead) return;
    const uint64_t t0 = tcu::globaltimer_ns();
    while (tcu::globaltimer_ns() - t0 < 1000000) {
    }
}
template <int N>
__device__ __forceinline__ void bar_sync(int id) {
    asm volatile("bar.sync %0, %1;" ::"r"(id), "n"(N) : "memory");
}

// ---- chunks with outputs ------------------------------------------------------------------------
// Eight warps work on the tiles.  A thread that issues products waits for the matrix unit to take them
// (about as long as they run), so another warp does that; it leaves its registers to the others (a group
// of four warps, three of which do nothing, as registers move by groups).  With keys and values of at most
// 64 two CTAs share an SM, and there one of the eight issues: the warp whose scores are all masked.
template <int DK, int DV>
constexpr bool kApart = DK + DV != 128;
template <int DK, int DV>
constexpr int kBlock = kApart<DK, DV> ? kCompute + 128 : kCompute;

template <int DK, int DV, int KP>
__global__ void __launch_bounds__(kBlock<DK, DV>, kApart<DK, DV> ? 1 : 2) tc_kernel(const __grid_constant__ Params p,
                                                                                 const __grid_constant__ Maps maps) {
    using S = Smem<DK, DV, KP>;
    constexpr bool APART = kApart<DK, DV>;
    // Where two CTAs share TMEM, the update takes the half of the scores that P leaves free; otherwise it has
    // columns of its own, and runs before P V while P is made.
    // With 128 keys, 64 columns and two planes there is room, in TMEM and in shared memory, for the scores of two
    // chunks, a P of its own and a second plane that leaves Q alone: the next chunk's scores then follow P V.
    constexpr bool AHEAD = S::kAhead;
    constexpr int kCols = APART ? 512 : 256, kSync = APART ? kCompute + 32 : kCompute;
    constexpr uint32_t kScoreCols = AHEAD ? 256 : 128;
    constexpr uint32_t cO1 = kScoreCols, cO2 = cO1 + DV, cU = APART ? cO2 + DV : 64, cP = AHEAD ? cU + DV : 0;
    auto scores_at = [](int c) { return AHEAD ? (uint32_t)(c & 1) * 128 : 0u; };
    constexpr int NC = Chain<DK, DV>::NC;
    enum { kValues = 2, kScores = 4, kPV = 5, kUpdate = 6 };  // barriers; 0 and 1: Q and K of the two stages
    extern __shared__ uint8_t raw[];
    uint8_t* smem = raw + (1024 - (tcu::smem_u32(raw) & 1023)) % 1024;
    uint8_t* state = smem + 2 * S::kStage;
    float* power = reinterpret_cast<float*>(smem + S::kPower);
    float* powk = power + 132;
    float* column = reinterpret_cast<float*>(smem + S::kWeights);  // lambda^(31-i), reversed lambda^i
    float* diagonal = column + 32;                                 // [31 + x]: lambda^x, reversed lambda^-x; 0 where masked
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::kBars);
    uint32_t* tmem_at = reinterpret_cast<uint32_t*>(bars + 7);
    const Waits wait{bars, tmem_at + 1};

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, quad = warp & 3, half = warp >> 2;
    const int h = blockIdx.y;
    const Unit u = block_unit(p, reinterpret_cast<int*>(power + 131));
    auto zero_outside = [&] {
        ssm::zero_outside<__nv_bfloat16>(p.seqs, p.heads * p.dv, ((int64_t)blockIdx.x * gridDim.y + h) * gridDim.z + blockIdx.z,
                                         (int64_t)gridDim.x * gridDim.y * gridDim.z, p.o);
    };
    if (!u.live) {
        zero_outside();
        return;
    }
    const Chain<DK, DV> chain(p, u);
    const bool reverse = p.seqs.reverse;
    const int chunks = (int)uniform((uint32_t)chain.chunks());
    const int last_tokens = (int)uniform((uint32_t)(chunks > 0 ? chain.tokens(chunks - 1) : 0));
    auto tokens = [&](int c) { return c + 1 < chunks ? kT : last_tokens; };  // every chunk but a sequence's last is full
    const float log_decay = p.log_decay[h];
    if (tid <= kT) {
        const float w = decay_power(log_decay, tid);
        power[tid] = w;
        powk[tid] = w * p.kv_scale;
    }
    if (tid >= 128 && tid < 192) {
        const int i = tid - 128, x = reverse ? 31 - i : i - 31;
        diagonal[i] = x >= 0 ? decay_power(log_decay, x) * p.kv_scale : 0.f;
        if (i < 32) column[i] = decay_power(log_decay, reverse ? i : 31 - i) * p.kv_scale;
    }
    if (tid == 0) {
#pragma unroll
        for (int i = 0; i < 7; ++i) tcu::mbar_init(&bars[i], 1);
        tcu::fence_barrier_init();
        tmem_at[1] = 0;
    }
    if (warp == 0) tcu::tmem_alloc(tmem_at, kCols);

    const int64_t states = (int64_t)p.dk * p.dv;
    // where the state before the first chunk comes from
    const float *initial = nullptr, *adds = nullptr;
    int before = 0;
    if (u.t0 == 0 || p.join) initial = p.initial ? p.initial + ((int64_t)u.s * p.heads + h) * states : nullptr;
    if (u.t0 > 0) {
        before = p.join ? (int)(u.t0 / p.segment) : 0;
        adds = p.states + ((u.slot - before) * p.heads + h) * states;
    }
    bool has_state = initial || adds;
    // is the state after a chunk wanted
    auto updates = [&](int c) { return c + 1 < chunks || (p.final_state && u.t1 >= u.e.len); };

    auto load_keys = [&](int c) {  // and queries
        if (*wait.dead) return;
        uint8_t* at = smem + (c & 1) * S::kStage;
        uint64_t* bar = &bars[c & 1];
        tcu::mbar_arrive_expect_tx(bar, 2 * S::kK);
        const int row = chain.row_at(c), b = chain.batch_at();
#pragma unroll
        for (int i = 0; i < DK / 64; ++i) {
            tcu::tma_load_4d(at + S::kKeys + i * kTileBytes, &maps.k, bar, i * 64, h, row, b);
            tcu::tma_load_4d(at + S::kQueries + i * kTileBytes, &maps.q, bar, i * 64, h, row, b);
        }
    };
    auto load_values = [&](int c) {
        if (*wait.dead) return;
        uint8_t* at = smem + (c & 1) * S::kStage;
        uint64_t* bar = &bars[kValues + (c & 1)];
        tcu::mbar_arrive_expect_tx(bar, S::kV);
        const int row = chain.row_at(c), b = chain.batch_at();
#pragma unroll
        for (int i = 0; i < DV / 64; ++i) tcu::tma_load_4d(at + i * kTileBytes, &maps.v, bar, chain.col0 + i * 64, h, row, b);
    };
    auto wait_values = [&](int c) { wait(kValues + (c & 1), (c >> 1) & 1); };
    auto store_tiles = [&](int c) {  // a full chunk's outputs
        const int row = chain.row_at(c), b = chain.batch_at();
#pragma unroll
        for (int i = 0; i < DV / 64; ++i)
            if (i * 64 < chain.cols) tma_store_4d(&maps.o, smem + (c & 1) * S::kStage + i * kTileBytes, chain.col0 + i * 64, h, row, b);
    };
    const uint32_t base = tcu::smem_u32(smem), state_addr = base + 2 * S::kStage;
    uint32_t tmem = 0;
    // The issuer's part, between the workers' steps.
    auto issue_scores = [&](int c) {
        const uint32_t kt = base + (c & 1) * S::kStage + S::kKeys, qt = kt + S::kK;
        wait(c & 1, (c >> 1) & 1);
        tcu::tc_fence_after_sync();
        constexpr uint32_t id = tcu::idesc_bf16_f32(128, 128);
        const uint64_t dq = desc(qt, 16), dk = desc(kt, 16);
#pragma unroll
        for (int kk = 0; kk < DK / 16; ++kk) {
            const uint32_t at = (kk / 4) * kTileBytes + (kk % 4) * 32;
            tcu::mma_bf16(tmem + scores_at(c), ahead(dq, at), ahead(dk, at), id, kk > 0);
        }
    };
    auto issue_state = [&](int c) {  // q S
        const uint32_t qt = base + (c & 1) * S::kStage + S::kQueries;
        constexpr uint32_t id = tcu::idesc_bf16_f32(128, DV) | kMajorB;
        const uint64_t dq = desc(qt, 16), ds = desc(state_addr, DK * 128);
#pragma unroll
        for (int kk = 0; kk < DK / 16; ++kk)
            tcu::mma_bf16(tmem + cO2, ahead(dq, (kk / 4) * kTileBytes + (kk % 4) * 32), ahead(ds, kk * 2048), id, kk > 0);
    };
    auto issue_start = [&] {
        for (int c = 0; c < min(chunks, 2); ++c) {
            load_keys(c);
            load_values(c);
        }
        if (chunks > 0) {
            issue_scores(0);
            if (AHEAD) tcu::mma_commit(&bars[kScores]);
            if (has_state) issue_state(0);
            if (!AHEAD) tcu::mma_commit(&bars[kScores]);
        }
    };
    auto issue_next = [&](int c) {  // after chunk c
        if (c + 1 < chunks) {
            if (!AHEAD) issue_scores(c + 1);
            issue_state(c + 1);
            if (!AHEAD) tcu::mma_commit(&bars[kScores]);
        }
        if (c + 2 < chunks) load_keys(c + 2);
    };
    auto load_rest = [&](int c) {  // the values of chunk c + 1, once the outputs of c - 1 have left
        if (c == 0) return;
        stores_read();
        if (c + 1 < chunks) load_values(c + 1);
    };
    auto issue_pv = [&](int c, int n) {
        const uint32_t vt = base + (c & 1) * S::kStage;
        wait_values(c);
        tcu::tc_fence_after_sync();
        constexpr uint32_t id = tcu::idesc_bf16_f32(128, DV) | kMajorB;
        const uint64_t dv = desc(vt, kTileBytes);
        if (n > kT - 16) {
#pragma unroll
            for (int kk = 0; kk < kT / 16; ++kk) mma_ts(tmem + cO1, tmem + cP + kk * 8, ahead(dv, kk * 2048), id, kk > 0);
        } else {
#pragma unroll 1
            for (int kk = 0; kk * 16 < n; ++kk) mma_ts(tmem + cO1, tmem + cP + kk * 8, ahead(dv, kk * 2048), id, kk > 0);
        }
        tcu::mma_commit(&bars[kPV]);  // and of q S before it
        if (AHEAD && c + 1 < chunks) {
            issue_scores(c + 1);
            tcu::mma_commit(&bars[kScores]);
        }
    };
    auto issue_u = [&](int c, int n) {
        const uint32_t vt = base + (c & 1) * S::kStage;
        wait_values(c);
        tcu::tc_fence_after_sync();
        issue_update<DK, DV, KP>(tmem + cU, vt + S::kKeys, AHEAD ? base + S::kPlane : vt + S::kQueries, state_addr, vt, n);
        tcu::mma_commit(&bars[kUpdate]);
    };
    // every step ends with the writes to shared memory fenced and the TMEM accesses ordered
    auto sync = [&] {
        tcu::tc_fence_before_sync();
        bar_sync<kSync>(1);
        tcu::tc_fence_after_sync();
    };
    auto sync_workers = [&] { bar_sync<kCompute>(2); };

    if (APART && uniform((uint32_t)warp) >= kCompute / 32) {
        if constexpr (APART) asm volatile("setmaxnreg.dec.sync.aligned.u32 104;");
        if (uniform((uint32_t)warp) == kCompute / 32) {
            bar_sync<kSync>(1);  // barriers, TMEM and the state are there
            tcu::tc_fence_after_sync();
            tmem = uniform(*tmem_at);
            if (elect()) issue_start();
            for (int c = 0; c < chunks; ++c) {
                const int n = tokens(c);
                bool stored = c == 0;
                if (updates(c)) {
                    __syncwarp();
                    sync();  // keys weighed
                    if (elect()) {
                        issue_u(c, n);
                        if (AHEAD && !stored) store_tiles(c - 1);
                    }
                    stored |= AHEAD;
                }
                if (!AHEAD) {
                    __syncwarp();
                    sync();  // scores read
                    if (elect() && !stored) store_tiles(c - 1);
                    stored = true;
                }
                __syncwarp();
                sync();  // P written
                if (elect()) {
                    if (!stored) store_tiles(c - 1);
                    issue_pv(c, n);
                    load_rest(c);
                }
                __syncwarp();
                sync();  // outputs read, state written
                if (elect()) issue_next(c);
            }
            if (chunks > 0) {
                __syncwarp();
                sync();  // the last outputs are in their tiles
                if (elect()) {
                    if (last_tokens == kT) store_tiles(chunks - 1);
                    stores_read();
                }
            }
            __syncwarp();
        }
    } else {
        if constexpr (APART) asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
        const bool issues = !APART && uniform((uint32_t)warp) == (reverse ? 3u : 4u);  // then one thread of the warp does
        float s[NC];
        // rows of 64 value columns, one a key: the contraction runs over keys
        auto put_state = [&] {
#pragma unroll
            for (int i = 0; i < NC; i += 8) {
                const int b = chain.b0 + i, a = chain.a;
                uint4 w;
                w.x = ssm::join(s[i], s[i + 1], __nv_bfloat16{});
                w.y = ssm::join(s[i + 2], s[i + 3], __nv_bfloat16{});
                w.z = ssm::join(s[i + 4], s[i + 5], __nv_bfloat16{});
                w.w = ssm::join(s[i + 6], s[i + 7], __nv_bfloat16{});
                *reinterpret_cast<uint4*>(state + (b / 64) * (DK * 128) + a * 128 + (((b % 64) / 8) ^ (a & 7)) * 16) = w;
            }
            tcu::fence_proxy_async_smem();
        };
        float* scratch = reinterpret_cast<float*>(smem);  // before the first tiles and after the last
        if (has_state) {
            chain.load_state(s, initial, adds, before, p.heads * states, log_decay, scratch, sync_workers);
            put_state();
        } else {
#pragma unroll
            for (int i = 0; i < NC; ++i) s[i] = 0.f;
        }
        tcu::fence_proxy_async_smem();
        sync();
        tmem = uniform(*tmem_at);
        const uint32_t tmem_lane = tmem + ((uint32_t)(quad * 32) << 16);
        if (issues && elect()) issue_start();
        const int row = quad * 32 + lane;  // of the scores and outputs
        for (int c = 0; c < chunks; ++c) {
            const int n = tokens(c);
            const int entry = p.entry && u.t0 == 0 && c == 0;
            uint8_t* vt = smem + (c & 1) * S::kStage;
            uint8_t *kt = vt + S::kKeys, *qt = vt + S::kQueries;
            const bool update = updates(c);
            const int pos = reverse ? n - 1 - row : row;
            wait(c & 1, (c >> 1) & 1);
            if (n < kT) {
                wait_values(c);
                clear_values<DV>(vt, n);
            }
            wait(kScores, c & 1);
            tcu::tc_fence_after_sync();
            auto weigh = [&] {
                weigh_keys<DK, KP>(kt, AHEAD ? smem + S::kPlane : qt, state, powk, n, reverse);
                sync();
                if (issues && elect()) {
                    issue_u(c, n);
                    load_rest(c);
                }
            };
            auto renew = [&] {
                wait(kUpdate, c & 1);
                tcu::tc_fence_after_sync();
                chain.update(s, tmem_lane + cU, power[n - entry]);
                if (c + 1 < chunks) put_state();
            };
            if (APART && update) weigh();
            // P: columns 64 half .. + 63 of this row, two blocks of 32
            uint32_t pw[2][16];
#pragma unroll
            for (int blk = 0; blk < 2; ++blk) {
                const int cb = half * 2 + blk, j0 = cb * 32;
                if ((reverse ? cb < quad : cb > quad) || j0 >= n) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) pw[blk][i] = 0;
                    continue;
                }
                uint32_t x[32];
                ld32(tmem_lane + scores_at(c) + j0, x);
                tcu::tmem_wait_ld();
                // columns of this block that exist: reversed, the ones past the sequence are not masked
                uint32_t on = reverse && n - j0 < 32 ? (1u << (n - j0)) - 1 : 0xffffffffu;
                if (cb == quad) {
                    on &= reverse ? 0xffffffffu << lane : 0xffffffffu >> (31 - lane);
                    const float* w = diagonal + 31 + lane;
#pragma unroll
                    for (int i = 0; i < 32; i += 2) {
                        const float2 v = fmul2(make_float2(__uint_as_float(x[i]), __uint_as_float(x[i + 1])), make_float2(w[-i], w[-i - 1]));
                        pw[blk][i / 2] = ssm::join(v.x, v.y, __nv_bfloat16{});
                    }
                } else {
                    // lambda^|i-j| = (from the row to the block's near edge) (within the block)
                    const float2 wr = splat2(power[reverse ? j0 - row : row - j0 - 31]);
#pragma unroll
                    for (int i = 0; i < 32; i += 4) {
                        const float4 wc = *reinterpret_cast<const float4*>(column + i);
                        const float2 v0 = fmul2(fmul2(make_float2(__uint_as_float(x[i]), __uint_as_float(x[i + 1])), make_float2(wc.x, wc.y)), wr);
                        const float2 v1 = fmul2(fmul2(make_float2(__uint_as_float(x[i + 2]), __uint_as_float(x[i + 3])), make_float2(wc.z, wc.w)), wr);
                        pw[blk][i / 2] = ssm::join(v0.x, v0.y, __nv_bfloat16{});
                        pw[blk][i / 2 + 1] = ssm::join(v1.x, v1.y, __nv_bfloat16{});
                    }
                }
                // what is masked is cleared, not multiplied by zero: it may not be finite
                if (cb == quad || on != 0xffffffffu) {
#pragma unroll
                    for (int i = 0; i < 32; i += 2)
                        pw[blk][i / 2] &= (on >> i & 1 ? 0xffffu : 0u) | (on >> (i + 1) & 1 ? 0xffff0000u : 0u);
                }
            }
            if (!AHEAD) {  // P takes the place of the scores' first half, which others may still be reading
                sync();
                if (c > 0 && issues && elect()) store_tiles(c - 1);
            }
            st16(tmem_lane + cP + half * 32, pw[0]);
            st16(tmem_lane + cP + half * 32 + 16, pw[1]);
            wait_st();
            sync();
            if (issues && elect()) issue_pv(c, n);
            if (update) {
                if (APART) renew(); else weigh();
            }
            // this row's outputs, DV / 2 columns
            uint32_t out[DV / 4];
            wait_values(c);
            wait(kPV, c & 1);
            tcu::tc_fence_after_sync();
            const float wi = row < n ? power[pos + 1 - entry] : 0.f;
#pragma unroll
            for (int blk = 0; blk < DV / 64; ++blk) {
                const int c0 = half * (DV / 2) + blk * 32;
                uint32_t x[32], y[32];
                ld32(tmem_lane + cO1 + c0, x);
                if (has_state) ld32(tmem_lane + cO2 + c0, y);
                tcu::tmem_wait_ld();
                float2 zero = splat2(0.f);  // NaN once a value is not finite
#pragma unroll
                for (int i = 0; i < 32; i += 2) {
                    float2 v = make_float2(__uint_as_float(x[i]), __uint_as_float(x[i + 1]));
                    zero = ffma2(v, splat2(0.f), zero);
                    if (has_state) v = ffma2(make_float2(__uint_as_float(y[i]), __uint_as_float(y[i + 1])), splat2(wi), v);
                    x[i] = __float_as_uint(v.x);
                    x[i + 1] = __float_as_uint(v.y);
                }
                // A value that is not finite must not reach the rows before it: 0 times it is NaN in the
                // product.  Such chunks are rare; their rows are summed again, term by term.
                if (__any_sync(0xffffffffu, !(zero.x + zero.y == 0.f))) {
                    float sum[32];
#pragma unroll
                    for (int i = 0; i < 32; ++i) sum[i] = has_state ? __uint_as_float(y[i]) * wi : 0.f;
#pragma unroll 1
                    for (int j = 0; j < n; ++j) {
                        float pr[2];
                        tcu::tmem_ld2(tmem_lane + cP + j / 4 * 2, pr);
                        tcu::tmem_wait_ld();
                        const uint32_t w = __float_as_uint(j & 2 ? pr[1] : pr[0]);
                        const float pv = __uint_as_float(j & 1 ? w & 0xffff0000u : w << 16);
                        if (reverse ? j >= row : j <= row) {
#pragma unroll
                            for (int i = 0; i < 32; i += 8) {
                                const int cc = c0 + i;
                                float b[8];
                                load8(reinterpret_cast<const __nv_bfloat16*>(vt + (cc / 64) * kTileBytes + j * 128 + (((cc % 64) / 8) ^ (j & 7)) * 16), b);
#pragma unroll
                                for (int e = 0; e < 8; ++e) sum[i + e] = fmaf(pv, b[e], sum[i + e]);
                            }
                        }
                        __syncwarp();
                    }
#pragma unroll
                    for (int i = 0; i < 32; ++i) x[i] = __float_as_uint(sum[i]);
                }
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    out[blk * 16 + i] = ssm::join(__uint_as_float(x[2 * i]) * p.out_scale, __uint_as_float(x[2 * i + 1]) * p.out_scale,
                                                  __nv_bfloat16{});
            }
            if (!APART && update) renew();
            has_state |= update;
            sync();
            if (issues && elect()) issue_next(c);
            // the rows of o where V was, in the swizzle of its tiles; they leave during the next chunk
#pragma unroll
            for (int i = 0; i < DV / 16; ++i) {
                const int ch = half * (DV / 16) + i;
                *reinterpret_cast<uint4*>(vt + (ch / 8) * kTileBytes + row * 128 + ((ch % 8) ^ (row & 7)) * 16) =
                    make_uint4(out[4 * i], out[4 * i + 1], out[4 * i + 2], out[4 * i + 3]);
            }
            tcu::fence_proxy_async_smem();
        }
        if (chunks > 0) {
            sync();
            const int c = chunks - 1, n = last_tokens;
            if (n < kT) {  // rows past these are another sequence's
                const uint8_t* from_tile = smem + (c & 1) * S::kStage;
                const int64_t step = (int64_t)p.heads * p.dv;
                __nv_bfloat16* to = static_cast<__nv_bfloat16*>(p.o) + (u.e.row + chain.first_row(c)) * step + (int64_t)h * p.dv + chain.col0;
                for (int i = tid; i < n * (DV / 8); i += kCompute) {
                    const int r = i / (DV / 8), ch = i % (DV / 8);
                    if (ch * 8 >= chain.cols) continue;
                    const uint4 v = *reinterpret_cast<const uint4*>(from_tile + (ch / 8) * kTileBytes + r * 128 + ((ch % 8) ^ (r & 7)) * 16);
                    *reinterpret_cast<uint4*>(to + r * step + ch * 8) = v;
                }
            }
            __syncwarp();
            if (issues && elect()) {
                if (n == kT) store_tiles(c);
                stores_read();
            }
        }
        if (p.final_state && u.t1 >= u.e.len) {
            // the stage that the last outputs do not lie in
            float* tile = reinterpret_cast<float*>(smem + (chunks & 1) * S::kStage);
            const float last = p.exit_decay && u.e.len > 0 ? decay_power(log_decay, 1) : 1.f;
            chain.store_state(s, p.final_state + ((int64_t)u.s * p.heads + h) * states, last, tile, sync_workers);
        }
    }
    if (tid == 0) settle(wait);  // warps without work have not waited for the flag to be set up
    tcu::tc_fence_before_sync();
    __syncthreads();
    if (warp == 0) tcu::tmem_dealloc(*tmem_at, kCols);
    zero_outside();
}

// ---- what a segment adds to the state -------------------------------------------------------------
template <int DK, int DV, int KP>
__global__ void __launch_bounds__(kCompute + 32, DK + DV == 128 ? 2 : 1) tc_states_kernel(const __grid_constant__ Params p,
                                                                                       const __grid_constant__ Maps maps) {
    using S = StatesSmem<DK, DV, KP>;
    constexpr int kCols = DV, NC = Chain<DK, DV>::NC;
    constexpr int kUpdate = S::kStages;
    extern __shared__ uint8_t raw[];
    uint8_t* smem = raw + (1024 - (tcu::smem_u32(raw) & 1023)) % 1024;
    float* powk = reinterpret_cast<float*>(smem + S::kPower);
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::kBars);
    uint32_t* tmem_at = reinterpret_cast<uint32_t*>(bars + S::kStages + 1);
    const Waits wait{bars, tmem_at + 1};
    const int tid = threadIdx.x, warp = tid >> 5, quad = warp & 3;
    const int h = blockIdx.y;
    const Unit u = block_unit(p, reinterpret_cast<int*>(powk + 131));
    if (!u.live || u.t1 >= u.e.len) return;  // the state after a sequence's last segment is nobody's start
    const Chain<DK, DV> chain(p, u);
    const bool reverse = p.seqs.reverse;
    const int chunks = (int)uniform((uint32_t)chain.chunks());
    const float log_decay = p.log_decay[h];
    if (tid <= kT) powk[tid] = decay_power(log_decay, tid) * p.kv_scale;
    const float decay = decay_power(log_decay, kT);  // all chunks of these segments are full
    if (tid == 0) {
#pragma unroll
        for (int i = 0; i <= S::kStages; ++i) tcu::mbar_init(&bars[i], 1);
        tcu::fence_barrier_init();
        tmem_at[1] = 0;
    }
    if (warp == 0) tcu::tmem_alloc(tmem_at, kCols);
    auto sync = [&] {
        tcu::tc_fence_before_sync();
        __syncthreads();
        tcu::tc_fence_after_sync();
    };
    sync();
    const uint32_t tmem = uniform(*tmem_at);
    auto planes_of = [&](int c) { return smem + S::kStages * S::kStage + (c % S::kBuffers) * S::kPlanes; };
    auto load_tiles = [&](int c) {
        if (*wait.dead) return;
        uint8_t* at = smem + c % S::kStages * S::kStage;
        uint64_t* bar = &bars[c % S::kStages];
        tcu::mbar_arrive_expect_tx(bar, S::kStage);
        const int row = chain.row_at(c), b = chain.batch_at();
#pragma unroll
        for (int i = 0; i < DV / 64; ++i) tcu::tma_load_4d(at + i * kTileBytes, &maps.v, bar, chain.col0 + i * 64, h, row, b);
#pragma unroll
        for (int i = 0; i < DK / 64; ++i) tcu::tma_load_4d(at + S::kV + i * kTileBytes, &maps.k, bar, i * 64, h, row, b);
    };
    if (uniform((uint32_t)warp) == kCompute / 32) {
        if (elect())
            for (int c = 0; c < min(chunks, S::kStages); ++c) load_tiles(c);
        for (int c = 0; c < chunks; ++c) {
            __syncwarp();
            sync();  // keys of chunk c weighed, product c - 1 read
            if (elect()) {
                const uint32_t vt = tcu::smem_u32(smem) + c % S::kStages * S::kStage, pl = tcu::smem_u32(planes_of(c));
                issue_update<DK, DV, KP>(tmem, vt + S::kV, pl, pl + S::kK, vt, kT);
                tcu::mma_commit(&bars[kUpdate]);
                if (c > 0 && c - 1 + S::kStages < chunks) load_tiles(c - 1 + S::kStages);
            }
        }
    } else {
        float s[NC];
#pragma unroll
        for (int i = 0; i < NC; ++i) s[i] = 0.f;
        auto weigh = [&](int c) {
            uint8_t *kt = smem + c % S::kStages * S::kStage + S::kV, *pl = planes_of(c);
            wait(c % S::kStages, c / S::kStages & 1);
            weigh_keys<DK, KP>(kt, pl, pl + S::kK, powk, kT, reverse);
        };
        weigh(0);
        for (int c = 0; c < chunks; ++c) {
            sync();
            if (S::kBuffers == 2 && c + 1 < chunks) weigh(c + 1);
            wait(kUpdate, c & 1);
            tcu::tc_fence_after_sync();
            chain.update(s, tmem + ((uint32_t)(quad * 32) << 16), decay);
            if (S::kBuffers == 1 && c + 1 < chunks) weigh(c + 1);
        }
        const int64_t states = (int64_t)p.dk * p.dv;
        chain.store_state(s, p.states + (u.slot * p.heads + h) * states, 1.f, reinterpret_cast<float*>(smem),
                          [&] { bar_sync<kCompute>(2); });
    }
    if (tid == 0) settle(wait);
    tcu::tc_fence_before_sync();
    __syncthreads();
    if (warp == 0) tcu::tmem_dealloc(tmem, kCols);
}

// ---- host ---------------------------------------------------------------------------------------
PFN_cuTensorMapEncodeTiled_v12000 encoder() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult q{};
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f);
    });
    return fn;
}

// Boxes of 64 columns by 128 tokens of one head and sequence.
bool encode(CUtensorMap* m, const Heads& t, const Params& p, int dim) {
    const bool packed = p.seqs.offsets != nullptr;
    const cuuint64_t dims[4] = {(cuuint64_t)dim, (cuuint64_t)p.heads, (cuuint64_t)p.seqs.length, (cuuint64_t)(packed ? 1 : p.seqs.count)};
    // an axis of one element may have any stride
    const int64_t widest = std::max<int64_t>({t.rows.token, t.head, 8});
    const int64_t st[3] = {p.heads > 1 ? t.head : widest, p.seqs.length > 1 ? t.rows.token : widest,
                           dims[3] > 1 ? t.rows.batch : widest};
    cuuint64_t strides[3];
    for (int i = 0; i < 3; ++i) {
        if (st[i] <= 0 || st[i] % 8 || st[i] >= (int64_t(1) << 38)) return false;
        strides[i] = (cuuint64_t)st[i] * 2;
    }
    const cuuint32_t box[4] = {64, 1, kT, 1}, es[4] = {1, 1, 1, 1};
    return encoder()(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(t.p), dims, strides, box, es,
                     CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int DK, int DV, int KP>
int launch(const Params& p, const Maps& m, int64_t units, bool outputs, cudaStream_t st) {
    const size_t smem = outputs ? Smem<DK, DV, KP>::kLaunch : StatesSmem<DK, DV, KP>::kLaunch;
    const void* fn = outputs ? reinterpret_cast<const void*>(&tc_kernel<DK, DV, KP>)
                             : reinterpret_cast<const void*>(&tc_states_kernel<DK, DV, KP>);
    if (!ensure_smem_attr(fn, smem)) return fail(VH_E_DEVICE, "linear attention: shared memory");
    const dim3 grid((unsigned)units, p.heads, (p.dv + DV - 1) / DV);
    if (outputs) tc_kernel<DK, DV, KP><<<grid, kBlock<DK, DV>, smem, st>>>(p, m);
    else tc_states_kernel<DK, DV, KP><<<grid, kCompute + 32, smem, st>>>(p, m);
    return launch_status(outputs ? "linear attention" : "linear attention: segment states");
}

template <int DK, int DV>
int run_dims(const Params& p, const Maps& m, int64_t units, bool exact, cudaStream_t st) {
    auto one = [&](bool outputs) {
        return exact ? launch<DK, DV, 3>(p, m, units, outputs, st) : launch<DK, DV, 2>(p, m, units, outputs, st);
    };
    if (p.segment) {
        if (int rc = one(false)) return rc;
        if (!p.join)
            if (int rc = enter_segments(p, st)) return rc;
    }
    return one(true);
}

}  // namespace

// The value columns a CTA takes: 64 where that makes up for chains that are fewer than the SMs (scores and
// weighted keys are then computed twice), else all.
static bool narrow_values(int64_t chains, int dv) { return dv <= 64 || 2 * chains <= sm_count(); }

// CTAs fill the card once: one an SM, two where keys and columns are at most 64.  Chains that are fewer
// than half of them are cut; packed sequences always are, as the host does not know their lengths.
int tc_segment_size(int64_t length, int batch, bool packed, int heads, int dk, int dv) {
    const bool narrow = narrow_values((int64_t)batch * heads, dv);
    const int64_t ctas = (int64_t)sm_count() * (dk <= 64 && narrow ? 2 : 1), rows = heads * (narrow ? (dv + 63) / 64 : 1);
    int64_t size;
    if (packed) {
        size = (length * rows + ctas - 1) / ctas;
    } else {
        const int64_t segs = ctas / (batch * rows);
        if (segs < 2) return 0;
        size = (length + segs - 1) / segs;
    }
    size = std::max<int64_t>((size + kT - 1) / kT * kT, 4 * kT);
    return size < length ? (int)size : 0;
}

bool tc_run(Params p, void* states, cudaStream_t st, int* rc) {
    if (p.q.vec != 8 || p.k.vec != 8 || p.v.vec != 8 || p.vec_o != 8 || p.seqs.length < kT || !encoder()) return false;
    Maps m;
    const int64_t row = (int64_t)p.heads * p.dv;
    const Heads o{p.o, {p.seqs.length * row, row}, p.dv, 8};
    if (!encode(&m.q, p.q, p, p.dk) || !encode(&m.k, p.k, p, p.dk) || !encode(&m.v, p.v, p, p.dv) || !encode(&m.o, o, p, p.dv)) return false;
    const bool packed = p.seqs.offsets != nullptr, exact = p.final_state != nullptr;
    p.segment = tc_segment_size(p.seqs.length, p.seqs.count, packed, p.heads, p.dk, p.dv);
    p.states = static_cast<float*>(states);
    // Sequences of a few segments add up their starts themselves, which saves a launch; long ones would read
    // the square of their number.
    p.join = p.segment && p.seqs.length <= 24 * (int64_t)p.segment;
    const int64_t units = p.segment ? ssm::slot_total(packed, p.seqs.length, p.seqs.count, p.segment) : p.seqs.count;
    const bool narrow = narrow_values((int64_t)p.seqs.count * p.heads, p.dv);
    if (p.dk <= 64) *rc = narrow ? run_dims<64, 64>(p, m, units, exact, st) : run_dims<64, 128>(p, m, units, exact, st);
    else *rc = narrow ? run_dims<128, 64>(p, m, units, exact, st) : run_dims<128, 128>(p, m, units, exact, st);
    return true;
}

unsigned tc_status(bool reset) {
    unsigned v = 0;
    if (cudaMemcpyFromSymbol(&v, g_status, sizeof(v)) != cudaSuccess) return 2;
    if (reset) {
        const unsigned zero = 0;
        cudaMemcpyToSymbol(g_status, &zero, sizeof(zero));
    }
    return v;
}

}  // namespace lin
}  // namespace vh
