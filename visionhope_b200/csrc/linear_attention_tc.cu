// Linear attention on tcgen05: bf16 rows whose addresses TMA takes, in chunks of 128 tokens.
//
// A CTA of 256 threads walks the chunks of one chain or segment (one head).  Per chunk, with the fp32
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
constexpr int kThreads = 256;
constexpr int kTileBytes = kT * 128;  // 128 rows of 64 bf16, 128-byte swizzle
constexpr uint64_t kWaitNs = 2000000000ull;

__device__ unsigned int g_status;  // non-zero once a bounded wait gave up

struct Maps {
    CUtensorMap q, k, v;
};

// ---- instructions that only this kernel uses ------------------------------------------------------
// Operands in 128-byte swizzle.  Rows of the contraction-contiguous kind: 8-row groups 1024 bytes apart.
// The other kind (64 contiguous elements of the outer axis a row, one row a step of the contraction):
// groups of 8 steps 1024 bytes apart, the next 64 outer elements `lead` bytes on.
__device__ __forceinline__ uint64_t desc(uint32_t addr, uint32_t lead) {
    return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)((lead >> 4) & 0x3FFFu) << 16) | ((uint64_t)(1024 >> 4) << 32) |
           (uint64_t(1) << 46) | (uint64_t(2) << 61);
}
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
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// ---- shared memory ------------------------------------------------------------------------------
// Two stages of tiles [K | V | Q], each of blocks of 64 columns; then the state's operand, which is also
// where the third plane of K~ goes.  The second plane goes where Q was, or, without Q, behind.
template <int DK, int DV, int KP, bool OUT>
struct Smem {
    static constexpr int kK = kTileBytes * (DK / 64), kV = kTileBytes * (DV / 64), kQ = OUT ? kK : 0;
    static constexpr int kStage = kK + kV + kQ;
    static constexpr int kState = OUT ? (KP == 3 && kK > DK * DV * 2 ? kK : DK * DV * 2) : kK * (KP - 1);
    static constexpr int kPower = 2 * kStage + kState;             // lambda^n, n = 0..128, and times kv_scale
    static constexpr int kBars = kPower + 2 * 132 * 4;             // 5 barriers, TMEM base, a flag
    static constexpr int kBytes = kBars + 64;
    static constexpr int kLaunch = kBytes + 1024;                  // the tiles start on 1024 bytes
    static_assert(kLaunch <= 232448, "shared memory of an SM");
};

template <int DK, int DV, int KP, bool OUT>
__global__ void __launch_bounds__(kThreads, DK + DV == 128 ? 2 : 1) tc_kernel(const __grid_constant__ Params p,
                                                                             const __grid_constant__ Maps maps) {
    using S = Smem<DK, DV, KP, OUT>;
    constexpr int kCols = DV == 64 ? 256 : 512;
    constexpr uint32_t cScore = 0, cO1 = 128, cO2 = 128 + DV, cU = DV == 64 ? 64 : 384;
    constexpr int NC = DK == 128 ? DV / 2 : DV / 4;  // state columns a thread
    extern __shared__ uint8_t raw[];
    uint8_t* smem = raw + (1024 - (tcu::smem_u32(raw) & 1023)) % 1024;
    uint8_t* state = smem + 2 * S::kStage;
    float* power = reinterpret_cast<float*>(smem + S::kPower);
    float* powk = power + 132;
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::kBars);  // tiles 0, tiles 1, scores, PV, U
    uint32_t* tmem_at = reinterpret_cast<uint32_t*>(bars + 5);
    volatile uint32_t* dead = tmem_at + 1;

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, quad = warp & 3, half = warp >> 2;
    const int h = blockIdx.y;
    Unit u = unit_at(p, blockIdx.x);
    if constexpr (OUT)
        ssm::zero_outside<__nv_bfloat16>(p.seqs, p.heads * p.dv, (int64_t)blockIdx.x * gridDim.y + h, (int64_t)gridDim.x * gridDim.y, p.o);
    if (!u.live || (!OUT && u.t1 >= u.e.len)) return;
    const bool reverse = p.seqs.reverse;
    const int chunks = (int)((u.t1 - u.t0 + kT - 1) / kT);
    const float log_decay = p.log_decay[h];
    if (tid <= kT) {
        const float w = decay_power(log_decay, tid);
        power[tid] = w;
        powk[tid] = w * p.kv_scale;
    }
    if (tid == 0) {
#pragma unroll
        for (int i = 0; i < 5; ++i) tcu::mbar_init(&bars[i], 1);
        tcu::fence_barrier_init();
        *dead = 0;
    }
    if (warp == 0) tcu::tmem_alloc(tmem_at, kCols);

    // this thread's part of the state: key row a, NC value columns from b0 on
    const int a = DK == 128 ? quad * 32 + lane : (quad & 1) * 32 + lane;
    const int b0 = DK == 128 ? half * NC : (half * 2 + (quad >> 1)) * NC;
    float s[NC];
    const int64_t states = (int64_t)p.dk * p.dv;
    const float* from = nullptr;
    int64_t fa = p.dv, fb = 1;
    if (OUT) {
        if (u.t0 == 0) {
            from = p.initial ? p.initial + ((int64_t)u.s * p.heads + h) * states : nullptr;
            fa = p.init_a;
            fb = p.init_b;
        } else {
            from = p.states + (u.slot * p.heads + h) * states;
        }
    }
#pragma unroll
    for (int i = 0; i < NC; ++i) s[i] = from && a < p.dk && b0 + i < p.dv ? from[a * fa + (b0 + i) * fb] : 0.f;
    bool has_state = from != nullptr;
    // rows of 64 value columns, one a key: the contraction runs over keys
    auto put_state = [&] {
#pragma unroll
        for (int i = 0; i < NC; i += 8) {
            const int b = b0 + i;
            uint4 w;
            w.x = ssm::join(s[i], s[i + 1], __nv_bfloat16{});
            w.y = ssm::join(s[i + 2], s[i + 3], __nv_bfloat16{});
            w.z = ssm::join(s[i + 4], s[i + 5], __nv_bfloat16{});
            w.w = ssm::join(s[i + 6], s[i + 7], __nv_bfloat16{});
            *reinterpret_cast<uint4*>(state + (b / 64) * (DK * 128) + a * 128 + (((b % 64) / 8) ^ (a & 7)) * 16) = w;
        }
        tcu::fence_proxy_async_smem();
    };
    if (OUT && has_state) put_state();
    tcu::tc_fence_before_sync();
    __syncthreads();
    tcu::tc_fence_after_sync();
    const uint32_t tmem = *tmem_at, tmem_lane = tmem + ((uint32_t)(quad * 32) << 16);
    const uint32_t base = tcu::smem_u32(smem), state_addr = tcu::smem_u32(state);

    auto wait = [&](int bar, uint32_t parity) {
        if (!tcu::mbar_wait(&bars[bar], parity, *dead ? 1000 : kWaitNs)) {
            *dead = 1;
            atomicOr(&g_status, 1u);
        }
    };
    auto tokens = [&](int c) { return (int)min((int64_t)kT, u.t1 - u.t0 - (int64_t)c * kT); };
    // the chunk's first row in memory, counted from the sequence's
    auto first_row = [&](int c) {
        const int64_t t = u.t0 + (int64_t)c * kT;
        return reverse ? u.e.len - t - tokens(c) : t;
    };
    auto load_tiles = [&](int c) {  // thread 0
        uint8_t* at = smem + (c & 1) * S::kStage;
        uint64_t* bar = &bars[c & 1];
        tcu::mbar_arrive_expect_tx(bar, S::kStage);
        const int row = (int)(first_row(c) + (p.seqs.offsets ? u.e.row : 0)), b = p.seqs.offsets ? 0 : u.s;
#pragma unroll
        for (int i = 0; i < DK / 64; ++i) tcu::tma_load_4d(at + i * kTileBytes, &maps.k, bar, i * 64, h, row, b);
#pragma unroll
        for (int i = 0; i < DV / 64; ++i) tcu::tma_load_4d(at + S::kK + i * kTileBytes, &maps.v, bar, i * 64, h, row, b);
        if constexpr (OUT) {
#pragma unroll
            for (int i = 0; i < DK / 64; ++i) tcu::tma_load_4d(at + S::kK + S::kV + i * kTileBytes, &maps.q, bar, i * 64, h, row, b);
        }
    };
    // scores and q S of chunk c (thread 0)
    auto first_products = [&](int c) {
        const uint32_t kt = base + (c & 1) * S::kStage, qt = kt + S::kK + S::kV;
        wait(c & 1, (c >> 1) & 1);
        tcu::tc_fence_after_sync();
        constexpr uint32_t id = tcu::idesc_bf16_f32(128, 128), id_state = tcu::idesc_bf16_f32(128, DV) | kMajorB;
#pragma unroll
        for (int kk = 0; kk < DK / 16; ++kk) {
            const uint32_t at = (kk / 4) * kTileBytes + (kk % 4) * 32;
            tcu::mma_bf16(tmem + cScore, desc(qt + at, 16), desc(kt + at, 16), id, kk > 0);
        }
        if (has_state) {
#pragma unroll
            for (int kk = 0; kk < DK / 16; ++kk) {
                const uint32_t at = (kk / 4) * kTileBytes + (kk % 4) * 32;
                tcu::mma_bf16(tmem + cO2, desc(qt + at, 16), desc(state_addr + kk * 2048, DK * 128), id_state, kk > 0);
            }
        }
        tcu::mma_commit(&bars[2]);
    };

    if (tid == 0) {
        if (chunks > 0) load_tiles(0);
        if (chunks > 1) load_tiles(1);
        if (OUT && chunks > 0) first_products(0);
    }

    for (int c = 0; c < chunks; ++c) {
        const int n = tokens(c);
        const int entry = p.entry && u.t0 == 0 && c == 0;
        uint8_t* stage = smem + (c & 1) * S::kStage;
        uint8_t *kt = stage, *vt = stage + S::kK, *qt = vt + S::kV;
        uint8_t* plane1 = OUT ? qt : state;
        uint8_t* plane2 = OUT ? state : state + S::kK;
        const uint32_t vt_addr = tcu::smem_u32(vt);
        const bool more = c + 1 < chunks;
        // the state after the last chunk of a sequence is only wanted where it is handed out
        const bool update = !OUT || more || (p.final_state && u.t1 >= u.e.len);
        wait(c & 1, (c >> 1) & 1);
        if (n < kT) {  // rows of another sequence: their products with zeros must be zeros
            for (int i = tid; i < (kT - n) * (DV / 8); i += kThreads) {
                const int r = n + i / (DV / 8), ch = i % (DV / 8);
                *reinterpret_cast<uint4*>(vt + (ch / 8) * kTileBytes + r * 128 + (ch % 8) * 16) = make_uint4(0, 0, 0, 0);
            }
            tcu::fence_proxy_async_smem();
        }
        const int row = quad * 32 + lane;           // of the scores and outputs
        const int pos = reverse ? n - 1 - row : row;
        if constexpr (OUT) {
            wait(2, c & 1);
            tcu::tc_fence_after_sync();
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
                ld32(tmem_lane + cScore + j0, x);
                tcu::tmem_wait_ld();
                if (cb == quad || n < kT) {
                    const int d0 = reverse ? j0 - row : row - j0;
#pragma unroll
                    for (int i = 0; i < 32; i += 2) {
                        float v[2];
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const int d = reverse ? d0 + i + e : d0 - i - e;
                            const bool on = d >= 0 && j0 + i + e < n;
                            v[e] = on ? __uint_as_float(x[i + e]) * powk[on ? d : 0] : 0.f;
                        }
                        pw[blk][i / 2] = ssm::join(v[0], v[1], __nv_bfloat16{});
                    }
                } else {
                    // lambda^|i-j| = (from the row to the block's near edge) (within the block)
                    const float wr = power[reverse ? j0 - row : row - j0 - 31];
                    const float2 wr2 = splat2(wr);
#pragma unroll
                    for (int i = 0; i < 32; i += 2) {
                        const float2 wc = reverse ? make_float2(powk[i], powk[i + 1]) : make_float2(powk[31 - i], powk[30 - i]);
                        const float2 v = fmul2(make_float2(__uint_as_float(x[i]), __uint_as_float(x[i + 1])), fmul2(wr2, wc));
                        pw[blk][i / 2] = ssm::join(v.x, v.y, __nv_bfloat16{});
                    }
                }
            }
            // P takes the place of the scores' first half, which others may still be reading
            tcu::tc_fence_before_sync();
            __syncthreads();
            tcu::tc_fence_after_sync();
            st16(tmem_lane + cScore + half * 32, pw[0]);
            st16(tmem_lane + cScore + half * 32 + 16, pw[1]);
            wait_st();
            tcu::tc_fence_before_sync();
            __syncthreads();
            if (tid == 0) {
                tcu::tc_fence_after_sync();
                constexpr uint32_t id = tcu::idesc_bf16_f32(128, DV) | kMajorB;
                const int steps = (n + 15) / 16;
                for (int kk = 0; kk < steps; ++kk)
                    mma_ts(tmem + cO1, tmem + cScore + kk * 8, desc(vt_addr + kk * 2048, kTileBytes), id, kk > 0);
                tcu::mma_commit(&bars[3]);
            }
        }
        if (update) {
            // planes of the weighted keys; rows past the sequence become zeros
#pragma unroll 2
            for (int i = tid; i < kT * DK / 8; i += kThreads) {
                const int j = i / 8 % kT;
                const float w = j < n ? powk[reverse ? j : n - 1 - j] : 0.f;
                const uint4 x = *reinterpret_cast<const uint4*>(kt + i * 16);
                const uint32_t words[4] = {x.x, x.y, x.z, x.w};
                uint32_t out[3][4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float lo = __uint_as_float(words[e] << 16) * w, hi = __uint_as_float(words[e] & 0xffff0000u) * w;
                    if (j >= n) lo = hi = 0.f;
#pragma unroll
                    for (int pl = 0; pl < KP; ++pl) {
                        const uint32_t b = ssm::join(lo, hi, __nv_bfloat16{});
                        out[pl][e] = b;
                        lo -= __uint_as_float(b << 16);
                        hi -= __uint_as_float(b & 0xffff0000u);
                    }
                }
                *reinterpret_cast<uint4*>(kt + i * 16) = make_uint4(out[0][0], out[0][1], out[0][2], out[0][3]);
                *reinterpret_cast<uint4*>(plane1 + i * 16) = make_uint4(out[1][0], out[1][1], out[1][2], out[1][3]);
                if constexpr (KP == 3)
                    *reinterpret_cast<uint4*>(plane2 + i * 16) = make_uint4(out[2][0], out[2][1], out[2][2], out[2][3]);
            }
            tcu::fence_proxy_async_smem();
            tcu::tc_fence_before_sync();
            __syncthreads();
            if (tid == 0) {
                tcu::tc_fence_after_sync();
                // 64 keys: a lead of 0 puts them into both halves of the 128 rows
                constexpr uint32_t id = tcu::idesc_bf16_f32(128, DV) | kMajorA | kMajorB, lead = DK == 128 ? kTileBytes : 0;
                const int steps = (n + 15) / 16;
                bool sum = false;
#pragma unroll
                for (int pl = KP - 1; pl >= 0; --pl) {
                    const uint32_t at = tcu::smem_u32(pl == 0 ? kt : pl == 1 ? plane1 : plane2);
                    for (int kk = 0; kk < steps; ++kk) {
                        tcu::mma_bf16(tmem + cU, desc(at + kk * 2048, lead), desc(vt_addr + kk * 2048, kTileBytes), id, sum);
                        sum = true;
                    }
                }
                tcu::mma_commit(&bars[4]);
            }
        }
        // this row's outputs, DV / 2 columns
        uint32_t out[DV / 4];
        if constexpr (OUT) {
            wait(3, c & 1);
            tcu::tc_fence_after_sync();
            const float wi = row < n ? power[pos + 1 - entry] : 0.f;
#pragma unroll
            for (int blk = 0; blk < DV / 64; ++blk) {
                const int c0 = half * (DV / 2) + blk * 32;
                uint32_t x[32], y[32];
                ld32(tmem_lane + cO1 + c0, x);
                if (has_state) ld32(tmem_lane + cO2 + c0, y);
                tcu::tmem_wait_ld();
                bool odd = false;
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    float v = __uint_as_float(x[i]);
                    odd |= !(fabsf(v) <= 3.4028234e38f);
                    if (has_state) v = fmaf(__uint_as_float(y[i]), wi, v);
                    x[i] = __float_as_uint(v);
                }
                // A value that is not finite must not reach the rows before it: 0 times it is NaN in the
                // product.  Such chunks are rare; their rows are summed again, term by term.
                if (__any_sync(0xffffffffu, odd)) {
                    float sum[32];
#pragma unroll
                    for (int i = 0; i < 32; ++i) sum[i] = has_state ? __uint_as_float(y[i]) * wi : 0.f;
                    for (int j0 = 0; j0 < n; j0 += 32) {
                        float pr[16];
                        tcu::tmem_ld16(tmem_lane + cScore + j0 / 2, pr);
                        tcu::tmem_wait_ld();
#pragma unroll
                        for (int jj = 0; jj < 32; ++jj) {
                            const int j = j0 + jj;
                            const uint32_t w = __float_as_uint(pr[jj / 2]);
                            const float pv = __uint_as_float(jj & 1 ? w & 0xffff0000u : w << 16);
                            if (j < n && (reverse ? j >= row : j <= row)) {
#pragma unroll
                                for (int i = 0; i < 32; ++i) {
                                    const int cc = c0 + i;
                                    const uint16_t b = *reinterpret_cast<const uint16_t*>(
                                        vt + (cc / 64) * kTileBytes + j * 128 + (((cc % 64) / 8) ^ (j & 7)) * 16 + (cc % 8) * 2);
                                    sum[i] = fmaf(pv, __uint_as_float((uint32_t)b << 16), sum[i]);
                                }
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
        }
        if (update) {
            wait(4, c & 1);
            tcu::tc_fence_after_sync();
            const float w = power[n - entry];
#pragma unroll
            for (int i0 = 0; i0 < NC; i0 += 16) {
                float x[16];
                tcu::tmem_ld16(tmem_lane + cU + b0 + i0, x);
                tcu::tmem_wait_ld();
#pragma unroll
                for (int i = 0; i < 16; ++i) s[i0 + i] = fmaf(s[i0 + i], w, x[i]);
            }
            has_state = true;
            if (OUT && more) put_state();
        }
        tcu::tc_fence_before_sync();
        __syncthreads();
        if (OUT && more && tid == 0) {
            tcu::tc_fence_after_sync();
            first_products(c + 1);
        }
        if constexpr (OUT) {
            // the rows of o through shared memory (where K was), 16 bytes in eight places by row
#pragma unroll
            for (int i = 0; i < DV / 16; ++i) {
                const int ch = half * (DV / 16) + i;
                *reinterpret_cast<uint4*>(kt + (ch / 8) * kTileBytes + row * 128 + ((ch % 8) ^ (row & 7)) * 16) =
                    make_uint4(out[4 * i], out[4 * i + 1], out[4 * i + 2], out[4 * i + 3]);
            }
            __syncthreads();
            const int64_t step = (int64_t)p.heads * p.dv;
            __nv_bfloat16* to = static_cast<__nv_bfloat16*>(p.o) + (u.e.row + first_row(c)) * step + (int64_t)h * p.dv;
            for (int i = tid; i < n * (DV / 8); i += kThreads) {
                const int r = i / (DV / 8), ch = i % (DV / 8);
                if (ch * 8 >= p.dv) continue;
                const uint4 v = *reinterpret_cast<const uint4*>(kt + (ch / 8) * kTileBytes + r * 128 + ((ch % 8) ^ (r & 7)) * 16);
                *reinterpret_cast<uint4*>(to + r * step + ch * 8) = v;
            }
            tcu::fence_proxy_async_smem();
            __syncthreads();
        }
        if (tid == 0 && c + 2 < chunks) {
            tcu::fence_proxy_async_smem();
            load_tiles(c + 2);
        }
    }

    float* to = nullptr;
    float last = 1.f;
    if constexpr (OUT) {
        if (p.final_state && u.t1 >= u.e.len) {
            to = p.final_state + ((int64_t)u.s * p.heads + h) * states;
            if (p.exit_decay && u.e.len > 0) last = decay_power(log_decay, 1);
        }
    } else {
        to = p.states + (u.slot * p.heads + h) * states;
    }
    if (to && a < p.dk) {
#pragma unroll
        for (int i = 0; i < NC; ++i)
            if (b0 + i < p.dv) to[(int64_t)a * p.dv + b0 + i] = s[i] * last;
    }
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

template <int DK, int DV, int KP, bool OUT>
int launch(const Params& p, const Maps& m, int64_t units, cudaStream_t st) {
    using L = Smem<DK, DV, KP, OUT>;
    const void* fn = reinterpret_cast<const void*>(&tc_kernel<DK, DV, KP, OUT>);
    if (!ensure_smem_attr(fn, L::kLaunch)) return fail(VH_E_DEVICE, "linear attention: shared memory");
    tc_kernel<DK, DV, KP, OUT><<<dim3((unsigned)units, p.heads), kThreads, L::kLaunch, st>>>(p, m);
    return launch_status(OUT ? "linear attention" : "linear attention: segment states");
}

template <int DK, int DV>
int run_dims(const Params& p, const Maps& m, int64_t units, bool exact, cudaStream_t st) {
    if (p.segment) {
        if (int rc = exact ? launch<DK, DV, 3, false>(p, m, units, st) : launch<DK, DV, 2, false>(p, m, units, st)) return rc;
        if (int rc = enter_segments(p, st)) return rc;
    }
    return exact ? launch<DK, DV, 3, true>(p, m, units, st) : launch<DK, DV, 2, true>(p, m, units, st);
}

}  // namespace

// CTAs fill the card once: one an SM, two where keys and values are at most 64.  Chains that are fewer
// than half of them are cut; packed sequences always are, as the host does not know their lengths.
int tc_segment_size(int64_t length, int batch, bool packed, int heads, int dk, int dv) {
    const int64_t ctas = (int64_t)sm_count() * (dk <= 64 && dv <= 64 ? 2 : 1), chains = (int64_t)batch * heads;
    int64_t size;
    if (packed) {
        size = (length * heads + ctas - 1) / ctas;
    } else {
        const int64_t segs = ctas / chains;
        if (segs < 2) return 0;
        size = (length + segs - 1) / segs;
    }
    size = std::max<int64_t>((size + kT - 1) / kT * kT, 4 * kT);
    return size < length ? (int)size : 0;
}

bool tc_run(Params p, void* states, cudaStream_t st, int* rc) {
    if (p.q.vec != 8 || p.k.vec != 8 || p.v.vec != 8 || p.vec_o != 8 || p.seqs.length < kT || !encoder()) return false;
    Maps m;
    if (!encode(&m.q, p.q, p, p.dk) || !encode(&m.k, p.k, p, p.dk) || !encode(&m.v, p.v, p, p.dv)) return false;
    const bool packed = p.seqs.offsets != nullptr, exact = p.final_state != nullptr;
    p.segment = tc_segment_size(p.seqs.length, p.seqs.count, packed, p.heads, p.dk, p.dv);
    p.states = static_cast<float*>(states);
    const int64_t units = p.segment ? ssm::slot_total(packed, p.seqs.length, p.seqs.count, p.segment) : p.seqs.count;
    if (p.dk <= 64) *rc = p.dv <= 64 ? run_dims<64, 64>(p, m, units, exact, st) : run_dims<64, 128>(p, m, units, exact, st);
    else *rc = p.dv <= 64 ? run_dims<128, 64>(p, m, units, exact, st) : run_dims<128, 128>(p, m, units, exact, st);
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
