// Linear attention with a decay for each head: whole and packed sequences, their gradients, and one
// token of cached streams.  The mathematics is in linear_attention.cuh.
#include <algorithm>

#include "abi_util.h"
#include "linear_attention.cuh"
#include "vhope.h"

namespace vh {
namespace lin {
namespace {

constexpr int kThreads = 128;

// ---- operands in 16 bits ------------------------------------------------------------------------
// The matrix products run on bf16 operands with fp32 sums.  An operand is NP planes that add up to
// its value: one for bf16 inputs (exact), two for fp16 (11 bits, exact), three for fp32 (24 bits,
// exact).  Each plane is the rounded rest of the ones before it, at most 2^-8 of their sum.  Products of
// planes a and b are kept while a + b < NP, which drops at most 2^-16 (two planes) or 2^-24 (three) of a
// product, with either sign.
template <typename T> constexpr int kPlanes = 3;
template <> constexpr int kPlanes<__nv_bfloat16> = 1;
template <> constexpr int kPlanes<__half> = 2;

template <int NP>
__device__ __forceinline__ void split2(float a, float b, uint32_t (&out)[NP]) {
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        out[i] = *reinterpret_cast<const uint32_t*>(&h);
        if (i + 1 < NP) {
            a -= __uint_as_float(out[i] << 16);
            b -= __uint_as_float(out[i] & 0xffff0000u);
        }
    }
}

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], const void* p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"((uint32_t)__cvta_generic_to_shared(p))
                 : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], const void* p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"((uint32_t)__cvta_generic_to_shared(p))
                 : "memory");
}
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// c += the products of planes of one k-step.  The matrix unit truncates its sums (a bias of up to 2^-23 of
// the sum for each instruction), so where several planes make up a value, or a sum lives on from chunk to
// chunk, a k-step is summed from zero, its small products first, and added to c by a rounded addition.
template <int NA, int NB, int KEEP>
__device__ __forceinline__ void product(float (&c0)[4], float (&c1)[4], const uint32_t (&a)[NA][4], const uint32_t (&b)[NB][4]) {
    if constexpr (NA == 1 && NB == 1) {
        mma(c0, a[0], b[0][0], b[0][1]);
        mma(c1, a[0], b[0][2], b[0][3]);
    } else {
        float d0[4] = {}, d1[4] = {};
#pragma unroll
        for (int sum = KEEP - 1; sum >= 0; --sum)
#pragma unroll
            for (int i = 0; i < NA; ++i) {
                const int j = sum - i;
                if (j < 0 || j >= NB) continue;
                mma(d0, a[i], b[j][0], b[j][1]);
                mma(d1, a[i], b[j][2], b[j][3]);
            }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            c0[i] += d0[i];
            c1[i] += d1[i];
        }
    }
}

// ---- shared memory ------------------------------------------------------------------------------
// Rows are 16 bytes longer than they hold, so that the eight rows of a matrix load lie in different
// banks.
template <typename T, int DK, bool OUT>
struct Layout {
    static constexpr int kNP = kPlanes<T>;
    static constexpr int kStages = kNP == 1 ? 2 : 1;
    static constexpr int kPitch = DK + 8, kVPitch = kTile + 8;
    static constexpr int kQ = kChunk * kPitch, kV = kChunk * kVPitch, kS = DK * kVPitch;  // elements a plane
    static constexpr int kStage = kNP * ((OUT ? 2 : 1) * kQ + kV);
    static constexpr int kElements = kStages * kStage + (OUT ? kNP * kS : 0);
    static constexpr size_t kBytes = (size_t)kElements * 2 + 2 * (kChunk + 2) * sizeof(float);
};

// Rows [0, n) of a tile of 64 tokens by W columns, of which `dim` exist, into its planes; the others are
// zero.  bf16 rows with aligned 16-byte pieces are copied asynchronously.
template <typename T, int W, int PITCH, int PLANE>
__device__ __forceinline__ void load_tile(uint16_t* dst, const T* src, int64_t step, int n, int dim, int vec) {
    constexpr int NP = kPlanes<T>;
    if constexpr (NP == 1) {
        if (vec == 8) {
            for (int i = threadIdx.x; i < kChunk * (W / 8); i += kThreads) {
                const int r = i / (W / 8), c = i % (W / 8) * 8;
                const bool live = r < n && c < dim;
                cp_async16_zfill(dst + r * PITCH + c, live ? src + r * step + c : src, live);
            }
            return;
        }
    }
    auto put = [&](int r, int c, const float (&v)[4]) {
        uint32_t lo[NP], hi[NP];
        split2<NP>(v[0], v[1], lo);
        split2<NP>(v[2], v[3], hi);
#pragma unroll
        for (int pl = 0; pl < NP; ++pl) *reinterpret_cast<uint2*>(dst + pl * PLANE + r * PITCH + c) = make_uint2(lo[pl], hi[pl]);
    };
    if (vec >= 4) {
        // several loads before the first is split; the places that do not exist read the tile's first
        constexpr int kAhead = 8;
#pragma unroll 1
        for (int i0 = threadIdx.x; i0 < kChunk * (W / 4); i0 += kAhead * kThreads) {
            float4 f[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                const int i = i0 + k * kThreads, r = i / (W / 4), c = i % (W / 4) * 4;
                f[k] = load4(r < n && c < dim ? src + r * step + c : src);
            }
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                const int i = i0 + k * kThreads, r = i / (W / 4), c = i % (W / 4) * 4;
                const bool live = r < n && c < dim;
                const float v[4] = {live ? f[k].x : 0.f, live ? f[k].y : 0.f, live ? f[k].z : 0.f, live ? f[k].w : 0.f};
                put(r, c, v);
            }
        }
        return;
    }
#pragma unroll 4
    for (int i = threadIdx.x; i < kChunk * (W / 4); i += kThreads) {
        const int r = i / (W / 4), c = i % (W / 4) * 4;
        float v[4] = {0.f, 0.f, 0.f, 0.f};
        if (r < n) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (c + e < dim) v[e] = to_f(src[r * step + c + e]);
        }
        put(r, c, v);
    }
}

// A chain, or a segment of one: a CTA walks its chunks, the state in the accumulators of its four
// warps (each a quarter of the key rows by 64 value columns) and, for the outputs, as a bf16 operand
// in shared memory.  OUT false computes only what the segment adds to the state.
//
// Four warps, because a chunk of 64 rows gives each of them 16 whole rows of scores, which then never leave its
// registers; 64 value columns, so that a state of 128 keys fits the accumulators.  Bound by latency (three
// sequences of 785 tokens, 5 heads of 48 and 72 in fp32, forward and backward: 186 us, tensor pipe 15 %).
//
// The state itself is fp32 throughout: a key's weight lambda^{n-1-j} is multiplied in fp32 and the
// product enters as three planes, so nothing of it is rounded.  As an operand of the outputs the
// state is rounded to NP planes, and so are the weighted scores: for bf16 inputs that is one rounding
// of 2^-9 on each term of o, as large as the rounding of o itself and independent of it.
template <typename T, int DK, bool OUT>
__global__ void __launch_bounds__(kThreads) chunk_kernel(Params p) {
    using L = Layout<T, DK, OUT>;
    constexpr int NP = L::kNP, P = L::kPitch, VP = L::kVPitch, MT = DK / 64;
    extern __shared__ __align__(16) uint16_t smem[];
    uint16_t* state = smem + L::kStages * L::kStage;
    float* power = reinterpret_cast<float*>(smem + L::kElements);  // lambda^n, n = 0..64
    float* powk = power + kChunk + 2;                              // times kv_scale

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t2 = (lane & 3) * 2;
    const int h = blockIdx.y, col0 = blockIdx.z * kTile, cols = min(kTile, p.dv - col0);
    const Unit u = block_unit(p, reinterpret_cast<int*>(power + kChunk + 1));
    if constexpr (OUT) {
        const int64_t block = ((int64_t)blockIdx.x * gridDim.y + h) * gridDim.z + blockIdx.z;
        ssm::zero_outside<T>(p.seqs, p.heads * p.dv, block, (int64_t)gridDim.x * gridDim.y * gridDim.z, p.o);
    }
    // the state after a sequence's last segment is nobody's start
    if (!u.live || (!OUT && u.t1 >= u.e.len)) return;

    const float log_decay = p.log_decay[h];
    if (tid <= kChunk) {
        const float w = decay_power(log_decay, tid);
        power[tid] = w;
        powk[tid] = w * p.kv_scale;
    }
    const T* q = static_cast<const T*>(p.q.p) + ssm::first_row(p.seqs, u.e, u.s, p.q.rows) + h * p.q.head;
    const T* k = static_cast<const T*>(p.k.p) + ssm::first_row(p.seqs, u.e, u.s, p.k.rows) + h * p.k.head;
    const T* v = static_cast<const T*>(p.v.p) + ssm::first_row(p.seqs, u.e, u.s, p.v.rows) + h * p.v.head + col0;
    const int64_t qs = ssm::row_step(p.seqs, p.q.rows), ks = ssm::row_step(p.seqs, p.k.rows),
                  vs = ssm::row_step(p.seqs, p.v.rows);

    // entering state: rows warp * DK / 4 + 16 mt + g (+ 8), columns 8 nt + t2 (+ 1)
    float s[MT][8][4];
    const bool first = u.t0 == 0;
    const int64_t states = (int64_t)p.dk * p.dv;
    const float* from = nullptr;
    int64_t fa = p.dv, fb = 1;
    if (OUT) {
        if (first) {
            from = p.initial ? p.initial + ((int64_t)u.s * p.heads + h) * states : nullptr;
            fa = p.init_a;
            fb = p.init_b;
        } else {
            from = p.states + (u.slot * p.heads + h) * states;
        }
    }
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int nt = 0; nt < 8; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int a = warp * (DK / 4) + mt * 16 + g + (e >> 1) * 8, b = nt * 8 + t2 + (e & 1);
                s[mt][nt][e] = from && a < p.dk && b < cols ? from[a * fa + (col0 + b) * fb] : 0.f;
            }
    bool has_state = from != nullptr;
    auto put_state = [&] {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int nt = 0; nt < 8; ++nt)
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    uint32_t w[NP];
                    split2<NP>(s[mt][nt][2 * half], s[mt][nt][2 * half + 1], w);
                    const int a = warp * (DK / 4) + mt * 16 + g + half * 8;
#pragma unroll
                    for (int pl = 0; pl < NP; ++pl)
                        *reinterpret_cast<uint32_t*>(state + pl * L::kS + a * VP + nt * 8 + t2) = w[pl];
                }
    };
    if (OUT && has_state) put_state();

    const int64_t tokens = u.t1 - u.t0;
    const int chunks = (int)((tokens + kChunk - 1) / kChunk);
    auto load_chunk = [&](int c) {
        const int64_t t = u.t0 + (int64_t)c * kChunk;
        const int n = (int)min((int64_t)kChunk, u.t1 - t);
        uint16_t* at = smem + (L::kStages == 2 && (c & 1) ? L::kStage : 0);
        load_tile<T, DK, P, L::kQ>(at, k + t * ks, ks, n, p.dk, p.k.vec);
        at += NP * L::kQ;
        load_tile<T, kTile, VP, L::kV>(at, v + t * vs, vs, n, cols, p.v.vec);
        at += NP * L::kV;
        if constexpr (OUT) load_tile<T, DK, P, L::kQ>(at, q + t * qs, qs, n, p.dk, p.q.vec);
        cp_async_commit();
    };
    if (L::kStages == 2 && chunks > 0) load_chunk(0);

    for (int c = 0; c < chunks; ++c) {
        const int64_t t = u.t0 + (int64_t)c * kChunk;
        const int n = (int)min((int64_t)kChunk, u.t1 - t);
        // a state that enters the sequence without a decay counts one power less in its first chunk
        const int entry = p.entry && t == 0;
        if (L::kStages == 2) {
            if (c + 1 < chunks) load_chunk(c + 1); else cp_async_commit();
            cp_async_wait<1>();
        } else {
            load_chunk(c);
        }
        __syncthreads();
        const uint16_t* kt = smem + (L::kStages == 2 && (c & 1) ? L::kStage : 0);
        const uint16_t* vt = kt + NP * L::kQ;
        if constexpr (OUT) {
            uint16_t* qt = const_cast<uint16_t*>(vt) + NP * L::kV;
            const int row0 = warp * 16;
            float o[8][4] = {}, sc[8][4] = {};
            // q S_0 and the scores q k^T, up to the diagonal
            auto from_state = [&](int kk, const uint32_t (&qa)[NP][4]) {
#pragma unroll
                for (int np = 0; np < 4; ++np) {
                    uint32_t b[NP][4];
#pragma unroll
                    for (int pb = 0; pb < NP; ++pb)
                        ldsm4t(b[pb], state + pb * L::kS + (kk * 16 + (lane & 15)) * VP + np * 16 + (lane >> 4) * 8);
                    product<NP, NP, NP>(o[2 * np], o[2 * np + 1], qa, b);
                }
            };
            auto load_q = [&](int kk, uint32_t (&qa)[NP][4]) {
#pragma unroll
                for (int pa = 0; pa < NP; ++pa)
                    ldsm4(qa[pa], qt + pa * L::kQ + (row0 + (lane & 15)) * P + kk * 16 + (lane >> 4) * 8);
            };
#pragma unroll
            for (int kk = 0; kk < DK / 16; ++kk) {
                uint32_t qa[NP][4];
                load_q(kk, qa);
                if (has_state) from_state(kk, qa);
#pragma unroll
                for (int np = 0; np < 4; ++np) {
                    if (np > warp) continue;
                    uint32_t b[NP][4];
#pragma unroll
                    for (int pb = 0; pb < NP; ++pb)
                        ldsm4(b[pb], kt + pb * L::kQ + (np * 16 + (lane & 7) + (lane >> 4) * 8) * P + kk * 16 + ((lane >> 3) & 1) * 8);
                    product<NP, NP, NP>(sc[2 * np], sc[2 * np + 1], qa, b);
                }
            }
            const int i0 = row0 + g, i1 = i0 + 8;
            // a NaN of the state stays one where its power is 0
            const float w0 = power[i0 + 1 - entry], w1 = power[i1 + 1 - entry];
            auto decay_rows = [&] {
#pragma unroll
                for (int nt = 0; nt < 8; ++nt) {
                    o[nt][0] *= w0; o[nt][1] *= w0;
                    o[nt][2] *= w1; o[nt][3] *= w1;
                }
            };
            if (has_state) decay_rows();
            // weighted scores as operands; what lies ahead of a row is selected away, not multiplied
            uint32_t pa_[4][NP][4];
#pragma unroll
            for (int np = 0; np < 4; ++np) {
                if (np > warp) continue;
#pragma unroll
                for (int hv = 0; hv < 2; ++hv) {
                    const int j = np * 16 + hv * 8 + t2;
                    float (&x)[4] = sc[2 * np + hv];
                    x[0] = i0 >= j ? x[0] * powk[i0 - j] : 0.f;
                    x[1] = i0 >= j + 1 ? x[1] * powk[i0 - j - 1] : 0.f;
                    x[2] = i1 >= j ? x[2] * powk[i1 - j] : 0.f;
                    x[3] = i1 >= j + 1 ? x[3] * powk[i1 - j - 1] : 0.f;
                    uint32_t lo[NP], hi[NP];
                    split2<NP>(x[0], x[1], lo);
                    split2<NP>(x[2], x[3], hi);
#pragma unroll
                    for (int pl = 0; pl < NP; ++pl) {
                        pa_[np][pl][2 * hv] = lo[pl];
                        pa_[np][pl][2 * hv + 1] = hi[pl];
                    }
                }
#pragma unroll
                for (int nq = 0; nq < 4; ++nq) {
                    uint32_t b[NP][4];
#pragma unroll
                    for (int pb = 0; pb < NP; ++pb)
                        ldsm4t(b[pb], vt + pb * L::kV + (np * 16 + (lane & 15)) * VP + nq * 16 + (lane >> 4) * 8);
                    product<NP, NP, NP>(o[2 * nq], o[2 * nq + 1], pa_[np], b);
                }
            }
            // A value that is not finite must not reach the rows before it: 0 times it is NaN in the
            // product above.  Such chunks are rare; their rows are summed again, term by term.
            bool odd = false;
#pragma unroll
            for (int nt = 0; nt < 8; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) odd |= !(fabsf(o[nt][e]) <= 3.4028234e38f);
            if (__any_sync(0xffffffffu, odd)) {
#pragma unroll
                for (int nt = 0; nt < 8; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[nt][e] = 0.f;
                if (has_state) {
#pragma unroll
                    for (int kk = 0; kk < DK / 16; ++kk) {
                        uint32_t qa[NP][4];
                        load_q(kk, qa);
                        from_state(kk, qa);
                    }
                    decay_rows();
                }
#pragma unroll
                for (int nj = 0; nj < 8; ++nj) {
                    if (nj / 2 > warp) continue;
#pragma unroll
                    for (int jj = 0; jj < 8; ++jj) {
                        const int j = nj * 8 + jj, src = g * 4 + jj / 2;
                        const float p0 = __shfl_sync(0xffffffffu, sc[nj][jj & 1], src);
                        const float p1 = __shfl_sync(0xffffffffu, sc[nj][2 + (jj & 1)], src);
#pragma unroll
                        for (int nt = 0; nt < 8; ++nt)
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                float x = 0.f;
#pragma unroll
                                for (int pl = NP - 1; pl >= 0; --pl)
                                    x += __uint_as_float((uint32_t)vt[pl * L::kV + j * VP + nt * 8 + t2 + e] << 16);
                                if (i0 >= j) o[nt][e] = fmaf(p0, x, o[nt][e]);
                                if (i1 >= j) o[nt][2 + e] = fmaf(p1, x, o[nt][2 + e]);
                            }
                    }
                }
            }
            // rows of o; 16-bit ones through the warp's own query rows, which it has read, into whole lines
            const int64_t out_step = (int64_t)p.heads * p.dv;
            T* out = static_cast<T*>(p.o) + (u.e.row + (p.seqs.reverse ? u.e.len - 1 - t : t)) * out_step + (int64_t)h * p.dv + col0;
            const int64_t os = p.seqs.reverse ? -out_step : out_step;
            bool staged = false;
            if constexpr (sizeof(T) == 2) {
                if (p.vec_o == 8) {
                    staged = true;
                    __syncwarp();
#pragma unroll
                    for (int nt = 0; nt < 8; ++nt)
#pragma unroll
                        for (int half = 0; half < 2; ++half)
                            *reinterpret_cast<uint32_t*>(qt + (row0 + g + half * 8) * P + nt * 8 + t2) =
                                ssm::join(o[nt][2 * half] * p.out_scale, o[nt][2 * half + 1] * p.out_scale, T{});
                    __syncwarp();
#pragma unroll
                    for (int it = 0; it < 4; ++it) {
                        const int r = row0 + it * 4 + (lane >> 3), cc = (lane & 7) * 8;
                        if (r < n && cc < cols)
                            *reinterpret_cast<uint4*>(out + r * os + cc) = *reinterpret_cast<const uint4*>(qt + r * P + cc);
                    }
                }
            }
            if (!staged) {
#pragma unroll
                for (int nt = 0; nt < 8; ++nt)
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const int r = row0 + g + half * 8, cc = nt * 8 + t2;
                        T* at = out + r * os + cc;
                        const float a = o[nt][2 * half] * p.out_scale, b = o[nt][2 * half + 1] * p.out_scale;
                        if (r >= n) continue;
                        if (sizeof(T) == 4 && p.vec_o >= 4) {
                            if (cc < cols) *reinterpret_cast<float2*>(at) = make_float2(a, b);
                        } else {
                            if (cc < cols) at[0] = from_f<T>(a);
                            if (cc + 1 < cols) at[1] = from_f<T>(b);
                        }
                    }
            }
        }
        // the state after the chunk
        {
            const float w = power[n - entry];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int nt = 0; nt < 8; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[mt][nt][e] *= w;
#pragma unroll
            for (int kk = 0; kk < kChunk / 16; ++kk) {
                if (kk * 16 >= n) continue;
                float wt[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int j = kk * 16 + t2 + (e & 1) + (e >> 1) * 8;
                    wt[e] = j < n ? powk[n - 1 - j] : 0.f;
                }
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    float x[8] = {};
#pragma unroll
                    for (int pl = NP - 1; pl >= 0; --pl) {
                        uint32_t r[4];
                        ldsm4t(r, kt + pl * L::kQ + (kk * 16 + (lane & 7) + (lane >> 4) * 8) * P + warp * (DK / 4) + mt * 16 +
                                      ((lane >> 3) & 1) * 8);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            x[2 * i] += __uint_as_float(r[i] << 16);
                            x[2 * i + 1] += __uint_as_float(r[i] & 0xffff0000u);
                        }
                    }
                    uint32_t a[3][4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        uint32_t w3[3];
                        split2<3>(x[2 * i] * wt[(i >> 1) * 2], x[2 * i + 1] * wt[(i >> 1) * 2 + 1], w3);
#pragma unroll
                        for (int pl = 0; pl < 3; ++pl) a[pl][i] = w3[pl];
                    }
#pragma unroll
                    for (int np = 0; np < 4; ++np) {
                        uint32_t b[NP][4];
#pragma unroll
                        for (int pb = 0; pb < NP; ++pb)
                            ldsm4t(b[pb], vt + pb * L::kV + (kk * 16 + (lane & 15)) * VP + np * 16 + (lane >> 4) * 8);
                        product<3, NP, 3>(s[mt][2 * np], s[mt][2 * np + 1], a, b);
                    }
                }
            }
        }
        has_state = true;
        __syncthreads();
        if (OUT && c + 1 < chunks) put_state();
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
    if (!to) return;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int nt = 0; nt < 8; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int a = warp * (DK / 4) + mt * 16 + g + (e >> 1) * 8, b = nt * 8 + t2 + (e & 1);
                if (a < p.dk && b < cols) to[(int64_t)a * p.dv + col0 + b] = s[mt][nt][e] * last;
            }
}

// From what each segment adds to the state before each of them, in place: a thread per element walks the
// segments of its sequence, 16 loads ahead (one pass over memory, bound by its latency; four elements a thread
// took 5.7 us instead of 3.7 for 32 segments of 8 chains of 64 x 64).
constexpr int kEnterAhead = 16;
__global__ void __launch_bounds__(256) enter_kernel(Params p) {
    const int s = blockIdx.x, h = blockIdx.y;
    const int states = p.dk * p.dv, i = blockIdx.z * 256 + threadIdx.x;
    const Seq e = ssm::seq_at(p.seqs, s);
    if (i >= states || e.len <= p.segment) return;
    const int64_t base = ssm::slot_base(p.seqs, s, e.row, p.segment);
    const float g = p.log_decay[h], step = decay_power(g, p.segment);
    const int a = i / p.dv, b = i - a * p.dv;
    float run = p.initial ? p.initial[((int64_t)s * p.heads + h) * states + a * p.init_a + b * p.init_b] : 0.f;
    float w = p.entry ? decay_power(g, p.segment - 1) : step;
    float* at = p.states + (base * p.heads + h) * states + i;
    const int64_t stride = (int64_t)p.heads * states;
    const int segs = (int)((e.len + p.segment - 1) / p.segment);
    float own[kEnterAhead];
    int j = 0;
    for (; j + kEnterAhead < segs; j += kEnterAhead) {
#pragma unroll
        for (int x = 0; x < kEnterAhead; ++x) own[x] = at[(j + x) * stride];
#pragma unroll
        for (int x = 0; x < kEnterAhead; ++x) {
            at[(j + x) * stride] = run;
            run = run * w + own[x];
            w = step;
        }
    }
#pragma unroll
    for (int x = 0; x < kEnterAhead; ++x) {  // the last segment adds to nobody's start
        if (j + x + 1 >= segs) break;
        own[x] = at[(j + x) * stride];
    }
#pragma unroll
    for (int x = 0; x < kEnterAhead; ++x) {
        if (j + x >= segs) break;
        at[(j + x) * stride] = run;
        if (j + x + 1 < segs) run = run * w + own[x];
        w = step;
    }
}

// ---- one token ----------------------------------------------------------------------------------
struct StepParams {
    Heads q, k, v;
    const float* log_decay;
    const float* state;
    float* state_out;
    const int32_t* slots_index;
    void* o;
    float scale;
    int32_t slots, batch, heads, dk, dv;
};

// A CTA per (stream, head): the state is read and written once, four columns a thread (V = 4) over key rows that
// the row groups share; the sums over key rows meet in shared memory.  Bound by the state's bytes (8 per
// element): 256 streams of 16 heads of 128 x 128 in 91 us, 5.9 TB/s.
template <typename T, int V>
__global__ void __launch_bounds__(256) step_kernel(StepParams p) {
    __shared__ float ks[kMaxDim], qs[kMaxDim];
    __shared__ float part[256 * V];
    const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
    const int slot = p.slots_index ? p.slots_index[b] : b;
    T* o = static_cast<T*>(p.o) + ((int64_t)b * p.heads + h) * p.dv;
    if (slot < 0 || slot >= p.slots) {
        for (int c = tid; c < p.dv; c += 256) o[c] = from_f<T>(0.f);
        return;
    }
    const float lambda = decay_power(p.log_decay[h], 1);
    const T* q = static_cast<const T*>(p.q.p) + (int64_t)b * p.q.rows.batch + h * p.q.head;
    const T* k = static_cast<const T*>(p.k.p) + (int64_t)b * p.k.rows.batch + h * p.k.head;
    const T* v = static_cast<const T*>(p.v.p) + (int64_t)b * p.v.rows.batch + h * p.v.head;
    for (int c = tid; c < p.dk; c += 256) {
        ks[c] = to_f(k[c]);
        qs[c] = to_f(q[c]);
    }
    __syncthreads();
    const int lanes = (p.dv + V - 1) / V, groups = 256 / lanes, gr = tid / lanes, c = tid % lanes * V;
    const int64_t base = ((int64_t)slot * p.heads + h) * p.dk * p.dv;
    float acc[V] = {}, vv[V];
#pragma unroll
    for (int e = 0; e < V; ++e) vv[e] = to_f(v[c + e]);
    if (gr < groups) {
#pragma unroll 4
        for (int r = gr; r < p.dk; r += groups) {
            const int64_t at = base + (int64_t)r * p.dv + c;
            float x[V];
            if constexpr (V == 4) {
                const float4 f = *reinterpret_cast<const float4*>(p.state + at);
                x[0] = f.x; x[1] = f.y; x[2] = f.z; x[3] = f.w;
            } else {
                x[0] = p.state[at];
            }
#pragma unroll
            for (int e = 0; e < V; ++e) {
                x[e] = fmaf(lambda, x[e], ks[r] * vv[e]);
                acc[e] = fmaf(qs[r], x[e], acc[e]);
            }
            if constexpr (V == 4) *reinterpret_cast<float4*>(p.state_out + at) = make_float4(x[0], x[1], x[2], x[3]);
            else p.state_out[at] = x[0];
        }
#pragma unroll
        for (int e = 0; e < V; ++e) part[gr * lanes * V + c + e] = acc[e];
    }
    __syncthreads();
    for (int i = tid; i < p.dv; i += 256) {
        float sum = 0.f;
        for (int r = 0; r < groups; ++r) sum += part[r * lanes * V + i];
        o[i] = from_f<T>(sum * p.scale);
    }
}

// ---- host ---------------------------------------------------------------------------------------
template <typename F>
int with_dtype(int dtype, F&& f) {
    if (dtype == VH_F32) return f(float{});
    if (dtype == VH_BF16) return f(__nv_bfloat16{});
    return f(__half{});
}

int check_sizes(const char* what, const vh_linear_attention_args* a, bool one_token) {
    if (!a) return fail(VH_E_ARG, "%s: null argument struct", what);
    if (!dtype_ok(a->dtype)) return fail(VH_E_DTYPE, "%s: dtype must be VH_F32, VH_BF16 or VH_F16", what);
    if (a->batch <= 0 || a->heads <= 0) return fail(VH_E_SHAPE, "%s: batch and heads must be positive", what);
    if (a->heads > 65535) return fail(VH_E_RANGE, "%s: at most 65535 heads", what);
    if (a->key_dim <= 0 || a->key_dim > kMaxDim || a->value_dim <= 0 || a->value_dim > kMaxDim)
        return fail(VH_E_SHAPE, "%s: key and value dims must be 1 to %d (got %d and %d)", what, kMaxDim, a->key_dim, a->value_dim);
    if (one_token) {
        if (a->batch > 65535) return fail(VH_E_RANGE, "%s: at most 65535 streams", what);
        return 0;
    }
    if (a->length < 0) return fail(VH_E_SHAPE, "%s: negative length", what);
    if (a->length > 0x7fffffff) return fail(VH_E_RANGE, "%s: at most 2^31 - 1 tokens a sequence", what);
    return 0;
}

int check_args(const char* what, const vh_linear_attention_args* a, bool one_token, bool backward) {
    if (!a) return fail(VH_E_ARG, "%s: null argument struct", what);
    if (!a->q || !a->k || !a->v || !a->log_decay || (!a->o && !backward)) return fail(VH_E_ARG, "%s: null pointer argument", what);
    if (int rc = check_sizes(what, a, one_token)) return rc;
    const size_t es = dtype_size(a->dtype);
    for (const void* t : {a->q, a->k, a->v, (const void*)a->o})
        if (t && !aligned(t, es)) return fail(VH_E_ALIGN, "%s: misaligned pointers", what);
    for (const void* t : {(const void*)a->log_decay, (const void*)a->initial_state, (const void*)a->final_state,
                          (const void*)a->seq_offsets})
        if (t && !aligned(t, 4)) return fail(VH_E_ALIGN, "%s: misaligned pointers", what);
    return 0;
}

// How many elements of [tokens, heads, dim] rows one aligned access may take.
int vec_of(const void* p, const Rows& r, int64_t head, int dim, int dtype, bool packed) {
    const int es = (int)dtype_size(dtype);
    for (int v : {8, 4}) {
        if (v * es > 16) continue;
        if (aligned(p, v * es) && dim % v == 0 && head % v == 0 && r.token % v == 0 && (packed || r.batch % v == 0)) return v;
    }
    return 1;
}

Heads heads_of(const void* p, int64_t batch, int64_t token, int64_t head, int dim, int dtype, bool packed) {
    Heads h{p, {batch, token}, head, 1};
    h.vec = vec_of(p, h.rows, head, dim, dtype, packed);
    return h;
}

Params base_params(const vh_linear_attention_args* a) {
    Params p{};
    const bool packed = a->seq_offsets != nullptr;
    p.seqs = {a->seq_offsets, a->length, a->batch, a->reverse != 0};
    p.q = heads_of(a->q, a->q_batch_stride, a->q_token_stride, a->q_head_stride, a->key_dim, a->dtype, packed);
    p.k = heads_of(a->k, a->k_batch_stride, a->k_token_stride, a->k_head_stride, a->key_dim, a->dtype, packed);
    p.v = heads_of(a->v, a->v_batch_stride, a->v_token_stride, a->v_head_stride, a->value_dim, a->dtype, packed);
    p.log_decay = a->log_decay;
    p.initial = a->initial_state;
    p.init_a = a->value_dim;
    p.init_b = 1;
    p.o = a->o;
    p.final_state = a->final_state;
    p.out_scale = a->scale;
    p.kv_scale = 1.f;
    p.heads = a->heads;
    p.dk = a->key_dim;
    p.dv = a->value_dim;
    return p;
}

// Tokens a segment, 0 for whole chains.  A CTA takes one segment of one head and 64 value columns, and
// two CTAs fit an SM: fewer chains than half as many are cut so that they fill the card once, into at least
// two chunks each (three sequences of 785 tokens, 5 heads of 48 and 72 in fp32, training: 255 us, with four
// chunks 434, with one 246).  Packed sequences are always cut, as the host does not know their lengths.
int segment_size(int64_t length, int batch, bool packed, int heads, int dv) {
    const int64_t ctas = 2 * (int64_t)sm_count(), lanes = (int64_t)heads * ((dv + kTile - 1) / kTile);
    if (!packed && 2 * batch * lanes > ctas) return 0;
    const int64_t tokens = packed ? length : (int64_t)batch * length;
    int64_t size = (tokens * lanes + ctas - 1) / ctas;
    size = std::max<int64_t>((size + kChunk - 1) / kChunk * kChunk, 2 * kChunk);
    return size < length ? (int)size : 0;
}

template <typename T, int DK, bool OUT>
int launch_chunks(const Params& p, int64_t units, cudaStream_t st) {
    using L = Layout<T, DK, OUT>;
    const void* fn = reinterpret_cast<const void*>(&chunk_kernel<T, DK, OUT>);
    if (!ensure_smem_attr(fn, L::kBytes)) return fail(VH_E_DEVICE, "linear attention: shared memory");
    const dim3 grid((unsigned)units, p.heads, (p.dv + kTile - 1) / kTile);
    chunk_kernel<T, DK, OUT><<<grid, kThreads, L::kBytes, st>>>(p);
    return launch_status(OUT ? "linear attention" : "linear attention: segment states");
}

// One pass of the operator over prepared parameters; `states` holds pass_bytes().
int run(Params p, int dtype, void* states, cudaStream_t st) {
    const bool packed = p.seqs.offsets != nullptr;
    p.vec_o = vec_of(p.o, {0, (int64_t)p.heads * p.dv}, p.dv, p.dv, dtype, true);
    int rc = 0;
    if (dtype == VH_BF16 && tc_run(p, states, st, &rc)) return rc;
    p.segment = segment_size(p.seqs.length, p.seqs.count, packed, p.heads, p.dv);
    p.states = static_cast<float*>(states);
    const int64_t units = p.segment ? ssm::slot_total(packed, p.seqs.length, p.seqs.count, p.segment) : p.seqs.count;
    return with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        const bool narrow = p.dk <= 64;
        if (p.segment) {
            if (int rc = narrow ? launch_chunks<T, 64, false>(p, units, st) : launch_chunks<T, 128, false>(p, units, st)) return rc;
            if (int rc = enter_segments(p, st)) return rc;
        }
        return narrow ? launch_chunks<T, 64, true>(p, units, st) : launch_chunks<T, 128, true>(p, units, st);
    });
}

// The states of a pass's segments, in whichever form it runs.
int64_t pass_bytes(const vh_linear_attention_args* a, int dk, int dv) {
    const bool packed = a->seq_offsets != nullptr;
    int64_t most = 0;
    for (int size : {segment_size(a->length, a->batch, packed, a->heads, dv),
                     a->dtype == VH_BF16 ? tc_segment_size(a->length, a->batch, packed, a->heads, dk, dv) : 0})
        if (size) most = std::max(most, ssm::slot_total(packed, a->length, a->batch, size) * a->heads * dk * dv * (int64_t)sizeof(float));
    return most;
}
int64_t fwd_bytes(const vh_linear_attention_args* a) { return pass_bytes(a, a->key_dim, a->value_dim); }
// the passes for dq and dk have the two dims the other way round
int64_t bwd_bytes(const vh_linear_attention_args* a) {
    return std::max(fwd_bytes(a), pass_bytes(a, a->value_dim, a->key_dim));
}

int check_workspace(const char* what, const void* ws, int64_t have, int64_t need) {
    if (need == 0) return 0;
    if (!ws || have < need) return fail(VH_E_ARG, "%s: workspace too small (%lld < %lld bytes)", what, (long long)have, (long long)need);
    if (!aligned(ws, 16)) return fail(VH_E_ALIGN, "%s: the workspace must be 16-byte aligned", what);
    return 0;
}

}  // namespace

int enter_segments(const Params& p, cudaStream_t st) {
    const int64_t states = (int64_t)p.dk * p.dv;
    enter_kernel<<<dim3(p.seqs.count, p.heads, (unsigned)((states + 255) / 256)), 256, 0, st>>>(p);
    return launch_status("linear attention: entering states");
}

}  // namespace lin
}  // namespace vh

using namespace vh;
using namespace vh::lin;

extern "C" int64_t vh_linear_attention_fwd_workspace_bytes(const vh_linear_attention_args* a) {
    clear_error();
    return check_sizes("vh_linear_attention_fwd_workspace_bytes", a, false) ? 0 : fwd_bytes(a);
}

extern "C" int vh_linear_attention_fwd(const vh_linear_attention_args* a, void* workspace, int64_t workspace_bytes,
                                       vh_stream_t stream) {
    clear_error();
    if (int rc = check_args("vh_linear_attention_fwd", a, false, false)) return rc;
    if (int rc = check_workspace("vh_linear_attention_fwd", workspace, workspace_bytes, fwd_bytes(a))) return rc;
    return run(base_params(a), a->dtype, workspace, static_cast<cudaStream_t>(stream));
}

extern "C" int64_t vh_linear_attention_bwd_workspace_bytes(const vh_linear_attention_args* a) {
    clear_error();
    return check_sizes("vh_linear_attention_bwd_workspace_bytes", a, false) ? 0 : bwd_bytes(a);
}

extern "C" int vh_linear_attention_bwd(const vh_linear_attention_args* a, const void* grad_o, const float* grad_final,
                                       void* grad_q, void* grad_k, void* grad_v, float* grad_initial, void* workspace,
                                       int64_t workspace_bytes, vh_stream_t stream) {
    clear_error();
    const char* what = "vh_linear_attention_bwd";
    if (int rc = check_args(what, a, false, true)) return rc;
    if (!grad_o || !grad_q || !grad_k || !grad_v) return fail(VH_E_ARG, "%s: null pointer argument", what);
    const size_t es = dtype_size(a->dtype);
    for (const void* t : {grad_o, (const void*)grad_q, (const void*)grad_k, (const void*)grad_v})
        if (!aligned(t, es)) return fail(VH_E_ALIGN, "%s: misaligned pointers", what);
    for (const void* t : {(const void*)grad_final, (const void*)grad_initial})
        if (t && !aligned(t, 4)) return fail(VH_E_ALIGN, "%s: misaligned pointers", what);
    if (int rc = check_workspace(what, workspace, workspace_bytes, bwd_bytes(a))) return rc;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool packed = a->seq_offsets != nullptr;
    const Params f = base_params(a);
    const int64_t row = (int64_t)a->heads * a->value_dim;
    const Heads go = heads_of(grad_o, a->length * row, row, a->value_dim, a->value_dim, a->dtype, packed);
    auto pass = [&](const Params& p) { return run(p, a->dtype, workspace, st); };
    // dq_t = scale S_t dO_t
    Params p = f;
    p.q = go; p.k = f.v; p.v = f.k;
    p.dk = f.dv; p.dv = f.dk;
    p.init_a = 1; p.init_b = f.dv;
    p.o = grad_q; p.final_state = nullptr;
    if (int rc = pass(p)) return rc;
    // G_t = scale q_t dO_t^T + lambda G_{t+1}, the gradient of the final state entering as it is:
    // dk_t = G_t v_t
    p = f;
    p.seqs.reverse = !f.seqs.reverse;
    p.q = f.v; p.k = go; p.v = f.q;
    p.dk = f.dv; p.dv = f.dk;
    p.initial = grad_final;
    p.init_a = 1; p.init_b = f.dv;
    p.entry = 1;
    p.out_scale = 1.f; p.kv_scale = a->scale;
    p.o = grad_k; p.final_state = nullptr;
    if (int rc = pass(p)) return rc;
    // dv_t = k_t G_t; before the first token the state's gradient is lambda G_1
    p = f;
    p.seqs.reverse = !f.seqs.reverse;
    p.q = f.k; p.k = f.q; p.v = go;
    p.initial = grad_final;
    p.entry = 1;
    p.out_scale = 1.f; p.kv_scale = a->scale;
    p.o = grad_v; p.final_state = grad_initial;
    p.exit_decay = 1;
    return pass(p);
}

extern "C" int vh_linear_attention_step(const vh_linear_attention_args* a, const float* state, float* state_out,
                                        const int32_t* slots_index, int32_t slots, vh_stream_t stream) {
    clear_error();
    const char* what = "vh_linear_attention_step";
    if (int rc = check_args(what, a, true, false)) return rc;
    if (!state || !state_out) return fail(VH_E_ARG, "%s: null state", what);
    if (!aligned(state, 4) || !aligned(state_out, 4)) return fail(VH_E_ALIGN, "%s: misaligned states", what);
    if (slots <= 0 || (!slots_index && slots < a->batch)) return fail(VH_E_SHAPE, "%s: %d slots for %d streams", what, slots, a->batch);
    StepParams p{};
    p.q = {a->q, {a->q_batch_stride, 0}, a->q_head_stride, 1};
    p.k = {a->k, {a->k_batch_stride, 0}, a->k_head_stride, 1};
    p.v = {a->v, {a->v_batch_stride, 0}, a->v_head_stride, 1};
    p.log_decay = a->log_decay;
    p.state = state;
    p.state_out = state_out;
    p.slots_index = slots_index;
    p.o = a->o;
    p.scale = a->scale;
    p.slots = slots;
    p.batch = a->batch;
    p.heads = a->heads;
    p.dk = a->key_dim;
    p.dv = a->value_dim;
    const bool wide = p.dv % 4 == 0 && aligned(state, 16) && aligned(state_out, 16);
    const dim3 grid(p.heads, p.batch);
    return with_dtype(a->dtype, [&](auto t) {
        using T = decltype(t);
        if (wide) step_kernel<T, 4><<<grid, 256, 0, static_cast<cudaStream_t>(stream)>>>(p);
        else step_kernel<T, 1><<<grid, 256, 0, static_cast<cudaStream_t>(stream)>>>(p);
        return launch_status("linear attention step");
    });
}
