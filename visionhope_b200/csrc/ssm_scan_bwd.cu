// Selective scan, backward (vh_ssm_scan_bwd).
//
// With p_t = s_t u_t, i_t = sum_n c_t h_t + D u_t (the output before its gate) and
// v_t = dy_t silu(z_t) (or dy_t):
//     g_t = c_t v_t + exp(s_{t+1} a) g_{t+1}          (the gradient of h_t, last token first)
//     dc_t = sum_channels v_t h_t                     db_t = sum_channels p_t g_t
//     q_t  = g_t exp(s_t a) h_{t-1}                   da = sum_t s_t q_t
//     ds_t = sum_n a q_t + u_t sum_n b_t g_t          du_t = s_t sum_n b_t g_t + D v_t
//     dz_t = dy_t i_t silu'(z_t)                      dD = sum_t v_t u_t
// ds_t goes through softplus' derivative to delta_t and delta_bias.  The products e h_{t-1} and
// the decays e = exp(s_t a) of a group of four tokens are computed once and kept in registers
// between the two directions.
//
// A warp owns a channel tile of a sequence (layout: ssm_scan.cuh) and walks its chunks of 32
// tokens from the last to the first.  The forward left the state before each chunk; the warp runs
// it forward again once, leaving the state before each group of four in shared memory, and then
// takes the groups in reverse, computing each again from its saved state.  Sums over channels
// (db, dc) leave one partial per channel tile, sums over tokens (da, dD, d delta_bias) one per
// sequence, and two small kernels add them in order.
#include <algorithm>
#include <type_traits>

#include "ssm_scan.cuh"

namespace vh {
namespace ssm {
namespace {

constexpr int kGroups = kCheckpoint / kGroup;  // groups in a chunk

struct BwdParams {
    ScanParams f;
    const void* dy;
    const float* dfinal;
    void *du, *ddelta, *dz;
    float* dinitial;
    float* part_bc;  // [tiles][tokens][2][N]
    float* part_a;   // [sequences][channels][N]
    float* part_d;   // [sequences][2][channels]: dD, d delta_bias
    int64_t tokens;
    int32_t vec;     // as f.vec, for dy and the outputs too
};

template <int NL>
struct BwdSmem {
    using K = Tile<NL>;
    float h[kGroups][32 * 16];
    float step[kGroup * K::CW], su[kGroup * K::CW], v[kGroup * K::CW];
    float bc[kGroup * 2 * K::N];
    float y[kGroup * K::CW], ds[kGroup * K::CW], gb[kGroup * K::CW];
};

// Sums four values (channels c of one token) over the state lanes into row[c of the tile].
template <int NL>
__device__ __forceinline__ void sum_states(float (&v)[4], int lane, float* row) {
    using K = Tile<NL>;
    reduce_scatter<4, NL, K::CL>(v, lane);
    constexpr int kKeep = NL >= 4 ? 1 : 4 / NL;
    const int j = lane / K::CL, k = lane % K::CL;
    const int first = j * 4 / NL;
    if (NL <= 4 || j % (NL / 4 > 0 ? NL / 4 : 1) == 0) {
#pragma unroll
        for (int i = 0; i < kKeep; ++i) row[4 * k + first + i] = v[i];
    }
}

template <typename T, int NL>
__global__ void __launch_bounds__(32 * kWarps, 2) scan_bwd_kernel(const BwdParams bp, int64_t items) {
    using K = Tile<NL>;
    constexpr int N = K::N, CW = K::CW, CE = K::CE, TE = K::TE, CL = K::CL;
    extern __shared__ __align__(16) unsigned char smem[];
    const ScanParams& p = bp.f;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int tiles = p.groups * p.tiles_per_group;
    const int64_t item = (int64_t)blockIdx.x * kWarps + warp;
    if (item >= items) return;
    BwdSmem<NL>& sm = reinterpret_cast<BwdSmem<NL>*>(smem)[warp];
    const int s = (int)(item / tiles), tile = (int)(item % tiles);
    const int group = tile / p.tiles_per_group;
    const int cbase = group * p.per_group + (tile % p.tiles_per_group) * CW;
    const int cend = (group + 1) * p.per_group;
    const Seq seq = seq_at(p.seqs, s);
    const LaneElems<NL> own(lane);
    const int n0 = 4 * (lane / CL), ct = 4 * (lane % CL), c0 = cbase + ct;
    const int ec = cbase + own.c0;

    const T* u = static_cast<const T*>(p.u) + first_row(p.seqs, seq, s, p.ur) + ec;
    const T* dl = static_cast<const T*>(p.delta) + first_row(p.seqs, seq, s, p.dr) + ec;
    const T* z = p.z ? static_cast<const T*>(p.z) + first_row(p.seqs, seq, s, p.zr) + ec : nullptr;
    const T* b = static_cast<const T*>(p.b) + first_row(p.seqs, seq, s, p.br) + group * p.bg;
    const T* c = static_cast<const T*>(p.c) + first_row(p.seqs, seq, s, p.cr) + group * p.cg;
    const int64_t us = row_step(p.seqs, p.ur), ds = row_step(p.seqs, p.dr), zs = row_step(p.seqs, p.zr);
    const int64_t bs = row_step(p.seqs, p.br), cs = row_step(p.seqs, p.cr);
    const Rows yr{p.seqs.length * p.channels, p.channels};
    const int64_t y0 = first_row(p.seqs, seq, s, yr) + ec, ys = row_step(p.seqs, yr);
    const T* dy = static_cast<const T*>(bp.dy) + y0;
    T* du = static_cast<T*>(bp.du) + y0;
    T* dd = static_cast<T*>(bp.ddelta) + y0;
    T* dz = bp.dz ? static_cast<T*>(bp.dz) + y0 : nullptr;
    const Rows tr{p.seqs.length, 1};
    float* pbc = bp.part_bc + ((int64_t)tile * bp.tokens + first_row(p.seqs, seq, s, tr)) * 2 * N;
    const int64_t ps = row_step(p.seqs, tr) * 2 * N;
    const float* ck = p.checkpoints + slot_base(p.seqs, s, seq.row, kCheckpoint) * p.channels * N;

    float a2[16], g[16], da[16];
    load_block<N>(p.a, c0, cend, n0, a2);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        a2[i] = to_log2(a2[i]);
        g[i] = da[i] = 0.f;
    }
    if (bp.dfinal) load_block<N>(bp.dfinal + (int64_t)s * p.channels * N, c0, cend, n0, g);
    float bias[CE], skip[CE], dskip[CE], dbias[CE];
#pragma unroll
    for (int i = 0; i < CE; ++i) {
        bias[i] = p.delta_bias && ec + i < cend ? p.delta_bias[ec + i] : 0.f;
        skip[i] = p.d_skip && ec + i < cend ? p.d_skip[ec + i] : 0.f;
        dskip[i] = dbias[i] = 0.f;
    }

    const int64_t chunks = (seq.len + kCheckpoint - 1) / kCheckpoint;
    for (int64_t ch = chunks - 1; ch >= 0; --ch) {
        const int64_t tc = ch * kCheckpoint;
        const int len = seq.len - tc < kCheckpoint ? (int)(seq.len - tc) : kCheckpoint;
        const int groups = (len + kGroup - 1) / kGroup;
        float h[16];
        load_block<N>(ck + ch * p.channels * N, c0, cend, n0, h);

        // forward over all groups but the last, whose state is not needed beyond its start
        for (int gi = 0; gi < groups; ++gi) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *reinterpret_cast<float4*>(&sm.h[gi][(i * 32 + lane) * 4]) =
                    make_float4(h[4 * i], h[4 * i + 1], h[4 * i + 2], h[4 * i + 3]);
            if (gi + 1 == groups) break;
            const int64_t t = tc + gi * kGroup;
#pragma unroll
            for (int e = 0; e < TE; ++e) {
                const int r = own.t0 + e;
                float ue[CE], de[CE];
                load_v<CE>(u + (t + r) * us, ec, cend, p.vec, ue);
                load_v<CE>(dl + (t + r) * ds, ec, cend, p.vec, de);
#pragma unroll
                for (int i = 0; i < CE; ++i) {
                    de[i] += bias[i];
                    if (p.softplus) de[i] = softplus(de[i]);
                    ue[i] *= de[i];
                }
                sts_v<CE>(sm.step + r * CW + own.c0, de);
                sts_v<CE>(sm.su + r * CW + own.c0, ue);
            }
            stage_bc<NL>(b + t * bs, c + t * cs, bs, cs, kGroup, p.vec_bc, lane, sm.bc);
            __syncwarp();
#pragma unroll
            for (int r = 0; r < kGroup; ++r) {
                float sv[4], pv[4], bv[4];
                lds4(sm.step + r * CW + ct, sv);
                lds4(sm.su + r * CW + ct, pv);
                lds4(sm.bc + r * 2 * N + n0, bv);
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int n = 0; n < 4; ++n) {
                        float& hh = h[4 * i + n];
                        hh = fmaf(pv[i], bv[n], exp2_fma(sv[i] * a2[4 * i + n]) * hh);
                    }
            }
            __syncwarp();
        }

        for (int gi = groups - 1; gi >= 0; --gi) {
            const int64_t t = tc + gi * kGroup;
            const int cnt = len - gi * kGroup < kGroup ? len - gi * kGroup : kGroup;
            float ue[TE][CE], ze[TE][CE], re[TE][CE], ye[TE][CE];  // u, z, delta + bias, dy
#pragma unroll
            for (int e = 0; e < TE; ++e) {
                const int r = own.t0 + e;
                float de[CE], pe[CE], ve[CE];
#pragma unroll
                for (int i = 0; i < CE; ++i) ue[e][i] = ze[e][i] = re[e][i] = ye[e][i] = de[i] = 0.f;
                if (r < cnt) {
                    load_v<CE>(u + (t + r) * us, ec, cend, p.vec, ue[e]);
                    load_v<CE>(dl + (t + r) * ds, ec, cend, p.vec, re[e]);
                    if (z) load_v<CE>(z + (t + r) * zs, ec, cend, p.vec, ze[e]);
                    load_v<CE>(dy + (t + r) * ys, ec, cend, bp.vec, ye[e]);
#pragma unroll
                    for (int i = 0; i < CE; ++i) {
                        re[e][i] += bias[i];
                        de[i] = p.softplus ? softplus(re[e][i]) : re[e][i];
                    }
                }
#pragma unroll
                for (int i = 0; i < CE; ++i) {
                    pe[i] = de[i] * ue[e][i];
                    ve[i] = z ? ye[e][i] * (ze[e][i] * sigmoid(ze[e][i])) : ye[e][i];
                }
                sts_v<CE>(sm.step + r * CW + own.c0, de);
                sts_v<CE>(sm.su + r * CW + own.c0, pe);
                sts_v<CE>(sm.v + r * CW + own.c0, ve);
            }
            stage_bc<NL>(b + t * bs, c + t * cs, bs, cs, cnt, p.vec_bc, lane, sm.bc);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float q[4];
                lds4(&sm.h[gi][(i * 32 + lane) * 4], q);
#pragma unroll
                for (int n = 0; n < 4; ++n) h[4 * i + n] = q[n];
            }
            __syncwarp();
            float e[kGroup][16], eh[kGroup][16];  // decays, and decays times the state before
            float dcs[kGroup][4];
#pragma unroll
            for (int r = 0; r < kGroup; ++r) {
                float sv[4], pv[4], vv[4], bv[4], cv[4], acc[4];
                lds4(sm.step + r * CW + ct, sv);
                lds4(sm.su + r * CW + ct, pv);
                lds4(sm.v + r * CW + ct, vv);
                lds4(sm.bc + r * 2 * N + n0, bv);
                lds4(sm.bc + r * 2 * N + N + n0, cv);
#pragma unroll
                for (int n = 0; n < 4; ++n) dcs[r][n] = acc[n] = 0.f;
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int n = 0; n < 4; ++n) {
                        float& hh = h[4 * i + n];
                        e[r][4 * i + n] = exp2_fma(sv[i] * a2[4 * i + n]);
                        eh[r][4 * i + n] = e[r][4 * i + n] * hh;
                        hh = fmaf(pv[i], bv[n], eh[r][4 * i + n]);
                        acc[i] = fmaf(cv[n], hh, acc[i]);
                        dcs[r][n] = fmaf(vv[i], hh, dcs[r][n]);
                    }
                if (z) sum_states<NL>(acc, lane, sm.y + r * CW);
            }
#pragma unroll
            for (int r = kGroup - 1; r >= 0; --r) {
                float sv[4], pv[4], vv[4], bv[4], cv[4], dsum[4], gsum[4], bcs[8];
                lds4(sm.step + r * CW + ct, sv);
                lds4(sm.su + r * CW + ct, pv);
                lds4(sm.v + r * CW + ct, vv);
                lds4(sm.bc + r * 2 * N + n0, bv);
                lds4(sm.bc + r * 2 * N + N + n0, cv);
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    dsum[n] = gsum[n] = bcs[n] = 0.f;
                    bcs[4 + n] = dcs[r][n];
                }
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int n = 0; n < 4; ++n) {
                        const int k = 4 * i + n;
                        g[k] = fmaf(cv[n], vv[i], g[k]);
                        const float q = g[k] * eh[r][k];
                        da[k] = fmaf(sv[i], q, da[k]);
                        dsum[i] = fmaf(a2[k], q, dsum[i]);
                        gsum[i] = fmaf(bv[n], g[k], gsum[i]);
                        bcs[n] = fmaf(pv[i], g[k], bcs[n]);
                        g[k] *= e[r][k];
                    }
                sum_states<NL>(dsum, lane, sm.ds + r * CW);
                sum_states<NL>(gsum, lane, sm.gb + r * CW);
                // db and dc of the thread's four states over the channel lanes
                reduce_scatter<8, CL, 1>(bcs, lane);
                if (r < cnt) {
                    constexpr int kKeep = CL >= 8 ? 1 : 8 / CL;
                    const int k = lane % CL, first = k * 8 / CL;
                    if (CL <= 8 || k % (CL / 8 > 0 ? CL / 8 : 1) == 0) {
#pragma unroll
                        for (int i = 0; i < kKeep; ++i) {
                            const int w = first + i;  // 0-3: db, 4-7: dc
                            pbc[(t + r) * ps + (w / 4) * N + n0 + w % 4] = bcs[i];
                        }
                    }
                }
            }
            __syncwarp();
#pragma unroll
            for (int x = 0; x < TE; ++x) {
                const int r = own.t0 + x;
                float yo[CE], dso[CE], gbo[CE], duo[CE], ddo[CE], dzo[CE];
                if (z) lds_v<CE>(sm.y + r * CW + own.c0, yo);
                lds_v<CE>(sm.ds + r * CW + own.c0, dso);
                lds_v<CE>(sm.gb + r * CW + own.c0, gbo);
                if (r < cnt) {
#pragma unroll
                    for (int i = 0; i < CE; ++i) {
                        float v = ye[x][i];
                        if (z) {
                            const float sg = sigmoid(ze[x][i]);
                            dzo[i] = ye[x][i] * fmaf(skip[i], ue[x][i], yo[i]) * (sg * (1.f + ze[x][i] * (1.f - sg)));
                            v *= ze[x][i] * sg;
                        }
                        const float st = p.softplus ? softplus(re[x][i]) : re[x][i];
                        duo[i] = fmaf(st, gbo[i], skip[i] * v);
                        ddo[i] = fmaf(ue[x][i], gbo[i], kLn2 * dso[i]);
                        if (p.softplus) ddo[i] *= sigmoid(re[x][i]);
                        dskip[i] = fmaf(v, ue[x][i], dskip[i]);
                        dbias[i] += ddo[i];
                    }
                    store_v<CE>(du + (t + r) * ys, ec, cend, bp.vec, duo);
                    store_v<CE>(dd + (t + r) * ys, ec, cend, bp.vec, ddo);
                    if (dz) store_v<CE>(dz + (t + r) * ys, ec, cend, bp.vec, dzo);
                }
            }
            __syncwarp();
        }
    }
    if (bp.dinitial) store_block<N>(bp.dinitial + (int64_t)s * p.channels * N, c0, cend, n0, g);
    store_block<N>(bp.part_a + (int64_t)s * p.channels * N, c0, cend, n0, da);
    // dD and d delta_bias over the lanes that share channels: those of one channel lane whose
    // elements differ in the token (lane distances CL * (lanes per token) and up)
    constexpr int kLanesPerToken = NL <= 4 ? 1 : NL / 4;
#pragma unroll
    for (int o = 16; o >= CL * kLanesPerToken; o >>= 1)
#pragma unroll
        for (int i = 0; i < CE; ++i) {
            dskip[i] += __shfl_xor_sync(0xffffffffu, dskip[i], o);
            dbias[i] += __shfl_xor_sync(0xffffffffu, dbias[i], o);
        }
    if (lane < CL * kLanesPerToken) {
        float* pd = bp.part_d + (int64_t)s * 2 * p.channels;
#pragma unroll
        for (int i = 0; i < CE; ++i)
            if (ec + i < cend) {
                pd[ec + i] = dskip[i];
                pd[p.channels + ec + i] = dbias[i];
            }
    }
}

// db and dc: the channel tiles' partials of each group added in order.
template <typename T>
__global__ void __launch_bounds__(256) sum_bc_kernel(const float* __restrict__ part, T* __restrict__ db, T* __restrict__ dc,
                                                     int64_t tokens, int groups, int tiles, int n) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;  // over [token][group][2][N]
    if (i >= tokens * groups * 2 * n) return;
    const int w = (int)(i % (2 * n));
    const int64_t tg = i / (2 * n);
    const int64_t t = tg / groups;
    const int gr = (int)(tg % groups);
    float sum = 0.f;
    for (int k = 0; k < tiles; ++k) sum += part[((int64_t)(gr * tiles + k) * tokens + t) * 2 * n + w];
    T* out = w < n ? db : dc;
    out[(t * groups + gr) * n + w % n] = from_f<T>(sum);
}

// out[i] = sum over `rows` of part[r][i], in order: 8 outputs by 32 row lanes per CTA.
__global__ void __launch_bounds__(256) sum_rows_kernel(const float* __restrict__ part, int64_t rows, int64_t stride,
                                                       int64_t count, float* __restrict__ out) {
    __shared__ float red[32][9];
    const int x = threadIdx.x % 8, r = threadIdx.x / 8;
    const int64_t i = (int64_t)blockIdx.x * 8 + x;
    float sum = 0.f;
    if (i < count)
        for (int64_t k = r; k < rows; k += 32) sum += part[k * stride + i];
    red[r][x] = sum;
    __syncthreads();
    for (int o = 16; o > 0; o >>= 1) {
        if (r < o) red[r][x] += red[r + o][x];
        __syncthreads();
    }
    if (r == 0 && i < count) out[i] = red[0][x];
}

struct Layout {
    int64_t tokens, bc, a, d, total;  // floats
};
Layout layout_of(const vh_ssm_scan_args* a) {
    Layout l;
    l.tokens = a->seq_offsets ? a->length : (int64_t)a->batch * a->length;
    const int cw = 128 / (a->states / 4), per = a->channels / a->groups;
    const int64_t tiles = (int64_t)a->groups * ((per + cw - 1) / cw);
    l.bc = tiles * l.tokens * 2 * a->states;
    l.a = (int64_t)a->batch * a->channels * a->states;
    l.d = (int64_t)a->batch * 2 * a->channels;
    l.total = l.bc + l.a + l.d;
    return l;
}

int check_bwd(const char* what, const vh_ssm_scan_bwd_args* a) {
    if (!a) return fail(VH_E_ARG, "%s: null argument struct", what);
    vh_ssm_scan_args f = a->fwd;
    if (!f.y) f.y = a->grad_u;  // the backward does not read y
    f.final_state = nullptr;
    if (int rc = check_scan_args(what, &f, false)) return rc;
    if (!f.checkpoints) return fail(VH_E_ARG, "%s: the forward's checkpoints are needed", what);
    if (!a->grad_y || !a->grad_u || !a->grad_delta || !a->grad_b || !a->grad_c || !a->grad_a || (f.z && !a->grad_z))
        return fail(VH_E_ARG, "%s: null pointer argument", what);
    const size_t es = dtype_size(f.dtype);
    const void* typed[] = {a->grad_y, a->grad_u, a->grad_delta, a->grad_z, a->grad_b, a->grad_c};
    for (const void* t : typed)
        if (t && !aligned(t, es)) return fail(VH_E_ALIGN, "%s: misaligned pointers", what);
    if ((a->grad_final && !aligned(a->grad_final, 16)) || (a->grad_initial && !aligned(a->grad_initial, 16)))
        return fail(VH_E_ALIGN, "%s: the states must be 16-byte aligned", what);
    return 0;
}

}  // namespace
}  // namespace ssm
}  // namespace vh

using namespace vh;
using namespace vh::ssm;

extern "C" int64_t vh_ssm_scan_bwd_workspace_bytes(const vh_ssm_scan_bwd_args* a) {
    if (check_bwd("vh_ssm_scan_bwd_workspace_bytes", a)) return 0;
    return layout_of(&a->fwd).total * 4;
}

extern "C" int vh_ssm_scan_bwd(const vh_ssm_scan_bwd_args* a, void* workspace, int64_t workspace_bytes,
                               vh_stream_t stream) {
    clear_error();
    if (int rc = check_bwd("vh_ssm_scan_bwd", a)) return rc;
    const vh_ssm_scan_args* f = &a->fwd;
    const Layout l = layout_of(f);
    if (!workspace || workspace_bytes < l.total * 4) return fail(VH_E_ARG, "vh_ssm_scan_bwd: workspace too small");
    if (!aligned(workspace, 16)) return fail(VH_E_ALIGN, "vh_ssm_scan_bwd: the workspace must be 16-byte aligned");
    BwdParams p{};
    vh_ssm_scan_args in = *f;
    in.y = a->grad_u;
    fill_scan_params(&in, &p.f);
    const size_t es = dtype_size(f->dtype);
    p.dy = a->grad_y; p.dfinal = a->grad_final;
    p.du = a->grad_u; p.ddelta = a->grad_delta; p.dz = f->z ? a->grad_z : nullptr; p.dinitial = a->grad_initial;
    p.part_a = static_cast<float*>(workspace);
    p.part_bc = p.part_a + l.a;
    p.part_d = p.part_bc + l.bc;
    p.tokens = l.tokens;
    p.vec = p.f.vec && aligned(a->grad_y, 4 * es) && aligned(a->grad_u, 4 * es) && aligned(a->grad_delta, 4 * es) &&
            (!p.dz || aligned(p.dz, 4 * es));
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int64_t items = (int64_t)f->batch * p.f.groups * p.f.tiles_per_group;
    const int64_t blocks = (items + kWarps - 1) / kWarps;
    if (blocks > 0x7fffffff) return fail(VH_E_RANGE, "vh_ssm_scan_bwd: too many channel tiles");
    return with_dtype(f->dtype, [&](auto t) {
        using T = decltype(t);
        int rc = with_states(f->states, [&](auto nl) {
            constexpr int NL = decltype(nl)::value;
            const size_t smem = sizeof(BwdSmem<NL>) * kWarps;
            const void* fn = reinterpret_cast<const void*>(&scan_bwd_kernel<T, NL>);
            if (!ensure_smem_attr(fn, smem))
                return fail(VH_E_DEVICE, "vh_ssm_scan_bwd: cannot reserve %zu bytes of shared memory", smem);
            scan_bwd_kernel<T, NL><<<(int)blocks, 32 * kWarps, smem, st>>>(p, items);
            return launch_status("selective scan backward");
        });
        if (rc) return rc;
        const int64_t outs = l.tokens * f->groups * 2 * f->states;
        if (outs > 0) {
            const int64_t grid = (outs + 255) / 256;
            if (grid > 0x7fffffff) return fail(VH_E_RANGE, "vh_ssm_scan_bwd: too many tokens");
            sum_bc_kernel<T><<<(int)grid, 256, 0, st>>>(p.part_bc, static_cast<T*>(a->grad_b), static_cast<T*>(a->grad_c),
                                                        l.tokens, f->groups, p.f.tiles_per_group, f->states);
            if ((rc = launch_status("selective scan backward: b, c"))) return rc;
        }
        auto rows = [&](const float* part, int64_t stride, int64_t count, float* out) {
            sum_rows_kernel<<<(int)((count + 7) / 8), 256, 0, st>>>(part, f->batch, stride, count, out);
            return launch_status("selective scan backward: parameters");
        };
        const int64_t dn = (int64_t)f->channels * f->states;
        if ((rc = rows(p.part_a, dn, dn, a->grad_a))) return rc;
        if (a->grad_d_skip && (rc = rows(p.part_d, 2 * f->channels, f->channels, a->grad_d_skip))) return rc;
        if (a->grad_delta_bias &&
            (rc = rows(p.part_d + f->channels, 2 * f->channels, f->channels, a->grad_delta_bias)))
            return rc;
        return 0;
    });
}
