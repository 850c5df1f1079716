// Selective scan, backward (vh_ssm_scan_bwd).
//
// With p_t = s_t u_t, e_t = exp(s_t a), i_t = sum_n c_t h_t + D u_t (the output before its gate)
// and v_t = dy_t silu(z_t) (or dy_t):
//     g_t = c_t v_t + e_{t+1} g_{t+1}                 (the gradient of h_t, last token first)
//     dc_t = sum_channels v_t h_t                     db_t = sum_channels p_t g_t
//     q_t  = e_t g_t h_{t-1}                          da = sum_t s_t q_t
//     ds_t = sum_n a q_t + u_t sum_n b_t g_t          du_t = s_t sum_n b_t g_t + D v_t
//     dz_t = dy_t i_t silu'(z_t)                      dD = sum_t v_t u_t
// ds_t goes through softplus' derivative to delta_t and delta_bias.
//
// A warp owns a channel tile (layout: ssm_scan.cuh) of a run of tokens and walks its chunks of 32
// tokens from the last to the first.  The forward left the state before each chunk; the warp runs
// the chunk forward once, leaving the state before each group of four in shared memory, and then
// takes the groups in reverse: four tokens forward again with their decays and states in
// registers, then back through them.  The states start from the forward's every 32 tokens, so
// the first of these passes takes all its decays from the special-function unit; the second one's
// carry the gradient along the whole sequence (see ssm_scan.cuh on the exponentials).  Sums over
// channels (db, dc) leave one partial per channel tile, sums over tokens (da, dD, d delta_bias)
// one per sequence or segment, and a small kernel adds them in order.
//
// 64 sequences of 784 tokens, 256 channels, 16 states, bf16 (12.8 M elements): 479 us, 377 of them
// this walk.  It is held by the 8 warps an SM that 255 registers and 27 KB of shared memory a warp
// leave: instruction issue is at 39 %, shared memory at 64 %, the special-function unit at 28 %, DRAM at
// 8 % (242 MB).  Two
// channels a thread would let 12 warps in, but at 289 M instructions for 186 M: 476 us against 440.
#include "ssm_scan.cuh"

namespace vh {
namespace ssm {
namespace {

constexpr int kGroups = kCheckpoint / kGroup;  // groups in a chunk
// Warps per CTA (neighbouring channel tiles): two CTAs an SM, in shared memory (fp32 groups take more of
// it) and registers.
template <typename T>
constexpr int kBwdWarps = sizeof(T) == 4 ? 3 : 4;

struct BwdParams {
    ScanParams f;
    const void* dy;
    const float* dfinal;
    void *du, *ddelta, *dz;
    float* dinitial;
    float* part_bc;  // [tiles][tokens][db, dc][state lane][4 states]
    float* part_a;   // [rows][tiles][512] in lane order; a row per sequence or segment
    float* part_d;   // [rows][2][tiles][CW]: dD, d delta_bias
    int64_t tokens;
    int32_t vec;     // as f.vec, for dy and the outputs too
};

// Shared memory of a warp.  A token's sums over lanes (ds, sum b g, db and dc) take the place of
// the state before it, once that is read.
template <typename T, int NL>
struct BwdRaw {
    typename Chain<T, NL>::Raw r;
    Pack<T, Tile<NL>::CE> dy[Tile<NL>::TE][32];
};
template <typename T, int NL>
struct OwnStage {
    BwdRaw<T, NL> raw;  // the next group, as loaded
    Stage<NL> s;
    float v[kGroup * Tile<NL>::CW];
};
template <typename T, int NL>
struct BwdStage : OwnStage<T, NL> {
    float h[kGroups][512];        // the states before the groups of a chunk
    float past[kGroup - 1][512];  // before the second to fourth token of the group at hand
    float y[512];
};

// Values in shared memory are read again after this, instead of being kept in registers.
__device__ __forceinline__ void reload() { asm volatile("" ::: "memory"); }

// db and dc of one token over the channel lanes: every lane leaves its four states of both, and
// output w = [db, dc][state lane][4 states] adds the CL parts.  A row is turned by its lane, so
// that neither side meets bank conflicts.  part: 256 floats.
template <int NL>
__device__ __forceinline__ void put_bc(float* part, int j, int k, const float (&db)[4], const float (&dc)[4]) {
    constexpr int R = 8 * NL;
    float* row = part + k * R;
    const int turn = 4 * k % R;
    *reinterpret_cast<float4*>(row + ((4 * j) ^ turn)) = make_float4(db[0], db[1], db[2], db[3]);
    *reinterpret_cast<float4*>(row + ((R / 2 + 4 * j) ^ turn)) = make_float4(dc[0], dc[1], dc[2], dc[3]);
}
// ... of the four tokens of a group, summed four outputs at a time and stored in that order.
// part(r): token r's parts; out: the group's first row, `ps` floats a token.
template <int NL, typename Part>
__device__ __forceinline__ void sum_bc(Part&& part, int lane, int64_t count, float* out, int64_t ps) {
    constexpr int R = 8 * NL, CL = Tile<NL>::CL, kQuads = kGroup * R / 4;
    constexpr int kSplit = kQuads < 32 ? 32 / kQuads : 1;  // lanes a quad: each takes some of the parts
#pragma unroll
    for (int m = 0; m < (kQuads + 31) / 32; ++m) {
        const int q = lane % kQuads + 32 * m, r = q / (R / 4), w = 4 * (q % (R / 4));
        const int k0 = kSplit > 1 ? lane / kQuads * (CL / kSplit) : 0;
        const float* rows = part(r);
        float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
        for (int i = 0; i < CL / kSplit; ++i) {
            float2 v[2];
            lds22(rows + (k0 + i) * R + (w ^ (4 * (k0 + i) % R)), v);
            sum[0] = fadd2(sum[0], v[0]);
            sum[1] = fadd2(sum[1], v[1]);
        }
#pragma unroll
        for (int o = 16; o >= kQuads; o >>= 1) {
            sum[0].x += __shfl_xor_sync(0xffffffffu, sum[0].x, o);
            sum[0].y += __shfl_xor_sync(0xffffffffu, sum[0].y, o);
            sum[1].x += __shfl_xor_sync(0xffffffffu, sum[1].x, o);
            sum[1].y += __shfl_xor_sync(0xffffffffu, sum[1].y, o);
        }
        if (r < count && (kSplit == 1 || lane < kQuads))
            *reinterpret_cast<float4*>(out + r * ps + w) = make_float4(sum[0].x, sum[0].y, sum[1].x, sum[1].y);
    }
}

// OWN: the first of the three kernels of a chain in segments: the segment's own gradient, that of
// the state before it when nothing enters from the right, and its sum of steps.
template <typename T, int NL, bool OWN>
__global__ void __launch_bounds__(32 * kBwdWarps<T>, OWN ? 4 : 2) scan_bwd_kernel(const BwdParams bp, const Segments seg, int64_t items) {
    using K = Tile<NL>;
    constexpr int N = K::N, CW = K::CW, CE = K::CE, TE = K::TE, CL = K::CL, P = kPairs<CE>;
    extern __shared__ __align__(16) unsigned char smem[];
    const ScanParams& p = bp.f;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    using Smem = std::conditional_t<OWN, OwnStage<T, NL>, BwdStage<T, NL>>;
    Smem& sm = reinterpret_cast<Smem*>(smem)[warp];
    const int64_t item = (int64_t)blockIdx.x * kBwdWarps<T> + warp;
    if (OWN) launch_dependents();
    Unit w;
    if (item >= items) return;
    const int tiles = p.groups * p.tiles_per_group;
    const int64_t unit = item;
    if (!unit_at(p, seg, item, w)) {  // a row of zeros
        if (!OWN) {
            for (int x = lane; x < 512; x += 32) bp.part_a[unit * 512 + x] = 0.f;
            for (int x = lane; x < CW; x += 32)
                bp.part_d[(w.slot * 2 * tiles + w.tile) * CW + x] = bp.part_d[((w.slot * 2 + 1) * tiles + w.tile) * CW + x] = 0.f;
        }
        return;
    }
    const Seq seq = w.seq;
    const int s = w.s, tile = w.tile;
    const int64_t t0 = w.t0, t1 = w.t1;
    Chain<T, NL> chn(p, seq, s, tile, lane);
    const int j = lane / CL, ct = 4 * (lane % CL), c0 = chn.cbase + ct;
    const int ec = chn.ec, cend = chn.cend, own_t = chn.own_t, own_c = chn.own_c;
    const Rows yr{p.seqs.length * p.channels, p.channels};
    const int64_t y0 = first_row(p.seqs, seq, s, yr) + ec, ys = row_step(p.seqs, yr);
    const T* dy = static_cast<const T*>(bp.dy) + y0;
    const bool gated = p.z != nullptr;
    float2 a2[8], g[8], da[8];
    float v16[16];
    const float most = mixed_limit(load_rates<NL>(p, c0, cend, j, v16));
    pair_up(v16, a2);
    const float* dfinal = bp.dfinal ? bp.dfinal + (int64_t)s * p.channels * N : nullptr;

    // dy's rows lie as y's; it moves with the chain's view, which stands at token `pos`
    const T* dyr = dy + (chn.left > 0 ? 0 : -(ec - (cend - (bp.vec ? CE : 1)))) + own_t * ys;
    int64_t pos = 0;
    // Fetches the group at `t` (of `count` tokens or more) behind the one at hand: a lane reads
    // back only what it fetched, and has read the group at hand by then.
    auto fetch_at = [&](int64_t t, int64_t tokens, bool all) {
        const int count = (int)min(tokens, (int64_t)kGroup);
        chn.move(t - pos);
        dyr += (t - pos) * ys;
        pos = t;
        if (all) {
            chn.template load<true>(sm.raw.r, count);
#pragma unroll
            for (int e = 0; e < TE; ++e) {
                const int64_t by = count >= kGroup ? e : min(e, count - 1 - own_t);
                fetch(&sm.raw.dy[e][lane], dyr + by * ys, chn.left, (bool)bp.vec);
            }
        } else {
            chn.template load<false>(sm.raw.r, count);
        }
        cp_async_commit();
    };
    // s, s u, B, C and v of the fetched group
    auto stage = [&](int64_t tokens, float2 (&sum)[P]) {
        const int count = (int)min(tokens, (int64_t)kGroup);
        const bool fast = chn.template stage<OWN, true>(sm.raw.r, count, sm.s, sum, most) && (OWN || count >= kGroup);
#pragma unroll
        for (int e = 0; e < TE; ++e) {
            float2 v2[P], z2[P];
            unpack<T, CE>(sm.raw.dy[e][lane], v2);
            if (gated) {
                unpack<T, CE>(sm.raw.r.z[e][lane], z2);
#pragma unroll
                for (int i = 0; i < P; ++i) v2[i] = fmul2(v2[i], fmul2(z2[i], sigmoid2(z2[i])));
            }
            chn.keep_real(e, count, v2);
            float f[CE];
            from_pairs<CE>(v2, f);
            sts_v<CE>(sm.v + (own_t + e) * CW + own_c, f);
        }
        return fast;
    };

    if constexpr (OWN) {
        // from its last token to its first: own = e_t (c_t v_t + own)
        float2 own[8];
        float2 sum[P];
#pragma unroll
        for (int i = 0; i < 8; ++i) own[i] = make_float2(0.f, 0.f);
#pragma unroll
        for (int i = 0; i < P; ++i) sum[i] = make_float2(0.f, 0.f);
        if (t0 > 0 && t0 < t1) {  // the first segment's own gradient is not needed
            int64_t t = t0 + (t1 - t0 - 1) / kGroup * kGroup;
            fetch_at(t, t1 - t, true);
            for (; t >= t0; t -= kGroup) {
                cp_async_wait<0>();
                const bool fast = stage(t1 - t, sum);
                __syncwarp();
                if (t > t0) fetch_at(t - kGroup, kGroup, true);
                auto pass = [&](auto mode) {
#pragma unroll
                    for (int r = kGroup - 1; r >= 0; --r) {
                        float2 sv[2], vv[2], c[4], e[8];
                        lds22(sm.s.step + r * CW + ct, sv);
                        lds22(sm.v + r * CW + ct, vv);
                        lds_dup4(sm.s.c(r, j), c);
                        decays<decltype(mode)::value>(sv, a2, e);
#pragma unroll
                        for (int i = 0; i < 4; ++i)
#pragma unroll
                            for (int q = 0; q < 2; ++q)
                                own[2 * i + q] = fmul2(e[2 * i + q], ffma2(c[i], vv[q], own[2 * i + q]));
                    }
                };
                if (fast) pass(std::integral_constant<int, kMixed>{});
                else pass(std::integral_constant<int, kChecked>{});
                __syncwarp();
            }
        }
        pair_down(own, v16);
        store_lanes(seg.state + unit * 512, lane, v16);
        sum_tokens<NL>(sum, lane, own_c, seg.sigma + unit * CW);
    } else {
        if (seg.state) {
            wait_for_previous();
            load_lanes(seg.state + unit * 512, lane, v16);
        } else if (dfinal) {
            load_block<NL>(dfinal, c0, cend, j, v16);
        } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) v16[i] = 0.f;
        }
        pair_up(v16, g);
#pragma unroll
        for (int i = 0; i < 8; ++i) da[i] = make_float2(0.f, 0.f);

        T* du = static_cast<T*>(bp.du) + y0;
        T* dd = static_cast<T*>(bp.ddelta) + y0;
        T* dz = bp.dz ? static_cast<T*>(bp.dz) + y0 : nullptr;
        const Rows tr{p.seqs.length, 1};
        float* pbc = bp.part_bc + ((int64_t)tile * bp.tokens + first_row(p.seqs, seq, s, tr)) * 2 * N;
        const int64_t ps = row_step(p.seqs, tr) * 2 * N;
        const float* ck = p.checkpoints + (slot_base(p.seqs, s, seq.row, kCheckpoint) * tiles + tile) * 512;
        float2 skip[P], dskip[P], dbias[P], unused[P];
        chn.load_params(p.d_skip, skip);
#pragma unroll
        for (int i = 0; i < P; ++i) dskip[i] = dbias[i] = unused[i] = make_float2(0.f, 0.f);

        const int64_t first = t0 / kCheckpoint, last = (t1 + kCheckpoint - 1) / kCheckpoint;
        if (t0 < t1) {  // the last chunk's first group
            const int64_t tc = (last - 1) * kCheckpoint;
            fetch_at(tc, t1 - tc, t1 - tc <= kGroup);
        }
        for (int64_t ch = last - 1; ch >= first && t0 < t1; --ch) {
            const int64_t tc = ch * kCheckpoint;
            const int64_t te = min(t1, tc + kCheckpoint);
            const int groups = (int)((te - tc + kGroup - 1) / kGroup);
            float2 h[8];
            load_lanes(ck + ch * tiles * 512, lane, v16);
            pair_up(v16, h);
            // forward over all groups but the last, whose state is not needed beyond its start
            {
                for (int gi = 0; gi < groups; ++gi) {
                    pair_down(h, v16);
                    store_lanes(sm.h[gi], lane, v16);
                    if (gi + 1 == groups) break;
                    cp_async_wait<0>();
                    chn.template stage<false, false>(sm.raw.r, kGroup, sm.s, unused);
                    __syncwarp();
                    const int64_t next = tc + (gi + 1) * kGroup;  // of the last group all, for the way back
                    fetch_at(next, te - next, gi + 2 == groups);
#pragma unroll
                    for (int r = 0; r < kGroup; ++r) {
                        float2 sv[2], pv[2], b[4], e[8];
                        lds22(sm.s.step + r * CW + ct, sv);
                        lds22(sm.s.su + r * CW + ct, pv);
                        lds_dup4(sm.s.b(r, j), b);
                        decays<kHardware>(sv, a2, e);
#pragma unroll
                        for (int i = 0; i < 4; ++i)
#pragma unroll
                            for (int q = 0; q < 2; ++q) h[2 * i + q] = ffma2(e[2 * i + q], h[2 * i + q], fmul2(pv[q], b[i]));
                    }
                    __syncwarp();
                }
            }
            for (int gi = groups - 1; gi >= 0; --gi) {
                const int64_t t = tc + gi * kGroup;
                cp_async_wait<0>();
                const bool fast = stage(te - t, unused);
                Pack<T, CE> nu[TE], nd[TE], nz[TE], ndy[TE];
#pragma unroll
                for (int x = 0; x < TE; ++x) {
                    nu[x] = sm.raw.r.u[x][lane];
                    nd[x] = sm.raw.r.d[x][lane];
                    ndy[x] = sm.raw.dy[x][lane];
                    if (gated) nz[x] = sm.raw.r.z[x][lane];
                }
                __syncwarp();
                if (gi > 0) fetch_at(t - kGroup, kGroup, true);
                else if (ch > first) fetch_at(tc - kCheckpoint, kGroup, false);
                auto pass = [&](auto mode) {
                    float2 e[kGroup][8];
                    float dcs[kGroup][4];
                    load_lanes(sm.h[gi], lane, v16);
                    pair_up(v16, h);
#pragma unroll
                    for (int r = 0; r < kGroup; ++r) {
                        reload();
                        float2 sv[2], pv[2], vv[2], b[4], c[4], acc[2], dc[4];
                        lds22(sm.s.step + r * CW + ct, sv);
                        lds22(sm.s.su + r * CW + ct, pv);
                        lds22(sm.v + r * CW + ct, vv);
                        lds_dup4(sm.s.b(r, j), b);
                        lds_dup4(sm.s.c(r, j), c);
                        decays<decltype(mode)::value>(sv, a2, e[r]);
                        acc[0] = acc[1] = make_float2(0.f, 0.f);
                        if (r > 0) {
                            pair_down(h, v16);
                            store_lanes(sm.past[r - 1], lane, v16);
                        }
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            dc[i] = make_float2(0.f, 0.f);
#pragma unroll
                            for (int q = 0; q < 2; ++q) {
                                float2& hh = h[2 * i + q];
                                hh = ffma2(e[r][2 * i + q], hh, fmul2(pv[q], b[i]));
                                acc[q] = ffma2(c[i], hh, acc[q]);
                                dc[i] = ffma2(vv[q], hh, dc[i]);
                            }
                            dcs[r][i] = dc[i].x + dc[i].y;
                        }
                        if (gated) put_part<NL>(sm.y + 128 * r, j, ct, acc);
                    }
                    // da takes 0 times the state before a missing token, which may be infinite
                    if (decltype(mode)::value == kChecked)
                        for (int64_t r = te - t; r < kGroup; ++r) clear_lanes(sm.past[r - 1], lane);
#pragma unroll
                    for (int r = kGroup - 1; r >= 0; --r) {
                        reload();
                        float2 sv[2], pv[2], vv[2], b[4], c[4], dsum[2], gsum[2], db[4];
                        float dbs[4];
                        lds22(sm.s.step + r * CW + ct, sv);
                        lds22(sm.s.su + r * CW + ct, pv);
                        lds22(sm.v + r * CW + ct, vv);
                        lds_dup4(sm.s.b(r, j), b);
                        lds_dup4(sm.s.c(r, j), c);
                        dsum[0] = dsum[1] = gsum[0] = gsum[1] = make_float2(0.f, 0.f);
                        load_lanes(r > 0 ? sm.past[r - 1] : sm.h[gi], lane, v16);
                        pair_up(v16, h);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            db[i] = make_float2(0.f, 0.f);
#pragma unroll
                            for (int q = 0; q < 2; ++q) {
                                const int k = 2 * i + q;
                                g[k] = ffma2(c[i], vv[q], g[k]);
                                gsum[q] = ffma2(b[i], g[k], gsum[q]);
                                db[i] = ffma2(pv[q], g[k], db[i]);
                                g[k] = fmul2(g[k], e[r][k]);
                                const float2 w = fmul2(g[k], h[k]);
                                da[k] = ffma2(sv[q], w, da[k]);
                                dsum[q] = ffma2(a2[k], w, dsum[q]);
                            }
                            dbs[i] = db[i].x + db[i].y;
                        }
                        __syncwarp();  // every lane has read the state that the sums replace
                        float* sums = r > 0 ? sm.past[r - 1] : sm.h[gi];
                        put_part<NL>(sums, j, ct, dsum);
                        put_part<NL>(sums + 128, j, ct, gsum);
                        put_bc<NL>(sums + 256, j, lane % CL, dbs, dcs[r]);
                    }
                };
                if (fast) pass(std::integral_constant<int, kMixed>{});
                else pass(std::integral_constant<int, kChecked>{});
                __syncwarp();
                auto sums_of = [&](int r) { return r > 0 ? sm.past[r - 1] : sm.h[gi]; };
                sum_bc<NL>([&](int r) { return sums_of(r) + 256; }, lane, te - t, pbc + t * ps, ps);
#pragma unroll
                for (int x = 0; x < TE; ++x) {
                    const int r = own_t + x;
                    const int64_t row = t + r;
                    float2 yo[P], dso[P], gbo[P], st2[P], du2[P], dd2[P], dz2[P], u2[P], r2[P], v2[P], z2[P];
                    float f[CE];
                    unpack<T, CE>(nu[x], u2);
                    unpack<T, CE>(nd[x], r2);
                    unpack<T, CE>(ndy[x], v2);
                    const float* sums = sums_of(r);
                    sum_parts<NL>(sums, own_c, dso);
                    sum_parts<NL>(sums + 128, own_c, gbo);
                    lds_v<CE>(sm.s.step + r * CW + own_c, f);
                    to_pairs<CE>(f, st2);
                    if (gated) {
                        sum_parts<NL>(sm.y + 128 * r, own_c, yo);
                        unpack<T, CE>(nz[x], z2);
#pragma unroll
                        for (int i = 0; i < P; ++i) {
                            // silu'(z) = sg (1 + z (1 - sg))
                            const float2 sg = sigmoid2(z2[i]), one = splat2(1.f);
                            const float2 slope = fmul2(sg, ffma2(z2[i], fsub2(one, sg), one));
                            dz2[i] = fmul2(fmul2(v2[i], ffma2(skip[i], u2[i], yo[i])), slope);
                            v2[i] = fmul2(v2[i], fmul2(z2[i], sg));
                        }
                    }
#pragma unroll
                    for (int i = 0; i < P; ++i) {
                        du2[i] = ffma2(st2[i], gbo[i], fmul2(skip[i], v2[i]));
                        dd2[i] = ffma2(u2[i], gbo[i], fmul2(splat2(kLn2), dso[i]));
                        if (p.softplus) dd2[i] = fmul2(dd2[i], sigmoid2(fadd2(r2[i], chn.bias[i])));
                    }
                    if (row < te) {
                        const int64_t off = row * ys;
                        float duo[CE], ddo[CE], dzo[CE];
                        from_pairs<CE>(du2, duo);
                        from_pairs<CE>(dd2, ddo);
                        from_pairs<CE>(dz2, dzo);
#pragma unroll
                        for (int i = 0; i < P; ++i) {
                            dskip[i] = ffma2(v2[i], u2[i], dskip[i]);
                            dbias[i] = fadd2(dbias[i], dd2[i]);
                        }
                        store_v<CE>(du + off, ec, cend, bp.vec, duo);
                        store_v<CE>(dd + off, ec, cend, bp.vec, ddo);
                        if (dz) store_v<CE>(dz + off, ec, cend, bp.vec, dzo);
                    }
                }
                __syncwarp();
            }
        }
        if (bp.dinitial && t0 == 0) {
            pair_down(g, v16);
            store_block<NL>(bp.dinitial + (int64_t)s * p.channels * N, c0, cend, j, v16);
        }
        pair_down(da, v16);
        store_lanes(bp.part_a + unit * 512, lane, v16);
        sum_tokens<NL>(dskip, lane, own_c, bp.part_d + (w.slot * 2 * tiles + tile) * CW);
        sum_tokens<NL>(dbias, lane, own_c, bp.part_d + ((w.slot * 2 + 1) * tiles + tile) * CW);
    }
}

// The sums that are left, in one launch (14 us at the sizes above; two took 9 and 13): blocks of da,
// dD and d delta_bias first (their columns are long), then blocks of db and dc.
struct Sums {
    float *da, *dd, *dbias;
    void *db, *dc;
    int64_t rows;  // of part_a and part_d
    int32_t row_blocks;
};

// db and dc: the channel tiles' partials of each group added in order.  A thread adds four states
// of one state lane j (j, j + N / 4, ...).  Rows of no sequence get zeros, in every gradient.
template <typename T, int NL>
__device__ __forceinline__ void sum_bc_tiles(const BwdParams& p, const Sums& to, int64_t block, int64_t blocks) {
    const float4* part = reinterpret_cast<const float4*>(p.part_bc);
    const int64_t tokens = p.tokens;
    const int groups = p.f.groups, tiles = p.f.tiles_per_group;
    constexpr int per = 2 * NL;
    zero_outside<T>(p.f.seqs, p.f.channels, block, blocks, p.du, p.ddelta, p.dz);
    const int64_t i = block * 256 + threadIdx.x;  // over [token][group][db, dc][state lane]
    if (i >= tokens * groups * per) return;
    const int w = (int)(i % per);
    const int64_t tg = i / per;
    const int64_t t = tg / groups;
    const int gr = (int)(tg % groups);
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    const bool none = Outside(p.f.seqs).has(t);
    for (int k = 0; k < tiles && !none; ++k) {
        const float4 v = part[((int64_t)(gr * tiles + k) * tokens + t) * per + w];
        sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
    }
    T* out = static_cast<T*>(w < NL ? to.db : to.dc) + (t * groups + gr) * 4 * NL + w % NL;
    out[0] = from_f<T>(sum.x);
    out[NL] = from_f<T>(sum.y);
    out[2 * NL] = from_f<T>(sum.z);
    out[3 * NL] = from_f<T>(sum.w);
}

// da, dD and d delta_bias: the partials' rows added in order, 8 outputs by 32 row lanes per block.
template <int NL>
__device__ __forceinline__ void sum_rows(const BwdParams& p, const Sums& to, float (&red)[32][9]) {
    constexpr int CW = Tile<NL>::CW, N = 4 * NL;
    const int tiles_per_group = p.f.tiles_per_group, tiles = p.f.groups * tiles_per_group, per_group = p.f.per_group;
    const int x = threadIdx.x % 8, r = threadIdx.x / 8;
    const int64_t i = (int64_t)blockIdx.x * 8 + x, na = (int64_t)tiles * 512, nd = (int64_t)tiles * CW;
    const float* src = i < na ? p.part_a + i : p.part_d + (i - na);
    const int64_t stride = i < na ? na : 2 * nd;
    float sum = 0.f;
    if (i < na + 2 * nd)
        for (int64_t k = r; k < to.rows; k += 32) sum += src[k * stride];
    red[r][x] = sum;
    __syncthreads();
    for (int o = 16; o > 0; o >>= 1) {
        if (r < o) red[r][x] += red[r + o][x];
        __syncthreads();
    }
    if (r != 0 || i >= na + 2 * nd) return;
    int tile, c, n = 0;
    if (i < na) {
        tile = (int)(i / 512);
        element<NL>((int)(i % 512), c, n);
    } else {
        tile = (int)((i - na) % nd / CW);
        c = (int)((i - na) % CW);
    }
    const int at = (tile % tiles_per_group) * CW + c;
    if (at >= per_group) return;
    const int ch = tile / tiles_per_group * per_group + at;
    if (i < na) to.da[(int64_t)ch * N + n] = red[0][x];
    else if (i < na + nd) { if (to.dd) to.dd[ch] = red[0][x]; }
    else if (to.dbias) to.dbias[ch] = red[0][x];
}

template <typename T, int NL>
__global__ void __launch_bounds__(256) sums_kernel(const BwdParams p, const Sums to) {
    __shared__ float red[32][9];
    wait_for_previous();
    if ((int)blockIdx.x < to.row_blocks) sum_rows<NL>(p, to, red);
    else sum_bc_tiles<T, NL>(p, to, (int64_t)blockIdx.x - to.row_blocks, (int64_t)gridDim.x - to.row_blocks);
}

struct Layout {
    int64_t tokens, rows, bc, a, d, total;  // floats
};
// Warps that a B200 holds of the backward kernel (two CTAs of three or four an SM).  Segments against
// whole chains of 784 tokens, by device time: bf16, 256 chains 251 against 567 us, 640 581 / 743, 768
// 707 / 750, 832 727 / 752; fp32, 512 573 / 724, 640 711 / 732, 768 846 / 735: whole chains from two
// thirds of the warps on (fp32's limit; bf16 would bear a few more segments).  Four segments a warp even
// out the last wave: 512 chains 480 us against 540 with one and 477 with two, 128 chains of 2048 tokens
// 308 / 332 / 324; eight 468 and 320.
int64_t bwd_warps(const vh_ssm_scan_args* a) { return (int64_t)(a->dtype == VH_F32 ? 6 : 8) * sm_count(); }

int bwd_segment_size(const vh_ssm_scan_args* a) { return segment_size(a, bwd_warps(a) * 2 / 3, 4 * bwd_warps(a), kCheckpoint); }

Layout layout_of(const vh_ssm_scan_args* a, int size) {
    Layout l;
    const bool packed = a->seq_offsets != nullptr;
    l.tokens = packed ? a->length : (int64_t)a->batch * a->length;
    const int64_t tiles = tile_count(a);
    l.rows = size ? slot_total(packed, a->length, a->batch, size) : a->batch;
    l.bc = tiles * l.tokens * 2 * a->states;
    l.a = l.rows * tiles * 512;
    l.d = l.rows * 2 * tiles * (128 / (a->states / 4));
    l.total = l.bc + l.a + l.d + segment_bytes(a, size) / 4;
    return l;
}

template <typename T, int NL>
int launch_bwd(const BwdParams& p, const Segments& g, cudaStream_t st) {
    constexpr int W = kBwdWarps<T>;
    const size_t smem = sizeof(BwdStage<T, NL>) * W, own = sizeof(OwnStage<T, NL>) * W;
    const int64_t items = (g.state ? g.slots : (int64_t)p.f.seqs.count) * p.f.groups * p.f.tiles_per_group;
    const int64_t blocks = (items + W - 1) / W;
    if (blocks > 0x7fffffff) return fail(VH_E_RANGE, "vh_ssm_scan_bwd: too many channel tiles");
    if (!ensure_smem_attr(reinterpret_cast<const void*>(&scan_bwd_kernel<T, NL, false>), smem) ||
        !ensure_smem_attr(reinterpret_cast<const void*>(&scan_bwd_kernel<T, NL, true>), own))
        return fail(VH_E_DEVICE, "vh_ssm_scan_bwd: cannot reserve %zu bytes of shared memory", smem);
    if (!g.state) {
        scan_bwd_kernel<T, NL, false><<<(int)blocks, 32 * W, smem, st>>>(p, g, items);
        return launch_status("selective scan backward");
    }
    scan_bwd_kernel<T, NL, true><<<(int)blocks, 32 * W, own, st>>>(p, g, items);
    if (int rc = launch_status("selective scan backward: own gradients")) return rc;
    if (int rc = enter_segments(p.f, 4 * NL, g, p.dfinal, true, st)) return rc;
    return launch_after("selective scan backward", scan_bwd_kernel<T, NL, false>, blocks, 32 * W, smem, st, p, g, items);
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
    for (const void* t : {(const void*)a->grad_final, (const void*)a->grad_initial, (const void*)a->grad_a,
                          (const void*)a->grad_d_skip, (const void*)a->grad_delta_bias})
        if (t && !aligned(t, 4)) return fail(VH_E_ALIGN, "%s: misaligned pointers", what);
    return 0;
}

}  // namespace
}  // namespace ssm
}  // namespace vh

using namespace vh;
using namespace vh::ssm;

extern "C" int64_t vh_ssm_scan_bwd_workspace_bytes(const vh_ssm_scan_bwd_args* a) {
    clear_error();
    if (check_bwd("vh_ssm_scan_bwd_workspace_bytes", a)) return 0;
    return layout_of(&a->fwd, bwd_segment_size(&a->fwd)).total * 4;
}

extern "C" int vh_ssm_scan_bwd(const vh_ssm_scan_bwd_args* a, void* workspace, int64_t workspace_bytes,
                               vh_stream_t stream) {
    clear_error();
    if (int rc = check_bwd("vh_ssm_scan_bwd", a)) return rc;
    const vh_ssm_scan_args* f = &a->fwd;
    const int size = bwd_segment_size(f);
    const Layout l = layout_of(f, size);
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
    Segments g;
    place_segments(f, size, static_cast<float*>(workspace) + l.a + l.bc + l.d, &g);
    p.tokens = l.tokens;
    p.vec = p.f.vec && aligned(a->grad_y, 4 * es) && aligned(a->grad_u, 4 * es) && aligned(a->grad_delta, 4 * es) &&
            (!p.dz || aligned(p.dz, 4 * es));
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int tiles = p.f.groups * p.f.tiles_per_group;
    return with_dtype(f->dtype, [&](auto t) {
        using T = decltype(t);
        return with_states(f->states, [&](auto nl) {
            constexpr int NL = decltype(nl)::value;
            if (int e = launch_bwd<T, NL>(p, g, st)) return e;
            const int64_t row_blocks = ((int64_t)tiles * (512 + 2 * Tile<NL>::CW) + 7) / 8;
            const int64_t bc_blocks = (l.tokens * f->groups * 2 * NL + 255) / 256;
            const Sums to{a->grad_a, a->grad_d_skip, a->grad_delta_bias, a->grad_b, a->grad_c, l.rows, (int32_t)row_blocks};
            return launch_after("selective scan backward: sums", sums_kernel<T, NL>, row_blocks + bc_blocks, 256, 0, st, p, to);
        });
    });
}
