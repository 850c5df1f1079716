// Selective scan, forward and one-token step (vh_ssm_scan_fwd, vh_ssm_scan_step).
#include "ssm_scan.cuh"

namespace vh {
namespace ssm {
namespace {

constexpr int kWarps = 4;        // one warp a chain: warps per CTA, neighbouring channel tiles
constexpr int kSplitWarps = 16;  // many warps a chain: warps per CTA, consecutive segments

// Four staged tokens; Y: also y's partial sums (pairs of channels, over the thread's states).
template <int NL, int MODE, bool Y>
__device__ __forceinline__ void advance(const Stage<NL>& st, int ct, int j, const float2 (&a2)[8], float2 (&h)[8],
                                        float (&acc)[16]) {
    using K = Tile<NL>;
#pragma unroll
    for (int r = 0; r < kGroup; ++r) {
        float2 s[2], su[2], b[4], e[8];
        lds22(st.step + r * K::CW + ct, s);
        lds22(st.su + r * K::CW + ct, su);
        lds_dup4(st.b(r, j), b);
        decays<MODE>(s, a2, e);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int p = 0; p < 2; ++p) h[2 * i + p] = ffma2(e[2 * i + p], h[2 * i + p], fmul2(su[p], b[i]));
        if constexpr (Y) {
            float2 c[4], y[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
            lds_dup4(st.c(r, j), c);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int p = 0; p < 2; ++p) y[p] = ffma2(c[i], h[2 * i + p], y[p]);
            acc[4 * r] = y[0].x; acc[4 * r + 1] = y[0].y; acc[4 * r + 2] = y[1].x; acc[4 * r + 3] = y[1].y;
        }
    }
}

// The forward scan.  A chain is a channel tile of a sequence.
// SPLIT = false: one warp walks a chain, four neighbouring chains a CTA.
// SPLIT = true, for few chains: the sixteen warps of a CTA, and the CTAs of a cluster, take
// consecutive segments of one chain.  Each warp first runs its segment from a zero state, without
// outputs.  A segment maps the state before it to exp(a sum s) h + own state, so the states before
// all segments follow from the sixteen own states and step sums of each CTA (512 threads, one
// state each) and the totals of the CTAs before it, read from their shared memory.  Then each
// warp runs its segment again from its true state.  Twice the exponentials, against the length
// of a chain divided by up to 128.
template <typename T, int NL, bool SPLIT>
__global__ void __launch_bounds__(32 * (SPLIT ? kSplitWarps : kWarps), SPLIT ? 1 : 3)
    scan_fwd_kernel(const ScanParams p, int64_t chains, int cluster) {
    using K = Tile<NL>;
    constexpr int CE = K::CE, TE = K::TE;
    constexpr int W = SPLIT ? kSplitWarps : kWarps;
    extern __shared__ __align__(16) unsigned char smem[];
    Stage<NL>* stages = reinterpret_cast<Stage<NL>*>(smem);
    // split only: what leaves and enters the segments
    float* states = reinterpret_cast<float*>(stages + 2 * W);
    SplitSmem<NL, W>& sp = *reinterpret_cast<SplitSmem<NL, W>*>(states + 512 * W);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int tiles = p.groups * p.tiles_per_group;
    const int64_t chain = SPLIT ? blockIdx.x / cluster : (int64_t)blockIdx.x * W + warp;
    if (!SPLIT && chain >= chains) return;
    const int s = (int)(chain / tiles), tile = (int)(chain % tiles);
    const Seq seq = seq_at(p.seqs, s);
    Chain<T, NL> ch(p, seq, s, tile, lane);
    const int j = lane / K::CL, ct = 4 * (lane % K::CL), c0 = ch.cbase + ct;  // the thread's 4 x 4 block
    const int ec = ch.ec, cend = ch.cend;
    Stage<NL>* st = stages + 2 * warp;
    const Rows yr{p.seqs.length * p.channels, p.channels};
    T* y = static_cast<T*>(p.y) + first_row(p.seqs, seq, s, yr) + ec;
    const int64_t ys = row_step(p.seqs, yr);
    float skip[CE];
#pragma unroll
    for (int i = 0; i < CE; ++i) skip[i] = p.d_skip && ec + i < cend ? p.d_skip[ec + i] : 0.f;
    const float* initial = p.initial ? p.initial + (int64_t)s * p.channels * K::N : nullptr;
    float2 a2[8], h[8];
    float v[16];
    const float top_a = load_rates<NL>(p, c0, cend, j, v);
    pair_up(v, a2);

    int64_t t0 = 0, t1 = seq.len;
    if constexpr (SPLIT) {
        if (warp == 0) store_lanes(sp.a2, lane, v);
        const int rank = blockIdx.x % cluster;
        const int seg = rank * W + warp, segs = cluster * W;
        const int64_t size = max((seq.len + segs - 1) / segs + kGroup - 1, (int64_t)4 * kGroup) / kGroup * kGroup;
        t0 = min(seq.len, seg * size);
        t1 = min(seq.len, t0 + size);
        float sum[CE];
#pragma unroll
        for (int i = 0; i < 8; ++i) h[i] = make_float2(0.f, 0.f);
#pragma unroll
        for (int i = 0; i < CE; ++i) sum[i] = 0.f;
        if (t1 < seq.len) {  // what leaves the last segment is not needed
            Chain<T, NL> at = ch;
            at.move(t0);
            typename Chain<T, NL>::Raw raw;
            at.template load<false>(raw, t1 - t0);
            int buf = 0;
            for (int64_t t = t0; t < t1; t += kGroup, buf ^= 1) {
                const float top = at.template stage<true>(raw, t1 - t, st[buf], sum);
                __syncwarp();
                at.move(kGroup);
                if (t + kGroup < t1) at.template load<false>(raw, t1 - t - kGroup);
                if (top * top_a <= 126.f) advance<NL, kMixed, false>(st[buf], ct, j, a2, h, v);
                else advance<NL, kChecked, false>(st[buf], ct, j, a2, h, v);
            }
            __syncwarp();
        }
        pair_down(h, v);
        store_lanes(states + 512 * warp, lane, v);
        sum_tokens<NL>(sum, lane, ch.own_c, sp.sigma[warp]);
        enter_segments<NL, W, false>(sp, [&](int w) { return states + 512 * w; }, initial, ch.cbase, cend, cluster, rank);
        load_lanes(states + 512 * warp, lane, v);
    } else if (initial) {
        load_block<NL>(initial, c0, cend, j, v);
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = 0.f;
    }
    pair_up(v, h);

    float* ck = p.checkpoints
                    ? p.checkpoints + (slot_base(p.seqs, s, seq.row, kCheckpoint) * tiles + tile) * 512 : nullptr;
    if (t0 < t1) {
        float unused[CE];
#pragma unroll
        for (int i = 0; i < CE; ++i) unused[i] = 0.f;
        ch.move(t0);
        y += (t0 + ch.own_t) * ys;
        typename Chain<T, NL>::Raw raw;
        ch.template load<true>(raw, t1 - t0);
        int buf = 0;
        for (int64_t t = t0; t < t1; t += kGroup, buf ^= 1) {
            if (ck && t % kCheckpoint == 0) {
                pair_down(h, v);
                store_lanes(ck + (t / kCheckpoint) * tiles * 512, lane, v);
            }
            const float top = ch.template stage<false>(raw, t1 - t, st[buf], unused);
            float ue[TE][CE], ze[TE][CE];
#pragma unroll
            for (int e = 0; e < TE; ++e) {
                raw.u[e].get(ue[e]);
                if (ch.gated) raw.z[e].get(ze[e]);
            }
            __syncwarp();
            ch.move(kGroup);
            if (t + kGroup < t1) ch.template load<true>(raw, t1 - t - kGroup);
            float acc[16];
            if (top * top_a <= 126.f) advance<NL, kMixed, true>(st[buf], ct, j, a2, h, acc);
            else advance<NL, kChecked, true>(st[buf], ct, j, a2, h, acc);
            reduce_scatter<16, NL, K::CL>(acc, lane);
#pragma unroll
            for (int e = 0; e < TE; ++e) {
                float out[CE];
#pragma unroll
                for (int i = 0; i < CE; ++i) {
                    out[i] = fmaf(skip[i], ue[e][i], acc[e * CE + i]);
                    if (ch.gated) out[i] *= ze[e][i] * sigmoid(ze[e][i]);
                }
                if (t + ch.own_t + e < t1) store_v<CE>(y + e * ys, ec, cend, p.vec, out);
            }
            y += kGroup * ys;
        }
    }
    // the last token's warp, or for an empty sequence the first one
    const bool ends = seq.len > 0 ? t0 < t1 && t1 == seq.len : (!SPLIT || (warp == 0 && blockIdx.x % cluster == 0));
    if (p.final_state && ends) {
        pair_down(h, v);
        store_block<NL>(p.final_state + (int64_t)s * p.channels * K::N, c0, cend, j, v);
    }
    if (SPLIT && cluster > 1) cluster_wait();
}

// One token per stream: a thread owns four states of one channel, N / 4 threads a channel.
template <typename T, int NL>
__global__ void __launch_bounds__(256) scan_step_kernel(const ScanParams p, const float* state,
                                                        float* state_out,
                                                        const int32_t* __restrict__ index, int32_t slots, int64_t rows) {
    constexpr int N = 4 * NL;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t row = i / NL;  // (stream, channel); whole groups of NL lanes are in or out together
    const int n0 = 4 * (int)(i % NL);
    const bool live = row < rows;
    const int s = live ? (int)(row / p.channels) : 0, c = live ? (int)(row % p.channels) : 0;
    const int slot = !live ? -1 : (index ? index[s] : s);
    const bool known = slot >= 0 && slot < slots;
    float part = 0.f, uu = 0.f, zz = 0.f;
    if (known) {
        const int g = c / p.per_group;
        uu = to_f(static_cast<const T*>(p.u)[s * p.ur.batch + c]);
        float st = to_f(static_cast<const T*>(p.delta)[s * p.dr.batch + c]) + (p.delta_bias ? p.delta_bias[c] : 0.f);
        if (p.z) zz = to_f(static_cast<const T*>(p.z)[s * p.zr.batch + c]);
        if (p.softplus) st = softplus(st);
        float av[4], hv[4], bv[4], cv[4];
        lds4(p.a + (int64_t)c * N + n0, av);
        lds4(state + ((int64_t)slot * p.channels + c) * N + n0, hv);
        load_v<4>(static_cast<const T*>(p.b) + s * p.br.batch + g * p.bg + n0, 0, 4, p.vec_bc, bv);
        load_v<4>(static_cast<const T*>(p.c) + s * p.cr.batch + g * p.cg + n0, 0, 4, p.vec_bc, cv);
        const float pu = st * uu;
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            hv[n] = fmaf(pu, bv[n], exp2_fma(st, to_log2(av[n])) * hv[n]);
            part = fmaf(cv[n], hv[n], part);
        }
        *reinterpret_cast<float4*>(state_out + ((int64_t)slot * p.channels + c) * N + n0) =
            make_float4(hv[0], hv[1], hv[2], hv[3]);
    }
#pragma unroll
    for (int o = NL / 2; o > 0; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
    if (live && n0 == 0) {
        float out = 0.f;
        if (known) {
            out = fmaf(p.d_skip ? p.d_skip[c] : 0.f, uu, part);
            if (p.z) out *= zz * sigmoid(zz);
        }
        static_cast<T*>(p.y)[(int64_t)s * p.channels + c] = from_f<T>(out);
    }
}

bool stride_ok(int64_t v, int m) { return v % m == 0; }

template <typename T, int NL>
int launch_fwd(const ScanParams& p, int64_t chains, cudaStream_t st) {
    // One warp a chain once there are two for each of the SM's four schedulers; fewer chains, and
    // packed sequences, whose lengths the host does not know, are split.
    const bool split = p.seqs.length > 4 * kGroup && (chains < 8 * sm_count() || p.seqs.offsets);
    if (!split) {
        const size_t smem = sizeof(Stage<NL>) * 2 * kWarps;
        if (!ensure_smem_attr(reinterpret_cast<const void*>(&scan_fwd_kernel<T, NL, false>), smem))
            return fail(VH_E_DEVICE, "vh_ssm_scan_fwd: cannot reserve %zu bytes of shared memory", smem);
        const int64_t blocks = (chains + kWarps - 1) / kWarps;
        if (blocks > 0x7fffffff) return fail(VH_E_RANGE, "vh_ssm_scan_fwd: too many channel tiles");
        scan_fwd_kernel<T, NL, false><<<(int)blocks, 32 * kWarps, smem, st>>>(p, chains, 1);
        return launch_status("selective scan");
    }
    const size_t smem = (sizeof(Stage<NL>) * 2 + 2048) * kSplitWarps + sizeof(SplitSmem<NL, kSplitWarps>);
    if (!ensure_smem_attr(reinterpret_cast<const void*>(&scan_fwd_kernel<T, NL, true>), smem))
        return fail(VH_E_DEVICE, "vh_ssm_scan_fwd: cannot reserve %zu bytes of shared memory", smem);
    static std::atomic<int> known[64][9];
    const int cluster = pick_cluster(scan_fwd_kernel<T, NL, true>, known, 32 * kSplitWarps, smem, chains,
                                     p.seqs.length, 4 * kGroup);
    return launch_cluster("selective scan", scan_fwd_kernel<T, NL, true>, chains * cluster, 32 * kSplitWarps, smem, cluster,
                          st, p, chains, cluster);
}

}  // namespace

int check_scan_args(const char* what, const vh_ssm_scan_args* a, bool one_token) {
    if (!a) return fail(VH_E_ARG, "%s: null argument struct", what);
    if (!a->u || !a->delta || !a->b || !a->c || !a->a || !a->y) return fail(VH_E_ARG, "%s: null pointer argument", what);
    if (!dtype_ok(a->dtype)) return fail(VH_E_DTYPE, "%s: dtype must be VH_F32, VH_BF16 or VH_F16", what);
    if (a->states != 4 && a->states != 8 && a->states != 16 && a->states != 32 && a->states != 64)
        return fail(VH_E_SHAPE, "%s: states must be 4, 8, 16, 32 or 64 (got %d)", what, a->states);
    if (a->batch <= 0 || a->channels <= 0 || a->groups <= 0)
        return fail(VH_E_SHAPE, "%s: batch, channels and groups must be positive", what);
    if (a->channels % a->groups)
        return fail(VH_E_SHAPE, "%s: channels (%d) must be a multiple of groups (%d)", what, a->channels, a->groups);
    const size_t es = dtype_size(a->dtype);
    const void* typed[] = {a->u, a->delta, a->z, a->b, a->c, a->y};
    for (const void* t : typed)
        if (t && !aligned(t, es)) return fail(VH_E_ALIGN, "%s: misaligned pointers", what);
    if (!aligned(a->a, 16) || (a->initial_state && !aligned(a->initial_state, 16)) ||
        (a->final_state && !aligned(a->final_state, 16)) || (a->checkpoints && !aligned(a->checkpoints, 16)))
        return fail(VH_E_ALIGN, "%s: a and the states must be 16-byte aligned", what);
    if (!one_token) {
        if (a->length < 0) return fail(VH_E_SHAPE, "%s: negative length", what);
        if (a->length > 0x7fffffff) return fail(VH_E_RANGE, "%s: at most 2^31 - 1 tokens a sequence", what);
        if (a->seq_offsets && !aligned(a->seq_offsets, 4)) return fail(VH_E_ALIGN, "%s: misaligned offsets", what);
    }
    return 0;
}

void fill_scan_params(const vh_ssm_scan_args* a, ScanParams* p) {
    p->u = a->u; p->delta = a->delta; p->z = a->z; p->b = a->b; p->c = a->c;
    p->ur = {a->u_batch_stride, a->u_token_stride};
    p->dr = {a->delta_batch_stride, a->delta_token_stride};
    p->zr = {a->z_batch_stride, a->z_token_stride};
    p->br = {a->b_batch_stride, a->b_token_stride};
    p->cr = {a->c_batch_stride, a->c_token_stride};
    p->bg = a->b_group_stride; p->cg = a->c_group_stride;
    p->a = a->a; p->d_skip = a->d_skip; p->delta_bias = a->delta_bias; p->initial = a->initial_state;
    p->y = a->y; p->final_state = a->final_state; p->checkpoints = a->checkpoints;
    p->seqs = {a->seq_offsets, a->length, a->batch, a->reverse != 0};
    p->channels = a->channels; p->groups = a->groups; p->per_group = a->channels / a->groups;
    const int nl = a->states / 4, cw = 128 / nl;
    p->tiles_per_group = (p->per_group + cw - 1) / cw;
    p->softplus = a->delta_softplus != 0;
    const size_t es = dtype_size(a->dtype);
    bool v = p->per_group % 4 == 0 && aligned(a->u, 4 * es) && aligned(a->delta, 4 * es) && aligned(a->y, 4 * es) &&
             (!a->z || aligned(a->z, 4 * es));
    for (int64_t st : {a->u_batch_stride, a->u_token_stride, a->delta_batch_stride, a->delta_token_stride})
        v = v && stride_ok(st, 4);
    if (a->z) v = v && stride_ok(a->z_batch_stride, 4) && stride_ok(a->z_token_stride, 4);
    p->vec = v;
    bool w = aligned(a->b, 4 * es) && aligned(a->c, 4 * es);
    for (int64_t st : {a->b_batch_stride, a->b_token_stride, a->b_group_stride, a->c_batch_stride, a->c_token_stride,
                       a->c_group_stride})
        w = w && stride_ok(st, 4);
    p->vec_bc = w;
}

// The checkpoints: a warp's states for every slot of 32 tokens and channel tile.
int64_t checkpoint_floats(const vh_ssm_scan_args* a) {
    const int cw = 128 / (a->states / 4), per = a->channels / a->groups;
    const int64_t tiles = (int64_t)a->groups * ((per + cw - 1) / cw);
    return slot_total(a->seq_offsets != nullptr, a->length, a->batch, kCheckpoint) * tiles * 512;
}

}  // namespace ssm
}  // namespace vh

using namespace vh;
using namespace vh::ssm;

extern "C" int64_t vh_ssm_scan_checkpoint_bytes(const vh_ssm_scan_args* a) {
    if (!a || a->batch <= 0 || a->length < 0 || a->channels <= 0 || a->groups <= 0 || a->channels % a->groups ||
        a->states < 4)
        return 0;
    return checkpoint_floats(a) * 4;
}

extern "C" int vh_ssm_scan_fwd(const vh_ssm_scan_args* a, vh_stream_t stream) {
    clear_error();
    if (int rc = check_scan_args("vh_ssm_scan_fwd", a, false)) return rc;
    ScanParams p;
    fill_scan_params(a, &p);
    const int64_t chains = (int64_t)a->batch * p.groups * p.tiles_per_group;
    return with_dtype(a->dtype, [&](auto t) {
        using T = decltype(t);
        return with_states(a->states, [&](auto nl) {
            return launch_fwd<T, decltype(nl)::value>(p, chains, static_cast<cudaStream_t>(stream));
        });
    });
}

extern "C" int vh_ssm_scan_step(const vh_ssm_scan_args* a, const float* state, float* state_out,
                                const int32_t* slots_index, int32_t slots, vh_stream_t stream) {
    clear_error();
    if (int rc = check_scan_args("vh_ssm_scan_step", a, true)) return rc;
    if (!state || !state_out) return fail(VH_E_ARG, "vh_ssm_scan_step: null state");
    if (!aligned(state, 16) || !aligned(state_out, 16))
        return fail(VH_E_ALIGN, "vh_ssm_scan_step: the states must be 16-byte aligned");
    if (slots <= 0 || (!slots_index && slots < a->batch))
        return fail(VH_E_SHAPE, "vh_ssm_scan_step: %d slots for %d streams", slots, a->batch);
    ScanParams p;
    fill_scan_params(a, &p);
    const int64_t rows = (int64_t)a->batch * a->channels;
    const int64_t blocks = (rows * (a->states / 4) + 255) / 256;
    if (blocks > 0x7fffffff) return fail(VH_E_RANGE, "vh_ssm_scan_step: too many channels");
    return with_dtype(a->dtype, [&](auto t) {
        using T = decltype(t);
        return with_states(a->states, [&](auto nl) {
            scan_step_kernel<T, decltype(nl)::value><<<(int)blocks, 256, 0, static_cast<cudaStream_t>(stream)>>>(
                p, state, state_out, slots_index, slots, rows);
            return launch_status("selective scan step");
        });
    });
}
