// Selective scan, forward and one-token step (vh_ssm_scan_fwd, vh_ssm_scan_step).
#include <type_traits>

#include "ssm_scan.cuh"

namespace vh {
namespace ssm {
namespace {

// The forward scan: one warp per (sequence, channel tile), tokens in order (layout: ssm_scan.cuh).
template <typename T, int NL>
__global__ void __launch_bounds__(32 * kWarps) scan_fwd_kernel(const ScanParams p, int64_t items) {
    using K = Tile<NL>;
    constexpr int N = K::N, CW = K::CW, CE = K::CE, TE = K::TE;
    __shared__ __align__(16) float s_step[kWarps][kGroup * CW];
    __shared__ __align__(16) float s_su[kWarps][kGroup * CW];
    __shared__ __align__(16) float s_bc[kWarps][kGroup * 2 * N];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int tiles = p.groups * p.tiles_per_group;
    const int64_t item = (int64_t)blockIdx.x * kWarps + warp;
    if (item >= items) return;
    const int s = (int)(item / tiles), tile = (int)(item % tiles);
    const int group = tile / p.tiles_per_group;
    const int cbase = group * p.per_group + (tile % p.tiles_per_group) * CW;
    const int cend = (group + 1) * p.per_group;
    const Seq seq = seq_at(p.seqs, s);
    const LaneElems<NL> own(lane);
    const int n0 = 4 * (lane / K::CL), c0 = cbase + 4 * (lane % K::CL);  // the thread's 4 x 4 block
    const int ec = cbase + own.c0;                                      // its elements' first channel
    float *step = s_step[warp], *su = s_su[warp], *bc = s_bc[warp];

    const T* u = static_cast<const T*>(p.u) + first_row(p.seqs, seq, s, p.ur) + ec;
    const T* dl = static_cast<const T*>(p.delta) + first_row(p.seqs, seq, s, p.dr) + ec;
    const T* z = p.z ? static_cast<const T*>(p.z) + first_row(p.seqs, seq, s, p.zr) + ec : nullptr;
    const T* b = static_cast<const T*>(p.b) + first_row(p.seqs, seq, s, p.br) + group * p.bg;
    const T* c = static_cast<const T*>(p.c) + first_row(p.seqs, seq, s, p.cr) + group * p.cg;
    const int64_t us = row_step(p.seqs, p.ur), ds = row_step(p.seqs, p.dr), zs = row_step(p.seqs, p.zr);
    const int64_t bs = row_step(p.seqs, p.br), cs = row_step(p.seqs, p.cr);
    const Rows yr{p.seqs.length * p.channels, p.channels};
    T* y = static_cast<T*>(p.y) + first_row(p.seqs, seq, s, yr) + ec;
    const int64_t ys = row_step(p.seqs, yr);

    float a2[16], h[16];
    load_block<N>(p.a, c0, cend, n0, a2);
#pragma unroll
    for (int i = 0; i < 16; ++i) a2[i] = to_log2(a2[i]);
    if (p.initial) load_block<N>(p.initial + (int64_t)s * p.channels * N, c0, cend, n0, h);
    else
#pragma unroll
        for (int i = 0; i < 16; ++i) h[i] = 0.f;
    float bias[CE], skip[CE];
#pragma unroll
    for (int i = 0; i < CE; ++i) {
        bias[i] = p.delta_bias && ec + i < cend ? p.delta_bias[ec + i] : 0.f;
        skip[i] = p.d_skip && ec + i < cend ? p.d_skip[ec + i] : 0.f;
    }
    float* ck = p.checkpoints ? p.checkpoints + slot_base(p.seqs, s, seq.row, kCheckpoint) * p.channels * N : nullptr;

    for (int64_t t = 0; t < seq.len; t += kGroup) {
        const int cnt = seq.len - t < kGroup ? (int)(seq.len - t) : kGroup;
        if (ck && t % kCheckpoint == 0) store_block<N>(ck + (t / kCheckpoint) * p.channels * N, c0, cend, n0, h);
        float ue[TE][CE], ze[TE][CE];
#pragma unroll
        for (int e = 0; e < TE; ++e) {
            const int r = own.t0 + e;
            float de[CE], prod[CE];
#pragma unroll
            for (int i = 0; i < CE; ++i) ue[e][i] = ze[e][i] = de[i] = 0.f;
            if (r < cnt) {
                load_v<CE>(u + (t + r) * us, ec, cend, p.vec, ue[e]);
                load_v<CE>(dl + (t + r) * ds, ec, cend, p.vec, de);
                if (z) load_v<CE>(z + (t + r) * zs, ec, cend, p.vec, ze[e]);
#pragma unroll
                for (int i = 0; i < CE; ++i) {
                    de[i] += bias[i];
                    if (p.softplus) de[i] = softplus(de[i]);
                }
            }
#pragma unroll
            for (int i = 0; i < CE; ++i) prod[i] = de[i] * ue[e][i];
            sts_v<CE>(step + r * CW + own.c0, de);
            sts_v<CE>(su + r * CW + own.c0, prod);
        }
        stage_bc<NL>(b + t * bs, c + t * cs, bs, cs, cnt, p.vec_bc, lane, bc);
        __syncwarp();
        float acc[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[i] = 0.f;
#pragma unroll
        for (int r = 0; r < kGroup; ++r) {
            float sv[4], pv[4], bv[4], cv[4];
            lds4(step + r * CW + 4 * (lane % K::CL), sv);
            lds4(su + r * CW + 4 * (lane % K::CL), pv);
            lds4(bc + r * 2 * N + n0, bv);
            lds4(bc + r * 2 * N + N + n0, cv);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    float& hh = h[4 * i + n];
                    hh = fmaf(pv[i], bv[n], exp2_fma(sv[i] * a2[4 * i + n]) * hh);
                    acc[4 * r + i] = fmaf(cv[n], hh, acc[4 * r + i]);
                }
        }
        __syncwarp();
        reduce_scatter<16, NL, K::CL>(acc, lane);
#pragma unroll
        for (int e = 0; e < TE; ++e) {
            const int r = own.t0 + e;
            float out[CE];
#pragma unroll
            for (int i = 0; i < CE; ++i) {
                out[i] = fmaf(skip[i], ue[e][i], acc[e * CE + i]);
                if (z) out[i] *= ze[e][i] * sigmoid(ze[e][i]);
            }
            if (r < cnt) store_v<CE>(y + (t + r) * ys, ec, cend, p.vec, out);
        }
    }
    if (p.final_state) store_block<N>(p.final_state + (int64_t)s * p.channels * N, c0, cend, n0, h);
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
            hv[n] = fmaf(pu, bv[n], exp2_fma(st * to_log2(av[n])) * hv[n]);
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

}  // namespace ssm
}  // namespace vh

using namespace vh;
using namespace vh::ssm;

extern "C" int64_t vh_ssm_scan_checkpoint_slots(const vh_ssm_scan_args* a) {
    if (!a || a->batch <= 0 || a->length < 0) return 0;
    return slot_total(a->seq_offsets != nullptr, a->length, a->batch, kCheckpoint);
}

extern "C" int64_t vh_ssm_scan_fwd_workspace_bytes(const vh_ssm_scan_args*) { return 0; }

extern "C" int vh_ssm_scan_fwd(const vh_ssm_scan_args* a, void*, int64_t, vh_stream_t stream) {
    clear_error();
    if (int rc = check_scan_args("vh_ssm_scan_fwd", a, false)) return rc;
    ScanParams p;
    fill_scan_params(a, &p);
    const int64_t items = (int64_t)a->batch * p.groups * p.tiles_per_group;
    const int64_t blocks = (items + kWarps - 1) / kWarps;
    if (blocks > 0x7fffffff) return fail(VH_E_RANGE, "vh_ssm_scan_fwd: too many channel tiles");
    return with_dtype(a->dtype, [&](auto t) {
        using T = decltype(t);
        return with_states(a->states, [&](auto nl) {
            scan_fwd_kernel<T, decltype(nl)::value>
                <<<(int)blocks, 32 * kWarps, 0, static_cast<cudaStream_t>(stream)>>>(p, items);
            return launch_status("selective scan");
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
