// Selective scan, forward and one-token step (vh_ssm_scan_fwd, vh_ssm_scan_step).
//
// The forward is bound by its exponentials and the arithmetic around them, not by memory: two
// images of 64 x 256 tokens, 384 channels, 16 states, bf16 (12.6 M elements, 103 MB) take 165 us,
// where the bytes would take 16 and the exponentials alone 45 for each of the two passes over a
// chain in segments.  The special-function unit is at 56 / 46 %, the FMA pipe at 57 / 52 % and
// instruction issue at 55 / 56 % in the first / last kernel (70 and about 90 us): their 105 M warp
// instructions alone would take 94 us at four a cycle and SM.
#include "ssm_scan.cuh"

namespace vh {
namespace ssm {
namespace {

constexpr int kWarps = 4;  // warps per CTA: neighbouring channel tiles

constexpr int kAhead = 2;  // groups fetched ahead (the latency of memory is about two groups' work)

// Shared memory of a warp.
template <typename T, int NL>
struct FwdSmem {
    Stage<NL> st[2];
    float part[512];
    typename Chain<T, NL>::Raw raw[kAhead + 1];
};

// Four staged tokens; Y: also y's partial sums over the thread's states, left in `part`.
template <int NL, int MODE, bool Y>
__device__ __forceinline__ void advance(const Stage<NL>& st, int ct, int j, const float2 (&a2)[8], float2 (&h)[8],
                                        float* part) {
    using K = Tile<NL>;
#pragma unroll
    for (int r = 0; r < kGroup; ++r) {
        float2 s[2], su[2], b[4], e[8];
        lds22(st.step + r * K::CW + ct, s);
        lds22(st.su + r * K::CW + ct, su);
        lds_dup4(st.b(r, j), b);
        decays<MODE, true>(s, a2, e);
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
            put_part<NL>(part + 128 * r, j, ct, y);
        }
    }
}

// The forward scan: a warp runs a channel tile of a sequence, or of a segment of one.
// OWN: the first of the three kernels of a chain in segments, without outputs: the segment's own
// state and sum of steps.
template <typename T, int NL, bool OWN>
__global__ void __launch_bounds__(32 * kWarps, 4) scan_fwd_kernel(const ScanParams p, const Segments g, int64_t items) {
    using K = Tile<NL>;
    constexpr int CE = K::CE, TE = K::TE;
    extern __shared__ __align__(16) unsigned char smem[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t item = (int64_t)blockIdx.x * kWarps + warp;
    if (OWN) launch_dependents();
    else zero_outside<T>(p.seqs, p.channels, blockIdx.x, gridDim.x, p.y);
    Unit w;
    if (item >= items || !unit_at(p, g, item, w)) return;
    const int tiles = p.groups * p.tiles_per_group;
    Chain<T, NL> ch(p, w.seq, w.s, w.tile, lane);
    const int j = lane / K::CL, ct = 4 * (lane % K::CL), c0 = ch.cbase + ct;  // the thread's 4 x 4 block
    const int ec = ch.ec, cend = ch.cend;
    FwdSmem<T, NL>& sm = reinterpret_cast<FwdSmem<T, NL>*>(smem)[warp];
    const int64_t unit = w.slot * tiles + w.tile;
    float2 a2[8], h[8];
    constexpr int P = kPairs<CE>;
    float v[16];
    float2 sum[P];
    const float most = mixed_limit(load_rates<NL>(p, c0, cend, j, v));
    pair_up(v, a2);
    ch.move(w.t0);
    // the last segment's own state is not needed
    const bool some = w.t0 < w.t1 && (!OWN || w.t1 < w.seq.len);
    // the first kAhead groups; every group is a commit of its own, empty past the end
    const int tokens = (int)(w.t1 - w.t0);
    int ahead = some ? tokens : 0;  // tokens still to fetch
    int slot = 0, next = 0;         // of the group at hand and the one fetched next
    auto fetch_next = [&]() {
        if (ahead > 0) {
            ch.template load<!OWN>(sm.raw[next], ahead);
            ch.advance();
            ahead -= kGroup;
        }
        cp_async_commit();
        next = next == kAhead ? 0 : next + 1;
    };
#pragma unroll
    for (int i = 0; i < kAhead; ++i) fetch_next();
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = 0.f;
#pragma unroll
    for (int i = 0; i < P; ++i) sum[i] = make_float2(0.f, 0.f);

    if constexpr (OWN) {
        pair_up(v, h);
        int buf = 0;
        for (int left = some ? tokens : 0; left > 0; left -= kGroup, buf ^= 1) {
            cp_async_wait<kAhead - 1>();
            const bool fast = ch.template stage<true, true>(sm.raw[slot], left, sm.st[buf], sum, most);
            slot = slot == kAhead ? 0 : slot + 1;
            __syncwarp();
            fetch_next();
            if (fast) advance<NL, kMixed, false>(sm.st[buf], ct, j, a2, h, nullptr);
            else advance<NL, kChecked, false>(sm.st[buf], ct, j, a2, h, nullptr);
        }
        pair_down(h, v);
        store_lanes(g.state + unit * 512, lane, v);
        sum_tokens<NL>(sum, lane, ch.own_c, g.sigma + unit * K::CW);
        return;
    }

    const Rows yr{p.seqs.length * p.channels, p.channels};
    const int64_t ys = row_step(p.seqs, yr);
    T* y = static_cast<T*>(p.y) + first_row(p.seqs, w.seq, w.s, yr) + ec + (w.t0 + ch.own_t) * ys;
    float2 skip[P];
    ch.load_params(p.d_skip, skip);
    if (g.state) {
        wait_for_previous();
        load_lanes(g.state + unit * 512, lane, v);
    } else if (p.initial) {
        load_block<NL>(p.initial + (int64_t)w.s * p.channels * K::N, c0, cend, j, v);
    }
    pair_up(v, h);
    float* ck = p.checkpoints ? p.checkpoints + (slot_base(p.seqs, w.s, w.seq.row, kCheckpoint) * tiles + w.tile) * 512
                              : nullptr;
    int buf = 0;
    if (ck) ck += (w.t0 + kCheckpoint - 1) / kCheckpoint * tiles * 512;
    int until = (int)((kCheckpoint - w.t0 % kCheckpoint) % kCheckpoint);  // tokens to the next saved state
    for (int left = tokens; left > 0; left -= kGroup, buf ^= 1) {
        if (ck) {
            if (until == 0) {
                pair_down(h, v);
                store_lanes(ck, lane, v);
                ck += (int64_t)tiles * 512;
                until = kCheckpoint;
            }
            until -= kGroup;
        }
        cp_async_wait<kAhead - 1>();
        const typename Chain<T, NL>::Raw& raw = sm.raw[slot];
        const bool fast = ch.template stage<false, true>(raw, left, sm.st[buf], sum, most);
        Pack<T, CE> nu[TE], nz[TE];
#pragma unroll
        for (int e = 0; e < TE; ++e) {
            nu[e] = raw.u[e][lane];
            if (ch.gated) nz[e] = raw.z[e][lane];
        }
        slot = slot == kAhead ? 0 : slot + 1;
        __syncwarp();
        fetch_next();
        if (fast) advance<NL, kMixed, true>(sm.st[buf], ct, j, a2, h, sm.part);
        else advance<NL, kChecked, true>(sm.st[buf], ct, j, a2, h, sm.part);
        __syncwarp();
#pragma unroll
        for (int e = 0; e < TE; ++e) {
            float2 y2[P], u2[P];
            sum_parts<NL>(sm.part + 128 * (ch.own_t + e), ch.own_c, y2);
            unpack<T, CE>(nu[e], u2);
#pragma unroll
            for (int i = 0; i < P; ++i) y2[i] = ffma2(skip[i], u2[i], y2[i]);
            if (ch.gated) {
                unpack<T, CE>(nz[e], u2);
#pragma unroll
                for (int i = 0; i < P; ++i) y2[i] = fmul2(y2[i], fmul2(u2[i], sigmoid2(u2[i])));
            }
            float out[CE];
            from_pairs<CE>(y2, out);
            if (ch.own_t + e < left) store_v<CE>(y + e * ys, ec, cend, p.vec, out);
        }
        y += kGroup * ys;
    }
    if (p.final_state && w.t1 == w.seq.len) {
        pair_down(h, v);
        store_block<NL>(p.final_state + (int64_t)w.s * p.channels * K::N, c0, cend, j, v);
    }
}

// What leaves a segment.  Zero stays zero, although a decay above 1 (a rate or a step against the sign) may
// be infinite over a whole segment.
__device__ __forceinline__ float carry(float decay, float state, float own) {
    return state == 0.f ? own : fmaf(decay, state, own);
}

// What enters every segment of a chain: a thread holds four states (one of four channels) and one
// of RUNS runs of segments.  It composes its run, the CTA chains the runs, and it walks its run
// again.  A CTA has 128 / PARTS of a chain's 128 such fours.
template <int NL, int RUNS, int PARTS>
__global__ void __launch_bounds__(RUNS * 128 / PARTS) enter_segments_kernel(const ScanParams p, const Segments g,
                                                                            const float* __restrict__ first, int right) {
    constexpr int kWide = 128 / PARTS;
    __shared__ float4 s_dec[RUNS][kWide], s_add[RUNS][kWide];
    constexpr int CW = Tile<NL>::CW, N = 4 * NL;
    launch_dependents();
    const int tiles = p.groups * p.tiles_per_group;
    const int64_t chain = blockIdx.x / PARTS;
    const int tile = (int)(chain % tiles), s = (int)(chain / tiles);
    const int run = threadIdx.x / kWide, lane = threadIdx.x % kWide;
    const int x = 4 * ((blockIdx.x % PARTS) * kWide + lane);
    int c, n;
    element<NL>(x, c, n);
    const int ch = tile / p.tiles_per_group * p.per_group + (tile % p.tiles_per_group) * CW + c;
    const int left = p.per_group - ((tile % p.tiles_per_group) * CW + c);
    float a2[4], in[4];  // in: what enters
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        a2[i] = i < left ? to_log2(p.a[(int64_t)(ch + i) * N + n]) : 0.f;
        in[i] = first && i < left ? first[((int64_t)s * p.channels + ch + i) * N + n] : 0.f;
    }
    const Seq seq = seq_at(p.seqs, s);
    const int segs = (int)slots_per_seq(seq.len, g.size), each = (segs + RUNS - 1) / RUNS;
    const int k0 = min(segs, run * each), k1 = min(segs, k0 + each);
    const int64_t base = slot_base(p.seqs, s, seq.row, g.size);
    // segment k of the walk: its states and its sums of steps
    const int64_t unit0 = (base + (right ? segs - 1 : 0)) * tiles + tile, by = right ? -tiles : tiles;
    float* state = g.state + unit0 * 512 + x;
    const float* sigma = g.sigma + unit0 * CW + c;
    wait_for_previous();
    if constexpr (RUNS > 1) {
        float dec[4] = {1.f, 1.f, 1.f, 1.f}, add[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
        for (int k = k0; k < k1; ++k) {
            float own[4], sg[4];
            lds4(state + k * by * 512, own);
            lds4(sigma + k * by * CW, sg);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float d = exp2_fma(sg[i], a2[i]);
                add[i] = carry(d, add[i], own[i]);
                dec[i] *= d;
            }
        }
        s_dec[run][lane] = make_float4(dec[0], dec[1], dec[2], dec[3]);
        s_add[run][lane] = make_float4(add[0], add[1], add[2], add[3]);
        __syncthreads();
        for (int r = 0; r < run; ++r) {
            const float4 d = s_dec[r][lane], e = s_add[r][lane];
            in[0] = carry(d.x, in[0], e.x);
            in[1] = carry(d.y, in[1], e.y);
            in[2] = carry(d.z, in[2], e.z);
            in[3] = carry(d.w, in[3], e.w);
        }
    }
    // four segments' loads at a time: the stores between them would hold the loads back
    for (int k = k0; k < k1; k += 4) {
        float own[4][4], sg[4][4];
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            const int64_t at = min(k + m, k1 - 1) * by;
            lds4(state + at * 512, own[m]);
            lds4(sigma + at * CW, sg[m]);
        }
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            if (k + m < k1)
                *reinterpret_cast<float4*>(state + (k + m) * by * 512) = make_float4(in[0], in[1], in[2], in[3]);
#pragma unroll
            for (int i = 0; i < 4; ++i) in[i] = carry(exp2_fma(sg[m][i], a2[i]), in[i], own[m][i]);
        }
    }
}

// One token per stream.  NL = N / 4 lanes share NL channels: a lane loads u, delta and z of its own
// channel and finishes its y, and holds four states of all NL channels; s and s u of a channel
// come from its lane, y's sums go back there.  A block keeps its channels' rates over several
// streams where registers allow.  Bound by latency: 256 streams of 2048 channels, 16 states, bf16,
// take 20 us for 71 MB (3.6 TB/s; the peak's 11 us would need more than the 32 warps of 64 registers
// an SM holds).  A softplus in every lane and rates read for every stream took 31.
template <typename T, int NL>
__global__ void __launch_bounds__(256, NL <= 4 ? 4 : 1) scan_step_kernel(const ScanParams p, const float* state, float* state_out,
                                                        const int32_t* __restrict__ index, int32_t slots) {
    constexpr int N = 4 * NL;
    constexpr bool kKeep = NL <= 4;
    const int c = blockIdx.x * 256 + threadIdx.x, lane = threadIdx.x & 31;
    const int j = lane % NL, first = c - j;
    const bool live = c < p.channels;
    const int group = min(c, p.channels - 1) / p.per_group;
    const float bias = live && p.delta_bias ? p.delta_bias[c] : 0.f, skip = live && p.d_skip ? p.d_skip[c] : 0.f;
    float a2[kKeep ? NL : 1][4];
    auto rates = [&](int i, float (&v)[4]) {
        lds4(p.a + (int64_t)min(first + i, p.channels - 1) * N + 4 * j, v);
#pragma unroll
        for (int n = 0; n < 4; ++n) v[n] = to_log2(v[n]);
    };
    if constexpr (kKeep)
#pragma unroll
        for (int i = 0; i < NL; ++i) rates(i, a2[i]);
    for (int s = blockIdx.y; s < p.seqs.count; s += gridDim.y) {
        const int slot = index ? index[s] : s;
        if (slot < 0 || slot >= slots) {  // the same for the whole block
            if (live) static_cast<T*>(p.y)[(int64_t)s * p.channels + c] = from_f<T>(0.f);
            continue;
        }
        const int64_t at = (int64_t)slot * p.channels * N + 4 * j;
        float h[NL][4];
#pragma unroll
        for (int i = 0; i < NL; ++i) lds4(state + at + (int64_t)min(first + i, p.channels - 1) * N, h[i]);
        float uu = 0.f, st = 0.f, zz = 0.f;
        if (live) {
            uu = to_f(static_cast<const T*>(p.u)[s * p.ur.batch + c]);
            st = to_f(static_cast<const T*>(p.delta)[s * p.dr.batch + c]) + bias;
            if (p.z) zz = to_f(static_cast<const T*>(p.z)[s * p.zr.batch + c]);
        }
        if (p.softplus) st = softplus(st);
        const float pu = st * uu;
        const T *pb = static_cast<const T*>(p.b) + s * p.br.batch, *pc = static_cast<const T*>(p.c) + s * p.cr.batch;
        float y[NL], bv[4], cv[4];
        int held = -1;
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            const float si = __shfl_sync(0xffffffffu, st, i, NL), pi = __shfl_sync(0xffffffffu, pu, i, NL);
            const int gi = p.groups == 1 ? 0 : __shfl_sync(0xffffffffu, group, i, NL);
            if (gi != held) {  // a group of lanes may straddle two groups of B and C
                load_four(pb + gi * p.bg + 4 * j, p.vec_bc, bv);
                load_four(pc + gi * p.cg + 4 * j, p.vec_bc, cv);
                held = gi;
            }
            float av[4];
            if constexpr (kKeep) {
#pragma unroll
                for (int n = 0; n < 4; ++n) av[n] = a2[i][n];
            } else {
                rates(i, av);
            }
            y[i] = 0.f;
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                h[i][n] = fmaf(exp2_fma(si, av[n]), h[i][n], pi * bv[n]);
                y[i] = fmaf(cv[n], h[i][n], y[i]);
            }
            if (first + i < p.channels)
                *reinterpret_cast<float4*>(state_out + at + (int64_t)(first + i) * N) =
                    make_float4(h[i][0], h[i][1], h[i][2], h[i][3]);
        }
        reduce_scatter<NL, NL, 1>(y, lane);
        if (live) {
            float out = fmaf(skip, uu, y[0]);
            if (p.z) out *= zz * sigmoid(zz);
            static_cast<T*>(p.y)[(int64_t)s * p.channels + c] = from_f<T>(out);
        }
    }
}

bool stride_ok(int64_t v, int m) { return v % m == 0; }

// Warps that a B200 holds of the forward kernel (four CTAs of four an SM).  Segments against whole
// chains of 784 tokens, bf16, by device time: 256 chains 99 against 211 us, 512 168 / 211, 704 223 /
// 256, 768 236 / 256, 832 262 / 257: whole chains from a third of the warps on.
int64_t fwd_warps() { return (int64_t)16 * sm_count(); }

int fwd_segment_size(const vh_ssm_scan_args* a) { return segment_size(a, fwd_warps() / 3, fwd_warps(), kGroup); }

template <typename T, int NL>
int launch_fwd(const ScanParams& p, const Segments& g, cudaStream_t st) {
    const int64_t tiles = (int64_t)p.groups * p.tiles_per_group;
    const int64_t items = (g.state ? g.slots : (int64_t)p.seqs.count) * tiles;
    const int64_t blocks = (items + kWarps - 1) / kWarps;
    if (blocks > 0x7fffffff) return fail(VH_E_RANGE, "vh_ssm_scan_fwd: too many channel tiles");
    const size_t smem = sizeof(FwdSmem<T, NL>) * kWarps;
    if (!ensure_smem_attr(reinterpret_cast<const void*>(&scan_fwd_kernel<T, NL, false>), smem) ||
        !ensure_smem_attr(reinterpret_cast<const void*>(&scan_fwd_kernel<T, NL, true>), smem))
        return fail(VH_E_DEVICE, "vh_ssm_scan_fwd: cannot reserve %zu bytes of shared memory", smem);
    if (!g.state) {
        scan_fwd_kernel<T, NL, false><<<(int)blocks, 32 * kWarps, smem, st>>>(p, g, items);
        return launch_status("selective scan");
    }
    scan_fwd_kernel<T, NL, true><<<(int)blocks, 32 * kWarps, smem, st>>>(p, g, items);
    if (int rc = launch_status("selective scan: own states")) return rc;
    if (int rc = enter_segments(p, 4 * NL, g, p.initial, false, st)) return rc;
    return launch_after("selective scan", scan_fwd_kernel<T, NL, false>, blocks, 32 * kWarps, smem, st, p, g, items);
}

}  // namespace

int check_scan_sizes(const char* what, const vh_ssm_scan_args* a, bool one_token) {
    if (!a) return fail(VH_E_ARG, "%s: null argument struct", what);
    if (!dtype_ok(a->dtype)) return fail(VH_E_DTYPE, "%s: dtype must be VH_F32, VH_BF16 or VH_F16", what);
    if (a->states != 4 && a->states != 8 && a->states != 16 && a->states != 32 && a->states != 64)
        return fail(VH_E_SHAPE, "%s: states must be 4, 8, 16, 32 or 64 (got %d)", what, a->states);
    if (a->batch <= 0 || a->channels <= 0 || a->groups <= 0)
        return fail(VH_E_SHAPE, "%s: batch, channels and groups must be positive", what);
    if (a->channels % a->groups)
        return fail(VH_E_SHAPE, "%s: channels (%d) must be a multiple of groups (%d)", what, a->channels, a->groups);
    if (one_token) return 0;
    if (a->length < 0) return fail(VH_E_SHAPE, "%s: negative length", what);
    if (a->length > 0x7fffffff) return fail(VH_E_RANGE, "%s: at most 2^31 - 1 tokens a sequence", what);
    return 0;
}

int check_scan_args(const char* what, const vh_ssm_scan_args* a, bool one_token) {
    if (!a) return fail(VH_E_ARG, "%s: null argument struct", what);
    if (!a->u || !a->delta || !a->b || !a->c || !a->a || !a->y) return fail(VH_E_ARG, "%s: null pointer argument", what);
    if (int rc = check_scan_sizes(what, a, one_token)) return rc;
    const size_t es = dtype_size(a->dtype);
    const void* typed[] = {a->u, a->delta, a->z, a->b, a->c, a->y};
    for (const void* t : typed)
        if (t && !aligned(t, es)) return fail(VH_E_ALIGN, "%s: misaligned pointers", what);
    if (one_token) {  // it reads its rates four at a time
        if (!aligned(a->a, 16)) return fail(VH_E_ALIGN, "%s: a must be 16-byte aligned", what);
        return 0;
    }
    for (const void* t : {(const void*)a->a, (const void*)a->d_skip, (const void*)a->delta_bias, (const void*)a->initial_state,
                          (const void*)a->final_state, (const void*)a->seq_offsets})
        if (t && !aligned(t, 4)) return fail(VH_E_ALIGN, "%s: misaligned pointers", what);
    if (a->checkpoints && !aligned(a->checkpoints, 16))
        return fail(VH_E_ALIGN, "%s: the checkpoints must be 16-byte aligned", what);
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

int64_t tile_count(const vh_ssm_scan_args* a) {
    const int cw = 128 / (a->states / 4), per = a->channels / a->groups;
    return (int64_t)a->groups * ((per + cw - 1) / cw);
}

// The checkpoints: a warp's states for every slot of 32 tokens and channel tile.
int64_t checkpoint_floats(const vh_ssm_scan_args* a) {
    return slot_total(a->seq_offsets != nullptr, a->length, a->batch, kCheckpoint) * tile_count(a) * 512;
}

int segment_size(const vh_ssm_scan_args* a, int64_t enough, int64_t warps, int step) {
    if (a->length == 0) return 0;
    const int64_t tiles = tile_count(a), tokens = a->seq_offsets ? a->length : (int64_t)a->batch * a->length;
    // The host does not know the lengths of packed sequences: any of them may hold most tokens, so
    // they are always cut, and twice as fine, because a sequence's last segment is a short one (17
    // sequences of 8192 tokens, 1024 channels: 132 us, against 134 as fine and 141 four times as).
    // With few segments to a chain one wave of warps is badly filled, and two are better (forward of
    // 512 chains of 784 tokens: 169 against 185 us; of 768: 235 / 291; but of 384: 140 / 132).
    if (a->seq_offsets) warps *= 2;
    else if (a->batch * tiles >= enough) return 0;
    else if (a->batch * tiles * 5 >= warps) warps *= 2;
    int64_t size = (tokens * tiles + warps - 1) / warps;
    size = std::max<int64_t>((size + step - 1) / step * step, kCheckpoint);
    if (!a->seq_offsets) {
        // segments of one length: a rounded-up number of them must not exceed the warps again
        while (a->batch * tiles * ((a->length + size - 1) / size) > warps) size += step;
        const int64_t segs = (a->length + size - 1) / size;
        size = std::max<int64_t>((((a->length + segs - 1) / segs) + step - 1) / step * step, kCheckpoint);
    }
    return size < a->length ? (int)size : 0;
}

int64_t segment_bytes(const vh_ssm_scan_args* a, int size) {
    if (size == 0) return 0;
    const int64_t units = slot_total(a->seq_offsets != nullptr, a->length, a->batch, size) * tile_count(a);
    return units * (512 + 128 / (a->states / 4)) * 4;
}

void place_segments(const vh_ssm_scan_args* a, int size, void* workspace, Segments* g) {
    *g = Segments{};
    if (size == 0) return;
    g->size = size;
    g->slots = slot_total(a->seq_offsets != nullptr, a->length, a->batch, size);
    g->state = static_cast<float*>(workspace);
    g->sigma = g->state + g->slots * tile_count(a) * 512;
}

int enter_segments(const ScanParams& p, int states, const Segments& g, const float* first, bool right, cudaStream_t st) {
    // Long chains, of which there are few, are cut into runs; a packed sequence may hold most of the
    // slots.  The forward's time with 1 / 4 / 16 runs: 7 segments of 128 chains 29 / 33 / 39 us, 18
    // of 128 122 / 117 / 122, 74 of 32 62 / 59 / 54, 98 of 24 183 / 172 / 164.
    const int64_t chains = (int64_t)p.seqs.count * p.groups * p.tiles_per_group;
    const int64_t segs = p.seqs.offsets ? std::min<int64_t>(g.slots, 4 * (g.slots / p.seqs.count + 1)) : g.slots / p.seqs.count;
    return with_states(states, [&](auto nl) {
        constexpr int NL = decltype(nl)::value;
        const char* what = "selective scan: entering states";
        if (segs <= 8) return launch_after(what, enter_segments_kernel<NL, 1, 1>, chains, 128, 0, st, p, g, first, (int)right);
        if (segs <= 32 || chains > 2 * sm_count())
            return launch_after(what, enter_segments_kernel<NL, 4, 1>, chains, 512, 0, st, p, g, first, (int)right);
        return launch_after(what, enter_segments_kernel<NL, 16, 4>, chains * 4, 512, 0, st, p, g, first, (int)right);
    });
}

}  // namespace ssm
}  // namespace vh

using namespace vh;
using namespace vh::ssm;

extern "C" int64_t vh_ssm_scan_checkpoint_bytes(const vh_ssm_scan_args* a) {
    clear_error();
    if (check_scan_sizes("vh_ssm_scan_checkpoint_bytes", a, false)) return 0;
    return checkpoint_floats(a) * 4;
}

extern "C" int64_t vh_ssm_scan_fwd_workspace_bytes(const vh_ssm_scan_args* a) {
    clear_error();
    if (check_scan_args("vh_ssm_scan_fwd_workspace_bytes", a, false)) return 0;
    return segment_bytes(a, fwd_segment_size(a));
}

extern "C" int vh_ssm_scan_fwd(const vh_ssm_scan_args* a, void* workspace, int64_t workspace_bytes, vh_stream_t stream) {
    clear_error();
    if (int rc = check_scan_args("vh_ssm_scan_fwd", a, false)) return rc;
    const int size = fwd_segment_size(a);
    const int64_t need = segment_bytes(a, size);
    if (need > 0 && (!workspace || workspace_bytes < need)) return fail(VH_E_ARG, "vh_ssm_scan_fwd: workspace too small");
    if (need > 0 && !aligned(workspace, 16))
        return fail(VH_E_ALIGN, "vh_ssm_scan_fwd: the workspace must be 16-byte aligned");
    ScanParams p;
    Segments g;
    fill_scan_params(a, &p);
    place_segments(a, size, workspace, &g);
    return with_dtype(a->dtype, [&](auto t) {
        using T = decltype(t);
        return with_states(a->states, [&](auto nl) {
            return launch_fwd<T, decltype(nl)::value>(p, g, static_cast<cudaStream_t>(stream));
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
    // streams share a block once there are four blocks an SM
    const int gx = (a->channels + 255) / 256;
    const int gy = std::min<int>(a->batch, std::max(1, 4 * sm_count() / gx));
    return with_dtype(a->dtype, [&](auto t) {
        using T = decltype(t);
        return with_states(a->states, [&](auto nl) {
            scan_step_kernel<T, decltype(nl)::value><<<dim3(gx, gy), 256, 0, static_cast<cudaStream_t>(stream)>>>(
                p, state, state_out, slots_index, slots);
            return launch_status("selective scan step");
        });
    });
}
