// Shared pieces of linear attention with a decay for each head (linear_attention.cu).
//
// Per sequence and head, with lambda = exp(log_decay) and a state S of [key dim, value dim]:
//     S_t = lambda S_{t-1} + kv_scale k_t v_t^T,    o_t = out_scale q_t^T S_t.
// Over a chunk of n tokens that starts from S_0:
//     o_i = out_scale (lambda^{i+1} q_i S_0 + kv_scale sum_{j<=i} lambda^{i-j} (q_i k_j) v_j)
//     S_n = lambda^n S_0 + kv_scale sum_j lambda^{n-1-j} k_j v_j^T
// which is four matrix products.  The gradients have the same form, so one kernel serves them too:
//     dq: queries dO, keys V, values K, state S^T, first token to last;
//     dk: queries V, keys dO, values Q, and dv: queries K, keys Q, values dO, from the last token to
//     the first, where the gradient of the final state enters without a decay (`entry`) and leaves
//     before the first token one decay further (`exit_decay`).
#pragma once

#include "ssm_common.cuh"

namespace vh {
namespace lin {

using ssm::Rows;
using ssm::Seq;
using ssm::Seqs;

constexpr int kChunk = 64;    // tokens a chunk
constexpr int kTile = 64;     // value columns a CTA
constexpr int kMaxDim = 128;  // keys and values a head

// One tensor [tokens, heads, dim] with unit stride last.
struct Heads {
    const void* p;
    Rows rows;
    int64_t head;
    int32_t vec;  // elements that one aligned access may take (8, 4 or 1)
};

struct Params {
    Seqs seqs;
    Heads q, k, v;
    const float* log_decay;           // [heads]
    const float* initial;             // or null: element (sequence, head, key a, value b) at
    int64_t init_a, init_b;           //   (s heads + h) dk dv + a init_a + b init_b
    void* o;                          // contiguous [tokens, heads, dv]
    float* final_state;               // contiguous [sequences, heads, dk, dv] or null
    float out_scale, kv_scale;
    int32_t heads, dk, dv;
    int32_t entry, exit_decay;        // see above
    int32_t vec_o;
    // chains in segments: the state before segment j of a sequence in `states` (0: whole chains)
    int32_t segment;
    float* states;                    // [slots, heads, dk, dv]
    int32_t join;                     // `states` holds what each segment adds: a start is the sum of those before it
};

// exp(log_decay) to the n-th.  A decay of 0 (log_decay -inf) leaves the power 0 at 1.
__device__ __forceinline__ float decay_power(float log_decay, int64_t n) {
    const float g = log_decay < -1e4f ? -1e4f : log_decay;
    return expf(g * (float)n);
}

// One unit of work: which tokens of which sequence.
struct Unit {
    int s;
    Seq e;
    int64_t slot, t0, t1;
    bool live;
};
// Of block column blockIdx.x; every thread takes part.  `found`: a word of shared memory.  Whose segment it is in packed sequences, the last
// sequence whose slots start at or before this one, is looked up by all threads at once: a binary search is
// five to ten loads one after another, and as long as a chunk.
__device__ __forceinline__ Unit block_unit(const Params& p, int* found) {
    Unit u;
    u.slot = blockIdx.x;
    if (p.segment == 0) {
        u.s = (int)u.slot;
    } else if (!p.seqs.offsets) {
        u.s = (int)(u.slot / ssm::slots_per_seq(p.seqs.length, p.segment));
    } else {
        if (threadIdx.x == 0) *found = 0;
        __syncthreads();
        int mine = 0;
        for (int s = threadIdx.x; s < p.seqs.count; s += blockDim.x) {
            int64_t row = p.seqs.offsets[s];
            row = row < 0 ? 0 : (row > p.seqs.length ? p.seqs.length : row);
            if (row / p.segment + s <= u.slot) mine = s;
        }
        if (mine > 0) atomicMax(found, mine);
        __syncthreads();
        u.s = *found;
    }
    u.e = ssm::seq_at(p.seqs, u.s);
    if (p.segment == 0) {
        u.t0 = 0;
        u.t1 = u.e.len;
        u.live = true;
        return u;
    }
    const int64_t j = u.slot - ssm::slot_base(p.seqs, u.s, u.e.row, p.segment);
    u.t0 = j * p.segment;
    u.t1 = min(u.e.len, u.t0 + p.segment);
    u.live = j >= 0 && (u.t0 < u.e.len || j == 0);
    return u;
}

// From what each segment adds to the state before each of them (linear_attention.cu).
int enter_segments(const Params& p, cudaStream_t st);

// The tcgen05 form (linear_attention_tc.cu).  tc_run does nothing and returns false where it does not
// apply; `states` holds the states of its segments.
int tc_segment_size(int64_t length, int batch, bool packed, int heads, int dk, int dv);
bool tc_run(Params p, void* states, cudaStream_t st, int* rc);
unsigned tc_status(bool reset);

}  // namespace lin
}  // namespace vh
