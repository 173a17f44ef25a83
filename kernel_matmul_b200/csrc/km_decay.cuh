// Linear attention with a decay for each head: arguments, work items and the arithmetic that the kernels of
// km_decay.cu (FMA pipe, scans, single tokens) and km_decay_tc.cu (tensor cores) share.
//
// A sequence is cut into chunks of C tokens.  With Z the state that meets the chunk's first token, already
// decayed to it, and t, s local to the chunk,
//   out_t = scale [ sum_{s <= t} e^{g (t - s)} (q_t . k_s) v_s + e^{g t} Z^T q_t ]
//   Z    <- e^{g e} Z + sum_s e^{g (e - s)} k_s v_s^T,    e = tokens of the chunk,
// so every exponent is that of a distance: nothing overflows however fast the decay, and the products over a
// chunk are matrix products.  The state after the last token takes e = tokens - 1 (forward), the gradient of the
// state before the first one e = tokens (reverse form, which runs over the tokens backwards).
//
// Where sequences and heads alone do not fill the device a sequence is cut into segments of several chunks:
// the segments' own states first (from zero), a scan over each sequence's segments, then all segments at once from
// their states.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "km_tcgen05.cuh"

namespace km {

struct Operand {  // strides in elements: sequence, group of heads, head in the group, token (or dk), value (or dv)
    char *data;
    int64_t seq, group, head, row, col;
    template <typename T>
    __device__ __forceinline__ T *at(int64_t s, int64_t hg, int64_t hi) const {
        return reinterpret_cast<T *>(data) + (s * seq + hg * group + hi * head);
    }
};

struct DecayArgs {
    Operand q, k, v, out, state_in, state_out;  // data == nullptr: absent
    const float *log_decay;
    const int32_t *starts;  // null: every sequence has `tokens` rows of its own
    int64_t sequences, tokens;
    unsigned group, heads;
    int dk, dv;
    unsigned segment;       // tokens of a segment (a multiple of the chunk; the sums of tokens and a segment fit 32 bits)
    int64_t slots;          // segments of all sequences, at most (less than 2^31, as all counts of this file)
    // What a segment adds to its sequence's state, then (decay_scan_kernel) the state the next one starts with: state_slots x heads
    // of (dk, dv) (gradient of the decays: two, Z and M); values (r, c) at r state_row + c state_col.
    float *states;
    int64_t state_slots;
    int state_row, state_col;
    float scale_in, scale_out;  // on k v^T, and on the result
    int reverse;
    int parts;                  // 16-bit parts of the decayed keys on the tensor cores
    int *gave_up;
    unsigned wait_polls;
};

inline Operand make_operand(const km_view *v) {
    if (v == nullptr || v->data == nullptr) return Operand{nullptr, 0, 0, 0, 0, 0};
    return Operand{static_cast<char *>(v->data), v->batch_stride[0], v->batch_stride[1], v->batch_stride[2], v->stride[0], v->stride[1]};
}

__device__ __forceinline__ float as_float(float x) { return x; }
__device__ __forceinline__ float as_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float as_float(__half x) { return __half2float(x); }
template <typename T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ float from_float<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }

// Decay per token as a power of two.  A decay of zero (g = -inf) must not meet a distance of 0 as inf * 0: from
// 2^-10000 on it is zero over any distance but that one.
__device__ __forceinline__ float log2_decay(float g) {
    g *= KM_LOG2E_F;
    return g < -10000.0f ? -10000.0f : g;
}

struct Segment {
    int seq, begin, length;  // its sequence: number, first row, rows (of all three there are less than 2^31)
    int first, count;        // its tokens inside the sequence (in the order in which they are gone through)
    int adds, start;         // places in `states` of what it adds (not of a last segment) and of its start (not of a first one)
    int spare, spares;       // rows of no sequence are shared by `spares` CTAs per head, of which this is number `spare`; -1: none
    bool used, last;
};

// Rows of sequence i: clamped, so that no `starts` leads out of the tensors.
__device__ __forceinline__ void sequence_rows(const DecayArgs &a, int64_t i, int64_t &begin, int64_t &length) {
    if (a.starts == nullptr) {
        begin = 0;
        length = a.tokens;
        return;
    }
    const int64_t lo = min(max((int64_t)a.starts[i], (int64_t)0), a.tokens);
    const int64_t hi = min(max((int64_t)a.starts[i + 1], lo), a.tokens);
    begin = lo;
    length = hi - lo;
}

__device__ __forceinline__ int segments_of(const DecayArgs &a, int64_t length) {
    return length <= a.segment ? 1 : (int)(((unsigned)length + (a.segment - 1u)) / a.segment);
}

// Packed sequences: sequence i, which starts at row b, has its segments in the slots from i + floor(b / segment) on and its states in the
// places from floor(b / segment) on.  A sequence of n rows has at most floor((b + n) / segment) - floor(b / segment) + 1 segments and
// one state less, so the next one's come behind, and neither needs a sum over the sequences before.  (No `starts` leads out of the slots and
// places there are; those that decrease may give two sequences the same ones.)
__device__ __forceinline__ int64_t first_place(const DecayArgs &a, int64_t i) {
    if (a.starts == nullptr) return i * (segments_of(a, a.tokens) - 1);
    return (unsigned)min(max((int64_t)a.starts[i], (int64_t)0), a.tokens) / a.segment;
}

// Segment number `slot` (one warp calls it, all lanes get the result).
__device__ __forceinline__ Segment find_segment(const DecayArgs &a, int64_t slot) {
    Segment r = {};
    r.spare = -1;
    int64_t index = 0, place = 0;
    if (a.starts == nullptr) {
        const int per = segments_of(a, a.tokens);
        r.seq = (int)((unsigned)slot / (unsigned)per);
        index = (int)slot - r.seq * per;
        place = (int64_t)r.seq * (per - 1);
    } else {
        // rows of no sequence: for the slots before the first sequence's and behind the last one's, or, if there are none, the last slot
        const int64_t begin = first_place(a, 0), end = a.sequences + first_place(a, a.sequences);
        int64_t spares = begin + (a.slots - end);
        if (slot < begin)
            r.spare = (int)slot;
        else if (slot >= end)
            r.spare = (int)(begin + (slot - end));
        else if (spares == 0 && slot == a.slots - 1)
            r.spare = 0, spares = 1;
        r.spares = (int)spares;
        // the last sequence whose first slot is not behind this one: 32 candidates at a time
        int64_t first = 0, count = a.sequences;
        bool found = false;
        for (int64_t step = count; step > 0 && !(found && step == 1);) {
            step = (count + 31) / 32;
            const int64_t i = first + (threadIdx.x & 31) * step;
            const unsigned hit = __ballot_sync(0xffffffffu, i < first + count && i + first_place(a, i) <= slot);
            if (hit == 0) break;
            const int64_t skip = (31 - __clz(hit)) * step;
            first += skip, count = min(step, count - skip);
            found = true;
        }
        if (!found) return r;
        r.seq = (int)first;
        place = first_place(a, first);
        index = slot - (first + place);
    }
    int64_t begin, length;
    sequence_rows(a, r.seq, begin, length);
    const int segments = segments_of(a, length);
    if (index >= segments) return r;  // (of packed sequences some slots are left over)
    r.used = true;
    r.begin = (int)begin, r.length = (int)length;
    r.first = (int)index * (int)a.segment;
    r.last = index == segments - 1;
    r.adds = (int)min(place + index, a.state_slots - 1);
    r.start = (int)min(place + index - 1, a.state_slots - 1);
    r.count = min(r.length - r.first, (int)a.segment);
    return r;
}

// Row of the tensors that holds token i (in the order in which the sequence is gone through).
__device__ __forceinline__ int64_t token_row(const DecayArgs &a, const Segment &s, int i) {
    return s.begin + (a.reverse ? s.length - 1 - i : i);
}

// Zeros into this CTA's share of the rows of no sequence.
template <typename O>
__device__ __forceinline__ void clear_spare_rows(const DecayArgs &a, const Segment &s, int64_t hg, int64_t hi) {
    const int64_t head_end = min(max((int64_t)a.starts[0], (int64_t)0), a.tokens);
    const int64_t tail = min(max((int64_t)a.starts[a.sequences], head_end), a.tokens);
    const int64_t rows = head_end + (a.tokens - tail);
    O *out = a.out.at<O>(0, hg, hi);
    for (int64_t i = s.spare; i < rows; i += s.spares) {
        const int64_t row = i < head_end ? i : tail + (i - head_end);
        for (int c = threadIdx.x; c < a.dv; c += blockDim.x) out[row * a.out.row + c * a.out.col] = from_float<O>(0.0f);
    }
}

int launch_decay_grad_tc(const km_decay_problem &p, const DecayArgs &a, const Operand &dout, const Operand &dstate, double *partials,
                         bool state_only, cudaStream_t stream);
int launch_decay_tc(const km_decay_problem &p, const DecayArgs &a, bool state_only, cudaStream_t stream);

}  // namespace km
