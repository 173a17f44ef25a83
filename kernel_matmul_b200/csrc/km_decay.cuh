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

// Segments of the sequences before `seq` (all lanes of a warp call it, all get the result).
__device__ __forceinline__ int segments_before(const DecayArgs &a, int64_t seq) {
    if (a.starts == nullptr) return (int)seq * segments_of(a, a.tokens);
    int sum = 0;
    for (int64_t i = threadIdx.x & 31; i < seq; i += 32) {
        int64_t begin, length;
        sequence_rows(a, i, begin, length);
        sum += segments_of(a, length);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    return sum;
}

// Segment number `slot` (one warp calls it, all lanes get the result).
__device__ __forceinline__ Segment find_segment(const DecayArgs &a, int64_t slot) {
    Segment r = {};
    r.spare = -1;
    int index = 0;
    if (a.starts == nullptr) {
        const int per = segments_of(a, a.tokens);
        r.seq = (int)((unsigned)slot / (unsigned)per);
        index = (int)slot - r.seq * per;
        r.used = true;
    } else {
        const int lane = threadIdx.x & 31;
        int before = 0;
        for (int64_t base = 0; base < a.sequences && !r.used; base += 32) {
            const int64_t i = base + lane;
            int64_t begin, length = 0;
            int n = 0;
            if (i < a.sequences) {
                sequence_rows(a, i, begin, length);
                n = segments_of(a, length);
            }
            int upto = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += v;
            }
            upto += before;
            const unsigned hit = __ballot_sync(0xffffffffu, slot < upto);
            if (hit != 0) {
                const int who = __ffs(hit) - 1;
                r.seq = (int)base + who;
                index = (int)slot - __shfl_sync(0xffffffffu, upto - n, who);
                r.used = true;
            }
            before = __shfl_sync(0xffffffffu, upto, 31);
        }
        if (!r.used) {
            r.spare = (int)(slot - before);
            r.spares = (int)(a.slots - before);
            return r;
        }
    }
    int64_t begin, length;
    sequence_rows(a, r.seq, begin, length);
    r.begin = (int)begin, r.length = (int)length;
    r.first = index * (int)a.segment;
    r.last = index == segments_of(a, length) - 1;
    // (a sequence of n segments has n - 1 states; bounded, should `starts` decrease and sequences overlap)
    r.adds = (int)min(slot - r.seq, a.state_slots - 1);
    r.start = (int)min(slot - r.seq - 1, a.state_slots - 1);
    r.count = min(r.length - r.first, (int)a.segment);
    // the very last slot is in use: its CTA sees to the rows of no sequence
    if (a.starts != nullptr && slot == a.slots - 1) r.spare = 0, r.spares = 1;
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
