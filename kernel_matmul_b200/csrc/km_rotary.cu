// Rotary positions: every pair (a, b) of a head's values turned by position * frequency.
//
// Bound by memory: each value is read and written once.  The angle belongs to (token, pair), not to the head, so a CTA
// takes a few tokens, evaluates the cosines and sines of all their pairs into shared memory once, and turns all heads of q
// and of k with them.  Angles: position * frequency and its reduction to a part of a turn in 64 bits (a position of 10^6
// leaves 2^-33 of a turn; in 32 bits it would be off by 0.06 rad), then sincospi in 32 bits on [-1, 1] half turns.
#include "km_decay.cuh"

namespace km {

struct RotaryOperand {
    const char *in;
    char *out;
    int64_t in_batch, in_head, in_token, in_col, out_batch, out_head, out_token, out_col;
};

struct RotaryArgs {
    RotaryOperand x[2];
    int heads[2];
    int64_t tokens;
    int dim, pairs, tile;  // tile: tokens of a CTA
    const void *positions;
    int64_t position_batch, position_token;
    int position_type, frequency_type;
    const void *frequencies;
    int inverse;
    float scale;
};

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Pack {
    T v[VEC];
};

// VEC = 1: any strides.  VEC > 1: VEC neighbouring values at once, which the host has found aligned.
template <typename T, int VEC, bool INTERLEAVED>
__global__ void __launch_bounds__(256) rotary_kernel(RotaryArgs a) {
    extern __shared__ float2 turns[];  // [token of the tile][pair]
    const int64_t tiles = (a.tokens + a.tile - 1) / a.tile;
    const int64_t batch = blockIdx.x / tiles, first = (blockIdx.x - batch * tiles) * a.tile;
    const int tokens = (int)min((int64_t)a.tile, a.tokens - first);
    for (int i = threadIdx.x; i < tokens * a.pairs; i += 256) {
        const int t = i / a.pairs, p = i - t * a.pairs;
        const int64_t at = batch * a.position_batch + (first + t) * a.position_token;
        const double pos = a.position_type == KM_TYPE_I64   ? (double)static_cast<const int64_t *>(a.positions)[at]
                           : a.position_type == KM_TYPE_I32 ? (double)static_cast<const int32_t *>(a.positions)[at]
                                                            : (double)static_cast<const float *>(a.positions)[at];
        const double f = a.frequency_type == KM_TYPE_F64 ? static_cast<const double *>(a.frequencies)[p]
                                                         : (double)static_cast<const float *>(a.frequencies)[p];
        const double half_turns = pos * f * 0.31830988618379067154;  // / pi
        float sn, cs;
        sincospif((float)(half_turns - 2.0 * rint(0.5 * half_turns)), &sn, &cs);
        turns[i] = make_float2(cs * a.scale, (a.inverse ? -sn : sn) * a.scale);
    }
    __syncthreads();
    // work units of a head: (half layout) VEC pairs each, then VEC copied values each; (interleaved) VEC / 2 pairs each
    constexpr int STEP = INTERLEAVED && VEC == 1 ? 2 : VEC;  // values of one side that a turning unit covers
    const int turning = INTERLEAVED ? 2 * a.pairs / STEP : a.pairs / STEP;
    const int rest = (a.dim - 2 * a.pairs) / VEC, units = turning + rest;
    const int heads = a.heads[0] + a.heads[1], total = tokens * heads * units;
    for (int i = threadIdx.x; i < total; i += 256) {
        const int th = i / units, u = i - th * units, t = th / heads;
        int h = th - t * heads;
        const int which = h >= a.heads[0];
        h -= which ? a.heads[0] : 0;
        const RotaryOperand &x = a.x[which];
        const T *in = reinterpret_cast<const T *>(x.in) + batch * x.in_batch + h * x.in_head + (first + t) * x.in_token;
        T *out = reinterpret_cast<T *>(x.out) + batch * x.out_batch + h * x.out_head + (first + t) * x.out_token;
        const float2 *angle = turns + t * a.pairs;
        if (u >= turning) {
            const int c = 2 * a.pairs + (u - turning) * VEC;
            if constexpr (VEC > 1)
                *reinterpret_cast<Pack<T, VEC> *>(out + c) = *reinterpret_cast<const Pack<T, VEC> *>(in + c);
            else
                out[c * x.out_col] = in[c * x.in_col];
        } else if constexpr (VEC == 1) {
            const int c0 = INTERLEAVED ? 2 * u : u, c1 = INTERLEAVED ? 2 * u + 1 : u + a.pairs;
            const float2 w = angle[u];
            const float p = as_float(in[c0 * x.in_col]), q = as_float(in[c1 * x.in_col]);
            out[c0 * x.out_col] = from_float<T>(p * w.x - q * w.y);
            out[c1 * x.out_col] = from_float<T>(p * w.y + q * w.x);
        } else if constexpr (INTERLEAVED) {
            const Pack<T, VEC> v = *reinterpret_cast<const Pack<T, VEC> *>(in + u * VEC);
            Pack<T, VEC> r;
#pragma unroll
            for (int j = 0; j < VEC; j += 2) {
                const float2 w = angle[(u * VEC + j) / 2];
                const float p = as_float(v.v[j]), q = as_float(v.v[j + 1]);
                r.v[j] = from_float<T>(p * w.x - q * w.y);
                r.v[j + 1] = from_float<T>(p * w.y + q * w.x);
            }
            *reinterpret_cast<Pack<T, VEC> *>(out + u * VEC) = r;
        } else {
            const Pack<T, VEC> v0 = *reinterpret_cast<const Pack<T, VEC> *>(in + u * VEC);
            const Pack<T, VEC> v1 = *reinterpret_cast<const Pack<T, VEC> *>(in + a.pairs + u * VEC);
            Pack<T, VEC> r0, r1;
#pragma unroll
            for (int j = 0; j < VEC; j++) {
                const float2 w = angle[u * VEC + j];
                const float p = as_float(v0.v[j]), q = as_float(v1.v[j]);
                r0.v[j] = from_float<T>(p * w.x - q * w.y);
                r1.v[j] = from_float<T>(p * w.y + q * w.x);
            }
            *reinterpret_cast<Pack<T, VEC> *>(out + u * VEC) = r0;
            *reinterpret_cast<Pack<T, VEC> *>(out + a.pairs + u * VEC) = r1;
        }
    }
}

template <typename T>
static int launch_rotary(RotaryArgs &a, int64_t batch, bool wide, bool interleaved, cudaStream_t s) {
    constexpr int VEC = 16 / sizeof(T);
    // Four tokens to a CTA where that still gives four CTAs per SM, else fewer: with 16 the last, partly filled wave of CTAs
    // costs too much (335 MB: 72 us; 8: 64, 4: 62.5, 2: 66).
    const int64_t rows = batch * a.tokens;
    a.tile = (int)std::max<int64_t>(1, std::min<int64_t>({4, rows / (4 * 148), 4096 / std::max(a.pairs, 1)}));  // (32 KB of angles at most)
    const int64_t ctas = batch * ceil_div(a.tokens, a.tile);
    KM_REQUIRE(ctas < (1LL << 31), KM_ERR_UNSUPPORTED, "km_rotary: more than 2^31 work items");
    auto kernel = wide ? (interleaved ? rotary_kernel<T, VEC, true> : rotary_kernel<T, VEC, false>)
                       : (interleaved ? rotary_kernel<T, 1, true> : rotary_kernel<T, 1, false>);
    kernel<<<(unsigned)ctas, 256, (size_t)a.tile * a.pairs * sizeof(float2), s>>>(a);
    KM_CHECK_LAUNCH("km_rotary launch");
    return KM_OK;
}

}  // namespace km

extern "C" int km_rotary(int32_t dtype, int64_t batch, int64_t tokens, const int64_t heads[2], int64_t dim, int64_t pairs,
                         const km_view in[2], const km_view out[2], int32_t position_type, const km_view *positions,
                         int32_t frequency_type, const void *frequencies, int32_t interleaved, int32_t inverse, float scale, void *stream) {
    using namespace km;
    KM_REQUIRE(heads && in && out && positions, KM_ERR_INVALID_ARGUMENT, "km_rotary: null argument");
    KM_REQUIRE(dtype >= KM_TYPE_F32 && dtype <= KM_TYPE_F16, KM_ERR_INVALID_ARGUMENT, "km_rotary: bad element type");
    KM_REQUIRE((position_type == KM_TYPE_I32 || position_type == KM_TYPE_I64 || position_type == KM_TYPE_F32) &&
                   (frequency_type == KM_TYPE_F32 || frequency_type == KM_TYPE_F64),
               KM_ERR_INVALID_ARGUMENT, "km_rotary: bad type of positions or frequencies");
    KM_REQUIRE(batch >= 0 && tokens >= 0 && heads[0] >= 0 && heads[1] >= 0 && pairs >= 0 && 2 * pairs <= dim, KM_ERR_INVALID_ARGUMENT,
               "km_rotary: bad sizes");
    KM_REQUIRE(dim <= 4096 && heads[0] + heads[1] <= 8192 && batch < (1LL << 31) && tokens < (1LL << 31) &&
                   (batch == 0 || tokens < (1LL << 40) / batch),
               KM_ERR_UNSUPPORTED, "km_rotary: at most 4096 values to a head, 8192 heads, 2^31 tokens");
    if (batch == 0 || tokens == 0 || dim == 0 || heads[0] + heads[1] == 0) return KM_OK;
    KM_REQUIRE(positions->data && (pairs == 0 || frequencies), KM_ERR_INVALID_ARGUMENT, "km_rotary: null pointer");
    RotaryArgs a = {};
    const int64_t vec = dtype == KM_TYPE_F32 ? 4 : 8;
    bool wide = dim % vec == 0 && (interleaved ? 2 * pairs : pairs) % vec == 0;
    for (int i = 0; i < 2; i++) {
        a.heads[i] = (int)heads[i];
        if (heads[i] == 0) continue;
        KM_REQUIRE(in[i].data && out[i].data, KM_ERR_INVALID_ARGUMENT, "km_rotary: null pointer");
        a.x[i] = RotaryOperand{static_cast<const char *>(in[i].data), static_cast<char *>(out[i].data),
                               in[i].batch_stride[0], in[i].batch_stride[1], in[i].stride[0], in[i].stride[1],
                               out[i].batch_stride[0], out[i].batch_stride[1], out[i].stride[0], out[i].stride[1]};
        const RotaryOperand &x = a.x[i];
        for (int64_t stride : {x.in_batch, x.in_head, x.in_token, x.out_batch, x.out_head, x.out_token}) wide = wide && stride % vec == 0;
        wide = wide && x.in_col == 1 && x.out_col == 1 && reinterpret_cast<uintptr_t>(x.in) % 16 == 0 &&
               reinterpret_cast<uintptr_t>(x.out) % 16 == 0;
    }
    a.tokens = tokens, a.dim = (int)dim, a.pairs = (int)pairs;
    a.positions = positions->data, a.position_batch = positions->batch_stride[0], a.position_token = positions->stride[0];
    a.position_type = position_type, a.frequency_type = frequency_type, a.frequencies = frequencies;
    a.inverse = inverse != 0, a.scale = scale;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (dtype == KM_TYPE_F32) return launch_rotary<float>(a, batch, wide, interleaved != 0, s);
    if (dtype == KM_TYPE_BF16) return launch_rotary<__nv_bfloat16>(a, batch, wide, interleaved != 0, s);
    return launch_rotary<__half>(a, batch, wide, interleaved != 0, s);
}
