// Linear attention with a decay for each head (km_decay.cuh has the method): the kernels on the FMA pipe, the scan
// over a sequence's segments, the gradient of the decays, sums over groups of heads and the recurrence for single tokens;
// the entry points for all of them.
#include "km_decay.cuh"

namespace km {

// ------------------------------------------------------------------------------------------------
// Whole sequences on the FMA pipe: fp32 operands (products of fp32 values have no exact form on the tensor cores), and the
// other types on path 1.  Chunks of 32 tokens, so that the products inside a chunk (32 x 32 x (dk + dv)) cost a quarter of those
// with the state (2 x 32 x dk x dv).  One CTA of 256 threads per (segment, head, 64 columns of v): the state's columns are
// independent, and two CTAs of half the columns fit an SM where one with all of them did.  The state is held in registers, ROWS x 4
// values per thread, for its update, and in shared memory for the product with q.  ROWS = 4: for dk up to 64, half of the work.
// The next chunk's values are on their way while a chunk is worked on.  Forwards and backwards (with decay_gradient_kernel), in us: 2 x 1001
// tokens, 6 heads of 40 and 72: 246 (all columns in one CTA, one load after the other: 361); 16 x 2048, 16 heads of 64: 3960 (9230);
// 4 x 4096, 16 heads of 128: 7720 (8930).  Bound by shared memory's bandwidth, of which a product takes 4 to 5 cycles for 4 of FMAs.
constexpr int FC = 32;          // tokens of a chunk
constexpr int FV = 64;          // columns of v of a CTA

// Rows [first, first + tokens) of an operand on the way to shared memory, zeros behind them and behind `dim`.
template <typename T, int WIDTH>
struct ChunkRows {
    static constexpr int STEP = 256 / WIDTH, N = FC / STEP;
    T x[N];
    __device__ __forceinline__ void fetch(const DecayArgs &a, const Segment &s, const Operand &o, int64_t hg, int64_t hi, int first, int tokens,
                                          int dim) {
        const T *src = o.at<T>(a.starts == nullptr ? s.seq : 0, hg, hi);
        const int c = threadIdx.x % WIDTH, t0 = threadIdx.x / WIDTH;
        const T *p = src + token_row(a, s, first + t0) * o.row + c * o.col;
        const int64_t step = (a.reverse ? -STEP : STEP) * o.row;
#pragma unroll
        for (int i = 0; i < N; i++) x[i] = t0 + i * STEP < tokens && c < dim ? p[i * step] : from_float<T>(0.0f);
    }
    template <int LD>
    __device__ __forceinline__ void put(float *dst) const {
        const int c = threadIdx.x % WIDTH, t0 = threadIdx.x / WIDTH;
#pragma unroll
        for (int i = 0; i < N; i++) dst[(t0 + i * STEP) * LD + c] = as_float(x[i]);
    }
};

template <int ROWS>
struct FmaSmem {
    static constexpr int LD = 16 * ROWS + 4;
    static constexpr int Q = 0, K = FC * LD, V = 2 * FC * LD, P = V + FC * (FV + 4), W = P + FC * 36, Z = W + FC, BYTES = (Z + 16 * ROWS * FV) * 4;
};

template <typename T, typename O, int ROWS, bool STATE_ONLY>
__global__ void __launch_bounds__(256, 2) decay_fma_kernel(DecayArgs a, int vblocks) {
    using L = FmaSmem<ROWS>;
    constexpr int LD = L::LD, LV = FV + 4;
    extern __shared__ __align__(16) float smem[];
    float *sq = smem + L::Q, *sk = smem + L::K, *sv = smem + L::V, *sp = smem + L::P, *sw = smem + L::W, *sz = smem + L::Z;
    const int vb = blockIdx.x % (unsigned)vblocks, v0 = vb * FV, cols = min(FV, a.dv - v0);
    const unsigned rest = blockIdx.x / (unsigned)vblocks;
    const int64_t h = rest % (unsigned)a.heads, slot = rest / (unsigned)a.heads;
    const int64_t hg = h / a.group, hi = h - hg * a.group;
    const Segment s = find_segment(a, slot);
    if (!STATE_ONLY && s.spare >= 0 && vb == 0) clear_spare_rows<O>(a, s, hg, hi);
    if (!s.used || (STATE_ONLY && s.last)) return;
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    const float g2 = log2_decay(a.log_decay[h]);
    const int dk4 = (a.dk + 3) & ~3;
    Operand v = a.v;
    v.data += v0 * v.col * (int64_t)sizeof(T);

    // state: rows ROWS ty + i, columns 4 tx .. + 3 of this CTA's
    float z[ROWS][4];
    const bool first_segment = s.first == 0;
    const float enter = first_segment && !a.reverse && s.length > 0 ? exp2f(g2) : 1.0f;
#pragma unroll
    for (int i = 0; i < ROWS; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int r = ROWS * ty + i, c = 4 * tx + j;
            float x = 0.0f;
            if (!STATE_ONLY && r < a.dk && c < cols) {
                if (!first_segment)
                    x = a.states[((int64_t)s.start * a.heads + h) * a.dk * a.dv + r * a.state_row + (v0 + c) * a.state_col];
                else if (a.state_in.data != nullptr)
                    x = a.state_in.at<float>(s.seq, hg, hi)[r * a.state_in.row + (v0 + c) * a.state_in.col] * enter;
            }
            z[i][j] = x;
        }
    ChunkRows<T, 16 * ROWS> nq, nk;
    ChunkRows<T, FV> nv;
    const auto fetch = [&](int first) {
        const int tokens = min(FC, s.first + s.count - first);
        if (!STATE_ONLY) nq.fetch(a, s, a.q, hg, hi, first, tokens, a.dk);
        nk.fetch(a, s, a.k, hg, hi, first, tokens, a.dk);
        nv.fetch(a, s, v, hg, hi, first, tokens, cols);
    };
    if (s.count > 0) fetch(s.first);

    for (int first = s.first; first < s.first + s.count; first += FC) {
        const int tokens = min(FC, s.first + s.count - first);
        const bool final = first + tokens == s.length;
        const int e = final && !a.reverse ? tokens - 1 : tokens;
        __syncthreads();
        if (!STATE_ONLY) nq.template put<LD>(sq);
        nk.template put<LD>(sk);
        nv.template put<LV>(sv);
        if (tid < FC) sw[tid] = exp2f(g2 * (float)max(e - tid, 0)) * a.scale_in;
        if (!STATE_ONLY) {
#pragma unroll
            for (int i = 0; i < ROWS; i++)
                *reinterpret_cast<float4 *>(sz + (ROWS * ty + i) * FV + 4 * tx) =
                    ROWS * ty + i < a.dk ? make_float4(z[i][0], z[i][1], z[i][2], z[i][3]) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);  // (not 0 * inf)
        }
        __syncthreads();
        if (first + FC < s.first + s.count) fetch(first + FC);
        if (!STATE_ONLY) {
            float p[2][2] = {};
#pragma unroll 2
            for (int c = 0; c < dk4; c += 4) {
                float4 x[2], y[2];
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    x[i] = *reinterpret_cast<const float4 *>(sq + (ty + 16 * i) * LD + c);
                    y[i] = *reinterpret_cast<const float4 *>(sk + (tx + 16 * i) * LD + c);
                }
#pragma unroll
                for (int i = 0; i < 2; i++)
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        p[i][j] = fmaf(x[i].x, y[j].x, p[i][j]);
                        p[i][j] = fmaf(x[i].y, y[j].y, p[i][j]);
                        p[i][j] = fmaf(x[i].z, y[j].z, p[i][j]);
                        p[i][j] = fmaf(x[i].w, y[j].w, p[i][j]);
                    }
            }
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    const int t = ty + 16 * i, u = tx + 16 * j;
                    sp[t * 36 + u] = t >= u ? p[i][j] * exp2f(g2 * (float)(t - u)) * (a.scale_in * a.scale_out) : 0.0f;
                }
            __syncthreads();
            float o[2][4] = {};
            const auto add = [&o](int i, float x, const float4 &y) {
                o[i][0] = fmaf(x, y.x, o[i][0]), o[i][1] = fmaf(x, y.y, o[i][1]);
                o[i][2] = fmaf(x, y.z, o[i][2]), o[i][3] = fmaf(x, y.w, o[i][3]);
            };
#pragma unroll 2
            for (int c = 0; c < dk4; c += 4) {
                float4 zz[4];
#pragma unroll
                for (int j = 0; j < 4; j++) zz[j] = *reinterpret_cast<const float4 *>(sz + (c + j) * FV + 4 * tx);
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const float4 x = *reinterpret_cast<const float4 *>(sq + (ty + 16 * i) * LD + c);
                    add(i, x.x, zz[0]), add(i, x.y, zz[1]), add(i, x.z, zz[2]), add(i, x.w, zz[3]);
                }
            }
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const float w = exp2f(g2 * (float)(ty + 16 * i)) * a.scale_out;
#pragma unroll
                for (int j = 0; j < 4; j++) o[i][j] *= w;
            }
#pragma unroll 2
            for (int u = 0; u < tokens; u += 4) {
                float4 vv[4];
#pragma unroll
                for (int j = 0; j < 4; j++) vv[j] = *reinterpret_cast<const float4 *>(sv + (u + j) * LV + 4 * tx);
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const int t = ty + 16 * i;
                    const float4 x = *reinterpret_cast<const float4 *>(sp + t * 36 + u);
                    if (u <= t) add(i, x.x, vv[0]);  // later tokens do not reach this one, not even as 0 * inf
                    if (u + 1 <= t) add(i, x.y, vv[1]);
                    if (u + 2 <= t) add(i, x.z, vv[2]);
                    if (u + 3 <= t) add(i, x.w, vv[3]);
                }
            }
            O *out = a.out.at<O>(a.starts == nullptr ? s.seq : 0, hg, hi) + v0 * a.out.col;
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const int t = ty + 16 * i;
                if (t >= tokens) continue;
                O *row = out + token_row(a, s, first + t) * a.out.row;
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (4 * tx + j < cols) row[(4 * tx + j) * a.out.col] = from_float<O>(o[i][j]);
            }
        }
        const float carry = exp2f(g2 * (float)e);
#pragma unroll
        for (int i = 0; i < ROWS; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) z[i][j] *= carry;
#pragma unroll 4
        for (int u = 0; u < tokens; u++) {
            const float w = sw[u];
            const float4 vv = *reinterpret_cast<const float4 *>(sv + u * LV + 4 * tx);
#pragma unroll
            for (int i = 0; i < ROWS; i += 4) {
                const float4 k4 = *reinterpret_cast<const float4 *>(sk + u * LD + ROWS * ty + i);
                const float x[4] = {k4.x * w, k4.y * w, k4.z * w, k4.w * w};
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    z[i + j][0] = fmaf(x[j], vv.x, z[i + j][0]), z[i + j][1] = fmaf(x[j], vv.y, z[i + j][1]);
                    z[i + j][2] = fmaf(x[j], vv.z, z[i + j][2]), z[i + j][3] = fmaf(x[j], vv.w, z[i + j][3]);
                }
            }
        }
    }
    if (STATE_ONLY || (s.last && a.state_out.data != nullptr)) {
#pragma unroll
        for (int i = 0; i < ROWS; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int r = ROWS * ty + i, c = 4 * tx + j;
                if (r >= a.dk || c >= cols) continue;
                if (STATE_ONLY)
                    a.states[(((int64_t)s.adds * a.heads + h) * a.dk + r) * a.dv + v0 + c] = z[i][j];
                else
                    a.state_out.at<float>(s.seq, hg, hi)[r * a.state_out.row + (v0 + c) * a.state_out.col] = z[i][j];
            }
    }
}

// ------------------------------------------------------------------------------------------------
// States at the start of each segment but the first, in place of what the segments before them add.  A thread takes four
// values of the state through the segments of a sequence, four segments loaded ahead: all is read and written once.
//
// TANGENT: of Z and, behind it, M = dZ/dg:  M <- e^{g n} (n Z + M) + own, n = tokens of a segment.
template <bool TANGENT>
__global__ void __launch_bounds__(256) decay_scan_kernel(DecayArgs a) {
    const unsigned h = blockIdx.x % a.heads, seq = blockIdx.x / a.heads;
    const unsigned hg = h / a.group, hi = h - hg * a.group;
    int64_t begin, length;
    sequence_rows(a, seq, begin, length);
    const int64_t place = first_place(a, seq);
    const int n = (int)min((int64_t)segments_of(a, length) - 1, a.state_slots - place);
    if (n <= 0) return;
    const float g2 = log2_decay(a.log_decay[h]);
    const float carry = exp2f(g2 * (float)a.segment), enter = a.reverse ? 1.0f : exp2f(g2);
    const int values = a.dk * a.dv, first = blockIdx.y * 1024 + threadIdx.x;
    constexpr int N = TANGENT ? 2 : 1;
    float z[4], m[4];
#pragma unroll
    for (int c = 0; c < 4; c++) {
        const int i = first + 256 * c;
        z[c] = m[c] = a.state_in.data != nullptr && i < values
                          ? enter * a.state_in.at<float>(seq, hg, hi)[(i / a.dv) * a.state_in.row + (i % a.dv) * a.state_in.col]
                          : 0.0f;
    }
    float *p = a.states + (place * a.heads + h) * N * values + first;
    const int64_t step = (int64_t)a.heads * N * values;
    const float tokens = (float)a.segment;
    for (int j = 0; j < n; j += 4) {
        float own[4][4], own_m[4][4];
#pragma unroll
        for (int u = 0; u < 4; u++)
#pragma unroll
            for (int c = 0; c < 4; c++) {
                const bool there = j + u < n && first + 256 * c < values;
                own[u][c] = there ? p[(j + u) * step + 256 * c] : 0.0f;
                own_m[u][c] = TANGENT && there ? p[(j + u) * step + values + 256 * c] : 0.0f;
            }
#pragma unroll
        for (int u = 0; u < 4; u++)
#pragma unroll
            for (int c = 0; c < 4; c++) {
                if (TANGENT) m[c] = fmaf(carry, fmaf(tokens, z[c], m[c]), own_m[u][c]);
                z[c] = fmaf(carry, z[c], own[u][c]);
                if (j + u < n && first + 256 * c < values) {
                    p[(j + u) * step + 256 * c] = z[c];
                    if (TANGENT) p[(j + u) * step + values + 256 * c] = m[c];
                }
            }
    }
}

// ------------------------------------------------------------------------------------------------
// Gradient of the log decays.  With M = dZ/dg the chunk's outputs change with g by
//   d out_t = scale [ sum_s (t - s) e^{g (t - s)} (q_t . k_s) v_s + e^{g t} (t Z + M)^T q_t ],
//   M <- e^{g e} (e Z + M) + sum_s (e - s) e^{g (e - s)} k_s v_s^T,
// and grad = sum_t dout_t . d out_t + <dstate, dM of the last state>: a sum of terms that are each as small as their
// distances, where differences of sums over tokens (t q.dq - s k.dk) would cancel to a part of 1 / tokens.
// One CTA per (segment, head, 32 columns of v): the states' columns are independent.  All in fp32, sums over chunks in fp64.
// STATE_ONLY: the states that a segment adds, from zero (before the scan).
constexpr int GV = 32;  // columns of v

// ROWS: groups of 32 rows of the state, 2 for dk up to 64: half of the work, and three CTAs to an SM instead of two.
template <int ROWS>
struct GradFmaSmem {
    static constexpr int LD = 32 * ROWS + 4, LV = GV + 4;
    static constexpr int Q = 0, K = FC * LD, V = 2 * FC * LD, D = V + FC * LV, W = D + FC * LV, Z = W + 2 * FC, M = Z + 32 * ROWS * LV,
                         BYTES = (M + 32 * ROWS * LV) * 4;
};

template <typename T, int ROWS, bool STATE_ONLY>
__global__ void __launch_bounds__(256, ROWS == 2 ? 3 : 2) decay_gradient_kernel(DecayArgs a, Operand dout, Operand dstate, int vblocks, double *partials) {
    using L = GradFmaSmem<ROWS>;
    constexpr int LD = L::LD, LV = L::LV;
    extern __shared__ __align__(16) float smem[];
    float *sq = smem + L::Q, *sk = smem + L::K, *sv = smem + L::V, *sd = smem + L::D, *sw = smem + L::W, *sz = smem + L::Z, *sm = smem + L::M;
    const int vb = blockIdx.x % vblocks;
    const unsigned rest = blockIdx.x / (unsigned)vblocks;
    const int64_t h = rest % a.heads, slot = rest / a.heads;
    const int64_t hg = h / a.group, hi = h - hg * a.group;
    const Segment s = find_segment(a, slot);
    if (!s.used || (STATE_ONLY && s.last)) {
        if (!STATE_ONLY && threadIdx.x == 0) partials[(h * a.slots + slot) * vblocks + vb] = 0.0;
        return;
    }
    const int tid = threadIdx.x, tx = tid & 7, ty = tid >> 3;  // columns 4 tx .. + 3, rows ty + 32 i
    const int cols = min(GV, a.dv - vb * GV), dk4 = (a.dk + 3) & ~3;
    const float g2 = log2_decay(a.log_decay[h]);
    Operand v = a.v, d = dout;
    v.data += vb * GV * v.col * (int64_t)sizeof(T);
    d.data += vb * GV * d.col * (int64_t)sizeof(T);
    const int64_t state = (int64_t)a.dk * a.dv;
    // Z, then M, where sequences are cut
    float *own = a.states + ((int64_t)s.adds * a.heads + h) * 2 * state + vb * GV;
    const float *start = a.states + ((int64_t)s.start * a.heads + h) * 2 * state + vb * GV;
    float z[ROWS][4], m[ROWS][4];
#pragma unroll
    for (int i = 0; i < ROWS; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int r = ty + 32 * i, c = 4 * tx + j;
            z[i][j] = m[i][j] = 0.0f;
            if (STATE_ONLY || r >= a.dk || c >= cols) continue;
            if (s.first > 0)
                z[i][j] = start[r * a.dv + c], m[i][j] = start[state + r * a.dv + c];
            else if (a.state_in.data != nullptr)
                z[i][j] = m[i][j] = exp2f(g2) * a.state_in.at<float>(s.seq, hg, hi)[r * a.state_in.row + (vb * GV + c) * a.state_in.col];
        }
    double total = 0.0;
    ChunkRows<T, 32 * ROWS> nq, nk;
    ChunkRows<T, GV> nv, nd;
    const auto fetch = [&](int first) {
        const int tokens = min(FC, s.first + s.count - first);
        if (!STATE_ONLY) nq.fetch(a, s, a.q, hg, hi, first, tokens, a.dk);
        nk.fetch(a, s, a.k, hg, hi, first, tokens, a.dk);
        nv.fetch(a, s, v, hg, hi, first, tokens, cols);
        if (!STATE_ONLY) nd.fetch(a, s, d, hg, hi, first, tokens, cols);
    };
    if (s.count > 0) fetch(s.first);
    for (int first = s.first; first < s.first + s.count; first += FC) {
        const int tokens = min(FC, s.first + s.count - first);
        const int e = first + tokens == s.length ? tokens - 1 : tokens;
        __syncthreads();
        if (!STATE_ONLY) nq.template put<LD>(sq);
        nk.template put<LD>(sk);
        nv.template put<LV>(sv);
        if (!STATE_ONLY) nd.template put<LV>(sd);
        if (tid < FC) {
            const float w = exp2f(g2 * (float)max(e - tid, 0));
            sw[2 * tid] = w, sw[2 * tid + 1] = w * (float)max(e - tid, 0);
        }
        if (!STATE_ONLY) {
#pragma unroll
            for (int i = 0; i < ROWS; i++) {
                const bool row = ty + 32 * i < a.dk;  // (zeros behind dk: not 0 * inf)
                const float4 none = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                *reinterpret_cast<float4 *>(sz + (ty + 32 * i) * LV + 4 * tx) = row ? make_float4(z[i][0], z[i][1], z[i][2], z[i][3]) : none;
                *reinterpret_cast<float4 *>(sm + (ty + 32 * i) * LV + 4 * tx) = row ? make_float4(m[i][0], m[i][1], m[i][2], m[i][3]) : none;
            }
        }
        __syncthreads();
        if (first + FC < s.first + s.count) fetch(first + FC);
        float sum = 0.0f;
        if (!STATE_ONLY) {  // inside the chunk: entries (t, u) with t = ty, u = tx + 8 i
            float p[4] = {}, r[4] = {};
            for (int c = 0; c < dk4; c += 4) {
                const float4 x = *reinterpret_cast<const float4 *>(sq + ty * LD + c);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float4 y = *reinterpret_cast<const float4 *>(sk + (tx + 8 * i) * LD + c);
                    p[i] = fmaf(x.x, y.x, fmaf(x.y, y.y, fmaf(x.z, y.z, fmaf(x.w, y.w, p[i]))));
                }
            }
            for (int c = 0; c < GV; c += 4) {
                const float4 x = *reinterpret_cast<const float4 *>(sd + ty * LV + c);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float4 y = *reinterpret_cast<const float4 *>(sv + (tx + 8 * i) * LV + c);
                    r[i] = fmaf(x.x, y.x, fmaf(x.y, y.y, fmaf(x.z, y.z, fmaf(x.w, y.w, r[i]))));
                }
            }
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int u = tx + 8 * i;
                if (ty > u) sum = fmaf((float)(ty - u) * exp2f(g2 * (float)(ty - u)) * p[i], r[i], sum);
            }
        }
        if (!STATE_ONLY) {  // from the states: row t = ty, columns 4 tx ..
            float x[4] = {}, y[4] = {};
            const auto add = [](float f, const float4 &v, float (&to)[4]) {
                to[0] = fmaf(f, v.x, to[0]), to[1] = fmaf(f, v.y, to[1]), to[2] = fmaf(f, v.z, to[2]), to[3] = fmaf(f, v.w, to[3]);
            };
#pragma unroll 2
            for (int c = 0; c < dk4; c += 4) {
                const float4 qv = *reinterpret_cast<const float4 *>(sq + ty * LD + c);
                const float f[4] = {qv.x, qv.y, qv.z, qv.w};
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    add(f[j], *reinterpret_cast<const float4 *>(sz + (c + j) * LV + 4 * tx), x);
                    add(f[j], *reinterpret_cast<const float4 *>(sm + (c + j) * LV + 4 * tx), y);
                }
            }
            const float w = exp2f(g2 * (float)ty);
            float part = 0.0f;
#pragma unroll
            for (int j = 0; j < 4; j++) part = fmaf(fmaf((float)ty, x[j], y[j]), sd[ty * LV + 4 * tx + j], part);
            if (ty < tokens) sum = fmaf(w, part, sum);
        }
        total += (double)sum * (double)a.scale_out;
        const float carry = exp2f(g2 * (float)e);
#pragma unroll
        for (int i = 0; i < ROWS; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                m[i][j] = carry * fmaf((float)e, z[i][j], m[i][j]);
                z[i][j] *= carry;
            }
#pragma unroll 4
        for (int u = 0; u < tokens; u++) {
            const float2 w = *reinterpret_cast<const float2 *>(sw + 2 * u);
            const float4 vv = *reinterpret_cast<const float4 *>(sv + u * LV + 4 * tx);
#pragma unroll
            for (int i = 0; i < ROWS; i++) {
                const float kk = sk[u * LD + ty + 32 * i], x = kk * w.x, y = kk * w.y;
                z[i][0] = fmaf(x, vv.x, z[i][0]), z[i][1] = fmaf(x, vv.y, z[i][1]), z[i][2] = fmaf(x, vv.z, z[i][2]),
                z[i][3] = fmaf(x, vv.w, z[i][3]);
                m[i][0] = fmaf(y, vv.x, m[i][0]), m[i][1] = fmaf(y, vv.y, m[i][1]), m[i][2] = fmaf(y, vv.z, m[i][2]),
                m[i][3] = fmaf(y, vv.w, m[i][3]);
            }
        }
    }
    if (STATE_ONLY) {
#pragma unroll
        for (int i = 0; i < ROWS; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int r = ty + 32 * i, c = 4 * tx + j;
                if (r < a.dk && c < cols) own[r * a.dv + c] = z[i][j], own[state + r * a.dv + c] = m[i][j];
            }
        return;
    }
    if (dstate.data != nullptr && s.last && s.length > 0) {
#pragma unroll
        for (int i = 0; i < ROWS; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int r = ty + 32 * i, c = 4 * tx + j;
                // (m holds e^{g e} (e Z + M) + ..: the derivative of the last state, whose Z is e^g S_0 with M = Z)
                if (r < a.dk && c < cols)
                    total += (double)m[i][j] * (double)dstate.at<float>(s.seq, hg, hi)[r * dstate.row + (vb * GV + c) * dstate.col];
            }
    }
    __shared__ double warp_sum[8];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    if ((tid & 31) == 0) warp_sum[tid >> 5] = total;
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < 8; w++) total += warp_sum[w];
        partials[(h * a.slots + slot) * vblocks + vb] = total;
    }
}

__global__ void __launch_bounds__(256) decay_gradient_finish_kernel(int64_t count, const double *partials, float *grad) {
    __shared__ double warp_sum[8];
    const int64_t h = blockIdx.x;
    double v = 0.0;
    for (int64_t i = threadIdx.x; i < count; i += 256) v += partials[h * count + i];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if ((threadIdx.x & 31) == 0) warp_sum[threadIdx.x >> 5] = v;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 8; w++) v += warp_sum[w];
        grad[h] = (float)v;
    }
}

// ------------------------------------------------------------------------------------------------
template <typename T>
__global__ void __launch_bounds__(256) group_sums_kernel(int64_t count, int64_t group, int64_t dim, const float *in, T *out) {
    for (int64_t i = blockIdx.x * 256LL + threadIdx.x; i < count; i += 256LL * gridDim.x) {
        const int64_t rg = i / dim, c = i - rg * dim;
        const float *p = in + rg * group * dim + c;
        float v = 0.0f;
        for (int64_t j = 0; j < group; j++) v += p[j * dim];
        out[i] = from_float<T>(v);
    }
}

// ------------------------------------------------------------------------------------------------
// One token: S <- e^g S + k v^T, out = scale S^T q.  Reading and writing the state is all the time there is.  A CTA of
// 256 threads per (row, head, COLS columns of v): a thread holds VEC neighbouring columns of every (256 VEC / COLS)-th
// row of the state, all of them loaded before the first is used; the sums over dk go through shared memory.
template <typename T, int VEC, int COLS>
__global__ void __launch_bounds__(256, COLS == 128 ? 2 : 4) decay_step_kernel(int64_t rows, int64_t pool, int64_t heads, int64_t group, int dk, int dv, Operand q,
                                                         Operand k, Operand v, Operand out, const float *log_decay, Operand states,
                                                         int slot_type, const void *slots, float scale) {
    constexpr int TX = COLS / VEC, TY = 256 / TX, N = (KM_DECAY_MAX_DIM + TY - 1) / TY;
    __shared__ float part[TY][COLS + 4];
    __shared__ float sq[KM_DECAY_MAX_DIM], sk[KM_DECAY_MAX_DIM];
    const int vblocks = (dv + COLS - 1) / COLS;
    const int vb = blockIdx.x % vblocks;
    const int64_t rest = blockIdx.x / vblocks, h = rest % heads;
    int64_t row = rest / heads;
    const int64_t hg = h / group, hi = h - hg * group;
    const int tid = threadIdx.x, tx = tid % TX, ty = tid / TX, col = vb * COLS + tx * VEC;
    const auto slot_of = [&](int64_t r) -> int64_t {
        if (slots == nullptr) return r;
        return slot_type == KM_TYPE_I32 ? static_cast<const int32_t *>(slots)[r] : static_cast<const int64_t *>(slots)[r];
    };
    const int64_t slot = slot_of(row);
    const bool valid = slot >= 0 && slot < pool;
    // rows with the same slot: the first one's CTA takes them all, in order
    bool again = false;
    if (slots != nullptr && valid) {
        bool earlier = false, later = false;
        for (int64_t r = tid; r < rows; r += 256) {
            const bool same = slot_of(r) == slot;
            earlier = earlier || (same && r < row);
            later = later || (same && r > row);
        }
        if (__syncthreads_or(earlier)) return;
        again = __syncthreads_or(later);
    }
    const bool mine = col < dv;
    if (!valid) {
        if (mine && ty == 0)
            for (int j = 0; j < VEC; j++)
                if (col + j < dv) out.at<T>(row, hg, hi)[col + j] = from_float<T>(0.0f);
        return;
    }
    const float decay = exp2f(log2_decay(log_decay[h]));
    float *state = states.at<float>(slot, hg, hi) + col;
    float s[N][VEC];
#pragma unroll
    for (int i = 0; i < N; i++) {
        const int r = ty + i * TY;
#pragma unroll
        for (int j = 0; j < VEC; j++) s[i][j] = 0.0f;
        if (mine && r < dk) {
            if constexpr (VEC == 4) {
                const float4 x = __ldcs(reinterpret_cast<const float4 *>(state + r * states.row));
                s[i][0] = x.x, s[i][1] = x.y, s[i][2] = x.z, s[i][3] = x.w;
            } else {
                s[i][0] = state[r * states.row];
            }
        }
    }
    for (;;) {
        for (int c = tid; c < dk; c += 256) {
            sq[c] = as_float(q.at<const T>(row, hg, hi)[c]);
            sk[c] = as_float(k.at<const T>(row, hg, hi)[c]);
        }
        float vv[VEC], o[VEC] = {};
#pragma unroll
        for (int j = 0; j < VEC; j++) vv[j] = col + j < dv ? as_float(v.at<const T>(row, hg, hi)[col + j]) : 0.0f;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; i++) {
            const int r = ty + i * TY;
            if (r < dk) {
                const float kk = sk[r], qq = sq[r];
#pragma unroll
                for (int j = 0; j < VEC; j++) {
                    s[i][j] = fmaf(decay, s[i][j], kk * vv[j]);
                    o[j] = fmaf(qq, s[i][j], o[j]);
                }
            }
        }
#pragma unroll
        for (int j = 0; j < VEC; j++) part[ty][tx * VEC + j] = o[j];
        __syncthreads();
        for (int c = tid; c < COLS; c += 256) {
            if (vb * COLS + c >= dv) continue;
            float sum = 0.0f;
#pragma unroll 8
            for (int y = 0; y < TY; y++) sum += part[y][c];
            out.at<T>(row, hg, hi)[vb * COLS + c] = from_float<T>(sum * scale);
        }
        if (!again) break;
        do row++;
        while (row < rows && slot_of(row) != slot);
        if (row >= rows) break;
    }
#pragma unroll
    for (int i = 0; i < N; i++) {
        const int r = ty + i * TY;
        if (mine && r < dk) {
            if constexpr (VEC == 4)
                __stcs(reinterpret_cast<float4 *>(state + r * states.row), make_float4(s[i][0], s[i][1], s[i][2], s[i][3]));
            else
                state[r * states.row] = s[i][0];
        }
    }
}

// ------------------------------------------------------------------------------------------ host

static int sm_count() {
    int dev = 0, sms = 148;
    if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    return sms;
}

struct DecayPlan {
    bool tc, split;
    int64_t segment, slots, states;  // states: places for those between segments, at most
};

static DecayPlan plan_of(const km_decay_problem &p) {
    DecayPlan r;
    r.tc = p.path == 2;
    const int64_t chunk = r.tc ? 128 : FC, sms = 148, heads = p.groups * p.group;
    const int64_t chunks = ceil_div(std::max<int64_t>(p.tokens, 1), chunk);
    // Chunks of a segment.  A cut costs the segments' own states (k and v once more) and the scan, about half of the
    // time again and some chunks' worth of launches.
    int64_t per = chunks;
    if (p.packed) {
        // lengths are known on the device only: segments of which all sequences together give two per SM, but of no fewer than
        // eight chunks, for which two further launches do not pay
        per = std::min(chunks, std::max<int64_t>(8, ceil_div(chunks * heads, 2 * sms)));
    } else {
        double best = (double)ceil_div(p.sequences * heads, sms) * (double)(chunks + 2);
        for (int64_t n = 2; n <= 64 && n <= chunks; n++) {
            const int64_t len = ceil_div(chunks, n), pieces = ceil_div(chunks, len);
            const double cost = (double)ceil_div(p.sequences * heads * pieces, sms) * (double)(len + 2) * 1.5 + 6.0;
            if (cost < best) best = cost, per = len;
        }
    }
    r.segment = per * chunk;
    r.split = per < chunks;
    r.slots = p.packed ? p.tokens / r.segment + p.sequences : p.sequences * ceil_div(std::max<int64_t>(p.tokens, 1), r.segment);
    r.states = r.split ? std::max<int64_t>(r.slots - p.sequences, 1) : 0;
    return r;
}

static int check_problem(const char *name, const km_decay_problem *p) {
    KM_REQUIRE(p != nullptr, KM_ERR_INVALID_ARGUMENT, "%s: null problem", name);
    KM_REQUIRE(p->dtype >= KM_TYPE_F32 && p->dtype <= KM_TYPE_F16 && (p->out_dtype == p->dtype || p->out_dtype == KM_TYPE_F32),
               KM_ERR_INVALID_ARGUMENT, "%s: bad element type", name);
    KM_REQUIRE(p->path == 1 || (p->path == 2 && p->dtype != KM_TYPE_F32), KM_ERR_UNSUPPORTED,
               "%s: path must be 1 (FMA pipe) or, for 16-bit types, 2 (tensor cores)", name);
    KM_REQUIRE(p->reverse >= 0 && p->reverse <= 2, KM_ERR_INVALID_ARGUMENT, "%s: reverse must be 0, 1 or 2", name);
    KM_REQUIRE(p->states == 0 || p->states == 2, KM_ERR_INVALID_ARGUMENT, "%s: states must be 0 or 2", name);
    KM_REQUIRE(p->sequences >= 0 && p->tokens >= 0 && p->groups >= 0 && p->group >= 1, KM_ERR_INVALID_ARGUMENT, "%s: bad sizes", name);
    KM_REQUIRE(p->dk >= 1 && p->dk <= KM_DECAY_MAX_DIM && p->dv >= 1 && p->dv <= KM_DECAY_MAX_DIM, KM_ERR_UNSUPPORTED,
               "%s: head sizes must be 1 to %d", name, KM_DECAY_MAX_DIM);
    const int64_t limit = (1LL << 31) - 4096;
    KM_REQUIRE(p->tokens < limit && p->sequences < limit && p->groups < limit && p->group < limit &&
                   p->groups * p->group < limit && p->sequences * (p->groups * p->group) < limit,
               KM_ERR_UNSUPPORTED, "%s: more than 2^31 tokens or (sequence, head) pairs", name);
    return KM_OK;
}

// What path 0 takes.
static km_decay_problem resolved(const km_decay_problem &p) {
    km_decay_problem r = p;
    if (r.path == 0) r.path = r.dtype == KM_TYPE_F32 ? 1 : 2;
    return r;
}

template <bool TANGENT>
static int launch_scan(const DecayArgs &a, cudaStream_t s) {
    decay_scan_kernel<TANGENT><<<dim3((unsigned)(a.sequences * a.heads), (unsigned)ceil_div(a.dk * a.dv, 1024)), 256, 0, s>>>(a);
    KM_CHECK_LAUNCH("decay_scan_kernel launch");
    return KM_OK;
}

template <typename T, typename O>
static int launch_fma(const DecayArgs &a, bool state_only, cudaStream_t s) {
    const bool few = a.dk <= 64;
    auto kernel = few ? state_only ? decay_fma_kernel<T, O, 4, true> : decay_fma_kernel<T, O, 4, false>
                      : state_only ? decay_fma_kernel<T, O, 8, true> : decay_fma_kernel<T, O, 8, false>;
    const int bytes = few ? FmaSmem<4>::BYTES : FmaSmem<8>::BYTES, vblocks = (int)ceil_div(a.dv, FV);
    cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (err != cudaSuccess) return cuda_fail(err, "decay_fma_kernel");
    KM_REQUIRE(a.slots * a.heads * vblocks < (1LL << 31), KM_ERR_UNSUPPORTED, "km_decay_attention: more than 2^31 work items");
    kernel<<<(unsigned)(a.slots * a.heads * vblocks), 256, bytes, s>>>(a, vblocks);
    KM_CHECK_LAUNCH("decay_fma_kernel launch");
    return KM_OK;
}

static int launch_main(const km_decay_problem &p, const DecayArgs &a, bool tc, bool state_only, cudaStream_t s) {
    if (tc) return launch_decay_tc(p, a, state_only, s);
    const bool wide = p.out_dtype == KM_TYPE_F32;
    if (p.dtype == KM_TYPE_F32) return launch_fma<float, float>(a, state_only, s);
    if (p.dtype == KM_TYPE_BF16)
        return wide ? launch_fma<__nv_bfloat16, float>(a, state_only, s) : launch_fma<__nv_bfloat16, __nv_bfloat16>(a, state_only, s);
    return wide ? launch_fma<__half, float>(a, state_only, s) : launch_fma<__half, __half>(a, state_only, s);
}

static DecayArgs make_args(const km_decay_problem &p, const km_view *q, const km_view *k, const km_view *v, const float *log_decay,
                           const int32_t *starts, const km_view *state_in) {
    DecayArgs a = {};
    a.q = make_operand(q), a.k = make_operand(k), a.v = make_operand(v);
    a.state_in = make_operand(state_in);
    a.log_decay = log_decay;
    a.starts = p.packed ? starts : nullptr;
    a.sequences = p.sequences, a.tokens = p.tokens, a.group = p.group, a.heads = p.groups * p.group;
    a.dk = (int)p.dk, a.dv = (int)p.dv;
    return a;
}

}  // namespace km

extern "C" size_t km_decay_attention_workspace_bytes(const km_decay_problem *problem) {
    using namespace km;
    if (problem == nullptr) return 0;
    const km_decay_problem p = resolved(*problem);
    if (check_problem("km_decay_attention_workspace_bytes", &p) != KM_OK) return 0;
    const DecayPlan plan = plan_of(p);
    return (size_t)plan.states * (size_t)(p.groups * p.group * p.dk * p.dv) * 4;
}

extern "C" int km_decay_attention(const km_decay_problem *problem, const km_view *q, const km_view *k, const km_view *v, const km_view *out,
                                  const float *log_decay, const int32_t *starts, const km_view *state_in, const km_view *state_out,
                                  void *workspace, size_t workspace_bytes, void *stream) {
    using namespace km;
    KM_REQUIRE(problem != nullptr, KM_ERR_INVALID_ARGUMENT, "km_decay_attention: null problem");
    const km_decay_problem p = resolved(*problem);
    int rc = check_problem("km_decay_attention", &p);
    if (rc != KM_OK) return rc;
    if (p.sequences == 0 || p.groups == 0) return KM_OK;
    KM_REQUIRE(q && k && v && out && log_decay && (!p.packed || starts), KM_ERR_INVALID_ARGUMENT, "km_decay_attention: null argument");
    KM_REQUIRE(p.tokens == 0 || (q->data && k->data && v->data && out->data), KM_ERR_INVALID_ARGUMENT, "km_decay_attention: null pointer");
    const DecayPlan plan = plan_of(p);
    const size_t need = km_decay_attention_workspace_bytes(problem);
    KM_REQUIRE(need == 0 || (workspace != nullptr && workspace_bytes >= need), KM_ERR_WORKSPACE,
               "km_decay_attention: workspace of %zu bytes needed, %zu given", need, workspace_bytes);
    KM_REQUIRE(need == 0 || reinterpret_cast<uintptr_t>(workspace) % 16 == 0, KM_ERR_WORKSPACE, "km_decay_attention: workspace must be 16-byte aligned");
    DecayArgs a = make_args(p, q, k, v, log_decay, starts, state_in);
    a.out = make_operand(out);
    a.state_out = make_operand(state_out);
    a.segment = (unsigned)plan.segment;
    a.slots = plan.slots;
    a.states = static_cast<float *>(workspace);
    a.state_slots = plan.states;
    a.state_row = p.states == 2 ? 1 : (int)p.dv, a.state_col = p.states == 2 ? (int)p.dk : 1;
    a.reverse = p.reverse == 1;
    a.scale_in = a.reverse ? p.scale : 1.0f;
    a.scale_out = a.reverse ? 1.0f : p.scale;
    // In bf16 the state, an fp32 result, needs three parts of the decayed keys; forward calls take them whether or not it is asked for, so that
    // the result is the same.  The passes of a gradient that return no state do with two (2^-17).
    a.parts = p.dtype == KM_TYPE_BF16 && (p.reverse == 0 || a.state_out.data != nullptr) ? 3 : 2;
    a.wait_polls = current_wait_polls();
    a.gave_up = plan.tc ? gave_up_word() : nullptr;
    KM_REQUIRE(a.slots * a.heads < (1LL << 31), KM_ERR_UNSUPPORTED, "km_decay_attention: more than 2^31 work items");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (plan.split && p.states == 0) {
        rc = launch_main(p, a, plan.tc, true, s);
        if (rc != KM_OK) return rc;
        rc = launch_scan<false>(a, s);
        if (rc != KM_OK) return rc;
    }
    return launch_main(p, a, plan.tc, false, s);
}

namespace km {

// Partial sums, and values of states, of the gradient of the decays.  (On the FMA pipe four CTAs share a head's columns.)
static size_t grad_sums(const km_decay_problem &p) {
    return (size_t)(p.groups * p.group) * (size_t)plan_of(p).slots * (size_t)(p.path == 2 ? 1 : ceil_div(p.dv, GV));
}
static size_t grad_states(const km_decay_problem &p) {
    return (size_t)plan_of(p).states * (size_t)(p.groups * p.group * p.dk * p.dv) * 2;
}

template <typename T, bool STATE_ONLY>
static int launch_grad_fma(const DecayArgs &a, const Operand &d, const Operand &ds, double *partials, cudaStream_t s) {
    auto kernel = a.dk <= 64 ? decay_gradient_kernel<T, 2, STATE_ONLY> : decay_gradient_kernel<T, 4, STATE_ONLY>;
    const int bytes = a.dk <= 64 ? GradFmaSmem<2>::BYTES : GradFmaSmem<4>::BYTES;
    const cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (err != cudaSuccess) return cuda_fail(err, "decay_gradient_kernel");
    const int vblocks = (int)ceil_div(a.dv, GV);
    kernel<<<(unsigned)(a.slots * a.heads * vblocks), 256, bytes, s>>>(a, d, ds, vblocks, partials);
    KM_CHECK_LAUNCH("decay_gradient_kernel launch");
    return KM_OK;
}

static int launch_grad(const km_decay_problem &p, const DecayArgs &a, const Operand &d, const Operand &ds, double *partials, bool state_only,
                       cudaStream_t s) {
    if (p.path == 2) return launch_decay_grad_tc(p, a, d, ds, partials, state_only, s);
    if (p.dtype == KM_TYPE_F32)
        return state_only ? launch_grad_fma<float, true>(a, d, ds, partials, s) : launch_grad_fma<float, false>(a, d, ds, partials, s);
    if (p.dtype == KM_TYPE_BF16)
        return state_only ? launch_grad_fma<__nv_bfloat16, true>(a, d, ds, partials, s) : launch_grad_fma<__nv_bfloat16, false>(a, d, ds, partials, s);
    return state_only ? launch_grad_fma<__half, true>(a, d, ds, partials, s) : launch_grad_fma<__half, false>(a, d, ds, partials, s);
}

}  // namespace km

extern "C" size_t km_decay_gradient_workspace_bytes(const km_decay_problem *problem) {
    using namespace km;
    if (problem == nullptr) return 0;
    const km_decay_problem p = resolved(*problem);
    if (check_problem("km_decay_gradient_workspace_bytes", &p) != KM_OK) return 0;
    return grad_sums(p) * sizeof(double) + grad_states(p) * sizeof(float);
}

extern "C" int km_decay_gradient(const km_decay_problem *problem, const km_view *q, const km_view *k, const km_view *v, const km_view *dout,
                                 const float *log_decay, const int32_t *starts, const km_view *state_in, const km_view *dstate, float *grad,
                                 void *workspace, size_t workspace_bytes, void *stream) {
    using namespace km;
    KM_REQUIRE(problem != nullptr, KM_ERR_INVALID_ARGUMENT, "km_decay_gradient: null problem");
    const km_decay_problem p = resolved(*problem);
    int rc = check_problem("km_decay_gradient", &p);
    if (rc != KM_OK) return rc;
    if (p.groups == 0) return KM_OK;
    KM_REQUIRE(q && k && v && dout && log_decay && grad && (!p.packed || starts), KM_ERR_INVALID_ARGUMENT, "km_decay_gradient: null argument");
    KM_REQUIRE(p.tokens == 0 || p.sequences == 0 || (q->data && k->data && v->data && dout->data), KM_ERR_INVALID_ARGUMENT,
               "km_decay_gradient: null pointer");
    const size_t need = km_decay_gradient_workspace_bytes(problem);
    KM_REQUIRE(need == 0 || (workspace != nullptr && workspace_bytes >= need), KM_ERR_WORKSPACE,
               "km_decay_gradient: workspace of %zu bytes needed, %zu given", need, workspace_bytes);
    KM_REQUIRE(need == 0 || reinterpret_cast<uintptr_t>(workspace) % 16 == 0, KM_ERR_WORKSPACE, "km_decay_gradient: workspace must be 16-byte aligned");
    DecayArgs a = make_args(p, q, k, v, log_decay, starts, state_in);
    a.scale_in = 1.0f, a.scale_out = p.scale;
    const Operand d = make_operand(dout), ds = make_operand(dstate);
    a.wait_polls = current_wait_polls();
    a.gave_up = p.path == 2 ? gave_up_word() : nullptr;
    const DecayPlan plan = plan_of(p);
    const int64_t sums = (int64_t)grad_sums(p) / a.heads, ctas = sums * a.heads;
    KM_REQUIRE(ctas < (1LL << 31), KM_ERR_UNSUPPORTED, "km_decay_gradient: more than 2^31 work items");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    double *partials = static_cast<double *>(workspace);
    a.segment = (unsigned)plan.segment;
    a.slots = plan.slots;
    a.state_slots = plan.states;
    a.states = reinterpret_cast<float *>(partials + ctas);
    if (ctas > 0) {
        if (plan.split) {
            rc = launch_grad(p, a, d, ds, partials, true, s);
            if (rc == KM_OK && p.sequences > 0) rc = launch_scan<true>(a, s);
            if (rc != KM_OK) return rc;
        }
        rc = launch_grad(p, a, d, ds, partials, false, s);
        if (rc != KM_OK) return rc;
    }
    decay_gradient_finish_kernel<<<a.heads, 256, 0, s>>>(sums, partials, grad);
    KM_CHECK_LAUNCH("decay_gradient_finish_kernel launch");
    return KM_OK;
}

extern "C" int km_group_sums(int32_t dtype, int64_t rows, int64_t groups, int64_t group, int64_t dim, const float *in, void *out, void *stream) {
    using namespace km;
    KM_REQUIRE(dtype >= KM_TYPE_F32 && dtype <= KM_TYPE_F16 && rows >= 0 && groups >= 0 && group >= 1 && dim >= 0, KM_ERR_INVALID_ARGUMENT,
               "km_group_sums: bad arguments");
    if (rows == 0 || groups == 0 || dim == 0) return KM_OK;
    const int64_t limit = 1LL << 60;  // values of `in`
    KM_REQUIRE(groups <= limit / rows && dim <= limit / (rows * groups) && group <= limit / (rows * groups * dim), KM_ERR_UNSUPPORTED,
               "km_group_sums: more than 2^60 values");
    const int64_t count = rows * groups * dim;
    KM_REQUIRE(in && out, KM_ERR_INVALID_ARGUMENT, "km_group_sums: null pointer");
    const unsigned ctas = (unsigned)std::min<int64_t>(ceil_div(count, 256), 8LL * sm_count());
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (dtype == KM_TYPE_F32)
        group_sums_kernel<float><<<ctas, 256, 0, s>>>(count, group, dim, in, static_cast<float *>(out));
    else if (dtype == KM_TYPE_BF16)
        group_sums_kernel<__nv_bfloat16><<<ctas, 256, 0, s>>>(count, group, dim, in, static_cast<__nv_bfloat16 *>(out));
    else
        group_sums_kernel<__half><<<ctas, 256, 0, s>>>(count, group, dim, in, static_cast<__half *>(out));
    KM_CHECK_LAUNCH("km_group_sums launch");
    return KM_OK;
}

namespace km {

template <typename T>
static int launch_step(int64_t rows, int64_t pool, int64_t heads, int64_t group, int dk, int dv, const Operand &q, const Operand &k,
                       const Operand &v, const Operand &out, const float *log_decay, const Operand &states, int slot_type,
                       const void *slots, float scale, cudaStream_t s) {
    // columns of 16 bytes where every row of every state starts on a boundary of 16 bytes
    const bool wide = dv % 4 == 0 && reinterpret_cast<uintptr_t>(states.data) % 16 == 0 && states.seq % 4 == 0 && states.group % 4 == 0 &&
                      states.head % 4 == 0 && states.row % 4 == 0;
    // few rows: 32 columns to a CTA, so that more SMs share a state
    const bool narrow = !wide || dv <= 32 || rows * heads < 4 * 148;
    const int64_t ctas = rows * heads * ceil_div(dv, narrow ? 32 : 128);
    KM_REQUIRE(ctas < (1LL << 31), KM_ERR_UNSUPPORTED, "km_decay_step: more than 2^31 work items");
    auto kernel = !wide ? decay_step_kernel<T, 1, 32> : narrow ? decay_step_kernel<T, 4, 32> : decay_step_kernel<T, 4, 128>;
    kernel<<<(unsigned)ctas, 256, 0, s>>>(rows, pool, heads, group, dk, dv, q, k, v, out, log_decay, states, slot_type, slots, scale);
    KM_CHECK_LAUNCH("km_decay_step launch");
    return KM_OK;
}

}  // namespace km

extern "C" int km_decay_step(int32_t dtype, int64_t rows, int64_t pool, int64_t groups, int64_t group, int64_t dk, int64_t dv,
                             const km_view *q, const km_view *k, const km_view *v, const km_view *out, const float *log_decay,
                             const km_view *states, int32_t slot_type, const void *slots, float scale, void *stream) {
    using namespace km;
    KM_REQUIRE(dtype >= KM_TYPE_F32 && dtype <= KM_TYPE_F16 && rows >= 0 && pool >= 0 && groups >= 0 && group >= 1, KM_ERR_INVALID_ARGUMENT,
               "km_decay_step: bad arguments");
    KM_REQUIRE(dk >= 1 && dk <= KM_DECAY_MAX_DIM && dv >= 1 && dv <= KM_DECAY_MAX_DIM, KM_ERR_UNSUPPORTED,
               "km_decay_step: head sizes must be 1 to %d", KM_DECAY_MAX_DIM);
    KM_REQUIRE(slots == nullptr ? rows <= pool : (slot_type == KM_TYPE_I32 || slot_type == KM_TYPE_I64), KM_ERR_INVALID_ARGUMENT,
               "km_decay_step: bad slots");
    KM_REQUIRE(rows < (1LL << 31) && groups < (1LL << 31) && group < (1LL << 31) && groups * group < (1LL << 31) &&
                   rows * (groups * group) < (1LL << 31),
               KM_ERR_UNSUPPORTED, "km_decay_step: more than 2^31 (row, head) pairs");
    if (rows == 0 || groups == 0) return KM_OK;
    KM_REQUIRE(q && k && v && out && log_decay && states && q->data && k->data && v->data && out->data, KM_ERR_INVALID_ARGUMENT,
               "km_decay_step: null argument");
    KM_REQUIRE(pool == 0 || states->data, KM_ERR_INVALID_ARGUMENT, "km_decay_step: null pointer");
    KM_REQUIRE(q->stride[1] == 1 && k->stride[1] == 1 && v->stride[1] == 1 && out->stride[1] == 1 && states->stride[1] == 1,
               KM_ERR_INVALID_ARGUMENT, "km_decay_step: values of a head must be contiguous");
    const Operand oq = make_operand(q), ok = make_operand(k), ov = make_operand(v), oo = make_operand(out), os = make_operand(states);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const int64_t heads = groups * group;
    if (dtype == KM_TYPE_F32)
        return launch_step<float>(rows, pool, heads, group, (int)dk, (int)dv, oq, ok, ov, oo, log_decay, os, slot_type, slots, scale, s);
    if (dtype == KM_TYPE_BF16)
        return launch_step<__nv_bfloat16>(rows, pool, heads, group, (int)dk, (int)dv, oq, ok, ov, oo, log_decay, os, slot_type, slots, scale, s);
    return launch_step<__half>(rows, pool, heads, group, (int)dk, (int)dv, oq, ok, ov, oo, log_decay, os, slot_type, slots, scale, s);
}
