// Gradient of the log decays on the tensor cores (km_decay.cu, decay_gradient_kernel, has the formula and why it takes a second
// state): 16-bit operands, chunks of 128 tokens, one CTA per (sequence, head).
//
// The gradient is an fp32 sum, so nothing of it may be rounded to 16 bits but the decayed operands, which go in parts: two in fp16
// (2^-22, scaled by powers of two to the top of its range: 2^-39 of a chunk's largest), three in bf16 (2^-25).  Per chunk, with d = t - s, e the exponent of the chunk's end and all accumulators fp32:
//   S = Q K^T, G = dO V^T:  sum over s < t of d e^{g d} S G, entry by entry in registers
//   U  = V^T K~, U' = V^T K':       K~ = e^{g (e - s)} K,  K' = (e - s) e^{g (e - s)} K
//   X  = dO^T Q~, X' = dO^T Q':     Q~ = e^{g t} Q,        Q' = t e^{g t} Q
//   sum += <X', Z> + <X, M>,  M <- e^{g e} (e Z + M) + U',  Z <- e^{g e} Z + U   with Z and M in registers
// (the products of the states with q and then dO are sums over the tokens first, so that neither state is an operand).
// Fourteen products of 128^3 with the three parts, 7200 cycles of the tensor pipe per chunk of a head with dk = dv = 128, and between
// them the parts have to be written into the only three tiles that Q, K, V and dO leave: the phases follow one another.
// (The products of half of the tokens under the writing of the other half's parts took 706 instead of 728 us for a training step of
// 4 x 4096 tokens with 16 heads, but small parts then come onto large sums, of which the tensor cores cut the last bits: an error of 5.9e-7 of
// the gradient for 2.2e-7.)
#include "km_decay_tc.cuh"

namespace km {

namespace {

constexpr int ARITH = 512, GRAD_THREADS = ARITH + 32;  // threads of arithmetic: four per lane of tensor memory; a warp of loads and products
// Powers of two by which K' and Q' are scaled so that their weights, d e^{g (d - steps)} for distances d of `steps` to 127, are at most one
// and the largest, at d = -1 / g or 1, above a half, as fp16 needs it.  (Q' has steps = 0; K', whose decays are relative to the
// chunk's last token, that token's distance from where the chunk's state is taken: 1, or 0 at the end of a sequence.)  A slow decay's is 1/128.
constexpr float SLOW = 1.0f / 128.0f;
__device__ __forceinline__ float weight_scale(float g2, int steps) {
    const float d = g2 < -0.0114f ? fmaxf(1.0f / (-0.69314718f * g2), 1.0f) : 127.0f;
    return exp2f(-fminf(fmaxf(ceilf(log2f(d) + g2 * (d - (float)steps)), -100.0f), 7.0f));
}
constexpr uint32_t COL_S = 0, COL_G = 128, COL_U = 256, COL_U1 = 384;  // X' over S, X over G

struct GradMaps {
    CUtensorMap map[4];  // q, k, v, dO
    int use[4], by_group[4], by_head[4], by_seq[4];
};

struct GradControl {
    uint64_t full, sg_full, ready, done, read, drain, meet;
    uint32_t tmem;
    int dead;
    float inner[16];  // 2^(g2 (15 - j))
    double sums[ARITH / 32];
    alignas(16) uint16_t largest[2][2][ARITH / 32];  // fp16: magnitudes of K and Q that a warp has seen, as bits, by parity of the chunk
};

template <int KB, int VB>
struct GradSmem {
    static constexpr int Q = 0, K = KB * BLOCK_BYTES, V = 2 * KB * BLOCK_BYTES, D = V + VB * BLOCK_BYTES, SPARE = D + VB * BLOCK_BYTES,
                         CONTROL = SPARE + 3 * KB * BLOCK_BYTES, BYTES = 1024 + CONTROL + (int)sizeof(GradControl);
    static_assert(BYTES <= 232448, "shared memory of an SM");
};

// 16 bytes of an operand times w in PARTS parts, each to its own tile.
template <typename T, int PARTS>
__device__ __forceinline__ void write_parts(uint4 x, float w, unsigned char *tile, int bytes) {
    const uint32_t in[4] = {x.x, x.y, x.z, x.w};
    uint32_t r[PARTS][4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const float2 v = unpack<T>(in[j]);
        f32x2 y = mul2(pack2(v.x, v.y), splat2(w));
#pragma unroll
        for (int i = 0; i < PARTS; i++) {
            float y0, y1;
            unpack2(y, y0, y1);
            r[i][j] = pack<T>(y0, y1);
            const float2 h = unpack<T>(r[i][j]);
            y = sub2(y, pack2(h.x, h.y));
        }
    }
#pragma unroll
    for (int i = 0; i < PARTS; i++) *reinterpret_cast<uint4 *>(tile + i * bytes) = make_uint4(r[i][0], r[i][1], r[i][2], r[i][3]);
}

}  // namespace

// STATE_ONLY: the states that a segment adds, from zero (before decay_scan_kernel).
template <typename T, int KB, int VB, bool STATE_ONLY>
__global__ void __launch_bounds__(GRAD_THREADS, 1) decay_grad_tc_kernel(const __grid_constant__ DecayArgs a, const __grid_constant__ Operand dout,
                                                                        const __grid_constant__ Operand dstate,
                                                                        const __grid_constant__ GradMaps maps, double *partials) {
    using L = GradSmem<KB, VB>;
    constexpr bool HALF = std::is_same<T, __half>::value;
    constexpr int PARTS = HALF ? 2 : 3;
    constexpr int NZ = KB * 16;  // of the states' rows: this thread's columns
    constexpr uint32_t type = std::is_same<T, __half>::value ? 0u : 1u;
    extern __shared__ unsigned char raw[];
    unsigned char *smem = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
    GradControl &ctl = *reinterpret_cast<GradControl *>(smem + L::CONTROL);
    const int64_t h = blockIdx.x % a.heads, slot = blockIdx.x / a.heads;
    const int64_t hg = h / a.group, hi = h - hg * a.group;
    const Segment s = find_segment(a, slot);
    if (!s.used || (STATE_ONLY && s.last)) {
        if (!STATE_ONLY && threadIdx.x == 0) partials[h * a.slots + slot] = 0.0;
        return;
    }
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, chunks = (s.count + TC - 1) / TC;
    const float g2 = log2_decay(a.log_decay[h]);
    const bool grows = HALF && g2 > 0.0f;
    const float query_part = HALF && !grows ? weight_scale(g2, 0) : SLOW;
    if (tid == 0) {
        mbar_init(&ctl.full, 33), mbar_init(&ctl.sg_full, 1), mbar_init(&ctl.done, 1), mbar_init(&ctl.drain, 1);
        mbar_init(&ctl.ready, ARITH), mbar_init(&ctl.read, ARITH), mbar_init(&ctl.meet, ARITH);
        ctl.dead = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == ARITH / 32) tmem_alloc(&ctl.tmem, 512);
    if (tid < 16) ctl.inner[tid] = exp2f(g2 * (float)(15 - tid));
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = ctl.tmem, base = smem_u32(smem);

    if (warp == ARITH / 32) {  // ------------------------------------------------------------------------------- loads and products
        constexpr uint32_t idesc0 = (1u << 4) | (type << 7) | (type << 10) | ((128u >> 4) << 24);
        constexpr uint32_t idesc_sg = idesc0 | ((128u >> 3) << 17);
        constexpr uint32_t idesc_u = idesc0 | ((uint32_t)(KB * 64 >> 3) << 17) | (1u << 15) | (1u << 16);
        constexpr uint32_t NEXT = BLOCK_BYTES;
        const int rows_seq = a.starts == nullptr ? s.seq : 0;
        unsigned bytes = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) bytes += maps.use[i] && !(STATE_ONLY && (i == 0 || i == 3)) ? (i < 2 ? KB : VB) * BLOCK_BYTES : 0;
        // sum over the tokens of A^T B: A (values on the lanes) as it lies in memory, B in parts
        const auto outer = [&](uint32_t col, uint32_t a_at) {
            const uint64_t at = tile_desc(base + a_at, VB == 2 ? NEXT : 0);
#pragma unroll 1
            for (int i = PARTS - 1; i >= 0; i--) {  // (small parts first: the tensor cores cut a sum's last bits off at every step)
                const uint64_t bt = tile_desc(base + L::SPARE + i * KB * BLOCK_BYTES, NEXT);
#pragma unroll
                for (int ks = 0; ks < TC / 16; ks++) mma_ss(tmem + col, at + ks * 128, bt + ks * 128, idesc_u, i < PARTS - 1 || ks > 0);
            }
        };
        const auto inner = [&](uint32_t col, uint32_t x, uint32_t y, int blocks) {
            const uint64_t xd = tile_desc(base + x, K_MAJOR_LBO), yd = tile_desc(base + y, K_MAJOR_LBO);
            for (int ks = 0; ks < blocks * 4; ks++) {
                const uint32_t at = ((ks >> 2) * BLOCK_BYTES + (ks & 3) * 32) >> 4;
                mma_ss(tmem + col, xd + at, yd + at, idesc_sg, ks > 0);
            }
        };
        constexpr int PHASES = STATE_ONLY ? 2 : 4;  // U, U', X, X'
        unsigned phase = 0;
        bool ok = true;
        int filled = 0;
        for (int it = 0; it < chunks && ok; it++) {
            const int tokens = min(TC, s.count - it * TC), row0 = chunk_row(a, s, it, tokens);
            if (lane == 0) mbar_expect_tx(&ctl.full, bytes);
            const auto fetch = [&](auto blocks, int i, const Operand &o, int at, int dim) {
                constexpr int BLOCKS = decltype(blocks)::value;
                if (maps.use[i]) {
                    const int head = maps.by_group[i] * (int)hg + maps.by_head[i] * (int)hi;
                    if (lane == 0)
                        for (int x = 0; x < BLOCKS; x++)
                            tma_load(smem + at + x * BLOCK_BYTES, maps.map[i], x * 64, head, row0, maps.by_seq[i] * rows_seq, &ctl.full);
                } else {
                    copy_tile<T, BLOCKS>(smem + at, o.at<const T>(rows_seq, hg, hi) + (int64_t)row0 * o.row, o.row, o.col, tokens, dim, lane);
                }
            };
            if (!STATE_ONLY) fetch(std::integral_constant<int, KB>(), 0, a.q, L::Q, a.dk);
            fetch(std::integral_constant<int, KB>(), 1, a.k, L::K, a.dk);
            fetch(std::integral_constant<int, VB>(), 2, a.v, L::V, a.dv);
            if (!STATE_ONLY) fetch(std::integral_constant<int, VB>(), 3, dout, L::D, a.dv);
            fence_async_smem();
            mbar_arrive(&ctl.full);
            filled++;
            ok = mbar_wait_warp(&ctl.full, it & 1, a.wait_polls) && (it == 0 || mbar_wait_warp(&ctl.read, (it - 1) & 1, a.wait_polls));
            if (!ok) break;
            tc_fence_after();
            if (lane == 0 && !STATE_ONLY) {
                inner(COL_S, L::Q, L::K, KB);
                inner(COL_G, L::D, L::V, VB);
                mma_commit(&ctl.sg_full);
            }
            __syncwarp();
            for (int i = 0; i < PHASES && ok; i++, phase++) {
                ok = mbar_wait_warp(&ctl.ready, phase & 1, a.wait_polls);
                if (!ok) break;
                tc_fence_after();
                if (lane == 0) {
                    outer(i == 0 ? COL_U : i == 1 ? COL_U1 : i == 2 ? COL_G : COL_S, i < 2 ? L::V : L::D);
                    mma_commit(&ctl.done);
                }
                __syncwarp();
                ok = mbar_wait_warp(&ctl.done, phase & 1, a.wait_polls);
            }
        }
        if (!ok) ctl.dead = 1;
        // no copy and no product may be in flight when the CTA ends
        if (filled > 0) mbar_wait_warp(&ctl.full, (filled - 1) & 1, TC_WAIT_POLLS);
        if (lane == 0) mma_commit(&ctl.drain);
        __syncwarp();
        mbar_wait_warp(&ctl.drain, 0, TC_WAIT_POLLS);
    } else {  // ---------------------------------------------------------------------------------------- arithmetic
        const int row = (warp & 3) * 32 + lane, part = warp >> 2, r0 = (warp & 3) * 32;
        const uint32_t lanes = tmem + ((uint32_t)(warp & 3) << 21);
        const bool state_row = row < VB * 64;
        const int64_t state = (int64_t)a.dk * a.dv;
        float *own = a.states + ((int64_t)s.adds * a.heads + h) * 2 * state;  // Z, then M (where sequences are cut)
        f32x2 z[NZ / 2], m[NZ / 2];
        {
            const float *from = nullptr, *from_m = nullptr;
            int64_t step = 0;
            float enter = 1.0f;
            if (!STATE_ONLY && row < a.dv) {
                if (s.first > 0) {
                    from = a.states + ((int64_t)s.start * a.heads + h) * 2 * state + row, from_m = from + state, step = a.dv;
                } else if (a.state_in.data != nullptr) {
                    from = from_m = a.state_in.at<const float>(s.seq, hg, hi) + row * a.state_in.col;
                    step = a.state_in.row, enter = exp2f(g2);
                }
            }
#pragma unroll
            for (int j = 0; j < NZ / 2; j++) {
                const int c = part * NZ + 2 * j;
                const bool one = from != nullptr && c < a.dk, two = from != nullptr && c + 1 < a.dk;
                z[j] = pack2(one ? from[c * step] * enter : 0.0f, two ? from[(c + 1) * step] * enter : 0.0f);
                m[j] = pack2(one ? from_m[c * step] * enter : 0.0f, two ? from_m[(c + 1) * step] * enter : 0.0f);
            }
        }
        double total = 0.0;
        unsigned phase = 0;
        bool ok = true;
        for (int it = 0; it < chunks; it++) {
            const int tokens = min(TC, s.count - it * TC);
            const int e = s.first + it * TC + tokens == s.length ? tokens - 1 : tokens;
            const int last = tokens - 1;  // decays are relative to the chunk's last token, the step beyond it is taken in fp32
            ok = mbar_wait_warp(&ctl.full, it & 1, a.wait_polls);
            if (!STATE_ONLY) ok = ok && mbar_wait_warp(&ctl.sg_full, it & 1, a.wait_polls);
            if (!ok) break;
            tc_fence_after();
            if (tokens < TC)  // rows behind the chunk may be another sequence's: not even 0 * inf may come in
                for (int p = tid; p < (STATE_ONLY ? 1 : 2) * VB * TC * 8; p += ARITH)
                    if (((p >> 3) & (TC - 1)) >= tokens) *reinterpret_cast<uint4 *>(smem + L::V + p * 16) = make_uint4(0, 0, 0, 0);
            // fp16: K~, K', Q~ and Q' are scaled by the chunk's largest key and query: values below fp16's normal range would leave
            // their low parts no bits
            const auto up = [&](int which) {
                if constexpr (!HALF) return 1.0f;
                static_assert(ARITH / 32 == 16, "two loads");
                const uint4 *m = reinterpret_cast<const uint4 *>(ctl.largest[it & 1][which]);
                return fp16_scale_of_bits(fp16_larger(fp16_largest(fp16_largest(0, m[0]), m[1])));
            };
            if (HALF) {
#pragma unroll
                for (int which = 0; which < (STATE_ONLY ? 1 : 2); which++) {
                    uint32_t m = 0;
                    for (int p = tid; p < KB * TC * 8; p += ARITH)
                        if (((p >> 3) & (TC - 1)) < tokens) m = fp16_largest(m, *reinterpret_cast<const uint4 *>(smem + (which ? L::Q : L::K) + p * 16));
                    m = __reduce_max_sync(0xffffffffu, fp16_larger(m));
                    if (lane == 0) ctl.largest[it & 1][which][warp] = (uint16_t)m;
                }
                mbar_arrive(&ctl.meet);
                ok = mbar_wait_warp(&ctl.meet, it & 1, a.wait_polls);
                if (!ok) break;
            }
            // an operand times `weight` of its token, in parts
            const auto parts = [&](int tile, auto weight) {
                const float f = up(tile == L::Q);
#pragma unroll 2
                for (int p = tid; p < KB * TC * 8; p += ARITH) {
                    const int t = (p >> 3) & (TC - 1);
                    uint4 x = *reinterpret_cast<const uint4 *>(smem + tile + p * 16);
                    if (t >= tokens) x = make_uint4(0, 0, 0, 0);
                    write_parts<T, PARTS>(x, HALF ? weight(t) * f : weight(t), smem + L::SPARE + p * 16, KB * BLOCK_BYTES);
                }
                fence_async_smem();
                mbar_arrive(&ctl.ready);
            };
            // (what grows in fp16 is taken relative to the largest, and the rest in fp32)
            const auto before_last = [&](int t) { return exp2f(g2 * (float)(max(last - t, 0) - (grows ? last : 0))); };
            const auto behind_first = [&](int t) { return exp2f(g2 * (float)(grows ? t - last : t)); };
            parts(L::K, before_last);
            // (under the products U)
            f32x2 sum = splat2(0.0f);
            if (!STATE_ONLY) {
#pragma unroll 1
                for (int c0 = part * 16; c0 <= r0 + 31; c0 += 64) {
                    uint32_t x[16], y[16];
                    tmem_ld16_nowait(lanes + COL_S + c0, x);
                    tmem_ld16_nowait(lanes + COL_G + c0, y);
                    const int d = row - c0;
                    const bool diagonal = c0 + 31 >= r0 + 16;  // (blocks of 16 columns that reach the diagonal of the warp's rows)
                    const f32x2 outer = splat2(exp2f(g2 * (float)max(d - 15, 0)));
                    tmem_ld_wait16(x);
                    tmem_ld_wait16(y);
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        const f32x2 dist = sub2(splat2((float)d), pack2((float)(2 * j), (float)(2 * j + 1)));
                        f32x2 w;
                        if (diagonal) {
                            w = ex2_approx2(mul2(splat2(g2), dist));
                        } else {
                            const float2 inside = *reinterpret_cast<const float2 *>(&ctl.inner[2 * j]);
                            w = mul2(outer, pack2(inside.x, inside.y));
                        }
                        f32x2 v = mul2(mul2(dist, w), mul2(pack2(__uint_as_float(x[2 * j]), __uint_as_float(x[2 * j + 1])),
                                                           pack2(__uint_as_float(y[2 * j]), __uint_as_float(y[2 * j + 1]))));
                        if (diagonal || tokens < TC) {  // what is behind the diagonal or the last token may be anything
                            float u0, u1;
                            unpack2(v, u0, u1);
                            v = pack2(2 * j < d && row < tokens ? u0 : 0.0f, 2 * j + 1 < d && row < tokens ? u1 : 0.0f);
                        }
                        sum = add2(sum, v);
                    }
                }
            }
            tc_fence_before();  // (S and G have been read before X goes over them)
            ok = mbar_wait_warp(&ctl.done, phase++ & 1, a.wait_polls);
            if (!ok) break;
            const float key_part = HALF && !grows ? weight_scale(g2, e - last) : SLOW;
            parts(L::K, [&](int t) { return before_last(t) * ((float)max(e - t, 0) * key_part); });
            ok = mbar_wait_warp(&ctl.done, phase++ & 1, a.wait_polls);
            if (!ok) break;
            if (!STATE_ONLY) {
                parts(L::Q, behind_first);
                ok = mbar_wait_warp(&ctl.done, phase++ & 1, a.wait_polls);
                if (!ok) break;
                parts(L::Q, [&](int t) { return behind_first(t) * ((float)t * query_part); });
                ok = mbar_wait_warp(&ctl.done, phase++ & 1, a.wait_polls);
                if (!ok) break;
            }
            tc_fence_after();
            const f32x2 carry = splat2(exp2f(g2 * (float)e)), steps = splat2((float)e), whole = splat2(1.0f / key_part);
            const float step = exp2f(g2 * (float)(grows ? e : e - last));
            const f32x2 beyond = splat2(HALF ? step / up(0) : step);
            const f32x2 back = splat2(HALF && !STATE_ONLY ? (grows ? exp2f(g2 * (float)last) : 1.0f) / up(1) : 1.0f);  // of X and X'
#pragma unroll
            for (int c = 0; c < NZ; c += 8) {
                uint32_t x[8], x1[8], u[8], u1[8];
                if (!STATE_ONLY) {
                    tmem_ld8_nowait(lanes + COL_G + part * NZ + c, x);
                    tmem_ld8_nowait(lanes + COL_S + part * NZ + c, x1);
                }
                tmem_ld8_nowait(lanes + COL_U + part * NZ + c, u);
                tmem_ld8_nowait(lanes + COL_U1 + part * NZ + c, u1);
                if (!STATE_ONLY) tmem_ld_wait8x2(x, x1);
                tmem_ld_wait8x2(u, u1);
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    f32x2 &zz = z[c / 2 + j], &mm = m[c / 2 + j];
                    const auto pair = [](const uint32_t &p, const uint32_t &q) { return pack2(__uint_as_float(p), __uint_as_float(q)); };
                    if (!STATE_ONLY && state_row) {  // (VB = 1: the other lanes repeat these)
                        const f32x2 p = pair(x[2 * j], x[2 * j + 1]), p1 = mul2(splat2(1.0f / query_part), pair(x1[2 * j], x1[2 * j + 1]));
                        sum = fma2(HALF ? mul2(back, p) : p, mm, sum);
                        sum = fma2(HALF ? mul2(back, p1) : p1, zz, sum);
                    }
                    mm = fma2(carry, fma2(steps, zz, mm), mul2(beyond, mul2(whole, pair(u1[2 * j], u1[2 * j + 1]))));
                    zz = fma2(carry, zz, mul2(beyond, pair(u[2 * j], u[2 * j + 1])));
                }
                // (done with these registers before the next loads)
#pragma unroll
                for (int j = 0; j < 4; j++) asm volatile("" : "+l"(z[c / 2 + j]), "+l"(m[c / 2 + j]));
            }
            tc_fence_before();
            mbar_arrive(&ctl.read);
            float u, v;
            unpack2(sum, u, v);
            total += (double)(u + v);
        }
        total *= (double)a.scale_out;
        if (!STATE_ONLY && dstate.data != nullptr && s.last && s.length > 0 && row < a.dv) {
            const float *from = dstate.at<const float>(s.seq, hg, hi) + row * dstate.col;
#pragma unroll
            for (int j = 0; j < NZ / 2; j++) {
                float u, v;
                unpack2(m[j], u, v);
                const int c = part * NZ + 2 * j;
                if (c < a.dk) total += (double)u * (double)from[c * dstate.row];
                if (c + 1 < a.dk) total += (double)v * (double)from[(c + 1) * dstate.row];
            }
        }
        if (STATE_ONLY && row < a.dv) {
#pragma unroll
            for (int j = 0; j < NZ / 2; j++) {
                float u, v, u1, v1;
                unpack2(z[j], u, v), unpack2(m[j], u1, v1);
                const int c = part * NZ + 2 * j;
                if (c < a.dk) own[c * a.dv + row] = u, own[state + c * a.dv + row] = u1;
                if (c + 1 < a.dk) own[(c + 1) * a.dv + row] = v, own[state + (c + 1) * a.dv + row] = v1;
            }
        }
        if (!ok) {  // gave up: say so, and leave nothing that looks like a result
            ctl.dead = 1;
            total = __longlong_as_double(0x7ff8000000000000LL);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
        if (lane == 0) ctl.sums[warp] = total;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == ARITH / 32) tmem_free(tmem, 512);
    if (tid == 0) {
        double v = 0.0;
        for (int w = 0; w < ARITH / 32; w++) v += ctl.sums[w];
        if (!STATE_ONLY) partials[h * a.slots + slot] = v;
        if (ctl.dead != 0 && a.gave_up != nullptr) {
            *reinterpret_cast<volatile int *>(a.gave_up) = GAVE_UP_DECAY;
            __threadfence_system();
        }
    }
}

template <typename T, int KB, int VB, bool STATE_ONLY>
static int launch_grad(const DecayArgs &a, const Operand &dout, const Operand &dstate, double *partials, cudaStream_t s) {
    auto kernel = decay_grad_tc_kernel<T, KB, VB, STATE_ONLY>;
    constexpr int bytes = GradSmem<KB, VB>::BYTES;
    const cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (err != cudaSuccess) return cuda_fail(err, "decay_grad_tc_kernel");
    GradMaps maps = {};
    const Operand *operands[4] = {&a.q, &a.k, &a.v, &dout};
    constexpr CUtensorMapDataType type = std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    for (int i = STATE_ONLY ? 1 : 0; i < (STATE_ONLY ? 3 : 4); i++)
        maps.use[i] = make_decay_map(&maps.map[i], a, *operands[i], i < 2 ? a.dk : a.dv, type, 2, 64, TC, &maps.by_group[i], &maps.by_head[i],
                                     &maps.by_seq[i]);
    kernel<<<(unsigned)(a.slots * a.heads), GRAD_THREADS, bytes, s>>>(a, dout, dstate, maps, partials);
    KM_CHECK_LAUNCH("decay_grad_tc_kernel launch");
    return KM_OK;
}

template <typename T, bool STATE_ONLY>
static int launch_grad_dims(const DecayArgs &a, const Operand &dout, const Operand &dstate, double *partials, cudaStream_t s) {
    if (a.dk <= 64)
        return a.dv <= 64 ? launch_grad<T, 1, 1, STATE_ONLY>(a, dout, dstate, partials, s) : launch_grad<T, 1, 2, STATE_ONLY>(a, dout, dstate, partials, s);
    return a.dv <= 64 ? launch_grad<T, 2, 1, STATE_ONLY>(a, dout, dstate, partials, s) : launch_grad<T, 2, 2, STATE_ONLY>(a, dout, dstate, partials, s);
}

int launch_decay_grad_tc(const km_decay_problem &p, const DecayArgs &a, const Operand &dout, const Operand &dstate, double *partials,
                         bool state_only, cudaStream_t s) {
    if (p.dtype == KM_TYPE_BF16)
        return state_only ? launch_grad_dims<__nv_bfloat16, true>(a, dout, dstate, partials, s)
                          : launch_grad_dims<__nv_bfloat16, false>(a, dout, dstate, partials, s);
    return state_only ? launch_grad_dims<__half, true>(a, dout, dstate, partials, s) : launch_grad_dims<__half, false>(a, dout, dstate, partials, s);
}

}  // namespace km
