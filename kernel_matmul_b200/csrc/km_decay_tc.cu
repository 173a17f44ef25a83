// Linear attention with a decay for each head on the tensor cores (km_decay.cuh has the method): 16-bit operands, chunks of
// 128 tokens, one CTA per (segment, head) that goes through its chunks with the state in registers.  Per chunk, with M = 128
// and fp32 accumulators in tensor memory (128 lanes):
//   S  = Q K^T            operands as they are in memory; lanes are tokens t
//   QZ = Q Z              Z: the state in 16 bits (below), dv x dk in shared memory
//   PV = P V              P = S with decays and mask, in 16 bits, from tensor memory
//   U  = V^T K~           K~ = K with decays e^{g (e - s)}, in two 16-bit parts; lanes are columns of v
//   out = PV + e^{g t} QZ,  Z <- e^{g e} Z + U     in fp32
// The tiles of Q, K and V have ONE layout, rows of 64 values (128 bytes, 128-byte swizzle), which the matrix unit takes either
// along the values (Q, K in S) or along the tokens (V in PV, V and K~ in U): nothing is transposed.
//
// Roundings to 16 bits: P and the state's copy in QZ, each once per term, half a step of the operands' type: as large as the
// rounding of the result.  Z itself and U stay in fp32; K~ = hi + lo (2^-17 relative in bf16), since its sum is the state, an fp32
// result.  fp16 has too few exponents for P and Z: both are scaled by powers of two per row, taken back in fp32.
//
// Bound by memory: a chunk of a head with dk = dv = 128 moves 128 KB and takes five products of 128^3 (1300 cycles of the tensor
// pipe), while its share of HBM takes 5600 cycles.  So everything is about keeping loads in flight: two stages of Q, K, V (96 KB
// each), each filled by a warp of its own through cp.async, which takes any row stride and zero-fills the rows behind
// the last token; K~ goes over K and Q once S and QZ have read them, P over S.
#include <type_traits>

#include "km_decay.cuh"

namespace km {

namespace {

constexpr int TC = 128;            // tokens of a chunk
constexpr int COMPUTE = 256;       // threads: two per lane of tensor memory
constexpr int LOADERS = 32;        // threads per stage
constexpr int THREADS = COMPUTE + 32 + 2 * LOADERS;
constexpr int BLOCK_BYTES = TC * 128;  // 128 rows of 64 values

template <int KB, int VB>
struct Smem {
    static constexpr int Q = 0, K = KB * BLOCK_BYTES, V = 2 * KB * BLOCK_BYTES, STAGE = (2 * KB + VB) * BLOCK_BYTES;
    static constexpr int Z = 2 * STAGE;                       // KB blocks of (64 VB rows of 64 values)
    static constexpr int REST = Z + KB * VB * 64 * 128;
    static constexpr int BYTES = 1024 + REST;
};

struct Control {
    uint64_t full[2], empty[2], s_full, qz_full, p_ready, o_full, z_ready, drain, meet;
    uint32_t tmem;
    int dead;
    __nv_bfloat16 z_scale[2][128];  // fp16: power of two that takes the scaling of Z's row back, by parity of the chunk
    float row_max[2][TC];           // fp16: largest of a row in each half
};

// tensor memory columns
constexpr uint32_t COL_S = 0, COL_PV = 128, COL_QZ = 256, COL_U = 384;

// Operand tiles, 128-byte swizzle (layout type 2).  Along the values (K-major): groups of 8 rows 1024 bytes apart.  Along the
// tokens (MN-major): `lbo` bytes to the next 64 values, 1024 to the next 8 tokens.
__device__ __forceinline__ uint64_t tile_desc(uint32_t addr, uint32_t lbo) {
    return smem_desc(addr, lbo, 1024) | (2ull << 61);
}
constexpr uint32_t K_MAJOR_LBO = 16;

// D (+)= A B, both operands in shared memory
__device__ __forceinline__ void mma_ss(uint32_t d_tmem, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t"
        ".reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %5, %5, %5}, p;\n\t"
        "}"
        :
        : "r"(d_tmem), "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(0u)
        : "memory");
}

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, "
        "%18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
          "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
          "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr)
        : "memory");
}
// The wait for the loads into `r`, tied to its registers (km_tcgen05.cuh, tmem_ld_wait16).
__device__ __forceinline__ void tmem_ld_wait32(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
                   "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]),
                   "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]),
                   "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
                 :
                 : "memory");
}

// two values as one word, the first in the low half, rounded to nearest
template <typename T>
__device__ __forceinline__ uint32_t pack(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return reinterpret_cast<const uint32_t &>(v);
}
template <>
__device__ __forceinline__ uint32_t pack<__half>(float a, float b) {
    const __half2 v = __floats2half2_rn(a, b);
    return reinterpret_cast<const uint32_t &>(v);
}
template <typename T>
__device__ __forceinline__ float2 unpack(uint32_t w);
template <>
__device__ __forceinline__ float2 unpack<__nv_bfloat16>(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 unpack<__half>(uint32_t w) {
    return __half22float2(reinterpret_cast<const __half2 &>(w));
}

// 2^n that brings a largest magnitude m to [2^13, 2^14) (fp16's range and as many of its small values as possible); 1 for 0 and
// for what is not finite
__device__ __forceinline__ float fp16_scale(float m) {
    const int e = (int)((__float_as_uint(m) >> 23) & 0xffu);
    if (e == 0 || e == 255) return 1.0f;
    return __uint_as_float((uint32_t)min(max(127 + 13 - (e - 127), 2), 252) << 23);  // (its inverse is a normal number too)
}

// One operand's rows into the stage, by the threads of the stage.
template <typename T, int BLOCKS>
__device__ __forceinline__ void load_tile(unsigned char *tile, const DecayArgs &a, const Segment &s, const Operand &o, int64_t hg,
                                          int64_t hi, int64_t first, int tokens, int dim, bool aligned, int tid) {
    constexpr int PIECES = BLOCKS * 8;  // of 16 bytes, in a row
    const T *src = o.at<const T>(a.starts == nullptr ? s.seq : 0, hg, hi);
    const int c = tid % PIECES, left = min(max(dim - c * 8, 0), 8);
    unsigned char *to = tile + (c >> 3) * BLOCK_BYTES;
    const int64_t step = (a.reverse ? -1 : 1) * o.row;
    const T *p = src + token_row(a, s, first) * o.row + (int64_t)c * 8 * o.col;
    for (int row = tid / PIECES; row < TC; row += LOADERS / PIECES) {
        unsigned char *dst = to + row * 128 + (((c & 7) ^ (row & 7)) << 4);
        const bool here = row < tokens && left > 0;
        const T *from = here ? p + row * step : src;
        if (aligned) {
            const unsigned bytes = here ? left * 2u : 0u;
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(from), "r"(bytes) : "memory");
        } else {
            union {
                T v[8];
                uint4 w;
            } x;
            x.w = make_uint4(0, 0, 0, 0);
            if (here)
                for (int j = 0; j < left; j++) x.v[j] = from[j * o.col];
            *reinterpret_cast<uint4 *>(dst) = x.w;
        }
    }
}

// Whether every row starts on a boundary of 16 bytes.
__device__ __forceinline__ bool rows_aligned(const Operand &o, int size) {
    return o.col == 1 && ((reinterpret_cast<uintptr_t>(o.data) | (uintptr_t)((o.seq | o.group | o.head | o.row) * size)) & 15) == 0;
}

}  // namespace

template <typename T, typename O, int KB, int VB, bool STATE_ONLY>
__global__ void __launch_bounds__(THREADS, 1) decay_tc_kernel(DecayArgs a) {
    using L = Smem<KB, VB>;
    constexpr bool HALF = std::is_same<T, __half>::value;
    constexpr int NZ = KB * 32;  // of the state's row: this thread's columns
    constexpr int NO = VB * 32;  // of a result's row
    extern __shared__ unsigned char raw[];
    unsigned char *smem = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
    Control &ctl = *reinterpret_cast<Control *>(smem + L::REST);

    const int64_t h = blockIdx.x % a.heads, slot = blockIdx.x / a.heads;
    const int64_t hg = h / a.group, hi = h - hg * a.group;
    const Segment s = find_segment(a, slot);
    if (!STATE_ONLY && s.spare >= 0) clear_spare_rows<O>(a, s, hg, hi);
    if (!s.used || (STATE_ONLY && s.last)) return;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int chunks = (int)((s.count + TC - 1) / TC);

    if (tid == 0) {
        for (int b = 0; b < 2; b++) {
            mbar_init(&ctl.full[b], LOADERS);
            mbar_init(&ctl.empty[b], 1);
        }
        mbar_init(&ctl.s_full, 1), mbar_init(&ctl.qz_full, 1), mbar_init(&ctl.o_full, 1), mbar_init(&ctl.drain, 1);
        mbar_init(&ctl.p_ready, COMPUTE), mbar_init(&ctl.z_ready, COMPUTE), mbar_init(&ctl.meet, COMPUTE);
        ctl.dead = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == COMPUTE / 32) tmem_alloc(&ctl.tmem, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = ctl.tmem;
    const uint32_t base = smem_u32(smem);
    const float g2 = log2_decay(a.log_decay[h]);

    if (warp > COMPUTE / 32) {  // ---------------------------------------------------------------- loads
        const int ltid = tid - COMPUTE - 32, b = ltid / LOADERS, mine = ltid % LOADERS;
        unsigned char *stage = smem + b * L::STAGE;
        const bool aq = rows_aligned(a.q, 2), ak = rows_aligned(a.k, 2), av = rows_aligned(a.v, 2);
        for (int it = b; it < chunks; it += 2) {
            if (it >= 2 && !mbar_wait_warp(&ctl.empty[b], ((it >> 1) + 1) & 1, a.wait_polls)) break;
            const int64_t first = s.first + (int64_t)it * TC;
            const int tokens = (int)min((int64_t)TC, s.first + s.count - first);
            load_tile<T, KB>(stage + L::K, a, s, a.k, hg, hi, first, tokens, a.dk, ak, mine);
            if (!STATE_ONLY) load_tile<T, KB>(stage + L::Q, a, s, a.q, hg, hi, first, tokens, a.dk, aq, mine);
            load_tile<T, VB>(stage + L::V, a, s, a.v, hg, hi, first, tokens, a.dv, av, mine);
            asm volatile("cp.async.wait_all;" ::: "memory");
            fence_async_smem();
            mbar_arrive(&ctl.full[b]);
        }
    } else if (warp == COMPUTE / 32) {  // ------------------------------------------------------------- matrix products
        constexpr uint32_t type = HALF ? 0u : 1u;
        constexpr uint32_t idesc0 = (1u << 4) | (type << 7) | (type << 10) | ((128u >> 4) << 24);
        constexpr uint32_t idesc_s = idesc0 | ((128u >> 3) << 17);
        constexpr uint32_t idesc_qz = idesc0 | ((uint32_t)(VB * 64 >> 3) << 17);
        constexpr uint32_t idesc_pv = idesc_qz | (1u << 16);
        constexpr uint32_t idesc_u = idesc0 | ((uint32_t)(KB * 64 >> 3) << 17) | (1u << 15) | (1u << 16);
        bool ok = true;
        for (int it = 0; it < chunks && ok; it++) {
            const int b = it & 1;
            const uint32_t q = base + b * L::STAGE + L::Q, k = base + b * L::STAGE + L::K, v = base + b * L::STAGE + L::V, z = base + L::Z;
            if (!STATE_ONLY) {
                ok = mbar_wait_warp(&ctl.full[b], (it >> 1) & 1, a.wait_polls);
                if (!ok) break;
                tc_fence_after();
                if (lane == 0) {
                    for (int ks = 0; ks < KB * 4; ks++) {
                        const uint32_t at = (ks >> 2) * BLOCK_BYTES + (ks & 3) * 32;
                        mma_ss(tmem + COL_S, tile_desc(q + at, K_MAJOR_LBO), tile_desc(k + at, K_MAJOR_LBO), idesc_s, ks > 0);
                    }
                    mma_commit(&ctl.s_full);
                }
                __syncwarp();
                ok = mbar_wait_warp(&ctl.z_ready, it & 1, a.wait_polls);
                if (!ok) break;
                tc_fence_after();
                if (lane == 0) {
                    for (int ks = 0; ks < KB * 4; ks++)
                        mma_ss(tmem + COL_QZ, tile_desc(q + (ks >> 2) * BLOCK_BYTES + (ks & 3) * 32, K_MAJOR_LBO),
                               tile_desc(z + (ks >> 2) * (VB * 64 * 128) + (ks & 3) * 32, K_MAJOR_LBO), idesc_qz, ks > 0);
                    mma_commit(&ctl.qz_full);
                }
                __syncwarp();
            }
            ok = mbar_wait_warp(&ctl.p_ready, it & 1, a.wait_polls);
            if (!ok) break;
            tc_fence_after();
            if (lane == 0) {
                const uint32_t next = BLOCK_BYTES;  // bytes to the next 64 values
                for (int ks = 0; ks < TC / 16; ks++) {
                    const uint64_t vt = tile_desc(v + ks * 2048, VB == 2 ? next : 0);  // (VB = 1: lanes 64 .. 127 repeat 0 .. 63)
                    mma_ss(tmem + COL_U, vt, tile_desc(k + ks * 2048, next), idesc_u, ks > 0);
                    mma_ss(tmem + COL_U, vt, tile_desc(q + ks * 2048, next), idesc_u, 1u);
                }
                if (!STATE_ONLY)
                    for (int ks = 0; ks < TC / 16; ks++)
                        mma_f16_ts(tmem + COL_PV, tmem + COL_S + (ks >> 2) * 64 + (ks & 3) * 8, tile_desc(v + ks * 2048, next), idesc_pv, ks > 0);
                mma_commit(&ctl.o_full);
                mma_commit(&ctl.empty[b]);
            }
            __syncwarp();
            // S of the next chunk goes over P
            ok = mbar_wait_warp(&ctl.o_full, it & 1, a.wait_polls);
        }
        // nothing may be in flight when tensor memory is freed
        if (lane == 0) mma_commit(&ctl.drain);
        __syncwarp();
        mbar_wait_warp(&ctl.drain, 0, TC_WAIT_POLLS);
    } else {  // ---------------------------------------------------------------------------------- arithmetic
        const int row = (warp & 3) * 32 + lane, half = warp >> 2;  // lane of tensor memory, half of the columns
        const uint32_t lanes = tmem + ((uint32_t)(warp & 3) << 21);
        const bool state_row = row < VB * 64;
        float z[NZ];
        const bool first_segment = s.first == 0;
        const float *from = nullptr;
        int64_t step = 0;
        if (!STATE_ONLY && row < a.dv) {
            if (!first_segment) {
                from = a.states + (slot * a.heads + h) * (int64_t)a.dk * a.dv + row;
                step = a.dv;
            } else if (a.state_in.data != nullptr) {
                from = a.state_in.at<const float>(s.seq, hg, hi) + row * a.state_in.col;
                step = a.state_in.row;
            }
        }
        const float enter = first_segment && !a.reverse && s.length > 0 ? exp2f(g2) : 1.0f;
#pragma unroll
        for (int j = 0; j < NZ; j++) {
            const int c = half * NZ + j;
            z[j] = from != nullptr && c < a.dk ? from[c * step] * enter : 0.0f;
        }
        // all arithmetic threads meet (false: gave up)
        unsigned meetings = 0;
        const auto meet = [&]() {
            mbar_arrive(&ctl.meet);
            return mbar_wait_warp(&ctl.meet, meetings++ & 1, a.wait_polls);
        };
        // the state's copy in 16 bits for the products of chunk `it`
        const auto publish = [&](int it) {
            float f = 1.0f;
            if (HALF) {
                float m = 0.0f;
#pragma unroll
                for (int j = 0; j < NZ; j++) m = fmaxf(m, fabsf(z[j]));
                ctl.row_max[half][row] = m;
                if (!meet()) return false;
                f = fp16_scale(fmaxf(m, ctl.row_max[half ^ 1][row]));
                if (half == 0) ctl.z_scale[it & 1][row] = __float2bfloat16_rn(1.0f / f);
                if (!meet()) return false;
            }
            if (!state_row) return true;
#pragma unroll
            for (int c = 0; c < NZ / 8; c++) {
                const int chunk = half * (NZ / 8) + c;  // of 8 values, in the row
                unsigned char *at = smem + L::Z + (chunk >> 3) * (VB * 64 * 128) + row * 128 + (((chunk & 7) ^ (row & 7)) << 4);
                *reinterpret_cast<uint4 *>(at) =
                    make_uint4(pack<T>(z[8 * c] * f, z[8 * c + 1] * f), pack<T>(z[8 * c + 2] * f, z[8 * c + 3] * f),
                               pack<T>(z[8 * c + 4] * f, z[8 * c + 5] * f), pack<T>(z[8 * c + 6] * f, z[8 * c + 7] * f));
            }
            return true;
        };
        bool ok = true;
        if (!STATE_ONLY) {
            ok = publish(0);
            fence_async_smem();
            mbar_arrive(&ctl.z_ready);
        }
        const bool out_aligned = rows_aligned(a.out, sizeof(O));
        const float intra = a.scale_in * a.scale_out;
        int it = 0;
        for (; it < chunks && ok; it++) {
            const int b = it & 1;
            const int64_t first = s.first + (int64_t)it * TC;
            const int tokens = (int)min((int64_t)TC, s.first + s.count - first);
            const int e = first + tokens == s.length && !a.reverse ? tokens - 1 : tokens;
            ok = mbar_wait_warp(&ctl.full[b], (it >> 1) & 1, a.wait_polls);
            if (!ok) break;
            float p_scale = 1.0f;  // fp16: takes the scaling of P's row back
            if (!STATE_ONLY) {
                ok = mbar_wait_warp(&ctl.s_full, it & 1, a.wait_polls);
                if (!ok) break;
                tc_fence_after();
                float f = intra;
                if (HALF) {  // scaling from the largest of the row's products: decays only make them smaller
                    float m = 0.0f;
#pragma unroll
                    for (int cb = 0; cb < 2; cb++) {
                        if (half * 64 + cb * 32 > (warp & 3) * 32 + 31) continue;
                        uint32_t r[32];
                        tmem_ld32(lanes + COL_S + half * 64 + cb * 32, r);
                        tmem_ld_wait32(r);
#pragma unroll
                        for (int j = 0; j < 32; j++) m = fmaxf(m, half * 64 + cb * 32 + j <= row ? fabsf(__uint_as_float(r[j])) : 0.0f);
                    }
                    ctl.row_max[half][row] = m;
                    ok = meet();
                    if (!ok) break;
                    const float up = fp16_scale(fabsf(intra) * fmaxf(m, ctl.row_max[half ^ 1][row]));
                    f *= up;
                    p_scale = 1.0f / up;
                }
#pragma unroll
                for (int cb = 0; cb < 2; cb++) {
                    const int c0 = half * 64 + cb * 32;
                    uint32_t w[16];
                    if (c0 > (warp & 3) * 32 + 31) {  // all of it later than all of these rows
#pragma unroll
                        for (int j = 0; j < 16; j++) w[j] = 0;
                    } else {
                        uint32_t r[32];
                        tmem_ld32(lanes + COL_S + c0, r);
                        tmem_ld_wait32(r);
#pragma unroll
                        for (int j = 0; j < 16; j++) {
                            const int d = row - (c0 + 2 * j);
                            const float x = d >= 0 ? __uint_as_float(r[2 * j]) * (f * ex2_approx(g2 * (float)d)) : 0.0f;
                            const float y = d >= 1 ? __uint_as_float(r[2 * j + 1]) * (f * ex2_approx(g2 * (float)(d - 1))) : 0.0f;
                            w[j] = pack<T>(x, y);
                        }
                    }
                    // (columns 0 .. 31 and 64 .. 95 of S: inside what this thread alone has read)
                    tmem_st16(lanes + COL_S + half * 64 + cb * 16, w);
                }
                tmem_st_wait();
                tc_fence_before();
                ok = mbar_wait_warp(&ctl.qz_full, it & 1, a.wait_polls);
                if (!ok) break;
            }
            // K~ over K, its low part over Q
            unsigned char *kt = smem + b * L::STAGE + L::K, *qt = smem + b * L::STAGE + L::Q;
#pragma unroll 4
            for (int p = tid; p < KB * TC * 8; p += COMPUTE) {
                const int t = (p >> 3) & (TC - 1);
                const float w = exp2f(g2 * (float)(e - t));
                const uint4 x = *reinterpret_cast<const uint4 *>(kt + p * 16);
                const uint32_t in[4] = {x.x, x.y, x.z, x.w};
                uint32_t hi4[4], lo4[4];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    float2 v = unpack<T>(in[j]);
                    // (rows behind the last token are zero, whatever their weight)
                    v.x = t < tokens ? v.x * w : 0.0f, v.y = t < tokens ? v.y * w : 0.0f;
                    hi4[j] = pack<T>(v.x, v.y);
                    const float2 r = unpack<T>(hi4[j]);
                    lo4[j] = pack<T>(v.x - r.x, v.y - r.y);
                }
                *reinterpret_cast<uint4 *>(kt + p * 16) = make_uint4(hi4[0], hi4[1], hi4[2], hi4[3]);
                *reinterpret_cast<uint4 *>(qt + p * 16) = make_uint4(lo4[0], lo4[1], lo4[2], lo4[3]);
            }
            fence_async_smem();
            mbar_arrive(&ctl.p_ready);

            ok = mbar_wait_warp(&ctl.o_full, it & 1, a.wait_polls);
            if (!ok) break;
            tc_fence_after();
            const float carry = exp2f(g2 * (float)e);
#pragma unroll
            for (int cb = 0; cb < NZ / 32; cb++) {
                uint32_t r[32];
                tmem_ld32(lanes + COL_U + half * NZ + cb * 32, r);
                tmem_ld_wait32(r);
#pragma unroll
                for (int j = 0; j < 32; j++) z[cb * 32 + j] = fmaf(carry, z[cb * 32 + j], a.scale_in * __uint_as_float(r[j]));
            }
            if (!STATE_ONLY) {
                ok = publish(it + 1);
                if (!ok) break;
                fence_async_smem();
                const float f = exp2f(g2 * (float)row) * a.scale_out;
                uint32_t out[VB][16];
                O *to = a.out.at<O>(a.starts == nullptr ? s.seq : 0, hg, hi) + token_row(a, s, first + row) * a.out.row;
                const bool store = row < tokens;
#pragma unroll
                for (int cb = 0; cb < VB; cb++) {
                    const int c0 = half * NO + cb * 32;
                    uint32_t x[32], y[32];
                    tmem_ld32(lanes + COL_PV + c0, x);
                    tmem_ld32(lanes + COL_QZ + c0, y);
                    tmem_ld_wait32(x);
                    tmem_ld_wait32(y);
                    float o[32];
#pragma unroll
                    for (int j = 0; j < 32; j++) {
                        float q = f * __uint_as_float(y[j]);
                        if (HALF) q *= __bfloat162float(ctl.z_scale[it & 1][c0 + j]);
                        o[j] = fmaf(p_scale, __uint_as_float(x[j]), q);
                    }
                    if constexpr (sizeof(O) == 2) {
#pragma unroll
                        for (int j = 0; j < 16; j++) out[cb][j] = pack<T>(o[2 * j], o[2 * j + 1]);
                    } else if (store) {
#pragma unroll
                        for (int j = 0; j < 32; j += 4) {
                            if (out_aligned && c0 + j + 4 <= a.dv) {
                                *reinterpret_cast<float4 *>(to + c0 + j) = make_float4(o[j], o[j + 1], o[j + 2], o[j + 3]);
                            } else {
#pragma unroll
                                for (int i = 0; i < 4; i++)
                                    if (c0 + j + i < a.dv) to[(c0 + j + i) * a.out.col] = o[j + i];
                            }
                        }
                    }
                }
                tc_fence_before();
                mbar_arrive(&ctl.z_ready);
                if constexpr (sizeof(O) == 2) {
                    if (store) {
#pragma unroll
                        for (int cb = 0; cb < VB; cb++)
#pragma unroll
                            for (int j = 0; j < 4; j++) {
                                const int c = half * NO + cb * 32 + j * 8;
                                if (out_aligned && c + 8 <= a.dv) {
                                    *reinterpret_cast<uint4 *>(to + c) = make_uint4(out[cb][4 * j], out[cb][4 * j + 1], out[cb][4 * j + 2], out[cb][4 * j + 3]);
                                } else {
#pragma unroll
                                    for (int i = 0; i < 8; i++)
                                        if (c + i < a.dv) {
                                            const uint32_t w = out[cb][4 * j + i / 2];
                                            reinterpret_cast<unsigned short *>(to)[(c + i) * a.out.col] = (unsigned short)(i & 1 ? w >> 16 : w);
                                        }
                                }
                            }
                    }
                }
            } else {
                tc_fence_before();
            }
        }
        if (!ok) {  // gave up: say so, and leave nothing that looks like a result
            ctl.dead = 1;
#pragma unroll
            for (int j = 0; j < NZ; j++) z[j] = __int_as_float(0x7fc00000);
            if (!STATE_ONLY)
                for (int64_t i = s.first + (int64_t)it * TC + row; i < s.first + s.count; i += TC) {
                    O *to = a.out.at<O>(a.starts == nullptr ? s.seq : 0, hg, hi) + token_row(a, s, i) * a.out.row;
                    for (int c = half * NO; c < min((half + 1) * NO, a.dv); c++) to[c * a.out.col] = from_float<O>(__int_as_float(0x7fc00000));
                }
        }
        if (row < a.dv && (STATE_ONLY || (s.last && a.state_out.data != nullptr))) {
            float *to = STATE_ONLY ? a.states + (slot * a.heads + h) * (int64_t)a.dk * a.dv + row
                                   : a.state_out.at<float>(s.seq, hg, hi) + row * a.state_out.col;
            const int64_t row_step = STATE_ONLY ? a.dv : a.state_out.row;
#pragma unroll
            for (int j = 0; j < NZ; j++)
                if (half * NZ + j < a.dk) to[(half * NZ + j) * row_step] = z[j];
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == COMPUTE / 32) tmem_free(tmem, 512);
    if (tid == 0 && ctl.dead != 0 && a.gave_up != nullptr) {
        *reinterpret_cast<volatile int *>(a.gave_up) = GAVE_UP_DECAY;
        __threadfence_system();
    }
}

template <typename T, typename O, int KB, int VB, bool STATE_ONLY>
static int launch_one(const DecayArgs &a, cudaStream_t s) {
    auto kernel = decay_tc_kernel<T, O, KB, VB, STATE_ONLY>;
    constexpr int bytes = Smem<KB, VB>::BYTES + (int)sizeof(Control);
    static_assert(bytes <= 232448, "shared memory of an SM");
    const cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (err != cudaSuccess) return cuda_fail(err, "decay_tc_kernel");
    kernel<<<(unsigned)(a.slots * a.heads), THREADS, bytes, s>>>(a);
    KM_CHECK_LAUNCH("decay_tc_kernel launch");
    return KM_OK;
}

template <typename T, typename O, int KB, int VB>
static int launch_dims(const DecayArgs &a, bool state_only, cudaStream_t s) {
    // (states alone do not depend on the type of the result)
    return state_only ? launch_one<T, T, KB, VB, true>(a, s) : launch_one<T, O, KB, VB, false>(a, s);
}

template <typename T, typename O>
static int launch_types(const DecayArgs &a, bool state_only, cudaStream_t s) {
    if (a.dk <= 64) return a.dv <= 64 ? launch_dims<T, O, 1, 1>(a, state_only, s) : launch_dims<T, O, 1, 2>(a, state_only, s);
    return a.dv <= 64 ? launch_dims<T, O, 2, 1>(a, state_only, s) : launch_dims<T, O, 2, 2>(a, state_only, s);
}

int launch_decay_tc(const km_decay_problem &p, const DecayArgs &a, bool state_only, cudaStream_t s) {
    const bool wide = p.out_dtype == KM_TYPE_F32;
    if (p.dtype == KM_TYPE_BF16)
        return wide ? launch_types<__nv_bfloat16, float>(a, state_only, s) : launch_types<__nv_bfloat16, __nv_bfloat16>(a, state_only, s);
    return wide ? launch_types<__half, float>(a, state_only, s) : launch_types<__half, __half>(a, state_only, s);
}

}  // namespace km
