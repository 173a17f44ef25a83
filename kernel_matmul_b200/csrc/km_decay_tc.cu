// Linear attention with a decay for each head on the tensor cores (km_decay.cuh has the method): 16-bit operands, chunks of
// 128 tokens, one CTA per (segment, head) that goes through its chunks with the state in registers.  Per chunk, with M = 128
// and fp32 accumulators in tensor memory (128 lanes):
//   S  = Q K^T            operands as they are in memory; lanes are tokens t
//   QZ = Q Z              Z: the state in 16 bits (below), dv x dk in shared memory
//   U  = V^T K~           K~ = K with decays to the chunk's last token, in parts (below); lanes are columns of v
//   PV = P V              P = S with decays and mask, in two 16-bit parts, from tensor memory
//   out = PV + e^{g t} QZ,  Z <- e^{g e} Z + U     in fp32
// The tiles of Q, K and V have ONE layout, rows of 64 values (128 bytes, 128-byte swizzle), which the matrix unit takes either
// along the values (Q, K in S) or along the tokens (V in PV, V and K~ in U): nothing is transposed.
//
// Roundings to 16 bits.  The state's copy in QZ is rounded once, half a step of the operands' type (its low part has no room in
// shared memory): the only one, besides the result's own, and as large as that.  P goes in two parts (one part made results of
// short sequences 1.4 - 1.6 times as wrong as their rounding).  Z itself and U stay in fp32 and are fp32 results: K~ goes in two
// parts in fp16 (2^-22) and three in bf16 (2^-25; two, 2^-17, in the passes of a gradient that return no state).  The tensor cores cut the last bits of a sum off at every step of 16 tokens,
// so small parts are added up first: final states are within 1.5e-7 (2-norm, as an fp32 evaluation is) instead of 5e-7, and
// 2.4e-6 with two parts of bf16.  fp16 has too few exponents for P, Z and K~: they are scaled by powers of two, P and Z per row, K~ per
// chunk (its low part is then good to 2^-39 of the chunk's largest key; unscaled, to 2^-25: keys of 1e-3 made states 3e-5 wrong), taken back in
// fp32.
//
// What bounds it: a chunk of a head with dk = dv = 128 moves 128 KB, 5600 cycles of its SM's share of HBM, but 670 KB through
// shared memory (products of 128^3 with both operands there take 64 KB each), 5200 cycles at 128 bytes each, and its phases depend
// on one another: S, then P and K~, then the products with V, then the next state and QZ.  They take 8000 cycles, or 6400 with one part
// of P and two of K~ (148 heads x 4096 tokens: 158 and 129 us, 3.9 and 4.8 TB/s of operands).  Three kinds of warps work at once on
// neighbouring phases; two stages of Q, K, V are filled through TMA; K~ goes over K, Q and Z once the products have read them, P
// over S.  What did not help: S of the next chunk before U, results drained from registers while U runs, K~ made before S is there
// (all within 3 %: shared memory is what they wait for).
#include "km_decay_tc.cuh"

namespace km {

namespace {

constexpr int GROUP = 256;    // threads of a group: two per lane of tensor memory
// warps 0 - 7: results and state; 8 - 15: operands; 16: matrix products; 17, 18: loads; 19: none
constexpr int MMA_WARP = 16, THREADS = 640;
// Registers: 640 threads are launched with 96 each, 61 440 in all, which the groups divide: 256 x 144 + 256 x 64 + 128 x 64.
constexpr int RESULT_REGS = 144, OPERAND_REGS = 64, OTHER_REGS = 64;
static_assert(256 * RESULT_REGS + 256 * OPERAND_REGS + 128 * OTHER_REGS <= THREADS * 96, "registers at launch");

template <int KB, int VB>
struct Smem {
    // (the Q tile is also where the results leave through: 8 warps' 4 KB)
    static constexpr int Q = 0, K = 2 * BLOCK_BYTES, V = K + KB * BLOCK_BYTES, STAGE = V + VB * BLOCK_BYTES;
    // the state: KB blocks of (64 VB rows of 64 values); between its product with q and its next value a third part of K~
    static constexpr int Z = 2 * STAGE;
    static constexpr int REST = Z + KB * BLOCK_BYTES;
    static constexpr int BYTES = 1024 + REST;
};

struct Control {
    uint64_t full[2], empty[2], q_empty[2], s_full, qz_full, p_ready, o_full, z_ready, drain, meet[2];
    uint32_t tmem;
    int dead;
    float inner[16];                // decays 2^(g2 (15 - j)), reverse 2^(g2 j)
    __nv_bfloat16 p_scale[2][TC];   // fp16: power of two that takes the scaling of P's row back, by parity of the chunk
    __nv_bfloat16 z_scale[2][128];  // fp16: power of two that takes the scaling of Z's row back, by parity of the chunk
    uint8_t row_max[2][2][TC];      // fp16: exponent of a row's largest magnitude in each half, for either group
    uint16_t key_max[2][GROUP / 32];  // fp16: largest magnitude of the keys that a warp has seen, as its bits, by parity of the chunk
    float key_scale[2];             // fp16: power of two that takes the scaling of K~ back
};

// tensor memory columns
constexpr uint32_t COL_S = 0, COL_PV = 128, COL_QZ = 256, COL_U = 384;

// The swizzle of rows of PITCH bytes, 128 or 64, on an offset from a boundary of 1024 bytes.
template <int PITCH>
__device__ __forceinline__ int swizzled(int offset) {
    static_assert(PITCH == 128 || PITCH == 64, "a row is as wide as the swizzle");
    return offset ^ (((offset >> 7) & (PITCH / 16 - 1)) << 4);
}

// Tensor maps of q, k, v (boxes of 64 values x 128 tokens) and the result (up to 128 bytes x 32 tokens), and which operands have
// one; the coordinates of a head and a sequence in them.
struct Maps {
    CUtensorMap q, k, v, out;
    int use[4], by_group[4], by_head[4], by_seq[4];
};

__device__ __forceinline__ void tma_store(const CUtensorMap &map, int x, int head, int row, int seq, const unsigned char *src) {
    asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.tile.bulk_group [%0, {%1, %2, %3, %4}], [%5];" ::"l"(&map), "r"(x), "r"(head), "r"(row),
                 "r"(seq), "r"(smem_u32(src))
                 : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
// Shared memory that this thread's stores read may be written again.
__device__ __forceinline__ void tma_store_wait() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }

// NaN into columns [c0, c1) of rows [first, end), by a warp.
template <typename O>
__device__ __noinline__ void poison_rows(O *out, int64_t row, int64_t col, int first, int end, int c0, int c1) {
    for (int i = first + (threadIdx.x & 31); i < end; i += 32)
        for (int c = c0; c < c1; c++) out[i * row + c * col] = from_float<O>(__int_as_float(0x7fc00000));
}

}  // namespace

template <typename T, typename O, int KB, int VB, bool STATE_ONLY>
__global__ void __launch_bounds__(THREADS, 1) decay_tc_kernel(const __grid_constant__ DecayArgs a, const __grid_constant__ Maps maps) {
    using L = Smem<KB, VB>;
    constexpr bool HALF = std::is_same<T, __half>::value;
    constexpr int NZ = KB * 32;  // of the state's row: this thread's columns
    constexpr int NO = VB * 32;  // of a result's row
    extern __shared__ unsigned char raw[];
    unsigned char *smem = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
    Control &ctl = *reinterpret_cast<Control *>(smem + L::REST);

    const int64_t h = blockIdx.x % (unsigned)a.heads, slot = blockIdx.x / (unsigned)a.heads;
    const int64_t hg = h / a.group, hi = h - hg * a.group;
    const Segment s = find_segment(a, slot);
    if (!STATE_ONLY && s.spare >= 0) clear_spare_rows<O>(a, s, hg, hi);
    if (!s.used || (STATE_ONLY && s.last)) return;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int chunks = (s.count + TC - 1) / TC;

    if (tid == 0) {
        for (int b = 0; b < 2; b++) {
            mbar_init(&ctl.full[b], STATE_ONLY ? 33 : 34);  // the loading warp's lanes, and its byte counts
            mbar_init(&ctl.empty[b], 1);
            mbar_init(&ctl.q_empty[b], GROUP);
            mbar_init(&ctl.meet[b], GROUP);
        }
        mbar_init(&ctl.s_full, 1), mbar_init(&ctl.qz_full, 1), mbar_init(&ctl.o_full, 1), mbar_init(&ctl.drain, 1);
        mbar_init(&ctl.p_ready, GROUP), mbar_init(&ctl.z_ready, GROUP);
        ctl.dead = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    const float g2 = log2_decay(a.log_decay[h]);
    const bool grows = HALF && g2 > 0.0f;  // (bf16 has the exponents of fp32)
    if (warp == MMA_WARP) tmem_alloc(&ctl.tmem, 512);
    if (warp == MMA_WARP + 1 && lane < 16) ctl.inner[lane] = exp2f(g2 * (float)(a.reverse ? lane : 15 - lane));
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = ctl.tmem;
    const uint32_t base = smem_u32(smem);
    // this thread's lane of tensor memory and half of the columns (of the two groups of eight warps)
    const int row = (warp & 3) * 32 + lane, half = (warp >> 2) & 1;
    const uint32_t lanes = tmem + ((uint32_t)(warp & 3) << 21);
    const int group = warp >> 3;
    // all threads of a group meet (false: gave up)
    unsigned meetings = 0;
    const auto meet = [&]() {
        mbar_arrive(&ctl.meet[group]);
        return mbar_wait_warp(&ctl.meet[group], meetings++ & 1, a.wait_polls);
    };

    if (warp >= MMA_WARP) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(OTHER_REGS));
    }
    if (warp > MMA_WARP + 2) {
    } else if (warp > MMA_WARP) {  // ---------------------------------------------------------------- loads
        const int b = warp - MMA_WARP - 1;
        unsigned char *stage = smem + b * L::STAGE;
        const int seq = a.starts == nullptr ? s.seq : 0;
        const auto fetch = [&](auto blocks, int which, const CUtensorMap &map, const Operand &o, unsigned char *tile, int row0, int tokens, int dim) {
            constexpr int BLOCKS = decltype(blocks)::value;
            if (maps.use[which]) {
                const int head = maps.by_group[which] * (int)hg + maps.by_head[which] * (int)hi;
                if (lane == 0)
                    for (int x = 0; x < BLOCKS; x++) tma_load(tile + x * BLOCK_BYTES, map, x * 64, head, row0, maps.by_seq[which] * seq, &ctl.full[b]);
            } else {
                copy_tile<T, BLOCKS>(tile, o.at<const T>(seq, hg, hi) + (int64_t)row0 * o.row, o.row, o.col, tokens, dim, lane);
            }
        };
        using Keys = std::integral_constant<int, KB>;
        using Values = std::integral_constant<int, VB>;
        const unsigned kv_bytes = ((maps.use[1] ? KB : 0) + (maps.use[2] ? VB : 0)) * BLOCK_BYTES, q_bytes = (maps.use[0] ? KB : 0) * BLOCK_BYTES;
        int filled = 0;
        bool ok = true;
        for (int it = b; it < chunks && ok; it += 2, filled++) {
            ok = it < 2 || mbar_wait_warp(&ctl.empty[b], ((it >> 1) + 1) & 1, a.wait_polls);
            if (!ok) break;
            const int tokens = min(TC, s.count - it * TC), row0 = chunk_row(a, s, it, tokens);
            if (lane == 0) mbar_expect_tx(&ctl.full[b], kv_bytes);
            fetch(Keys(), 1, maps.k, a.k, stage + L::K, row0, tokens, a.dk);
            fetch(Values(), 2, maps.v, a.v, stage + L::V, row0, tokens, a.dv);
            if (!STATE_ONLY) {
                ok = it < 2 || mbar_wait_warp(&ctl.q_empty[b], ((it >> 1) + 1) & 1, a.wait_polls);
                if (!ok) *reinterpret_cast<volatile int *>(&ctl.dead) = 1;  // (before the others can see this stage as full)
                if (lane == 0) mbar_expect_tx(&ctl.full[b], ok ? q_bytes : 0u);
                if (ok) fetch(Keys(), 0, maps.q, a.q, stage + L::Q, row0, tokens, a.dk);
            }
            fence_async_smem();
            mbar_arrive(&ctl.full[b]);
        }
        // no copy may be in flight when the CTA ends
        if (filled > 0) mbar_wait_warp(&ctl.full[b], (filled - 1) & 1, TC_WAIT_POLLS);
    } else if (warp == MMA_WARP) {  // ------------------------------------------------------------- matrix products
        constexpr uint32_t type = HALF ? 0u : 1u;
        constexpr uint32_t idesc0 = (1u << 4) | (type << 7) | (type << 10) | ((128u >> 4) << 24);
        constexpr uint32_t idesc_s = idesc0 | ((128u >> 3) << 17);
        constexpr uint32_t idesc_qz = idesc0 | ((uint32_t)(VB * 64 >> 3) << 17);
        constexpr uint32_t idesc_pv = idesc_qz | (1u << 16);
        constexpr uint32_t idesc_u = idesc0 | ((uint32_t)(KB * 64 >> 3) << 17) | (1u << 15) | (1u << 16);
        bool ok = true;
        for (int it = 0; it < chunks && ok; it++) {
            const int b = it & 1;
            // (an offset of n bytes inside a tile is n >> 4 in its descriptor)
            const uint64_t qd = tile_desc(base + b * L::STAGE + L::Q, K_MAJOR_LBO), kd = tile_desc(base + b * L::STAGE + L::K, K_MAJOR_LBO);
            if (!STATE_ONLY) {
                ok = mbar_wait_warp(&ctl.full[b], (it >> 1) & 1, a.wait_polls);
                if (!ok) break;
                tc_fence_after();
                if (lane == 0) {
#pragma unroll
                    for (int ks = 0; ks < KB * 4; ks++) {
                        const uint32_t at = ((ks >> 2) * BLOCK_BYTES + (ks & 3) * 32) >> 4;
                        mma_ss(tmem + COL_S, qd + at, kd + at, idesc_s, ks > 0);
                    }
                    mma_commit(&ctl.s_full);
                }
                __syncwarp();
                ok = mbar_wait_warp(&ctl.z_ready, it & 1, a.wait_polls);
                if (!ok) break;
                tc_fence_after();
                if (lane == 0) {
                    const uint64_t zd = tile_desc(base + L::Z, K_MAJOR_LBO);
#pragma unroll
                    for (int ks = 0; ks < KB * 4; ks++)
                        mma_ss(tmem + COL_QZ, qd + (((ks >> 2) * BLOCK_BYTES + (ks & 3) * 32) >> 4),
                               zd + (((ks >> 2) * (VB * 64 * 128) + (ks & 3) * 32) >> 4), idesc_qz, ks > 0);
                    mma_commit(&ctl.qz_full);
                }
                __syncwarp();
            }
            ok = mbar_wait_warp(&ctl.p_ready, it & 1, a.wait_polls);
            // (states alone: U of the chunk before has been read)
            if (ok && STATE_ONLY && it > 0) ok = mbar_wait_warp(&ctl.z_ready, (it - 1) & 1, a.wait_polls);
            if (!ok) break;
            tc_fence_after();
            if (lane == 0) {
                // along the tokens: 16 of them are 2048 bytes
                const uint64_t vd = tile_desc(base + b * L::STAGE + L::V, BLOCK_BYTES);
                const uint64_t vt = tile_desc(base + b * L::STAGE + L::V, VB == 2 ? BLOCK_BYTES : 0);  // (VB = 1: lanes 64 .. 127 repeat 0 .. 63)
                const uint64_t kt = tile_desc(base + b * L::STAGE + L::K, BLOCK_BYTES), lt = tile_desc(base + b * L::STAGE + L::Q, BLOCK_BYTES);
                // (the tensor cores cut a sum's last bits off at every step: small parts first, so that most steps have little to lose)
                bool begun = false;
                if (!HALF && a.parts == 3) {
                    const uint64_t zt = tile_desc(base + L::Z, BLOCK_BYTES);
#pragma unroll
                    for (int ks = 0; ks < TC / 16; ks++) mma_ss(tmem + COL_U, vt + ks * 128, zt + ks * 128, idesc_u, ks > 0);
                    begun = true;
                }
#pragma unroll
                for (int ks = 0; ks < TC / 16; ks++) mma_ss(tmem + COL_U, vt + ks * 128, lt + ks * 128, idesc_u, begun || ks > 0);
#pragma unroll
                for (int ks = 0; ks < TC / 16; ks++) mma_ss(tmem + COL_U, vt + ks * 128, kt + ks * 128, idesc_u, 1u);
                if (!STATE_ONLY) {
#pragma unroll
                    for (int i = 8; i >= 0; i -= 8)  // P's low part, then its high part
#pragma unroll
                        for (int ks = 0; ks < TC / 16; ks++)
                            mma_f16_ts(tmem + COL_PV, tmem + COL_S + ks * 16 + i, vd + ks * 128, idesc_pv, i == 0 || ks > 0);
                }
                mma_commit(&ctl.o_full);
                mma_commit(&ctl.empty[b]);
            }
            __syncwarp();
            // S of the next chunk goes over P
            if (!STATE_ONLY) ok = mbar_wait_warp(&ctl.o_full, it & 1, a.wait_polls);
        }
        // nothing may be in flight when tensor memory is freed
        if (lane == 0) mma_commit(&ctl.drain);
        __syncwarp();
        mbar_wait_warp(&ctl.drain, 0, TC_WAIT_POLLS);
    } else if (group == 1) {  // ------------------------------------------------------------------------ operands: P and K~
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(OPERAND_REGS));
        const int mine = tid - GROUP, r0 = (warp & 3) * 32;  // (first of the warp's rows)
        bool ok = true;
        for (int it = 0; it < chunks; it++) {
            const int b = it & 1, tokens = min(TC, s.count - it * TC);
            ok = mbar_wait_warp(&ctl.full[b], (it >> 1) & 1, a.wait_polls);
            if (!ok) break;
            if (tokens < TC) {  // what lies behind the chunk may be another sequence's: not even 0 * inf may come in
                unsigned char *vt = smem + b * L::STAGE + L::V;
                for (int p = mine; p < VB * TC * 8; p += GROUP)
                    if (((p >> 3) & (TC - 1)) >= tokens) *reinterpret_cast<uint4 *>(vt + p * 16) = make_uint4(0, 0, 0, 0);
            }
            float key_up = 1.0f;
            // K~ is scaled by the chunk's largest key: values below fp16's normal range would leave their low parts no bits
            if (HALF) {
                const unsigned char *kt = smem + b * L::STAGE + L::K + mine * 16;
                uint32_t largest = 0;
#pragma unroll
                for (int i = 0; i < KB * 4; i++) {
                    const uint4 x = *reinterpret_cast<const uint4 *>(kt + i * (GROUP * 16));
                    if ((mine >> 3) + 32 * (i & 3) < tokens) largest = fp16_largest(largest, x);
                }
                const uint32_t top = __reduce_max_sync(0xffffffffu, fp16_larger(largest));
                if (lane == 0) ctl.key_max[it & 1][warp & 7] = (uint16_t)top;
            }
            if (!STATE_ONLY) {
                ok = mbar_wait_warp(&ctl.s_full, it & 1, a.wait_polls);
                if (!ok) break;
                tc_fence_after();
                // Blocks of 32 rows x 16 columns: `side` < 0 for those before the diagonal in time (all of which count), 0 on it.  In the
                // reverse form the columns from `tokens` on, rows of the tensors behind the sequence, are on that side too: `live` of
                // a block's columns are this chunk's, and the others, which may hold anything, are no part of the row.
                // (The loops of this kernel are not unrolled further than registers demand: three kinds of warps run their code
                // at once, and unrolled it did not fit the instruction cache.)
                float up = 1.0f;
                if (HALF) {  // scaling from the largest of the row's products, times what a block's can grow by at most (decays only make them smaller)
                    float m = 0.0f;
#pragma unroll 1
                    for (int c0 = half * 16; c0 < TC; c0 += 32) {
                        const int side = a.reverse ? r0 - (c0 & ~31) : (c0 & ~31) - r0, d = row - c0, live = a.reverse ? tokens - c0 : 16;
                        if (side > 0 || live <= 0) continue;
                        const int lo = a.reverse ? d : 0, hi = a.reverse ? live - 1 : d;  // the row's columns of the block
                        uint32_t r[16];
                        tmem_ld16_nowait(lanes + COL_S + c0, r);
                        tmem_ld_wait16(r);
                        float largest = 0.0f;
#pragma unroll
                        for (int j = 0; j < 16; j++)
                            largest = fmaxf(largest, j >= lo && j <= hi ? fabsf(__uint_as_float(r[j])) : 0.0f);
                        if (grows) largest *= ex2_approx(g2 * (float)max(a.reverse ? 15 - d : d, 0));  // (its farthest column)
                        m = fmaxf(m, largest);
                    }
                    ctl.row_max[1][half][row] = (uint8_t)exponent_of(m);
                    ok = meet();
                    if (!ok) break;
                    up = fp16_scale(max(exponent_of(m), (int)ctl.row_max[1][half ^ 1][row]));
                    if (half == 0) ctl.p_scale[it & 1][row] = __float2bfloat16_rn(1.0f / up);
                }
#pragma unroll 1
                for (int c0 = half * 16; c0 < TC; c0 += 32) {
                    const int side = a.reverse ? r0 - (c0 & ~31) : (c0 & ~31) - r0, d = row - c0, live = a.reverse ? tokens - c0 : 16;
                    uint32_t w[16];  // eight words of high parts, eight of low ones
                    if (side > 0 || live <= 0) {
#pragma unroll
                        for (int j = 0; j < 16; j++) w[j] = 0;
                    } else {
                        uint32_t r[16];
                        tmem_ld16_nowait(lanes + COL_S + c0, r);
                        if (side < 0 && live >= 16) {
                            // decay = 2^(g2 (distance to the block's nearer edge)) 2^(g2 (inside the block))
                            const f32x2 outer = splat2(ex2_approx(g2 * (float)(a.reverse ? -d : d - 15)) * up);
                            tmem_ld_wait16(r);
#pragma unroll
                            for (int j = 0; j < 8; j++) {
                                const float2 inner = *reinterpret_cast<const float2 *>(&ctl.inner[2 * j]);
                                float u, v;
                                unpack2(mul2(mul2(pack2(inner.x, inner.y), outer), pack2(__uint_as_float(r[2 * j]), __uint_as_float(r[2 * j + 1]))), u, v);
                                two_parts<T>(u, v, w[j], w[j + 8]);
                            }
                        } else {  // entry by entry
                            const int lo = a.reverse ? d : 0, hi = a.reverse ? live - 1 : d;
                            const f32x2 g22 = splat2(a.reverse ? -g2 : g2), d2 = splat2((float)d), up2 = splat2(up);
                            tmem_ld_wait16(r);
#pragma unroll
                            for (int j = 0; j < 8; j++) {
                                const f32x2 x = ex2_approx2(mul2(g22, sub2(d2, pack2((float)(2 * j), (float)(2 * j + 1)))));
                                float u, v;
                                unpack2(mul2(HALF ? mul2(x, up2) : x, pack2(__uint_as_float(r[2 * j]), __uint_as_float(r[2 * j + 1]))), u, v);
                                two_parts<T>(2 * j >= lo && 2 * j <= hi ? u : 0.0f, 2 * j + 1 >= lo && 2 * j + 1 <= hi ? v : 0.0f, w[j], w[j + 8]);
                            }
                        }
                    }
                    tmem_st16(lanes + COL_S + c0, w);  // (over the 16 columns that have been read)
                }
                tmem_st_wait();
                tc_fence_before();
            }
            if (HALF) {
                if (STATE_ONLY) ok = meet();  // (else they have met for the rows of S)
                if (!ok) break;
                uint32_t top = 0;
#pragma unroll
                for (int i = 0; i < GROUP / 32; i++) top = max(top, (uint32_t)ctl.key_max[it & 1][i]);
                key_up = fp16_scale_of_bits(top);
                if (mine == 0) ctl.key_scale[it & 1] = 1.0f / key_up;
            }
            // K~ over K, its low part over Q and, if there is one, its lowest over Z, which QZ has read by now
            const bool three = !HALF && a.parts == 3;
            if (!STATE_ONLY)
                ok = mbar_wait_warp(&ctl.qz_full, it & 1, a.wait_polls);
            else if (three && it > 0)  // (nothing but U of the chunk before holds Z's only tile)
                ok = mbar_wait_warp(&ctl.o_full, (it - 1) & 1, a.wait_polls);
            if (!ok) break;
            unsigned char *kt = smem + b * L::STAGE + L::K + mine * 16, *qt = smem + b * L::STAGE + L::Q + mine * 16;
#pragma unroll
            for (int i = 0; i < KB * 4; i++) {
                uint4 x = *reinterpret_cast<const uint4 *>(kt + i * (GROUP * 16));
                const int m = (mine >> 3) + 32 * (i & 3);
                // (rows behind the last token are zero, whatever is in them)
                if (m >= tokens) x = make_uint4(0, 0, 0, 0);
                // decay to the chunk's last token; where it grows in fp16, relative to that of the chunk's first
                const float decay = exp2f(g2 * (float)(max(a.reverse ? m : tokens - 1 - m, 0) - (grows ? tokens - 1 : 0)));
                const f32x2 w = splat2(HALF ? decay * key_up : decay);
                const uint32_t in[4] = {x.x, x.y, x.z, x.w};
                uint32_t high[4], low[4], lowest[4];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float2 v = unpack<T>(in[j]);
                    const f32x2 y = mul2(pack2(v.x, v.y), w);
                    float y0, y1;
                    unpack2(y, y0, y1);
                    high[j] = pack<T>(y0, y1);
                    float2 r = unpack<T>(high[j]);
                    const f32x2 rest = sub2(y, pack2(r.x, r.y));
                    unpack2(rest, y0, y1);
                    low[j] = pack<T>(y0, y1);
                    if (!HALF) {
                        r = unpack<T>(low[j]);
                        unpack2(sub2(rest, pack2(r.x, r.y)), y0, y1);
                        lowest[j] = pack<T>(y0, y1);
                    }
                }
                if (three) *reinterpret_cast<uint4 *>(smem + L::Z + mine * 16 + i * (GROUP * 16)) = make_uint4(lowest[0], lowest[1], lowest[2], lowest[3]);
                *reinterpret_cast<uint4 *>(kt + i * (GROUP * 16)) = make_uint4(high[0], high[1], high[2], high[3]);
                *reinterpret_cast<uint4 *>(qt + i * (GROUP * 16)) = make_uint4(low[0], low[1], low[2], low[3]);
            }
            fence_async_smem();
            // (states alone: no further ahead than one chunk, of which key_scale has two)
            if (HALF && STATE_ONLY && it > 0) ok = mbar_wait_warp(&ctl.z_ready, (it - 1) & 1, a.wait_polls);
            if (!ok) break;
            mbar_arrive(&ctl.p_ready);
        }
        if (!ok) ctl.dead = 1;
    } else {  // ---------------------------------------------------------------------------------- results and state
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(RESULT_REGS));
        const bool state_row = row < VB * 64;
        f32x2 z[NZ / 2];
        const bool first_segment = s.first == 0;
        const float *from = nullptr;
        int64_t step = 0;
        if (!STATE_ONLY && row < a.dv) {
            if (!first_segment) {
                from = a.states + ((int64_t)s.start * a.heads + h) * a.dk * a.dv + row * a.state_col;
                step = a.state_row;
            } else if (a.state_in.data != nullptr) {
                from = a.state_in.at<const float>(s.seq, hg, hi) + row * a.state_in.col;
                step = a.state_in.row;
            }
        }
        const float enter = first_segment && !a.reverse && s.length > 0 ? exp2f(g2) : 1.0f;
#pragma unroll
        for (int j = 0; j < NZ / 2; j++) {
            const int c = half * NZ + 2 * j;
            z[j] = pack2(from != nullptr && c < a.dk ? from[c * step] * enter : 0.0f,
                         from != nullptr && c + 1 < a.dk ? from[(c + 1) * step] * enter : 0.0f);
        }
        // the state's copy in 16 bits for the products of chunk `it`
        const auto publish = [&](int it) {
            float f = 1.0f;
            if (HALF) {
                float m = 0.0f;
#pragma unroll
                for (int j = 0; j < NZ / 2; j++) {
                    float u, v;
                    unpack2(z[j], u, v);
                    m = fmaxf(m, fmaxf(fabsf(u), fabsf(v)));
                }
                ctl.row_max[0][half][row] = (uint8_t)exponent_of(m);
                if (!meet()) return false;
                f = fp16_scale(max(exponent_of(m), (int)ctl.row_max[0][half ^ 1][row]));
                if (half == 0) ctl.z_scale[it & 1][row] = __float2bfloat16_rn(1.0f / f);
                if (!meet()) return false;
            }
            if (!state_row) return true;
            const f32x2 f2 = splat2(f);
#pragma unroll
            for (int c = 0; c < NZ / 8; c++) {
                const int chunk = half * (NZ / 8) + c;  // of 8 values, in the row
                unsigned char *at = smem + L::Z + (chunk >> 3) * (VB * 64 * 128) + row * 128 + (((chunk & 7) ^ (row & 7)) << 4);
                uint32_t w[4];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    float u, v;
                    unpack2(HALF ? mul2(z[4 * c + j], f2) : z[4 * c + j], u, v);
                    w[j] = pack<T>(u, v);
                }
                *reinterpret_cast<uint4 *>(at) = make_uint4(w[0], w[1], w[2], w[3]);
            }
            return true;
        };
        bool ok = true;
        if (!STATE_ONLY) {
            ok = publish(0);
            fence_async_smem();
            mbar_arrive(&ctl.z_ready);
        }
        // how results leave: rounds of CB columns, 16 bytes (VALUES) of a row by a lane, ROWS rows at once
        constexpr int PER = 128 / (int)sizeof(O), CB = NO < PER ? NO : PER, VALUES = 16 / (int)sizeof(O), ACROSS = CB / VALUES, ROWS = 32 / ACROSS;
        constexpr int PITCH = CB * (int)sizeof(O);
        const bool out_aligned = rows_aligned(a.out, sizeof(O));
        O *const out = a.out.data == nullptr ? nullptr : a.out.at<O>(a.starts == nullptr ? s.seq : 0, hg, hi);
        const float intra = a.scale_in * a.scale_out;
        float inter = 0.0f;  // decay of the state to this row
        int it = 0;
        for (; it < chunks && ok; it++) {
            const int b = it & 1, tokens = min(TC, s.count - it * TC);
            const int e = s.first + it * TC + tokens == s.length && !a.reverse ? tokens - 1 : tokens;
            const float carry = exp2f(g2 * (float)e);
            if (it == 0 || tokens < TC) inter = exp2f(g2 * (float)(a.reverse ? tokens - 1 - row : row)) * a.scale_out;
            ok = mbar_wait_warp(&ctl.o_full, it & 1, a.wait_polls);
            if (HALF) ok = ok && mbar_wait_warp(&ctl.p_ready, it & 1, a.wait_polls);  // (p_scale, key_scale; long complete)
            ok = ok && *reinterpret_cast<volatile int *>(&ctl.dead) == 0;
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            tc_fence_after();
            // (K~ is decayed to the chunk's last token, which keeps its largest entries in fp16's range; the step beyond it, and those that growing
            // keys are short of, are taken here)
            const float beyond = a.scale_in * exp2f(g2 * (float)(grows ? e : e - tokens + 1));
            const f32x2 carry2 = splat2(carry), in2 = splat2(HALF ? beyond * ctl.key_scale[it & 1] : beyond);
#pragma unroll
            for (int cb = 0; cb < NZ / 16; cb++) {
                uint32_t r[16];
                tmem_ld16_nowait(lanes + COL_U + half * NZ + cb * 16, r);
                tmem_ld_wait16(r);
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    f32x2 &to = z[cb * 8 + j];
                    to = fma2(carry2, to, mul2(in2, pack2(__uint_as_float(r[2 * j]), __uint_as_float(r[2 * j + 1]))));
                }
                // (done with r before the next load: registers)
#pragma unroll
                for (int j = 0; j < 8; j++) asm volatile("" : "+l"(z[cb * 8 + j]));
            }
            if (STATE_ONLY) {
                tc_fence_before();
                mbar_arrive(&ctl.z_ready);
                continue;
            }
            ok = publish(it + 1);
            if (!ok) break;
            fence_async_smem();
            // Results leave through the stage's Q tile (K~'s low part has been read), a warp's 32 rows of up to 128 bytes at a
            // time, by TMA: with all of shared memory in use there is next to no L1 for stores of the threads (a chunk's results
            // took them 3000 cycles).  The rows around a sequence's end and what has no map do take that way.
            const float fp = HALF ? intra * __bfloat162float(ctl.p_scale[it & 1][row]) : intra;
            unsigned char *box = smem + b * L::STAGE + L::Q + warp * 4096;
            const int r0 = (warp & 3) * 32, to_row = chunk_row(a, s, it, tokens);
            const bool by_map = maps.use[3] && r0 + 32 <= tokens;
            static_assert(L::K >= 8 * 4096, "a box for each warp");
#pragma unroll
            for (int round = 0; round < NO / CB; round++) {
                if (round > 0) __syncwarp();
#pragma unroll 1
                for (int cb = 0; cb < CB; cb += 16) {
                    const int c0 = half * NO + round * CB + cb;
                    uint32_t x[16], y[16];
                    tmem_ld16_nowait(lanes + COL_PV + c0, x);
                    tmem_ld16_nowait(lanes + COL_QZ + c0, y);
                    tmem_ld_wait16(x);
                    tmem_ld_wait16(y);
                    const f32x2 fp2 = splat2(fp), inter2 = splat2(inter);
                    uint32_t w[sizeof(O) == 2 ? 8 : 16];
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        f32x2 q = mul2(inter2, pack2(__uint_as_float(y[2 * j]), __uint_as_float(y[2 * j + 1])));
                        if (HALF) {
                            const float2 f = unpack<__nv_bfloat16>(*reinterpret_cast<const uint32_t *>(&ctl.z_scale[it & 1][c0 + 2 * j]));
                            q = mul2(q, pack2(f.x, f.y));
                        }
                        float u, v;
                        unpack2(fma2(fp2, pack2(__uint_as_float(x[2 * j]), __uint_as_float(x[2 * j + 1])), q), u, v);
                        if constexpr (sizeof(O) == 2) {
                            w[j] = pack<T>(u, v);
                        } else {
                            w[2 * j] = __float_as_uint(u), w[2 * j + 1] = __float_as_uint(v);
                        }
                    }
#pragma unroll
                    for (int j = 0; j < 16 / VALUES; j++)
                        *reinterpret_cast<uint4 *>(box + swizzled<PITCH>(lane * PITCH + (cb / VALUES + j) * 16)) =
                            make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
                }
                const int x0 = half * NO + round * CB;
                if (by_map) fence_async_smem();
                if (round == NO / CB - 1) {
                    tc_fence_before();
                    mbar_arrive(&ctl.z_ready);
                }
                __syncwarp();
                if (by_map) {
                    if (lane == 0 && x0 < a.dv) {
                        tma_store(maps.out, x0, maps.by_group[3] * (int)hg + maps.by_head[3] * (int)hi, to_row + r0,
                                  maps.by_seq[3] * (a.starts == nullptr ? s.seq : 0), box);
                        tma_store_wait();
                    }
                    continue;
                }
                const int piece = lane % ACROSS, c = x0 + piece * VALUES, t0 = r0 + lane / ACROSS;
                O *to = out + (int64_t)(to_row + t0) * a.out.row + c * a.out.col;
#pragma unroll 1
                for (int i = 0; i < 32 / ROWS; i++, to += ROWS * a.out.row) {
                    const uint4 w = *reinterpret_cast<const uint4 *>(box + swizzled<PITCH>((i * ROWS + lane / ACROSS) * PITCH + piece * 16));
                    if (t0 + i * ROWS >= tokens || c >= a.dv) continue;
                    if (out_aligned && c + VALUES <= a.dv) {
                        *reinterpret_cast<uint4 *>(to) = w;
                    } else {
                        O x[VALUES];
                        memcpy(x, &w, 16);
#pragma unroll
                        for (int j = 0; j < VALUES; j++)
                            if (c + j < a.dv) to[j * a.out.col] = x[j];
                    }
                }
            }
            // The next copy into this tile is TMA's: it has to come after what the threads wrote and read here.  (Results that went by a
            // map are behind such a fence already.)
            if (!by_map) fence_async_smem();
            mbar_arrive(&ctl.q_empty[b]);
        }
        if (row < a.dv && (STATE_ONLY || (s.last && a.state_out.data != nullptr))) {
            float *to = STATE_ONLY ? a.states + ((int64_t)s.adds * a.heads + h) * a.dk * a.dv + row
                                   : a.state_out.at<float>(s.seq, hg, hi) + row * a.state_out.col;
            const int64_t row_step = STATE_ONLY ? a.dv : a.state_out.row;
#pragma unroll
            for (int j = 0; j < NZ / 2; j++) {
                float u, v;
                unpack2(z[j], u, v);
#pragma unroll
                for (int i = 0; i < 2; i++)
                    if (half * NZ + 2 * j + i < a.dk) to[(half * NZ + 2 * j + i) * row_step] = ok ? (i ? v : u) : __int_as_float(0x7fc00000);
            }
        }
        if (!ok) {  // gave up: say so, and leave nothing that looks like a result
            ctl.dead = 1;
            if (!STATE_ONLY)
                poison_rows<O>(out, a.out.row, a.out.col, a.reverse ? s.begin + s.length - s.first - s.count : s.begin + s.first + it * TC,
                               a.reverse ? s.begin + s.length - s.first - it * TC : s.begin + s.first + s.count, half * NO, min((half + 1) * NO, a.dv));
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == MMA_WARP) tmem_free(tmem, 512);
    if (tid == 0 && ctl.dead != 0 && a.gave_up != nullptr) {
        *reinterpret_cast<volatile int *>(a.gave_up) = GAVE_UP_DECAY;
        __threadfence_system();
    }
}

bool make_decay_map(CUtensorMap *map, const DecayArgs &a, const Operand &o, int dim, CUtensorMapDataType type, int size, int width, int rows,
                     int *by_group, int *by_head, int *by_seq) {
    using Encode = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                                const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static const Encode encode = [] {
        void *f = nullptr;
        cudaDriverEntryPointQueryResult found = cudaDriverEntryPointSymbolNotFound;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &found) != cudaSuccess || found != cudaDriverEntryPointSuccess)
            f = nullptr;
        return reinterpret_cast<Encode>(f);
    }();
    if (encode == nullptr || a.tokens < 1) return false;
    if (o.col != 1 || o.row <= 0 || o.seq < 0 || o.group < 0 || o.head < 0) return false;
    if ((reinterpret_cast<uintptr_t>(o.data) | (uintptr_t)((o.seq | o.group | o.head | o.row) * size)) & 15) return false;
    // heads: all of them (stride o.head), one to a group (stride o.group), or one in all
    const int64_t groups = a.heads / a.group;
    int64_t heads = 1, head_stride = 16;
    *by_group = *by_head = 0;
    if (o.head != 0 && a.group > 1) {
        if (o.group != o.head * a.group && groups > 1) return false;
        heads = a.heads, head_stride = o.head;
        *by_group = (int)a.group, *by_head = 1;
    } else if (o.group != 0 && groups > 1) {
        heads = groups, head_stride = o.group;
        *by_group = 1;
    }
    const bool batch = a.starts == nullptr && a.sequences > 1 && o.seq != 0;
    *by_seq = batch ? 1 : 0;
    const cuuint64_t sizes[4] = {(cuuint64_t)dim, (cuuint64_t)heads, (cuuint64_t)a.tokens, (cuuint64_t)(batch ? a.sequences : 1)};
    const cuuint64_t strides[3] = {(cuuint64_t)(head_stride * size), (cuuint64_t)(o.row * size), (cuuint64_t)((batch ? o.seq : 16) * size)};
    for (cuuint64_t stride : strides)
        if (stride >= (1ull << 40)) return false;
    const cuuint32_t box[4] = {(cuuint32_t)width, 1, (cuuint32_t)rows, 1}, ones[4] = {1, 1, 1, 1};
    return encode(map, type, 4, o.data, sizes, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  width * size == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, typename O, int KB, int VB, bool STATE_ONLY>
static int launch_one(const DecayArgs &a, cudaStream_t s) {
    auto kernel = decay_tc_kernel<T, O, KB, VB, STATE_ONLY>;
    constexpr int bytes = Smem<KB, VB>::BYTES + (int)sizeof(Control);
    static_assert(bytes <= 232448, "shared memory of an SM");
    const cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (err != cudaSuccess) return cuda_fail(err, "decay_tc_kernel");
    Maps maps = {};
    const Operand *operands[3] = {&a.q, &a.k, &a.v};
    CUtensorMap *map[3] = {&maps.q, &maps.k, &maps.v};
    constexpr CUtensorMapDataType type = std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    for (int i = STATE_ONLY ? 1 : 0; i < 3; i++)
        maps.use[i] = make_decay_map(map[i], a, *operands[i], i == 2 ? a.dv : a.dk, type, 2, 64, TC, &maps.by_group[i], &maps.by_head[i], &maps.by_seq[i]);
    if (!STATE_ONLY)
        maps.use[3] = make_decay_map(&maps.out, a, a.out, a.dv, sizeof(O) == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : type, (int)sizeof(O),
                               std::min(VB * 32, 128 / (int)sizeof(O)), 32, &maps.by_group[3], &maps.by_head[3], &maps.by_seq[3]);
    kernel<<<(unsigned)(a.slots * a.heads), THREADS, bytes, s>>>(a, maps);
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
