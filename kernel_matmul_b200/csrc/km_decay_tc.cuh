// What the tensor-core kernels of the linear attention with decay share (km_decay_tc.cu, km_decay_grad_tc.cu): tiles of 128
// tokens in shared memory, products of them, their loads.
#pragma once

#include <cuda.h>

#include <type_traits>

#include "km_decay.cuh"

namespace km {

namespace {

constexpr int TC = 128;       // tokens of a chunk
constexpr int BLOCK_BYTES = TC * 128;  // 128 rows of 64 values

// Tiles hold rows in the order of memory, in the reverse form too, which goes through the chunks from the last: row `m` of
// a chunk of n tokens is token m, or token n - 1 - m in the order in which the sequence is gone through.
__device__ __forceinline__ int chunk_row(const DecayArgs &a, const Segment &s, int chunk, int tokens) {
    const int first = s.first + chunk * TC;
    return s.begin + (a.reverse ? s.length - first - tokens : first);
}

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

__device__ __forceinline__ void tmem_ld8_nowait(uint32_t taddr, uint32_t (&r)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr)
                 : "memory");
}
// The wait for loads into `p` and `q`, tied to their registers (km_tcgen05.cuh, tmem_ld_wait16).
__device__ __forceinline__ void tmem_ld_wait8x2(uint32_t (&p)[8], uint32_t (&q)[8]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(p[0]), "+r"(p[1]), "+r"(p[2]), "+r"(p[3]), "+r"(p[4]), "+r"(p[5]), "+r"(p[6]), "+r"(p[7]), "+r"(q[0]), "+r"(q[1]),
                   "+r"(q[2]), "+r"(q[3]), "+r"(q[4]), "+r"(q[5]), "+r"(q[6]), "+r"(q[7])
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

// Two values in two parts: high (rounded to nearest) and what that leaves.
template <typename T>
__device__ __forceinline__ void two_parts(float a, float b, uint32_t &high, uint32_t &low) {
    high = pack<T>(a, b);
    const float2 h = unpack<T>(high);
    low = pack<T>(a - h.x, b - h.y);
}

__device__ __forceinline__ int exponent_of(float m) { return (int)((__float_as_uint(m) >> 23) & 0xffu); }
// 2^n that brings a largest magnitude of (biased) exponent e to [2^13, 2^14) (fp16's range and as many of its small values as
// possible); 1 for 0 and for what is not finite
__device__ __forceinline__ float fp16_scale(int e) {
    if (e == 0 || e == 255) return 1.0f;
    return __uint_as_float((uint32_t)min(max(127 + 13 - (e - 127), 2), 252) << 23);  // (its inverse is a normal number too)
}
// The larger magnitudes of pairs of fp16 values, as bits; those of a word's two as one.
__device__ __forceinline__ uint32_t fp16_largest(uint32_t so_far, const uint4 &x) {
    const uint32_t p = __vmaxu2(x.x & 0x7fff7fffu, x.y & 0x7fff7fffu), q = __vmaxu2(x.z & 0x7fff7fffu, x.w & 0x7fff7fffu);
    return __vmaxu2(so_far, __vmaxu2(p, q));
}
__device__ __forceinline__ uint32_t fp16_larger(uint32_t pair) { return max(pair >> 16, pair & 0xffffu); }
__device__ __forceinline__ float fp16_scale_of_bits(uint32_t bits) {
    return fp16_scale(exponent_of(__half2float(__ushort_as_half((unsigned short)bits))));
}

// Whether every row starts on a boundary of 16 bytes.
__device__ __forceinline__ bool rows_aligned(const Operand &o, int size) {
    return o.col == 1 && ((reinterpret_cast<uintptr_t>(o.data) | (uintptr_t)((o.seq | o.group | o.head | o.row) * size)) & 15) == 0;
}

__device__ __forceinline__ void tma_load(unsigned char *dst, const CUtensorMap &map, int x, int head, int row, int seq, uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(
            smem_u32(dst)),
        "l"(&map), "r"(x), "r"(head), "r"(row), "r"(seq), "r"(smem_u32(bar))
        : "memory");
}

// Rows [0, tokens) of a tile without a tensor map (rows or values that do not lie on boundaries of 16 bytes), by a warp; zeros
// behind them.  `src` is the head's value (row `first`, 0).
template <typename T, int BLOCKS>
__device__ __noinline__ void copy_tile(unsigned char *tile, const T *src, int64_t row, int64_t col, int tokens, int dim, int lane) {
    constexpr int PIECES = BLOCKS * 8;
    for (int i = lane; i < TC * PIECES; i += 32) {
        const int r = i / PIECES, c = i % PIECES;
        union {
            T v[8];
            uint4 w;
        } x;
        x.w = make_uint4(0, 0, 0, 0);
        if (r < tokens)
            for (int j = 0; j < min(dim - c * 8, 8); j++) x.v[j] = src[r * row + (c * 8 + j) * col];
        *reinterpret_cast<uint4 *>(tile + (c >> 3) * BLOCK_BYTES + r * 128 + (((c & 7) ^ (r & 7)) << 4)) = x.w;
    }
}

}  // namespace

// The tensor map of one operand (boxes of `width` values x `rows` tokens), if its rows and values allow one, and the coordinates
// of a head and a sequence in it (km_decay_tc.cu).
bool make_decay_map(CUtensorMap *map, const DecayArgs &a, const Operand &o, int dim, CUtensorMapDataType type, int size, int width, int rows,
                    int *by_group, int *by_head, int *by_seq);

}  // namespace km
