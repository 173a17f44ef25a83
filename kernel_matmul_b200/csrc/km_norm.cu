// The 2-norm over many tensors, and clipping to it.
//
// Bound by memory: the norm reads every value once; the scaling pass, which runs only where the factor is not one, reads
// and writes them once more.  All tensors go into one launch (their table travels in the kernel's parameters, so that nothing is
// copied beforehand and a captured graph holds it): chunks of NORM_CHUNK bytes, dealt to a fixed number of CTAs, one
// partial sum per CTA, added in a fixed order: deterministic.
//
// Squares are summed in fp32 inside a chunk and in fp64 beyond it.  A chunk whose sum overflows or is so small that squares
// may have been lost below the smallest fp32 is summed again in fp64: values from 1e-38 to 3e38 have their norm.
#include <vector>

#include "km_decay.cuh"

namespace km {

// Tensors to a launch: 21 KB of parameters, or, where 64 do, 1.3 KB (a launch copies them: 5 us of host time for the long table).
constexpr int NORM_TENSORS = 1024, NORM_FEW = 64;
constexpr int64_t NORM_CHUNK = 65536;   // bytes
constexpr int NORM_CTAS = 148 * 4;
constexpr int NORM_THREADS = 512;

template <int N>
struct NormTable {
    int count;
    int64_t chunks;
    void *data[N];
    int64_t elements[N];
    uint32_t first[N];  // number of the tensor's first chunk
    uint8_t type[N];
};

struct NormChunk {
    char *data;
    int64_t elements;
    int type;
};

template <int N>
__device__ __forceinline__ NormChunk norm_chunk(const NormTable<N> &t, int64_t chunk) {
    int lo = 0, hi = t.count - 1;  // the last tensor whose first chunk is not behind
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if ((int64_t)t.first[mid] <= chunk)
            lo = mid;
        else
            hi = mid - 1;
    }
    const int size = t.type[lo] == KM_TYPE_F32 ? 4 : 2;
    const int64_t per = NORM_CHUNK / size, skip = (chunk - t.first[lo]) * per;
    return {static_cast<char *>(t.data[lo]) + skip * size, min(per, t.elements[lo] - skip), t.type[lo]};
}

template <typename T>
__device__ __forceinline__ float squares(const uint4 &w) {
    float s = 0.0f;
    if constexpr (sizeof(T) == 4) {
        const float x[4] = {__uint_as_float(w.x), __uint_as_float(w.y), __uint_as_float(w.z), __uint_as_float(w.w)};
#pragma unroll
        for (int i = 0; i < 4; i++) s = fmaf(x[i], x[i], s);
    } else {
        T x[8];
        memcpy(x, &w, 16);
#pragma unroll
        for (int i = 0; i < 8; i++) s = fmaf(as_float(x[i]), as_float(x[i]), s);
    }
    return s;
}

// Sum of this thread's squares; `lost`: whether they may have fallen out of fp32's range (a sum of exact zeros has not).
template <typename T>
__device__ __forceinline__ float chunk_squares(const NormChunk &c, bool &lost) {
    constexpr int VEC = 16 / sizeof(T);
    const T *p = reinterpret_cast<const T *>(c.data);
    // plain loads up to the first boundary of 16 bytes and behind the last
    const int lead = (int)min(c.elements, (int64_t)(((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / sizeof(T)));
    const int words = (int)((c.elements - lead) / VEC), tail = (int)(c.elements - lead) - words * VEC;
    const uint4 *w = reinterpret_cast<const uint4 *>(p + lead);
    float s[4] = {};
    uint32_t bits = 0;
    bool odd = false;
    int i = threadIdx.x;
    for (; i + 3 * NORM_THREADS < words; i += 4 * NORM_THREADS) {
        uint4 v[4];
#pragma unroll
        for (int j = 0; j < 4; j++) v[j] = w[i + j * NORM_THREADS];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            s[j] += squares<T>(v[j]);
            bits |= v[j].x | v[j].y | v[j].z | v[j].w;
        }
    }
    for (; i < words; i += NORM_THREADS) {
        const uint4 v = w[i];
        s[0] += squares<T>(v);
        bits |= v.x | v.y | v.z | v.w;
    }
    if ((int)threadIdx.x < lead) {
        const float x = as_float(p[threadIdx.x]);
        s[1] = fmaf(x, x, s[1]);
        odd = odd || x != 0.0f;
    }
    if ((int)threadIdx.x < tail) {
        const float x = as_float(p[lead + words * VEC + threadIdx.x]);
        s[2] = fmaf(x, x, s[2]);
        odd = odd || x != 0.0f;
    }
    const float sum = (s[0] + s[1]) + (s[2] + s[3]);
    odd = odd || (bits & (sizeof(T) == 4 ? 0x7fffffffu : 0x7fff7fffu)) != 0;
    lost = !(sum <= 1e36f) || (sum < 1e-30f && odd);
    return sum;
}

template <typename T>
__device__ double chunk_squares_f64(const NormChunk &c) {
    const T *p = reinterpret_cast<const T *>(c.data);
    double s = 0.0;
    for (int64_t i = threadIdx.x; i < c.elements; i += NORM_THREADS) {
        const double x = (double)as_float(p[i]);
        s = fma(x, x, s);
    }
    return s;
}

__device__ __forceinline__ double block_sum(double v, double *scratch) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.0;
    for (int w = 0; w < NORM_THREADS / 32; w++) v += scratch[w];
    return v;
}

template <int N>
__global__ void __launch_bounds__(NORM_THREADS) norm_squares_kernel(const __grid_constant__ NormTable<N> t, double *partials) {
    __shared__ double scratch[NORM_THREADS / 32];
    double sum = 0.0;
    for (int64_t chunk = blockIdx.x; chunk < t.chunks; chunk += gridDim.x) {
        const NormChunk c = norm_chunk(t, chunk);
        bool lost;
        const float s = c.type == KM_TYPE_F32    ? chunk_squares<float>(c, lost)
                        : c.type == KM_TYPE_BF16 ? chunk_squares<__nv_bfloat16>(c, lost)
                                                 : chunk_squares<__half>(c, lost);
        if (__syncthreads_or(lost)) {
            sum += c.type == KM_TYPE_F32    ? chunk_squares_f64<float>(c)
                   : c.type == KM_TYPE_BF16 ? chunk_squares_f64<__nv_bfloat16>(c)
                                            : chunk_squares_f64<__half>(c);
        } else {
            sum += (double)s;
        }
    }
    sum = block_sum(sum, scratch);
    if (threadIdx.x == 0) partials[blockIdx.x] = sum;
}

template <typename T>
__device__ __forceinline__ void scale_chunk(const NormChunk &c, float f, float power) {
    constexpr int VEC = 16 / sizeof(T);
    T *p = reinterpret_cast<T *>(c.data);
    const int lead = (int)min(c.elements, (int64_t)(((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / sizeof(T)));
    const int words = (int)((c.elements - lead) / VEC), tail = (int)(c.elements - lead) - words * VEC;
    uint4 *w = reinterpret_cast<uint4 *>(p + lead);
    const auto scaled = [f, power](uint4 v) {
        T x[VEC];
        memcpy(x, &v, 16);
#pragma unroll
        for (int i = 0; i < VEC; i++) x[i] = from_float<T>(as_float(x[i]) * f * power);
        memcpy(&v, x, 16);
        return v;
    };
    int i = threadIdx.x;
    for (; i + 3 * NORM_THREADS < words; i += 4 * NORM_THREADS) {
        uint4 v[4];
#pragma unroll
        for (int j = 0; j < 4; j++) v[j] = w[i + j * NORM_THREADS];
#pragma unroll
        for (int j = 0; j < 4; j++) w[i + j * NORM_THREADS] = scaled(v[j]);
    }
    for (; i < words; i += NORM_THREADS) w[i] = scaled(w[i]);
    if ((int)threadIdx.x < lead) p[threadIdx.x] = from_float<T>(as_float(p[threadIdx.x]) * f * power);
    if ((int)threadIdx.x < tail) {
        T *q = p + lead + words * VEC + threadIdx.x;
        *q = from_float<T>(as_float(*q) * f * power);
    }
}

// Every CTA adds the partial sums by itself (a few KB from L2), in the same order.  Chunks are gone through from the last:
// what the first pass read last may still be in L2.
template <int N>
__global__ void __launch_bounds__(NORM_THREADS) norm_finish_kernel(const __grid_constant__ NormTable<N> t, const double *partials, int count,
                                                                  int scale, double max_norm, double eps, float *norm) {
    __shared__ double scratch[NORM_THREADS / 32];
    grid_wait();
    double v = 0.0;
    for (int i = threadIdx.x; i < count; i += NORM_THREADS) v += partials[i];
    const double n = sqrt(block_sum(v, scratch));
    if (norm != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)n;
    if (!scale) return;
    const double factor = max_norm / (n + eps);
    if (factor >= 1.0) return;
    // (a factor near the smallest fp32 values or below them, as for gradients of 1e38, in two)
    const float power = factor < 1e-30 ? 0x1p-100f : 1.0f, f = (float)(factor / (double)power);
    for (int64_t chunk = t.chunks - 1 - (int64_t)blockIdx.x; chunk >= 0; chunk -= gridDim.x) {
        const NormChunk c = norm_chunk(t, chunk);
        if (c.type == KM_TYPE_F32)
            scale_chunk<float>(c, f, power);
        else if (c.type == KM_TYPE_BF16)
            scale_chunk<__nv_bfloat16>(c, f, power);
        else
            scale_chunk<__half>(c, f, power);
    }
}

template <int N>
static int norm_launches(int64_t count, void *const *tensors, const int64_t *elements, const int32_t *types, int32_t scale_in_place, double max_norm,
                         double eps, float *norm, double *partials, cudaStream_t s) {
    static thread_local NormTable<N> table;  // (which a launch copies)
    int used = 0;
    const auto fill = [&](int64_t first) -> int {
        table.count = 0, table.chunks = 0;
        for (int64_t i = first; i < std::min(count, first + N); i++) {
            if (elements[i] == 0) continue;
            const int j = table.count++;
            table.data[j] = tensors[i], table.elements[j] = elements[i], table.type[j] = (uint8_t)types[i];
            table.first[j] = (uint32_t)table.chunks;
            table.chunks += ceil_div(elements[i], NORM_CHUNK / (types[i] == KM_TYPE_F32 ? 4 : 2));
            KM_REQUIRE(table.chunks < (1LL << 32), KM_ERR_UNSUPPORTED, "km_global_norm: more than 2^48 bytes");
        }
        return KM_OK;
    };
    const int64_t launches = std::max<int64_t>(1, ceil_div(count, N));
    for (int64_t l = 0; l < launches; l++) {
        const int rc = fill(l * N);
        if (rc != KM_OK) return rc;
        const int ctas = (int)std::min<int64_t>(table.chunks, NORM_CTAS);
        if (ctas == 0) continue;
        norm_squares_kernel<N><<<ctas, NORM_THREADS, 0, s>>>(table, partials + used);
        KM_CHECK_LAUNCH("norm_squares_kernel launch");
        used += ctas;
    }
    for (int64_t l = 0; l < (scale_in_place ? launches : 1); l++) {
        if (launches > 1) {
            const int rc = fill(l * N);
            if (rc != KM_OK) return rc;
        }
        const int ctas = scale_in_place ? (int)std::max<int64_t>(1, std::min<int64_t>(table.chunks, NORM_CTAS)) : 1;
        const int rc = launch_chained("norm_finish_kernel launch", norm_finish_kernel<N>, dim3((unsigned)ctas), NORM_THREADS, 0, s, table,
                                      (const double *)partials, used, (int)scale_in_place, max_norm, eps, l == 0 ? norm : (float *)nullptr);
        if (rc != KM_OK) return rc;
    }
    return KM_OK;
}

}  // namespace km

extern "C" size_t km_global_norm_workspace_bytes(int64_t count) {
    using namespace km;
    return (size_t)std::max<int64_t>(1, ceil_div(std::max<int64_t>(count, 0), NORM_TENSORS)) * NORM_CTAS * sizeof(double);
}

extern "C" int km_global_norm(int64_t count, void *const *tensors, const int64_t *elements, const int32_t *types, int32_t scale_in_place,
                              double max_norm, double eps, float *norm, void *workspace, size_t workspace_bytes, void *stream) {
    using namespace km;
    KM_REQUIRE(count >= 0 && norm != nullptr && (count == 0 || (tensors && elements && types)), KM_ERR_INVALID_ARGUMENT,
               "km_global_norm: bad arguments");
    KM_REQUIRE(workspace != nullptr && workspace_bytes >= km_global_norm_workspace_bytes(count), KM_ERR_WORKSPACE,
               "km_global_norm: workspace of %zu bytes needed", km_global_norm_workspace_bytes(count));
    KM_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, KM_ERR_WORKSPACE, "km_global_norm: workspace must be 16-byte aligned");
    for (int64_t i = 0; i < count; i++) {
        KM_REQUIRE(elements[i] >= 0 && types[i] >= KM_TYPE_F32 && types[i] <= KM_TYPE_F16 && (elements[i] == 0 || tensors[i] != nullptr),
                   KM_ERR_INVALID_ARGUMENT, "km_global_norm: bad tensor %lld", (long long)i);
        KM_REQUIRE(reinterpret_cast<uintptr_t>(tensors[i]) % (types[i] == KM_TYPE_F32 ? 4 : 2) == 0 && elements[i] < (1LL << 40),
                   KM_ERR_INVALID_ARGUMENT, "km_global_norm: bad tensor %lld", (long long)i);
    }
    const auto run = count <= NORM_FEW ? km::norm_launches<NORM_FEW> : km::norm_launches<NORM_TENSORS>;
    return run(count, tensors, elements, types, scale_in_place, max_norm, eps, norm, static_cast<double *>(workspace), static_cast<cudaStream_t>(stream));
}
