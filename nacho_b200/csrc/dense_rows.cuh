// What the operators around a router share: element types of dense rows, vectors of them, and blocks of 128 in 8-bit
// floating point.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "block_utils.cuh"

namespace nb200 {

// ---- rows of floats --------------------------------------------------------------------

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// V neighbouring elements, loaded and stored as one word.
template <typename T, int V>
struct alignas(sizeof(T) * V) Vec {
    T v[V];
};

// 16 bytes of a row as a thread handles them: words of V elements, `pitch` elements apart (neighbouring threads have neighbouring words), so that
// rows of any alignment keep as much on its way per thread.
template <typename T, int V>
struct Chunk {
    static constexpr int WORDS = 16 / (int)sizeof(T) / V, N = WORDS * V;
    Vec<T, V> w[WORDS];

    __device__ __forceinline__ void load(const T *row, int64_t c, int64_t pitch, int64_t cols) {
#pragma unroll
        for (int u = 0; u < WORDS; ++u)
            if (u == 0 || c + u * pitch < cols) w[u] = *reinterpret_cast<const Vec<T, V> *>(row + c + u * pitch);
    }
    __device__ __forceinline__ void store(T *row, int64_t c, int64_t pitch, int64_t cols) const {
#pragma unroll
        for (int u = 0; u < WORDS; ++u)
            if (u == 0 || c + u * pitch < cols) *reinterpret_cast<Vec<T, V> *>(row + c + u * pitch) = w[u];
    }
    __device__ __forceinline__ float get(int i) const { return to_float(w[i / V].v[i % V]); }
    __device__ __forceinline__ void set(int i, float f) { w[i / V].v[i % V] = from_float<T>(f); }
    // Whether element i lies in the row.
    __device__ __forceinline__ static bool there(int i, int64_t c, int64_t pitch, int64_t cols) { return i < V || c + i / V * pitch < cols; }
};

inline size_t type_size(int type) { return type == NB200_F32 ? 4 : 2; }

inline bool dense_ok(const nb200_dense *x) {
    return x && x->rows >= 0 && x->cols >= 0 && x->stride >= 0 && (x->rows == 0 || x->cols == 0 || x->data) && x->type >= NB200_F32 && x->type <= NB200_BF16 &&
           reinterpret_cast<uintptr_t>(x->data) % type_size(x->type) == 0;
}

// The widest word, 16 bytes at most, by which all rows of all given matrices can be accessed (in bytes). Rows are read whole, so the width
// has to divide too.
inline int word_bytes(std::initializer_list<const nb200_dense *> all) {
    int word = 16;
    for (const nb200_dense *x : all) {
        const uint64_t size = type_size(x->type);
        const uint64_t bits = reinterpret_cast<uintptr_t>(x->data) | (x->rows > 1 ? x->stride * size : 0) | x->cols * size;
        while (bits % word) word /= 2;
    }
    return word;
}

inline int sm_count() {
    static const int count = [] {
        int dev = 0, n = 0;
        if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) n = 148;
        return n;
    }();
    return count;
}

// Calls f(T{}) with the element type.
template <typename F>
int with_type(int type, F f) {
    if (type == NB200_F32) return f(float{});
    if (type == NB200_F16) return f(__half{});
    return f(__nv_bfloat16{});
}

// Calls f(std::integral_constant<int, V>) for words of `word` bytes, no fewer than an element's.
template <typename T, typename F>
int with_vector(int word, F f) {
    if (word == 16) return f(std::integral_constant<int, 16 / sizeof(T)>{});
    if (word == 8) return f(std::integral_constant<int, 8 / sizeof(T)>{});
    if constexpr (sizeof(T) == 2)
        if (word == 4) return f(std::integral_constant<int, 2>{});
    return f(std::integral_constant<int, 1>{});
}

// ---- 8-bit blocks ----------------------------------------------------------------------

constexpr int BLOCK8 = 128;
constexpr float TOP8 = 448.f;           // the largest e4m3 number
constexpr uint32_t FLOOR8 = 0x08800000;  // 2^-110: 448 / m stays finite, m / 448 a normal number

__host__ __device__ __forceinline__ int64_t blocks_of(int64_t n) { return (n + BLOCK8 - 1) / BLOCK8; }
__host__ __device__ __forceinline__ int64_t padded_rows(int64_t rows) { return (rows + 7) & ~int64_t(7); }

// Byte offset of piece p (16 codes) of row r in a column block. The place of a piece turns with the row as the 128-byte swizzle of
// the tensor cores' shared-memory tiles has it, so that a tile is a plain copy of consecutive memory.
__device__ __forceinline__ int64_t piece_at(int64_t r, int p) { return r * BLOCK8 + ((p ^ (int)(r & 7)) << 4); }

// Magnitudes are compared as integers, in which a NaN is above everything.
__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// The two factors of a block whose largest magnitude is m.
struct Factors {
    float scale, inverse;
};
__device__ __forceinline__ Factors factors_of(uint32_t m) {
    const float top = __uint_as_float(max(m, FLOOR8));
    return {__fdiv_rn(top, TOP8), __fdiv_rn(TOP8, top)};
}

__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d, float inverse) {
    const __nv_fp8x2_storage_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a * inverse, b * inverse), __NV_SATFINITE, __NV_E4M3);
    const __nv_fp8x2_storage_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c * inverse, d * inverse), __NV_SATFINITE, __NV_E4M3);
    return (uint32_t)lo | (uint32_t)hi << 16;
}

inline bool fp8_ok(const nb200_fp8 *m) {
    return m && nb200_fp8_value_count(m) >= 0 && (nb200_fp8_value_count(m) == 0 || (m->values && m->scales)) &&
           reinterpret_cast<uintptr_t>(m->values) % 16 == 0 && reinterpret_cast<uintptr_t>(m->scales) % 16 == 0;
}

// Eight neighbouring elements of a row from column c on, zeros from column `cols` on. V: what one load brings.
template <typename T, int V>
__device__ __forceinline__ Vec<T, 8> load8(const T *row, int64_t c, int64_t cols) {
    Vec<T, 8> out;
#pragma unroll
    for (int i = 0; i < 8; i += V) {
        Vec<T, V> w;
        if (c + i < cols) {
            w = *reinterpret_cast<const Vec<T, V> *>(row + c + i);
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) w.v[j] = from_float<T>(0.f);
        }
#pragma unroll
        for (int j = 0; j < V; ++j) out.v[i + j] = w.v[j];
    }
    return out;
}

// The factors of U blocks (a power of two) of 16 threads, which all have their largest magnitudes: every thread divides for one of them, a division
// being as much as a dozen other instructions.
template <int U>
__device__ __forceinline__ void share_factors(unsigned threads, const uint32_t (&m)[U], Factors (&f)[U]) {
    const int lane = lane_id();
    uint32_t mine = m[0];
#pragma unroll
    for (int u = 1; u < U; ++u) mine = (lane & (U - 1)) == u ? m[u] : mine;
    const Factors own = factors_of(mine);
#pragma unroll
    for (int u = 0; u < U; ++u) {
        f[u].scale = __shfl_sync(threads, own.scale, (lane & 16) + u);
        f[u].inverse = __shfl_sync(threads, own.inverse, (lane & 16) + u);
    }
}

// Eight neighbouring codes, and the largest magnitude of eight elements.
template <typename T>
__device__ __forceinline__ uint2 codes8(const Vec<T, 8> &v, float inverse) {
    return make_uint2(codes4(to_float(v.v[0]), to_float(v.v[1]), to_float(v.v[2]), to_float(v.v[3]), inverse),
                      codes4(to_float(v.v[4]), to_float(v.v[5]), to_float(v.v[6]), to_float(v.v[7]), inverse));
}
template <typename T>
__device__ __forceinline__ uint32_t magnitude8(const Vec<T, 8> &v) {
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max(m, magnitude(to_float(v.v[j])));
    return m;
}

}  // namespace nb200
