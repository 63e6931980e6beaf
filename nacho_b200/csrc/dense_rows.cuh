// What the operators around a router share: element types of dense rows, vectors of them, and blocks of 128 in 8-bit
// floating point.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <initializer_list>
#include <type_traits>

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

// What the runtime is asked once per device and kernel (a microsecond each time): a limit of dynamic shared memory that has been raised, and how
// many CTAs of so many threads an SM holds.
int allow_shared_memory(const void *kernel, size_t bytes);
int resident_ctas(const void *kernel, int threads);
template <typename... P>
int allow_shared(void (*kernel)(P...), size_t bytes) { return allow_shared_memory(reinterpret_cast<const void *>(kernel), bytes); }

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

// Eight neighbouring elements of a row as the words they lie in (kept whole: element by element the compiler takes them apart and puts them
// together again, which was most of what quantising did).
template <typename T>
struct Eight {
    static constexpr int WORDS = sizeof(T) * 2;
    uint32_t w[WORDS];

    // From column c on, zeros from column `cols` on. V: what one load brings.
    template <int V>
    __device__ __forceinline__ void load(const T *row, int64_t c, int64_t cols) {
        constexpr int BYTES = V * sizeof(T);
        if constexpr (BYTES >= 4) {
            constexpr int EACH = BYTES / 4;
#pragma unroll
            for (int i = 0; i < WORDS; i += EACH) {
                Vec<uint32_t, EACH> in{};
                if (c + i * (4 / (int)sizeof(T)) < cols) in = *reinterpret_cast<const Vec<uint32_t, EACH> *>(row + c + i * (4 / (int)sizeof(T)));
#pragma unroll
                for (int j = 0; j < EACH; ++j) w[i + j] = in.v[j];
            }
        } else {
            const uint16_t *from = reinterpret_cast<const uint16_t *>(row + c);
#pragma unroll
            for (int i = 0; i < WORDS; ++i) {
                const uint32_t lo = c + 2 * i < cols ? from[2 * i] : 0, hi = c + 2 * i + 1 < cols ? from[2 * i + 1] : 0;
                w[i] = lo | hi << 16;
            }
        }
    }
    __device__ __forceinline__ float get(int i) const {
        if constexpr (sizeof(T) == 4) return __uint_as_float(w[i]);
        else if constexpr (std::is_same<T, __half>::value) return __half2float(__ushort_as_half((unsigned short)(i & 1 ? w[i / 2] >> 16 : w[i / 2])));
        else return __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
    }
};

// Largest magnitudes. They are compared as integers, in which a NaN is above everything; those of 16-bit types two at a time, since what
// quantises is bound by its instructions. `bits` is the larger one as a 32-bit number's.
template <typename T>
struct Top {
    uint32_t v = 0;

    __device__ __forceinline__ static uint32_t larger(uint32_t a, uint32_t b) {
        if constexpr (sizeof(T) == 2) {
            uint32_t m;
            asm("max.u16x2 %0, %1, %2;" : "=r"(m) : "r"(a), "r"(b));
            return m;
        } else {
            return max(a, b);
        }
    }
    __device__ __forceinline__ void add(uint32_t word) { v = larger(v, word & (sizeof(T) == 2 ? 0x7fff7fffu : 0x7fffffffu)); }
    __device__ __forceinline__ void add(const Eight<T> &x) {
#pragma unroll
        for (int i = 0; i < Eight<T>::WORDS; ++i) add(x.w[i]);
    }
    // With that of the thread `distance` lanes away.
    __device__ __forceinline__ void join(unsigned threads, int distance) { v = larger(v, __shfl_xor_sync(threads, v, distance)); }
    __device__ __forceinline__ static uint32_t as_float(uint32_t half) {
        if constexpr (std::is_same<T, __half>::value) return __float_as_uint(__half2float(__ushort_as_half((unsigned short)half)));
        else return half << 16;
    }
    __device__ __forceinline__ uint32_t bits() const {
        if constexpr (sizeof(T) == 2) return as_float(max(v & 0xffffu, v >> 16));
        else return v;
    }
};

// The two factors of a block whose largest magnitude is m.
struct Factors {
    float scale, inverse;
};
__device__ __forceinline__ Factors factors_of(uint32_t m) {
    const float top = __uint_as_float(max(m, FLOOR8));
    return {__fdiv_rn(top, TOP8), __fdiv_rn(TOP8, top)};
}

__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d, float inverse) {
    uint32_t q;
    asm("{\n\t.reg .b16 lo, hi;\n\t"
        "cvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\n\t"
        "cvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\n\t"
        "mov.b32 %0, {lo, hi};\n\t}"
        : "=r"(q)
        : "f"(a * inverse), "f"(b * inverse), "f"(c * inverse), "f"(d * inverse));
    return q;
}

inline bool fp8_ok(const nb200_fp8 *m) {
    return m && nb200_fp8_value_count(m) >= 0 && (nb200_fp8_value_count(m) == 0 || (m->values && m->scales)) &&
           reinterpret_cast<uintptr_t>(m->values) % 16 == 0 && reinterpret_cast<uintptr_t>(m->scales) % 16 == 0;
}

// The factors of U blocks (a power of two) of G neighbouring threads, which all have their largest magnitudes: every thread divides for one of them, a
// division being as much as a dozen other instructions.
template <int U, int G>
__device__ __forceinline__ void share_factors(unsigned threads, const uint32_t (&m)[U], Factors (&f)[U]) {
    const int lane = lane_id();
    uint32_t mine = m[0];
#pragma unroll
    for (int u = 1; u < U; ++u) mine = (lane & (U - 1)) == u ? m[u] : mine;
    const Factors own = factors_of(mine);
#pragma unroll
    for (int u = 0; u < U; ++u) {
        f[u].scale = __shfl_sync(threads, own.scale, (lane & (32 - G)) + u);
        f[u].inverse = __shfl_sync(threads, own.inverse, (lane & (32 - G)) + u);
    }
}

// Eight neighbouring codes.
template <typename T>
__device__ __forceinline__ uint2 codes8(const Eight<T> &v, float inverse) {
    return make_uint2(codes4(v.get(0), v.get(1), v.get(2), v.get(3), inverse), codes4(v.get(4), v.get(5), v.get(6), v.get(7), inverse));
}

// A thread's eighth of a block of 128 columns: 16 elements, a piece of the codes. What eight threads share costs half of what 16 would.
template <typename T>
struct Piece {
    Eight<T> lo, hi;

    template <int V>
    __device__ __forceinline__ void load(const T *row, int64_t c, int64_t cols) {
        lo.template load<V>(row, c, cols);
        hi.template load<V>(row, c + 8, cols);
    }
    // The block's largest magnitude; `threads`: its eight.
    __device__ __forceinline__ uint32_t top(unsigned threads) const {
        Top<T> t;
        t.add(lo), t.add(hi);
        t.join(threads, 4), t.join(threads, 2), t.join(threads, 1);
        return t.bits();
    }
    __device__ __forceinline__ uint4 codes(float inverse) const {
        const uint2 a = codes8(lo, inverse), b = codes8(hi, inverse);
        return make_uint4(a.x, a.y, b.x, b.y);
    }
};

}  // namespace nb200
