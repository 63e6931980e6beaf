// The norm over many tensors, and their elements scaled by it: norm = sqrt(sum x^2), z = x min(1, max_norm / (norm + 1e-6)).
//
// Device memory bounds it: what is larger than L2 is read twice and written once. Two kernels per 512 tensors: one sums squares, a double per CTA; the
// other adds those up, every CTA for itself and in the same order (a few KB out of L2, which needs neither an atomic nor a cleared counter), and scales. It goes
// through the tensors from the last to the first, so that what the first kernel has read last comes from L2.
#include <algorithm>
#include <cmath>

#include "dense_rows.cuh"

namespace nb200 {
namespace {

constexpr int NT = 256, TURNS = 4;              // threads; 16-byte chunks that a thread has on its way
constexpr int CHUNK_BYTES = NT * TURNS * 16;    // what a CTA takes at a time, of the elements' own type
constexpr int MAX_CTAS = 4 * 148 * 2;           // partial sums of a launch

// A launch's tensors lie in its parameters: a captured graph has them with it.
template <int N>
struct Spans {
    const void *from[N];
    void *to[N];
    int64_t count[N];
    int32_t first[N + 1];  // chunks of the tensors in front
    uint8_t type[N], to_type[N], words[N];
    int n;
};

__host__ __device__ constexpr int64_t chunk_elements(int type) { return CHUNK_BYTES / (type == NB200_F32 ? 4 : 2); }

// The tensor that a chunk belongs to; `at`: one that lies in front of it or is it.
template <int N>
__device__ __forceinline__ int span_of(const Spans<N> &s, int chunk) {
    int lo = 0, hi = s.n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (s.first[mid] <= chunk) lo = mid;
        else hi = mid;
    }
    return lo;
}

// Squares of N elements: in 32 bits, unless those run over or lose what there is.
template <typename T, int V>
__device__ __forceinline__ double squares(const Chunk<T, V> (&x)[TURNS], int64_t c, int64_t step, int64_t pitch, int64_t count) {
    constexpr int N = Chunk<T, V>::N;
    float sum = 0.f;
#pragma unroll
    for (int u = 0; u < TURNS; ++u)
        if (c + u * step < count) {
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (Chunk<T, V>::there(i, c + u * step, pitch, count)) sum = __fmaf_rn(x[u].get(i), x[u].get(i), sum);
        }
    if (sum > 0x1p-90f && sum < 0x1p126f) return sum;
    double exact = 0.0;
#pragma unroll
    for (int u = 0; u < TURNS; ++u)
        if (c + u * step < count) {
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (Chunk<T, V>::there(i, c + u * step, pitch, count)) exact += (double)x[u].get(i) * (double)x[u].get(i);
        }
    return exact;
}

// A CTA's chunk as its threads have it: TURNS words (or several, of V elements, a CTA's width apart) each.
template <typename T, int V, typename F>
__device__ __forceinline__ void with_chunk(const T *from, int64_t begin, int64_t count, F f) {
    constexpr int64_t pitch = (int64_t)NT * V, step = (int64_t)NT * Chunk<T, V>::N;
    const int64_t c = begin + (int64_t)threadIdx.x * V;
    Chunk<T, V> x[TURNS];
#pragma unroll
    for (int u = 0; u < TURNS; ++u)
        if (c + u * step < count) x[u].load(from, c + u * step, pitch, count);
    f(x, c, step, pitch);
}

template <typename F>
__device__ __forceinline__ void with_span(int type, bool words, F f) {
    if (type == NB200_F32) words ? f(float{}, std::integral_constant<int, 4>{}) : f(float{}, std::integral_constant<int, 1>{});
    else if (type == NB200_F16) words ? f(__half{}, std::integral_constant<int, 8>{}) : f(__half{}, std::integral_constant<int, 1>{});
    else words ? f(__nv_bfloat16{}, std::integral_constant<int, 8>{}) : f(__nv_bfloat16{}, std::integral_constant<int, 1>{});
}

__device__ __forceinline__ double cta_sum(double v, double *tmp) {
#pragma unroll
    for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(FULL_MASK, v, d);
    if (lane_id() == 0) tmp[warp_id()] = v;
    __syncthreads();
    v = 0.0;
#pragma unroll
    for (int i = 0; i < NT / 32; ++i) v += tmp[i];
    return v;
}

template <int N>
__global__ void __launch_bounds__(NT, 4) k_squares(const __grid_constant__ Spans<N> s, double *partial) {
    __shared__ double tmp[NT / 32];
    trigger_dependents();
    wait_for_previous();
    double sum = 0.0;
    const int chunks = s.first[s.n];
    for (int chunk = blockIdx.x; chunk < chunks; chunk += gridDim.x) {
        const int k = span_of(s, chunk);
        with_span(s.type[k], s.words[k], [&](auto e, auto v) {
            using T = decltype(e);
            const int64_t count = s.count[k];
            with_chunk<T, decltype(v)::value>(static_cast<const T *>(s.from[k]), (chunk - s.first[k]) * chunk_elements(s.type[k]), count,
                                              [&](auto &x, int64_t c, int64_t step, int64_t pitch) { sum += squares(x, c, step, pitch, count); });
        });
    }
    sum = cta_sum(sum, tmp);
    if (threadIdx.x == 0) partial[blockIdx.x] = sum;
}

template <int N>
__global__ void __launch_bounds__(NT, 4) k_scale(const __grid_constant__ Spans<N> s, const double *partial, int partials, float max_norm, float *norm) {
    __shared__ double tmp[NT / 32];
    trigger_dependents();
    wait_for_previous();
    double sum = 0.0;
    for (int i = threadIdx.x; i < partials; i += NT) sum += ld_late(partial + i);
    sum = cta_sum(sum, tmp);
    const float root = (float)sqrt(sum), wanted = __fdiv_rn(max_norm, root + 1e-6f);
    const float factor = root < __uint_as_float(0x7f800000u) && wanted < 1.f ? wanted : 1.f;
    if (blockIdx.x == 0 && threadIdx.x == 0 && norm) *norm = root;
    const int chunks = s.first[s.n];
    for (int chunk = chunks - 1 - blockIdx.x; chunk >= 0; chunk -= gridDim.x) {
        const int k = span_of(s, chunk);
        if (factor == 1.f && s.from[k] == s.to[k]) continue;
        with_span(s.type[k], s.words[k], [&](auto e, auto v) {
            using T = decltype(e);
            constexpr int V = decltype(v)::value;
            const int64_t count = s.count[k];
            with_chunk<T, V>(static_cast<const T *>(s.from[k]), (chunk - s.first[k]) * chunk_elements(s.type[k]), count, [&](auto &x, int64_t c, int64_t step, int64_t pitch) {
                auto each = [&](auto put) {
#pragma unroll
                    for (int u = 0; u < TURNS; ++u)
                        if (c + u * step < count) {
#pragma unroll
                            for (int i = 0; i < Chunk<T, V>::N; ++i)
                                if (Chunk<T, V>::there(i, c + u * step, pitch, count)) put(u, i, factor == 1.f ? x[u].get(i) : x[u].get(i) * factor);
                        }
                };
                if (s.to_type[k] == s.type[k]) {
                    if (factor != 1.f) each([&](int u, int i, float f) { x[u].set(i, f); });
#pragma unroll
                    for (int u = 0; u < TURNS; ++u)
                        if (c + u * step < count) x[u].store(static_cast<T *>(s.to[k]), c + u * step, pitch, count);
                } else {
                    auto at = [&](int u, int i) { return c + u * step + i / V * pitch + i % V; };
                    if (s.to_type[k] == NB200_F32) each([&](int u, int i, float f) { static_cast<float *>(s.to[k])[at(u, i)] = f; });
                    else if (s.to_type[k] == NB200_F16) each([&](int u, int i, float f) { static_cast<__half *>(s.to[k])[at(u, i)] = __float2half_rn(f); });
                    else each([&](int u, int i, float f) { static_cast<__nv_bfloat16 *>(s.to[k])[at(u, i)] = __float2bfloat16_rn(f); });
                }
            });
        });
    }
}

constexpr int FEW = 32, MANY = 512;

bool span_ok(const nb200_span &s) {
    if (s.count < 0 || s.type < NB200_F32 || s.type > NB200_BF16 || s.to_type < NB200_F32 || s.to_type > NB200_BF16) return false;
    if (s.count == 0) return true;
    return s.from && s.to && reinterpret_cast<uintptr_t>(s.from) % type_size(s.type) == 0 && reinterpret_cast<uintptr_t>(s.to) % type_size(s.to_type) == 0 &&
           (s.from != s.to || s.type == s.to_type);
}

int64_t launches_of(int64_t n) { return n <= FEW ? 1 : (n + MANY - 1) / MANY; }

template <int N>
int clip(const nb200_span *spans, int64_t n, float max_norm, float *norm, double *partial, cudaStream_t stream) {
    const int64_t launches = std::max<int64_t>(1, (n + N - 1) / N);
    auto fill = [&](int64_t l, Spans<N> &s) {
        s.n = (int)std::min<int64_t>(N, n - l * N);
        int64_t chunks = 0;
        for (int i = 0; i < s.n; ++i) {
            const nb200_span &x = spans[l * N + i];
            s.from[i] = x.from, s.to[i] = x.to, s.count[i] = x.count, s.type[i] = (uint8_t)x.type, s.to_type[i] = (uint8_t)x.to_type;
            // words of 16 bytes; the last one need not be whole if the next element is where another word would begin
            const bool even = x.count * type_size(x.type) % 16 == 0 && reinterpret_cast<uintptr_t>(x.from) % 16 == 0;
            s.words[i] = even && (x.type != x.to_type || reinterpret_cast<uintptr_t>(x.to) % 16 == 0);
            s.first[i] = (int32_t)chunks;
            chunks += (x.count + chunk_elements(x.type) - 1) / chunk_elements(x.type);
            if (chunks > INT32_MAX) return (int)NB200_E_UNSUPPORTED;
        }
        for (int i = s.n; i <= N; ++i) s.first[i] = (int32_t)chunks;
        return (int)NB200_OK;
    };
    int partials = 0, st;
    Spans<N> s;
    for (int64_t l = 0; l < launches; ++l) {
        if ((st = fill(l, s))) return st;
        const int ctas = std::max(1, std::min(s.first[N], MAX_CTAS));
        LaunchScope scope("clip_squares", stream);
        NB200_CUDA(launch_overlapped(k_squares<N>, dim3((unsigned)ctas), dim3(NT), 0, stream, s, partial + partials));
        partials += ctas;
    }
    for (int64_t l = launches - 1; l >= 0; --l) {
        if (launches > 1) fill(l, s);
        LaunchScope scope("clip_scale", stream);
        NB200_CUDA(launch_overlapped(k_scale<N>, dim3((unsigned)std::max(1, std::min(s.first[N], MAX_CTAS))), dim3(NT), 0, stream, s, partial, partials, max_norm, norm));
    }
    return NB200_OK;
}

}  // namespace
}  // namespace nb200

using namespace nb200;

extern "C" {

int64_t nb200_clip_scratch(const nb200_span *spans, int64_t n) {
    if (n < 0 || (n > 0 && !spans) || n > INT32_MAX) return -1;
    for (int64_t i = 0; i < n; ++i)
        if (!span_ok(spans[i])) return -1;
    return std::max<int64_t>(1, launches_of(n)) * MAX_CTAS * (int64_t)sizeof(double);
}

int nb200_clip(const nb200_span *spans, int64_t n, float max_norm, float *norm, void *scratch, int64_t scratch_bytes, void *stream_) {
    const int64_t bytes = nb200_clip_scratch(spans, n);
    if (bytes < 0 || !norm || !(max_norm >= 0.f) || !scratch || reinterpret_cast<uintptr_t>(scratch) % 256 != 0) return NB200_E_BADARG;
    if (scratch_bytes < bytes) return NB200_E_CAPACITY;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    double *partial = static_cast<double *>(scratch);
    return n <= FEW ? clip<FEW>(spans, n, max_norm, norm, partial, stream) : clip<MANY>(spans, n, max_norm, norm, partial, stream);
}

}  // extern "C"
