// The norm over many tensors, and their elements scaled by it: norm = sqrt(sum x^2), z = x min(1, max_norm / (norm + 1e-6)).
//
// Device memory bounds it: what is larger than L2 is read twice and written once (500 M 16-bit elements 498 us, 3 GB at 0.92 of a copy). Two kernels per 512
// tensors: one sums squares, a double per CTA; the other adds those up, every CTA for itself and in the same order (a few KB out of L2, which needs neither an
// atomic nor a cleared counter), and scales. It goes through the tensors from the last to the first, so that what the first kernel has read last comes from L2.
#include <algorithm>
#include <cmath>

#include "dense_rows.cuh"

namespace nb200 {
namespace {

constexpr int NT = 256, TURNS = 4;              // threads; 16-byte chunks that a thread has on its way
constexpr int CHUNK_BYTES = NT * TURNS * 16;    // what a CTA takes at a time, of the elements' own type
// CTAs that are at work at once (500 M elements: summed 161 us, with eight per SM 167; scaled 345 us with four, 325 with eight).
int sum_ctas() { return 4 * sm_count(); }
int scale_ctas() { return 8 * sm_count(); }

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

// The tensor that a chunk belongs to.
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

// What a thread has of a CTA's chunk: TURNS pieces of V elements, a CTA's width apart, of the `count` elements from `from` on. The words are kept whole: as
// elements of 16 bits they would take a register each, and spill.
template <typename T, int V>
struct Mine {
    static constexpr int STEP = NT * V, WORDS = V * (int)sizeof(T) < 4 ? 1 : V * (int)sizeof(T) / 4;
    uint32_t w[TURNS][WORDS];

    __device__ __forceinline__ void load(const T *from, int at, int count) {
#pragma unroll
        for (int u = 0; u < TURNS; ++u) {
            Vec<uint32_t, WORDS> in{};
            if (at + u * STEP < count) {
                if constexpr (V * sizeof(T) == 2) in.v[0] = *reinterpret_cast<const uint16_t *>(from + at + u * STEP);
                else in = *reinterpret_cast<const Vec<uint32_t, WORDS> *>(from + at + u * STEP);
            }
#pragma unroll
            for (int i = 0; i < WORDS; ++i) w[u][i] = in.v[i];
        }
    }
    __device__ __forceinline__ float get(int u, int i) const {
        if constexpr (sizeof(T) == 4) return __uint_as_float(w[u][i]);
        else if constexpr (std::is_same<T, __half>::value) return __half2float(__ushort_as_half((unsigned short)(i & 1 ? w[u][i / 2] >> 16 : w[u][i / 2])));
        else return __uint_as_float(i & 1 ? w[u][i / 2] & 0xffff0000u : w[u][i / 2] << 16);
    }
    // The sum of the squares: in 32 bits, unless those run over or lose what there is.
    __device__ __forceinline__ double squares() const {
        float part[TURNS] = {};
#pragma unroll
        for (int u = 0; u < TURNS; ++u)
#pragma unroll
            for (int i = 0; i < V; ++i) part[u] = __fmaf_rn(get(u, i), get(u, i), part[u]);
        const float sum = (part[0] + part[1]) + (part[2] + part[3]);
        if (sum > 0x1p-90f && sum < 0x1p126f) return sum;
        double exact = 0.0;
#pragma unroll
        for (int u = 0; u < TURNS; ++u)
#pragma unroll
            for (int i = 0; i < V; ++i) exact += (double)get(u, i) * (double)get(u, i);
        return exact;
    }
    // Elements go over times the factor (1 changes none of them).
    template <typename Z>
    __device__ __forceinline__ void store(Z *to, int at, int count, float factor) const {
#pragma unroll
        for (int u = 0; u < TURNS; ++u) {
            if (at + u * STEP >= count) break;
            Z *const z = to + at + u * STEP;
            if constexpr (V == 1) {
                z[0] = from_float<Z>(get(u, 0) * factor);
            } else if constexpr (sizeof(Z) == 4) {
#pragma unroll
                for (int i = 0; i < V; i += 4)
                    __stcs(reinterpret_cast<float4 *>(z + i), make_float4(get(u, i) * factor, get(u, i + 1) * factor, get(u, i + 2) * factor, get(u, i + 3) * factor));
            } else {
                Vec<uint32_t, V / 2> out;
#pragma unroll
                for (int i = 0; i < V; i += 2) out.v[i / 2] = pack2<Z>(get(u, i) * factor, get(u, i + 1) * factor);
                if constexpr (V == 8) __stcs(reinterpret_cast<uint4 *>(z), make_uint4(out.v[0], out.v[1], out.v[2], out.v[3]));
                else __stcs(reinterpret_cast<uint2 *>(z), make_uint2(out.v[0], out.v[1]));
            }
        }
    }
};
static_assert(TURNS == 4, "");

template <typename F>
__device__ __forceinline__ void with_type_of(int type, F f) {
    if (type == NB200_F32) f(float{});
    else if (type == NB200_F16) f(__half{});
    else f(__nv_bfloat16{});
}

// A chunk of a tensor, by words of V elements and behind the last whole one of the tensor by single elements: f(Mine, where in the chunk, up to where).
template <typename T, int V, typename F>
__device__ __forceinline__ void with_chunk(const T *from, int count, F f) {
    const int whole = count / V * V;
#pragma unroll 1
    for (int at = threadIdx.x * V; at < whole; at += TURNS * Mine<T, V>::STEP) {
        Mine<T, V> mine;
        mine.load(from, at, whole);
        f(mine, at, whole);
    }
    if (V > 1 && (int)threadIdx.x < count - whole) {
        Mine<T, 1> mine;
        mine.load(from, whole + threadIdx.x, whole + threadIdx.x + 1);
        f(mine, whole + (int)threadIdx.x, whole + (int)threadIdx.x + 1);
    }
}
template <typename T>
__device__ __forceinline__ double sum_chunk(const T *from, int count, bool words) {
    double sum = 0.0;
    auto add = [&](const auto &mine, int, int) { sum += mine.squares(); };
    if (words) with_chunk<T, 16 / sizeof(T)>(from, count, add);
    else with_chunk<T, 1>(from, count, add);
    return sum;
}
template <typename T, typename Z>
__device__ __forceinline__ void scale_chunk(const T *from, Z *to, int count, bool words, float factor) {
    auto put = [&](const auto &mine, int at, int stop) { mine.store(to, at, stop, factor); };
    if (words) with_chunk<T, 16 / sizeof(T)>(from, count, put);
    else with_chunk<T, 1>(from, count, put);
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

// Neighbouring CTAs have neighbouring chunks, and all of them move through the tensors together: with ranges of their own, reads and writes of 1184
// places at once, scaling 500 M elements took 493 us.
template <int N>
__global__ void __launch_bounds__(NT, 4) k_squares(const __grid_constant__ Spans<N> s, double *partial) {
    __shared__ double tmp[NT / 32];
    trigger_dependents();
    wait_for_previous();
    double sum = 0.0;
    const int chunks = s.first[s.n];
    int k = span_of(s, blockIdx.x);
    for (int chunk = blockIdx.x; chunk < chunks; chunk += gridDim.x) {
        while (s.first[k + 1] <= chunk) ++k;
        with_type_of(s.type[k], [&](auto e) {
            using T = decltype(e);
            constexpr int64_t EACH = CHUNK_BYTES / sizeof(T);
            const int64_t at = (chunk - s.first[k]) * EACH;
            sum += sum_chunk(static_cast<const T *>(s.from[k]) + at, (int)min(EACH, s.count[k] - at), s.words[k]);
        });
    }
    sum = cta_sum(sum, tmp);
    if (threadIdx.x == 0) partial[blockIdx.x] = sum;
}

template <int N>
__global__ void __launch_bounds__(NT, 8) k_scale(const __grid_constant__ Spans<N> s, const double *partial, int partials, float max_norm, float *norm) {
    __shared__ double tmp[NT / 32];
    trigger_dependents();
    wait_for_previous();
    double sum = 0.0;
    for (int i = threadIdx.x; i < partials; i += NT) sum += ld_late(partial + i);
    sum = cta_sum(sum, tmp);
    const float root = (float)sqrt(sum), wanted = __fdiv_rn(max_norm, root + 1e-6f);
    const float factor = root < __uint_as_float(0x7f800000u) && wanted < 1.f ? wanted : 1.f;
    if (blockIdx.x == 0 && threadIdx.x == 0) *norm = root;
    int chunk = s.first[s.n] - 1 - (int)blockIdx.x;
    if (chunk < 0) return;
    for (int k = span_of(s, chunk); chunk >= 0; chunk -= gridDim.x) {
        while (s.first[k] > chunk) --k;
        if (factor == 1.f && s.from[k] == s.to[k]) continue;
        with_type_of(s.type[k], [&](auto e) {
            using T = decltype(e);
            constexpr int64_t EACH = CHUNK_BYTES / sizeof(T);
            const int64_t at = (chunk - s.first[k]) * EACH;
            const T *const from = static_cast<const T *>(s.from[k]) + at;
            const int count = (int)min(EACH, s.count[k] - at);
            with_type_of(s.to_type[k], [&](auto z) { scale_chunk(from, static_cast<decltype(z) *>(s.to[k]) + at, count, s.words[k], factor); });
        });
    }
}

constexpr int FEW = 32, SOME = 128, MANY = 512;  // tensors of a launch: what its parameters hold is copied with it

// With a pointer to the tensors: passed by value they are copied three times on the way, 14 KB of them in a microsecond each.
int launch_spans(const char *name, const void *kernel, int ctas, void **args, cudaStream_t stream) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)ctas), cfg.blockDim = dim3(NT), cfg.stream = stream;
    cudaLaunchAttribute early{};
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &early, cfg.numAttrs = 1;
    LaunchScope scope(name, stream);
    NB200_CUDA(cudaLaunchKernelExC(&cfg, kernel, args));
    return NB200_OK;
}

bool span_ok(const nb200_span &s) {
    if (s.count < 0 || s.type < NB200_F32 || s.type > NB200_BF16 || s.to_type < NB200_F32 || s.to_type > NB200_BF16) return false;
    if (s.count == 0) return true;
    return s.from && s.to && (reinterpret_cast<uintptr_t>(s.from) & (type_size(s.type) - 1)) == 0 && (reinterpret_cast<uintptr_t>(s.to) & (type_size(s.to_type) - 1)) == 0 &&
           (s.from != s.to || s.type == s.to_type);
}

int64_t launches_of(int64_t n) { return n <= SOME ? 1 : (n + MANY - 1) / MANY; }

template <int N>
int clip(const nb200_span *spans, int64_t n, float max_norm, float *norm, double *partial, cudaStream_t stream) {
    const int64_t launches = std::max<int64_t>(1, (n + N - 1) / N);
    auto fill = [&](int64_t l, Spans<N> &s) {
        s.n = (int)std::min<int64_t>(N, n - l * N);
        int64_t chunks = 0;
        for (int i = 0; i < s.n; ++i) {
            const nb200_span &x = spans[l * N + i];
            s.from[i] = x.from, s.to[i] = x.to, s.count[i] = x.count, s.type[i] = (uint8_t)x.type, s.to_type[i] = (uint8_t)x.to_type;
            s.words[i] = reinterpret_cast<uintptr_t>(x.from) % 16 == 0 && reinterpret_cast<uintptr_t>(x.to) % 16 == 0;
            s.first[i] = (int32_t)chunks;
            chunks += x.type == NB200_F32 ? (x.count + chunk_elements(NB200_F32) - 1) / chunk_elements(NB200_F32) : (x.count + chunk_elements(NB200_F16) - 1) / chunk_elements(NB200_F16);
            if (chunks > INT32_MAX) return (int)NB200_E_UNSUPPORTED;
        }
        for (int i = s.n; i <= N; ++i) s.first[i] = (int32_t)chunks;
        return (int)NB200_OK;
    };
    int partials = 0, st;
    Spans<N> s;
    for (int64_t l = 0; l < launches; ++l) {
        if ((st = fill(l, s))) return st;
        const int ctas = std::max(1, std::min(s.first[N], sum_ctas()));
        double *const at = partial + partials;
        void *args[] = {&s, const_cast<double **>(&at)};
        if ((st = launch_spans("clip_squares", reinterpret_cast<const void *>(k_squares<N>), ctas, args, stream))) return st;
        partials += ctas;
    }
    for (int64_t l = launches - 1; l >= 0; --l) {
        if (launches > 1) fill(l, s);
        const double *const sums = partial;
        void *args[] = {&s, const_cast<const double **>(&sums), &partials, &max_norm, &norm};
        if ((st = launch_spans("clip_scale", reinterpret_cast<const void *>(k_scale<N>), std::max(1, std::min(s.first[N], scale_ctas())), args, stream))) return st;
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
    return std::max<int64_t>(1, launches_of(n)) * sum_ctas() * (int64_t)sizeof(double);
}

int nb200_clip(const nb200_span *spans, int64_t n, float max_norm, float *norm, void *scratch, int64_t scratch_bytes, void *stream_) {
    const int64_t bytes = nb200_clip_scratch(spans, n);
    if (bytes < 0 || !norm || !(max_norm >= 0.f) || !scratch || reinterpret_cast<uintptr_t>(scratch) % 256 != 0) return NB200_E_BADARG;
    if (scratch_bytes < bytes) return NB200_E_CAPACITY;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    double *partial = static_cast<double *>(scratch);
    if (n <= FEW) return clip<FEW>(spans, n, max_norm, norm, partial, stream);
    return n <= SOME ? clip<SOME>(spans, n, max_norm, norm, partial, stream) : clip<MANY>(spans, n, max_norm, norm, partial, stream);
}

}  // extern "C"
