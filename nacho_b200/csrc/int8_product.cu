// Rows in 8-bit integers with a scale each, and products of them: y[i, n] = sa[i] sw[n] sum_k a[i, k] w[n, k], the sum in whole numbers.
#include "few_rows.cuh"
#include "tile_product.cuh"

namespace nb200 {
namespace {

constexpr int NT = 256;
constexpr float TOP_INT8 = 127.f;

int64_t pitch_of(int64_t cols) { return (cols + 31) / 32 * 32; }
int64_t all_rows(const nb200_int8 *m) { return (int64_t)m->groups * m->rows; }
bool int8_ok(const nb200_int8 *m) {
    return m && m->groups >= 0 && m->rows >= 0 && m->cols >= 0 && nb200_int8_value_count(m) >= 0 && (all_rows(m) == 0 || m->scales) &&
           (nb200_int8_value_count(m) == 0 || m->values) && reinterpret_cast<uintptr_t>(m->values) % 16 == 0 && reinterpret_cast<uintptr_t>(m->scales) % 4 == 0;
}

__device__ __forceinline__ uint32_t int_codes4(float a, float b, float c, float d, float inverse) {
    const int i0 = __float2int_rn(a * inverse), i1 = __float2int_rn(b * inverse), i2 = __float2int_rn(c * inverse), i3 = __float2int_rn(d * inverse);
    return __byte_perm(__byte_perm(i0, i1, 0x0040), __byte_perm(i2, i3, 0x0040), 0x5410);
}

// The largest magnitude of what THREADS neighbouring threads have (8, 32, or all of a CTA), for all of them.
template <int THREADS>
__device__ __forceinline__ uint32_t row_top(uint32_t mine) {
    if constexpr (THREADS == 8) {
        const unsigned eight = 0xffu << (threadIdx.x & 24);
#pragma unroll
        for (int d = 4; d; d >>= 1) mine = max(mine, __shfl_xor_sync(eight, mine, d));
        return mine;
    }
    mine = __reduce_max_sync(FULL_MASK, mine);
    if constexpr (THREADS == 32) return mine;
    __shared__ uint32_t top[NT / 32];
    if (lane_id() == 0) top[warp_id()] = mine;
    __syncthreads();
    mine = 0;
#pragma unroll
    for (int i = 0; i < NT / 32; ++i) mine = max(mine, top[i]);
    return mine;
}

// The factor of a row's codes, and its scale. A row that holds a NaN or an infinity stands for NaNs: its codes are zeros and its scale is none.
__device__ __forceinline__ float row_factor(uint32_t top, float *scale) {
    const bool finite = top < 0x7f800000u;
    const float largest = __uint_as_float(max(top, FLOOR8));
    *scale = finite ? __fdiv_rn(largest, TOP_INT8) : __uint_as_float(0x7fc00000u);
    return finite ? __fdiv_rn(TOP_INT8, largest) : 0.f;
}

// THREADS threads have a row: they read it for its largest magnitude and again, out of registers as far as KEEP pieces of 16 elements a thread go, for its
// codes. (32768 rows of 2048 by CTAs 64 us, by warps 30, a copy's time; 52620 rows of 128 by warps 13, by eighths of them 5.)
template <typename T, int V, int THREADS, int KEEP>
__global__ void __launch_bounds__(NT) k_int8_rows(const T *x, int64_t stride, int64_t rows, int64_t cols, int8_t *values, int64_t pitch, float *scales) {
    wait_for_previous();
    trigger_dependents();
    const int64_t r = (int64_t)blockIdx.x * (NT / THREADS) + threadIdx.x / THREADS;
    const int sub = threadIdx.x % THREADS;
    if (r >= rows) return;  // whole rows' threads
    const T *const row = x + r * stride;
    Piece<T> kept[KEEP];
    Top<T> m;
#pragma unroll
    for (int i = 0; i < KEEP; ++i) {
        kept[i].template load<V>(row, ((int64_t)i * THREADS + sub) * 16, cols);
        m.add(kept[i].lo), m.add(kept[i].hi);
    }
    if constexpr (THREADS == NT)
        for (int64_t c = ((int64_t)KEEP * THREADS + sub) * 16; c < cols; c += THREADS * 16) {
            Piece<T> p;
            p.template load<V>(row, c, cols);
            m.add(p.lo), m.add(p.hi);
        }
    float scale;
    const float factor = row_factor(row_top<THREADS>(m.bits()), &scale);
    if (sub == 0) scales[r] = scale;
    auto put = [&](const Piece<T> &p, int64_t c) {
        uint32_t w[4] = {0, 0, 0, 0};
        if (factor != 0.f) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                w[i] = int_codes4(p.lo.get(4 * i), p.lo.get(4 * i + 1), p.lo.get(4 * i + 2), p.lo.get(4 * i + 3), factor);
                w[2 + i] = int_codes4(p.hi.get(4 * i), p.hi.get(4 * i + 1), p.hi.get(4 * i + 2), p.hi.get(4 * i + 3), factor);
            }
        }
        *reinterpret_cast<uint4 *>(values + r * pitch + c) = make_uint4(w[0], w[1], w[2], w[3]);
    };
#pragma unroll
    for (int i = 0; i < KEEP; ++i) {
        const int64_t c = ((int64_t)i * THREADS + sub) * 16;
        if (c < pitch) put(kept[i], c);
    }
    if constexpr (THREADS == NT)
        for (int64_t c = ((int64_t)KEEP * THREADS + sub) * 16; c < pitch; c += THREADS * 16) {
            Piece<T> p;
            p.template load<V>(row, c, cols);
            put(p, c);
        }
}

// The same for rows that lie on no boundary: a thread has four elements at a time and KEEP fours in registers. (8192 rows of 8191 in 48 us, of 8192 in 32. With 16 elements
// in a row a thread, read one by one, they took 73; with each four taken apart before the next was asked for, 91.)
template <typename T, int THREADS, int KEEP>
__global__ void __launch_bounds__(NT) k_int8_rows_odd(const T *x, int64_t stride, int64_t rows, int64_t cols_, int8_t *values, int64_t pitch_, float *scales) {
    wait_for_previous();
    trigger_dependents();
    const int64_t r = (int64_t)blockIdx.x * (NT / THREADS) + threadIdx.x / THREADS;
    const uint32_t sub = threadIdx.x % THREADS, cols = (uint32_t)cols_, pitch = (uint32_t)pitch_;
    if (r >= rows) return;
    const T *const row = x + r * stride;
    int8_t *const codes = values + r * pitch_;
    float kept[KEEP][4];
    uint32_t m = 0;
    auto add = [&](const float (&v)[4]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
    };
    {
        Four<T> raw[KEEP];
#pragma unroll
        for (int u = 0; u < KEEP; ++u) raw[u].load(row, (sub + u * THREADS) * 4, cols);
#pragma unroll
        for (int u = 0; u < KEEP; ++u) {
            raw[u].get(row, kept[u]);
            add(kept[u]);
        }
    }
    auto later = [&](uint32_t c, float (&v)[4]) {
        Four<T> raw;
        raw.load(row, c, cols);
        raw.get(row, v);
    };
    const uint32_t rest = KEEP * THREADS * 4, turns = pitch > rest ? (pitch - rest + THREADS * 4 - 1) / (THREADS * 4) : 0;  // for whole warps
    for (uint32_t i = 0; i < turns; ++i) {
        float v[4];
        later(rest + (i * THREADS + sub) * 4, v);
        add(v);
    }
    float scale;
    const float factor = row_factor(row_top<THREADS>(m), &scale);
    if (sub == 0) scales[r] = scale;
    auto put = [&](uint32_t c, const float (&v)[4]) {
        if (c < pitch) *reinterpret_cast<uint32_t *>(codes + c) = factor != 0.f ? int_codes4(v[0], v[1], v[2], v[3], factor) : 0;
    };
#pragma unroll
    for (int u = 0; u < KEEP; ++u) put((sub + u * THREADS) * 4, kept[u]);
    for (uint32_t i = 0; i < turns; ++i) {
        float v[4];
        later(rest + (i * THREADS + sub) * 4, v);
        put(rest + (i * THREADS + sub) * 4, v);
    }
}

__global__ void __launch_bounds__(NT) k_int8_unpack(const int8_t *values, int64_t pitch, const float *scales, int64_t rows, int64_t cols, float *z) {
    wait_for_previous();
    trigger_dependents();
    const int64_t all = rows * cols;
    for (int64_t i = (int64_t)blockIdx.x * NT + threadIdx.x; i < all; i += (int64_t)gridDim.x * NT) {
        const int64_t r = i / cols;
        z[i] = (float)values[r * pitch + i - r * cols] * scales[r];
    }
}

}  // namespace
}  // namespace nb200

using namespace nb200;

extern "C" {

int64_t nb200_int8_pitch(const nb200_int8 *m) { return m && m->cols >= 0 ? pitch_of(m->cols) : -1; }

int64_t nb200_int8_value_count(const nb200_int8 *m) {
    if (!m || m->groups < 0 || m->rows < 0 || m->cols < 0) return -1;
    const int64_t rows = all_rows(m), pitch = pitch_of(m->cols);
    if (rows > 0 && pitch > INT64_MAX / rows) return -1;
    return rows * pitch;
}

int nb200_int8_quantise(const nb200_dense *x, nb200_int8 *z, void *stream_) {
    if (!dense_ok(x) || !int8_ok(z) || x->rows != all_rows(z) || x->cols != z->cols) return NB200_E_BADARG;
    if (x->rows == 0) return NB200_OK;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    if (x->rows > INT32_MAX) return NB200_E_UNSUPPORTED;
    return with_type(x->type, [&](auto e) {
        using T = decltype(e);
        return with_vector<T>(word_bytes({x}), [&](auto v) {
            constexpr int V = decltype(v)::value;
            auto go = [&](auto kernel, int64_t rows_each) -> int {
                LaunchScope scope("int8_rows", stream);
                NB200_CUDA(launch_overlapped(kernel, dim3((unsigned)((x->rows + rows_each - 1) / rows_each)), dim3(NT), 0, stream, static_cast<const T *>(x->data), x->stride, x->rows,
                                             x->cols, z->values, pitch_of(x->cols), z->scales));
                return NB200_OK;
            };
            // As few threads per row as hold it in registers.
            if constexpr (V == 1) {
                if (x->cols <= 1024) return go(k_int8_rows_odd<T, 32, 8>, NT / 32);
                return go(k_int8_rows_odd<T, NT, 8>, 1);
            } else {
                if (x->cols <= 256) return go(k_int8_rows<T, V, 8, 2>, NT / 8);
                if (x->cols <= 1024) return go(k_int8_rows<T, V, 32, 2>, NT / 32);
                if (x->cols <= 2048) return go(k_int8_rows<T, V, 32, 4>, NT / 32);
                return go(k_int8_rows<T, V, NT, sizeof(T) == 2 ? 2 : 1>, 1);
            }
        });
    });
}

int nb200_int8_pack(const int8_t *codes, const float *scales, nb200_int8 *z, void *stream_) {
    if (!int8_ok(z) || (all_rows(z) > 0 && !scales) || (nb200_int8_value_count(z) > 0 && !codes)) return NB200_E_BADARG;
    const int64_t rows = all_rows(z), cols = z->cols, pitch = pitch_of(cols);
    if (rows == 0) return NB200_OK;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    NB200_CUDA(cudaMemcpyAsync(z->scales, scales, (size_t)rows * sizeof(float), cudaMemcpyDeviceToDevice, stream));
    if (cols == 0) return NB200_OK;
    if (pitch > cols) NB200_CUDA(cudaMemset2DAsync(z->values + cols, (size_t)pitch, 0, (size_t)(pitch - cols), (size_t)rows, stream));
    NB200_CUDA(cudaMemcpy2DAsync(z->values, (size_t)pitch, codes, (size_t)cols, (size_t)cols, (size_t)rows, cudaMemcpyDeviceToDevice, stream));
    return NB200_OK;
}

int nb200_int8_unpack(const nb200_int8 *a, float *z, void *stream_) {
    if (!int8_ok(a) || (all_rows(a) > 0 && a->cols > 0 && !z)) return NB200_E_BADARG;
    const int64_t rows = all_rows(a);
    if (rows == 0 || a->cols == 0) return NB200_OK;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    LaunchScope scope("int8_unpack", stream);
    const int64_t ctas = std::min<int64_t>((rows * a->cols + NT - 1) / NT, sm_count() * 64ll);
    NB200_CUDA(launch_overlapped(k_int8_unpack, dim3((unsigned)ctas), dim3(NT), 0, stream, a->values, pitch_of(a->cols), a->scales, rows, a->cols, z));
    return NB200_OK;
}

static int int8_product(const nb200_int8 *a, const nb200_int8 *w, const int32_t *offsets, nb200_dense *y, bool starve, void *stream_) {
    if (!int8_ok(a) || !int8_ok(w) || !dense_ok(y) || a->groups != 1 || a->cols != w->cols || y->rows != a->rows || y->cols != w->rows || (!offsets && w->groups != 1)) return NB200_E_BADARG;
    if (w->groups > NB200_MAX_EXPERTS || a->cols > NB200_MAX_INT8_COLUMNS || a->rows > INT32_MAX - 1024 || w->rows > INT32_MAX / 2 - 1024) return NB200_E_UNSUPPORTED;
    if (y->rows == 0 || y->cols == 0) return NB200_OK;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    const int64_t stride = y->rows > 1 ? y->stride : y->cols, pitch = pitch_of(a->cols), groups = w->groups;
    int st;
    if (groups == 0 || a->cols == 0) {
        // nothing is summed; a row or a channel that stands for NaNs (its scale is one) is zeros too
        const size_t size = type_size(y->type);
        NB200_CUDA(cudaMemset2DAsync(y->data, (size_t)stride * size, 0, (size_t)y->cols * size, (size_t)y->rows, stream));
        return NB200_OK;
    }
    return with_type(y->type, [&](auto e) -> int {
        using T = decltype(e);
        if (!starve && few_rows(y->rows, groups, all_rows(w) * pitch, 1)) {
            const FewArgs args{a->values, w->values, pitch, pitch, offsets, w->groups, a->rows, w->rows, 16, (int)pitch, y->data, nullptr, stride, a->scales, w->scales, false};
            return launch_few_rows<Sum::S8, false, 16, T>("int8_few", args, stream);
        }
        TileMaps maps{};
        TileArgs args{};
        int clusters[2];
        if ((st = tile_clusters<Sum::S8, Form::ROWS, false, T>(clusters))) return st;
        args.offsets = offsets, args.groups = w->groups, args.rows = a->rows, args.wide = w->rows, args.blocks = (int)((a->cols + 127) / 128);
        args.pairs = (int)all_pairs();
        const TileWork::Way way = TileWork{a->rows, groups, (w->rows + TILE_M - 1) / TILE_M, args.blocks}.best(args.pairs, clusters);
        args.tile_n = way.n, args.parts = way.parts;
        if ((st = describe_rows(&maps.wide, CU_TENSOR_MAP_DATA_TYPE_UINT8, w->values, 1, pitch, w->rows, groups, pitch, 128)) ||
            (st = describe_narrow(&maps, &args, CU_TENSOR_MAP_DATA_TYPE_UINT8, a->values, 1, pitch, a->rows, pitch)) || (st = describe_result(&maps.y, &args.words, map_type(y->type), *y, 1)))
            return st;
        args.starve = starve;
        args.y = y->data, args.stride = stride, args.row_scale = a->scales, args.col_scale = w->scales;
        return launch_tiles<Sum::S8, Form::ROWS, false, T>("int8_product", args, maps, stream);
    });
}

int nb200_int8_product(const nb200_int8 *a, const nb200_int8 *w, const int32_t *offsets, nb200_dense *y, void *stream) { return int8_product(a, w, offsets, y, false, stream); }

int nb200_selftest_tiles_timeout(const nb200_int8 *a, const nb200_int8 *w, nb200_dense *y, void *stream) { return int8_product(a, w, nullptr, y, true, stream); }

}  // extern "C"
