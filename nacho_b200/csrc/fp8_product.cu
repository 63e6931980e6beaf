// Products of 8-bit matrices with a scale per block of 128:
//     y[i, n] = sum_b sa[i, b] sw[n / 128, b] sum_{k in block b} a[i, k] w[n, k],
// all rows by one matrix or every group of rows by its own, and the gradient for the weights of the latter,
//     z[g][n, k] = sum_b sd[n, b] sx[k, b] sum_{i in block b} dy[i, n] x[i, k],   b over blocks of 128 rows of group g.
#include <algorithm>
#include <type_traits>

#include "dense_rows.cuh"

namespace nb200 {
namespace {

constexpr int NT = 256;

// An operand: [group][block][row][128 codes], and where the scale of (group, block, row) lies.
struct Operand {
    const uint8_t *values;
    const float *scales;
    int64_t blocks, pad;        // per group; rows to a multiple of 8
    int64_t scale_pitch;        // scales per block
    int scale_shift;            // rows per scale, as a power of two

    __device__ const uint8_t *block(int64_t g, int64_t b) const { return values + (g * blocks + b) * pad * BLOCK8; }
    __device__ float scale(int64_t g, int64_t b, int64_t r) const { return ld_late(scales + (g * blocks + b) * scale_pitch + (r >> scale_shift)); }
};

__device__ __forceinline__ float2 pair_of(uint32_t two) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(two & 0xffff), __NV_E4M3);
    return __half22float2(__half2(h));
}

// Sum over one block of 128.
__device__ float dot128(const uint8_t *a, int64_t ra, const uint8_t *b, int64_t rb) {
    float sum = 0.f;
    for (int p = 0; p < 8; ++p) {
        const uint4 qa = *reinterpret_cast<const uint4 *>(a + piece_at(ra, p)), qb = *reinterpret_cast<const uint4 *>(b + piece_at(rb, p));
        const uint32_t wa[4] = {qa.x, qa.y, qa.z, qa.w}, wb[4] = {qb.x, qb.y, qb.z, qb.w};
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float2 u = pair_of(wa[j / 2] >> (j % 2 * 16)), v = pair_of(wb[j / 2] >> (j % 2 * 16));
            sum = __fmaf_rn(u.x, v.x, sum);
            sum = __fmaf_rn(u.y, v.y, sum);
        }
    }
    return sum;
}

// A thread per element of the result.
template <typename T>
__global__ void __launch_bounds__(NT) k_product_simple(Operand a, Operand w, const int32_t *offsets, int groups, int64_t rows, int64_t cols, T *y, int64_t stride) {
    wait_for_previous();
    trigger_dependents();
    const int64_t all = rows * cols;
    for (int64_t i = (int64_t)blockIdx.x * NT + threadIdx.x; i < all; i += (int64_t)gridDim.x * NT) {
        const int64_t r = i / cols, n = i - r * cols;
        int g = 0;
        if (offsets) {
            while (g < groups && ld_late(offsets + g + 1) <= r) ++g;
            if (r < ld_late(offsets)) g = groups;
        }
        float sum = 0.f;
        if (g < groups)
            for (int64_t b = 0; b < a.blocks; ++b) sum = __fmaf_rn(a.scale(0, b, r) * w.scale(g, b, n), dot128(a.block(0, b), r, w.block(g, b), n), sum);
        y[r * stride + n] = from_float<T>(sum);
    }
}

__global__ void __launch_bounds__(NT) k_grad_w_simple(Operand d, Operand x, const int32_t *first_block, int groups, int64_t rows, int64_t cols, float *z) {
    wait_for_previous();
    trigger_dependents();
    const int64_t all = groups * rows * cols;
    for (int64_t i = (int64_t)blockIdx.x * NT + threadIdx.x; i < all; i += (int64_t)gridDim.x * NT) {
        const int64_t g = i / (rows * cols), n = i / cols % rows, k = i % cols;
        float sum = 0.f;
        for (int64_t b = ld_late(first_block + g); b < ld_late(first_block + g + 1); ++b)
            sum = __fmaf_rn(d.scale(0, b, n) * x.scale(0, b, k), dot128(d.block(0, b), n, x.block(0, b), k), sum);
        z[i] = sum;
    }
}

// ---- operands of the gradient ------------------------------------------------------------

// Blocks of 128 rows, counted from each group's first: where a group's blocks begin, and every block's rows {first, how many}. One CTA.
__global__ void __launch_bounds__(1024) k_group_blocks(const int32_t *offsets, int groups, int rows, int bound, int32_t *first_block, int2 *block) {
    __shared__ int tmp[33];
    wait_for_previous();
    trigger_dependents();
    int base = 0;
    for (int g0 = 0; g0 < groups; g0 += 1024) {
        const int g = g0 + threadIdx.x;
        int from = 0, to = 0;
        if (g < groups) {
            from = offsets ? min(max(ld_late(offsets + g), 0), rows) : 0;
            to = offsets ? min(max(ld_late(offsets + g + 1), from), rows) : rows;
        }
        int sum;
        const int at = base + block_excl_sum<1024>((to - from + BLOCK8 - 1) / BLOCK8, tmp, sum);
        if (g < groups) {
            first_block[g] = min(at, bound);
            for (int b = 0; from + b * BLOCK8 < to && at + b < bound; ++b) block[at + b] = make_int2(from + b * BLOCK8, min(BLOCK8, to - from - b * BLOCK8));
        }
        base += sum;
    }
    if (threadIdx.x == 0) first_block[groups] = min(base, bound);
    for (int b = base + threadIdx.x; b < bound; b += 1024) block[b] = make_int2(0, 0);
}

// x by blocks of rows: column c becomes row c of the result, a scale for it per block. A CTA per block and 128 columns.
template <typename T, int V>
__global__ void __launch_bounds__(NT) k_fp8_columns(const T *x, int64_t stride, int64_t cols, const int2 *block, uint8_t *values, float *scales) {
    extern __shared__ unsigned char raw[];
    constexpr int PITCH = BLOCK8 + 4 / sizeof(T);  // a word more: both directions without conflicts
    T *tile = reinterpret_cast<T *>(raw);
    wait_for_previous();
    trigger_dependents();
    const int64_t chunks = blocks_of(cols), b = blockIdx.x / chunks, c0 = blockIdx.x % chunks * BLOCK8, pad = padded_rows(cols);
    const int2 rows = *(block + b);
    if (rows.y == 0) return;
    for (int i = threadIdx.x; i < BLOCK8 * (BLOCK8 / V); i += NT) {
        const int r = i / (BLOCK8 / V), c = i % (BLOCK8 / V) * V;
        Vec<T, V> v;
        if (r < rows.y && c0 + c < cols) {
            v = *reinterpret_cast<const Vec<T, V> *>(x + (int64_t)(rows.x + r) * stride + c0 + c);
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) v.v[j] = from_float<T>(0.f);
        }
#pragma unroll
        for (int j = 0; j < V; ++j) tile[r * PITCH + c + j] = v.v[j];
    }
    __syncthreads();
    // two threads per column, 64 rows each, in different halves of a warp's pairs
    const int c = threadIdx.x / 2, part = threadIdx.x & 1;
    uint32_t m = 0;
    for (int r = 0; r < 64; ++r) m = max(m, magnitude(to_float(tile[(part * 64 + r) * PITCH + c])));
    m = max(m, __shfl_xor_sync(FULL_MASK, m, 1));
    const Factors f = factors_of(m);
    if (c0 + c >= cols) return;
    uint8_t *to = values + b * pad * BLOCK8;
    for (int p = 0; p < 4; ++p) {
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const T *at = tile + (part * 64 + p * 16 + j * 4) * PITCH + c;
            w[j] = codes4(to_float(at[0]), to_float(at[PITCH]), to_float(at[2 * PITCH]), to_float(at[3 * PITCH]), f.inverse);
        }
        *reinterpret_cast<uint4 *>(to + piece_at(c0 + c, part * 4 + p)) = make_uint4(w[0], w[1], w[2], w[3]);
    }
    if (part == 0) scales[b * pad + c0 + c] = f.scale;
}

// ---- host ------------------------------------------------------------------------------

dim3 grid_of(int64_t ctas) { return dim3((unsigned)std::max<int64_t>(1, std::min<int64_t>(ctas, 148 * 64))); }

struct GradScratch {
    int32_t *first_block;
    int2 *block;
    uint8_t *d, *x;
    float *ds, *xs;
    size_t bytes;
    int64_t bound;  // blocks at most

    GradScratch(void *base, const nb200_dense *dy, const nb200_dense *xx, int32_t groups) {
        Carver c(base);
        bound = dy->rows / BLOCK8 + groups;
        first_block = c.take<int32_t>((size_t)groups + 1);
        block = c.take<int2>((size_t)bound);
        d = c.take<uint8_t>((size_t)(bound * padded_rows(dy->cols) * BLOCK8));
        ds = c.take<float>((size_t)(bound * padded_rows(dy->cols)));
        x = c.take<uint8_t>((size_t)(bound * padded_rows(xx->cols) * BLOCK8));
        xs = c.take<float>((size_t)(bound * padded_rows(xx->cols)));
        bytes = c.used();
    }
};

bool grad_ok(const nb200_dense *dy, const nb200_dense *x, int32_t groups) {
    return dense_ok(dy) && dense_ok(x) && dy->rows == x->rows && dy->type == x->type && groups >= 0 && dy->rows <= INT32_MAX - BLOCK8 && dy->cols <= INT32_MAX && x->cols <= INT32_MAX;
}

int quantise_columns(const nb200_dense *x, const int2 *block, int64_t bound, uint8_t *values, float *scales, cudaStream_t stream) {
    const int64_t ctas = bound * blocks_of(x->cols);
    if (ctas == 0) return NB200_OK;
    if (ctas > INT32_MAX) return NB200_E_UNSUPPORTED;
    return with_type(x->type, [&](auto e) {
        using T = decltype(e);
        return with_vector<T>(word_bytes({x}), [&](auto v) {
            constexpr int V = decltype(v)::value;
            const size_t smem = sizeof(T) * BLOCK8 * (BLOCK8 + 4 / sizeof(T));
            if (smem > 48 * 1024) NB200_CUDA(cudaFuncSetAttribute(k_fp8_columns<T, V>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
            LaunchScope scope("fp8_columns", stream);
            NB200_CUDA(launch_overlapped(k_fp8_columns<T, V>, dim3((unsigned)ctas), dim3(NT), smem, stream, static_cast<const T *>(x->data), x->stride, x->cols, block, values,
                                         scales));
            return (int)NB200_OK;
        });
    });
}

}  // namespace
}  // namespace nb200

using namespace nb200;

extern "C" {

int nb200_fp8_product(const nb200_fp8 *a, const nb200_fp8 *w, const int32_t *offsets, nb200_dense *y, void *stream_) {
    if (!fp8_ok(a) || !fp8_ok(w) || !dense_ok(y) || a->tiled || !w->tiled || a->cols != w->cols || y->rows != a->rows || y->cols != w->rows) return NB200_E_BADARG;
    if (!offsets && w->groups != 1) return NB200_E_BADARG;
    if (w->groups > NB200_MAX_EXPERTS) return NB200_E_UNSUPPORTED;
    if (y->rows == 0 || y->cols == 0) return NB200_OK;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    const Operand oa{a->values, a->scales, blocks_of(a->cols), padded_rows(a->rows), padded_rows(a->rows), 0};
    const Operand ow{w->values, w->scales, blocks_of(w->cols), padded_rows(w->rows), blocks_of(w->rows), 7};
    return with_type(y->type, [&](auto e) {
        using T = decltype(e);
        LaunchScope scope("fp8_product", stream);
        NB200_CUDA(launch_overlapped(k_product_simple<T>, grid_of((y->rows * y->cols + NT - 1) / NT), dim3(NT), 0, stream, oa, ow, offsets, w->groups, y->rows, y->cols,
                                     static_cast<T *>(y->data), y->stride));
        return (int)NB200_OK;
    });
}

int64_t nb200_fp8_product_grad_w_scratch(const nb200_dense *dy, const nb200_dense *x, int32_t groups) {
    return grad_ok(dy, x, groups) ? (int64_t)GradScratch(nullptr, dy, x, groups).bytes : -1;
}

int nb200_fp8_product_grad_w(const nb200_dense *dy, const nb200_dense *x, int32_t groups, const int32_t *offsets, float *z, void *scratch, int64_t scratch_bytes, void *stream_) {
    if (!grad_ok(dy, x, groups) || (!offsets && groups != 1)) return NB200_E_BADARG;
    if (groups > NB200_MAX_EXPERTS) return NB200_E_UNSUPPORTED;
    if (groups == 0 || dy->cols == 0 || x->cols == 0) return NB200_OK;
    const GradScratch s(scratch, dy, x, groups);
    if (!z || !scratch || reinterpret_cast<uintptr_t>(scratch) % 256 != 0) return NB200_E_BADARG;
    if (scratch_bytes < (int64_t)s.bytes) return NB200_E_CAPACITY;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    {
        LaunchScope scope("group_blocks", stream);
        NB200_CUDA(launch_overlapped(k_group_blocks, dim3(1), dim3(1024), 0, stream, offsets, groups, (int)dy->rows, (int)s.bound, s.first_block, s.block));
    }
    int st;
    if ((st = quantise_columns(dy, s.block, s.bound, s.d, s.ds, stream))) return st;
    if ((st = quantise_columns(x, s.block, s.bound, s.x, s.xs, stream))) return st;
    const Operand od{s.d, s.ds, s.bound, padded_rows(dy->cols), padded_rows(dy->cols), 0};
    const Operand ox{s.x, s.xs, s.bound, padded_rows(x->cols), padded_rows(x->cols), 0};
    LaunchScope scope("fp8_grad_w", stream);
    NB200_CUDA(launch_overlapped(k_grad_w_simple, grid_of(((int64_t)groups * dy->cols * x->cols + NT - 1) / NT), dim3(NT), 0, stream, od, ox, s.first_block, groups, dy->cols,
                                 x->cols, z));
    return NB200_OK;
}

}  // extern "C"
