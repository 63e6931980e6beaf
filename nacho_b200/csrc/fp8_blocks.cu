// Matrices in 8-bit floating point with a scale per block of 128: from dense rows, from codes that exist, back to 32 bits, and the
// transpose of tiles. All of it is bound by device memory: one pass, whole 128-byte lines of codes.
#include <algorithm>
#include <type_traits>

#include "dense_rows.cuh"

namespace nb200 {
namespace {

constexpr int NT = 256;

// Extents and arrays of a matrix as kernels see them.
struct Blocks {
    int rows, cols, groups;
    int64_t kb, pad, nb;  // column blocks, padded rows, row blocks
    uint8_t *values;
    float *scales;

    __device__ uint8_t *block(int g, int64_t b) const { return values + (g * kb + b) * pad * BLOCK8; }
};

Blocks blocks(const nb200_fp8 *m) { return {m->rows, m->cols, m->groups, blocks_of(m->cols), padded_rows(m->rows), blocks_of(m->rows), m->values, m->scales}; }

// 16 threads have a row's block of 128 columns: a load of eight elements each, the largest magnitude by four exchanges, eight codes each.
template <typename T, int V>
__global__ void __launch_bounds__(NT) k_fp8_rows(Blocks z, const T *x, int64_t stride) {
    wait_for_previous();
    trigger_dependents();
    const int sub = threadIdx.x & 15;
    const unsigned half = 0xffffu << (threadIdx.x & 16);
    const int64_t all = (int64_t)z.rows * z.kb;
    for (int64_t i = (int64_t)blockIdx.x * (NT / 16) + threadIdx.x / 16; i < all; i += (int64_t)gridDim.x * (NT / 16)) {
        const int64_t r = i / z.kb, b = i - r * z.kb;
        float v[8];
        load8<T, V>(x + r * stride, b * BLOCK8 + sub * 8, z.cols, v);
        uint32_t m = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) m = max(m, magnitude(v[j]));
#pragma unroll
        for (int d = 8; d; d >>= 1) m = max(m, __shfl_xor_sync(half, m, d));
        const Factors f = factors_of(m);
        *reinterpret_cast<uint2 *>(z.block(0, b) + piece_at(r, sub >> 1) + (sub & 1) * 8) =
            make_uint2(codes4(v[0], v[1], v[2], v[3], f.inverse), codes4(v[4], v[5], v[6], v[7], f.inverse));
        if (sub == 0) z.scales[b * z.pad + r] = f.scale;
    }
}

// A CTA per 128 x 128; the tile stays in registers between the search for its largest magnitude and the codes.
template <typename T, int V>
__global__ void __launch_bounds__(NT) k_fp8_tiles(Blocks z, const T *x, int64_t stride) {
    __shared__ uint32_t top;
    wait_for_previous();
    trigger_dependents();
    const int sub = threadIdx.x & 15;
    const int64_t per_group = z.kb * z.nb;
    const int g = (int)(blockIdx.x / per_group);
    const int64_t b = blockIdx.x % per_group / z.nb, n = blockIdx.x % z.nb;
    if (threadIdx.x == 0) top = 0;
    __syncthreads();
    float v[8][8];
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int64_t r = n * BLOCK8 + i * 16 + threadIdx.x / 16;
        load8<T, V>(x + ((int64_t)g * z.rows + min(r, (int64_t)z.rows - 1)) * stride, b * BLOCK8 + sub * 8, r < z.rows ? z.cols : 0, v[i]);
#pragma unroll
        for (int j = 0; j < 8; ++j) m = max(m, magnitude(v[i][j]));
    }
    m = __reduce_max_sync(FULL_MASK, m);
    if (lane_id() == 0) atomicMax(&top, m);
    __syncthreads();
    const Factors f = factors_of(top);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int64_t r = n * BLOCK8 + i * 16 + threadIdx.x / 16;
        if (r < z.rows)
            *reinterpret_cast<uint2 *>(z.block(g, b) + piece_at(r, sub >> 1) + (sub & 1) * 8) =
                make_uint2(codes4(v[i][0], v[i][1], v[i][2], v[i][3], f.inverse), codes4(v[i][4], v[i][5], v[i][6], v[i][7], f.inverse));
    }
    if (threadIdx.x == 0) z.scales[(g * z.nb + n) * z.kb + b] = f.scale;
}

// Eight threads have a row's block: 16 codes each. `wide`: the rows of the given codes can be read in words of 16.
__global__ void __launch_bounds__(NT) k_fp8_pack(Blocks z, const uint8_t *codes, const float *scales, bool tiled, bool wide) {
    wait_for_previous();
    trigger_dependents();
    const int p = threadIdx.x & 7;
    const int64_t rows = (int64_t)z.groups * z.rows, all = rows * z.kb;
    for (int64_t i = (int64_t)blockIdx.x * (NT / 8) + threadIdx.x / 8; i < all; i += (int64_t)gridDim.x * (NT / 8)) {
        const int64_t row = i / z.kb, b = i - row * z.kb, c = b * BLOCK8 + p * 16;
        const int g = (int)(row / z.rows);
        const int64_t r = row - (int64_t)g * z.rows;
        const uint8_t *from = codes + row * z.cols;
        uint4 q = make_uint4(0, 0, 0, 0);
        if (wide) {
            if (c < z.cols) q = *reinterpret_cast<const uint4 *>(from + c);
        } else {
            uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < 16; ++j)
                if (c + j < z.cols) w[j / 4] |= (uint32_t)from[c + j] << (j % 4 * 8);
            q = make_uint4(w[0], w[1], w[2], w[3]);
        }
        *reinterpret_cast<uint4 *>(z.block(g, b) + piece_at(r, p)) = q;
        if (tiled) {
            if (p == 0 && r % BLOCK8 == 0) z.scales[(g * z.nb + r / BLOCK8) * z.kb + b] = scales[(g * z.nb + r / BLOCK8) * z.kb + b];
        } else if (p == 0) {
            z.scales[b * z.pad + r] = scales[r * z.kb + b];
        }
    }
}

__global__ void __launch_bounds__(NT) k_fp8_unpack(Blocks a, bool tiled, float *z) {
    wait_for_previous();
    trigger_dependents();
    const int64_t rows = (int64_t)a.groups * a.rows, all = rows * a.cols;
    for (int64_t i = (int64_t)blockIdx.x * NT + threadIdx.x; i < all; i += (int64_t)gridDim.x * NT) {
        const int64_t row = i / a.cols, c = i - row * a.cols, b = c / BLOCK8;
        const int g = (int)(row / a.rows), at = (int)(c % BLOCK8);
        const int64_t r = row - (int64_t)g * a.rows;
        __nv_fp8_e4m3 q;
        q.__x = a.block(g, b)[piece_at(r, at / 16) + at % 16];
        z[i] = float(q) * (tiled ? a.scales[(g * a.nb + r / BLOCK8) * a.kb + b] : a.scales[b * a.pad + r]);
    }
}

// A CTA per tile: read by rows, turned in shared memory, written by rows of the transpose.
__global__ void __launch_bounds__(NT) k_fp8_transpose(Blocks a, Blocks z) {
    __shared__ uint8_t tile[BLOCK8][BLOCK8 + 4];
    wait_for_previous();
    trigger_dependents();
    const int64_t per_group = a.kb * a.nb;
    const int g = (int)(blockIdx.x / per_group);
    const int64_t b = blockIdx.x % per_group / a.nb, n = blockIdx.x % a.nb;
    for (int i = threadIdx.x; i < BLOCK8 * 8; i += NT) {
        const int r = i / 8, p = i % 8;
        uint4 q = make_uint4(0, 0, 0, 0);
        if (n * BLOCK8 + r < a.rows) q = *reinterpret_cast<const uint4 *>(a.block(g, b) + piece_at(n * BLOCK8 + r, p));
        uint32_t *to = reinterpret_cast<uint32_t *>(&tile[r][p * 16]);
        to[0] = q.x, to[1] = q.y, to[2] = q.z, to[3] = q.w;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < BLOCK8 * 8; i += NT) {
        const int c = i % BLOCK8, p = i / BLOCK8;  // row c of the transpose; its 16 codes from rows p * 16 on
        const int64_t row = b * BLOCK8 + c;
        if (row >= z.rows) continue;
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            w[j] = tile[p * 16 + j * 4][c] | tile[p * 16 + j * 4 + 1][c] << 8 | tile[p * 16 + j * 4 + 2][c] << 16 | (uint32_t)tile[p * 16 + j * 4 + 3][c] << 24;
        *reinterpret_cast<uint4 *>(z.block(g, n) + piece_at(row, p)) = make_uint4(w[0], w[1], w[2], w[3]);
    }
    if (threadIdx.x == 0) z.scales[(g * z.nb + b) * z.kb + n] = a.scales[(g * a.nb + n) * a.kb + b];
}

dim3 grid_of(int64_t ctas) { return dim3((unsigned)std::max<int64_t>(1, std::min<int64_t>(ctas, sm_count() * 64ll))); }

constexpr int64_t MAX_CTAS = (1ll << 31) - 1;

}  // namespace
}  // namespace nb200

using namespace nb200;

extern "C" {

int64_t nb200_fp8_value_count(const nb200_fp8 *m) {
    if (!m || m->groups < 0 || m->rows < 0 || m->cols < 0 || (!m->tiled && m->groups != 1)) return -1;
    return m->groups * blocks_of(m->cols) * padded_rows(m->rows) * BLOCK8;
}

int64_t nb200_fp8_scale_count(const nb200_fp8 *m) {
    if (nb200_fp8_value_count(m) < 0) return -1;
    return m->tiled ? m->groups * blocks_of(m->cols) * blocks_of(m->rows) : blocks_of(m->cols) * padded_rows(m->rows);
}

int nb200_fp8_quantise(const nb200_dense *x, nb200_fp8 *z, void *stream_) {
    if (!dense_ok(x) || !fp8_ok(z) || x->cols != z->cols || x->rows != (int64_t)z->groups * z->rows) return NB200_E_BADARG;
    if (x->rows == 0 || x->cols == 0) return NB200_OK;
    const Blocks m = blocks(z);
    const int64_t tiles = m.groups * m.kb * m.nb;
    if (z->tiled && tiles > MAX_CTAS) return NB200_E_UNSUPPORTED;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    return with_type(x->type, [&](auto e) {
        using T = decltype(e);
        return with_vector<T>(word_bytes({x}), [&](auto v) {
            constexpr int V = decltype(v)::value;
            const T *data = static_cast<const T *>(x->data);
            if (z->tiled) {
                LaunchScope scope("fp8_tiles", stream);
                NB200_CUDA(launch_overlapped(k_fp8_tiles<T, V>, dim3((unsigned)tiles), dim3(NT), 0, stream, m, data, x->stride));
            } else {
                LaunchScope scope("fp8_rows", stream);
                NB200_CUDA(launch_overlapped(k_fp8_rows<T, V>, grid_of((m.rows * m.kb + NT / 16 - 1) / (NT / 16)), dim3(NT), 0, stream, m, data, x->stride));
            }
            return (int)NB200_OK;
        });
    });
}

int nb200_fp8_pack(const uint8_t *codes, const float *scales, nb200_fp8 *z, void *stream_) {
    if (!fp8_ok(z)) return NB200_E_BADARG;
    if ((int64_t)z->groups * z->rows == 0 || z->cols == 0) return NB200_OK;
    if (!codes || !scales) return NB200_E_BADARG;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    const Blocks m = blocks(z);
    const bool wide = reinterpret_cast<uintptr_t>(codes) % 16 == 0 && z->cols % 16 == 0;
    LaunchScope scope("fp8_pack", stream);
    NB200_CUDA(launch_overlapped(k_fp8_pack, grid_of(((int64_t)m.groups * m.rows * m.kb + NT / 8 - 1) / (NT / 8)), dim3(NT), 0, stream, m, codes, scales, z->tiled != 0, wide));
    return NB200_OK;
}

int nb200_fp8_unpack(const nb200_fp8 *a, float *z, void *stream_) {
    if (!fp8_ok(a)) return NB200_E_BADARG;
    if ((int64_t)a->groups * a->rows == 0 || a->cols == 0) return NB200_OK;
    if (!z) return NB200_E_BADARG;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    const Blocks m = blocks(a);
    LaunchScope scope("fp8_unpack", stream);
    NB200_CUDA(launch_overlapped(k_fp8_unpack, grid_of(((int64_t)m.groups * m.rows * m.cols + NT - 1) / NT), dim3(NT), 0, stream, m, a->tiled != 0, z));
    return NB200_OK;
}

int nb200_fp8_transpose(const nb200_fp8 *a, nb200_fp8 *z, void *stream_) {
    if (!fp8_ok(a) || !fp8_ok(z) || !a->tiled || !z->tiled || a->groups != z->groups || a->rows != z->cols || a->cols != z->rows) return NB200_E_BADARG;
    const Blocks m = blocks(a), t = blocks(z);
    const int64_t tiles = m.groups * m.kb * m.nb;
    if (tiles == 0) return NB200_OK;
    if (tiles > MAX_CTAS) return NB200_E_UNSUPPORTED;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    LaunchScope scope("fp8_transpose", stream);
    NB200_CUDA(launch_overlapped(k_fp8_transpose, dim3((unsigned)tiles), dim3(NT), 0, stream, m, t));
    return NB200_OK;
}

}  // extern "C"
