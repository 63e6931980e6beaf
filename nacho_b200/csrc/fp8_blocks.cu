// Matrices in 8-bit floating point with a scale per block of 128: from dense rows, from codes that exist, back to 32 bits, and the
// transpose of tiles. One pass each, whole 128-byte lines of codes. 16 matrices of 2048 x 2048 become tiles in 36 us, 0.85 of a copy.
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

// A CTA has 32 rows by two blocks, eight threads a row's block of 128 columns. So a block's 32 rows of codes are written as one stretch, and so are
// their scales. 16384 x 2048 of 16 bits take 19 us, 0.81 of a copy; with sixteen threads a block 22 (72 instead of 62 % of the issue slots).
constexpr int ROWS8 = 32, BLOCKS8 = 2;

template <typename T, int V>
__global__ void __launch_bounds__(NT) k_fp8_rows(Blocks z, int chunks, const T *x, int64_t stride) {
    wait_for_previous();
    trigger_dependents();
    const int sub = threadIdx.x & 7;
    const unsigned eight = 0xffu << (threadIdx.x & 24);
    const int64_t r = (int64_t)(blockIdx.x / chunks) * ROWS8 + threadIdx.x / 8;
    const int64_t b0 = (int64_t)(blockIdx.x % chunks) * BLOCKS8;
    if (r >= z.rows) return;
    Piece<T> v[BLOCKS8];
#pragma unroll
    for (int u = 0; u < BLOCKS8; ++u) v[u].template load<V>(x + r * stride, (b0 + u) * BLOCK8 + sub * 16, z.cols);
    uint32_t m[BLOCKS8];
    Factors f[BLOCKS8];
#pragma unroll
    for (int u = 0; u < BLOCKS8; ++u) m[u] = v[u].top(eight);
    share_factors<BLOCKS8, 8>(eight, m, f);
#pragma unroll
    for (int u = 0; u < BLOCKS8; ++u) {
        const int64_t b = b0 + u;
        if (b >= z.kb) break;
        *reinterpret_cast<uint4 *>(z.block(0, b) + piece_at(r, sub)) = v[u].codes(f[u].inverse);
        if (sub == 0) z.scales[b * z.pad + r] = f[u].scale;
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
    Eight<T> v[8];
    Top<T> mine;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int64_t r = n * BLOCK8 + i * 16 + threadIdx.x / 16;
        v[i].template load<V>(x + ((int64_t)g * z.rows + min(r, (int64_t)z.rows - 1)) * stride, b * BLOCK8 + sub * 8, r < z.rows ? z.cols : 0);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) mine.add(v[i]);
    const uint32_t m = __reduce_max_sync(FULL_MASK, mine.bits());
    if (lane_id() == 0) atomicMax(&top, m);
    __syncthreads();
    const Factors f = factors_of(top);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int64_t r = n * BLOCK8 + i * 16 + threadIdx.x / 16;
        if (r < z.rows)
            *reinterpret_cast<uint2 *>(z.block(g, b) + piece_at(r, sub >> 1) + (sub & 1) * 8) = codes8(v[i], f.inverse);
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

// A CTA per tile: read by rows into shared memory, words of four codes turned four by four, written by rows of the transpose. Word w of row r lies at
// place w ^ (r / 4), so that a warp reads a column of words without conflicts.
__global__ void __launch_bounds__(NT) k_fp8_transpose(Blocks a, Blocks z) {
    __shared__ uint32_t tile[BLOCK8][32];
    wait_for_previous();
    trigger_dependents();
    const int per_group = (int)(a.kb * a.nb), g = blockIdx.x / per_group, b = blockIdx.x % per_group / (int)a.nb, n = blockIdx.x % (int)a.nb;
    uint4 q[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = i * 32 + threadIdx.x / 8;
        q[i] = make_uint4(0, 0, 0, 0);
        if ((int64_t)n * BLOCK8 + r < a.rows) q[i] = *reinterpret_cast<const uint4 *>(a.block(g, b) + piece_at((int64_t)n * BLOCK8 + r, threadIdx.x & 7));
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = i * 32 + threadIdx.x / 8, w = (threadIdx.x & 7) * 4, turn = r / 4;
        tile[r][w ^ turn] = q[i].x, tile[r][(w + 1) ^ turn] = q[i].y, tile[r][(w + 2) ^ turn] = q[i].z, tile[r][(w + 3) ^ turn] = q[i].w;
    }
    __syncthreads();
    const int lane = lane_id();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int w = i * 8 + warp_id();  // rows 4w .. 4w + 3 of the transpose, their codes 4 lane .. 4 lane + 3
        uint32_t r[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) r[k] = tile[lane * 4 + k][w ^ lane];
        const uint32_t lo01 = __byte_perm(r[0], r[1], 0x5140), lo23 = __byte_perm(r[2], r[3], 0x5140), hi01 = __byte_perm(r[0], r[1], 0x7362),
                       hi23 = __byte_perm(r[2], r[3], 0x7362);
        const uint32_t turned[4] = {__byte_perm(lo01, lo23, 0x5410), __byte_perm(lo01, lo23, 0x7632), __byte_perm(hi01, hi23, 0x5410), __byte_perm(hi01, hi23, 0x7632)};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int64_t row = (int64_t)b * BLOCK8 + w * 4 + k;
            if (row < z.rows) *reinterpret_cast<uint32_t *>(z.block(g, n) + piece_at(row, lane / 4) + lane % 4 * 4) = turned[k];
        }
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
    int64_t all;  // a division to look ahead would take longer than all else that a call checks
    return __builtin_mul_overflow(m->groups * padded_rows(m->rows), blocks_of(m->cols) * BLOCK8, &all) ? -1 : all;
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
    const int64_t chunks = (m.kb + BLOCKS8 - 1) / BLOCKS8, row_ctas = (m.rows + ROWS8 - 1) / ROWS8 * chunks;
    if ((z->tiled ? tiles : row_ctas) > MAX_CTAS) return NB200_E_UNSUPPORTED;
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
                NB200_CUDA(launch_overlapped(k_fp8_rows<T, V>, dim3((unsigned)row_ctas), dim3(NT), 0, stream, m, (int)chunks, data, x->stride));
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
