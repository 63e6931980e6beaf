// Products of few rows with large weights, whose bytes are all that such a product takes: up to 16 rows of weights (and for gated ones as many more) per CTA, the summed
// axis shared by its eight warps. Weights go from memory into the registers of the matrix instructions (16 x 8, the legacy form: nothing here is
// bound by their rate), without a stop in shared memory: with 16 bytes a thread, four threads have 64 bytes of a row, and which of a step's columns are called
// first is the same for both operands.
#pragma once

#include "activation.cuh"
#include "dense_rows.cuh"
#include "product_waits.cuh"

namespace nb200 {

constexpr int FEW_NT = 256, FEW_WARPS = FEW_NT / 32;

struct FewArgs {
    const void *x, *w;
    int64_t x_stride, w_stride;  // elements
    const int32_t *offsets;
    int groups, rows;
    int wide;   // hidden, or columns of y
    int each;   // columns of the result per CTA, at most 16
    int inner;  // elements of a row (padding counted where it holds zeros)
    void *y, *both;
    int64_t stride;
    const float *row_scale, *col_scale;
    bool gelu;
};

// 16 rows by 32 bytes of weights (as words 0, 1 of two rows) times 32 bytes of 8 rows.
template <Sum SUM>
__device__ __forceinline__ void mma_few(uint32_t (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if constexpr (SUM == Sum::S8)
        asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else if constexpr (SUM == Sum::F16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 16 bytes of a row from element c on, zeros from element `inner` on, in words of V elements.
template <typename E, int V>
__device__ __forceinline__ uint4 load16(const E *row, int64_t c, int64_t inner) {
    if constexpr (sizeof(E) == 2) {
        Eight<E> v;
        v.template load<V>(row, c, inner);
        return make_uint4(v.w[0], v.w[1], v.w[2], v.w[3]);
    } else {
        return c < inner ? *reinterpret_cast<const uint4 *>(row + c) : make_uint4(0, 0, 0, 0);
    }
}

// A CTA per group and `each` columns of the result; NB rows of the group in a turn over the weights.
template <Sum SUM, bool GATED, int NB, int V, typename T>
__global__ void __launch_bounds__(FEW_NT, 2) k_few(const FewArgs args) {
    using E = std::conditional_t<SUM == Sum::S8, int8_t, std::conditional_t<SUM == Sum::F16, __half, __nv_bfloat16>>;
    constexpr int R = GATED ? 2 : 1, Q = NB / 8, U = NB == 32 ? 2 : R == 1 && NB == 8 ? 8 : 4;
    constexpr int PER = 64 / (int)sizeof(E), PIECE = PER / 4;  // elements of a row in a step, and a thread's
    __shared__ uint32_t part[FEW_WARPS][R][NB][17];
    const int warp = warp_id(), lane = lane_id(), g = blockIdx.y, col = blockIdx.x * args.each;
    trigger_dependents();
    wait_for_previous();
    const int lo = args.offsets ? min(max(ld_late(args.offsets + g), 0), args.rows) : 0;
    const int hi = args.offsets ? min(max(ld_late(args.offsets + g + 1), lo), args.rows) : args.rows;
    const E *const x = static_cast<const E *>(args.x);
    const E *w[R][2];
    bool there[R][2];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int c = col + lane / 4 + 8 * i;
            there[r][i] = c < args.wide && lane / 4 + 8 * i < args.each;
            w[r][i] = static_cast<const E *>(args.w) + (((int64_t)g * R + r) * args.wide + (there[r][i] ? c : 0)) * args.w_stride;
        }
    T *const y = static_cast<T *>(args.y);
    for (int row0 = lo; row0 < hi; row0 += NB) {
        const int count = min(NB, hi - row0);
        uint32_t acc[R][Q][4] = {};
        for (int64_t c0 = (int64_t)warp * PER; c0 < args.inner; c0 += (int64_t)FEW_WARPS * PER * U) {
            uint4 a[U][R][2], b[U][Q];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t c = c0 + (int64_t)u * FEW_WARPS * PER + (lane & 3) * PIECE;
#pragma unroll
                for (int r = 0; r < R; ++r)
#pragma unroll
                    for (int i = 0; i < 2; ++i) a[u][r][i] = load16<E, V>(w[r][i], c, there[r][i] ? args.inner : 0);
#pragma unroll
                for (int q = 0; q < Q; ++q) {
                    const int n = q * 8 + lane / 4;
                    b[u][q] = load16<E, V>(x + (int64_t)(row0 + min(n, count - 1)) * args.x_stride, c, n < count ? args.inner : 0);
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int q = 0; q < Q; ++q)
#pragma unroll
                    for (int r = 0; r < R; ++r) {
                        mma_few<SUM>(acc[r][q], a[u][r][0].x, a[u][r][1].x, a[u][r][0].y, a[u][r][1].y, b[u][q].x, b[u][q].y);
                        mma_few<SUM>(acc[r][q], a[u][r][0].z, a[u][r][1].z, a[u][r][0].w, a[u][r][1].w, b[u][q].z, b[u][q].w);
                    }
        }
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int q = 0; q < Q; ++q)
#pragma unroll
                for (int i = 0; i < 4; ++i) part[warp][r][q * 8 + (lane & 3) * 2 + (i & 1)][lane / 4 + (i / 2) * 8] = acc[r][q][i];
        __syncthreads();
        for (int i = threadIdx.x; i < count * 16; i += FEW_NT) {
            const int n = i / 16, c = i % 16;
            if (c >= args.each || col + c >= args.wide) continue;
            const int64_t row = row0 + n;
            if constexpr (SUM == Sum::S8) {
                int sum = 0;
#pragma unroll
                for (int k = 0; k < FEW_WARPS; ++k) sum += (int)part[k][0][n][c];
                y[row * args.stride + col + c] = from_float<T>(scaled(sum, ld_late(args.row_scale + row), ld_late(args.col_scale + (int64_t)g * args.wide + col + c)));
            } else {
                float sum[R] = {};
#pragma unroll
                for (int r = 0; r < R; ++r)
#pragma unroll
                    for (int k = 0; k < FEW_WARPS; ++k) sum[r] += __uint_as_float(part[k][r][n][c]);
                if constexpr (GATED) {
                    y[row * args.stride + col + c] = from_float<T>(sum[0] * logistic(act_inner(sum[0], args.gelu)) * sum[1]);
                    if (args.both) {
                        T *const both = static_cast<T *>(args.both) + row * 2 * args.wide + col + c;
                        both[0] = from_float<T>(sum[0]);
                        both[args.wide] = from_float<T>(sum[1]);
                    }
                } else {
                    y[row * args.stride + col + c] = from_float<T>(sum[0]);
                }
            }
        }
        __syncthreads();
    }
    if (args.offsets) {  // rows of no group
        const int64_t rows = args.rows, begin = min(max((int64_t)ld_late(args.offsets), (int64_t)0), rows), end = min(max((int64_t)ld_late(args.offsets + args.groups), begin), rows);
        const int64_t cta = (int64_t)blockIdx.y * gridDim.x + blockIdx.x, ctas = (int64_t)gridDim.x * gridDim.y;
        auto clear = [&](int64_t from, int64_t to) {
            for (int64_t r = from + cta; r < to; r += ctas) {
                for (int64_t c = threadIdx.x; c < args.wide; c += FEW_NT) y[r * args.stride + c] = from_float<T>(0.f);
                if (GATED && args.both)
                    for (int64_t c = threadIdx.x; c < 2 * (int64_t)args.wide; c += FEW_NT) static_cast<T *>(args.both)[r * 2 * args.wide + c] = from_float<T>(0.f);
            }
        };
        clear(0, begin);
        clear(end, rows);
    }
}

// Whether so few rows go this way, by the rows of a group and the bytes of all weights, of elements of `size` bytes (us on a B200, out of device memory, this way and by tiles of the tensor
// cores; hidden x width or columns x width):
//   - with groups while there are four rows for each (16 bits: 64 experts of 1024 x 2048 with a row each 82 and 91, with 4 rows 88 and 93, with 8 rows 92 and 93; where one of them
//     has 64 of 256 rows 92 and 93, 128 of them 98 and 92, and where it has all of them, which eight by eight read its weights again, 85 and 18); integers, of which a CTA has half
//     the bytes, never (64 experts of 2048 x 2048 with 3 rows 79 and 47);
//   - one group of up to 8 rows always (16 bits: 8192 x 8192 43 and 48; integers: 4096 x 4096 5.2 and 10, 14336 x 4096 15.2 and 14.9); more rows, whose own bytes all CTAs read, while the
//     weights are small. 16 bits, 16 rows: 4096 x 4096 16.4 and 17.0, 4094 x 4098 28 and 45, 8192 x 4096 31 and 28; 32 rows: 1100 x 1500 10 and 14, 2048 x 2048 11.7 and 10.5, 2044 x 2052,
//     whose rows would be copied to boundaries first, 14 and 19. Integers, 16 rows: 6144 x 4096 10.4 and 11.0, 8192 x 4096 11 and 12, 11000 x 4096 15 and 13; 32 rows: 4096 x 4096 8.5 and
//     10.4, 5000 x 4096 14 and 11.
// The kernel of 16 rows with gates and values spills 60 bytes a thread where words have 16 bytes, 128 to 384 where they have fewer; those of 8 and 32 rows 40 to 192 with words of 4 and 2.
inline bool few_rows(int64_t rows, int64_t groups, int64_t bytes, int size) {
    if (groups != 1) return size > 1 && rows <= 4 * groups;
    return rows <= (bytes <= (size > 1 ? 24ll : 18ll) << 20 ? 32 : bytes <= (size > 1 ? 96ll : 34ll) << 20 ? 16 : 8);
}

template <Sum SUM, bool GATED, int V, typename T>
int launch_few_rows(const char *name, const FewArgs &args, cudaStream_t stream) {
    Workspace *ws = nullptr;
    if (const int st = report_of(stream, &ws)) return st;  // an earlier product's: nothing here waits for anything
    auto go = [&](auto rows) -> int {
        constexpr int NB = decltype(rows)::value;
        // Two CTAs per SM are at work at once. Where there are few rounds of them, a CTA takes fewer than 16 columns so that all rounds are full: 4096 columns
        // are 256 CTAs of 16, of which 108 SMs get two and 40 one, or 293 of 14.
        const int64_t room = 2 * sm_count(), ctas = ((int64_t)args.wide + 15) / 16 * args.groups, rounds = (ctas + room - 1) / room;
        FewArgs a = args;
        a.each = 16;
        if (rounds <= 4) {
            const int64_t per = std::max<int64_t>(1, rounds * room / args.groups);
            a.each = (int)std::min<int64_t>(16, (args.wide + per - 1) / per);
        }
        LaunchScope scope(name, stream);
        NB200_CUDA(launch_overlapped(k_few<SUM, GATED, NB, V, T>, dim3((unsigned)((args.wide + a.each - 1) / a.each), (unsigned)args.groups), dim3(FEW_NT), 0, stream, a));
        return NB200_OK;
    };
    if (args.groups != 1 || args.rows <= 8) return go(std::integral_constant<int, 8>{});
    if (args.rows <= 16) return go(std::integral_constant<int, 16>{});
    return go(std::integral_constant<int, 32>{});
}

}  // namespace nb200
