// Products of 8-bit matrices with a scale per block of 128:
//     y[i, n] = sum_b sa[i, b] sw[n / 128, b] sum_{k in block b} a[i, k] w[n, k],
// all rows by one matrix or every group of rows by its own, and the gradient for the weights of the latter,
//     z[g][n, k] = sum_b sd[n, b] sx[k, b] sum_{i in block b} dy[i, n] x[i, k],   b over blocks of 128 rows of group g.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "dense_rows.cuh"
#include "tensor_core.cuh"

namespace nb200 {
namespace {

constexpr int NT = 256;

// An operand, [group][block of 128][row][128 codes], with its scales: of a row per block [block][row], or per 128 x 128 [group][row block][block].
struct Operand {
    const uint8_t *values;
    const float *scales;
    int64_t blocks, pad;  // per group; rows to a multiple of 8
    int64_t row_blocks;

    __device__ const uint8_t *block(int64_t g, int64_t b) const { return values + (g * blocks + b) * pad * BLOCK8; }
    __device__ const float *row_scales(int64_t b) const { return scales + b * pad; }
    __device__ const float *tile_scales(int64_t g, int64_t n) const { return scales + (g * row_blocks + min(n, row_blocks - 1)) * blocks; }
};

// ---- tiles on the tensor cores -------------------------------------------------------------

constexpr int STORE_WARPS = 8, THREADS = (STORE_WARPS + 4) * 32;
// Registers a thread: 168 at launch (65536 / 384), then 216 for the two groups of four warps that hold sums and 72 for the third: 64512 as before.
constexpr int REGS_SUMS = 216, REGS_OTHERS = 72;
static_assert(256 * REGS_SUMS + 128 * REGS_OTHERS <= 168 * THREADS, "");
constexpr uint64_t PATIENCE = 2000000000, SHORT_PATIENCE = 20000000;  // ns, after which a wait gives up (microseconds are usual); the self-test's

// A CTA has 128 rows of the result and 128 columns, in a pair 256. Both CTAs of a pair have the same columns, each brings half of their codes.
template <bool PAIR>
struct Shape {
    static constexpr int CTAS = PAIR ? 2 : 1, BM = 128 * CTAS, BN = 128 * CTAS;  // a tile of the result
    static constexpr int A_ROWS = 128, B_ROWS = 128;                             // what a CTA brings per block
    static constexpr int STAGES = 4, SUMS = 512 / BN;                            // blocks under way; places for their sums in tensor memory
    // Scales are written into a place STAGES + SUMS + 1 blocks after it was used before: by then the matrix instructions of STAGES blocks earlier are
    // done, which had to wait until every warp had said that it has read the sums of SUMS blocks before those. It says so once it has read all scales of
    // the block before (of that block itself the columns' last ones may still be missing).
    static constexpr int SCALES = STAGES + SUMS + 1;
    static constexpr int PANEL = PAIR ? 8 : 16;  // tiles that share columns follow one another: 2048 rows, then the next columns

    // What a CTA has in shared memory; tiles and the stores' staging begin at 1024-byte boundaries.
    struct Shared {
        uint8_t a[STAGES][A_ROWS * BLOCK8];
        uint8_t b[STAGES][B_ROWS * BLOCK8];
        uint8_t out[STORE_WARPS][2][32 * 128];
        float scale[SCALES][A_ROWS], col_scale[SCALES][BN];  // the latter for the gradient
        uint64_t full[STAGES], empty[STAGES];      // a stage's copies have landed (in the leader's: in both CTAs); its matrix instructions are done
        uint64_t sum_full[SUMS], sum_empty[SUMS];  // a block's sums lie in tensor memory; they have been read
        uint64_t drained;
        uint32_t tmem;
        int failed;
    };
    static constexpr size_t SHARED_BYTES = sizeof(Shared) + 1024;
    static_assert(SHARED_BYTES <= 227 * 1024, "");
};

// Which of N places is next, and in which phase of its barriers.
template <int N>
struct Ring {
    int at = 0;
    uint32_t phase = 0;
    __device__ void next() {
        if (++at == N) at = 0, phase ^= 1;
    }
};

// A tile of the result: its group, first row (a multiple of 8) and column, the rows that count, and the blocks that are summed.
struct Tile {
    int g, row, from, to, col;
    int first_block, blocks;
};

// The order of the tiles of `high` x `wide`: panels of rows, column by column.
template <int PANEL>
__device__ __forceinline__ void place_tile(int within, int high, int wide, int *row, int *col) {
    const unsigned panel = (unsigned)within / (unsigned)(PANEL * wide), width = min((unsigned)PANEL, (unsigned)high - panel * PANEL);
    const unsigned rest = (unsigned)within - panel * PANEL * wide, column = rest / width;
    *row = (int)(panel * PANEL + rest - column * width);
    *col = (int)column;
}

// Where a tile lies, found by a whole warp: groups 32 at a time, whose tiles it counts. Tiles are asked for in rising order. `most`: as many as there
// are with offsets that rise; others end there.
template <int BM, int BN, int PANEL>
struct Walk {
    const int32_t *offsets;
    int groups, blocks, rows, col_tiles, most;
    int chunk = -32, base = 0, incl = 0;  // tiles of the groups before this chunk; of this chunk's groups up to the lane's
    int from = 0, to = 0;

    __device__ Walk(const int32_t *o, int g, int b, int r, int c, int m) : offsets(o), groups(g), blocks(b), rows(r), col_tiles((c + BN - 1) / BN), most(m) {}

    __device__ static int row_tiles(int from, int to) { return to > from ? (to - (from & ~7) + BM - 1) / BM : 0; }

    __device__ bool find(int tile, Tile &t) {
        if (tile >= most) return false;
        int total;
        while (total = __shfl_sync(FULL_MASK, incl, 31), tile >= base + total) {
            base += total;
            chunk += 32;
            if (chunk >= groups) return false;
            const int g = chunk + lane_id();
            from = to = 0;
            if (g < groups) {
                from = offsets ? min(max(ld_late(offsets + g), 0), rows) : 0;
                to = offsets ? min(max(ld_late(offsets + g + 1), from), rows) : rows;
            }
            incl = warp_incl_sum(min(row_tiles(from, to) * col_tiles, most));
        }
        const int src = __ffs(__ballot_sync(FULL_MASK, base + incl > tile)) - 1;
        t.g = chunk + src;
        t.from = __shfl_sync(FULL_MASK, from, src);
        t.to = __shfl_sync(FULL_MASK, to, src);
        const int high = row_tiles(t.from, t.to);
        place_tile<PANEL>(tile - base - (__shfl_sync(FULL_MASK, incl, src) - high * col_tiles), high, col_tiles, &t.row, &t.col);
        t.row = (t.from & ~7) + t.row * BM;
        t.col *= BN;
        t.first_block = 0, t.blocks = blocks;
        return true;
    }
};

// The same for the gradient, whose groups have a result each, all of one size, and blocks of their own.
template <int BM, int BN, int PANEL>
struct GradWalk {
    const int32_t *first_block;
    int groups, rows, cols;

    __device__ bool find(int tile, Tile &t) {
        const int high = (rows + BM - 1) / BM, wide = (cols + BN - 1) / BN;
        t.g = (int)((unsigned)tile / (unsigned)(high * wide));
        if (t.g >= groups) return false;
        place_tile<PANEL>(tile - t.g * high * wide, high, wide, &t.row, &t.col);
        t.row *= BM, t.col *= BN, t.from = 0, t.to = rows;
        t.first_block = ld_late(first_block + t.g);
        t.blocks = ld_late(first_block + t.g + 1) - t.first_block;
        return true;
    }
};

__device__ __forceinline__ uint64_t now_ns() {
    uint64_t t;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
    return t;
}

// For a whole warp; false for all of it once one of its threads, or another warp of the CTA, has given up.
template <bool SELFTEST = false>
__device__ __forceinline__ bool wait_for(uint64_t *bar, uint32_t parity, volatile int *failed) {
    uint64_t start = 0;
    for (int i = 1;; ++i) {
        if (__all_sync(FULL_MASK, mbar_try_wait(bar, parity))) return true;
        if (i % 64) continue;
        if (__any_sync(FULL_MASK, *failed)) return false;
        if (!start) start = now_ns();
        if (__any_sync(FULL_MASK, now_ns() - start > (SELFTEST ? SHORT_PATIENCE : PATIENCE))) break;
    }
    *failed = 1;
    return false;
}

// After a give-up: what is still on its way lands first, or never will.
__device__ __forceinline__ void drain(uint64_t *bar, uint32_t parity) {
    for (const uint64_t start = now_ns(); now_ns() - start < SHORT_PATIENCE && !mbar_try_wait(bar, parity);) {}
}

// 32 rows of a warp, N columns from `col` on, from registers to memory, through two places in shared memory of 128 bytes of every row. WORD: rows
// can be written in words of so many bytes. With 16 the copy engine stores a place while the next one is filled, for which all 32 rows have to count (`base`: the
// row of the matrix at which the group's rows begin; `last`: there are no rows behind the group's). Otherwise the warp reads the place again and writes
// whole lines: 8192 x 32768 x 2048 521 us that way for all rows, 610 without shared memory.
template <typename T, int WORD, int N>
__device__ __forceinline__ void store_rows(const float (&acc)[N], uint8_t (*places)[32 * 128], int &turn, const CUtensorMap *matrix, int base, bool last, T *y, int64_t stride,
                                           int row, int from, int to, int col, int cols) {
    constexpr bool WIDE = WORD == 16;
    constexpr int PER = 128 / sizeof(T), EACH = 16 / sizeof(T);  // columns at a time; in 16 bytes
    const int lane = lane_id();
    if (row + 32 <= from || row >= to) return;
    const bool whole = WIDE && row >= from && (row + 32 <= to || last);
#pragma unroll
    for (int c = 0; c < N; c += PER) {
        if (col + c >= cols) break;
        uint8_t *place = places[turn];
        turn ^= 1;
        if (WIDE && elected()) stores_read_but<1>();
        __syncwarp();
#pragma unroll
        for (int p = 0; p < 8; ++p) {
            Vec<T, EACH> v;
#pragma unroll
            for (int j = 0; j < EACH; ++j) v.v[j] = from_float<T>(acc[c + p * EACH + j]);
            *reinterpret_cast<Vec<T, EACH> *>(place + piece_at(lane, p)) = v;
        }
        if (whole) {
            fence_async_shared();
            __syncwarp();
            if (elected()) store_tile(matrix, place, col + c, base + row);
        } else if constexpr (WIDE) {
            __syncwarp();
            const int p = lane & 7;
            const bool there = col + c + p * EACH < cols;
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
                const int r = i + lane / 8;
                if (there && row + r >= from && row + r < to)
                    *reinterpret_cast<uint4 *>(y + (int64_t)(row + r) * stride + col + c + p * EACH) = *reinterpret_cast<const uint4 *>(place + piece_at(r, p));
            }
        } else {
            constexpr int IN_WORD = WORD / sizeof(T);
            __syncwarp();
#pragma unroll 8
            for (int r = 0; r < 32; ++r) {
                const bool there = row + r >= from && row + r < to;
#pragma unroll
                for (int i = 0; i < PER; i += 32 * IN_WORD) {
                    const int j = i + lane * IN_WORD;
                    if (there && col + c + j < cols)
                        *reinterpret_cast<Vec<T, IN_WORD> *>(y + (int64_t)(row + r) * stride + col + c + j) =
                            *reinterpret_cast<const Vec<T, IN_WORD> *>(place + piece_at(r, j / EACH) + j % EACH * sizeof(T));
                }
            }
        }
        if (WIDE && elected()) close_stores();  // an empty group where the warp has written itself
    }
}

// One CTA per SM; they take tiles of 128 x 128 (a pair of them 256 x 256) in turn. One warp brings blocks of both operands into shared
// memory (plain bulk copies: a tile of a block is consecutive memory), one issues the matrix instructions, whose sums of a block land in
// tensor memory, and eight multiply the sums of earlier blocks by their scales into registers, half of a tile's columns of a row per thread: scales
// differ from block to block, so the sums have to leave tensor memory every 128 columns.
//
// GRAD: the sums run over a group's blocks of rows of dy and x, `offsets` says where those begin, and columns have a scale each. The scales of
// both are multiplied for every element, which is as much arithmetic again.
// SELFTEST: the first block's copies are left out, so that every warp's wait runs out.
template <typename T, int WORD, bool PAIR, bool GRAD, bool SELFTEST = false>
__device__ __forceinline__ void product(const Operand &a, const Operand &w, const int32_t *offsets, int groups, int64_t rows, int64_t cols, T *y, int64_t stride,
                                        int most, unsigned long long *report, const CUtensorMap *matrix) {
    using S = Shape<PAIR>;
    constexpr bool WIDE = WORD == 16;
    constexpr int STAGES = S::STAGES, SUMS = S::SUMS, BN = S::BN, N = BN / 2, W = 16;
    extern __shared__ uint8_t raw[];
    typename S::Shared &sh = *reinterpret_cast<typename S::Shared *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
    const int warp = warp_id(), lane = lane_id();
    const int rank = PAIR ? (int)cluster_rank() : 0;
    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) mbar_init(&sh.full[s], PAIR && rank == 0 ? 2 : 1), mbar_init(&sh.empty[s], 1);
        for (int s = 0; s < SUMS; ++s) mbar_init(&sh.sum_full[s], 1), mbar_init(&sh.sum_empty[s], STORE_WARPS * S::CTAS);
        mbar_init(&sh.drained, 1);
        mbar_fence_init();
        sh.failed = 0;
    }
    if (warp == STORE_WARPS) tmem_alloc<PAIR>(&sh.tmem, 512);
    tmem_fence_before();
    __syncthreads();
    if constexpr (PAIR) cluster_sync();  // nobody arrives at a barrier that is not there yet
    tmem_fence_after();
    const uint32_t tmem = *(volatile uint32_t *)&sh.tmem;
    volatile int *failed = &sh.failed;
    trigger_dependents();
    wait_for_previous();

    const int first = blockIdx.x / S::CTAS, step = gridDim.x / S::CTAS;
    auto tiles = [&] {
        if constexpr (GRAD) return GradWalk<S::BM, BN, S::PANEL>{offsets, groups, (int)rows, (int)cols};
        else return Walk<S::BM, BN, S::PANEL>(offsets, groups, (int)a.blocks, (int)rows, (int)cols, most);
    };
    if (warp < STORE_WARPS) {
        // sums and stores: warps w and w + 4 have the lanes of tensor memory that every fourth warp can reach, and a half of the columns each
        more_registers<REGS_SUMS>();
        auto walk = tiles();
        Tile t;
        const int lanes = warp & 3, half = warp >> 2;
        int turn = 0;
        Ring<SUMS> sums;
        Ring<S::SCALES> place;
        const uint32_t base = tmem + ((uint32_t)(lanes * 32) << 16) + half * N;
        for (int tile = first; walk.find(tile, t); tile += step) {
            float acc[N];
#pragma unroll
            for (int j = 0; j < N; ++j) acc[j] = 0.f;
            const int64_t row = t.row + rank * 128 + lanes * 32, col = t.col + half * N;
            // The scales of the columns' tiles: each lane has a block's, of 32 blocks, and asks for those of the next 32. The scales of rows (for the
            // gradient, of columns too) come with the copies, which the matrix instructions have waited for and this warp waits for those.
            const float *sw = GRAD ? nullptr : w.tile_scales(t.g, col / BLOCK8);
            float tile_scale = 0.f, next_scale = !GRAD && lane < t.blocks ? ld_late(sw + lane) : 0.f;
            bool fine = true;
            for (int b = 0; b < t.blocks; ++b, sums.next(), place.next()) {
                if (!GRAD && b % 32 == 0) {
                    tile_scale = next_scale;
                    next_scale = b + 32 + lane < t.blocks ? ld_late(sw + b + 32 + lane) : 0.f;
                }
                if (!(fine = wait_for<SELFTEST>(&sh.sum_full[sums.at], sums.phase, failed))) break;
                tmem_fence_after();
                const uint32_t at = base + sums.at * BN;
                // W columns are on their way while W others are added: with 32 the registers are short (8192^3 490 us, with 16 468)
                uint32_t v[N / W][W];
                tmem_load(at, v[0]);
                float s = sh.scale[place.at][lanes * 32 + lane];
                if constexpr (!GRAD) s *= __shfl_sync(FULL_MASK, tile_scale, b % 32);
#pragma unroll
                for (int q = 0; q < N / W; ++q) {
                    tmem_wait_loads(v[q]);
                    if (q + 1 < N / W) {
                        tmem_load(at + (q + 1) * W, v[q + 1]);
                    } else {
                        tmem_fence_before();
                        __syncwarp();
                        if (lane == 0) {
                            if constexpr (PAIR) mbar_arrive_leader(&sh.sum_empty[sums.at]);
                            else mbar_arrive(&sh.sum_empty[sums.at]);
                        }
                    }
                    if constexpr (GRAD) {
                        const float4 *columns = reinterpret_cast<const float4 *>(&sh.col_scale[place.at][half * N + q * W]);
#pragma unroll
                        for (int j = 0; j < W; j += 4) {
                            const float4 c = columns[j / 4];
                            add_scaled(acc[q * W + j], acc[q * W + j + 1], v[q][j], v[q][j + 1], s, c.x, c.y);
                            add_scaled(acc[q * W + j + 2], acc[q * W + j + 3], v[q][j + 2], v[q][j + 3], s, c.z, c.w);
                        }
                    } else {
#pragma unroll
                        for (int j = 0; j < W; ++j) acc[q * W + j] = __fmaf_rn(__uint_as_float(v[q][j]), s, acc[q * W + j]);
                    }
                }
            }
            if (!fine) break;
            if (col < cols)
                store_rows<T, WORD, N>(acc, sh.out[warp], turn, matrix, GRAD ? t.g * (int)rows : 0, GRAD ? t.g == groups - 1 : t.to == rows, GRAD ? y + t.g * rows * stride : y,
                                       stride, (int)row, t.from, t.to, (int)col, (int)cols);
        }
        if (WIDE && elected()) stores_done();
        __syncwarp();
        // rows of no group
        if (!GRAD && offsets) {
            const int64_t lo = min(max((int64_t)ld_late(offsets), (int64_t)0), rows), hi = min(max((int64_t)ld_late(offsets + groups), lo), rows);
            for (int64_t r = blockIdx.x * STORE_WARPS + warp; r < rows; r += (int64_t)gridDim.x * STORE_WARPS)
                if (r < lo || r >= hi)
                    for (int64_t c = lane; c < cols; c += 32) y[r * stride + c] = from_float<T>(0.f);
        }
    } else {
        fewer_registers<REGS_OTHERS>();
        auto walk = tiles();
        Tile t;
        Ring<STAGES> stage;
        Ring<S::SCALES> place;
        bool fine = true;
        if (warp == STORE_WARPS + 1) {  // copies
            for (int tile = first; fine && walk.find(tile, t); tile += step) {
                const int64_t row = t.row + rank * S::A_ROWS, col = t.col + rank * S::B_ROWS;
                const uint32_t a_bytes = (uint32_t)min((int64_t)S::A_ROWS, max(a.pad - row, (int64_t)0)) * BLOCK8;
                const uint32_t b_bytes = (uint32_t)min((int64_t)S::B_ROWS, max(w.pad - col, (int64_t)0)) * BLOCK8;
                const uint32_t scale_bytes = a_bytes / BLOCK8 * sizeof(float);
                const uint32_t col_bytes = GRAD ? (uint32_t)min((int64_t)BN, w.pad - t.col) * sizeof(float) : 0;
                const float *from_scales = a.row_scales(t.first_block) + row, *from_col_scales = w.row_scales(t.first_block) + t.col;
                const uint8_t *from_a = a.block(0, t.first_block) + row * BLOCK8, *from_b = w.block(GRAD ? 0 : t.g, t.first_block) + col * BLOCK8;
                for (int b = 0; b < t.blocks; ++b, stage.next(), place.next()) {
                    if (!(fine = wait_for<SELFTEST>(&sh.empty[stage.at], stage.phase ^ 1, failed))) break;
                    if (elected() && !(SELFTEST && b == 0)) {
                        mbar_arrive_expect_tx(&sh.full[stage.at], a_bytes + b_bytes + scale_bytes + col_bytes);
                        if (a_bytes) {
                            bulk_load(sh.a[stage.at], from_a, a_bytes, &sh.full[stage.at]);
                            bulk_load(sh.scale[place.at], from_scales, scale_bytes, &sh.full[stage.at]);
                        }
                        if (GRAD) bulk_load(sh.col_scale[place.at], from_col_scales, col_bytes, &sh.full[stage.at]);
                        if (b_bytes) bulk_load(sh.b[stage.at], from_b, b_bytes, &sh.full[stage.at]);
                    }
                    __syncwarp();
                    from_a += a.pad * BLOCK8, from_b += w.pad * BLOCK8, from_scales += a.pad, from_col_scales += w.pad;
                }
            }
            if (!fine)  // nothing may land in shared memory that is no longer this CTA's
                for (int s = 0; s < STAGES; ++s) drain(&sh.full[s], s < stage.at ? stage.phase : stage.phase ^ 1);
        } else if (warp == STORE_WARPS && rank == 0) {  // matrix instructions
            const uint64_t tile_a = tile_descriptor(smem_u32(sh.a[0])), tile_b = tile_descriptor(smem_u32(sh.b[0]));
            Ring<SUMS> sums;
            for (int tile = first; fine && walk.find(tile, t); tile += step) {
                for (int b = 0; b < t.blocks; ++b, stage.next(), sums.next()) {
                    if (!(fine = wait_for<SELFTEST>(&sh.full[stage.at], stage.phase, failed))) break;
                    if (!(fine = wait_for<SELFTEST>(&sh.sum_empty[sums.at], sums.phase ^ 1, failed))) break;
                    tmem_fence_after();
                    if (elected()) {
                        const uint64_t da = tile_a + (uint64_t)(stage.at * (S::A_ROWS * BLOCK8 >> 4)), db = tile_b + (uint64_t)(stage.at * (S::B_ROWS * BLOCK8 >> 4));
#pragma unroll
                        for (int k = 0; k < BLOCK8 / 32; ++k) mma_e4m3<PAIR>(tmem + sums.at * BN, da + 2 * k, db + 2 * k, product_descriptor(S::BM, BN), k > 0);
                        mma_commit<PAIR>(&sh.empty[stage.at]);
                        mma_commit<PAIR>(&sh.sum_full[sums.at]);
                    }
                    __syncwarp();
                }
            }
            if (!fine) {
                if (elected()) mma_commit<PAIR>(&sh.drained);
                __syncwarp();
                drain(&sh.drained, 0);
            }
        } else if (PAIR && warp == STORE_WARPS) {  // tells the leader of the copies that have landed here
            for (int tile = first; fine && walk.find(tile, t); tile += step) {
                for (int b = 0; b < t.blocks; ++b, stage.next()) {
                    if (!(fine = wait_for<SELFTEST>(&sh.full[stage.at], stage.phase, failed))) break;
                    if (elected()) mbar_arrive_leader(&sh.full[stage.at]);
                    __syncwarp();
                }
            }
        }
    }
    tmem_fence_before();
    __syncthreads();
    if constexpr (PAIR) cluster_sync();  // no arrival is on its way to a CTA that is gone
    if (warp == STORE_WARPS) {
        tmem_fence_after();
        tmem_free<PAIR>(tmem, 512);
        if (lane == 0 && *failed) publish_result_word(report, 1, blockIdx.x);
    }
}

template <typename T, int WORD, bool GRAD>
__global__ void __launch_bounds__(THREADS, 1) k_product(Operand a, Operand w, const int32_t *offsets, int groups, int64_t rows, int64_t cols, T *y, int64_t stride,
                                                        int most, unsigned long long *report, const __grid_constant__ CUtensorMap matrix) {
    product<T, WORD, false, GRAD>(a, w, offsets, groups, rows, cols, y, stride, most, report, &matrix);
}
__global__ void __launch_bounds__(THREADS, 1) k_product_selftest(Operand a, Operand w, const int32_t *offsets, int groups, int64_t rows, int64_t cols, float *y, int64_t stride,
                                                                 unsigned long long *report) {
    product<float, 4, false, false, true>(a, w, offsets, groups, rows, cols, y, stride, 1 << 20, report, nullptr);
}
template <typename T, int WORD, bool GRAD>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS, 1) k_product_pair(Operand a, Operand w, const int32_t *offsets, int groups, int64_t rows, int64_t cols, T *y,
                                                                                       int64_t stride, int most, unsigned long long *report, const __grid_constant__ CUtensorMap matrix) {
    product<T, WORD, true, GRAD>(a, w, offsets, groups, rows, cols, y, stride, most, report, &matrix);
}

// ---- few rows per group ------------------------------------------------------------------

// The operands change sides: 128 rows of weights against NB rows, 16 to 128, of a group, so that a CTA brings hardly more than the weights, which is
// all that a product of few rows takes: one CTA per group and 128 columns of the result, several to an SM. Where there are not enough of them, the
// CTAs of a cluster have a part of the blocks each (SPLIT) and add their sums, in order, through one another's shared memory. A group of more rows
// than NB (than NB times the grid's third extent) takes several turns over its weights.
template <int NB, bool SPLIT>
struct FewShape {
    static constexpr int STAGES = 4, SUMS = 4, SCALES = STAGES + SUMS, COLUMNS = SUMS * NB;  // of tensor memory
    struct Shared {
        uint8_t w[STAGES][128 * BLOCK8];
        uint8_t a[STAGES][NB * BLOCK8];
        float scale[SCALES][NB];
        float part[SPLIT ? NB : 1][128];
        uint64_t full[STAGES], empty[STAGES], sum_full[SUMS], sum_empty[SUMS], drained;
        uint32_t tmem;
        int failed;
    };
    static constexpr size_t SHARED_BYTES = sizeof(Shared) + 1024;
};
constexpr int FEW_THREADS = 6 * 32;

template <typename T, int NB, bool SPLIT>
__global__ void __launch_bounds__(FEW_THREADS, NB == 16 ? 3 : NB == 128 ? 1 : 2) k_product_few(Operand a, Operand w, const int32_t *offsets, int groups, int64_t rows, int64_t cols, T *y, int64_t stride,
                                                             int tiles_each, unsigned long long *report) {
    using S = FewShape<NB, SPLIT>;
    constexpr int STAGES = S::STAGES, SUMS = S::SUMS, W = NB < 32 ? 16 : 32;
    extern __shared__ uint8_t raw[];
    typename S::Shared &sh = *reinterpret_cast<typename S::Shared *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
    const int warp = warp_id(), lane = lane_id();
    const int slices = SPLIT ? (int)cluster_size() : 1, slice = SPLIT ? (int)cluster_rank() : 0;
    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) mbar_init(&sh.full[s], 1), mbar_init(&sh.empty[s], 1);
        for (int s = 0; s < SUMS; ++s) mbar_init(&sh.sum_full[s], 1), mbar_init(&sh.sum_empty[s], 4);
        mbar_init(&sh.drained, 1);
        mbar_fence_init();
        sh.failed = 0;
    }
    if (warp == 4) tmem_alloc<false>(&sh.tmem, S::COLUMNS);
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    const uint32_t tmem = *(volatile uint32_t *)&sh.tmem;
    volatile int *failed = &sh.failed;
    trigger_dependents();
    wait_for_previous();

    const int g = blockIdx.y;
    const int64_t first_col = (int64_t)(blockIdx.x / slices) * tiles_each * 128, end_col = min(first_col + (int64_t)tiles_each * 128, cols);
    const int64_t from = offsets ? min(max((int64_t)ld_late(offsets + g), (int64_t)0), rows) : 0;
    const int64_t to = offsets ? min(max((int64_t)ld_late(offsets + g + 1), from), rows) : rows;
    const int first = (int)(a.blocks * slice / slices), blocks = (int)(a.blocks * (slice + 1) / slices) - first;
    Ring<STAGES> stage;
    Ring<SUMS> sums;
    Ring<S::SCALES> place;
    bool fine = true;
    for (int64_t col = first_col; col < end_col; col += 128) {
        for (int64_t row = (from & ~int64_t(7)) + (int64_t)blockIdx.z * NB; row < to; row += (int64_t)gridDim.z * NB) {
            if (warp == 5) {  // copies
                const uint32_t a_bytes = (uint32_t)min((int64_t)NB, a.pad - row) * BLOCK8, w_bytes = (uint32_t)min((int64_t)128, w.pad - col) * BLOCK8;
                const uint32_t scale_bytes = a_bytes / BLOCK8 * sizeof(float);
                for (int b = first; fine && b < first + blocks; ++b, stage.next(), place.next()) {
                    if (!(fine = wait_for(&sh.empty[stage.at], stage.phase ^ 1, failed))) break;
                    if (elected()) {
                        mbar_arrive_expect_tx(&sh.full[stage.at], a_bytes + w_bytes + scale_bytes);
                        bulk_load(sh.w[stage.at], w.block(g, b) + col * BLOCK8, w_bytes, &sh.full[stage.at]);
                        bulk_load(sh.a[stage.at], a.block(0, b) + row * BLOCK8, a_bytes, &sh.full[stage.at]);
                        bulk_load(sh.scale[place.at], a.row_scales(b) + row, scale_bytes, &sh.full[stage.at]);
                    }
                    __syncwarp();
                }
            } else if (warp == 4) {  // matrix instructions
                const uint64_t tile_w = tile_descriptor(smem_u32(sh.w[0])), tile_a = tile_descriptor(smem_u32(sh.a[0]));
                for (int b = 0; fine && b < blocks; ++b, stage.next(), sums.next()) {
                    if (!(fine = wait_for(&sh.full[stage.at], stage.phase, failed))) break;
                    if (!(fine = wait_for(&sh.sum_empty[sums.at], sums.phase ^ 1, failed))) break;
                    tmem_fence_after();
                    if (elected()) {
                        const uint64_t dw = tile_w + (uint64_t)(stage.at * (128 * BLOCK8 >> 4)), da = tile_a + (uint64_t)(stage.at * (NB * BLOCK8 >> 4));
    #pragma unroll
                        for (int k = 0; k < BLOCK8 / 32; ++k) mma_e4m3<false>(tmem + sums.at * NB, dw + 2 * k, da + 2 * k, product_descriptor(128, NB), k > 0);
                        mma_commit<false>(&sh.empty[stage.at]);
                        mma_commit<false>(&sh.sum_full[sums.at]);
                    }
                    __syncwarp();
                }
            } else {  // sums and stores: a thread has a column of the result
                float acc[NB];
    #pragma unroll
                for (int j = 0; j < NB; ++j) acc[j] = 0.f;
                const float *sw = w.tile_scales(g, col / BLOCK8) + first;
                float tile_scale = 0.f, next_scale = lane < blocks ? ld_late(sw + lane) : 0.f;
                for (int b = 0; fine && b < blocks; ++b, sums.next(), place.next()) {
                    if (b % 32 == 0) {
                        tile_scale = next_scale;
                        next_scale = b + 32 + lane < blocks ? ld_late(sw + b + 32 + lane) : 0.f;
                    }
                    const float s = __shfl_sync(FULL_MASK, tile_scale, b % 32);
                    if (!(fine = wait_for(&sh.sum_full[sums.at], sums.phase, failed))) break;
                    tmem_fence_after();
                    const uint32_t at = tmem + ((uint32_t)(warp * 32) << 16) + sums.at * NB;
                    uint32_t v[NB / W][W];
                    tmem_load(at, v[0]);
    #pragma unroll
                    for (int q = 0; q < NB / W; ++q) {
                        float row_scale[W];
    #pragma unroll
                        for (int j = 0; j < W; j += 4) *reinterpret_cast<float4 *>(row_scale + j) = *reinterpret_cast<const float4 *>(&sh.scale[place.at][q * W + j]);
                        tmem_wait_loads(v[q]);
                        if (q + 1 < NB / W) {
                            tmem_load(at + (q + 1) * W, v[q + 1]);
                        } else {
                            tmem_fence_before();
                            __syncwarp();
                            if (lane == 0) mbar_arrive(&sh.sum_empty[sums.at]);
                        }
    #pragma unroll
                        for (int j = 0; j < W; ++j) acc[q * W + j] = __fmaf_rn(__uint_as_float(v[q][j]), s * row_scale[j], acc[q * W + j]);
                    }
                }
                const int64_t n = col + threadIdx.x;
                if constexpr (SPLIT) {
    #pragma unroll
                    for (int j = 0; j < NB; ++j) sh.part[j][threadIdx.x] = acc[j];
                } else if (fine && n < cols) {
    #pragma unroll
                    for (int j = 0; j < NB; ++j)
                        if (row + j >= from && row + j < to) y[(row + j) * stride + n] = from_float<T>(acc[j]);
                }
            }
            if constexpr (SPLIT) {
                cluster_sync();
                // Eight loads of the others' parts are on their way at a time: one by one they took longer than the product.
                if (threadIdx.x < 128 && fine && col + threadIdx.x < cols)
                    for (int j = slice; j < NB; j += slices) {
                        if (row + j < from || row + j >= to) continue;
                        float part[8], sum = 0.f;
    #pragma unroll
                        for (int r = 0; r < 8; ++r) part[r] = r < slices ? load_remote(&sh.part[j][threadIdx.x], r) : 0.f;
    #pragma unroll
                        for (int r = 0; r < 8; ++r) sum += part[r];
                        y[(row + j) * stride + col + threadIdx.x] = from_float<T>(sum);
                    }
                cluster_sync();  // the parts have been read, also those of a CTA that ends here
            }
        }
    }
    if (offsets && warp < 4) {  // rows of no group
        const int64_t lo = min(max((int64_t)ld_late(offsets), (int64_t)0), rows), hi = min(max((int64_t)ld_late(offsets + groups), lo), rows);
        const int64_t cta = ((int64_t)blockIdx.z * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x, ctas = (int64_t)gridDim.x * gridDim.y * gridDim.z;
        auto clear = [&](int64_t begin, int64_t end) {
            for (int64_t r = begin + cta; r < end; r += ctas)
                for (int64_t c = threadIdx.x; c < cols; c += 128) y[r * stride + c] = from_float<T>(0.f);
        };
        clear(0, lo);
        clear(hi, rows);
    }
    if (!fine && warp == 5)
        for (int s = 0; s < STAGES; ++s) drain(&sh.full[s], s < stage.at ? stage.phase : stage.phase ^ 1);
    if (!fine && warp == 4) {
        if (elected()) mma_commit<false>(&sh.drained);
        __syncwarp();
        drain(&sh.drained, 0);
    }
    tmem_fence_before();
    __syncthreads();
    if (warp == 4) {
        tmem_fence_after();
        tmem_free<false>(tmem, S::COLUMNS);
        if (lane == 0 && *failed) publish_result_word(report, 1, blockIdx.x);
    }
}

// ---- operands of the gradient ------------------------------------------------------------

// Blocks of 128 rows, counted from each group's first: where a group's blocks begin, and every block's rows {first, how many}. One CTA. Offsets that fall
// stand for up to 2^35 blocks, which are counted in two parts of 12 and more bits; those from `bound` on are left out.
__global__ void __launch_bounds__(1024) k_group_blocks(const int32_t *offsets, int groups, int rows, int bound, int32_t *first_block, int2 *block) {
    __shared__ int tmp[66];
    wait_for_previous();
    trigger_dependents();
    int64_t base = 0;
    for (int g0 = 0; g0 < groups; g0 += 1024) {
        const int g = g0 + threadIdx.x;
        int from = 0, to = 0;
        if (g < groups) {
            from = offsets ? min(max(ld_late(offsets + g), 0), rows) : 0;
            to = offsets ? min(max(ld_late(offsets + g + 1), from), rows) : rows;
        }
        const int n = (to - from + BLOCK8 - 1) / BLOCK8;
        int high, low, all_high, all_low;
        block_excl_sum2<1024>(n >> 12, n & 4095, tmp, high, low, all_high, all_low);
        const int64_t at = base + ((int64_t)high << 12) + low;
        if (g < groups) {
            first_block[g] = (int)min(at, (int64_t)bound);
            for (int b = 0; from + b * BLOCK8 < to && at + b < bound; ++b) block[at + b] = make_int2(from + b * BLOCK8, min(BLOCK8, to - from - b * BLOCK8));
        }
        base += ((int64_t)all_high << 12) + all_low;
    }
    if (threadIdx.x == 0) first_block[groups] = (int)min(base, (int64_t)bound);
    for (int64_t b = base + threadIdx.x; b < bound; b += 1024) block[b] = make_int2(0, 0);
}

// x by blocks of rows: column c becomes row c of the result, a scale for it per block. A CTA per block and 128 columns: a thread has eight columns of
// eight rows, the largest magnitude of a column comes from 16 threads by way of shared memory, and the codes go through shared memory to whole
// lines. There the eight codes of a column and eight rows p lie at place p ^ (column / 8) of the column's, which spreads a warp over the banks.
// ROWS: the same elements quantised along the columns too, which reads them once for both: the 16 threads of a row have its block of 128.
template <typename T, int V, bool ROWS>
__global__ void __launch_bounds__(NT, sizeof(T) == 2 ? 3 : 2) k_fp8_columns(const T *x, int64_t stride, int64_t cols, const int2 *block, uint8_t *values, float *scales,
                                                                              uint8_t *row_values, float *row_scales, int64_t row_pad) {
    __shared__ uint32_t top[NT / 32][BLOCK8];  // words
    __shared__ alignas(16) float inverse[BLOCK8];
    __shared__ alignas(16) uint2 codes[BLOCK8][16];
    wait_for_previous();
    trigger_dependents();
    const int64_t chunks = blocks_of(cols), b = blockIdx.x / chunks, c0 = blockIdx.x % chunks * BLOCK8, pad = padded_rows(cols);
    const int2 rows = *(block + b);
    if (rows.y == 0) return;
    const int sub = threadIdx.x & 15, part = threadIdx.x / 16;
    Eight<T> v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int r = part * 8 + i;
        v[i].template load<V>(x + (int64_t)(rows.x + min(r, rows.y - 1)) * stride, c0 + sub * 8, r < rows.y ? cols : 0);
    }
    if constexpr (ROWS) {
        const unsigned half = 0xffffu << (threadIdx.x & 16);
        uint32_t top_of[8];
        Factors f[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            Top<T> row;
            row.add(v[i]);
#pragma unroll
            for (int d = 8; d; d >>= 1) row.join(half, d);
            top_of[i] = row.bits();
        }
        share_factors<8, 16>(half, top_of, f);
        const int64_t at = c0 / BLOCK8 * row_pad + rows.x;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int r = part * 8 + i;
            if (r >= rows.y) break;
            *reinterpret_cast<uint2 *>(row_values + c0 / BLOCK8 * row_pad * BLOCK8 + piece_at(rows.x + r, sub >> 1) + (sub & 1) * 8) = codes8(v[i], f[i].inverse);
            if (sub == 0) row_scales[at + r] = f[i].scale;
        }
    }
    // words of a row: a column each, or two neighbours
    constexpr int WORDS = Eight<T>::WORDS, EACH = 4 / sizeof(T);
    Top<T> m[WORDS];
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < WORDS; ++j) m[j].add(v[i].w[j]);
#pragma unroll
    for (int j = 0; j < WORDS; ++j) {
        m[j].join(FULL_MASK, 16);
        if (lane_id() < 16) top[warp_id()][sub * WORDS + j] = m[j].v;
    }
    __syncthreads();
    if (threadIdx.x < BLOCK8) {
        Top<T> column;
#pragma unroll
        for (int w = 0; w < NT / 32; ++w) column.add(top[w][threadIdx.x / EACH]);
        const uint32_t all = sizeof(T) == 2 ? Top<T>::as_float(threadIdx.x & 1 ? column.v >> 16 : column.v & 0xffffu) : column.v;
        const Factors f = factors_of(all);
        inverse[threadIdx.x] = f.inverse;
        if (c0 + threadIdx.x < cols) scales[b * pad + c0 + threadIdx.x] = f.scale;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float f = inverse[sub * 8 + j];
        codes[sub * 8 + j][part ^ sub] =
            make_uint2(codes4(v[0].get(j), v[1].get(j), v[2].get(j), v[3].get(j), f), codes4(v[4].get(j), v[5].get(j), v[6].get(j), v[7].get(j), f));
    }
    __syncthreads();
    uint8_t *to = values + b * pad * BLOCK8;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int c = i * 32 + threadIdx.x / 8, p = threadIdx.x & 7, turn = c / 8;
        const uint4 q = *reinterpret_cast<const uint4 *>(&codes[c][(p ^ (turn >> 1)) * 2]);
        if (c0 + c < cols) *reinterpret_cast<uint4 *>(to + piece_at(c0 + c, p)) = turn & 1 ? make_uint4(q.z, q.w, q.x, q.y) : q;
    }
}

// ---- host ------------------------------------------------------------------------------

// The word by which a product of this stream says that a wait gave up. The call does not wait for its kernel, so the next one on the stream
// finds it and returns the error in its place.
int report_of(cudaStream_t stream, Workspace **ws) {
    int st;
    if ((st = acquire_workspace(stream, 0, ws, REPORT_SLOT))) return st;
    volatile unsigned long long *word = reinterpret_cast<volatile unsigned long long *>((*ws)->host) + 32;
    const unsigned long long said = *word;
    if (!(said & RW_VALID)) return NB200_OK;
    *word = 0;
    return note_timeout(3, (int)(said & RW_VALUE_MASK), "an earlier 8-bit product");
}

// Slices of the summed axis, CTAs of a cluster, for `tiles` CTAs' worth of work: more while the SMs are not all busy (where one CTA fills an SM: while
// they would not be more than the SMs), eight at most, of four blocks at least. 256 tiles of 8 blocks
// take 9 us in one slice and 15 in two, 32 tiles of 32 blocks that fill an SM 11 us in four and 21 in eight.
int slices_of(int64_t tiles, int64_t blocks, bool one_per_sm) {
    int s = 1;
    while (s < 8 && (one_per_sm ? 2 : 1) * tiles * s < sm_count() && blocks >= 8 * s) s *= 2;
    return s;
}

template <typename T, int NB>
int launch_few(const Operand &a, const Operand &w, const int32_t *offsets, int groups, const nb200_dense &y, cudaStream_t stream) {
    Workspace *ws = nullptr;
    int st;
    if ((st = report_of(stream, &ws))) return st;
    unsigned long long *report = reinterpret_cast<unsigned long long *>(ws->host) + 32;
    const int64_t wide = blocks_of(y.cols);
    // One group's turns over its weights have CTAs of their own; of several groups, whose rows nobody knows here, up to four while SMs are free for them.
    const int64_t used = std::min<int64_t>(groups, y.rows);
    int64_t turns = groups == 1 ? (y.rows + NB - 1) / NB : 1;
    while (groups > 1 && turns < 4 && wide * used * turns < 2 * sm_count()) turns *= 2;
    const int slices = slices_of(wide * used * (groups == 1 ? turns : 1), a.blocks, NB >= 64);
    // Short sums: a CTA takes several tiles of columns, one after another, while that leaves eight CTAs for every SM. (Its copies run ahead from tile to tile,
    // where a CTA's first take a microsecond or two: 112 experts of 3584 x 512 with 15 rows each 71 -> 60 us.)
    int each = 1;
    while (slices == 1 && each < 8 && a.blocks * each <= 8 && wide * used * turns >= (int64_t)16 * each * sm_count()) each *= 2;
    if (wide * slices > INT32_MAX || turns > 65535) return NB200_E_UNSUPPORTED;
    auto go = [&](auto kernel, size_t smem) -> int {
        if ((st = allow_shared(kernel, smem))) return st;
        LaunchScope scope("fp8_product_few", stream);
        NB200_CUDA(launch_overlapped_clusters(slices, kernel, dim3((unsigned)((wide + each - 1) / each * slices), (unsigned)groups, (unsigned)turns), dim3(FEW_THREADS), smem, stream, a, w,
                                              offsets, groups, y.rows, y.cols, static_cast<T *>(y.data), y.stride, each, report));
        return NB200_OK;
    };
    if constexpr (NB < 64)  // of more rows, long sums of so few tiles that they are always shared
        if (slices == 1) return go(k_product_few<T, NB, false>, FewShape<NB, false>::SHARED_BYTES);
    return go(k_product_few<T, NB, true>, FewShape<NB, true>::SHARED_BYTES);
}

// The result as the copy engine sees it: boxes of 32 rows by 128 bytes.
int describe(const nb200_dense &y, CUtensorMap *map) {
    typedef CUresult (*encode_fn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *, const cuuint32_t *,
                                  CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static std::atomic<encode_fn> known{nullptr};
    encode_fn encode = known.load(std::memory_order_acquire);
    if (!encode) {
        void *found = nullptr;
        cudaDriverEntryPointQueryResult how = cudaDriverEntryPointSymbolNotFound;
        NB200_CUDA(cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &found, 12000, cudaEnableDefault, &how));
        if (how != cudaDriverEntryPointSuccess || !found) return note_cuda_error(cudaErrorNotSupported, "cuTensorMapEncodeTiled");
        encode = reinterpret_cast<encode_fn>(found);
        known.store(encode, std::memory_order_release);
    }
    const CUtensorMapDataType type = y.type == NB200_F32   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                     : y.type == NB200_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                           : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    const cuuint64_t extents[2] = {(cuuint64_t)y.cols, (cuuint64_t)y.rows}, pitch[1] = {(cuuint64_t)(y.rows > 1 ? y.stride : y.cols) * type_size(y.type)};
    const cuuint32_t box[2] = {(cuuint32_t)(128 / type_size(y.type)), 32}, steps[2] = {1, 1};
    if (encode(map, type, 2, y.data, extents, pitch, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
        return note_cuda_error(cudaErrorInvalidValue, "cuTensorMapEncodeTiled");
    return NB200_OK;
}

// `tiles` of the shape that `pair` selects, at most.
template <typename T, bool GRAD>
int launch_product(const char *name, bool pair, int64_t tiles, const Operand &a, const Operand &w, const int32_t *offsets, int groups, const nb200_dense &y, cudaStream_t stream) {
    Workspace *ws = nullptr;
    int st;
    if ((st = report_of(stream, &ws))) return st;
    unsigned long long *report = reinterpret_cast<unsigned long long *>(ws->host) + 32;
    // As far as the copy engine counts a matrix (2^40 bytes from row to row); a result beyond that is written in words of its elements.
    const bool wide = word_bytes({&y}) == 16 && y.stride < int64_t(1) << 36 && y.rows < int64_t(1) << 31;
    CUtensorMap matrix{};
    if (wide && (st = describe(y, &matrix))) return st;
    auto go = [&](auto kernel, size_t smem, int ctas) -> int {
        if ((st = allow_shared(kernel, smem))) return st;
        LaunchScope scope(name, stream);
        NB200_CUDA(launch_overlapped(kernel, dim3((unsigned)std::min<int64_t>(tiles * ctas, sm_count() / ctas * ctas)), dim3(THREADS), smem, stream, a, w, offsets, groups,
                                     GRAD ? y.rows / groups : y.rows, y.cols, static_cast<T *>(y.data), y.stride, (int)tiles, report, matrix));
        return NB200_OK;
    };
    const int word = wide ? 16 : std::min(word_bytes({&y}), 4);
    auto sized = [&](auto bytes) {
        constexpr int WORD = decltype(bytes)::value;
        return pair ? go(k_product_pair<T, WORD, GRAD>, Shape<true>::SHARED_BYTES, 2) : go(k_product<T, WORD, GRAD>, Shape<false>::SHARED_BYTES, 1);
    };
    if (word == 16) return sized(std::integral_constant<int, 16>{});
    if constexpr (sizeof(T) == 2)
        if (word == 2) return sized(std::integral_constant<int, 2>{});
    return sized(std::integral_constant<int, 4>{});
}

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

// `rows`: x quantised by rows too, or none.
int quantise_columns(const nb200_dense *x, const int2 *block, int64_t bound, uint8_t *values, float *scales, const nb200_fp8 *rows, cudaStream_t stream) {
    const int64_t ctas = bound * blocks_of(x->cols);
    if (ctas == 0) return NB200_OK;
    if (ctas > INT32_MAX) return NB200_E_UNSUPPORTED;
    return with_type(x->type, [&](auto e) {
        using T = decltype(e);
        return with_vector<T>(word_bytes({x}), [&](auto v) {
            constexpr int V = decltype(v)::value;
            auto kernel = rows ? k_fp8_columns<T, V, true> : k_fp8_columns<T, V, false>;
            LaunchScope scope(rows ? "fp8_columns_rows" : "fp8_columns", stream);
            NB200_CUDA(launch_overlapped(kernel, dim3((unsigned)ctas), dim3(NT), 0, stream, static_cast<const T *>(x->data), x->stride, x->cols, block, values, scales,
                                         rows ? rows->values : nullptr, rows ? rows->scales : nullptr, padded_rows(x->rows)));
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
    const Operand oa{a->values, a->scales, blocks_of(a->cols), padded_rows(a->rows), 0};
    const Operand ow{w->values, w->scales, blocks_of(w->cols), padded_rows(w->rows), blocks_of(w->rows)};
    // Which kernel, by the rows of a group and the work there is (us on a B200, n x inner):
    //   - few rows: with groups while NB rows are three times the mean, so that hardly a group takes two turns (32 groups of 2048 x 2048: 28 against
    //     34 with 16 rows each, 35 against 34 with 24); one group up to 32 rows (4096 x 4096: 7 to 8 against 17), and where the sums are long enough
    //     to be worth sharing, up to 64 (4096 x 4096: 12 against 17; 1024 x 2048: 10 either way; 2048 x 1024: 13 against 7) and beyond, while
    //     tiles leave more than half of the SMs idle, so that a cluster shares them (128 rows, 1024 x 8192: 13 against 30; 4096 x 4096: 17 either
    //     way; at half, 9472 x 8192, nothing is shared: 42 against 29);
    //   - pairs of CTAs from where single ones have a second tile (4096 x 4096, 512 rows: 19 against 18; 768 rows: 20 against 31) and groups fill
    //     most of 128 rows (32 groups of 2048 x 2048 with 96 rows: 41 against 36, with 128 rows: 42 against 50);
    //   - no groups: the tiles' kernel, which finds none and clears the rows, all of them rows of no group.
    // tiles at most: a group may begin and end inside tiles
    const int64_t groups = w->groups, mean = groups ? (y->rows + groups - 1) / groups : 0, singles = blocks_of(y->rows) * blocks_of(y->cols);
    const bool one = groups == 1, idle = 2 * singles < sm_count(), pair = mean >= 112 && singles > sm_count();
    const int64_t side = pair ? 256 : 128, tiles = ((y->rows + side - 1) / side + 2 * groups) * ((y->cols + side - 1) / side);
    if (tiles > INT32_MAX / 64 || y->rows > INT32_MAX - 1024 || y->cols > INT32_MAX - 1024) return NB200_E_UNSUPPORTED;
    return with_type(y->type, [&](auto e) {
        using T = decltype(e);
        if (groups == 0) return launch_product<T, false>("fp8_product", false, tiles, oa, ow, offsets, 0, *y, stream);
        if (mean <= (one ? 16 : 5)) return launch_few<T, 16>(oa, ow, offsets, w->groups, *y, stream);
        if (mean <= (one ? 32 : 20)) return launch_few<T, 32>(oa, ow, offsets, w->groups, *y, stream);
        if (one && idle && mean <= 64 && oa.blocks >= 24) return launch_few<T, 64>(oa, ow, offsets, 1, *y, stream);
        if (one && idle && oa.blocks >= 48) return launch_few<T, 128>(oa, ow, offsets, 1, *y, stream);
        return launch_product<T, false>("fp8_product", pair, tiles, oa, ow, offsets, w->groups, *y, stream);
    });
}

int nb200_selftest_product_timeout(const nb200_fp8 *a, const nb200_fp8 *w, nb200_dense *y, void *stream_) {
    if (!fp8_ok(a) || !fp8_ok(w) || !dense_ok(y) || a->tiled || !w->tiled || w->groups != 1 || a->cols != w->cols || y->rows != a->rows || y->cols != w->rows ||
        y->type != NB200_F32 || y->rows == 0 || y->cols == 0 || a->cols == 0)
        return NB200_E_BADARG;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    Workspace *ws = nullptr;
    int st;
    if ((st = report_of(stream, &ws))) return st;
    const Operand oa{a->values, a->scales, blocks_of(a->cols), padded_rows(a->rows), 0};
    const Operand ow{w->values, w->scales, blocks_of(w->cols), padded_rows(w->rows), blocks_of(w->rows)};
    if ((st = allow_shared(k_product_selftest, Shape<false>::SHARED_BYTES))) return st;
    LaunchScope scope("fp8_product_selftest", stream);
    NB200_CUDA(launch_overlapped(k_product_selftest, dim3(1), dim3(THREADS), Shape<false>::SHARED_BYTES, stream, oa, ow, (const int32_t *)nullptr, 1, y->rows, y->cols,
                                 static_cast<float *>(y->data), y->stride, reinterpret_cast<unsigned long long *>(ws->host) + 32));
    return NB200_OK;
}

int64_t nb200_fp8_product_grad_w_scratch(const nb200_dense *dy, const nb200_dense *x, int32_t groups) {
    return grad_ok(dy, x, groups) ? (int64_t)GradScratch(nullptr, dy, x, groups).bytes : -1;
}

int nb200_fp8_product_grad_w(const nb200_dense *dy, const nb200_dense *x, int32_t groups, const int32_t *offsets, float *z, nb200_fp8 *dy_rows, void *scratch,
                             int64_t scratch_bytes, void *stream_) {
    if (!grad_ok(dy, x, groups) || (!offsets && groups != 1)) return NB200_E_BADARG;
    if (dy_rows && (!fp8_ok(dy_rows) || dy_rows->tiled || dy_rows->groups != 1 || dy_rows->rows != dy->rows || dy_rows->cols != dy->cols)) return NB200_E_BADARG;
    if (groups > NB200_MAX_EXPERTS) return NB200_E_UNSUPPORTED;
    if (groups == 0 || dy->cols == 0 || (x->cols == 0 && !dy_rows)) return NB200_OK;
    const GradScratch s(scratch, dy, x, groups);
    if ((!z && x->cols > 0) || !scratch || reinterpret_cast<uintptr_t>(scratch) % 256 != 0) return NB200_E_BADARG;
    if (scratch_bytes < (int64_t)s.bytes) return NB200_E_CAPACITY;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    {
        LaunchScope scope("group_blocks", stream);
        NB200_CUDA(launch_overlapped(k_group_blocks, dim3(1), dim3(1024), 0, stream, offsets, groups, (int)dy->rows, (int)s.bound, s.first_block, s.block));
    }
    int st;
    if ((st = quantise_columns(dy, s.block, s.bound, s.d, s.ds, dy_rows, stream))) return st;
    if (x->cols == 0) return NB200_OK;
    if ((st = quantise_columns(x, s.block, s.bound, s.x, s.xs, nullptr, stream))) return st;
    const Operand od{s.d, s.ds, s.bound, padded_rows(dy->cols), 0};
    const Operand ox{s.x, s.xs, s.bound, padded_rows(x->cols), 0};
    const nb200_dense result{(int64_t)groups * dy->cols, x->cols, x->cols, NB200_F32, z};
    const bool pair = dy->cols > 128 && x->cols > 128;
    const int64_t side = pair ? 256 : 128, tiles = groups * ((dy->cols + side - 1) / side) * ((x->cols + side - 1) / side);
    if (tiles > INT32_MAX / 64 || dy->cols > INT32_MAX - 1024 || x->cols > INT32_MAX - 1024) return NB200_E_UNSUPPORTED;
    return launch_product<float, true>("fp8_grad_w", pair, tiles, od, ox, s.first_block, groups, result, stream);
}

}  // extern "C"
