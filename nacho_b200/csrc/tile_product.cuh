// Products on the tensor cores whose sums stay in tensor memory until a tile is done: 16-bit floats and 8-bit integers. Tokens, which groups share
// unevenly, lie on the narrow side of the matrix instructions (N, any multiple of 32), weights on the wide one (M = 256), so that a group's
// last tile does hardly more work than its rows need.
//   GATED:   h[t, j] = act(sum_k x[t, k] w[g][j, k]) * sum_k x[t, k] w[g][hidden + j, k], and both sums where they are kept
//   ROWS:    y[t, j] = sum_k x[t, k] w[g][j, k], the second operand by rows or turned
//   WEIGHTS: z[g][m, n] = sum over the tokens t of group g of d[t, m] x[t, n]
#pragma once

#include <algorithm>
#include <type_traits>

#include "activation.cuh"
#include "dense_rows.cuh"
#include "product_waits.cuh"

namespace nb200 {

enum class Form { GATED, ROWS, WEIGHTS };

constexpr int TILE_STORE_WARPS = 8, TILE_THREADS = (TILE_STORE_WARPS + 4) * 32;
enum { TILE_MMA_WARP = TILE_STORE_WARPS, TILE_COPY_WARP, TILE_PLACE_WARP, TILE_TAIL_WARP };
constexpr int TILE_M = 256, TILE_N = 256, TILE_STEP = 32, TILE_PANEL = 8;  // of a pair of CTAs; the narrow side comes in steps; row tiles that follow one another

struct TileArgs {
    const int32_t *offsets;  // groups + 1, or none: one group of all rows
    int groups, rows;
    int wide;    // the result's extent on the side of M: hidden, columns of y, rows of z
    int across;  // WEIGHTS: columns of z
    int blocks;  // of 128 bytes along the summed axis (not WEIGHTS)
    int tile_n;  // TILE_N at most
    int pairs;   // of CTAs that the launch may take
    int parts;   // pairs that share a tile's blocks
    int b_bytes, stages;  // of the narrow operand in a stage; stages
    int most;    // tiles, at most
    void *y;
    int64_t stride;
    void *both;  // GATED: [rows][2 hidden] or none
    const float *row_scale, *col_scale;  // S8: of the rows, of every group's columns
    bool gelu;
    bool words;  // results in words of 16 bytes, whole tiles by the copy engine
    bool whole_wide;    // a block of the wide operand comes by one copy: 64 rows of gates and 64 of values, or 128 columns of a turned one
    bool whole_narrow;  // a whole tile's of the narrow one
    bool beside;  // nothing here depends on the kernel in front, which has itself waited for all that was before it: no wait but at the end
    unsigned long long *report;
    uint64_t patience;
    bool starve;  // a self-test: the first block's copies are left out
};

// The operands and the results as the copy engine sees them: boxes of rows of 128 bytes. Results: y [rows][columns], both [rows][2][hidden], z [group][rows][columns].
struct TileMaps {
    CUtensorMap wide, narrow, narrow_whole, y, both;  // narrow_whole: boxes of half a tile's narrow side
};

// A tile of the result: its group (-1: there are no more), where its rows begin and how many there are (for WEIGHTS: its columns), its first column (row), and the blocks that are summed.
struct Place {
    int g, from, count, col, blocks;
    int first, last;  // WEIGHTS: the group's tokens
};

// What a CTA of a pair has in shared memory; tiles begin at 1024-byte boundaries.
struct TileShared {
    static constexpr int STAGES = 8, SUMS = 2, PLACES = 4;  // blocks under way, at most; places for a tile's sums in tensor memory; tiles known ahead
    static constexpr int A_BYTES = 128 * 128;   // of a block: 128 rows of the wide side (turned: two blocks of 64 by 64 of the summed axis)
    static constexpr int STAGE_BYTES = 160 * 1024;
    uint8_t stage[STAGE_BYTES];            // of both operands' blocks, the wide one's first; `b_bytes` of the narrow one (half of the tile's narrow side)
    uint8_t out[2][24 * 1024];             // tiles of 32 rows by 128 bytes on their way out, of four warps each
    uint64_t full[STAGES], empty[STAGES];  // the leader's: a stage's copies of both CTAs have landed; its matrix instructions are done
    uint64_t landed[STAGES];               // this CTA's copies have, of a block whose tail is to be cleared
    uint64_t sum_full[SUMS], sum_empty[SUMS];  // a tile's sums lie in tensor memory; they have been read
    uint64_t place_full[PLACES], place_empty[PLACES];  // a tile's place is known; all warps know it
    uint64_t drained;
    Place place[PLACES];
    uint32_t tmem;
    int failed;
};
constexpr size_t TILE_SHARED_BYTES = sizeof(TileShared) + 1024;
static_assert(TILE_SHARED_BYTES <= 227 * 1024, "");

// Where a tile lies, found by a whole warp: groups 32 at a time, whose tiles it counts. Tiles are asked for in rising order. `most`: as many as there
// are with offsets that rise; others end there.
template <Form FORM>
struct TileWalk {
    const TileArgs &p;
    int per_tile;  // columns of the result in a tile
    int chunk = -32, base = 0, incl = 0, from = 0, to = 0;

    __device__ explicit TileWalk(const TileArgs &args) : p(args), per_tile(FORM == Form::GATED ? TILE_M / 2 : TILE_M) {}

    __device__ void range(int g, int &lo, int &hi) const {
        lo = p.offsets ? min(max(ld_late(p.offsets + g), 0), p.rows) : 0;
        hi = p.offsets ? min(max(ld_late(p.offsets + g + 1), lo), p.rows) : p.rows;
    }
    __device__ bool find(int tile, Place &t) {
        if (tile >= p.most) return false;
        const int wide = (p.wide + per_tile - 1) / per_tile;
        int row, col;
        if constexpr (FORM == Form::WEIGHTS) {
            const int narrow = (p.across + p.tile_n - 1) / p.tile_n;
            t.g = (int)((unsigned)tile / (unsigned)(narrow * wide));
            if (t.g >= p.groups) return false;
            range(t.g, t.first, t.last);
            place_tile<TILE_PANEL>(tile - t.g * narrow * wide, narrow, wide, &row, &col);
            t.from = row * p.tile_n;
            t.count = min(p.tile_n, p.across - t.from);
            t.blocks = (t.last - t.first + 63) / 64;
        } else {
            int total;
            while (total = __shfl_sync(FULL_MASK, incl, 31), tile >= base + total) {
                base += total;
                chunk += 32;
                if (chunk >= p.groups) return false;
                const int g = chunk + lane_id();
                from = to = 0;
                if (g < p.groups) range(g, from, to);
                incl = warp_incl_sum((int)min((int64_t)((to - from + p.tile_n - 1) / p.tile_n) * wide, (int64_t)p.most));
            }
            const int src = __ffs(__ballot_sync(FULL_MASK, base + incl > tile)) - 1;
            const int begin = __shfl_sync(FULL_MASK, from, src), end = __shfl_sync(FULL_MASK, to, src), high = (end - begin + p.tile_n - 1) / p.tile_n;
            t.g = chunk + src;
            place_tile<TILE_PANEL>(tile - base - (__shfl_sync(FULL_MASK, incl, src) - high * wide), high, wide, &row, &col);
            t.from = begin + row * p.tile_n;
            t.count = min(p.tile_n, end - t.from);
            t.blocks = p.blocks;
        }
        t.col = col * per_tile;
        return true;
    }
};

// The tiles of a pair of CTAs: one of every round of as many as there are pairs, another place in each, since groups' last tiles, which cost less, may come
// at a distance that divides the round (experts of 1000 rows: every fourth tile, and half of 74 pairs got all of them).
struct Turns {
    int base = 0, place, pairs, turn;
    __device__ Turns(int pair, int all) : place(pair), pairs(all), turn(31 % all) {}
    __device__ int tile() const { return base + place; }
    __device__ void next() {
        base += pairs;
        place += turn;
        if (place >= pairs) place -= pairs;
    }
};

// ---- the kernel ------------------------------------------------------------------------

// The four warps that share half of a tile's columns meet.
__device__ __forceinline__ void half_sync(int half) { asm volatile("barrier.cta.sync %0, 128;" ::"r"(half + 1) : "memory"); }
// And learn whether all of them are fine.
__device__ __forceinline__ bool half_all(int half, bool fine) {
    uint32_t all;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.u32 p, %1, 0;\n\t"
        "barrier.cta.red.and.pred q, %2, 128, p;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(all)
        : "r"((uint32_t)fine), "r"(half + 1)
        : "memory");
    return all != 0;
}

// Fragments of 16 lanes of M by 32 columns of N into tiles of 128-byte rows laid out as the copy engine takes them. By columns: row n of the tile, 16 elements
// from the 16-byte piece `piece` on.
template <typename T>
__device__ __forceinline__ void put_columns(uint8_t *tile, int piece, const float (&v)[16]) {
    const int q = lane_id() >> 3, r = lane_id() & 7;
#pragma unroll
    for (int j = 0; j < 4; j += 2) {
        const int row = 8 * (j + q / 2) + r;
        store_matrices<true>(tile + piece_at(row, piece + (q & 1)), pack2<T>(v[4 * j], v[4 * j + 1]), pack2<T>(v[4 * j + 2], v[4 * j + 3]), pack2<T>(v[4 * j + 4], v[4 * j + 5]),
                             pack2<T>(v[4 * j + 6], v[4 * j + 7]));
    }
}
// By lanes: rows `row` .. row + 15, 32 elements from `piece` on.
template <typename T>
__device__ __forceinline__ void put_lanes(uint8_t *tile, int row, int piece, const float (&v)[16]) {
    const int q = lane_id() >> 3, r = lane_id() & 7;
#pragma unroll
    for (int j = 0; j < 4; j += 2)
        store_matrices<false>(tile + piece_at(row + 8 * (q & 1) + r, piece + j + q / 2), pack2<T>(v[4 * j], v[4 * j + 1]), pack2<T>(v[4 * j + 2], v[4 * j + 3]),
                              pack2<T>(v[4 * j + 4], v[4 * j + 5]), pack2<T>(v[4 * j + 6], v[4 * j + 7]));
}
// Stores that depend on a condition, without a branch: a warp whose threads part and meet again at each of them takes 200 cycles a row.
__device__ __forceinline__ void store_if(bool yes, void *p, uint32_t v) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %2, 0;\n\t@p st.global.u32 [%0], %1;\n\t}" ::"l"(p), "r"(v), "r"((uint32_t)yes) : "memory");
}
__device__ __forceinline__ void store_if(bool yes, void *p, uint16_t v) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %2, 0;\n\t@p st.global.u16 [%0], %1;\n\t}" ::"l"(p), "h"(v), "r"((uint32_t)yes) : "memory");
}
// Rows first, first + step, .. below `rows` (32 at most) of such a tile to memory, `cols` elements of each: in words of 16 bytes, or of 4, which begin at a row's
// first or second element, whichever lies on a boundary.
template <int STEP, typename T>
__device__ __forceinline__ void flush(const uint8_t *tile, bool words, T *to, int64_t stride, int first, int rows, int cols) {
    const int lane = lane_id();
    if (words) {
        const int p = lane & 7;
        for (int r = first + lane / 8 * STEP; r < rows; r += 4 * STEP)
            if (p * 8 < cols) *reinterpret_cast<uint4 *>(to + r * stride + p * 8) = *reinterpret_cast<const uint4 *>(tile + piece_at(r, p));
        return;
    }
    const int end = min(cols, 64);
    if (end <= 0) return;
    T *row = to + first * stride;
#pragma unroll
    for (int i = 0; i < 32; i += 8 * STEP) {
        uint32_t w[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) w[k] = *reinterpret_cast<const uint32_t *>(tile + piece_at(first + i + k * STEP, lane / 4) + (lane & 3) * 4);
#pragma unroll
        for (int k = 0; k < 8; ++k, row += STEP * stride) {
            const uint32_t next = __shfl_down_sync(FULL_MASK, w[k], 1);
            const bool there = first + i + k * STEP < rows, odd = reinterpret_cast<uintptr_t>(row) & 2;
            const int e = 2 * lane + odd;
            const uint32_t out = odd ? __funnelshift_r(w[k], next, 16) : w[k];
            store_if(there && e + 1 < end, row + e, out);
            store_if(there && e + 1 == end, row + e, (uint16_t)out);
            store_if(there && odd && lane == 0, row, (uint16_t)w[k]);
        }
    }
}

// What becomes of a tile's sums: 32 columns of the warp's 32 lanes at a time, as fragments (first of the upper, then of the lower 16 lanes; where results are
// 32-bit, all of a thread's lane). Four warps, the ones that share half of the columns, store together.
template <Sum SUM, Form FORM, typename T>
struct Finish {
    static constexpr bool GATED = FORM == Form::GATED, WIDE = std::is_same<T, float>::value;
    const TileArgs &args;
    const TileMaps &maps;
    uint8_t *const out;
    const int rank, lanes, half;
    int turn = 0;
    float col_scale[4] = {};

    __device__ T *y() const { return static_cast<T *>(args.y); }

    __device__ __forceinline__ void begin(const Place &t) {
        if constexpr (SUM == Sum::S8) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int c = t.col + rank * 128 + lanes * 32 + (WIDE ? lane_id() : lane_id() / 4 + 8 * i);
                if (c < args.wide) col_scale[i] = ld_late(args.col_scale + (int64_t)t.g * args.wide + c);
            }
        }
    }
    __device__ __forceinline__ void value(const uint32_t (&v)[32], int first, float row_scale, float (&f)[16]) const {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            if constexpr (SUM == Sum::S8) f[i] = scaled((int)v[first + i], __shfl_sync(FULL_MASK, row_scale, i / 4 * 8 + (lane_id() & 3) * 2 + (i & 1)), col_scale[first / 8 + (i & 2) / 2]);
            else f[i] = __uint_as_float(v[first + i]);
        }
    }

    // GATED, ROWS: rows t.from + c .. of the result
    __device__ __forceinline__ void rows(const Place &t, int c, const uint32_t (&v)[32]) {
        const int lane = lane_id(), left = t.count - c, row = t.from + c;
        float row_scale = 0.f;
        if constexpr (SUM == Sum::S8) row_scale = lane < left ? ld_late(args.row_scale + row + lane) : 0.f;
        if constexpr (WIDE) {
            const int col = t.col + rank * 128 + lanes * 32 + lane;
#pragma unroll
            for (int j = 0; j < 32; ++j) {
                const float f = SUM == Sum::S8 ? scaled((int)v[j], __shfl_sync(FULL_MASK, row_scale, j), col_scale[0]) : __uint_as_float(v[j]);
                if (j < left && col < args.wide) y()[(int64_t)(row + j) * args.stride + col] = f;
            }
        } else {
            constexpr int TILES = GATED ? 3 : 2;  // of 64 columns: of h, gates and values, or two of y
            const int col = t.col + (GATED ? rank * 64 : rank * 128), wide = args.wide;
            // behind the group's last row there is no other's row, or these 32 are all the group's
            const bool whole = args.words && (left >= 32 || t.from + t.count == args.rows);
            uint8_t *const place = out + turn * TILES * 4096;
            turn ^= 1;
            float lo[16], hi[16];
            value(v, 0, row_scale, lo);
            value(v, 16, row_scale, hi);
            if (lanes == 0 && elected()) stores_read_but<1>();
            half_sync(half);  // this place has been read
            if constexpr (GATED) {
                if (args.both) {
                    put_columns<T>(place + 4096, lanes * 2, lo);
                    put_columns<T>(place + 2 * 4096, lanes * 2, hi);
                }
                float h[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) h[i] = lo[i] * logistic(act_inner(lo[i], args.gelu)) * hi[i];
                put_columns<T>(place, lanes * 2, h);
            } else {
                put_columns<T>(place + (lanes >> 1) * 4096, (lanes & 1) * 4, lo);
                put_columns<T>(place + (lanes >> 1) * 4096, (lanes & 1) * 4 + 2, hi);
            }
            if (whole) fence_async_shared();
            half_sync(half);
            if (whole) {
                if (lanes == 0 && col < wide && elected()) {
                    store_tile3(&maps.y, place, col, row, 0);
                    if constexpr (GATED) {
                        if (args.both) store_tile3(&maps.both, place + 4096, col, 0, row), store_tile3(&maps.both, place + 2 * 4096, col, 1, row);
                    } else {
                        if (col + 64 < wide) store_tile3(&maps.y, place + 4096, col + 64, row, 0);
                    }
                }
            } else {
                const int count = min(32, left);
                T *const to = y() + (int64_t)row * args.stride + col;
                flush<4>(place, args.words, to, args.stride, lanes, count, wide - col);
                if constexpr (GATED) {
                    if (args.both) {
                        T *const both = static_cast<T *>(args.both) + (int64_t)row * 2 * wide + col;
                        flush<4>(place + 4096, args.words, both, 2 * (int64_t)wide, lanes, count, wide - col);
                        flush<4>(place + 2 * 4096, args.words, both + wide, 2 * (int64_t)wide, lanes, count, wide - col);
                    }
                } else {
                    flush<4>(place + 4096, args.words, to + 64, args.stride, lanes, count, wide - col - 64);
                }
            }
            if (lanes == 0 && elected()) close_stores();  // an empty group where the warps have written themselves
        }
    }

    // WEIGHTS: columns t.from + c .. of 32 rows, 64 of them in two parts. (Written by the threads, a row each, without a stop in shared memory, both gradients of 16
    // experts took 535 us where this takes 520.)
    __device__ __forceinline__ void columns(const Place &t, int c, const uint32_t (&v)[2][32]) {
        const int row = t.col + rank * 128 + lanes * 32;
        uint8_t *const place = out + lanes * 6144;
        if (args.words && elected()) stores_read_but<0>();
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float lo[16], hi[16];
            value(v[i], 0, 0.f, lo);
            value(v[i], 16, 0.f, hi);
            put_lanes<T>(place, 0, 4 * i, lo);
            put_lanes<T>(place, 16, 4 * i, hi);
        }
        if (args.words) {
            fence_async_shared();
            __syncwarp();
            if (row < args.wide && elected()) store_tile3(&maps.y, place, t.from + c, row, t.g), close_stores();
        } else {
            __syncwarp();
            flush<1>(place, false, y() + ((int64_t)t.g * args.wide + row) * args.stride + t.from + c, args.stride, 0, min(32, args.wide - row), t.count - c);
            __syncwarp();
        }
    }

    __device__ __forceinline__ void end() {
        if (args.words && elected()) stores_done();
        __syncwarp();
    }
};

// Which of `all` places is next, and in which phase of its barriers.
struct Stages {
    int all, at = 0;
    uint32_t phase = 0;
    __device__ explicit Stages(int n) : all(n) {}
    __device__ void next() {
        if (++at == all) at = 0, phase ^= 1;
    }
};

// Pairs of CTAs, one CTA per SM, take tiles of 256 x 256 at most in turn. One warp finds out where they lie, some ahead of the others (half a dozen divisions and
// the group's offsets: found by every warp for itself at the tile's beginning, the matrix instructions of short sums waited for it), one brings blocks of 128
// bytes of both operands into shared memory (the copy engine's tiled form, which turns them as the tensor cores take them and fills up with zeros what lies
// beyond a matrix), one issues the matrix instructions, and eight read the sums of a whole tile while those of the next one are made: tensor memory holds two.
// 4096 x 8192 x 4096 gated, both sums kept: 504 K cycles with the tensor cores busy 95 %, which the power cap makes 322 to 345 us alone and 406 to 426 in call after call; without them
// kept 502 K cycles and 96 %. 8192^3 in integers: 498 K cycles, 300 to 322 us alone.
//
// GATED: 16 rows of gates and 16 of values alternate in the wide operand's tile, so that a gate and its value lie 16 lanes apart in tensor memory and fragments
// of both land in the same thread.
// WEIGHTS: the last block of a group's tokens runs into the next group's. Steps of 16 tokens that are not the group's are left out, and in the last step the rows
// behind its last token are cleared in shared memory.
// SPLIT: where there are tiles for a part of the SMs only, the pairs of a cluster have a part of a tile's blocks each and add up their sums, in order, through
// one another's shared memory.
template <Sum SUM, Form FORM, bool A_TURNED, bool SPLIT, typename T>
__global__ void __launch_bounds__(TILE_THREADS, 1) k_tiles(const TileArgs args, const __grid_constant__ TileMaps maps) {
    constexpr int SUMS = TileShared::SUMS;
    constexpr bool B_TURNED = FORM == Form::WEIGHTS, GATED = FORM == Form::GATED, WIDE = std::is_same<T, float>::value;
    constexpr int PER_BLOCK = SUM == Sum::S8 ? 128 : 64, UNIT = FORM == Form::WEIGHTS ? 64 : 32;  // elements of a block; columns that are finished at once
    extern __shared__ uint8_t raw[];
    TileShared &sh = *reinterpret_cast<TileShared *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
    const int warp = warp_id(), lane = lane_id(), cta = (int)cluster_rank(), rank = cta & 1, leader = cta & ~1, part = cta >> 1, parts = SPLIT ? (int)cluster_size() / 2 : 1;
    if (threadIdx.x == 0) {
        for (int s = 0; s < args.stages; ++s) mbar_init(&sh.landed[s], 1), mbar_init(&sh.full[s], FORM == Form::WEIGHTS ? 2 : 1), mbar_init(&sh.empty[s], 1);
        for (int s = 0; s < SUMS; ++s) mbar_init(&sh.sum_full[s], 1), mbar_init(&sh.sum_empty[s], TILE_STORE_WARPS * 2);
        for (int s = 0; s < TileShared::PLACES; ++s) mbar_init(&sh.place_full[s], 1), mbar_init(&sh.place_empty[s], TILE_STORE_WARPS + 1 + (rank == 0) + (FORM == Form::WEIGHTS));
        mbar_init(&sh.drained, 1);
        mbar_fence_init();
        sh.failed = 0;
        ask_for_map(&maps.wide), ask_for_map(B_TURNED ? &maps.narrow : &maps.narrow_whole);
    }
    if (warp == TILE_MMA_WARP) tmem_alloc<true>(&sh.tmem, 512);
    tmem_fence_before();
    __syncthreads();
    cluster_sync();  // nobody arrives at a barrier that is not there yet
    tmem_fence_after();
    const uint32_t tmem = *(volatile uint32_t *)&sh.tmem;
    volatile int *failed = &sh.failed;
    // In this order: what starts beside this kernel then finds everything complete that was in front of it.
    if (!args.beside) wait_for_previous();
    trigger_dependents();

    Place t{};
    Ring<TileShared::PLACES> places;
    // The next tile, for a whole warp; false once a wait has given up.
    auto next_place = [&] {
        if (!wait_for(&sh.place_full[places.at], places.phase, failed, args.patience)) return false;
        t = sh.place[places.at];
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.place_empty[places.at]);
        places.next();
        return true;
    };
    const int stage_bytes = TileShared::A_BYTES + args.b_bytes;
    auto stage_a = [&](int s) { return sh.stage + s * stage_bytes; };
    auto stage_b = [&](int s) { return sh.stage + s * stage_bytes + TileShared::A_BYTES; };
    // Columns of N that the tile's matrix instructions have, half of which each CTA of the pair brings; the pair's part of the blocks.
    auto narrow = [&] { return (t.count + TILE_STEP - 1) / TILE_STEP * TILE_STEP; };
    auto first_block = [&] { return SPLIT ? (int)((int64_t)t.blocks * part / parts) : 0; };
    auto end_block = [&] { return SPLIT ? (int)((int64_t)t.blocks * (part + 1) / parts) : t.blocks; };
    // Tokens of block b if it is a group's last one and its last step of 16 is not whole, else 0.
    auto tail_rows = [&](int b) {
        const int rows = FORM == Form::WEIGHTS ? t.last - t.first - b * 64 : 64;
        return rows < 64 && rows % 16 ? rows : 0;
    };
    // The last block of a group's tokens has `rows` of them: what follows up to the next 16 is cleared in this CTA's halves of both operands.
    auto clear_tail = [&](int stage, int n, int rows) {
        const int stop = (rows + 15) / 16 * 16, chunks = (n / 2 + 63) / 64;
        for (int r = rows + lane / 8; r < stop; r += 4) {
            const int at = r * 128 + (lane & 7) * 16;
#pragma unroll
            for (int i = 0; i < 2; ++i) *reinterpret_cast<uint4 *>(stage_a(stage) + i * 8192 + at) = make_uint4(0, 0, 0, 0);
            for (int i = 0; i < chunks; ++i) *reinterpret_cast<uint4 *>(stage_b(stage) + i * 8192 + at) = make_uint4(0, 0, 0, 0);
        }
        fence_async_shared();
        __syncwarp();
    };
    const int lanes = warp & 3, half = warp >> 2;
    Finish<SUM, FORM, T> finish{args, maps, sh.out[half & 1], rank, lanes, half};
    bool fine = true;
    if (warp < TILE_STORE_WARPS) {
        Ring<SUMS> sums;
        for (;;) {
            fine = next_place();
            const int n = narrow();
            const bool any = fine && t.g >= 0 && end_block() > first_block();
            if (any) {
                fine = wait_for(&sh.sum_full[sums.at], sums.phase, failed, args.patience);
                tmem_fence_after();
            }
            fine = half_all(half, fine);  // nobody waits for a warp that has given up
            if (!fine || t.g < 0) break;
            const uint32_t base = tmem + ((uint32_t)(lanes * 32) << 16) + sums.at * TILE_N;
            auto load = [&](int c, uint32_t (&v)[32]) {
                if (!any || c >= n) {
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[i] = 0;
                } else if constexpr (WIDE) {
                    tmem_load(base + c, v);
                    tmem_wait_loads(v);
                } else {
                    uint32_t lo[16], hi[16];
                    tmem_load_fragments(base + c, lo);
                    tmem_load_fragments(base + c + (16u << 16), hi);
                    tmem_wait_loads(lo);
                    tmem_wait_loads(hi);
#pragma unroll
                    for (int i = 0; i < 16; ++i) v[i] = lo[i], v[16 + i] = hi[i];
                }
            };
            auto all_read = [&] {  // the tile's place is free again, as far as this warp goes
                if (!any) return;
                tmem_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_at<false>(&sh.sum_empty[sums.at], leader);
            };
            if (!SPLIT) finish.begin(t);
            for (int c = half * UNIT; c < n; c += 2 * UNIT) {
                uint32_t v[UNIT / 32][32];
#pragma unroll
                for (int i = 0; i < UNIT / 32; ++i) load(c + 32 * i, v[i]);
                if constexpr (SPLIT) {
                    // behind the last matrix instruction the stages are free
#pragma unroll
                    for (int i = 0; i < UNIT / 32; ++i)
                        if (c + 32 * i < n)
#pragma unroll
                            for (int k = 0; k < 32; ++k) reinterpret_cast<uint32_t *>(sh.stage)[((c / 32 + i) * 4 + lanes) * 1024 + k * 32 + lane] = v[i][k];
                } else {
                    if (c + 2 * UNIT >= n) all_read();
                    if constexpr (FORM == Form::WEIGHTS) finish.columns(t, c, v);
                    else finish.rows(t, c, v[0]);
                }
            }
            if (SPLIT) break;  // one tile per cluster
            if (half * UNIT >= n) all_read();  // a narrow tile is the other half's
            if (any) sums.next();
        }
        if (!SPLIT) finish.end();
        // rows of no group
        if (FORM != Form::WEIGHTS && args.offsets) {
            T *const y = static_cast<T *>(args.y);
            const int64_t rows = args.rows, lo = min(max((int64_t)ld_late(args.offsets), (int64_t)0), rows), hi = min(max((int64_t)ld_late(args.offsets + args.groups), lo), rows);
            for (int64_t r = blockIdx.x * TILE_STORE_WARPS + warp; r < rows; r += (int64_t)gridDim.x * TILE_STORE_WARPS) {
                if (r >= lo && r < hi) continue;
                for (int64_t c = lane; c < args.wide; c += 32) y[r * args.stride + c] = from_float<T>(0.f);
                if (GATED && args.both)
                    for (int64_t c = lane; c < 2 * (int64_t)args.wide; c += 32) static_cast<T *>(args.both)[r * 2 * args.wide + c] = from_float<T>(0.f);
            }
        }
    } else {
        Stages stage(args.stages);
        if (warp == TILE_PLACE_WARP) {
            Turns turns((int)blockIdx.x / (2 * parts), (int)gridDim.x / (2 * parts));
            TileWalk<FORM> walk(args);
            for (bool more = true; more; turns.next(), places.next()) {
                if (!wait_for(&sh.place_empty[places.at], places.phase ^ 1, failed, args.patience)) break;
                more = walk.find(turns.tile(), t);
                if (!more) t.g = -1;
                if (lane == 0) {
                    sh.place[places.at] = t;
                    mbar_arrive(&sh.place_full[places.at]);
                }
                __syncwarp();
            }
        } else if (warp == TILE_COPY_WARP) {
            while ((fine = next_place()) && t.g >= 0) {
                const int n = narrow(), mine = n / 2;
                const uint32_t bytes = TileShared::A_BYTES + (B_TURNED ? (mine + 63) / 64 * 8192 : (mine + 31) / 32 * 4096);
                const int begin = t.from + rank * mine, end = end_block();
                for (int b = first_block(); b < end; ++b, stage.next()) {
                    if (!(fine = wait_for(&sh.empty[stage.at], stage.phase ^ 1, failed, args.patience))) break;
                    if (elected() && !(args.starve && b == 0)) {
                        // Both CTAs' copies report to the leader, which expects them; those of a block whose tail is to be cleared to their own CTA.
                        const bool tail = tail_rows(b) > 0;
                        const uint32_t bar = tail ? smem_u32(&sh.landed[stage.at]) : remote_barrier(&sh.full[stage.at], leader);
                        if (tail) mbar_arrive_expect_tx(&sh.landed[stage.at], bytes);
                        else if (rank == 0) mbar_arrive_expect_tx(&sh.full[stage.at], 2 * bytes);
                        if (FORM == Form::WEIGHTS && !tail && rank == 0) mbar_arrive(&sh.full[stage.at]);  // of two, for the two warps that clear tails
                        const int k = FORM == Form::WEIGHTS ? t.first + b * 64 : b * PER_BLOCK;
                        uint8_t *const to_a = stage_a(stage.at), *const to_b = stage_b(stage.at);
                        if constexpr (GATED) {
                            const int col = t.col + rank * 64;
                            if (args.whole_wide) {
                                load_tile5(to_a, &maps.wide, k, col / 16, t.g, bar);
                            } else {
#pragma unroll
                                for (int i = 0; i < 4; ++i) {
                                    load_tile(to_a + i * 4096, &maps.wide, k, col + 16 * i, t.g, bar);
                                    load_tile(to_a + i * 4096 + 2048, &maps.wide, k, args.wide + col + 16 * i, t.g, bar);
                                }
                            }
                        } else if constexpr (A_TURNED) {
                            const int col = t.col + rank * 128, g = FORM == Form::WEIGHTS ? 0 : t.g;
                            if (args.whole_wide) {
                                load_tile4(to_a, &maps.wide, k, col / 64, g, bar);
                            } else {
                                load_tile(to_a, &maps.wide, col, k, g, bar);
                                load_tile(to_a + 8192, &maps.wide, col + 64, k, g, bar);
                            }
                        } else {
                            load_tile(to_a, &maps.wide, k, t.col + rank * 128, t.g, bar);
                        }
                        if constexpr (B_TURNED) {
                            if (args.whole_narrow && n == args.tile_n) load_tile4(to_b, &maps.narrow_whole, k, begin / 64, 0, bar);
                            else
                                for (int i = 0; i < mine; i += 64) load_tile(to_b + i * 128, &maps.narrow, begin + i, k, 0, bar);
                        } else if (args.whole_narrow && n == args.tile_n) {
                            load_tile(to_b, &maps.narrow_whole, k, begin, 0, bar);
                        } else {
                            for (int i = 0; i < mine; i += 32) load_tile(to_b + i * 128, &maps.narrow, k, begin + i, 0, bar);
                        }
                    }
                    __syncwarp();
                }
                if (!fine) break;
            }
            if (!fine)  // nothing may land in shared memory that is no longer this CTA's: what was to come until then has, or never will
                for (const uint64_t start = now_ns(); now_ns() - start < SHORT_PATIENCE;) {}
        } else if (warp == TILE_MMA_WARP && rank == 0) {
            const uint64_t tile_a = A_TURNED ? turned_descriptor(smem_u32(stage_a(0))) : tile_descriptor(smem_u32(stage_a(0)));
            const uint64_t tile_b = B_TURNED ? turned_descriptor(smem_u32(stage_b(0))) : tile_descriptor(smem_u32(stage_b(0)));
            const uint32_t both = 3u << leader;
            Ring<SUMS> sums;
            while ((fine = next_place()) && t.g >= 0) {
                const int n = narrow(), begin = first_block(), end = end_block();
                const uint32_t shape = sum_descriptor<SUM>(A_TURNED, B_TURNED, TILE_M) | (uint32_t)(n >> 3) << 17;
                if (begin == end) continue;
                if (!(fine = wait_for(&sh.sum_empty[sums.at], sums.phase ^ 1, failed, args.patience))) break;
                for (int b = begin; b < end; ++b, stage.next()) {
                    if (!(fine = wait_for(&sh.full[stage.at], stage.phase, failed, args.patience))) break;
                    const int rows = FORM == Form::WEIGHTS ? t.last - t.first - b * 64 : 64;
                    // The other CTA's warp has written there too. The phase is over: not to see that would be a fault, which ends as a wait that gives up does.
                    if (tail_rows(b) && !(fine = __all_sync(FULL_MASK, mbar_acquire_cluster(&sh.full[stage.at], stage.phase)))) {
                        *failed = 1;
                        break;
                    }
                    tmem_fence_after();
                    if (elected()) {
                        const uint64_t da = tile_a + (uint64_t)(stage.at * (stage_bytes >> 4)), db = tile_b + (uint64_t)(stage.at * (stage_bytes >> 4));
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            if (FORM != Form::WEIGHTS || k * 16 < rows)
                                mma_pair<SUM>(tmem + sums.at * TILE_N, da + (A_TURNED ? 128 : 2) * k, db + (B_TURNED ? 128 : 2) * k, shape, b > begin || k > 0);
                        mma_commit_pair(&sh.empty[stage.at], both);
                        if (b + 1 == end) mma_commit_pair(&sh.sum_full[sums.at], both);
                    }
                    __syncwarp();
                }
                if (!fine) break;
                sums.next();
            }
            if (!fine) {
                if (elected()) mma_commit_pair(&sh.drained, both);
                __syncwarp();
                drain(&sh.drained, 0);
            }
        } else if (FORM == Form::WEIGHTS && warp == TILE_TAIL_WARP) {
            uint32_t phases = 0;  // of the stages' `landed`
            while ((fine = next_place()) && t.g >= 0) {
                const int n = narrow(), begin = first_block(), end = end_block();
                for (int b = begin; b < end; ++b, stage.next()) {
                    const int rows = tail_rows(b);
                    if (!rows) continue;
                    if (!(fine = wait_for(&sh.landed[stage.at], phases >> stage.at & 1, failed, args.patience))) break;
                    phases ^= 1u << stage.at;
                    clear_tail(stage.at, n, rows);
                    if (elected()) mbar_arrive_at<true>(&sh.full[stage.at], leader);
                    __syncwarp();
                }
                if (!fine) break;
            }
        }
    }
    if constexpr (SPLIT) {
        cluster_sync();
        if (warp < TILE_STORE_WARPS && half_all(half, fine && t.g >= 0)) {
            const int n = narrow();
            finish.begin(t);
            for (int c = (half + 2 * part) * UNIT; c < n; c += 2 * parts * UNIT) {
                uint32_t v[UNIT / 32][32];
#pragma unroll
                for (int i = 0; i < UNIT / 32; ++i) {
                    const uint32_t *const mine = reinterpret_cast<const uint32_t *>(sh.stage) + ((c / 32 + i) * 4 + lanes) * 1024 + lane;
#pragma unroll
                    for (int k = 0; k < 32; ++k) v[i][k] = 0;
                    for (int p = 0; p < parts && c + 32 * i < n; ++p) {
                        uint32_t w[32];
#pragma unroll
                        for (int k = 0; k < 32; ++k) w[k] = __float_as_uint(load_remote(reinterpret_cast<const float *>(mine + k * 32), 2 * p + rank));
#pragma unroll
                        for (int k = 0; k < 32; ++k) v[i][k] = SUM == Sum::S8 ? v[i][k] + w[k] : __float_as_uint(__uint_as_float(v[i][k]) + __uint_as_float(w[k]));
                    }
                }
                if constexpr (FORM == Form::WEIGHTS) finish.columns(t, c, v);
                else finish.rows(t, c, v[0]);
            }
            finish.end();
        }
    }
    tmem_fence_before();
    __syncthreads();
    cluster_sync();  // no arrival is on its way to a CTA that is gone
    if (warp == TILE_MMA_WARP) {
        tmem_fence_after();
        tmem_free<true>(tmem, 512);
        if (lane == 0 && *failed) publish_result_word(args.report, 1, REPORT_OTHER | blockIdx.x);
    }
    if (args.beside) finish_after_previous();
}

// ---- host ------------------------------------------------------------------------------

// Whether the copy engine can read the rows: 16-byte boundaries, rows that do not overlap, less than 2^40 bytes from row to row and group to group.
inline bool tiles_readable(const nb200_dense &x, int64_t groups) {
    const int64_t size = (int64_t)type_size(x.type), per_group = groups ? x.rows / groups : 0;
    return reinterpret_cast<uintptr_t>(x.data) % 16 == 0 && (x.rows <= 1 || (x.stride * size % 16 == 0 && x.stride >= x.cols && x.stride < (int64_t(1) << 40) / size)) &&
           (groups <= 1 || per_group * x.stride < (int64_t(1) << 40) / size);
}

// `groups` matrices of rows, one after another, in boxes of `box_rows` rows of 128 bytes.
inline int describe_rows(CUtensorMap *map, CUtensorMapDataType type, void *data, int64_t size, int64_t cols, int64_t rows, int64_t groups, int64_t stride, int box_rows) {
    const cuuint64_t extents[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)groups};
    const cuuint64_t pitch = (cuuint64_t)(rows * groups > 1 ? stride : (cols * size + 15) / 16 * 16 / size) * size;
    const cuuint64_t pitches[2] = {pitch, groups > 1 ? pitch * (cuuint64_t)rows : pitch};
    const cuuint32_t box[3] = {(cuuint32_t)(128 / size), (cuuint32_t)box_rows, 1};
    return encode_matrix(map, type, 3, data, extents, pitches, box);
}
// The engine takes a copy for every block of an operand, not so much its bytes: with boxes of 16 and 32 rows, 12 copies for a block, 4096 x 8192 x 4096 gated (alone, sums not kept)
// took 368 us, with the largest ones 337.

// The narrow operand by rows, in boxes for parts of a tile and for half of a whole one.
inline int describe_narrow(TileMaps *maps, TileArgs *args, CUtensorMapDataType type, void *data, int64_t size, int64_t cols, int64_t rows, int64_t stride) {
    args->whole_narrow = true;
    const int st = describe_rows(&maps->narrow, type, data, size, cols, rows, 1, stride, 32);
    return st ? st : describe_rows(&maps->narrow_whole, type, data, size, cols, rows, 1, stride, args->tile_n / 2);
}
// A turned operand of 16-bit elements in blocks of 64 columns by 64 rows, `blocks` of them in a box, if its columns are sixty-fours (a row's last block would reach into
// the next row, the last row's beyond the matrix).
inline int describe_turned(CUtensorMap *map, bool *whole, CUtensorMapDataType type, void *data, int64_t cols, int64_t rows, int64_t groups, int64_t stride, int blocks) {
    *whole = cols % 64 == 0 && blocks > 0;
    if (!*whole) return NB200_OK;
    const cuuint64_t pitch = (cuuint64_t)(rows * groups > 1 ? stride : cols) * 2;
    const cuuint64_t extents[4] = {64, (cuuint64_t)rows, (cuuint64_t)cols / 64, (cuuint64_t)groups}, pitches[3] = {pitch, 128, groups > 1 ? pitch * (cuuint64_t)rows : pitch};
    const cuuint32_t box[4] = {64, 64, (cuuint32_t)blocks, 1};
    return encode_matrix(map, type, 4, data, extents, pitches, box);
}
// A result of `groups` matrices, if whole tiles of it can leave through the copy engine.
inline int describe_result(CUtensorMap *map, bool *words, CUtensorMapDataType type, const nb200_dense &y, int64_t groups) {
    const int64_t stride = y.rows > 1 ? y.stride : y.cols, limit = (int64_t(1) << 40) / 2, rows = y.rows / groups;
    *words = y.type != NB200_F32 && word_bytes({&y}) == 16 && stride < limit && (groups == 1 || rows * stride < limit);
    return *words ? describe_rows(map, type, y.data, 2, y.cols, rows, groups, stride, 32) : (int)NB200_OK;
}
inline CUtensorMapDataType map_type(int type) { return type == NB200_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16; }

inline int64_t all_pairs() { return std::max(1, sm_count() / 2); }

// A product as tiles: `rows` on the narrow side of all groups together, `wide_tiles` beside one another on the wide one, `blocks` summed for each. `results`: what the products wait
// for while a tile leaves, in the cost's rows of blocks.
struct TileWork {
    int64_t rows, groups, wide_tiles, blocks, results = 0;

    // How it goes on so many pairs of CTAs: the narrow side of its tiles, a multiple of 64, the pairs that share a tile's blocks, and what the busiest pair then has to
    // bring, in rows of blocks: 256 of the wide side and n of the narrow one for every tile and block (1330 of them take a microsecond); adding up parts takes as long
    // as 50 for each of the n columns.
    struct Way {
        int n, parts;
        double cost;
    };
    // Tiles at most, however the groups share the rows: each one that has any may leave one tile unfilled.
    int64_t most(int n) const { return (rows + std::min(groups, rows) * (n - 1)) / n * wide_tiles; }

    // Parts: as many pairs as find room for all tiles at once, of at least eight blocks each (`clusters`: of four and eight CTAs that the device holds. A second round
    // costs more than parts give: 16 tiles of 32 blocks take 19 us in four parts, of which the device holds fewer than 16, and 10 in two). A launch has a cluster for
    // every tile that there can be.
    Way best(int64_t pairs, const int (&clusters)[2]) const {
        const int64_t mean = (rows + groups - 1) / groups;
        Way way{0, 1, 0};
        for (int n = TILE_N; n >= 64; n -= 64) {
            const int64_t each_group = (mean + n - 1) / n * wide_tiles, tiles = std::min(groups, rows) * each_group, all = std::max(groups * each_group, most(n));
            const int64_t each = TILE_M + std::min<int64_t>(n, mean);
            for (int k = 0; k < 3; ++k) {
                const int parts = 1 << k;
                if (parts > 1 && (all * parts > pairs || all > clusters[k - 1] || blocks < 8 * parts)) break;
                const double cost = (double)((tiles + pairs - 1) / pairs) * ((double)each * (double)((blocks + parts - 1) / parts) + (double)results) + (parts > 1 ? 50 * std::min<int64_t>(n, mean) : 0);
                // One group's tiles are no wider than its rows: a stage then has that much more room for others, and a tile comes by one copy. Groups share the rows
                // unevenly: the wider side is for those that have more.
                if (way.n == 0 || cost < way.cost || (groups == 1 && cost == way.cost && parts == way.parts)) way = Way{n, parts, cost};
            }
        }
        return way;
    }
};

// Clusters of four and of eight CTAs that the device holds (all these kernels have the same threads and shared memory).
template <Sum SUM, Form FORM, bool A_TURNED, typename T>
int tile_clusters(int (&clusters)[2]) {
    auto split = k_tiles<SUM, FORM, A_TURNED, true, T>;
    if (const int st = allow_shared(split, TILE_SHARED_BYTES)) return st;
    for (int k = 0; k < 2; ++k) clusters[k] = resident_clusters(reinterpret_cast<const void *>(split), 4 << k, TILE_THREADS, TILE_SHARED_BYTES);
    return NB200_OK;
}

template <Sum SUM, Form FORM, bool A_TURNED, typename T>
int launch_tiles(const char *name, TileArgs args, const TileMaps &maps, cudaStream_t stream) {
    Workspace *ws = nullptr;
    int st;
    if ((st = report_of(stream, &ws))) return st;
    args.report = reinterpret_cast<unsigned long long *>(ws->host) + 32;
    const int64_t per_tile = FORM == Form::GATED ? TILE_M / 2 : TILE_M, wide = (args.wide + per_tile - 1) / per_tile;
    const TileWork work = FORM == Form::WEIGHTS ? TileWork{args.across, 1, args.groups * wide, 0} : TileWork{args.rows, args.groups, wide, 0};
    const int64_t tiles = work.most(args.tile_n);
    if (tiles > INT32_MAX / 64 || args.rows > INT32_MAX - 1024 || args.wide > INT32_MAX / 2 - 1024 || args.across > INT32_MAX - 1024) return NB200_E_UNSUPPORTED;
    args.most = (int)tiles;
    args.patience = args.starve ? SHORT_PATIENCE : PATIENCE;
    args.b_bytes = FORM == Form::WEIGHTS ? (args.tile_n / 2 + 63) / 64 * 8192 : args.tile_n / 2 * 128;
    args.stages = std::min(TileShared::STAGES, TileShared::STAGE_BYTES / (TileShared::A_BYTES + args.b_bytes));
    auto split = k_tiles<SUM, FORM, A_TURNED, true, T>;
    const int parts = args.parts;
    const int64_t ctas = parts > 1 ? tiles * 2 * parts : 2 * std::max<int64_t>(1, std::min<int64_t>(tiles, args.pairs));
    auto go = [&](auto kernel) -> int {
        if ((st = allow_shared(kernel, TILE_SHARED_BYTES))) return st;
        LaunchScope scope(name, stream);
        NB200_CUDA(launch_overlapped_clusters(2 * parts, kernel, dim3((unsigned)ctas), dim3(TILE_THREADS), TILE_SHARED_BYTES, stream, args, maps));
        return NB200_OK;
    };
    return parts > 1 ? go(split) : go(k_tiles<SUM, FORM, A_TURNED, false, T>);
}

}  // namespace nb200
