// What kernels of products on the tensor cores share: rings of barriers, waits that end, the order of tiles, and the word by which a kernel whose call
// has returned says that a wait gave up.
#pragma once

#include "block_utils.cuh"
#include "tensor_core.cuh"

namespace nb200 {

constexpr uint64_t PATIENCE = 2000000000, SHORT_PATIENCE = 20000000;  // ns, after which a wait gives up (microseconds are usual); the self-test's

// Which of N places is next, and in which phase of its barriers.
template <int N>
struct Ring {
    int at = 0;
    uint32_t phase = 0;
    __device__ void next() {
        if (++at == N) at = 0, phase ^= 1;
    }
};

// The order of the tiles of `high` x `wide`: panels of rows, column by column.
template <int PANEL>
__device__ __forceinline__ void place_tile(int within, int high, int wide, int *row, int *col) {
    const unsigned panel = (unsigned)within / (unsigned)(PANEL * wide), width = min((unsigned)PANEL, (unsigned)high - panel * PANEL);
    const unsigned rest = (unsigned)within - panel * PANEL * wide, column = rest / width;
    *row = (int)(panel * PANEL + rest - column * width);
    *col = (int)column;
}

__device__ __forceinline__ uint64_t now_ns() {
    uint64_t t;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
    return t;
}

// For a whole warp; false for all of it once one of its threads, or another warp of the CTA, has given up after `patience` ns.
__device__ __forceinline__ bool wait_for(uint64_t *bar, uint32_t parity, volatile int *failed, uint64_t patience) {
    uint64_t start = 0;
    for (int i = 1;; ++i) {
        if (__all_sync(FULL_MASK, mbar_try_wait(bar, parity))) return true;
        if (i % 64) continue;
        if (__any_sync(FULL_MASK, *failed)) return false;
        if (!start) start = now_ns();
        if (__any_sync(FULL_MASK, now_ns() - start > patience)) break;
    }
    *failed = 1;
    return false;
}
template <bool SELFTEST = false>
__device__ __forceinline__ bool wait_for(uint64_t *bar, uint32_t parity, volatile int *failed) {
    return wait_for(bar, parity, failed, SELFTEST ? SHORT_PATIENCE : PATIENCE);
}

// After a give-up: what is still on its way lands first, or never will.
__device__ __forceinline__ void drain(uint64_t *bar, uint32_t parity) {
    for (const uint64_t start = now_ns(); now_ns() - start < SHORT_PATIENCE && !mbar_try_wait(bar, parity);) {}
}

// ---- host ------------------------------------------------------------------------------

// The word by which a product of this stream says that a wait gave up. The call does not wait for its kernel, so the next one on the stream
// finds it and returns the error in its place. Its value is the CTA, with REPORT_OTHER where that was no product of 8-bit floating point.
constexpr unsigned long long REPORT_OTHER = 1ull << 32;
int report_of(cudaStream_t stream, Workspace **ws);

// A matrix (or several of them, `rank` 3 to 5) as the copy engine sees it, in boxes of rows of 128 bytes, turned as the tensor cores take them; what lies
// beyond it is read as zeros.
int encode_matrix(CUtensorMap *map, CUtensorMapDataType type, int rank, void *data, const cuuint64_t *extents, const cuuint64_t *pitches, const cuuint32_t *box);

}  // namespace nb200
