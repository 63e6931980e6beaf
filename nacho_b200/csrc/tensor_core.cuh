// Thin wrappers over the sm_100a tensor-core PTX that the products use: tensor memory, descriptors of shared-memory tiles,
// matrix instructions with 32-bit sums (on e4m3, 16-bit and 8-bit integer operands), and the barriers they complete on.
#pragma once

#include <cuda.h>

#include "tma.cuh"

namespace nb200 {

// PAIR: by two CTAs of a cluster together (their ranks 0 and 1, the first leads), each with its own half of the operands and of the result.

// ---- tensor memory ---------------------------------------------------------------------

// One warp (of each CTA) takes `columns` (a power of two from 32 to 512) of all 128 lanes and later gives them back. The address lands in
// shared memory.
template <bool PAIR>
__device__ __forceinline__ void tmem_alloc(uint32_t *address, uint32_t columns) {
    if constexpr (PAIR) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(address)), "r"(columns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(address)), "r"(columns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
}
template <bool PAIR>
__device__ __forceinline__ void tmem_free(uint32_t address, uint32_t columns) {
    if constexpr (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(address), "r"(columns) : "memory");
    else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(address), "r"(columns) : "memory");
}

// 16 or 32 columns of this warp's 32 lanes: thread i gets lane i's. The words are there after tmem_wait_loads, which names them so that
// nothing uses them before.
__device__ __forceinline__ void tmem_load(uint32_t address, uint32_t (&v)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]),
                   "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
                 : "r"(address)
                 : "memory");
}
__device__ __forceinline__ void tmem_wait_loads(uint32_t (&v)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), "+r"(v[8]), "+r"(v[9]), "+r"(v[10]),
                   "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15])
                 :
                 : "memory");
}
__device__ __forceinline__ void tmem_load(uint32_t address, uint32_t (&v)[32]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
                 "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]),
                   "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]),
                   "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
                 : "r"(address)
                 : "memory");
}
__device__ __forceinline__ void tmem_wait_loads(uint32_t (&v)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), "+r"(v[8]), "+r"(v[9]), "+r"(v[10]),
                   "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15]), "+r"(v[16]), "+r"(v[17]), "+r"(v[18]), "+r"(v[19]), "+r"(v[20]),
                   "+r"(v[21]), "+r"(v[22]), "+r"(v[23]), "+r"(v[24]), "+r"(v[25]), "+r"(v[26]), "+r"(v[27]), "+r"(v[28]), "+r"(v[29]), "+r"(v[30]), "+r"(v[31])
                 :
                 : "memory");
}

// 32 columns of 16 of this warp's lanes (the address is that of the first, the warp's own or 16 further) as matrix fragments of 8 x 8: thread i gets
// of lanes i / 4 and i / 4 + 8 the columns 8 j + 2 (i % 4) and the next one as v[4 j] .. v[4 j + 1] and v[4 j + 2] .. v[4 j + 3].
__device__ __forceinline__ void tmem_load_fragments(uint32_t address, uint32_t (&v)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]),
                   "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
                 : "r"(address)
                 : "memory");
}

// Orders tensor-memory accesses with the barrier operations of other threads.
__device__ __forceinline__ void tmem_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// ---- one thread of a warp --------------------------------------------------------------

// True for one thread of a converged warp, always the same. Matrix instructions and copies take their addresses from registers that a warp shares: in a
// branch on the lane's number the compiler makes them so one by one (600 cycles for the instructions of a block), in this one they are.
__device__ __forceinline__ bool elected() {
    uint32_t yes;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(yes));
    return yes != 0;
}

// ---- operands --------------------------------------------------------------------------

// A tile of rows of 128 bytes, one after another from a 1024-byte boundary on, whose 16-byte pieces are turned by row % 8 (the 128-byte
// swizzle): start address and distance of 8 rows in units of 16 bytes, version 1, swizzle code 2. A step of 32 bytes along the rows adds 2.
__device__ __forceinline__ uint64_t tile_descriptor(uint32_t smem_address) {
    return (uint64_t)((smem_address >> 4) & 0x3fff) | 1ull << 16 | (uint64_t)(1024 >> 4) << 32 | 1ull << 46 | 2ull << 61;
}

// e4m3 times e4m3, sums in 32 bits, both operands by rows along the summed axis.
__host__ __device__ constexpr uint32_t product_descriptor(int m, int n) { return 1u << 4 | (uint32_t)(n >> 3) << 17 | (uint32_t)(m >> 4) << 24; }

// d (+)= a b^T over 32 columns of the operands. One thread issues it, of a pair the leader's; the addresses are the same in both CTAs.
template <bool PAIR>
__device__ __forceinline__ void mma_e4m3(uint32_t d, uint64_t a, uint64_t b, uint32_t shape, bool add) {
    if constexpr (PAIR)
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.u32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
            "l"(a), "l"(b), "r"(shape), "r"((uint32_t)add)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.u32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
            "l"(a), "l"(b), "r"(shape), "r"((uint32_t)add)
            : "memory");
}

// What 16-bit and integer products multiply.
enum class Sum { F16, BF16, S8 };

// The same where the tile's rows run across the summed axis: blocks of 64 elements of 16 bits, each 64 rows of 128 bytes, 8192 bytes apart. A step of
// 16 along the summed axis is 16 rows and adds 128.
__device__ __forceinline__ uint64_t turned_descriptor(uint32_t smem_address) {
    return (uint64_t)((smem_address >> 4) & 0x3fff) | (uint64_t)(8192 >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | 1ull << 46 | 2ull << 61;
}
template <Sum SUM>
__host__ __device__ constexpr uint32_t sum_descriptor(bool a_turned, bool b_turned, int m) {
    return (SUM == Sum::S8 ? 2u << 4 | 1u << 7 | 1u << 10 : SUM == Sum::BF16 ? 1u << 4 | 1u << 7 | 1u << 10 : 1u << 4) | (a_turned ? 1u << 15 : 0u) | (b_turned ? 1u << 16 : 0u) |
           (uint32_t)(m >> 4) << 24;
}

// d (+)= a b^T over 32 bytes of the operands' rows (16 rows of turned ones), by a pair of CTAs; its leader's thread issues it. `shape`: the
// descriptor above with n >> 3 at bit 17.
template <Sum SUM>
__device__ __forceinline__ void mma_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t shape, bool add) {
    if constexpr (SUM == Sum::S8)
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.u32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
            "l"(a), "l"(b), "r"(shape), "r"((uint32_t)add)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.u32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
            "l"(a), "l"(b), "r"(shape), "r"((uint32_t)add)
            : "memory");
}

// The barrier (at this place in both CTAs of a pair) gets an arrival when all matrix instructions that this thread has issued so far are done.
template <bool PAIR>
__device__ __forceinline__ void mma_commit(uint64_t *bar) {
    if constexpr (PAIR)
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)), "h"((uint16_t)3) : "memory");
    else asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// The same for pairs in clusters of several: `ctas` has a bit for each CTA of the pair.
__device__ __forceinline__ void mma_commit_pair(uint64_t *bar, uint32_t ctas) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)), "h"((uint16_t)ctas) : "memory");
}

// ---- loads and stores of tiles -------------------------------------------------------------------

__device__ __forceinline__ void ask_for_map(const CUtensorMap *matrix) { asm volatile("prefetch.tensormap [%0];" ::"l"(matrix) : "memory"); }
// The place of this CTA's barrier in the cluster's CTA `rank`.
__device__ __forceinline__ uint32_t remote_barrier(const uint64_t *bar, int rank) {
    uint32_t at;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(bar)), "r"(rank));
    return at;
}
// A tile of rows of 128 bytes from the place (x, y) of matrix z, where nothing is below zero; what lies beyond the matrix comes as zeros. It lands in this CTA; the
// barrier that counts its bytes is one of the pair's, in either CTA.
__device__ __forceinline__ void load_tile(void *smem, const CUtensorMap *matrix, int x, int y, int z, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem_u32(smem)), "l"(matrix),
                 "r"(x), "r"(y), "r"(z), "r"(bar)
                 : "memory");
}

// The same of a matrix of four extents, from its first column on.
__device__ __forceinline__ void load_tile4(void *smem, const CUtensorMap *matrix, int y, int z, int group, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.4d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(smem_u32(smem)), "l"(matrix),
                 "r"(0), "r"(y), "r"(z), "r"(group), "r"(bar)
                 : "memory");
}
// The same of a matrix of five extents, of which the second and third begin at zero.
__device__ __forceinline__ void load_tile5(void *smem, const CUtensorMap *matrix, int x, int z, int group, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.5d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %3, %4, %5}], [%6];" ::"r"(smem_u32(smem)),
                 "l"(matrix), "r"(x), "r"(0), "r"(z), "r"(group), "r"(bar)
                 : "memory");
}

// Four matrices of 8 x 8 words of 16 bits from the warp's registers (thread i has two neighbours of row i / 4) to shared memory, row r of matrix m to
// the 16 bytes at the address that thread 8 m + r gives; TURNED: their columns.
template <bool TURNED>
__device__ __forceinline__ void store_matrices(void *row, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    if constexpr (TURNED) asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(smem_u32(row)), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
    else asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(smem_u32(row)), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

// A tile of rows of 128 bytes from shared memory, laid out as above, to the place (x, y) of a matrix; what lies beyond the matrix is left out. The
// thread that starts such stores also closes them into groups and waits until all but its last N groups have been read (or written).
__device__ __forceinline__ void store_tile(const CUtensorMap *matrix, const void *smem, int x, int y) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%2, %3}], [%1];" ::"l"(matrix), "r"(smem_u32(smem)), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ void store_tile3(const CUtensorMap *matrix, const void *smem, int x, int y, int z) {
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(matrix), "r"(smem_u32(smem)), "r"(x), "r"(y), "r"(z) : "memory");
}
__device__ __forceinline__ void close_stores() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void stores_read_but() { asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void stores_done() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

// ---- barriers within a cluster -----------------------------------------------------------

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
    uint32_t n;
    asm volatile("mov.u32 %0, %cluster_nctaid.x;" : "=r"(n));
    return n;
}
// What lies at this place in the shared memory of the cluster's CTA `rank`.
__device__ __forceinline__ float load_remote(const float *p, int rank) {
    float v;
    asm volatile(
        "{\n\t.reg .b32 remote;\n\t"
        "mapa.shared::cluster.u32 remote, %1, %2;\n\t"
        "ld.shared::cluster.f32 %0, [remote];\n\t}"
        : "=f"(v)
        : "r"(smem_u32(p)), "r"(rank)
        : "memory");
    return v;
}
// An arrival at the barrier that lies at this place in the first CTA of the cluster. It orders what the tensor cores and the copy engine do, on
// both sides of which their own fences and barriers stand; ordinary accesses would need a release and an acquire of the cluster's scope, which
// wait for all memory of the thread: with those an 8192^3 product took 1102 us.
__device__ __forceinline__ void mbar_arrive_leader(uint64_t *bar) {
    asm volatile(
        "{\n\t.reg .b32 remote;\n\t"
        "mapa.shared::cluster.u32 remote, %0, 0;\n\t"
        "mbarrier.arrive.shared::cluster.b64 _, [remote];\n\t}" ::"r"(smem_u32(bar))
        : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint64_t *bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// The same at the cluster's CTA `rank`. RELEASE: for ordinary stores to shared memory that matrix instructions of that CTA read (behind
// fence_async_shared; its other side is mbar_acquire_cluster).
template <bool RELEASE>
__device__ __forceinline__ void mbar_arrive_at(uint64_t *bar, int rank) {
    if constexpr (RELEASE)
        asm volatile(
            "{\n\t.reg .b32 remote;\n\t"
            "mapa.shared::cluster.u32 remote, %0, %1;\n\t"
            "mbarrier.arrive.release.cluster.shared::cluster.b64 _, [remote];\n\t}" ::"r"(smem_u32(bar)),
            "r"(rank)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .b32 remote;\n\t"
            "mapa.shared::cluster.u32 remote, %0, %1;\n\t"
            "mbarrier.arrive.shared::cluster.b64 _, [remote];\n\t}" ::"r"(smem_u32(bar)),
            "r"(rank)
            : "memory");
}
// Whether a phase of this CTA's barrier is over; if so, what arrivals with RELEASE stand for is there.
__device__ __forceinline__ bool mbar_acquire_cluster(uint64_t *bar, uint32_t parity) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return done != 0;
}
// All threads of all CTAs of the cluster meet.
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// ---- sums ------------------------------------------------------------------------------

// a += v * (s * c) for two neighbours at once: half the instructions where every element has factors of its own.
__device__ __forceinline__ void add_scaled(float &a0, float &a1, uint32_t v0, uint32_t v1, float s, float c0, float c1) {
    asm("{\n\t.reg .b64 a, v, s, c;\n\t"
        "mov.b64 a, {%0, %1};\n\t"
        "mov.b64 v, {%2, %3};\n\t"
        "mov.b64 s, {%4, %4};\n\t"
        "mov.b64 c, {%5, %6};\n\t"
        "mul.rn.f32x2 c, s, c;\n\t"
        "fma.rn.f32x2 a, v, c, a;\n\t"
        "mov.b64 {%0, %1}, a;\n\t}"
        : "+f"(a0), "+f"(a1)
        : "r"(v0), "r"(v1), "f"(s), "f"(c0), "f"(c1));
}

// ---- registers -------------------------------------------------------------------------

// Four neighbouring warps together change how many registers each of their threads has. What the warps of a block end up with must not be
// more than the block was launched with.
template <int N>
__device__ __forceinline__ void fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }

}  // namespace nb200
