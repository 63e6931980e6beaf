/*
 * nacho_b200 — C ABI of the B200 (sm_100a) sparse-kernel library.
 *
 * Drop-in boundary for the GPU hot path of the nacho sparse tensor algebra compiler: each
 * entry point below stands where one of nacho's emitted host drivers
 * `<kernel>::<kernel>_gpu_i32_f32(a, b[, c], num_blocks, threads_per_block)` stands today
 * (emitter: src/backend/stitch_and_generate_gpu.cpp:142-185, signature
 * src/backend/stitch_and_generate.cpp:278-290), and is what the emitted nanobind wrappers
 * `gpu_<kernel>_f32` (src/backend/generate_bindings.cpp:288-331) would call instead.
 *
 * Conventions shared by every entry point
 *   - All indices are int32 and all values float32 (src/backend/stitch_and_generate.cpp:235-236).
 *   - Every array pointer is a DEVICE pointer on the current CUDA device, 4-byte aligned,
 *     contiguous. Operands are borrowed and never written (runtime/nacho_nb.h:73-78).
 *   - Operands must hold sorted, duplicate-free columns / coordinates, as nacho requires.
 *   - `stream` is a cudaStream_t passed as void* (NULL = the legacy default stream, which is
 *     what nacho's drivers use, src/backend/stitch_and_generate_gpu.cpp:163-167).
 *   - Every call returns an nb200_status; 0 is success. Nothing throws and nothing aborts.
 *   - The calls block the host until the result lengths are known (a kernel writes them to pinned
 *     host memory), like nacho's drivers do; on return kernels may still be running, and the result is
 *     complete in stream order.
 *   - num_blocks / threads_per_block are accepted for signature compatibility
 *     (src/backend/generate_bindings.cpp:317-327); the kernels size their own grids, so the
 *     two values are ignored.
 *
 * Two flavours per operator
 *   nb200_<op>_f32       allocates each result array separately with cudaMallocAsync on
 *                        `stream`, so that each can be released independently with
 *                        nb200_free_async (= cudaFreeAsync), the ownership nacho's adopt_gpu
 *                        capsules expect (runtime/nacho_nb.h:50-58,
 *                        runtime/cuda_utils/cuda_utils.cu:7-11). A zero-length array is
 *                        returned as NULL (runtime/nacho_nb.h:37-45).
 *   nb200_<op>_f32_into  writes into caller-owned arrays of a stated capacity (for callers
 *                        whose framework owns device memory, e.g. torch tensors) and reports
 *                        the used lengths. If a capacity is too small the call returns
 *                        NB200_E_CAPACITY with the needed lengths filled in and the value /
 *                        index arrays untouched.
 */
#ifndef NACHO_B200_H
#define NACHO_B200_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define NB200_VERSION 100

typedef enum nb200_status {
    NB200_OK = 0,
    NB200_E_BADARG = 1,     /* null pointer, negative size, mismatched shapes */
    NB200_E_CUDA = 2,       /* a CUDA runtime call failed; see nb200_last_cuda_error() */
    NB200_E_OVERFLOW = 3,   /* a result length or work count does not fit int32 */
    NB200_E_CAPACITY = 4,   /* caller-provided result arrays are too small */
    NB200_E_TIMEOUT = 5,    /* a bounded device-side wait gave up (no hang, context intact) */
    NB200_E_NOMEM = 6,      /* device allocation failed */
    NB200_E_UNSUPPORTED = 7 /* size beyond a documented limit of the entry point */
} nb200_status;

/* CSR matrix: the field set of nacho's emitted CSR structs
 * {dim_i_size, dim_j_size, dim_j_offsets, dim_j_length, dim_j_indices, values, nnz}
 * (src/backend/tensor.cpp:13-61, include/backend/tensor.h:78-81). */
typedef struct nb200_csr {
    int32_t rows;     /* dim_i_size */
    int32_t cols;     /* dim_j_size */
    int32_t nnz;      /* dim_j_length */
    int32_t *row_ptr; /* dim_j_offsets, rows + 1 entries */
    int32_t *col;     /* dim_j_indices, nnz entries */
    float *val;       /* values, nnz entries */
} nb200_csr;

/* COO3 tensor: three parallel coordinate arrays + values
 * (src/backend/tensor.cpp:13-61 for the Compressed_non_unique, Singleton, Singleton levels of
 * compiler.cpp:60-64). */
typedef struct nb200_coo3 {
    int32_t dims[3];
    int32_t nnz;
    int32_t *i, *j, *k; /* dim_{i,j,k}_indices, nnz entries each */
    float *val;
} nb200_coo3;

/* CSF3 tensor: three compressed levels (compiler.cpp:44-48); the outermost level has no
 * offsets array (src/backend/tensor.cpp:35-39). */
typedef struct nb200_csf3 {
    int32_t dims[3];
    int32_t n_i, n_j, n_k; /* dim_{i,j,k}_length */
    int32_t *i_idx;        /* dim_i_indices, n_i */
    int32_t *j_ptr;        /* dim_j_offsets, n_i + 1 */
    int32_t *j_idx;        /* dim_j_indices, n_j */
    int32_t *k_ptr;        /* dim_k_offsets, n_j + 1 */
    int32_t *k_idx;        /* dim_k_indices, n_k */
    float *val;            /* values, n_k */
} nb200_csf3;

/* 2-D coordinate list: the field set of nacho's emitted COO structs (Compressed_non_unique +
 * Singleton_unique levels, compiler.cpp:50-53): parallel row / column arrays sorted by (i, j). */
typedef struct nb200_coo {
    int32_t rows, cols;
    int32_t nnz;
    int32_t *i, *j; /* dim_{i,j}_indices, nnz entries each */
    float *val;
} nb200_coo;

/* DCSR matrix: both levels compressed (compiler.cpp:38-42): only the rows that hold entries are
 * stored, with their row numbers. */
typedef struct nb200_dcsr {
    int32_t rows, cols;
    int32_t n_i, nnz; /* dim_i_length, dim_j_length */
    int32_t *i_idx;   /* dim_i_indices, n_i */
    int32_t *j_ptr;   /* dim_j_offsets, n_i + 1 */
    int32_t *j_idx;   /* dim_j_indices, nnz */
    float *val;       /* values, nnz */
} nb200_dcsr;

/* ---- library -------------------------------------------------------------------------- */

int nb200_version(void);
const char *nb200_strerror(int status);
/* Text of the last CUDA error seen by the calling thread's most recent failing call; after
 * NB200_E_TIMEOUT, which bounded device-side wait gave up and at which tile. */
const char *nb200_last_cuda_error(void);
/* Release a result array of an allocating entry point: cudaFreeAsync(p, stream); NULL is
 * ignored. Replaces cudaFreeWrapper (runtime/cuda_utils/cuda_utils.cu:7-11). */
int nb200_free_async(void *p, void *stream);
/* Release the per-device scratch pools the library keeps between calls. */
int nb200_release_workspaces(void);
/* Number of kernels this library has launched in this process so far. */
uint64_t nb200_launch_count(void);

/* Per-kernel device timing. While enabled, every kernel launch of the library is bracketed
 * by CUDA events on its stream. nb200_profile_read synchronises those events and reports,
 * for the kernel called `name`, the launches and their summed duration since the last
 * nb200_profile_reset; nb200_profile_names writes a comma-separated list of kernel names.
 * `on`: 0 ends it. 2 times the launches that calls make anyway. 1 (or any other value) times merges
 * that find their tile cuts themselves (calls that wait for their result, of up to about 65 million
 * entries) as two launches, the search for the cuts and the merge proper: more than such a call takes. */
int nb200_profile_enable(int on);
int nb200_profile_reset(void);
int nb200_profile_read(const char *name, int64_t *launches, double *total_ms);
int nb200_profile_names(char *buf, size_t buf_len);

/* ---- CSR element-wise ------------------------------------------------------------------- */

/* Z = A + B, sorted union per row; a position present in both holds a + b, explicit zeros
 * are kept. Replaces csr_add::csr_add_gpu_i32_f32 (kernel declared at compiler.cpp:112;
 * partition src/backend/partition.cpp:813-993, count/fill src/backend/compute.cpp:152-411).
 * Result: row_ptr rows+1, col/val nnz. Capacity that always suffices: nnz(A) + nnz(B). */
int nb200_csr_add_f32(const nb200_csr *a, const nb200_csr *b, nb200_csr *z,
                      int32_t num_blocks, int32_t threads_per_block, void *stream);
int nb200_csr_add_f32_into(const nb200_csr *a, const nb200_csr *b, nb200_csr *z,
                           int64_t capacity, void *stream);

/* Z = A + B for callers that must not trigger any device or pinned-host allocation while they
 * run -- code inside a framework's memory-pool callback or an out-of-memory handler, plug-ins
 * living under a fixed memory budget that the host application has already handed out, and
 * latency-critical loops where an allocator call could take a lock or synchronise the device.
 * Has no counterpart in the reference, whose drivers allocate on every call.
 *
 * Same result as nb200_csr_add_f32_into, but the scratch memory of the kernels (tile cuts and
 * the cross-tile counters) is a fixed 1 MiB array inside the library's device image instead of
 * a pool that grows on demand. The call makes no cudaMalloc / cudaFree / cudaHostAlloc and
 * calls no allocating library routine; the caller provides every operand and result array.
 * Limits and rules:
 *   - nnz(A) + nnz(B) may not exceed 159350784 entries;
 *     larger inputs return NB200_E_UNSUPPORTED and nothing is launched.
 *   - `capacity` (entries in z->col / z->val) must be at least nnz(A) + nnz(B); otherwise
 *     NB200_E_CAPACITY. z->row_ptr holds rows + 1 entries.
 *   - The first call on each device looks up the array's device address and raises the
 *     kernel's shared-memory limit; make that first call before any stream capture begins.
 *   - All calls on a device share the one array: it is re-zeroed at the start of each call,
 *     and two calls that overlap on the GPU (different streams, different host threads)
 *     would corrupt each other. Serialise them.
 *   - Launches made here are not counted by nb200_launch_count nor timed by the profile. */
int nb200_csr_add_f32_noalloc(const nb200_csr *a, const nb200_csr *b, nb200_csr *z,
                              int64_t capacity, void *stream);

/* Asynchronous forms of add and multiply: like the _into forms with a capacity of at least the
 * worst case (nnz(A) + nnz(B) for add, min(nnz(A), nnz(B)) for multiply; less returns
 * NB200_E_CAPACITY), but the call returns as soon as its kernels are queued. The result length and
 * the device-side status arrive, in stream order, in three int64 DEVICE words:
 * device_result[0] = nnz(Z), device_result[1] = an nb200_status (NB200_OK, NB200_E_TIMEOUT or
 * NB200_E_OVERFLOW), device_result[2] = the row count (so that the three words are a row block's
 * whole contribution to a stitch and can be all-gathered as they are). z->nnz is left 0. For callers that consume the length on the device -- a
 * multi-GPU stitch that all-gathers the block lengths, a pipeline that launches the next operator
 * from the same stream -- and must not stall the host once per call. The reference has no
 * counterpart: its drivers read every length back (src/backend/stitch_and_generate_gpu.cpp:660-671). */
int nb200_csr_add_f32_async(const nb200_csr *a, const nb200_csr *b, nb200_csr *z, int64_t capacity,
                            int64_t *device_result, void *stream);
int nb200_csr_mul_f32_async(const nb200_csr *a, const nb200_csr *b, nb200_csr *z, int64_t capacity,
                            int64_t *device_result, void *stream);

/* Z = A .* B, sorted intersection per row, value a * b. Replaces
 * csr_mul::csr_mul_gpu_i32_f32 (compiler.cpp:116; src/backend/compute.cpp:434-440). An empty
 * result has an all-zero row_ptr (src/backend/stitch_and_generate.cpp:168-220).
 * Capacity that always suffices: min(nnz(A), nnz(B)). */
int nb200_csr_mul_f32(const nb200_csr *a, const nb200_csr *b, nb200_csr *z,
                      int32_t num_blocks, int32_t threads_per_block, void *stream);
int nb200_csr_mul_f32_into(const nb200_csr *a, const nb200_csr *b, nb200_csr *z,
                           int64_t capacity, void *stream);

/* Host-buffer forms of add and multiply: every pointer in a, b and z is a HOST pointer (pinned
 * memory gives full PCIe speed; pageable memory works but copies synchronously). The matrices
 * are streamed through the current device in row blocks of about 12 M operand entries on three
 * internal streams, so that the upload of one block, the merge of the previous one and the
 * download of the one before overlap. z->row_ptr (rows + 1), z->col and z->val (`capacity`
 * entries each) are the caller's; on return z->nnz is the result length and the arrays are
 * complete (the call synchronises its own streams). NB200_E_CAPACITY if the result does not fit.
 * Calls on one device take turns (the library holds a per-device lock for the whole call); on any
 * error return the call has first waited for every copy it had queued, so the host buffers are no
 * longer read or written once it is back.
 * The reference has no counterpart: its operators take device tensors only. */
int nb200_csr_add_f32_host(const nb200_csr *a, const nb200_csr *b, nb200_csr *z, int64_t capacity);
int nb200_csr_mul_f32_host(const nb200_csr *a, const nb200_csr *b, nb200_csr *z, int64_t capacity);

/* Z = (A + B) + C, left-to-right association, in one call. Replaces
 * csr_add_3::csr_add_3_gpu_i32_f32 (compiler.cpp:114; src/backend/compute.cpp:426-432).
 * Capacity that always suffices: nnz(A) + nnz(B) + nnz(C). */
int nb200_csr_add_3_f32(const nb200_csr *a, const nb200_csr *b, const nb200_csr *c,
                        nb200_csr *z, int32_t num_blocks, int32_t threads_per_block,
                        void *stream);
int nb200_csr_add_3_f32_into(const nb200_csr *a, const nb200_csr *b, const nb200_csr *c,
                             nb200_csr *z, int64_t capacity, void *stream);
/* The sum A + B is formed on the way: 8 bytes per entry of A and of B. The forms above keep it in the library's scratch
 * pool, where the room stays taken until nb200_release_workspaces (three times 67 million entries: 1.3 GB). _lent is
 * _into with scratch of the caller's: at least nb200_csr_add_3_f32_scratch(a, b, c) bytes (0 for operands that the call
 * would refuse) on a 256-byte boundary, in use until the work queued on `stream` is done. */
int64_t nb200_csr_add_3_f32_scratch(const nb200_csr *a, const nb200_csr *b, const nb200_csr *c);
int nb200_csr_add_3_f32_lent(const nb200_csr *a, const nb200_csr *b, const nb200_csr *c, nb200_csr *z,
                             int64_t capacity, void *scratch, int64_t scratch_bytes, void *stream);

/* ---- SpGEMM ----------------------------------------------------------------------------- */

/* C = A * B by expand-sort-compress; columns sorted per row, explicit zeros kept, rows
 * without products empty. Replaces spgemm::spgemm_gpu_i32_f32 (compiler.cpp:145-148;
 * expand src/backend/compute.cpp:526-611, sort/compress
 * src/backend/stitch_and_generate_gpu.cpp:14-139,257-363). Unlike the reference, product
 * counts are 64-bit (a product count above 2^31 is fine as long as nnz(C) fits int32) and
 * rows with at most 256 products sum equal-column products in a fixed order (ascending j);
 * longer rows accumulate with float32 atomics (as the reference does for every row). No
 * product is written to device memory. Scratch: 24 bytes per row, 8 per entry of A, for matrices wider
 * than 262144 columns a pointer table of one int32 per row of B and 262144 columns of width; and, where
 * there is room, a bitmap of the result's columns for every row of more than 256 products (8 GiB at
 * most), 40 bytes for each of them where there are 8192 and more, and, for more than 32 M products that
 * read the entries of B 16 to 32 times, 16 bytes and more per entry of B for other forms of it. */
int nb200_spgemm_f32(const nb200_csr *a, const nb200_csr *b, nb200_csr *c, int32_t num_blocks,
                     int32_t threads_per_block, void *stream);
/* Two-step form for caller-owned memory: _symbolic fills c->row_ptr (rows + 1, caller-owned)
 * and c->nnz; the caller then provides col/val of c->nnz entries to _numeric.
 * `products` (may be NULL) receives the number of scalar products. A _numeric call that follows
 * a _symbolic call on the same arrays, device and stream, with no other call of this library on
 * that stream in between, reuses what _symbolic left in the scratch pool (row bins and the column
 * bitmaps of the long rows, up to 8 GiB) instead of computing it again; any other order of calls
 * is equally valid and recomputes. That reuse assumes the patterns of A and B (row offsets and
 * columns) are unchanged between the two calls -- their values may differ -- and that c->row_ptr is
 * the array _symbolic filled; a caller that rewrites a pattern in place must call _symbolic again. */
int nb200_spgemm_f32_symbolic(const nb200_csr *a, const nb200_csr *b, nb200_csr *c,
                              int64_t *products, void *stream);
int nb200_spgemm_f32_numeric(const nb200_csr *a, const nb200_csr *b, nb200_csr *c,
                             void *stream);

/* One-call forms for caller-owned memory.
 *
 * _with asks for the result's arrays when it knows how many entries they need: `take(ctx, entries, &col, &val)` is called
 * on the calling thread, hands out two arrays of that many entries that may be used on `stream`, and returns NB200_OK, or
 * a status with which the call then ends. It must not throw, nor call this library on `stream`. c->row_ptr is the
 * caller's; c->col / c->val are set to the arrays in use, of which the first c->nnz entries are. An empty result
 * takes none. A request refused with NB200_E_NOMEM is made once more if the call holds other forms of B, which it gives back
 * first. Matrices of short rows (at most 8 entries in a row of A and 32 products) are multiplied in one pass into an
 * entry per product: if `take` refuses that with NB200_E_NOMEM they are counted first, like any others, and if fewer
 * than half of the entries are in use, `take` is called again for nnz(C) entries, to which the result moves (the arrays
 * of the first call are read until the work queued on `stream` is done; a refusal leaves the result where it is).
 *
 * _into takes any capacity that holds the result (less returns NB200_E_CAPACITY with c->nnz filled in). _bound sets
 * *capacity to the number of entries with which _into runs in one pass, or to 0 where it has to count first. */
typedef int (*nb200_take_fn)(void *ctx, int64_t entries, int32_t **col, float **val);
int nb200_spgemm_f32_with(const nb200_csr *a, const nb200_csr *b, nb200_csr *c, nb200_take_fn take, void *ctx, void *stream);
int nb200_spgemm_f32_bound(const nb200_csr *a, const nb200_csr *b, int64_t *capacity, void *stream);
int nb200_spgemm_f32_into(const nb200_csr *a, const nb200_csr *b, nb200_csr *c, int64_t capacity, void *stream);

/* Masked SpGEMM: Z_ik = sum_j a_ij * b_jk * c_ik on the positions the mask C stores and at least
 * one product reaches (explicit zeros kept, columns in C's order). Replaces
 * sssmm::sssmm_gpu_i32_f32 (compiler.cpp:150-153). The mask drives the accumulation: every product
 * looks its column up in C's row and is added -- as (a * b) * c, the reference's expression -- to
 * that position or dropped, so nothing outside the mask is formed; float32 atomics in arrival
 * order, as the reference's compress. z->row_ptr holds rows(A) + 1 entries; `capacity` entries in
 * z->col / z->val, nnz(C) always suffices (less returns NB200_E_CAPACITY with z->nnz filled in).
 * Scratch: 8 bytes per entry of C. */
int nb200_sssmm_f32_into(const nb200_csr *a, const nb200_csr *b, const nb200_csr *c, nb200_csr *z,
                         int64_t capacity, void *stream);

/* ---- 3-mode tensor add ------------------------------------------------------------------ */

/* Z = A + B over lexicographically sorted unique (i, j, k). Replaces
 * coo3d_add::coo3d_add_gpu_i32_f32 (compiler.cpp:138; merged coordinate level
 * src/Compile.cpp:66-154). Capacity that always suffices: nnz(A) + nnz(B). */
int nb200_coo3d_add_f32(const nb200_coo3 *a, const nb200_coo3 *b, nb200_coo3 *z,
                        int32_t num_blocks, int32_t threads_per_block, void *stream);
int nb200_coo3d_add_f32_into(const nb200_coo3 *a, const nb200_coo3 *b, nb200_coo3 *z,
                             int64_t capacity, void *stream);

/* Z = A + B for CSF3 operands. Replaces csf_add::csf_add_gpu_i32_f32 (compiler.cpp:135).
 * Capacities that always suffice (for _into): i_idx n_i(A)+n_i(B); j_ptr that + 1;
 * j_idx n_j(A)+n_j(B); k_ptr that + 1; k_idx / val n_k(A)+n_k(B). The _into form takes the
 * three capacities (entries of i_idx, j_idx, k_idx); j_ptr / k_ptr must hold one entry more
 * than cap_i / cap_j, and cap_k must be at least n_k(A)+n_k(B) (the merge works in place in
 * the result's k_idx / val arrays). Any extents up to 2^31 - 1 per mode work, here and for COO3:
 * coordinates that fit 63 bits together are merged as packed 64-bit keys, wider ones as
 * (i, j) / k word pairs (the reference's three-int32 tuple compare, src/backend/tensor.cpp:447-560). */
int nb200_csf_add_f32(const nb200_csf3 *a, const nb200_csf3 *b, nb200_csf3 *z,
                      int32_t num_blocks, int32_t threads_per_block, void *stream);
int nb200_csf_add_f32_into(const nb200_csf3 *a, const nb200_csf3 *b, nb200_csf3 *z,
                           int64_t cap_i, int64_t cap_j, int64_t cap_k, void *stream);

/* ---- the rest of the element-wise family, and the inner products ------------------------- */

/* The kernels nacho declares beside the six above over 2-D coordinate lists and doubly compressed
 * rows (compiler.cpp:118-126) and the two full reductions (compiler.cpp:141-143), in the
 * caller-owned-memory form only. Results are bit-identical to nacho's CPU kernels: sorted union /
 * intersection, explicit zeros kept.
 *   coo_add / coo_mul    Z = A (+|.*) B over sorted unique (i, j) lists; `capacity` entries in
 *                        z->i / z->j / z->val (always enough: nnz(A)+nnz(B), min(nnz(A), nnz(B))).
 *   coo_csr_add          Z = A + B with A in CSR and B a coordinate list; Z in CSR.
 *   dcsr_add / dcsr_mul  DCSR operands and result. `cap_i` entries in z->i_idx (z->j_ptr one more)
 *                        must cover the worst case, min(n_i(A)+n_i(B), rows) for the sum and
 *                        min(n_i(A), n_i(B)) for the product; `capacity` as for CSR. The product
 *                        keeps every row that BOTH operands store, with an empty column range where
 *                        their columns do not meet, as nacho's level-by-level intersection does.
 * These run the CSR merge kernels on the operands' own column / value arrays. Scratch: a few int32 per
 * matrix row for the coordinate lists (their row offsets are rebuilt), per STORED row for DCSR. */
int nb200_coo_add_f32_into(const nb200_coo *a, const nb200_coo *b, nb200_coo *z, int64_t capacity, void *stream);
int nb200_coo_mul_f32_into(const nb200_coo *a, const nb200_coo *b, nb200_coo *z, int64_t capacity, void *stream);
int nb200_coo_csr_add_f32_into(const nb200_csr *a, const nb200_coo *b, nb200_csr *z, int64_t capacity, void *stream);
int nb200_dcsr_add_f32_into(const nb200_dcsr *a, const nb200_dcsr *b, nb200_dcsr *z, int64_t cap_i, int64_t capacity,
                            void *stream);
int nb200_dcsr_mul_f32_into(const nb200_dcsr *a, const nb200_dcsr *b, nb200_dcsr *z, int64_t cap_i, int64_t capacity,
                            void *stream);

/* z[0] = sum over the coordinates both tensors hold of a * b, one float32 in DEVICE memory (nacho
 * returns a one-element tensor). Replaces inner_prod::inner_prod_gpu_i32_f32 (CSF3 operands) and
 * inner_prod_coo::inner_prod_coo_gpu_i32_f32 (COO3 operands); append-reduction
 * src/backend/compute.cpp:498-525. Each product is a float32 multiply as in nacho; the products
 * are summed in double and rounded once, where nacho adds float32 atomically in arrival order, so
 * the two agree to float32 rounding of the sum, not bit for bit. Extents must pack into 63 bits. */
int nb200_inner_prod_f32(const nb200_csf3 *a, const nb200_csf3 *b, float *z, void *stream);
int nb200_inner_prod_coo_f32(const nb200_coo3 *a, const nb200_coo3 *b, float *z, void *stream);

/* ---- around a router ---------------------------------------------------------------------- */

/* A router's decision is a CSR matrix R of tokens x experts whose values are the gate weights. The entry points
 * below bring dense rows (one per token) into the order of the experts, multiply every expert's rows with its
 * weights in 8-bit floating point, and bring them back. They have no counterpart in the reference.
 *   - Rows of R may be empty or hold any number of entries, in any order of experts (duplicates count twice).
 *     An entry whose column lies outside [0, cols) is dropped: it has no slot and takes part in nothing.
 *   - None of the calls waits for the device: all result lengths are known before. They can be captured in a CUDA
 *     graph once a call of their kind has been made on the stream (a product's first one there allocates 512 bytes of
 *     pinned memory for its report), and use no device memory but what the caller gives them, so graphs may be
 *     replayed on any stream, beside one another and after calls of any size.
 *   - Sums are 32-bit, in a fixed order: the same call gives the same bits. */

/* Dense rows in device memory: element (r, c) lies at data[r * stride + c]. */
typedef enum nb200_type { NB200_F32 = 0, NB200_F16 = 1, NB200_BF16 = 2 } nb200_type;
typedef struct nb200_dense {
    int64_t rows, cols, stride;
    int32_t type; /* nb200_type; data is aligned to the type's size */
    void *data;
} nb200_dense;

/* The order of the experts: entries of R sorted by expert, entries of one expert in storage order. Kept entries take
 * the slots 0 .. offsets[experts] - 1; the slots behind those belong to nobody. */
typedef struct nb200_expert_order {
    int32_t tokens, experts, entries;
    int32_t *row_ptr; /* R's own, tokens + 1 */
    int32_t *offsets; /* experts + 1: where each expert's slots begin */
    int32_t *rows;    /* entries: the token of every slot, -1 for a slot of nobody (and counts while the order is made) */
    int32_t *slots;   /* entries: the slot of every entry of R, -1 for a dropped one */
} nb200_expert_order;

#define NB200_MAX_EXPERTS 4096

/* Matrices in 8-bit floating point (e4m3) with a 32-bit scale for every 128 columns of a row (tiled = 0; one group) or for
 * every 128 x 128 (tiled = 1). With m the largest magnitude of a block, at least 2^-110: scale = m / 448, code =
 * e4m3(x * (448 / m)), both quotients rounded to 32 bits; a block that holds a NaN or an infinity stands for NaNs.
 * values: [group][column block][row, to a multiple of 8][128 codes], column blocks filled up with zeros. The 16-byte piece p of
 *         a row's 128 codes lies at place p ^ (row % 8). 16-byte aligned.
 * scales: tiled = 0: [column block][row, to a multiple of 8]; tiled = 1: [group][row block][column block]. 16-byte aligned. */
typedef struct nb200_fp8 {
    int32_t groups, rows, cols, tiled;
    uint8_t *values;
    float *scales;
} nb200_fp8;

/* Lengths of the two arrays for the extents in `m`, -1 if those are not possible. */
int64_t nb200_fp8_value_count(const nb200_fp8 *m);
int64_t nb200_fp8_scale_count(const nb200_fp8 *m);

/* order of R, and (where x is not NULL) xs[slot] = x[token], zeros for slots of nobody. order->row_ptr is set to R's. The
 * other three arrays are the caller's. The form with fp8 rows quantises on the way. At most NB200_MAX_EXPERTS columns, and
 * 2^31 - 1025 tokens and entries. */
int nb200_expert_sort(const nb200_csr *r, const nb200_dense *x, nb200_expert_order *order, nb200_dense *xs, void *stream);
int nb200_expert_sort_fp8(const nb200_csr *r, const nb200_dense *x, nb200_expert_order *order, nb200_fp8 *xs, void *stream);
/* y[t] = sum over the kept entries e of token t of w[e] * z[slot(e)]; w = NULL stands for ones (the gradient of the sort). */
int nb200_expert_unsort(const nb200_expert_order *order, const float *w, const nb200_dense *z, nb200_dense *y, void *stream);
/* Its gradients: dz[slot(e)] = w[e] * dy[t] (zeros for slots of nobody), dw[e] = <dy[t], z[slot(e)]> (0 where dropped). */
int nb200_expert_unsort_grad(const nb200_expert_order *order, const float *w, const nb200_dense *z, const nb200_dense *dy,
                             nb200_dense *dz, float *dw, void *stream);

/* Quantises. The rows of x are those of z, group after group. */
int nb200_fp8_quantise(const nb200_dense *x, nb200_fp8 *z, void *stream);
/* Takes over codes and scales that exist: codes [groups * rows][cols] one after another, scales [rows][column blocks]
 * (tiled = 0) or [groups][row blocks][column blocks] (tiled = 1). */
int nb200_fp8_pack(const uint8_t *codes, const float *scales, nb200_fp8 *z, void *stream);
/* The 32-bit values that a matrix stands for, [groups * rows][cols] one after another. */
int nb200_fp8_unpack(const nb200_fp8 *a, float *z, void *stream);
/* Every group's transpose; tiled = 1 only. */
int nb200_fp8_transpose(const nb200_fp8 *a, nb200_fp8 *z, void *stream);

/* The products' waits for copies and matrix instructions are bounded (two seconds, where microseconds are usual). One that gave up is reported by
 * the next product called on the stream, which returns NB200_E_TIMEOUT and does nothing. One in a graph reports to the stream that it was captured
 * on, wherever the graph is replayed.
 *
 * y[i] = a[i] * w[g]^T: rows a (tiled = 0), weights w (tiled = 1) with as many columns, y of a->rows x w->rows in any type. With
 * `offsets` (w->groups + 1 of them, rising, in device memory) rows offsets[g] .. offsets[g + 1] - 1 take group g and rows
 * in front of the first or behind the last are zeros, all rows where there are no groups; without it there is one group. Products of a block of 128 columns are summed on
 * the tensor cores and the blocks, times their two scales, in 32 bits. */
int nb200_fp8_product(const nb200_fp8 *a, const nb200_fp8 *w, const int32_t *offsets, nb200_dense *y, void *stream);
/* The gradient for the weights: z[g] = sum over the rows i of group g of dy[i]^T x[i], z = [groups][dy->cols][x->cols] 32-bit. Both
 * operands are quantised along the rows, a scale for every column and 128 rows counted from the group's first. With
 * `dy_rows` (or NULL), the rows of dy that belong to a group are quantised into it as nb200_fp8_quantise would, in the same pass: the left operand of
 * the gradient for x, dy * w, whose right one is nb200_fp8_transpose of w. Rows of no group are left as they are. */
int nb200_fp8_product_grad_w(const nb200_dense *dy, const nb200_dense *x, int32_t groups, const int32_t *offsets, float *z,
                             nb200_fp8 *dy_rows, void *scratch, int64_t scratch_bytes, void *stream);
/* Bytes of scratch, 256-byte aligned device memory, that it needs: the quantised operands; -1 for impossible operands. */
int64_t nb200_fp8_product_grad_w_scratch(const nb200_dense *dy, const nb200_dense *x, int32_t groups);

/* ---- gated layers ------------------------------------------------------------------------- */

/* The gated half of a feed-forward layer, dense or by expert, in 16 bits: with g = x Wg^T and u = x Wu^T, h = act(g) u. w holds `groups` matrices of
 * 2 * hidden x x->cols, one after another (w->rows = groups * 2 * hidden): first the hidden rows of Wg, then those of Wu. All operands of a call are of one type,
 * float16 or bfloat16; sums are 32-bit, in a fixed order, and rounded once. `offsets` as in the products above: groups + 1 of them, rising, rows of no
 * group are zeros; without it there is one group. None of the calls waits for the device, and they can be captured as the products can.
 * act: v s(v) with the logistic function s (silu), or v s(2 sqrt(2 / pi) (v + 0.044715 v^3)), the tanh form of gelu. */
typedef enum nb200_activation { NB200_SILU = 0, NB200_GELU = 1 } nb200_activation;

/* both: NULL, or [g u] rounded to the type (2 * hidden columns, rows one after another), which the backward pass takes. scratch: 256-byte aligned device
 * memory of nb200_gated_product_scratch bytes (rows that the copy engine cannot read are copied there; mostly 0); -1 for impossible operands. */
int nb200_gated_product(const nb200_dense *x, const nb200_dense *w, int32_t groups, const int32_t *offsets, int32_t activation, nb200_dense *h,
                        nb200_dense *both, void *scratch, int64_t scratch_bytes, void *stream);
int64_t nb200_gated_product_scratch(const nb200_dense *x, const nb200_dense *w, int32_t groups);
/* Gradients: with dboth = [dh u act'(g), dh act(g)] rounded to the type, dx = dboth w (zeros for rows of no group) and, for every group, its matrix of
 * dw = dboth^T x over the group's rows (zeros where it has none), dw laid out as w without gaps between groups. */
int nb200_gated_product_grad(const nb200_dense *dh, const nb200_dense *both, const nb200_dense *x, const nb200_dense *w, int32_t groups,
                             const int32_t *offsets, int32_t activation, nb200_dense *dx, nb200_dense *dw, void *scratch, int64_t scratch_bytes,
                             void *stream);
int64_t nb200_gated_product_grad_scratch(const nb200_dense *x, const nb200_dense *w, int32_t groups);

/* ---- products in 8-bit integers ------------------------------------------------------------ */

/* Rows of 8-bit integers with a 32-bit scale each. With m the largest magnitude of a row, at least 2^-110: scale = m / 127, code = x * (127 / m) rounded to
 * the nearest whole number (ties to even), the quotients and the product rounded to 32 bits. A row that holds a NaN or an infinity stands for NaNs.
 * values: [groups * rows][nb200_int8_pitch codes], filled up with zeros, 16-byte aligned. scales: [groups * rows]. */
typedef struct nb200_int8 {
    int32_t groups, rows, cols;
    int8_t *values;
    float *scales;
} nb200_int8;

#define NB200_MAX_INT8_COLUMNS 131071 /* a product's sums fit 32 bits, whatever the codes */

int64_t nb200_int8_pitch(const nb200_int8 *m);
/* Bytes of values for the extents in `m`, -1 if those are not possible. */
int64_t nb200_int8_value_count(const nb200_int8 *m);
/* Quantises. The rows of x are those of z, group after group. */
int nb200_int8_quantise(const nb200_dense *x, nb200_int8 *z, void *stream);
/* Takes over codes [groups * rows][cols] and scales [groups * rows] that exist. */
int nb200_int8_pack(const int8_t *codes, const float *scales, nb200_int8 *z, void *stream);
/* The 32-bit values that a matrix stands for, [groups * rows][cols] one after another. */
int nb200_int8_unpack(const nb200_int8 *a, float *z, void *stream);
/* y[i, n] = sa[i] sw[n] sum_k a[i, k] w[g][n, k]: rows a (one group) and channels w (a group per expert), y of any type; offsets as above. The sum is
 * exact, its product with the two scales rounded to 32 bits each time. At most NB200_MAX_INT8_COLUMNS columns. */
int nb200_int8_product(const nb200_int8 *a, const nb200_int8 *w, const int32_t *offsets, nb200_dense *y, void *stream);

/* ---- the norm of gradients ------------------------------------------------------------------ */

/* One of many tensors: `count` elements of a type at `from`, and where the scaled ones go, as another type if need be. `from` and `to` may be the same
 * place (of one type); otherwise nothing that is written may overlap anything else. */
typedef struct nb200_span {
    const void *from;
    void *to;
    int64_t count;
    int32_t type, to_type;
} nb200_span;

/* norm = the root of the sum of all squares, one float32 in device memory; every element goes over times max_norm / (norm + 1e-6) where that is below 1,
 * unchanged otherwise, and unchanged if the norm is no finite number. Sums in a fixed order, 64-bit beyond a few elements. `spans` is host memory; scratch:
 * 256-byte aligned device memory of nb200_clip_scratch bytes. Does not wait for the device; can be captured. */
int nb200_clip(const nb200_span *spans, int64_t n, float max_norm, float *norm, void *scratch, int64_t scratch_bytes, void *stream);
int64_t nb200_clip_scratch(const nb200_span *spans, int64_t n);

/* ---- self-test -------------------------------------------------------------------------- */

/* Exercises the give-up path of the bounded device-side waits without faulting or hanging the
 * GPU: runs the single-pass CSR add on (a, b) WITHOUT its first tile and with a look-back limit of
 * `polls` polls, so that the second tile waits for a count nobody publishes, gives up, records it
 * and lets its successors through. Needs operands of at least three tiles (a few thousand entries
 * each); `capacity` >= nnz(A) + nnz(B). Returns NB200_E_TIMEOUT when the path works (the contents
 * of z are then meaningless, but every write stayed inside its arrays); the context stays usable.
 * Has no counterpart in the reference, which has no device-side waits. */
int nb200_selftest_lookback_timeout(const nb200_csr *a, const nb200_csr *b, nb200_csr *z,
                                    int64_t capacity, int32_t polls, void *stream);

/* A give-up that comes late: all tiles run, but a tile waits for its output base for `polls` polls only, while the
 * counts it depends on do arrive. Returns NB200_E_TIMEOUT, or NB200_OK with a result that is whole. */
int nb200_selftest_late_give_up(const nb200_csr *a, const nb200_csr *b, nb200_csr *z,
                                int64_t capacity, int32_t polls, void *stream);

/* For calls that queue several merges, each of which reads the one before it on the device: the FIRST merge
 * of a three-operand add, and of a CSF3 add level by level, runs without its first tile and gives up. The merges behind
 * it must read none of its results and the call must return NB200_E_TIMEOUT. Needs 24000 entries in A and B (of
 * the CSF3 tensors: slices); capacities of the worst case. */
int nb200_selftest_chain_timeout(const nb200_csr *a, const nb200_csr *b, const nb200_csr *c, nb200_csr *z,
                                 int64_t capacity, int32_t polls, void *stream);
int nb200_selftest_levels_timeout(const nb200_csf3 *a, const nb200_csf3 *b, nb200_csf3 *z, int64_t cap_i, int64_t cap_j,
                                  int64_t cap_k, int32_t polls, void *stream);

/* For the 8-bit products, whose calls do not wait for their kernels: a product that is never given its first block, so that every wait in it gives
 * up after 20 ms. It writes nothing and returns NB200_OK; once it has ended, the NEXT product on the stream returns NB200_E_TIMEOUT in its
 * place, and the one after that works. y is 32-bit. */
int nb200_selftest_product_timeout(const nb200_fp8 *a, const nb200_fp8 *w, nb200_dense *y, void *stream);

/* The same for the kernel of gated products, their gradients and integer products of more than a few rows. */
int nb200_selftest_tiles_timeout(const nb200_int8 *a, const nb200_int8 *w, nb200_dense *y, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* NACHO_B200_H */
