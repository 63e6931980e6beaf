// Tokens sorted by expert and back. R (CSR, tokens x experts) is a router's decision; its entries sorted by expert, stably, say where
// the copies of a token's row go, and a token's result is the weighted sum of the rows at its entries' slots:
//     slot(e) = |{e' kept: c_e' < c_e}| + |{e' < e: c_e' = c_e}|,   xs[slot(e)] = x[t_e],   y[t] = sum_e w_e z[slot(e)].
// All of it walks token by token, so that a token's row is read (or written) once however many experts it has, and no sum
// needs atomics: the entries of a token are added in storage order.
#include <algorithm>
#include <type_traits>

#include "dense_rows.cuh"

namespace nb200 {
namespace {

constexpr int NT = 256;

// R and its order as kernels see them. `first` .. `last` is the range of entries that belong to rows of R: row offsets may point into
// larger arrays.
struct Order {
    const int32_t *row_ptr, *expert;
    int32_t *offsets, *rows, *slots;
    int32_t tokens, experts, entries;

    __device__ int entry_of(int t) const { return min(max(ld_late(row_ptr + t), 0), entries); }
    __device__ int key(int e) const {  // dropped entries have the key behind the last expert
        const int c = ld_late(expert + e);
        return c >= 0 && c < experts ? c : experts;
    }
    __device__ int slot(int e) const {
        const int s = ld_late(slots + e);
        return s < entries ? s : -1;
    }
    __device__ int kept() const { return min(max(ld_late(offsets + experts), 0), entries); }
};

// ---- the order -------------------------------------------------------------------------

constexpr int MAX_TILES = 256, AT_ONCE = 8;  // entries per thread that are on their way together

// How often each key occurs in this CTA's tile of entries: counts[tile][key]. They lie where the order's rows come to lie once all slots are known: a
// call has no memory of its own that another stream, or a later call beside a captured graph, could have too.
template <typename C>
__global__ void __launch_bounds__(NT) k_order_count(Order o, int tile) {
    extern __shared__ int32_t hist[];
    wait_for_previous();
    trigger_dependents();
    for (int k = threadIdx.x; k < o.experts; k += NT) hist[k] = 0;
    __syncthreads();
    const int64_t begin = (int64_t)blockIdx.x * tile;
    const int64_t from = max(begin, (int64_t)o.entry_of(0)), to = min(begin + tile, (int64_t)o.entry_of(o.tokens));
    for (int64_t e = from + threadIdx.x; e < to; e += NT) {
        const int k = o.key((int)e);
        if (k < o.experts) atomicAdd(&hist[k], 1);
    }
    __syncthreads();
    C *counts = reinterpret_cast<C *>(o.rows) + (int64_t)blockIdx.x * o.experts;
    for (int k = threadIdx.x; k < o.experts; k += NT) counts[k] = (C)hist[k];
}

// Slots of a tile's entries. Every warp has a stretch of the tile and a counter per expert, which starts at the slots in front of its stretch:
// those of all smaller experts, of this expert's entries in the tiles before, and of the warps before.
template <typename C>
__global__ void __launch_bounds__(NT) k_order_place(Order o, int tile, int tiles) {
    extern __shared__ int32_t next[];  // [warp][expert], then the experts' totals and their entries in the tiles before
    __shared__ int tmp[33];
    int32_t *total = next + (NT / 32) * o.experts, *before = total + o.experts;
    wait_for_previous();
    trigger_dependents();
    const int w = warp_id(), lane = lane_id();
    int32_t *mine = next + w * o.experts;
    for (int k = threadIdx.x; k < (NT / 32) * o.experts; k += NT) next[k] = 0;
    __syncthreads();
    const int64_t begin = (int64_t)blockIdx.x * tile + (int64_t)w * (tile / (NT / 32));
    const int64_t end = min(begin + tile / (NT / 32), (int64_t)o.entries);
    const int lo = o.entry_of(0), hi = o.entry_of(o.tokens);
    auto key_of = [&](int64_t e) { return e < end && e >= lo && e < hi ? o.key((int)e) : o.experts; };
    for (int64_t e0 = begin + lane; e0 - lane < end; e0 += 32 * AT_ONCE) {
        int key[AT_ONCE];
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u) key[u] = key_of(e0 + 32 * u);
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u)
            if (key[u] < o.experts) atomicAdd(&mine[key[u]], 1);
    }
    // an expert's entries in all tiles and in the tiles before, all threads over all counts, eight of them on their way at a time
    for (int k = threadIdx.x; k < 2 * o.experts; k += NT) total[k] = 0;
    __syncthreads();
    const C *counts = reinterpret_cast<const C *>(o.rows);
    const int64_t all = (int64_t)tiles * o.experts, mine_too = (int64_t)blockIdx.x * o.experts;
    for (int64_t i0 = threadIdx.x; i0 < all; i0 += 8 * NT) {
        int c[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) c[u] = i0 + u * NT < all ? ld_late(counts + i0 + u * NT) : 0;
#pragma unroll
        for (int u = 0; u < 8; ++u)
            if (c[u]) {
                const int k = (int)((i0 + u * NT) % o.experts);
                atomicAdd(&total[k], c[u]);
                if (i0 + u * NT < mine_too) atomicAdd(&before[k], c[u]);
            }
    }
    __syncthreads();
    int base = 0;
    for (int k0 = 0; k0 < o.experts; k0 += NT) {
        const int k = k0 + threadIdx.x;
        int sum;
        const int at = base + block_excl_sum<NT>(k < o.experts ? total[k] : 0, tmp, sum);
        if (k < o.experts) {
            if (blockIdx.x == 0) o.offsets[k] = at;
            int from = at + before[k];
            for (int v = 0; v < NT / 32; ++v) {
                const int c = next[v * o.experts + k];
                next[v * o.experts + k] = from;
                from += c;
            }
        }
        base += sum;
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) o.offsets[o.experts] = base;
    __syncthreads();
    for (int64_t e0 = begin + lane; e0 - lane < end; e0 += 32 * AT_ONCE) {
        int key[AT_ONCE];
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u) key[u] = key_of(e0 + 32 * u);
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u) {
            const int k = key[u];
            const unsigned same = __match_any_sync(FULL_MASK, k);
            const int rank = __popc(same & ((1u << lane) - 1));
            int slot = -1;
            if (k < o.experts) slot = mine[k] + rank;
            __syncwarp();
            if (k < o.experts && rank == 0) mine[k] += __popc(same);
            __syncwarp();
            if (e0 + 32 * u < end) o.slots[e0 + 32 * u] = slot;
        }
    }
}

// ---- moving rows -----------------------------------------------------------------------

// `tpr` threads (a power of two from 32 to NT) have a token together; a CTA has NT / tpr tokens at a time. Loops over tokens and slots count without a
// sign: the last of them may lie less than a step below 2^31.
struct Team {
    int size, lane;
    unsigned first, step;  // first token, distance to the next
    __device__ explicit Team(int tpr) : size(tpr), lane(threadIdx.x & (tpr - 1)), first(blockIdx.x * (NT / tpr) + threadIdx.x / tpr), step(gridDim.x * (NT / tpr)) {}
};

template <typename T, int V>
__device__ __forceinline__ void copy_rows(const Order &o, const Team &team, int t, const T *x, int64_t stride, int64_t cols, T *xs) {
    constexpr int U = 4;
    using C = Chunk<T, V>;
    const int64_t pitch = (int64_t)team.size * V;
    const int e0 = o.entry_of(t), e1 = o.entry_of(t + 1);
    if (team.lane == 0)
        for (int e = e0; e < e1; ++e) {
            const int s = o.slot(e);
            if (s >= 0) o.rows[s] = t;
        }
    if (e0 >= e1) return;
    for (int64_t c = team.lane * V; c < cols; c += pitch * C::WORDS * U) {
        C v[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (c + u * C::WORDS * pitch < cols) v[u].load(x + t * stride, c + u * C::WORDS * pitch, pitch, cols);
        for (int e = e0; e < e1; ++e) {
            const int s = o.slot(e);
            if (s < 0) continue;
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (c + u * C::WORDS * pitch < cols) v[u].store(xs + s * cols, c + u * C::WORDS * pitch, pitch, cols);
        }
    }
}

template <typename T, int V>
__device__ __forceinline__ void clear_rows(const Order &o, int kept, const Team &team, int64_t cols, T *xs) {
    for (unsigned s = kept + team.first; s < (unsigned)o.entries; s += team.step) {
        if (o.rows && team.lane == 0) o.rows[s] = -1;
        for (int64_t c = team.lane * V; c < cols; c += team.size * V) {
            Vec<T, V> zero;
#pragma unroll
            for (int j = 0; j < V; ++j) zero.v[j] = from_float<T>(0.f);
            *reinterpret_cast<Vec<T, V> *>(xs + s * cols + c) = zero;
        }
    }
}

template <typename T, int V>
__global__ void __launch_bounds__(NT) k_sort_rows(Order o, int tpr, const T *x, int64_t stride, int64_t cols, T *xs) {
    wait_for_previous();
    trigger_dependents();
    const Team team(tpr);
    for (unsigned t = team.first; t < (unsigned)o.tokens; t += team.step) copy_rows<T, V>(o, team, t, x, stride, cols, xs);
    clear_rows<T, V>(o, o.kept(), team, cols, xs);
}

__device__ __forceinline__ void clear_rows8(const Order &o, int kept, const Team &team, int64_t kb, uint8_t *codes, float *scales) {
    const int sub = team.lane & 15;
    const int64_t pad = padded_rows(o.entries);
    for (unsigned s = kept + team.first; s < (unsigned)o.entries; s += team.step) {
        if (team.lane == 0) o.rows[s] = -1;
        for (int64_t b = team.lane >> 4; b < kb; b += team.size >> 4) {
            *reinterpret_cast<uint2 *>(codes + b * pad * BLOCK8 + piece_at(s, sub >> 1) + (sub & 1) * 8) = make_uint2(0, 0);
            if (sub == 0) scales[b * pad + s] = 0.f;
        }
    }
}

// The entries of the tokens a team works on, asked for early: row offsets two tokens ahead, the slots of up to N entries one ahead, so that a
// token's rows can be asked for at once; weights with the rows, as they are needed no earlier. Nothing here looks at a loaded word before
// the token's turn.
template <int N>
struct Entries {
    const Order &o;
    const float *w;
    unsigned t, step;
    int e0, e1, next0, next1, slot[N], raw[N];
    float weight[N];

    __device__ Entries(const Order &order, const float *weights, unsigned first, unsigned distance) : o(order), w(weights), t(first - distance), step(distance) {
        next0 = o.entry_of(min(first, (unsigned)o.tokens)), next1 = o.entry_of(min(first + 1, (unsigned)o.tokens));
        ask();
    }
    __device__ void ask() {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            raw[i] = -1;
            if (next0 + i < next1) raw[i] = ld_late(o.slots + next0 + i);
        }
    }
    __device__ int clamped(int s) const { return s < o.entries ? s : -1; }
    // The next token, if there is one.
    __device__ bool advance() {
        t += step;
        if (t >= (unsigned)o.tokens) return false;
        const int64_t after = min((int64_t)t + step, (int64_t)o.tokens);
        e0 = next0, e1 = next1;
        next0 = ld_late(o.row_ptr + after), next1 = ld_late(o.row_ptr + min(after + 1, (int64_t)o.tokens));
#pragma unroll
        for (int i = 0; i < N; ++i) {
            slot[i] = clamped(raw[i]);
            weight[i] = w && e0 + i < e1 ? ld_late(w + e0 + i) : 1.f;
        }
        return true;
    }
    // To be called when the rows of this token are on their way.
    __device__ void ask_next() {
        next0 = min(max(next0, 0), o.entries), next1 = min(max(next1, 0), o.entries);
        ask();
    }
};

// The same into 8-bit rows: eight threads have a block of 128 columns, quantise it once and write it to all of the token's slots. 65536
// rows of 4096 from 16384 tokens of 16 bits take 85 us (411 MB, 0.74 of a copy's rate): a thread has one block's loads on their way and waits for them.
template <typename T, int V, int N>
__global__ void __launch_bounds__(NT, 4) k_sort_rows_fp8(Order o, int tpr, const T *x, int64_t stride, int64_t cols, uint8_t *codes, float *scales) {
    wait_for_previous();
    trigger_dependents();
    const Team team(tpr);
    const int sub = team.lane & 7, mine = team.lane >> 3, blocks = team.size >> 3;
    const unsigned eight = 0xffu << (threadIdx.x & 24);
    const int64_t pad = padded_rows(o.entries);
    const int kb = (int)blocks_of(cols);
    auto place_of = [&](int s) { return codes + piece_at(s, sub); };
    Entries<N> at(o, nullptr, team.first, team.step);
    while (at.advance()) {
        const T *row = x + at.t * stride;
        uint8_t *place[N];  // kept where registers last
        if constexpr (N == 4) {
#pragma unroll
            for (int i = 0; i < N; ++i) place[i] = place_of(at.slot[i]);
        }
        for (int b = mine; b < kb; b += blocks) {
            Piece<T> v;
            v.template load<V>(row, (int64_t)b * BLOCK8 + sub * 16, cols);
            if (b == mine) {
                if (team.lane == 0)
                    for (int e = at.e0; e < at.e1; ++e) {
                        const int s = o.slot(e);
                        if (s >= 0) o.rows[s] = at.t;
                    }
                at.ask_next();
            }
            const Factors f = factors_of(v.top(eight));
            const uint4 q = v.codes(f.inverse);
            const int64_t block = (int64_t)b * pad;
            auto put = [&](uint8_t *to, int s) {
                if (s < 0) return;
                *reinterpret_cast<uint4 *>(to + block * BLOCK8) = q;
                if (sub == 0) scales[block + s] = f.scale;
            };
#pragma unroll
            for (int i = 0; i < N; ++i) put(N == 4 ? place[i] : place_of(at.slot[i]), at.slot[i]);
            for (int e = at.e0 + N; e < at.e1; ++e) {
                const int s = o.slot(e);
                put(place_of(s), s);
            }
        }
        if (mine >= kb) at.ask_next();
    }
    clear_rows8(o, o.kept(), team, kb, codes, scales);
}

// y[t] = sum of w[e] * z[slot(e)]. The rows of up to N entries are on their way together. Bound by device memory as long as nothing spills: three CTAs
// of 80 registers to an SM (N = 4) take 65536 rows of 4096 back in 110 us, 93 % of a copy; four of 64 registers 153.
template <typename T, int V, int N>
__global__ void __launch_bounds__(NT, N == 8 ? 2 : 3) k_unsort_rows(Order o, int tpr, const float *w, const T *z, int64_t stride, T *y, int64_t y_stride, int64_t cols) {
    wait_for_previous();
    trigger_dependents();
    const Team team(tpr);
    using C = Chunk<T, V>;
    const int64_t pitch = (int64_t)team.size * V;
    Entries<N> at(o, w, team.first, team.step);
    while (at.advance()) {
        bool asked = false;
        for (int64_t c = team.lane * V; c < cols; c += pitch * C::WORDS) {
            float sum[C::N];
            C v[N];
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (at.slot[i] >= 0) v[i].load(z + at.slot[i] * stride, c, pitch, cols);
            if (!asked) at.ask_next(), asked = true;
#pragma unroll
            for (int j = 0; j < C::N; ++j) sum[j] = 0.f;
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (at.slot[i] >= 0) {
#pragma unroll
                    for (int j = 0; j < C::N; ++j) sum[j] = __fmaf_rn(at.weight[i], v[i].get(j), sum[j]);
                }
            for (int e = at.e0 + N; e < at.e1; ++e) {
                const int s = o.slot(e);
                if (s < 0) continue;
                C more;
                more.load(z + s * stride, c, pitch, cols);
                const float g = w ? ld_late(w + e) : 1.f;
#pragma unroll
                for (int j = 0; j < C::N; ++j) sum[j] = __fmaf_rn(g, more.get(j), sum[j]);
            }
            C out;
#pragma unroll
            for (int j = 0; j < C::N; ++j) out.set(j, sum[j]);
            out.store(y + at.t * y_stride, c, pitch, cols);
        }
        if (!asked) at.ask_next();
    }
}

// dz[slot(e)] = w[e] * dy[t] and dw[e] = <dy[t], z[slot(e)]>, N entries of a token at a time. Sums over the columns: every thread its own,
// then the warp's by exchanges, then the team's warps' in order, in shared memory that two batches in turn have.
template <typename T, int V, int N>
__global__ void __launch_bounds__(NT, N == 8 ? 2 : 3) k_unsort_grad(Order o, int tpr, const float *w, const T *z, int64_t z_stride, const T *dy, int64_t dy_stride, T *dz, float *dw,
                                                    int64_t cols) {
    __shared__ float part[2][NT / 32][N];
    wait_for_previous();
    trigger_dependents();
    const Team team(tpr);
    using C = Chunk<T, V>;
    const int64_t pitch = (int64_t)team.size * V;
    const int warps = tpr / 32, name = 1 + threadIdx.x / tpr;
    int turn = 0;
    Entries<N> at(o, w, team.first, team.step);
    while (at.advance()) {
        bool asked = false;
        for (int e = at.e0; e < at.e1; e += N, turn ^= 1) {
            if (e > at.e0)  // more than N entries: these were not asked for early
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    at.slot[i] = e + i < at.e1 ? o.slot(e + i) : -1;
                    at.weight[i] = at.slot[i] >= 0 ? ld_late(w + e + i) : 0.f;
                }
            float dot[N];
#pragma unroll
            for (int i = 0; i < N; ++i) dot[i] = 0.f;
            for (int64_t c = team.lane * V; c < cols; c += pitch * C::WORDS) {
                C d, v[N];
                d.load(dy + at.t * dy_stride, c, pitch, cols);
#pragma unroll
                for (int i = 0; i < N; ++i)
                    if (at.slot[i] >= 0) v[i].load(z + at.slot[i] * z_stride, c, pitch, cols);
                if (!asked) at.ask_next(), asked = true;
#pragma unroll
                for (int i = 0; i < N; ++i)
                    if (at.slot[i] >= 0) {
                        C out;
#pragma unroll
                        for (int j = 0; j < C::N; ++j) {
                            if (C::there(j, c, pitch, cols)) dot[i] = __fmaf_rn(d.get(j), v[i].get(j), dot[i]);
                            out.set(j, at.weight[i] * d.get(j));
                        }
                        out.store(dz + at.slot[i] * cols, c, pitch, cols);
                    }
            }
#pragma unroll
            for (int i = 0; i < N; ++i)
                for (int d = 16; d; d >>= 1) dot[i] += __shfl_xor_sync(FULL_MASK, dot[i], d);
            if (warps > 1) {
                if (lane_id() == 0)
#pragma unroll
                    for (int i = 0; i < N; ++i) part[turn][warp_id()][i] = dot[i];
                asm volatile("bar.sync %0, %1;" ::"r"(name), "r"(tpr) : "memory");
                if (team.lane < N) {
                    float sum = 0.f;
                    for (int v = 0; v < warps; ++v) sum += part[turn][warp_id() + v][team.lane];
                    if (e + team.lane < at.e1) dw[e + team.lane] = o.slot(e + team.lane) >= 0 ? sum : 0.f;
                }
            } else if (team.lane == 0) {
#pragma unroll
                for (int i = 0; i < N; ++i)
                    if (e + i < at.e1) dw[e + i] = at.slot[i] >= 0 ? dot[i] : 0.f;
            }
        }
        if (!asked) at.ask_next();
    }
    Order tail = o;
    tail.rows = nullptr;
    clear_rows<T, V>(tail, o.kept(), team, cols, dz);
    // entries of no row: views into larger arrays
    const int lo = o.entry_of(0), hi = o.entry_of(o.tokens);
    for (unsigned e = blockIdx.x * NT + threadIdx.x; e < (unsigned)o.entries; e += gridDim.x * NT)
        if (e < (unsigned)lo || e >= (unsigned)hi) dw[e] = 0.f;
}

// ---- few entries: all in one launch ------------------------------------------------------

// Up to this many entries, every CTA counts all of them: that takes less than a launch. Its own tokens' entries follow from the totals and
// from the counts of those in front of them. Order and rows of 2048 16-bit elements, us, by 8 / 64 / 256 experts: 2048 entries 7.6 / 9.8 / 10.4 where
// two launches for the order in front take 11.5 / 11.3 / 11.4; 4096 entries 10.8 / 14.5 / 15.5 against 11.5 / 11.6 / 12.2.
constexpr int FEW_ENTRIES = 2560;

// Slots of the entries of tokens t0 .. t1 - 1, the offsets, and how many entries are kept (returned). counts: two words per expert.
__device__ int place_few(const Order &o, int t0, int t1, int32_t *counts) {
    __shared__ int tmp[33];
    int32_t *total = counts, *next = counts + o.experts;
    const int lane = lane_id();
    const int lo = o.entry_of(0), hi = o.entry_of(o.tokens), e0 = o.entry_of(t0), e1 = o.entry_of(t1);
    for (int k = threadIdx.x; k < 2 * o.experts; k += NT) counts[k] = 0;
    __syncthreads();
    for (int e = lo + (int)threadIdx.x; e - lane < hi; e += NT) {
        const int k = e < hi ? o.key(e) : o.experts;
        const unsigned same = __match_any_sync(FULL_MASK, k);
        const unsigned before = __ballot_sync(FULL_MASK, e < e0);
        if (k < o.experts && (same & ((1u << lane) - 1)) == 0) {
            atomicAdd(&total[k], __popc(same));
            if (same & before) atomicAdd(&next[k], __popc(same & before));
        }
    }
    __syncthreads();
    int kept = 0;
    for (int k0 = 0; k0 < o.experts; k0 += NT) {
        const int k = k0 + threadIdx.x;
        int sum;
        const int at = kept + block_excl_sum<NT>(k < o.experts ? total[k] : 0, tmp, sum);
        if (k < o.experts) {
            next[k] += at;
            if (blockIdx.x == 0) o.offsets[k] = at;
        }
        kept += sum;
    }
    if (blockIdx.x == 0) {
        if (threadIdx.x == 0) o.offsets[o.experts] = kept;
        for (int e = threadIdx.x; e < o.entries; e += NT)
            if (e < lo || e >= hi) o.slots[e] = -1;  // entries of no row
    }
    __syncthreads();
    if (warp_id() == 0)
        for (int e = e0 + lane; e - lane < e1; e += 32) {
            const int k = e < e1 ? o.key(e) : o.experts;
            const unsigned same = __match_any_sync(FULL_MASK, k);
            const int rank = __popc(same & ((1u << lane) - 1));
            const int slot = k < o.experts ? next[k] + rank : -1;
            __syncwarp();
            if (k < o.experts && rank == 0) next[k] += __popc(same);
            __syncwarp();
            if (e < e1) o.slots[e] = slot;
        }
    __syncthreads();
    return kept;
}

template <typename T, int V>
__global__ void __launch_bounds__(NT) k_sort_few(Order o, int per_cta, int tpr, const T *x, int64_t stride, int64_t cols, T *xs) {
    extern __shared__ int32_t counts[];
    wait_for_previous();
    trigger_dependents();
    const int t0 = (int)min(blockIdx.x * (unsigned)per_cta, (unsigned)o.tokens), t1 = (int)min((unsigned)t0 + per_cta, (unsigned)o.tokens);
    const int kept = place_few(o, t0, t1, counts);
    Team team(tpr);
    for (int t = t0 + (int)threadIdx.x / tpr; t < t1; t += NT / tpr) copy_rows<T, V>(o, team, t, x, stride, cols, xs);
    clear_rows<T, V>(o, kept, team, cols, xs);
}

template <typename T, int V>
__global__ void __launch_bounds__(NT) k_sort_few_fp8(Order o, int per_cta, int tpr, const T *x, int64_t stride, int64_t cols, uint8_t *codes, float *scales) {
    extern __shared__ int32_t counts[];
    wait_for_previous();
    trigger_dependents();
    const int t0 = (int)min(blockIdx.x * (unsigned)per_cta, (unsigned)o.tokens), t1 = (int)min((unsigned)t0 + per_cta, (unsigned)o.tokens);
    const int kept = place_few(o, t0, t1, counts);
    const Team team(tpr);
    const int sub = team.lane & 15;
    const unsigned half = 0xffffu << (threadIdx.x & 16);
    const int64_t pad = padded_rows(o.entries), kb = blocks_of(cols);
    for (int t = t0 + (int)threadIdx.x / tpr; t < t1; t += NT / tpr) {
        const int e0 = o.entry_of(t), e1 = o.entry_of(t + 1);
        for (int e = e0 + team.lane; e < e1; e += tpr) {
            const int s = o.slot(e);
            if (s >= 0) o.rows[s] = t;
        }
        for (int64_t b = team.lane >> 4; b < kb; b += team.size >> 4) {
            Eight<T> v;
            v.template load<V>(x + t * stride, b * BLOCK8 + sub * 8, cols);
            Top<T> top;
            top.add(v);
#pragma unroll
            for (int d = 8; d; d >>= 1) top.join(half, d);
            const Factors f = factors_of(top.bits());
            const uint2 q = codes8(v, f.inverse);
            for (int e = e0; e < e1; ++e) {
                const int s = o.slot(e);
                if (s < 0) continue;
                *reinterpret_cast<uint2 *>(codes + b * pad * BLOCK8 + piece_at(s, sub >> 1) + (sub & 1) * 8) = q;
                if (sub == 0) scales[b * pad + s] = f.scale;
            }
        }
    }
    clear_rows8(o, kept, team, kb, codes, scales);
}

// ---- host ------------------------------------------------------------------------------

// Threads per token for rows that take `loads` of 16 bytes: up to four each (the way back of 131072 rows of 8 KB 187 us, with two each 191, with eight
// 186, but odd rows of 4 KB 14.6, 14.8 and 18.3), and two each while all tokens together leave most of the GPU free.
int team_of(int64_t loads, int64_t tokens) {
    int t = 32;
    while (t < NT && (4 * t < loads || (2 * t < loads && tokens * t < (int64_t)sm_count() * 512))) t *= 2;
    return t;
}

dim3 grid_of(int64_t teams, int tpr) {
    const int64_t ctas = (teams * tpr + NT - 1) / NT;
    return dim3((unsigned)std::max<int64_t>(1, std::min<int64_t>(ctas, (int64_t)sm_count() * 64)));
}

// As many CTAs as can be at work at once, or fewer where there are fewer teams' worth of tokens.
template <typename... P>
dim3 resident_grid(void (*kernel)(P...), int64_t teams, int tpr) {
    const int per_sm = resident_ctas(reinterpret_cast<const void *>(kernel), NT);
    const int64_t ctas = (teams * tpr + NT - 1) / NT;
    return dim3((unsigned)std::max<int64_t>(1, std::min<int64_t>(ctas, (int64_t)sm_count() * per_sm)));
}

// Entries per token that kernels hold at a time: what an average token has, 4 or 8.
bool many_entries(const Order &o) { return (int64_t)o.entries > 4 * (int64_t)o.tokens; }

int check_order(const nb200_expert_order *o, bool slots_given) {
    if (!o || o->tokens < 0 || o->experts < 0 || o->entries < 0 || !o->row_ptr || !o->offsets) return NB200_E_BADARG;
    if (o->entries > 0 && (!o->slots || (!slots_given && !o->rows))) return NB200_E_BADARG;
    // the last numbers in front of 2^31 are what kernels that look a few entries or tokens ahead may count up to
    return o->experts > NB200_MAX_EXPERTS || o->tokens > INT32_MAX - 1024 || o->entries > INT32_MAX - 1024 ? NB200_E_UNSUPPORTED : NB200_OK;
}

Order order_of(const nb200_expert_order *o, const int32_t *expert) {
    return {o->row_ptr, expert, o->offsets, o->rows, o->slots, o->tokens, o->experts, o->entries};
}

int check_routing(const nb200_csr *r, nb200_expert_order *order) {
    if (!r || !order || r->rows < 0 || r->cols < 0 || r->nnz < 0 || !r->row_ptr || (r->nnz > 0 && !r->col)) return NB200_E_BADARG;
    order->row_ptr = r->row_ptr;
    order->tokens = r->rows, order->experts = r->cols, order->entries = r->nnz;
    return check_order(order, false);
}

// The launch for few entries: two CTAs to an SM at most, since each counts all entries.
struct Few {
    int per_cta;
    dim3 grid;
    size_t smem;
    Few(const Order &o, int tpr) {
        const int teams = NT / tpr, most = 2 * sm_count();
        per_cta = (int)std::max<int64_t>(teams, ((int64_t)o.tokens + most - 1) / most);
        grid = dim3((unsigned)std::max<int64_t>(1, ((int64_t)o.tokens + per_cta - 1) / per_cta));
        smem = sizeof(int32_t) * 2 * o.experts;
    }
};

// The entries of a CTA, a multiple of the warps' 32 each, and how many CTAs there are: as few entries as leave no more than MAX_TILES CTAs and
// tables of counts, 16 bits each while a tile's entries can be counted in those, that fit into the order's `rows` (up to 2560 experts they do with 2048).
struct OrderTiles {
    int tile = 2048, tiles;
    OrderTiles(int64_t entries, int64_t experts) {  // entries > FEW_ENTRIES, so that one table fits
        auto fits = [&] {
            tiles = (int)((entries + tile - 1) / tile);
            return tiles <= MAX_TILES && tiles * experts * (narrow() ? 2 : 4) <= entries * 4;
        };
        while (!fits()) tile *= 2;
    }
    bool narrow() const { return tile < 1 << 16; }
};
static_assert(2 * NB200_MAX_EXPERTS <= 4 * FEW_ENTRIES, "");

template <typename C>
int make_order(const Order &o, int tile, int tiles, cudaStream_t stream) {
    int st;
    const size_t count_smem = sizeof(int32_t) * o.experts, place_smem = sizeof(int32_t) * o.experts * (NT / 32 + 2);
    if (place_smem > 32 * 1024 && (st = allow_shared(k_order_place<C>, place_smem))) return st;
    {
        LaunchScope scope("order_count", stream);
        NB200_CUDA(launch_overlapped(k_order_count<C>, dim3(tiles), dim3(NT), count_smem, stream, o, tile));
    }
    LaunchScope scope("order_place", stream);
    NB200_CUDA(launch_overlapped(k_order_place<C>, dim3(tiles), dim3(NT), place_smem, stream, o, tile, tiles));
    return NB200_OK;
}
int make_order(const Order &o, cudaStream_t stream) {
    const OrderTiles cut(o.entries, o.experts);
    return cut.narrow() ? make_order<uint16_t>(o, cut.tile, cut.tiles, stream) : make_order<int32_t>(o, cut.tile, cut.tiles, stream);
}

}  // namespace
}  // namespace nb200

using namespace nb200;

extern "C" {

int nb200_expert_sort(const nb200_csr *r, const nb200_dense *x, nb200_expert_order *order, nb200_dense *xs, void *stream_) {
    int st;
    if ((st = check_routing(r, order))) return st;
    if (x && (!dense_ok(x) || !dense_ok(xs) || x->rows != r->rows || xs->rows != r->nnz || xs->cols != x->cols || xs->type != x->type || xs->stride != xs->cols))
        return NB200_E_BADARG;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    const Order o = order_of(order, r->col);
    const nb200_dense none{r->rows, 0, 0, NB200_F32, nullptr};
    if (!x) x = &none, xs = const_cast<nb200_dense *>(&none);
    if (o.entries > FEW_ENTRIES && (st = make_order(o, stream))) return st;
    const int word = word_bytes({x, xs}), tpr = team_of((x->cols * type_size(x->type) + 15) / 16, o.tokens);
    return with_type(x->type, [&](auto e) {
        using T = decltype(e);
        return with_vector<T>(word, [&](auto v) {
            if (o.entries <= FEW_ENTRIES) {
                const Few few(o, tpr);
                LaunchScope scope("sort_few", stream);
                NB200_CUDA(launch_overlapped(k_sort_few<T, decltype(v)::value>, few.grid, dim3(NT), few.smem, stream, o, few.per_cta, tpr, static_cast<const T *>(x->data),
                                             x->stride, x->cols, static_cast<T *>(xs->data)));
                return (int)NB200_OK;
            }
            LaunchScope scope("sort_rows", stream);
            NB200_CUDA(launch_overlapped(k_sort_rows<T, decltype(v)::value>, grid_of(o.tokens, tpr), dim3(NT), 0, stream, o, tpr, static_cast<const T *>(x->data), x->stride, x->cols,
                                         static_cast<T *>(xs->data)));
            return (int)NB200_OK;
        });
    });
}

int nb200_expert_sort_fp8(const nb200_csr *r, const nb200_dense *x, nb200_expert_order *order, nb200_fp8 *xs, void *stream_) {
    int st;
    if ((st = check_routing(r, order))) return st;
    if (!dense_ok(x) || !fp8_ok(xs) || x->rows != r->rows || xs->groups != 1 || xs->tiled || xs->rows != r->nnz || xs->cols != x->cols) return NB200_E_BADARG;
    if (x->cols == 0) return nb200_expert_sort(r, nullptr, order, nullptr, stream_);  // the kernels below fill in the order beside a token's first block
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    const Order o = order_of(order, r->col);
    const bool all_in_one = o.entries <= FEW_ENTRIES;
    if (!all_in_one && (st = make_order(o, stream))) return st;
    const int word = word_bytes({x}), tpr = team_of(blocks_of(x->cols) * 32, o.tokens);
    return with_type(x->type, [&](auto e) {
        using T = decltype(e);
        return with_vector<T>(word, [&](auto v) {
            if (all_in_one) {
                const Few few(o, tpr);
                LaunchScope scope("sort_few_fp8", stream);
                NB200_CUDA(launch_overlapped(k_sort_few_fp8<T, decltype(v)::value>, few.grid, dim3(NT), few.smem, stream, o, few.per_cta, tpr, static_cast<const T *>(x->data),
                                             x->stride, x->cols, xs->values, xs->scales));
                return (int)NB200_OK;
            }
            auto kernel = many_entries(o) ? k_sort_rows_fp8<T, decltype(v)::value, 8> : k_sort_rows_fp8<T, decltype(v)::value, 4>;
            LaunchScope scope("sort_rows_fp8", stream);
            NB200_CUDA(launch_overlapped(kernel, resident_grid(kernel, o.tokens, tpr), dim3(NT), 0, stream, o, tpr, static_cast<const T *>(x->data), x->stride, x->cols, xs->values,
                                         xs->scales));
            return (int)NB200_OK;
        });
    });
}

int nb200_expert_unsort(const nb200_expert_order *order, const float *w, const nb200_dense *z, nb200_dense *y, void *stream_) {
    int st;
    if ((st = check_order(order, true))) return st;
    if (!dense_ok(z) || !dense_ok(y) || z->rows != order->entries || y->rows != order->tokens || y->cols != z->cols || y->type != z->type) return NB200_E_BADARG;
    if (y->rows == 0 || y->cols == 0) return NB200_OK;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    const Order o = order_of(order, nullptr);
    const int word = word_bytes({z, y}), tpr = team_of((z->cols * type_size(z->type) + 15) / 16, o.tokens);
    return with_type(z->type, [&](auto e) {
        using T = decltype(e);
        return with_vector<T>(word, [&](auto v) {
            auto kernel = many_entries(o) ? k_unsort_rows<T, decltype(v)::value, 8> : k_unsort_rows<T, decltype(v)::value, 4>;
            LaunchScope scope("unsort_rows", stream);
            NB200_CUDA(launch_overlapped(kernel, resident_grid(kernel, o.tokens, tpr), dim3(NT), 0, stream, o, tpr, w, static_cast<const T *>(z->data), z->stride,
                                         static_cast<T *>(y->data), y->stride, z->cols));
            return (int)NB200_OK;
        });
    });
}

int nb200_expert_unsort_grad(const nb200_expert_order *order, const float *w, const nb200_dense *z, const nb200_dense *dy, nb200_dense *dz, float *dw, void *stream_) {
    int st;
    if ((st = check_order(order, true))) return st;
    if (!dense_ok(z) || !dense_ok(dy) || !dense_ok(dz) || z->rows != order->entries || dz->rows != z->rows || dy->rows != order->tokens || dy->cols != z->cols ||
        dz->cols != z->cols || dy->type != z->type || dz->type != z->type || dz->stride != dz->cols || (order->entries > 0 && (!w || !dw)))
        return NB200_E_BADARG;
    if (order->entries == 0) return NB200_OK;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    const Order o = order_of(order, nullptr);
    const int word = word_bytes({z, dy, dz}), tpr = team_of((z->cols * type_size(z->type) + 15) / 16, o.tokens);
    return with_type(z->type, [&](auto e) {
        using T = decltype(e);
        return with_vector<T>(word, [&](auto v) {
            auto kernel = many_entries(o) ? k_unsort_grad<T, decltype(v)::value, 8> : k_unsort_grad<T, decltype(v)::value, 4>;
            LaunchScope scope("unsort_grad", stream);
            NB200_CUDA(launch_overlapped(kernel, resident_grid(kernel, std::max<int64_t>(o.tokens, 1), tpr), dim3(NT), 0, stream, o, tpr, w,
                                         static_cast<const T *>(z->data), z->stride, static_cast<const T *>(dy->data), dy->stride, static_cast<T *>(dz->data), dw, z->cols));
            return (int)NB200_OK;
        });
    });
}

}  // extern "C"
