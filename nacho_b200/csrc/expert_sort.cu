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
constexpr int ORDER_SLOT = 8;  // of the scratch pool

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

constexpr int MAX_TILES = 256;

// How often each key occurs in this CTA's tile of entries: counts[key][tile].
__global__ void __launch_bounds__(NT) k_order_count(Order o, int tile, int tiles, int32_t *counts) {
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
    for (int k = threadIdx.x; k < o.experts; k += NT) counts[(int64_t)k * tiles + blockIdx.x] = hist[k];
}

// Slots of a tile's entries. Every warp has a stretch of the tile and a counter per expert, which starts at the slots in front of its stretch:
// those of all smaller experts, of this expert's entries in the tiles before, and of the warps before.
__global__ void __launch_bounds__(NT) k_order_place(Order o, int tile, int tiles, const int32_t *counts) {
    extern __shared__ int32_t next[];  // [warp][expert], then the experts' totals
    __shared__ int tmp[33];
    int32_t *total = next + (NT / 32) * o.experts;
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
    for (int64_t e = begin + lane; e - lane < end; e += 32) {
        const int k = key_of(e);
        if (k < o.experts) atomicAdd(&mine[k], 1);
    }
    // this expert's entries in all tiles and in the tiles before, a warp per expert
    __syncthreads();
    for (int k = w; k < o.experts; k += NT / 32) {
        int all = 0, before = 0;
        for (int j = lane; j < tiles; j += 32) {
            const int c = ld_late(counts + (int64_t)k * tiles + j);
            all += c;
            before += j < (int)blockIdx.x ? c : 0;
        }
        all = __reduce_add_sync(FULL_MASK, all);
        before = __reduce_add_sync(FULL_MASK, before);
        if (lane == 0) {
            total[k] = all;
            for (int v = 0; v < NT / 32; ++v) {
                const int c = next[v * o.experts + k];
                next[v * o.experts + k] = before;
                before += c;
            }
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
            for (int v = 0; v < NT / 32; ++v) next[v * o.experts + k] += at;
        }
        base += sum;
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) o.offsets[o.experts] = base;
    __syncthreads();
    for (int64_t e = begin + lane; e - lane < end; e += 32) {
        const int k = key_of(e);
        const unsigned same = __match_any_sync(FULL_MASK, k);
        const int rank = __popc(same & ((1u << lane) - 1));
        int slot = -1;
        if (k < o.experts) slot = mine[k] + rank;
        __syncwarp();
        if (k < o.experts && rank == 0) mine[k] += __popc(same);
        __syncwarp();
        if (e < end) o.slots[e] = slot;
    }
}

// ---- moving rows -----------------------------------------------------------------------

// `tpr` threads (a power of two from 32 to NT) have a token together; a CTA has NT / tpr tokens at a time.
struct Team {
    int size, lane, first, step;  // first token, distance to the next
    __device__ explicit Team(int tpr) : size(tpr), lane(threadIdx.x & (tpr - 1)), first(blockIdx.x * (NT / tpr) + threadIdx.x / tpr), step(gridDim.x * (NT / tpr)) {}
};

template <typename T, int V>
__device__ __forceinline__ void copy_rows(const Order &o, const Team &team, int t, const T *x, int64_t stride, int64_t cols, T *xs) {
    constexpr int U = 4;
    const int e0 = o.entry_of(t), e1 = o.entry_of(t + 1);
    if (team.lane == 0)
        for (int e = e0; e < e1; ++e) {
            const int s = o.slot(e);
            if (s >= 0) o.rows[s] = t;
        }
    if (e0 >= e1) return;
    for (int64_t c = team.lane * V; c < cols; c += (int64_t)team.size * V * U) {
        Vec<T, V> v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t at = c + (int64_t)u * team.size * V;
            if (at < cols) v[u] = *reinterpret_cast<const Vec<T, V> *>(x + t * stride + at);
        }
        for (int e = e0; e < e1; ++e) {
            const int s = o.slot(e);
            if (s < 0) continue;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t at = c + (int64_t)u * team.size * V;
                if (at < cols) *reinterpret_cast<Vec<T, V> *>(xs + s * cols + at) = v[u];
            }
        }
    }
}

template <typename T, int V>
__device__ __forceinline__ void clear_rows(const Order &o, const Team &team, int64_t cols, T *xs) {
    for (int s = o.kept() + team.first; s < o.entries; s += team.step) {
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
    for (int t = team.first; t < o.tokens; t += team.step) copy_rows<T, V>(o, team, t, x, stride, cols, xs);
    clear_rows<T, V>(o, team, cols, xs);
}

// The same into 8-bit rows: 16 threads have a block of 128 columns, quantise it once and write it to all of the token's slots.
template <typename T, int V>
__global__ void __launch_bounds__(NT) k_sort_rows_fp8(Order o, int tpr, const T *x, int64_t stride, int64_t cols, uint8_t *codes, float *scales) {
    wait_for_previous();
    trigger_dependents();
    const Team team(tpr);
    const int sub = team.lane & 15;
    const unsigned half = 0xffffu << (threadIdx.x & 16);
    const int64_t pad = padded_rows(o.entries), kb = blocks_of(cols);
    for (int t = team.first; t < o.tokens; t += team.step) {
        const int e0 = o.entry_of(t), e1 = o.entry_of(t + 1);
        if (team.lane == 0)
            for (int e = e0; e < e1; ++e) {
                const int s = o.slot(e);
                if (s >= 0) o.rows[s] = t;
            }
        if (e0 >= e1) continue;
        for (int64_t b = team.lane >> 4; b < kb; b += team.size >> 4) {
            float v[8];
            load8<T, V>(x + t * stride, b * BLOCK8 + sub * 8, cols, v);
            uint32_t m = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) m = max(m, magnitude(v[j]));
#pragma unroll
            for (int d = 8; d; d >>= 1) m = max(m, __shfl_xor_sync(half, m, d));
            const Factors f = factors_of(m);
            const uint2 q = make_uint2(codes4(v[0], v[1], v[2], v[3], f.inverse), codes4(v[4], v[5], v[6], v[7], f.inverse));
            for (int e = e0; e < e1; ++e) {
                const int s = o.slot(e);
                if (s < 0) continue;
                *reinterpret_cast<uint2 *>(codes + b * pad * BLOCK8 + piece_at(s, sub >> 1) + (sub & 1) * 8) = q;
                if (sub == 0) scales[b * pad + s] = f.scale;
            }
        }
    }
    for (int s = o.kept() + team.first; s < o.entries; s += team.step) {
        if (team.lane == 0) o.rows[s] = -1;
        for (int64_t b = team.lane >> 4; b < kb; b += team.size >> 4) {
            *reinterpret_cast<uint2 *>(codes + b * pad * BLOCK8 + piece_at(s, sub >> 1) + (sub & 1) * 8) = make_uint2(0, 0);
            if (sub == 0) scales[b * pad + s] = 0.f;
        }
    }
}

// y[t] = sum of w[e] * z[slot(e)]. The rows of up to N entries are on their way together.
template <typename T, int V>
__global__ void __launch_bounds__(NT) k_unsort_rows(Order o, int tpr, const float *w, const T *z, int64_t stride, T *y, int64_t y_stride, int64_t cols) {
    constexpr int N = 4;
    wait_for_previous();
    trigger_dependents();
    const Team team(tpr);
    for (int t = team.first; t < o.tokens; t += team.step) {
        const int e0 = o.entry_of(t), e1 = o.entry_of(t + 1);
        for (int64_t c = team.lane * V; c < cols; c += team.size * V) {
            float sum[V];
#pragma unroll
            for (int j = 0; j < V; ++j) sum[j] = 0.f;
            for (int e = e0; e < e1; e += N) {
                Vec<T, V> v[N];
                int s[N];
                float g[N];
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    s[i] = e + i < e1 ? o.slot(e + i) : -1;
                    g[i] = s[i] >= 0 && w ? ld_late(w + e + i) : 1.f;
                }
#pragma unroll
                for (int i = 0; i < N; ++i)
                    if (s[i] >= 0) v[i] = *reinterpret_cast<const Vec<T, V> *>(z + s[i] * stride + c);
#pragma unroll
                for (int i = 0; i < N; ++i)
                    if (s[i] >= 0) {
#pragma unroll
                        for (int j = 0; j < V; ++j) sum[j] = __fmaf_rn(g[i], to_float(v[i].v[j]), sum[j]);
                    }
            }
            Vec<T, V> out;
#pragma unroll
            for (int j = 0; j < V; ++j) out.v[j] = from_float<T>(sum[j]);
            *reinterpret_cast<Vec<T, V> *>(y + t * y_stride + c) = out;
        }
    }
}

// dz[slot(e)] = w[e] * dy[t] and dw[e] = <dy[t], z[slot(e)]>, N entries of a token at a time. Sums over the columns: every thread its own,
// then the team's, in a fixed order.
template <typename T, int V>
__global__ void __launch_bounds__(NT) k_unsort_grad(Order o, int tpr, const float *w, const T *z, int64_t z_stride, const T *dy, int64_t dy_stride, T *dz, float *dw,
                                                    int64_t cols) {
    constexpr int N = 4;
    __shared__ float part[NT / 32][N];
    wait_for_previous();
    trigger_dependents();
    const Team team(tpr);
    // All threads of a CTA take the same number of rounds, since teams of several warps meet at barriers.
    for (int t0 = team.first - (int)threadIdx.x / tpr; t0 < o.tokens; t0 += team.step) {
        const int t = t0 + (int)threadIdx.x / tpr;
        const bool there = t < o.tokens;
        const int e0 = there ? o.entry_of(t) : 0, e1 = there ? o.entry_of(t + 1) : 0;
        for (int e = e0; __syncthreads_or(e < e1); e += N) {
            float dot[N];
            int s[N];
            float g[N];
#pragma unroll
            for (int i = 0; i < N; ++i) {
                dot[i] = 0.f;
                s[i] = e + i < e1 ? o.slot(e + i) : -1;
                g[i] = s[i] >= 0 ? ld_late(w + e + i) : 0.f;
            }
            if (e < e1)
                for (int64_t c = team.lane * V; c < cols; c += team.size * V) {
                    const Vec<T, V> d = *reinterpret_cast<const Vec<T, V> *>(dy + t * dy_stride + c);
                    Vec<T, V> v[N];
#pragma unroll
                    for (int i = 0; i < N; ++i)
                        if (s[i] >= 0) v[i] = *reinterpret_cast<const Vec<T, V> *>(z + s[i] * z_stride + c);
#pragma unroll
                    for (int i = 0; i < N; ++i)
                        if (s[i] >= 0) {
                            Vec<T, V> out;
#pragma unroll
                            for (int j = 0; j < V; ++j) {
                                dot[i] = __fmaf_rn(to_float(d.v[j]), to_float(v[i].v[j]), dot[i]);
                                out.v[j] = from_float<T>(g[i] * to_float(d.v[j]));
                            }
                            *reinterpret_cast<Vec<T, V> *>(dz + s[i] * cols + c) = out;
                        }
                }
#pragma unroll
            for (int i = 0; i < N; ++i)
                for (int d = 16; d; d >>= 1) dot[i] += __shfl_xor_sync(FULL_MASK, dot[i], d);
            if (tpr > 32) {
                if (lane_id() == 0)
#pragma unroll
                    for (int i = 0; i < N; ++i) part[warp_id()][i] = dot[i];
                __syncthreads();
                if (team.lane == 0)
#pragma unroll
                    for (int i = 0; i < N; ++i) {
                        dot[i] = 0.f;
                        for (int v = 0; v < tpr / 32; ++v) dot[i] += part[warp_id() + v][i];
                    }
            }
            if (team.lane == 0)
#pragma unroll
                for (int i = 0; i < N; ++i)
                    if (e + i < e1) dw[e + i] = s[i] >= 0 ? dot[i] : 0.f;
        }
    }
    Order tail = o;
    tail.rows = nullptr;
    clear_rows<T, V>(tail, team, cols, dz);
    // entries of no row: views into larger arrays
    const int lo = o.entry_of(0), hi = o.entry_of(o.tokens);
    for (int e = blockIdx.x * NT + threadIdx.x; e < o.entries; e += gridDim.x * NT)
        if (e < lo || e >= hi) dw[e] = 0.f;
}

// ---- host ------------------------------------------------------------------------------

// Threads per token for rows of `words` loads: one load each, whole warps from 32 on.
int team_of(int64_t words) {
    int t = 32;
    while (t < NT && t < words) t *= 2;
    return t;
}

dim3 grid_of(int64_t teams, int tpr) {
    const int64_t ctas = (teams * tpr + NT - 1) / NT;
    return dim3((unsigned)std::max<int64_t>(1, std::min<int64_t>(ctas, (int64_t)sm_count() * 64)));
}

int check_order(const nb200_expert_order *o, bool slots_given) {
    if (!o || o->tokens < 0 || o->experts < 0 || o->entries < 0 || !o->row_ptr || !o->offsets) return NB200_E_BADARG;
    if (o->entries > 0 && (!o->slots || (!slots_given && !o->rows))) return NB200_E_BADARG;
    return o->experts > NB200_MAX_EXPERTS ? NB200_E_UNSUPPORTED : NB200_OK;
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

int make_order(const Order &o, cudaStream_t stream) {
    int tile = 2048;  // a multiple of the warps' 32 each
    while ((o.entries + (int64_t)tile - 1) / tile > MAX_TILES) tile *= 2;
    const int tiles = std::max(1, (o.entries + tile - 1) / tile);
    Workspace *ws = nullptr;
    int st;
    if ((st = acquire_workspace(stream, sizeof(int32_t) * (size_t)tiles * std::max(o.experts, 1), &ws, ORDER_SLOT))) return st;
    int32_t *counts = static_cast<int32_t *>(ws->dev);
    const size_t count_smem = sizeof(int32_t) * o.experts, place_smem = sizeof(int32_t) * o.experts * (NT / 32 + 1);
    if (place_smem > 48 * 1024) NB200_CUDA(cudaFuncSetAttribute(k_order_place, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)place_smem));
    {
        LaunchScope scope("order_count", stream);
        NB200_CUDA(launch_overlapped(k_order_count, dim3(tiles), dim3(NT), count_smem, stream, o, tile, tiles, counts));
    }
    LaunchScope scope("order_place", stream);
    NB200_CUDA(launch_overlapped(k_order_place, dim3(tiles), dim3(NT), place_smem, stream, o, tile, tiles, counts));
    return NB200_OK;
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
    if ((st = make_order(o, stream))) return st;
    const nb200_dense none{r->rows, 0, 0, NB200_F32, nullptr};
    if (!x) x = &none, xs = const_cast<nb200_dense *>(&none);
    const int word = word_bytes({x, xs}), tpr = team_of(x->cols * type_size(x->type) / word / 4);
    return with_type(x->type, [&](auto e) {
        using T = decltype(e);
        return with_vector<T>(word, [&](auto v) {
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
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    const Order o = order_of(order, r->col);
    if ((st = make_order(o, stream))) return st;
    const int word = word_bytes({x}), tpr = team_of(blocks_of(x->cols) * 16);
    return with_type(x->type, [&](auto e) {
        using T = decltype(e);
        return with_vector<T>(word, [&](auto v) {
            LaunchScope scope("sort_rows_fp8", stream);
            NB200_CUDA(launch_overlapped(k_sort_rows_fp8<T, decltype(v)::value>, grid_of(o.tokens, tpr), dim3(NT), 0, stream, o, tpr, static_cast<const T *>(x->data), x->stride,
                                         x->cols, xs->values, xs->scales));
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
    const int word = word_bytes({z, y}), tpr = team_of(z->cols * type_size(z->type) / word);
    return with_type(z->type, [&](auto e) {
        using T = decltype(e);
        return with_vector<T>(word, [&](auto v) {
            LaunchScope scope("unsort_rows", stream);
            NB200_CUDA(launch_overlapped(k_unsort_rows<T, decltype(v)::value>, grid_of(o.tokens, tpr), dim3(NT), 0, stream, o, tpr, w, static_cast<const T *>(z->data), z->stride,
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
    const int word = word_bytes({z, dy, dz}), tpr = team_of(z->cols * type_size(z->type) / word);
    return with_type(z->type, [&](auto e) {
        using T = decltype(e);
        return with_vector<T>(word, [&](auto v) {
            LaunchScope scope("unsort_grad", stream);
            NB200_CUDA(launch_overlapped(k_unsort_grad<T, decltype(v)::value>, grid_of(std::max<int64_t>(o.tokens, 1), tpr), dim3(NT), 0, stream, o, tpr, w,
                                         static_cast<const T *>(z->data), z->stride, static_cast<const T *>(dy->data), dy->stride, static_cast<T *>(dz->data), dw, z->cols));
            return (int)NB200_OK;
        });
    });
}

}  // extern "C"
