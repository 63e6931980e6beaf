// The gated half of a feed-forward layer, dense or by expert, in 16 bits with 32-bit sums:
//     g = x Wg^T, u = x Wu^T, h = act(g) u,
// both products, the activation and their product in one kernel, and its gradients
//     dg = dh u act'(g), du = dh act(g), dx = dg Wg + du Wu, dWg = dg^T x, dWu = du^T x.
#include "few_rows.cuh"
#include "tile_product.cuh"

namespace nb200 {
namespace {

constexpr int NT = 256;

// Rows at a distance that the copy engine takes, of up to two matrices: `first` CTAs have the first one's. A thread has 16 bytes of a row where rows lie on boundaries of four.
struct Align {
    const void *x;
    int64_t stride, rows, cols;
    void *z;
    int64_t pitch;
};
template <typename T, int V>
__global__ void __launch_bounds__(NT) k_align_rows(const Align a, const Align b, int first, bool beside) {
    // beside the kernel in front, which has waited for what is read here
    if (!beside) wait_for_previous();
    trigger_dependents();
    const bool second = (int)blockIdx.x >= first;
    const Align &m = second ? b : a;
    const int64_t cta = blockIdx.x - (second ? first : 0), ctas = second ? gridDim.x - first : first;
    if constexpr (V == 1) {
        // rows on no boundary: a warp has 128 elements of a row at a time, TURNS of them on their way
        constexpr int TURNS = 4;
        const int64_t per_row = (m.pitch + 127) / 128, all = m.rows * per_row, step = ctas * (NT / 32);
        for (int64_t i = cta * (NT / 32) + warp_id(); i < all; i += TURNS * step) {
            Four<T> raw[TURNS];
            auto place = [&](int u, int64_t *r) {
                const int64_t at = i + u * step < all ? i + u * step : i;
                *r = at / per_row;
                return (uint32_t)(at - *r * per_row) * 128 + lane_id() * 4;
            };
            int64_t r;
#pragma unroll
            for (int u = 0; u < TURNS; ++u) {
                const uint32_t c = place(u, &r);
                raw[u].load(static_cast<const T *>(m.x) + r * m.stride, c, (uint32_t)m.cols);
            }
#pragma unroll
            for (int u = 0; u < TURNS; ++u) {
                const uint32_t c = place(u, &r);
                float v[4];
                raw[u].get(static_cast<const T *>(m.x) + r * m.stride, v);
                if (i + u * step < all && c < m.pitch) *reinterpret_cast<uint2 *>(static_cast<T *>(m.z) + r * m.pitch + c) = make_uint2(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]));
            }
        }
    } else {
        const int64_t pieces = m.pitch / 8, all = m.rows * pieces, step = ctas * NT;
        for (int64_t i = cta * NT + threadIdx.x; i < all; i += step) {
            const int64_t r = i / pieces, c = (i - r * pieces) * 8;
            Eight<T> v;
            v.template load<V>(static_cast<const T *>(m.x) + r * m.stride, c, m.cols);
            *reinterpret_cast<uint4 *>(static_cast<T *>(m.z) + r * m.pitch + c) = make_uint4(v.w[0], v.w[1], v.w[2], v.w[3]);
        }
    }
    if (beside) finish_after_previous();
}

// [dg du] of one element, from dh and [g u].
__device__ __forceinline__ void gate_grad(float d, float g, float u, bool gelu, float *dg, float *du) {
    float rest;  // the logistic function of -|p(g)|, s that of p(g)
    const float s = logistic(act_inner(g, gelu), &rest), slope = rest * (1.f - rest);  // s (1 - s)
    const float more = slope == 0.f ? 0.f : g * slope * (gelu ? __fmaf_rn(3.f * GELU3 * g, g, GELU1) : 1.f);
    *dg = d * u * (s + more);
    *du = d * (g * s);
}

// dboth = [dg du], rounded to 16 bits for the tensor cores: each element is off by half a step of the type at most, before the products, and so are the gradients once more behind them.
// Both together are 1.4 times as far from 64 bits as gradients that are rounded once (bfloat16 0.0023 of the root of the squares' mean and 0.0017, float16 0.00029 and 0.00021). Kept
// whole, dboth would have to be multiplied in two parts, twice the operations. Device memory bounds it (16384 rows of 2048: 336 MB in 56 to 59 us, 0.9 of a copy) where rows are read in
// words of 16 bytes, which are kept whole.
template <typename T, int V>
__global__ void __launch_bounds__(NT) k_gate_grad(const T *dh, int64_t dh_stride, const T *both, int64_t both_stride, int64_t rows, int64_t hidden, bool gelu, T *z, int64_t pitch) {
    wait_for_previous();
    trigger_dependents();
    // a warp has 32 chunks of 16 bytes of a row at a time, whose words its threads take in turn
    constexpr int N = Chunk<T, V>::N, p = 32 * V;
    const int64_t per_row = (hidden + 32 * N - 1) / (32 * N), all = rows * per_row;
    for (int64_t i = (int64_t)blockIdx.x * (NT / 32) + warp_id(); i < all; i += (int64_t)gridDim.x * (NT / 32)) {
        const int64_t r = i / per_row, c = (i - r * per_row) * (32 * N) + lane_id() * V;
        if (c >= hidden) continue;
        const T *const from_d = dh + r * dh_stride, *const from_g = both + r * both_stride, *const from_u = from_g + hidden;
        T *const to_g = z + r * pitch, *const to_u = to_g + hidden;
        if constexpr (V == 8) {
            Eight<T> d, g, u;
            d.template load<8>(from_d, c, hidden), g.template load<8>(from_g, c, hidden), u.template load<8>(from_u, c, hidden);
            uint32_t a[4], b[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                float dg[2], du[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) gate_grad(d.get(2 * k + e), g.get(2 * k + e), u.get(2 * k + e), gelu, &dg[e], &du[e]);
                a[k] = pack2<T>(dg[0], dg[1]), b[k] = pack2<T>(du[0], du[1]);
            }
            *reinterpret_cast<uint4 *>(to_g + c) = make_uint4(a[0], a[1], a[2], a[3]);
            *reinterpret_cast<uint4 *>(to_u + c) = make_uint4(b[0], b[1], b[2], b[3]);
        } else {
            Chunk<T, V> d, g, u, dg, du;
            d.load(from_d, c, p, hidden), g.load(from_g, c, p, hidden), u.load(from_u, c, p, hidden);
#pragma unroll
            for (int k = 0; k < N; ++k) {
                if (!Chunk<T, V>::there(k, c, p, hidden)) continue;
                float a, b;
                gate_grad(d.get(k), g.get(k), u.get(k), gelu, &a, &b);
                dg.set(k, a), du.set(k, b);
            }
            dg.store(to_g, c, p, hidden), du.store(to_u, c, p, hidden);
        }
    }
}

unsigned grid_of(int64_t threads) { return (unsigned)std::max<int64_t>(1, std::min<int64_t>((threads + NT - 1) / NT, sm_count() * 16ll)); }

int64_t pitch_of(int64_t cols) { return (cols + 7) / 8 * 8; }

bool act_ok(int32_t activation) { return activation == NB200_SILU || activation == NB200_GELU; }
bool operands_ok(const nb200_dense *x, const nb200_dense *w, int32_t groups, const int32_t *offsets) {
    return dense_ok(x) && dense_ok(w) && x->type != NB200_F32 && x->type == w->type && groups >= 0 && x->cols == w->cols && (offsets || groups == 1) &&
           (groups == 0 ? w->rows == 0 : w->rows % groups == 0 && w->rows / groups % 2 == 0);
}

template <typename F>
int with_half(int type, F f) {
    return type == NB200_F16 ? f(__half{}) : f(__nv_bfloat16{});
}
template <typename T>
constexpr Sum sum_of = std::is_same<T, __half>::value ? Sum::F16 : Sum::BF16;

// Rows and weights as the copy engine reads them: as they are, or copied to where there is room.
int aligned(const nb200_dense &x, void *to_x, const nb200_dense &w, void *to_w, nb200_dense *ax, nb200_dense *aw, bool beside, cudaStream_t stream) {
    *ax = x, *aw = w;
    Align copies[2] = {};
    int n = 0, word = 16;
    int64_t ctas[2] = {0, 0};
    auto add = [&](const nb200_dense &from, void *to, nb200_dense *z) {
        if (!to) return;
        z->data = to, z->stride = pitch_of(from.cols);
        copies[n] = Align{from.data, from.stride, from.rows, from.cols, to, z->stride};
        ctas[n++] = grid_of(from.rows * (z->stride / 8));
        word = std::min(word, word_bytes({&from}));
    };
    add(x, to_x, ax);
    add(w, to_w, aw);
    if (n == 0) return NB200_OK;
    return with_half(x.type, [&](auto e) {
        using T = decltype(e);
        return with_vector<T>(word, [&](auto v) {
            LaunchScope scope("align_rows", stream);
            NB200_CUDA(launch_overlapped(k_align_rows<T, decltype(v)::value>, dim3((unsigned)(ctas[0] + ctas[1])), dim3(NT), 0, stream, copies[0], copies[1], (int)ctas[0], beside));
            return (int)NB200_OK;
        });
    });
}

bool few(const nb200_dense *x, const nb200_dense *w, int64_t groups) { return few_rows(x->rows, groups, w->rows * w->cols * 2, 2); }

struct ForwardScratch {
    uint8_t *x = nullptr, *w = nullptr;
    size_t bytes = 0;

    ForwardScratch(void *base, const nb200_dense *xx, const nb200_dense *ww, int64_t groups) {
        if (few(xx, ww, groups)) return;
        Carver c(base);
        if (!tiles_readable(*xx, 1)) x = c.take<uint8_t>((size_t)(xx->rows * pitch_of(xx->cols)) * 2);
        if (!tiles_readable(*ww, groups)) w = c.take<uint8_t>((size_t)(ww->rows * pitch_of(ww->cols)) * 2);
        bytes = c.used();
    }
};

struct GradScratch {
    uint8_t *d, *x = nullptr, *w = nullptr;
    size_t bytes;

    GradScratch(void *base, const nb200_dense *xx, const nb200_dense *ww, int64_t groups) {
        Carver c(base);
        d = c.take<uint8_t>((size_t)(xx->rows * pitch_of(groups ? ww->rows / groups : 0)) * 2);
        if (!tiles_readable(*xx, 1)) x = c.take<uint8_t>((size_t)(xx->rows * pitch_of(xx->cols)) * 2);
        if (!tiles_readable(*ww, groups)) w = c.take<uint8_t>((size_t)(ww->rows * pitch_of(ww->cols)) * 2);
        bytes = c.used();
    }
};

// The two products of the gradient, which do not wait for one another: with all pairs of CTAs each, or, where their tiles would leave many of them idle, rows' gradient with the pairs
// that it needs and the weights' with the rest, as far as that keeps up (128 rows of 4096 x 4096: one after the other 48 us, beside one another 39; 1003 rows by 1101 hidden units and a
// width of 1100: 37 and 27; 14 rows of 4992 x 768: the weights' gradient on all 62 pairs that are left 21.5 us, on 20 to 40 of them, beside which the next kernel's CTAs find room, 18.7).
// Tiles wait for their results to leave, where they sum little for longer than for their blocks, and longest where warps store them (`words` false). The constants, in rows of blocks, are
// those by which the plans of 200 products, of one row to some ten thousand, come nearest to the best of some twenty plans that were measured for each: 1.8 % on the mean.
struct GradPlan {
    static constexpr int64_t RESULTS_X = 1280, ODD_RESULTS_X = 4096, RESULTS_W = 1536, ODD_RESULTS_W = 6144, LAUNCH = 8000;  // for a tile; for a kernel that follows another
    TileWork::Way x, w;
    int pairs_x, pairs_w;

    GradPlan(int64_t rows, int64_t width, int64_t hidden, int64_t groups, bool words, const int (&clusters)[2]) {
        const int64_t high = (2 * hidden + TILE_M - 1) / TILE_M, all = all_pairs();
        const TileWork work_x{rows, groups, (width + TILE_M - 1) / TILE_M, (2 * hidden + 63) / 64, words ? RESULTS_X : ODD_RESULTS_X};
        const TileWork work_w{width, 1, groups * high, ((rows + groups - 1) / groups + 63) / 64, words ? RESULTS_W : ODD_RESULTS_W};
        x = work_x.best(all, clusters), w = work_w.best(all, clusters);
        pairs_x = pairs_w = (int)all;
        double least = (x.cost + w.cost) * 15 / 16 + LAUNCH;  // the shares of the pairs do not change on the way: they have to give more than a little
        for (int k = 1; k < 8; ++k) {
            const int64_t part = all * k / 8;
            if (part < 1 || part >= all) continue;
            // clusters have to find room beside the other product's CTAs
            const int half[2] = {clusters[0] * k / 8, clusters[1] * k / 8};
            const TileWork::Way a = work_x.best(part, half);
            const int64_t mine = std::min(part, work_x.most(a.n) * a.parts), other = all - mine;
            const int rest[2] = {(int)(clusters[0] * other / all) - 1, (int)(clusters[1] * other / all) - 1};
            const TileWork::Way b = work_w.best(other, rest);
            if (std::max(a.cost, b.cost) >= least) continue;
            least = std::max(a.cost, b.cost), x = a, w = b, pairs_x = (int)mine, pairs_w = (int)other;
            if (a.parts > 1 && b.parts == 1 && b.cost < a.cost) {
                // beside clusters in as many rounds as three quarters of their time hold
                const int64_t tiles = work_w.most(b.n), now = (tiles + other - 1) / other, rounds = std::max(now, (int64_t)(a.cost * 3 / 4 * now / b.cost));
                pairs_w = (int)((tiles + rounds - 1) / rounds);
            }
        }
    }
};

int zeros(const nb200_dense &y, cudaStream_t stream) {
    if (y.rows == 0 || y.cols == 0) return NB200_OK;
    const size_t size = type_size(y.type);
    NB200_CUDA(cudaMemset2DAsync(y.data, (size_t)(y.rows > 1 ? y.stride : y.cols) * size, 0, (size_t)y.cols * size, (size_t)y.rows, stream));
    return NB200_OK;
}

}  // namespace
}  // namespace nb200

using namespace nb200;

extern "C" {

int64_t nb200_gated_product_scratch(const nb200_dense *x, const nb200_dense *w, int32_t groups) {
    if (!dense_ok(x) || !dense_ok(w) || groups < 0) return -1;
    return (int64_t)ForwardScratch(nullptr, x, w, groups).bytes;
}

int nb200_gated_product(const nb200_dense *x, const nb200_dense *w, int32_t groups, const int32_t *offsets, int32_t activation, nb200_dense *h, nb200_dense *both, void *scratch,
                        int64_t scratch_bytes, void *stream_) {
    if (!operands_ok(x, w, groups, offsets) || !act_ok(activation) || !dense_ok(h) || h->rows != x->rows || h->type != x->type) return NB200_E_BADARG;
    const int64_t hidden = groups ? w->rows / groups / 2 : h->cols;
    if (h->cols != hidden || (both && (!dense_ok(both) || both->rows != x->rows || both->cols != 2 * hidden || both->type != x->type || (both->rows > 1 && both->stride != both->cols))))
        return NB200_E_BADARG;
    if (groups > NB200_MAX_EXPERTS || hidden > INT32_MAX / 2 - 1024 || x->rows > INT32_MAX - 1024 || x->cols > INT32_MAX - 1024) return NB200_E_UNSUPPORTED;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    if (x->rows == 0 || hidden == 0) return NB200_OK;
    int st;
    if (groups == 0 || x->cols == 0) {
        if ((st = zeros(*h, stream)) || (both && (st = zeros(*both, stream)))) return st;
        return NB200_OK;
    }
    const bool gelu = activation == NB200_GELU;
    if (few(x, w, groups)) {
        const FewArgs args{x->data, w->data, x->rows > 1 ? x->stride : x->cols, w->rows > 1 ? w->stride : w->cols, offsets, groups, (int)x->rows, (int)hidden, 16, (int)x->cols, h->data,
                           both ? both->data : nullptr, h->rows > 1 ? h->stride : h->cols, nullptr, nullptr, gelu};
        return with_half(x->type, [&](auto e) {
            using T = decltype(e);
            return with_vector<T>(word_bytes({x, w}), [&](auto v) { return launch_few_rows<sum_of<T>, true, decltype(v)::value, T>("gated_few", args, stream); });
        });
    }
    const ForwardScratch s(scratch, x, w, groups);
    if (s.bytes && (!scratch || reinterpret_cast<uintptr_t>(scratch) % 256 != 0)) return NB200_E_BADARG;
    if (scratch_bytes < (int64_t)s.bytes) return NB200_E_CAPACITY;
    nb200_dense ax, aw;
    if ((st = aligned(*x, s.x, *w, s.w, &ax, &aw, false, stream))) return st;
    TileMaps maps{};
    TileArgs args{};
    int clusters[2];
    if ((st = with_half(x->type, [&](auto e) { return tile_clusters<sum_of<decltype(e)>, Form::GATED, false, decltype(e)>(clusters); }))) return st;
    args.offsets = offsets, args.groups = groups, args.rows = (int)x->rows, args.wide = (int)hidden, args.blocks = (int)((x->cols + 63) / 64);
    args.pairs = (int)all_pairs();
    const TileWork::Way way = TileWork{x->rows, groups, (hidden + TILE_M / 2 - 1) / (TILE_M / 2), args.blocks}.best(args.pairs, clusters);
    args.tile_n = way.n, args.parts = way.parts;
    // Sixteen rows of gates and sixteen of values in turn: as one box where the hidden units are sixteens, else by boxes of 16 rows.
    args.whole_wide = hidden % 16 == 0;
    if (args.whole_wide) {
        const cuuint64_t pitch = (cuuint64_t)(w->rows > 1 ? aw.stride : pitch_of(w->cols)) * 2;
        const cuuint64_t extents[5] = {(cuuint64_t)w->cols, 16, 2, (cuuint64_t)hidden / 16, (cuuint64_t)groups}, pitches[4] = {pitch, pitch * hidden, pitch * 16, pitch * 2 * hidden};
        const cuuint32_t box[5] = {64, 16, 2, 4, 1};
        st = encode_matrix(&maps.wide, map_type(w->type), 5, aw.data, extents, pitches, box);
    } else {
        st = describe_rows(&maps.wide, map_type(w->type), aw.data, 2, w->cols, 2 * hidden, groups, aw.stride, 16);
    }
    if (st || (st = describe_narrow(&maps, &args, map_type(x->type), ax.data, 2, x->cols, x->rows, ax.stride)) || (st = describe_result(&maps.y, &args.words, map_type(x->type), *h, 1))) return st;
    if (both) {
        args.words = args.words && word_bytes({both}) == 16;
        // gates and values as two matrices, so that a tile of one ends where the other begins
        const cuuint64_t extents[3] = {(cuuint64_t)hidden, 2, (cuuint64_t)x->rows}, pitches[2] = {(cuuint64_t)hidden * 2, (cuuint64_t)hidden * 4};
        const cuuint32_t box[3] = {64, 1, 32};
        if (args.words && (st = encode_matrix(&maps.both, map_type(x->type), 3, both->data, extents, pitches, box))) return st;
    }
    args.y = h->data, args.stride = h->rows > 1 ? h->stride : h->cols, args.both = both ? both->data : nullptr, args.gelu = gelu;
    return with_half(x->type, [&](auto e) {
        using T = decltype(e);
        return launch_tiles<sum_of<T>, Form::GATED, false, T>("gated_product", args, maps, stream);
    });
}

int64_t nb200_gated_product_grad_scratch(const nb200_dense *x, const nb200_dense *w, int32_t groups) {
    if (!dense_ok(x) || !dense_ok(w) || groups < 0) return -1;
    return (int64_t)GradScratch(nullptr, x, w, groups).bytes;
}

int nb200_gated_product_grad(const nb200_dense *dh, const nb200_dense *both, const nb200_dense *x, const nb200_dense *w, int32_t groups, const int32_t *offsets, int32_t activation,
                             nb200_dense *dx, nb200_dense *dw, void *scratch, int64_t scratch_bytes, void *stream_) {
    if (!operands_ok(x, w, groups, offsets) || !act_ok(activation) || !dense_ok(dh) || !dense_ok(both) || !dense_ok(dx) || !dense_ok(dw)) return NB200_E_BADARG;
    const int type = x->type;
    const int64_t hidden = groups ? w->rows / groups / 2 : dh->cols;
    if (dh->type != type || both->type != type || dx->type != type || dw->type != type || dh->rows != x->rows || both->rows != x->rows || dh->cols != hidden || both->cols != 2 * hidden ||
        dx->rows != x->rows || dx->cols != x->cols || dw->rows != w->rows || dw->cols != w->cols)
        return NB200_E_BADARG;
    if (groups > NB200_MAX_EXPERTS || hidden > INT32_MAX / 2 - 1024 || x->rows > INT32_MAX - 1024 || x->cols > INT32_MAX / 2 - 1024) return NB200_E_UNSUPPORTED;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    int st;
    if (x->cols == 0) return NB200_OK;
    if (x->rows == 0 || hidden == 0 || groups == 0) {
        if ((st = zeros(*dx, stream)) || (st = zeros(*dw, stream))) return st;
        return NB200_OK;
    }
    const GradScratch s(scratch, x, w, groups);
    if (!scratch || reinterpret_cast<uintptr_t>(scratch) % 256 != 0) return NB200_E_BADARG;
    if (scratch_bytes < (int64_t)s.bytes) return NB200_E_CAPACITY;
    const int64_t pitch = pitch_of(2 * hidden);
    const bool gelu = activation == NB200_GELU;
    // du begins `hidden` elements behind dg, and so does u behind g
    nb200_dense half = *both;
    half.cols = hidden, half.data = static_cast<uint8_t *>(both->data) + hidden * 2;
    nb200_dense to{x->rows, hidden, pitch, type, s.d + hidden * 2};
    return with_half(type, [&](auto e) -> int {
        using T = decltype(e);
        st = with_vector<T>(word_bytes({dh, both, &half, &to}), [&](auto v) {
            constexpr int V = decltype(v)::value;
            LaunchScope scope("gate_grad", stream);
            NB200_CUDA(launch_overlapped(k_gate_grad<T, V>, dim3(grid_of(x->rows * ((hidden + 255) / 256) * 32)), dim3(NT), 0, stream, static_cast<const T *>(dh->data), dh->stride,
                                         static_cast<const T *>(both->data), both->stride, x->rows, hidden, gelu, reinterpret_cast<T *>(s.d), pitch));
            return (int)NB200_OK;
        });
        if (st) return st;
        // Copies for the copy engine are made beside that kernel, and the weights' gradient beside the other one: neither has anything from the kernel in front.
        nb200_dense ax, aw;
        if ((st = aligned(*x, s.x, *w, s.w, &ax, &aw, true, stream))) return st;
        int clusters[2];
        if ((st = tile_clusters<sum_of<T>, Form::WEIGHTS, true, T>(clusters))) return st;
        const GradPlan plan(x->rows, x->cols, hidden, groups, word_bytes({dw}) == 16, clusters);
        TileMaps maps{};
        TileArgs args{};
        args.offsets = offsets, args.groups = groups, args.rows = (int)x->rows;
        // dx: the weights' columns on the wide side
        args.wide = (int)x->cols, args.blocks = (int)((2 * hidden + 63) / 64), args.tile_n = plan.x.n, args.parts = plan.x.parts, args.pairs = plan.pairs_x;
        args.y = dx->data, args.stride = dx->rows > 1 ? dx->stride : dx->cols;
        if ((st = describe_turned(&maps.wide, &args.whole_wide, map_type(type), aw.data, w->cols, 2 * hidden, groups, aw.stride, 2)) ||
            (!args.whole_wide && (st = describe_rows(&maps.wide, map_type(type), aw.data, 2, w->cols, 2 * hidden, groups, aw.stride, 64))) ||
            (st = describe_narrow(&maps, &args, map_type(type), s.d, 2, 2 * hidden, x->rows, pitch)) || (st = describe_result(&maps.y, &args.words, map_type(type), *dx, 1)))
            return st;
        if ((st = launch_tiles<sum_of<T>, Form::ROWS, true, T>("gated_grad_x", args, maps, stream))) return st;
        // dw: both operands turned
        args.beside = true;
        args.wide = (int)(2 * hidden), args.across = (int)x->cols, args.tile_n = plan.w.n, args.parts = plan.w.parts, args.pairs = plan.pairs_w;
        args.y = dw->data, args.stride = dw->rows > 1 ? dw->stride : dw->cols;
        if ((st = describe_turned(&maps.wide, &args.whole_wide, map_type(type), s.d, 2 * hidden, x->rows, 1, pitch, 2)) ||
            (!args.whole_wide && (st = describe_rows(&maps.wide, map_type(type), s.d, 2, 2 * hidden, x->rows, 1, pitch, 64))) ||
            (st = describe_rows(&maps.narrow, map_type(type), ax.data, 2, x->cols, x->rows, 1, ax.stride, 64)) ||
            (st = describe_turned(&maps.narrow_whole, &args.whole_narrow, map_type(type), ax.data, x->cols, x->rows, 1, ax.stride, args.tile_n % 128 == 0 ? args.tile_n / 128 : 0)) ||
            (st = describe_result(&maps.y, &args.words, map_type(type), *dw, groups)))
            return st;
        return launch_tiles<sum_of<T>, Form::WEIGHTS, true, T>("gated_grad_w", args, maps, stream);
    });
}

}  // extern "C"
