// The addition to the residual stream with its RMS norm, and its pullback.
//
//   forward    s = hidden + residual,   y = s * rsqrt(mean(s^2) + eps) * weight
//   pullback   i = rsqrt(mean(s^2) + eps), u = s i, p = g_y * weight:   g_s = i (p - u mean(u p)) + g_s',   g_weight = sum over rows of g_y u
//
// Everything between load and store is fp32, the sum that the norm sees included: it is rounded only where it is stored.  y comes in the
// type of `hidden`, or in 8 bits (e4m3) with one scale a row, max|y| / 448.
//
// Bound by memory: a row is read once and kept in registers, eight neighbouring elements a lane and piece, by as many lanes (8 ... 1024) as
// hold it in one or two pieces: few registers a lane leave room for the waves that hide the loads.  Pieces are loaded at any alignment (an
// element's own is enough); one that runs past the end of its row goes element by element, so every width takes the same kernel.
// Forward 5003 x 8192 in bf16 with 8-bit output: 55 us, 5.2 TB/s; 8192 x 768 in bf16 with an fp32 stream 13 ... 14 us, 5.3 ... 5.8 TB/s, part of it
// from the cache, and backwards 20.5 us, 4.9 TB/s, and 4 for the fold of the weight's gradient.  One row: 2.4 us.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "lbi_block_rows.h"

namespace lbi {
namespace block_norm {
namespace {

// NT threads a row (beyond 64: up to NT, the workgroup's), PIECES pieces a lane.  TAIL: D is no whole number of pieces.  Results may be inputs:
// all of a row is read before any of it is written.
template <typename T, typename R, bool SCALED, bool TAIL, int NT, int PIECES>
__global__ __launch_bounds__(NT * SIDE<NT>) void norm_kernel(const T* hidden, const R* residual, const void* __restrict__ weight,
                                                             void* normed, R* stream_out, float* __restrict__ scales, long long rows, int D,
                                                             float eps, int weight_wide) {
    __shared__ float spare[2][NT <= 64 ? 1 : NT / 64];
    const int threads = NT <= 64 ? NT : (int)blockDim.x, t = threadIdx.x % threads;
    const long long row = (long long)blockIdx.x * SIDE<NT> + threadIdx.x / threads;
    if (row >= rows) return;  // all lanes of a row, and with barriers below the row is the workgroup's only one
    Raw<T> h[PIECES];
    Raw<R> r[PIECES];
    Eight s[PIECES], w[PIECES];
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
        const int c = (p * threads + t) * PIECE;
        if (c < D) h[p] = load8<TAIL>(hidden + row * D + c, D - c);
    }
    if (residual)
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            const int c = (p * threads + t) * PIECE;
            if (c < D) r[p] = load8<TAIL>(residual + row * D + c, D - c);
        }
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
        const int c = (p * threads + t) * PIECE;
        if (c < D) w[p] = load_weight<TAIL, T>(weight, c, D - c, weight_wide != 0);
    }
    float sum = 0.0f;
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
        const int c = (p * threads + t) * PIECE;
        if (c >= D) continue;
        s[p] = h[p].wide();
        if (residual) {
            const Eight more = r[p].wide();
#pragma unroll
            for (int e = 0; e < PIECE; ++e) s[p].v[e] += more.v[e];
        }
        if (stream_out) store8<TAIL>(stream_out + row * D + c, s[p], D - c);
#pragma unroll
        for (int e = 0; e < PIECE; ++e) sum = fmaf(s[p].v[e], s[p].v[e], sum);
    }
    const float inv = rsqrtf(over_row<Add, NT>(sum, spare[0]) / (float)D + eps);
    float most = 0.0f;
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
        const int c = (p * threads + t) * PIECE;
        if (c >= D) continue;
#pragma unroll
        for (int e = 0; e < PIECE; ++e) {
            s[p].v[e] = s[p].v[e] * inv * w[p].v[e];
            if (SCALED) most = larger(most, fabsf(s[p].v[e]));
        }
        if (!SCALED) store8<TAIL>(static_cast<T*>(normed) + row * D + c, s[p], D - c);
    }
    if constexpr (SCALED) {
        most = over_row<Larger, NT>(most, spare[1]);
        // a row of zeros has the scale 1; no scale is below the smallest normal number, whose reciprocal is still one
        const float scale = most == 0.0f ? 1.0f : larger(most / E4M3_MOST, SMALLEST_NORMAL), back = 1.0f / scale;
        if (t == 0) scales[row] = scale;
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            const int c = (p * threads + t) * PIECE;
            if (c >= D) continue;
#pragma unroll
            for (int e = 0; e < PIECE; ++e) s[p].v[e] *= back;
            store8_e4m3<TAIL>(static_cast<unsigned char*>(normed) + row * D + c, s[p], D - c);
        }
    }
}

// A workgroup takes the rows of one slab, NT threads a row, and leaves its share of the weight's gradient in `partials` [slabs, D].  The next
// row is on its way while one is worked on; its loads stand in no branch, since the compiler waits for every load under way where branches meet
// (past the end of a row or of the slab they fetch again what is there, and nothing uses it).  MORE: there is a g_stream.  Results may be inputs here too.
template <typename T, typename R, bool MORE, bool TAIL, int NT, int PIECES>
__global__ __launch_bounds__(NT * SIDE<NT>) void norm_pullback_kernel(const T* g_normed, const R* stream, const R* g_stream,
                                                                      const void* __restrict__ weight, T* g_hidden, R* g_residual,
                                                                      float* __restrict__ partials, long long rows, int D, float eps,
                                                                      int weight_wide, int slab) {
    extern __shared__ __align__(16) float lds[];  // SIDE > 1: [SIDE][D]
    __shared__ float spare[2][NT <= 64 ? 1 : NT / 64][2];
    const int threads = NT <= 64 ? NT : (int)blockDim.x, t = threadIdx.x % threads, side = threadIdx.x / threads;
    const long long first = (long long)blockIdx.x * slab, last = first + slab < rows ? first + slab : rows;
    struct Row {
        Raw<R> x[PIECES], more[PIECES];
        Raw<T> g[PIECES];
    };
    auto bring = [&](long long row) __attribute__((always_inline)) {
        Row r;
        const long long from = (row < last ? row : last - 1) * D;
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            const int at = (p * threads + t) * PIECE, c = at < D ? at : 0;
            r.x[p] = load8<TAIL>(stream + from + c, D - c);
            r.g[p] = load8<TAIL>(g_normed + from + c, D - c);
            if constexpr (MORE) r.more[p] = load8<TAIL>(g_stream + from + c, D - c);
        }
        return r;
    };
    constexpr bool AHEAD = NT * PIECES <= 1024;  // the widest rows leave no registers for it
    Row next;
    if constexpr (AHEAD) next = bring(first + side);
    Eight w[PIECES], total[PIECES];
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
        const int c = (p * threads + t) * PIECE;
        if (c < D) w[p] = load_weight<TAIL, T>(weight, c, D - c, weight_wide != 0);
#pragma unroll
        for (int e = 0; e < PIECE; ++e) total[p].v[e] = 0.0f;
    }
    int turn = 0;
    for (long long row = first + side; row < last; row += SIDE<NT>, turn ^= 1) {
        const Row now = AHEAD ? next : bring(row);
        if constexpr (AHEAD) next = bring(row + SIDE<NT>);
        float squares = 0.0f, along = 0.0f;
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            if ((p * threads + t) * PIECE >= D) continue;
            const Eight x = now.x[p].wide(), g = now.g[p].wide();
#pragma unroll
            for (int e = 0; e < PIECE; ++e) {
                squares = fmaf(x.v[e], x.v[e], squares);
                along = fmaf(x.v[e], g.v[e] * w[p].v[e], along);
            }
        }
        sums_over_row<NT>(squares, along, spare[turn]);
        const float inv = rsqrtf(squares / (float)D + eps), mean = along * inv / (float)D;
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            const int c = (p * threads + t) * PIECE;
            if (c >= D) continue;
            const Eight x = now.x[p].wide(), g = now.g[p].wide();
            Eight out, more;
            if constexpr (MORE) more = now.more[p].wide();
#pragma unroll
            for (int e = 0; e < PIECE; ++e) {
                const float unit = x.v[e] * inv;
                total[p].v[e] = fmaf(g.v[e], unit, total[p].v[e]);
                out.v[e] = inv * (g.v[e] * w[p].v[e] - unit * mean);
                if constexpr (MORE) out.v[e] += more.v[e];
            }
            if (g_residual) store8<TAIL>(g_residual + row * D + c, out, D - c);
            if (g_hidden) store8<TAIL>(g_hidden + row * D + c, out, D - c);
        }
    }
    if constexpr (SIDE<NT> > 1) {
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            const int c = (p * threads + t) * PIECE;
            if (c < D) store8<TAIL>(lds + side * D + c, total[p], D - c);
        }
        __syncthreads();
        for (int c = threadIdx.x; c < D; c += 256) {
            float sum = lds[c];
#pragma unroll
            for (int q = 1; q < SIDE<NT>; ++q) sum += lds[q * D + c];
            partials[(size_t)blockIdx.x * D + c] = sum;
        }
    } else {
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            const int c = (p * threads + t) * PIECE;
            if (c < D) store8<TAIL>(partials + (size_t)blockIdx.x * D + c, total[p], D - c);
        }
    }
}

// Slabs of the pullback, and the rows of one: four workgroups a CU of narrow rows, two of wide ones, whose shares of the weight's gradient
// would be as many bytes as a twentieth of the rows themselves.
int slab_rows(int64_t rows, int64_t D) {
    const int64_t slabs = D <= 1024 ? 1024 : 512;
    const int64_t least = D <= 512 ? 2048 / D : 1;  // rows that a workgroup holds side by side, about
    return (int)std::max<int64_t>((rows + slabs - 1) / slabs, least);
}
int slab_count(int64_t rows, int64_t D) { return (int)((rows + slab_rows(rows, D) - 1) / slab_rows(rows, D)); }

int check(const char* who, int64_t rows, int64_t D, int dtype, int stream, int weight) {
    if (rows < 0 || D < 1) return fail(LBI_ERR_INVALID, "%s: bad size (rows=%lld D=%lld)", who, (long long)rows, (long long)D);
    if (!dtype_size(dtype) || (stream != dtype && stream != LBI_F32) || (weight != dtype && weight != LBI_F32))
        return fail(LBI_ERR_INVALID, "%s: bad dtype (%d; residual stream %d and weight %d are of the same or fp32)", who, dtype, stream, weight);
    if (D > MOST_COLUMNS || rows >= MOST_ROWS)
        return fail(LBI_ERR_UNSUPPORTED, "%s: rows of up to %lld columns, fewer than 2^31 of them", who, (long long)MOST_COLUMNS);
    return LBI_OK;
}

}  // namespace
}  // namespace block_norm
}  // namespace lbi

extern "C" int lbi_residual_rmsnorm(const void* hidden, const void* residual, const void* weight, void* normed, void* residual_out,
                                    float* scales, int64_t rows, int64_t D, float eps, int dtype, int residual_dtype, int weight_dtype,
                                    void* stream) {
    using namespace lbi;
    using namespace lbi::block_norm;
    clear_error();
    if (int bad = check("lbi_residual_rmsnorm", rows, D, dtype, residual_dtype, weight_dtype)) return bad;
    if (rows == 0) return LBI_OK;
    if (!hidden || !weight || !normed) return fail(LBI_ERR_INVALID, "lbi_residual_rmsnorm: null pointer");
    if (!aligned(hidden, dtype) || (!scales && !aligned(normed, dtype)) || !aligned(residual, residual_dtype) || !aligned(weight, weight_dtype) ||
        !aligned(residual_out, residual_dtype) || !aligned(scales, LBI_F32))
        return fail(LBI_ERR_INVALID, "lbi_residual_rmsnorm: a tensor is not aligned to its elements");
    const size_t size = dtype_size(dtype), of_stream = dtype_size(residual_dtype);
    const Place y(normed, rows * D, scales ? 1 : size), s(residual_out, rows * D, of_stream);
    for (const Place& in : {Place(hidden, rows * D, size), Place(residual, rows * D, of_stream)})
        if ((y.meets(in) && !y.is(in)) || (s.meets(in) && !s.is(in)) || y.meets(s))
            return fail(LBI_ERR_INVALID, "lbi_residual_rmsnorm: a result overlaps another tensor");
    return by_types(dtype, residual_dtype, [&](auto t, auto r) {
        using T = typename decltype(t)::type;
        using R = typename decltype(r)::type;
        return by_width<false>(D, [&](auto form) {
            constexpr int NT = decltype(form)::NT, PIECES = decltype(form)::PIECES, COUNT = SIDE<NT>;
            const auto kernel = D % PIECE ? (scales ? norm_kernel<T, R, true, true, NT, PIECES> : norm_kernel<T, R, false, true, NT, PIECES>)
                                          : (scales ? norm_kernel<T, R, true, false, NT, PIECES> : norm_kernel<T, R, false, false, NT, PIECES>);
            const int threads = threads_of<NT, PIECES>(D) * COUNT;
            const int64_t most = (MOST_THREADS / threads) * COUNT;  // rows of a launch
            for (int64_t first = 0; first < rows; first += most) {
                const int64_t count = std::min(rows - first, most);
                const auto from = [&](auto* p) { return p ? p + first * D : p; };
                void* y = scales ? static_cast<void*>(from(static_cast<unsigned char*>(normed))) : static_cast<void*>(from(static_cast<T*>(normed)));
                hipLaunchKernelGGL(kernel, dim3((unsigned)((count + COUNT - 1) / COUNT)), dim3((unsigned)threads), 0, static_cast<hipStream_t>(stream),
                                   from(static_cast<const T*>(hidden)), from(static_cast<const R*>(residual)), weight, y,
                                   from(static_cast<R*>(residual_out)), scales ? scales + first : nullptr, (long long)count, (int)D, eps,
                                   (int)(weight_dtype == LBI_F32));
                LBI_HIP_CHECK(hipGetLastError());
            }
            return (int)LBI_OK;
        });
    });
}

extern "C" size_t lbi_residual_rmsnorm_pullback_workspace_bytes(int64_t rows, int64_t D) {
    using namespace lbi::block_norm;
    if (rows < 0 || D < 1 || D > MOST_COLUMNS || rows >= MOST_ROWS) return 0;
    return (size_t)slab_count(rows, D) * (size_t)D * sizeof(float);
}

extern "C" int lbi_residual_rmsnorm_pullback(const void* g_normed, const void* residual_out, const void* g_residual_out, const void* weight,
                                             void* g_hidden, void* g_residual, float* g_weight, void* workspace, size_t workspace_bytes,
                                             int64_t rows, int64_t D, float eps, int dtype, int residual_dtype, int weight_dtype,
                                             void* stream) {
    using namespace lbi;
    using namespace lbi::block_norm;
    clear_error();
    if (int bad = check("lbi_residual_rmsnorm_pullback", rows, D, dtype, residual_dtype, weight_dtype)) return bad;
    if (!g_weight || (rows && (!g_normed || !residual_out || !weight || (!g_hidden && !g_residual))))
        return fail(LBI_ERR_INVALID, "lbi_residual_rmsnorm_pullback: null pointer");
    const int slabs = slab_count(rows, D);
    const size_t need = lbi_residual_rmsnorm_pullback_workspace_bytes(rows, D);
    if (need && (!workspace || workspace_bytes < need))
        return fail(LBI_ERR_WORKSPACE, "lbi_residual_rmsnorm_pullback: workspace of %zu bytes needed, %zu given", need, workspace_bytes);
    if (!aligned(g_normed, dtype) || !aligned(residual_out, residual_dtype) || !aligned(g_residual_out, residual_dtype) ||
        !aligned(weight, weight_dtype) || !aligned(g_hidden, dtype) || !aligned(g_residual, residual_dtype) || !aligned(g_weight, LBI_F32) ||
        !aligned(workspace, LBI_F32))
        return fail(LBI_ERR_INVALID, "lbi_residual_rmsnorm_pullback: a tensor is not aligned to its elements");
    const size_t size = dtype_size(dtype), of_stream = dtype_size(residual_dtype);
    const Place out(g_hidden, rows * D, size), more(g_residual, rows * D, of_stream);
    for (const Place& in : {Place(g_normed, rows * D, size), Place(residual_out, rows * D, of_stream), Place(g_residual_out, rows * D, of_stream)})
        if ((out.meets(in) && !out.is(in)) || (more.meets(in) && !more.is(in)) || (out.meets(more) && !out.is(more)))
            return fail(LBI_ERR_INVALID, "lbi_residual_rmsnorm_pullback: a result overlaps another tensor");
    float* partials = static_cast<float*>(workspace);
    if (rows) {
        const int status = by_types(dtype, residual_dtype, [&](auto t, auto r) {
            using T = typename decltype(t)::type;
            using R = typename decltype(r)::type;
            return by_width<true>(D, [&](auto form) {
                constexpr int NT = decltype(form)::NT, PIECES = decltype(form)::PIECES, COUNT = SIDE<NT>;
                const size_t bytes = COUNT > 1 ? COUNT * (size_t)D * sizeof(float) : 0;  // 16 KiB at most
                const auto kernel = D % PIECE ? (g_residual_out ? norm_pullback_kernel<T, R, true, true, NT, PIECES>
                                                                : norm_pullback_kernel<T, R, false, true, NT, PIECES>)
                                              : (g_residual_out ? norm_pullback_kernel<T, R, true, false, NT, PIECES>
                                                                : norm_pullback_kernel<T, R, false, false, NT, PIECES>);
                hipLaunchKernelGGL(kernel, dim3((unsigned)slabs), dim3((unsigned)(threads_of<NT, PIECES>(D) * COUNT)), bytes,
                                   static_cast<hipStream_t>(stream), static_cast<const T*>(g_normed), static_cast<const R*>(residual_out),
                                   static_cast<const R*>(g_residual_out), weight, static_cast<T*>(g_hidden), static_cast<R*>(g_residual),
                                   partials, (long long)rows, (int)D, eps, (int)(weight_dtype == LBI_F32), slab_rows(rows, D));
                LBI_HIP_CHECK(hipGetLastError());
                return (int)LBI_OK;
            });
        });
        if (status) return status;
    }
    const bool wide = D >= 4096;  // enough columns to fill the chip in whole lines
    const auto fold = wide ? fold_kernel<32, 32> : fold_kernel<16, 64>;
    hipLaunchKernelGGL(fold, dim3((unsigned)((D + (wide ? 31 : 15)) / (wide ? 32 : 16))), dim3(1024), 0, static_cast<hipStream_t>(stream),
                       partials, g_weight, slabs, (int)D);
    LBI_HIP_CHECK(hipGetLastError());
    return LBI_OK;
}
