// The addition to the residual stream with its RMS norm, and its pullback.
//
//   forward    s = hidden + residual,   y = s * rsqrt(mean(s^2) + eps) * weight
//   pullback   i = rsqrt(mean(s^2) + eps), u = s i, p = g_y * weight:   g_s = i (p - u mean(u p)) + g_s',   g_weight = sum over rows of g_y u
//
// Everything between load and store is fp32, the sum that the norm sees included: it is rounded only where it is stored.  y comes in the
// type of `hidden`, or in 8 bits (e4m3) with one scale a row, max|y| / 448.
//
// Bound by memory: a row is read once and kept in registers, eight neighbouring elements a lane and piece, by one wave up to 2048 columns,
// by a workgroup of 256 or 512 threads beyond.  Pieces are loaded at any alignment (an element's own is enough); one that runs past the
// end of its row goes element by element, so every width takes the same kernel.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "lbi_attn_mfma.h"

namespace lbi {
namespace block_norm {
namespace {

using attn_mfma::Mma;

constexpr int PIECE = 8;
constexpr float E4M3_MOST = 448.0f;
constexpr float SMALLEST_NORMAL = 1.17549435e-38f;

typedef unsigned u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned u32x2_any __attribute__((ext_vector_type(2), aligned(1)));

struct Eight { float v[PIECE]; };

// Eight elements from `p` on, `left` of which are in the row (the others are zero).
__device__ __forceinline__ Eight load8(const float* p, int left) {
    Eight r;
    if (left >= PIECE) {
        const f32x4_any a = reinterpret_cast<const f32x4_any*>(p)[0], b = reinterpret_cast<const f32x4_any*>(p + 4)[0];
#pragma unroll
        for (int e = 0; e < 4; ++e) r.v[e] = a[e], r.v[4 + e] = b[e];
    } else {
#pragma unroll
        for (int e = 0; e < PIECE; ++e) r.v[e] = e < left ? p[e] : 0.0f;
    }
    return r;
}
template <typename T> __device__ __forceinline__ Eight load8(const T* p, int left) {
    Eight r;
    if (left >= PIECE) {
        const u32x4_any a = *reinterpret_cast<const u32x4_any*>(p);
#pragma unroll
        for (int e = 0; e < 4; ++e) r.v[2 * e] = Mma<T>::lo(a[e]), r.v[2 * e + 1] = Mma<T>::hi(a[e]);
    } else {
#pragma unroll
        for (int e = 0; e < PIECE; ++e) r.v[e] = e < left ? to_f32(p[e]) : 0.0f;
    }
    return r;
}
__device__ __forceinline__ void store8(float* p, const Eight& x, int left) {
    if (left >= PIECE) {
        reinterpret_cast<f32x4_any*>(p)[0] = f32x4_any{x.v[0], x.v[1], x.v[2], x.v[3]};
        reinterpret_cast<f32x4_any*>(p + 4)[0] = f32x4_any{x.v[4], x.v[5], x.v[6], x.v[7]};
    } else {
#pragma unroll
        for (int e = 0; e < PIECE; ++e)
            if (e < left) p[e] = x.v[e];
    }
}
template <typename T> __device__ __forceinline__ void store8(T* p, const Eight& x, int left) {
    u32x4_any words;
#pragma unroll
    for (int e = 0; e < 4; ++e) words[e] = Mma<T>::pack2(x.v[2 * e], x.v[2 * e + 1]);
    if (left >= PIECE) {
        *reinterpret_cast<u32x4_any*>(p) = words;
    } else {
        unsigned short* raw = reinterpret_cast<unsigned short*>(p);
#pragma unroll
        for (int e = 0; e < PIECE; ++e)
            if (e < left) raw[e] = (unsigned short)(words[e / 2] >> (16 * (e % 2)));
    }
}
__device__ __forceinline__ void store8_e4m3(unsigned char* p, const Eight& x, int left) {
    u32x2_any words;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(x.v[4 * e], x.v[4 * e + 1], 0, false);
        words[e] = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(x.v[4 * e + 2], x.v[4 * e + 3], w, true);
    }
    if (left >= PIECE) {
        *reinterpret_cast<u32x2_any*>(p) = words;
    } else {
#pragma unroll
        for (int e = 0; e < PIECE; ++e)
            if (e < left) p[e] = (unsigned char)(words[e / 4] >> (8 * (e % 4)));
    }
}

// The larger one; not a number if either is none.
__device__ __forceinline__ float larger(float a, float b) { return b > a || b != b ? b : a; }

struct Add { static __device__ __forceinline__ float of(float a, float b) { return a + b; } };
struct Larger { static __device__ __forceinline__ float of(float a, float b) { return larger(a, b); } };

// One value over the NT threads that share a row, the same in all of them: lanes by exchange, waves in order.  `spare`: NT / 64 floats that no
// other exchange of the row uses.
template <typename Op, int NT> __device__ __forceinline__ float over_row(float x, float* spare) {
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) x = Op::of(x, __shfl_xor(x, off, 64));
    if constexpr (NT > 64) {
        if ((threadIdx.x & 63) == 0) spare[threadIdx.x >> 6] = x;
        __syncthreads();
        x = spare[0];
#pragma unroll
        for (int w = 1; w < NT / 64; ++w) x = Op::of(x, spare[w]);
    }
    return x;
}

template <typename T> __device__ __forceinline__ Eight load_weight(const void* weight, int c, int left, bool wide) {
    return wide ? load8(static_cast<const float*>(weight) + c, left) : load8(static_cast<const T*>(weight) + c, left);
}

// NT threads a row (a workgroup of 256 holds four rows of 64), PIECES pieces a lane.
template <typename T, typename R, bool SCALED, int NT, int PIECES>
__global__ __launch_bounds__(NT < 256 ? 256 : NT) void norm_kernel(const T* __restrict__ hidden, const R* __restrict__ residual,
                                                                   const void* __restrict__ weight, void* __restrict__ normed,
                                                                   R* __restrict__ stream_out, float* __restrict__ scales, long long rows,
                                                                   int D, float eps, int weight_wide) {
    __shared__ float spare[2][NT / 64];
    const int t = threadIdx.x % NT;
    const long long row = NT < 256 ? (long long)blockIdx.x * (256 / NT) + threadIdx.x / NT : (long long)blockIdx.x;
    if (row >= rows) return;  // whole waves, and no barrier below is theirs alone
    Eight s[PIECES], w[PIECES];
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
        const int c = (p * NT + t) * PIECE;
        if (c < D) s[p] = load8(hidden + row * D + c, D - c);
    }
    if (residual) {
        Eight r[PIECES];
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            const int c = (p * NT + t) * PIECE;
            if (c < D) r[p] = load8(residual + row * D + c, D - c);
        }
#pragma unroll
        for (int p = 0; p < PIECES; ++p)
#pragma unroll
            for (int e = 0; e < PIECE; ++e) s[p].v[e] += r[p].v[e];
    }
    float sum = 0.0f;
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
        const int c = (p * NT + t) * PIECE;
        if (c >= D) continue;
        w[p] = load_weight<T>(weight, c, D - c, weight_wide != 0);
        if (stream_out) store8(stream_out + row * D + c, s[p], D - c);
#pragma unroll
        for (int e = 0; e < PIECE; ++e) sum = fmaf(s[p].v[e], s[p].v[e], sum);
    }
    const float inv = rsqrtf(over_row<Add, NT>(sum, spare[0]) / (float)D + eps);
    float most = 0.0f;
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
        const int c = (p * NT + t) * PIECE;
        if (c >= D) continue;
#pragma unroll
        for (int e = 0; e < PIECE; ++e) {
            s[p].v[e] = s[p].v[e] * inv * w[p].v[e];
            if (SCALED) most = larger(most, fabsf(s[p].v[e]));
        }
        if (!SCALED) store8(static_cast<T*>(normed) + row * D + c, s[p], D - c);
    }
    if constexpr (SCALED) {
        most = over_row<Larger, NT>(most, spare[1]);
        // a row of zeros has the scale 1; no scale is below the smallest normal number, whose reciprocal is still one
        const float scale = most == 0.0f ? 1.0f : larger(most / E4M3_MOST, SMALLEST_NORMAL), back = 1.0f / scale;
        if (t == 0) scales[row] = scale;
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            const int c = (p * NT + t) * PIECE;
            if (c >= D) continue;
#pragma unroll
            for (int e = 0; e < PIECE; ++e) s[p].v[e] *= back;
            store8_e4m3(static_cast<unsigned char*>(normed) + row * D + c, s[p], D - c);
        }
    }
}

// A workgroup takes the rows of one slab, NT threads a row, and leaves its share of the weight's gradient in `partials` [slabs, D].
template <typename T, typename R, int NT, int PIECES>
__global__ __launch_bounds__(NT < 256 ? 256 : NT) void norm_pullback_kernel(const T* __restrict__ g_normed, const R* __restrict__ stream,
                                                                            const R* __restrict__ g_stream, const void* __restrict__ weight,
                                                                            T* __restrict__ g_hidden, R* __restrict__ g_residual,
                                                                            float* __restrict__ partials, long long rows, int D, float eps,
                                                                            int weight_wide, int slab) {
    constexpr int SIDE = NT < 256 ? 256 / NT : 1;  // rows side by side
    extern __shared__ __align__(16) float lds[];   // SIDE > 1: [SIDE][D]
    __shared__ float spare[2][2][NT / 64];
    const int t = threadIdx.x % NT, side = threadIdx.x / NT;
    const long long first = (long long)blockIdx.x * slab, last = first + slab < rows ? first + slab : rows;
    Eight w[PIECES], total[PIECES];
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
        const int c = (p * NT + t) * PIECE;
        if (c < D) w[p] = load_weight<T>(weight, c, D - c, weight_wide != 0);
#pragma unroll
        for (int e = 0; e < PIECE; ++e) total[p].v[e] = 0.0f;
    }
    int turn = 0;
    for (long long row = first + side; row < last; row += SIDE, turn ^= 1) {
        Eight x[PIECES], g[PIECES], more[PIECES];
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            const int c = (p * NT + t) * PIECE;
            if (c >= D) continue;
            x[p] = load8(stream + row * D + c, D - c);
            g[p] = load8(g_normed + row * D + c, D - c);
            if (g_stream) more[p] = load8(g_stream + row * D + c, D - c);
        }
        float squares = 0.0f, along = 0.0f;
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            if ((p * NT + t) * PIECE >= D) continue;
#pragma unroll
            for (int e = 0; e < PIECE; ++e) {
                squares = fmaf(x[p].v[e], x[p].v[e], squares);
                along = fmaf(x[p].v[e], g[p].v[e] * w[p].v[e], along);
            }
        }
        squares = over_row<Add, NT>(squares, spare[turn][0]);
        along = over_row<Add, NT>(along, spare[turn][1]);
        const float inv = rsqrtf(squares / (float)D + eps), mean = along * inv / (float)D;
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            const int c = (p * NT + t) * PIECE;
            if (c >= D) continue;
            Eight out;
#pragma unroll
            for (int e = 0; e < PIECE; ++e) {
                const float unit = x[p].v[e] * inv;
                total[p].v[e] = fmaf(g[p].v[e], unit, total[p].v[e]);
                out.v[e] = inv * (g[p].v[e] * w[p].v[e] - unit * mean) + (g_stream ? more[p].v[e] : 0.0f);
            }
            if (g_residual) store8(g_residual + row * D + c, out, D - c);
            if (g_hidden) store8(g_hidden + row * D + c, out, D - c);
        }
    }
    if constexpr (SIDE > 1) {
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            const int c = (p * NT + t) * PIECE;
            if (c < D) store8(lds + side * D + c, total[p], D - c);
        }
        __syncthreads();
        for (int c = threadIdx.x; c < D; c += 256) {
            float sum = lds[c];
#pragma unroll
            for (int q = 1; q < SIDE; ++q) sum += lds[q * D + c];
            partials[(size_t)blockIdx.x * D + c] = sum;
        }
    } else {
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            const int c = (p * NT + t) * PIECE;
            if (c < D) store8(partials + (size_t)blockIdx.x * D + c, total[p], D - c);
        }
    }
}

// out[c] = sum over slabs of partials[slab][c]: 16 columns a workgroup, 64 threads a column, whose sums are added in order.
constexpr int FOLD_COLUMNS = 16, FOLD_PARTS = 64;
__global__ __launch_bounds__(FOLD_COLUMNS * FOLD_PARTS) void fold_kernel(const float* __restrict__ partials, float* __restrict__ out, int slabs,
                                                                         int D) {
    __shared__ float part[FOLD_PARTS][FOLD_COLUMNS];
    const int col = threadIdx.x % FOLD_COLUMNS, q = threadIdx.x / FOLD_COLUMNS, c = blockIdx.x * FOLD_COLUMNS + col;
    float sum = 0.0f;
    if (c < D)
#pragma unroll 8
        for (int s = q; s < slabs; s += FOLD_PARTS) sum += partials[(size_t)s * D + c];
    part[q][col] = sum;
    __syncthreads();
    for (int half = FOLD_PARTS / 2; half >= 1; half /= 2) {
        if (q < half) part[q][col] += part[q + half][col];
        __syncthreads();
    }
    if (q == 0 && c < D) out[c] = part[0][col];
}

constexpr int64_t MOST_COLUMNS = 512 * 4 * PIECE, MOST_ROWS = (int64_t)1 << 31;
constexpr int SLABS = 512;  // two workgroups a CU

// rows of a slab of the pullback, and how many slabs that makes
int slab_rows(int64_t rows) { return (int)std::max<int64_t>((rows + SLABS - 1) / SLABS, 4); }
int slab_count(int64_t rows) { return (int)((rows + slab_rows(rows) - 1) / slab_rows(rows)); }

template <int NT_, int PIECES_> struct Form { static constexpr int NT = NT_, PIECES = PIECES_; };
// What holds a row of D columns in registers.
template <typename F> int by_width(int64_t D, F&& launch) {
    if (D <= 512) return launch(Form<64, 1>{});
    if (D <= 1024) return launch(Form<64, 2>{});
    if (D <= 2048) return launch(Form<64, 4>{});
    if (D <= 4096) return launch(Form<256, 2>{});
    if (D <= 8192) return launch(Form<256, 4>{});
    return launch(Form<512, 4>{});
}

template <typename T> struct Type { using type = T; };
// dtype: of hidden, normed and their cotangents; stream: of the residual stream, the same or fp32.
template <typename F> int by_types(int dtype, int stream, F&& launch) {
    if (dtype == LBI_F32) return launch(Type<float>{}, Type<float>{});
    if (dtype == LBI_F16) return stream == LBI_F16 ? launch(Type<_Float16>{}, Type<_Float16>{}) : launch(Type<_Float16>{}, Type<float>{});
    return stream == LBI_BF16 ? launch(Type<bf16_raw>{}, Type<bf16_raw>{}) : launch(Type<bf16_raw>{}, Type<float>{});
}

int check(const char* who, int64_t rows, int64_t D, int dtype, int stream, int weight) {
    if (rows < 0 || D < 1) return fail(LBI_ERR_INVALID, "%s: bad size (rows=%lld D=%lld)", who, (long long)rows, (long long)D);
    if (!dtype_size(dtype) || (stream != dtype && stream != LBI_F32) || (weight != dtype && weight != LBI_F32))
        return fail(LBI_ERR_INVALID, "%s: bad dtype (%d; residual stream %d and weight %d are of the same or fp32)", who, dtype, stream, weight);
    if (D > MOST_COLUMNS || rows >= MOST_ROWS)
        return fail(LBI_ERR_UNSUPPORTED, "%s: rows of up to %lld columns, fewer than 2^31 of them", who, (long long)MOST_COLUMNS);
    return LBI_OK;
}

bool aligned(const void* p, int dtype) { return reinterpret_cast<uintptr_t>(p) % (dtype_size(dtype)) == 0; }

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
    return by_types(dtype, residual_dtype, [&](auto t, auto r) {
        using T = typename decltype(t)::type;
        using R = typename decltype(r)::type;
        return by_width(D, [&](auto form) {
            constexpr int NT = decltype(form)::NT, PIECES = decltype(form)::PIECES, SIDE = NT < 256 ? 256 / NT : 1;
            const auto kernel = scales ? norm_kernel<T, R, true, NT, PIECES> : norm_kernel<T, R, false, NT, PIECES>;
            hipLaunchKernelGGL(kernel, dim3((unsigned)((rows + SIDE - 1) / SIDE)), dim3(NT * SIDE), 0, static_cast<hipStream_t>(stream),
                               static_cast<const T*>(hidden), static_cast<const R*>(residual), weight, normed, static_cast<R*>(residual_out),
                               scales, (long long)rows, (int)D, eps, (int)(weight_dtype == LBI_F32));
            LBI_HIP_CHECK(hipGetLastError());
            return (int)LBI_OK;
        });
    });
}

extern "C" size_t lbi_residual_rmsnorm_pullback_workspace_bytes(int64_t rows, int64_t D) {
    using namespace lbi::block_norm;
    if (rows < 0 || D < 1 || D > MOST_COLUMNS || rows >= MOST_ROWS) return 0;
    return (size_t)slab_count(rows) * (size_t)D * sizeof(float);
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
    const int slabs = slab_count(rows);
    const size_t need = lbi_residual_rmsnorm_pullback_workspace_bytes(rows, D);
    if (need && (!workspace || workspace_bytes < need))
        return fail(LBI_ERR_WORKSPACE, "lbi_residual_rmsnorm_pullback: workspace of %zu bytes needed, %zu given", need, workspace_bytes);
    if (!aligned(g_normed, dtype) || !aligned(residual_out, residual_dtype) || !aligned(g_residual_out, residual_dtype) ||
        !aligned(weight, weight_dtype) || !aligned(g_hidden, dtype) || !aligned(g_residual, residual_dtype) || !aligned(g_weight, LBI_F32) ||
        !aligned(workspace, LBI_F32))
        return fail(LBI_ERR_INVALID, "lbi_residual_rmsnorm_pullback: a tensor is not aligned to its elements");
    float* partials = static_cast<float*>(workspace);
    if (rows) {
        const int status = by_types(dtype, residual_dtype, [&](auto t, auto r) {
            using T = typename decltype(t)::type;
            using R = typename decltype(r)::type;
            return by_width(D, [&](auto form) {
                constexpr int NT = decltype(form)::NT, PIECES = decltype(form)::PIECES, SIDE = NT < 256 ? 256 / NT : 1;
                const size_t bytes = SIDE > 1 ? SIDE * (size_t)D * sizeof(float) : 0;  // 32 KiB at most
                hipLaunchKernelGGL((norm_pullback_kernel<T, R, NT, PIECES>), dim3((unsigned)slabs), dim3(NT * SIDE), bytes,
                                   static_cast<hipStream_t>(stream), static_cast<const T*>(g_normed), static_cast<const R*>(residual_out),
                                   static_cast<const R*>(g_residual_out), weight, static_cast<T*>(g_hidden), static_cast<R*>(g_residual),
                                   partials, (long long)rows, (int)D, eps, (int)(weight_dtype == LBI_F32), slab_rows(rows));
                LBI_HIP_CHECK(hipGetLastError());
                return (int)LBI_OK;
            });
        });
        if (status) return status;
    }
    hipLaunchKernelGGL(fold_kernel, dim3((unsigned)((D + FOLD_COLUMNS - 1) / FOLD_COLUMNS)), dim3(FOLD_COLUMNS * FOLD_PARTS), 0,
                       static_cast<hipStream_t>(stream), partials, g_weight, slabs, (int)D);
    LBI_HIP_CHECK(hipGetLastError());
    return LBI_OK;
}
