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

// Eight elements as stored.  They are widened only where they are used: a conversion right behind its load would wait for it, and the loads of
// a row would come one after the other (2000 x 8192 in bf16, pullback: 46 -> 32 us).
template <typename T> struct Raw {
    u32x4_any w;
    __device__ __forceinline__ Eight wide() const {
        Eight r;
#pragma unroll
        for (int e = 0; e < 4; ++e) r.v[2 * e] = Mma<T>::lo(w[e]), r.v[2 * e + 1] = Mma<T>::hi(w[e]);
        return r;
    }
};
template <> struct Raw<float> {
    f32x4_any a, b;
    __device__ __forceinline__ Eight wide() const { return Eight{{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]}}; }
};
// From `p` on, `left` of which are in the row (TAIL: perhaps fewer than eight; the others are zero).
template <bool TAIL> __device__ __forceinline__ Raw<float> load8(const float* p, int left) {
    Raw<float> r;
    if (!TAIL || left >= PIECE) {
        r.a = reinterpret_cast<const f32x4_any*>(p)[0];
        r.b = reinterpret_cast<const f32x4_any*>(p + 4)[0];
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            r.a[e] = e < left ? p[e] : 0.0f;
            r.b[e] = 4 + e < left ? p[4 + e] : 0.0f;
        }
    }
    return r;
}
template <bool TAIL, typename T> __device__ __forceinline__ Raw<T> load8(const T* p, int left) {
    Raw<T> r;
    if (!TAIL || left >= PIECE) {
        r.w = *reinterpret_cast<const u32x4_any*>(p);
    } else {
        const unsigned short* raw = reinterpret_cast<const unsigned short*>(p);
#pragma unroll
        for (int e = 0; e < 4; ++e) r.w[e] = (2 * e < left ? raw[2 * e] : 0u) | (2 * e + 1 < left ? (unsigned)raw[2 * e + 1] << 16 : 0u);
    }
    return r;
}
template <bool TAIL> __device__ __forceinline__ void store8(float* p, const Eight& x, int left) {
    if (!TAIL || left >= PIECE) {
        reinterpret_cast<f32x4_any*>(p)[0] = f32x4_any{x.v[0], x.v[1], x.v[2], x.v[3]};
        reinterpret_cast<f32x4_any*>(p + 4)[0] = f32x4_any{x.v[4], x.v[5], x.v[6], x.v[7]};
    } else {
#pragma unroll
        for (int e = 0; e < PIECE; ++e)
            if (e < left) p[e] = x.v[e];
    }
}
template <bool TAIL, typename T> __device__ __forceinline__ void store8(T* p, const Eight& x, int left) {
    u32x4_any words;
#pragma unroll
    for (int e = 0; e < 4; ++e) words[e] = Mma<T>::pack2(x.v[2 * e], x.v[2 * e + 1]);
    if (!TAIL || left >= PIECE) {
        *reinterpret_cast<u32x4_any*>(p) = words;
    } else {
        unsigned short* raw = reinterpret_cast<unsigned short*>(p);
#pragma unroll
        for (int e = 0; e < PIECE; ++e)
            if (e < left) raw[e] = (unsigned short)(words[e / 2] >> (16 * (e % 2)));
    }
}
template <bool TAIL> __device__ __forceinline__ void store8_e4m3(unsigned char* p, const Eight& x, int left) {
    u32x2_any words;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(x.v[4 * e], x.v[4 * e + 1], 0, false);
        words[e] = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(x.v[4 * e + 2], x.v[4 * e + 3], w, true);
    }
    if (!TAIL || left >= PIECE) {
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

// One value over the threads that share a row, the same in all of them: lanes by exchange, waves in order.  Rows of up to 64 threads have NT of
// them, wider ones the whole workgroup, which is at most NT.  `spare`: NT / 64 floats that no other exchange of the row uses.
template <typename Op, int NT> __device__ __forceinline__ float over_row(float x, float* spare) {
#pragma unroll
    for (int off = (NT < 64 ? NT : 64) / 2; off >= 1; off >>= 1) x = Op::of(x, __shfl_xor(x, off, 64));
    if constexpr (NT > 64) {
        if ((threadIdx.x & 63) == 0) spare[threadIdx.x >> 6] = x;
        __syncthreads();
        x = spare[0];
        for (int w = 1; w < (int)blockDim.x / 64; ++w) x = Op::of(x, spare[w]);
    }
    return x;
}

// Two sums at once.
template <int NT> __device__ __forceinline__ void sums_over_row(float& x, float& y, float (*spare)[2]) {
#pragma unroll
    for (int off = (NT < 64 ? NT : 64) / 2; off >= 1; off >>= 1) {
        const float a = __shfl_xor(x, off, 64), b = __shfl_xor(y, off, 64);
        x += a;
        y += b;
    }
    if constexpr (NT > 64) {
        if ((threadIdx.x & 63) == 0) spare[threadIdx.x >> 6][0] = x, spare[threadIdx.x >> 6][1] = y;
        __syncthreads();
        x = spare[0][0];
        y = spare[0][1];
        for (int w = 1; w < (int)blockDim.x / 64; ++w) x += spare[w][0], y += spare[w][1];
    }
}

// rows that a workgroup holds side by side: 256 threads of rows that need no more than a wave each, one row otherwise
template <int NT> constexpr int SIDE = NT <= 64 ? 256 / NT : 1;

template <bool TAIL, typename T> __device__ __forceinline__ Eight load_weight(const void* weight, int c, int left, bool wide) {
    return wide ? load8<TAIL>(static_cast<const float*>(weight) + c, left).wide() : load8<TAIL>(static_cast<const T*>(weight) + c, left).wide();
}

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

// out[c] = sum over slabs of partials[slab][c]: COLUMNS columns a workgroup, PARTS threads a column, whose sums are added in order.
template <int COLUMNS, int PARTS>
__global__ __launch_bounds__(COLUMNS * PARTS) void fold_kernel(const float* __restrict__ partials, float* __restrict__ out, int slabs, int D) {
    __shared__ float part[PARTS][COLUMNS];
    const int col = threadIdx.x % COLUMNS, q = threadIdx.x / COLUMNS, c = blockIdx.x * COLUMNS + col;
    float sum = 0.0f;
    if (c < D)
#pragma unroll 8
        for (int s = q; s < slabs; s += PARTS) sum += partials[(size_t)s * D + c];
    part[q][col] = sum;
    __syncthreads();
    for (int half = PARTS / 2; half >= 1; half /= 2) {
        if (q < half) part[q][col] += part[q + half][col];
        __syncthreads();
    }
    if (q == 0 && c < D) out[c] = part[0][col];
}

constexpr int64_t MOST_COLUMNS = 1024 * 2 * PIECE, MOST_ROWS = (int64_t)1 << 31;
constexpr int64_t MOST_THREADS = ((int64_t)1 << 32) - 1;  // of a launch

// Slabs of the pullback, and the rows of one: four workgroups a CU of narrow rows, two of wide ones, whose shares of the weight's gradient
// would be as many bytes as a twentieth of the rows themselves.
int slab_rows(int64_t rows, int64_t D) {
    const int64_t slabs = D <= 1024 ? 1024 : 512;
    const int64_t least = D <= 512 ? 2048 / D : 1;  // rows that a workgroup holds side by side, about
    return (int)std::max<int64_t>((rows + slabs - 1) / slabs, least);
}
int slab_count(int64_t rows, int64_t D) { return (int)((rows + slab_rows(rows, D) - 1) / slab_rows(rows, D)); }

template <int NT_, int PIECES_> struct Form { static constexpr int NT = NT_, PIECES = PIECES_; };
// Threads of a row: as few waves as hold it where that is more than one.
template <int NT, int PIECES> int threads_of(int64_t D) {
    return NT <= 64 ? NT : (int)((D + 64 * PIECE * PIECES - 1) / (64 * PIECE * PIECES)) * 64;
}
// What holds a row of D columns in registers.
template <bool PULLBACK, typename F> int by_width(int64_t D, F&& launch) {
    if (D <= 64) return launch(Form<8, 1>{});
    if (D <= 128) return launch(Form<16, 1>{});
    if (D <= 256) return launch(Form<32, 1>{});
    if (D <= 512) return launch(Form<64, 1>{});
    if (D <= 1024) return launch(Form<64, 2>{});
    // a slab's rows come one after the other: twice the waves (6000 x 5120 in fp16: 74 -> 68 us, and 53 with the next row ahead)
    if (D <= 8192) return launch(Form<PULLBACK ? 1024 : 512, PULLBACK ? 1 : 2>{});
    return launch(Form<1024, 2>{});
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

// A tensor of so many bytes; none if it is not given.
struct Place {
    uintptr_t at;
    uint64_t bytes;
    Place(const void* p, int64_t elements, size_t size) : at(reinterpret_cast<uintptr_t>(p)), bytes(p ? (uint64_t)elements * size : 0) {}
    bool meets(const Place& o) const { return bytes && o.bytes && at < o.at + o.bytes && o.at < at + bytes; }
    bool is(const Place& o) const { return at == o.at && bytes == o.bytes; }
};

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
