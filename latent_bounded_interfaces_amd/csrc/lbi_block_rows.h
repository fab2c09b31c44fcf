// Rows in registers: what the kernels of a block's norms share.  A row is taken in pieces of eight neighbouring elements a lane, by as many
// lanes as hold it; loads and stores at any alignment of the elements.
#pragma once

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
