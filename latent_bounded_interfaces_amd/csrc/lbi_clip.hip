// Clipping of a list of gradients by their global 2-norm:  n = sqrt(sum of all squares),  out = g * min(1, max_norm / (n + 1e-6)).
//
// Two kernels: one leaves the sums of squares of its workgroups in the workspace, the other adds them (every workgroup for itself: a
// thousand numbers out of the cache cost less than a launch) and scales.  Both walk the same chunks of up to CHUNK elements of one tensor,
// the table of tensors coming as a kernel argument, TABLE tensors a launch, so nothing is copied to the device and the call can be captured.
// Squares are formed and added in 64 bits: no gradient of fp32 overflows or vanishes in them, and the norm does not depend on how the chunks
// fall (fp32 sums of eight would be no faster).  Chunks go to workgroups in a fixed order and sums are added in a fixed order: reruns are bit-identical.
//
// Bound by memory: 162 M elements of bf16 are read twice, which the caches cannot hold, and written once, 980 MB in 194 us, the rate of a
// large copy.  A call of a few small tensors is two launches, 4 + 5 us.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <new>
#include <vector>

#include "lbi_attn_mfma.h"

namespace lbi {
namespace clip {
namespace {

using attn_mfma::Mma;

constexpr int THREADS = 256, PIECE = 8, UNROLL = 4, CHUNK = THREADS * PIECE * UNROLL;
constexpr int TABLE = 140, MOST_GROUPS = 1024;
constexpr double SMALLEST_NORMAL = 1.1754943508222875e-38;  // of fp32

typedef unsigned u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));

struct Table {
    const void* in[TABLE];
    void* out[TABLE];
    long long count_type[TABLE];  // elements * 4 + type
    unsigned first[TABLE];        // chunk with which the tensor begins
    int tensors;
    unsigned chunks;
};
static_assert(sizeof(Table) <= 4000, "kernel arguments");

struct Piece {  // a chunk's part of a tensor
    const void* in;
    void* out;
    long long at;
    int count, dtype;
};
// the tensor that a chunk lies in: the last one that begins no later
__device__ __forceinline__ Piece piece_of(const Table& table, unsigned chunk) {
    int low = 0, high = table.tensors - 1;
    while (low < high) {
        const int mid = (low + high + 1) / 2;
        if (table.first[mid] <= chunk) low = mid;
        else high = mid - 1;
    }
    const long long at = (long long)(chunk - table.first[low]) * CHUNK, left = (table.count_type[low] >> 2) - at;
    return Piece{table.in[low], table.out[low], at, (int)(left < CHUNK ? left : CHUNK), (int)(table.count_type[low] & 3)};
}

struct Eight { float v[PIECE]; };
__device__ __forceinline__ Eight load8(const float* p) {
    const f32x4_any a = reinterpret_cast<const f32x4_any*>(p)[0], b = reinterpret_cast<const f32x4_any*>(p + 4)[0];
    return Eight{{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]}};
}
template <typename T> __device__ __forceinline__ Eight load8(const T* p) {
    const u32x4_any a = *reinterpret_cast<const u32x4_any*>(p);
    Eight r;
#pragma unroll
    for (int e = 0; e < 4; ++e) r.v[2 * e] = Mma<T>::lo(a[e]), r.v[2 * e + 1] = Mma<T>::hi(a[e]);
    return r;
}
__device__ __forceinline__ void store8(float* p, const Eight& x) {
    reinterpret_cast<f32x4_any*>(p)[0] = f32x4_any{x.v[0], x.v[1], x.v[2], x.v[3]};
    reinterpret_cast<f32x4_any*>(p + 4)[0] = f32x4_any{x.v[4], x.v[5], x.v[6], x.v[7]};
}
template <typename T> __device__ __forceinline__ void store8(T* p, const Eight& x) {
    u32x4_any w;
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = Mma<T>::pack2(x.v[2 * e], x.v[2 * e + 1]);
    *reinterpret_cast<u32x4_any*>(p) = w;
}
__device__ __forceinline__ void store1(float* p, float x) { *p = x; }
template <typename T> __device__ __forceinline__ void store1(T* p, float x) {
    *reinterpret_cast<unsigned short*>(p) = (unsigned short)Mma<T>::pack2(x, 0.0f);
}

template <typename T> __device__ __forceinline__ double squares_of(const T* p, int count) {
    double sum[UNROLL] = {};
    if (count == CHUNK) {
        Eight x[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) x[u] = load8(p + (u * THREADS + threadIdx.x) * PIECE);
#pragma unroll
        for (int u = 0; u < UNROLL; ++u)
#pragma unroll
            for (int e = 0; e < PIECE; ++e) sum[u] = fma((double)x[u].v[e], (double)x[u].v[e], sum[u]);
    } else {
        for (int i = threadIdx.x * PIECE; i < count; i += THREADS * PIECE) {
            if (i + PIECE <= count) {
                const Eight x = load8(p + i);
#pragma unroll
                for (int e = 0; e < PIECE; ++e) sum[0] = fma((double)x.v[e], (double)x.v[e], sum[0]);
            } else {
                for (int e = i; e < count; ++e) sum[0] = fma((double)to_f32(p[e]), (double)to_f32(p[e]), sum[0]);
            }
        }
    }
    return (sum[0] + sum[1]) + (sum[2] + sum[3]);
}

// times * 2^exponent: a factor below fp32's smallest normal number, which has few of its digits left there, is held in two, any other in `times`
// alone.
struct Factor {
    float times;
    int exponent;
    __device__ __forceinline__ float operator()(float x) const { return ldexpf(x * times, exponent); }
};
template <typename T> __device__ __forceinline__ void scale(const T* p, T* out, int count, Factor factor) {
    if (count == CHUNK) {
        Eight x[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) x[u] = load8(p + (u * THREADS + threadIdx.x) * PIECE);
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
#pragma unroll
            for (int e = 0; e < PIECE; ++e) x[u].v[e] = factor(x[u].v[e]);
            store8(out + (u * THREADS + threadIdx.x) * PIECE, x[u]);
        }
    } else {
        for (int i = threadIdx.x * PIECE; i < count; i += THREADS * PIECE) {
            if (i + PIECE <= count) {
                Eight x = load8(p + i);
#pragma unroll
                for (int e = 0; e < PIECE; ++e) x.v[e] = factor(x.v[e]);
                store8(out + i, x);
            } else {
                for (int e = i; e < count; ++e) store1(out + e, factor(to_f32(p[e])));
            }
        }
    }
}

// The sum over a workgroup, the same in all of its threads.
__device__ __forceinline__ double over_group(double x, double* spare) {
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) x += __shfl_xor(x, off, 64);
    if ((threadIdx.x & 63) == 0) spare[threadIdx.x >> 6] = x;
    __syncthreads();
    return (spare[0] + spare[1]) + (spare[2] + spare[3]);
}

__global__ __launch_bounds__(THREADS) void squares_kernel(Table table, double* __restrict__ sums) {
    __shared__ double spare[THREADS / 64];
    double sum = 0.0;
    for (unsigned chunk = blockIdx.x; chunk < table.chunks; chunk += gridDim.x) {
        const Piece p = piece_of(table, chunk);
        if (p.dtype == LBI_F32) sum += squares_of(static_cast<const float*>(p.in) + p.at, p.count);
        else if (p.dtype == LBI_F16) sum += squares_of(static_cast<const _Float16*>(p.in) + p.at, p.count);
        else sum += squares_of(static_cast<const bf16_raw*>(p.in) + p.at, p.count);
    }
    sum = over_group(sum, spare);
    if (threadIdx.x == 0) sums[blockIdx.x] = sum;
}

__global__ __launch_bounds__(THREADS) void scale_kernel(Table table, const double* __restrict__ sums, int n_sums, double max_norm,
                                                        float* __restrict__ norm_out) {
    __shared__ double spare[THREADS / 64];
    double sum = 0.0;
    for (int i = threadIdx.x; i < n_sums; i += THREADS) sum += sums[i];
    const double norm = sqrt(over_group(sum, spare)), ratio = max_norm / (norm + 1e-6);
    Factor factor{(float)(ratio > 1.0 ? 1.0 : ratio), 0};  // not a number stays one
    if (ratio < SMALLEST_NORMAL) factor.times = (float)frexp(ratio, &factor.exponent);
    if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = (float)norm;
    for (unsigned chunk = blockIdx.x; chunk < table.chunks; chunk += gridDim.x) {
        const Piece p = piece_of(table, chunk);
        if (!p.out || (p.in == p.out && factor.times == 1.0f)) continue;
        if (p.dtype == LBI_F32) scale(static_cast<const float*>(p.in) + p.at, static_cast<float*>(p.out) + p.at, p.count, factor);
        else if (p.dtype == LBI_F16) scale(static_cast<const _Float16*>(p.in) + p.at, static_cast<_Float16*>(p.out) + p.at, p.count, factor);
        else scale(static_cast<const bf16_raw*>(p.in) + p.at, static_cast<bf16_raw*>(p.out) + p.at, p.count, factor);
    }
}

// The next TABLE tensors of the list that have elements.
Table table_of(const lbi_gradient* list, int64_t n, int64_t& first) {
    Table table;
    table.tensors = 0;
    table.chunks = 0;
    for (; first < n && table.tensors < TABLE; ++first) {
        const lbi_gradient& g = list[first];
        if (g.count == 0) continue;
        table.in[table.tensors] = g.in;
        table.out[table.tensors] = g.out;
        table.count_type[table.tensors] = (long long)g.count * 4 + g.dtype;
        table.first[table.tensors++] = table.chunks;
        table.chunks += (unsigned)((g.count + CHUNK - 1) / CHUNK);
    }
    return table;
}
int groups_of(const Table& table) { return (int)std::min<unsigned>(table.chunks, MOST_GROUPS); }

constexpr int64_t MOST_ELEMENTS = (int64_t)1 << 40;  // of a list: more than any memory holds, and 32 bits count its chunks

int check(const char* who, const lbi_gradient* list, int64_t n) {
    if (n < 0 || (n && !list)) return fail(LBI_ERR_INVALID, "%s: bad list", who);
    int64_t all = 0;
    for (int64_t i = 0; i < n; ++i) {
        const lbi_gradient& g = list[i];
        if (g.dtype < LBI_F32 || g.dtype > LBI_BF16) return fail(LBI_ERR_INVALID, "%s: bad dtype %lld", who, (long long)g.dtype);
        if (g.count < 0 || g.count > MOST_ELEMENTS || (all += g.count) > MOST_ELEMENTS)
            return fail(LBI_ERR_INVALID, "%s: bad size %lld", who, (long long)g.count);
        if (g.count && !g.in) return fail(LBI_ERR_INVALID, "%s: null pointer", who);
        const uintptr_t grid = dtype_size((int)g.dtype);
        if (reinterpret_cast<uintptr_t>(g.in) % grid || reinterpret_cast<uintptr_t>(g.out) % grid)
            return fail(LBI_ERR_INVALID, "%s: a tensor is not aligned to its elements", who);
    }
    return LBI_OK;
}

struct Range {
    uintptr_t begin, end;
    int64_t of;
};

// Whether no result lies on another one, nor on an input other than its own, which it then covers exactly.
bool apart(const lbi_gradient* list, int64_t n) {
    std::vector<Range> outs;
    outs.reserve((size_t)n);
    const auto bytes = [&](int64_t i) { return (uintptr_t)list[i].count * dtype_size((int)list[i].dtype); };
    for (int64_t i = 0; i < n; ++i)
        if (list[i].out && list[i].count) {
            const uintptr_t at = reinterpret_cast<uintptr_t>(list[i].out);
            outs.push_back({at, at + bytes(i), i});
        }
    std::sort(outs.begin(), outs.end(), [](const Range& a, const Range& b) { return a.begin < b.begin; });
    for (size_t i = 1; i < outs.size(); ++i)
        if (outs[i].begin < outs[i - 1].end) return false;
    for (int64_t i = 0; i < n; ++i) {
        if (!list[i].count) continue;
        const uintptr_t begin = reinterpret_cast<uintptr_t>(list[i].in), end = begin + bytes(i);
        auto hit = std::upper_bound(outs.begin(), outs.end(), begin, [](uintptr_t at, const Range& r) { return at < r.end; });
        for (; hit != outs.end() && hit->begin < end; ++hit)
            if (hit->of != i || hit->begin != begin) return false;
    }
    return true;
}

}  // namespace
}  // namespace clip
}  // namespace lbi

extern "C" size_t lbi_clip_gradients_workspace_bytes(int64_t n) {
    using namespace lbi::clip;
    return (size_t)(std::max<int64_t>(n, 0) / TABLE + 1) * MOST_GROUPS * sizeof(double);
}

extern "C" int lbi_clip_gradients(const lbi_gradient* gradients, int64_t n, float max_norm, float* norm, void* workspace,
                                  size_t workspace_bytes, void* stream) {
    using namespace lbi;
    using namespace lbi::clip;
    clear_error();
    if (int bad = check("lbi_clip_gradients", gradients, n)) return bad;
    if (!(max_norm >= 0.0f)) return fail(LBI_ERR_INVALID, "lbi_clip_gradients: max_norm must not be negative");
    if (!norm) return fail(LBI_ERR_INVALID, "lbi_clip_gradients: null pointer");
    if (reinterpret_cast<uintptr_t>(norm) % 4 || reinterpret_cast<uintptr_t>(workspace) % 8)
        return fail(LBI_ERR_INVALID, "lbi_clip_gradients: norm or workspace is not aligned");
    const size_t need = lbi_clip_gradients_workspace_bytes(n);
    if (!workspace || workspace_bytes < need)
        return fail(LBI_ERR_WORKSPACE, "lbi_clip_gradients: workspace of %zu bytes needed, %zu given", need, workspace_bytes);
    try {
        if (!apart(gradients, n)) return fail(LBI_ERR_INVALID, "lbi_clip_gradients: a result overlaps another tensor");
    } catch (const std::bad_alloc&) {
        return fail(LBI_ERR_INVALID, "lbi_clip_gradients: out of host memory");
    }
    const hipStream_t on = static_cast<hipStream_t>(stream);
    double* sums = static_cast<double*>(workspace);
    int n_sums = 0;
    for (int64_t first = 0; first < n;) {
        const Table table = table_of(gradients, n, first);
        if (!table.tensors) continue;
        hipLaunchKernelGGL(squares_kernel, dim3((unsigned)groups_of(table)), dim3(THREADS), 0, on, table, sums + n_sums);
        LBI_HIP_CHECK(hipGetLastError());
        n_sums += groups_of(table);
    }
    bool told = false;
    for (int64_t first = 0; first < n || !told; told = true) {
        const Table table = table_of(gradients, n, first);
        if (!table.tensors && told) continue;
        hipLaunchKernelGGL(scale_kernel, dim3((unsigned)std::max(groups_of(table), 1)), dim3(THREADS), 0, on, table, sums, n_sums,
                           (double)max_norm, told ? nullptr : norm);
        LBI_HIP_CHECK(hipGetLastError());
    }
    return LBI_OK;
}
