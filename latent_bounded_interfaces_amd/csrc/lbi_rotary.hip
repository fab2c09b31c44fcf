// Rotary positions: a packed projection's queries and keys turned into heads, and back.
//
//   forward    (x1, x2) -> (x1 cos - x2 sin, x1 sin + x2 cos) for each pair of the first R elements of a head, the others as they are
//   pullback   the same with -sin, after the heads that share a key or value are added up, into the packed projection's cotangent
//
// A pair is (c, c + R/2), or (2 c, 2 c + 1) if interleaved.  cos and sin are tables of fp32 over positions; a position past their end turns to
// NaN.  Arithmetic is fp32, each result is rounded once.
//
// Bound by memory: every element is read and written once, a thread to a piece of 16 bytes or to a pair of them, wherever they start (a projection
// that starts on an odd element takes 7 to 16 % longer; an element each would take 1.7 to 2.7 times as long), and an element each where a head's
// parts are no whole pieces; the tables come from the caches, once a thread.  8 x 1024 tokens of 12 + 2 x 12 heads of 64 in bf16: 12.5 us, 4.0 TB/s; the pullback
// of 4 x 4096 tokens of 16 + 2 x 4 heads of 128, whose key and value cotangents come for 16 heads: 77 us, 3.9 TB/s.  One token: 2.2 us.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "lbi_common.h"

namespace lbi {
namespace rotary {
namespace {

constexpr int64_t MOST_UNITS = (int64_t)1 << 31;  // of a launch: what the divisions below take

// n / d for n < 2^31 by a multiplication: a thread moves a piece or two, next to which the processor's own divisions count.
struct Divisor {
    unsigned d, factor, shift;
    Divisor(unsigned d_ = 1) : d(d_), factor(0), shift(0) {
        while (((uint64_t)1 << shift) < d) ++shift;
        factor = (unsigned)((((uint64_t)1 << 32) * (((uint64_t)1 << shift) - d)) / d + 1);
    }
    __device__ __forceinline__ unsigned of(unsigned n) const { return (__umulhi(n, factor) + n) >> shift; }
};

// N elements that start on any of them.
template <typename T, int N> struct Piece;
template <int N> struct Piece<float, N> { typedef float type __attribute__((ext_vector_type(N), aligned(4))); };
template <int N> struct Piece<_Float16, N> { typedef _Float16 type __attribute__((ext_vector_type(N), aligned(2))); };
template <int N> struct Piece<bf16_raw, N> { typedef unsigned short type __attribute__((ext_vector_type(N), aligned(2))); };

template <typename T> __device__ __forceinline__ float widen(T x) { return (float)x; }
template <> __device__ __forceinline__ float widen(unsigned short x) { return __uint_as_float((unsigned)x << 16); }
template <typename T> __device__ __forceinline__ auto narrow(float x) {
    if constexpr (std::is_same_v<T, bf16_raw>) return f32_to_bf16_bits(x);
    else return (T)x;
}

struct Call {
    const void *q, *k, *v;  // forward: the packed projection in q; pullback: [B, P, heads, T, D]
    void *out, *out_k;      // forward: [B, H, T, D] and [B, Hkv, T, D]; pullback: [B, P, T, (H + 2 Hkv) D]
    const float *cos, *sin;  // [table, R / 2]
    const void* positions;   // [B, T], NULL: 0, 1, ...; 8 bytes each if positions_wide
    int64_t stride_b, stride_t;  // of the packed projection
    int64_t table, first_row;
    unsigned units;  // of this launch
    Divisor places, heads, by_t, by_p;
    unsigned first_bp, first_t;  // of the launch's first row
    int positions_wide, P, T, H, Hkv, shared, D, R, interleaved;  // shared: heads of k and v that are added up
};

__device__ __forceinline__ int64_t row_of_table(const Call& c, int64_t b, int64_t t) {
    int64_t at = t;
    if (c.positions) at = c.positions_wide ? static_cast<const int64_t*>(c.positions)[b * c.T + t] : (int64_t)static_cast<const int*>(c.positions)[b * c.T + t];
    return at >= 0 && at < c.table ? at : -1;
}

// N elements from `p` on, `shared` times `apart` elements apart, added up; four are asked for at once.
template <typename T, int N> __device__ __forceinline__ void load(const T* p, int shared, int64_t apart, float* x) {
    typedef typename Piece<T, N>::type piece;
#pragma unroll
    for (int e = 0; e < N; ++e) x[e] = 0.0f;
    for (int s = 0; s < shared; s += 4) {
        piece own[4];
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (s + k < shared) own[k] = *reinterpret_cast<const piece*>(p + (s + k) * apart);
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (s + k < shared)
#pragma unroll
                for (int e = 0; e < N; ++e) x[e] += widen(own[k][e]);
    }
}
template <typename T, int N> __device__ __forceinline__ void load(const T* p, float* x) {
    const typename Piece<T, N>::type own = *reinterpret_cast<const typename Piece<T, N>::type*>(p);
#pragma unroll
    for (int e = 0; e < N; ++e) x[e] = widen(own[e]);
}
template <typename T, int N> __device__ __forceinline__ void store(T* p, const float* x) {
    typedef typename Piece<T, N>::type piece;
    piece own;
#pragma unroll
    for (int e = 0; e < N; ++e) own[e] = narrow<T>(x[e]);
    *reinterpret_cast<piece*>(p) = own;
}

// A unit is a place of a head of a row: half layout, pairs of pieces of the turned part, then the pieces of the rest; interleaved, the pieces in order.
template <typename T, int N, bool BACK> __global__ __launch_bounds__(256) void rotary_kernel(Call c) {
    const unsigned id = blockIdx.x * 256 + threadIdx.x;
    if (id >= c.units) return;
    const int turned = c.interleaved ? c.R / N : c.R / 2 / N;  // places of a head's turned part
    const int heads = c.H + (BACK ? 2 : 1) * c.Hkv;
    const unsigned rest = c.places.of(id), row_here = c.heads.of(rest);
    const int place = (int)(id - rest * c.places.d), head = (int)(rest - row_here * c.heads.d);
    const int64_t row = c.first_row + row_here;  // of [B, P, T]
    const unsigned tokens = c.first_t + row_here, bp_here = c.by_t.of(tokens);
    const int t = (int)(tokens - bp_here * c.by_t.d);
    const int64_t bp = c.first_bp + bp_here, b = BACK ? c.by_p.of((unsigned)bp) : bp;
    const bool is_q = head < c.H, is_v = head >= c.H + c.Hkv;
    const int own = is_q ? head : is_v ? head - c.H - c.Hkv : head - c.H;
    const int shared = is_q ? 1 : c.shared;
    const auto bring = [&](auto count, const T* p, float* x) __attribute__((always_inline)) {
        constexpr int COUNT = decltype(count)::value;
        if (!BACK || shared == 1) load<T, COUNT>(p, x);
        else load<T, COUNT>(p, shared, (int64_t)c.T * c.D, x);
    };
    using Pieces = std::integral_constant<int, N>;
    using One = std::integral_constant<int, 1>;

    const T* from;
    T* to;
    if constexpr (BACK) {
        const int count = is_q ? c.H : c.Hkv * c.shared;
        from = static_cast<const T*>(is_q ? c.q : is_v ? c.v : c.k) + ((bp * count + own * shared) * c.T + t) * c.D;
        to = static_cast<T*>(c.out) + (row * heads + head) * c.D;
    } else {
        from = static_cast<const T*>(c.q) + b * c.stride_b + t * c.stride_t + (int64_t)head * c.D;
        to = static_cast<T*>(is_q ? c.out : c.out_k) + ((b * (is_q ? c.H : c.Hkv) + own) * c.T + t) * c.D;
    }
    float x[N], y[N];
    if (place >= turned) {
        const int at = c.R + (place - turned) * N;
        bring(Pieces{}, from + at, x);
        store<T, N>(to + at, x);
        return;
    }
    const int64_t line = is_v ? 0 : row_of_table(c, b, t);
    const float nan = __builtin_nanf("");
    if (c.interleaved) {
        if constexpr (N % 2 == 0) {
            bring(Pieces{}, from + place * N, x);
            if (!is_v) {
                const float *cs = c.cos + line * (c.R / 2) + place * (N / 2), *sn = c.sin + line * (c.R / 2) + place * (N / 2);
#pragma unroll
                for (int e = 0; e < N / 2; ++e) {
                    const float co = line < 0 ? nan : cs[e], si = line < 0 ? nan : BACK ? -sn[e] : sn[e];
                    y[2 * e] = x[2 * e] * co - x[2 * e + 1] * si;
                    y[2 * e + 1] = x[2 * e] * si + x[2 * e + 1] * co;
                }
            } else {
#pragma unroll
                for (int e = 0; e < N; ++e) y[e] = x[e];
            }
            store<T, N>(to + place * N, y);
        } else {  // one element: its pair's other one is next to it
            const int at = place, other = at ^ 1;
            bring(One{}, from + at, x);
            if (!is_v) {
                bring(One{}, from + other, y);
                const float co = line < 0 ? nan : c.cos[line * (c.R / 2) + at / 2];
                float si = line < 0 ? nan : c.sin[line * (c.R / 2) + at / 2];
                if ((at & 1) == 0) si = -si;
                if (BACK) si = -si;
                x[0] = x[0] * co + y[0] * si;
            }
            store<T, 1>(to + at, x);
        }
        return;
    }
    const int at = place * N, half = c.R / 2;
    bring(Pieces{}, from + at, x);
    bring(Pieces{}, from + at + half, y);
    if (!is_v) {
        const float *cs = c.cos + line * half + at, *sn = c.sin + line * half + at;
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const float co = line < 0 ? nan : cs[e], si = line < 0 ? nan : BACK ? -sn[e] : sn[e];
            const float a = x[e], o = y[e];
            x[e] = a * co - o * si;
            y[e] = a * si + o * co;
        }
    }
    store<T, N>(to + at, x);
    store<T, N>(to + at + half, y);
}

bool off(const void* p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to != 0; }

template <typename T, int N, bool BACK> int launch(Call c, int64_t rows, hipStream_t stream) {
    const int64_t places = (c.interleaved ? c.R / N : c.R / 2 / N) + (c.D - c.R) / N, heads = c.H + (BACK ? 2 : 1) * c.Hkv;
    if (places * heads >= MOST_UNITS) return fail(LBI_ERR_UNSUPPORTED, "rotary positions: too many elements of a token");
    c.places = Divisor((unsigned)places), c.heads = Divisor((unsigned)heads), c.by_t = Divisor((unsigned)c.T), c.by_p = Divisor((unsigned)c.P);
    const int64_t most = std::min((MOST_UNITS - 1) / (places * heads), MOST_UNITS / 2);  // rows of a launch
    for (int64_t first = 0; first < rows; first += most) {
        const int64_t count = std::min(rows - first, most) * places * heads;
        c.first_row = first, c.first_bp = (unsigned)(first / c.T), c.first_t = (unsigned)(first % c.T);
        c.units = (unsigned)count;
        hipLaunchKernelGGL((rotary_kernel<T, N, BACK>), dim3((unsigned)((count + 255) / 256)), dim3(256), 0, stream, c);
        LBI_HIP_CHECK(hipGetLastError());
    }
    return LBI_OK;
}

template <typename T, bool BACK> int by_pieces(const Call& c, int64_t rows, hipStream_t stream) {
    constexpr int N = 16 / sizeof(T);
    const bool whole = c.D % N == 0 && (c.interleaved ? c.R : c.R / 2) % N == 0;
    return whole ? launch<T, N, BACK>(c, rows, stream) : launch<T, 1, BACK>(c, rows, stream);
}
template <bool BACK> int by_type(const Call& c, int64_t rows, int dtype, hipStream_t stream) {
    if (dtype == LBI_F32) return by_pieces<float, BACK>(c, rows, stream);
    return dtype == LBI_F16 ? by_pieces<_Float16, BACK>(c, rows, stream) : by_pieces<bf16_raw, BACK>(c, rows, stream);
}

int check(const char* who, int64_t B, int64_t P, int64_t T, int64_t H, int64_t Hkv, int64_t D, int64_t R, int64_t table, const void* positions, int dtype) {
    if (B < 0 || P < 0 || T < 0 || H < 1 || Hkv < 1 || D < 1 || R < 0 || R > D || table < 0)
        return fail(LBI_ERR_INVALID, "%s: bad size (B=%lld P=%lld T=%lld H=%lld Hkv=%lld D=%lld R=%lld table=%lld)", who, (long long)B, (long long)P,
                    (long long)T, (long long)H, (long long)Hkv, (long long)D, (long long)R, (long long)table);
    if (H % Hkv) return fail(LBI_ERR_INVALID, "%s: H=%lld not a multiple of Hkv=%lld", who, (long long)H, (long long)Hkv);
    if (R % 2) return fail(LBI_ERR_INVALID, "%s: rotary embedding needs an even part of a head, got %lld", who, (long long)R);
    if (!dtype_size(dtype)) return fail(LBI_ERR_INVALID, "%s: bad dtype %d", who, dtype);
    if (!positions && table < T) return fail(LBI_ERR_INVALID, "%s: tables of %lld positions for %lld tokens", who, (long long)table, (long long)T);
    if (D > (int64_t)1 << 16 || H > (int64_t)1 << 16 || T >= (int64_t)1 << 30 || P >= (int64_t)1 << 31 || B >= (int64_t)1 << 31 ||
        B * P >= (int64_t)1 << 31 || B * P * T >= (int64_t)1 << 40)
        return fail(LBI_ERR_UNSUPPORTED, "%s: too many elements", who);
    return LBI_OK;
}

}  // namespace
}  // namespace rotary
}  // namespace lbi

extern "C" int lbi_rotary(const void* qkv, const float* cos, const float* sin, const void* positions, void* q, void* k, int64_t B, int64_t T, int64_t H,
                          int64_t Hkv, int64_t D, int64_t R, int64_t table, int64_t stride_b, int64_t stride_t, int positions_wide, int interleaved,
                          int dtype, void* stream) {
    using namespace lbi;
    using namespace lbi::rotary;
    clear_error();
    if (int bad = check("lbi_rotary", B, 1, T, H, Hkv, D, R, table, positions, dtype)) return bad;
    if (!B || !T) return LBI_OK;
    if (!qkv || !q || !k || (R && table && (!cos || !sin))) return fail(LBI_ERR_INVALID, "lbi_rotary: null pointer");
    const size_t size = dtype_size(dtype);
    if (off(qkv, size) || off(q, size) || off(k, size) || off(cos, 4) || off(sin, 4) || off(positions, positions_wide ? 8 : 4))
        return fail(LBI_ERR_INVALID, "lbi_rotary: a tensor is not aligned to its elements");
    Call c{};
    c.q = qkv, c.out = q, c.out_k = k, c.cos = cos, c.sin = sin, c.positions = positions;
    c.stride_b = stride_b, c.stride_t = stride_t, c.table = table, c.positions_wide = positions_wide != 0;
    c.P = 1, c.T = (int)T, c.H = (int)H, c.Hkv = (int)Hkv, c.shared = 1, c.D = (int)D, c.R = (int)R, c.interleaved = interleaved != 0;
    return by_type<false>(c, B * T, dtype, static_cast<hipStream_t>(stream));
}

extern "C" int lbi_rotary_pullback(const void* dq, const void* dk, const void* dv, const float* cos, const float* sin, const void* positions, void* g_qkv,
                                   int64_t B, int64_t P, int64_t T, int64_t H, int64_t Hkv, int64_t kv_heads, int64_t D, int64_t R, int64_t table,
                                   int positions_wide, int interleaved, int dtype, void* stream) {
    using namespace lbi;
    using namespace lbi::rotary;
    clear_error();
    if (int bad = check("lbi_rotary_pullback", B, P, T, H, Hkv, D, R, table, positions, dtype)) return bad;
    if (kv_heads != H && kv_heads != Hkv)
        return fail(LBI_ERR_INVALID, "lbi_rotary_pullback: dk and dv of %lld heads, neither H=%lld nor Hkv=%lld", (long long)kv_heads, (long long)H, (long long)Hkv);
    if (!B || !P || !T) return LBI_OK;
    if (!dq || !dk || !dv || !g_qkv || (R && table && (!cos || !sin))) return fail(LBI_ERR_INVALID, "lbi_rotary_pullback: null pointer");
    const size_t size = dtype_size(dtype);
    if (off(dq, size) || off(dk, size) || off(dv, size) || off(g_qkv, size) || off(cos, 4) || off(sin, 4) || off(positions, positions_wide ? 8 : 4))
        return fail(LBI_ERR_INVALID, "lbi_rotary_pullback: a tensor is not aligned to its elements");
    Call c{};
    c.q = dq, c.k = dk, c.v = dv, c.out = g_qkv, c.cos = cos, c.sin = sin, c.positions = positions;
    c.table = table, c.positions_wide = positions_wide != 0;
    c.P = (int)P, c.T = (int)T, c.H = (int)H, c.Hkv = (int)Hkv, c.shared = (int)(kv_heads / Hkv), c.D = (int)D, c.R = (int)R, c.interleaved = interleaved != 0;
    return by_type<true>(c, B * P * T, dtype, static_cast<hipStream_t>(stream));
}
