// The kernels of linear attention over chunks (lbi_linear_attn.h has the mathematics).
//
// A workgroup takes the chunks of one segment of one chain one after the other.  Each of its waves holds 16 columns of the state, in fp32 and in
// registers for the whole segment, and never exchanges them: the accumulators of X, packed, are the operand of the next readout.
//   1  waves 0 ... 3: the scores of 16 tokens i each with all j <= i, times l^(i-j), rounded to 16 bits into LDS
//   2  every wave: out^T of its columns = X^T a^T, times l^(i+1), plus c^T scores^T
//   3  every wave: X = l^64 X + b^T (l^(63-j) c), the decayed c in planes of 16 bits that add up to 16 or 24 significant bits (22 in half precision)
// The next chunk's tiles are on their way into the other half of the LDS meanwhile, past the registers.
#pragma once

#include "lbi_linear_attn.h"
#include "lbi_scan_planes.h"

namespace lbi {
namespace linear_attn {

constexpr float LOG2E = 1.4426950408889634f;
constexpr unsigned NOWHERE = 0x80000000u;  // an offset past the end of every buffer

// Everything that this wave has in LDS is there, for all waves; transfers from and to memory stay under way.
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

template <typename T> struct Mma16;
template <> struct Mma16<bf16_raw> {
    static __device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
};
template <> struct Mma16<_Float16> {
    static __device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
};

// The power of two that brings values of up to `most` below 2^14, as (down, up): half precision ends at 65504, and the sums of linear
// attention, which no softmax bounds, do not.
struct Pow2 { float down, up; };
__device__ __forceinline__ Pow2 into_range(float most) {
    int e = (int)(__float_as_uint(most) >> 23) - 127 - 13;
    e = e < -100 ? -100 : e > 100 ? 0 : e;  // infinities and NaN as they are
    return Pow2{__uint_as_float((unsigned)(127 - e) << 23), __uint_as_float((unsigned)(127 + e) << 23)};
}
__device__ __forceinline__ float over_wave_max(float x) {
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) x = fmaxf(x, __shfl_xor(x, off, 64));
    return x;
}

__device__ __forceinline__ int length_of(const Call& call, int b) {
    if (!call.lengths) return call.T;
    const long long n = call.lengths_wide ? static_cast<const long long*>(call.lengths)[b] : (long long)static_cast<const int*>(call.lengths)[b];
    return n < 0 ? 0 : n > call.T ? call.T : (int)n;
}
// log_decay of a head; -inf (no memory at all) as a number whose product with 0 is 0
__device__ __forceinline__ float rate_of(const Call& call, int h) {
    const float l = call.log_decay[h];
    return l < -1e30f ? -1e30f : l;
}

// A tile of 64 tokens, rows of DIM 16-bit elements in LDS (16-byte pieces, swizzled as in lbi_attn_mfma.h).  VEC: by transfers of 16 bytes past the
// registers, zeros past the end of a row and behind the last token; otherwise, rows that start on any element, an element at a time.
template <typename T, int DIM, int THREADS, bool VEC> struct Tile {
    static constexpr int PIECES = DIM / 8, N = CHUNK * PIECES / THREADS;
    const T* base;
    int64_t st;
    int dim;
    unsigned full[N];  // offsets of this lane's pieces from the first token in memory of a whole chunk
    __device__ __forceinline__ unsigned piece_of(int u, int count, bool reverse) const {
        const int id = u * THREADS + (int)threadIdx.x, r = id / PIECES, slot = id % PIECES;
        const int chunk = tile_off<DIM>(r, slot) / 16 % PIECES;  // the swizzle is its own inverse
        const int64_t at = (int64_t)(reverse ? count - 1 - r : r) * st + chunk * 8;
        return r < count && chunk * 8 < dim ? (unsigned)(at * 2) : NOWHERE;
    }
    __device__ __forceinline__ Tile(const T* base_, int64_t st_, int dim_, bool reverse) : base(base_), st(st_), dim(dim_) {
        if constexpr (VEC)
#pragma unroll
            for (int u = 0; u < N; ++u) full[u] = piece_of(u, CHUNK, reverse);
    }
    // local tokens first ... first + count - 1 of the n that count
    __device__ __forceinline__ void bring(char* tile, unsigned tile_at, bool reverse, int n, int first, int count) const {
        const T* from = base + (int64_t)(reverse ? n - first - count : first) * st;
        if constexpr (VEC) {
            const auto source = scan_planes::rows(from, 0x7fffffffu);
            const unsigned to = tile_at + (threadIdx.x >> 6) * 1024;
#pragma unroll
            for (int u = 0; u < N; ++u) {
                unsigned from_at = full[u];
                if (__builtin_expect(count < CHUNK, 0)) from_at = piece_of(u, count, reverse);
                scan_planes::dma16(source, from_at, 0, to + u * THREADS * 16);
            }
        } else {
#pragma unroll
            for (int u = 0; u < N; ++u) {
                const int id = u * THREADS + (int)threadIdx.x, r = id / PIECES, c = id % PIECES * 8;
                const unsigned short* raw = reinterpret_cast<const unsigned short*>(from + (int64_t)(reverse ? count - 1 - r : r) * st + c);
                u32x4 words = {0, 0, 0, 0};
                if (r < count)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        words[e] = (c + 2 * e < dim ? raw[2 * e] : 0u) | (c + 2 * e + 1 < dim ? (unsigned)raw[2 * e + 1] << 16 : 0u);
                *reinterpret_cast<u32x4*>(tile + tile_off<DIM>(r, c / 8)) = words;
            }
        }
    }
};

// eight neighbouring elements of row r
template <int DIM> __device__ __forceinline__ u32x4 nat(const char* tile, int r, int chunk) {
    return *reinterpret_cast<const u32x4*>(tile + tile_off<DIM>(r, chunk));
}
// elements 4 g ... 4 g + 3 and 16 + 4 g ... of the 32 from column 32 ks on: the order in which accumulators hold the rows of two tiles
template <int DIM> __device__ __forceinline__ u32x4 split(const char* tile, int r, int ks, int g) {
    const u32x2 lo = *reinterpret_cast<const u32x2*>(tile + tile_off<DIM>(r, 4 * ks + (g >> 1)) + 8 * (g & 1));
    const u32x2 hi = *reinterpret_cast<const u32x2*>(tile + tile_off<DIM>(r, 4 * ks + 2 + (g >> 1)) + 8 * (g & 1));
    return u32x4{lo[0], lo[1], hi[0], hi[1]};
}
// rows row0 ... row0 + 7 of column col0 + lane % 16
template <int DIM> __device__ __forceinline__ u32x4 turned(const char* tile, int row0, int col0) {
    const int s = threadIdx.x & 15, chunk = (col0 >> 3) + ((s & 3) >> 1), sub = (s & 1) << 3, row = row0 + (s >> 2);
    typedef __attribute__((address_space(3))) attn_mfma::s16x4* lds_ptr;
    const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(tile + tile_off<DIM>(row, chunk) + sub)));
    const u32x2 hi = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(tile + tile_off<DIM>(row + 4, chunk) + sub)));
    return u32x4{lo[0], lo[1], hi[0], hi[1]};
}

// unit -> (chain, sequence, direction, head, segment): the workgroups that read the same tensors next to each other on one XCD
struct Unit { int chain, b, p, h, segment, number; };
__device__ __forceinline__ bool unit_of(const Call& call, int segments, Unit& u) {
    const int total = call.chains * call.B * call.P * call.H * segments, per = (int)(gridDim.x >> 3);
    int id = (int)(blockIdx.x & 7) * per + (int)(blockIdx.x >> 3);
    if (id >= total) return false;
    u.chain = id % call.chains;
    id /= call.chains;
    u.segment = id % segments;
    id /= segments;
    u.p = id % call.P;
    id /= call.P;
    u.h = id % call.H;
    u.b = id / call.H;
    u.number = ((u.chain * call.B + u.b) * call.P + u.p) * call.H + u.h;
    return true;
}

template <int DA, int DC, bool OUT> constexpr int stage_bytes() { return CHUNK * 2 * ((OUT ? 2 : 1) * DA + DC); }
template <int DA, int DC, bool OUT> constexpr int lds_bytes() { return 2 * stage_bytes<DA, DC, OUT>() + (OUT ? CHUNK * CHUNK * 2 : 0); }

// OUT false: only the state that a segment leaves behind, from zero, into its slot.
template <typename T, int DA, int DC, bool VEC, bool OUT, int PLANES>
__global__ __launch_bounds__(4 * DC, 2) void chunk_kernel(Call call) {
    constexpr bool HALF = std::is_same_v<T, _Float16>;
    constexpr int THREADS = 4 * DC, KS = DA / 32, MT = DA / 16, STAGE = stage_bytes<DA, DC, OUT>();
    extern __shared__ __align__(16) char lds[];  // two of: b, c, a; then the scores
    __shared__ float score_up[4];
    char* const tp = lds + 2 * STAGE;
    Unit u;
    if (!unit_of(call, OUT ? call.segments : call.segments - 1, u)) return;
    const Chain& ch = call.chain[u.chain];
    const int n = length_of(call, u.b), w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), m = threadIdx.x & 15, g = (threadIdx.x >> 4) & 3;
    const int begin = u.segment * call.segment, end = begin + call.segment < n ? begin + call.segment : n;  // of the tokens that count
    auto at = [&](const View& v) { return static_cast<const T*>(v.p) + u.b * v.sb + u.p * v.sp + (u.h / v.group) * v.sh; };
    const bool reverse = ch.reverse != 0;
    const float rate = rate_of(call, u.h), rate2 = rate * LOG2E;
    const int shift = ch.shift, Da = ch.Da, Dc = ch.Dc, col = 16 * w + m;

    const Tile<T, DA, THREADS, VEC> a(OUT ? at(ch.a) : nullptr, ch.a.st, Da, reverse), b(at(ch.b), ch.b.st, Da, reverse);
    const Tile<T, DC, THREADS, VEC> c(at(ch.c), ch.c.st, Dc, reverse);
    const unsigned lds0 = (unsigned)(size_t)(__attribute__((address_space(3))) char*)lds;
    auto bring = [&](int stage, int from) {
        const int count = end - from < CHUNK ? end - from : CHUNK, to = stage * STAGE;
        b.bring(lds + to, lds0 + to, reverse, n, from, count);
        c.bring(lds + to + CHUNK * 2 * DA, lds0 + to + CHUNK * 2 * DA, reverse, n, from, count);
        if constexpr (OUT) a.bring(lds + to + CHUNK * 2 * (DA + DC), lds0 + to + CHUNK * 2 * (DA + DC), reverse, n, from, count);
    };
    if (begin < end) bring(0, begin);

    // l to the power of tokens apart, as products of l^0 ... l^31 of this lane's place and of l^16, l^32, l^48
    const float l16 = exp2f(rate2 * 16.0f), l32 = exp2f(rate2 * 32.0f), l48 = exp2f(rate2 * 48.0f);
    const float read0 = exp2f(rate2 * (float)(m + 1 - shift));
    float near[4], far[4], keep[8];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int apart = m - 4 * g - r;
        near[r] = exp2f(rate2 * (float)(apart < 0 ? 0 : apart));
        far[r] = exp2f(rate2 * (float)(16 + apart));
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) keep[e] = exp2f(rate2 * (float)(31 - 8 * g - e + shift));
    float fade = expm1f(rate * (float)CHUNK);  // X + X (l^64 - 1) keeps what rounding l^64 near 1 would add up over many chunks

    f32x4 x[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) x[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    // This wave's columns of a state in memory, strides in elements: all asked for before any is waited for, zeros past the dimensions.
    auto place = [&](int i, int r, unsigned sr, unsigned sc) __attribute__((always_inline)) {
        const int row = 16 * i + 4 * g + r;
        return row < Da && col < Dc ? 4 * (row * sr + col * sc) : NOWHERE;
    };
    auto state_at = [&](const float* p, unsigned sr, unsigned sc, auto&& use) __attribute__((always_inline)) {
        const auto from = scan_planes::rows(p, 0x7fffffffu);
        float v[MT][4];
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) v[i][r] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(from, place(i, r, sr, sc), 0, 0));
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) x[i][r] = use(x[i][r], v[i][r]);
    };
    if constexpr (OUT) {
        if (ch.first.p && (u.segment == 0 || !call.joined)) {
            const float scale = ch.first_scale;
            state_at(ch.first.p + u.b * ch.first.sb + u.p * ch.first.sp + u.h * ch.first.sh, (unsigned)ch.first.sr, (unsigned)ch.first.sc,
                     [&](float, float v) __attribute__((always_inline)) { return v * scale; });
        }
        const float* slots = call.segment_states + (int64_t)u.number * (call.segments - 1) * Da * Dc;
        for (int s = call.joined ? u.segment - 1 : 0; s >= 0 && s < u.segment; ++s) {  // what the segments before add, the first one first
            int tokens = n - s * call.segment;
            tokens = tokens < 0 ? 0 : tokens > call.segment ? call.segment : tokens;
            const float left = call.joined ? -1.0f : expm1f(rate * (float)tokens);
            state_at(slots + (int64_t)s * Da * Dc, (unsigned)Dc, 1, [&](float x_, float v) __attribute__((always_inline)) { return fmaf(x_, left, x_) + v; });
        }
    }
    scan_planes::wait_vm<0>();

    const unsigned out_at = (unsigned)(((int64_t)(reverse ? 15 - m : m) * ch.out.st + 16 * w + 4 * g) * 2), out_tile = (unsigned)(32 * ch.out.st);
    int stage = 0, from = begin;
    auto chunk = [&](auto whole_tag) __attribute__((always_inline)) {
        constexpr bool WHOLE = decltype(whole_tag)::value;  // 64 tokens
        lds_barrier();  // this chunk's tiles are there, and everyone is done with the ones before
        if (WHOLE && from + CHUNK < end) bring(stage ^ 1, from + CHUNK);
        const char *tb = lds + stage * STAGE, *tc = tb + CHUNK * 2 * DA, *ta = tc + CHUNK * 2 * DC;
        const int count = WHOLE ? CHUNK : end - from;

        f32x4 acc[4];
        Pow2 state_by = {1.0f, 1.0f};
        if constexpr (OUT) {
            if (w < 4) {
                f32x4 s[4];
#pragma unroll
                for (int t = 0; t < 4; ++t) s[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    const u32x4 mine = nat<DA>(ta, 16 * w + m, 4 * ks + g);
#pragma unroll
                    for (int t = 0; t < 4; ++t) s[t] = Mma16<T>::mma(nat<DA>(tb, 16 * t + m, 4 * ks + g), mine, s[t]);
                }
                float most = 0.0f;
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    const float more = w - t == 2 ? l16 : w - t == 3 ? l32 : 1.0f;
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        s[t][r] = t < w ? s[t][r] * (far[r] * more) : t == w && m >= 4 * g + r ? s[t][r] * near[r] : 0.0f;
                        if constexpr (HALF) most = fmaxf(most, fabsf(s[t][r]));
                    }
                }
                if constexpr (HALF) {
                    const Pow2 by = into_range(over_wave_max(most));
                    if ((threadIdx.x & 63) == 0) score_up[w] = by.up;
#pragma unroll
                    for (int t = 0; t < 4; ++t) s[t] *= by.down;
                }
#pragma unroll
                for (int t = 0; t < 4; ++t)
                    *reinterpret_cast<u32x2*>(tp + tile_off<CHUNK>(16 * w + m, 2 * t + (g >> 1)) + 8 * (g & 1)) =
                        u32x2{Mma<T>::pack2(s[t][0], s[t][1]), Mma<T>::pack2(s[t][2], s[t][3])};
            }
            // what the state in front of the chunk gives
            if constexpr (HALF) {
                float most = 0.0f;
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r) most = fmaxf(most, fabsf(x[i][r]));
                state_by = into_range(over_wave_max(most));
            }
#pragma unroll
            for (int t = 0; t < 4; ++t) acc[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                const f32x4 lo = x[2 * ks] * state_by.down, hi = x[2 * ks + 1] * state_by.down;
                const u32x4 state = {Mma<T>::pack2(lo[0], lo[1]), Mma<T>::pack2(lo[2], lo[3]), Mma<T>::pack2(hi[0], hi[1]), Mma<T>::pack2(hi[2], hi[3])};
#pragma unroll
                for (int t = 0; t < 4; ++t) acc[t] = Mma16<T>::mma(state, split<DA>(ta, 16 * t + m, ks, g), acc[t]);
            }
        }

        u32x4 raws[2];  // the chunk's c: as it is for the scores, decayed for the state
        if constexpr (!WHOLE) fade = expm1f(rate * (float)count);
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) x[i][r] = fmaf(x[i][r], fade, x[i][r]);
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            const u32x4 raw = turned<DC>(tc, 32 * ks + 8 * g, 16 * w);
            if constexpr (OUT) raws[ks] = raw;
            float left[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int tokens = count - 1 - (32 * ks + 8 * g + e);
                left[e] = !WHOLE ? exp2f(rate2 * (float)((tokens < 0 ? 0 : tokens) + shift)) : ks == 0 ? keep[e] * l32 : keep[e];
            }
            u32x4 plane[PLANES];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float lo = Mma<T>::lo(raw[e]) * left[2 * e], hi = Mma<T>::hi(raw[e]) * left[2 * e + 1];
#pragma unroll
                for (int q = 0; q < PLANES; ++q) {
                    const unsigned word = Mma<T>::pack2(lo, hi);
                    plane[q][e] = word;
                    lo -= Mma<T>::lo(word), hi -= Mma<T>::hi(word);
                }
            }
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                const u32x4 bt = turned<DA>(tb, 32 * ks + 8 * g, 16 * i);
#pragma unroll
                for (int q = PLANES - 1; q >= 0; --q) x[i] = Mma16<T>::mma(bt, plane[q], x[i]);
            }
        }

        if constexpr (OUT) {
            lds_barrier();  // the scores are there
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                float by = read0 * (t == 0 ? 1.0f : t == 1 ? l16 : t == 2 ? l32 : l48);
                if constexpr (HALF) by *= state_by.up / score_up[t];
                acc[t] *= by;
            }
#pragma unroll
            for (int ks = 0; ks < 2; ++ks)
#pragma unroll
                for (int t = 2 * ks; t < 4; ++t) acc[t] = Mma16<T>::mma(raws[ks], nat<CHUNK>(tp, 16 * t + m, 4 * ks + g), acc[t]);
            T* const out = const_cast<T*>(at(ch.out)) + (int64_t)(reverse ? n - from - count : from) * ch.out.st;
            const auto to = scan_planes::rows(out, 0x7fffffffu);
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const int i = 16 * t + m, row = reverse ? count - 1 - i : i, first = 16 * w + 4 * g;
                float by = ch.scale;
                if constexpr (HALF) by *= score_up[t];
                const u32x2 words = {Mma<T>::pack2(acc[t][0] * by, acc[t][1] * by), Mma<T>::pack2(acc[t][2] * by, acc[t][3] * by)};
                if constexpr (VEC && WHOLE) {  // each wave has the same number of stores under way, whatever there is to store
                    __builtin_amdgcn_raw_buffer_store_b64(words, to, first < Dc ? out_at : NOWHERE, out_tile * (reverse ? 3 - t : t), 0);
                } else if constexpr (VEC) {
                    __builtin_amdgcn_raw_buffer_store_b64(words, to, i < count && first < Dc ? (unsigned)(((int64_t)row * ch.out.st + first) * 2) : NOWHERE, 0, 0);
                } else if (i < count) {
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (first + r < Dc) reinterpret_cast<unsigned short*>(out + row * ch.out.st)[first + r] = (unsigned short)(words[r / 2] >> (16 * (r % 2)));
                }
            }
        }
        scan_planes::wait_vm<OUT && VEC ? 4 : 0>();  // the next tiles; this chunk's stores may still be under way
    };
    for (; from + CHUNK <= end; from += CHUNK, stage ^= 1) chunk(std::true_type{});
    if (from < end) chunk(std::false_type{});
    if constexpr (OUT) {  // rows behind the sequence
        T* out = const_cast<T*>(at(ch.out));
        const int stop = begin + call.segment < call.T ? begin + call.segment : call.T, past = begin > n ? begin : n;
        for (int64_t i = (int64_t)past * Dc + threadIdx.x; i < (int64_t)stop * Dc; i += THREADS)
            reinterpret_cast<unsigned short*>(out)[i / Dc * ch.out.st + i % Dc] = 0;
    }
    auto leave = [&](float* p, unsigned sr, unsigned sc, float scale) __attribute__((always_inline)) {
        const auto to = scan_planes::rows(p, 0x7fffffffu);
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float v = x[i][r] * scale;
                __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(v), to, place(i, r, sr, sc), 0, 0);
            }
    };
    if constexpr (OUT) {
        if (ch.last.p && u.segment == call.segments - 1)
            leave(ch.last.p + u.b * ch.last.sb + u.p * ch.last.sp + u.h * ch.last.sh, (unsigned)ch.last.sr, (unsigned)ch.last.sc, ch.last_scale);
    } else {
        leave(call.segment_states + ((int64_t)u.number * (call.segments - 1) + u.segment) * Da * Dc, (unsigned)Dc, 1, 1.0f);
    }
}

// Slot s of each unit holds what segment s adds; they become the states behind the segments.  BATCH slots are asked for at once.
template <typename T> __global__ __launch_bounds__(256) void join_kernel(Call call) {
    constexpr int BATCH = 8;
    const int of_chain = call.B * call.P * call.H, slots = call.segments - 1;
    int id = (int)blockIdx.y;
    const int number = id;
    const Chain& ch = call.chain[id / of_chain];
    id %= of_chain;
    const int h = id % call.H, p = id / call.H % call.P, b = id / call.H / call.P;
    const int e = (int)(blockIdx.x * 256 + threadIdx.x), count = ch.Da * ch.Dc;
    if (e >= count) return;
    const int n = length_of(call, b);
    const float rate = rate_of(call, h), whole = expm1f(rate * (float)call.segment);
    float* slot = call.segment_states + (int64_t)number * slots * count + e;
    float x = 0.0f;
    if (ch.first.p) x = ch.first.p[b * ch.first.sb + p * ch.first.sp + h * ch.first.sh + e / ch.Dc * ch.first.sr + e % ch.Dc * ch.first.sc] * ch.first_scale;
    for (int from = 0; from < slots; from += BATCH) {
        float more[BATCH];
#pragma unroll
        for (int s = 0; s < BATCH; ++s) more[s] = slot[(int64_t)(from + s < slots ? from + s : slots - 1) * count];
#pragma unroll
        for (int s = 0; s < BATCH; ++s) {
            if (from + s >= slots) break;
            const int left = n - (from + s) * call.segment;
            const float fade = left >= call.segment ? whole : expm1f(rate * (float)(left < 0 ? 0 : left));
            x = fmaf(x, fade, x) + more[s];
            slot[(int64_t)(from + s) * count] = x;
        }
    }
}

}  // namespace linear_attn
}  // namespace lbi
