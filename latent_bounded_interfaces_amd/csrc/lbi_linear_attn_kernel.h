// The kernels of linear attention over chunks (lbi_linear_attn.h has the mathematics).
//
// A workgroup takes the chunks of one segment of one chain one after the other; its four waves hold a quarter of the state's columns each, in
// fp32 and in registers for the whole segment, and never exchange it: the accumulators of X, packed, are the operand of the next readout.
//   1  wave w: pairs of tokens i = 16 w ... 16 w + 15 with all j <= i, times l^(i-j), rounded to 16 bits into LDS
//   2  every wave: out^T of its columns = X^T a^T, times l^(i+1), plus c^T pairs^T
//   3  every wave: X = l^64 X + b^T (l^(63-j) c), the decayed c in planes of 16 bits whose sum has 16 (22 in half precision) significant bits
// The next chunk's tiles are on their way in registers meanwhile.
#pragma once

#include "lbi_linear_attn.h"

namespace lbi {
namespace linear_attn {

constexpr float LOG2E = 1.4426950408889634f;

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

// Tile of 64 tokens x W elements: rows of 16-byte pieces, DIM / 8 of them, from tensors whose rows start on any element (!VEC: and whose
// widths are any).
template <typename T, int DIM, bool VEC> struct Tile {
    static constexpr int PIECES = DIM / 8, N = CHUNK * PIECES / 256;
    u32x4 regs[N];
    // local tokens first ... first + 63; what is at or past `end` and columns past `dim` are zero
    __device__ __forceinline__ void fetch(const T* base, int64_t st, bool reverse, int n, int first, int end, int dim) {
        const T* from = base + (reverse ? (int64_t)(n - first - CHUNK) : (int64_t)first) * st;
#pragma unroll
        for (int u = 0; u < N; ++u) {
            const int id = threadIdx.x + 256 * u, r = id / PIECES, c = id % PIECES * 8;
            const T* p = from + (int64_t)(reverse ? CHUNK - 1 - r : r) * st + c;
            regs[u] = u32x4{0, 0, 0, 0};
            if (first + r < end && c < dim) {
                if constexpr (VEC) {
                    regs[u] = *reinterpret_cast<const u32x4*>(p);
                } else {
                    const unsigned short* raw = reinterpret_cast<const unsigned short*>(p);
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        regs[u][e] = (c + 2 * e < dim ? raw[2 * e] : 0u) | (c + 2 * e + 1 < dim ? (unsigned)raw[2 * e + 1] << 16 : 0u);
                }
            }
        }
    }
    __device__ __forceinline__ void commit(char* tile) const {
#pragma unroll
        for (int u = 0; u < N; ++u) {
            const int id = threadIdx.x + 256 * u;
            *reinterpret_cast<u32x4*>(tile + tile_off<DIM>(id / PIECES, id % PIECES)) = regs[u];
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

// OUT false: only the state that a segment leaves behind, from zero, into the slot of the next one.
template <typename T, int DA, int DC, bool VEC, bool OUT, int PLANES>
__global__ __launch_bounds__(256, 2) void chunk_kernel(Call call) {
    constexpr bool HALF = std::is_same_v<T, _Float16>;
    constexpr int KS = DA / 32, MT = DA / 16, NT = DC / 64;  // steps and tiles of the state: rows, this wave's columns
    __shared__ __align__(16) char lds[(OUT ? CHUNK * DA * 2 : 0) + CHUNK * DA * 2 + CHUNK * DC * 2 + (OUT ? CHUNK * CHUNK * 2 : 0)];
    __shared__ float pair_up[4];
    char* const tb = lds;
    char* const tc = tb + CHUNK * DA * 2;
    char* const ta = tc + CHUNK * DC * 2;
    char* const tp = ta + CHUNK * DA * 2;
    Unit u;
    if (!unit_of(call, OUT ? call.segments : call.segments - 1, u)) return;
    const Chain& ch = call.chain[u.chain];
    const int n = length_of(call, u.b), w = threadIdx.x >> 6, m = threadIdx.x & 15, g = (threadIdx.x >> 4) & 3;
    const int begin = u.segment * call.segment, end = begin + call.segment < n ? begin + call.segment : n;  // of the tokens that count
    const int stop = OUT ? (begin + call.segment < call.T ? begin + call.segment : call.T) : end;           // of the rows written
    auto at = [&](const View& v) { return static_cast<const T*>(v.p) + u.b * v.sb + u.p * v.sp + (u.h / v.group) * v.sh; };
    const T *a = OUT ? at(ch.a) : nullptr, *b = at(ch.b), *c = at(ch.c);
    const bool reverse = ch.reverse != 0;
    const float rate = rate_of(call, u.h), rate2 = rate * LOG2E;
    const int shift = ch.shift, Da = ch.Da, Dc = ch.Dc;
    const int col0 = w * (DC / 4);

    float pair[4][4], read[4], keep[2][8];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int apart = 16 * w + m - (16 * t + 4 * g + r);
            pair[t][r] = apart < 0 ? 0.0f : exp2f(rate2 * (float)apart);
        }
        read[t] = exp2f(rate2 * (float)(16 * t + m + 1 - shift));
    }
    auto weigh = [&](int count) {  // of a chunk of `count` tokens
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int left = count - 1 - (32 * ks + 8 * g + e);
                keep[ks][e] = exp2f(rate2 * (float)((left < 0 ? 0 : left) + shift));
            }
    };
    weigh(CHUNK);
    float fade = expm1f(rate * (float)CHUNK);  // X + X (l^64 - 1) keeps what rounding l^64 near 1 would add up over many chunks

    f32x4 x[MT][NT];
    const float* first = OUT ? (call.segments > 1 ? call.segment_states : ch.first.p) : nullptr;
    if (OUT && first) {
        int64_t sr = Dc, sc = 1;
        float factor = 1.0f;
        if (call.segments > 1) {
            first += ((int64_t)u.number * call.segments + u.segment) * Da * Dc;
        } else {
            first += u.b * ch.first.sb + u.p * ch.first.sp + u.h * ch.first.sh;
            sr = ch.first.sr, sc = ch.first.sc, factor = ch.first_scale;
        }
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int row = 16 * i + 4 * g + r, col = col0 + 16 * j + m;
                    x[i][j][r] = row < Da && col < Dc ? first[row * sr + col * sc] * factor : 0.0f;
                }
    } else {
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j) x[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    if constexpr (OUT) {  // pairs of later tokens stay zero
        for (int i = threadIdx.x; i < CHUNK * CHUNK * 2 / 16; i += 256) reinterpret_cast<u32x4*>(tp)[i] = u32x4{0, 0, 0, 0};
    }

    Tile<T, DA, VEC> na, nb;
    Tile<T, DC, VEC> nc;
    auto bring = [&](int from) {
        if constexpr (OUT) na.fetch(a, ch.a.st, reverse, n, from, end, Da);
        nb.fetch(b, ch.b.st, reverse, n, from, end, Da);
        nc.fetch(c, ch.c.st, reverse, n, from, end, Dc);
    };
    if (begin < end) bring(begin);
    for (int from = begin; from < end; from += CHUNK) {
        __syncthreads();  // everyone is done with the tiles
        if constexpr (OUT) na.commit(ta);
        nb.commit(tb);
        nc.commit(tc);
        __syncthreads();
        if (from + CHUNK < end) bring(from + CHUNK);
        const int count = end - from < CHUNK ? end - from : CHUNK;

        f32x4 acc[OUT ? NT : 1][4];
        float bring_up = 1.0f;
        if constexpr (OUT) {
            f32x4 s[4];
#pragma unroll
            for (int t = 0; t < 4; ++t) s[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                const u32x4 mine = nat<DA>(ta, 16 * w + m, 4 * ks + g);
#pragma unroll
                for (int t = 0; t < 4; ++t)
                    if (t <= w) s[t] = Mma16<T>::mma(nat<DA>(tb, 16 * t + m, 4 * ks + g), mine, s[t]);
            }
            float down = 1.0f;
            if constexpr (HALF) {
                float most = 0.0f;
#pragma unroll
                for (int t = 0; t < 4; ++t)
#pragma unroll
                    for (int r = 0; r < 4; ++r) most = fmaxf(most, fabsf(s[t][r] * pair[t][r]));
                const Pow2 by = into_range(over_wave_max(most));
                down = by.down;
                if ((threadIdx.x & 63) == 0) pair_up[w] = by.up;
            }
#pragma unroll
            for (int t = 0; t < 4; ++t)
                if (t <= w) {
                    float v[4];
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        v[r] = 16 * w + m < 16 * t + 4 * g + r ? 0.0f : s[t][r] * pair[t][r];
                        if constexpr (HALF) v[r] *= down;
                    }
                    *reinterpret_cast<u32x2*>(tp + tile_off<CHUNK>(16 * w + m, 2 * t + (g >> 1)) + 8 * (g & 1)) =
                        u32x2{Mma<T>::pack2(v[0], v[1]), Mma<T>::pack2(v[2], v[3])};
                }
            // what the state in front of the chunk gives
            if constexpr (HALF) {
                float most = 0.0f;
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int j = 0; j < NT; ++j)
#pragma unroll
                        for (int r = 0; r < 4; ++r) most = fmaxf(most, fabsf(x[i][j][r]));
                const Pow2 by = into_range(over_wave_max(most));
                down = by.down;
                bring_up = by.up;
            }
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int t = 0; t < 4; ++t) acc[j][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                u32x4 state[NT];
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    const f32x4 lo = x[2 * ks][j] * down, hi = x[2 * ks + 1][j] * down;
                    state[j] = u32x4{Mma<T>::pack2(lo[0], lo[1]), Mma<T>::pack2(lo[2], lo[3]), Mma<T>::pack2(hi[0], hi[1]), Mma<T>::pack2(hi[2], hi[3])};
                }
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    const u32x4 mine = split<DA>(ta, 16 * t + m, ks, g);
#pragma unroll
                    for (int j = 0; j < NT; ++j) acc[j][t] = Mma16<T>::mma(state[j], mine, acc[j][t]);
                }
            }
            __syncthreads();  // the pairs are there
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                float by = read[t];
                if constexpr (HALF) by *= bring_up / pair_up[t];
#pragma unroll
                for (int j = 0; j < NT; ++j) acc[j][t] *= by;
            }
        }

        // the chunk's c: as it is for the pairs, decayed for the state
        if (count < CHUNK) {
            weigh(count);
            fade = expm1f(rate * (float)count);
        }
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r) x[i][j][r] = fmaf(x[i][j][r], fade, x[i][j][r]);
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            u32x4 plane[PLANES][NT];
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const u32x4 raw = turned<DC>(tc, 32 * ks + 8 * g, col0 + 16 * j);
                if constexpr (OUT)
#pragma unroll
                    for (int t = 2 * ks; t < 4; ++t) acc[j][t] = Mma16<T>::mma(raw, nat<CHUNK>(tp, 16 * t + m, 4 * ks + g), acc[j][t]);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float lo = Mma<T>::lo(raw[e]) * keep[ks][2 * e], hi = Mma<T>::hi(raw[e]) * keep[ks][2 * e + 1];
#pragma unroll
                    for (int q = 0; q < PLANES; ++q) {
                        const unsigned word = Mma<T>::pack2(lo, hi);
                        plane[q][j][e] = word;
                        lo -= Mma<T>::lo(word), hi -= Mma<T>::hi(word);
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                const u32x4 bt = turned<DA>(tb, 32 * ks + 8 * g, 16 * i);
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int q = PLANES - 1; q >= 0; --q) x[i][j] = Mma16<T>::mma(bt, plane[q][j], x[i][j]);
            }
        }

        if constexpr (OUT) {
            T* out = const_cast<T*>(at(ch.out));
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const int i = from + 16 * t + m;
                float by = ch.scale;
                if constexpr (HALF) by *= pair_up[t];
                if (i < end) {
                    T* row = out + (int64_t)(reverse ? n - 1 - i : i) * ch.out.st;
#pragma unroll
                    for (int j = 0; j < NT; ++j) {
                        const int col = col0 + 16 * j + 4 * g;
                        const u32x2 words = {Mma<T>::pack2(acc[j][t][0] * by, acc[j][t][1] * by), Mma<T>::pack2(acc[j][t][2] * by, acc[j][t][3] * by)};
                        if constexpr (VEC) {
                            if (col < Dc) *reinterpret_cast<u32x2*>(row + col) = words;
                        } else {
#pragma unroll
                            for (int r = 0; r < 4; ++r)
                                if (col + r < Dc) reinterpret_cast<unsigned short*>(row)[col + r] = (unsigned short)(words[r / 2] >> (16 * (r % 2)));
                        }
                    }
                }
            }
        }
    }
    if constexpr (OUT) {  // rows behind the sequence
        T* out = const_cast<T*>(at(ch.out));
        const int past = begin > n ? begin : n;
        for (int64_t i = (int64_t)past * Dc + threadIdx.x; i < (int64_t)stop * Dc; i += 256)
            reinterpret_cast<unsigned short*>(out)[i / Dc * ch.out.st + i % Dc] = 0;
    }
    float* last = nullptr;
    int64_t sr = Dc, sc = 1;
    float factor = 1.0f;
    if constexpr (OUT) {
        if (ch.last.p && u.segment == call.segments - 1) {
            last = ch.last.p + u.b * ch.last.sb + u.p * ch.last.sp + u.h * ch.last.sh;
            sr = ch.last.sr, sc = ch.last.sc, factor = ch.last_scale;
        }
    } else {
        last = call.segment_states + ((int64_t)u.number * call.segments + u.segment + 1) * Da * Dc;
    }
    if (last) {
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int row = 16 * i + 4 * g + r, col = col0 + 16 * j + m;
                    if (row < Da && col < Dc) last[row * sr + col * sc] = x[i][j][r] * factor;
                }
    }
}

// Slot s + 1 of each unit holds what segment s adds; with the first state in slot 0 they become the states in front of the segments.
template <typename T> __global__ __launch_bounds__(256) void join_kernel(Call call) {
    const int of_chain = call.B * call.P * call.H;
    int id = (int)blockIdx.y;
    const int number = id;
    const Chain& ch = call.chain[id / of_chain];
    id %= of_chain;
    const int h = id % call.H, p = id / call.H % call.P, b = id / call.H / call.P;
    const int e = (int)(blockIdx.x * 256 + threadIdx.x), count = ch.Da * ch.Dc;
    if (e >= count) return;
    const int n = length_of(call, b);
    const float rate = rate_of(call, h);
    float* slot = call.segment_states + (int64_t)number * call.segments * count + e;
    float x = 0.0f;
    if (ch.first.p) x = ch.first.p[b * ch.first.sb + p * ch.first.sp + h * ch.first.sh + e / ch.Dc * ch.first.sr + e % ch.Dc * ch.first.sc] * ch.first_scale;
    for (int s = 0; s < call.segments; ++s) {
        const float more = s + 1 < call.segments ? slot[(int64_t)(s + 1) * count] : 0.0f;
        slot[(int64_t)s * count] = x;
        int tokens = n - s * call.segment;
        tokens = tokens < 0 ? 0 : tokens > call.segment ? call.segment : tokens;
        x = fmaf(x, expm1f(rate * (float)tokens), x) + more;
    }
}

}  // namespace linear_attn
}  // namespace lbi
