// The kernels of linear attention over chunks (lbi_linear_attn.h has the mathematics).
//
// A workgroup takes the chunks of one segment of one chain one after the other.  Each of its four waves holds a quarter of the state's columns, in
// fp32 and in registers for the whole segment, and never exchanges them: the accumulators of X, packed, are the operand of the next readout.
//   1  wave w: the scores of tokens i = 16 w ... 16 w + 15 with all j <= i, times l^(i-j), rounded to 16 bits into LDS
//   2  every wave: X^T a^T of its columns, the readout of the state in front of the chunk
//   3  behind a barrier: out^T = l^(i+1) readout + c^T scores^T, from registers and the scores alone
//   4  every wave: X = l^64 X + b^T (l^(63-j) c), the decayed c in planes of 16 bits that add up to 16 or 24 significant bits, while
//      the results go out
// Half precision ends at 65504 and 2^-24, so its operands are brought into range by powers of two: a query's scores, a column's copy of the state, and
// a column's decayed c (22 bits of those down to 2^-16 of the column's largest, 2^-38 of that below), each by its own.  The chunk's sum comes in the last one's
// power and joins X with it taken out, a readout goes from the second's into the first's.  Without, an fp32 state of values of 1e-5 was off by 0.002 to 0.005 and
// a column of 2^-39 of its neighbour was lost (us, without / with: 512 chains of 4096 tokens of 128 474 / 483, split ones 105 / 115, a basis of 4 587 / 622).
// Below 2^-38 of the largest of its sum an operand is lost all the same.
// The scores and the copy of the state are operands of 16 bits, one rounding each, as the inputs are: what they add to the results is as much as rounding the results
// does (2-norm of the error, bf16 2.35e-3 where that alone is 1.66e-3, half precision 2.9e-4 and 2.1e-4).  In two planes each, results are as near as that one
// rounding, at 44 more of 124 products a chunk (us, so / in one plane: 96 chains of 1024 tokens of 64 31 / 25, 64 of 4096 of 128 130 / 112, 512 521 / 487, the pullback below
// 636 / 510); the scores alone in two leave 2.17e-3 (28, 117, 489, 546).  Calls of one chunk, which lose nothing by it, take two.
// b has two tiles in LDS and the next chunk's comes in from the start of this one; a and c have one, which is free behind 2's barrier.  72 KB for heads of
// 128, so that two workgroups share a CU, whose vector work then runs beside the other's products.
//
// Bound by memory in long calls that fill the chip: 512 chains of 4096 tokens of 128 457 to 487 us, 4.4 to 4.7 TB/s, 1024 of 2048 of 64 235 us, 4.6 TB/s, of the 4.9 that
// a copy reaches.  The pullback of 4 directions for 4 x 16 heads of 4096 of 128, three chains each, takes 464 to 540 us, card by card (1.28 GB, 2.6 TB/s): 768 workgroups are one and a
// half rounds of the 512 that fit, and a chunk's 124 products and 400 vector instructions a wave take 159 and 129 us of the SIMDs in all.  All tiles
// asked for behind the last barrier had it at 541 us; a second tile of c instead of b's gained with one workgroup a CU
// and lost with two; eight waves of 16 columns, priorities of waves, results past the caches (4 to 40 % slower) did not pay.
#pragma once

#include "lbi_linear_attn.h"
#include "lbi_scan_planes.h"

namespace lbi {
namespace linear_attn {

constexpr float LOG2E = 1.4426950408889634f;
constexpr unsigned NOWHERE = 0x80000000u;  // an offset past the end of every buffer

// Everything that this wave has in LDS is there, for all waves; transfers from and to memory stay under way.
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// Where 16-byte piece `piece` of row r lies in a tile of DIM 16-bit elements a row (64 or 128).  The swizzle is its own inverse; by measurement neither
// pieces of 16 bytes (whose banks the LDS arbitrates for lanes 0-3, 12-15, 20-27 together, then 4-11, 16-19, 28-31), nor halves of them, nor transposed reads of 4
// rows meet in a bank.
template <int DIM> __device__ __forceinline__ int tile_off(int r, int piece) {
    const int x = DIM == 128 ? r : r >> 1, q = DIM == 128 ? (x >> 2) & 3 : (x >> 1) & 3;
    const int low = ((q & 1) << 1) ^ (q >> 1) ^ (q & 2);
    return r * (DIM * 2) + ((piece ^ (DIM == 128 ? (x & 3) << 2 | low : (x & 1) << 2 | low)) << 4);
}

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

// The power of two that brings values of up to `most` below 2^14: half precision ends at 65504, and the sums of linear
// attention, which no softmax bounds, do not.  Values below the power `least` lose digits; every finite one is taken.
struct Pow2 {
    int e;
    __device__ __forceinline__ float down() const { return __uint_as_float((unsigned)(127 - e) << 23); }
    __device__ __forceinline__ float up() const { return __uint_as_float((unsigned)(127 + e) << 23); }
};
constexpr int LEAST = -100;
__device__ __forceinline__ Pow2 into_range(float most, int least = LEAST) {
    const int e = (int)(__float_as_uint(most) >> 23) - 127 - 13;
    return Pow2{e < least ? least : e > 114 ? 0 : e};  // infinities and NaN as they are
}
// Over the lanes that hold one column of a state, of an operand's tokens, or one query's scores.
__device__ __forceinline__ float over_rows_max(float x) {
    x = fmaxf(x, __shfl_xor(x, 16, 64));
    return fmaxf(x, __shfl_xor(x, 32, 64));
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

// So many 16-bit elements that start on any of them: the memory takes such pieces as a whole, too.
template <int N> struct Any { typedef unsigned short type __attribute__((ext_vector_type(N), aligned(2))); };
template <int N> using Anywhere = typename Any<N>::type;

// A tile of 64 tokens, rows of DIM 16-bit elements in LDS (16-byte pieces, swizzled as in lbi_attn_mfma.h).  VEC: by transfers of 16 bytes past the
// registers, zeros past the end of a row and behind the last token; otherwise, rows that start on any element, by loads of the same size where they
// are whole.
template <typename T, int DIM, int THREADS, bool VEC> struct Tile {
    static constexpr int PIECES = DIM / 8, N = CHUNK * PIECES / THREADS;
    const T* next;  // where the chunk that is brought next lies in memory (reverse: as if it were whole)
    int64_t st;
    int dim;
    unsigned whole;  // offset of this lane's first piece (reverse: its last) of a whole chunk; the others lie so many whole rows further, in the same columns
    __device__ __forceinline__ unsigned piece_of(int u, int count, bool reverse) const {
        const int id = u * THREADS + (int)threadIdx.x, r = id / PIECES, slot = id % PIECES;
        const int chunk = tile_off<DIM>(r, slot) / 16 % PIECES;  // the swizzle is its own inverse
        const unsigned at = (unsigned)((reverse ? count - 1 - r : r) * (int)st + chunk * 8) * 2;
        return r < count && chunk * 8 < dim ? at : NOWHERE;
    }
    __device__ __forceinline__ Tile(const T* base, int64_t st_, int dim_, bool reverse, int64_t chunk_at) : next(base + chunk_at * st_), st(st_), dim(dim_) {
        static_assert(THREADS / PIECES % 16 == 0, "the swizzle repeats after 16 rows");
        whole = VEC ? piece_of(reverse ? N - 1 : 0, CHUNK, reverse) : 0;
    }
    // The next `count` tokens; `wave`: threadIdx.x / 64.
    __device__ __forceinline__ void bring(char* tile, unsigned tile_at, bool reverse, int count, int wave) {
        if constexpr (VEC) {
            const unsigned to = tile_at + wave * 1024;
            if (__builtin_expect(count == CHUNK, 1)) {
                const auto source = scan_planes::rows(next, 0x7fffffffu);
#pragma unroll
                for (int u = 0; u < N; ++u)
                    scan_planes::dma16(source, whole, (unsigned)((reverse ? N - 1 - u : u) * (THREADS / PIECES) * (int)st * 2), to + u * THREADS * 16);
            } else {
                const auto source = scan_planes::rows(next + (reverse ? (CHUNK - count) * st : 0), 0x7fffffffu);
#pragma unroll
                for (int u = 0; u < N; ++u) scan_planes::dma16(source, piece_of(u, count, reverse), 0, to + u * THREADS * 16);
            }
        } else {
            const T* const from = next + (reverse ? (CHUNK - count) * st : 0);
            int thread = (int)threadIdx.x;
            asm volatile("" : "+v"(thread));  // (what is made of it stays in the loop over the chunks: in front of it, each would take a register)
#pragma unroll
            for (int u = 0; u < N; ++u) {
                const int id = u * THREADS + thread, r = id / PIECES, c = id % PIECES * 8;
                const unsigned short* raw = reinterpret_cast<const unsigned short*>(from + (int64_t)(reverse ? count - 1 - r : r) * st + c);
                u32x4 words = {0, 0, 0, 0};
                if (r < count && c + 8 <= dim) words = __builtin_bit_cast(u32x4, *reinterpret_cast<const Anywhere<8>*>(raw));
                else if (r < count)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        words[e] = (c + 2 * e < dim ? raw[2 * e] : 0u) | (c + 2 * e + 1 < dim ? (unsigned)raw[2 * e + 1] << 16 : 0u);
                *reinterpret_cast<u32x4*>(tile + tile_off<DIM>(r, c / 8)) = words;
            }
        }
        next += reverse ? -CHUNK * st : CHUNK * st;
    }
};

// Places of a lane in a tile, from which all that it reads lie an exclusive or of constants (pieces) and a constant (rows) away.
typedef __attribute__((address_space(3))) char* lds_ptr;
template <int DIM> struct Places {
    unsigned nat_, split_, turned_, halved_;
    __device__ __forceinline__ Places(int m, int g)
        : nat_(tile_off<DIM>(m, g)), split_(tile_off<DIM>(m, g >> 1) + 8 * (g & 1)), turned_(tile_off<DIM>(8 * g + (m >> 2), (m & 3) >> 1) + ((m & 1) << 3)),
          halved_(tile_off<DIM>(8 * g + (m >> 2), m & 3)) {}
    // row 16 t + m, elements 32 ks + 8 g ... + 7
    __device__ __forceinline__ u32x4 nat(lds_ptr tile, int t, int ks) const {
        return *(__attribute__((address_space(3))) const u32x4*)(tile + (nat_ ^ (ks << 6)) + t * 32 * DIM);
    }
    // row 16 t + m, elements 32 ks + 4 g ... + 3 and 16 further: the order in which accumulators hold the rows of two tiles
    __device__ __forceinline__ u32x4 split(lds_ptr tile, int t, int ks) const {
        // (volatile: two rows' halves in one instruction would have to be taken apart again)
        typedef __attribute__((address_space(3))) const volatile u32x2* half;
        const u32x2 lo = *(half)(tile + (split_ ^ (ks << 6)) + t * 32 * DIM), hi = *(half)(tile + (split_ ^ (ks << 6) ^ 32) + t * 32 * DIM);
        return u32x4{lo[0], lo[1], hi[0], hi[1]};
    }
    // column `col` + m (a multiple of 16), rows 32 ks + 8 g ... + 7; of HALVES 2, column `col` + 8 (m / 4) + 4 half + m % 4 of 32
    template <int HALVES = 1> __device__ __forceinline__ u32x4 turned(lds_ptr tile, int ks, int col, int half = 0) const {
        typedef __attribute__((address_space(3))) attn_mfma::s16x4* four;
        const unsigned at = (HALVES == 1 ? turned_ : halved_) ^ (col << 1);
        const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((four)(tile + at + 8 * half + ks * 64 * DIM)));
        const u32x2 hi = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((four)(tile + (at ^ 32) + 8 * half + ks * 64 * DIM + 8 * DIM)));
        return u32x4{lo[0], lo[1], hi[0], hi[1]};
    }
};

// unit -> (chain, sequence, direction, head, segment): the workgroups that read the same tensors next to each other on one XCD
struct Unit { int chain, b, p, h, segment, number; };
__device__ __forceinline__ bool unit_of(const Call& call, int segments, Unit& u) {
    const int total = call.chains * call.B * call.P * call.H * segments, per = (int)(gridDim.x >> 3);
    int id = (int)(blockIdx.x & 7) * per + (int)(blockIdx.x >> 3);
    if (id >= total) return false;
    const auto digit = [&](int base) __attribute__((always_inline)) {  // (in scalar registers, and so is all that is read by it)
        const int rest = __builtin_amdgcn_readfirstlane(id / base), of = id - rest * base;
        id = rest;
        return of;
    };
    u.chain = digit(call.chains);
    u.segment = digit(segments);
    u.p = digit(call.P);
    u.h = digit(call.H);
    u.b = id;
    u.number = ((u.chain * call.B + u.b) * call.P + u.p) * call.H + u.h;
    return true;
}

// Two tiles of b; of c one and a's and the scores, or two of c where only the state is wanted.
template <int DA, int DC, bool OUT> constexpr int lds_bytes() { return CHUNK * 2 * (OUT ? 3 * DA + DC + CHUNK : 2 * (DA + DC)); }

// OUT false: only the state that a segment, or half of one, leaves behind, from zero, into its slot.  TWICE: calls of one chunk, with the scores and the copy of the state in two
// planes; the scores' second one has the place of b's second tile.
template <typename T, int DA, int DC, bool VEC, bool OUT, int PLANES, bool TWICE>
__global__ __launch_bounds__(256, OUT && DA == 64 && DC == 64 ? 3 : 2) void chunk_kernel(Call call) {
    constexpr bool HALF = std::is_same_v<T, _Float16>;
    constexpr int OPERANDS = TWICE ? 2 : 1;  // planes of the scores and of the state's copy
    constexpr int KS = DA / 32, MT = DA / 16, NT = DC / 64;  // steps and tiles of the state: rows, this wave's columns
    constexpr int TILE_A = CHUNK * 2 * DA, TILE_C = CHUNK * 2 * DC, AT_C = 2 * TILE_A, AT_A = AT_C + TILE_C, AT_P = AT_A + TILE_A;
    extern __shared__ __align__(16) char lds[];  // b, b, c, a, the scores; b, b, c, c
    __shared__ int score_by[HALF ? CHUNK : 1];  // exponents, a query each
    Unit u;
    if (!unit_of(call, OUT ? call.segments : call.slots(), u)) return;
    const Chain& ch = call.chain[u.chain];
    const int n = length_of(call, u.b), w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), m = threadIdx.x & 15, g = (threadIdx.x >> 4) & 3;
    const int begin = OUT ? u.segment * call.segment : call.slot_at(u.segment), stop = OUT ? begin + call.segment : call.slot_at(u.segment + 1);
    const int end = stop < n ? stop : n;  // of the tokens that count
    auto at = [&](const View& v) { return static_cast<const T*>(v.p) + u.b * v.sb + u.p * v.sp + (u.h / v.group) * v.sh; };
    const bool reverse = ch.reverse != 0;
    const float rate = rate_of(call, u.h), rate2 = rate * LOG2E;
    const int shift = ch.shift, Da = ch.Da, Dc = ch.Dc, col0 = w * (DC / 4);

    const int64_t chunk_at = reverse ? (int64_t)n - begin - CHUNK : begin;
    Tile<T, DA, 256, VEC> a(OUT ? at(ch.a) : nullptr, ch.a.st, Da, reverse, chunk_at), b(at(ch.b), ch.b.st, Da, reverse, chunk_at);
    Tile<T, DC, 256, VEC> c(at(ch.c), ch.c.st, Dc, reverse, chunk_at);
    const unsigned lds0 = (unsigned)(size_t)(__attribute__((address_space(3))) char*)lds;
    auto bring_b = [&](int stage, int from) __attribute__((always_inline)) {
        b.bring(lds + stage * TILE_A, lds0 + stage * TILE_A, reverse, end - from < CHUNK ? end - from : CHUNK, w);
    };
    auto bring_rest = [&](int stage, int from) __attribute__((always_inline)) {
        const int count = end - from < CHUNK ? end - from : CHUNK, to = AT_C + (OUT ? 0 : stage * TILE_C);
        c.bring(lds + to, lds0 + to, reverse, count, w);
        if constexpr (OUT) a.bring(lds + AT_A, lds0 + AT_A, reverse, count, w);
    };
    if (begin < end) {
        bring_b(0, begin);
        bring_rest(0, begin);
    }

    // l to the power of tokens apart (and the result's scale): of this lane's scores, 0 for later tokens, of its readouts and of its rows of c
    const float l16 = exp2f(rate2 * 16.0f), l32 = exp2f(rate2 * 32.0f), l48 = exp2f(rate2 * 48.0f);
    const float read0 = exp2f(rate2 * (float)(m + 1 - shift)) * ch.scale;
    float apart[OUT ? 4 : 1][4], keep[8];
    if constexpr (OUT)
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int tokens = 16 * (w - t) + m - 4 * g - r;
                apart[t][r] = tokens < 0 ? 0.0f : exp2f(rate2 * (float)tokens) * ch.scale;
            }
#pragma unroll
    for (int e = 0; e < 8; ++e) keep[e] = exp2f(rate2 * (float)(31 - 8 * g - e + shift));
    // half precision: the least power of scores whose inverse times the scale is a number (only a scale of 2^26 and more raises it)
    const int by_scale = (int)(__float_as_uint(ch.scale) >> 23 & 255) - 126 - 126, least_score = by_scale > LEAST ? by_scale : LEAST;
    // Of the state, over a chunk: a fused multiply-add beside each readout's operands for decays near 1, and for others, which that one then leaves as they are, a
    // product behind them, in a branch that those near 1 do not take (us, fused for all / so: half precision, a basis of 4 623 / 632, 512 chains of 4096 of 128
    // 484 / 490; bf16 the same).
    Fade fade(rate * (float)CHUNK);

    f32x4 x[MT][NT];
    auto each = [&](auto&& f) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r) f(i, j, r);
    };
    each([&](int i, int j, int r) __attribute__((always_inline)) { x[i][j][r] = 0.0f; });
    // This wave's columns of a state in memory, strides in elements: f(row tile, column tile, register, offset in bytes), no place for what lies past
    // the dimensions.
    auto of_state = [&](unsigned sr, unsigned sc, auto&& f) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            const int col = col0 + (NT == 1 ? m : 8 * (m >> 2) + 4 * j + (m & 3));
            unsigned at_row = col < Dc ? 4 * (4 * g * sr + col * sc) : NOWHERE;
#pragma unroll
            for (int i = 0; i < MT; ++i) {
#pragma unroll
                for (int r = 0; r < 4; ++r) f(i, j, r, 16 * i + 4 * g + r < Da ? at_row + 4 * r * sr : NOWHERE);
                at_row += 64 * sr;
            }
        }
    };
    auto state_at = [&](const float* p, unsigned sr, unsigned sc, auto&& use) __attribute__((always_inline)) {
        const auto from = scan_planes::rows(p, 0x7fffffffu);
        float v[MT][NT][4];  // all asked for before any is waited for
        of_state(sr, sc, [&](int i, int j, int r, unsigned place) __attribute__((always_inline)) {
            v[i][j][r] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(from, place, 0, 0));
        });
        each([&](int i, int j, int r) __attribute__((always_inline)) { x[i][j][r] = use(x[i][j][r], v[i][j][r]); });
    };
    if constexpr (OUT) {
        if (ch.first.p && (u.segment == 0 || !call.joined)) {
            const float scale = ch.first_scale;
            state_at(ch.first.p + u.b * ch.first.sb + u.p * ch.first.sp + u.h * ch.first.sh, (unsigned)ch.first.sr, (unsigned)ch.first.sc,
                     [&](float, float v) __attribute__((always_inline)) { return v * scale; });
        }
        const float* slots = call.segment_states + (int64_t)u.number * call.slots() * Da * Dc;
        const int before = u.segment << call.halved;
        for (int s = call.joined ? before - 1 : 0; s >= 0 && s < before; ++s) {  // what the slots before add, the first one first
            const int from = call.slot_at(s), most = call.slot_at(s + 1) - from;
            int tokens = n - from;
            tokens = tokens < 0 ? 0 : tokens > most ? most : tokens;
            Fade over(rate * (float)tokens);
            if (call.joined) over.by = over.kept = 0.0f;
            state_at(slots + (int64_t)s * Da * Dc, (unsigned)Dc, 1, [&](float x_, float v) __attribute__((always_inline)) { return over.of(x_) + v; });
        }
    }
    scan_planes::wait_vm<0>();

    const int64_t out_st = ch.out.st;
    T* next_out = OUT ? const_cast<T*>(at(ch.out)) + chunk_at * out_st : nullptr;
    const int first_col = col0 + 4 * NT * g;  // of the 4 NT neighbouring ones that this lane has of a row
    const unsigned out_at = (unsigned)((reverse ? 15 - m : m) * (int)out_st + first_col) * 2;  // in sixteen rows of a whole chunk
    Places<DA> in_a(m, g);  // and in b's
    Places<DC> in_c(m, g);
    Places<CHUNK> in_p(m, g);
    int stage = 0, from = begin;
    auto chunk = [&](auto whole_tag) __attribute__((always_inline)) {
        constexpr bool WHOLE = decltype(whole_tag)::value;  // 64 tokens
        lds_barrier();  // this chunk's tiles are there
        const lds_ptr tb = (lds_ptr)lds + stage * TILE_A, tc = (lds_ptr)lds + AT_C + (OUT ? 0 : stage * TILE_C), ta = (lds_ptr)lds + AT_A, tp = (lds_ptr)lds + AT_P, tp2 = (lds_ptr)lds + TILE_A;
        // (what is made of them stays in this loop: in front of it, each would take a register)
        asm volatile("" : "+v"(in_a.nat_), "+v"(in_a.split_), "+v"(in_a.turned_), "+v"(in_p.nat_), "+v"(in_p.split_), "+v"(NT == 1 ? in_c.turned_ : in_c.halved_));
        const int count = WHOLE ? CHUNK : end - from;
        const bool more_tokens = WHOLE && !TWICE && from + CHUNK < end;
        if (more_tokens) {
            bring_b(stage ^ 1, from + CHUNK);
            if (!OUT) bring_rest(stage ^ 1, from + CHUNK);
        }

        // What a wave issues between its products runs beside them: each stretch below, between fences, holds the vector work of a later one.
        u32x4 raw[2][NT];  // the chunk's c: as it is for the scores, decayed for the state
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
            for (int j = 0; j < NT; ++j) raw[ks][j] = in_c.template turned<NT>(tc, ks, col0, j);
        u32x4 plane[2][PLANES][NT];
        auto left = [&](int ks, int at_e) __attribute__((always_inline)) {
            const int tokens = count - 1 - (32 * ks + 8 * g + at_e);
            return !WHOLE ? exp2f(rate2 * (float)((tokens < 0 ? 0 : tokens) + shift)) : ks == 0 ? keep[at_e] * l32 : keep[at_e];
        };
        Pow2 decayed_by[NT];  // half precision: of this lane's columns
        auto decayed_into_range = [&]() __attribute__((always_inline)) {
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                float most = 0.0f;
#pragma unroll
                for (int ks = 0; ks < 2; ++ks)
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const unsigned word = raw[ks][j][e / 2];
                        most = fmaxf(most, fabsf((e % 2 ? Mma<T>::hi(word) : Mma<T>::lo(word)) * left(ks, e)));
                    }
                decayed_by[j] = into_range(over_rows_max(most));
            }
        };
        // words e of the decayed c of step ks, column tile j
        auto decay = [&](int ks, int j, int e) __attribute__((always_inline)) {
            float lo = Mma<T>::lo(raw[ks][j][e]) * left(ks, 2 * e), hi = Mma<T>::hi(raw[ks][j][e]) * left(ks, 2 * e + 1);
            if constexpr (HALF) lo *= decayed_by[j].down(), hi *= decayed_by[j].down();
#pragma unroll
            for (int q = 0; q < PLANES; ++q) {
                const unsigned word = Mma<T>::pack2(lo, hi);
                plane[ks][q][j][e] = word;
                lo -= Mma<T>::lo(word), hi -= Mma<T>::hi(word);
            }
        };
        if constexpr (!WHOLE) fade = Fade(rate * (float)count);
        const float near_one = fade.kept != 0.0f ? fade.by : 0.0f;
        auto move_on = [&](int i) __attribute__((always_inline)) {  // rows 16 i ... of the state, past the chunk's tokens
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r) x[i][j][r] = fmaf(x[i][j][r], near_one, x[i][j][r]);
        };

        f32x4 acc[NT][4];
        Pow2 state_by[NT];  // half precision: of this lane's columns
        if constexpr (OUT) {
            f32x4 s[4];
#pragma unroll
            for (int t = 0; t < 4; ++t) s[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                const u32x4 mine = in_a.nat(ta, w, ks);
#pragma unroll
                for (int t = 0; t < 4; ++t) s[t] = Mma16<T>::mma(in_a.nat(tb, t, ks), mine, s[t]);
            }
            if constexpr (HALF) {
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    float of_state = 0.0f;
#pragma unroll
                    for (int i = 0; i < MT; ++i)
#pragma unroll
                        for (int r = 0; r < 4; ++r) of_state = fmaxf(of_state, fabsf(x[i][j][r]));
                    state_by[j] = into_range(over_rows_max(of_state));
                }
            }
            u32x4 state[2][OPERANDS][NT];  // this step's rows of the state as an operand, and the next one's
            auto pack = [&](int ks) __attribute__((always_inline)) {
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    const float by = HALF ? state_by[j].down() : 1.0f;
                    const f32x4 lo = x[2 * ks][j] * by, hi = x[2 * ks + 1][j] * by;
                    float v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
#pragma unroll
                    for (int e = 0; e < 4; ++e)
#pragma unroll
                        for (int q = 0; q < OPERANDS; ++q) {
                            const unsigned word = Mma<T>::pack2(v[2 * e], v[2 * e + 1]);
                            state[ks & 1][q][j][e] = word;
                            v[2 * e] -= Mma<T>::lo(word), v[2 * e + 1] -= Mma<T>::hi(word);
                        }
                }
                move_on(2 * ks);
                move_on(2 * ks + 1);
            };
            pack(0);
            u32x4 tokens[4];
#pragma unroll
            for (int t = 0; t < 4; ++t) tokens[t] = in_a.split(ta, t, 0);
            LBI_PHASE_FENCE();
            // the scores, rounded, beside the readout's first step
            float most = 0.0f;
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    s[t][r] = m - 4 * g >= 16 * (t - w) + r ? s[t][r] * apart[t][r] : 0.0f;
                    if constexpr (HALF) most = fmaxf(most, fabsf(s[t][r]));
                }
            if constexpr (HALF) {
                const Pow2 by = into_range(over_rows_max(most), least_score);
                if (g == 0) score_by[16 * w + m] = by.e;
#pragma unroll
                for (int t = 0; t < 4; ++t) s[t] *= by.down();
            }
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int q = 0; q < OPERANDS; ++q) {
                    const u32x2 words = {Mma<T>::pack2(s[t][0], s[t][1]), Mma<T>::pack2(s[t][2], s[t][3])};
                    *(__attribute__((address_space(3))) u32x2*)((q == 0 ? tp : tp2) + (in_p.split_ ^ (t << 5)) + w * 32 * CHUNK) = words;
                    s[t] -= f32x4{Mma<T>::lo(words[0]), Mma<T>::hi(words[0]), Mma<T>::lo(words[1]), Mma<T>::hi(words[1])};
                }
            if constexpr (HALF) {
                decayed_into_range();
            }
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int t = 0; t < 4; ++t) acc[j][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                constexpr int EARLY = NT == 1 ? 4 : 2;  // tokens' tiles that are read a step ahead: what the registers hold
                u32x4 more[EARLY];
                if (ks > 0)
#pragma unroll
                    for (int t = EARLY; t < 4; ++t) tokens[t] = in_a.split(ta, t, ks);
                if (ks + 1 < KS)
#pragma unroll
                    for (int t = 0; t < EARLY; ++t) more[t] = in_a.split(ta, t, ks + 1);
#pragma unroll
                for (int q = OPERANDS - 1; q >= 0; --q)
#pragma unroll
                    for (int t = 0; t < 4; ++t)
#pragma unroll
                        for (int j = 0; j < NT; ++j) acc[j][t] = Mma16<T>::mma(state[ks & 1][q][j], tokens[t], acc[j][t]);
                if (ks + 1 < KS) pack(ks + 1);
#pragma unroll
                for (int p = ks * 4 * NT / KS; p < (ks + 1) * 4 * NT / KS; ++p) decay(0, p / 4, p % 4);
                if constexpr (WHOLE && !HALF)
#pragma unroll
                    for (int i = 0; i < 4 * NT; ++i) {
                        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                        __builtin_amdgcn_sched_group_barrier(0x002, 6, 0);
                    }
                LBI_PHASE_FENCE();
                if (ks + 1 < KS)
#pragma unroll
                    for (int t = 0; t < EARLY; ++t) tokens[t] = more[t];
            }
            if constexpr (HALF)
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float up = Pow2{__shfl(state_by[j].e, 4 * g + r, 64)}.up();  // the state's columns are rows here
#pragma unroll
                        for (int t = 0; t < 4; ++t) acc[j][t][r] *= up;
                    }
        } else {
            if constexpr (HALF) decayed_into_range();
#pragma unroll
            for (int p = 0; p < (HALF ? 8 : 4) * NT; ++p) decay(p / (4 * NT), p / 4 % NT, p % 4);
#pragma unroll
            for (int i = 0; i < MT; ++i) move_on(i);
        }

        T* const out = OUT ? next_out + (WHOLE || !reverse ? 0 : (CHUNK - count) * out_st) : nullptr;
        const auto to = scan_planes::rows(out, 0x7fffffffu);
        auto store = [&](int t) __attribute__((always_inline)) {  // sixteen rows
            const int i = 16 * t + m, row = reverse ? count - 1 - i : i;
            const float by = HALF ? Pow2{score_by[16 * t + m]}.up() : 1.0f;
            unsigned words[2 * NT];
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                words[2 * j] = Mma<T>::pack2(acc[j][t][0] * by, acc[j][t][1] * by);
                words[2 * j + 1] = Mma<T>::pack2(acc[j][t][2] * by, acc[j][t][3] * by);
            }
            if constexpr (VEC) {  // each wave has the same number of stores under way, whatever there is to store
                const unsigned place = WHOLE ? (first_col < Dc ? out_at : NOWHERE)
                                             : (i < count && first_col < Dc ? (unsigned)(row * (int)out_st + first_col) * 2 : NOWHERE);
                const unsigned tile = WHOLE ? (unsigned)((reverse ? 3 - t : t) * 32 * (int)out_st) : 0;
                if constexpr (NT == 1) __builtin_amdgcn_raw_buffer_store_b64(u32x2{words[0], words[1]}, to, place, tile, 0);
                else __builtin_amdgcn_raw_buffer_store_b128(u32x4{words[0], words[1], words[2], words[3]}, to, place, tile, 0);
            } else if (i < count && first_col + 4 * NT <= Dc) {
                typedef unsigned whole __attribute__((ext_vector_type(2 * NT)));
                whole all;
#pragma unroll
                for (int e = 0; e < 2 * NT; ++e) all[e] = words[e];
                *reinterpret_cast<Anywhere<4 * NT>*>(out + row * out_st + first_col) = __builtin_bit_cast(Anywhere<4 * NT>, all);
            } else if (i < count) {
#pragma unroll
                for (int r = 0; r < 4 * NT; ++r)
                    if (first_col + r < Dc) reinterpret_cast<unsigned short*>(out + row * out_st)[first_col + r] = (unsigned short)(words[r / 2] >> (16 * (r % 2)));
            }
        };
        if constexpr (OUT) {
            next_out += reverse ? -CHUNK * out_st : CHUNK * out_st;
            lds_barrier();  // the scores are there, and everyone is done with a and c
            u32x4 scores[OPERANDS][2][4];  // (read before the next tiles are asked for, which they would wait behind)
#pragma unroll
            for (int q = 0; q < OPERANDS; ++q)
#pragma unroll
                for (int ks = 0; ks < 2; ++ks)
#pragma unroll
                    for (int t = 2 * ks; t < 4; ++t) scores[q][ks][t] = in_p.nat(q == 0 ? tp : tp2, t, ks);
            LBI_PHASE_FENCE();
            if (more_tokens) bring_rest(0, from + CHUNK);
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                float by = read0 * (t == 0 ? 1.0f : t == 1 ? l16 : t == 2 ? l32 : l48);
                // Into the scores' power, which what reads the state out has room for (least_score).  A readout that is past fp32 then would be past half
                // precision as a result: scores of so small a power add less than 2^-64 to it.
                if constexpr (HALF) by *= Pow2{score_by[16 * t + m]}.down();
#pragma unroll
                for (int j = 0; j < NT; ++j) acc[j][t] *= by;
            }
#pragma unroll
            for (int q = OPERANDS - 1; q >= 0; --q)
#pragma unroll
                for (int ks = 0; ks < 2; ++ks)
#pragma unroll
                    for (int t = 2 * ks; t < 4; ++t)
#pragma unroll
                        for (int j = 0; j < NT; ++j) acc[j][t] = Mma16<T>::mma(raw[ks][j], scores[q][ks][t], acc[j][t]);
            if constexpr (HALF) {
                if constexpr (!VEC) LBI_PHASE_FENCE();
#pragma unroll
                for (int p = 0; p < 4 * NT; ++p) decay(1, p / 4, p % 4);
            }
            LBI_PHASE_FENCE();
        }

        if (fade.kept == 0.0f) each([&](int i, int j, int r) __attribute__((always_inline)) { x[i][j][r] *= fade.by; });
        // In half precision the sum of a chunk comes in the power of two of its decayed values: both steps of a row tile, then onto the state.
        const auto step_of = [](int step) __attribute__((always_inline)) { return HALF ? step % 2 : step / MT; };
        const auto tile_of = [](int step) __attribute__((always_inline)) { return HALF ? step / 2 : step % MT; };
        if (TWICE)
#pragma unroll
            for (int t = 0; t < 4; ++t) store(t);
        if (TWICE && !ch.last.p) return;  // nobody wants the state behind the only chunk
        u32x4 rows = in_a.turned(tb, 0, 0);
        f32x4 added[HALF ? NT : 1];
#pragma unroll
        for (int step = 0; step < 2 * MT; ++step) {
            const int ks = step_of(step), i = tile_of(step);
            u32x4 more;
            if (step + 1 < 2 * MT) more = in_a.turned(tb, step_of(step + 1), 16 * tile_of(step + 1));
            if (HALF && ks == 0)
#pragma unroll
                for (int j = 0; j < NT; ++j) added[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int q = PLANES - 1; q >= 0; --q)
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    f32x4& sum = HALF ? added[j] : x[i][j];
                    sum = Mma16<T>::mma(rows, plane[ks][q][j], sum);
                }
            if (HALF && ks == 1)
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int r = 0; r < 4; ++r) x[i][j][r] = fmaf(added[j][r], decayed_by[j].up(), x[i][j][r]);
            if (!HALF && ks == 0)
#pragma unroll
                for (int p = i * 4 * NT / MT; p < (i + 1) * 4 * NT / MT; ++p) decay(1, p / 4, p % 4);
            if constexpr (OUT && !TWICE)
                if (ks == 1 && i < 4) store(i);
            if constexpr (WHOLE)
#pragma unroll
                for (int n_ = 0; n_ < PLANES * NT; ++n_) {
                    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                    __builtin_amdgcn_sched_group_barrier(0x002, 4, 0);
                }
            LBI_PHASE_FENCE();
            rows = more;
        }

        scan_planes::wait_vm<OUT && VEC ? 4 : 0>();  // the next tiles; this chunk's stores may still be under way
        stage ^= 1;
    };
    for (; from + CHUNK <= end; from += CHUNK) chunk(std::true_type{});
    if (from < end) chunk(std::false_type{});
    if constexpr (OUT) {  // rows behind the sequence
        T* const out = const_cast<T*>(at(ch.out));
        const int last = stop < call.T ? stop : call.T, past = begin > n ? begin : n;
        const int c8 = (int)threadIdx.x % (DC / 8) * 8;
        for (int i = past + (int)threadIdx.x / (DC / 8); i < last; i += 256 / (DC / 8)) {
            T* const row = out + i * out_st + c8;
            if (VEC && c8 < Dc) *reinterpret_cast<u32x4*>(row) = u32x4{0, 0, 0, 0};
            if constexpr (!VEC)
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (c8 + e < Dc) reinterpret_cast<unsigned short*>(row)[e] = 0;
        }
    }
    auto leave = [&](float* p, unsigned sr, unsigned sc, float scale) __attribute__((always_inline)) {
        const auto to = scan_planes::rows(p, 0x7fffffffu);
        of_state(sr, sc, [&](int i, int j, int r, unsigned place) __attribute__((always_inline)) {
            const float v = x[i][j][r] * scale;
            __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(v), to, place, 0, 0);
        });
    };
    if constexpr (OUT) {
        if (ch.last.p && u.segment == call.segments - 1)
            leave(ch.last.p + u.b * ch.last.sb + u.p * ch.last.sp + u.h * ch.last.sh, (unsigned)ch.last.sr, (unsigned)ch.last.sc, ch.last_scale);
    } else {
        leave(call.segment_states + ((int64_t)u.number * call.slots() + u.segment) * Da * Dc, (unsigned)Dc, 1, 1.0f);
    }
}

// Slot s of each unit holds what segment s adds; they become the states behind the segments.  BATCH slots are asked for at once.
template <typename T> __global__ __launch_bounds__(256) void join_kernel(Call call) {
    constexpr int BATCH = 8;
    const int of_chain = call.B * call.P * call.H, slots = call.slots();
    int id = (int)blockIdx.y;
    const int number = id;
    const Chain& ch = call.chain[id / of_chain];
    id %= of_chain;
    const int h = id % call.H, p = id / call.H % call.P, b = id / call.H / call.P;
    const int e = (int)(blockIdx.x * 256 + threadIdx.x), count = ch.Da * ch.Dc;
    if (e >= count) return;
    const int n = length_of(call, b);
    const float rate = rate_of(call, h);
    const Fade whole(rate * (float)call.segment);
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
            x = (left >= call.segment ? whole : Fade(rate * (float)(left < 0 ? 0 : left))).of(x) + more[s];
            slot[(int64_t)(from + s) * count] = x;
        }
    }
}

}  // namespace linear_attn
}  // namespace lbi
