// The gated MLP of a Transformer block and its pullback, in one 16-bit type, sums in fp32:
//
//   forward    z = x W1^T + b1,  [u | g] = z,  a = u * g * sigmoid(g),  out = a W2^T + b2
//   pullback   g_a = g_out W2;  g_u = g_a silu(g), g_g = g_a u silu'(g);  g_x = [g_u | g_g] W1;  g_W1 = [g_u | g_g]^T x;  g_W2 = g_out^T a
//
// All six products are one kernel, and the last two one launch: a workgroup of four waves owns a tile of results, 32 FM x 32 FN of them a wave, and
// takes 64 terms of the sums a step through LDS, in a ring of two or three steps.  Operands arrive by buffer_load ... lds, whole 128-byte lines
// (what lies past the end of an operand is zero, so ragged sizes take the same loop); one whose terms lie side by side is read in 16-byte
// pieces, one whose terms are its rows through transposing reads.  The product is formed as C^T: a lane ends up with four neighbouring columns
// of one row.  Up and gate of one column meet in one lane, so the gate costs no pass of its own in either direction.
//
// Bound by the matrix units' issue in large calls (6007 rows, 4096 -> 2 x 11008 -> 4096 in bf16: 1.37 ms, 1.19 PFLOP/s), by starts, ends and results on
// their way out in ordinary ones (8192 rows, 768 -> 2 x 2048 -> 768, fc1_output kept: 98 us, 0.79 PFLOP/s), by the weights' way through the chip in small ones.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>
#include <utility>

#include "lbi_attn_mfma.h"
#include "lbi_attn_dkdv128.h"
#include "lbi_block_mlp_layout.h"

namespace lbi {
namespace block_mlp {
namespace {

using attn_mfma::Mma;
using attn_mfma::s16x4;
using attn_mfma::swz;
using attn_mfma::tile_off;
using attn_mfma::u32x2;
using attn_mfma::u32x4;

constexpr int NT = 256;  // threads
constexpr unsigned PAST_END = 1u << 31;  // no operand's step reaches this far
constexpr int PIECE = 1024;  // bytes that a wave's load brings: 8 rows of 64 terms, or 8 terms of 64 columns

template <int N> using Count = std::integral_constant<int, N>;

struct Task {
    const void *a, *b, *bias;  // A [M, K] or, by rows, [K, M]; B [N, K] or, by rows, [K, N]; GATED: B [2N, K]
    void *out, *z;             // GATED: z [M, 2N] written if given; UNGATED: z [M, 2N] read, out [M, 2N]
    long long M, N, K;
    long long own;             // GATED, UNGATED: the first of N that are not padding; the next product sums over the others too, which must be 0
    int m_tiles, n_tiles;
    struct {  // both operands by rows: a second product over the same K, whose tiles follow those of the first
        const void *a, *b;
        void* out;
        long long M, N;
        int m_tiles, n_tiles;
    } second;
    float* partial;
    int tiles;              // of both
    int whole;              // tiles that one workgroup each sums up; the others' sums are cut into `parts` ranges of `part_steps` steps
    int parts, part_steps;
};
// The product that tile `at` belongs to becomes the task's, and `at` its own tile.
__device__ __forceinline__ void turn_to(Task& task, int& at) {
    const int of_first = task.m_tiles * task.n_tiles;
    if (at < of_first) return;
    at -= of_first;
    task.a = task.second.a, task.b = task.second.b, task.out = task.second.out, task.M = task.second.M, task.N = task.second.N;
    task.m_tiles = task.second.m_tiles, task.n_tiles = task.second.n_tiles;
}

__device__ __forceinline__ float sigmoid(float x) { return 1.0f / (1.0f + __expf(-x)); }

struct Eight { float v[8]; };
__device__ __forceinline__ Eight operator+(const Eight& a, const Eight& b) {
    Eight r;
#pragma unroll
    for (int e = 0; e < 8; ++e) r.v[e] = a.v[e] + b.v[e];
    return r;
}
template <typename T> __device__ __forceinline__ Eight wide8(const u32x4& w) {
    return Eight{{Mma<T>::lo(w[0]), Mma<T>::hi(w[0]), Mma<T>::lo(w[1]), Mma<T>::hi(w[1]), Mma<T>::lo(w[2]), Mma<T>::hi(w[2]),
                  Mma<T>::lo(w[3]), Mma<T>::hi(w[3])}};
}
template <typename T> __device__ __forceinline__ Eight load8(const T* p) { return wide8<T>(*reinterpret_cast<const u32x4*>(p)); }
template <typename T> __device__ __forceinline__ void store8(T* p, const Eight& x) {
    *reinterpret_cast<u32x4*>(p) = u32x4{Mma<T>::pack2(x.v[0], x.v[1]), Mma<T>::pack2(x.v[2], x.v[3]), Mma<T>::pack2(x.v[4], x.v[5]),
                                         Mma<T>::pack2(x.v[6], x.v[7])};
}
__device__ __forceinline__ void store8(float* p, const Eight& x) {
    reinterpret_cast<f32x4*>(p)[0] = f32x4{x.v[0], x.v[1], x.v[2], x.v[3]};
    reinterpret_cast<f32x4*>(p)[1] = f32x4{x.v[4], x.v[5], x.v[6], x.v[7]};
}
__device__ __forceinline__ Eight load8(const float* p) {
    const f32x4 a = reinterpret_cast<const f32x4*>(p)[0], b = reinterpret_cast<const f32x4*>(p)[1];
    return Eight{{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]}};
}

// What finishing eight columns of one row reads beside their sums, as stored: the bias (GATED: up's and gate's; zero where there is none) or
// UNGATED up and gate.  Read ahead, and in no branch: at the end of one the compiler would wait for it, one eight after the other.
struct Beside { u32x4 a, b; };
template <typename T, Finish FINISH> __device__ __forceinline__ Beside beside(const Task& task, long long row, long long col) {
    const long long N = task.N;
    Beside r{};
    if (col >= N) col = 0;
    if constexpr (FINISH == UNGATED) {
        const T* z = static_cast<const T*>(task.z) + (row < task.M ? row : 0) * 2 * N + col;
        r.a = *reinterpret_cast<const u32x4*>(z);
        r.b = *reinterpret_cast<const u32x4*>(z + N);
    } else if (const T* bias = static_cast<const T*>(task.bias)) {
        r.a = *reinterpret_cast<const u32x4*>(bias + col);
        if constexpr (FINISH == GATED) r.b = *reinterpret_cast<const u32x4*>(bias + N + col);
    }
    return r;
}
// Zero where a column is padding.  The sums there are products with zeros, which an infinity on the other side makes NaN.
__device__ __forceinline__ void drop_padding(const Task& task, long long col, Eight& x) {
    if (col + 8 <= task.own) return;
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (col + e >= task.own) x.v[e] = 0.0f;
}
// Eight columns of one row of the result, from their sums (GATED: up's and gate's).
template <typename T, Finish FINISH>
__device__ __forceinline__ void finish(const Task& task, long long row, long long col, const Eight& x, const Eight& y, const Beside& more) {
    const long long N = task.N;
    if (row >= task.M || col >= N) return;
    T* out = static_cast<T*>(task.out);
    const Eight a = wide8<T>(more.a), b = wide8<T>(more.b);
    if constexpr (FINISH == PLAIN) {
        store8(out + row * N + col, x + a);
    } else if constexpr (FINISH == GATED) {
        const Eight up = x + a, gate = y + b;
        Eight act;
#pragma unroll
        for (int e = 0; e < 8; ++e) act.v[e] = up.v[e] * (gate.v[e] * sigmoid(gate.v[e]));
        drop_padding(task, col, act);
        store8(out + row * N + col, act);
        if (T* z = static_cast<T*>(task.z)) {
            store8(z + row * 2 * N + col, up);
            store8(z + row * 2 * N + N + col, gate);
        }
    } else {
        Eight g_up, g_gate;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float open = sigmoid(b.v[e]);
            g_up.v[e] = x.v[e] * (b.v[e] * open);
            g_gate.v[e] = x.v[e] * a.v[e] * (open * (1.0f + b.v[e] * (1.0f - open)));
        }
        drop_padding(task, col, g_up);
        drop_padding(task, col, g_gate);
        store8(out + row * 2 * N + col, g_up);
        store8(out + row * 2 * N + N + col, g_gate);
    }
}

template <typename F, int... I> __host__ __device__ __forceinline__ void each(F&& f, std::integer_sequence<int, I...>) { (f(Count<I>{}), ...); }
// f(Count<0>{}), ... f(Count<N - 1>{})
template <int N, typename F> __host__ __device__ __forceinline__ void each(F&& f) { each(f, std::make_integer_sequence<int, N>{}); }

// 1 KiB from memory to LDS by one wave: lane l brings the 16 bytes at `off` of what `words` describe, zeros past its end.
template <int AT> __device__ __forceinline__ void bring(const u32x4& words, unsigned off, unsigned lds) {
    asm volatile("s_add_u32 m0, %0, %1\n\ts_nop 0\n\tbuffer_load_dwordx4 %2, %3, 0 offen lds"
                 :
                 : "s"(lds), "i"(AT), "v"(off), "s"(words)
                 : "memory", "scc");
}

// Where an operand's steps lie: the bytes from its tile's part of a step to the end of the tile (terms side by side) or of the operand (by rows).
struct Source {
    const char* at;
    long long left, step;
    __device__ __forceinline__ void skip(int steps) {
        at += steps * step;
        left -= steps * step;
    }
    // words 0 and 1 the address, 2 the bytes that may be read, 3 the format (32 bits); then on to the next step
    __device__ __forceinline__ u32x4 next(bool there) {
        constexpr long long most = PAST_END - 16;
        const u32x4 words = {(unsigned)(size_t)at, (unsigned)((size_t)at >> 32) & 0xffffu, there ? (unsigned)(left < most ? left : most) : 0u, 4u << 15};
        skip(1);
        return words;
    }
};

// Ids equal mod 8 share an L2: they get neighbouring places.
__device__ __forceinline__ int place(int id, int count) {
    const int lot = count / 8, left = count % 8, x = id % 8;
    return x * lot + min(x, left) + id / 8;
}
// Place -> tile: eight rows of tiles at a time.
__device__ __forceinline__ void tile_at(int at, int m_tiles, int n_tiles, int& mt, int& nt) {
    constexpr int ROWS = 8;
    const int band = at / (ROWS * n_tiles), in = at - band * ROWS * n_tiles, rows = min(ROWS, m_tiles - band * ROWS);
    mt = band * ROWS + in % rows;
    nt = in / rows;
}
// What one wave leaves of 32 rows of a part of a tile: columns in eights, GATED up's first.
template <int FM, int FN> __device__ __forceinline__ size_t partial_at(int item, int wave, int i) {
    return ((size_t)(item * 4 + wave) * FM + i) * (32 * 32 * FN);
}

template <typename T, int FM, int FN, int DEEP, bool A_ROWS, bool B_ROWS, Finish FINISH>  // ..._ROWS: the terms are the operand's rows
__global__ __launch_bounds__(NT) void product_kernel(Task task) {
    constexpr int BM = 64 * FM, BN = 64 * FN;  // rows and columns of B's tile
    constexpr int A_BYTES = BM * 128, SLOT = A_BYTES + BN * 128, READS = FM + FN, LOADS = 2 * READS;
    extern __shared__ __align__(16) char lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int m = lane & 31, h = lane >> 5, wm = wave >> 1, wn = wave & 1;
    constexpr int WIDE = FINISH == GATED ? BN / 2 : BN;
    const long long K = task.K;
    const int steps = (int)((K + STEP - 1) / STEP);
    int at, first = 0, last = steps, item = -1;
    if ((int)blockIdx.x < task.whole) {
        at = place((int)blockIdx.x, task.whole);
    } else {
        const int rest = task.tiles - task.whole, p = place((int)blockIdx.x - task.whole, rest * task.parts), part = p / rest;
        at = task.whole + p % rest;
        first = part * task.part_steps;
        last = min(first + task.part_steps, steps);
        item = p;
    }
    if constexpr (A_ROWS && B_ROWS) turn_to(task, at);
    const long long M = task.M, N = task.N;
    int mt, nt;
    tile_at(at, task.m_tiles, task.n_tiles, mt, nt);
    const long long row0 = (long long)mt * BM, col0 = (long long)nt * WIDE;
    const unsigned row_bytes = (unsigned)K * 2;
    const int a_rows = (int)(M - row0 < BM ? M - row0 : BM), b_cols = (int)(N - col0 < WIDE ? N - col0 : WIDE);
    Source a_src = A_ROWS ? Source{static_cast<const char*>(task.a) + row0 * 2, (K * M - row0) * 2, STEP * M * 2}
                          : Source{static_cast<const char*>(task.a) + row0 * K * 2, (long long)a_rows * row_bytes, STEP * 2};
    Source b_src = B_ROWS ? Source{static_cast<const char*>(task.b) + col0 * 2, (K * N - col0) * 2, STEP * N * 2}
                          : Source{static_cast<const char*>(task.b) + col0 * K * 2, (long long)b_cols * row_bytes, STEP * 2};
    a_src.skip(first);
    b_src.skip(first);
    // Each wave brings every fourth piece.  GATED: B's tile is up's rows, then gate's, the same pieces further on.
    unsigned a_off[2 * FM], b_off[FINISH == GATED ? FN : 2 * FN];
    constexpr int B_OFFS = FINISH == GATED ? FN : 2 * FN;
    const int chunk = (lane & 7) ^ swz<64>(8 * wave + lane / 8);  // the same for each of the wave's pieces: they are 32 rows apart
#pragma unroll
    for (int u = 0; u < 2 * FM; ++u) {
        const int q = wave + 4 * u, col = 64 * (q / 8) + 8 * chunk;
        if constexpr (A_ROWS) a_off[u] = col < a_rows ? (unsigned)((8 * (q % 8) + lane / 8) * M + col) * 2 : PAST_END;
        else a_off[u] = (unsigned)(8 * q + lane / 8) * row_bytes + chunk * 16;
    }
#pragma unroll
    for (int u = 0; u < B_OFFS; ++u) {
        const int q = wave + 4 * u, col = 64 * (q / 8) + 8 * chunk;
        if constexpr (B_ROWS) b_off[u] = col < b_cols ? (unsigned)((8 * (q % 8) + lane / 8) * N + col) * 2 : PAST_END;
        else b_off[u] = (unsigned)(8 * q + lane / 8) * row_bytes + chunk * 16;
    }
    const int rest_terms = (int)(K % STEP), cut = rest_terms ? steps - 1 : -1;  // the step that ends early
    const unsigned past = 8 * chunk >= rest_terms ? PAST_END : 0;
    const unsigned lds_wave = (unsigned)(size_t)(__attribute__((address_space(3))) char*)lds + wave * PIECE;
    u32x4 a_words, b_words, gate_words;
    auto aim = [&](int it) __attribute__((always_inline)) {  // at the loads of step `it`, which follows the last one aimed at
        a_words = a_src.next(it < last);
        b_words = b_src.next(it < last);
        if constexpr (FINISH == GATED) {
            const size_t gate = ((size_t)b_words[1] << 32 | b_words[0]) + (size_t)(N * K * 2);
            gate_words = u32x4{(unsigned)gate, (unsigned)(gate >> 32) & 0xffffu, b_words[2], b_words[3]};
        }
        if (it == cut) {  // the last step of all: what comes behind it reads nothing
            if constexpr (!A_ROWS)
#pragma unroll
                for (int u = 0; u < 2 * FM; ++u) a_off[u] |= past;
            if constexpr (!B_ROWS)
#pragma unroll
                for (int u = 0; u < B_OFFS; ++u) b_off[u] |= past;
        }
    };
    // The loads of a step, one after the other: U below 2 FM A's, then B's.
    auto fetch = [&](auto slot_, auto u_) __attribute__((always_inline)) {
        constexpr int SLOT_AT = decltype(slot_)::value * SLOT, U = decltype(u_)::value, V = U - 2 * FM;
        if constexpr (U < 2 * FM) bring<SLOT_AT + U * 4 * PIECE>(a_words, a_off[U], lds_wave);
        else if constexpr (V < B_OFFS) bring<SLOT_AT + A_BYTES + V * 4 * PIECE>(b_words, b_off[V], lds_wave);
        else bring<SLOT_AT + A_BYTES + V * 4 * PIECE>(gate_words, b_off[V - B_OFFS], lds_wave);
    };
    // first row of B's tile (column of the product) of a wave's j-th fragment
    auto b_row = [&](int j) __attribute__((always_inline)) {
        if (FINISH == GATED) return (j / (FN / 2)) * WIDE + 16 * FN * wn + 32 * (j % (FN / 2));
        return 32 * FN * wn + 32 * j;
    };
    // Where a lane reads.  Terms side by side: a row is 128 bytes, its 16-byte pieces swapped by row, which 32 rows further on is the same; a
    // place for each quarter of a step.  By rows: 64 columns are 8 KiB, 16 terms 2 KiB; two places for each fragment.
    int a_lane[A_ROWS ? 2 * FM : 4], b_lane[B_ROWS ? 2 * FN : 4];
    auto by_rows = [&](int n0, int half) __attribute__((always_inline)) {
        const int s = lane & 15, term = 8 * h + (s >> 2) + 4 * half, c = (n0 % 64 >> 3) + 2 * ((lane >> 4) & 1) + ((s & 3) >> 1);
        return n0 / 64 * 8 * PIECE + tile_off<64>(term, c) + ((s & 1) << 3);
    };
#pragma unroll
    for (int u = 0; u < (A_ROWS ? 2 * FM : 4); ++u) a_lane[u] = A_ROWS ? by_rows(32 * FM * wm + 32 * (u / 2), u % 2) : tile_off<64>(32 * FM * wm + m, 2 * u + h);
#pragma unroll
    for (int u = 0; u < (B_ROWS ? 2 * FN : 4); ++u)
        b_lane[u] = A_BYTES + (B_ROWS ? by_rows(b_row(u / 2), u % 2) : tile_off<64>((FINISH == GATED ? 16 : 32) * FN * wn + m, 2 * u + h));
    auto transposed = [&](int lo_at, int hi_at) __attribute__((always_inline)) {
        typedef __attribute__((address_space(3))) s16x4* lds_ptr;
        const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(lds + lo_at)));
        const u32x2 hi = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(lds + hi_at)));
        return u32x4{lo[0], lo[1], hi[0], hi[1]};
    };
    // Small tiles multiply little in a step: the fragments of a whole one are read while the last one's are multiplied (77 x 2048 x 5632 in tiles of
    // 64 x 128: 36 us by quarters, 27 by steps).
    constexpr bool AHEAD = FM == 1;
    constexpr int SETS = AHEAD ? 8 : 2;
    u32x4 af[SETS][FM], bf[SETS][FN];
    // The reads of a quarter of a step, in the order in which the products need them: A's first fragment, B's, A's others.
    auto read = [&](auto set_, auto ks_, auto slot_, auto u_) __attribute__((always_inline)) {
        constexpr int set = decltype(set_)::value, ks = decltype(ks_)::value, from = decltype(slot_)::value * SLOT, U = decltype(u_)::value;
        if constexpr (U == 0 || U > FN) {
            constexpr int i = U == 0 ? 0 : U - FN;
            if constexpr (A_ROWS) af[set][i] = transposed(a_lane[2 * i] + (from + ks * 2048), a_lane[2 * i + 1] + (from + ks * 2048));
            else af[set][i] = *reinterpret_cast<const u32x4*>(lds + a_lane[ks] + (from + i * 4096));
        } else {
            constexpr int j = U - 1, further = FINISH == GATED ? j / (FN / 2) * WIDE * 128 + j % (FN / 2) * 4096 : j * 4096;
            if constexpr (B_ROWS) bf[set][j] = transposed(b_lane[2 * j] + (from + ks * 2048), b_lane[2 * j + 1] + (from + ks * 2048));
            else bf[set][j] = *reinterpret_cast<const u32x4*>(lds + b_lane[ks] + (from + further));
        }
    };
    f32x16 acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;
    // The products of a quarter of a step, and behind each what may run beside it (the compiler would put a read right before its use).
    auto multiply = [&](auto set_, auto beside) __attribute__((always_inline)) {
        constexpr int set = decltype(set_)::value;
        each<FM * FN>([&](auto n) __attribute__((always_inline)) {
            constexpr int i = decltype(n)::value / FN, j = decltype(n)::value % FN, BESIDE = (READS + FM * FN - 1) / (FM * FN);
            acc[i][j] = Mma<T>::mma(bf[set][j], af[set][i], acc[i][j]);
            __builtin_amdgcn_sched_barrier(0);
            each<BESIDE>([&](auto e) __attribute__((always_inline)) {
                constexpr int U = decltype(n)::value * BESIDE + decltype(e)::value;
                if constexpr (U < READS) beside(Count<U>{});
            });
            __builtin_amdgcn_sched_barrier(0);
        });
    };
    // This wave's loads of the next step have landed and its reads of this one are done, and behind the barrier everyone's.
    auto meet = [&]() __attribute__((always_inline)) {
        __builtin_amdgcn_s_waitcnt(attn_mfma::waitcnt_vm((DEEP - 2) * LOADS));
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    };
    // The ring is filled, up to half of its last step; that one's other half goes beside the first products.
    each<DEEP>([&](auto s) __attribute__((always_inline)) {
        aim(first + decltype(s)::value);
        each<(decltype(s)::value == DEEP - 1 && !AHEAD ? READS : LOADS)>([&](auto u) __attribute__((always_inline)) { fetch(s, u); });
    });
    __builtin_amdgcn_s_waitcnt(attn_mfma::waitcnt_vm(AHEAD ? (DEEP - 1) * LOADS : (DEEP - 2) * LOADS + READS));
    asm volatile("s_barrier" ::: "memory");
    if constexpr (AHEAD) {
        each<4>([&](auto ks) __attribute__((always_inline)) { each<READS>([&](auto u) __attribute__((always_inline)) { read(ks, ks, Count<0>{}, u); }); });
        auto step = [&](auto n, int it) __attribute__((always_inline)) {
            constexpr int S = decltype(n)::value % DEEP, NEXT = (S + 1) % DEEP, now = decltype(n)::value % 2 * 4, then = 4 - now;
            meet();
            aim(it + DEEP);
            each<4>([&](auto ks) __attribute__((always_inline)) {
                constexpr int KS = decltype(ks)::value;
                multiply(Count<now + KS>{}, [&](auto u) __attribute__((always_inline)) {
                    read(Count<then + KS>{}, ks, Count<NEXT>{}, u);
                    if constexpr (KS % 2) fetch(Count<S>{}, Count<KS / 2 * READS + decltype(u)::value>{});
                });
            });
        };
        constexpr int TURN = DEEP % 2 ? 2 * DEEP : DEEP;  // after which places and sets are as before
        for (int it = first;;) {
            bool more = true;
            each<TURN>([&](auto n) __attribute__((always_inline)) {
                if (more) {
                    step(n, it);
                    more = ++it < last;
                }
            });
            if (!more) break;
        }
    } else {
        each<READS>([&](auto u) __attribute__((always_inline)) { read(Count<0>{}, Count<0>{}, Count<0>{}, u); });
        auto step = [&](auto s, int it) __attribute__((always_inline)) {
            constexpr int S = decltype(s)::value, NEXT = (S + 1) % DEEP, BEFORE = (S + DEEP - 1) % DEEP;
            // A step's place is free for the one a ring later from the barrier on.  Half of its loads go beside the quarter behind it, half
            // beside the quarter after that: all at once they queue up and hold up the products (tiles of 256 x 256, 6007 x 4096 x 11008:
            // 525 -> 486 us).
            multiply(Count<0>{}, [&](auto u) __attribute__((always_inline)) {
                read(Count<1>{}, Count<1>{}, s, u);
                fetch(Count<BEFORE>{}, Count<READS + decltype(u)::value>{});
            });
            multiply(Count<1>{}, [&](auto u) __attribute__((always_inline)) { read(Count<0>{}, Count<2>{}, s, u); });
            multiply(Count<0>{}, [&](auto u) __attribute__((always_inline)) { read(Count<1>{}, Count<3>{}, s, u); });
            meet();
            aim(it + DEEP);
            multiply(Count<1>{}, [&](auto u) __attribute__((always_inline)) {
                read(Count<0>{}, Count<0>{}, Count<NEXT>{}, u);
                fetch(s, u);
            });
        };
        if constexpr (DEEP == 2) {
            for (int it = first; it < last; it += 2) {  // behind the last of an odd number of steps comes one of zeros
                step(Count<0>{}, it);
                step(Count<1>{}, it + 1);
            }
        } else {
            for (int it = first;;) {
                bool more = true;
                each<DEEP>([&](auto n) __attribute__((always_inline)) {
                    if (more) {
                        step(n, it);
                        more = ++it < last;
                    }
                });
                if (!more) break;
            }
        }
    }
    // Nothing is under way into LDS any more, and behind the barrier nothing is read from it: from here on each wave has a part of its own, in
    // which 32 rows of its results turn from four columns a lane to eight, so that a wave's stores (and z's loads) are whole lines.
    __builtin_amdgcn_s_waitcnt(attn_mfma::waitcnt_vm(0));
    asm volatile("s_barrier" ::: "memory");
    constexpr int ROW = 32 * FN + 4;  // floats
    constexpr int WIDTH = (FINISH == GATED ? 16 : 32) * FN, EIGHTS = WIDTH / 8, TURNS = 32 * EIGHTS / 64;
    float* turn = reinterpret_cast<float*>(lds) + wave * 32 * ROW;
    const auto row_of = [&](int i, int u) { return row0 + 32 * FM * wm + 32 * i + (64 * u + lane) / EIGHTS; };
    const auto col_of = [&](int u) { return col0 + WIDTH * wn + (64 * u + lane) % EIGHTS * 8; };
    Beside more[2][TURNS];
#pragma unroll
    for (int u = 0; u < TURNS; ++u) more[0][u] = beside<T, FINISH>(task, row_of(0, u), col_of(u));
#pragma unroll
    for (int i = 0; i < FM; ++i) {
        if (FINISH == UNGATED && i + 1 < FM)
#pragma unroll
            for (int u = 0; u < TURNS; ++u) more[(i + 1) & 1][u] = beside<T, FINISH>(task, row_of(i + 1, u), col_of(u));
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int g = 0; g < 4; ++g)  // lane (m, h): columns 8 g + 4 h ... + 3 of row m
                *reinterpret_cast<f32x4*>(turn + m * ROW + 32 * j + 8 * g + 4 * h) =
                    f32x4{acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]};
#pragma unroll
        for (int u = 0; u < TURNS; ++u) {
            const int eight = 64 * u + lane, r = eight / EIGHTS, c = eight % EIGHTS * 8;
            const Eight x = load8(turn + r * ROW + c);
            Eight y{};
            if constexpr (FINISH == GATED) y = load8(turn + r * ROW + WIDTH + c);
            if (item < 0) {
                finish<T, FINISH>(task, row_of(i, u), col_of(u), x, y, more[FINISH == UNGATED ? i & 1 : 0][u]);
            } else {
                float* to = task.partial + partial_at<FM, FN>(item, wave, i) + eight * 8;
                store8(to, x);
                if constexpr (FINISH == GATED) store8(to + 32 * WIDTH, y);
            }
        }
    }
}

// Adds the parts of the tiles whose sums were cut, in order, and finishes them: a thread takes eight columns of a row.
template <typename T, int FM, int FN, Finish FINISH, bool PAIR> __global__ __launch_bounds__(256) void add_parts_kernel(Task task) {
    constexpr int WIDTH = (FINISH == GATED ? 16 : 32) * FN, EIGHTS = WIDTH / 8, COUNT = 32 * EIGHTS;
    const int rest = task.tiles - task.whole;
    const int id = blockIdx.x * 256 + threadIdx.x, eight = id % COUNT, i = id / COUNT % FM, wave = id / (COUNT * FM) % 4, tile = id / (COUNT * FM * 4);
    if (tile >= rest) return;
    int at = task.whole + tile, mt, nt;
    if constexpr (PAIR) turn_to(task, at);
    tile_at(at, task.m_tiles, task.n_tiles, mt, nt);
    const long long row = (long long)mt * 64 * FM + 32 * FM * (wave >> 1) + 32 * i + eight / EIGHTS;
    const long long col = (long long)nt * (FINISH == GATED ? 32 : 64) * FN + WIDTH * (wave & 1) + eight % EIGHTS * 8;
    if (row >= task.M || col >= task.N) return;
    const Beside more = beside<T, FINISH>(task, row, col);
    Eight x{}, y{};
#pragma unroll 4
    for (int part = 0; part < task.parts; ++part) {
        const float* from = task.partial + partial_at<FM, FN>(part * rest + tile, wave, i) + eight * 8;
        x = x + load8(from);
        if constexpr (FINISH == GATED) y = y + load8(from + 32 * WIDTH);
    }
    finish<T, FINISH>(task, row, col, x, y, more);
}

// Products of a few rows, both operands' terms side by side: a weight comes through once, and what counts is that all of the chip asks for it
// at once.  KW waves share the sums of COLUMNS columns (GATED: pairs of them) of all rows, each lane 16 bytes of every 512 KW terms; lanes are
// added by exchange, waves in order.  One token, 768 -> 2 x 2048 -> 768 in bf16: 4.8 and 2.3 us (64 x 128 tiles: 7.5 and 8.6), from
// memory 5.7 and 3.1.
constexpr int COLUMNS = 2;
template <typename T, int ROWS, Finish FINISH, int KW> __global__ __launch_bounds__(256) void few_rows_kernel(Task task) {
    constexpr int HALVES = FINISH == GATED ? 2 : 1;
    __shared__ float sums[4][HALVES][COLUMNS][ROWS];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, kw = wave % KW;
    const long long M = task.M, N = task.N, K = task.K, col0 = ((long long)blockIdx.x * (4 / KW) + wave / KW) * COLUMNS;
    const T* x = static_cast<const T*>(task.a);
    const T* w = static_cast<const T*>(task.b);
    const T *x_row[ROWS], *w_row[HALVES][COLUMNS];  // past the end: the last one again
#pragma unroll
    for (int r = 0; r < ROWS; ++r) x_row[r] = x + (r < M ? r : M - 1) * K;
#pragma unroll
    for (int s = 0; s < HALVES; ++s)
#pragma unroll
        for (int c = 0; c < COLUMNS; ++c) w_row[s][c] = w + (s * N + (col0 + c < N ? col0 + c : N - 1)) * K;
    float acc[HALVES][COLUMNS][ROWS] = {};
#pragma unroll 2
    for (long long k = (kw * 64 + lane) * 8; k < K; k += KW * 512) {
        Eight wv[HALVES][COLUMNS];
#pragma unroll
        for (int s = 0; s < HALVES; ++s)
#pragma unroll
            for (int c = 0; c < COLUMNS; ++c) wv[s][c] = load8(w_row[s][c] + k);
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            const Eight xv = load8(x_row[r] + k);
#pragma unroll
            for (int s = 0; s < HALVES; ++s)
#pragma unroll
                for (int c = 0; c < COLUMNS; ++c)
#pragma unroll
                    for (int e = 0; e < 8; ++e) acc[s][c][r] = fmaf(wv[s][c].v[e], xv.v[e], acc[s][c][r]);
        }
    }
#pragma unroll
    for (int s = 0; s < HALVES; ++s)
#pragma unroll
        for (int c = 0; c < COLUMNS; ++c)
#pragma unroll
            for (int r = 0; r < ROWS; ++r) {
#pragma unroll
                for (int off = 32; off >= 1; off >>= 1) acc[s][c][r] += __shfl_xor(acc[s][c][r], off, 64);
                if (lane == 0) sums[wave][s][c][r] = acc[s][c][r];
            }
    __syncthreads();
    const int c = lane / ROWS, r = lane % ROWS;
    const long long col = col0 + c;
    if (kw || c >= COLUMNS || r >= M || col >= N) return;
    float total[HALVES];
#pragma unroll
    for (int s = 0; s < HALVES; ++s) {
        total[s] = sums[wave][s][c][r];
#pragma unroll
        for (int q = 1; q < KW; ++q) total[s] += sums[wave + q][s][c][r];
        if (task.bias) total[s] += to_f32(static_cast<const T*>(task.bias)[s * N + col]);
    }
    const auto store = [](T* p, float v) { *reinterpret_cast<unsigned short*>(p) = (unsigned short)Mma<T>::pack2(v, 0.0f); };
    T* out = static_cast<T*>(task.out) + r * N + col;
    if constexpr (FINISH == PLAIN) {
        store(out, total[0]);
    } else {
        store(out, col < task.own ? total[0] * (total[1] * sigmoid(total[1])) : 0.0f);
        if (T* z = static_cast<T*>(task.z)) {
            store(z + r * 2 * N + col, total[0]);
            store(z + r * 2 * N + N + col, total[1]);
        }
    }
}

template <typename T, Finish FINISH> int launch_few(const Task& task, hipStream_t stream) {
    const auto with = [&](auto rows, auto kw) {
        constexpr int ROWS = decltype(rows)::value, KW = decltype(kw)::value, COUNT = COLUMNS * (4 / KW);
        hipLaunchKernelGGL((few_rows_kernel<T, ROWS, FINISH, KW>), dim3((unsigned)((task.N + COUNT - 1) / COUNT)), dim3(256), 0, stream, task);
        LBI_HIP_CHECK(hipGetLastError());
        return (int)LBI_OK;
    };
    const auto with_rows = [&](auto rows) {  // sums so long that a wave's share takes two loads and more are shared
        if (task.K <= 1024) return with(rows, Count<1>{});
        return task.K <= 2048 ? with(rows, Count<2>{}) : with(rows, Count<4>{});
    };
    if (task.M <= 1) return with_rows(Count<1>{});
    if (task.M <= 2) return with_rows(Count<2>{});
    return with_rows(Count<4>{});
}

template <typename T, int FM, int FN, int DEEP, bool A_ROWS, bool B_ROWS, Finish FINISH> int launch_tile(Task task, hipStream_t stream) {
    constexpr auto kernel = product_kernel<T, FM, FN, DEEP, A_ROWS, B_ROWS, FINISH>;
    constexpr size_t bytes = (size_t)DEEP * 8192 * (FM + FN);
    static_assert(bytes >= 4 * 32 * (32 * FN + 4) * sizeof(float), "the turn of the results fits the ring");
    if (int status = ensure_dynamic_lds<kernel>(bytes)) return status;
    constexpr int ROWS = 64 * FM, WIDE = FINISH == GATED ? 32 * FN : 64 * FN;
    task.m_tiles = (int)((task.M + ROWS - 1) / ROWS), task.n_tiles = (int)((task.N + WIDE - 1) / WIDE);
    task.second.m_tiles = (int)((task.second.M + ROWS - 1) / ROWS), task.second.n_tiles = (int)((task.second.N + WIDE - 1) / WIDE);
    const int rest = task.tiles - task.whole;
    hipLaunchKernelGGL(kernel, dim3((unsigned)(task.whole + rest * task.parts)), dim3(NT), bytes, stream, task);
    if (rest) {
        const int eights = rest * 4 * FM * 32 * (FINISH == GATED ? 2 : 4) * FN;
        hipLaunchKernelGGL((add_parts_kernel<T, FM, FN, FINISH, A_ROWS && B_ROWS>), dim3((unsigned)((eights + 255) / 256)), dim3(256), 0, stream, task);
    }
    LBI_HIP_CHECK(hipGetLastError());
    return LBI_OK;
}

// `partial`: l.bytes()
template <typename T, bool A_ROWS, bool B_ROWS, Finish FINISH> int launch(const Layout& l, Task task, void* partial, hipStream_t stream) {
    if (l.form == NONE) return fail(LBI_ERR_UNSUPPORTED, "lbi_gated_mlp: too many tiles");
    task.partial = static_cast<float*>(partial);
    task.tiles = l.tiles, task.whole = l.whole, task.parts = l.parts, task.part_steps = l.part_steps;
    if constexpr (!A_ROWS && !B_ROWS)
        if (l.form == FEW_ROWS) return launch_few<T, FINISH>(task, stream);
    int status = LBI_OK;
    each<FORMS>([&](auto f) {
        constexpr Form form = forms[decltype(f)::value];
        if constexpr (FINISH != GATED || form.fn % 2 == 0)
            if (l.form == decltype(f)::value) status = launch_tile<T, form.fm, form.fn, form.deep, A_ROWS, B_ROWS, FINISH>(task, stream);
    });
    return status;
}

// Sums over the rows of matrices [rows, N]: the gradients of the biases, both in one launch.  A workgroup takes 64 columns of one, eight to a
// thread's load, and a slab of rows.  The slabs' sums are added by a second launch, where there is more than one.  6007 rows of 13824 and 2560
// columns in fp16: 36 us, 5.5 TB/s, and 5 (one matrix after the other, four launches: 51).
constexpr int SUM_COLUMNS = 64, SUM_SLAB = 256;
struct Sum {
    const void* x;
    void* out;
    float* partials;  // [slabs, N]
    long long N;
    int first;  // workgroup (in x) with which it begins
};
struct Sums {
    Sum sum[2];
    long long rows;
    int slabs;
};
template <typename T> __device__ __forceinline__ void store_sum(const Sum& s, long long col, float total) {
    static_cast<unsigned short*>(s.out)[col] = (unsigned short)Mma<T>::pack2(total, 0.0f);
}
template <typename T> __global__ __launch_bounds__(256) void column_sums_kernel(Sums all) {
    __shared__ float part[32][SUM_COLUMNS + 1];
    const Sum& s = all.sum[(int)blockIdx.x >= all.sum[1].first];
    const T* x = static_cast<const T*>(s.x);
    const long long N = s.N, rows = all.rows, col0 = (long long)((int)blockIdx.x - s.first) * SUM_COLUMNS;
    const int c = threadIdx.x % 8 * 8, r = threadIdx.x / 8;
    const long long col = col0 + c, first = (long long)blockIdx.y * SUM_SLAB;
    float sum[8] = {};
    if (col < N)
#pragma unroll
        for (int u = 0; u < SUM_SLAB / 32; ++u) {
            const long long row = first + r + 32 * u;
            if (row < rows) {
                const u32x4 w = *reinterpret_cast<const u32x4*>(x + row * N + col);
#pragma unroll
                for (int e = 0; e < 4; ++e) sum[2 * e] += Mma<T>::lo(w[e]), sum[2 * e + 1] += Mma<T>::hi(w[e]);
            }
        }
#pragma unroll
    for (int e = 0; e < 8; ++e) part[r][c + e] = sum[e];
    __syncthreads();
    const long long mine = col0 + threadIdx.x;
    if (threadIdx.x < SUM_COLUMNS && mine < N) {
        float total = 0.0f;
        for (int q = 0; q < 32; ++q) total += part[q][threadIdx.x];
        if (all.slabs == 1) store_sum<T>(s, mine, total);
        else s.partials[(long long)blockIdx.y * N + mine] = total;
    }
}
template <typename T> __global__ __launch_bounds__(256) void add_slabs_kernel(Sums all) {
    __shared__ float part[16][17];
    const int c = threadIdx.x % 16, q = threadIdx.x / 16;
    const Sum& s = all.sum[(int)blockIdx.x >= 4 * all.sum[1].first];
    const long long col = (long long)((int)blockIdx.x - 4 * s.first) * 16 + c;
    float sum = 0.0f;
    if (col < s.N)
        for (int slab = q; slab < all.slabs; slab += 16) sum += s.partials[(long long)slab * s.N + col];
    part[q][c] = sum;
    __syncthreads();
    if (q == 0 && col < s.N) {
        for (int p = 1; p < 16; ++p) sum += part[p][c];
        store_sum<T>(s, col, sum);
    }
}
int slabs_of(int64_t rows) { return (int)((rows + SUM_SLAB - 1) / SUM_SLAB); }
// Of one matrix or two; an `out` that is not given takes its matrix out.
template <typename T> int column_sums(Sum a, Sum b, int64_t rows, hipStream_t stream) {
    if (!a.out) std::swap(a, b);
    if (!a.out) return LBI_OK;
    const int of_a = (int)((a.N + SUM_COLUMNS - 1) / SUM_COLUMNS), of_b = b.out ? (int)((b.N + SUM_COLUMNS - 1) / SUM_COLUMNS) : 0;
    a.first = 0, b.first = of_a;
    const Sums all{{a, b}, (long long)rows, slabs_of(rows)};
    hipLaunchKernelGGL((column_sums_kernel<T>), dim3((unsigned)(of_a + of_b), (unsigned)all.slabs), dim3(256), 0, stream, all);
    if (all.slabs > 1) hipLaunchKernelGGL((add_slabs_kernel<T>), dim3(4 * (unsigned)(of_a + of_b)), dim3(256), 0, stream, all);
    LBI_HIP_CHECK(hipGetLastError());
    return LBI_OK;
}

// Widths that are no whole 16-byte pieces run on copies padded with zeros, which change neither results nor gradients: one launch pads all
// operands, one cuts all results (padded one by one, a fill and a copy each, a call for two rows of 503 -> 2 x 159 -> 503 took 48 us, now 20).
struct Copy {
    const void* from;
    void* to;
    long long from_rows, from_columns, from_ld, to_rows, to_columns, to_ld, first;  // first: row of the launch with which it begins
};
struct Copies {
    Copy copy[8];
    int count;
    int lanes;  // of a row: a wave, or all four waves of a workgroup
    long long rows;
};
typedef unsigned u32x4_any __attribute__((ext_vector_type(4), aligned(2)));

__global__ __launch_bounds__(256) void copy_kernel(Copies all) {
    const int lane = threadIdx.x % all.lanes;
    const long long row = (long long)blockIdx.x * (256 / all.lanes) + threadIdx.x / all.lanes;
    if (row >= all.rows) return;
    int n = 0;
    while (n + 1 < all.count && all.copy[n + 1].first <= row) ++n;
    const Copy& c = all.copy[n];
    const long long r = row - c.first, there = r < c.from_rows ? c.from_columns : 0;
    const unsigned short* from = static_cast<const unsigned short*>(c.from) + r * c.from_ld;
    unsigned short* to = static_cast<unsigned short*>(c.to) + r * c.to_ld;
    for (long long col = lane * 8; col < c.to_columns; col += all.lanes * 8) {
        u32x4_any w = {0, 0, 0, 0};
        if (col + 8 <= there) {
            w = *reinterpret_cast<const u32x4_any*>(from + col);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                w[e] = (col + 2 * e < there ? from[col + 2 * e] : 0u) | (col + 2 * e + 1 < there ? (unsigned)from[col + 2 * e + 1] << 16 : 0u);
        }
        if (col + 8 <= c.to_columns) {
            *reinterpret_cast<u32x4_any*>(to + col) = w;
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (col + e < c.to_columns) to[col + e] = (unsigned short)(w[e / 2] >> (16 * (e % 2)));
        }
    }
}

size_t up(size_t bytes) { return (bytes + 255) / 256 * 256; }

// The copies of a call, and what they take of the workspace.  Without a base it only counts.
struct Padding {
    char* base;
    size_t bytes = 0;
    Copies in{}, out{};
    static int64_t eights(int64_t n) { return (n + 7) / 8 * 8; }
    static void add(Copies& list, const Copy& c) {
        list.copy[list.count] = c;
        list.copy[list.count++].first = list.rows;
        list.rows += c.to_rows;
    }
    // Room for `halves` matrices [rows, columns] behind one another, padded; where nothing is to pad, the tensor itself.
    void* room(const void* tensor, int64_t rows, int64_t columns, int64_t padded_rows, int64_t padded_columns, int halves) {
        if (!tensor || (rows == padded_rows && columns == padded_columns)) return const_cast<void*>(tensor);
        void* at = base + bytes;
        bytes += up((size_t)halves * padded_rows * padded_columns * 2);
        return at;
    }
    // Matrices one behind the other.
    const void* operand(const void* tensor, int64_t rows, int64_t columns, int64_t padded_rows, int64_t padded_columns, int halves = 1) {
        char* at = static_cast<char*>(room(tensor, rows, columns, padded_rows, padded_columns, halves));
        if (at != tensor)
            for (int half = 0; half < halves; ++half)
                add(in, {static_cast<const char*>(tensor) + half * rows * columns * 2, at + half * padded_rows * padded_columns * 2, rows, columns,
                         columns, padded_rows, padded_columns, padded_columns, 0});
        return at;
    }
    void* result(void* tensor, int64_t rows, int64_t columns, int64_t padded_rows, int64_t padded_columns, int halves = 1) {
        char* at = static_cast<char*>(room(tensor, rows, columns, padded_rows, padded_columns, halves));
        if (at != tensor)
            for (int half = 0; half < halves; ++half)
                add(out, {at + half * padded_rows * padded_columns * 2, static_cast<char*>(tensor) + half * rows * columns * 2, padded_rows,
                          padded_columns, padded_columns, rows, columns, columns, 0});
        return at;
    }
    // Two matrices side by side, [rows, 2 columns].
    const void* side_by_side(const void* tensor, int64_t rows, int64_t columns, int64_t padded) {
        char* at = static_cast<char*>(room(tensor, rows, columns, rows, padded, 2));
        if (at != tensor)
            for (int half = 0; half < 2; ++half)
                add(in, {static_cast<const char*>(tensor) + half * columns * 2, at + half * padded * 2, rows, columns, 2 * columns, rows, padded,
                         2 * padded, 0});
        return at;
    }
    void* result_side_by_side(void* tensor, int64_t rows, int64_t columns, int64_t padded) {
        char* at = static_cast<char*>(room(tensor, rows, columns, rows, padded, 2));
        if (at != tensor)
            for (int half = 0; half < 2; ++half)
                add(out, {at + half * padded * 2, static_cast<char*>(tensor) + half * columns * 2, rows, columns, 2 * padded, rows, columns,
                          2 * columns, 0});
        return at;
    }
    // Few long rows take a workgroup each (952 of 4063 ... 10799 columns: 15.0 -> 9.9 us), others a wave (7832 of 1001 ... 2811: 12.8 us, not 16.9).
    static int run(Copies list, hipStream_t stream) {
        if (!list.rows) return LBI_OK;
        long long columns = 0;
        for (int n = 0; n < list.count; ++n) columns = std::max(columns, list.copy[n].to_columns);
        list.lanes = columns >= 1024 && list.rows < 8 * device_compute_units() ? 256 : 64;
        const int rows = 256 / list.lanes;
        hipLaunchKernelGGL(copy_kernel, dim3((unsigned)((list.rows + rows - 1) / rows)), dim3(256), 0, stream, list);
        LBI_HIP_CHECK(hipGetLastError());
        return LBI_OK;
    }
};

constexpr int64_t MOST_WIDTH = 1 << 20, MOST_ROWS = 1 << 23;

int check(const char* who, int64_t rows, int64_t D, int64_t hidden, int64_t width, int dtype) {
    if (rows < 0 || D < 1 || hidden < 1 || width < 1)
        return fail(LBI_ERR_INVALID, "%s: bad size (rows=%lld D=%lld hidden=%lld width=%lld)", who, (long long)rows, (long long)D,
                    (long long)hidden, (long long)width);
    if (dtype != LBI_F16 && dtype != LBI_BF16) return fail(LBI_ERR_UNSUPPORTED, "%s: needs half or bfloat16", who);
    if (std::max({D, hidden, width}) > MOST_WIDTH || rows > MOST_ROWS)
        return fail(LBI_ERR_UNSUPPORTED, "%s: widths up to 2^20, rows up to 2^23", who);
    return LBI_OK;
}
bool on_grid(std::initializer_list<const void*> tensors) {
    for (const void* p : tensors)
        if (reinterpret_cast<uintptr_t>(p) % 16) return false;
    return true;
}

struct Forward {
    const void *x, *fc1_weight, *fc1_bias, *fc2_weight, *fc2_bias;
    void *fc1_output, *down_input, *out;
    int64_t rows, D, hidden, width;
};
struct Pullback {
    const void *g_out, *x, *fc1_output, *down_input, *fc1_weight, *fc2_weight;
    void *g_x, *g_fc1_weight, *g_fc2_weight, *g_fc1_bias, *g_fc2_bias;
    int64_t rows, D, hidden, width;
};

// The calls as they run: tensors padded where that is needed, the products' layouts, the workspace.
struct ForwardPlan {
    Padding pad;
    Forward t;
    Layout fc1, fc2;
    size_t partial;
    ForwardPlan(const Forward& c, void* workspace) : pad{static_cast<char*>(workspace)}, t(c) {
        const int cus = device_compute_units();
        t.D = Padding::eights(c.D), t.hidden = Padding::eights(c.hidden), t.width = Padding::eights(c.width);
        t.x = pad.operand(c.x, c.rows, c.D, c.rows, t.D);
        t.fc1_weight = pad.operand(c.fc1_weight, c.hidden, c.D, t.hidden, t.D, 2);
        t.fc1_bias = pad.operand(c.fc1_bias, 1, c.hidden, 1, t.hidden, 2);
        t.fc2_weight = pad.operand(c.fc2_weight, c.width, c.hidden, t.width, t.hidden);
        t.fc2_bias = pad.operand(c.fc2_bias, 1, c.width, 1, t.width);
        t.fc1_output = pad.result_side_by_side(c.fc1_output, c.rows, c.hidden, t.hidden);
        t.down_input = pad.result(c.down_input, c.rows, c.hidden, c.rows, t.hidden);
        t.out = pad.result(c.out, c.rows, c.width, c.rows, t.width);
        fc1 = layout_of(cus, t.rows, t.hidden, t.D, GATED, 0);
        fc2 = layout_of(cus, t.rows, t.width, t.hidden, PLAIN, 0);
        partial = pad.bytes;
    }
    size_t bytes() const { return partial + up(std::max(fc1.bytes(), fc2.bytes())); }
};
struct PullbackPlan {
    Padding pad;
    Pullback t;
    Layout a, x, weights;
    size_t g_fc1, sums, partial;
    PullbackPlan(const Pullback& c, void* workspace) : pad{static_cast<char*>(workspace)}, t(c) {
        const int cus = device_compute_units();
        t.D = Padding::eights(c.D), t.hidden = Padding::eights(c.hidden), t.width = Padding::eights(c.width);
        t.g_out = pad.operand(c.g_out, c.rows, c.width, c.rows, t.width);
        t.x = pad.operand(c.x, c.rows, c.D, c.rows, t.D);
        t.fc1_output = pad.side_by_side(c.fc1_output, c.rows, c.hidden, t.hidden);
        t.down_input = pad.operand(c.down_input, c.rows, c.hidden, c.rows, t.hidden);
        t.fc1_weight = pad.operand(c.fc1_weight, c.hidden, c.D, t.hidden, t.D, 2);
        t.fc2_weight = pad.operand(c.fc2_weight, c.width, c.hidden, t.width, t.hidden);
        t.g_x = pad.result(c.g_x, c.rows, c.D, c.rows, t.D);
        t.g_fc1_weight = pad.result(c.g_fc1_weight, c.hidden, c.D, t.hidden, t.D, 2);
        t.g_fc2_weight = pad.result(c.g_fc2_weight, c.width, c.hidden, t.width, t.hidden);
        t.g_fc1_bias = pad.result(c.g_fc1_bias, 1, c.hidden, 1, t.hidden, 2);
        t.g_fc2_bias = pad.result(c.g_fc2_bias, 1, c.width, 1, t.width);
        a = layout_of(cus, t.rows, t.hidden, t.width, UNGATED, 1);
        x = layout_of(cus, t.rows, t.D, 2 * t.hidden, PLAIN, 1);
        weights = layout_of(cus, 2 * t.hidden, t.D, t.rows, PLAIN, 2, t.width, t.hidden);
        g_fc1 = pad.bytes;
        sums = g_fc1 + up((size_t)t.rows * 2 * t.hidden * 2);
        partial = sums + up((size_t)slabs_of(t.rows) * (2 * t.hidden + t.width) * sizeof(float));
    }
    size_t bytes() const { return partial + up(std::max({a.bytes(), x.bytes(), weights.bytes()})); }
};

// Every tensor given: what a plan that only counts is told.
const void* const SOME = reinterpret_cast<const void*>(256);
void* const SOME_RESULT = reinterpret_cast<void*>(256);

}  // namespace
}  // namespace block_mlp
}  // namespace lbi

extern "C" size_t lbi_gated_mlp_workspace_bytes(int64_t rows, int64_t D, int64_t hidden, int64_t width) {
    using namespace lbi::block_mlp;
    if (check("lbi_gated_mlp", rows, D, hidden, width, LBI_BF16) || rows == 0) return 0;
    return ForwardPlan({SOME, SOME, SOME, SOME, SOME, SOME_RESULT, SOME_RESULT, SOME_RESULT, rows, D, hidden, width}, nullptr).bytes();
}

extern "C" int lbi_gated_mlp(const void* x, const void* fc1_weight, const void* fc1_bias, const void* fc2_weight, const void* fc2_bias,
                             void* fc1_output, void* down_input, void* out, void* workspace, size_t workspace_bytes, int64_t rows,
                             int64_t D, int64_t hidden, int64_t width, int dtype, void* stream) {
    using namespace lbi;
    using namespace lbi::block_mlp;
    clear_error();
    if (int bad = check("lbi_gated_mlp", rows, D, hidden, width, dtype)) return bad;
    if (rows == 0) return LBI_OK;
    if (!x || !fc1_weight || !fc2_weight || !down_input || !out) return fail(LBI_ERR_INVALID, "lbi_gated_mlp: null pointer");
    if (!on_grid({x, fc1_weight, fc1_bias, fc2_weight, fc2_bias, fc1_output, down_input, out}) || reinterpret_cast<uintptr_t>(workspace) % 256)
        return fail(LBI_ERR_INVALID, "lbi_gated_mlp: tensors must be 16-byte aligned, the workspace 256");
    const ForwardPlan p({x, fc1_weight, fc1_bias, fc2_weight, fc2_bias, fc1_output, down_input, out, rows, D, hidden, width}, workspace);
    const size_t need = p.bytes();
    if (need && (!workspace || workspace_bytes < need))
        return fail(LBI_ERR_WORKSPACE, "lbi_gated_mlp: workspace of %zu bytes needed, %zu given", need, workspace_bytes);
    const hipStream_t on = static_cast<hipStream_t>(stream);
    const auto run = [&](auto type) {
        using T = decltype(type);
        const Forward& t = p.t;
        void* partial = static_cast<char*>(workspace) + p.partial;
        if (int s = launch<T, false, false, GATED>(p.fc1, {t.x, t.fc1_weight, t.fc1_bias, t.down_input, t.fc1_output, rows, t.hidden, t.D, hidden}, partial,
                                                     on))
            return s;
        return launch<T, false, false, PLAIN>(p.fc2, {t.down_input, t.fc2_weight, t.fc2_bias, t.out, nullptr, rows, t.width, t.hidden}, partial, on);
    };
    if (int s = Padding::run(p.pad.in, on)) return s;
    if (int s = dtype == LBI_F16 ? run(_Float16{}) : run(bf16_raw{})) return s;
    return Padding::run(p.pad.out, on);
}

extern "C" size_t lbi_gated_mlp_vjp_workspace_bytes(int64_t rows, int64_t D, int64_t hidden, int64_t width) {
    using namespace lbi::block_mlp;
    if (check("lbi_gated_mlp_vjp", rows, D, hidden, width, LBI_BF16) || rows == 0) return 0;
    return PullbackPlan({SOME, SOME, SOME, SOME, SOME, SOME, SOME_RESULT, SOME_RESULT, SOME_RESULT, SOME_RESULT, SOME_RESULT, rows, D, hidden, width},
                        nullptr).bytes();
}

extern "C" int lbi_gated_mlp_vjp(const void* g_out, const void* x, const void* fc1_output, const void* down_input, const void* fc1_weight,
                                 const void* fc2_weight, void* g_x, void* g_fc1_weight, void* g_fc2_weight, void* g_fc1_bias,
                                 void* g_fc2_bias, void* workspace, size_t workspace_bytes, int64_t rows, int64_t D, int64_t hidden,
                                 int64_t width, int dtype, void* stream) {
    using namespace lbi;
    using namespace lbi::block_mlp;
    clear_error();
    if (int bad = check("lbi_gated_mlp_vjp", rows, D, hidden, width, dtype)) return bad;
    if (rows == 0) return fail(LBI_ERR_UNSUPPORTED, "lbi_gated_mlp_vjp: no rows");
    if (!g_out || !x || !fc1_output || !down_input || !fc1_weight || !fc2_weight || !g_x || !g_fc1_weight || !g_fc2_weight)
        return fail(LBI_ERR_INVALID, "lbi_gated_mlp_vjp: null pointer");
    if (!on_grid({g_out, x, fc1_output, down_input, fc1_weight, fc2_weight, g_x, g_fc1_weight, g_fc2_weight, g_fc1_bias, g_fc2_bias}) ||
        reinterpret_cast<uintptr_t>(workspace) % 256)
        return fail(LBI_ERR_INVALID, "lbi_gated_mlp_vjp: tensors must be 16-byte aligned, the workspace 256");
    const PullbackPlan p({g_out, x, fc1_output, down_input, fc1_weight, fc2_weight, g_x, g_fc1_weight, g_fc2_weight, g_fc1_bias, g_fc2_bias, rows, D,
                          hidden, width}, workspace);
    if (!workspace || workspace_bytes < p.bytes())
        return fail(LBI_ERR_WORKSPACE, "lbi_gated_mlp_vjp: workspace of %zu bytes needed, %zu given", p.bytes(), workspace_bytes);
    const hipStream_t on = static_cast<hipStream_t>(stream);
    char* base = static_cast<char*>(workspace);
    void *g_fc1 = base + p.g_fc1, *partial = base + p.partial;
    float* sums = reinterpret_cast<float*>(base + p.sums);
    const auto run = [&](auto type) {
        using T = decltype(type);
        const Pullback& t = p.t;
        void* z = const_cast<void*>(t.fc1_output);
        if (int s = launch<T, false, true, UNGATED>(p.a, {t.g_out, t.fc2_weight, nullptr, g_fc1, z, rows, t.hidden, t.width, hidden}, partial, on)) return s;
        if (int s = launch<T, false, true, PLAIN>(p.x, {g_fc1, t.fc1_weight, nullptr, t.g_x, nullptr, rows, t.D, 2 * t.hidden}, partial, on)) return s;
        // Both weights' gradients are sums over the rows: one list of tiles, with one last round (the whole call for one row of 768 / 2048: 33 -> 29 us, 16000
        // of 256 / 1024 122 -> 112, 8192 of 768 / 2048 241 -> 230; 6007 of 2560 / 6912, whose products fill the chip alone, 1290 -> 1310).
        Task weights{g_fc1, t.x, nullptr, t.g_fc1_weight, nullptr, 2 * t.hidden, t.D, rows};
        weights.second = {t.g_out, t.down_input, t.g_fc2_weight, t.width, t.hidden};
        if (int s = launch<T, true, true, PLAIN>(p.weights, weights, partial, on)) return s;
        return column_sums<T>({g_fc1, t.g_fc1_bias, sums, 2 * t.hidden, 0}, {t.g_out, t.g_fc2_bias, sums + slabs_of(rows) * 2 * t.hidden, t.width, 0}, rows, on);
    };
    if (int s = Padding::run(p.pad.in, on)) return s;
    if (int s = dtype == LBI_F16 ? run(_Float16{}) : run(bf16_raw{})) return s;
    return Padding::run(p.pad.out, on);
}
