// The gated MLP of a Transformer block and its pullback, in one 16-bit type, sums in fp32:
//
//   forward    z = x W1^T + b1,  [u | g] = z,  a = u * g * sigmoid(g),  out = a W2^T + b2
//   pullback   g_a = g_out W2;  g_u = g_a silu(g), g_g = g_a u silu'(g);  g_x = [g_u | g_g] W1
//
// (the weights' gradients are lbi_weight_gradient's).  All four products are one kernel: a workgroup of four waves owns a tile of results,
// 32 FM x 32 FN of them a wave, and takes 32 terms of the sums a step through LDS, in a ring of four steps.  Operands arrive by
// buffer_load ... lds (what lies past the end of an operand is zero, so ragged sizes take the same loop); one whose terms lie side by side is
// read in 16-byte pieces, one whose terms are its rows through transposing reads.  The product is formed as C^T: a lane ends up with four
// neighbouring columns of one row.  Up and gate of one column meet in one lane, so the gate costs no pass of its own in either direction.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "lbi_attn_mfma.h"
#include "lbi_attn_dkdv128.h"

namespace lbi {
namespace block_mlp {
namespace {

using attn_mfma::Mma;
using attn_mfma::s16x4;
using attn_mfma::swz;
using attn_mfma::tile_off;
using attn_mfma::u32x2;
using attn_mfma::u32x4;

constexpr int STEP = 32, RING = 4, NT = 256;
constexpr unsigned PAST_END = 1u << 31;
constexpr int PIECE = 1024;  // bytes that a wave's load brings: 16 rows of 32 terms, or 8 terms of 64 columns

// What becomes of the sums.
enum Finish {
    PLAIN,   // out = C + bias
    GATED,   // C is up and gate of one column: activation, and z where it is kept
    UNGATED  // C is the activation's cotangent: that of z
};

struct Task {
    const void *a, *b, *bias;  // A [M, K]; B [N, K] or, transposed, [K, N]; GATED: B [2N, K]
    void *out, *z;             // GATED: z [M, 2N] written if given; UNGATED: z [M, 2N] read, out [M, 2N]
    long long M, N, K;
    int m_tiles, n_tiles;
};

__device__ __forceinline__ float sigmoid(float x) { return 1.0f / (1.0f + __expf(-x)); }

template <typename T> __device__ __forceinline__ f32x4 load_four(const T* p) {
    const u32x2 w = *reinterpret_cast<const u32x2*>(p);
    return f32x4{Mma<T>::lo(w[0]), Mma<T>::hi(w[0]), Mma<T>::lo(w[1]), Mma<T>::hi(w[1])};
}
template <typename T> __device__ __forceinline__ void store_four(T* p, f32x4 v) {
    *reinterpret_cast<u32x2*>(p) = u32x2{Mma<T>::pack2(v[0], v[1]), Mma<T>::pack2(v[2], v[3])};
}

// 1 KiB from memory to LDS by one wave: lane l brings the 16 bytes at `base` + `off`, zeros from `bytes` on.
__device__ __forceinline__ void bring(const char* base, unsigned off, unsigned bytes, unsigned lds) {
    attn_mfma::dma_tile<true>(base, off, bytes, lds);
}

// Rows of an operand whose terms lie side by side.  In LDS a row of a step is 64 bytes, four rows a bank line, its four chunks swapped by row.
__device__ __forceinline__ int row_chunk(int row, int chunk) { return row * 64 + ((chunk ^ ((row >> 2) & 3)) << 4); }

// Workgroup -> tile.  Ids equal mod 8 share an L2: they get neighbouring tiles, eight rows of them at a time.
__device__ __forceinline__ void tile_of(int id, int m_tiles, int n_tiles, int& mt, int& nt) {
    const int count = m_tiles * n_tiles, lot = count / 8, left = count % 8, x = id % 8;
    const int at = x * lot + min(x, left) + id / 8;
    constexpr int ROWS = 8;
    const int band = at / (ROWS * n_tiles), in = at - band * ROWS * n_tiles, rows = min(ROWS, m_tiles - band * ROWS);
    mt = band * ROWS + in % rows;
    nt = in / rows;
}

template <typename T, int FM, int FN, bool B_ROWS, Finish FINISH>  // B_ROWS: the terms of B are its rows
__global__ __launch_bounds__(NT) void product_kernel(Task task) {
    constexpr int BM = 64 * FM, BN = 64 * FN;  // rows and columns of B's tile
    constexpr int A_BYTES = BM * 64, SLOT = A_BYTES + BN * 64, LOADS = FM + FN;
    extern __shared__ __align__(16) char lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int m = lane & 31, h = lane >> 5, wm = wave >> 1, wn = wave & 1;
    constexpr int COLUMNS = FINISH == GATED ? BN / 2 : BN;
    const long long M = task.M, N = task.N, K = task.K;
    int mt, nt;
    tile_of((int)blockIdx.x, task.m_tiles, task.n_tiles, mt, nt);
    const long long row0 = (long long)mt * BM, col0 = (long long)nt * COLUMNS;
    const int steps = (int)((K + STEP - 1) / STEP);
    const unsigned row_bytes = (unsigned)K * 2;
    // sources: A's rows, B's rows (GATED: up's and gate's) or B's terms
    const int a_rows = (int)(M - row0 < BM ? M - row0 : BM), b_cols = (int)(N - col0 < COLUMNS ? N - col0 : COLUMNS);
    const char* a_src = static_cast<const char*>(task.a) + row0 * K * 2;
    const char* b_src = static_cast<const char*>(task.b) + (B_ROWS ? col0 : col0 * K) * 2;
    unsigned a_off[FM], b_off[FN];
    const char* b_from[FN];
    const int chunk = (lane & 3) ^ ((lane >> 4) & 3);
#pragma unroll
    for (int u = 0; u < FM; ++u) {
        const int row = 16 * (wave + 4 * u) + lane / 4;
        a_off[u] = row < a_rows ? (unsigned)row * row_bytes + chunk * 16 : PAST_END;
    }
#pragma unroll
    for (int u = 0; u < FN; ++u) {
        const int q = wave + 4 * u;
        b_from[u] = b_src;
        if constexpr (B_ROWS) {
            const int term = 8 * (q % 4) + lane / 8, col = 64 * (q / 4) + 8 * ((lane % 8) ^ swz<64>(term));
            b_off[u] = col < b_cols ? (unsigned)(term * N + col) * 2 : PAST_END;
        } else {
            int row = 16 * q + lane / 4;
            if (FINISH == GATED && 16 * q >= COLUMNS) {  // the same for the whole wave
                row -= COLUMNS;
                b_from[u] += N * K * 2;
            }
            b_off[u] = row < b_cols ? (unsigned)row * row_bytes + chunk * 16 : PAST_END;
        }
    }
    const unsigned lds0 = (unsigned)(size_t)(__attribute__((address_space(3))) char*)lds;
    auto fetch = [&](int it, int slot) __attribute__((always_inline)) {
        const unsigned to = lds0 + slot * SLOT + wave * PIECE;
        const bool there = it < steps;
        const long long k = (long long)it * STEP;
        const bool cut = k + 8 * chunk >= K;  // pieces past the end of a row
        const unsigned a_bytes = there ? (unsigned)(a_rows * (long long)row_bytes - k * 2) : 0;
#pragma unroll
        for (int u = 0; u < FM; ++u) bring(a_src + k * 2, cut ? PAST_END : a_off[u], a_bytes, to + u * 4 * PIECE);
        if constexpr (B_ROWS) {
            const long long terms = K - k < STEP ? K - k : STEP;
            const unsigned b_bytes = there ? (unsigned)((terms * N - col0) * 2) : 0;
#pragma unroll
            for (int u = 0; u < FN; ++u) bring(b_src + k * N * 2, b_off[u], b_bytes, to + A_BYTES + u * 4 * PIECE);
        } else {
            const unsigned b_bytes = there ? (unsigned)(b_cols * (long long)row_bytes - k * 2) : 0;
#pragma unroll
            for (int u = 0; u < FN; ++u) bring(b_from[u] + k * 2, cut ? PAST_END : b_off[u], b_bytes, to + A_BYTES + u * 4 * PIECE);
        }
    };
    // first row of B's tile (column of the product) of a wave's j-th fragment
    auto b_row = [&](int j) __attribute__((always_inline)) {
        if (FINISH == GATED) return (j / (FN / 2)) * COLUMNS + 16 * FN * wn + 32 * (j % (FN / 2));
        return 32 * FN * wn + 32 * j;
    };
    u32x4 af[2][FM], bf[2][FN];
    auto read = [&](int ks, int slot) __attribute__((always_inline)) {
        const char* at_a = lds + slot * SLOT;
        const char* at_b = at_a + A_BYTES;
#pragma unroll
        for (int i = 0; i < FM; ++i)
            af[ks][i] = *reinterpret_cast<const u32x4*>(at_a + row_chunk(32 * FM * wm + 32 * i + m, 2 * ks + h));
#pragma unroll
        for (int j = 0; j < FN; ++j) {
            if constexpr (B_ROWS) {
                const int n0 = b_row(j);
                const char* tile = at_b + n0 / 64 * 4 * PIECE;
                const int s = lane & 15, term = 16 * ks + 8 * h + (s >> 2), c = (n0 % 64 >> 3) + 2 * ((lane >> 4) & 1) + ((s & 3) >> 1);
                typedef __attribute__((address_space(3))) s16x4* lds_ptr;
                const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(tile + tile_off<64>(term, c) + ((s & 1) << 3))));
                const u32x2 hi = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(tile + tile_off<64>(term + 4, c) + ((s & 1) << 3))));
                bf[ks][j] = u32x4{lo[0], lo[1], hi[0], hi[1]};
            } else {
                bf[ks][j] = *reinterpret_cast<const u32x4*>(at_b + row_chunk(b_row(j) + m, 2 * ks + h));
            }
        }
    };
    f32x16 acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;
    auto multiply = [&](int ks) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j) acc[i][j] = Mma<T>::mma(bf[ks][j], af[ks][i], acc[i][j]);
    };
#pragma unroll
    for (int u = 0; u < RING; ++u) fetch(u, u);
    __builtin_amdgcn_s_waitcnt(attn_mfma::waitcnt_vm((RING - 1) * LOADS));
    asm volatile("s_barrier" ::: "memory");
    read(0, 0);
    int slot = 0;
    for (int it = 0; it < steps; ++it) {
        const int next = slot + 1 == RING ? 0 : slot + 1;
        read(1, slot);
        multiply(0);
        // this wave's loads of the next step have landed and its reads of this one are done, and behind the barrier everyone's: the next
        // step can be read, and this one's place filled
        __builtin_amdgcn_s_waitcnt(attn_mfma::waitcnt_vm((RING - 2) * LOADS));
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        fetch(it + RING, slot);
        read(0, next);
        multiply(1);
        slot = next;
    }
    __builtin_amdgcn_s_waitcnt(attn_mfma::waitcnt_vm(0));  // nothing is under way into LDS when the workgroup ends
    // lane (m, h): columns 8 g + 4 h ... + 3 of row m of each 32 x 32 results
    const T* bias = static_cast<const T*>(task.bias);
    T* out = static_cast<T*>(task.out);
    T* z = static_cast<T*>(task.z);
#pragma unroll
    for (int i = 0; i < FM; ++i) {
        const long long row = row0 + 32 * FM * wm + 32 * i + m;
        if (row >= M) continue;
#pragma unroll
        for (int j = 0; j < (FINISH == GATED ? FN / 2 : FN); ++j)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const long long col = col0 + b_row(j) + 8 * g + 4 * h;
                if (col >= N) continue;
                auto four = [&](const f32x16& c) { return f32x4{c[4 * g], c[4 * g + 1], c[4 * g + 2], c[4 * g + 3]}; };
                f32x4 c = four(acc[i][j]);
                if constexpr (FINISH == PLAIN) {
                    if (bias) {
                        const f32x4 b = load_four(bias + col);
#pragma unroll
                        for (int e = 0; e < 4; ++e) c[e] += b[e];
                    }
                    store_four(out + row * N + col, c);
                } else if constexpr (FINISH == GATED) {
                    f32x4 gate = four(acc[i][j + FN / 2]), act;
                    if (bias) {
                        const f32x4 b = load_four(bias + col), bg = load_four(bias + N + col);
#pragma unroll
                        for (int e = 0; e < 4; ++e) c[e] += b[e], gate[e] += bg[e];
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) act[e] = c[e] * (gate[e] * sigmoid(gate[e]));
                    store_four(out + row * N + col, act);
                    if (z) {
                        store_four(z + row * 2 * N + col, c);
                        store_four(z + row * 2 * N + N + col, gate);
                    }
                } else {
                    const f32x4 up = load_four(z + row * 2 * N + col), gate = load_four(z + row * 2 * N + N + col);
                    f32x4 g_up, g_gate;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float open = sigmoid(gate[e]);
                        g_up[e] = c[e] * (gate[e] * open);
                        g_gate[e] = c[e] * up[e] * (open * (1.0f + gate[e] * (1.0f - open)));
                    }
                    store_four(out + row * 2 * N + col, g_up);
                    store_four(out + row * 2 * N + N + col, g_gate);
                }
            }
    }
}

template <typename T, int FM, int FN, bool B_ROWS, Finish FINISH> int launch_tile(Task task, hipStream_t stream) {
    constexpr auto kernel = product_kernel<T, FM, FN, B_ROWS, FINISH>;
    constexpr int BM = 64 * FM, COLUMNS = FINISH == GATED ? 32 * FN : 64 * FN;
    constexpr size_t bytes = (size_t)RING * 4096 * (FM + FN);
    if (int status = ensure_dynamic_lds<kernel>(bytes)) return status;
    task.m_tiles = (int)((task.M + BM - 1) / BM);
    task.n_tiles = (int)((task.N + COLUMNS - 1) / COLUMNS);
    hipLaunchKernelGGL(kernel, dim3((unsigned)(task.m_tiles * task.n_tiles)), dim3(NT), bytes, stream, task);
    LBI_HIP_CHECK(hipGetLastError());
    return LBI_OK;
}

template <typename T, bool B_ROWS, Finish FINISH> int launch(const Task& task, hipStream_t stream) {
    return launch_tile<T, 2, 2, B_ROWS, FINISH>(task, stream);
}

// Sums over the rows of x [rows, N]: the gradient of a bias.  A workgroup takes 64 columns, eight to a thread's load, and a slab of rows;
// the slabs' sums go to `partials` [slabs, N].
constexpr int SUM_COLUMNS = 64, SUM_SLAB = 256;
template <typename T>
__global__ __launch_bounds__(256) void column_sums_kernel(const T* __restrict__ x, float* __restrict__ partials, long long rows, long long N) {
    __shared__ float part[32][SUM_COLUMNS + 1];
    const int c = threadIdx.x % 8 * 8, r = threadIdx.x / 8;
    const long long col = (long long)blockIdx.x * SUM_COLUMNS + c, first = (long long)blockIdx.y * SUM_SLAB;
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
    if (threadIdx.x < SUM_COLUMNS && (long long)blockIdx.x * SUM_COLUMNS + threadIdx.x < N) {
        float total = 0.0f;
        for (int q = 0; q < 32; ++q) total += part[q][threadIdx.x];
        partials[(long long)blockIdx.y * N + (long long)blockIdx.x * SUM_COLUMNS + threadIdx.x] = total;
    }
}
template <typename T>
__global__ __launch_bounds__(256) void add_slabs_kernel(const float* __restrict__ partials, T* __restrict__ out, int slabs, long long N) {
    __shared__ float part[16][17];
    const int c = threadIdx.x % 16, q = threadIdx.x / 16;
    const long long col = (long long)blockIdx.x * 16 + c;
    float sum = 0.0f;
    if (col < N)
        for (int s = q; s < slabs; s += 16) sum += partials[(long long)s * N + col];
    part[q][c] = sum;
    __syncthreads();
    if (q == 0 && col < N) {
        for (int p = 1; p < 16; ++p) sum += part[p][c];
        *reinterpret_cast<unsigned short*>(out + col) = (unsigned short)Mma<T>::pack2(sum, 0.0f);
    }
}
int slabs_of(int64_t rows) { return (int)((rows + SUM_SLAB - 1) / SUM_SLAB); }
template <typename T> int column_sums(const void* x, void* out, float* partials, int64_t rows, int64_t N, hipStream_t stream) {
    const int slabs = slabs_of(rows);
    hipLaunchKernelGGL((column_sums_kernel<T>), dim3((unsigned)((N + SUM_COLUMNS - 1) / SUM_COLUMNS), (unsigned)slabs), dim3(256), 0, stream,
                       static_cast<const T*>(x), partials, (long long)rows, (long long)N);
    hipLaunchKernelGGL((add_slabs_kernel<T>), dim3((unsigned)((N + 15) / 16)), dim3(256), 0, stream, partials, static_cast<T*>(out), slabs,
                       (long long)N);
    LBI_HIP_CHECK(hipGetLastError());
    return LBI_OK;
}

constexpr int64_t MOST_WIDTH = 1 << 20, MOST_ROWS = 1 << 23;

int check(const char* who, int64_t rows, int64_t D, int64_t hidden, int64_t width, int dtype) {
    if (rows < 0 || D < 0 || hidden < 0 || width < 0)
        return fail(LBI_ERR_INVALID, "%s: bad size (rows=%lld D=%lld hidden=%lld width=%lld)", who, (long long)rows, (long long)D,
                    (long long)hidden, (long long)width);
    if (dtype != LBI_F16 && dtype != LBI_BF16) return fail(LBI_ERR_UNSUPPORTED, "%s: needs half or bfloat16", who);
    if (D < 8 || hidden < 8 || width < 8 || D % 8 || hidden % 8 || width % 8 || std::max({D, hidden, width}) > MOST_WIDTH || rows > MOST_ROWS)
        return fail(LBI_ERR_UNSUPPORTED, "%s: widths are multiples of 8, up to 2^20, rows up to 2^23", who);
    return LBI_OK;
}
bool on_grid(std::initializer_list<const void*> tensors) {
    for (const void* p : tensors)
        if (reinterpret_cast<uintptr_t>(p) % 16) return false;
    return true;
}

size_t up(size_t bytes) { return (bytes + 255) / 256 * 256; }
struct Parts {  // of the pullback's workspace, in bytes
    size_t g_fc1, sums, gradient;
};
Parts parts_of(int64_t rows, int64_t D, int64_t hidden, int64_t width) {
    return {up((size_t)rows * 2 * hidden * 2), up((size_t)slabs_of(rows) * std::max(2 * hidden, width) * sizeof(float)),
            up(std::max(lbi_weight_gradient_workspace_bytes(2 * hidden, D, rows), lbi_weight_gradient_workspace_bytes(width, hidden, rows)))};
}

}  // namespace
}  // namespace block_mlp
}  // namespace lbi

extern "C" int lbi_gated_mlp(const void* x, const void* fc1_weight, const void* fc1_bias, const void* fc2_weight, const void* fc2_bias,
                             void* fc1_output, void* down_input, void* out, int64_t rows, int64_t D, int64_t hidden, int64_t width,
                             int dtype, void* stream) {
    using namespace lbi;
    using namespace lbi::block_mlp;
    clear_error();
    if (int bad = check("lbi_gated_mlp", rows, D, hidden, width, dtype)) return bad;
    if (rows == 0) return LBI_OK;
    if (!x || !fc1_weight || !fc2_weight || !down_input || !out) return fail(LBI_ERR_INVALID, "lbi_gated_mlp: null pointer");
    if (!on_grid({x, fc1_weight, fc1_bias, fc2_weight, fc2_bias, fc1_output, down_input, out}))
        return fail(LBI_ERR_INVALID, "lbi_gated_mlp: tensors must be 16-byte aligned");
    const hipStream_t on = static_cast<hipStream_t>(stream);
    const auto run = [&](auto t) {
        using T = decltype(t);
        if (int status = launch<T, false, GATED>(Task{x, fc1_weight, fc1_bias, down_input, fc1_output, rows, hidden, D, 0, 0}, on)) return status;
        return launch<T, false, PLAIN>(Task{down_input, fc2_weight, fc2_bias, out, nullptr, rows, width, hidden, 0, 0}, on);
    };
    return dtype == LBI_F16 ? run(_Float16{}) : run(bf16_raw{});
}

extern "C" size_t lbi_gated_mlp_vjp_workspace_bytes(int64_t rows, int64_t D, int64_t hidden, int64_t width) {
    using namespace lbi::block_mlp;
    if (check("lbi_gated_mlp_vjp", rows, D, hidden, width, LBI_BF16) || rows == 0) return 0;
    const Parts p = parts_of(rows, D, hidden, width);
    return p.g_fc1 + p.sums + p.gradient;
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
    const Parts p = parts_of(rows, D, hidden, width);
    if (!workspace || workspace_bytes < p.g_fc1 + p.sums + p.gradient)
        return fail(LBI_ERR_WORKSPACE, "lbi_gated_mlp_vjp: workspace of %zu bytes needed, %zu given", p.g_fc1 + p.sums + p.gradient, workspace_bytes);
    const hipStream_t on = static_cast<hipStream_t>(stream);
    char* g_fc1 = static_cast<char*>(workspace);
    float* sums = reinterpret_cast<float*>(g_fc1 + p.g_fc1);
    char* gradient = g_fc1 + p.g_fc1 + p.sums;
    const auto run = [&](auto t) {
        using T = decltype(t);
        if (int s = launch<T, true, UNGATED>(Task{g_out, fc2_weight, nullptr, g_fc1, const_cast<void*>(fc1_output), rows, hidden, width, 0, 0}, on)) return s;
        if (int s = launch<T, true, PLAIN>(Task{g_fc1, fc1_weight, nullptr, g_x, nullptr, rows, D, 2 * hidden, 0, 0}, on)) return s;
        if (g_fc1_bias)
            if (int s = column_sums<T>(g_fc1, g_fc1_bias, sums, rows, 2 * hidden, on)) return s;
        if (g_fc2_bias)
            if (int s = column_sums<T>(g_out, g_fc2_bias, sums, rows, width, on)) return s;
        return (int)LBI_OK;
    };
    if (int s = dtype == LBI_F16 ? run(_Float16{}) : run(bf16_raw{})) return s;
    if (int s = lbi_weight_gradient(g_fc1, x, g_fc1_weight, gradient, p.gradient, 2 * hidden, D, rows, dtype, stream)) return s;
    return lbi_weight_gradient(g_out, down_input, g_fc2_weight, gradient, p.gradient, width, hidden, rows, dtype, stream);
}
