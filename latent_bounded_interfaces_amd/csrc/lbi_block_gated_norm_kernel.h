// The norms behind a block's branch and in front of the next one, with the branch's gate and the residual's scale, and their pullback.
//
//   forward    u = b i1 w1, i1 = rsqrt(mean(b^2) + eps);   s = alpha r + gate u;   y = s i2 w2, i2 = rsqrt(mean(s^2) + eps)
//   pullback   n = s i2, p = g_y w2:       g_s = i2 (p - n mean(n p)) + g_s',   g_r = alpha g_s,   g_w2 = sum over rows of g_y n
//              m = b i1, q = gate g_s w1:  g_b = i1 (q - m mean(m q)),   g_gate = g_s m w1,   g_w1 = sum over rows of gate g_s m
//
// Everything between load and store is fp32: y is the norm of the sum before its rounding.  The gate is one row for all rows, one for each
// `per_gate` of them (then its gradient is a sum, too), or one for each.
//
// Bound by memory: one pass, a row in the registers of the lanes that share it (lbi_block_rows.h).  Forward, 8192 x 768 in bf16 with an fp32 stream: 16.5 us,
// 4.6 TB/s; pullback, 5015 x 2048 in bf16: 29 us, 4.3 TB/s, and 5 us for the sums over the slabs.
#pragma once

#include "lbi_block_gated_norm.h"
#include "lbi_block_rows.h"

namespace lbi {
namespace block_norm {
namespace {

template <typename T, typename R, bool GATED, bool TAIL, int NT, int PIECES>
__global__ __launch_bounds__(NT * SIDE<NT>) void gated_norm_kernel(const T* branch, const R* residual, const T* __restrict__ gate,
                                                                   const void* __restrict__ post_weight, const void* __restrict__ weight, T* normed,
                                                                   R* stream_out, unsigned first, unsigned rows, unsigned per_gate, int D, float eps, float alpha,
                                                                   int post_wide, int wide) {
    __shared__ float spare[2][NT <= 64 ? 1 : NT / 64];
    const int threads = NT <= 64 ? NT : (int)blockDim.x, t = threadIdx.x % threads;
    const unsigned row = first + blockIdx.x * SIDE<NT> + threadIdx.x / threads;
    if (row >= rows) return;  // all lanes of a row, and with barriers below the row is the workgroup's only one
    const int64_t from = (int64_t)row * D, of_gate = GATED ? (int64_t)(row / per_gate) * D : 0;
    Raw<T> b[PIECES], k[PIECES];
    Raw<R> r[PIECES];
    Eight w1[PIECES], w2[PIECES], s[PIECES];
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
        const int c = (p * threads + t) * PIECE;
        if (c >= D) continue;
        b[p] = load8<TAIL>(branch + from + c, D - c);
        r[p] = load8<TAIL>(residual + from + c, D - c);
        if constexpr (GATED) k[p] = load8<TAIL>(gate + of_gate + c, D - c);
    }
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
        const int c = (p * threads + t) * PIECE;
        if (c >= D) continue;
        w1[p] = load_weight<TAIL, T>(post_weight, c, D - c, post_wide != 0);
        w2[p] = load_weight<TAIL, T>(weight, c, D - c, wide != 0);
    }
    float sum = 0.0f;
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
        if ((p * threads + t) * PIECE >= D) continue;
        s[p] = b[p].wide();
#pragma unroll
        for (int e = 0; e < PIECE; ++e) sum = fmaf(s[p].v[e], s[p].v[e], sum);
    }
    const float inv1 = rsqrtf(over_row<Add, NT>(sum, spare[0]) / (float)D + eps);
    sum = 0.0f;
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
        const int c = (p * threads + t) * PIECE;
        if (c >= D) continue;
        const Eight more = r[p].wide();
        Eight open;
        if constexpr (GATED) open = k[p].wide();
#pragma unroll
        for (int e = 0; e < PIECE; ++e) {
            float u = s[p].v[e] * inv1 * w1[p].v[e];
            if constexpr (GATED) u *= open.v[e];
            s[p].v[e] = fmaf(alpha, more.v[e], u);
            sum = fmaf(s[p].v[e], s[p].v[e], sum);
        }
        store8<TAIL>(stream_out + from + c, s[p], D - c);
    }
    const float inv2 = rsqrtf(over_row<Add, NT>(sum, spare[1]) / (float)D + eps);
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
        const int c = (p * threads + t) * PIECE;
        if (c >= D) continue;
#pragma unroll
        for (int e = 0; e < PIECE; ++e) s[p].v[e] = s[p].v[e] * inv2 * w2[p].v[e];
        store8<TAIL>(normed + from + c, s[p], D - c);
    }
}

// COUNT sums over the threads of a row, the same in all of them.
template <int COUNT, int NT> __device__ __forceinline__ void sums(float (&x)[COUNT], float (*spare)[COUNT]) {
#pragma unroll
    for (int off = (NT < 64 ? NT : 64) / 2; off >= 1; off >>= 1)
#pragma unroll
        for (int i = 0; i < COUNT; ++i) x[i] += __shfl_xor(x[i], off, 64);
    if constexpr (NT > 64) {
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int i = 0; i < COUNT; ++i) spare[threadIdx.x >> 6][i] = x[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < COUNT; ++i) x[i] = spare[0][i];
        for (int w = 1; w < (int)blockDim.x / 64; ++w)
#pragma unroll
            for (int i = 0; i < COUNT; ++i) x[i] += spare[w][i];
    }
}

enum Gate { SHARED, EACH };  // SHARED: by the rows of a slab; none at all is one of ones whose gradient nobody wants

// A workgroup takes the rows of one slab, which lies within the rows of one gate, SIDE of them at a time, and keeps the sums over them in registers.
template <typename T, typename R, int GATE, bool MORE, bool TAIL, int NT, int PIECES>
__global__ __launch_bounds__(NT * SIDE<NT>) void gated_norm_pullback_kernel(const T* g_normed, const T* branch, const R* stream, const R* g_stream,
                                                                            const T* __restrict__ gate, const void* __restrict__ post_weight,
                                                                            const void* __restrict__ weight, T* g_branch, R* g_residual, T* g_gate,
                                                                            Partials partials, unsigned first_slab, int64_t per_gate, int slabs_per_gate, int slab, int D,
                                                                            float eps, float alpha, int post_wide, int wide) {
    extern __shared__ __align__(16) float lds[];  // SIDE > 1: [SIDE][D]
    __shared__ float spare[2][NT <= 64 ? 1 : NT / 64][3], spare2[2][NT <= 64 ? 1 : NT / 64][1];
    const int threads = NT <= 64 ? NT : (int)blockDim.x, t = threadIdx.x % threads, side = threadIdx.x / threads;
    const unsigned own = first_slab + blockIdx.x;
    const int64_t group = own / slabs_per_gate, ends = (group + 1) * per_gate;
    const int64_t first = group * per_gate + (int64_t)(own % slabs_per_gate) * slab, last = first + slab < ends ? first + slab : ends;
    struct Row {
        Raw<R> x[PIECES], more[PIECES];
        Raw<T> g[PIECES], b[PIECES], k[PIECES];
    };
    auto bring = [&](int64_t row) __attribute__((always_inline)) {
        Row r;
        const int64_t from = (row < last ? row : last - 1) * D;
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            const int at = (p * threads + t) * PIECE, c = at < D ? at : 0;
            r.x[p] = load8<TAIL>(stream + from + c, D - c);
            r.g[p] = load8<TAIL>(g_normed + from + c, D - c);
            r.b[p] = load8<TAIL>(branch + from + c, D - c);
            if constexpr (MORE) r.more[p] = load8<TAIL>(g_stream + from + c, D - c);
            if constexpr (GATE == EACH) r.k[p] = load8<TAIL>(gate + from + c, D - c);
        }
        return r;
    };
    Eight of_post[PIECES], of_pre[PIECES], of_gate[PIECES];
#pragma unroll
    for (int p = 0; p < PIECES; ++p)
#pragma unroll
        for (int e = 0; e < PIECE; ++e) of_post[p].v[e] = of_pre[p].v[e] = of_gate[p].v[e] = 0.0f;
    constexpr bool AHEAD = NT * PIECES <= 1024;  // the widest rows leave no registers for it, nor for the weights
    Row next;
    if constexpr (AHEAD) next = bring(first + side);
    struct Fixed { Eight w1, w2, open; };
    auto fixed_of = [&](int p) __attribute__((always_inline)) {
        Fixed f;
        const int at = (p * threads + t) * PIECE, c = at < D ? at : 0;
        f.w1 = load_weight<TAIL, T>(post_weight, c, D - c, post_wide != 0);
        f.w2 = load_weight<TAIL, T>(weight, c, D - c, wide != 0);
        if constexpr (GATE == SHARED) {
#pragma unroll
            for (int e = 0; e < PIECE; ++e) f.open.v[e] = 1.0f;
            if (gate) f.open = load8<TAIL>(gate + group * D + c, D - c).wide();
        }
        return f;
    };
    Fixed held[PIECES];
    if constexpr (AHEAD)
#pragma unroll
        for (int p = 0; p < PIECES; ++p) held[p] = fixed_of(p);
    int turn = 0;
    for (int64_t row = first + side; row < last; row += SIDE<NT>, turn ^= 1) {
        const Row now = AHEAD ? next : bring(row);
        if constexpr (AHEAD) next = bring(row + SIDE<NT>);
        float three[3] = {0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            if ((p * threads + t) * PIECE >= D) continue;
            const Fixed f = AHEAD ? held[p] : fixed_of(p);
            const Eight x = now.x[p].wide(), g = now.g[p].wide(), b = now.b[p].wide();
#pragma unroll
            for (int e = 0; e < PIECE; ++e) {
                three[0] = fmaf(x.v[e], x.v[e], three[0]);
                three[1] = fmaf(x.v[e], g.v[e] * f.w2.v[e], three[1]);
                three[2] = fmaf(b.v[e], b.v[e], three[2]);
            }
        }
        sums<3, NT>(three, spare[turn]);
        const float inv = rsqrtf(three[0] / (float)D + eps), mean = three[1] * inv / (float)D, inv1 = rsqrtf(three[2] / (float)D + eps);
        Eight g_s[PIECES];
        float one[1] = {0.0f};
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            const int c = (p * threads + t) * PIECE;
            if (c >= D) continue;
            const Fixed f = AHEAD ? held[p] : fixed_of(p);
            const Eight x = now.x[p].wide(), g = now.g[p].wide(), b = now.b[p].wide();
            Eight more, open, out;
            if constexpr (MORE) more = now.more[p].wide();
            if constexpr (GATE == EACH) open = now.k[p].wide();
            if constexpr (GATE == SHARED) open = f.open;
#pragma unroll
            for (int e = 0; e < PIECE; ++e) {
                const float unit = x.v[e] * inv;
                of_pre[p].v[e] = fmaf(g.v[e], unit, of_pre[p].v[e]);
                float total = inv * (g.v[e] * f.w2.v[e] - unit * mean);
                if constexpr (MORE) total += more.v[e];
                out.v[e] = alpha * total;
                g_s[p].v[e] = total * open.v[e];
                const float m = b.v[e] * inv1;
                of_post[p].v[e] = fmaf(g_s[p].v[e], m, of_post[p].v[e]);
                if constexpr (GATE == SHARED) of_gate[p].v[e] = fmaf(total * f.w1.v[e], m, of_gate[p].v[e]);
                if constexpr (GATE == EACH) more.v[e] = total * f.w1.v[e] * m;
                g_s[p].v[e] *= f.w1.v[e];
                one[0] = fmaf(m, g_s[p].v[e], one[0]);
            }
            store8<TAIL>(g_residual + row * D + c, out, D - c);
            if constexpr (GATE == EACH) store8<TAIL>(g_gate + row * D + c, more, D - c);
        }
        sums<1, NT>(one, spare2[turn]);
        const float mean1 = one[0] / (float)D;
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            const int c = (p * threads + t) * PIECE;
            if (c >= D) continue;
            const Eight b = now.b[p].wide();
            Eight out;
#pragma unroll
            for (int e = 0; e < PIECE; ++e) out.v[e] = inv1 * (g_s[p].v[e] - b.v[e] * inv1 * mean1);
            store8<TAIL>(g_branch + row * D + c, out, D - c);
        }
    }
    auto leave = [&](Eight (&total)[PIECES], float* to) __attribute__((always_inline)) {
        if constexpr (SIDE<NT> > 1) {
            __syncthreads();
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
                to[(size_t)own * D + c] = sum;
            }
        } else {
#pragma unroll
            for (int p = 0; p < PIECES; ++p) {
                const int c = (p * threads + t) * PIECE;
                if (c < D) store8<TAIL>(to + (size_t)own * D + c, total[p], D - c);
            }
        }
    };
    leave(of_post, partials.post);
    leave(of_pre, partials.pre);
    if constexpr (GATE == SHARED)
        if (gate) leave(of_gate, partials.gate);
}

// Threads and pieces that hold a row of D columns; the pullback, whose rows are six tensors and three sums, in as few waves as have the registers for the next
// row too (us, 5015 rows of bf16: of 2048 256 threads of one piece 33 and of two 37, 1024 of one 44; of 4096 256 of two 58, 512 of one 68; of 8192 512 of two 122,
// 1024 of one 167; of 1000 rows of 768 64 of two 12, 256 of one 14).  Past 8192 columns 1024 threads leave 128 registers each, and 33 to 112 of what a row takes are kept
// in memory: 5015 x 16384 of bf16 469 us, 1000 of fp32 181, 2.3 times their bytes (5015 x 8192 of bf16 97 us, 0.96).
template <bool PULLBACK, typename F> int by_row(int64_t D, F&& launch) {
    if (D <= 128) return launch(Form<16, 1>{});
    if (D <= 512) return launch(Form<64, 1>{});
    if (D <= 1024) return launch(Form<64, 2>{});
    if constexpr (PULLBACK) {
        if (D <= 2048) return launch(Form<256, 1>{});
        if (D <= 4096) return launch(Form<256, 2>{});
    }
    if (D <= 8192) return launch(Form<512, 2>{});
    return launch(Form<1024, 2>{});
}

template <typename T, typename R> int forward(const Forward& f, hipStream_t stream) {
    return by_row<false>(f.D, [&](auto form) {
        constexpr int NT = decltype(form)::NT, PIECES = decltype(form)::PIECES, COUNT = SIDE<NT>;
        const auto kernel = f.D % PIECE ? (f.gate ? gated_norm_kernel<T, R, true, true, NT, PIECES> : gated_norm_kernel<T, R, false, true, NT, PIECES>)
                                        : (f.gate ? gated_norm_kernel<T, R, true, false, NT, PIECES> : gated_norm_kernel<T, R, false, false, NT, PIECES>);
        const int threads = threads_of<NT, PIECES>(f.D) * COUNT;
        const int64_t most = (MOST_THREADS / threads) * COUNT;  // rows of a launch
        for (int64_t first = 0; first < f.rows; first += most) {
            hipLaunchKernelGGL(kernel, dim3((unsigned)((std::min(f.rows - first, most) + COUNT - 1) / COUNT)), dim3((unsigned)threads), 0, stream,
                               static_cast<const T*>(f.branch), static_cast<const R*>(f.residual), static_cast<const T*>(f.gate), f.post_weight, f.weight,
                               static_cast<T*>(f.normed), static_cast<R*>(f.residual_out), (unsigned)first, (unsigned)f.rows,
                               (unsigned)std::max<int64_t>(f.per_gate, 1), (int)f.D, f.eps, f.residual_scale, f.post_wide, f.wide);
            LBI_HIP_CHECK(hipGetLastError());
        }
        return (int)LBI_OK;
    });
}

template <typename T, typename R> int pullback(const Pullback& f, hipStream_t stream) {
    return by_row<true>(f.D, [&](auto form) {
        constexpr int NT = decltype(form)::NT, PIECES = decltype(form)::PIECES, COUNT = SIDE<NT>;
        const auto launch = [&](auto kernel) {
            const size_t bytes = COUNT > 1 ? COUNT * (size_t)f.D * sizeof(float) : 0;  // 16 KiB at most
            const int threads = threads_of<NT, PIECES>(f.D) * COUNT;
            const int64_t slabs = f.plan.slabs(), most = MOST_THREADS / threads;  // slabs of a launch
            for (int64_t first = 0; first < slabs; first += most) {
                hipLaunchKernelGGL(kernel, dim3((unsigned)std::min(slabs - first, most)), dim3((unsigned)threads), bytes, stream,
                                   static_cast<const T*>(f.g_normed), static_cast<const T*>(f.branch), static_cast<const R*>(f.residual_out),
                                   static_cast<const R*>(f.g_residual_out), static_cast<const T*>(f.gate), f.post_weight, f.weight,
                                   static_cast<T*>(f.g_branch), static_cast<R*>(f.g_residual), static_cast<T*>(f.g_gate), f.partials, (unsigned)first,
                                   f.plan.per_gate, f.plan.slabs_per_gate, f.plan.slab, (int)f.D, f.eps, f.residual_scale, f.post_wide, f.wide);
                LBI_HIP_CHECK(hipGetLastError());
            }
            return (int)LBI_OK;
        };
        const auto by_gate = [&](auto more, auto tail) {
            constexpr bool MORE = decltype(more)::value, TAIL = decltype(tail)::value;
            return f.each ? launch(gated_norm_pullback_kernel<T, R, EACH, MORE, TAIL, NT, PIECES>)
                          : launch(gated_norm_pullback_kernel<T, R, SHARED, MORE, TAIL, NT, PIECES>);
        };
        const auto by_tail = [&](auto more) { return f.D % PIECE ? by_gate(more, std::true_type{}) : by_gate(more, std::false_type{}); };
        return f.g_residual_out ? by_tail(std::true_type{}) : by_tail(std::false_type{});
    });
}

}  // namespace
}  // namespace block_norm
}  // namespace lbi
