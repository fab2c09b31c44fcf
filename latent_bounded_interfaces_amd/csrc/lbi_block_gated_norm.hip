// The norms behind and before a block with its gate and residual scale: the C entries (lbi_block_gated_norm_kernel.h has the mathematics).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "lbi_block_gated_norm.h"
#include "lbi_block_rows.h"

namespace lbi {
namespace block_norm {
namespace {

// out[c] = sum over slabs of the shares: sum 0 is g_post_weight, 1 g_weight, 2 + g that of gate g, over its own slabs only.  COLUMNS columns a
// workgroup, PARTS threads a column, whose sums are added in order.
template <int COLUMNS, int PARTS>
__global__ __launch_bounds__(COLUMNS * PARTS) void gated_fold_kernel(Partials partials, float* __restrict__ post, float* __restrict__ pre,
                                                                     float* __restrict__ gate, int64_t first, int64_t slabs, int slabs_per_gate, int D) {
    __shared__ float part[PARTS][COLUMNS];
    const int col = threadIdx.x % COLUMNS, q = threadIdx.x / COLUMNS, c = blockIdx.x * COLUMNS + col;
    const int64_t which = first + blockIdx.y, g = which - 2, count = which < 2 ? slabs : slabs_per_gate;
    const float* from = which == 0 ? partials.post : which == 1 ? partials.pre : partials.gate + g * slabs_per_gate * D;
    float* to = which == 0 ? post : which == 1 ? pre : gate + g * D;
    float sum = 0.0f;
    if (c < D)
#pragma unroll 8
        for (int64_t s = q; s < count; s += PARTS) sum += from[s * D + c];
    part[q][col] = sum;
    __syncthreads();
    for (int half = PARTS / 2; half >= 1; half /= 2) {
        if (q < half) part[q][col] += part[q + half][col];
        __syncthreads();
    }
    if (q == 0 && c < D) to[c] = part[0][col];
}

// As many slabs in all as fill the chip a few times, none across two gates.
Plan plan_of(int64_t rows, int64_t D, int64_t per_gate) {
    const bool summed = per_gate > 0;
    Plan p;
    p.per_gate = summed ? per_gate : std::max<int64_t>(rows, 1);
    p.gates = summed ? rows / per_gate : 1;
    // One slab a CU for short sums over narrow rows and for the widest rows, two otherwise (us, one / two, bf16 with a gate for each of 5 sequences: 5015 rows of
    // 768 20 / 22, 40000 94 / 88, 1000 12 / 17; 5015 of 2048 44 / 33, of 4096 62 / 58, of 8192 117 / 123; four take 22 to 40 % longer, but 40000 x 1024).
    const int64_t cus = device_compute_units(), slabs = D > 4096 || (D <= 1024 && rows <= 16384) ? cus : 2 * cus, least = D <= 512 ? 2048 / D : 1;
    p.slab = (int)std::min<int64_t>(std::max<int64_t>((rows + slabs - 1) / slabs, least), p.per_gate);
    p.slabs_per_gate = (int)((p.per_gate + p.slab - 1) / p.slab);
    return p;
}
size_t partial_bytes(const Plan& p, int64_t rows, int64_t D, bool summed) { return rows ? (size_t)p.slabs() * D * sizeof(float) * (summed ? 3 : 2) : 0; }

int check_gated(const char* who, int64_t rows, int64_t D, int64_t per_gate, int dtype, int stream, int post_weight, int weight) {
    if (rows < 0 || D < 1 || per_gate < 0 || (per_gate && rows % per_gate))
        return fail(LBI_ERR_INVALID, "%s: bad size (rows=%lld D=%lld rows a gate=%lld)", who, (long long)rows, (long long)D, (long long)per_gate);
    if (!dtype_size(dtype) || (stream != dtype && stream != LBI_F32) || (post_weight != dtype && post_weight != LBI_F32) ||
        (weight != dtype && weight != LBI_F32))
        return fail(LBI_ERR_INVALID, "%s: bad dtype (%d; residual stream %d and weights %d, %d are of the same or fp32)", who, dtype, stream, post_weight, weight);
    if (D > MOST_COLUMNS || rows >= MOST_ROWS)
        return fail(LBI_ERR_UNSUPPORTED, "%s: rows of up to %lld columns, fewer than 2^31 of them", who, (long long)MOST_COLUMNS);
    return LBI_OK;
}

}  // namespace
}  // namespace block_norm
}  // namespace lbi

extern "C" int lbi_gated_residual_rmsnorm(const void* branch, const void* residual, const void* gate, const void* post_weight, const void* weight,
                                          void* normed, void* residual_out, int64_t rows, int64_t D, int64_t per_gate, float eps, float residual_scale,
                                          int dtype, int residual_dtype, int post_weight_dtype, int weight_dtype, void* stream) {
    using namespace lbi;
    using namespace lbi::block_norm;
    clear_error();
    if (int bad = check_gated("lbi_gated_residual_rmsnorm", rows, D, per_gate, dtype, residual_dtype, post_weight_dtype, weight_dtype)) return bad;
    if (rows == 0) return LBI_OK;
    if (!branch || !residual || !post_weight || !weight || !normed || !residual_out)
        return fail(LBI_ERR_INVALID, "lbi_gated_residual_rmsnorm: null pointer");
    if (!aligned(branch, dtype) || !aligned(normed, dtype) || !aligned(gate, dtype) || !aligned(residual, residual_dtype) ||
        !aligned(residual_out, residual_dtype) || !aligned(post_weight, post_weight_dtype) || !aligned(weight, weight_dtype))
        return fail(LBI_ERR_INVALID, "lbi_gated_residual_rmsnorm: a tensor is not aligned to its elements");
    const size_t size = dtype_size(dtype), of_stream = dtype_size(residual_dtype);
    const Place y(normed, rows * D, size), s(residual_out, rows * D, of_stream);
    for (const Place& in : {Place(branch, rows * D, size), Place(residual, rows * D, of_stream)})
        if ((y.meets(in) && !y.is(in)) || (s.meets(in) && !s.is(in)) || y.meets(s))
            return fail(LBI_ERR_INVALID, "lbi_gated_residual_rmsnorm: a result overlaps another tensor");
    for (const Place& in : {Place(gate, (per_gate ? rows / per_gate : rows) * D, size), Place(post_weight, D, dtype_size(post_weight_dtype)), Place(weight, D, dtype_size(weight_dtype))})
        if (y.meets(in) || s.meets(in)) return fail(LBI_ERR_INVALID, "lbi_gated_residual_rmsnorm: a result overlaps another tensor");
    const Forward f{branch, residual, gate, post_weight, weight, normed, residual_out, rows, D, per_gate, eps, residual_scale,
                    post_weight_dtype == LBI_F32, weight_dtype == LBI_F32};
    const auto s_ = static_cast<hipStream_t>(stream);
    const bool same = residual_dtype == dtype;
    return dtype == LBI_F32 ? forward_f32(f, s_) : dtype == LBI_F16 ? forward_f16(f, same, s_) : forward_bf16(f, same, s_);
}

extern "C" size_t lbi_gated_residual_rmsnorm_pullback_workspace_bytes(int64_t rows, int64_t D, int64_t per_gate) {
    using namespace lbi::block_norm;
    if (rows < 1 || D < 1 || per_gate < 0 || D > MOST_COLUMNS || rows >= MOST_ROWS || (per_gate && rows % per_gate)) return 0;
    return partial_bytes(plan_of(rows, D, per_gate), rows, D, per_gate > 0);
}

extern "C" int lbi_gated_residual_rmsnorm_pullback(const void* g_normed, const void* branch, const void* residual_out, const void* g_residual_out,
                                                   const void* gate, const void* post_weight, const void* weight, void* g_branch, void* g_residual,
                                                   void* g_gate, float* g_post_weight, float* g_weight, void* workspace, size_t workspace_bytes,
                                                   int64_t rows, int64_t D, int64_t per_gate, float eps, float residual_scale, int dtype,
                                                   int residual_dtype, int post_weight_dtype, int weight_dtype, void* stream) {
    using namespace lbi;
    using namespace lbi::block_norm;
    const char* const who = "lbi_gated_residual_rmsnorm_pullback";
    clear_error();
    if (int bad = check_gated(who, rows, D, per_gate, dtype, residual_dtype, post_weight_dtype, weight_dtype)) return bad;
    const bool summed = gate && per_gate > 0;
    if (!g_post_weight || !g_weight || (gate && !g_gate) ||
        (rows && (!g_normed || !branch || !residual_out || !post_weight || !weight || !g_branch || !g_residual)))
        return fail(LBI_ERR_INVALID, "%s: null pointer", who);
    const Plan plan = plan_of(rows, D, gate ? per_gate : 0);
    const size_t need = partial_bytes(plan, rows, D, summed);
    if (need && (!workspace || workspace_bytes < need)) return fail(LBI_ERR_WORKSPACE, "%s: workspace of %zu bytes needed, %zu given", who, need, workspace_bytes);
    if (!aligned(g_normed, dtype) || !aligned(branch, dtype) || !aligned(gate, dtype) || !aligned(residual_out, residual_dtype) ||
        !aligned(g_residual_out, residual_dtype) || !aligned(post_weight, post_weight_dtype) || !aligned(weight, weight_dtype) || !aligned(g_branch, dtype) ||
        !aligned(g_residual, residual_dtype) || !aligned(g_gate, summed ? LBI_F32 : dtype) || !aligned(g_post_weight, LBI_F32) ||
        !aligned(g_weight, LBI_F32) || !aligned(workspace, LBI_F32))
        return fail(LBI_ERR_INVALID, "%s: a tensor is not aligned to its elements", who);
    const size_t size = dtype_size(dtype), of_stream = dtype_size(residual_dtype);
    const int64_t gates = per_gate ? rows / per_gate : rows;
    const Place results[] = {Place(g_branch, rows * D, size), Place(g_residual, rows * D, of_stream), Place(gate ? g_gate : nullptr, gates * D, summed ? 4 : size),
                             Place(g_post_weight, D, 4), Place(g_weight, D, 4), Place(workspace, (int64_t)need, 1)};
    const Place inputs[] = {Place(g_normed, rows * D, size), Place(branch, rows * D, size), Place(residual_out, rows * D, of_stream),
                            Place(g_residual_out, rows * D, of_stream), Place(gate, gates * D, size), Place(post_weight, D, dtype_size(post_weight_dtype)),
                            Place(weight, D, dtype_size(weight_dtype))};
    for (const Place& out : results) {
        for (const Place& in : inputs)
            if (out.meets(in)) return fail(LBI_ERR_INVALID, "%s: a result overlaps another tensor", who);
        for (const Place& other : results)
            if (&out != &other && out.meets(other)) return fail(LBI_ERR_INVALID, "%s: a result overlaps another tensor", who);
    }
    const auto s = static_cast<hipStream_t>(stream);
    const int64_t slabs = rows ? plan.slabs() : 0;
    float* const shares = static_cast<float*>(workspace);
    const Partials partials{shares, shares + slabs * D, shares + 2 * slabs * D};
    if (rows) {
        const Pullback f{g_normed, branch, residual_out, g_residual_out, gate, post_weight, weight, g_branch, g_residual, summed ? nullptr : g_gate,
                         partials, plan, D, eps, residual_scale, gate && !summed, post_weight_dtype == LBI_F32, weight_dtype == LBI_F32};
        const bool same = residual_dtype == dtype;
        const int status = dtype == LBI_F32 ? pullback_f32(f, s) : dtype == LBI_F16 ? pullback_f16(f, same, s) : pullback_bf16(f, same, s);
        if (status) return status;
    }
    // one launch for all sums, in so many more as there are gates past what a launch numbers
    const int64_t outs = 2 + (summed && rows ? plan.gates : 0);
    // Enough columns to fill the chip in whole lines (us of a pullback of 5015 rows, 16 / 64 columns: 768 wide 29.7 / 29.8, 2048 35 / 33, 8192 179 / 167; of 64 of
    // 1024 10.1 / 10.6).
    const bool wide = D > 1024;
    for (int64_t first = 0; first < outs; first += 65535) {
        const auto fold = wide ? gated_fold_kernel<64, 16> : gated_fold_kernel<16, 64>;
        hipLaunchKernelGGL(fold, dim3((unsigned)((D + (wide ? 63 : 15)) / (wide ? 64 : 16)), (unsigned)std::min<int64_t>(outs - first, 65535)), dim3(1024),
                           0, s, partials, g_post_weight, g_weight, static_cast<float*>(g_gate), first, slabs, plan.slabs_per_gate, (int)D);
        LBI_HIP_CHECK(hipGetLastError());
    }
    return LBI_OK;
}
