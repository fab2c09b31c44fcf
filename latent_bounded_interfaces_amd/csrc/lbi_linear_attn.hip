// Linear attention with a decay for each head: the C entries, and the kernel for single tokens.
//
//   prompts    S_t = l S_{t-1} + k_t v_t^T,   out_t = scale q_t S_t          lbi_linear_attention (lbi_linear_attn_kernel.h)
//   pullback   of the same for P cotangents of out, from q, k and v          lbi_linear_attention_pullback
//   tokens     one step of it for each sequence, the state in place          lbi_linear_attention_step
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <utility>

#include "lbi_linear_attn.h"

namespace lbi {
namespace linear_attn {

int run_bf16(const Call& call, bool exact, hipStream_t stream);
int run_f16(const Call& call, hipStream_t stream);

namespace {

// Chains of a launch: a workgroup of 256 threads each (several of few only), in eights, and a launch has fewer than 2^32 threads.
constexpr int64_t MOST_UNITS = ((int64_t)1 << 24) - 8;

int run(const Call& call, int dtype, bool exact, hipStream_t stream) {
    return dtype == LBI_F16 ? run_f16(call, stream) : run_bf16(call, exact, stream);
}

// Segments that a chain is cut into: as many as give a workgroup to each CU, since one alone on a CU takes a chunk in about 0.6 of the time of two that
// share it, and the states in front of the segments are a pass over b and c and a join on top.  Two segments pay for that from 32 chunks on only.
// us, with 1 / 2 / 3 / 4 / 8 / 16 / 32 segments: 64 chains of 4096 tokens of 128 173 / 153 / 123 / 106 / 118 / 154 / 201, 16 of 8192 of 128 327 / 266 / 183 / 142 /
// 88 / 64 / 72, 12 of 8192 of 64 163 / 133 / 95 / 74 / 47 / 33 / 33; with 1 / 2 / 3 / 4: 80 of 2048 of 128 89 / 81 / 66 / 73, 96 of 4096 of 64 90 / 81 / 79 / 73,
// of 1024 of 128 48 / 51 / 54 / 54; 128 of 4096 of 128 182 / 179 / 179 / 182; 192 of 2048 of 128 118 / 147 / 153 / 154.
void cut(Call& call, int64_t units, int64_t T) {
    const int64_t chunks = (T + CHUNK - 1) / CHUNK, cus = device_compute_units(), each = cus / std::max<int64_t>(units, 1);
    const int64_t wanted = each < 2 || chunks < (each == 2 ? 32 : 4) ? 1 : std::min(each, chunks / 2);
    const int64_t of = std::max<int64_t>((chunks + wanted - 1) / wanted, 1);
    call.segments = std::max((int)((chunks + of - 1) / of), 1);
    call.segment = (int)of * CHUNK;
    // The states' pass takes half a segment a workgroup where that, too, gives each CU one at most, which is with two segments (us, whole / half: 96 chains of 4096 of
    // 128 147 / 132, of 64 79 / 69, 128 of 4096 of 128 171 / 163); more workgroups than CUs lose (80 of 4096 of 128 117 / 121, 16 of 8192 of 128 64 / 72).
    call.halved = of >= 4 && 2 * units * (call.segments - 1) <= cus;
    call.half = (int)((of + 1) / 2) * CHUNK;
}
size_t states_bytes(int64_t units, int64_t T, int64_t Da, int64_t Dc) {
    Call call{};
    cut(call, units, T);
    return (size_t)units * call.slots() * Da * Dc * sizeof(float);
}
void cut(Call& call, float* workspace) {
    cut(call, (int64_t)call.chains * call.B * call.P * call.H, call.T);
    call.segment_states = workspace;
    // A workgroup adds up to fourteen slots by itself: a launch costs what it saves there (us, by itself / by a launch: 11 segments 42 / 42 and
    // 79 / 80, 16 71 / 70 and 38 / 35, 32 91 / 73).
    call.joined = !call.halved && call.slots() > 14;
}

bool any_null(std::initializer_list<const void*> pointers) {
    return std::any_of(pointers.begin(), pointers.end(), [](const void* p) { return !p; });
}
bool off(const void* p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to != 0; }

int check(const char* who, const lbi_linear_attention_call* call, bool pullback) {
    if (!call) return fail(LBI_ERR_INVALID, "%s: null pointer", who);
    const auto& c = *call;
    if (c.B < 0 || c.H < 1 || c.Hkv < 1 || c.T < 0 || c.Dk < 1 || c.Dv < 1 || (pullback && c.P < 0))
        return fail(LBI_ERR_INVALID, "%s: bad size (B=%lld H=%lld Hkv=%lld T=%lld Dk=%lld Dv=%lld)", who, (long long)c.B, (long long)c.H,
                    (long long)c.Hkv, (long long)c.T, (long long)c.Dk, (long long)c.Dv);
    if (c.H % c.Hkv) return fail(LBI_ERR_INVALID, "%s: H=%lld not a multiple of Hkv=%lld", who, (long long)c.H, (long long)c.Hkv);
    if (c.dtype != LBI_F16 && c.dtype != LBI_BF16) return fail(dtype_size(c.dtype) ? LBI_ERR_UNSUPPORTED : LBI_ERR_INVALID, "%s: bad dtype %d", who, c.dtype);
    if (c.Dk > MOST_DIM || c.Dv > MOST_DIM) return fail(LBI_ERR_UNSUPPORTED, "%s: head dims of up to %d", who, MOST_DIM);
    const int64_t basis = pullback ? std::max<int64_t>(c.P, 1) : 1, chains = !pullback ? 1 : c.Dk == c.Dv ? 3 : 2;
    if (c.T >= (int64_t)1 << 30 || c.B >= (int64_t)1 << 20 || c.H >= (int64_t)1 << 16 || basis >= (int64_t)1 << 20 ||
        chains * c.B * c.H * basis > MOST_UNITS)
        return fail(LBI_ERR_UNSUPPORTED, "%s: too many sequences, heads and directions, or too many tokens", who);
    if (!std::isfinite(c.scale) || !std::isfinite(1.0f / c.scale))  // the pullback's chains begin with the state's cotangent over the scale
        return fail(LBI_ERR_INVALID, "%s: scale must be finite and not zero, and so must its inverse", who);
    return LBI_OK;
}

int check_workspace(const char* who, size_t need, const void* workspace, size_t bytes) {
    if (need && (!workspace || bytes < need)) return fail(LBI_ERR_WORKSPACE, "%s: workspace of %zu bytes needed, %zu given", who, need, bytes);
    if (need && off(workspace, 4)) return fail(LBI_ERR_INVALID, "%s: a tensor is not aligned to its elements", who);
    return LBI_OK;
}

View shared(const void* p, const int64_t* stride, int64_t group) { return View{p, stride[0], 0, stride[1], stride[2], (int)group}; }
// contiguous [B, P, H, T, width]
View dense(const void* p, const lbi_linear_attention_call& c, int64_t width) {
    return View{p, c.P * c.H * c.T * width, c.H * c.T * width, c.T * width, width, 1};
}
Call base(const lbi_linear_attention_call& c, int64_t basis) {
    Call call{};
    call.log_decay = c.log_decay;
    call.lengths = c.lengths;
    call.lengths_wide = c.lengths_wide != 0;
    call.B = (int)c.B, call.P = (int)basis, call.H = (int)c.H, call.T = (int)c.T;
    return call;
}

// One token of each head: a workgroup takes COLS columns of a head's state, VEC neighbouring ones a thread, and as many rows side by side as it
// has threads left.  Bound by memory: the state is read and written once; all of a thread's share is asked for before any of it is used.
// 1600 heads of 128 x 128 (210 MB in and out): 32.5 us, 6.4 TB/s, part of it from the last-level cache.  One sequence of 12 heads: 3.3 us, latency.
template <typename T, int COLS, int VEC, int ROUNDS>
__global__ __launch_bounds__(256) void step_kernel(const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v,
                                                   const float* __restrict__ log_decay, float* state, const unsigned char* __restrict__ active,
                                                   T* __restrict__ out, int H, int group, int Dk, int Dv, float scale) {
    constexpr int LANES = COLS / VEC, SIDE = 256 / LANES;
    typedef float vec __attribute__((ext_vector_type(VEC), aligned(4 * VEC)));
    __shared__ float sums[SIDE][COLS];
    const int bh = blockIdx.x, h = bh % H, b = bh / H, col = (int)blockIdx.y * COLS + threadIdx.x % LANES * VEC, row0 = threadIdx.x / LANES;
    const int64_t kv = (int64_t)b * (H / group) + h / group;
    float* s = state + (int64_t)bh * Dk * Dv;
    const bool on = !active || active[b];
    float part[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) part[e] = 0.0f;
    if (on && col < Dv) {
        vec x[ROUNDS];
        float kk[ROUNDS], qq[ROUNDS], vv[VEC];
#pragma unroll
        for (int i = 0; i < ROUNDS; ++i) {
            const int row = row0 + i * SIDE, from = row < Dk ? row : 0;
            x[i] = *reinterpret_cast<const vec*>(s + from * Dv + col);
            kk[i] = to_f32(k[kv * Dk + from]);
            qq[i] = to_f32(q[(int64_t)bh * Dk + from]);
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e) vv[e] = to_f32(v[kv * Dv + col + e]);
        const Fade fade(log_decay[h]);
#pragma unroll
        for (int i = 0; i < ROUNDS; ++i) {
            const int row = row0 + i * SIDE;
            if (row >= Dk) continue;
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                x[i][e] = fmaf(kk[i], vv[e], fade.of(x[i][e]));
                part[e] = fmaf(qq[i], x[i][e], part[e]);
            }
            *reinterpret_cast<vec*>(s + row * Dv + col) = x[i];
        }
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) sums[row0][threadIdx.x % LANES * VEC + e] = part[e];
    __syncthreads();
    for (int c = threadIdx.x; c < COLS; c += 256) {
        const int to = (int)blockIdx.y * COLS + c;
        if (to >= Dv) continue;
        float sum = sums[0][c];
#pragma unroll
        for (int r = 1; r < SIDE; ++r) sum += sums[r][c];
        sum *= scale;
        T* o = out + (int64_t)bh * Dv + to;
        if constexpr (std::is_same_v<T, bf16_raw>) o->bits = f32_to_bf16_bits(sum);
        else *o = (T)sum;
    }
}

template <typename T, int COLS, int VEC>
int launch_step(const void* q, const void* k, const void* v, const float* log_decay, float* state, const unsigned char* active, void* out, int64_t B,
                int64_t H, int64_t Hkv, int64_t Dk, int64_t Dv, float scale, hipStream_t stream) {
    constexpr int SIDE = 256 / (COLS / VEC);
    const auto kernel = Dk <= 64 ? step_kernel<T, COLS, VEC, (64 + SIDE - 1) / SIDE> : step_kernel<T, COLS, VEC, (128 + SIDE - 1) / SIDE>;
    hipLaunchKernelGGL(kernel, dim3((unsigned)(B * H), (unsigned)((Dv + COLS - 1) / COLS)), dim3(256), 0, stream, static_cast<const T*>(q),
                       static_cast<const T*>(k), static_cast<const T*>(v), log_decay, state, active, static_cast<T*>(out), (int)H, (int)(H / Hkv), (int)Dk,
                       (int)Dv, scale);
    LBI_HIP_CHECK(hipGetLastError());
    return LBI_OK;
}

}  // namespace
}  // namespace linear_attn
}  // namespace lbi

extern "C" size_t lbi_linear_attention_workspace_bytes(const lbi_linear_attention_call* c) {
    using namespace lbi::linear_attn;
    if (check("lbi_linear_attention_workspace_bytes", c, false)) return 0;
    if (!c->B || !c->T) return 0;
    return states_bytes(c->B * c->H, c->T, c->Dk, c->Dv);
}

extern "C" int lbi_linear_attention(const lbi_linear_attention_call* c, void* workspace, size_t workspace_bytes, void* stream) {
    using namespace lbi;
    using namespace lbi::linear_attn;
    clear_error();
    if (int bad = check("lbi_linear_attention", c, false)) return bad;
    if (!c->B) return LBI_OK;
    if (any_null({c->log_decay}) || (c->T && any_null({c->q, c->k, c->v, c->out}))) return fail(LBI_ERR_INVALID, "lbi_linear_attention: null pointer");
    if (off(c->q, 2) || off(c->k, 2) || off(c->v, 2) || off(c->out, 2) || off(c->state, 4) || off(c->state_out, 4) || off(c->log_decay, 4) ||
        off(c->lengths, c->lengths_wide ? 8 : 4))
        return fail(LBI_ERR_INVALID, "lbi_linear_attention: a tensor is not aligned to its elements");
    if (int bad = check_workspace("lbi_linear_attention", lbi_linear_attention_workspace_bytes(c), workspace, workspace_bytes)) return bad;
    clear_error();
    Call call = base(*c, 1);
    call.chains = 1;
    Chain& ch = call.chain[0];
    ch.a = shared(c->q, c->q_stride, 1);
    ch.b = shared(c->k, c->k_stride, c->H / c->Hkv);
    ch.c = shared(c->v, c->v_stride, c->H / c->Hkv);
    ch.out = shared(c->out, c->out_stride, 1);
    const auto states = [&](const float* p) { return States{const_cast<float*>(p), c->H * c->Dk * c->Dv, 0, c->Dk * c->Dv, c->Dv, 1}; };
    ch.first = states(c->state), ch.last = states(c->state_out);
    ch.first_scale = ch.last_scale = 1.0f;
    ch.scale = c->scale;
    ch.Da = (int)c->Dk, ch.Dc = (int)c->Dv, ch.reverse = 0, ch.shift = 0;
    cut(call, static_cast<float*>(workspace));
    return run(call, c->dtype, true, static_cast<hipStream_t>(stream));
}

extern "C" size_t lbi_linear_attention_pullback_workspace_bytes(const lbi_linear_attention_call* c) {
    using namespace lbi::linear_attn;
    if (check("lbi_linear_attention_pullback_workspace_bytes", c, true)) return 0;
    if (!c->B || !c->T || !c->P) return 0;
    const int64_t units = c->B * c->P * c->H;
    if (c->Dk == c->Dv) return states_bytes(3 * units, c->T, c->Dk, c->Dv);
    return std::max(states_bytes(2 * units, c->T, c->Dv, c->Dk), states_bytes(units, c->T, c->Dk, c->Dv));
}

extern "C" int lbi_linear_attention_pullback(const lbi_linear_attention_call* c, void* workspace, size_t workspace_bytes, void* stream) {
    using namespace lbi;
    using namespace lbi::linear_attn;
    clear_error();
    if (int bad = check("lbi_linear_attention_pullback", c, true)) return bad;
    if (!c->B || !c->P) return LBI_OK;
    if (any_null({c->log_decay}) || (c->T && any_null({c->q, c->k, c->v, c->g_out, c->dq, c->dk, c->dv})))
        return fail(LBI_ERR_INVALID, "lbi_linear_attention_pullback: null pointer");
    if (off(c->q, 2) || off(c->k, 2) || off(c->v, 2) || off(c->g_out, 2) || off(c->dq, 2) || off(c->dk, 2) || off(c->dv, 2) || off(c->state, 4) ||
        off(c->g_state, 4) || off(c->d_state, 4) || off(c->log_decay, 4) || off(c->lengths, c->lengths_wide ? 8 : 4))
        return fail(LBI_ERR_INVALID, "lbi_linear_attention_pullback: a tensor is not aligned to its elements");
    if (int bad = check_workspace("lbi_linear_attention_pullback", lbi_linear_attention_pullback_workspace_bytes(c), workspace, workspace_bytes)) return bad;
    clear_error();
    const int64_t group = c->H / c->Hkv, of_state = c->Dk * c->Dv;
    const View q = shared(c->q, c->q_stride, 1), k = shared(c->k, c->k_stride, group), v = shared(c->v, c->v_stride, group);
    const View gv = View{c->g_out, c->g_out_stride[0], c->g_out_stride[1], c->g_out_stride[2], c->g_out_stride[3], 1};
    // of the forward's first state, one for all directions, and of the cotangents of the last and the first
    const States none{}, first{const_cast<float*>(c->state), c->H * of_state, 0, of_state, 1, c->Dv};
    const auto cotangent = [&](const float* p, bool turned) {
        return States{const_cast<float*>(p), c->P * c->H * of_state, c->H * of_state, of_state, turned ? 1 : c->Dv, turned ? c->Dv : 1};
    };
    Call call = base(*c, c->P);
    const int dk = (int)c->Dk, dv = (int)c->Dv;
    const float s = c->scale;
    const Chain of_q{gv, v, k, dense(c->dq, *c, dk), first, none, 1.0f, 1.0f, s, dv, dk, 0, 0};
    const Chain of_k{v, gv, q, dense(c->dk, *c, dk), cotangent(c->g_state, true), none, 1.0f / s, s, s, dv, dk, 1, 1};
    const Chain of_v{k, q, gv, dense(c->dv, *c, dv), cotangent(c->g_state, false), cotangent(c->d_state, false), 1.0f / s, s, s, dk, dv, 1, 1};
    const bool exact = c->d_state != nullptr;
    const auto go = [&](std::initializer_list<Chain> chains) {
        call.chains = 0;
        for (const Chain& ch : chains) call.chain[call.chains++] = ch;
        cut(call, static_cast<float*>(workspace));
        return run(call, c->dtype, exact, static_cast<hipStream_t>(stream));
    };
    if (dk == dv) return go({of_q, of_k, of_v});
    if (int bad = go({of_q, of_k})) return bad;
    return go({of_v});
}

extern "C" int lbi_linear_attention_step(const void* q, const void* k, const void* v, const float* log_decay, float* state, const unsigned char* active,
                                         void* out, int64_t B, int64_t H, int64_t Hkv, int64_t Dk, int64_t Dv, float scale, int dtype, void* stream) {
    using namespace lbi;
    using namespace lbi::linear_attn;
    clear_error();
    if (B < 0 || H < 1 || Hkv < 1 || Dk < 1 || Dv < 1)
        return fail(LBI_ERR_INVALID, "lbi_linear_attention_step: bad size (B=%lld H=%lld Hkv=%lld Dk=%lld Dv=%lld)", (long long)B, (long long)H,
                    (long long)Hkv, (long long)Dk, (long long)Dv);
    if (H % Hkv) return fail(LBI_ERR_INVALID, "lbi_linear_attention_step: H=%lld not a multiple of Hkv=%lld", (long long)H, (long long)Hkv);
    const size_t size = dtype_size(dtype);
    if (!size) return fail(LBI_ERR_INVALID, "lbi_linear_attention_step: bad dtype %d", dtype);
    if (Dk > MOST_DIM || Dv > MOST_DIM) return fail(LBI_ERR_UNSUPPORTED, "lbi_linear_attention_step: head dims of up to %d", MOST_DIM);
    if (B >= (int64_t)1 << 24 || H >= (int64_t)1 << 16 || B * H >= (int64_t)1 << 24)
        return fail(LBI_ERR_UNSUPPORTED, "lbi_linear_attention_step: too many sequences and heads");
    if (!B) return LBI_OK;
    if (any_null({q, k, v, log_decay, state, out})) return fail(LBI_ERR_INVALID, "lbi_linear_attention_step: null pointer");
    if (off(q, size) || off(k, size) || off(v, size) || off(out, size) || off(state, 4) || off(log_decay, 4))
        return fail(LBI_ERR_INVALID, "lbi_linear_attention_step: a tensor is not aligned to its elements");
    const int64_t heads = B * H, kv_heads = B * Hkv;
    const std::pair<const void*, uint64_t> places[] = {{state, heads * Dk * Dv * 4}, {out, heads * Dv * size}, {q, heads * Dk * size}, {k, kv_heads * Dk * size},
                                                       {v, kv_heads * Dv * size},    {log_decay, H * 4},        {active, B}};
    for (int w = 0; w < 2; ++w)  // what is written: state and out, which other workgroups of a head read beside
        for (int o = w + 1; o < 7; ++o) {
            const uintptr_t here = reinterpret_cast<uintptr_t>(places[w].first), there = reinterpret_cast<uintptr_t>(places[o].first);
            if (there && here < there + places[o].second && there < here + places[w].second)
                return fail(LBI_ERR_INVALID, "lbi_linear_attention_step: a result overlaps another tensor");
        }
    // Wide heads that give at most one workgroup to a CU are cut into blocks of 16 columns (us, 16 / 128 columns: 16 heads of 128 x 128 3.6 / 4.4, 256
    // 7.0 / 7.9, 320 8.9 / 8.4, 1600 44 / 33); heads of 64 x 64 gain nothing (12 of them 3.4 / 3.2, 64 3.3 / 3.3).
    const bool in_fours = Dv % 4 == 0 && !off(state, 16), few = Dv > 64 && B * H <= device_compute_units();
    const auto go = [&](auto t) {
        using T = decltype(t);
        const auto with = [&](auto launch) { return launch(q, k, v, log_decay, state, active, out, B, H, Hkv, Dk, Dv, scale, static_cast<hipStream_t>(stream)); };
        if (!in_fours) return with(launch_step<T, 64, 1>);
        if (few) return with(launch_step<T, 16, 4>);
        return Dv > 64 ? with(launch_step<T, 128, 4>) : with(launch_step<T, 64, 4>);
    };
    if (dtype == LBI_F32) return go(float{});
    return dtype == LBI_F16 ? go(_Float16{}) : go(bf16_raw{});
}
