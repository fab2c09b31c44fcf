// Launches of lbi_linear_attn_kernel.h for one type: which tiles and copies a call takes.
#pragma once

#include "lbi_linear_attn_kernel.h"

namespace lbi {
namespace linear_attn {

template <typename T, int DA, int DC, bool VEC, bool OUT, int PLANES, bool TWICE>
int launch_chunks(const Call& call, int64_t workgroups, hipStream_t stream) {
    constexpr auto kernel = chunk_kernel<T, DA, DC, VEC, OUT, PLANES, TWICE>;
    constexpr size_t bytes = lds_bytes<DA, DC, OUT>();
    if (int rc = ensure_dynamic_lds<kernel>(bytes)) return rc;
    hipLaunchKernelGGL(kernel, dim3((unsigned)((workgroups + 7) / 8 * 8)), dim3(256), bytes, stream, call);
    LBI_HIP_CHECK(hipGetLastError());
    return LBI_OK;
}

template <typename T, int DA, int DC, bool VEC, int PLANES, bool TWICE>
int launch(const Call& call, hipStream_t stream) {
    const int64_t units = (int64_t)call.chains * call.B * call.P * call.H;
    if constexpr (!TWICE) {  // (calls of one chunk are not cut)
        if (call.segments > 1) {
            if (int rc = launch_chunks<T, DA, DC, VEC, false, PLANES, false>(call, units * call.slots(), stream)) return rc;
            if (call.joined) {
                const int elements = call.chain[0].Da * call.chain[0].Dc;
                hipLaunchKernelGGL(join_kernel<T>, dim3((unsigned)((elements + 255) / 256), (unsigned)units), dim3(256), 0, stream, call);
                LBI_HIP_CHECK(hipGetLastError());
            }
        }
    }
    return launch_chunks<T, DA, DC, VEC, true, PLANES, TWICE>(call, units * call.segments, stream);
}

template <typename T, bool VEC, int PLANES, bool TWICE> int by_dims(const Call& call, hipStream_t stream) {
    const bool wide_a = call.chain[0].Da > 64, wide_c = call.chain[0].Dc > 64;
    if (wide_a) return wide_c ? launch<T, 128, 128, VEC, PLANES, TWICE>(call, stream) : launch<T, 128, 64, VEC, PLANES, TWICE>(call, stream);
    return wide_c ? launch<T, 64, 128, VEC, PLANES, TWICE>(call, stream) : launch<T, 64, 64, VEC, PLANES, TWICE>(call, stream);
}

// Calls of up to so many tokens, one chunk, take the scores and the copy of the state in two planes, and so round their results once: a row then rests on few
// scores, and all of its elements share the rounding of each.  They cost as much as in one (us, one / two: 16 chains of 64 tokens of 128 12.3 / 12.2, 4096 197 / 190, of
// 64 57 / 57, in half precision 55 / 60, 16384 of 8 tokens of 64 186 / 193; pullbacks, which leave out the state that nobody wants, too, 180 / 164, 96 / 88, 107 / 98, 397 /
// 331), longer calls do not (chunk_kernel's comment).
constexpr int MOST_TWICE = CHUNK;

// Offsets within a chunk are 32 bits.
constexpr int64_t MOST_STRIDE = (int64_t)1 << 23;

// Whether rows can be taken in whole 16-byte pieces on their grid, which transfers past the registers need; others are loaded and written to LDS, a chunk's loads
// with nothing beside them (us, on the grid / off it: 96 chains of 1024 x 64 28 / 65, 512 of 4096 x 128 473 / 757, pullbacks 39 / 69 and 1080 / 2070).
inline bool in_pieces(const Call& call) {
    for (int i = 0; i < call.chains; ++i) {
        const Chain& ch = call.chain[i];
        if (ch.Da % 8 || ch.Dc % 8) return false;
        for (const View* v : {&ch.a, &ch.b, &ch.c, &ch.out})
            if (reinterpret_cast<uintptr_t>(v->p) % 16 || v->sb % 8 || v->sp % 8 || v->sh % 8 || v->st % 8 || v->st < 0 || v->st >= MOST_STRIDE) return false;
    }
    return true;
}

template <typename T, int PLANES, bool TWICE> int by_pieces(const Call& call, hipStream_t stream) {
    return in_pieces(call) ? by_dims<T, true, PLANES, TWICE>(call, stream) : by_dims<T, false, PLANES, TWICE>(call, stream);
}

}  // namespace linear_attn
}  // namespace lbi
