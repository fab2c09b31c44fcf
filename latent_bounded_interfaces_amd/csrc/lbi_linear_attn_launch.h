// Launches of lbi_linear_attn_kernel.h for one type: which tiles and copies a call takes.
#pragma once

#include "lbi_linear_attn_kernel.h"

namespace lbi {
namespace linear_attn {

template <typename T, int DA, int DC, bool VEC, int PLANES>
int launch(const Call& call, hipStream_t stream) {
    const int64_t units = (int64_t)call.chains * call.B * call.P * call.H;
    const auto grid = [](int64_t workgroups) { return dim3((unsigned)((workgroups + 7) / 8 * 8)); };
    if (call.segments > 1) {
        hipLaunchKernelGGL((chunk_kernel<T, DA, DC, VEC, false, PLANES>), grid(units * (call.segments - 1)), dim3(256), 0, stream, call);
        LBI_HIP_CHECK(hipGetLastError());
        const int elements = call.chain[0].Da * call.chain[0].Dc;
        hipLaunchKernelGGL(join_kernel<T>, dim3((unsigned)((elements + 255) / 256), (unsigned)units), dim3(256), 0, stream, call);
        LBI_HIP_CHECK(hipGetLastError());
    }
    hipLaunchKernelGGL((chunk_kernel<T, DA, DC, VEC, true, PLANES>), grid(units * call.segments), dim3(256), 0, stream, call);
    LBI_HIP_CHECK(hipGetLastError());
    return LBI_OK;
}

template <typename T, bool VEC, int PLANES> int by_dims(const Call& call, hipStream_t stream) {
    const bool wide_a = call.chain[0].Da > 64, wide_c = call.chain[0].Dc > 64;
    if (wide_a) return wide_c ? launch<T, 128, 128, VEC, PLANES>(call, stream) : launch<T, 128, 64, VEC, PLANES>(call, stream);
    return wide_c ? launch<T, 64, 128, VEC, PLANES>(call, stream) : launch<T, 64, 64, VEC, PLANES>(call, stream);
}

// Whether rows can be taken in whole 16-byte pieces.
inline bool in_pieces(const Call& call) {
    for (int i = 0; i < call.chains; ++i) {
        const Chain& ch = call.chain[i];
        if (ch.Da % 8 || ch.Dc % 8) return false;
        for (const View* v : {&ch.a, &ch.b, &ch.c, &ch.out})
            if (reinterpret_cast<uintptr_t>(v->p) % 16 || v->sb % 8 || v->sp % 8 || v->sh % 8 || v->st % 8) return false;
    }
    return true;
}

template <typename T, int PLANES> int by_pieces(const Call& call, hipStream_t stream) {
    return in_pieces(call) ? by_dims<T, true, PLANES>(call, stream) : by_dims<T, false, PLANES>(call, stream);
}

}  // namespace linear_attn
}  // namespace lbi
