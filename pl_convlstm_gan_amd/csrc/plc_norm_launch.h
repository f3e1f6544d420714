// Launches of the group norm, one translation unit per element type (plc_norm_f32.hip, ...); the plan is made in
// plc_layers.hip.
#pragma once
#include "plc_host.h"
#include "plc_norm_kernels.h"

struct NormPlan {
    int v;               // channels of a unit
    int ku, threads;     // resident form: units of a thread (0: split form), threads of a workgroup
    bool stream;         // split form: the tensors are larger than what the caches keep between two passes
    size_t part_g, part_c, total;     // workspace
};

PLC_HIDDEN int plc_norm_launch_f32(const NormArgs& a, const NormPlan& pl, bool backward, hipStream_t st);
PLC_HIDDEN int plc_norm_launch_bf16(const NormArgs& a, const NormPlan& pl, bool backward, hipStream_t st);
PLC_HIDDEN int plc_norm_launch_f16(const NormArgs& a, const NormPlan& pl, bool backward, hipStream_t st);

#ifdef PLC_NORM_TYPE
namespace {
template <class T, int V, int FORM>
int norm_launch(NormArgs a, const NormPlan& pl, bool backward, hipStream_t st) {
    const unsigned blocks = (unsigned)a.N * a.tiles * a.splits;
    const int nch = a.ut * V, params = a.dw || a.db ? cdiv(a.C, NORM_PARAM_CH) : 0;
    const int f = (int)sizeof(float);
    if (pl.ku) {
        const int lds = (5 * nch + norm_lds_floats(pl.threads, a.ut, V, 1)) * f;
        const dim3 grid(blocks), block(pl.threads);
        if (!backward) {
            if (pl.ku == 4) hipLaunchKernelGGL((plc_norm_fwd_resident_kernel<T, V, FORM, 4>), grid, block, lds, st, a);
            else hipLaunchKernelGGL((plc_norm_fwd_resident_kernel<T, V, FORM, 16>), grid, block, lds, st, a);
        } else {
            if (pl.ku == 4) hipLaunchKernelGGL((plc_norm_bwd_resident_kernel<T, V, FORM, 4>), grid, block, lds, st, a);
            else hipLaunchKernelGGL((plc_norm_bwd_resident_kernel<T, V, FORM, 8>), grid, block, lds, st, a);
            if (params) hipLaunchKernelGGL(plc_norm_params_kernel<T>, dim3(params), dim3(256), 0, st, a);
        }
    } else if (!backward) {
        hipLaunchKernelGGL((plc_norm_stats_kernel<T, V>), dim3(blocks), dim3(256), (nch + norm_lds_floats(256, a.ut, V, 2)) * f, st, a);
        hipLaunchKernelGGL((plc_norm_fwd_kernel<T, V, FORM>), dim3(blocks), dim3(256), 2 * nch * f, st, a);
    } else {
        hipLaunchKernelGGL((plc_norm_bwd_sums_kernel<T, V, FORM>), dim3(blocks), dim3(256), (3 * nch + norm_lds_floats(256, a.ut, V, 1)) * f, st, a);
        a.param_blocks = params;
        const int lds = 4 * nch * f, need = 512 * (int)sizeof(double);
        const dim3 grid(blocks + params);
        if (V * sizeof(T) == 16 && pl.stream) hipLaunchKernelGGL((plc_norm_bwd_kernel<T, V, FORM, V * sizeof(T) == 16>), grid, dim3(256), lds < need ? need : lds, st, a);
        else hipLaunchKernelGGL((plc_norm_bwd_kernel<T, V, FORM, false>), grid, dim3(256), lds < need ? need : lds, st, a);
    }
    PLC_HIP(hipGetLastError());
    return PLC_OK;
}

template <class T, int V>
int norm_form(const NormArgs& a, const NormPlan& pl, bool backward, hipStream_t st) {
    // (the widest vectors with the activation and dropout compiled in; the others are for few shapes)
    if constexpr (V * sizeof(T) == 16) {
        switch (a.act + (a.drop.thr ? 3 : 0)) {
            case 0: return norm_launch<T, V, 0>(a, pl, backward, st);
            case 1: return norm_launch<T, V, 1>(a, pl, backward, st);
            case 2: return norm_launch<T, V, 2>(a, pl, backward, st);
            case 3: return norm_launch<T, V, 3>(a, pl, backward, st);
            case 4: return norm_launch<T, V, 4>(a, pl, backward, st);
            default: return norm_launch<T, V, 5>(a, pl, backward, st);
        }
    } else {
        return norm_launch<T, V, -1>(a, pl, backward, st);
    }
}
template <class T>
int norm_type(const NormArgs& a, const NormPlan& pl, bool backward, hipStream_t st) {
    switch (pl.v) {
        case 8: if constexpr (sizeof(T) == 2) return norm_form<T, 8>(a, pl, backward, st);
        case 4: return norm_form<T, 4>(a, pl, backward, st);
        case 2: if constexpr (sizeof(T) == 2) return norm_form<T, 2>(a, pl, backward, st);
        default: return norm_form<T, 1>(a, pl, backward, st);
    }
}
}  // namespace
#endif
