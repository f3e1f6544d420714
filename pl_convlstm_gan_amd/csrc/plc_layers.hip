// C ABI of the layer operators (see include/plconvlstm.h): gated linear recurrence, group norm with an activation,
// dropout from a counter-based generator.  Argument checks, choice of the variant, launches; no allocation, no
// synchronisation, no state.
#include <math.h>
#include <string.h>

#include "plc_host.h"
#include "plc_dropout_kernels.h"
#include "plc_norm_kernels.h"
#include "plc_scan_kernels.h"

static int dtype_size(int dtype) { return dtype == PLC_F32 ? 4 : (dtype == PLC_BF16 || dtype == PLC_F16 ? 2 : 0); }
// a launch counts its work-items in 32 bits
static bool grid_ok(long long blocks, int threads) { return blocks >= 0 && blocks * threads < (1ll << 32); }

// largest number of elements of a vector access, at most `v`, that every one of the given addresses and strides allows
struct VecRule {
    int v;
    void pointer(const void* p, int e) { while (v > 1 && ((uintptr_t)p & ((v * e > 16 ? 16 : v * e) - 1))) v /= 2; }
    void stride(long long s) { while (v > 1 && s % v) v /= 2; }
};

#define PLC_BY_TYPE(dtype, CALL)            \
    switch (dtype) {                        \
        case PLC_F32: CALL(float); break;   \
        case PLC_BF16: CALL(plc_bf16); break; \
        default: CALL(plc_f16); break;      \
    }

// ---------------------------------------------------------------------------------------------
// dropout
// ---------------------------------------------------------------------------------------------
static PlcDrop drop_of(double p, unsigned long long seed, unsigned long long offset) {
    PlcDrop d;
    d.seed = seed;
    d.offset = offset;
    d.thr = (uint32_t)floor(p * 65536.0 + 0.5);
    d.scale = d.thr < 65536 ? (float)(65536.0 / (65536.0 - d.thr)) : 0.0f;
    return d;
}

extern "C" int plc_dropout(const void* x, const void* residual, void* y, long long n, int dtype, double p,
                           unsigned long long seed, unsigned long long offset, const long long* offset_ptr,
                           long long* used_offset, void* stream) {
    const int e = dtype_size(dtype);
    PLC_REQUIRE(e, "dropout: unknown element type %d", dtype);
    PLC_REQUIRE(n >= 0, "dropout: negative size");
    PLC_REQUIRE(p >= 0.0 && p <= 1.0, "dropout: p = %g is not a probability", p);
    if (n == 0) return PLC_OK;
    PLC_REQUIRE(x && y, "dropout: null tensor pointer");
    PLC_REQUIRE((((uintptr_t)x | (uintptr_t)y | (uintptr_t)residual) & (e - 1)) == 0, "dropout: misaligned tensor pointer");
    DropoutArgs a;
    a.n = n;
    a.x = x;
    a.r = residual;
    a.y = y;
    a.drop = drop_of(p, seed, offset);
    a.offset_ptr = offset_ptr;
    a.used_offset = used_offset;
    const long long blocks = (n + 2047) / 2048;
    if (!grid_ok(blocks, 256)) return plc_fail(PLC_EUNSUPPORTED, "dropout: %lld elements are more than one launch covers", n);
    const bool wide = aligned16(x) && aligned16(y) && aligned16(residual);
#define CALL(T)                                                                                                        \
    if (wide) hipLaunchKernelGGL((plc_dropout_kernel<T, 8>), dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, a); \
    else hipLaunchKernelGGL((plc_dropout_kernel<T, 1>), dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, a)
    PLC_BY_TYPE(dtype, CALL)
#undef CALL
    PLC_HIP(hipGetLastError());
    return PLC_OK;
}

// ---------------------------------------------------------------------------------------------
// gated linear recurrence
// ---------------------------------------------------------------------------------------------
extern "C" size_t plc_gated_scan_states_bytes(int B, int T, long long D) {
    if (B <= 0 || T <= 0 || D <= 0) return 0;
    return (size_t)B * ((T + SCAN_K - 1) / SCAN_K - 1) * (size_t)D * 4;
}

extern "C" size_t plc_gated_scan_workspace_bytes(const plc_scan_desc* d, int backward) {
    (void)d;
    (void)backward;
    return 0;
}

static int scan_check(const plc_scan_desc* d, bool backward, ScanArgs* a, int* v) {
    PLC_REQUIRE(d, "gated scan: null descriptor");
    const int e = dtype_size(d->dtype);
    PLC_REQUIRE(e, "gated scan: unknown element type %d", d->dtype);
    PLC_REQUIRE(d->B >= 0 && d->T >= 0 && d->D >= 0, "gated scan: negative size");
    memset(a, 0, sizeof(*a));
    if (d->B == 0 || d->D == 0) return PLC_OK;
    const bool any = d->T > 0;
    PLC_REQUIRE(!any || (d->x && d->f), "gated scan: null input pointer");
    PLC_REQUIRE(!any || (backward ? (d->dy && d->dx && d->df) : d->y != nullptr), "gated scan: null output pointer");
    PLC_REQUIRE(!backward || d->T <= SCAN_K || d->states, "gated scan: the backward pass needs the states the forward pass stored");
    a->B = d->B; a->T = d->T; a->D = d->D;
    a->coupled = d->coupled != 0;
    a->x = d->x; a->x_sb = d->x_batch; a->x_st = d->x_step;
    a->f = d->f; a->f_sb = d->f_batch; a->f_st = d->f_step;
    a->dy = d->dy; a->dy_sb = d->dy_batch; a->dy_st = d->dy_step;
    a->h0 = d->h0; a->dh_last = d->dh_last;
    a->lengths = d->lengths;
    a->y = d->y; a->dx = d->dx; a->df = d->df;
    a->h_last = d->h_last; a->dh0 = d->dh0; a->states = d->states;
    const void* types[] = {d->x, d->f, d->y, backward ? d->dy : nullptr, backward ? d->dx : nullptr, backward ? d->df : nullptr};
    const void* floats[] = {d->h0, d->h_last, d->states, backward ? d->dh_last : nullptr, backward ? d->dh0 : nullptr};
    for (const void* p : types) PLC_REQUIRE(((uintptr_t)p & (e - 1)) == 0, "gated scan: misaligned tensor pointer");
    for (const void* p : floats) PLC_REQUIRE(((uintptr_t)p & 3) == 0, "gated scan: misaligned state pointer");
    VecRule r{16 / e};
    for (const void* p : types) r.pointer(p, e);
    for (const void* p : floats) r.pointer(p, 4);
    r.stride(d->D);
    r.stride(d->x_batch); r.stride(d->x_step); r.stride(d->f_batch); r.stride(d->f_step);
    if (backward) { r.stride(d->dy_batch); r.stride(d->dy_step); }
    *v = r.v;
    return PLC_OK;
}

template <class T>
static int scan_launch(const ScanArgs& a, bool backward, int v, hipStream_t st) {
    const long long lanes = a.B * (a.D / v), blocks = (lanes + 255) / 256;
    if (!grid_ok(blocks, 256)) return plc_fail(PLC_EUNSUPPORTED, "gated scan: %lld lanes are more than one launch covers", lanes);
    const dim3 grid((unsigned)blocks), block(256);
#define CALL(V)                                                                                  \
    if (backward) hipLaunchKernelGGL((plc_scan_bwd_kernel<T, V>), grid, block, 0, st, a);        \
    else hipLaunchKernelGGL((plc_scan_fwd_kernel<T, V>), grid, block, 0, st, a)
    switch (v) {
        case 8: if constexpr (sizeof(T) == 2) { CALL(8); } break;
        case 4: CALL(4); break;
        case 2: CALL(2); break;
        default: CALL(1); break;
    }
#undef CALL
    PLC_HIP(hipGetLastError());
    return PLC_OK;
}

static int scan_run(const plc_scan_desc* d, bool backward, void* stream) {
    ScanArgs a;
    int v = 1;
    const int rc = scan_check(d, backward, &a, &v);
    if (rc || a.B == 0 || a.D == 0) return rc;
    // (four channels at most: with eight, the sixteen steps a lane holds in registers exceed them)
    if (v > 4) v = 4;
    switch (d->dtype) {
        case PLC_F32: return scan_launch<float>(a, backward, v, (hipStream_t)stream);
        case PLC_BF16: return scan_launch<plc_bf16>(a, backward, v, (hipStream_t)stream);
        default: return scan_launch<plc_f16>(a, backward, v, (hipStream_t)stream);
    }
}

extern "C" int plc_gated_scan_fwd(const plc_scan_desc* d, void* stream) { return scan_run(d, false, stream); }
extern "C" int plc_gated_scan_bwd(const plc_scan_desc* d, void* stream) { return scan_run(d, true, stream); }

// ---------------------------------------------------------------------------------------------
// group norm with an activation
// ---------------------------------------------------------------------------------------------
static int norm_geometry(const plc_norm_desc* d, NormArgs* a, int* v) {
    PLC_REQUIRE(d, "group norm: null descriptor");
    const int e = dtype_size(d->dtype);
    PLC_REQUIRE(e, "group norm: unknown element type %d", d->dtype);
    PLC_REQUIRE(d->N >= 0 && d->HW >= 0 && d->C > 0, "group norm: bad size");
    PLC_REQUIRE(d->G > 0 && d->C % d->G == 0, "group norm: %d channels do not divide into %d groups", d->C, d->G);
    PLC_REQUIRE(d->act >= PLC_ACT_NONE && d->act <= PLC_ACT_SILU, "group norm: unknown activation %d", d->act);
    PLC_REQUIRE(d->layout == PLC_NHWC || d->layout == PLC_CB8, "group norm: unknown layout %d", d->layout);
    PLC_REQUIRE(d->layout == PLC_NHWC || d->C % 8 == 0, "group norm: the CB8 layout takes whole blocks of 8 channels, not %d", d->C);
    PLC_REQUIRE(d->eps >= 0.0f, "group norm: negative eps");
    PLC_REQUIRE(d->p >= 0.0 && d->p <= 1.0, "group norm: p = %g is not a probability", d->p);
    memset(a, 0, sizeof(*a));
    a->N = d->N; a->C = d->C; a->G = d->G; a->HW = d->HW;
    a->cg = d->C / d->G;
    VecRule r{8};
    r.stride(d->C);
    const void* types[] = {d->x, d->y, d->dy, d->dx};
    for (const void* p : types) PLC_REQUIRE(((uintptr_t)p & (e - 1)) == 0, "group norm: misaligned tensor pointer");
    for (const void* p : types) r.pointer(p, e);
    PLC_REQUIRE(d->layout == PLC_NHWC || r.v == 8, "group norm: CB8 tensors must be 16-byte aligned");
    *v = r.v;
    a->U = d->C / r.v;
    a->img = (long long)d->HW * d->C;
    if (d->layout == PLC_NHWC) {
        a->us = r.v;
        a->ps = d->C;
        a->ut = a->U < 256 ? a->U : 256;
    } else {
        a->us = 8ll * d->HW;
        a->ps = 8;
        a->ut = 1;
    }
    a->tiles = cdiv(a->U, a->ut);
    const int rows = 256 / a->ut;
    // pixel ranges: enough workgroups for the chip, at least one round of loads each, at most 64 partial sums for the
    // second pass to add
    const long long want = 2048, per = (long long)d->N * a->tiles;
    long long s = per > 0 ? (want + per - 1) / per : 1;
    const long long most = d->HW > 0 ? (d->HW + NORM_P * rows - 1) / (NORM_P * rows) : 1;
    s = s > most ? most : s;
    s = s > 64 ? 64 : (s < 1 ? 1 : s);
    a->px_split = d->HW > 0 ? (int)((d->HW + s - 1) / s) : 1;
    a->splits = d->HW > 0 ? cdiv(d->HW, a->px_split) : 1;
    a->px_chunk = a->px_split;
    a->chunks = a->splits;
    a->act = d->act;
    a->eps = d->eps;
    a->x = d->x; a->dy = d->dy; a->y = d->y; a->dx = d->dx;
    a->w = d->weight; a->b = d->bias; a->dw = d->dweight; a->db = d->dbias;
    a->stats = d->stats;
    a->part = (float*)d->workspace;
    a->drop = drop_of(d->p, d->seed, d->offset);
    a->offset_ptr = d->offset_ptr;
    a->used_offset = d->used_offset;
    return PLC_OK;
}

static size_t norm_workspace(const NormArgs& a) { return (size_t)a.N * a.splits * a.C * 2 * sizeof(float); }

extern "C" size_t plc_group_norm_workspace_bytes(const plc_norm_desc* d) {
    NormArgs a;
    int v;
    if (norm_geometry(d, &a, &v) != PLC_OK) return 0;
    return norm_workspace(a);
}

static int norm_check(const plc_norm_desc* d, bool backward, NormArgs* a, int* v) {
    const int rc = norm_geometry(d, a, v);
    if (rc) return rc;
    const bool any = d->N > 0 && d->HW > 0;
    PLC_REQUIRE(!any || (d->x && d->stats && (backward ? d->dy && d->dx : d->y != nullptr)), "group norm: null tensor pointer");
    PLC_REQUIRE(!any || d->workspace, "group norm: null workspace");
    PLC_REQUIRE((((uintptr_t)d->weight | (uintptr_t)d->bias | (uintptr_t)d->stats | (uintptr_t)d->workspace |
                  (uintptr_t)d->dweight | (uintptr_t)d->dbias) & 3) == 0, "group norm: misaligned float pointer");
    if (any && d->workspace_bytes < norm_workspace(*a))
        return plc_fail(PLC_EWORKSPACE, "group norm: workspace %zu < %zu bytes", d->workspace_bytes, norm_workspace(*a));
    const long long blocks = (long long)a->N * a->tiles * (a->splits > a->chunks ? a->splits : a->chunks) + cdiv(a->C, NORM_PARAM_CH);
    if (!grid_ok(blocks, 256)) return plc_fail(PLC_EUNSUPPORTED, "group norm: %d samples are more than one launch covers", d->N);
    return PLC_OK;
}

template <class T, int V>
static int norm_launch(NormArgs a, bool backward, hipStream_t st) {
    const unsigned per = (unsigned)a.N * a.tiles;
    const int nch = a.ut * V;
    const int sum_lds = (2 * nch + 256 * V * (backward ? 2 : 1)) * (int)sizeof(float);
    if (!backward) {
        hipLaunchKernelGGL((plc_norm_stats_kernel<T, V>), dim3(per * a.splits), dim3(256), sum_lds, st, a);
        hipLaunchKernelGGL((plc_norm_fwd_kernel<T, V>), dim3(per * a.chunks), dim3(256), 2 * (nch + 1) * sizeof(float), st, a);
    } else {
        hipLaunchKernelGGL((plc_norm_bwd_sums_kernel<T, V>), dim3(per * a.splits), dim3(256), sum_lds, st, a);
        a.param_blocks = a.dw || a.db ? cdiv(a.C, NORM_PARAM_CH) : 0;
        int lds = 4 * (nch + 1) * (int)sizeof(float);
        if (lds < 2 * 256 * (int)sizeof(double)) lds = 2 * 256 * (int)sizeof(double);
        hipLaunchKernelGGL((plc_norm_bwd_kernel<T, V>), dim3(per * a.chunks + a.param_blocks), dim3(256), lds, st, a);
    }
    PLC_HIP(hipGetLastError());
    return PLC_OK;
}

__global__ void plc_norm_clear_kernel(float* a, float* b, int n) {
    const int i = blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= n) return;
    if (a) a[i] = 0.0f;
    if (b) b[i] = 0.0f;
}

static int norm_run(const plc_norm_desc* d, bool backward, void* stream) {
    NormArgs a;
    int v = 1;
    const int rc = norm_check(d, backward, &a, &v);
    if (rc) return rc;
    hipStream_t st = (hipStream_t)stream;
    if (a.N == 0 || a.HW == 0) {          // no element: the parameters' gradients are sums over nothing
        if (backward && (a.dw || a.db)) {
            hipLaunchKernelGGL(plc_norm_clear_kernel, dim3(cdiv(a.C, 256)), dim3(256), 0, st, a.dw, a.db, a.C);
            PLC_HIP(hipGetLastError());
        }
        return PLC_OK;
    }
#define CALL(T)                                             \
    switch (v) {                                            \
        case 8: return norm_launch<T, 8>(a, backward, st);  \
        case 4: return norm_launch<T, 4>(a, backward, st);  \
        case 2: return norm_launch<T, 2>(a, backward, st);  \
        default: return norm_launch<T, 1>(a, backward, st); \
    }
    PLC_BY_TYPE(d->dtype, CALL)
#undef CALL
    return PLC_OK;
}

extern "C" int plc_group_norm_fwd(const plc_norm_desc* d, void* stream) { return norm_run(d, false, stream); }
extern "C" int plc_group_norm_bwd(const plc_norm_desc* d, void* stream) { return norm_run(d, true, stream); }
