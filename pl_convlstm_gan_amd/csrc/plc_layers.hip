// C ABI of the layer operators (see include/plconvlstm.h): gated linear recurrence, group norm with an activation,
// dropout from a counter-based generator.  Argument checks, choice of the variant, launches; no allocation, no
// synchronisation, no state.
#include <math.h>
#include <string.h>

#include "plc_host.h"
#include "plc_dropout_kernels.h"
#include "plc_norm_launch.h"
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

// Whether an operator that reads its inputs once reads them past the caches.  It pays for tensors whose inputs and output
// together do not fit the 256 MB behind the L2s while each alone does: the output stays there, for whoever reads it next.
// In us, kept against streamed, in brackets with a reader of the output behind it:
//   scan forward, bf16   84 MB 49.5 (81.8) 53.9 (79.3)   126 MB 83.5 (129) 79.4 (119)   168 MB 110 (167) 97 (150)   335 MB 218 (320) 230 (343)
//   dropout + residual   84 MB 42.9 (70.8) 44.2 (70.0)   126 MB 69.2 (112) 62.0 (102)   168 MB 91.6 (151) 87.3 (138)   335 MB 177 (286) 168 (291)
//   dropout              84 MB 31.1 (56.5) 28.9 (53.2)   126 MB 44.4 (85.5) 41.6 (80.0)   168 MB 58.8 (115) 57.7 (111)   250 MB 84.3 (167) 85.1 (170)   335 MB 112 (219) 112 (226)
// (Dropout alone has one input; the one range serves both.  fp32 dropout does not stream at any size: a lane moves 32 bytes of it
// in two accesses, and the form was not built for it.)
// (Not where a backward pass will read the scan's inputs again: a training pass of 168 MB tensors takes 316 us with it, 309 without.)
static bool streams(double bytes) { return bytes > 100e6 && bytes < 256e6; }

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
    PLC_REQUIRE((((uintptr_t)offset_ptr | (uintptr_t)used_offset) & 7) == 0, "dropout: misaligned offset pointer");
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
    const bool wide = aligned16(x) && aligned16(y) && aligned16(residual), large = streams((double)n * e);
#define CALL(T)                                                                                                        \
    if (wide && large) hipLaunchKernelGGL((plc_dropout_kernel<T, 8, sizeof(T) == 2>), dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, a); \
    else if (wide) hipLaunchKernelGGL((plc_dropout_kernel<T, 8, false>), dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, a); \
    else hipLaunchKernelGGL((plc_dropout_kernel<T, 1, false>), dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, a)
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

static int scan_check(const plc_scan_desc* d, bool backward, ScanArgs* a, int* v) {
    PLC_REQUIRE(d, "gated scan: null descriptor");
    const int e = dtype_size(d->dtype);
    PLC_REQUIRE(e, "gated scan: unknown element type %d", d->dtype);
    PLC_REQUIRE(d->B >= 0 && d->T >= 0 && d->D >= 0, "gated scan: negative size");
    if (d->T > 1 << 30) return plc_fail(PLC_EUNSUPPORTED, "gated scan: %d steps are more than 2^30", d->T);
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

// How a call runs: channels per lane, and segments of time (1: one lane walks the whole sequence).
//
// One pass costs about 0.11 us a step (a block of SCAN_K steps is one trip to memory) until the rows fill the memory; the
// split form costs three launches, 8 us, and reads its inputs twice.  So time is split for long sequences of narrow rows.
// Forward/backward in us, split against one pass, rows of n = B x D numbers (4 samples):
//   n = 512, bf16:    T = 64   8.1/8.4 against  6.6/9.3     T = 96   8.1/8.3 against  8.8/12.9    T = 1024   9.2/9.4 against  73/140
//   n = 16000, fp32:  T = 96  14.3/15.7 against 13.2/16.8   T = 128 15.0/16.5 against 16.8/21.2   T = 1024  71/104  against 179/228
//   n = 80000, bf16:  T = 128 28.8/36.7 against 20.2/32.4   T = 256 49.1/69.4 against 55.9/73.1   T = 1024 197/272  against 221/288
//   n = 80000, fp32:  T = 128 42.2/61.6 against 33.2/45.5   T = 256 92/128    against 64.5/94.5   (one pass at every length)
//
// Without the split, lanes take fewer channels until 1024 waves share the rows: more loads are in flight.  With 16 x 40000
// bf16 of 4 samples four channels per lane cost 6.9/9.0 us, two 6.2/8.3; 24 x 8192 fp32 of 8 samples 8.6/13.7 with four, 6.4/8.3 with one.
// Eight channels (16 bytes of a 16-bit type) pay forward once 4096 waves are left; backward they cost registers, and with
// them the waves that hide the loads (10 x 2097152 bf16 of 4 samples: 250 us against 190).
static void scan_plan(ScanArgs* a, int e, int vmax, bool backward, int* v) {
    const long long n = (long long)a->B * a->D;
    *v = vmax < 4 ? vmax : 4;
    a->nseg = 1;
    a->seg = a->T;
    if (n * e <= 160 << 10 && a->T >= 80 + n * e / 1024) {
        *v = vmax >= 2 && n >= 1024 ? 2 : 1;
        const long long most = a->T >= 1 << 18 ? 64 * 4 * SCAN_RUN : 64 * SCAN_RUN;
        long long want = 4096 * 64ll / (n / *v);
        want = want > most ? most : (want < 1 ? 1 : want);
        long long seg = (a->T + want - 1) / want;
        seg = (seg + SCAN_K - 1) / SCAN_K * SCAN_K;
        a->seg = (int)seg;
        a->nseg = (int)((a->T + seg - 1) / seg);
    } else if (vmax == 8 && !backward && n / 8 / 64 >= 4096) {
        *v = 8;
    } else {
        while (*v > 1 && n / *v / 64 < 1024) *v /= 2;
    }
}

template <bool BACKWARD, int R>
static void scan_carry_runs(const ScanArgs& a, hipStream_t st) {
    constexpr int CH = scan_carry_channels(R);
    hipLaunchKernelGGL((plc_scan_carry_kernel<BACKWARD, R>), dim3((unsigned)(((long long)a.B * a.D + CH - 1) / CH)), dim3(R * CH), 0, st, a);
}
template <bool BACKWARD>
static void scan_carry(const ScanArgs& a, hipStream_t st) {
    if (a.nseg <= 4) scan_carry_runs<BACKWARD, 1>(a, st);
    else if (a.nseg <= 32) scan_carry_runs<BACKWARD, 4>(a, st);
    else if (a.nseg <= 16 * SCAN_RUN) scan_carry_runs<BACKWARD, 16>(a, st);
    else scan_carry_runs<BACKWARD, 64>(a, st);
}

template <class T, int V, bool COUPLED, bool BACKWARD>
static int scan_launch(const ScanArgs& a, hipStream_t st) {
    const long long lanes = a.B * (a.D / V);
    if (a.nseg > 1) {
        const dim3 grid((unsigned)((lanes * a.nseg + 255) / 256)), block(256);
        hipLaunchKernelGGL((plc_scan_segments_kernel<T, V, COUPLED, BACKWARD>), grid, block, 0, st, a);
        scan_carry<BACKWARD>(a, st);
        hipLaunchKernelGGL((plc_scan_split_kernel<T, V, COUPLED, BACKWARD>), grid, block, 0, st, a);
    } else {
        const long long blocks = (lanes + 255) / 256;
        if (!grid_ok(blocks, 256)) return plc_fail(PLC_EUNSUPPORTED, "gated scan: %lld lanes are more than one launch covers", lanes);
        const dim3 grid((unsigned)blocks), block(256);
        if (BACKWARD) hipLaunchKernelGGL((plc_scan_bwd_kernel<T, V, COUPLED>), grid, block, 0, st, a);
        else if (V * sizeof(T) == 16 && !a.states && streams((double)a.B * a.T * a.D * sizeof(T)))
            hipLaunchKernelGGL((plc_scan_fwd_kernel<T, V, COUPLED, V * sizeof(T) == 16>), grid, block, 0, st, a);
        else hipLaunchKernelGGL((plc_scan_fwd_kernel<T, V, COUPLED, false>), grid, block, 0, st, a);
    }
    PLC_HIP(hipGetLastError());
    return PLC_OK;
}

static size_t scan_workspace(const ScanArgs& a) { return a.nseg > 1 ? (size_t)a.nseg * 2 * a.B * (size_t)a.D * 4 : 0; }

extern "C" size_t plc_gated_scan_workspace_bytes(const plc_scan_desc* d, int backward) {
    ScanArgs a;
    int v = 1;
    if (scan_check(d, backward != 0, &a, &v) || a.B == 0 || a.D == 0) return 0;
    scan_plan(&a, dtype_size(d->dtype), v, backward != 0, &v);
    return scan_workspace(a);
}

template <class T, int V>
static int scan_pick(const ScanArgs& a, bool backward, hipStream_t st) {
    if (a.coupled) return backward ? scan_launch<T, V, true, true>(a, st) : scan_launch<T, V, true, false>(a, st);
    return backward ? scan_launch<T, V, false, true>(a, st) : scan_launch<T, V, false, false>(a, st);
}
template <class T>
static int scan_type(const ScanArgs& a, bool backward, int v, hipStream_t st) {
    switch (v) {
        case 8: if constexpr (sizeof(T) == 2) return scan_pick<T, 8>(a, backward, st);
        case 4: return scan_pick<T, 4>(a, backward, st);
        case 2: return scan_pick<T, 2>(a, backward, st);
        default: return scan_pick<T, 1>(a, backward, st);
    }
}

static int scan_run(const plc_scan_desc* d, bool backward, void* stream) {
    ScanArgs a;
    int v = 1;
    const int rc = scan_check(d, backward, &a, &v);
    if (rc || a.B == 0 || a.D == 0) return rc;
    scan_plan(&a, dtype_size(d->dtype), v, backward, &v);
    const size_t need = scan_workspace(a);
    if (need) {
        if (!d->workspace || d->workspace_bytes < need)
            return plc_fail(PLC_EWORKSPACE, "gated scan: workspace %zu < %zu bytes", d->workspace ? d->workspace_bytes : 0, need);
        PLC_REQUIRE(aligned16(d->workspace), "gated scan: workspace must be 16-byte aligned");
        a.agg = (float*)d->workspace;
    }
    switch (d->dtype) {
        case PLC_F32: return scan_type<float>(a, backward, v, (hipStream_t)stream);
        case PLC_BF16: return scan_type<plc_bf16>(a, backward, v, (hipStream_t)stream);
        default: return scan_type<plc_f16>(a, backward, v, (hipStream_t)stream);
    }
}

extern "C" int plc_gated_scan_fwd(const plc_scan_desc* d, void* stream) { return scan_run(d, false, stream); }
extern "C" int plc_gated_scan_bwd(const plc_scan_desc* d, void* stream) { return scan_run(d, true, stream); }

// ---------------------------------------------------------------------------------------------
// group norm with an activation
// ---------------------------------------------------------------------------------------------
static int gcd(int a, int b) { return b ? gcd(b, a % b) : a; }

static int norm_plan(const plc_norm_desc* d, bool backward, NormArgs* a, NormPlan* pl) {
    PLC_REQUIRE(d, "group norm: null descriptor");
    const int e = dtype_size(d->dtype);
    PLC_REQUIRE(e, "group norm: unknown element type %d", d->dtype);
    PLC_REQUIRE(d->N >= 0 && d->HW >= 0 && d->C > 0, "group norm: bad size");
    PLC_REQUIRE(d->G > 0 && d->C % d->G == 0, "group norm: %d channels do not divide into %d groups", d->C, d->G);
    PLC_REQUIRE(d->act >= PLC_ACT_NONE && d->act <= PLC_ACT_SILU, "group norm: unknown activation %d", d->act);
    PLC_REQUIRE(d->layout == PLC_NHWC || d->layout == PLC_CB8, "group norm: unknown layout %d", d->layout);
    PLC_REQUIRE(d->layout == PLC_NHWC || d->C % 8 == 0, "group norm: the CB8 layout takes whole blocks of 8 channels, not %d", d->C);
    PLC_REQUIRE(d->layout == PLC_NHWC || e == 2, "group norm: the CB8 layout holds 16-bit elements");
    PLC_REQUIRE(d->eps >= 0.0f, "group norm: negative eps");
    PLC_REQUIRE(d->p >= 0.0 && d->p <= 1.0, "group norm: p = %g is not a probability", d->p);
    PLC_REQUIRE((((uintptr_t)d->offset_ptr | (uintptr_t)d->used_offset) & 7) == 0, "group norm: misaligned offset pointer");
    if (d->HW > 1 << 30) return plc_fail(PLC_EUNSUPPORTED, "group norm: %d pixels are more than 2^30", d->HW);
    const void* types[] = {d->x, d->y, d->dy, d->dx};
    for (const void* p : types) PLC_REQUIRE(((uintptr_t)p & (e - 1)) == 0, "group norm: misaligned tensor pointer");
    memset(a, 0, sizeof(*a));
    memset(pl, 0, sizeof(*pl));
    a->N = d->N; a->C = d->C; a->G = d->G; a->HW = d->HW;
    a->cg = d->C / d->G;
    VecRule r{16 / e};
    r.stride(d->C);
    for (const void* p : types) r.pointer(p, e);
    PLC_REQUIRE(d->layout == PLC_NHWC || r.v == 8, "group norm: CB8 tensors must be 16-byte aligned");
    int v = r.v;
    if (e == 4 && v == 2) v = 1;       // (fp32 is compiled for 4 and 1)
    // the smallest run of units that holds whole groups; a group of more than 256 units is taken in parts, for which a
    // unit has to lie within one group
    int m0 = a->cg / gcd(v, a->cg);
    a->parts = 1;
    if (m0 > 256) {
        if (d->layout == PLC_NHWC) v = gcd(v, a->cg);
        if (e == 4 && v == 2) v = 1;
        PLC_REQUIRE(a->cg % v == 0, "group norm: CB8 groups of more than 2048 channels must be whole blocks");
        m0 = a->cg / v;
        a->gu = m0;
        a->parts = cdiv(m0, 256);
    }
    pl->v = v;
    a->U = d->C / v;
    a->img = (long long)d->HW * d->C;
    a->px_first = d->layout == PLC_CB8;
    a->us = a->px_first ? 8ll * d->HW : v;
    a->ps = a->px_first ? 8 : d->C;
    a->splits = 1;
    a->px_split = d->HW;
    // Resident form (one launch, x read once).  A thread keeps up to four units; or, forward 9 .. 16 and backward 5 .. 8, with
    // 512 threads, where a workgroup per CU (backward two) is left.  Rows as wide as 128 bytes while enough tiles are left.
    // Forward/backward in us against the split form (32 channels in 8 groups, bf16, unless said otherwise):
    //   5 x 15 x 12, fp32          3.9/7.7 against  9.3/10.4      8 x 512 channels in 32 groups, 32 x 32   8.9/17.0 against 23.6/25.6
    //   128 x 32 x 64             16.9/23.7 against 18.5/24.6      32 x 512 channels in 32 groups, 32 x 32 27.8/44 against 33.3/52.5
    //   512 x 40 x 40, 1 group    23.5/57.7 against 34.4/58.0
    // A tensor beyond the caches (20 MB) is another matter.  There the workgroups' loads, sums and stores have to overlap:
    // workgroups of more than 256 threads with four units each do not (512 x 8 channels x 64 x 64: 30.3/47.6 against 23.6/37.5),
    // and rows of less than 64 bytes that are part of longer ones move lines more than once (512 x 30 x 24, fp32, 16-byte rows:
    // 27.9/59.5 against 29.2/46.9).
    const int ku_max = backward ? 8 : 16;
    const double bytes = (double)a->N * (double)a->img * e;
    const bool large = bytes > 20e6;
    pl->stream = bytes > 64e6;
    if (a->parts == 1 && m0 <= 64 && d->HW > 0 && (long long)d->HW * m0 <= 512ll * ku_max) {
        int widest = m0;
        if (!a->px_first)
            while (a->U % (widest * 2) == 0 && widest * v * e < 128) widest *= 2;
        for (int limit = 4; limit <= ku_max && !pl->ku; limit = limit == 4 ? ku_max : 2 * ku_max)
            for (int ut = widest; ut >= m0; ut /= 2) {
                const int most = limit == 4 ? 1024 : 512, need = cdiv(d->HW, most / ut);
                const long long tiles = (long long)d->N * (a->U / ut);
                const bool lines = ut * v * e >= 64;
                if (need > limit) continue;
                if (limit == 4) {
                    if (tiles < 256 && ut / 2 >= m0) continue;
                    if (large && !((lines || ut == a->U || a->px_first) && cdiv(d->HW, 256 / ut) <= 4)) continue;
                } else if (tiles < (backward ? 512 : 256) || need <= ku_max / 2 || (backward && !lines)) {
                    continue;
                }
                a->ut = ut;
                pl->ku = limit;
                pl->threads = most;
                for (int n = 64; n < most; n *= 2)
                    if (n >= ut && cdiv(d->HW, n / ut) <= 4) {
                        pl->threads = n;
                        break;
                    }
                break;
            }
    }
    if (pl->ku == 0) {
        // Split form.  NHWC: whole rows up to 256 units; CB8: the smallest tile.
        if (a->parts > 1) a->ut = cdiv(a->gu, a->parts);
        else a->ut = a->px_first ? m0 : (a->U < 256 ? a->U : 256 / m0 * m0);
        pl->threads = 256;
        const int rows = 256 / a->ut, p = backward ? NORM_PB : NORM_P;
        a->tiles = a->parts > 1 ? a->G * a->parts : cdiv(a->U, a->ut);
        // Pixel ranges: two rounds of loads each at least, at most 256 per sample, and enough for 4096 workgroups: with 40 samples
        // of 256 x 256 x 32 in bf16 1024 of them cost 120/203 us, 2048 110/186, 4096 105/175, 8192 105/171; smaller calls do not differ.
        const long long per = (long long)d->N * a->tiles, want = per > 0 ? (4096 + per - 1) / per : 1;
        const long long most = d->HW > 0 ? (d->HW + 2 * p * rows - 1) / (2 * p * rows) : 1;
        long long s = want < most ? want : most;
        s = s > 256 ? 256 : (s < 1 ? 1 : s);
        a->px_split = d->HW > 0 ? (int)((d->HW + s - 1) / s) : 1;
        a->splits = d->HW > 0 ? cdiv(d->HW, a->px_split) : 1;
    }
    a->tiles = a->parts > 1 ? a->G * a->parts : cdiv(a->U, a->ut);
    a->act = d->act;
    a->eps = d->eps;
    a->x = d->x; a->dy = d->dy; a->y = d->y; a->dx = d->dx;
    a->w = d->weight; a->b = d->bias; a->dw = d->dweight; a->db = d->dbias;
    a->stats = d->stats;
    a->drop = drop_of(d->p, d->seed, d->offset);
    a->offset_ptr = d->offset_ptr;
    a->used_offset = d->used_offset;
    pl->part_g = 0;
    pl->part_c = align256((size_t)a->N * a->G * a->splits * a->parts * 2 * sizeof(float));
    pl->total = pl->part_c + (backward ? (size_t)a->N * a->splits * a->C * 2 * sizeof(float) : 0);
    return PLC_OK;
}

extern "C" size_t plc_group_norm_workspace_bytes(const plc_norm_desc* d, int backward) {
    NormArgs a;
    NormPlan pl;
    if (norm_plan(d, backward != 0, &a, &pl) != PLC_OK) return 0;
    return pl.total;
}

static int norm_check(const plc_norm_desc* d, bool backward, NormArgs* a, NormPlan* pl) {
    const int rc = norm_plan(d, backward, a, pl);
    if (rc) return rc;
    const bool any = d->N > 0 && d->HW > 0;
    PLC_REQUIRE(!any || (d->x && d->stats && (backward ? d->dy && d->dx : d->y != nullptr)), "group norm: null tensor pointer");
    PLC_REQUIRE(!any || d->workspace, "group norm: null workspace");
    PLC_REQUIRE((((uintptr_t)d->weight | (uintptr_t)d->bias | (uintptr_t)d->stats | (uintptr_t)d->dweight | (uintptr_t)d->dbias) & 3) == 0,
                "group norm: misaligned float pointer");
    PLC_REQUIRE(aligned16(d->workspace), "group norm: workspace must be 16-byte aligned");
    if (any && d->workspace_bytes < pl->total)
        return plc_fail(PLC_EWORKSPACE, "group norm: workspace %zu < %zu bytes", d->workspace_bytes, pl->total);
    a->part_g = (float*)((char*)d->workspace + pl->part_g);
    a->part_c = (float*)((char*)d->workspace + pl->part_c);
    const long long blocks = (long long)a->N * a->tiles * a->splits + cdiv(a->C, NORM_PARAM_CH);
    if (!grid_ok(blocks, pl->threads)) return plc_fail(PLC_EUNSUPPORTED, "group norm: %d samples are more than one launch covers", d->N);
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
    NormPlan pl;
    const int rc = norm_check(d, backward, &a, &pl);
    if (rc) return rc;
    hipStream_t st = (hipStream_t)stream;
    if (a.N == 0 || a.HW == 0) {          // no element: the parameters' gradients are sums over nothing
        if (backward && (a.dw || a.db)) {
            hipLaunchKernelGGL(plc_norm_clear_kernel, dim3(cdiv(a.C, 256)), dim3(256), 0, st, a.dw, a.db, a.C);
            PLC_HIP(hipGetLastError());
        }
        return PLC_OK;
    }
    switch (d->dtype) {
        case PLC_F32: return plc_norm_launch_f32(a, pl, backward, st);
        case PLC_BF16: return plc_norm_launch_bf16(a, pl, backward, st);
        default: return plc_norm_launch_f16(a, pl, backward, st);
    }
}

extern "C" int plc_group_norm_fwd(const plc_norm_desc* d, void* stream) { return norm_run(d, false, stream); }
extern "C" int plc_group_norm_bwd(const plc_norm_desc* d, void* stream) { return norm_run(d, true, stream); }
