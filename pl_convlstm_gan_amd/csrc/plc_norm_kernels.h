// Group norm with an activation and, in the same pass, dropout; channels-last tensors.
//
//   m, v      mean and biased variance of x over the pixels and the C/G channels of a group of one sample
//   xh = (x - m) r, r = 1 / sqrt(v + eps);  z = w_c xh + b_c;  y = act(z) * (keep ? scale : 0)
//   backward: dz = dy (keep ? scale : 0) act'(z);  db_c = sum dz;  dw_c = sum dz xh;
//             dx = r (w dz - mean(w dz) - xh mean(w dz xh)), the means over the group
//
// A tensor is a set of V-channel units: unit u of pixel p of sample n lies at n * img + u * us + p * ps (elements).
// That covers [N][HW][C] (us = V, ps = C) and the engine's CB8 ([N][C/8][HW][8]: us = 8 HW, ps = 8).  A workgroup
// takes `ut` neighbouring units of one sample: NHWC as many as make whole rows, CB8 one plane, so that its lanes read
// consecutive memory either way.
#pragma once
#include "plc_layers_common.h"

enum { NORM_ACT_NONE = 0, NORM_ACT_RELU = 1, NORM_ACT_SILU = 2 };

struct NormArgs {
    int N, C, G, HW;
    int cg;                       // C / G
    int U;                        // units of a sample: C / V
    int ut;                       // units of a workgroup; rows of threads: blockDim / ut
    int tiles;                    // workgroups along the units
    int splits, px_split;         // statistics passes: pixel ranges of a sample and their length
    int chunks, px_chunk;         // output passes
    int param_blocks;             // backward output pass: leading workgroups that sum dw and db
    long long img, us, ps;
    int act;
    float eps;
    const void *x, *dy;
    const float *w, *b;           // [C] or null (1 and 0)
    void *y, *dx;
    float* stats;                 // [N][G][2]: mean, 1 / sqrt(v + eps)
    float* part;                  // [N][splits][C][2]: forward mean and sum of squared differences, backward sum dz, dz xh
    float *dw, *db;               // [C] or null
    PlcDrop drop;                 // thr == 0: no dropout
    const long long* offset_ptr;  // device: drop.offset, or null
    long long* used_offset;       // device: receives the offset this call used, or null
};

// workgroup -> (sample, tile of units, pixel range): one dimension, so that the number of samples is not limited by a
// grid dimension's 16 bits
struct NormBlock {
    int n, tile, range;
};
__device__ __forceinline__ NormBlock norm_block(const NormArgs& a, unsigned i, int ranges) {
    NormBlock b;
    const unsigned q = i / (unsigned)ranges;
    b.range = (int)(i - q * (unsigned)ranges);
    b.n = (int)(q / (unsigned)a.tiles);
    b.tile = (int)(q - (unsigned)b.n * (unsigned)a.tiles);
    return b;
}

struct NormTid {
    int u, r, rows;               // unit within the workgroup, row, number of rows
    bool on;
};
__device__ __forceinline__ NormTid norm_tid(const NormArgs& a) {
    NormTid t;
    t.rows = blockDim.x / a.ut;
    t.u = threadIdx.x % a.ut;
    t.r = threadIdx.x / a.ut;
    t.on = t.r < t.rows;
    return t;
}

// Sum over the rows of a workgroup of NV values per channel: every thread brings v[NV][V] of its unit, out[k][ut * V]
// (LDS) receives the sums.  Fixed order.  scratch: NV * rows * ut * V floats (LDS); ends with a barrier.
template <int V, int NV>
__device__ __forceinline__ void norm_sum_rows(const NormTid& t, int ut, const float (&v)[NV][V], float* scratch, float* out) {
    const int nch = ut * V, n = t.rows * nch;
    if (t.on) {
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i) scratch[k * n + t.r * nch + t.u * V + i] = v[k][i];
    }
    __syncthreads();
    for (int half = t.rows; half > 1;) {
        const int lower = (half + 1) / 2;
        for (int i = threadIdx.x; i < (half - lower) * nch; i += blockDim.x)
#pragma unroll
            for (int k = 0; k < NV; ++k) scratch[k * n + i] += scratch[k * n + i + lower * nch];
        __syncthreads();
        half = lower;
    }
    for (int i = threadIdx.x; i < nch; i += blockDim.x)
#pragma unroll
        for (int k = 0; k < NV; ++k) out[k * nch + i] = scratch[k * n + i];
    __syncthreads();
}

// ---- forward, first pass: per channel of a pixel range, mean and sum of squared differences from it ------------
// Blocks of NORM_P pixels are reduced around their own mean and merged by the parallel form of the variance
// (Chan, Golub, LeVeque 1983): sums of squares around 0 would cancel where the mean is far from 0.
constexpr int NORM_P = 4;

template <class T, int V>
__global__ __launch_bounds__(256) void plc_norm_stats_kernel(NormArgs a) {
    extern __shared__ __align__(16) float lds[];
    const NormTid t = norm_tid(a);
    const NormBlock blk = norm_block(a, blockIdx.x, a.splits);
    const int n = blk.n, u0 = blk.tile * a.ut;
    const int nu = a.U - u0 < a.ut ? a.U - u0 : a.ut;
    const int p0 = blk.range * a.px_split, p1 = p0 + a.px_split < a.HW ? p0 + a.px_split : a.HW;
    const T* x = (const T*)a.x + n * a.img + (long long)(u0 + t.u) * a.us;
    float mean[V], m2[V], count = 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) mean[i] = m2[i] = 0.0f;
    if (t.on && t.u < nu) {
        for (int p = p0 + t.r; p < p1; p += NORM_P * t.rows) {
            PlcVec<T, V> raw[NORM_P];
#pragma unroll
            for (int j = 0; j < NORM_P; ++j)
                if (p + j * t.rows < p1) raw[j] = plc_load<T, V>(x + (long long)(p + j * t.rows) * a.ps);
            const int m = min(NORM_P, (p1 - p + t.rows - 1) / t.rows);
            const float inv = 1.0f / (float)m, frac = (float)m / (count + (float)m), cross = count * frac;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                float s = 0.0f, q = 0.0f;
#pragma unroll
                for (int j = 0; j < NORM_P; ++j) s += j < m ? (float)raw[j].e[i] : 0.0f;
                const float c = s * inv;
#pragma unroll
                for (int j = 0; j < NORM_P; ++j) {
                    const float d = j < m ? (float)raw[j].e[i] - c : 0.0f;
                    q = __builtin_fmaf(d, d, q);
                }
                const float delta = c - mean[i];
                mean[i] = __builtin_fmaf(delta, frac, mean[i]);
                m2[i] += __builtin_fmaf(delta * delta, cross, q);
            }
            count += (float)m;
        }
    }
    // the rows of the workgroup: mean = sum n_r mean_r / n, then sum of m2_r + n_r (mean_r - mean)^2
    const int nch = a.ut * V, total = p1 - p0;
    float* sums = lds;
    float* scratch = lds + 2 * nch;
    float v[1][V];
#pragma unroll
    for (int i = 0; i < V; ++i) v[0][i] = count * mean[i];
    norm_sum_rows<V, 1>(t, a.ut, v, scratch, sums);
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const float d = t.on ? mean[i] - sums[t.u * V + i] / (float)total : 0.0f;
        v[0][i] = __builtin_fmaf(count * d, d, m2[i]);
    }
    norm_sum_rows<V, 1>(t, a.ut, v, scratch, sums + nch);
    float* part = a.part + (((long long)n * a.splits + blk.range) * a.C + (long long)u0 * V) * 2;
    for (int i = threadIdx.x; i < nu * V; i += blockDim.x) {
        part[2 * i] = sums[i] / (float)total;
        part[2 * i + 1] = sums[nch + i];
    }
}

// ---- the groups that a workgroup's channels touch: mean and r from the partials, into LDS -----------------------
// st[2 g'], g' counted from the first group of the workgroup.  One wave per group, lanes over (split, channel).
__device__ __forceinline__ float norm_wave_sum(float v) {
#pragma unroll
    for (int m = 32; m > 0; m >>= 1) v += __shfl_xor(v, m);
    return v;
}

__device__ __forceinline__ void norm_group_stats(const NormArgs& a, int n, int c0, int c1, float* st, bool keep) {
    const int g0 = c0 / a.cg, g1 = (c1 - 1) / a.cg;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, waves = blockDim.x >> 6;
    const long long items = (long long)a.splits * a.cg;
    const float whole = (float)a.px_split, last = (float)(a.HW - (long long)(a.splits - 1) * a.px_split);
    for (int g = g0 + wave; g <= g1; g += waves) {
        const float* part = a.part + ((long long)n * a.splits * a.C + (long long)g * a.cg) * 2;
        float s = 0.0f;
        for (long long i = lane; i < items; i += 64) {
            const long long sp = i / a.cg, c = i - sp * a.cg;
            s = __builtin_fmaf(sp == a.splits - 1 ? last : whole, part[(sp * a.C + c) * 2], s);
        }
        const float m = (float)a.HW * (float)a.cg, mean = norm_wave_sum(s) / m;
        float q = 0.0f;
        for (long long i = lane; i < items; i += 64) {
            const long long sp = i / a.cg, c = i - sp * a.cg;
            const float d = part[(sp * a.C + c) * 2] - mean;
            q += part[(sp * a.C + c) * 2 + 1] + (sp == a.splits - 1 ? last : whole) * d * d;
        }
        const float var = norm_wave_sum(q) / m, r = 1.0f / sqrtf(var + a.eps);
        if (lane == 0) {
            st[2 * (g - g0)] = mean;
            st[2 * (g - g0) + 1] = r;
            if (keep) {
                a.stats[((long long)n * a.G + g) * 2] = mean;
                a.stats[((long long)n * a.G + g) * 2 + 1] = r;
            }
        }
    }
    __syncthreads();
}

__device__ __forceinline__ float norm_act(float z, int act) {
    if (act == NORM_ACT_RELU) return z > 0.0f ? z : (z != z ? z : 0.0f);
    if (act == NORM_ACT_SILU) {
        float s, q;
        plc_sigmoid_pair(z, s, q);
        return z * s;
    }
    return z;
}
// act'(z); ReLU's is 0 at 0
__device__ __forceinline__ float norm_act_slope(float z, int act) {
    if (act == NORM_ACT_RELU) return z > 0.0f ? 1.0f : (z != z ? z : 0.0f);
    if (act == NORM_ACT_SILU) {
        float s, q;
        plc_sigmoid_pair(z, s, q);
        return __builtin_fmaf(z * s, q, s);
    }
    return 1.0f;
}

__device__ __forceinline__ PlcDrop norm_drop(const NormArgs& a) {
    PlcDrop d = a.drop;
    if (d.thr && a.offset_ptr) d.offset = (uint64_t)*a.offset_ptr;
    return d;
}

// (elements are counted in [N][HW][C] order whatever the layout, so that one seed gives one mask)
template <int V>
__device__ __forceinline__ uint32_t norm_keep(const NormArgs& a, const PlcDrop& d, int n, int p, int u) {
    return plc_keep_bits<V>(d, ((uint64_t)n * a.HW + p) * a.C + (uint64_t)u * V);
}

// per-channel constants of a thread's unit: group mean, r, weight, bias
template <int V>
struct NormUnit {
    float mean[V], r[V], w[V], b[V];
};
template <int V>
__device__ __forceinline__ void norm_unit(const NormArgs& a, int c0, int c, const float* st, NormUnit<V>& k) {
    const int g0 = c0 / a.cg;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int g = (c + i) / a.cg - g0;
        k.mean[i] = st[2 * g];
        k.r[i] = st[2 * g + 1];
        k.w[i] = a.w ? a.w[c + i] : 1.0f;
        k.b[i] = a.b ? a.b[c + i] : 0.0f;
    }
}

// ---- forward, second pass ---------------------------------------------------------------------------------------
template <class T, int V>
__global__ __launch_bounds__(256) void plc_norm_fwd_kernel(NormArgs a) {
    extern __shared__ __align__(16) float lds[];
    const NormTid t = norm_tid(a);
    const NormBlock blk = norm_block(a, blockIdx.x, a.chunks);
    const int n = blk.n, u0 = blk.tile * a.ut;
    const int nu = a.U - u0 < a.ut ? a.U - u0 : a.ut;
    norm_group_stats(a, n, u0 * V, (u0 + nu) * V, lds, blk.range == 0);
    const PlcDrop drop = norm_drop(a);
    if (a.used_offset && blockIdx.x == 0 && threadIdx.x == 0) *a.used_offset = (long long)drop.offset;
    if (!t.on || t.u >= nu) return;
    NormUnit<V> k;
    norm_unit<V>(a, u0 * V, (u0 + t.u) * V, lds, k);
    const long long at = n * a.img + (long long)(u0 + t.u) * a.us;
    const T* x = (const T*)a.x + at;
    T* y = (T*)a.y + at;
    const int p0 = blk.range * a.px_chunk, p1 = p0 + a.px_chunk < a.HW ? p0 + a.px_chunk : a.HW;
    for (int p = p0 + t.r; p < p1; p += NORM_P * t.rows) {
        PlcVec<T, V> raw[NORM_P];
#pragma unroll
        for (int j = 0; j < NORM_P; ++j)
            if (p + j * t.rows < p1) raw[j] = plc_load<T, V>(x + (long long)(p + j * t.rows) * a.ps);
#pragma unroll
        for (int j = 0; j < NORM_P; ++j) {
            const int pj = p + j * t.rows;
            if (pj >= p1) break;
            const uint32_t keep = drop.thr ? norm_keep<V>(a, drop, n, pj, u0 + t.u) : 0;
            float o[V];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float z = __builtin_fmaf(((float)raw[j].e[i] - k.mean[i]) * k.r[i], k.w[i], k.b[i]);
                o[i] = norm_act(z, a.act);
                if (drop.thr) o[i] = (keep >> i) & 1 ? o[i] * drop.scale : 0.0f;
            }
            plc_store<T, V>(y + (long long)pj * a.ps, plc_from_float<T, V>(o));
        }
    }
}

// ---- backward, first pass: per channel of a pixel range, sum dz and sum dz xh -----------------------------------
template <class T, int V>
__device__ __forceinline__ void norm_dz(const NormArgs& a, const NormUnit<V>& k, const PlcDrop& drop, int n, int p, int u,
                                        const PlcVec<T, V>& xr, const PlcVec<T, V>& gr, float (&xh)[V], float (&dz)[V]) {
    const uint32_t keep = drop.thr ? norm_keep<V>(a, drop, n, p, u) : 0;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        xh[i] = ((float)xr.e[i] - k.mean[i]) * k.r[i];
        const float z = __builtin_fmaf(xh[i], k.w[i], k.b[i]);
        float g = (float)gr.e[i];
        if (drop.thr) g = (keep >> i) & 1 ? g * drop.scale : 0.0f;
        dz[i] = a.act == NORM_ACT_NONE ? g : g * norm_act_slope(z, a.act);
    }
}

__device__ __forceinline__ void norm_load_stats(const NormArgs& a, int n, int c0, int c1, float* st) {
    const int g0 = c0 / a.cg, g1 = (c1 - 1) / a.cg;
    for (int i = threadIdx.x; i < 2 * (g1 - g0 + 1); i += blockDim.x) st[i] = a.stats[((long long)n * a.G + g0) * 2 + i];
    __syncthreads();
}

template <class T, int V>
__global__ __launch_bounds__(256) void plc_norm_bwd_sums_kernel(NormArgs a) {
    extern __shared__ __align__(16) float lds[];
    const NormTid t = norm_tid(a);
    const NormBlock blk = norm_block(a, blockIdx.x, a.splits);
    const int n = blk.n, u0 = blk.tile * a.ut;
    const int nu = a.U - u0 < a.ut ? a.U - u0 : a.ut, nch = a.ut * V;
    norm_load_stats(a, n, u0 * V, (u0 + nu) * V, lds);
    const PlcDrop drop = norm_drop(a);
    float v[2][V];
#pragma unroll
    for (int i = 0; i < V; ++i) v[0][i] = v[1][i] = 0.0f;
    const int p0 = blk.range * a.px_split, p1 = p0 + a.px_split < a.HW ? p0 + a.px_split : a.HW;
    if (t.on && t.u < nu) {
        NormUnit<V> k;
        norm_unit<V>(a, u0 * V, (u0 + t.u) * V, lds, k);
        const long long at = n * a.img + (long long)(u0 + t.u) * a.us;
        const T *x = (const T*)a.x + at, *dy = (const T*)a.dy + at;
        for (int p = p0 + t.r; p < p1; p += NORM_P * t.rows) {
            PlcVec<T, V> xr[NORM_P], gr[NORM_P];
#pragma unroll
            for (int j = 0; j < NORM_P; ++j)
                if (p + j * t.rows < p1) {
                    xr[j] = plc_load<T, V>(x + (long long)(p + j * t.rows) * a.ps);
                    gr[j] = plc_load<T, V>(dy + (long long)(p + j * t.rows) * a.ps);
                }
#pragma unroll
            for (int j = 0; j < NORM_P; ++j) {
                if (p + j * t.rows >= p1) break;
                float xh[V], dz[V];
                norm_dz<T, V>(a, k, drop, n, p + j * t.rows, u0 + t.u, xr[j], gr[j], xh, dz);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    v[0][i] += dz[i];
                    v[1][i] = __builtin_fmaf(dz[i], xh[i], v[1][i]);
                }
            }
        }
    }
    __syncthreads();          // (the statistics in LDS make room for the sums)
    float* sums = lds;
    norm_sum_rows<V, 2>(t, a.ut, v, lds + 2 * nch, sums);
    float* part = a.part + (((long long)n * a.splits + blk.range) * a.C + (long long)u0 * V) * 2;
    for (int i = threadIdx.x; i < nu * V; i += blockDim.x) {
        part[2 * i] = sums[i];
        part[2 * i + 1] = sums[nch + i];
    }
}

// ---- backward, second pass: dx; the leading workgroups sum dw and db over samples and ranges -------------------
// dw, db: 16 channels per workgroup, 16 threads each; the sums over many samples run in 64 bits.
constexpr int NORM_PARAM_CH = 16;

__device__ __forceinline__ void norm_param_block(const NormArgs& a, int block, double* scratch) {
    const int c = block * NORM_PARAM_CH + (threadIdx.x & 15), row = threadIdx.x >> 4, rows = blockDim.x >> 4;
    double sb = 0.0, sw = 0.0;
    if (c < a.C)
        for (long long i = row; i < (long long)a.N * a.splits; i += rows) {
            sb += (double)a.part[(i * a.C + c) * 2];
            sw += (double)a.part[(i * a.C + c) * 2 + 1];
        }
    scratch[threadIdx.x] = sb;
    scratch[blockDim.x + threadIdx.x] = sw;
    __syncthreads();
    if (row == 0 && c < a.C) {
        for (int i = 1; i < rows; ++i) {
            sb += scratch[i * 16 + threadIdx.x];
            sw += scratch[blockDim.x + i * 16 + threadIdx.x];
        }
        if (a.db) a.db[c] = (float)sb;
        if (a.dw) a.dw[c] = (float)sw;
    }
}

template <class T, int V>
__global__ __launch_bounds__(256) void plc_norm_bwd_kernel(NormArgs a) {
    extern __shared__ __align__(16) float lds[];
    if ((int)blockIdx.x < a.param_blocks) {
        norm_param_block(a, blockIdx.x, (double*)lds);
        return;
    }
    const NormTid t = norm_tid(a);
    const NormBlock blk = norm_block(a, blockIdx.x - a.param_blocks, a.chunks);
    const int n = blk.n, u0 = blk.tile * a.ut;
    const int nu = a.U - u0 < a.ut ? a.U - u0 : a.ut;
    // means over the group of w dz and w dz xh: one wave per group
    const int g0 = u0 * V / a.cg, g1 = ((u0 + nu) * V - 1) / a.cg;
    float* st = lds;
    float* means = lds + 2 * (g1 - g0 + 1);
    {
        const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, waves = blockDim.x >> 6;
        const long long items = (long long)a.splits * a.cg;
        for (int g = g0 + wave; g <= g1; g += waves) {
            float s0 = 0.0f, s1 = 0.0f;
            for (long long i = lane; i < items; i += 64) {
                const long long sp = i / a.cg;
                const int c = g * a.cg + (int)(i - sp * a.cg);
                const float* part = a.part + (((long long)n * a.splits + sp) * a.C + c) * 2;
                const float w = a.w ? a.w[c] : 1.0f;
                s0 = __builtin_fmaf(w, part[0], s0);
                s1 = __builtin_fmaf(w, part[1], s1);
            }
            s0 = norm_wave_sum(s0);
            s1 = norm_wave_sum(s1);
            const float m = (float)a.HW * (float)a.cg;
            if (lane == 0) {
                means[2 * (g - g0)] = s0 / m;
                means[2 * (g - g0) + 1] = s1 / m;
            }
        }
    }
    norm_load_stats(a, n, u0 * V, (u0 + nu) * V, st);       // (ends with a barrier)
    if (!t.on || t.u >= nu) return;
    const PlcDrop drop = norm_drop(a);
    NormUnit<V> k;
    norm_unit<V>(a, u0 * V, (u0 + t.u) * V, st, k);
    float c1[V], c2[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int g = ((u0 + t.u) * V + i) / a.cg - g0;
        c1[i] = means[2 * g];
        c2[i] = means[2 * g + 1];
    }
    const long long at = n * a.img + (long long)(u0 + t.u) * a.us;
    const T *x = (const T*)a.x + at, *dy = (const T*)a.dy + at;
    T* dx = (T*)a.dx + at;
    const int p0 = blk.range * a.px_chunk, p1 = p0 + a.px_chunk < a.HW ? p0 + a.px_chunk : a.HW;
    for (int p = p0 + t.r; p < p1; p += NORM_P * t.rows) {
        PlcVec<T, V> xr[NORM_P], gr[NORM_P];
#pragma unroll
        for (int j = 0; j < NORM_P; ++j)
            if (p + j * t.rows < p1) {
                xr[j] = plc_load<T, V>(x + (long long)(p + j * t.rows) * a.ps);
                gr[j] = plc_load<T, V>(dy + (long long)(p + j * t.rows) * a.ps);
            }
#pragma unroll
        for (int j = 0; j < NORM_P; ++j) {
            if (p + j * t.rows >= p1) break;
            float xh[V], dz[V], o[V];
            norm_dz<T, V>(a, k, drop, n, p + j * t.rows, u0 + t.u, xr[j], gr[j], xh, dz);
#pragma unroll
            for (int i = 0; i < V; ++i) o[i] = k.r[i] * (__builtin_fmaf(k.w[i], dz[i], -c1[i]) - xh[i] * c2[i]);
            plc_store<T, V>(dx + (long long)(p + j * t.rows) * a.ps, plc_from_float<T, V>(o));
        }
    }
}
