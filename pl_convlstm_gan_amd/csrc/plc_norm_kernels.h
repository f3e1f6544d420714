// Group norm with an activation and, in the same pass, dropout; channels-last tensors.
//
//   m, v      mean and biased variance of x over the pixels and the C/G channels of a group of one sample
//   xh = (x - m) r, r = 1 / sqrt(v + eps);  z = w_c xh + b_c;  y = act(z) * (keep ? scale : 0)
//   backward: dz = dy (keep ? scale : 0) act'(z);  db_c = sum dz;  dw_c = sum dz xh;
//             dx = r (w dz - mean(w dz) - xh mean(w dz xh)), the means over the group
//
// A tensor is a set of V-channel units of at most 16 bytes: unit u of pixel p of sample n lies at n * img + u * us + p * ps
// (elements).  That covers [N][HW][C] (us = V, ps = C) and the engine's CB8 ([N][C/8][HW][8]: us = 8 HW, ps = 8).
// A workgroup takes a tile of neighbouring units that holds whole groups (a group wider than a tile: a part of one) and
// runs with its lanes along the memory's fast direction, units first in NHWC, pixels first in CB8.
//
// Two forms.  Resident: the tile's pixels of a sample stay in the registers of one workgroup between the statistics and
// the output, one launch.  Split: a first launch writes partial sums over ranges of pixels, the second adds them up
// (every workgroup for its own groups) and makes the output, reading its inputs a second time.
//
// What bounds it: memory.  40 samples of 256 x 256 x 32 bf16, forward: statistics 33.9 us (168 MB: 5.0 TB/s), output 51.3
// (336 MB: 6.5 TB/s), where one copy of the tensor would take 64; the second reading is the price of a sum over a sample that no
// workgroup holds.  Joining the workgroups of a sample inside one launch (partial sums exchanged through memory) read once and
// was slower, 157 us, as was going through the tensor in chunks of samples that fit the caches (113 to 182).
// 80 samples of 128 x 128 x 32 with silu and dropout: 20.1 + 43.4 us forward, 56.0 + 54.1 backward; there the generator (ten
// rounds per eight elements) and the exponential cost as much as the memory.
// Resident: 5 x 15 x 12 x 32 fp32 4.2 us forward, one launch of 40 workgroups of a wave, all latency; 8 x 32 x 32 x 512 fp16 9.5 us
// forward (17 MB: 1.8 TB/s) and 15 + 4 backward, the last a launch of its own for dw and db, which are sums over samples that
// different workgroups hold.
// Narrow units (a C without a common factor with the vector) cost the generator, which is called per unit: 40 x 256 x 256 bf16 with
// dropout, forward/backward, 32 channels 96/163 us, 30 (units of two) 165/279, 31 (of one) 294/515; without it 87/147, 87/179, 105/200.
// Many groups cost the split form's joining of the partial sums, which every workgroup does for all groups of its tile:
// 4 x 128 x 128 x 512 bf16 61/77 us with 32 groups, 405/265 with 512.
#pragma once
#include "plc_layers_common.h"

enum { NORM_ACT_NONE = 0, NORM_ACT_RELU = 1, NORM_ACT_SILU = 2 };

struct NormArgs {
    int N, C, G, HW;
    int cg;                       // C / G
    int U;                        // units of a sample: C / V
    int ut;                       // units of a tile at most
    int parts;                    // 1: a tile holds whole groups; else: tiles of one group
    int gu;                       // parts > 1: units of a group
    int tiles;                    // of a sample
    int splits, px_split;         // pixel ranges of a sample and their length
    int px_first;                 // lanes run along pixels (CB8)
    int param_blocks;             // backward output pass: leading workgroups that sum dw and db
    long long img, us, ps;
    int act;
    float eps;
    const void *x, *dy;
    const float *w, *b;           // [C] or null (1 and 0)
    void *y, *dx;
    float* stats;                 // [N][G][2]: mean, 1 / sqrt(v + eps)
    float* part_g;                // [N][G][splits * parts][2]: forward mean and sum of squared differences, backward sums of w dz, w dz xh
    float* part_c;                // backward: [N * splits][C][2]: sums of dz, dz xh
    float *dw, *db;               // [C] or null
    PlcDrop drop;                 // thr == 0: no dropout
    const long long* offset_ptr;  // device: drop.offset, or null
    long long* used_offset;       // device: receives the offset this call used, or null
};

// workgroup -> (sample, tile, pixel range): one dimension, so that the number of samples is not limited by a grid
// dimension's 16 bits
struct NormBlock {
    int n, range;
    int u0, nu;                   // the tile's units
    int g0, ng;                   // its groups
    int part;
};
template <int V>
__device__ __forceinline__ NormBlock norm_block(const NormArgs& a, unsigned i, int ranges) {
    NormBlock b;
    const unsigned q = i / (unsigned)ranges;
    b.range = (int)(i - q * (unsigned)ranges);
    b.n = (int)(q / (unsigned)a.tiles);
    const int tile = (int)(q - (unsigned)b.n * (unsigned)a.tiles);
    if (a.parts == 1) {
        b.part = 0;
        b.u0 = tile * a.ut;
        b.nu = min(a.ut, a.U - b.u0);
        b.g0 = b.u0 * V / a.cg;
        b.ng = b.nu * V / a.cg;
    } else {
        b.g0 = tile / a.parts;
        b.ng = 1;
        b.part = tile - b.g0 * a.parts;
        b.u0 = b.g0 * a.gu + b.part * a.ut;
        b.nu = min(a.ut, a.gu - b.part * a.ut);
    }
    return b;
}

// thread -> (unit of the tile, row): a row is one pixel of a round, and threads beyond whole rows are idle
struct NormTid {
    int u, r, rows;
    bool on;
};
__device__ __forceinline__ NormTid norm_tid(const NormArgs& a, const NormBlock& b) {
    NormTid t;
    t.rows = blockDim.x / b.nu;
    t.u = a.px_first ? threadIdx.x / t.rows : threadIdx.x % b.nu;
    t.r = a.px_first ? threadIdx.x % t.rows : threadIdx.x / b.nu;
    t.on = t.u < b.nu && t.r < t.rows;
    return t;
}

// ---- sums over lanes ----------------------------------------------------------------------------------------------
// Lane shifts inside the vector unit: shuffles go through LDS, at about ten times the latency, and every workgroup needs a few
// of these before it can do anything else.
template <int CTRL, int ROWS>
__device__ __forceinline__ float norm_lane_add(float v) {
    const int moved = __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, ROWS, 0xf, false);
    return v + __builtin_bit_cast(float, moved);
}
// sum of the lanes that agree modulo NU (a power of two up to 16), in every lane
template <int NU>
__device__ __forceinline__ float norm_lane_sum(float v) {
    if (NU <= 8) v = norm_lane_add<0x128, 0xf>(v);      // row_ror:8, 4, 2, 1: rotations within 16 lanes
    if (NU <= 4) v = norm_lane_add<0x124, 0xf>(v);
    if (NU <= 2) v = norm_lane_add<0x122, 0xf>(v);
    if (NU <= 1) v = norm_lane_add<0x121, 0xf>(v);
    // rows of 16: v_permlane16_swap of a value with itself leaves (rows 0 0 2 2, rows 1 1 3 3), v_permlane32_swap the halves
    // (the results go through scalars: a bit cast of a vector's element reads element 0)
    const unsigned x = __builtin_bit_cast(unsigned, v);
    const auto p = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    const unsigned p0 = p[0], p1 = p[1];
    v = __builtin_bit_cast(float, p0) + __builtin_bit_cast(float, p1);
    const unsigned y = __builtin_bit_cast(unsigned, v);
    const auto q = __builtin_amdgcn_permlane32_swap(y, y, false, false);
    const unsigned q0 = q[0], q1 = q[1];
    return __builtin_bit_cast(float, q0) + __builtin_bit_cast(float, q1);
}
__device__ __forceinline__ float norm_wave_sum(float v) { return norm_lane_sum<1>(v); }

// sum over a workgroup of up to 16 waves, in every thread; scratch: 16 floats of LDS that nothing else uses; one barrier
__device__ __forceinline__ float norm_block_sum(float v, float* scratch) {
    v = norm_wave_sum(v);
    if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = v;
    __syncthreads();
    float s = 0.0f;
    for (int w = 0; w < (int)(blockDim.x >> 6); ++w) s += scratch[w];
    return s;
}

// Sums over the rows where the lanes of a wave that hold one unit are those that agree modulo nu (NHWC rows of 1, 2, 4, 8 or 16 units;
// CB8 tiles of one): added across the lanes, then one value per wave.  Three barriers and no more LDS than the result times the
// number of waves; the general form below has five (three where a channel is one thread's) and moves every value through LDS.
template <int V, int NV, int NU>
__device__ __forceinline__ void norm_sum_waves(const float (&v)[NV][V], float* scratch, float* out) {
    constexpr int nch = NU * V;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, waves = blockDim.x >> 6;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float s = norm_lane_sum<NU>(v[k][i]);
            if (lane < NU) scratch[(wave * NV + k) * nch + lane * V + i] = s;
        }
    __syncthreads();
    for (int c = threadIdx.x; c < NV * nch; c += blockDim.x) {
        float s = 0.0f;
        for (int w = 0; w < waves; ++w) s += scratch[w * NV * nch + c];
        out[c] = s;
    }
    __syncthreads();
}

// ---- sums over the rows of a workgroup --------------------------------------------------------------------------
// Every thread brings NV values per channel of its unit; out[k * nch + channel of the tile] (LDS) receives their sums over
// the rows, in a fixed order: a thread per (channel, share of the rows), then one per channel.  Scratch: NV * V * (threads +
// tile units) floats, padded so that the lanes of a wave read different banks.  Begins and ends with a barrier.
template <int V, int NV>
__device__ __forceinline__ void norm_sum_rows(const NormTid& t, bool px_first, int nu, const float (&v)[NV][V], float* scratch, float* out) {
    if (nu == 1) return norm_sum_waves<V, NV, 1>(v, scratch, out);
    if (!px_first) {
        if (nu == 2) return norm_sum_waves<V, NV, 2>(v, scratch, out);
        if (nu == 4) return norm_sum_waves<V, NV, 4>(v, scratch, out);
        if (nu == 8) return norm_sum_waves<V, NV, 8>(v, scratch, out);
        if (nu == 16) return norm_sum_waves<V, NV, 16>(v, scratch, out);
    }
    const int nch = nu * V, pitch = blockDim.x + nu;
    __syncthreads();
    if (t.on) {
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i) scratch[(k * V + i) * pitch + t.r * nu + t.u] = v[k][i];
    }
    __syncthreads();
    const int shares = max(1, min(t.rows, (int)blockDim.x / nch));
    float s[NV];
    for (int base = 0; base < nch * shares; base += blockDim.x) {            // (one round unless the tile has more channels than threads)
        const int id = base + threadIdx.x, ch = id % nch, share = id / nch;
        const bool mine = id < nch * shares;
        const int i = ch / nu, u = ch - i * nu;
#pragma unroll
        for (int k = 0; k < NV; ++k) s[k] = 0.0f;
        if (mine)
#pragma unroll 8
            for (int r = share; r < t.rows; r += shares)
#pragma unroll
                for (int k = 0; k < NV; ++k) s[k] += scratch[(k * V + i) * pitch + r * nu + u];
        if (shares == 1) {
            if (mine)
#pragma unroll
                for (int k = 0; k < NV; ++k) out[k * nch + u * V + i] = s[k];
        } else {
            __syncthreads();
            if (mine)
#pragma unroll
                for (int k = 0; k < NV; ++k) scratch[k * (nch * shares) + id] = s[k];
            __syncthreads();
            for (int c = threadIdx.x; c < nch; c += blockDim.x) {
                const int ci = c / nu, cu = c - ci * nu;
#pragma unroll
                for (int k = 0; k < NV; ++k) {
                    float q = 0.0f;
#pragma unroll 8
                    for (int h = 0; h < shares; ++h) q += scratch[k * (nch * shares) + h * nch + c];
                    out[k * nch + cu * V + ci] = q;
                }
            }
        }
    }
    __syncthreads();
}
// floats of LDS for the above: out and scratch
__host__ __device__ constexpr int norm_lds_floats(int threads, int nu, int V, int NV) { return NV * nu * V + NV * V * (threads + nu); }

// ---- activation -------------------------------------------------------------------------------------------------
__device__ __forceinline__ float norm_sigmoid(float z) {
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.44269504088896341f * z));
}
// What a kernel is compiled for: FORM = activation + 3 * dropout, or -1, which asks the arguments for every element (the
// vector widths that few shapes take).  Compiled in, an element has no branch.
template <int FORM>
__device__ __forceinline__ int norm_form_act(const NormArgs& a) { return FORM >= 0 ? FORM % 3 : a.act; }
template <int FORM>
__device__ __forceinline__ bool norm_form_drop(const NormArgs& a) { return FORM >= 0 ? FORM >= 3 : a.drop.thr != 0; }

__device__ __forceinline__ float norm_act(float z, int act) {
    if (act == NORM_ACT_RELU) return z > 0.0f ? z : (z != z ? z : 0.0f);
    if (act == NORM_ACT_SILU) return z * norm_sigmoid(z);
    return z;
}
// silu'(z)
__device__ __forceinline__ float norm_silu_slope(float z) {
    const float s = norm_sigmoid(z);
    return __builtin_fmaf(z * s, 1.0f - s, s);
}

template <int FORM>
__device__ __forceinline__ PlcDrop norm_drop(const NormArgs& a) {
    PlcDrop d = a.drop;
    if (norm_form_drop<FORM>(a) && a.offset_ptr) d.offset = (uint64_t)*a.offset_ptr;
    return d;
}
// (elements are counted in [N][HW][C] order whatever the layout, so that one seed gives one mask)
template <int V>
__device__ __forceinline__ uint32_t norm_keep(const NormArgs& a, const PlcDrop& d, int n, int p, int u) {
    return plc_keep_bits<V>(d, ((uint64_t)n * a.HW + p) * a.C + (uint64_t)u * V);
}

// per-channel constants of a thread's unit.  The difference x - mean is formed first (the mean may be many deviations from
// 0), r and the weight are one factor.
template <int V>
struct NormUnit {
    float mean[V], r[V], rw[V], b[V];
};
template <int V>
__device__ __forceinline__ void norm_unit(const NormArgs& a, const NormBlock& blk, int u, const float* st, NormUnit<V>& k) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int c = (blk.u0 + u) * V + i, g = c / a.cg - blk.g0;
        k.mean[i] = st[2 * g];
        k.r[i] = st[2 * g + 1];
        k.rw[i] = k.r[i] * (a.w ? a.w[c] : 1.0f);
        k.b[i] = a.b ? a.b[c] : 0.0f;
    }
}

template <class T, int V, int FORM>
__device__ __forceinline__ PlcVec<T, V> norm_out(const NormArgs& a, const NormUnit<V>& k, const PlcDrop& drop, int n, int p, int u,
                                                 const PlcVec<T, V>& x) {
    const bool drops = norm_form_drop<FORM>(a);
    const int act = norm_form_act<FORM>(a);
    const uint32_t keep = drops ? norm_keep<V>(a, drop, n, p, u) : 0;
    float o[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        o[i] = norm_act(__builtin_fmaf(x.get(i) - k.mean[i], k.rw[i], k.b[i]), act);
        if (drops) o[i] = (keep >> i) & 1 ? o[i] * drop.scale : 0.0f;
    }
    return plc_from_float<T, V>(o);
}

// d = x - mean and dz of one unit
template <class T, int V, int FORM>
__device__ __forceinline__ void norm_dz(const NormArgs& a, const NormUnit<V>& k, const PlcDrop& drop, int n, int p, int u,
                                        const PlcVec<T, V>& xr, const PlcVec<T, V>& gr, float (&d)[V], float (&dz)[V]) {
    const bool drops = norm_form_drop<FORM>(a);
    const int act = norm_form_act<FORM>(a);
    const uint32_t keep = drops ? norm_keep<V>(a, drop, n, p, u) : 0;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        d[i] = xr.get(i) - k.mean[i];
        const float z = __builtin_fmaf(d[i], k.rw[i], k.b[i]), g = gr.get(i);
        if (act == NORM_ACT_RELU) dz[i] = z > 0.0f ? g : 0.0f;
        else if (act == NORM_ACT_SILU) dz[i] = g * norm_silu_slope(z);
        else dz[i] = g;
        if (drops) dz[i] = (keep >> i) & 1 ? dz[i] * drop.scale : 0.0f;
    }
}

__device__ __forceinline__ void norm_load_stats(const NormArgs& a, const NormBlock& blk, float* st) {
    for (int i = threadIdx.x; i < 2 * blk.ng; i += blockDim.x) st[i] = a.stats[((long long)blk.n * a.G + blk.g0) * 2 + i];
    __syncthreads();
}

// Calls f(first pixel, number of pixels, loaded units) for rounds of P pixels of a thread; whole rounds carry no conditions,
// so that all their loads are in flight at once.
template <class T, int V, int P, int NT, bool STREAM, class F>
__device__ __forceinline__ void norm_rounds(const T* const (&src)[NT], long long ps, int p0, int p1, int rows, F f) {
    PlcVec<T, V> raw[NT][P];
    int p = p0;
    for (; p + (P - 1) * rows < p1; p += P * rows) {
#pragma unroll
        for (int j = 0; j < P; ++j)
#pragma unroll
            for (int k = 0; k < NT; ++k) raw[k][j] = plc_load<T, V, STREAM>(src[k] + (long long)(p + j * rows) * ps);
#pragma unroll
        for (int j = 0; j < P; ++j) {
            PlcVec<T, V> one[NT];
#pragma unroll
            for (int k = 0; k < NT; ++k) one[k] = raw[k][j];
            f(p + j * rows, one);
            // (pixel by pixel: left alone, the compiler works on all of them at once, at twice the registers)
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    if (p < p1) {
#pragma unroll
        for (int j = 0; j < P; ++j)
            if (p + j * rows < p1) {
#pragma unroll
                for (int k = 0; k < NT; ++k) raw[k][j] = plc_load<T, V, STREAM>(src[k] + (long long)(p + j * rows) * ps);
            }
#pragma unroll
        for (int j = 0; j < P; ++j)
            if (p + j * rows < p1) {
                PlcVec<T, V> one[NT];
#pragma unroll
                for (int k = 0; k < NT; ++k) one[k] = raw[k][j];
                f(p + j * rows, one);
                __builtin_amdgcn_sched_barrier(0);
            }
    }
}

// ---- split form, forward, first pass ----------------------------------------------------------------------------
// Per channel of a pixel range, mean and sum of squared differences from it: blocks of NORM_P pixels are reduced around
// their own mean and merged by the parallel form of the variance (Chan, Golub, LeVeque 1983), since sums of squares around 0
// would cancel where the mean is far from 0.  The channels of a group are merged the same way at the end.
constexpr int NORM_P = 8;             // pixels a thread has in flight (forward); half of it for two tensors

template <class T, int V>
__global__ __launch_bounds__(256) void plc_norm_stats_kernel(NormArgs a) {
    extern __shared__ __align__(16) float lds[];
    const NormBlock blk = norm_block<V>(a, blockIdx.x, a.splits);
    const NormTid t = norm_tid(a, blk);
    const int p0 = blk.range * a.px_split, p1 = min(p0 + a.px_split, a.HW);
    const T* x = (const T*)a.x + blk.n * a.img + (long long)(blk.u0 + t.u) * a.us;
    float mean[V], m2[V], count = 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) mean[i] = m2[i] = 0.0f;
    if (t.on) {
        auto merge = [&](int m, const PlcVec<T, V> (&raw)[NORM_P], bool full) {
            const float inv = full ? 1.0f / NORM_P : 1.0f / (float)m, frac = (float)m * __builtin_amdgcn_rcpf(count + (float)m), cross = count * frac;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                float s = 0.0f, q = 0.0f;
#pragma unroll
                for (int j = 0; j < NORM_P; ++j) s += full || j < m ? raw[j].get(i) : 0.0f;
                const float c = s * inv;
#pragma unroll
                for (int j = 0; j < NORM_P; ++j) {
                    const float d = full || j < m ? raw[j].get(i) - c : 0.0f;
                    q = __builtin_fmaf(d, d, q);
                }
                const float delta = c - mean[i];
                mean[i] = __builtin_fmaf(delta, frac, mean[i]);
                m2[i] += __builtin_fmaf(delta * delta, cross, q);
            }
            count += (float)m;
        };
        int p = p0 + t.r;
        for (; p + (NORM_P - 1) * t.rows < p1; p += NORM_P * t.rows) {
            PlcVec<T, V> raw[NORM_P];
#pragma unroll
            for (int j = 0; j < NORM_P; ++j) raw[j] = plc_load<T, V>(x + (long long)(p + j * t.rows) * a.ps);
            merge(NORM_P, raw, true);
        }
        if (p < p1) {
            PlcVec<T, V> raw[NORM_P];
#pragma unroll
            for (int j = 0; j < NORM_P; ++j)
                if (p + j * t.rows < p1) raw[j] = plc_load<T, V>(x + (long long)(p + j * t.rows) * a.ps);
            merge((p1 - p + t.rows - 1) / t.rows, raw, false);
        }
    }
    // The rows of the workgroup, around the mean of the first row (the pivot is one of the means that are merged, so its
    // own difference counts in the result and the subtraction loses at most a factor of the number of rows).
    const int nch = blk.nu * V;
    float* pivot = lds;
    float* sums = lds + nch;
    float* scratch = sums + 2 * nch;
    if (t.on && t.r == 0)
#pragma unroll
        for (int i = 0; i < V; ++i) pivot[t.u * V + i] = mean[i];
    __syncthreads();
    float v[2][V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const float d = t.on && count > 0.0f ? mean[i] - pivot[t.u * V + i] : 0.0f;
        v[0][i] = count * d;
        v[1][i] = __builtin_fmaf(count * d, d, m2[i]);
    }
    norm_sum_rows<V, 2>(t, a.px_first, blk.nu, v, scratch, sums);
    // channels -> groups, one wave per group
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, waves = blockDim.x >> 6, entries = a.splits * a.parts;
    const int width = a.parts == 1 ? a.cg : nch;
    const float px = (float)(p1 - p0), inv_px = 1.0f / px, inv_w = 1.0f / (float)width;
    for (int g = wave; g < blk.ng; g += waves) {
        float s = 0.0f;
        for (int c = lane; c < width; c += 64) s += pivot[g * a.cg + c] + sums[g * a.cg + c] * inv_px;
        const float m = norm_wave_sum(s) * inv_w;
        float q = 0.0f;
        for (int c = lane; c < width; c += 64) {
            const float d0 = sums[g * a.cg + c] * inv_px, d = pivot[g * a.cg + c] + d0 - m;
            q += sums[nch + g * a.cg + c] + px * (d * d - d0 * d0);
        }
        q = norm_wave_sum(q);
        if (lane == 0) {
            float* out = a.part_g + (((long long)blk.n * a.G + blk.g0 + g) * entries + blk.range * a.parts + blk.part) * 2;
            out[0] = m;
            out[1] = fmaxf(q, 0.0f) + (q != q ? q : 0.0f);
        }
    }
}

// pixels times channels of partial sum e of a group
__device__ __forceinline__ float norm_entry_count(const NormArgs& a, int V, int e) {
    const int range = e / a.parts, part = e - range * a.parts;
    const int px = min(a.px_split, a.HW - range * a.px_split);
    const int ch = a.parts == 1 ? a.cg : min(a.ut, a.gu - part * a.ut) * V;
    return (float)px * (float)ch;
}

// ---- split form, forward, second pass ---------------------------------------------------------------------------
// Nothing it touches is needed in the caches afterwards, and what the first pass left of x there is: loads and stores stream.
// 32 channels in 8 groups, both passes together, in brackets with an operator that reads y behind them, against loads and stores that
// stay: bf16 40 x 256 x 256 84.4 (152) us against 104 (162), 12 x 256 x 256 30.0 (47.1) against 31.5 (48.1), 20 x 128 x 128 18.7 (28.1)
// against 20.5 (28.5), 2 x 256 x 256 15.1 (21.2) against 16.0 (21.5), 4 x 128 x 128 14.5 (18.7) both; fp32 2 x 256 x 256 15.4 (22.8)
// against 16.6 (22.7).  (Streaming in the first pass too, 40 x 256 x 256: 93.8 where this took 86.4.)
template <class T, int V, int FORM>
__global__ __launch_bounds__(256) void plc_norm_fwd_kernel(NormArgs a) {
    extern __shared__ __align__(16) float st[];
    const NormBlock blk = norm_block<V>(a, blockIdx.x, a.splits);
    const NormTid t = norm_tid(a, blk);
    {   // the tile's groups: mean and r from the partial sums, one wave per group
        const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, waves = blockDim.x >> 6, entries = a.splits * a.parts;
        const float m = (float)a.HW * (float)a.cg;
        for (int g = wave; g < blk.ng; g += waves) {
            const float* part = a.part_g + ((long long)blk.n * a.G + blk.g0 + g) * entries * 2;
            float s = 0.0f, q = 0.0f;
            for (int e = lane; e < entries; e += 64) s = __builtin_fmaf(norm_entry_count(a, V, e), part[2 * e], s);
            const float mean = norm_wave_sum(s) / m;
            for (int e = lane; e < entries; e += 64) {
                const float d = part[2 * e] - mean;
                q += __builtin_fmaf(norm_entry_count(a, V, e) * d, d, part[2 * e + 1]);
            }
            const float r = 1.0f / sqrtf(norm_wave_sum(q) / m + a.eps);
            if (lane == 0) {
                st[2 * g] = mean;
                st[2 * g + 1] = r;
                if (blk.range == 0 && blk.part == 0) {
                    a.stats[((long long)blk.n * a.G + blk.g0 + g) * 2] = mean;
                    a.stats[((long long)blk.n * a.G + blk.g0 + g) * 2 + 1] = r;
                }
            }
        }
        __syncthreads();
    }
    const PlcDrop drop = norm_drop<FORM>(a);
    if (a.used_offset && blockIdx.x == 0 && threadIdx.x == 0) *a.used_offset = (long long)drop.offset;
    if (!t.on) return;
    NormUnit<V> k;
    norm_unit<V>(a, blk, t.u, st, k);
    const int u = blk.u0 + t.u;
    const long long at = blk.n * a.img + (long long)u * a.us;
    const T* x = (const T*)a.x + at;
    T* y = (T*)a.y + at;
    const int p0 = blk.range * a.px_split, p1 = min(p0 + a.px_split, a.HW);
    const T* const src[1] = {x};
    norm_rounds<T, V, NORM_P, 1, true>(src, a.ps, p0 + t.r, p1, t.rows, [&](int p, const PlcVec<T, V> (&v)[1]) {
        plc_store<T, V, true>(y + (long long)p * a.ps, norm_out<T, V, FORM>(a, k, drop, blk.n, p, u, v[0]));
    });
}

// ---- backward: sums of a tile ------------------------------------------------------------------------------------
// v[0] = sum dz, v[1] = sum dz (x - mean) of a thread -> part_c (per channel) and, per group, the sums of w dz and w dz xh:
// into part_g (split) or as means into LDS (resident)
template <int V>
__device__ __forceinline__ void norm_bwd_reduce(const NormArgs& a, const NormBlock& blk, const NormTid& t, const NormUnit<V>& k,
                                                float (&v)[2][V], float* sums, float* scratch, float* means) {
#pragma unroll
    for (int i = 0; i < V; ++i) v[1][i] *= k.r[i];
    const int nch = blk.nu * V, c0 = blk.u0 * V;
#pragma unroll
    for (int j = 0; j < 2; ++j) {         // (one after the other: half the LDS)
        float one[1][V];
#pragma unroll
        for (int i = 0; i < V; ++i) one[0][i] = v[j][i];
        norm_sum_rows<V, 1>(t, a.px_first, blk.nu, one, scratch, sums + j * nch);
    }
    float* out = a.part_c + (((long long)blk.n * a.splits + blk.range) * a.C + c0) * 2;
    for (int i = threadIdx.x; i < nch; i += blockDim.x) {
        out[2 * i] = sums[i];
        out[2 * i + 1] = sums[nch + i];
    }
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, waves = blockDim.x >> 6, entries = a.splits * a.parts;
    const int width = a.parts == 1 ? a.cg : nch;
    for (int g = wave; g < blk.ng; g += waves) {
        float s0 = 0.0f, s1 = 0.0f;
        for (int c = lane; c < width; c += 64) {
            const float w = a.w ? a.w[c0 + g * a.cg + c] : 1.0f;
            s0 = __builtin_fmaf(w, sums[g * a.cg + c], s0);
            s1 = __builtin_fmaf(w, sums[nch + g * a.cg + c], s1);
        }
        s0 = norm_wave_sum(s0);
        s1 = norm_wave_sum(s1);
        if (lane == 0) {
            if (means) {
                const float m = (float)a.HW * (float)a.cg;
                means[2 * g] = s0 / m;
                means[2 * g + 1] = s1 / m;
            } else {
                float* pg = a.part_g + (((long long)blk.n * a.G + blk.g0 + g) * entries + blk.range * a.parts + blk.part) * 2;
                pg[0] = s0;
                pg[1] = s1;
            }
        }
    }
}

// dx = rw dz - r c1 - (x - mean) r^2 c2
template <int V>
struct NormMeans {
    float k1[V], k2[V];
};
template <int V>
__device__ __forceinline__ void norm_means(const NormArgs& a, const NormBlock& blk, int u, const float* means, const NormUnit<V>& k, NormMeans<V>& q) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int g = ((blk.u0 + u) * V + i) / a.cg - blk.g0;
        q.k1[i] = k.r[i] * means[2 * g];
        q.k2[i] = k.r[i] * k.r[i] * means[2 * g + 1];
    }
}
template <class T, int V>
__device__ __forceinline__ PlcVec<T, V> norm_dx(const NormUnit<V>& k, const NormMeans<V>& q, const float (&d)[V], const float (&dz)[V]) {
    float o[V];
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = __builtin_fmaf(-d[i], q.k2[i], __builtin_fmaf(k.rw[i], dz[i], -q.k1[i]));
    return plc_from_float<T, V>(o);
}

// ---- split form, backward, first pass ----------------------------------------------------------------------------
constexpr int NORM_PB = NORM_P / 2;

template <class T, int V, int FORM>
__global__ __launch_bounds__(256) void plc_norm_bwd_sums_kernel(NormArgs a) {
    extern __shared__ __align__(16) float lds[];
    const NormBlock blk = norm_block<V>(a, blockIdx.x, a.splits);
    const NormTid t = norm_tid(a, blk);
    const int nch = blk.nu * V;
    float* st = lds;
    norm_load_stats(a, blk, st);
    const PlcDrop drop = norm_drop<FORM>(a);
    float v[2][V];
    NormUnit<V> k;
#pragma unroll
    for (int i = 0; i < V; ++i) v[0][i] = v[1][i] = k.r[i] = 0.0f;
    const int p0 = blk.range * a.px_split, p1 = min(p0 + a.px_split, a.HW);
    if (t.on) {
        norm_unit<V>(a, blk, t.u, st, k);
        const int u = blk.u0 + t.u;
        const long long at = blk.n * a.img + (long long)u * a.us;
        const T *x = (const T*)a.x + at, *dy = (const T*)a.dy + at;
        const T* const src[2] = {x, dy};
        norm_rounds<T, V, NORM_PB, 2, false>(src, a.ps, p0 + t.r, p1, t.rows, [&](int p, const PlcVec<T, V> (&q)[2]) {
            float d[V], dz[V];
            norm_dz<T, V, FORM>(a, k, drop, blk.n, p, u, q[0], q[1], d, dz);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                v[0][i] += dz[i];
                v[1][i] = __builtin_fmaf(dz[i], d[i], v[1][i]);
            }
        });
    }
    norm_bwd_reduce<V>(a, blk, t, k, v, lds + 2 * nch, lds + 4 * nch, nullptr);
}

// ---- backward: dw and db from the per-channel sums of samples and ranges ------------------------------------------
// 16 channels per workgroup of 256, 16 threads each; the sums over many samples run in 64 bits.
constexpr int NORM_PARAM_CH = 16;

__device__ __forceinline__ void norm_param_block(const NormArgs& a, int block, double* scratch) {
    const int c = block * NORM_PARAM_CH + (threadIdx.x & 15), row = threadIdx.x >> 4;
    double sb = 0.0, sw = 0.0;
    const long long n = (long long)a.N * a.splits;
    if (c < a.C) {
#pragma unroll 8
        for (long long i = row; i < n; i += 16) {
            const PlcVec<float, 2> q = plc_load<float, 2>(a.part_c + (i * a.C + c) * 2);
            sb += (double)q.get(0);
            sw += (double)q.get(1);
        }
    }
    scratch[threadIdx.x] = sb;
    scratch[256 + threadIdx.x] = sw;
    __syncthreads();
    if (row == 0 && c < a.C) {
        for (int i = 1; i < 16; ++i) {
            sb += scratch[i * 16 + threadIdx.x];
            sw += scratch[256 + i * 16 + threadIdx.x];
        }
        if (a.db) a.db[c] = (float)sb;
        if (a.dw) a.dw[c] = (float)sw;
    }
}
template <class T>        // (T only tells the translation units' copies apart)
__global__ __launch_bounds__(256) void plc_norm_params_kernel(NormArgs a) {
    __shared__ double scratch[512];
    norm_param_block(a, blockIdx.x, scratch);
}

// ---- split form, backward, second pass: dx; the leading workgroups sum dw and db -----------------------------------
// STREAM as in the forward pass, for tensors that the caches do not hold: 40 x 256 x 256 152 us against 174, 80 x 128 x 128 with silu
// 82 against 88; small ones lose by it (2 x 256 x 256 18.3 against 17.6, with a reader of dx behind it 27.2 against 25.1).
template <class T, int V, int FORM, bool STREAM>
__global__ __launch_bounds__(256) void plc_norm_bwd_kernel(NormArgs a) {
    extern __shared__ __align__(16) float lds[];
    if ((int)blockIdx.x < a.param_blocks) {
        norm_param_block(a, blockIdx.x, (double*)lds);
        return;
    }
    const NormBlock blk = norm_block<V>(a, blockIdx.x - a.param_blocks, a.splits);
    const NormTid t = norm_tid(a, blk);
    float* st = lds;
    float* means = lds + 2 * blk.ng;
    {
        const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, waves = blockDim.x >> 6, entries = a.splits * a.parts;
        const float m = (float)a.HW * (float)a.cg;
        for (int g = wave; g < blk.ng; g += waves) {
            const float* part = a.part_g + ((long long)blk.n * a.G + blk.g0 + g) * entries * 2;
            float s0 = 0.0f, s1 = 0.0f;
            for (int e = lane; e < entries; e += 64) {
                s0 += part[2 * e];
                s1 += part[2 * e + 1];
            }
            s0 = norm_wave_sum(s0);
            s1 = norm_wave_sum(s1);
            if (lane == 0) {
                means[2 * g] = s0 / m;
                means[2 * g + 1] = s1 / m;
            }
        }
    }
    norm_load_stats(a, blk, st);       // (ends with a barrier)
    if (!t.on) return;
    const PlcDrop drop = norm_drop<FORM>(a);
    NormUnit<V> k;
    NormMeans<V> q;
    norm_unit<V>(a, blk, t.u, st, k);
    norm_means<V>(a, blk, t.u, means, k, q);
    const int u = blk.u0 + t.u;
    const long long at = blk.n * a.img + (long long)u * a.us;
    const T *x = (const T*)a.x + at, *dy = (const T*)a.dy + at;
    T* dx = (T*)a.dx + at;
    const int p0 = blk.range * a.px_split, p1 = min(p0 + a.px_split, a.HW);
    const T* const src[2] = {x, dy};
    norm_rounds<T, V, NORM_PB, 2, STREAM>(src, a.ps, p0 + t.r, p1, t.rows, [&](int p, const PlcVec<T, V> (&v)[2]) {
        float d[V], dz[V];
        norm_dz<T, V, FORM>(a, k, drop, blk.n, p, u, v[0], v[1], d, dz);
        plc_store<T, V, STREAM>(dx + (long long)p * a.ps, norm_dx<T, V>(k, q, d, dz));
    });
}

// ---- resident form -----------------------------------------------------------------------------------------------
// One workgroup per (sample, tile of whole groups); a thread keeps KU units.  Neighbouring tiles share cache lines, so they
// are given to workgroups of one XCD (workgroups go round the XCDs one by one).
__device__ __forceinline__ unsigned norm_xcd_order(unsigned i, unsigned n) {
    const unsigned per = n / 8, rest = n % 8, x = i % 8;
    return x * per + min(x, rest) + i / 8;
}

template <class T, int V, int FORM, int KU>
__global__ __launch_bounds__(KU == 4 ? 1024 : 512) void plc_norm_fwd_resident_kernel(NormArgs a) {
    extern __shared__ __align__(16) float lds[];
    const NormBlock blk = norm_block<V>(a, norm_xcd_order(blockIdx.x, gridDim.x), 1);
    const NormTid t = norm_tid(a, blk);
    const int nch = blk.nu * V, u = blk.u0 + t.u;
    const long long at = blk.n * a.img + (long long)u * a.us;
    const T* x = (const T*)a.x + at;
    float* st = lds;
    float* sums = lds + 2 * blk.ng;
    float* scratch = sums + nch;
    const PlcDrop drop = norm_drop<FORM>(a);
    if (a.used_offset && blockIdx.x == 0 && threadIdx.x == 0) *a.used_offset = (long long)drop.offset;
    PlcVec<T, V> raw[KU];
#pragma unroll
    for (int j = 0; j < KU; ++j)
        if (t.on && t.r + j * t.rows < a.HW) raw[j] = plc_load<T, V>(x + (long long)(t.r + j * t.rows) * a.ps);
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, waves = blockDim.x >> 6;
    const float inv = 1.0f / ((float)a.HW * (float)a.cg);
    float* const stats = a.stats + ((long long)blk.n * a.G + blk.g0) * 2;
    if (blk.ng == 1) {
        // the tile is one group: one number per thread, not one per channel
        float s = 0.0f, q = 0.0f;
#pragma unroll
        for (int j = 0; j < KU; ++j)
            if (t.on && t.r + j * t.rows < a.HW)
#pragma unroll
                for (int i = 0; i < V; ++i) s += raw[j].get(i);
        const float m = norm_block_sum(s, scratch) * inv;
#pragma unroll
        for (int j = 0; j < KU; ++j)
            if (t.on && t.r + j * t.rows < a.HW)
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float d = raw[j].get(i) - m;
                    q = __builtin_fmaf(d, d, q);
                }
        const float r = 1.0f / sqrtf(norm_block_sum(q, scratch + 16) * inv + a.eps);
        if (threadIdx.x == 0) {
            st[0] = stats[0] = m;
            st[1] = stats[1] = r;
        }
        __syncthreads();
    } else {
        float v[1][V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            v[0][i] = 0.0f;
#pragma unroll
            for (int j = 0; j < KU; ++j)
                if (t.on && t.r + j * t.rows < a.HW) v[0][i] += raw[j].get(i);
        }
        norm_sum_rows<V, 1>(t, a.px_first, blk.nu, v, scratch, sums);
        for (int g = wave; g < blk.ng; g += waves) {
            float s = 0.0f;
            for (int c = lane; c < a.cg; c += 64) s += sums[g * a.cg + c];
            s = norm_wave_sum(s);
            if (lane == 0) st[2 * g] = s * inv;
        }
        __syncthreads();
        float mean[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            mean[i] = t.on ? st[2 * ((u * V + i) / a.cg - blk.g0)] : 0.0f;
            v[0][i] = 0.0f;
#pragma unroll
            for (int j = 0; j < KU; ++j)
                if (t.on && t.r + j * t.rows < a.HW) {
                    const float d = raw[j].get(i) - mean[i];
                    v[0][i] = __builtin_fmaf(d, d, v[0][i]);
                }
        }
        norm_sum_rows<V, 1>(t, a.px_first, blk.nu, v, scratch, sums);
        for (int g = wave; g < blk.ng; g += waves) {
            float s = 0.0f;
            for (int c = lane; c < a.cg; c += 64) s += sums[g * a.cg + c];
            s = norm_wave_sum(s);
            if (lane == 0) {
                const float r = 1.0f / sqrtf(s * inv + a.eps);
                st[2 * g + 1] = r;
                stats[2 * g] = st[2 * g];
                stats[2 * g + 1] = r;
            }
        }
        __syncthreads();
    }
    if (!t.on) return;
    NormUnit<V> k;
    norm_unit<V>(a, blk, t.u, st, k);
    T* y = (T*)a.y + at;
#pragma unroll
    for (int j = 0; j < KU; ++j) {
        const int p = t.r + j * t.rows;
        if (p < a.HW) plc_store<T, V>(y + (long long)p * a.ps, norm_out<T, V, FORM>(a, k, drop, blk.n, p, u, raw[j]));
    }
}

template <class T, int V, int FORM, int KU>
__global__ __launch_bounds__(KU == 4 ? 1024 : 512) void plc_norm_bwd_resident_kernel(NormArgs a) {
    extern __shared__ __align__(16) float lds[];
    const NormBlock blk = norm_block<V>(a, norm_xcd_order(blockIdx.x, gridDim.x), 1);
    const NormTid t = norm_tid(a, blk);
    const int nch = blk.nu * V, u = blk.u0 + t.u;
    const long long at = blk.n * a.img + (long long)u * a.us;
    const T *x = (const T*)a.x + at, *dy = (const T*)a.dy + at;
    float* st = lds;
    float* means = st + 2 * blk.ng;
    float* sums = means + 2 * blk.ng;
    float* scratch = sums + 2 * nch;
    PlcVec<T, V> xr[KU], gr[KU];
#pragma unroll
    for (int j = 0; j < KU; ++j)
        if (t.on && t.r + j * t.rows < a.HW) {
            xr[j] = plc_load<T, V>(x + (long long)(t.r + j * t.rows) * a.ps);
            gr[j] = plc_load<T, V>(dy + (long long)(t.r + j * t.rows) * a.ps);
        }
    norm_load_stats(a, blk, st);
    const PlcDrop drop = norm_drop<FORM>(a);
    float v[2][V];
    NormUnit<V> k;
#pragma unroll
    for (int i = 0; i < V; ++i) v[0][i] = v[1][i] = k.r[i] = 0.0f;
    if (t.on) {
        norm_unit<V>(a, blk, t.u, st, k);
#pragma unroll
        for (int j = 0; j < KU; ++j) {
            const int p = t.r + j * t.rows;
            if (p < a.HW) {
                float d[V], dz[V];
                norm_dz<T, V, FORM>(a, k, drop, blk.n, p, u, xr[j], gr[j], d, dz);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    v[0][i] += dz[i];
                    v[1][i] = __builtin_fmaf(dz[i], d[i], v[1][i]);
                }
            }
        }
    }
    norm_bwd_reduce<V>(a, blk, t, k, v, sums, scratch, means);
    __syncthreads();
    if (!t.on) return;
    NormMeans<V> q;
    norm_means<V>(a, blk, t.u, means, k, q);
    T* dx = (T*)a.dx + at;
#pragma unroll
    for (int j = 0; j < KU; ++j) {
        const int p = t.r + j * t.rows;
        if (p < a.HW) {
            float d[V], dz[V];
            norm_dz<T, V, FORM>(a, k, drop, blk.n, p, u, xr[j], gr[j], d, dz);
            plc_store<T, V>(dx + (long long)p * a.ps, norm_dx<T, V>(k, q, d, dz));
        }
    }
}
