// Gated linear recurrence over time, h_t = s_t h_{t-1} + (1 - s_t) x_t ("coupled") or h_t = s_t h_{t-1} + x_t, with
// s_t = sigmoid(f_t): the gates do not depend on h, so the whole sequence is known before the recurrence starts.
//
// Layout: [B][T][D], D innermost; a lane owns V channels of one sample.  The state is fp32 from the first step to
// the last, whatever the type of x, f and y.
#pragma once
#include "plc_layers_common.h"

// Steps a lane holds in registers at a time: their loads are all requested before the first is used, and the
// backward pass rebuilds the states of one such block from the state in front of it.
constexpr int SCAN_K = 16;

struct ScanArgs {
    int B, T;
    long long D;
    int coupled;
    const void *x, *f, *dy;
    long long x_sb, x_st, f_sb, f_st, dy_sb, dy_st;   // element strides of a sample and of a step
    const float *h0, *dh_last;      // [B][D] or null (zeros)
    const int* lengths;             // [B] or null (all T); taken into 0 .. T
    void *y, *dx, *df;              // [B][T][D]
    float *h_last, *dh0;            // [B][D] or null
    float* states;                  // [B][ceil(T / SCAN_K) - 1][D]: the state in front of block 1, 2, ...; or null
};

// One step.  The coupled form is a mean of h and x with weights s and q = 1 - s: it starts from the one with the larger
// weight and moves by the smaller weight times the difference, which is exact at h = x and at s = 0 and 1, and loses
// nothing of a gate near 1 (q is not formed by subtraction).
__device__ __forceinline__ float scan_step(float h, float x, float s, float q, bool coupled) {
    if (!coupled) return __builtin_fmaf(s, h, x);
    const bool open = q < s;
    const float d = x - h;
    return __builtin_fmaf(open ? q : -s, d, open ? h : x);
}

struct ScanLane {
    long long b, d;
    int n;            // steps of this sample
};
template <int V>
__device__ __forceinline__ bool scan_lane(const ScanArgs& a, ScanLane& l) {
    const long long per = a.D / V, i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= per * a.B) return false;
    l.b = i / per;
    l.d = (i - l.b * per) * V;
    l.n = a.T;
    if (a.lengths) {
        const int n = a.lengths[l.b];
        l.n = n < 0 ? 0 : (n > a.T ? a.T : n);
    }
    return true;
}

template <int V>
__device__ __forceinline__ void scan_load_state(const float* p, long long b, long long D, long long d, float (&h)[V]) {
    if (p) {
        plc_to_float<float, V>(plc_load<float, V>(p + b * D + d), h);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) h[i] = 0.0f;
    }
}

// forward, one lane from the first step to the last
template <class T, int V>
__global__ __launch_bounds__(256) void plc_scan_fwd_kernel(ScanArgs a) {
    ScanLane l;
    if (!scan_lane<V>(a, l)) return;
    const T* x = (const T*)a.x + l.b * a.x_sb + l.d;
    const T* f = (const T*)a.f + l.b * a.f_sb + l.d;
    T* y = (T*)a.y + l.b * a.T * a.D + l.d;
    float h[V];
    scan_load_state<V>(a.h0, l.b, a.D, l.d, h);
    const int blocks = (a.T + SCAN_K - 1) / SCAN_K;
    for (int k = 0; k < blocks; ++k) {
        const int t0 = k * SCAN_K;
        if (k > 0 && a.states)
            plc_store<float, V>(a.states + (l.b * (blocks - 1) + k - 1) * a.D + l.d, plc_from_float<float, V>(h));
        PlcVec<T, V> xr[SCAN_K], fr[SCAN_K];
#pragma unroll
        for (int j = 0; j < SCAN_K; ++j)
            if (t0 + j < l.n) {
                xr[j] = plc_load<T, V>(x + (t0 + j) * a.x_st);
                fr[j] = plc_load<T, V>(f + (t0 + j) * a.f_st);
            }
#pragma unroll
        for (int j = 0; j < SCAN_K; ++j) {
            if (t0 + j >= a.T) break;
            float o[V];
            if (t0 + j < l.n) {
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    float s, q;
                    plc_sigmoid_pair((float)fr[j].e[i], s, q);
                    h[i] = scan_step(h[i], (float)xr[j].e[i], s, q, a.coupled);
                    o[i] = h[i];
                }
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i) o[i] = 0.0f;
            }
            plc_store<T, V>(y + (t0 + j) * a.D, plc_from_float<T, V>(o));
        }
    }
    if (a.h_last) plc_store<float, V>(a.h_last + l.b * a.D + l.d, plc_from_float<float, V>(h));
}

// backward of one block of steps: rebuilds h in fp32 from the state in front of it, then walks it from the end.
// p: what the steps behind the block pass to their previous state (s_{t+1} g_{t+1}); on return, what this block
// passes on.
template <class T, int V>
__device__ __forceinline__ void scan_bwd_block(const ScanArgs& a, const ScanLane& l, int t0, float (&h)[V], float (&p)[V]) {
    const T* x = (const T*)a.x + l.b * a.x_sb + l.d;
    const T* f = (const T*)a.f + l.b * a.f_sb + l.d;
    const T* dy = (const T*)a.dy + l.b * a.dy_sb + l.d;
    T* dx = (T*)a.dx + l.b * a.T * a.D + l.d;
    T* df = (T*)a.df + l.b * a.T * a.D + l.d;
    PlcVec<T, V> xr[SCAN_K], fr[SCAN_K], gr[SCAN_K];
#pragma unroll
    for (int j = 0; j < SCAN_K; ++j)
        if (t0 + j < l.n) {
            xr[j] = plc_load<T, V>(x + (t0 + j) * a.x_st);
            fr[j] = plc_load<T, V>(f + (t0 + j) * a.f_st);
            gr[j] = plc_load<T, V>(dy + (t0 + j) * a.dy_st);
        }
    float before[SCAN_K][V];        // the state in front of each step
#pragma unroll
    for (int j = 0; j < SCAN_K; ++j)
        if (t0 + j < l.n) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                float s, q;
                plc_sigmoid_pair((float)fr[j].e[i], s, q);
                before[j][i] = h[i];
                h[i] = scan_step(h[i], (float)xr[j].e[i], s, q, a.coupled);
            }
        }
#pragma unroll
    for (int j = SCAN_K - 1; j >= 0; --j) {
        if (t0 + j >= a.T) continue;
        float ox[V], of[V];
        if (t0 + j < l.n) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                float s, q;
                plc_sigmoid_pair((float)fr[j].e[i], s, q);
                const float g = (float)gr[j].e[i] + p[i];
                const float m = a.coupled ? before[j][i] - (float)xr[j].e[i] : before[j][i];
                ox[i] = a.coupled ? q * g : g;
                of[i] = g * m * (s * q);
                p[i] = s * g;
            }
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) ox[i] = of[i] = 0.0f;
        }
        plc_store<T, V>(dx + (t0 + j) * a.D, plc_from_float<T, V>(ox));
        plc_store<T, V>(df + (t0 + j) * a.D, plc_from_float<T, V>(of));
    }
}

// backward, one lane from the last step to the first
template <class T, int V>
__global__ __launch_bounds__(256) void plc_scan_bwd_kernel(ScanArgs a) {
    ScanLane l;
    if (!scan_lane<V>(a, l)) return;
    float p[V];
    scan_load_state<V>(a.dh_last, l.b, a.D, l.d, p);
    const int blocks = (a.T + SCAN_K - 1) / SCAN_K;
    for (int k = blocks - 1; k >= 0; --k) {
        float h[V];
        if (k > 0) scan_load_state<V>(a.states + (l.b * (blocks - 1) + k - 1) * a.D, 0, 0, l.d, h);
        else scan_load_state<V>(a.h0, l.b, a.D, l.d, h);
        scan_bwd_block<T, V>(a, l, k * SCAN_K, h, p);
    }
    if (a.dh0) plc_store<float, V>(a.dh0 + l.b * a.D + l.d, plc_from_float<float, V>(p));
}
