// Gated linear recurrence over time, h_t = s_t h_{t-1} + (1 - s_t) x_t ("coupled") or h_t = s_t h_{t-1} + x_t, with
// s_t = sigmoid(f_t): the gates do not depend on h, so the whole sequence is known before the recurrence starts.
//
// Layout: [B][T][D], D innermost; a lane owns V channels of one sample.  The state is fp32 from the first step to
// the last, whatever the type of x, f and y: 16-bit tensors are rounded when a value is stored as y, dx or df and nowhere else.
//
// What bounds it: memory, once there are rows enough.  Forward 3 tensors of B T D elements plus a state every SCAN_K steps,
// backward 5.  8 x 10 x 128 x 128 x 32 bf16 forward without states 47 us, 285 MB: 6.1 TB/s (a large copy runs at 5.2, reading
// alone at 6 to 7).  4 x 10 x 256 x 256 x 32 bf16 forward with states 122 us (604 MB), backward 196 us (973 MB): 5.0 TB/s both.
#pragma once
#include "plc_layers_common.h"

// Steps a lane holds in registers at a time: their loads are all requested before the first is used, and the
// backward pass rebuilds the states of one such block from the state in front of it.  Measured on 4 x 10 x 256 x 256 x 32 bf16
// and 2 x 500 x 20000 bf16: 16 steps need more registers than a lane has (backward 660 us against 190), 4 steps are as
// fast at T = 10 but slower at T = 500 and store twice the states.
constexpr int SCAN_K = 8;
constexpr int SCAN_RUN = 16;          // split form, carry kernel: segments a thread holds in registers

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
    int seg, nseg;                  // split form: steps of a segment (a multiple of SCAN_K) and their number
    float* agg;                     // split form: [nseg][2][B * D], what a segment does to the state: h -> A h + S
};

// The gate as one number, w = -(1 - s) for s > 1/2 and s otherwise: the smaller of the two weights with the sign telling
// which it is.  Both weights follow from it to half a step (1 - |w| >= 1/2), so one register keeps what two would.
// e = exp(-|f|) in (0, 1], |w| = e / (1 + e).  For fp32 tensors the product |f| log2(e) is taken in two parts; for 16-bit
// ones its rounding (|f| 2^-24 relative in e, hence at most 0.4 2^-24 in |w|) is far below their own.
template <class T>
__device__ __forceinline__ float scan_gate(float f) {
    const float e = sizeof(T) == 4 ? plc_exp_neg(-__builtin_fabsf(f)) : __builtin_amdgcn_exp2f(-1.44269504088896341f * __builtin_fabsf(f));
    return __builtin_copysignf(e * __builtin_amdgcn_rcpf(1.0f + e), -f);
}
__device__ __forceinline__ bool scan_open(float w) { return __builtin_bit_cast(int, w) < 0; }     // (-0.0: s = 1)
__device__ __forceinline__ float scan_s(float w) { return scan_open(w) ? 1.0f + w : w; }

// One step.  The coupled form is a mean of h and x: it starts from the one with the larger weight and moves by the smaller
// weight times the difference, which is exact at h = x and at s = 0 and 1, and loses nothing of a gate near 1.  (The price: an
// infinite x, or an x - h beyond fp32's range, gives an infinity or a NaN where the two products would give their sum.)
template <bool COUPLED>
__device__ __forceinline__ float scan_step(float h, float x, float w) {
    if (!COUPLED) return __builtin_fmaf(scan_s(w), h, x);
    return __builtin_fmaf(-w, x - h, scan_open(w) ? h : x);
}

struct ScanLane {
    long long b, d;
    int n;            // steps of this sample
};
template <int V>
__device__ __forceinline__ bool scan_lane(const ScanArgs& a, long long i, ScanLane& l) {
    const long long per = a.D / V;
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
__device__ __forceinline__ void scan_load_state(const float* p, long long at, float (&h)[V]) {
    if (p) {
        plc_to_float<float, V>(plc_load<float, V>(p + at), h);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) h[i] = 0.0f;
    }
}

// Rows t0 .. t0 + SCAN_K - 1 of one tensor.  Not FULL: the block reaches behind some lane's sample.  Its loads are not
// conditional all the same (they would wait for one another); a row behind the sequence becomes its last one, which is
// memory of the tensor, and what is loaded there is not used.
template <class T, int V, bool FULL, bool STREAM = false>
__device__ __forceinline__ void scan_rows(const ScanArgs& a, const void* base, long long sb, long long st, const ScanLane& l, int t0, PlcVec<T, V> (&r)[SCAN_K]) {
    const T* p = (const T*)base + l.b * sb + l.d + t0 * st;
    const int most = a.T - 1 - t0;
#pragma unroll
    for (int j = 0; j < SCAN_K; ++j) r[j] = plc_load<T, V, STREAM>(p + (FULL ? j : min(j, most)) * st);
}

// ---- forward ----------------------------------------------------------------------------------------------------
// one block of steps from state h; rows between the sample's length and T get 0
template <class T, int V, bool COUPLED, bool FULL, bool STREAM>
__device__ __forceinline__ void scan_fwd_block(const ScanArgs& a, const ScanLane& l, int t0, float (&h)[V]) {
    PlcVec<T, V> xr[SCAN_K], fr[SCAN_K];
    scan_rows<T, V, FULL, STREAM>(a, a.f, a.f_sb, a.f_st, l, t0, fr);
    scan_rows<T, V, FULL, STREAM>(a, a.x, a.x_sb, a.x_st, l, t0, xr);
    T* y = (T*)a.y + (l.b * a.T + t0) * a.D + l.d;
#pragma unroll
    for (int j = 0; j < SCAN_K; ++j) {
        if (!FULL && t0 + j >= a.T) break;
        float o[V];
        const bool on = FULL || t0 + j < l.n;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float next = scan_step<COUPLED>(h[i], xr[j].get(i), scan_gate<T>(fr[j].get(i)));
            h[i] = on ? next : h[i];
            o[i] = on ? next : 0.0f;
        }
        plc_store<T, V>(y + j * a.D, plc_from_float<T, V>(o));
    }
}
// a block behind every lane's sample
template <class T, int V>
__device__ __forceinline__ void scan_zero_block(const ScanArgs& a, T* y, const ScanLane& l, int t0) {
    float o[V];
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = 0.0f;
    y += (l.b * a.T + t0) * a.D + l.d;
#pragma unroll
    for (int j = 0; j < SCAN_K; ++j)
        if (t0 + j < a.T) plc_store<T, V>(y + j * a.D, plc_from_float<T, V>(o));
}
template <class T, int V, bool COUPLED, bool STREAM>
__device__ __forceinline__ void scan_fwd_range(const ScanArgs& a, const ScanLane& l, int t0, int t1, float (&h)[V]) {
    const int blocks = (a.T + SCAN_K - 1) / SCAN_K;
    for (int t = t0; t < t1; t += SCAN_K) {
        const int k = t / SCAN_K;
        if (k > 0 && a.states) plc_store<float, V>(a.states + (l.b * (blocks - 1) + k - 1) * a.D + l.d, plc_from_float<float, V>(h));
        if (__all(t + SCAN_K <= l.n)) scan_fwd_block<T, V, COUPLED, true, STREAM>(a, l, t, h);
        else if (__any(t < l.n)) scan_fwd_block<T, V, COUPLED, false, STREAM>(a, l, t, h);
        else scan_zero_block<T, V>(a, (T*)a.y, l, t);
    }
}

// one lane from the first step to the last; STREAM: x and f do not stay in the caches
template <class T, int V, bool COUPLED, bool STREAM>
__global__ __launch_bounds__(256) void plc_scan_fwd_kernel(ScanArgs a) {
    ScanLane l;
    if (!scan_lane<V>(a, (long long)blockIdx.x * blockDim.x + threadIdx.x, l)) return;
    float h[V];
    scan_load_state<V>(a.h0, l.b * a.D + l.d, h);
    scan_fwd_range<T, V, COUPLED, STREAM>(a, l, 0, a.T, h);
    if (a.h_last) plc_store<float, V>(a.h_last + l.b * a.D + l.d, plc_from_float<float, V>(h));
}

// ---- backward ---------------------------------------------------------------------------------------------------
// One block of steps: rebuilds the states in fp32 from the one in front of it, then walks it from the end.
// p: what the steps behind the block pass to their previous state (s_{t+1} g_{t+1}); on return, what this block
// passes on.  Between the two walks a step is two numbers per channel: its gate, and the factor of df (h_{t-1} - x_t or
// h_{t-1}); x and f are not kept.
template <class T, int V, bool COUPLED, bool FULL>
__device__ __forceinline__ void scan_bwd_block(const ScanArgs& a, const ScanLane& l, int t0, float (&h)[V], float (&p)[V]) {
    PlcVec<T, V> gr[SCAN_K];
    float w[SCAN_K][V], m[SCAN_K][V];
    {
        PlcVec<T, V> xr[SCAN_K], fr[SCAN_K];
        scan_rows<T, V, FULL>(a, a.f, a.f_sb, a.f_st, l, t0, fr);
        scan_rows<T, V, FULL>(a, a.x, a.x_sb, a.x_st, l, t0, xr);
        scan_rows<T, V, FULL>(a, a.dy, a.dy_sb, a.dy_st, l, t0, gr);
#pragma unroll
        for (int j = 0; j < SCAN_K; ++j) {
            const bool on = FULL || t0 + j < l.n;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float x = xr[j].get(i);
                w[j][i] = scan_gate<T>(fr[j].get(i));
                m[j][i] = COUPLED ? h[i] - x : h[i];
                const float next = scan_step<COUPLED>(h[i], x, w[j][i]);
                h[i] = on ? next : h[i];
            }
        }
    }
    T* dx = (T*)a.dx + (l.b * a.T + t0) * a.D + l.d;
    T* df = (T*)a.df + (l.b * a.T + t0) * a.D + l.d;
#pragma unroll
    for (int j = SCAN_K - 1; j >= 0; --j) {
        if (!FULL && t0 + j >= a.T) continue;
        const bool on = FULL || t0 + j < l.n;
        float ox[V], of[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float small = __builtin_fabsf(w[j][i]), large = 1.0f - small;
            const bool open = scan_open(w[j][i]);
            const float s = open ? large : small, g = gr[j].get(i) + p[i];
            ox[i] = on ? (COUPLED ? (open ? small : large) * g : g) : 0.0f;
            of[i] = on ? g * m[j][i] * (small * large) : 0.0f;
            p[i] = on ? s * g : p[i];
        }
        plc_store<T, V>(dx + j * a.D, plc_from_float<T, V>(ox));
        plc_store<T, V>(df + j * a.D, plc_from_float<T, V>(of));
    }
}
template <class T, int V, bool COUPLED>
__device__ __forceinline__ void scan_bwd_range(const ScanArgs& a, const ScanLane& l, int t0, int t1, float (&p)[V]) {
    const int blocks = (a.T + SCAN_K - 1) / SCAN_K;
    for (int k = (t1 - 1) / SCAN_K; k >= t0 / SCAN_K; --k) {
        float h[V];
        if (k > 0) scan_load_state<V>(a.states, (l.b * (blocks - 1) + k - 1) * a.D + l.d, h);
        else scan_load_state<V>(a.h0, l.b * a.D + l.d, h);
        if (!__any(k * SCAN_K < l.n)) {
            scan_zero_block<T, V>(a, (T*)a.dx, l, k * SCAN_K);
            scan_zero_block<T, V>(a, (T*)a.df, l, k * SCAN_K);
            continue;
        }
        if (__all((k + 1) * SCAN_K <= l.n)) scan_bwd_block<T, V, COUPLED, true>(a, l, k * SCAN_K, h, p);
        else scan_bwd_block<T, V, COUPLED, false>(a, l, k * SCAN_K, h, p);
    }
}

// one lane from the last step to the first
template <class T, int V, bool COUPLED>
__global__ __launch_bounds__(256) void plc_scan_bwd_kernel(ScanArgs a) {
    ScanLane l;
    if (!scan_lane<V>(a, (long long)blockIdx.x * blockDim.x + threadIdx.x, l)) return;
    float p[V];
    scan_load_state<V>(a.dh_last, l.b * a.D + l.d, p);
    if (a.T > 0) scan_bwd_range<T, V, COUPLED>(a, l, 0, a.T, p);
    if (a.dh0) plc_store<float, V>(a.dh0 + l.b * a.D + l.d, plc_from_float<float, V>(p));
}

// ---- split form: few channels, many steps -----------------------------------------------------------------------
// A segment of steps does h -> A h + S to the state (A the product of its gates), and the same to the gradient that runs
// backwards, p -> A p + S.  The first launch computes A and S of every segment, the second turns them into the state in
// front of (the gradient behind) each, the third walks the segments as above.  x and f (f and dy) are read twice, the second
// time mostly from the cache; in return every segment runs at once.  Lanes run over (segment, channels): a row of few
// channels does not leave lanes of a wave idle.
// 4 x 32768 x 96 bf16 with lengths: 12.8 + 5.8 + 18.7 us (75 MB that cannot be done without, 126 MB moved); 8 x 3653 x 48 fp32
// forward 5.3 + 6.2 + 5.5 us, backward 4.6 + 5.9 + 6.1: three launches of which none is bound by memory.
template <int V>
__device__ __forceinline__ bool scan_item(const ScanArgs& a, ScanLane& l, int& k) {
    const unsigned lanes = (unsigned)(a.B * (a.D / V)), i = blockIdx.x * blockDim.x + threadIdx.x;
    k = (int)(i / lanes);
    return k < a.nseg && scan_lane<V>(a, i - (unsigned)k * lanes, l);
}

template <class T, int V, bool COUPLED, bool BACKWARD, bool FULL>
__device__ __forceinline__ void scan_agg_block(const ScanArgs& a, const ScanLane& l, int t0, float (&A)[V], float (&S)[V]) {
    PlcVec<T, V> fr[SCAN_K], vr[SCAN_K];
    scan_rows<T, V, FULL>(a, a.f, a.f_sb, a.f_st, l, t0, fr);
    if (BACKWARD) scan_rows<T, V, FULL>(a, a.dy, a.dy_sb, a.dy_st, l, t0, vr);
    else scan_rows<T, V, FULL>(a, a.x, a.x_sb, a.x_st, l, t0, vr);
#pragma unroll
    for (int jj = 0; jj < SCAN_K; ++jj) {
        const int j = BACKWARD ? SCAN_K - 1 - jj : jj;
        const bool on = FULL || t0 + j < l.n;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float w = scan_gate<T>(fr[j].get(i)), v = vr[j].get(i), s = scan_s(w);
            const float next = BACKWARD ? s * (v + S[i]) : scan_step<COUPLED>(S[i], v, w);
            A[i] = on ? A[i] * s : A[i];
            S[i] = on ? next : S[i];
        }
    }
}

template <class T, int V, bool COUPLED, bool BACKWARD>
__global__ __launch_bounds__(256) void plc_scan_segments_kernel(ScanArgs a) {
    ScanLane l;
    int k;
    if (!scan_item<V>(a, l, k)) return;
    float A[V], S[V];
#pragma unroll
    for (int i = 0; i < V; ++i) A[i] = 1.0f, S[i] = 0.0f;
    const int t0 = k * a.seg, t1 = min(t0 + a.seg, a.T), blocks = (t1 - t0 + SCAN_K - 1) / SCAN_K;
    for (int q = 0; q < blocks; ++q) {
        const int t = t0 + (BACKWARD ? blocks - 1 - q : q) * SCAN_K;
        if (__all(t + SCAN_K <= l.n)) scan_agg_block<T, V, COUPLED, BACKWARD, true>(a, l, t, A, S);
        else if (__any(t < l.n)) scan_agg_block<T, V, COUPLED, BACKWARD, false>(a, l, t, A, S);
    }
    float* agg = a.agg + (long long)k * 2 * a.B * a.D + l.b * a.D + l.d;
    plc_store<float, V>(agg, plc_from_float<float, V>(A));
    plc_store<float, V>(agg + (long long)a.B * a.D, plc_from_float<float, V>(S));
}

// (A, S) of the segments -> what each starts from, in A's place.  R threads per channel, each a run of segments: folded, the
// runs joined in order through LDS, walked again.  A run of up to SCAN_RUN segments is read once and kept (the launch picks
// R so that a run stays short: 16 segments cost 10.7 us in runs of 16, 8.3 in runs of four; only more than 64 * SCAN_RUN
// segments are read twice).  One launch of its own: the fold inside the last kernel, repeated by every workgroup, took
// 441 us for 1 x 1000000 x 16 where the three launches take 86.
constexpr int scan_carry_channels(int R) { return R == 64 ? 16 : 256 / R; }

template <bool BACKWARD, int R>
__global__ __launch_bounds__(R * scan_carry_channels(R)) void plc_scan_carry_kernel(ScanArgs a) {
    constexpr int CH = scan_carry_channels(R);
    __shared__ float part[2][R][CH];
    const int ch = threadIdx.x % CH, run = threadIdx.x / CH;
    const long long n = (long long)a.B * a.D, c = (long long)blockIdx.x * CH + ch;
    const int share = (a.nseg + R - 1) / R, q0 = min(run * share, a.nseg), q1 = min(q0 + share, a.nseg);
    float* agg = a.agg + c;
    auto at = [&](int q) { return (long long)(BACKWARD ? a.nseg - 1 - q : q) * 2 * n; };
    float A = 1.0f, S = 0.0f, ra[SCAN_RUN], rs[SCAN_RUN];
    auto load = [&](int q) {
#pragma unroll
        for (int j = 0; j < SCAN_RUN; ++j)
            if (q + j < q1) ra[j] = agg[at(q + j)], rs[j] = agg[at(q + j) + n];
    };
    if (c < n)
        for (int q = q0; q < q1; q += SCAN_RUN) {
            load(q);
#pragma unroll
            for (int j = 0; j < SCAN_RUN; ++j)
                if (q + j < q1) {
                    S = __builtin_fmaf(ra[j], S, rs[j]);
                    A *= ra[j];
                }
        }
    if (R > 1) {
        part[0][run][ch] = A;
        part[1][run][ch] = S;
        __syncthreads();
    }
    if (c >= n) return;
    const float* first = BACKWARD ? a.dh_last : a.h0;
    float h = first ? first[c] : 0.0f;
#pragma unroll 8
    for (int r = 0; r < run; ++r) h = __builtin_fmaf(part[0][r][ch], h, part[1][r][ch]);
    for (int q = q0; q < q1; q += SCAN_RUN) {
        if (share > SCAN_RUN) load(q);
#pragma unroll
        for (int j = 0; j < SCAN_RUN; ++j)
            if (q + j < q1) {
                agg[at(q + j)] = h;
                h = __builtin_fmaf(ra[j], h, rs[j]);
            }
    }
}

template <class T, int V, bool COUPLED, bool BACKWARD>
__global__ __launch_bounds__(256) void plc_scan_split_kernel(ScanArgs a) {
    ScanLane l;
    int k;
    if (!scan_item<V>(a, l, k)) return;
    float h[V];
    scan_load_state<V>(a.agg, (long long)k * 2 * a.B * a.D + l.b * a.D + l.d, h);
    const int t0 = k * a.seg, t1 = min(t0 + a.seg, a.T);
    if (BACKWARD) {
        scan_bwd_range<T, V, COUPLED>(a, l, t0, t1, h);
        if (k == 0 && a.dh0) plc_store<float, V>(a.dh0 + l.b * a.D + l.d, plc_from_float<float, V>(h));
    } else {
        scan_fwd_range<T, V, COUPLED, false>(a, l, t0, t1, h);
        if (k == a.nseg - 1 && a.h_last) plc_store<float, V>(a.h_last + l.b * a.D + l.d, plc_from_float<float, V>(h));
    }
}
