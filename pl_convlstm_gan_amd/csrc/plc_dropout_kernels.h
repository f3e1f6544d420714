// Dropout whose mask is computed from a counter instead of being stored: y = keep ? x * scale : 0, plus a residual.
// The backward pass runs the same kernel on dy.  A dropped element is exactly 0, also where x is not finite.
// The product and the residual's sum are fp32; y is rounded once.
// Bound by memory: 84 M bf16 elements 56.9 us (336 MB: 5.9 TB/s); ten rounds of the generator serve eight elements,
// so that one lane makes one 16-byte store (8 fp32 elements: two).  Small calls cost their launch: 1 M odd fp16 elements with a
// residual 3.0 us.
#pragma once
#include "plc_layers_common.h"

struct DropoutArgs {
    long long n;
    const void *x, *r;            // r: residual or null
    void* y;
    PlcDrop drop;
    const long long* offset_ptr;  // device: drop.offset, or null
    long long* used_offset;       // device: receives the offset this call used, or null
};

// one lane per call of the generator: eight consecutive elements, moved as vectors of VEC
template <class T, int VEC, bool STREAM>
__global__ __launch_bounds__(256) void plc_dropout_kernel(DropoutArgs a) {
    PlcDrop d = a.drop;
    if (a.offset_ptr) d.offset = (uint64_t)*a.offset_ptr;
    if (a.used_offset && blockIdx.x == 0 && threadIdx.x == 0) *a.used_offset = (long long)d.offset;
    const long long j = (long long)blockIdx.x * blockDim.x + threadIdx.x, e0 = j * 8;
    if (e0 >= a.n) return;
    const T *x = (const T*)a.x + e0, *r = a.r ? (const T*)a.r + e0 : nullptr;
    T* y = (T*)a.y + e0;
    const uint32_t keep = plc_keep_bits<8>(d, e0);
    if (VEC == 8 && e0 + 8 <= a.n) {
        const PlcVec<T, 8> v = plc_load<T, 8, STREAM>(x);
        PlcVec<T, 8> w = v;
        if (r) w = plc_load<T, 8>(r);
        float o[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            o[i] = (keep >> i) & 1 ? v.get(i) * d.scale : 0.0f;
            if (r) o[i] += w.get(i);
        }
        plc_store<T, 8>(y, plc_from_float<T, 8>(o));
    } else {
        for (int i = 0; i < 8 && e0 + i < a.n; ++i) {
            float o = (keep >> i) & 1 ? (float)x[i] * d.scale : 0.0f;
            if (r) o += (float)r[i];
            y[i] = (T)o;
        }
    }
}
