// Device helpers of the layer operators (gated linear recurrence, group norm, dropout): element types, vector
// loads and stores, the sigmoid, the counter-based generator.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

typedef __bf16 plc_bf16;
typedef _Float16 plc_f16;

template <bool WHOLE>
struct PlcWord {
    typedef uint32_t type;
};
template <>
struct PlcWord<false> {
    typedef unsigned short type;
};

// V consecutive elements of T, moved as one access of V * sizeof(T) bytes (16 at most; wider ones as several).  They are
// kept as the words that were loaded and unpacked where they are used: held as separate 16-bit values, each would take a
// register of its own.
template <class T, int V>
struct alignas(V * sizeof(T) > 16 ? 16 : V * sizeof(T)) PlcVec {
    static constexpr int NW = V * sizeof(T) >= 4 ? V * sizeof(T) / 4 : 1;
    using Word = typename PlcWord<(V * sizeof(T) >= 4)>::type;
    Word w[NW];
    __device__ __forceinline__ float get(int i) const {
        if constexpr (sizeof(T) == 4) {
            return __builtin_bit_cast(float, w[i]);
        } else {
            const uint32_t q = (uint32_t)w[i >> 1];
            if constexpr (__is_same(T, plc_bf16)) return __builtin_bit_cast(float, (i & 1) ? q & 0xffff0000u : q << 16);
            else return (float)__builtin_bit_cast(plc_f16, (unsigned short)((i & 1) ? q >> 16 : q & 0xffffu));
        }
    }
};

// STREAM: the access does not keep its line in the caches (whole vectors only); for tensors that are too large to be
// found there again.
typedef uint32_t plc_u32x4 __attribute__((ext_vector_type(4)));
template <class T, int V, bool STREAM = false>
__device__ __forceinline__ PlcVec<T, V> plc_load(const T* p) {
    if constexpr (STREAM && sizeof(PlcVec<T, V>) == 16) return __builtin_bit_cast(PlcVec<T, V>, __builtin_nontemporal_load(reinterpret_cast<const plc_u32x4*>(p)));
    else return *reinterpret_cast<const PlcVec<T, V>*>(p);
}
template <class T, int V, bool STREAM = false>
__device__ __forceinline__ void plc_store(T* p, const PlcVec<T, V>& v) {
    if constexpr (STREAM && sizeof(PlcVec<T, V>) == 16) __builtin_nontemporal_store(__builtin_bit_cast(plc_u32x4, v), reinterpret_cast<plc_u32x4*>(p));
    else *reinterpret_cast<PlcVec<T, V>*>(p) = v;
}
template <class T, int V>
__device__ __forceinline__ void plc_to_float(const PlcVec<T, V>& v, float (&o)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = v.get(i);
}
// (conversions from fp32 round to nearest even: results and gradients leave in the inputs' type, rounded once)
template <class T, int V>
__device__ __forceinline__ PlcVec<T, V> plc_from_float(const float (&v)[V]) {
    PlcVec<T, V> o;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < V; ++i) o.w[i] = __builtin_bit_cast(uint32_t, v[i]);
    } else if constexpr (V == 1) {
        o.w[0] = __builtin_bit_cast(unsigned short, (T)v[0]);
    } else {
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
            typedef float F2 __attribute__((ext_vector_type(2)));
            typedef T T2 __attribute__((ext_vector_type(2)));
            const F2 f = {v[2 * i], v[2 * i + 1]};
            o.w[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(f, T2));
        }
    }
    return o;
}

// exp(x) for x <= 0, to about one unit in the last place: the product x log2(e) is taken in two parts, so that the
// rounding of its leading part does not grow with |x| (v_exp_f32 alone would be off by |x| 2^-24).
__device__ __forceinline__ float plc_exp_neg(float x) {
    const float t = x * 1.44269504088896341f;
    // the rest of the product; t is -inf when x is, where the difference has no value
    const float lo = __builtin_fmaf(x, 1.44269504088896341f, -t) + x * 1.92596299112661746e-8f;
    const float e = __builtin_amdgcn_exp2f(t);
    return t < -126.0f ? e : __builtin_fmaf(e * 0.693147180559945309f, lo, e);
}

// Philox4x32-10 (Salmon, Moraes, Dror, Shaw: Parallel random numbers: as easy as 1, 2, 3; SC 2011): 128 random bits
// that depend on the counter and the key alone.
__device__ __forceinline__ uint4 plc_philox(uint64_t lo, uint64_t hi, uint64_t key) {
    uint32_t c0 = (uint32_t)lo, c1 = (uint32_t)(lo >> 32), c2 = (uint32_t)hi, c3 = (uint32_t)(hi >> 32);
    uint32_t k0 = (uint32_t)key, k1 = (uint32_t)(key >> 32);
#pragma unroll
    for (int i = 0; i < 10; ++i) {
        const uint64_t m0 = (uint64_t)0xD2511F53u * c0, m1 = (uint64_t)0xCD9E8D57u * c2;
        c0 = (uint32_t)(m1 >> 32) ^ c1 ^ k0;
        c2 = (uint32_t)(m0 >> 32) ^ c3 ^ k1;
        c1 = (uint32_t)m1;
        c3 = (uint32_t)m0;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return make_uint4(c0, c1, c2, c3);
}

// What decides which elements are dropped: element e of the tensor takes the 16-bit value e & 7 of
// Philox(counter = (e >> 3, offset), key = seed) and stays when that is at least `thr`.  16 bits resolve a
// probability to 2^-17; the scale is formed from the resolved one, so the mean is kept exactly.  One call of the
// generator (about 20 quarter-rate multiplies) then serves eight elements: with 32 bits per element the
// generator and not the memory would bound a 16-bit tensor.
struct PlcDrop {
    uint64_t seed, offset;
    uint32_t thr;         // 0: nothing is dropped, 65536: everything
    float scale;          // 65536 / (65536 - thr)
};
// bit i: element e0 + i stays (i < V; e0 is a multiple of V, so its V values lie in one call)
template <int V>
__device__ __forceinline__ uint32_t plc_keep_bits(const PlcDrop& d, uint64_t e0) {
    const uint4 r = plc_philox(e0 >> 3, d.offset, d.seed);
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
    uint32_t bits = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t u = (i & 1) ? w[i >> 1] >> 16 : w[i >> 1] & 0xffffu;
        bits |= (u >= d.thr ? 1u : 0u) << i;
    }
    return bits >> (uint32_t)(e0 & 7);
}
