// cat_rows.h -- what the categorical-policy kernels (cat_loss.hip,
// cat_sample.hip) share: element types, reductions, argument checks.
#pragma once
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>

#include "rtenv.h"

extern "C" int rt_internal_fail(int code, const char* msg);

namespace rtcat {

// ---- element types ---------------------------------------------------------
struct F32 {
    using raw = float;
    static __device__ __forceinline__ float get(raw r) { return r; }
    static __device__ __forceinline__ raw put(float f) { return f; }
};
struct BF16 {
    using raw = uint16_t;
    static __device__ __forceinline__ float get(raw r) { return __uint_as_float((uint32_t)r << 16); }
    // round to nearest even, NaN kept a (quiet) NaN
    static __device__ __forceinline__ raw put(float f) {
        const uint32_t b = __float_as_uint(f);
        if (f != f) return (raw)((b >> 16) | 0x40);
        return (raw)((b + 0x7fff + ((b >> 16) & 1)) >> 16);
    }
};
struct F16 {
    using raw = uint16_t;
    static __device__ __forceinline__ float get(raw r) { return (float)__builtin_bit_cast(_Float16, r); }
    static __device__ __forceinline__ raw put(float f) { return __builtin_bit_cast(raw, (_Float16)f); }
};

// ---- 2^t in 64 bits --------------------------------------------------------
// t <= 0 or NaN.  t = n + f, |f| <= 1/2; the Taylor sum of exp(f ln 2) up to
// f^11 leaves (ln 2 / 2)^12 / 12! < 7e-15.
__device__ __forceinline__ double exp2_64(double t) {
    t = t < -1100.0 ? -1100.0 : t;
    const double n = rint(t), f = t - n;
    double p = 4.44553827187081e-10;  // (ln 2)^11 / 11!, and so on down
    p = fma(p, f, 7.054911620801121e-09);
    p = fma(p, f, 1.0178086009239696e-07);
    p = fma(p, f, 1.3215486790144305e-06);
    p = fma(p, f, 1.5252733804059838e-05);
    p = fma(p, f, 0.00015403530393381606);
    p = fma(p, f, 0.0013333558146428441);
    p = fma(p, f, 0.009618129107628477);
    p = fma(p, f, 0.055504108664821576);
    p = fma(p, f, 0.2402265069591007);
    p = fma(p, f, 0.6931471805599453);
    p = fma(p, f, 1.0);
    return ldexp(p, (int)n);
}

// ---- reductions ------------------------------------------------------------
template <class T>
__device__ __forceinline__ T wave_sum(T v) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    return v;
}
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));  // NaN loses; the sums keep it
    return v;
}

// Whole-block reductions through one LDS slot per wave; every thread gets the
// result, and the slots may be used again at once.
template <int THREADS, class T>
__device__ __forceinline__ T block_sum(T v, T* slots) {
    v = wave_sum(v);
    if constexpr (THREADS == 64) return v;
    if ((threadIdx.x & 63) == 0) slots[threadIdx.x >> 6] = v;
    __syncthreads();
    T r = slots[0];
#pragma unroll
    for (int i = 1; i < THREADS / 64; ++i) r += slots[i];
    __syncthreads();
    return r;
}
template <int THREADS>
__device__ __forceinline__ float block_max(float v, float* slots) {
    v = wave_max(v);
    if constexpr (THREADS == 64) return v;
    if ((threadIdx.x & 63) == 0) slots[threadIdx.x >> 6] = v;
    __syncthreads();
    float r = slots[0];
#pragma unroll
    for (int i = 1; i < THREADS / 64; ++i) r = fmaxf(r, slots[i]);
    __syncthreads();
    return r;
}

// ---- argument checks -------------------------------------------------------
inline int elem_size(int32_t dtype) { return dtype == RT_DT_F32 ? 4 : 2; }
inline bool bad_type(int32_t dtype) { return dtype != RT_DT_F32 && dtype != RT_DT_BF16 && dtype != RT_DT_F16; }

inline const char* logits_fault(const rt_cat_logits* l) {
    if (!l || !l->x) return "NULL logits";
    if (bad_type(l->dtype)) return "logits type is not one of RT_DT_*";
    if (l->rows < 1 || l->rows > INT32_MAX) return "rows out of range";
    if (l->vocab < 1 || l->vocab > RT_CAT_MAX_VOCAB) return "vocab out of range";
    if (l->row_stride < 0) return "negative row stride";
    if ((uintptr_t)l->x % elem_size(l->dtype)) return "logits not aligned to their element";
    return nullptr;
}

inline int launched() {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? RT_OK : rt_internal_fail(RT_ELAUNCH, hipGetErrorString(e));
}

}  // namespace rtcat
