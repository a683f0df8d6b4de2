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
    static __device__ __forceinline__ raw put(float f) { return __builtin_bit_cast(raw, (__bf16)f); }
    static __device__ __forceinline__ uint32_t put2(float lo, float hi) {  // one instruction for both
        typedef float f2 __attribute__((ext_vector_type(2)));
        typedef __bf16 b2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2{lo, hi}), b2));
    }
};
struct F16 {
    using raw = uint16_t;
    static __device__ __forceinline__ float get(raw r) { return (float)__builtin_bit_cast(_Float16, r); }
    static __device__ __forceinline__ raw put(float f) { return __builtin_bit_cast(raw, (_Float16)f); }
    static __device__ __forceinline__ uint32_t put2(float lo, float hi) { return put(lo) | (uint32_t)put(hi) << 16; }
};

// ---- 2^t in 64 bits --------------------------------------------------------
// t <= 1100 (where 2^t is infinite) or NaN.  t = n + f, |f| <= 1/2, n from the
// sum with 1.5 2^52, whose low word holds it (a NaN's is any number); the Taylor
// sum of exp(f ln 2) up to f^11 leaves (ln 2 / 2)^12 / 12! < 7e-15.
__device__ __forceinline__ double exp2_64(double t) {
    const double kWhole = 6755399441055744.0;  // 1.5 2^52
    t = t < -1100.0 ? -1100.0 : t;
    const double sum = t + kWhole, f = t - (sum - kWhole);
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
    return ldexp(p, (int)(uint32_t)__builtin_bit_cast(uint64_t, sum));
}

// e^x of any x: infinite past the doubles, and for +inf
__device__ __forceinline__ double exp_64(double x) {
    const double t = x * 1.4426950408889634;
    return exp2_64(t > 1100.0 ? 1100.0 : t);
}

// log s, 1 <= s <= 2^20 or NaN: the hardware's log2, corrected by what it
// leaves.  Floats below 20 are 2^-19 apart, the instruction is within one of
// them, and s was rounded to f32 before: d < 2^-18, and log(1 + d) up to d^3
// leaves d^4 / 4 < 2^-74.
__device__ __forceinline__ double log_64(double s) {
    const double y = (double)__builtin_amdgcn_logf((float)s);
    const double d = s * exp2_64(-y) - 1.0;
    return y * 0.6931471805599453 + d * (1.0 - d * (0.5 - d * 0.3333333333333333));
}

// ---- reductions ------------------------------------------------------------
// A value from the lane that the DPP control names: within 16 lanes an exchange
// costs one VALU move and no trip through LDS.
template <int CTRL, class T>
__device__ __forceinline__ T dpp(T v) {
    constexpr int kWords = sizeof(T) / 4;
    struct Words { int w[kWords]; } x = __builtin_bit_cast(Words, v);
#pragma unroll
    for (int i = 0; i < kWords; ++i) x.w[i] = __builtin_amdgcn_update_dpp(0, x.w[i], CTRL, 0xf, 0xf, true);
    return __builtin_bit_cast(T, x);
}
// op over G lanes (a power of two), every lane gets the result: the two swaps
// within four lanes, the mirrors of 8 and 16, then LDS permutes.
template <int G, class T, class Op>
__device__ __forceinline__ T lanes(T v, Op op) {
    if constexpr (G >= 2) v = op(v, dpp<0xb1>(v));
    if constexpr (G >= 4) v = op(v, dpp<0x4e>(v));
    if constexpr (G >= 8) v = op(v, dpp<0x141>(v));
    if constexpr (G >= 16) v = op(v, dpp<0x140>(v));
    if constexpr (G >= 32) v = op(v, __shfl_xor(v, 16));
    if constexpr (G >= 64) v = op(v, __shfl_xor(v, 32));
    return v;
}
template <int G, class T>
__device__ __forceinline__ T lanes_sum(T v) {
    return lanes<G>(v, [](T a, T b) { return a + b; });
}
template <int G>
__device__ __forceinline__ float lanes_max(float v) {  // NaN loses; the sums keep it
    return lanes<G>(v, [](float a, float b) { return fmaxf(a, b); });
}
template <class T>
__device__ __forceinline__ T wave_sum(T v) { return lanes_sum<64>(v); }
__device__ __forceinline__ float wave_max(float v) { return lanes_max<64>(v); }

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

// ---- rows as 16-byte pieces ------------------------------------------------
// A row as 16-byte pieces that are aligned wherever the row starts, and the
// few entries before and after them ("edges", at most 2 (PER - 1) <= 14: one
// per thread).
template <class D>
struct Span {
    static constexpr int kPer = 16 / (int)sizeof(typename D::raw);
    const typename D::raw* x;
    int32_t head, pieces, edges;

    __device__ Span(const typename D::raw* row, int32_t V) : x(row) {
        head = min(V, (int32_t)((0 - (uintptr_t)row) % 16 / sizeof(typename D::raw)));
        pieces = (V - head) / kPer;
        edges = V - pieces * kPer;
    }
    __device__ __forceinline__ int32_t edge(int t) const { return t < head ? t : pieces * kPer + t; }
    __device__ __forceinline__ uint4 piece(int32_t i) const {
        return *reinterpret_cast<const uint4*>(x + head + (int64_t)i * kPer);
    }
};

template <class D>
struct Unpack {
    static constexpr int kPer = 16 / (int)sizeof(typename D::raw);
    float v[kPer];
    __device__ __forceinline__ explicit Unpack(const uint4& r) {
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            if constexpr (kPer == 4) v[i] = __uint_as_float(w[i]);
            else v[i] = D::get((typename D::raw)(i & 1 ? w[i / 2] >> 16 : w[i / 2] & 0xffff));
        }
    }
    __device__ __forceinline__ float max() const {
        float m = v[0];
#pragma unroll
        for (int i = 1; i < kPer; ++i) m = fmaxf(m, v[i]);
        return m;
    }
};

// Rows of V <= 32 entries into LDS, V | 1 words apart; eight trips to memory at
// once (one by one they were most of what such a row took).
template <class D, int THREADS>
__device__ __forceinline__ void load_tile(float* tile, const typename D::raw* x, int64_t stride, int32_t rows, int32_t V) {
    constexpr int kAhead = 8;
    const float per = 1.0f / (float)V;  // (i + 1/2) / V is 1/64 or more away from a whole number
    for (int32_t from = threadIdx.x; from < rows * V; from += kAhead * THREADS) {
        typename D::raw v[kAhead];
        int32_t at[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            const int32_t i = from + k * THREADS, r = (int32_t)(((float)i + 0.5f) * per), c = i - r * V;
            at[k] = r * (V | 1) + c;
            if (i < rows * V) v[k] = x[r * stride + c];
        }
#pragma unroll
        for (int k = 0; k < kAhead; ++k)
            if (from + k * THREADS < rows * V) tile[at[k]] = D::get(v[k]);
    }
}

// 16 bytes of entries that add nothing
template <class D>
__device__ __forceinline__ uint4 nothing() {
    if constexpr (sizeof(typename D::raw) == 4) return make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u);
    const uint32_t two = (uint32_t)D::put(-INFINITY) * 0x10001u;
    return make_uint4(two, two, two, two);
}

// ---- launches --------------------------------------------------------------
// A dimension of a launch has less than 2^32 threads: past 2^20 blocks the grid
// has a second one, and block_index() may then be behind the last block.
inline dim3 grid_of(int64_t blocks) {
    constexpr int64_t kMost = 1 << 20;
    if (blocks <= kMost) return dim3((unsigned)blocks);
    return dim3((unsigned)kMost, (unsigned)((blocks + kMost - 1) / kMost));
}
__device__ __forceinline__ int64_t block_index() { return (int64_t)blockIdx.y << 20 | blockIdx.x; }

// ---- argument checks -------------------------------------------------------
inline int elem_size(int32_t dtype) { return dtype == RT_DT_F32 ? 4 : 2; }
inline bool bad_type(int32_t dtype) { return dtype != RT_DT_F32 && dtype != RT_DT_BF16 && dtype != RT_DT_F16; }

inline const char* logits_fault(const rt_cat_logits* l) {
    if (!l || !l->x) return "NULL logits";
    if (bad_type(l->dtype)) return "logits type is not one of RT_DT_*";
    if (l->rows < 1 || l->rows > INT32_MAX) return "rows out of range";
    if (l->vocab < 1 || l->vocab > RT_CAT_MAX_VOCAB) return "vocab out of range";
    if (l->row_stride < 0) return "negative row stride";
    if (l->row_stride > INT64_MAX / 16 / l->rows) return "row stride out of range";
    if ((uintptr_t)l->x % elem_size(l->dtype)) return "logits not aligned to their element";
    return nullptr;
}

inline int launched() {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? RT_OK : rt_internal_fail(RT_ELAUNCH, hipGetErrorString(e));
}

}  // namespace rtcat
