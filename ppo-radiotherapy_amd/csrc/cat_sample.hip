// cat_sample.hip -- one action per row of logits from given random numbers,
// under temperature, top-k, top-p and min-p.
//
// Which entry a number falls to is decided at borders between sums of
// exponentials, so the weights are whole numbers, w = 2^40 exp((x - m) / T)
// rounded: their sums are exact in 64 bits (vocab <= 2^20), the same in every
// order, and atomics on them change nothing.
//
// The three filters are prefixes of one order (falling logits, equal ones by
// index), so their intersection is the shortest of them: a least key, and
// where entries equal to it are cut apart, a last index.  The key is found
// digit by digit from a histogram of the entries (top-k) or of their weights
// (top-p) in LDS; then the running weight by index is searched segment by
// segment.
#include <string>

#include "cat_rows.h"

namespace {

using namespace rtcat;

constexpr double kUnit = 1099511627776.0;  // 2^40
constexpr int kBins = 2048;                // of one digit: 11 bits

struct Args {
    const void* x;
    int64_t stride;
    int32_t vocab;
    rt_cat_sampling p;
    int64_t* action;
    float *logprob, *kept;
};

// Keys order like the numbers: -0 as +0, no NaN.
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float of_key(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}

struct Weigher {
    double m, inv_t;
    __device__ __forceinline__ uint64_t operator()(float x) const {
        return x == -INFINITY ? 0 : (uint64_t)rint(exp(((double)x - m) * inv_t) * kUnit);
    }
};

template <int THREADS>
struct Shared {
    uint64_t hist[kBins];
    uint64_t slots[THREADS / 64];
    float fslots[THREADS / 64];
    uint64_t found[2];
    int32_t where;
};

// The bin, from the highest down, in which a running sum reaches `want`
// (want >= 1 and <= the sum of all bins): the bin, and the sum above it.
template <int THREADS>
__device__ int find_bin(Shared<THREADS>& s, uint64_t want, uint64_t* above) {
    constexpr int kPer = kBins / THREADS;
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    uint64_t mine = 0;  // thread 0 has the highest bins
#pragma unroll
    for (int i = 0; i < kPer; ++i) mine += s.hist[kBins - 1 - (tid * kPer + i)];
    uint64_t run = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint64_t v = __shfl_up(run, o);
        if (lane >= o) run += v;
    }
    if (lane == 63) s.slots[w] = run;
    __syncthreads();
    uint64_t before = run - mine;
    for (int i = 0; i < w; ++i) before += s.slots[i];
    if (before < want && want <= before + mine) {
        for (int i = 0; i < kPer; ++i) {
            const int b = kBins - 1 - (tid * kPer + i);
            const uint64_t h = s.hist[b];
            if (want <= before + h) {
                s.where = b;
                s.found[0] = before;
                break;
            }
            before += h;
        }
    }
    __syncthreads();
    *above = s.found[0];
    const int b = s.where;
    __syncthreads();
    return b;
}

// The key at which the running sum of `weight` over falling keys reaches
// `want`, and the sum above that key.  `weight` is 0 for entries that do not
// take part.
template <int THREADS, bool SHORT, class Get, class Weight>
__device__ uint32_t find_key(Shared<THREADS>& s, int32_t V, Get get, Weight weight, uint64_t want, uint64_t* above) {
    uint32_t prefix = 0;
    uint64_t over = 0;
    // 16-bit types fill the upper 21 bits of a key at most: the last digit follows from the sign
    for (int level = 0; level < (SHORT ? 2 : 3); ++level) {
        const int shift = level == 0 ? 21 : level == 1 ? 10 : 0, bits = level == 2 ? 10 : 11;
        for (int i = threadIdx.x; i < kBins; i += THREADS) s.hist[i] = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < V; i += THREADS) {
            const float x = get(i);
            const uint32_t k = key_of(x);
            if (level && (k >> (shift + bits)) != prefix) continue;
            const uint64_t w = weight(x, k);
            if (w) atomicAdd(reinterpret_cast<unsigned long long*>(&s.hist[(k >> shift) & ((1u << bits) - 1)]), (unsigned long long)w);
        }
        __syncthreads();
        uint64_t a;
        const int b = find_bin<THREADS>(s, want - over, &a);
        over += a;
        prefix = prefix << bits | (uint32_t)b;
    }
    if (SHORT) prefix = prefix << 10 | (prefix >> 21 ? 0u : 0x3ffu);
    *above = over;
    return prefix;
}

// The entry, by index, at which the running sum of `weight` first exceeds
// `target` (target < the sum of all): the block halves its way down, each wave
// summing a part of the segment that holds it.
template <int THREADS, class Weight>
__device__ int32_t find_index(Shared<THREADS>& s, int32_t V, Weight weight, uint64_t target) {
    constexpr int kWaves = THREADS / 64;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    int32_t lo = 0, len = V;
    while (len > 64) {
        const int32_t part = (len + kWaves - 1) / kWaves;
        const int32_t a = min(lo + w * part, lo + len), b = min(a + part, lo + len);
        uint64_t sum = 0;
        for (int32_t i = a + lane; i < b; i += 64) sum += weight(i);
        sum = wave_sum(sum);
        if (lane == 0) s.slots[w] = sum;
        __syncthreads();
        uint64_t before = 0;
        int at = 0;
        for (; at < kWaves - 1; ++at) {
            if (target < before + s.slots[at]) break;
            before += s.slots[at];
        }
        __syncthreads();
        target -= before;
        const int32_t from = min(lo + at * part, lo + len);
        len = min(part, lo + len - from);
        lo = from;
    }
    // one wave's worth: all waves do the same
    uint64_t run = lane < len ? weight(lo + lane) : 0;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint64_t v = __shfl_up(run, o);
        if (lane >= o) run += v;
    }
    const uint64_t over = __ballot(lane < len && run > target);
    return lo + (over ? __ffsll((long long)over) - 1 : len - 1);
}

template <class D, int THREADS>
__global__ __launch_bounds__(THREADS) void k_cat_sample(Args A) {
    __shared__ Shared<THREADS> s;
    constexpr bool kShort = sizeof(typename D::raw) == 2;
    const int64_t n = blockIdx.x;
    const int32_t V = A.vocab;
    const auto* row = static_cast<const typename D::raw*>(A.x) + n * A.stride;
    const auto get = [&](int32_t i) { return D::get(row[i]); };
    const float T = A.p.temperature ? A.p.temperature[n] : A.p.temperature_all;
    const int32_t K = A.p.top_k ? A.p.top_k[n] : A.p.top_k_all;
    const float P = A.p.top_p ? A.p.top_p[n] : A.p.top_p_all;
    const float Q = A.p.min_p ? A.p.min_p[n] : A.p.min_p_all;

    float m = -INFINITY;
    uint32_t odd = 0;
    for (int i = threadIdx.x; i < V; i += THREADS) {
        const float v = get(i);
        m = fmaxf(m, v);
        odd |= v != v || v == INFINITY;
    }
    m = block_max<THREADS>(m, s.fslots);
    odd = (uint32_t)__syncthreads_or((int)odd);
    if (odd || m == -INFINITY) {
        if (threadIdx.x == 0) {
            A.action[n] = -1;
            A.logprob[n] = A.kept[n] = NAN;
        }
        return;
    }
    if (!(T > 0.0f)) {
        const uint32_t top = key_of(m);
        const int32_t a = find_index<THREADS>(s, V, [&](int32_t i) { return (uint64_t)(key_of(get(i)) == top); }, 0);
        if (threadIdx.x == 0) {
            A.action[n] = a;
            A.logprob[n] = A.kept[n] = 0.0f;
        }
        return;
    }
    const Weigher weigh{(double)m, 1.0 / (double)T};
    uint64_t all = 0;
    for (int i = threadIdx.x; i < V; i += THREADS) all += weigh(get(i));
    all = block_sum<THREADS>(all, s.slots);

    // the least key that is kept, and how many of the entries equal to it
    uint32_t cut = 0;
    uint64_t ties = UINT64_MAX, mass = all;
    if (K > 0 && K < V) {
        uint64_t above;
        cut = find_key<THREADS, kShort>(s, V, get, [](float, uint32_t) { return (uint64_t)1; }, (uint64_t)K, &above);
        ties = (uint64_t)K - above;
        mass = 0;
        if (P < 1.0f) {
            for (int i = threadIdx.x; i < V; i += THREADS)
                if (key_of(get(i)) > cut) mass += weigh(get(i));
            mass = block_sum<THREADS>(mass, s.slots) + ties * weigh(of_key(cut));
        }
    }
    if (P < 1.0f) {
        const double part = ceil((double)P * (double)mass);
        const uint64_t want = part >= 1.0 ? (uint64_t)part : 1;
        const uint32_t from = cut;
        uint64_t above;
        const uint32_t k = find_key<THREADS, kShort>(
            s, V, get, [&](float x, uint32_t key) { return key >= from ? weigh(x) : 0; }, want, &above);
        const uint64_t w = weigh(of_key(k));
        const uint64_t need = (want - above + w - 1) / w;
        if (k > cut || need < ties) ties = need;
        cut = k;
    }
    const double theta = Q >= 1.0f ? 0.0 : Q > 0.0f ? (double)T * log((double)Q) : -INFINITY;
    // entries equal to the cut: the last index that is kept
    int32_t last = V;
    if (ties != UINT64_MAX) {
        uint64_t equal = 0;
        for (int i = threadIdx.x; i < V; i += THREADS) equal += key_of(get(i)) == cut;
        equal = block_sum<THREADS>(equal, s.slots);
        if (ties < equal)
            last = find_index<THREADS>(s, V, [&](int32_t i) { return (uint64_t)(key_of(get(i)) == cut); }, ties - 1);
    }
    const auto kept = [&](int32_t i) -> uint64_t {
        const float x = get(i);
        const uint32_t k = key_of(x);
        if (k < cut || (k == cut && i > last) || (double)x - (double)m < theta) return 0;
        return weigh(x);
    };
    uint64_t left = 0;
    for (int i = threadIdx.x; i < V; i += THREADS) left += kept(i);
    left = block_sum<THREADS>(left, s.slots);
    const float u = A.p.u[n];
    const double hit = floor((u > 0.0f ? (double)u : 0.0) * (double)left);
    const uint64_t target = hit < (double)left ? (uint64_t)hit : left - 1;
    const int32_t a = find_index<THREADS>(s, V, kept, target < left ? target : left - 1);
    if (threadIdx.x == 0) {
        const double z = ((double)get(a) - (double)m) / (double)T;
        A.action[n] = a;
        A.logprob[n] = (float)(z - log((double)all / kUnit));
        A.kept[n] = (float)(z - log((double)left / kUnit));
    }
}

template <class D>
int run_sample(const Args& a, int64_t rows, hipStream_t st) {
    if (a.vocab > 4096)
        hipLaunchKernelGGL((k_cat_sample<D, 1024>), dim3((unsigned)rows), dim3(1024), 0, st, a);
    else
        hipLaunchKernelGGL((k_cat_sample<D, 256>), dim3((unsigned)rows), dim3(256), 0, st, a);
    return launched();
}

int bad(const char* what) { return rt_internal_fail(RT_EINVAL, (std::string("rt_cat_sample: ") + what).c_str()); }

}  // namespace

extern "C" int64_t rt_cat_sample_workspace_bytes(int64_t rows, int32_t vocab, int32_t dtype) {
    if (rows < 1 || rows > INT32_MAX || vocab < 1 || vocab > RT_CAT_MAX_VOCAB || bad_type(dtype)) return -1;
    return 0;
}

extern "C" int rt_cat_sample(const rt_cat_logits* logits, const rt_cat_sampling* params, int64_t* action_d,
                             float* logprob_d, float* kept_logprob_d, void* workspace_d, int64_t workspace_bytes,
                             void* stream) {
    if (const char* f = logits_fault(logits)) return bad(f);
    if (!params || !params->u) return bad("NULL parameters");
    if (!action_d || !logprob_d || !kept_logprob_d) return bad("NULL output");
    const int64_t need = rt_cat_sample_workspace_bytes(logits->rows, logits->vocab, logits->dtype);
    if (need > 0 && (!workspace_d || (uintptr_t)workspace_d % 16 || workspace_bytes < need))
        return bad("workspace NULL, not 16-B aligned or too small");
    const Args a{logits->x, logits->row_stride, logits->vocab, *params, action_d, logprob_d, kept_logprob_d};
    const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    if (logits->dtype == RT_DT_F32) return run_sample<F32>(a, logits->rows, st);
    if (logits->dtype == RT_DT_BF16) return run_sample<BF16>(a, logits->rows, st);
    return run_sample<F16>(a, logits->rows, st);
}
