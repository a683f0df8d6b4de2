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
// where entries equal to it are cut apart, a last index.
//
// By the row's length: a lane has a row of up to 32 entries; a team of 64 to
// 1024 threads holds one of up to 9216 in registers; a longer one is shared by
// blocks.  There bf16 rows go by counts of each number (two launches, one pass
// over the row and a second one over a part of it), f32 and f16 rows by bins
// (four launches, three passes).
#include <algorithm>
#include <string>
#include <type_traits>

#include "cat_rows.h"

namespace {

using namespace rtcat;

constexpr int kBins = 2048;  // of a histogram; 11 bits of a key
constexpr int kList = 4096;  // entries around a cut that a block can have

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

// 2^40 2^((x - m) c), c = log2(e) / T, as a whole number.  The product's whole
// part n comes of its sum with 1.5 2^52 and is added to the exponent; 2^40 e^(f
// ln 2), |f| <= 1/2, is the Taylor sum up to f^11 (within 7e-15 of it); the sum
// with 2^52 rounds to a whole number, half to even, that its low bits hold.
constexpr double kUnit = 1099511627776.0;  // 2^40
struct Weigher {
    double m, c, least;  // least: of x - m, where nothing is left of the weight
    __device__ Weigher(double m, double c) : m(m), c(c), least(-1000.0 / c) {}
    __device__ __forceinline__ uint64_t operator()(float x) const {
        const double kWhole = 6755399441055744.0;  // 1.5 2^52
        const double d = fmax((double)x - m, least), t = fma(d, c, kWhole), f = fma(d, c, kWhole - t);
        double p = kUnit * 4.44553827187081e-10;  // (ln 2)^11 / 11!, and so on down
        p = fma(p, f, kUnit * 7.054911620801121e-09);
        p = fma(p, f, kUnit * 1.0178086009239696e-07);
        p = fma(p, f, kUnit * 1.3215486790144305e-06);
        p = fma(p, f, kUnit * 1.5252733804059838e-05);
        p = fma(p, f, kUnit * 0.00015403530393381606);
        p = fma(p, f, kUnit * 0.0013333558146428441);
        p = fma(p, f, kUnit * 0.009618129107628477);
        p = fma(p, f, kUnit * 0.055504108664821576);
        p = fma(p, f, kUnit * 0.2402265069591007);
        p = fma(p, f, kUnit * 0.6931471805599453);
        p = fma(p, f, kUnit);
        const uint64_t n = (uint64_t)(uint32_t)__builtin_bit_cast(uint64_t, t) << 52;  // modulo 2^64, as the exponent is
        const double w = __builtin_bit_cast(double, __builtin_bit_cast(uint64_t, p) + n);
        return __builtin_bit_cast(uint64_t, w + 4503599627370496.0) - 0x4330000000000000ull;
    }
};

template <int THREADS>
struct Shared {
    uint64_t hist[kBins];
    uint64_t slots[THREADS / 64];
    uint64_t found[2];
    int32_t where;
};

// The bin, from the highest down, in which a running sum reaches `want` (want
// >= 1 and <= the sum of all bins): the bin, and the sum above it.
template <int THREADS>
__device__ int find_bin(Shared<THREADS>& s, uint64_t want, uint64_t* above) {
    constexpr int kPer = kBins / THREADS;
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    uint64_t mine = 0;
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

// A wave's part of a row, in the order of the index: whole pieces, the first
// wave also what lies before them, the last what lies behind.
template <class D>
struct Part {
    int32_t from, to, first, last;  // pieces; entries
    __device__ Part(const Span<D>& row, int32_t V, int w, int waves) {
        const int32_t per = (row.pieces + waves - 1) / waves;
        from = min(w * per, row.pieces);
        to = min(from + per, row.pieces);
        first = w == 0 ? 0 : row.head + from * Span<D>::kPer;
        last = w == waves - 1 ? V : row.head + to * Span<D>::kPer;
    }
};

// f(x, i) for every entry of a part; the lanes of one wave together, kAhead
// pieces at a time, -inf where a lane has none.  `skip` says of a maximum
// whether all that is not above it can be left out.
struct Never {
    __device__ __forceinline__ bool operator()(float) const { return false; }
};
template <int kAhead, class D, class F, class Skip = Never>
__device__ __forceinline__ void walk(const Span<D>& row, const Part<D>& p, F f, Skip skip = Skip()) {
    const int lane = threadIdx.x & 63;
    constexpr int kPer = Span<D>::kPer;
    const int32_t a = row.head + p.from * kPer, b = row.head + p.to * kPer;
    if (p.first < a) f(p.first + lane < a ? D::get(row.x[p.first + lane]) : -INFINITY, p.first + lane);
    if (b < p.last) f(b + lane < p.last ? D::get(row.x[b + lane]) : -INFINITY, b + lane);
    for (int32_t at = p.from; at < p.to; at += 64 * kAhead) {
        const int32_t i = at + lane;
        uint4 r[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) r[k] = i + 64 * k < p.to ? row.piece(i + 64 * k) : nothing<D>();
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            const Unpack<D> x(r[k]);
            if constexpr (!std::is_same_v<Skip, Never>)
                if (!__any(!skip(x.max()))) continue;
#pragma unroll
            for (int j = 0; j < kPer; ++j) f(x.v[j], row.head + (i + 64 * k) * kPer + j);
        }
    }
}

// The key at which the running sum of `weight` over falling keys reaches
// `want`, and the sum above that key, digit by digit.  `weight` is 0 for
// entries that do not take part.
template <class D, int THREADS, class Weight>
__device__ __forceinline__ uint32_t find_key(Shared<THREADS>& s, const Span<D>& row, const Part<D>& part, Weight weight,
                                             uint64_t want, uint64_t* above) {
    constexpr bool kShort = sizeof(typename D::raw) == 2;
    uint32_t prefix = 0;
    uint64_t over = 0;
    // 16-bit types fill the upper 22 bits of a key at most: the last digit follows from the sign
#pragma unroll 1
    for (int level = 0; level < (kShort ? 2 : 3); ++level) {
        const int shift = level == 0 ? 21 : level == 1 ? 10 : 0, bits = level == 2 ? 10 : 11;
        for (int i = threadIdx.x; i < kBins; i += THREADS) s.hist[i] = 0;
        __syncthreads();
        walk<1>(row, part, [&](float x, int32_t i) {
            const uint32_t k = key_of(x);
            const uint64_t w = level && (k >> (shift + bits)) != prefix ? 0 : weight(x, k, i);
            const int b = (int)(k >> shift & ((1u << bits) - 1));
            const uint64_t who = __ballot(w != 0);
            if (!who) return;
            // equal logits are what brings a row here: one addition where all lanes have one bin
            if (__all(!w || b == __shfl(b, __ffsll((long long)who) - 1))) {
                const uint64_t sum = wave_sum(w);
                if (__ffsll((long long)who) - 1 == (int)(threadIdx.x & 63))
                    atomicAdd(reinterpret_cast<unsigned long long*>(&s.hist[b]), (unsigned long long)sum);
            } else if (w) {
                atomicAdd(reinterpret_cast<unsigned long long*>(&s.hist[b]), (unsigned long long)w);
            }
        });
        __syncthreads();
        uint64_t a;
        const int b = find_bin<THREADS>(s, want - over, &a);
        over += a;
        prefix = prefix << bits | (uint32_t)b;
    }
    if (kShort) prefix = prefix << 10 | (prefix >> 21 ? 0u : 0x3ffu);
    *above = over;
    return prefix;
}

// The entry, by index, at which the running sum of `weight` first exceeds
// `target` (target < the sum of all): the block halves its way down, each wave
// summing a part of the segment that holds it.
template <int THREADS, class Weight>
__device__ int32_t find_index(Shared<THREADS>& s, int32_t lo, int32_t len, Weight weight, uint64_t target) {
    constexpr int kWaves = THREADS / 64;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
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

// What a row is asked for.
struct Ask {
    float T, P, Q, u;
    int32_t K;
    __device__ Ask(const rt_cat_sampling& p, int64_t n, int32_t V)
        : T(p.temperature ? p.temperature[n] : p.temperature_all), P(p.top_p ? p.top_p[n] : p.top_p_all),
          Q(p.min_p ? p.min_p[n] : p.min_p_all), u(p.u[n]), K(p.top_k ? p.top_k[n] : p.top_k_all) {
        if (K >= V) K = 0;
    }
    __device__ double least() const {  // of x - m
        return Q >= 1.0f ? 0.0 : Q > 0.0f ? (double)T * log((double)Q) : -INFINITY;
    }
    __device__ uint64_t limit(uint64_t mass) const {  // of the weight before the last that top-p keeps
        const double part = ceil((double)P * (double)mass);
        return part >= 1.0 ? (uint64_t)part : 1;
    }
    __device__ uint64_t target(uint64_t left) const {
        const double hit = floor((u > 0.0f ? (double)u : 0.0) * (double)left);
        const uint64_t t = hit < (double)left ? (uint64_t)hit : left - 1;
        return t < left ? t : left - 1;
    }
};

__device__ __forceinline__ void answer(const Args& A, int64_t n, int32_t a, double z, uint64_t all, uint64_t left) {
    A.action[n] = a;
    A.logprob[n] = (float)(z - log((double)all / kUnit));
    A.kept[n] = (float)(z - log((double)left / kUnit));
}

// ---- any row, slowly -------------------------------------------------------
// By one block, the key digit by digit from a histogram over the whole row: for
// f32 and f16 rows whose cut falls among more entries than a list holds (many
// equal logits, a very large k) and for temperatures past the bins' range.
// 780 us for a row of 131072 equal f32 logits under top-k and top-p, where the
// entries add to one place of LDS.
template <class D, int THREADS>
__device__ __forceinline__ void slow_row(const Args& A, int64_t n, const Ask& ask, float m, Shared<THREADS>& s) {
    const int32_t V = A.vocab;
    const Span<D> row(static_cast<const typename D::raw*>(A.x) + n * A.stride, V);
    const Part<D> part(row, V, threadIdx.x >> 6, THREADS / 64);
    const Weigher weigh((double)m, fmax(1.4426950408889634 / (double)ask.T, 1e-300));
    const auto sum = [&](auto f) {
        uint64_t v = 0;
        walk<1>(row, part, [&](float x, int32_t i) { v += f(x, i); });
        return block_sum<THREADS>(v, s.slots);
    };
    // the entry at which the running sum of f, by index, first exceeds `target`: its wave's part, then there
    const auto search = [&](auto f, uint64_t target) {
        uint64_t v = 0;
        walk<1>(row, part, [&](float x, int32_t i) { v += f(x, i); });
        v = wave_sum(v);
        if ((threadIdx.x & 63) == 0) s.slots[threadIdx.x >> 6] = v;
        __syncthreads();
        int w = 0;
        for (; w < THREADS / 64 - 1 && target >= s.slots[w]; ++w) target -= s.slots[w];
        __syncthreads();
        const Part<D> p(row, V, w, THREADS / 64);
        return find_index<THREADS>(s, p.first, p.last - p.first, [&](int32_t i) { return f(D::get(row.x[i]), i); }, target);
    };
    const uint64_t all = sum([&](float x, int32_t) { return weigh(x); });

    // the least key that is kept, and how many of the entries equal to it
    uint32_t cut = 0;
    uint64_t ties = UINT64_MAX, mass = all, above;
    if (ask.K > 0) {
        cut = find_key<D, THREADS>(s, row, part, [&](float x, uint32_t, int32_t) { return (uint64_t)(x > -INFINITY); },
                                   min((uint64_t)ask.K, sum([](float x, int32_t) { return (uint64_t)(x > -INFINITY); })), &above);
        ties = (uint64_t)ask.K - above;
        if (ask.P < 1.0f)
            mass = sum([&](float x, int32_t) { return key_of(x) > cut ? weigh(x) : 0; }) +
                   min(ties, sum([&](float x, int32_t) { return (uint64_t)(key_of(x) == cut); })) * weigh(of_key(cut));
    }
    if (ask.P < 1.0f) {
        const uint64_t want = ask.limit(mass);
        const uint32_t from = cut;
        const uint32_t k = find_key<D, THREADS>(
            s, row, part, [&](float x, uint32_t key, int32_t) { return key >= from ? weigh(x) : 0; }, want, &above);
        const uint64_t w = weigh(of_key(k));
        const uint64_t need = (want - above + w - 1) / w;
        if (k > cut || need < ties) ties = need;
        cut = k;
    }
    const double theta = ask.least();
    // entries equal to the cut: the last index that is kept
    int32_t last = V;
    if (ties != UINT64_MAX && ties < sum([&](float x, int32_t) { return (uint64_t)(key_of(x) == cut); }))
        last = search([&](float x, int32_t) { return (uint64_t)(key_of(x) == cut); }, ties - 1);
    const auto kept = [&](float x, int32_t i) -> uint64_t {
        const uint32_t k = key_of(x);
        return k < cut || (k == cut && i > last) || (double)x - (double)m < theta ? 0 : weigh(x);
    };
    const uint64_t left = sum(kept);
    const int32_t a = search(kept, ask.target(left));
    if (threadIdx.x == 0) answer(A, n, a, ((double)D::get(row.x[a]) - (double)m) / (double)ask.T, all, left);
}

// An entry's place in the order, larger first: key, then index from below.
__device__ __forceinline__ uint64_t rank_of(float x, int32_t i) { return (uint64_t)key_of(x) << 32 | (uint32_t)~i; }

// Bins of falling logits, by t = (m - x) / (T ln 2): the last holds what weighs
// nothing (2^(40 - 41.5) < 1/2).  Each step of the arithmetic keeps the order,
// so a bin's entries come before those of the next.
struct Binner {
    float m, scale, last;
    __device__ __forceinline__ int operator()(float x) const { return (int)fminf((m - x) * scale, last); }
    // the least number whose bin is not behind b >= 0, by a wave: 64 keys at a time
    __device__ uint32_t least_key(int b) const {
        uint32_t lo = 0x00800000u, hi = key_of(m);  // from the lowest finite one
        while (lo < hi) {
            const uint32_t step = (hi - lo) / 64 + 1;
            const uint32_t k = min((uint64_t)hi, lo + (uint64_t)step * (threadIdx.x & 63));
            const uint64_t reached = __ballot((*this)(of_key(k)) <= b);
            const int first = reached ? __ffsll((long long)reached) - 1 : 64;
            const uint32_t below = lo + step * (uint32_t)(first - 1);
            if (first == 0) return lo;
            if (first < 64) hi = (uint32_t)min((uint64_t)hi, (uint64_t)below + step);
            lo = below + 1;
        }
        return lo;
    }
    // the numbers of bins [from, to], which are not empty of numbers
    __device__ void range(int from, int to, float* least, float* most) const {
        *least = of_key(least_key(to));
        *most = from > 0 ? of_key(least_key(from - 1) - 1) : m;
    }
};

constexpr float kMostT = 1e30f;  // above, numbers that the bins cannot tell apart weigh something

// What is known of a row when its maximum is.
struct Head {
    float m;
    double c, theta;
    Weigher weigh;
    __device__ Head(const Ask& ask, float m)
        : m(m), c(fmax(1.4426950408889634 / (double)ask.T, 1e-300)), theta(ask.least()), weigh((double)m, c) {}
    __device__ __forceinline__ bool likely(float x) const { return !((double)x - (double)m < theta); }  // min-p keeps it
    // entries in bins before this one are kept by min-p, those two or more behind it are not: the bin of
    // the least logit, with one to spare for its rounding
    __device__ int sure_bin(const Binner& bin) const { return theta == -INFINITY ? kBins : max(bin((float)((double)m + theta)) - 1, 0); }
    // Bins 0 to `last` over what weighs something, or over `reach` where that is less.
    __device__ Binner binner(int last, float reach) const {
        const double scale = fmax(c / 41.5, 1.0 / (double)reach);  // reach 0: infinite, as it is clamped
        return Binner{m, (float)fmin(fmax(scale * last, 1e-30), 3e38), (float)last};
    }
};

__device__ __forceinline__ void no_answer(const Args& A, int64_t n) {
    A.action[n] = -1;
    A.logprob[n] = A.kept[n] = NAN;
}

template <class D, int THREADS>
__device__ void greedy(const Args& A, int64_t n, float m, int32_t lo, int32_t len, const Span<D>& row, Shared<THREADS>& s) {
    const uint32_t top = key_of(m);
    const int32_t a = find_index<THREADS>(s, lo, len, [&](int32_t i) { return (uint64_t)(key_of(D::get(row.x[i])) == top); }, 0);
    if (threadIdx.x == 0) {
        A.action[n] = a;
        A.logprob[n] = A.kept[n] = 0.0f;
    }
}

// Between a wave's accesses to LDS that other lanes of it made: they keep their
// order in the hardware, the compiler has to keep it too.
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// ---- the cut, among entries in registers -----------------------------------
// A team of one to sixteen waves, and what they tell each other.
template <int THREADS>
struct Team {
    static constexpr int kWaves = THREADS / 64;
    struct Slots { uint64_t v[2][kWaves]; };
    Slots& s;
    int turn = 0;  // two sets in turn: one barrier for each exchange

    __device__ explicit Team(Slots& s) : s(s) {}
    // v from every wave, combined
    template <class T, class Op>
    __device__ __forceinline__ T all(T v, Op op) {
        v = lanes<64>(v, op);
        if constexpr (kWaves > 1) {
            uint64_t* slot = s.v[turn];
            turn ^= 1;
            if ((threadIdx.x & 63) == 0) slot[threadIdx.x >> 6] = (uint64_t)v;
            __syncthreads();
            v = (T)slot[0];
#pragma unroll
            for (int i = 1; i < kWaves; ++i) v = op(v, (T)slot[i]);
        }
        return v;
    }
    template <class T>
    __device__ __forceinline__ T sum(T v) {
        return all(v, [](T a, T b) { return a + b; });
    }
    __device__ __forceinline__ uint32_t top(uint32_t v) {
        return all(v, [](uint32_t a, uint32_t b) { return max(a, b); });
    }
    __device__ __forceinline__ void sync() {
        if constexpr (kWaves > 1) __syncthreads();
        else wave_sync();
    }
    // the sum of the threads before this one; `total` of all
    __device__ __forceinline__ uint64_t before(uint64_t v, uint64_t* total) {
        const int lane = threadIdx.x & 63;
        uint64_t run = v;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const uint64_t q = __shfl_up(run, o);
            if (lane >= o) run += q;
        }
        uint64_t all = __shfl(run, 63), at = run - v;
        if constexpr (kWaves > 1) {
            uint64_t* slot = s.v[turn];
            turn ^= 1;
            if (lane == 0) slot[threadIdx.x >> 6] = all;
            __syncthreads();
            all = 0;
#pragma unroll
            for (int i = 0; i < kWaves; ++i) {
                if (i < (int)(threadIdx.x >> 6)) at += slot[i];
                all += slot[i];
            }
        }
        *total = all;
        return at;
    }
};

// A thread's entries: E of them, in registers; or every `step`-th of a list, in
// a loop that stays one (a kernel that runs once a row spends its time on
// fetching code).
template <int E>
struct Held {
    template <class F>
    __device__ __forceinline__ void operator()(F f) const {
#pragma unroll
        for (int e = 0; e < E; ++e) f(e);
    }
};
struct Listed {
    int from, to, step;
    template <class F>
    __device__ __forceinline__ void operator()(F f) const {
#pragma unroll 1
        for (int i = from; i < to; i += step) f(i);
    }
};

// The key at which the sum of value(e), over falling keys, reaches `want` (1 <=
// want <= the sum of all), and the sum above it.  A histogram by bin(e) (larger
// keys have no larger bin) says in which bin; there, the largest key that is
// left, and then the middle of what is left, each with its sum: most bins have
// an entry or two.  The first kMiddles middles are those of `middle`, which
// suits the bin; numbers next to 0 can be more than a hundred halvings apart,
// but any two keys are 32, so from then on the keys are halved, and the search
// ends in kMiddles + 33 steps.  hist: BINS places of LDS.
constexpr int kMiddles = 16;

template <int BINS, class K, class T, class Each, class Key, class Bin, class Value, class Middle>
__device__ __forceinline__ K team_key(T& team, uint64_t* hist, Each each, Key key, Bin bin, Value value, uint64_t want, Middle middle,
                                      uint64_t* above) {
    constexpr int kThreads = T::kWaves * 64, kPer = BINS / kThreads;
    const int t = threadIdx.x % kThreads;
#pragma unroll
    for (int i = 0; i < kPer; ++i) hist[t + i * kThreads] = 0;
    team.sync();
    each([&](int e) {
        if (const uint64_t v = value(e))
            atomicAdd(reinterpret_cast<unsigned long long*>(hist + bin(e)), (unsigned long long)v);
    });
    team.sync();
    uint64_t mine = 0, total;
#pragma unroll
    for (int i = 0; i < kPer; ++i) mine += hist[t * kPer + i];
    uint64_t at = team.before(mine, &total);
    uint32_t where = 0;
    uint64_t over = 0;
    if (at < want && want <= at + mine) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const uint64_t v = hist[t * kPer + i];
            if (at < want && want <= at + v) {
                where = t * kPer + i;
                over = at;
            }
            at += v;
        }
    }
    where = team.top(where);
    over = team.sum(over);
    // the sum of keys >= lo reaches `want`, that of keys >= hi does not
    K k = 0, lo = ~(K)0;
    each([&](int e) {
        const bool here = value(e) && (uint32_t)bin(e) == where;
        k = here ? max(k, key(e)) : k;
        lo = here ? min(lo, key(e)) : lo;
    });
    k = team.all(k, [](K a, K b) { return max(a, b); });
    lo = team.all(lo, [](K a, K b) { return min(a, b); });
    const auto from = [&](K least) {
        uint64_t s = 0;
        each([&](int e) { s += key(e) >= least ? value(e) : 0; });
        return team.sum(s);
    };
    for (int step = 0; step < kMiddles + 33; ++step) {
        uint64_t sum = from(k);
        if (sum >= want) {
            *above = over;
            return k;
        }
        K hi = k;
        over = sum;
        K mid = middle(lo, hi);
        if (step >= kMiddles || mid <= lo || mid >= hi) mid = lo + (hi - lo) / 2;  // lo <= mid < hi
        sum = from(mid);
        if (sum >= want) {
            lo = mid;
        } else {
            hi = mid;
            over = sum;
        }
        k = 0;
        each([&](int e) { k = key(e) < hi ? max(k, key(e)) : k; });
        k = team.all(k, [](K a, K b) { return max(a, b); });
    }
    *above = over;  // (not reached)
    return lo;
}

// The key half way between the numbers of two keys (those around 0 have most of
// the keys).
__device__ __forceinline__ uint32_t middle_key(uint32_t lo, uint32_t hi) {
    return key_of(0.5f * of_key(lo) + 0.5f * of_key(hi));
}

// ---- long rows of f32 and f16, by parts ------------------------------------
// Up to 64 blocks share a row, one launch for each thing that all of it has to
// be known for: the maximum; the weights, and a histogram of them where there
// is a cut to find; the entries around the cut; the answer, by one block.
// 63 x 50021 f32, top-p: 5 + 13 + 11 + 15 us, 43 together (f16 46; 12.6 MB: 2.5 us of
// HBM).  The weights are bound by f64 arithmetic and LDS additions, the others
// by the trips to memory and barriers that follow one another.
constexpr int kParts = 64, kPartWaves = 4;

struct RowSpace {
    float top[kParts], low[kParts];             // largest (NaN: a NaN or +inf) and least finite logit
    uint64_t all[kParts * kPartWaves];          // the weight of each wave's part
    uint64_t kept[kParts * kPartWaves];         // what of it is surely kept
    uint64_t coarse[kParts][64];                // the histogram of each part by 32 bins
    uint64_t list[kList];
    int32_t many, pad[15];
};
constexpr int kCoarse = kBins / 64;

struct Batch {
    Args a;
    RowSpace* space;  // of row `first`
    uint64_t* hist;   // [row][part][kBins]
    int64_t first;
    int32_t parts;
};

// The maximum of the row, and how far its least finite logit is below; from
// those of its parts, by each wave.  NaN for a row without an answer.
struct Extent {
    float m, reach;
    __device__ __forceinline__ Extent(const RowSpace& r, int32_t parts) {
        const int lane = threadIdx.x & 63;
        const float top = lane < parts ? r.top[lane] : -INFINITY, low = lane < parts ? r.low[lane] : INFINITY;
        m = wave_max(top);
        reach = m + wave_max(-low);
        if (__any(top != top) || m == -INFINITY) m = NAN;
    }
};

__device__ __forceinline__ bool cuts(const Ask& ask) { return ask.K > 0 || ask.P < 1.0f; }

// The lane at which the running sum of v reaches `want`, and the sum before it.
__device__ __forceinline__ int lane_of(uint64_t v, uint64_t want, uint64_t* before) {
    uint64_t run = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint64_t q = __shfl_up(run, o);
        if ((int)(threadIdx.x & 63) >= o) run += q;
    }
    const int lane = __ffsll((long long)__ballot(run >= want)) - 1;
    *before = __shfl(run - v, lane);
    return lane;
}

// Where the cut falls: its bin, what is wanted, the sum before the bin and in
// it.
struct Near {
    int bin;
    uint64_t want, before, in;
    // whether a list can hold what has to be in it
    __device__ bool fits(const Ask& ask) const { return ask.K <= 0 || before + in <= kList; }
};

// By the whole block: 64 coarse bins, then the 32 of one, each the sum of all
// parts (which write their own: adding them up in memory took longer).  Every
// thread has a bin of every THREADS / 64-th part, or / 32-nd.
template <int THREADS>
struct NearRoom {
    uint64_t sums[THREADS];
    Near near;
};

template <int THREADS>
__device__ __forceinline__ void find_near(const Ask& ask, const RowSpace& r, const uint64_t* hist, int32_t parts,
                                          NearRoom<THREADS>& room) {
    const int tid = threadIdx.x, lane = tid & 63;
    Near n;
    uint64_t v = 0, more;
#pragma unroll 4
    for (int p = tid / 64; p < parts; p += THREADS / 64) v += r.coarse[p][lane];
    room.sums[tid] = v;
    __syncthreads();
    if (tid < 64) {
        v = 0;
#pragma unroll
        for (int i = 0; i < THREADS / 64; ++i) v += room.sums[i * 64 + lane];
        // entries that weigh nothing are not in the histogram: they stand behind all others, and keeping
        // them or not changes nothing
        n.want = ask.K > 0 ? min((uint64_t)ask.K, wave_sum(v)) : ask.limit(wave_sum(v));
        n.bin = lane_of(v, n.want, &n.before) * kCoarse;
        if (tid == 0) room.near = n;
    }
    __syncthreads();
    n = room.near;
    v = 0;
#pragma unroll 4
    for (int p = tid / kCoarse; p < parts; p += THREADS / kCoarse) v += hist[p * kBins + n.bin + tid % kCoarse];
    room.sums[tid] = v;
    __syncthreads();
    if (tid < 64) {
        v = 0;
        if (lane < kCoarse)
#pragma unroll
            for (int i = 0; i < THREADS / kCoarse; ++i) v += room.sums[i * kCoarse + lane];
        const int f = lane_of(v, n.want - n.before, &more);
        n.bin += f;
        n.before += more;
        n.in = __shfl(v, f);
        if (tid == 0) room.near = n;
    }
    __syncthreads();
}

template <class D>
__global__ __launch_bounds__(256) void k_cat_sample_top(Batch b) {
    __shared__ float fs[4];
    const int64_t r = blockIdx.x / b.parts, n = b.first + r;
    const int32_t p = blockIdx.x % b.parts, V = b.a.vocab;
    const int w = threadIdx.x >> 6;
    const Span<D> row(static_cast<const typename D::raw*>(b.a.x) + n * b.a.stride, V);
    const Part<D> part(row, V, p * kPartWaves + w, b.parts * kPartWaves);
    RowSpace& to = b.space[r];
    float m = -INFINITY, low = INFINITY;
    int odd = 0;
    walk<2>(row, part, [&](float x, int32_t) {
        m = fmaxf(m, x);
        low = fminf(low, x == -INFINITY ? INFINITY : x);
        odd |= !(x < INFINITY);
    });
    m = block_max<256>(m, fs);
    low = -block_max<256>(-low, fs);
    odd = __syncthreads_or(odd);
    if (threadIdx.x == 0) {
        to.top[p] = odd ? NAN : m;
        to.low[p] = low;
        if (p == 0) to.many = 0;
    }
}

template <class D>
__global__ __launch_bounds__(256) void k_cat_sample_weigh(Batch b) {
    __shared__ uint64_t hist[kBins + 64];  // behind the bins, a place for each lane's entries that weigh nothing
    const int64_t r = blockIdx.x / b.parts, n = b.first + r;
    const int32_t p = blockIdx.x % b.parts, V = b.a.vocab;
    const int tid = threadIdx.x, w = tid >> 6, seg = p * kPartWaves + w;
    const Span<D> row(static_cast<const typename D::raw*>(b.a.x) + n * b.a.stride, V);
    const Part<D> part(row, V, seg, b.parts * kPartWaves);
    RowSpace& to = b.space[r];
    const Extent extent(to, b.parts);
    const float m = extent.m;
    const Ask ask(b.a.p, n, V);
    if (m != m || !(ask.T > 0.0f)) return;
    const Head h(ask, m);
    uint64_t all = 0, kept = 0;
    if (cuts(ask)) {
        const Binner bin = h.binner(kBins - 1, extent.reach);
        const bool count = ask.K > 0;
        for (int i = tid; i < kBins; i += 256) hist[i] = 0;
        __syncthreads();
        walk<2>(row, part, [&](float x, int32_t) {
            const uint64_t v = h.weigh(x);
            all += v;
            const int at = v ? bin(x) : kBins + (tid & 63);
            atomicAdd(reinterpret_cast<unsigned long long*>(&hist[at]), (unsigned long long)(count ? 1 : v));
        });
        __syncthreads();
        uint64_t* own = b.hist + (r * b.parts + p) * (int64_t)kBins;
#pragma unroll
        for (int i = tid; i < kBins; i += 256) {
            own[i] = hist[i];
            const uint64_t sum = lanes_sum<kCoarse>(hist[i]);
            if (i % kCoarse == 0) to.coarse[p][i / kCoarse] = sum;
        }
    } else {
        if (h.theta == -INFINITY) {
            walk<2>(row, part, [&](float x, int32_t) { all += h.weigh(x); });
            kept = all;
        } else {
            walk<2>(row, part, [&](float x, int32_t) {
                const uint64_t v = h.weigh(x);
                all += v;
                kept += h.likely(x) ? v : 0;
            });
        }
    }
    all = wave_sum(all);
    kept = wave_sum(kept);
    if ((tid & 63) == 0) {
        to.all[seg] = all;
        to.kept[seg] = kept;
    }
}

// Sum of n <= 256 numbers, by each wave for itself.
__device__ __forceinline__ uint64_t sum_of(const uint64_t* v, int n) {
    uint64_t s = 0;
    for (int i = threadIdx.x & 63; i < n; i += 64) s += v[i];
    return wave_sum(s);
}

template <class D>
__global__ __launch_bounds__(256) void k_cat_sample_near(Batch b) {
    constexpr int kOwn = 256;
    __shared__ NearRoom<256> room;
    __shared__ uint64_t own[kPartWaves][kOwn];  // a wave's entries, added to the row's list at once
    const int64_t r = blockIdx.x / b.parts, n = b.first + r;
    const int32_t p = blockIdx.x % b.parts, V = b.a.vocab;
    const int tid = threadIdx.x, w = tid >> 6, seg = p * kPartWaves + w;
    const Span<D> row(static_cast<const typename D::raw*>(b.a.x) + n * b.a.stride, V);
    const Part<D> part(row, V, seg, b.parts * kPartWaves);
    RowSpace& to = b.space[r];
    const Extent extent(to, b.parts);
    const float m = extent.m;
    const Ask ask(b.a.p, n, V);
    if (m != m || !(ask.T > 0.0f) || !cuts(ask) || ask.T > kMostT) return;
    const Head h(ask, m);
    const Binner bin = h.binner(kBins - 1, extent.reach);
    int many = 0;
    find_near<256>(ask, to, b.hist + r * b.parts * (int64_t)kBins, b.parts, room);
    const Near& near = room.near;
    if (!near.fits(ask)) return;
    const int at = near.bin;
    uint64_t kept = 0;
    // top-k: all up to the bin of the cut.  top-p: that bin; what stands before it is known by parts, but for
    // the bins where min-p cuts.  Bins as ranges of numbers: most entries are neither
    const int sure = h.sure_bin(bin);
    const bool last_bins = at > kBins - 64;  // where the weights end
    float low, high, low_p = INFINITY, high_p = -INFINITY;
    bin.range(ask.K > 0 ? 0 : at, at, &low, &high);
    if (ask.K <= 0 && min(sure + 2, at - 1) >= sure) bin.range(sure, min(sure + 2, at - 1), &low_p, &high_p);
    walk<2>(row, part, [&](float x, int32_t i) {
        const bool listed = x >= low && x <= high, split = x >= low_p && x <= high_p;
        if (!__any(listed || split)) return;
        // behind the entries of this wave: its lanes in turn
        const bool add = listed && (!last_bins || h.weigh(x));
        const uint64_t who = __ballot(add);
        if (add) {
            const int o = many + __popcll(who & ((1ull << (tid & 63)) - 1));
            if (o < kOwn) {
                own[w][o] = rank_of(x, i);
            } else {
                const int l = atomicAdd(&to.many, 1);
                if (l < kList) to.list[l] = rank_of(x, i);
            }
        }
        many += __popcll(who);
        if (split && h.likely(x)) kept += h.weigh(x);
    }, [&](float x) { return x < fminf(low, low_p); });
    kept = wave_sum(kept);
    if ((tid & 63) == 0) to.kept[seg] = kept;
    wave_sync();
    const int mine = min(many, kOwn);
    int first = 0;
    if ((tid & 63) == 0 && mine) first = atomicAdd(&to.many, mine);
    first = __shfl(first, 0);
    for (int i = tid & 63; i < mine; i += 64)
        if (first + i < kList) to.list[first + i] = own[w][i];
}

// Which of the equal shares of a row has an entry.
template <class D>
__device__ __forceinline__ int share_of(const Span<D>& row, int shares, int32_t i) {
    const int32_t per = (row.pieces + shares - 1) / shares, piece = (i - row.head) / Span<D>::kPer;
    return i < row.head ? 0 : piece >= row.pieces ? shares - 1 : piece / per;
}

// What is known at the end: the least rank that is kept, by top-p, or the answer.
struct Verdict {
    uint64_t cut;
    int32_t action;  // -1: still to be found
    float x;
    uint64_t left;
};

// What the block that answers has of a row.
template <int THREADS>
struct Room {
    uint64_t hist[kBins];
    uint64_t list[kList], weight[kList];  // ranks, and what of their weight is kept
    uint64_t segs[kParts * kPartWaves];   // the weight of what is kept, by shares of the row
    NearRoom<THREADS> near;
    Verdict verdict;
};

// From the list, by a team: top-k rows whole, of top-p rows the cut, and the
// weight of what the list has of the kept ones on to their shares of the row.
template <class D, int THREADS, int BINS, class R>
__device__ __forceinline__ Verdict settle(Team<THREADS>& team, R& room, const Ask& ask, const Head& h, int many,
                                          const Span<D>& row, int waves, int group, int32_t V) {
    const Near& near = room.near.near;
    const int t = threadIdx.x % THREADS;
    const Listed each{t, many, THREADS};
    const auto key = [&](int i) { return (uint32_t)(room.list[i] >> 32); };
    const auto turned = [&](int i) { return (uint32_t)room.list[i]; };  // by index, the first ones highest
    const auto weight = [&](int i) { return room.weight[i]; };
    uint32_t top = 0, low = UINT32_MAX;
    each([&](int i) {
        room.weight[i] = h.weigh(of_key(key(i)));
        top = max(top, key(i));
        low = min(low, key(i));
    });
    top = team.top(top);
    low = team.all(low, [](uint32_t a, uint32_t b) { return min(a, b); });
    const float first = of_key(top), reach = first - of_key(low);
    const Binner fine{first, reach > 0.0f ? fminf((float)(BINS - 1) / reach, 3e38f) : 0.0f, (float)(BINS - 1)};
    const auto place = [&](int i) { return fine(of_key(key(i))); };
    const int shift = max(0, 32 - __clz((uint32_t)V) - (31 - __clz(BINS)));  // V >> shift < BINS
    const auto slot = [&](int i) { return (int)(~turned(i) >> shift); };
    const auto middle = [](uint32_t lo, uint32_t hi) { return lo + (hi - lo) / 2; };
    uint64_t above, cut = 0;
    // Two rounds at most: by number, then by weight.  What is behind the cut loses its weight: smaller
    // keys, and of the entries equal to it all but the first `ties`.
#pragma unroll 1
    for (int round = ask.K > 0 ? 0 : 1; round < (ask.P < 1.0f ? 2 : 1); ++round) {
        uint64_t want = ask.K > 0 ? near.want : near.want - near.before;
        if (round == 1 && ask.K > 0) {
            uint64_t mass = 0;
            each([&](int i) { mass += weight(i); });
            want = ask.limit(team.sum(mass));
        }
        const auto value = [&](int i) { return round == 0 ? (uint64_t)(room.weight[i] != 0) : room.weight[i]; };
        // (a bin of 16-bit logits often has one number, many times)
        const uint32_t c = top == low ? (above = 0, top)
                                      : team_key<BINS, uint32_t>(team, room.hist, each, key, place, value, want, middle_key, &above);
        const uint64_t one = round == 0 ? 1 : h.weigh(of_key(c)), ties = (want - above + one - 1) / one;
        const auto tie = [&](int i) { return (uint64_t)(key(i) == c && room.weight[i]); };
        uint64_t equal = 0;
        each([&](int i) { equal += tie(i); });
        uint32_t last = 0;
        if (ties < team.sum(equal)) last = team_key<BINS, uint32_t>(team, room.hist, each, turned, slot, tie, ties, middle, &above);
        each([&](int i) {
            if (key(i) < c || (key(i) == c && turned(i) < last)) room.weight[i] = 0;
        });
        cut = (uint64_t)c << 32 | last;
    }
    uint64_t left = 0;
    each([&](int i) {
        if (!h.likely(of_key(key(i)))) room.weight[i] = 0;
        left += weight(i);
    });
    if (ask.K > 0) {  // all that is kept is here
        left = team.sum(left);
        const uint32_t found = team_key<BINS, uint32_t>(team, room.hist, each, turned, slot, weight, ask.target(left) + 1, middle, &above);
        uint32_t k = 0;
        each([&](int i) { k = turned(i) == found && weight(i) ? key(i) : k; });
        return Verdict{cut, (int32_t)~found, of_key(team.top(k)), left};
    }
    each([&](int i) {
        if (const uint64_t w = weight(i))
            atomicAdd(reinterpret_cast<unsigned long long*>(&room.segs[share_of(row, waves, (int32_t)~turned(i)) / group]),
                      (unsigned long long)w);
    });
    return Verdict{cut, -1, 0.0f, 0};
}

template <class D>
__global__ __launch_bounds__(512) void k_cat_sample_answer(Batch b) {
    constexpr int kThreads = 512;
    __shared__ Shared<kThreads> s;
    __shared__ Team<kThreads>::Slots slots;
    __shared__ Team<64>::Slots one;
    __shared__ Room<kThreads> room;
    uint64_t* const segs = room.segs;
    const int64_t n = b.first + blockIdx.x;
    const int32_t V = b.a.vocab, waves = b.parts * kPartWaves;
    const int tid = threadIdx.x;
    const Span<D> row(static_cast<const typename D::raw*>(b.a.x) + n * b.a.stride, V);
    const RowSpace& r = b.space[blockIdx.x];
    // one trip to memory for all of this
    const Extent extent(r, b.parts);
    const float m = extent.m;
    const Ask ask(b.a.p, n, V);
    const uint64_t v_all = tid < waves ? r.all[tid] : 0, v_kept = tid < waves ? r.kept[tid] : 0;
    const int many = r.many;
    if (m != m) {
        if (tid == 0) no_answer(b.a, n);
        return;
    }
    if (!(ask.T > 0.0f)) {
        int p = 0;
        while (p < b.parts - 1 && r.top[p] != m) ++p;
        const int32_t from = Part<D>(row, V, p * kPartWaves, waves).first;
        const int32_t to = Part<D>(row, V, (p + 1) * kPartWaves - 1, waves).last;
        return greedy<D, kThreads>(b.a, n, m, from, to - from, row, s);
    }
    const Head h(ask, m);
    Team<kThreads> team(slots);
    // top-p rows have the weight of what is kept by whole parts, others by each wave's
    const int group = ask.K <= 0 && ask.P < 1.0f ? kPartWaves : 1, shares = waves / group;
    if (group == 1) {
        if (tid < waves) segs[tid] = v_kept;
    } else {
        const uint64_t of_part = lanes_sum<kPartWaves>(v_kept);
        if (tid < waves && tid % kPartWaves == 0) segs[tid / kPartWaves] = of_part;
    }
    const uint64_t all = team.sum(v_all);
    Verdict v{0, -1, 0.0f, 0};
    if (cuts(ask)) {
        if (many <= kList)
            for (int i = tid; i < many; i += kThreads) room.list[i] = r.list[i];
        find_near<kThreads>(ask, r, b.hist + blockIdx.x * (int64_t)b.parts * kBins, b.parts, room.near);
        const Near& near = room.near.near;
        const int sure = h.sure_bin(h.binner(kBins - 1, extent.reach));
        if (ask.T > kMostT || !near.fits(ask) || many > kList) return slow_row<D, kThreads>(b.a, n, ask, m, s);
        __syncthreads();
        if (group > 1) {  // the bins before both cuts, of each part: whole coarse ones, and the rest
            const int end = min(near.bin, sure), coarse = end / kCoarse;
            const int lane = tid & 63;
            for (int p = tid >> 6; p < b.parts; p += kThreads / 64) {
                const uint64_t* fine = b.hist + (blockIdx.x * (int64_t)b.parts + p) * kBins + coarse * kCoarse;
                uint64_t known = lane < coarse ? r.coarse[p][lane] : 0;
                if (lane < end % kCoarse) known += fine[lane];
                known = wave_sum(known);
                if (lane == 0) segs[p] += known;
            }
        }
        __syncthreads();
        if (ask.K <= 0 && near.bin > sure + 2) {
            // min-p cuts before top-p does
        } else if (many <= 128) {  // one wave is faster than the barriers of eight
            if (tid < 64) {
                Team<64> wave(one);
                v = settle<D, 64, 256>(wave, room, ask, h, many, row, waves, group, V);
                if (tid == 0) room.verdict = v;
            }
            __syncthreads();
            v = room.verdict;
        } else {
            v = settle<D, kThreads, kBins>(team, room, ask, h, many, row, waves, group, V);
        }
    }
    if (v.action >= 0) {
        if (tid == 0) answer(b.a, n, v.action, ((double)v.x - (double)m) / (double)ask.T, all, v.left);
        return;
    }
    __syncthreads();
    const uint64_t left = sum_of(segs, shares);
    uint64_t target = ask.target(left);
    int at = 0;
    for (; at < shares - 1 && target >= segs[at]; ++at) target -= segs[at];
    // that share of the row, by waves, and one wave's of it in equal shares for the threads
    const auto weight = [&](float x, int32_t i) -> uint64_t { return rank_of(x, i) < v.cut || !h.likely(x) ? 0 : h.weigh(x); };
    const int32_t per_wave = (row.pieces + waves - 1) / waves, from_piece = min(at * group * per_wave, row.pieces);
    Part<D> p(row, V, at * group, waves);
    int32_t first = p.first, end = Part<D>(row, V, at * group + group - 1, waves).last;
    uint64_t before, total;
    if (end - first > 2 * kThreads) {
        constexpr int kWaves = kThreads / 64;
        const int w = tid >> 6;
        const int32_t to_piece = min(from_piece + group * per_wave, row.pieces), per = (to_piece - from_piece + kWaves - 1) / kWaves;
        const auto wave_part = [&](int k) {
            Part<D> q = p;
            q.from = min(from_piece + k * per, to_piece);
            q.to = min(q.from + per, to_piece);
            q.first = k == 0 ? first : row.head + q.from * Span<D>::kPer;
            q.last = k == kWaves - 1 ? end : row.head + q.to * Span<D>::kPer;
            return q;
        };
        uint64_t sum = 0;
        walk<1>(row, wave_part(w), [&](float x, int32_t i) { sum += weight(x, i); });
        sum = wave_sum(sum);
        if ((tid & 63) == 0) s.slots[w] = sum;
        __syncthreads();
        int k = 0;
        for (; k < kWaves - 1 && target >= s.slots[k]; ++k) target -= s.slots[k];
        const Part<D> q = wave_part(k);
        first = q.first;
        end = q.last;
    }
    const int32_t per = (end - first + kThreads - 1) / kThreads;
    const int32_t from = min(first + tid * per, end), to = min(from + per, end);
    uint64_t sum = 0;
    for (int32_t i = from; i < to; ++i) sum += weight(D::get(row.x[i]), i);
    before = team.before(sum, &total);
    if (before <= target && target < before + sum) {
        int32_t i = from;
        for (; i < to - 1; ++i) {
            before += weight(D::get(row.x[i]), i);
            if (target < before) break;
        }
        answer(b.a, n, i, ((double)D::get(row.x[i]) - (double)m) / (double)ask.T, all, left);
    }
}

// ---- long rows of bf16, by counts ------------------------------------------
// A bf16 row has few different numbers, so how often each one occurs says all
// about it: one pass counts them, before the maximum is known, with integers
// alone; weights are worked out once for each number and not for each entry
// (the 20 f64 operations of a weight for each of 256 x 131072 entries took
// 47 us, a pass that counts reads them at HBM's pace).  The cut comes exactly
// from the counts, ties included; what is left is to find an index in one part
// of the row, with the weights by number in LDS.
//
// A place for each number with 2^-36 < |x| < 2^12 and for -2^-36, largest
// first, 0 in the middle.  -inf is not counted.  Rows with other numbers that
// weigh something go the slow way.
//
// 256 x 131072, filters of all kinds: 22 us for the counts (67 MB: 3 TB/s),
// 23 us for the rest by one block a row, 8 of them in the search of a part, the
// others in loads and barriers that follow one another.  One row of 131072: 7
// and 19 us.  Fewer parts make the search longer, more of them the counts: at
// 256 rows six in place of three took 47 us in all, not 43.
constexpr int kSigned = 48 * 128, kPlaces = 2 * kSigned, kZero = kSigned - 1;
constexpr uint32_t kLowBits = (127 - 36) << 23;  // of the lowest magnitude; as its positive number's place is 0's
enum { kOdd = 1, kAbove = 2, kBelow = 4, kBetween = 8 };  // NaN or +inf; past the places

// The place of x, or -1 and what is the matter with it.
__device__ __forceinline__ int place_of(float x, uint32_t* flags) {
    const uint32_t b = __float_as_uint(x), t = (b & 0x7fffffffu) - kLowBits;
    if (t < (uint32_t)kSigned << 16 && b != kLowBits) return kSigned + ((int)(t >> 16) ^ ~((int32_t)b >> 31));
    if (x == 0.0f) return kZero;
    if (x != -INFINITY) *flags |= !(x < INFINITY) ? kOdd : x >= 4096.0f ? kAbove : x <= -4096.0f ? kBelow : kBetween;
    return -1;
}
__device__ __forceinline__ float number_at(int place) {
    if (place == kZero) return 0.0f;
    const int s = place < kSigned ? -1 : 0;
    return __uint_as_float((kLowBits + ((uint32_t)((place - kSigned) ^ s) << 16)) | (s ? 0u : 0x80000000u));
}

constexpr int kBinade = 128, kBinades = kPlaces / kBinade;
constexpr int kMostCounts = 32, kCountWaves = 8, kPickWaves = 16;

struct Counts {
    Args a;
    uint32_t* many;  // [row of the batch][part][kPlaces / 2]: two counts, a part has less than 2^16 entries
    uint4* has;      // [row][part]: a bit for each binade that has entries (only those are in `many`); the flags
    int64_t first;
    int32_t parts;
};

// 48 KB of LDS: three blocks of eight waves on a CU.
__global__ __launch_bounds__(512) void k_cat_sample_count(Counts b) {
    __shared__ __align__(16) uint32_t many[kPlaces];
    __shared__ uint32_t has[4];
    const int64_t r = blockIdx.x / b.parts, n = b.first + r;
    const int32_t p = blockIdx.x % b.parts, V = b.a.vocab;
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const Span<BF16> row(static_cast<const uint16_t*>(b.a.x) + n * b.a.stride, V);
    const Part<BF16> part(row, V, p * kCountWaves + w, b.parts * kCountWaves);
    for (int i = tid; i < kPlaces / 4; i += 512) reinterpret_cast<uint4*>(many)[i] = make_uint4(0, 0, 0, 0);
    if (tid < 4) has[tid] = 0;
    __syncthreads();
    uint32_t flags = 0;
    walk<4>(row, part, [&](float x, int32_t) {
        const int at = place_of(x, &flags);
        if (at >= 0) atomicAdd(&many[at], 1u);
    });
    if (flags) atomicOr(&has[3], flags);
    __syncthreads();
    uint32_t* to = b.many + blockIdx.x * (int64_t)(kPlaces / 2);
    for (int i = w; i < kBinades; i += kCountWaves) {
        const uint2 c = reinterpret_cast<const uint2*>(many + i * kBinade)[lane];
        if (!__any(c.x | c.y)) continue;
        to[i * (kBinade / 2) + lane] = c.x | c.y << 16;
        if (lane == 0) atomicOr(&has[i / 32], 1u << i % 32);
    }
    __syncthreads();
    if (tid == 0) b.has[blockIdx.x] = make_uint4(has[0], has[1], has[2], has[3]);
}

// A row with numbers that have no place: the key, and then the index, of each
// cut by halving, a pass over the row for every step (131072 entries: 0.2 ms
// without a cut, 1.2 with one, 2.1 with two).  In little code and few
// registers: it stands in the kernel that every row goes through, and with
// slow_row() there that one spilled (20 us more for each call).
template <class T>
__device__ __forceinline__ void other_row(const Args& A, int64_t n, const Ask& ask, T& team) {
    constexpr int kThreads = T::kWaves * 64;
    const int32_t V = A.vocab;
    const uint16_t* const x = static_cast<const uint16_t*>(A.x) + n * A.stride;
    const auto key = [](float v) { return key_of(v) >> 16; };
    uint32_t top = 0;
    for (int32_t i = threadIdx.x; i < V; i += kThreads) top = max(top, key_of(BF16::get(x[i])));
    const float m = of_key(team.top(top));
    const bool greedily = !(ask.T > 0.0f);
    const Head h(ask, m);
    // over the entries before `end`, of those with a larger key than `least`, or that one and an index up to `last`:
    // how many they are, or what they weigh
    const auto pass = [&](uint32_t least, int32_t last, int32_t end, bool by_number, double theta) {
        uint64_t v = 0;
#pragma unroll 1
        for (int32_t i = threadIdx.x; i < end; i += 4 * kThreads) {
            uint64_t four = 0xff80ff80ff80ff80ull;  // -inf
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (i + j * kThreads < end) four ^= (uint64_t)(x[i + j * kThreads] ^ 0xff80) << 16 * j;
#pragma unroll 1
            for (int j = 0; j < 4; ++j, four >>= 16) {
                const float f = BF16::get((uint16_t)four);
                const uint32_t k = key(f);
                const bool in = k > least || (k == least && i + j * kThreads <= last);
                v += !in || (double)f - (double)m < theta ? 0 : by_number ? (uint64_t)(f > -INFINITY) : h.weigh(f);
            }
        }
        return team.sum(v);
    };
    uint32_t cut = 0;
    int32_t last = V - 1;
    uint64_t all = 0, left = 0;
    if (greedily) {
        cut = key(m);
    } else {
        all = left = pass(0, last, V, false, -INFINITY);
#pragma unroll 1
        for (int round = 0; round < 2; ++round) {  // top-k, top-p
            const bool by_number = round == 0;
            if (by_number ? ask.K <= 0 : !(ask.P < 1.0f)) continue;
            const uint64_t want = by_number ? min((uint64_t)ask.K, pass(0, last, V, true, -INFINITY)) : ask.limit(left);
            uint32_t c = 0;
#pragma unroll 1
            for (uint32_t bit = 0x8000; bit; bit >>= 1)
                if ((c | bit) <= cut || pass(c | bit, V, V, by_number, -INFINITY) >= want) c |= bit;
            int32_t lo = 0, hi = c == cut ? last : V - 1;
#pragma unroll 1
            while (lo < hi) {
                const int32_t mid = (lo + hi) / 2;
                if (pass(c, mid, V, by_number, -INFINITY) >= want) hi = mid;
                else lo = mid + 1;
            }
            cut = c;
            last = lo;
            left = pass(cut, last, V, false, -INFINITY);
        }
        left = pass(cut, last, V, false, h.theta);
    }
    const uint64_t target = greedily ? 0 : ask.target(left);
    int32_t lo = 0, hi = V - 1;
#pragma unroll 1
    while (lo < hi) {
        const int32_t mid = (lo + hi) / 2;
        if (pass(cut, last, mid + 1, greedily, greedily ? -INFINITY : h.theta) > target) hi = mid;
        else lo = mid + 1;
    }
    if (threadIdx.x) return;
    if (greedily) {
        A.action[n] = lo;
        A.logprob[n] = A.kept[n] = 0.0f;
    } else {
        answer(A, n, lo, ((double)BF16::get(x[lo]) - (double)m) / (double)ask.T, all, left);
    }
}

// One block for a row.  The binades in turn for the waves: those that have
// entries are next to one another.  The counts stay in registers for the second
// use, of up to eight parts; loops over a wave's binades that are not unrolled,
// and cuts found by every wave for itself, where a barrier would cost more.
__global__ __launch_bounds__(1024) void k_cat_sample_pick(Counts b) {
    constexpr int kThreads = 64 * kPickWaves, kOwn = kBinades / kPickWaves, kAhead = 8;
    static_assert(kOwn * kPickWaves == kBinades && kPickWaves == 16, "two binades of a wave in each word of a mask");
    __shared__ struct {
        uint64_t weight[kPlaces];  // of a number; and how many there are.  Not set where a binade has none
        uint32_t many[kPlaces];
    } room;
    __shared__ Team<kThreads>::Slots slots;
    __shared__ uint64_t mass_of[kBinades], sums[kPickWaves][kMostCounts];
    __shared__ uint32_t many_of[kBinades], ties_of[kPickWaves];
    const int64_t n = b.first + blockIdx.x;
    const int32_t V = b.a.vocab, parts = b.parts;
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const Span<BF16> row(static_cast<const uint16_t*>(b.a.x) + n * b.a.stride, V);
    const uint32_t* const counts = b.many + (int64_t)blockIdx.x * parts * (kPlaces / 2) + lane;
    const Ask ask(b.a.p, n, V);
    const uint4 has = lane < parts ? b.has[blockIdx.x * parts + lane] : make_uint4(0, 0, 0, 0);
    const uint32_t has_word[4] = {has.x, has.y, has.z, has.w};
    const auto any_of = [](uint32_t v) { return lanes<64>(v, [](uint32_t a, uint32_t b) { return a | b; }); };
    const auto binade = [&](int i) { return w + kPickWaves * i; };  // the wave's i-th
    uint32_t held[kAhead][kOwn];  // of kAhead parts, in one trip to memory; all that there are, mostly
    const auto load = [&](int from) {
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
#pragma unroll
            for (int i = 0; i < kOwn; ++i) held[j][i] = 0;
            if (from + j < parts)
#pragma unroll
                for (int i = 0; i < kOwn; ++i) {
                    const uint32_t bits = __builtin_amdgcn_readlane(has_word[i / 2], from + j);
                    if (bits >> (w + kPickWaves * (i & 1)) & 1)
                        held[j][i] = counts[(from + j) * (kPlaces / 2) + binade(i) * (kBinade / 2)];
                }
        }
    };
    uint32_t first = kPlaces;
    {
        uint2 many[kOwn] = {};
#pragma unroll 1
        for (int from = 0; from < parts; from += kAhead) {
            load(from);
#pragma unroll
            for (int j = 0; j < kAhead; ++j)
#pragma unroll
                for (int i = 0; i < kOwn; ++i) many[i].x += held[j][i] & 0xffff, many[i].y += held[j][i] >> 16;
        }
#pragma unroll
        for (int i = kOwn - 1; i >= 0; --i) {
            const int at = binade(i) * kBinade + 2 * lane;
            reinterpret_cast<uint2*>(room.many)[at / 2] = many[i];
            first = many[i].x ? at : many[i].y ? at + 1 : first;
        }
    }
    const uint32_t flags = any_of(has.w);
    if (flags & kOdd) {
        if (tid == 0) no_answer(b.a, n);
        return;
    }
    Team<kThreads> team(slots);
    first = team.all(first, [](uint32_t a, uint32_t b) { return min(a, b); });
    if (first == kPlaces && !flags) {
        if (tid == 0) no_answer(b.a, n);
        return;
    }
    const bool greedily = !(ask.T > 0.0f);
    float m = first < kPlaces ? number_at(first) : 0.0f;
    if (flags) {
        const Weigher weigh((double)m, fmax(1.4426950408889634 / (double)(greedily ? 1.0f : ask.T), 1e-300));
        if (first == kPlaces || flags & kAbove || (flags & kBetween && (m <= 0.0f || weigh(0x1p-36f))) ||
            (flags & kBelow && weigh(-4096.0f)))
            return other_row(b.a, n, ask, team);
    }
    const Head h(ask, m);
    uint32_t mine = 0;  // a bit for each of the wave's binades that have entries
#pragma unroll
    for (int i = 0; i < kOwn; ++i) mine |= (any_of(has_word[i / 2]) >> (w + kPickWaves * (i & 1)) & 1) << i;
    mine = __builtin_amdgcn_readfirstlane(mine);
#pragma unroll 1
    for (int i = 0; i < kOwn; ++i) {
        uint64_t mass = 0;
        uint32_t many = 0;
        if (mine >> i & 1) {
            const int at = binade(i) * kBinade + 2 * lane;
            const uint2 c = reinterpret_cast<const uint2*>(room.many)[at / 2];
            uint64_t v0 = at == (int)first, v1 = at + 1 == (int)first;
            if (!greedily) {
                v0 = h.weigh(number_at(at));
                v1 = h.weigh(number_at(at + 1));
            }
            room.weight[at] = v0;
            room.weight[at + 1] = v1;
            mass = wave_sum(c.x * v0 + c.y * v1);
            many = wave_sum((v0 ? c.x : 0) + (v1 ? c.y : 0));
        }
        if (lane == 0) {
            mass_of[binade(i)] = mass;
            many_of[binade(i)] = many;
        }
    }
    __syncthreads();
    // The cut, by every wave for itself.
    const auto pair = [&](int i, bool by_number, uint64_t* low) {  // of places i, i + 1
        const uint2 c = reinterpret_cast<const uint2*>(room.many)[i / 2];
        const uint64_t v0 = room.weight[i], v1 = room.weight[i + 1];
        *low = c.x * (by_number ? (uint64_t)(v0 != 0) : v0);
        return *low + c.y * (by_number ? (uint64_t)(v1 != 0) : v1);
    };
    // the place at which the running sum reaches `want`, and how much of that place is wanted
    const auto find = [&](uint64_t want, bool by_number, uint64_t* need) {
        uint64_t v = 0, low = 0, before, more;
        if (lane < kBinades / 2) {
            low = by_number ? many_of[2 * lane] : mass_of[2 * lane];
            v = low + (by_number ? many_of[2 * lane + 1] : mass_of[2 * lane + 1]);
        }
        int at = lane_of(v, want, &before);
        low = __shfl(low, at);
        const bool odd = want > before + low;
        want -= before + (odd ? low : 0);
        const int base = (2 * at + odd) * kBinade;
        v = pair(base + 2 * lane, by_number, &low);
        at = lane_of(v, want, &more);
        want -= more;
        low = __shfl(low, at);
        const bool second = want > low;
        *need = want - (second ? low : 0);
        return base + 2 * at + second;
    };
    const auto mass_before = [&](int place) {
        uint64_t v = 0, low;
        const int whole = place / kBinade, at = whole * kBinade + 2 * lane;
        if (lane < kBinades / 2)
            v = (2 * lane < whole ? mass_of[2 * lane] : 0) + (2 * lane + 1 < whole ? mass_of[2 * lane + 1] : 0);
        if (at < place) {  // (the binade of a place that was found has entries)
            const uint64_t both = pair(at, false, &low);
            v += at + 1 < place ? both : low;
        }
        return wave_sum(v);
    };
    const uint64_t all = wave_sum(lane < kBinades / 2 ? mass_of[2 * lane] + mass_of[2 * lane + 1] : 0);
    // Kept are the places before `cut`, and of its entries the first `ties` by index.
    int cut = kPlaces;
    uint64_t ties = 0, left = all, need;
    if (!greedily) {
        if (ask.K > 0) {
            const uint64_t many = wave_sum(lane < kBinades / 2 ? many_of[2 * lane] + many_of[2 * lane + 1] : 0);
            if ((uint64_t)ask.K < many) {
                cut = find(ask.K, true, &ties);
                left = mass_before(cut) + ties * room.weight[cut];
            }
        }
        if (ask.P < 1.0f) {
            cut = find(ask.limit(left), false, &need);
            const uint64_t one = room.weight[cut];
            ties = (need + one - 1) / one;
            left = mass_before(cut) + ties * one;
        }
        if (h.theta > -INFINITY) {  // a place that has entries and is the last that min-p keeps, or the one behind it
            int lo = 0, step = kPlaces / 64;  // lo is kept
            for (; step > 0; step = step == 1 ? 0 : max(step / 64, 1)) {
                const int at = lo + step * (lane + 1);
                const uint64_t gone = __ballot(at >= kPlaces || !h.likely(number_at(at)));
                lo += step * (gone ? __ffsll((long long)gone) - 1 : 64);
            }
            const int end = lo + 1;
            if (end <= cut) {
                cut = end;
                ties = 0;
                left = 0;
            }
        }
    }
    // What is kept of each part: before the cut by each wave's binades, of the ties by a lane for each part.
    uint32_t tied = 0;
    if (ties && lane < parts && ((cut < 4096 ? has.x : cut < 8192 ? has.y : has.z) >> cut / kBinade % 32 & 1))
        tied = b.many[((int64_t)blockIdx.x * parts + lane) * (kPlaces / 2) + cut / 2] >> (cut & 1 ? 16 : 0) & 0xffff;
#pragma unroll 1
    for (int from = 0; from < parts; from += kAhead) {
        if (parts > kAhead) load(from);
        uint64_t s[kAhead] = {};
#pragma unroll
        for (int i = 0; i < kOwn; ++i) {
            const int at = binade(i) * kBinade + 2 * lane;
            if (!(mine >> i & 1) || binade(i) * kBinade >= cut) continue;
            const uint64_t v0 = at < cut ? room.weight[at] : 0, v1 = at + 1 < cut ? room.weight[at + 1] : 0;
#pragma unroll
            for (int j = 0; j < kAhead; ++j)
                if (from + j < parts) s[j] += (held[j][i] & 0xffff) * v0 + (held[j][i] >> 16) * v1;
        }
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            if (from + j >= parts) break;
            const uint64_t sum = __any(s[j] != 0) ? wave_sum(s[j]) : 0;
            if (lane == 0) sums[w][from + j] = sum;
        }
    }
    __syncthreads();
    uint64_t v = 0, target, before;
    uint32_t rest = 0;
    if (lane < parts)
#pragma unroll
        for (int i = 0; i < kPickWaves; ++i) v += sums[i][lane];
    if (ties) {
        uint32_t run = tied;
#pragma unroll
        for (int o = 1; o < kMostCounts; o <<= 1) {
            const uint32_t q = __shfl_up(run, o);
            if (lane >= o) run += q;
        }
        run -= tied;
        rest = run < ties ? (uint32_t)ties - run : 0;  // of part `lane`, those that are kept
        v += min(rest, tied) * room.weight[cut];
    }
    left = wave_sum(v);
    target = greedily ? 0 : ask.target(left);
    const int p = lane_of(v, target + 1, &before);
    target -= before;
    rest = __shfl(rest, p);
    // In that part, by waves and then by threads: the weight of what is not a tie, and the ties, of which the
    // first `rest` count (where some but not all of them do)
    if (ties && rest >= __shfl(tied, p)) {
        ++cut;
        rest = 0;
    }
    const uint64_t tie_weight = rest ? room.weight[cut] : 0;
    float least = number_at(cut - (rest ? 0 : 1));  // that counts
    // Numbers up to 2^-36 that weigh nothing have no place (nor has 2^-36, whose place is 0's and may not be
    // set): from the next one on
    if (flags & kBetween) least = fmaxf(least, 0x1.02p-36f);
    const auto add = [&](float x, uint64_t& s, uint32_t& t) {
        if (!(x >= least)) return;
        const uint32_t q = __float_as_uint(x + 0.0f);  // -0 as +0
        const int at = kSigned + ((int)((max(q & 0x7fffffffu, kLowBits) - kLowBits) >> 16) ^ ~((int32_t)q >> 31));
        if (at == cut) ++t;
        else s += room.weight[at];
    };
    const auto weight = [&](uint64_t s, uint32_t t) { return s + min(t, rest) * tie_weight; };
    const int32_t per_wave = (row.pieces + parts * kCountWaves - 1) / (parts * kCountWaves);
    const int32_t from_piece = min(p * kCountWaves * per_wave, row.pieces), to_piece = min(from_piece + kCountWaves * per_wave, row.pieces);
    const int32_t per = (to_piece - from_piece + kPickWaves - 1) / kPickWaves;
    const auto wave_part = [&](int k) {
        Part<BF16> q(row, V, 0, 1);
        q.from = min(from_piece + k * per, to_piece);
        q.to = min(q.from + per, to_piece);
        q.first = p == 0 && k == 0 ? 0 : row.head + q.from * Span<BF16>::kPer;
        q.last = p == parts - 1 && k == kPickWaves - 1 ? V : row.head + q.to * Span<BF16>::kPer;
        return q;
    };
    uint64_t s = 0;
    uint32_t t = 0;
    {
        const Part<BF16> q = wave_part(w);
        constexpr int kBatch = 6;
        const int32_t a = row.head + q.from * Span<BF16>::kPer, z = row.head + q.to * Span<BF16>::kPer;
        if (q.first + lane < a) add(BF16::get(row.x[q.first + lane]), s, t);
        if (z + lane < q.last) add(BF16::get(row.x[z + lane]), s, t);
        for (int32_t at = q.from; at < q.to; at += 64 * kBatch) {
            uint4 r[kBatch];
#pragma unroll
            for (int k = 0; k < kBatch; ++k) r[k] = at + 64 * k + lane < q.to ? row.piece(at + 64 * k + lane) : nothing<BF16>();
#pragma unroll
            for (int k = 0; k < kBatch; ++k) {
                if (at + 64 * k >= q.to) break;
                const Unpack<BF16> x(r[k]);
#pragma unroll
                for (int j = 0; j < Span<BF16>::kPer; ++j) add(x.v[j], s, t);
            }
        }
    }
    s = wave_sum(s);
    if (rest) t = wave_sum(t);
    __syncthreads();
    if (lane == 0) {
        sums[w][0] = s;
        ties_of[w] = t;
    }
    __syncthreads();
    s = 0;
    t = 0;
    int k = 0;
    for (; k < kPickWaves - 1 && weight(s + sums[k][0], t + ties_of[k]) <= target; ++k) {
        s += sums[k][0];
        t += ties_of[k];
    }
    const Part<BF16> q = wave_part(k);
    const int32_t each = (q.last - q.first + kThreads - 1) / kThreads;
    const int32_t from = min(q.first + tid * each, q.last), to = min(from + each, q.last);
    uint64_t own = 0;
    uint32_t own_ties = 0;
    for (int32_t i = from; i < to; ++i) add(BF16::get(row.x[i]), own, own_ties);
    uint64_t total;
    s += team.before(own, &total);
    if (rest) t += (uint32_t)team.before(own_ties, &total);
    if (weight(s, t) <= target && target < weight(s + own, t + own_ties)) {
        int32_t i = from;
        for (; i < to - 1; ++i) {
            add(BF16::get(row.x[i]), s, t);
            if (target < weight(s, t)) break;
        }
        if (greedily) {
            b.a.action[n] = i;
            b.a.logprob[n] = b.a.kept[n] = 0.0f;
        } else {
            answer(b.a, n, i, ((double)BF16::get(row.x[i]) - (double)m) / (double)ask.T, all, left);
        }
    }
}

// ---- short rows ------------------------------------------------------------
// Up to 32 entries: one lane per row, the block's rows in LDS (an odd number of
// words apart: no two lanes on one bank).  The order is not sorted: an entry's
// place in it is how many stand before it, and what is kept is a 32-bit mask.
// 24576 x 11 f32: 8 us, a launch and one chain of f64 weights.
constexpr int kTiny = 32;

template <class D>
__global__ __launch_bounds__(64) void k_cat_sample_tiny(Args A, int64_t rows) {
    __shared__ float tile[64 * (kTiny + 1)];
    __shared__ uint64_t weight[64 * (kTiny + 1)];
    const int tid = threadIdx.x;
    const int32_t V = A.vocab, pitch = V | 1;
    const int64_t n0 = (int64_t)blockIdx.x * 64, n = n0 + tid;
    const int32_t here = (int32_t)min((int64_t)64, rows - n0);
    load_tile<D, 64>(tile, static_cast<const typename D::raw*>(A.x) + n0 * A.stride, A.stride, here, V);
    __syncthreads();
    if (tid >= here) return;
    const float* x = tile + tid * pitch;
    uint64_t* wt = weight + tid * pitch;
    const Ask ask(A.p, n, V);
    float m = x[0];
    int32_t first = 0;
    bool odd = !(x[0] < INFINITY);
    for (int i = 1; i < V; ++i) {
        odd |= !(x[i] < INFINITY);
        if (x[i] > m) {
            m = x[i];
            first = i;
        }
    }
    if (odd || m == -INFINITY) {
        A.action[n] = -1;
        A.logprob[n] = A.kept[n] = NAN;
        return;
    }
    if (!(ask.T > 0.0f)) {
        A.action[n] = first;
        A.logprob[n] = A.kept[n] = 0.0f;
        return;
    }
    const Weigher weigh((double)m, fmax(1.4426950408889634 / (double)ask.T, 1e-300));
    uint64_t all = 0;
    for (int i = 0; i < V; ++i) {
        wt[i] = weigh(x[i]);
        all += wt[i];
    }
    uint32_t keep = 0xffffffffu >> (32 - V);
    uint64_t mass = all;
    if (ask.K > 0) {
        mass = 0;
        for (int i = 0; i < V; ++i) {
            int ahead = 0;
            for (int j = 0; j < V; ++j) ahead += x[j] > x[i] || (x[j] == x[i] && j < i);
            if (ahead >= ask.K) keep &= ~(1u << i);
            else mass += wt[i];
        }
    }
    if (ask.P < 1.0f) {
        const uint64_t limit = ask.limit(mass);
        for (int i = 0; i < V; ++i) {
            uint64_t before = 0;
            for (int j = 0; j < V; ++j) before += x[j] > x[i] || (x[j] == x[i] && j < i) ? wt[j] : 0;
            if (before >= limit) keep &= ~(1u << i);
        }
    }
    const double theta = ask.least();
    uint64_t left = 0;
    for (int i = 0; i < V; ++i) {
        if ((double)x[i] - (double)m < theta) keep &= ~(1u << i);
        if (keep >> i & 1) left += wt[i];
    }
    const uint64_t target = ask.target(left);
    uint64_t run = 0;
    int32_t a = 0;
    for (; a < V - 1; ++a) {
        if (keep >> a & 1) run += wt[a];
        if (run > target) break;
    }
    answer(A, n, a, ((double)x[a] - (double)m) / (double)ask.T, all, left);
}

// ---- rows that are held ----------------------------------------------------
// Up to 9216 entries: a team of one to sixteen waves has the row in registers,
// nine entries a thread at most (with 17 the weights spill).  Thread t has the
// entries [t per, (t + 1) per), so the order by index is that of the threads;
// the row passes through LDS on its way there (per is odd: no bank conflicts).
// The cut is found by team_key; each exchange is one barrier.  65536 x 64 f32:
// 50 us without a filter, 85 with top-p (17 MB: 3.6 us of HBM), bound by the issue
// of vector instructions, 460 and 862 a wave and row: 1.05 and 1.14 a cycle and
// CU, waves waiting for their turn more than half of their time.  A weight is some
// 30 of them, the rest are exchanges of 64 bits between 64 lanes that have an entry
// each.  4096 x 2048: 30 and 63 us (33.5 MB: 6.7), 0.60 and 0.74 a cycle, the rest
// barriers and dependent steps.
template <class D, int THREADS, int E>
__global__ __launch_bounds__(THREADS < 256 ? 256 : THREADS) void k_cat_sample_held(Args A, int64_t rows) {
    constexpr int kRows = THREADS == 64 ? 4 : 1;  // of a block
    constexpr int kFine = THREADS == 64 ? 256 : THREADS == 256 ? 1024 : kBins;
    __shared__ uint64_t hist[kRows][kFine];
    extern __shared__ __align__(16) float staged[];
    __shared__ typename Team<THREADS>::Slots slots;
    Team<THREADS> team(slots);
    const int t = threadIdx.x % THREADS;
    const int64_t n = block_index() * kRows + threadIdx.x / THREADS;
    const int32_t V = A.vocab, per = ((V + THREADS - 1) / THREADS) | 1;
    const bool in = n < rows;
    float* mine = staged + threadIdx.x / THREADS * per * THREADS;
    if (in) {
        const auto* row = static_cast<const typename D::raw*>(A.x) + n * A.stride;
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (t + THREADS * e < V) mine[t + THREADS * e] = D::get(row[t + THREADS * e]);
    }
    __syncthreads();
    if (!in) return;  // a wave of a block whose waves have a row each, or all of a block
    float x[E];
    uint32_t top = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const bool here = e < per && t * per + e < V;
        x[e] = here ? mine[t * per + e] : -INFINITY;
        top = max(top, x[e] < INFINITY ? key_of(x[e]) : UINT32_MAX);
    }
    top = team.top(top);
    const float m = of_key(top);
    if (top == UINT32_MAX || m == -INFINITY) {  // a NaN or +inf, or nothing
        if (t == 0) no_answer(A, n);
        return;
    }
    const Ask ask(A.p, n, V);
    uint64_t total;
    if (!(ask.T > 0.0f)) {
        int32_t first = -1;
#pragma unroll
        for (int e = E - 1; e >= 0; --e) first = key_of(x[e]) == top ? t * per + e : first;
        if (team.before(first >= 0, &total) == 0 && first >= 0) {
            A.action[n] = first;
            A.logprob[n] = A.kept[n] = 0.0f;
        }
        return;
    }
    const Head h(ask, m);
    uint64_t wt[E], all = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        wt[e] = h.weigh(x[e]);  // 0 where there is no entry
        all += wt[e];
        if (e & 1) __builtin_amdgcn_sched_barrier(0);  // two chains at a time: more only need registers
    }
    all = team.sum(all);
    // What is not kept loses its weight.  Of the entries equal to the cut, and not lost yet, the first
    // `ties` by index stay.
    const auto drop = [&](uint32_t cut, uint64_t ties) {
        uint32_t many = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) many += key_of(x[e]) == cut && wt[e];
        uint64_t at = team.before(many, &total);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const uint32_t k = key_of(x[e]);
            const bool tie = k == cut && wt[e];
            if (k < cut || (tie && at >= ties)) wt[e] = 0;
            at += tie;
        }
    };
    uint64_t mass = all;
    const Binner bin = h.binner(kFine - 1, INFINITY);
    const auto key = [&](int e) { return key_of(x[e]); };
    const auto place = [&](int e) { return bin(x[e]); };
    uint64_t* mine_hist = hist[threadIdx.x / THREADS];
    int32_t many = 0;
    if (ask.K > 0) {
#pragma unroll
        for (int e = 0; e < E; ++e) many += wt[e] != 0;
        many = team.sum(many);
    }
    if (ask.K > 0 && ask.K < many) {  // else top-k drops nothing that weighs
        uint64_t above;
        const uint32_t cut = team_key<kFine, uint32_t>(
            team, mine_hist, Held<E>{}, key, place, [&](int e) { return (uint64_t)(wt[e] != 0); }, (uint64_t)ask.K, middle_key, &above);
        drop(cut, (uint64_t)ask.K - above);
        mass = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) mass += wt[e];
        mass = team.sum(mass);
    }
    if (ask.P < 1.0f) {
        uint64_t above;
        const uint64_t want = ask.limit(mass);
        const uint32_t cut = team_key<kFine, uint32_t>(team, mine_hist, Held<E>{}, key, place, [&](int e) { return wt[e]; }, want,
                                                          middle_key, &above);
        const uint64_t each = h.weigh(of_key(cut));
        drop(cut, (want - above + each - 1) / each);
    }
    uint64_t sum = 0, left;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        if (!h.likely(x[e])) wt[e] = 0;
        sum += wt[e];
    }
    uint64_t at = team.before(sum, &left);
    const uint64_t target = ask.target(left);
    if (at <= target && target < at + sum) {
        float xa = 0.0f;
        int32_t a = -1;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            if (at <= target && target < at + wt[e]) {
                a = t * per + e;
                xa = x[e];
            }
            at += wt[e];
        }
        answer(A, n, a, ((double)xa - (double)m) / (double)ask.T, all, left);
    }
}

constexpr int kHeld = 9216;

template <class D>
void launch_held(const Args& a, int64_t rows, hipStream_t st) {
    const auto go = [&](auto kernel, int threads) {
        const int per = ((a.vocab + threads - 1) / threads) | 1, many = threads == 64 ? 4 : 1;
        hipLaunchKernelGGL(kernel, grid_of((rows + many - 1) / many), dim3(threads * many),
                           (size_t)per * threads * many * sizeof(float), st, a, rows);
    };
    const int32_t V = a.vocab;
    if (V <= 64) go(k_cat_sample_held<D, 64, 1>, 64);
    else if (V <= 64 * 3) go(k_cat_sample_held<D, 64, 3>, 64);
    else if (V <= 64 * 5) go(k_cat_sample_held<D, 64, 5>, 64);
    else if (V <= 64 * 9) go(k_cat_sample_held<D, 64, 9>, 64);
    else if (V <= 256 * 5) go(k_cat_sample_held<D, 256, 5>, 256);
    else if (V <= 256 * 9) go(k_cat_sample_held<D, 256, 9>, 256);
    else if (V <= 512 * 9) go(k_cat_sample_held<D, 512, 9>, 512);
    else go(k_cat_sample_held<D, 1024, 9>, 1024);
}

// Rows of one round: what their histograms and lists take is bounded, and they
// fill the card.
constexpr int64_t kBatch = 512;

int64_t batch_of(int64_t rows) { return std::min(rows, kBatch); }
// 1536 blocks of 256 threads are on the card at once (six on a CU, by their registers: 2048 took 20 %
// longer); 16 entries for each thread at least (63 x 50021 f32, top-p: 44 us, with eight 52: every part has a
// histogram to write and to read)
int32_t parts_of(int64_t rows, int32_t vocab) {
    return (int32_t)std::min<int64_t>({std::max<int64_t>(1536 / batch_of(rows), 1), vocab / 4096, kParts});
}

// 768 blocks of 512 threads are on the card at once; two pieces for each thread at least, and counts in 16 bits
int32_t counts_of(int64_t rows, int32_t vocab) {
    const int64_t most = std::min(vocab / 8192, 8), least = (vocab + 57343) / 57344;
    return (int32_t)std::max(least, std::min(768 / batch_of(rows), most));
}

int run_counts(const Args& a, int64_t rows, void* space, hipStream_t st) {
    const int64_t many = batch_of(rows);
    const int32_t parts = counts_of(rows, a.vocab);
    uint32_t* const counts = static_cast<uint32_t*>(space);
    for (int64_t first = 0; first < rows; first += many) {
        const Counts b{a, counts, reinterpret_cast<uint4*>(counts + many * parts * (kPlaces / 2)), first, parts};
        const unsigned here = (unsigned)std::min(many, rows - first);
        hipLaunchKernelGGL(k_cat_sample_count, dim3(here * parts), dim3(512), 0, st, b);
        hipLaunchKernelGGL(k_cat_sample_pick, dim3(here), dim3(64 * kPickWaves), 0, st, b);
    }
    return launched();
}

template <class D>
int run_parts(const Args& a, int64_t rows, void* space, hipStream_t st) {
    const bool cut = a.p.top_k || a.p.top_k_all > 0 || a.p.top_p || a.p.top_p_all < 1.0f;
    const int64_t many = batch_of(rows);
    const int32_t parts = parts_of(rows, a.vocab);
    RowSpace* const rooms = static_cast<RowSpace*>(space);
    for (int64_t first = 0; first < rows; first += many) {
        const Batch b{a, rooms, reinterpret_cast<uint64_t*>(rooms + many), first, parts};
        const unsigned here = (unsigned)std::min(many, rows - first), blocks = here * parts;
        hipLaunchKernelGGL(k_cat_sample_top<D>, dim3(blocks), dim3(256), 0, st, b);
        hipLaunchKernelGGL(k_cat_sample_weigh<D>, dim3(blocks), dim3(256), 0, st, b);
        if (cut) hipLaunchKernelGGL(k_cat_sample_near<D>, dim3(blocks), dim3(256), 0, st, b);
        hipLaunchKernelGGL(k_cat_sample_answer<D>, dim3(here), dim3(512), 0, st, b);
    }
    return launched();
}

template <class D>
int run_sample(const Args& a, int64_t rows, void* space, hipStream_t st) {
    if (a.vocab <= kTiny) {
        hipLaunchKernelGGL(k_cat_sample_tiny<D>, dim3((unsigned)((rows + 63) / 64)), dim3(64), 0, st, a, rows);
        return launched();
    }
    if (a.vocab <= kHeld) {
        launch_held<D>(a, rows, st);
        return launched();
    }
    if constexpr (std::is_same_v<D, BF16>) return run_counts(a, rows, space, st);
    else return run_parts<D>(a, rows, space, st);
}

int bad(const char* what) { return rt_internal_fail(RT_EINVAL, (std::string("rt_cat_sample: ") + what).c_str()); }

}  // namespace

extern "C" int64_t rt_cat_sample_workspace_bytes(int64_t rows, int32_t vocab, int32_t dtype) {
    if (rows < 1 || rows > INT32_MAX || vocab < 1 || vocab > RT_CAT_MAX_VOCAB || bad_type(dtype)) return -1;
    if (vocab <= kHeld) return 0;
    if (dtype == RT_DT_BF16)
        return batch_of(rows) * counts_of(rows, vocab) * (kPlaces / 2 * (int64_t)sizeof(uint32_t) + (int64_t)sizeof(uint4));
    const int64_t hist = parts_of(rows, vocab) * kBins * (int64_t)sizeof(uint64_t);
    return batch_of(rows) * ((int64_t)sizeof(RowSpace) + hist);
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
    if (logits->dtype == RT_DT_F32) return run_sample<F32>(a, logits->rows, workspace_d, st);
    if (logits->dtype == RT_DT_BF16) return run_sample<BF16>(a, logits->rows, workspace_d, st);
    return run_sample<F16>(a, logits->rows, workspace_d, st);
}
