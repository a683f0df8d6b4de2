// cat_loss.hip -- losses of a categorical policy from its logits, with their
// gradients: the clipped PPO loss (train.py:200-226, 243, for actions drawn
// from a row of logits) and distillation from a teacher's top logits.
//
// Both need of a row x of V logits the same sums, with m = max x and
// z = (x - m) / T:   S = sum exp z,   U = sum z exp z,   and give a dense
// gradient of one form,  p_v (E lp_v + F),  lp_v = z_v - log S,  p = exp lp,
// plus something at a few named entries: C at the action (PPO), or -C q_j at
// each of the teacher's (distillation, where E = 0).  A row's state is
// therefore five numbers: m, log S, E, F, C.
#include <algorithm>
#include <string>
#include <type_traits>

#include "cat_rows.h"

namespace {

using namespace rtcat;

// (m and log S apart: their sum would lose log S beside a lowest-value m)
struct RowState {
    double m, logs, e, f, c;
};

struct Out {
    float *loss, *logprob, *entropy, *stats, *kl;
    void* grad;
    int64_t grad_stride;
    double* state;
};

struct Logits {
    const void* x;
    int64_t rows, stride;
    int32_t vocab;
};

// ---- the two losses --------------------------------------------------------
struct Ppo {
    rt_cat_ppo_batch b;
    double t, inv, low, high, ent, klc;  // inv = 1 / t
    static constexpr int terms = 7;
    static constexpr bool ppo = true;

    __device__ int32_t k() const { return 0; }
    __device__ bool ignored(int64_t n, int32_t V) const {
        const int64_t a = b.actions[n];
        return a < 0 || a >= V || (b.weights && b.weights[n] == 0.0f);
    }
    // What a row has beside its logits, asked for before their sums are known.
    struct Given { float w, adv, old, ref; };
    __device__ Given given(int64_t n) const {
        return Given{b.weights ? b.weights[n] : 0.0f, b.advantages[n], b.old_logprobs[n], b.ref_logprobs ? b.ref_logprobs[n] : 0.0f};
    }
    // From the row's log-probability of its action and its entropy: the state, and the weighted terms.
    __device__ RowState finish(const Given& g, int64_t rows, double m, double logs, double lp, double h, double* term) const {
        const double w = b.weights ? (double)g.w : 1.0 / (double)rows;
        const double A = g.adv, lr = lp - (double)g.old, r = exp_64(lr);
        const double lo = 1.0 - low, hi = 1.0 + high;
        const double rc = r < lo ? lo : r > hi ? hi : r;
        const double one = -A * r, two = -A * rc;
        const double pg = one >= two ? one : two > one ? two : one + two;  // the larger, NaN if one is
        double c = one >= two ? one : two > one ? 0.0 : pg, kl = 0.0;
        if (b.ref_logprobs) {
            const double away = (double)g.ref - lp, q = exp_64(away);
            kl = q - away - 1.0;
            if (klc != 0.0) c += klc * (1.0 - q);
        }
        term[0] = w * (pg - ent * h + (klc != 0.0 ? klc * kl : 0.0));
        term[1] = w * pg;
        term[2] = w * kl;
        term[3] = w * h;
        term[4] = w * -lr;
        term[5] = w * ((r - 1.0) - lr);
        term[6] = r < lo || r > hi ? w : 0.0;
        RowState s;
        s.m = m;
        s.logs = logs;
        s.c = w * c * inv;
        s.e = w * ent * inv;
        s.f = s.e * h - s.c;
        return s;
    }
};

struct Distill {
    rt_cat_teacher b;
    double t, inv;  // inv = 1 / t
    static constexpr int terms = 1;
    static constexpr bool ppo = false;

    __device__ bool ignored(int64_t n, int32_t) const { return b.weights && b.weights[n] == 0.0f; }
    __device__ int32_t k() const { return b.k; }
    struct Given { float w; };
    __device__ Given given(int64_t n) const { return Given{b.weights ? b.weights[n] : 0.0f}; }
    __device__ double weight(const Given& g, int64_t rows) const { return b.weights ? (double)g.w : 1.0 / (double)rows; }
};

template <class D>
__device__ __forceinline__ const typename D::raw* row_of(const Logits& l, int64_t n) {
    return static_cast<const typename D::raw*>(l.x) + n * l.stride;
}

template <class D>
__device__ __forceinline__ uint4 pack(const float* v) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(typename D::raw) == 4) w[i] = __float_as_uint(v[i]);
        else w[i] = D::put2(v[2 * i], v[2 * i + 1]);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// ---- a row's sums ----------------------------------------------------------
// In units of log 2: t = (x - m) c, c = log2(e) / T.  exp2 is the hardware's
// (within one unit of the last place, 0 below 2^-126); up to eight terms are
// added in f32, those sums in f64.  c is rounded to f32 (2^-25 of t), and so are
// x - m, of f32 logits, and t (2^-24 each): together they move log S by less than
// 1.25 2^-23 of the row's entropy, and exp2 moves it by 2^-23 at most: about what
// the f32 outputs resolve.  In f64 (20 operations an entry) each pass over 4096 x
// 131072 would take 270 us of arithmetic, where memory takes 215.
struct Sums {
    double s, u;  // sum 2^t and sum t 2^t
};

// What a block's waves tell each other about a row, each place written once.
template <int THREADS>
struct Slots {
    float top[THREADS / 64];
    Sums sums[THREADS / 64];
    RowState state;
};

__device__ __forceinline__ float scale_of(double inv) { return (float)fmin(1.4426950408889634 * inv, 3.0e38); }

// t for a factor beside 2^t: where 2^t is 0 anyway it must stay finite.  2^t
// itself is taken of the plain t, so that a NaN reaches the sums.
__device__ __forceinline__ float finite_t(float t) { return fmaxf(t, -200.0f); }

// The compiler is to unpack a held piece again each time it is used, not to
// keep its entries as f32 (at 16 pieces of bf16 that is 128 more registers, and
// spills).
__device__ __forceinline__ void keep_packed(uint4& r) { asm volatile("" : "+v"(r.x), "+v"(r.y), "+v"(r.z), "+v"(r.w)); }

template <class D, bool U>
__device__ __forceinline__ void add_piece(const uint4& r, float m, float c, Sums& a) {
    const Unpack<D> x(r);
    float s = 0.0f, u = 0.0f;
#pragma unroll
    for (int i = 0; i < Unpack<D>::kPer; ++i) {
        const float t = (x.v[i] - m) * c, e = __builtin_amdgcn_exp2f(t);
        s += e;
        if (U) u = fmaf(e, finite_t(t), u);
    }
    a.s += (double)s;
    if (U) a.u += (double)u;
}

template <bool U>
__device__ __forceinline__ void move_to(Sums& a, double by) {  // by = (old m - new m) c <= 0
    const double f = exp2(by);
    if (U) a.u = f == 0.0 ? 0.0 : f * (a.u + by * a.s);
    a.s *= f;
}

constexpr int kBatch = 4;  // pieces a thread has in flight where a row is streamed

// The maximum and sums of pieces [from, to) of a row, and of its edges where
// `edges` is set.  The first THREADS * HELD pieces stay in `held`; what is left
// is streamed before, each thread with a maximum of its own.  The result is the same
// in every thread.  A part of nothing but -inf: m = -inf and sums 0, or NaN
// where it has one.
template <class D, int THREADS, int HELD, bool U>
__device__ __forceinline__ void row_sums(const Span<D>& row, int32_t from, int32_t to, bool edges, float c, uint4* held,
                                         Slots<THREADS>& slots, float* m_out, Sums* out) {
    const int tid = threadIdx.x;
    float top = -INFINITY, mine = -INFINITY;  // of what is held; of what is streamed
    Sums a{0.0, 0.0};
    float xe = -INFINITY;
    if (edges && tid < row.edges) xe = D::get(row.x[row.edge(tid)]);
    for (int32_t i = from + HELD * THREADS + tid; i < to; i += kBatch * THREADS) {
        uint4 r[kBatch];
#pragma unroll
        for (int k = 0; k < kBatch; ++k) r[k] = i + k * THREADS < to ? row.piece(i + k * THREADS) : nothing<D>();
        float bm = mine;
#pragma unroll
        for (int k = 0; k < kBatch; ++k) bm = fmaxf(bm, Unpack<D>(r[k]).max());
        if (bm > mine) {
            if (mine > -INFINITY) move_to<U>(a, ((double)mine - (double)bm) * (double)c);
            mine = bm;
        }
        if (mine > -INFINITY) {
#pragma unroll
            for (int k = 0; k < kBatch; ++k) {
                keep_packed(r[k]);
                add_piece<D, U>(r[k], mine, c, a);
            }
        } else {  // only -inf so far, or a NaN
            float bad = 0.0f;
#pragma unroll
            for (int k = 0; k < kBatch; ++k) {
                const Unpack<D> x(r[k]);
#pragma unroll
                for (int j = 0; j < Unpack<D>::kPer; ++j) bad = x.v[j] != x.v[j] ? x.v[j] : bad;
            }
            a.s += (double)bad;
        }
    }
#pragma unroll
    for (int k = 0; k < HELD; ++k) {
        const int32_t i = from + k * THREADS + tid;
        held[k] = i < to ? row.piece(i) : nothing<D>();
    }
    top = fmaxf(xe, mine);
#pragma unroll
    for (int k = 0; k < HELD; ++k) top = fmaxf(top, Unpack<D>(held[k]).max());
    top = wave_max(top);
    if constexpr (THREADS > 64) {
        if ((tid & 63) == 0) slots.top[tid >> 6] = top;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < THREADS / 64; ++i) top = fmaxf(top, slots.top[i]);
    }
    const float m = top;
    if (m == -INFINITY) {
        float bad = xe != xe ? xe : 0.0f;
#pragma unroll
        for (int k = 0; k < HELD; ++k) {
            keep_packed(held[k]);
            const Unpack<D> x(held[k]);
#pragma unroll
            for (int j = 0; j < Unpack<D>::kPer; ++j) bad = x.v[j] != x.v[j] ? x.v[j] : bad;
        }
        a.s += (double)bad;
    } else {
        if (mine > -INFINITY && mine != m) move_to<U>(a, ((double)mine - (double)m) * (double)c);
#pragma unroll
        for (int k = 0; k < HELD; ++k) {
            keep_packed(held[k]);
            add_piece<D, U>(held[k], m, c, a);
        }
        const float t = (xe - m) * c, e = __builtin_amdgcn_exp2f(t);
        if (edges && tid < row.edges) {
            a.s += (double)e;
            if (U) a.u += (double)(e * finite_t(t));
        }
    }
    a.s = wave_sum(a.s);
    if (U) a.u = wave_sum(a.u);
    if constexpr (THREADS > 64) {
        if ((tid & 63) == 0) slots.sums[tid >> 6] = a;
        __syncthreads();
        a = slots.sums[0];
#pragma unroll
        for (int i = 1; i < THREADS / 64; ++i) {
            a.s += slots.sums[i].s;
            a.u += slots.sums[i].u;
        }
    }
    *out = a;
    *m_out = m;
}

// ---- a row's gradient ------------------------------------------------------
// scale p (E lp + F) = 2^t (a t + b); rounded once to the logits' type.  In f32
// with the hardware's exp2, also for short rows whose sums are in f64: an entry is
// off by |t| 2^-22 of its size and a few roundings; against 64 bits all outputs are
// 4.4e-8 and 5.7e-8 off (196608 x 11, 32768 x 64), with f64 throughout 2.5e-8 and
// 3.2e-8.
// What a term C or -C q leaves at a named entry is rounded at the size of C.
// Below 2^-126 of the scale a gradient is 0.
struct Slope {
    float m, c, a, b;
};

__device__ __forceinline__ Slope slope_of(const RowState& s, double t_inv, double scale) {
    const double inv = scale * exp_64(-s.logs);
    return Slope{(float)s.m, scale_of(t_inv), (float)(inv * s.e * 0.6931471805599453), (float)(inv * (s.f - s.e * s.logs))};
}

template <bool E>
__device__ __forceinline__ float slope_at(const Slope& g, float x) {
    const float t = (x - g.m) * g.c, e = __builtin_amdgcn_exp2f(t);
    return E ? e * fmaf(finite_t(t), g.a, g.b) : e * g.b;
}

// How a gradient's pieces are stored.
enum { kPlain, kStream, kSingle };

// Rows of logits and gradient that start alike within 16 bytes take whole
// pieces.  A gradient that is larger than half the 256 MB behind the L2 goes
// past it: the logits that are read twice stay there (4096 x 131072 bf16, PPO:
// 441 us, plain stores 476); a smaller one is likely read from there next.
__device__ __forceinline__ int store_mode(const void* g, const void* x, int64_t bytes) {
    return (((uintptr_t)g ^ (uintptr_t)x) & 15) ? kSingle : bytes > (128ll << 20) ? kStream : kPlain;
}

template <class D>
__device__ __forceinline__ void store_piece(typename D::raw* g, const Span<D>& row, int32_t i, int mode, const uint4& r) {
    typename D::raw* at = g + row.head + (int64_t)i * Span<D>::kPer;
    if (mode == kStream) {
        typedef uint32_t u4 __attribute__((ext_vector_type(4)));
        __builtin_nontemporal_store(u4{r.x, r.y, r.z, r.w}, reinterpret_cast<u4*>(at));
    } else if (mode == kPlain) {
        *reinterpret_cast<uint4*>(at) = r;
    } else {
        const typename D::raw* v = reinterpret_cast<const typename D::raw*>(&r);
#pragma unroll
        for (int k = 0; k < Span<D>::kPer; ++k) at[k] = v[k];
    }
}

template <class D, bool E>
__device__ __forceinline__ uint4 slope_piece(const uint4& r, const Slope& sl) {
    const Unpack<D> x(r);
    float v[Unpack<D>::kPer];
#pragma unroll
    for (int k = 0; k < Unpack<D>::kPer; ++k) v[k] = slope_at<E>(sl, x.v[k]);
    return pack<D>(v);
}

// The dense gradient of pieces [from, to) of a row that are not held; a row
// that is ignored gets zeros and is not read.
template <class D, bool E, int THREADS>
__device__ __forceinline__ void put_pieces(typename D::raw* g, const Span<D>& row, int32_t from, int32_t to, int mode,
                                           const Slope& sl, bool skip) {
    if (skip) {
        for (int32_t i = from + (int)threadIdx.x; i < to; i += THREADS) store_piece<D>(g, row, i, mode, make_uint4(0, 0, 0, 0));
        return;
    }
    for (int32_t i = from + (int)threadIdx.x; i < to; i += kBatch * THREADS) {
        uint4 r[kBatch];
#pragma unroll
        for (int k = 0; k < kBatch; ++k)
            if (i + k * THREADS < to) r[k] = row.piece(i + k * THREADS);
#pragma unroll
        for (int k = 0; k < kBatch; ++k)
            if (i + k * THREADS < to) store_piece<D>(g, row, i + k * THREADS, mode, slope_piece<D, E>(r[k], sl));
    }
}

// What a block holds of a row's teacher, k entries of each (dynamic LDS):
// those outside the vocabulary have idx -1 and q 0.
struct Teacher {
    double *lq, *q;
    float* v;      // the logits at idx, then the gradient there
    int32_t* idx;
    __device__ Teacher(char* lds, int32_t k)
        : lq(reinterpret_cast<double*>(lds)), q(lq + k), v(reinterpret_cast<float*>(q + k)),
          idx(reinterpret_cast<int32_t*>(v + k)) {}
    static size_t bytes(int32_t k) { return (size_t)k * 24; }
};

// By one wave: the entries, their probabilities q, and sum q.  lse: the
// teacher's normaliser, NaN for one that is still to be found.
template <class D>
__device__ double teacher_load(const Distill& op, int64_t n, int32_t V, const typename D::raw* x, Teacher& te,
                               double* lse) {
    const int lane = threadIdx.x & 63;
    const int64_t at = n * op.b.k;
    const double inv = op.inv;
    float m = -INFINITY;
    for (int j = lane; j < op.b.k; j += 64) {
        const int64_t i = op.b.idx[at + j];
        const bool in = i >= 0 && i < V;
        const float t = in ? op.b.logits[at + j] : -INFINITY;
        te.idx[j] = in ? (int32_t)i : -1;
        te.lq[j] = t;
        te.v[j] = in ? D::get(x[i]) : 0.0f;
        m = fmaxf(m, t);
    }
    if (op.b.lse) {
        *lse = op.b.lse[n];
    } else {
        m = wave_max(m);
        if (m == -INFINITY) m = 0.0f;
        double s = 0.0;
        for (int j = lane; j < op.b.k; j += 64) s += exp2_64((te.lq[j] - (double)m) * (1.4426950408889634 * inv));
        s = wave_sum(s);
        *lse = s == 0.0 ? 0.0 : (double)m * inv + log_64(s);
    }
    double Q = 0.0;
    for (int j = lane; j < op.b.k; j += 64) {
        const double lq = te.idx[j] < 0 ? -INFINITY : te.lq[j] * inv - *lse, q = exp_64(lq);
        te.lq[j] = lq;
        te.q[j] = q;
        Q += q;
    }
    return wave_sum(Q);
}

// ---- from the sums to the loss ---------------------------------------------
// By one wave: the row's state, its outputs, its terms of the sums over rows.
__device__ __forceinline__ RowState ppo_row(const Ppo& op, const Out& o, const Ppo::Given& given, int64_t n, int64_t rows,
                                            float m, double S, double U, float xa, bool write, double* term) {
    const double logs = log_64(S), lp = ((double)xa - (double)m) * op.inv - logs;
    const double h = logs - 0.6931471805599453 * (U / S);
    const RowState st = op.finish(given, rows, m, logs, lp, h, term);
    if (write) {
        o.logprob[n] = (float)lp;
        o.entropy[n] = (float)h;
    }
    return st;
}

__device__ __forceinline__ RowState distill_row(const Distill& op, const Out& o, const Distill::Given& given, int64_t n,
                                                int64_t rows, float m, double S, const Teacher& te, double lse, double Q,
                                                bool write, double* term) {
    const int lane = threadIdx.x & 63;
    const double logs = log_64(S), inv = op.inv;
    double kl = 0.0;
    for (int j = lane; j < op.b.k; j += 64) {
        const double q = te.q[j];
        if (te.idx[j] >= 0 && q != 0.0) kl += q * (te.lq[j] - (((double)te.v[j] - (double)m) * inv - logs));
    }
    kl = wave_sum(kl);
    const double w = op.weight(given, rows);
    if (write) o.kl[n] = (float)kl;
    term[0] = w * kl;
    // E is 0 throughout: its place keeps the teacher's normaliser for the backward pass
    return RowState{m, logs, lse, w * Q * inv, w * inv};
}

template <class Op>
__device__ __forceinline__ RowState finish_row(const Op& op, const Out& o, const typename Op::Given& given, int64_t n,
                                               int64_t rows, bool skip, float m,
                                               const Sums& sums, float xa, const Teacher& te, double lse, double Q,
                                               bool write, double* terms) {
    const int tid = threadIdx.x;
    RowState st{0.0, INFINITY, 0.0, 0.0, 0.0};  // log S +inf: a row that adds nothing
    double term[Op::terms] = {};
    write = write && tid == 0;
    if constexpr (Op::ppo) {
        if (!skip) st = ppo_row(op, o, given, n, rows, m, sums.s, sums.u, xa, write, term);
        else if (write) o.logprob[n] = o.entropy[n] = 0.0f;
    } else {
        if (!skip) st = distill_row(op, o, given, n, rows, m, sums.s, te, lse, Q, write, term);
        else if (write) o.kl[n] = 0.0f;
    }
    if (write) {
#pragma unroll
        for (int k = 0; k < Op::terms; ++k) terms[n * Op::terms + k] = term[k];
        if (o.state) *reinterpret_cast<RowState*>(o.state + n * RT_CAT_ROW_STATE) = st;
    }
    return st;
}

template <class Op>
__device__ __forceinline__ Slope op_slope(const Op& op, RowState s, double scale) {
    if (!Op::ppo) s.e = 0.0;
    return slope_of(s, op.inv, scale);
}

// The gradient at the teacher's entries, in the place of their logits: the
// dense part and all that names the same entry, in the entries' order.
template <int THREADS>
__device__ __forceinline__ void named_slopes(const Teacher& te, int32_t k, int32_t first, int32_t last, const Slope& sl,
                                             float each) {
    for (int j = threadIdx.x; j < k; j += THREADS) {
        const int32_t at = te.idx[j];
        if (at < first || at >= last) continue;
        double q = 0.0;
        for (int i = 0; i < k; ++i) q += te.idx[i] == at ? te.q[i] : 0.0;
        te.v[j] = slope_at<false>(sl, te.v[j]) - each * (float)q;
    }
}

extern __shared__ __align__(16) char teacher_lds[];

// ---- one block per row -----------------------------------------------------
// HELD pieces of every thread stay in registers between the sums and the
// gradient; longer rows are read again for the rest, mostly from the 256 MB
// behind the L2.  4096 x 131072 bf16, PPO with gradient: 441 us for 2.1 GB, 4.9
// TB/s, where a copy of that size reaches 5.0.  2048 x 50021 f16, loss alone: 52
// us for 205 MB, 3.9 TB/s.
template <class D, class Op, int THREADS, int HELD>
__global__ __launch_bounds__(THREADS) void k_cat_row(Logits l, Op op, Out o, double* terms) {
    __shared__ Slots<THREADS> slots;
    Teacher te(teacher_lds, Op::ppo ? 0 : op.k());
    const int64_t n = block_index();
    if (n >= l.rows) return;
    const int tid = threadIdx.x;
    const auto* x = row_of<D>(l, n);
    const Span<D> row(x, l.vocab);
    uint4 held[HELD ? HELD : 1];
    float m = -INFINITY, xa = 0.0f;
    Sums sums{0.0, 0.0};
    bool skip = op.ignored(n, l.vocab);
    const auto given = op.given(n);
    double lse = 0.0, Q = 0.0;
    if (!skip) {
        if constexpr (Op::ppo) xa = D::get(x[op.b.actions[n]]);
        else if (tid < 64) Q = teacher_load<D>(op, n, l.vocab, x, te, &lse);
        row_sums<D, THREADS, HELD, Op::ppo>(row, 0, row.pieces, true, scale_of(op.inv), held, slots, &m, &sums);
        skip = m == -INFINITY && sums.s == 0.0;
    }
    if (tid < 64) {
        const RowState st = finish_row(op, o, given, n, l.rows, skip, m, sums, xa, te, lse, Q, true, terms);
        if (tid == 0) slots.state = st;
    }
    if (!o.grad) return;
    auto* g = static_cast<typename D::raw*>(o.grad) + n * o.grad_stride;
    float xe = 0.0f;
    if (tid < row.edges) xe = D::get(x[row.edge(tid)]);
    __syncthreads();
    const RowState st = slots.state;
    const Slope sl = op_slope(op, st, 1.0);
    if constexpr (!Op::ppo) {
        if (!skip) named_slopes<THREADS>(te, op.b.k, 0, l.vocab, sl, (float)st.c);
        __syncthreads();
    }
    // the gradient may lie in the logits' own memory: from here on only what is not held is read, each
    // entry by the thread that writes it
    const int mode = store_mode(g, x, l.rows * l.vocab * (int64_t)sizeof(typename D::raw));
    if (!skip) {
#pragma unroll
        for (int k = 0; k < HELD; ++k) {
            const int32_t i = k * THREADS + tid;
            keep_packed(held[k]);
            if (i < row.pieces) store_piece<D>(g, row, i, mode, slope_piece<D, Op::ppo>(held[k], sl));
        }
    }
    put_pieces<D, Op::ppo, THREADS>(g, row, skip ? 0 : HELD * THREADS, row.pieces, mode, sl, skip);
    if (tid < row.edges) g[row.edge(tid)] = D::put(skip ? 0.0f : slope_at<Op::ppo>(sl, xe));
    if (skip) return;
    __syncthreads();
    if constexpr (Op::ppo) {
        if (tid == 0) g[op.b.actions[n]] = D::put(slope_at<true>(sl, xa) + (float)st.c);
    } else {
        for (int j = tid; j < op.b.k; j += THREADS)
            if (te.idx[j] >= 0) g[te.idx[j]] = D::put(te.v[j]);
    }
}

// ---- a row by parts --------------------------------------------------------
// Few long rows leave most of the card idle at one block each, so several have
// a part of a row: its sums first, then, each block from all parts' sums, the
// part's gradient.  The backward pass is the second step alone, from the state.
// 8 x 131072 bf16: 4 + 5 us, each a launch and two trips to memory, the whole
// call 28 (39 by one block a row).  Backward, 1023 x 32003 f32: 39 us for 262 MB, 6.7 TB/s (the
// logits lie in cache from the forward pass).
struct PartSums {
    double m;
    Sums sums;
};

struct Piece {  // [from, to) of the pieces, [first, last) of the entries
    int32_t from, to, first, last;
    template <class D>
    __device__ Piece(const Span<D>& row, int32_t V, int32_t part, int32_t parts) {
        const int32_t per = (row.pieces + parts - 1) / parts;
        from = min(part * per, row.pieces);
        to = min(from + per, row.pieces);
        // the first part also has the entries before the pieces, the last those behind
        first = part == 0 ? 0 : row.head + from * Span<D>::kPer;
        last = part == parts - 1 ? V : row.head + to * Span<D>::kPer;
    }
};

template <class D, class Op>
__global__ __launch_bounds__(256) void k_cat_part(Logits l, Op op, PartSums* to, int32_t parts) {
    __shared__ Slots<256> slots;
    const int64_t n = blockIdx.x / parts;
    const int32_t part = blockIdx.x % parts;
    const Span<D> row(row_of<D>(l, n), l.vocab);
    if (op.ignored(n, l.vocab)) return;
    const Piece p(row, l.vocab, part, parts);
    uint4 held[2];
    float m;
    Sums sums;
    row_sums<D, 256, 2, Op::ppo>(row, p.from, p.to, part == 0, scale_of(op.inv), held, slots, &m, &sums);
    if (threadIdx.x == 0) to[blockIdx.x] = PartSums{m, sums};
}

// By one wave: the sums of a row from those of its parts (at most 64).
template <bool U>
__device__ __forceinline__ Sums join(const PartSums* from, int32_t parts, float c, float* m) {
    const int lane = threadIdx.x & 63;
    PartSums p{-INFINITY, Sums{0.0, 0.0}};
    if (lane < parts) p = from[lane];
    *m = wave_max((float)p.m);
    // a part of nothing but -inf has sums 0 or NaN, which stay
    if (p.m > -INFINITY) move_to<U>(p.sums, (p.m - (double)*m) * (double)c);
    p.sums.s = wave_sum(p.sums.s);
    if (U) p.sums.u = wave_sum(p.sums.u);
    return p.sums;
}

template <class D, class Op, bool JOIN>
__global__ __launch_bounds__(256) void k_cat_grad(Logits l, Op op, Out o, const PartSums* from, double* terms,
                                                  const RowState* state, const float* gout, int32_t parts) {
    constexpr int kThreads = 256;
    __shared__ RowState share;
    Teacher te(teacher_lds, Op::ppo ? 0 : op.k());
    const uint32_t blocks = JOIN && !o.grad ? 1 : parts, block = (uint32_t)block_index();  // of a row; rows parts < 2^31
    const int64_t n = block / blocks;
    const int32_t part = (int32_t)(block % blocks);
    if (n >= l.rows) return;
    const int tid = threadIdx.x;
    const auto* x = row_of<D>(l, n);
    const Span<D> row(x, l.vocab);
    const Piece p(row, l.vocab, part, parts);
    RowState st;
    if constexpr (JOIN) {
        if (tid < 64) {
            bool skip = op.ignored(n, l.vocab);
            const auto given = op.given(n);
            float m = -INFINITY, xa = 0.0f;
            double lse = 0.0, Q = 0.0;
            Sums sums{0.0, 0.0};
            if (!skip) {
                if constexpr (Op::ppo) xa = D::get(x[op.b.actions[n]]);
                else Q = teacher_load<D>(op, n, l.vocab, x, te, &lse);
                sums = join<Op::ppo>(from + n * parts, parts, scale_of(op.inv), &m);
                skip = m == -INFINITY && sums.s == 0.0;
            }
            st = finish_row(op, o, given, n, l.rows, skip, m, sums, xa, te, lse, Q, part == 0, terms);
            if (tid == 0) share = st;
        }
        if (!o.grad) return;
        __syncthreads();
        st = share;
    } else {
        st = state[n];
    }
    const bool skip = st.logs == INFINITY;
    auto* g = static_cast<typename D::raw*>(o.grad) + n * o.grad_stride;
    const double scale = gout ? (double)*gout : 1.0;
    const Slope sl = op_slope(op, st, scale);
    const float each = (float)(scale * st.c);
    int64_t a = -1;
    float va = 0.0f;
    if constexpr (Op::ppo) {
        if (!skip && tid == 0) {
            a = op.b.actions[n];
            if (a >= p.first && a < p.last) va = slope_at<true>(sl, D::get(x[a])) + each;
            else a = -1;
        }
    } else if (!skip) {
        if constexpr (!JOIN) {
            for (int j = tid; j < op.b.k; j += kThreads) {
                const int64_t i = op.b.idx[n * op.b.k + j];
                const bool in = i >= p.first && i < p.last;
                te.idx[j] = in ? (int32_t)i : -1;
                te.q[j] = in ? exp_64((double)op.b.logits[n * op.b.k + j] * op.inv - st.e) : 0.0;
                te.v[j] = in ? D::get(x[i]) : 0.0f;
            }
            __syncthreads();
        }
        named_slopes<kThreads>(te, op.b.k, p.first, p.last, sl, each);
    }
    const int mode = store_mode(g, x, l.rows * l.vocab * (int64_t)sizeof(typename D::raw));
    const int32_t e = tid < row.edges ? row.edge(tid) : -1;
    const bool mine = e >= p.first && e < p.last;
    float xe = 0.0f;
    if (mine) xe = D::get(x[e]);
    __syncthreads();
    put_pieces<D, Op::ppo, kThreads>(g, row, p.from, p.to, mode, sl, skip);
    if (mine) g[e] = D::put(skip ? 0.0f : slope_at<Op::ppo>(sl, xe));
    if (skip) return;
    __syncthreads();
    if constexpr (Op::ppo) {
        if (a >= 0) g[a] = D::put(va);
    } else {
        for (int j = tid; j < op.b.k; j += kThreads)
            if (te.idx[j] >= p.first && te.idx[j] < p.last) g[te.idx[j]] = D::put(te.v[j]);
    }
}

// ---- short rows ------------------------------------------------------------
// Up to 1024 entries: many rows, so more of them lie next to the border of the
// clip, and the memory they need is small beside the arithmetic of a row: the
// sums are in f64 throughout.  Bound by the issue of vector instructions: 32768 x
// 64 f32 with 8 of a teacher's entries 15.5 us (17 MB: 4 us), 827 of them a wave
// of four rows, 0.94 a cycle and CU.

// The sums of a block's rows, in a fixed order.
template <int TERMS>
__device__ __forceinline__ void block_terms(const double* term, double (*ds)[TERMS], double* to) {
#pragma unroll
    for (int k = 0; k < TERMS; ++k) {
        const double r = wave_sum(term[k]);
        if ((threadIdx.x & 63) == 0) ds[threadIdx.x >> 6][k] = r;
    }
    __syncthreads();
    const int k = threadIdx.x;
    if (k < TERMS) to[block_index() * TERMS + k] = ds[0][k] + ds[1][k] + ds[2][k] + ds[3][k];
}

// G lanes per row, E entries each, in registers.  GIVEN: the backward pass,
// from the state.
template <class D, class Op, int G, int E, bool GIVEN>
__global__ __launch_bounds__(256) void k_cat_short(Logits l, Op op, Out o, double* terms, const RowState* state,
                                                   const float* gout) {
    __shared__ double ds[4][Op::terms];
    const int t = threadIdx.x % G;
    const int64_t n0 = block_index() * (256 / G), n = n0 + threadIdx.x / G;
    if (n0 >= l.rows) return;
    const bool in = n < l.rows;
    const int32_t V = l.vocab;
    const auto* x = row_of<D>(l, in ? n : 0);
    double term[Op::terms] = {};
    RowState st{0.0, INFINITY, 0.0, 0.0, 0.0};
    bool skip = !in || (GIVEN ? false : op.ignored(n, V));
    typename Op::Given given{};
    if (!GIVEN && in) given = op.given(n);
    if (GIVEN && in) {
        st = state[n];
        skip = st.logs == INFINITY;
    }
    // the lane's first entry of the teacher's, asked for before the logits are waited for
    struct { int32_t i; float t, x; } first{-1, 0.0f, 0.0f};
    const int64_t at = Op::ppo || !in ? 0 : n * op.k();
    if constexpr (!Op::ppo) {
        if (!skip && t < op.b.k) {
            const int64_t i = op.b.idx[at + t];
            first.t = op.b.logits[at + t];
            if (i >= 0 && i < V) first.i = (int32_t)i;
        }
    }
    float v[E], m = -INFINITY;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int32_t i = t + G * e;
        v[e] = !skip && i < V ? D::get(x[i]) : -INFINITY;
    }
    if (!Op::ppo && !GIVEN && first.i >= 0) first.x = D::get(x[first.i]);
#pragma unroll
    for (int e = 0; e < E; ++e) m = fmaxf(m, v[e]);
    if constexpr (!GIVEN) {
        const double c = 1.4426950408889634 * op.inv;
        m = lanes_max<G>(m);
        const float mf = m == -INFINITY ? 0.0f : m;
        double S = 0.0, U = 0.0;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const double z = ((double)v[e] - (double)mf) * c, p = exp2_64(z);
            S += p;
            if (Op::ppo) U = fma(p, z < -1100.0 ? -1100.0 : z, U);
        }
        S = lanes_sum<G>(S);
        if (Op::ppo) U = lanes_sum<G>(U);
        skip = skip || S == 0.0;
        if constexpr (Op::ppo) {
            if (!skip) {
                st = ppo_row(op, o, given, n, l.rows, m, S, U, D::get(x[op.b.actions[n]]), t == 0, term);
            } else if (in && t == 0) {
                o.logprob[n] = o.entropy[n] = 0.0f;
            }
        } else {
            double kl = 0.0, Q = 0.0, lse = 0.0;
            const double logs = log_64(S), w = skip ? 0.0 : op.weight(given, l.rows);
            // f(the teacher's logit, the student's) for the lane's entries
            const auto entries = [&](auto f) {
                if (first.i >= 0) f(first.t, first.x);
                for (int j = t + G; j < op.b.k; j += G) {
                    const int64_t i = op.b.idx[at + j];
                    if (i >= 0 && i < V) f(op.b.logits[at + j], D::get(x[i]));
                }
            };
            if (op.b.lse) {
                if (!skip) lse = op.b.lse[n];
            } else {
                float tm = -INFINITY;
                entries([&](float tl, float) { tm = fmaxf(tm, tl); });
                tm = lanes_max<G>(tm);
                if (tm == -INFINITY) tm = 0.0f;
                entries([&](float tl, float) { lse += exp2_64(((double)tl - (double)tm) * c); });
                lse = lanes_sum<G>(lse);
                lse = lse == 0.0 ? 0.0 : (double)tm * op.inv + log_64(lse);
            }
            if (!skip) {
                entries([&](float tl, float xl) {
                    const double lq = (double)tl * op.inv - lse, q = exp_64(lq);
                    if (q != 0.0) kl += q * (lq - (((double)xl - (double)m) * op.inv - logs));
                    Q += q;
                });
            }
            kl = lanes_sum<G>(kl);
            Q = lanes_sum<G>(Q);
            if (!skip) {
                st = RowState{m, logs, lse, w * Q * op.inv, w * op.inv};
                term[0] = w * kl;
            }
            if (in && t == 0) o.kl[n] = (float)kl;
        }
        if (in && t == 0 && o.state) *reinterpret_cast<RowState*>(o.state + n * RT_CAT_ROW_STATE) = st;
        if (t) {
#pragma unroll
            for (int k = 0; k < Op::terms; ++k) term[k] = 0.0;
        }
        block_terms<Op::terms>(term, ds, terms);
    }
    if (!o.grad || !in) return;
    auto* g = static_cast<typename D::raw*>(o.grad) + n * o.grad_stride;
    const double scale = gout ? (double)*gout : 1.0;
    float named[E] = {};
    if constexpr (!Op::ppo) {
        // the teacher's entries in turn, each met by the lane that has its place (q of one entry that is named
        // again and again is added in f32: 1024 times, 24 2^-24 off)
        for (int j0 = 0; j0 < op.b.k; j0 += G) {
            int32_t idx = j0 ? -1 : first.i;
            float tl = first.t;
            if (j0 && !skip && j0 + t < op.b.k) {
                const int64_t i = op.b.idx[at + j0 + t];
                tl = op.b.logits[at + j0 + t];
                if (i >= 0 && i < V) idx = (int32_t)i;
            }
            const float q = skip || idx < 0 ? 0.0f : (float)exp_64((double)tl * op.inv - st.e);
            if (skip) idx = -1;
            const int many = min(G, op.b.k - j0);
            for (int j = 0; j < many; ++j) {
                const int32_t bi = __shfl(idx, j, G);
                const float bq = __shfl(q, j, G);
#pragma unroll
                for (int e = 0; e < E; ++e) named[e] += bi == t + G * e ? bq : 0.0f;
            }
        }
    } else if (!skip) {
        const int64_t a = op.b.actions[n];
#pragma unroll
        for (int e = 0; e < E; ++e) named[e] = a == t + G * e ? 1.0f : 0.0f;
    }
    const Slope sl = op_slope(op, st, scale);
    const float each = (float)(Op::ppo ? scale * st.c : -scale * st.c);
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int32_t i = t + G * e;
        if (i < V) g[i] = D::put(skip ? 0.0f : slope_at<Op::ppo>(sl, v[e]) + (named[e] != 0.0f ? each * named[e] : 0.0f));
    }
}

// Up to 32 entries: one lane per row, so that the arithmetic of a row (log,
// exp, divisions) is done once and not by every lane that has a part of it.
// The block's rows pass through LDS (rows an odd number of words apart: no two
// lanes on one bank), where the accesses to memory are those of one long row.
// 196608 x 11 f32, PPO with gradient: 14 us for 23 MB, 0.64 vector instructions a
// cycle and CU: twelve waves on it, each a chain of f64 steps.
constexpr int kTiny = 32;

template <class D, class Op, bool GIVEN>
__global__ __launch_bounds__(256) void k_cat_tiny(Logits l, Op op, Out o, double* terms, const RowState* state,
                                                  const float* gout) {
    __shared__ double ds[4][Op::terms];
    __shared__ float tile[256 * (kTiny + 1)];
    const int tid = threadIdx.x;
    const int32_t V = l.vocab, pitch = V | 1;
    const int64_t n0 = block_index() * 256, n = n0 + tid;
    if (n0 >= l.rows) return;
    const int32_t here = (int32_t)min((int64_t)256, l.rows - n0);
    const bool in = tid < here;
    RowState st{0.0, INFINITY, 0.0, 0.0, 0.0};
    bool skip = !in || (GIVEN ? false : op.ignored(n, V));
    typename Op::Given given{};
    if (!GIVEN && in) given = op.given(n);
    if (GIVEN && in) {
        st = state[n];
        skip = st.logs == INFINITY;
    }
    load_tile<D, 256>(tile, row_of<D>(l, n0), l.stride, here, V);
    __syncthreads();
    float* x = tile + tid * pitch;
    double term[Op::terms] = {};
    if constexpr (!GIVEN) {
        if (!skip) {
            const double c = 1.4426950408889634 * op.inv;
            float m = x[0];
            for (int i = 1; i < V; ++i) m = fmaxf(m, x[i]);
            const float mf = m == -INFINITY ? 0.0f : m;
            double S = 0.0, U = 0.0;
            for (int i = 0; i < V; ++i) {
                const double z = ((double)x[i] - (double)mf) * c, p = exp2_64(z);
                S += p;
                if (Op::ppo) U = fma(p, z < -1100.0 ? -1100.0 : z, U);
            }
            skip = S == 0.0;
            if (!skip) {
                if constexpr (Op::ppo) {
                    st = ppo_row(op, o, given, n, l.rows, m, S, U, x[op.b.actions[n]], true, term);
                } else {
                    const double logs = log_64(S), w = op.weight(given, l.rows);
                    const int64_t at = n * op.b.k;
                    double lse = 0.0, kl = 0.0, Q = 0.0;
                    if (op.b.lse) {
                        lse = op.b.lse[n];
                    } else {
                        float tm = -INFINITY;
                        for (int j = 0; j < op.b.k; ++j) {
                            const int64_t i = op.b.idx[at + j];
                            if (i >= 0 && i < V) tm = fmaxf(tm, op.b.logits[at + j]);
                        }
                        if (tm == -INFINITY) tm = 0.0f;
                        for (int j = 0; j < op.b.k; ++j) {
                            const int64_t i = op.b.idx[at + j];
                            if (i >= 0 && i < V) lse += exp2_64(((double)op.b.logits[at + j] - (double)tm) * c);
                        }
                        lse = lse == 0.0 ? 0.0 : (double)tm * op.inv + log_64(lse);
                    }
                    for (int j = 0; j < op.b.k; ++j) {
                        const int64_t i = op.b.idx[at + j];
                        if (i < 0 || i >= V) continue;
                        const double lq = (double)op.b.logits[at + j] * op.inv - lse, q = exp_64(lq);
                        if (q != 0.0) kl += q * (lq - (((double)x[i] - (double)m) * op.inv - logs));
                        Q += q;
                    }
                    st = RowState{m, logs, lse, w * Q * op.inv, w * op.inv};
                    term[0] = w * kl;
                    o.kl[n] = (float)kl;
                }
            }
        }
        if (in && skip) {
            if constexpr (Op::ppo) o.logprob[n] = o.entropy[n] = 0.0f;
            else o.kl[n] = 0.0f;
        }
        if (in && o.state) *reinterpret_cast<RowState*>(o.state + n * RT_CAT_ROW_STATE) = st;
        block_terms<Op::terms>(term, ds, terms);
    }
    if (!o.grad) return;
    if (in) {
        const double scale = gout ? (double)*gout : 1.0;
        const Slope sl = op_slope(op, st, scale);
        const float each = (float)(scale * st.c);
        for (int i = 0; i < V; ++i) x[i] = skip ? 0.0f : slope_at<Op::ppo>(sl, x[i]);
        if (!skip) {
            if constexpr (Op::ppo) {
                const int64_t a = op.b.actions[n];
                if (a >= 0 && a < V) x[a] += each;
            } else {
                const int64_t at = n * op.b.k;
                for (int j = 0; j < op.b.k; ++j) {
                    const int64_t i = op.b.idx[at + j];
                    const float q = (float)exp_64((double)op.b.logits[at + j] * op.inv - st.e);
                    if (i >= 0 && i < V && q != 0.0f) x[i] -= each * q;
                }
            }
        }
    }
    __syncthreads();
    const float per = 1.0f / (float)V;
    for (int32_t i = tid; i < here * V; i += 256) {
        const int32_t r = (int32_t)(((float)i + 0.5f) * per), c = i - r * V;  // as load_tile's
        static_cast<typename D::raw*>(o.grad)[(n0 + r) * o.grad_stride + c] = D::put(tile[r * pitch + c]);
    }
}

constexpr int kShort = 1024;

template <class Op>
bool tiny(const Op& op, int32_t V) {
    if constexpr (Op::ppo) return V <= kTiny;
    else return V <= kTiny && op.b.k <= kTiny;
}

// Launches the kernel for short rows; how many blocks it had.
template <class D, class Op, bool GIVEN>
int64_t launch_short(const Logits& l, const Op& op, const Out& o, double* ws, const RowState* state, const float* gout,
                     hipStream_t st) {
    const auto go = [&](auto kernel, int per_block) {
        const int64_t blocks = (l.rows + per_block - 1) / per_block;
        hipLaunchKernelGGL(kernel, grid_of(blocks), dim3(256), 0, st, l, op, o, ws, state, gout);
        return blocks;
    };
    const int32_t V = l.vocab;
    if (tiny(op, V)) return go(k_cat_tiny<D, Op, GIVEN>, 256);
    if (V <= 64) return go(k_cat_short<D, Op, 16, 4, GIVEN>, 16);
    if (V <= 128) return go(k_cat_short<D, Op, 16, 8, GIVEN>, 16);
    if (V <= 256) return go(k_cat_short<D, Op, 64, 4, GIVEN>, 4);
    if (V <= 512) return go(k_cat_short<D, Op, 64, 8, GIVEN>, 4);
    return go(k_cat_short<D, Op, 64, 16, GIVEN>, 4);
}

// ---- sums over the rows ----------------------------------------------------
// Every thread a fixed set of rows, then a fixed tree: the same bits every
// time.  One block, or, past 4096 rows (one block takes 50 us for 65536), one
// for each 1024 rows that leave their sums for it.
constexpr int64_t kFold = 1024;

template <int TERMS>
__global__ __launch_bounds__(1024) void k_cat_total(const double* terms, int64_t n, int64_t per, double* sums, float* loss,
                                                    float* stats) {
    __shared__ double part[16][TERMS];
    const int64_t from = blockIdx.x * per, to = min(from + per, n);
    double s[TERMS] = {};
    for (int64_t i = from + threadIdx.x; i < to; i += 1024)
#pragma unroll
        for (int k = 0; k < TERMS; ++k) s[k] += terms[i * TERMS + k];
#pragma unroll
    for (int k = 0; k < TERMS; ++k) {
        const double r = wave_sum(s[k]);
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6][k] = r;
    }
    __syncthreads();
    const int k = threadIdx.x;
    if (k >= TERMS) return;
    double r = part[0][k];
#pragma unroll
    for (int i = 1; i < 16; ++i) r += part[i][k];
    if (sums) sums[blockIdx.x * TERMS + k] = r;
    else if (k == 0) *loss = (float)r;
    else stats[k - 1] = (float)r;
}

// per-row terms of the sums over rows: the loss and up to six statistics; and of each kFold rows
int64_t terms_bytes(int64_t rows) { return (rows + (rows + kFold - 1) / kFold) * Ppo::terms * (int64_t)sizeof(double); }

template <int TERMS>
void launch_total(const double* terms, int64_t n, double* sums, const Out& o, hipStream_t st) {
    const auto go = [&](const double* from, int64_t n, int64_t blocks, int64_t per, double* to) {
        hipLaunchKernelGGL((k_cat_total<TERMS>), dim3((unsigned)blocks), dim3(1024), 0, st, from, n, per, to, o.loss, o.stats);
    };
    if (n > 4 * kFold) {
        const int64_t blocks = (n + kFold - 1) / kFold;
        go(terms, n, blocks, kFold, sums);
        terms = sums;
        n = blocks;
    }
    go(terms, n, 1, n, nullptr);
}

size_t teacher_bytes(const Ppo&) { return 0; }
size_t teacher_bytes(const Distill& op) { return Teacher::bytes(op.b.k); }

template <class D, class Op, int THREADS, int HELD>
void launch_row(const Logits& l, const Op& op, const Out& o, double* ws, hipStream_t st) {
    hipLaunchKernelGGL((k_cat_row<D, Op, THREADS, HELD>), grid_of(l.rows), dim3(THREADS), teacher_bytes(op), st, l, op, o,
                       ws);
}

// How many blocks share a row: as many as bring the card 1024 blocks, with two
// pieces for every thread.
constexpr int kMostParts = 64;
int64_t parts_of(int64_t rows, int32_t vocab, int32_t per) {
    return std::max<int64_t>(1, std::min({1024 / rows, (int64_t)(vocab / per / 512), (int64_t)kMostParts}));
}

template <class D, class Op>
void launch_parts(const Logits& l, const Op& op, const Out& o, double* ws, int64_t parts, hipStream_t st) {
    PartSums* sums = reinterpret_cast<PartSums*>(ws + terms_bytes(l.rows) / sizeof(double));
    const unsigned all = (unsigned)(l.rows * parts);
    hipLaunchKernelGGL((k_cat_part<D, Op>), dim3(all), dim3(256), 0, st, l, op, sums, (int32_t)parts);
    hipLaunchKernelGGL((k_cat_grad<D, Op, true>), dim3(o.grad ? all : (unsigned)l.rows), dim3(256), teacher_bytes(op), st, l,
                       op, o, sums, ws, nullptr, nullptr, (int32_t)parts);
}

template <class D, class Op>
int run_loss(const Logits& l, const Op& op, const Out& o, double* ws, hipStream_t st) {
    const int32_t pieces = l.vocab / Span<D>::kPer;
    int64_t parts = l.rows;
    if (l.vocab <= kShort) parts = launch_short<D, Op, false>(l, op, o, ws, nullptr, nullptr, st);
    // (not where the gradient takes the logits' place: a block reads entries of other blocks' parts)
    else if (const int64_t many = parts_of(l.rows, l.vocab, Span<D>::kPer); many > 1 && o.grad != l.x)
        launch_parts<D>(l, op, o, ws, many, st);
    // Short rows leave most of a block idle between its barriers, long ones need many threads to be in
    // flight; what is held beyond a row's length is computed for nothing.  Measured, PPO with gradient, us
    // (rows x entries; threads x pieces):
    //   65536 x 2048 bf16:   64 x 4 178, 128 x 4 243, 256 x 8 477, 512 x 8 996
    //   16384 x 8192 bf16:   64 x 8 133, 128 x 8 130, 256 x 8 163, 512 x 8 306
    //   8000 x 32000 bf16:   64 x 8 285, 128 x 8 239, 256 x 8 218, 512 x 8 258
    //   2048 x 131072 bf16:  64 x 8 338, 128 x 8 313, 256 x 8 284, 512 x 8 258, 1024 x 8 286
    else if (pieces <= 64 * 4) launch_row<D, Op, 64, 4>(l, op, o, ws, st);
    else if (pieces <= 64 * 8) launch_row<D, Op, 64, 8>(l, op, o, ws, st);
    else if (!o.grad) launch_row<D, Op, 256, 0>(l, op, o, ws, st);
    else if (pieces <= 128 * 8) launch_row<D, Op, 128, 8>(l, op, o, ws, st);
    else if (pieces <= 256 * 16) launch_row<D, Op, 256, 8>(l, op, o, ws, st);
    else launch_row<D, Op, 512, 8>(l, op, o, ws, st);
    launch_total<Op::terms>(ws, parts, ws + l.rows * Op::terms, o, st);
    return launched();
}

template <class Op>
int pick_loss(int dtype, const Logits& l, const Op& op, const Out& o, double* ws, hipStream_t st) {
    if (dtype == RT_DT_F32) return run_loss<F32>(l, op, o, ws, st);
    if (dtype == RT_DT_BF16) return run_loss<BF16>(l, op, o, ws, st);
    return run_loss<F16>(l, op, o, ws, st);
}

template <class D, class Op>
int run_backward(const Logits& l, const Op& op, const double* state, const float* gout, void* grad, int64_t stride,
                 hipStream_t st) {
    if (l.vocab <= kShort) {
        Out o{};
        o.grad = grad;
        o.grad_stride = stride;
        launch_short<D, Op, true>(l, op, o, nullptr, reinterpret_cast<const RowState*>(state), gout, st);
        return launched();
    }
    // 256 threads, eight pieces each, fewer where there are few rows
    const int64_t parts = std::max(parts_of(l.rows, l.vocab, Span<D>::kPer),
                                   std::max<int64_t>(1, std::min<int64_t>(l.vocab / (2048 * Span<D>::kPer), INT32_MAX / l.rows)));
    Out o{};
    o.grad = grad;
    o.grad_stride = stride;
    hipLaunchKernelGGL((k_cat_grad<D, Op, false>), grid_of(l.rows * parts), dim3(256), teacher_bytes(op), st, l, op, o,
                       nullptr, nullptr, reinterpret_cast<const RowState*>(state), gout, (int32_t)parts);
    return launched();
}

template <class Op>
int pick_backward(int dtype, const Logits& l, const Op& op, const double* state, const float* gout, void* grad,
                  int64_t stride, hipStream_t st) {
    if (dtype == RT_DT_F32) return run_backward<F32>(l, op, state, gout, grad, stride, st);
    if (dtype == RT_DT_BF16) return run_backward<BF16>(l, op, state, gout, grad, stride, st);
    return run_backward<F16>(l, op, state, gout, grad, stride, st);
}

int bad(const char* who, const char* what) {
    return rt_internal_fail(RT_EINVAL, (std::string(who) + ": " + what).c_str());
}

const char* grad_fault(const rt_cat_logits* l, const void* grad, int64_t stride) {
    const int64_t es = elem_size(l->dtype);
    if (stride < l->vocab) return "gradient rows overlap (stride < vocab)";
    if (stride > INT64_MAX / 16 / l->rows) return "gradient stride out of range";
    if ((uintptr_t)grad % es) return "gradient not aligned to its element";
    if (grad == l->x) return stride == l->row_stride || l->rows == 1 ? nullptr : "in-place gradient with another stride";
    const uintptr_t x0 = (uintptr_t)l->x, x1 = x0 + ((l->rows - 1) * l->row_stride + l->vocab) * es;
    const uintptr_t g0 = (uintptr_t)grad, g1 = g0 + ((l->rows - 1) * stride + l->vocab) * es;
    if (g0 >= x1 || x0 >= g1) return nullptr;
    // rows of one buffer, the gradient's between the logits': how far behind a row of the logits one starts
    const int64_t step = stride * es, row = l->vocab * es, apart = (int64_t)(g0 - x0) % step, behind = apart < 0 ? apart + step : apart;
    return stride == l->row_stride && behind >= row && behind + row <= step ? nullptr : "gradient overlaps the logits";
}

bool finite_pos(float v) { return v > 0.0f && std::isfinite(v); }

const char* teacher_fault(const rt_cat_teacher* t) {
    if (!t || !t->idx || !t->logits) return "NULL teacher";
    if (t->k < 1 || t->k > RT_CAT_MAX_TOP) return "teacher entries out of range";
    return finite_pos(t->temperature) ? nullptr : "temperature is not a positive number";
}

const char* workspace_fault(const rt_cat_logits* l, const void* ws, int64_t bytes) {
    if (!ws || (uintptr_t)ws % 16) return "workspace NULL or not 16-B aligned";
    return bytes < rt_cat_loss_workspace_bytes(l->rows, l->vocab, l->dtype) ? "workspace too small" : nullptr;
}

}  // namespace

extern "C" int64_t rt_cat_loss_workspace_bytes(int64_t rows, int32_t vocab, int32_t dtype) {
    if (rows < 1 || rows > INT32_MAX || vocab < 1 || vocab > RT_CAT_MAX_VOCAB || bad_type(dtype)) return -1;
    const int64_t parts = parts_of(rows, vocab, 16 / elem_size(dtype));
    return terms_bytes(rows) + (parts > 1 ? rows * parts * (int64_t)sizeof(PartSums) : 0);
}

extern "C" int rt_cat_ppo(const rt_cat_logits* logits, const rt_cat_ppo_batch* batch, const rt_cat_ppo_hparams* hp,
                          const rt_cat_ppo_out* out, void* workspace_d, int64_t workspace_bytes, void* stream) {
    const char* me = "rt_cat_ppo";
    if (const char* f = logits_fault(logits)) return bad(me, f);
    if (!batch || !batch->actions || !batch->old_logprobs || !batch->advantages) return bad(me, "NULL batch");
    if (!hp || !finite_pos(hp->temperature)) return bad(me, "temperature is not a positive number");
    if (!(hp->clip_low >= 0.0f) || !(hp->clip_high >= 0.0f)) return bad(me, "negative clip");
    if (!std::isfinite(hp->ent_coef) || !std::isfinite(hp->kl_coef)) return bad(me, "coefficient is not finite");
    if (hp->kl_coef != 0.0f && !batch->ref_logprobs) return bad(me, "kl_coef without ref_logprobs");
    if (!out || !out->loss || !out->logprob || !out->entropy || !out->stats) return bad(me, "NULL output");
    if (out->grad)
        if (const char* f = grad_fault(logits, out->grad, out->grad_stride)) return bad(me, f);
    if (const char* f = workspace_fault(logits, workspace_d, workspace_bytes)) return bad(me, f);
    const Logits l{logits->x, logits->rows, logits->row_stride, logits->vocab};
    const Ppo op{*batch, hp->temperature, 1.0 / hp->temperature, hp->clip_low, hp->clip_high, hp->ent_coef, hp->kl_coef};
    const Out o{out->loss, out->logprob, out->entropy, out->stats, nullptr, out->grad, out->grad_stride, out->row_state};
    return pick_loss(logits->dtype, l, op, o, static_cast<double*>(workspace_d), reinterpret_cast<hipStream_t>(stream));
}

extern "C" int rt_cat_ppo_backward(const rt_cat_logits* logits, const int64_t* actions_d, float temperature,
                                   const double* row_state_d, const float* grad_loss_d, void* grad_d,
                                   int64_t grad_stride, void* stream) {
    const char* me = "rt_cat_ppo_backward";
    if (const char* f = logits_fault(logits)) return bad(me, f);
    if (!actions_d || !row_state_d || !grad_d) return bad(me, "NULL argument");
    if (!finite_pos(temperature)) return bad(me, "temperature is not a positive number");
    if (const char* f = grad_fault(logits, grad_d, grad_stride)) return bad(me, f);
    const Logits l{logits->x, logits->rows, logits->row_stride, logits->vocab};
    Ppo op{};
    op.b.actions = actions_d;
    op.t = temperature;
    op.inv = 1.0 / op.t;
    return pick_backward(logits->dtype, l, op, row_state_d, grad_loss_d, grad_d, grad_stride,
                         reinterpret_cast<hipStream_t>(stream));
}

extern "C" int rt_cat_distill(const rt_cat_logits* logits, const rt_cat_teacher* teacher,
                              const rt_cat_distill_out* out, void* workspace_d, int64_t workspace_bytes,
                              void* stream) {
    const char* me = "rt_cat_distill";
    if (const char* f = logits_fault(logits)) return bad(me, f);
    if (const char* f = teacher_fault(teacher)) return bad(me, f);
    if (!out || !out->loss || !out->kl) return bad(me, "NULL output");
    if (out->grad)
        if (const char* f = grad_fault(logits, out->grad, out->grad_stride)) return bad(me, f);
    if (const char* f = workspace_fault(logits, workspace_d, workspace_bytes)) return bad(me, f);
    const Logits l{logits->x, logits->rows, logits->row_stride, logits->vocab};
    const Distill op{*teacher, teacher->temperature, 1.0 / teacher->temperature};
    const Out o{out->loss, nullptr, nullptr, nullptr, out->kl, out->grad, out->grad_stride, out->row_state};
    return pick_loss(logits->dtype, l, op, o, static_cast<double*>(workspace_d), reinterpret_cast<hipStream_t>(stream));
}

extern "C" int rt_cat_distill_backward(const rt_cat_logits* logits, const rt_cat_teacher* teacher,
                                       const double* row_state_d, const float* grad_loss_d, void* grad_d,
                                       int64_t grad_stride, void* stream) {
    const char* me = "rt_cat_distill_backward";
    if (const char* f = logits_fault(logits)) return bad(me, f);
    if (const char* f = teacher_fault(teacher)) return bad(me, f);
    if (!row_state_d || !grad_d) return bad(me, "NULL argument");
    if (const char* f = grad_fault(logits, grad_d, grad_stride)) return bad(me, f);
    const Logits l{logits->x, logits->rows, logits->row_stride, logits->vocab};
    const Distill op{*teacher, teacher->temperature, 1.0 / teacher->temperature};
    return pick_backward(logits->dtype, l, op, row_state_d, grad_loss_d, grad_d, grad_stride,
                         reinterpret_cast<hipStream_t>(stream));
}
