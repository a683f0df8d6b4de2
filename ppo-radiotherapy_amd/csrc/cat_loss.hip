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
    double t, low, high, ent, klc;
    static constexpr int terms = 7;
    static constexpr bool ppo = true;

    __device__ bool ignored(int64_t n, int32_t V) const {
        const int64_t a = b.actions[n];
        return a < 0 || a >= V || (b.weights && b.weights[n] == 0.0f);
    }
    // From the row's log-probability of its action and its entropy: the state, and the weighted terms.
    __device__ RowState finish(int64_t n, int64_t rows, double m, double logs, double lp, double h, double* term) const {
        const double w = b.weights ? (double)b.weights[n] : 1.0 / (double)rows;
        const double A = b.advantages[n], lr = lp - (double)b.old_logprobs[n], r = exp(lr);
        const double lo = 1.0 - low, hi = 1.0 + high;
        const double rc = r < lo ? lo : r > hi ? hi : r;
        const double one = -A * r, two = -A * rc;
        const double pg = one >= two ? one : two > one ? two : one + two;  // the larger, NaN if one is
        double c = one >= two ? one : two > one ? 0.0 : pg, kl = 0.0;
        if (b.ref_logprobs) {
            const double away = (double)b.ref_logprobs[n] - lp, q = exp(away);
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
        s.c = w * c / t;
        s.e = w * ent / t;
        s.f = s.e * h - s.c;
        return s;
    }
};

struct Distill {
    rt_cat_teacher b;
    double t;
    static constexpr int terms = 1;
    static constexpr bool ppo = false;

    __device__ bool ignored(int64_t n, int32_t) const { return b.weights && b.weights[n] == 0.0f; }
    __device__ double weight(int64_t n, int64_t rows) const {
        return b.weights ? (double)b.weights[n] : 1.0 / (double)rows;
    }
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
        else w[i] = (uint32_t)D::put(v[2 * i]) | (uint32_t)D::put(v[2 * i + 1]) << 16;
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// 16 bytes of entries that add nothing
template <class D>
__device__ __forceinline__ uint4 nothing() {
    if constexpr (sizeof(typename D::raw) == 4) return make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u);
    const uint32_t two = (uint32_t)D::put(-INFINITY) * 0x10001u;
    return make_uint4(two, two, two, two);
}

// ---- a row's sums ----------------------------------------------------------
// In units of log 2: t = (x - m) c, c = log2(e) / T.  exp2 is the hardware's
// (within one unit of the last place); up to eight terms are added in f32,
// those sums in f64.  c is rounded to f32 (2^-25 of t) and so is t (2^-24):
// together they move log S by less than 2^-23 of the row's entropy, less than
// the f32 outputs resolve.
struct Sums {
    double s, u;  // sum 2^t and sum t 2^t
};

__device__ __forceinline__ float scale_of(double t) { return (float)fmin(1.4426950408889634 / t, 3.0e38); }

// t for a factor beside 2^t: where 2^t is 0 anyway it must stay finite.  2^t
// itself is taken of the plain t, so that a NaN reaches the sums.
__device__ __forceinline__ float finite_t(float t) { return fmaxf(t, -200.0f); }

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
// is streamed, each thread with a maximum of its own.  The result is the same
// in every thread.  A part of nothing but -inf: m = -inf and sums 0, or NaN
// where it has one.
template <class D, int THREADS, int HELD, bool U>
__device__ void row_sums(const Span<D>& row, int32_t from, int32_t to, bool edges, float c, uint4* held, float* fs,
                         double* ds, float* m_out, Sums* out) {
    const int tid = threadIdx.x;
    float top = -INFINITY, mine = -INFINITY;  // of what is held; of what is streamed
    Sums a{0.0, 0.0};
    float xe = -INFINITY;
    if (edges && tid < row.edges) xe = D::get(row.x[row.edge(tid)]);
#pragma unroll
    for (int k = 0; k < HELD; ++k) {
        const int32_t i = from + k * THREADS + tid;
        held[k] = i < to ? row.piece(i) : nothing<D>();
    }
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
            for (int k = 0; k < kBatch; ++k) add_piece<D, U>(r[k], mine, c, a);
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
    top = fmaxf(xe, mine);
#pragma unroll
    for (int k = 0; k < HELD; ++k) top = fmaxf(top, Unpack<D>(held[k]).max());
    const float m = block_max<THREADS>(top, fs);
    if (m == -INFINITY) {
        float bad = xe != xe ? xe : 0.0f;
#pragma unroll
        for (int k = 0; k < HELD; ++k) {
            const Unpack<D> x(held[k]);
#pragma unroll
            for (int j = 0; j < Unpack<D>::kPer; ++j) bad = x.v[j] != x.v[j] ? x.v[j] : bad;
        }
        a.s += (double)bad;
    } else {
        if (mine > -INFINITY && mine != m) move_to<U>(a, ((double)mine - (double)m) * (double)c);
#pragma unroll
        for (int k = 0; k < HELD; ++k) add_piece<D, U>(held[k], m, c, a);
        const float t = (xe - m) * c, e = __builtin_amdgcn_exp2f(t);
        if (edges && tid < row.edges) {
            a.s += (double)e;
            if (U) a.u += (double)(e * finite_t(t));
        }
    }
    out->s = block_sum<THREADS>(a.s, ds);
    out->u = U ? block_sum<THREADS>(a.u, ds) : 0.0;
    *m_out = m;
}

// ---- a row's gradient ------------------------------------------------------
// scale p (E lp + F) = 2^t (a t + b), f32; rounded once to the logits' type.
struct Slope {
    float m, c, a, b;
};

__device__ __forceinline__ Slope slope_of(const RowState& s, double t, double scale) {
    const double inv = scale * exp(-s.logs);
    return Slope{(float)s.m, scale_of(t), (float)(inv * s.e * 0.6931471805599453), (float)(inv * (s.f - s.e * s.logs))};
}

template <bool E>
__device__ __forceinline__ float slope_at(const Slope& g, float x) {
    const float t = (x - g.m) * g.c, e = __builtin_amdgcn_exp2f(t);
    return E ? e * fmaf(finite_t(t), g.a, g.b) : e * g.b;
}

template <class D, bool E>
__device__ __forceinline__ void put_piece(typename D::raw* g, const Span<D>& row, int32_t i, bool aligned, const uint4& r,
                                          const Slope& sl, bool skip) {
    const Unpack<D> x(r);
    float v[Unpack<D>::kPer];
#pragma unroll
    for (int k = 0; k < Unpack<D>::kPer; ++k) v[k] = skip ? 0.0f : slope_at<E>(sl, x.v[k]);
    typename D::raw* at = g + row.head + (int64_t)i * Span<D>::kPer;
    if (aligned) {
        *reinterpret_cast<uint4*>(at) = pack<D>(v);
    } else {
#pragma unroll
        for (int k = 0; k < Span<D>::kPer; ++k) at[k] = D::put(v[k]);
    }
}

// The same numbers at one entry, in f64.
template <class Op, class D>
__device__ double dense_at(const Op& op, const RowState& s, const typename D::raw* x, int64_t i) {
    const double lp = ((double)D::get(x[i]) - s.m) / op.t - s.logs, p = exp(lp);
    return p == 0.0 ? 0.0 : p * ((Op::ppo ? s.e : 0.0) * lp + s.f);
}

// What a block holds of a row's teacher: the entries inside the vocabulary
// (others idx -1, q 0).
struct Teacher {
    int32_t idx[RT_CAT_MAX_TOP];
    double q[RT_CAT_MAX_TOP];  // log q, then q
};
struct NoTeacher {};

// log of the teacher's normaliser
template <int THREADS>
__device__ double teacher_lse(const Distill& op, int64_t n, int32_t V, float* fs, double* ds) {
    if (op.b.lse) return op.b.lse[n];
    const int64_t at = n * op.b.k;
    float m = -INFINITY;
    for (int j = threadIdx.x; j < op.b.k; j += THREADS) {
        const int64_t i = op.b.idx[at + j];
        if (i >= 0 && i < V) m = fmaxf(m, op.b.logits[at + j]);
    }
    m = block_max<THREADS>(m, fs);
    if (m == -INFINITY) m = 0.0f;
    double s = 0.0;
    for (int j = threadIdx.x; j < op.b.k; j += THREADS) {
        const int64_t i = op.b.idx[at + j];
        if (i >= 0 && i < V) s += exp(((double)op.b.logits[at + j] - (double)m) / op.t);
    }
    s = block_sum<THREADS>(s, ds);
    return s == 0.0 ? 0.0 : (double)m / op.t + log(s);
}

// The teacher's entries and their log-probabilities into LDS.
template <int THREADS>
__device__ void teacher_load(const Distill& op, int64_t n, int32_t V, double lse, Teacher& te) {
    const int64_t at = n * op.b.k;
    for (int j = threadIdx.x; j < op.b.k; j += THREADS) {
        const int64_t i = op.b.idx[at + j];
        const bool in = i >= 0 && i < V;
        te.idx[j] = in ? (int32_t)i : -1;
        te.q[j] = in ? (double)op.b.logits[at + j] / op.t - lse : -INFINITY;
    }
    __syncthreads();
}

// What the named entries' gradient is on top of the dense part: each is
// computed whole, before anything is written (the gradient may lie in the
// logits' own memory), and stored over the dense value.
template <int THREADS>
struct Named {
    static constexpr int kMost = (RT_CAT_MAX_TOP + THREADS - 1) / THREADS;
    int32_t at[kMost];
    float v[kMost];
};

// first, last: the entries that this block writes
template <class D, class Op, int THREADS, class Te>
__device__ void named_find(const Op& op, int64_t n, const RowState& s, double scale, bool skip, const Te& te,
                           const typename D::raw* x, Named<THREADS>& e, int32_t first, int32_t last) {
    const int tid = threadIdx.x;
    if constexpr (Op::ppo) {
        e.at[0] = -1;
        if (!skip && tid == 0) {
            const int64_t a = op.b.actions[n];
            if (a >= first && a < last) {
                e.at[0] = (int32_t)a;
                e.v[0] = (float)(scale * (dense_at<Op, D>(op, s, x, a) + s.c));
            }
        }
    } else {
#pragma unroll
        for (int k = 0; k < Named<THREADS>::kMost; ++k) {
            const int j = tid + k * THREADS;
            e.at[k] = !skip && j < op.b.k ? te.idx[j] : -1;
            if (e.at[k] < first || e.at[k] >= last) e.at[k] = -1;
            if (e.at[k] < 0) continue;
            double q = 0.0;
            for (int i = 0; i < op.b.k; ++i)
                if (te.idx[i] == e.at[k]) q += te.q[i];
            e.v[k] = (float)(scale * (dense_at<Op, D>(op, s, x, e.at[k]) - s.c * q));
        }
    }
}

template <class D, class Op, int THREADS>
__device__ void named_put(const Named<THREADS>& e, typename D::raw* g) {
#pragma unroll
    for (int k = 0; k < (Op::ppo ? 1 : Named<THREADS>::kMost); ++k)
        if (e.at[k] >= 0) g[e.at[k]] = D::put(e.v[k]);
}

// ---- from the sums to the loss ---------------------------------------------
// The row's outputs, its terms of the sums over rows, and its state.  Every
// thread of the block calls it; every thread gets the state.
template <class D, class Op, int THREADS, class Te>
__device__ RowState finish_row(const Logits& l, const Op& op, const Out& o, int64_t n, bool skip, float m,
                               const Sums& sums, const typename D::raw* x, Te& te, double* terms, bool write, float* fs,
                               double* ds, RowState* share) {
    const int tid = threadIdx.x;
    RowState st{0.0, INFINITY, 0.0, 0.0, 0.0};  // log S +inf: a row that adds nothing
    if constexpr (Op::ppo) {
        if (tid < 64) {
            double term[Op::terms] = {}, lp = 0.0, h = 0.0;
            if (!skip) {
                const double logs = log(sums.s);
                lp = ((double)D::get(x[op.b.actions[n]]) - (double)m) / op.t - logs;
                h = logs - 0.6931471805599453 * (sums.u / sums.s);
                st = op.finish(n, l.rows, m, logs, lp, h, term);
            }
            if (tid == 0) {
                *share = st;
                if (write) {
                    o.logprob[n] = (float)lp;
                    o.entropy[n] = (float)h;
                    for (int k = 0; k < Op::terms; ++k) terms[n * Op::terms + k] = term[k];
                }
            }
        }
        __syncthreads();
        st = *share;
    } else {
        double kl = 0.0;
        if (!skip) {
            const double logs = log(sums.s), lse = teacher_lse<THREADS>(op, n, l.vocab, fs, ds);
            teacher_load<THREADS>(op, n, l.vocab, lse, te);
            double Q = 0.0;
            for (int j = tid; j < op.b.k; j += THREADS) {
                const double lq = te.q[j], q = exp(lq);
                if (te.idx[j] >= 0 && q != 0.0) kl += q * (lq - (((double)D::get(x[te.idx[j]]) - (double)m) / op.t - logs));
                Q += q;
                te.q[j] = q;
            }
            Q = block_sum<THREADS>(Q, ds);
            kl = block_sum<THREADS>(kl, ds);
            const double w = op.weight(n, l.rows);
            // E is 0 throughout: its place keeps the teacher's normaliser for the backward pass
            st = RowState{m, logs, lse, w * Q / op.t, w / op.t};
            if (tid == 0 && write) terms[n] = w * kl;
        } else if (tid == 0 && write) {
            terms[n] = 0.0;
        }
        if (tid == 0 && write) o.kl[n] = (float)kl;
    }
    if (tid == 0 && write && o.state) *reinterpret_cast<RowState*>(o.state + n * RT_CAT_ROW_STATE) = st;
    return st;
}

template <class Op>
__device__ __forceinline__ Slope op_slope(const Op& op, RowState s, double scale) {
    if (!Op::ppo) s.e = 0.0;
    return slope_of(s, op.t, scale);
}

// ---- one block per row -----------------------------------------------------
// The row is read once: HELD pieces of every thread stay in registers between
// the sums and the gradient, which longer rows read again.
template <class D, class Op, int THREADS, int HELD>
__global__ __launch_bounds__(THREADS) void k_cat_row(Logits l, Op op, Out o, double* terms) {
    __shared__ float fs[THREADS / 64];
    __shared__ double ds[THREADS / 64];
    __shared__ RowState share;
    __shared__ std::conditional_t<Op::ppo, NoTeacher, Teacher> te;
    const int64_t n = blockIdx.x;
    const int tid = threadIdx.x;
    const auto* x = row_of<D>(l, n);
    const Span<D> row(x, l.vocab);
    uint4 held[HELD ? HELD : 1];
    float m = -INFINITY;
    Sums sums{0.0, 0.0};
    bool skip = op.ignored(n, l.vocab);
    if (!skip) {
        row_sums<D, THREADS, HELD, Op::ppo>(row, 0, row.pieces, true, scale_of(op.t), held, fs, ds, &m, &sums);
        skip = m == -INFINITY && sums.s == 0.0;
    }
    const RowState st = finish_row<D, Op, THREADS>(l, op, o, n, skip, m, sums, x, te, terms, true, fs, ds, &share);
    if (!o.grad) return;
    auto* g = static_cast<typename D::raw*>(o.grad) + n * o.grad_stride;
    Named<THREADS> named;
    named_find<D, Op, THREADS>(op, n, st, 1.0, skip, te, x, named, 0, l.vocab);
    const Slope sl = op_slope(op, st, 1.0);
    const bool aligned = (((uintptr_t)g ^ (uintptr_t)x) & 15) == 0;
    float xe = 0.0f;
    if (tid < row.edges) xe = D::get(x[row.edge(tid)]);
    __syncthreads();
#pragma unroll
    for (int k = 0; k < HELD; ++k) {
        const int32_t i = k * THREADS + tid;
        if (i < row.pieces) put_piece<D, Op::ppo>(g, row, i, aligned, held[k], sl, skip);
    }
    for (int32_t i = HELD * THREADS + tid; i < row.pieces; i += THREADS)
        put_piece<D, Op::ppo>(g, row, i, aligned, row.piece(i), sl, skip);
    if (tid < row.edges) g[row.edge(tid)] = D::put(skip ? 0.0f : slope_at<Op::ppo>(sl, xe));
    __syncthreads();
    named_put<D, Op, THREADS>(named, g);
}

// ---- a row's gradient from its state, by parts -----------------------------
template <class D, class Op, int THREADS>
__global__ __launch_bounds__(THREADS) void k_cat_backward(Logits l, Op op, const RowState* state, const float* gout,
                                                          void* grad, int64_t grad_stride, int32_t parts) {
    __shared__ std::conditional_t<Op::ppo, NoTeacher, Teacher> te;
    const int64_t n = blockIdx.x / parts;
    const int32_t part = blockIdx.x % parts;
    const int tid = threadIdx.x;
    const auto* x = row_of<D>(l, n);
    auto* g = static_cast<typename D::raw*>(grad) + n * grad_stride;
    const Span<D> row(x, l.vocab);
    const RowState st = state[n];
    const bool skip = st.logs == INFINITY;
    const double scale = gout ? (double)*gout : 1.0;
    const int32_t per = (row.pieces + parts - 1) / parts;
    const int32_t from = min(part * per, row.pieces), to = min(from + per, row.pieces);
    // the first part also has the entries before the pieces, the last those behind
    const int32_t first = part == 0 ? 0 : row.head + from * Span<D>::kPer;
    const int32_t last = part == parts - 1 ? l.vocab : row.head + to * Span<D>::kPer;
    if constexpr (!Op::ppo) {
        if (!skip) {
            teacher_load<THREADS>(op, n, l.vocab, st.e, te);
            for (int j = tid; j < op.b.k; j += THREADS) te.q[j] = exp(te.q[j]);
            __syncthreads();
        }
    }
    Named<THREADS> named;
    named_find<D, Op, THREADS>(op, n, st, scale, skip, te, x, named, first, last);
    const Slope sl = op_slope(op, st, scale);
    const bool aligned = (((uintptr_t)g ^ (uintptr_t)x) & 15) == 0;
    const int32_t e = tid < row.edges ? row.edge(tid) : -1;
    const bool mine = e >= first && e < last;
    float xe = 0.0f;
    if (mine) xe = D::get(x[e]);
    __syncthreads();
    for (int32_t i = from + tid; i < to; i += THREADS)
        put_piece<D, Op::ppo>(g, row, i, aligned, skip ? nothing<D>() : row.piece(i), sl, skip);
    if (mine) g[e] = D::put(skip ? 0.0f : slope_at<Op::ppo>(sl, xe));
    __syncthreads();
    named_put<D, Op, THREADS>(named, g);
}

// ---- short rows ------------------------------------------------------------
// Up to 1024 entries: many rows, so more of them lie next to the border of the
// clip, and the memory they need is small beside the arithmetic of a row: the
// sums are in f64 throughout.

// From the state, or from a row's sums, to the state and the terms; what the
// two kernels below share.  Every lane of the G that have the row calls it.
__device__ __forceinline__ RowState ppo_row(const Ppo& op, const Out& o, int64_t n, int64_t rows, float m, double S,
                                            double U, float xa, bool write, double* term) {
    const double logs = log(S), lp = ((double)xa - (double)m) / op.t - logs;
    const double h = logs - 0.6931471805599453 * (U / S);
    const RowState st = op.finish(n, rows, m, logs, lp, h, term);
    if (write) {
        o.logprob[n] = (float)lp;
        o.entropy[n] = (float)h;
    }
    return st;
}

// The sums of a block's rows, in a fixed order.
template <int TERMS>
__device__ __forceinline__ void block_terms(const double* term, double* ds, double* to) {
#pragma unroll
    for (int k = 0; k < TERMS; ++k) {
        const double r = block_sum<256>(term[k], ds);
        if (threadIdx.x == 0) to[(int64_t)blockIdx.x * TERMS + k] = r;
    }
}

// G lanes per row, E entries each, in registers.  GIVEN: the backward pass,
// from the state.
template <class D, class Op, int G, int E, bool GIVEN>
__global__ __launch_bounds__(256) void k_cat_short(Logits l, Op op, Out o, double* terms, const RowState* state,
                                                   const float* gout) {
    __shared__ double ds[4];
    const int t = threadIdx.x % G;
    const int64_t n = (int64_t)blockIdx.x * (256 / G) + threadIdx.x / G;
    const bool in = n < l.rows;
    const int32_t V = l.vocab;
    const auto* x = row_of<D>(l, in ? n : 0);
    double term[Op::terms] = {};
    RowState st{0.0, INFINITY, 0.0, 0.0, 0.0};
    bool skip = !in || (GIVEN ? false : op.ignored(n, V));
    if (GIVEN && in) {
        st = state[n];
        skip = st.logs == INFINITY;
    }
    float v[E], m = -INFINITY;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int32_t i = t + G * e;
        v[e] = !skip && i < V ? D::get(x[i]) : -INFINITY;
        m = fmaxf(m, v[e]);
    }
    if constexpr (!GIVEN) {
        const double c = 1.4426950408889634 / op.t;
#pragma unroll
        for (int d = G / 2; d; d >>= 1) m = fmaxf(m, __shfl_xor(m, d));
        const float mf = m == -INFINITY ? 0.0f : m;
        double S = 0.0, U = 0.0;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const double z = ((double)v[e] - (double)mf) * c, p = exp2_64(z);
            S += p;
            if (Op::ppo) U = fma(p, z < -1100.0 ? -1100.0 : z, U);
        }
#pragma unroll
        for (int d = G / 2; d; d >>= 1) {
            S += __shfl_xor(S, d);
            if (Op::ppo) U += __shfl_xor(U, d);
        }
        skip = skip || S == 0.0;
        if constexpr (Op::ppo) {
            if (!skip) {
                st = ppo_row(op, o, n, l.rows, m, S, U, D::get(x[op.b.actions[n]]), t == 0, term);
            } else if (in && t == 0) {
                o.logprob[n] = o.entropy[n] = 0.0f;
            }
        } else {
            double kl = 0.0, Q = 0.0, lse = 0.0;
            const double logs = log(S), w = skip ? 0.0 : op.weight(n, l.rows);
            const int64_t at = in ? n * op.b.k : 0;
            if (op.b.lse) {
                if (!skip) lse = op.b.lse[n];
            } else {
                float tm = -INFINITY;
                for (int j = t; j < op.b.k; j += G) {
                    const int64_t i = op.b.idx[at + j];
                    if (i >= 0 && i < V) tm = fmaxf(tm, op.b.logits[at + j]);
                }
#pragma unroll
                for (int d = G / 2; d; d >>= 1) tm = fmaxf(tm, __shfl_xor(tm, d));
                if (tm == -INFINITY) tm = 0.0f;
                for (int j = t; j < op.b.k; j += G) {
                    const int64_t i = op.b.idx[at + j];
                    if (i >= 0 && i < V) lse += exp2_64(((double)op.b.logits[at + j] - (double)tm) * c);
                }
#pragma unroll
                for (int d = G / 2; d; d >>= 1) lse += __shfl_xor(lse, d);
                lse = lse == 0.0 ? 0.0 : (double)tm / op.t + log(lse);
            }
            if (!skip) {
                for (int j = t; j < op.b.k; j += G) {
                    const int64_t i = op.b.idx[at + j];
                    if (i < 0 || i >= V) continue;
                    const double lq = (double)op.b.logits[at + j] / op.t - lse, q = exp(lq);
                    if (q != 0.0) kl += q * (lq - (((double)D::get(x[i]) - (double)m) / op.t - logs));
                    Q += q;
                }
            }
#pragma unroll
            for (int d = G / 2; d; d >>= 1) {
                kl += __shfl_xor(kl, d);
                Q += __shfl_xor(Q, d);
            }
            if (!skip) {
                st = RowState{m, logs, lse, w * Q / op.t, w / op.t};
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
        // the teacher's entries in turn, each met by the lane that has its place
        const int64_t at = n * op.b.k;
        for (int j0 = 0; j0 < op.b.k; j0 += G) {
            int32_t idx = -1;
            float q = 0.0f;
            if (!skip && j0 + t < op.b.k) {
                const int64_t i = op.b.idx[at + j0 + t];
                if (i >= 0 && i < V) {
                    idx = (int32_t)i;
                    q = (float)exp((double)op.b.logits[at + j0 + t] / op.t - st.e);
                }
            }
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
constexpr int kTiny = 32;

template <class D, class Op, bool GIVEN>
__global__ __launch_bounds__(256) void k_cat_tiny(Logits l, Op op, Out o, double* terms, const RowState* state,
                                                  const float* gout) {
    __shared__ double ds[4];
    __shared__ float tile[256 * (kTiny + 1)];
    const int tid = threadIdx.x;
    const int32_t V = l.vocab, pitch = V | 1;
    const int64_t n0 = (int64_t)blockIdx.x * 256, n = n0 + tid;
    const int32_t here = (int32_t)min((int64_t)256, l.rows - n0);
    const float per = 1.0f / (float)V;  // (i + 1/2) / V is 1/64 or more away from a whole number
    for (int32_t i = tid; i < here * V; i += 256) {
        const int32_t r = (int32_t)(((float)i + 0.5f) * per), c = i - r * V;
        tile[r * pitch + c] = D::get(row_of<D>(l, n0 + r)[c]);
    }
    __syncthreads();
    const bool in = tid < here;
    float* x = tile + tid * pitch;
    double term[Op::terms] = {};
    RowState st{0.0, INFINITY, 0.0, 0.0, 0.0};
    bool skip = !in || (GIVEN ? false : op.ignored(n, V));
    if (GIVEN && in) {
        st = state[n];
        skip = st.logs == INFINITY;
    }
    if constexpr (!GIVEN) {
        if (!skip) {
            const double c = 1.4426950408889634 / op.t;
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
                    st = ppo_row(op, o, n, l.rows, m, S, U, x[op.b.actions[n]], true, term);
                } else {
                    const double logs = log(S), w = op.weight(n, l.rows);
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
                        lse = lse == 0.0 ? 0.0 : (double)tm / op.t + log(lse);
                    }
                    for (int j = 0; j < op.b.k; ++j) {
                        const int64_t i = op.b.idx[at + j];
                        if (i < 0 || i >= V) continue;
                        const double lq = (double)op.b.logits[at + j] / op.t - lse, q = exp(lq);
                        if (q != 0.0) kl += q * (lq - (((double)x[i] - (double)m) / op.t - logs));
                        Q += q;
                    }
                    st = RowState{m, logs, lse, w * Q / op.t, w / op.t};
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
                    const float q = (float)exp((double)op.b.logits[at + j] / op.t - st.e);
                    if (i >= 0 && i < V && q != 0.0f) x[i] -= each * q;
                }
            }
        }
    }
    __syncthreads();
    for (int32_t i = tid; i < here * V; i += 256) {
        const int32_t r = (int32_t)(((float)i + 0.5f) * per), c = i - r * V;
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
        hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(256), 0, st, l, op, o, ws, state, gout);
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
// One block; every thread a fixed set of rows, then a fixed tree: the same
// bits every time.
template <int TERMS>
__global__ __launch_bounds__(1024) void k_cat_total(const double* terms, int64_t n, float* loss, float* stats) {
    __shared__ double ds[16];
    double s[TERMS] = {};
    for (int64_t i = threadIdx.x; i < n; i += 1024)
        for (int k = 0; k < TERMS; ++k) s[k] += terms[i * TERMS + k];
    for (int k = 0; k < TERMS; ++k) {
        const double r = block_sum<1024>(s[k], ds);
        if (threadIdx.x == 0) {
            if (k == 0) *loss = (float)r;
            else stats[k - 1] = (float)r;
        }
    }
}

// per-row terms of the sums over rows: the loss and up to six statistics
int64_t terms_bytes(int64_t rows) { return rows * Ppo::terms * (int64_t)sizeof(double); }

template <class D, class Op, int THREADS, int HELD>
void launch_row(const Logits& l, const Op& op, const Out& o, double* ws, hipStream_t st) {
    hipLaunchKernelGGL((k_cat_row<D, Op, THREADS, HELD>), dim3((unsigned)l.rows), dim3(THREADS), 0, st, l, op, o, ws);
}

template <class D, class Op>
int run_loss(const Logits& l, const Op& op, const Out& o, double* ws, hipStream_t st) {
    const int32_t pieces = l.vocab / Span<D>::kPer;
    int64_t parts = l.rows;
    if (l.vocab <= kShort) parts = launch_short<D, Op, false>(l, op, o, ws, nullptr, nullptr, st);
    else if (!o.grad) launch_row<D, Op, 256, 0>(l, op, o, ws, st);
    else if (pieces <= 256 * 4) launch_row<D, Op, 256, 4>(l, op, o, ws, st);
    else if (pieces <= 256 * 16) launch_row<D, Op, 256, 16>(l, op, o, ws, st);
    else if (pieces <= 512 * 16) launch_row<D, Op, 512, 16>(l, op, o, ws, st);
    else launch_row<D, Op, 1024, 16>(l, op, o, ws, st);
    hipLaunchKernelGGL((k_cat_total<Op::terms>), dim3(1), dim3(1024), 0, st, ws, parts, o.loss, o.stats);
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
    // 256 threads, eight pieces each
    const int64_t parts = std::max<int64_t>(1, std::min<int64_t>(l.vocab / (2048 * Span<D>::kPer), INT32_MAX / l.rows));
    hipLaunchKernelGGL((k_cat_backward<D, Op, 256>), dim3((unsigned)(l.rows * parts)), dim3(256), 0, st, l, op,
                       reinterpret_cast<const RowState*>(state), gout, grad, stride, (int32_t)parts);
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
    if ((uintptr_t)grad % es) return "gradient not aligned to its element";
    if (grad == l->x) return stride == l->row_stride || l->rows == 1 ? nullptr : "in-place gradient with another stride";
    const uintptr_t x0 = (uintptr_t)l->x, x1 = x0 + ((l->rows - 1) * l->row_stride + l->vocab) * es;
    const uintptr_t g0 = (uintptr_t)grad, g1 = g0 + ((l->rows - 1) * stride + l->vocab) * es;
    return g0 < x1 && x0 < g1 ? "gradient overlaps the logits" : nullptr;
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
    return terms_bytes(rows);
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
    const Ppo op{*batch, hp->temperature, hp->clip_low, hp->clip_high, hp->ent_coef, hp->kl_coef};
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
    const Distill op{*teacher, teacher->temperature};
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
    return pick_backward(logits->dtype, l, Distill{*teacher, teacher->temperature}, row_state_d, grad_loss_d, grad_d,
                         grad_stride, reinterpret_cast<hipStream_t>(stream));
}
