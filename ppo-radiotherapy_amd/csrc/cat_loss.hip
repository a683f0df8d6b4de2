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
#include <string>

#include "cat_rows.h"

namespace {

using namespace rtcat;

constexpr int kThreads = 256;

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

// What a block holds of a row's teacher: the entries inside the vocabulary
// (others idx -1, q 0).
struct Teacher {
    int32_t idx[RT_CAT_MAX_TOP];
    double q[RT_CAT_MAX_TOP];   // first log q, then q
};

template <class D>
__device__ __forceinline__ const typename D::raw* row_of(const Logits& l, int64_t n) {
    return static_cast<const typename D::raw*>(l.x) + n * l.stride;
}

// The teacher's entries and their log-probabilities into LDS.
template <int THREADS>
__device__ void teacher_load(const Distill& op, int64_t n, int32_t V, Teacher& te, float* fs, double* ds) {
    const int64_t at = n * op.b.k;
    float m = -INFINITY;
    for (int j = threadIdx.x; j < op.b.k; j += THREADS) {
        const int64_t i = op.b.idx[at + j];
        const bool in = i >= 0 && i < V;
        te.idx[j] = in ? (int32_t)i : -1;
        te.q[j] = in ? (double)op.b.logits[at + j] : -INFINITY;
        if (in) m = fmaxf(m, op.b.logits[at + j]);
    }
    double lse;
    if (op.b.lse) {
        lse = op.b.lse[n];
    } else {
        m = block_max<THREADS>(m, fs);
        if (m == -INFINITY) m = 0.0f;
        double s = 0.0;
        for (int j = threadIdx.x; j < op.b.k; j += THREADS) s += exp((te.q[j] - (double)m) / op.t);
        s = block_sum<THREADS>(s, ds);
        lse = s == 0.0 ? 0.0 : (double)m / op.t + log(s);
    }
    for (int j = threadIdx.x; j < op.b.k; j += THREADS) te.q[j] = te.idx[j] < 0 ? -INFINITY : te.q[j] / op.t - lse;
    __syncthreads();
}

// ---- one block per row -----------------------------------------------------
// d loss / d x at the entries that are named, on top of the dense part: each
// value is computed whole before any is written (the gradient may lie in the
// logits' own memory) and rounded once.
constexpr int kNamed = RT_CAT_MAX_TOP / kThreads;

template <class D, class Op, int THREADS>
__device__ void write_grad(const Logits& l, const Op& op, int64_t n, const RowState& s, double scale, bool skip,
                           const Teacher* te, typename D::raw* g) {
    const auto* x = row_of<D>(l, n);
    const int32_t V = l.vocab;
    const int tid = threadIdx.x;
    const auto dense = [&](int32_t i) {
        const double lp = ((double)D::get(x[i]) - s.m) / op.t - s.logs, p = exp(lp);
        return p == 0.0 ? 0.0 : p * (s.e * lp + s.f);
    };
    int32_t at[kNamed];
    float v[kNamed];
    if constexpr (Op::ppo) {
        at[0] = -1;
        if (!skip && tid == 0) {
            at[0] = (int32_t)op.b.actions[n];
            v[0] = (float)(scale * (dense(at[0]) + s.c));
        }
    } else {
#pragma unroll
        for (int k = 0; k < kNamed; ++k) {
            const int j = tid + k * THREADS;
            at[k] = !skip && j < op.b.k ? te->idx[j] : -1;
            if (at[k] < 0) continue;
            double q = 0.0;
            for (int i = 0; i < op.b.k; ++i)
                if (te->idx[i] == at[k]) q += te->q[i];
            v[k] = (float)(scale * (dense(at[k]) - s.c * q));
        }
    }
    __syncthreads();
    for (int i = tid; i < V; i += THREADS) g[i] = D::put(skip ? 0.0f : (float)(scale * dense(i)));
    __syncthreads();
#pragma unroll
    for (int k = 0; k < (Op::ppo ? 1 : kNamed); ++k)
        if (at[k] >= 0) g[at[k]] = D::put(v[k]);
}

template <class D, class Op, int THREADS>
__global__ __launch_bounds__(THREADS) void k_cat_row(Logits l, Op op, Out o, double* terms) {
    __shared__ float fs[THREADS / 64];
    __shared__ double ds[THREADS / 64];
    __shared__ Teacher te;
    const int64_t n = blockIdx.x;
    const int32_t V = l.vocab;
    const int tid = threadIdx.x;
    const auto* x = row_of<D>(l, n);

    bool skip = op.ignored(n, V);
    float m = -INFINITY;
    double S = 0.0, U = 0.0;
    if (!skip) {
        float nan = 0.0f;
        for (int i = tid; i < V; i += THREADS) {
            const float v = D::get(x[i]);
            m = fmaxf(m, v);
            nan += v != v ? 1.0f : 0.0f;
        }
        m = block_max<THREADS>(m, fs);
        nan = block_sum<THREADS>(nan, fs);
        skip = m == -INFINITY && nan == 0.0f;
    }
    if (!skip) {
        for (int i = tid; i < V; i += THREADS) {
            const double z = ((double)D::get(x[i]) - (double)m) / op.t, e = exp(z);
            S += e;
            if (Op::ppo && e != 0.0) U += e * z;
        }
        S = block_sum<THREADS>(S, ds);
        if (Op::ppo) U = block_sum<THREADS>(U, ds);
    }
    double term[Op::terms] = {};
    RowState st{0.0, INFINITY, 0.0, 0.0, 0.0};  // log S +inf: a row that adds nothing
    const double logs = log(S);
    if constexpr (Op::ppo) {
        double lp = 0.0, h = 0.0;
        if (!skip) {
            lp = ((double)D::get(x[op.b.actions[n]]) - (double)m) / op.t - logs;
            h = logs - U / S;
            st = op.finish(n, l.rows, m, logs, lp, h, term);
        }
        if (tid == 0) {
            o.logprob[n] = (float)lp;
            o.entropy[n] = (float)h;
        }
    } else {
        double kl = 0.0, Q = 0.0;
        if (!skip) {
            teacher_load<THREADS>(op, n, V, te, fs, ds);
            for (int j = tid; j < op.b.k; j += THREADS) {
                const double lq = te.q[j], q = exp(lq);
                if (te.idx[j] >= 0 && q != 0.0) kl += q * (lq - (((double)D::get(x[te.idx[j]]) - (double)m) / op.t - logs));
                Q += q;
                te.q[j] = q;
            }
            Q = block_sum<THREADS>(Q, ds);
            kl = block_sum<THREADS>(kl, ds);
            const double w = op.weight(n, l.rows);
            st = RowState{m, logs, 0.0, w * Q / op.t, w / op.t};
            term[0] = w * kl;
        }
        if (tid == 0) o.kl[n] = (float)kl;
    }
    if (tid == 0) {
        for (int k = 0; k < Op::terms; ++k) terms[n * Op::terms + k] = term[k];
        if (o.state) {
            double* s = o.state + n * RT_CAT_ROW_STATE;
            s[0] = st.m;
            s[1] = st.logs;
            s[2] = st.e;
            s[3] = st.f;
            s[4] = st.c;
        }
    }
    if (o.grad)
        write_grad<D, Op, THREADS>(l, op, n, st, 1.0, skip, &te, static_cast<typename D::raw*>(o.grad) + n * o.grad_stride);
}

template <class D, class Op, int THREADS>
__global__ __launch_bounds__(THREADS) void k_cat_backward(Logits l, Op op, const double* state, const float* gout,
                                                          void* grad, int64_t grad_stride) {
    __shared__ float fs[THREADS / 64];
    __shared__ double ds[THREADS / 64];
    __shared__ Teacher te;
    const int64_t n = blockIdx.x;
    const double* s = state + n * RT_CAT_ROW_STATE;
    const RowState st{s[0], s[1], s[2], s[3], s[4]};
    const bool skip = st.logs == INFINITY;
    if constexpr (!Op::ppo) {
        if (!skip) {
            teacher_load<THREADS>(op, n, l.vocab, te, fs, ds);
            for (int j = threadIdx.x; j < op.b.k; j += THREADS) te.q[j] = exp(te.q[j]);
            __syncthreads();
        }
    }
    write_grad<D, Op, THREADS>(l, op, n, st, gout ? (double)*gout : 1.0, skip, &te,
                               static_cast<typename D::raw*>(grad) + n * grad_stride);
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

template <class D, class Op>
int run_loss(const Logits& l, const Op& op, const Out& o, double* ws, hipStream_t st) {
    hipLaunchKernelGGL((k_cat_row<D, Op, kThreads>), dim3((unsigned)l.rows), dim3(kThreads), 0, st, l, op, o, ws);
    hipLaunchKernelGGL((k_cat_total<Op::terms>), dim3(1), dim3(1024), 0, st, ws, l.rows, o.loss, o.stats);
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
    hipLaunchKernelGGL((k_cat_backward<D, Op, kThreads>), dim3((unsigned)l.rows), dim3(kThreads), 0, st, l, op, state,
                       gout, grad, stride);
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
