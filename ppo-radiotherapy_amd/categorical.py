"""Operators of categorical policies: sampling, the PPO loss, distillation.

The Gaussian agent's rollout and update steps (rt_policy_sample, rt_ppo_grad;
train.py:143-149, 197-246) for a policy that picks one entry of a row of
logits: a discretised beam action ([..., bins]) or a token ([..., vocab]).

    a = sample(logits, u, temperature=0.8, top_k=50, top_p=0.9)                   # rollout
    out = ppo_loss(logits, a.action, a.logprob, adv, temperature=0.8)             # update, autograd
    out.loss.backward()
    out, grad = ppo_loss_grad(logits, a.action, a.logprob, adv, temperature=0.8)  # the same in one pass over the logits
    out = distill_loss(logits, idx, top_logits, temperature=2.0)                  # from a teacher's top logits

Logits are float32, bfloat16 or float16 on the GPU, entries of a row adjacent
(stride 1), leading dimensions any that collapse to evenly spaced rows; -inf
marks an entry that cannot be taken.  Everything is enqueued on the current
stream of the logits' device, nothing synchronises, and all but the autograd
forms can be captured in a graph (there take the `_grad` forms, and
`logits.backward(grad)` for what lies before).  The definitions stand in
include/rtenv.h; wrong arguments raise ValueError or TypeError, those that the
library itself refuses (a gradient that overlaps the logits) RtError, before
anything is launched.
"""
from __future__ import annotations

import ctypes
import functools
import math
from typing import NamedTuple

import torch
from torch.autograd import forward_ad

from . import _lib

_DTYPES = {torch.float32: _lib.DT_F32, torch.bfloat16: _lib.DT_BF16, torch.float16: _lib.DT_F16}


class Sample(NamedTuple):
    action: torch.Tensor        # int64 [...], -1 where a row has no distribution
    logprob: torch.Tensor       # f32 [...]: log softmax(logits / T) of the action
    kept_logprob: torch.Tensor  # f32 [...]: the same over the kept entries alone


class PpoLoss(NamedTuple):
    loss: torch.Tensor     # f32 scalar
    logprob: torch.Tensor  # f32 [...]
    entropy: torch.Tensor  # f32 [...]
    stats: torch.Tensor    # f32 [6]: pg_loss, kl, entropy, old_approx_kl, approx_kl, clipfrac


class DistillLoss(NamedTuple):
    loss: torch.Tensor  # f32 scalar
    kl: torch.Tensor    # f32 [...]


class _Rows:
    """Logits as evenly spaced rows, and the checks every operator makes."""

    __slots__ = ("x", "lead", "n", "vocab", "stride", "device", "dtype")

    def __init__(self, logits: torch.Tensor):
        if not isinstance(logits, torch.Tensor):
            raise TypeError("logits: expected a tensor")
        self.dtype = _DTYPES.get(logits.dtype, -1)
        if self.dtype < 0:
            raise TypeError(f"logits: {logits.dtype} is not one of float32, bfloat16, float16")
        shape = logits.shape
        if not shape or shape[-1] < 1:
            raise ValueError(f"logits: shape {tuple(shape)} has no entries in a row")
        if not logits.is_cuda:
            raise ValueError("logits: expected a tensor on the GPU")
        self.x, self.device = logits, logits.device
        self.lead, self.vocab = shape[:-1], shape[-1]
        self.n = shape[0] if len(shape) == 2 else math.prod(self.lead)
        if self.vocab > _lib.CAT_MAX_VOCAB:
            raise ValueError(f"logits: {self.vocab} entries in a row, at most {_lib.CAT_MAX_VOCAB}")
        if self.n > 2**31 - 1:
            raise ValueError(f"logits: {self.n} rows, at most 2^31 - 1")
        self.stride = self.vocab
        if logits.is_contiguous():
            return
        strides = logits.stride()
        if self.vocab > 1 and strides[-1] != 1:
            raise ValueError("logits: the entries of a row are not adjacent (stride 1)")
        # the leading dimensions, from the last: each as far apart as all rows before it together
        rows = 1
        for size, step in zip(reversed(self.lead), reversed(strides[:-1])):
            if size == 1 or self.n == 0:
                continue
            if rows == 1:
                self.stride = step
            elif step != self.stride * rows:
                raise ValueError("logits: the leading dimensions do not collapse to evenly spaced rows")
            rows *= size

    def arg(self):
        return _lib.RtCatLogits(self.x.data_ptr(), self.n, self.stride, self.vocab, self.dtype)

    def per_row(self, t, name: str, dtype=torch.float32, tail=()):
        """`t` ([...] or [..., k]) as the kernels read it, or None."""
        if t is None:
            return None
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name}: expected a tensor")
        if t.shape != (self.lead + tail if tail else self.lead):
            raise ValueError(f"{name}: shape {tuple(t.shape)}, expected {tuple(self.lead + tail)}")
        if t.device != self.device:
            raise ValueError(f"{name}: on {t.device}, the logits on {self.device}")
        if t.dtype == dtype and t.is_contiguous():
            return t
        if dtype.is_floating_point != t.dtype.is_floating_point or t.dtype == torch.bool or t.is_complex():
            raise TypeError(f"{name}: {t.dtype}")
        return t.detach().to(dtype).contiguous()

    def empty(self, dtype=torch.float32):
        return torch.empty(self.lead, dtype=dtype, device=self.device)

    def grad_buffer(self, out):
        """(tensor of the logits' shape, row stride) that a gradient is written to."""
        if out is None:
            # rows placed like the logits' modulo 16 bytes, so that both sides take wide accesses
            size = self.x.element_size()
            lead, extra = self.x.data_ptr() % 16 // size, (self.stride - self.vocab) % (16 // size)
            if not lead and not extra:
                return torch.empty(self.x.shape, dtype=self.x.dtype, device=self.device), self.vocab
            stride = self.vocab + extra
            flat = torch.empty(lead + max(self.n, 1) * stride, dtype=self.x.dtype, device=self.device)
            return flat.as_strided((self.n, self.vocab), (stride, 1), lead).view(self.x.shape), stride
        if not isinstance(out, torch.Tensor) or out.shape != self.x.shape or out.dtype != self.x.dtype or out.device != self.device:
            raise ValueError("out: expected a tensor of the logits' shape, type and device")
        if out.requires_grad:
            raise ValueError("out: requires grad")
        o = _Rows(out)
        if self.n > 1 and o.stride < self.vocab:
            raise ValueError("out: rows overlap")
        if not out.is_inference():
            torch.autograd.graph.increment_version(out)  # as an operation in place: autograd's check sees it
        return out, max(o.stride, self.vocab)

    def call(self, fn, what: str, *args):
        """fn(*args, stream) on the logits' device and its current stream."""
        here = torch.cuda.current_device()
        if here == self.device.index:
            _lib.check(fn(*args, _raw_stream(here) or None), what)
        else:
            with torch.cuda.device(self.device):
                _lib.check(fn(*args, _raw_stream(self.device.index) or None), what)


# the handle alone: building torch's Stream object costs more than a launch
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


@functools.lru_cache(maxsize=256)
def _workspace_bytes(name: str, rows: int, vocab: int, dtype: int) -> int:
    return int(getattr(_lib.load(), name)(rows, vocab, dtype))


def _workspace(name: str, r: _Rows):
    n = _workspace_bytes(name, r.n, r.vocab, r.dtype)
    return torch.empty(n, dtype=torch.uint8, device=r.device) if n else None, n


def _coef(v, name: str, low=None, positive=False) -> float:
    """v as the kernels get it, in 32 bits."""
    x = float(v)
    f = ctypes.c_float(x).value
    if not math.isfinite(f) or (low is not None and x < low) or (positive and f <= 0):
        raise ValueError(f"{name}: {x}")
    return f


_SAMPLING_OFF = {"temperature": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0}


@functools.lru_cache(maxsize=256)
def _sampling(temperature, top_k, top_p, min_p):
    """The parameters of all rows, checked."""
    if not 0 <= top_k < 2**31 or int(top_k) != top_k:
        raise ValueError(f"top_k: {top_k}")
    return (_coef(temperature, "temperature", low=0.0), int(top_k), _coef(top_p, "top_p", low=0.0),
            _coef(min_p, "min_p", low=0.0))


def sample(logits, u, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0) -> Sample:
    """One action per row from uniform numbers u in [0, 1) (rt_cat_sample).

    temperature, top_k, top_p and min_p are numbers or tensors of one value per
    row; temperature 0 takes the largest logit.  Equal logits rank by index.
    Rows without a distribution (a NaN, +inf, nothing but -inf) get action -1
    and NaN."""
    r = _Rows(logits)
    u = r.per_row(u, "u")
    if u is None:
        raise TypeError("u: expected a tensor")
    params = {"temperature": temperature, "top_k": top_k, "top_p": top_p, "min_p": min_p}
    rows = {}
    for name, v in params.items():
        if isinstance(v, torch.Tensor):
            if name == "top_k" and v.dtype == torch.int64:
                v = v.clamp(0, 2**31 - 1)
            rows[name] = r.per_row(v, name, torch.int32 if name == "top_k" else torch.float32)
            params[name] = _SAMPLING_OFF[name]
    p = _lib.RtCatSampling(u.data_ptr(), *((_lib.ptr(rows.get(k)) for k in params) if rows else (None,) * 4),
                           *_sampling(*params.values()))
    out = Sample(r.empty(torch.int64), r.empty(), r.empty())
    if r.n == 0:
        return out
    ws, n = _workspace("rt_cat_sample_workspace_bytes", r)
    r.call(_lib.load().rt_cat_sample, "rt_cat_sample", ctypes.byref(r.arg()), ctypes.byref(p), out.action.data_ptr(),
           out.logprob.data_ptr(), out.kept_logprob.data_ptr(), _lib.ptr(ws), n)
    return out


@functools.lru_cache(maxsize=256)
def _ppo_hparams(temperature, low, high, ent_coef, kl_coef):
    return _lib.RtCatPpoHparams(_coef(temperature, "temperature", positive=True), _coef(low, "clip_coef", low=0.0),
                                _coef(high, "clip_coef_high", low=0.0), _coef(ent_coef, "ent_coef"),
                                _coef(kl_coef, "kl_coef"))


class _Ppo:
    """The arguments of a PPO loss, checked and laid out."""

    def __init__(self, logits, actions, old_logprobs, advantages, weights, ref_logprobs, temperature, clip_coef,
                 clip_coef_high, ent_coef, kl_coef):
        r = self.r = _Rows(logits)
        if actions is None or old_logprobs is None or advantages is None:
            raise TypeError("actions, old_logprobs, advantages: expected tensors")
        self.actions = r.per_row(actions, "actions", torch.int64)
        self.held = (r.per_row(old_logprobs, "old_logprobs"), r.per_row(advantages, "advantages"),
                     r.per_row(weights, "weights"), r.per_row(ref_logprobs, "ref_logprobs"))
        self.hp = _ppo_hparams(float(temperature), float(clip_coef),
                               float(clip_coef if clip_coef_high is None else clip_coef_high), float(ent_coef), float(kl_coef))
        if self.hp.kl_coef != 0.0 and ref_logprobs is None:
            raise ValueError("kl_coef without ref_logprobs")

    def run(self, grad=None, stride=0, keep=False):
        """(PpoLoss, row state or None); the gradient into `grad`."""
        r = self.r
        f32 = dict(dtype=torch.float32, device=r.device)
        res = PpoLoss(torch.empty((), **f32), r.empty(), r.empty(), torch.empty(6, **f32))
        state = torch.empty((r.n, _lib.CAT_ROW_STATE), dtype=torch.float64, device=r.device) if keep else None
        if r.n == 0:
            res.loss.zero_()
            res.stats.zero_()
            return res, state
        ws, n = _workspace("rt_cat_loss_workspace_bytes", r)
        batch = _lib.RtCatPpoBatch(self.actions.data_ptr(), *map(_lib.ptr, self.held))
        out = _lib.RtCatPpoOut(res.loss.data_ptr(), res.logprob.data_ptr(), res.entropy.data_ptr(),
                               res.stats.data_ptr(), _lib.ptr(grad), stride, _lib.ptr(state))
        r.call(_lib.load().rt_cat_ppo, "rt_cat_ppo", ctypes.byref(r.arg()), ctypes.byref(batch), ctypes.byref(self.hp),
               ctypes.byref(out), _lib.ptr(ws), n)
        return res, state


class _Final(torch.autograd.Function):
    """A gradient by `logits` that is not differentiated: trying to raises."""

    @staticmethod
    def forward(ctx, grad, logits):
        return grad

    @staticmethod
    def backward(ctx, g):
        raise RuntimeError("ppo_loss and distill_loss are differentiated once only")


def _no_capture(device):
    # A captured backward pass ends the process where an eager graph of the same leaves is alive (their
    # nodes keep its stream): nothing here can tell.
    if torch.cuda.current_device() == device.index:
        capturing = torch.cuda.is_current_stream_capturing()
    else:
        with torch.cuda.device(device):
            capturing = torch.cuda.is_current_stream_capturing()
    if capturing:
        raise RuntimeError("logits require grad while a graph is captured: take the _grad form")


def _once(backward):
    def run(ctx, gloss):
        _no_capture(gloss.device)
        if not torch.is_grad_enabled():  # no graph of the gradient is asked for
            return backward(ctx, gloss), None
        with torch.no_grad():
            grad = backward(ctx, gloss)
        return _Final.apply(grad, ctx.saved_tensors[0]), None

    return staticmethod(run)


def _differentiated(logits) -> bool:
    if forward_ad.unpack_dual(logits).tangent is not None:
        raise RuntimeError("ppo_loss and distill_loss have no forward mode: the logits' tangent would be lost")
    return torch.is_grad_enabled() and logits.requires_grad


def _with_grad(fn, logits, op):
    _no_capture(logits.device)
    loss = fn.apply(logits, op)
    return op.rest._replace(loss=loss)


class _PpoFn(torch.autograd.Function):
    """The loss alone: the other results go by `op`."""

    @staticmethod
    def forward(ctx, logits, op):
        op.rest, state = op.run(keep=True)
        ctx.temperature = op.hp.temperature
        ctx.save_for_backward(logits, op.actions, state)
        return op.rest.loss

    @_once
    def backward(ctx, gloss):
        logits, actions, state = ctx.saved_tensors
        r = _Rows(logits)
        grad, stride = r.grad_buffer(None)
        if r.n == 0:
            return grad
        if gloss.dtype != torch.float32:
            gloss = gloss.float()
        r.call(_lib.load().rt_cat_ppo_backward, "rt_cat_ppo_backward", ctypes.byref(r.arg()), actions.data_ptr(),
               ctx.temperature, state.data_ptr(), gloss.data_ptr(), grad.data_ptr(), stride)
        return grad


def ppo_loss(logits, actions, old_logprobs, advantages, *, weights=None, ref_logprobs=None, temperature=1.0,
             clip_coef=0.2, clip_coef_high=None, ent_coef=0.0, kl_coef=0.0) -> PpoLoss:
    """The clipped PPO loss of a categorical policy (rt_cat_ppo): the weighted
    sum over rows of the surrogate, - ent_coef * entropy, + kl_coef * the KL
    estimate against ref_logprobs.

    temperature: the one that old_logprobs (and ref_logprobs) were taken at, as
    sample's logprob.  weights: one per row, None: 1 / rows each.  A row with
    weight 0 or an action outside the vocabulary is ignored.  Only `loss` is
    differentiable, and only with respect to the logits."""
    op = _Ppo(logits, actions, old_logprobs, advantages, weights, ref_logprobs, temperature, clip_coef,
              clip_coef_high, ent_coef, kl_coef)
    if _differentiated(logits):
        return _with_grad(_PpoFn, logits, op)
    return op.run()[0]


def ppo_loss_grad(logits, actions, old_logprobs, advantages, *, weights=None, ref_logprobs=None, temperature=1.0,
                  clip_coef=0.2, clip_coef_high=None, ent_coef=0.0, kl_coef=0.0, out=None):
    """(ppo_loss, its gradient by the logits) in one call, outside autograd.

    out: where the gradient goes: memory apart from the logits, other columns of
    their buffer, or the logits themselves."""
    op = _Ppo(logits, actions, old_logprobs, advantages, weights, ref_logprobs, temperature, clip_coef,
              clip_coef_high, ent_coef, kl_coef)
    grad, stride = op.r.grad_buffer(out)
    return op.run(grad, stride)[0], grad


class _Distill:
    def __init__(self, logits, idx, top, weights, teacher_lse, temperature):
        r = self.r = _Rows(logits)
        if not isinstance(idx, torch.Tensor) or idx.dim() != len(r.lead) + 1:
            raise ValueError("teacher_idx: expected a tensor [..., k]")
        self.k = k = idx.shape[-1]
        if not 1 <= k <= _lib.CAT_MAX_TOP:
            raise ValueError(f"teacher_idx: {k} entries in a row, expected 1 to {_lib.CAT_MAX_TOP}")
        if top is None:
            raise TypeError("teacher_logits: expected a tensor")
        self.idx = r.per_row(idx, "teacher_idx", torch.int64, (k,))
        self.top = r.per_row(top, "teacher_logits", torch.float32, (k,))
        self.lse = r.per_row(teacher_lse, "teacher_lse")
        self.weights = r.per_row(weights, "weights")
        self.temperature = _coef(temperature, "temperature", positive=True)

    def arg(self):
        return _lib.RtCatTeacher(self.idx.data_ptr(), self.top.data_ptr(), _lib.ptr(self.lse),
                                 _lib.ptr(self.weights), self.k, self.temperature)

    def run(self, grad=None, stride=0, keep=False):
        r = self.r
        res = DistillLoss(torch.empty((), dtype=torch.float32, device=r.device), r.empty())
        state = torch.empty((r.n, _lib.CAT_ROW_STATE), dtype=torch.float64, device=r.device) if keep else None
        if r.n == 0:
            res.loss.zero_()
            return res, state
        ws, n = _workspace("rt_cat_loss_workspace_bytes", r)
        out = _lib.RtCatDistillOut(res.loss.data_ptr(), res.kl.data_ptr(), _lib.ptr(grad), stride, _lib.ptr(state))
        r.call(_lib.load().rt_cat_distill, "rt_cat_distill", ctypes.byref(r.arg()), ctypes.byref(self.arg()),
               ctypes.byref(out), _lib.ptr(ws), n)
        return res, state


class _DistillFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, op):
        op.rest, state = op.run(keep=True)
        ctx.k, ctx.temperature = op.k, op.temperature
        ctx.save_for_backward(logits, op.idx, op.top, state)  # (weights and lse are in the state)
        return op.rest.loss

    @_once
    def backward(ctx, gloss):
        logits, idx, top, state = ctx.saved_tensors  # raises where one of them was changed in place
        r = _Rows(logits)
        grad, stride = r.grad_buffer(None)
        if r.n == 0:
            return grad
        if gloss.dtype != torch.float32:
            gloss = gloss.float()
        teacher = _lib.RtCatTeacher(idx.data_ptr(), top.data_ptr(), None, None, ctx.k, ctx.temperature)
        r.call(_lib.load().rt_cat_distill_backward, "rt_cat_distill_backward", ctypes.byref(r.arg()),
               ctypes.byref(teacher), state.data_ptr(), gloss.data_ptr(), grad.data_ptr(), stride)
        return grad


def distill_loss(logits, teacher_idx, teacher_logits, *, weights=None, teacher_lse=None, temperature=1.0) -> DistillLoss:
    """KL from a teacher's top logits (rt_cat_distill), both sides at
    `temperature`: sum_n w_n sum_j q_j (log q_j - log softmax(x / T)[idx_j]).

    teacher_idx, teacher_logits [..., k]: entries outside the vocabulary (-1)
    are unused.  teacher_lse: the teacher's logsumexp(logits / T) over its whole
    vocabulary; without it its probabilities are normalised over the k.
    weights: as ppo_loss.  Only `loss` is differentiable, by the logits."""
    op = _Distill(logits, teacher_idx, teacher_logits, weights, teacher_lse, temperature)
    if _differentiated(logits):
        return _with_grad(_DistillFn, logits, op)
    return op.run()[0]


def distill_loss_grad(logits, teacher_idx, teacher_logits, *, weights=None, teacher_lse=None, temperature=1.0, out=None):
    """(distill_loss, its gradient by the logits) in one call, outside autograd; `out` as ppo_loss_grad."""
    op = _Distill(logits, teacher_idx, teacher_logits, weights, teacher_lse, temperature)
    grad, stride = op.r.grad_buffer(out)
    return op.run(grad, stride)[0], grad
