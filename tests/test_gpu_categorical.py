"""Categorical-policy operators (ppo_radiotherapy_amd.categorical) on the GPU
against their definitions in 64 bits (tests/cat_plain.py): sampling, the PPO
loss and distillation, with their gradients, over row lengths, types, strides
and special rows."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

import cat_plain as P  # noqa: E402

INF, NAN = math.inf, math.nan
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
# one entry, one lane's worth, around a wave, around a block's tile, odd and large
VOCABS = [1, 2, 3, 11, 16, 17, 63, 64, 65, 127, 300, 1000, 1024, 1025, 4096, 4097, 8191, 20011, 50021]


@pytest.fixture(scope="module")
def C():
    import _rtpkg  # noqa: F401
    from ppo_radiotherapy_amd import categorical

    return categorical


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def rows(n, v, dtype, seed, pad=0, off=0, kind="normal"):
    """[n, v] logits inside a wider buffer whose other places hold NaN."""
    g = gen(seed)
    flat = torch.full((off + n * (v + pad),), NAN, dtype=dtype, device="cuda")
    x = flat.as_strided((n, v), (v + pad, 1), off)
    if kind == "ties":       # few distinct values: every cut falls among equals
        x.copy_(torch.randint(-3, 4, (n, v), generator=g, device="cuda"))
    elif kind == "flat":
        x.fill_(1.5)
    elif kind == "peaked":
        x.copy_(torch.randn(n, v, generator=g, device="cuda") * 8)
    else:
        x.copy_(torch.randn(n, v, generator=g, device="cuda") * 2)
    return x


def check_sample(C, x, u, par):
    n = x.shape[0]
    got = C.sample(x, u, **par)
    full = {k: (t.cpu().numpy() if torch.is_tensor(t) else np.full(n, t)) for k, t in
            ({"temperature": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0} | par).items()}
    a, lp, kp = P.sample(x.double().cpu().numpy(), u.double().cpu().numpy(), full["temperature"].astype(np.float32),
                         full["top_k"], full["top_p"].astype(np.float32), full["min_p"].astype(np.float32))
    assert got.action.dtype == torch.int64 and got.logprob.dtype == torch.float32
    np.testing.assert_array_equal(got.action.cpu().numpy(), a)
    # whole-number sums: what is left is the rounding of the result, and of exp and log (2^-50)
    for mine, want in ((got.logprob, lp), (got.kept_logprob, kp)):
        mine = mine.double().cpu().numpy()
        np.testing.assert_array_equal(np.isnan(mine), np.isnan(want))
        ok = ~np.isnan(want)
        assert (np.abs(mine - want)[ok] <= 2.0 ** -24 * np.abs(want[ok]) + 2.0 ** -40).all()
    return got


FILTERS = {
    "none": {}, "k": {"top_k": 7}, "k1": {"top_k": 1}, "p": {"top_p": 0.8}, "p0": {"top_p": 0.0},
    "min_p": {"min_p": 0.1}, "min_p1": {"min_p": 1.0}, "k+p": {"top_k": 20, "top_p": 0.7, "temperature": 0.7},
    "all": {"top_k": 300, "top_p": 0.95, "min_p": 0.01, "temperature": 1.7}, "greedy": {"temperature": 0.0},
    "big k": {"top_k": 3000, "top_p": 0.97},
}


@pytest.mark.parametrize("v", VOCABS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_sample_lengths(C, v, dtype):
    for i, (name, par) in enumerate(FILTERS.items()):
        x = rows(5, v, dtype, 100 * v + i, pad=(0, 3, 8)[i % 3], off=i % 2)
        u = torch.rand(5, generator=gen(v + i), device="cuda")
        check_sample(C, x, u, par)


@pytest.mark.parametrize("kind", ["ties", "flat", "peaked"])
@pytest.mark.parametrize("v", [5, 64, 700, 5000, 33000])
@pytest.mark.parametrize("dtype", DTYPES)
def test_sample_ties_and_peaks(C, kind, v, dtype):
    for i, par in enumerate(FILTERS.values()):
        x = rows(4, v, dtype, v + i, kind=kind)
        check_sample(C, x, torch.rand(4, generator=gen(i), device="cuda"), par)


@pytest.mark.parametrize("v", [11, 1000, 9000, 20000])
def test_sample_extreme_numbers(C, v):
    """u at and beyond its ends; per-row parameters at and beyond theirs."""
    u = torch.tensor([0.0, 2.0 ** -24, 0.5, 1 - 2.0 ** -24, 1.0, 3.0, -1.0, NAN, INF], device="cuda")
    n = len(u)
    x = rows(n, v, torch.float32, 3)
    check_sample(C, x, u, {})
    check_sample(C, x, u, {"top_k": 3, "top_p": 0.5})
    t = torch.tensor([1e-38, 1e-45, 1e30, INF, NAN, -1.0, 0.0, 1.0, 3.0], device="cuda")
    k = torch.tensor([0, -5, v, v + 1, 2 ** 31 - 1, 1, 2, v - 1, 5], dtype=torch.int32, device="cuda")
    p = torch.tensor([NAN, 1.0, 1e-30, -1.0, 2.0, 1 - 2.0 ** -24, 0.3, 0.5, 0.9], device="cuda")
    q = torch.tensor([NAN, -1.0, 0.0, 2.0, 1.0, 1e-30, 0.5, 0.01, 0.1], device="cuda")
    u = torch.rand(n, generator=gen(1), device="cuda")
    for par in ({"temperature": t}, {"top_k": k}, {"top_p": p}, {"min_p": q},
                {"temperature": t, "top_k": k, "top_p": p, "min_p": q}):
        check_sample(C, x, u, par)
    check_sample(C, x, u, {"top_k": k.long() * 4})


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v", [3, 70, 1500, 20000])
def test_sample_special_rows(C, dtype, v):
    low = torch.finfo(dtype).min
    x = rows(12, v, dtype, 9)
    x[0] = -INF
    x[1, 1:] = -INF
    x[2, :-1] = -INF
    x[3, v // 2] = NAN
    x[4, -1] = INF
    x[5] = NAN
    x[6] = low
    x[7, 1:] = low
    x[8, ::2] = -INF
    x[9] = torch.finfo(dtype).max
    x[10] = 0.0
    x[10, ::2] = -0.0
    x[11] = -INF
    x[11, v // 2] = low
    u = torch.rand(12, generator=gen(2), device="cuda")
    for par in FILTERS.values():
        check_sample(C, x, u, par)


@pytest.mark.parametrize("v", [9217, 70000, 200003])
def test_sample_bf16_of_every_magnitude(C, v):
    """Numbers from the least to the largest that bf16 has, those that weigh something and those that do not."""
    x = rows(13, v, torch.bfloat16, 15, pad=3, off=1)
    odd = torch.randperm(v, generator=gen(16), device="cuda")[:400]
    bits = lambda lo, hi: torch.randint(lo, hi, (400,), generator=gen(17), device="cuda").short().view(torch.bfloat16)  # noqa: E731
    x[0, odd] = bits(1, 128)                  # subnormal
    x[1] *= 2.0 ** -20
    x[2] *= 2.0 ** -40                        # next to one another, all weigh the same or nearly
    x[3, odd] = bits(0x4580, 0x4680)          # 2^12 and more
    x[4, odd] = -bits(0x4580, 0x7f80)
    x[5] = -(x[5].abs() * 2.0 ** 13)          # nothing above -2^12
    x[5] = x[5].clamp(max=-5000.0)
    x[6] = -x[6].abs() - 5.0                  # all negative, tiny ones on top
    x[6, odd] = -bits(1, 0x2d80)
    x[7, odd] = bits(1, 0x2d80)               # tiny ones where they weigh nothing
    x[7, odd[0]] = 100.0
    x[8] = -INF
    x[8, odd] = bits(0, 0x7f80)
    x[9] = -INF
    x[9, odd] = bits(1, 0x2d80)
    x[10] = -INF
    x[10, odd] = -bits(0x4580, 0x7f80)
    x[11, odd] = bits(0x2d80, 0x2e00)         # the borders of 2^-36
    x[12, odd] = bits(0x4570, 0x4580)         # and of 2^12
    u = torch.rand(13, generator=gen(18), device="cuda")
    for par in (*FILTERS.values(), {"temperature": 3000.0}, {"temperature": 1e32, "top_p": 0.5}, {"temperature": 1e-3, "top_k": 40}):
        check_sample(C, x, u, par)


@pytest.mark.parametrize("v", [57343, 57345, 114688, 2 ** 20])
def test_sample_more_equal_logits_than_16_bits_count(C, v):
    for i, par in enumerate(FILTERS.values()):
        x = rows(2, v, torch.bfloat16, 19, off=i % 2, kind="flat")
        x[1, v // 3:] = -2.0
        check_sample(C, x, torch.rand(2, generator=gen(20 + i), device="cuda"), par)


def test_sample_large_batches(C):
    """More rows than a grid holds at once, wide rows of every filter side by side, and one long row."""
    g = gen(4)
    x = torch.randn(30001, 11, generator=g, device="cuda")
    check_sample(C, x, torch.rand(30001, generator=g, device="cuda"), {})
    n, v = 40, 131072
    x = (torch.randn(n, v, generator=g, device="cuda") * 2).bfloat16()
    pick = lambda *s: torch.tensor(s, device="cuda")[torch.randint(len(s), (n,), generator=g, device="cuda")]  # noqa: E731
    par = {"temperature": pick(0.0, 0.5, 1.0, 2.0), "top_k": pick(0, 1, 50, 5000).int(),
           "top_p": pick(1.0, 0.95, 0.5), "min_p": pick(0.0, 0.05)}
    check_sample(C, x, torch.rand(n, generator=g, device="cuda"), par)
    x = torch.randn(1, 2 ** 20, generator=g, device="cuda")
    for par in ({}, {"top_p": 0.9}, {"top_k": 100}, {"top_k": 100000, "top_p": 0.5}):
        check_sample(C, x, torch.rand(1, generator=g, device="cuda"), par)


def test_sample_frequencies(C):
    """Equal steps of u meet each kept entry as often as its probability says (within one step)."""
    n = 4096
    x = torch.randn(1, 37, generator=gen(5), device="cuda")
    u = (torch.arange(n, device="cuda") + 0.5) / n
    a = C.sample(x.expand(n, 37), u, top_k=10, temperature=1.3).action
    top = x[0].topk(10)
    p = torch.softmax(top.values.double() / 1.3, 0)
    count = torch.bincount(a, minlength=37)
    assert int(count.sum()) == int(count[top.indices].sum()) == n
    assert ((count[top.indices] - p * n).abs() <= 1.0).all()


def small_numbers(kind, n, v, seed):
    """Rows whose numbers next to 0 spread over many binades."""
    g = gen(seed)
    if kind == "logsigmoid":    # half of them within 1e-6 of 0
        return torch.nn.functional.logsigmoid(30 * torch.randn(n, v, generator=g, device="cuda"))
    if kind == "powers":        # a binade each, and zeros behind them
        x = torch.zeros(n, v, device="cuda")
        many = min(v, 150)
        x[:, :many] = 2.0 ** (27 - torch.arange(many, device="cuda", dtype=torch.float64)).float()
        return torch.gather(x, 1, torch.rand(n, v, generator=g, device="cuda").argsort(1))
    x = 10.0 ** -(3 + 35 * torch.rand(n, v, generator=g, device="cuda", dtype=torch.float64))
    if kind == "both":
        x *= torch.where(torch.rand(n, v, generator=g, device="cuda") < 0.5, -1.0, 1.0)
    else:
        x = -x
    return x.float()


@pytest.mark.parametrize("kind", ["logsigmoid", "below", "both", "powers"])
@pytest.mark.parametrize("v", [40, 300, 2000, 9000, 20000])
@pytest.mark.parametrize("dtype", DTYPES)
def test_sample_cut_among_small_numbers(C, kind, v, dtype):
    """The cut between numbers that one bin holds and that are tens of binades apart."""
    x = small_numbers(kind, 4, v, v).to(dtype)
    t = 1e10 if kind == "powers" else 1.0
    for i, par in enumerate(({"top_k": 7}, {"top_k": 100}, {"top_k": 129}, {"top_k": 140}, {"top_k": 400}, {"top_k": 1500},
                             {"top_p": 0.613}, {"top_p": 0.03}, {"top_k": 300, "top_p": 0.37})):
        check_sample(C, x, torch.rand(4, generator=gen(i), device="cuda"), par | {"temperature": t})


@pytest.mark.parametrize("v", [9300, 70001])
def test_sample_bf16_at_the_border_of_the_places(C, v):
    """2^-36, which has no place of its own and weighs nothing, and is the only number near 0, in rows after others of
    zeros."""
    n = 600 if v < 10000 else 520
    x = torch.zeros(n, v, dtype=torch.bfloat16, device="cuda")
    x[512:] = 2.0 ** -36
    x[512:, v // 2] = 100.0
    x[512:, v - 3] = 99.5
    x[515, 7:] = 100.0
    u = torch.rand(n, generator=gen(n), device="cuda")
    for par in ({}, {"temperature": 0.0}, {"temperature": 2.0, "min_p": 1e-30}, {"top_k": v - 1}):
        check_sample(C, x, u, par)


# ---- losses ---------------------------------------------------------------
def ppo_inputs(n, v, seed, logits):
    g = gen(seed)
    a = torch.randint(0, v, (n,), generator=g, device="cuda")
    lp = torch.log_softmax(logits.double().nan_to_num(0, 0, -30), 1).gather(1, a[:, None])[:, 0]
    old = (lp + 0.3 * torch.randn(n, generator=g, device="cuda")).float()
    ref = (lp + 0.2 * torch.randn(n, generator=g, device="cuda")).float()
    adv = torch.randn(n, generator=g, device="cuda")
    w = torch.rand(n, generator=g, device="cuda")
    return a, old, adv, w, ref


def teacher_inputs(n, v, k, seed):
    g = gen(seed)
    idx = torch.randint(0, v, (n, k), generator=g, device="cuda")
    return idx, torch.randn(n, k, generator=g, device="cuda") * 3, torch.rand(n, generator=g, device="cuda")


def near(got, want, names):
    for k in names:
        value, tol = want[k]
        d = (got[k].double() - value).abs()
        # also the value rounded to the output's type, which past the type's range is an infinity
        same = (got[k] == value.to(got[k].dtype)) | (got[k].isnan() & value.isnan())
        bad = ~(same | (d <= tol))
        assert not bad.any(), f"{k}: {int(bad.sum())} of {bad.numel()} off, the worst by {float((d / tol.clamp(min=1e-300))[bad].max()):.3g} of its tolerance"


def run_ppo(C, x, a, old, adv, grad=True, **kw):
    r, g = C.ppo_loss_grad(x, a, old, adv, **kw)
    return r._asdict() | {"grad": g}


@pytest.mark.parametrize("v", VOCABS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_ppo_lengths(C, v, dtype):
    for i, (n, pad, off) in enumerate([(1, 0, 0), (6, 0, 1), (70, 5, 0), (9, 8, 3)]):
        x = rows(n, v, dtype, v + i, pad, off, kind=("normal", "peaked", "normal", "flat")[i])
        a, old, adv, w, ref = ppo_inputs(n, v, v + i, x)
        want = P.ppo(x, a, old, adv, w, ref, 0.9, 0.2, 0.3, 0.01, 0.1)
        got = run_ppo(C, x, a, old, adv, weights=w, ref_logprobs=ref, temperature=0.9, clip_coef=0.2,
                      clip_coef_high=0.3, ent_coef=0.01, kl_coef=0.1)
        near(got, want, ("loss", "stats", "logprob", "entropy", "grad"))
        # the loss alone, and the gradient through autograd with a factor behind it
        alone = C.ppo_loss(x, a, old, adv, weights=w, ref_logprobs=ref, temperature=0.9, clip_coef=0.2,
                           clip_coef_high=0.3, ent_coef=0.01, kl_coef=0.1)
        near(alone._asdict(), want, ("loss", "stats", "logprob", "entropy"))
        want = P.ppo(x, a, old, adv, None, None, 1.0, 0.2, 0.2, 0.0, 0.0, scale=-2.5)
        leaf = x.detach().requires_grad_()
        r = C.ppo_loss(leaf, a, old, adv)
        near(r._asdict(), want, ("loss", "stats", "logprob", "entropy"))
        g, = torch.autograd.grad(-2.5 * r.loss, leaf)
        near({"grad": g}, want, ("grad",))


@pytest.mark.parametrize("v,k", [(1, 1), (2, 3), (11, 4), (17, 16), (64, 8), (65, 65), (300, 256), (1000, 33), (1025, 7),
                                 (4097, 64), (20011, 1024), (50021, 33)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_distill_lengths(C, v, k, dtype):
    for i, (n, pad, off) in enumerate([(1, 0, 0), (6, 0, 1), (70, 5, 0), (9, 8, 3)]):
        x = rows(n, v, dtype, v + i, pad, off, kind=("normal", "peaked", "normal", "flat")[i])
        idx, top, w = teacher_inputs(n, v, k, v + i)
        lse = torch.logsumexp(top / 2.0, 1) + 0.3 if i % 2 else None
        if i > 1:
            idx[0] = -1                # a teacher without entries
            idx[1, k // 2:] = v + 5    # ... with fewer
            top[1, k // 2:] = NAN
            idx[2] = int(idx[2, 0])         # the same index throughout
            top[3, 0] = -INF
        want = P.distill(x, idx, top, w, lse, 2.0)
        r, g = C.distill_loss_grad(x, idx, top, weights=w, teacher_lse=lse, temperature=2.0)
        near(r._asdict() | {"grad": g}, want, ("loss", "kl", "grad"))
        want = P.distill(x, idx, top, None, lse, 2.0, scale=3.0)
        leaf = x.detach().requires_grad_()
        r = C.distill_loss(leaf, idx, top, teacher_lse=lse, temperature=2.0)
        g, = torch.autograd.grad(3.0 * r.loss, leaf)
        near(r._asdict() | {"grad": g}, want, ("loss", "kl", "grad"))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v", [5, 100, 3000, 40000])
def test_losses_special_rows(C, dtype, v):
    """Masked entries, rows of nothing, ignored rows whose numbers are NaN, a NaN that counts."""
    n = 10
    x = rows(n, v, dtype, 21)
    low = torch.finfo(dtype).min
    a, old, adv, w, ref = ppo_inputs(n, v, 21, x)
    x[0] = -INF
    x[1, 1:] = -INF
    a[1] = 0
    x[2, ::2] = -INF
    a[2] = 1
    x[3] = NAN
    w[3] = 0.0
    x[4] = INF
    a[4] = -1
    a[5] = v
    x[6] = low
    x[7, 1:] = low
    a[7] = 0
    x[8] = torch.finfo(dtype).max
    kw = dict(weights=w, ref_logprobs=ref, ent_coef=0.02, kl_coef=0.1)
    want = P.ppo(x, a, old, adv, w, ref, ent=0.02, klc=0.1)
    near(run_ppo(C, x, a, old, adv, **kw), want, ("loss", "stats", "logprob", "entropy", "grad"))
    leaf = x.detach().requires_grad_()
    g, = torch.autograd.grad(C.ppo_loss(leaf, a, old, adv, **kw).loss, leaf)
    near({"grad": g}, want, ("grad",))
    assert not g[[0, 3, 4, 5]].any()

    x[4] = 1.0
    idx, top, w = teacher_inputs(n, v, 3, 22)
    w[3] = 0.0
    idx[1] = 0
    idx[2] = torch.tensor([1, 3, 1])
    want = P.distill(x, idx, top, w)
    r, g = C.distill_loss_grad(x, idx, top, weights=w)
    near(r._asdict() | {"grad": g}, want, ("loss", "kl", "grad"))
    leaf = x.detach().requires_grad_()
    g, = torch.autograd.grad(C.distill_loss(leaf, idx, top, weights=w).loss, leaf)
    near({"grad": g}, want, ("grad",))

    # a NaN in a row that counts, and all of one: the loss and that row say so, the others do not notice
    for fill in (slice(1, 2), slice(None)):
        y = rows(3, v, dtype, 23)
        y[1, fill] = NAN
        a, old, adv, w, _ = ppo_inputs(3, v, 23, y)
        r, g = C.ppo_loss_grad(y, a, old, adv)
        assert r.loss.isnan() and r.logprob.isnan().tolist() == [False, True, False]
        assert g.isnan().any(1).tolist() == [False, True, False]
        idx, top, _ = teacher_inputs(3, v, 2, 24)
        r, g = C.distill_loss_grad(y, idx, top)
        assert r.loss.isnan() and r.kl.isnan().tolist() == [False, True, False]
        assert g.isnan().any(1).tolist() == [False, True, False]


def test_distill_impossible_entry(C):
    """A student that rules out what the teacher names: infinite, with a finite gradient."""
    x = torch.zeros(2, 4, device="cuda")
    x[0, 2] = -INF
    idx = torch.tensor([[2, 0], [2, 0]], device="cuda")
    r, g = C.distill_loss_grad(x, idx, torch.zeros(2, 2, device="cuda"))
    assert r.loss == INF and r.kl[0] == INF and r.kl[1].isfinite()
    assert torch.allclose(g[0].double(), torch.tensor([1 / 6 - 1 / 4, 1 / 6, -1 / 4, 1 / 6], device="cuda", dtype=torch.float64), atol=2.0 ** -20)


def test_ppo_clip_sides(C):
    """The clipped side has no gradient, the other has; both signs of the advantage."""
    x = torch.randn(4, 9, generator=gen(6), device="cuda")
    a = torch.tensor([0, 1, 2, 3], device="cuda")
    lp = torch.log_softmax(x.double(), 1).gather(1, a[:, None])[:, 0]
    old = (lp - torch.tensor([0.5, 0.5, -0.5, -0.5], device="cuda")).float()
    adv = torch.tensor([1.0, -1.0, 1.0, -1.0], device="cuda")
    r, g = C.ppo_loss_grad(x, a, old, adv, clip_coef=0.2)
    assert g.any(1).tolist() == [False, True, True, False] and r.stats[5] == 1.0


def test_gradients_against_differences(C):
    """Along random directions, the oracle's loss in 64 bits changes by what the kernels' gradients say."""
    n, v = 7, 53
    x = torch.randn(n, v, generator=gen(7), device="cuda")
    a, old, adv, w, ref = ppo_inputs(n, v, 7, x)
    idx, top, _ = teacher_inputs(n, v, 5, 7)
    g1 = C.ppo_loss_grad(x, a, old, adv, weights=w, ref_logprobs=ref, temperature=1.3, ent_coef=0.1, kl_coef=0.2)[1]
    g2 = C.distill_loss_grad(x, idx, top, weights=w, temperature=1.7)[1]
    f1 = lambda y: P.ppo(y, a, old, adv, w, ref, 1.3, 0.2, 0.2, 0.1, 0.2)["loss"][0]  # noqa: E731
    f2 = lambda y: P.distill(y, idx, top, w, None, 1.7)["loss"][0]  # noqa: E731
    for s in range(5):
        d = torch.randn(n, v, generator=gen(70 + s), device="cuda", dtype=torch.float64)
        for f, g in ((f1, g1), (f2, g2)):
            h = 1e-5  # truncation h^2, cancellation 2^-52 / h
            slope = (f(x.double() + h * d) - f(x.double() - h * d)) / (2 * h)
            size = (g.double() * d).abs().sum()
            assert abs(float(slope - (g.double() * d).sum())) <= 1e-6 * float(size) + 1e-8


@pytest.mark.parametrize("v", [11, 300, 5000, 60000])
def test_shapes_strides_and_places(C, v):
    """Leading dimensions, broadcast rows, one row, no rows, gradients into given memory and in place."""
    g = gen(8)
    x = torch.randn(4, 3, v + 2, generator=g, device="cuda")[..., 1:-1]
    u = torch.rand(4, 3, generator=g, device="cuda")
    flat = x.reshape(12, v)
    s, t = C.sample(x, u, top_k=5), C.sample(flat, u.reshape(12), top_k=5)
    assert s.action.shape == (4, 3) and torch.equal(s.action.reshape(12), t.action)
    a, old, adv, w, _ = ppo_inputs(12, v, 8, flat)
    shape = lambda q: q.reshape(4, 3)  # noqa: E731
    r1, g1 = C.ppo_loss_grad(x, shape(a), shape(old), shape(adv))
    r2, g2 = C.ppo_loss_grad(flat, a, old, adv)
    assert g1.shape == x.shape and torch.equal(g1.reshape(12, v), g2) and torch.equal(r1.loss, r2.loss)
    one = C.ppo_loss_grad(flat[0], a[0], old[0], adv[0])[1]
    two = C.ppo_loss_grad(flat[:1], a[:1], old[:1], adv[:1])[1]
    assert one.shape == (v,) and torch.equal(one, two[0])
    # broadcast rows: the gradient of the row they come from is the sum
    base = flat[:1].clone().requires_grad_()
    C.ppo_loss(base.expand(12, v), a, old, adv).loss.backward()
    many = C.ppo_loss_grad(flat[:1].repeat(12, 1), a, old, adv)[1]
    assert torch.allclose(base.grad[0].double(), many.double().sum(0), rtol=0, atol=12 * 2.0 ** -22 * float(many.abs().max()))
    # given memory: what lies between the rows stays
    for dtype in DTYPES:
        y = flat.to(dtype)
        ref = C.ppo_loss_grad(y, a, old, adv)[1]
        wide = torch.full((12, v + 7), 5.0, dtype=dtype, device="cuda")
        got = C.ppo_loss_grad(y, a, old, adv, out=wide[:, 2:v + 2])[1]
        assert torch.equal(got, ref) and (wide[:, :2] == 5).all() and (wide[:, v + 2:] == 5).all()
        idx, top, w = teacher_inputs(12, v, 4, 8)
        idx[0] = 0
        # in place: the bits of a gradient elsewhere, from the same rows (where a row starts within 16 bytes
        # decides which entries are added first, so not from a copy that lies differently)
        z = y.clone()
        want = C.distill_loss_grad(z, idx, top)[1]
        assert torch.equal(C.distill_loss_grad(z, idx, top, out=z)[1], want) and torch.equal(z, want)
        z = torch.nn.functional.pad(y, (1, 2))[:, 1:-2]
        want = C.ppo_loss_grad(z, a, old, adv)[1]
        near({"grad": want}, P.ppo(z, a, old, adv), ("grad",))
        C.ppo_loss_grad(z, a, old, adv, out=z)
        assert torch.equal(z, want)
    none = torch.empty(0, v, device="cuda", requires_grad=True)
    e = torch.empty(0, device="cuda")
    assert C.sample(none, e).action.shape == (0,)
    r = C.ppo_loss(none, e.long(), e, e)
    r.loss.backward()
    assert r.loss == 0 and none.grad.shape == (0, v)
    r, gr = C.distill_loss_grad(none, torch.empty(0, 3, dtype=torch.int64, device="cuda"), torch.empty(0, 3, device="cuda"))
    assert r.loss == 0 and gr.shape == (0, v)


@pytest.mark.parametrize("n", [1, 2, 5, 33, 200])
@pytest.mark.parametrize("v,dtype", [(8192, torch.float32), (20011, torch.bfloat16), (131073, torch.float16), (2 ** 20, torch.bfloat16)])
def test_few_long_rows(C, n, v, dtype):
    """Rows that several blocks share: every operator, loss alone, gradient elsewhere, in place and through autograd."""
    if n * v > 2 ** 25:
        n = max(1, 2 ** 25 // v)
    x = rows(n, v, dtype, n + v, pad=5, off=1)
    x[0, : v // 2] = -INF
    a, old, adv, w, ref = ppo_inputs(n, v, n, x)
    a[0] = v - 1
    kw = dict(weights=w, ref_logprobs=ref, ent_coef=0.05, kl_coef=0.1, temperature=1.2)
    want = P.ppo(x, a, old, adv, w, ref, 1.2, 0.2, 0.2, 0.05, 0.1)
    near(run_ppo(C, x, a, old, adv, **kw), want, ("loss", "stats", "logprob", "entropy", "grad"))
    near(C.ppo_loss(x, a, old, adv, **kw)._asdict(), want, ("loss", "stats", "logprob", "entropy"))
    leaf = x.detach().requires_grad_()
    g, = torch.autograd.grad(C.ppo_loss(leaf, a, old, adv, **kw).loss, leaf)
    near({"grad": g}, want, ("grad",))
    y = x.clone()
    r, g = C.ppo_loss_grad(y, a, old, adv, out=y, **kw)
    near(r._asdict() | {"grad": y}, want, ("loss", "logprob", "grad"))
    idx, top, _ = teacher_inputs(n, v, 70, n)
    idx[:, 1] = idx[:, 0]
    idx[0, 2], idx[0, 3], idx[0, 4] = v - 1, v - 2, -1
    idx[0] = torch.where(idx[0] >= 0, idx[0].clamp(min=v // 2), -1)
    want = P.distill(x, idx, top, w, None, 1.5)
    r, g = C.distill_loss_grad(x, idx, top, weights=w, temperature=1.5)
    near(r._asdict() | {"grad": g}, want, ("loss", "kl", "grad"))
    near(C.distill_loss(x, idx, top, weights=w, temperature=1.5)._asdict(), want, ("loss", "kl"))
    g, = torch.autograd.grad(C.distill_loss(leaf, idx, top, weights=w, temperature=1.5).loss, leaf)
    near({"grad": g}, want, ("grad",))
    y = x.clone()
    C.distill_loss_grad(y, idx, top, weights=w, temperature=1.5, out=y)
    near({"grad": y}, want, ("grad",))
    x = x[:9]
    u = torch.rand(len(x), generator=gen(n), device="cuda")
    for par in ({}, {"top_k": 40, "top_p": 0.9}, {"top_p": 0.95}, {"min_p": 0.05}, {"temperature": 0.0}, {"top_k": 1500}):
        check_sample(C, x, u, par)


def test_rows_past_32_bits(C):
    """Rows that start more than 2^32 bytes and 2^31 elements into their buffer."""
    v, n = 131072, 16500
    x = torch.zeros(n, v, dtype=torch.bfloat16, device="cuda")
    tail = rows(4, v, torch.bfloat16, 31)
    x[-4:] = tail
    a, old, adv, w, _ = ppo_inputs(4, v, 31, tail)
    pad = lambda t, fill: torch.cat([torch.full((n - 4,), fill, dtype=t.dtype, device="cuda"), t])  # noqa: E731
    want = P.ppo(tail, a, old, adv, w)
    r, g = C.ppo_loss_grad(x, pad(a, -1), pad(old, 0.0), pad(adv, 0.0), weights=pad(w, 1.0), out=x)
    near({"loss": r.loss, "logprob": r.logprob[-4:], "grad": g[-4:]}, want, ("loss", "logprob", "grad"))
    assert not g[:-4].any()


def test_repeated_runs_are_bitwise_equal(C):
    for v in (11, 500, 50021):
        x = rows(33, v, torch.bfloat16, 41)
        a, old, adv, w, ref = ppo_inputs(33, v, 41, x)
        first = run_ppo(C, x, a, old, adv, weights=w, ent_coef=0.1)
        idx, top, _ = teacher_inputs(33, v, 9, 41)
        second, grad = C.distill_loss_grad(x, idx, top)
        u = torch.rand(33, generator=gen(1), device="cuda")
        third = C.sample(x, u, top_p=0.9)
        for _ in range(5):
            again = run_ppo(C, x, a, old, adv, weights=w, ent_coef=0.1)
            assert all(torch.equal(again[k], first[k]) for k in first)
            r, g = C.distill_loss_grad(x, idx, top)
            assert torch.equal(g, grad) and torch.equal(r.loss, second.loss)
            assert all(torch.equal(p, q) for p, q in zip(C.sample(x, u, top_p=0.9), third))


@pytest.mark.parametrize("v", [11, 2000, 60000])
def test_graph_and_stream(C, v):
    """Captured on a stream of its own, replayed on changing inputs with eager work between, two graphs side by side."""
    n = 13
    x = torch.empty(n, v, dtype=torch.bfloat16, device="cuda")
    u = torch.empty(n, device="cuda")
    a, old, adv, w, _ = ppo_inputs(n, v, 51, rows(n, v, torch.bfloat16, 51))
    idx, top, _ = teacher_inputs(n, v, 6, 51)

    def step():
        s = C.sample(x, u, top_k=40, top_p=0.9)
        r, g = C.ppo_loss_grad(x, s.action, s.logprob, adv, weights=w, ent_coef=0.01)
        d, h = C.distill_loss_grad(x, idx, top, temperature=1.5)
        return [*s, *r, g, *d, h]

    def fill(seed):
        x.copy_(rows(n, v, torch.bfloat16, seed))
        u.copy_(torch.rand(n, generator=gen(seed), device="cuda"))

    fill(0)
    step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, out))
    for seed in range(1, 5):
        fill(seed)
        want = step()
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            for p, q in zip(out, want):
                assert torch.equal(p, q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_changed_inputs_are_noticed(C):
    """Autograd's own check: logits or actions changed in place between the loss and its gradient."""
    x = torch.randn(3, 20, device="cuda", requires_grad=True)
    y = x * 1.0
    a, old, adv, _, _ = ppo_inputs(3, 20, 61, x.detach())
    r = C.ppo_loss(y, a, old, adv)
    with torch.no_grad():
        y.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        r.loss.backward()


def test_second_derivatives_are_refused(C):
    x = torch.randn(3, 20, device="cuda", requires_grad=True)
    a, old, adv, _, _ = ppo_inputs(3, 20, 64, x.detach())
    idx, top, _ = teacher_inputs(3, 20, 4, 64)
    for loss in (lambda: C.ppo_loss(x, a, old, adv).loss, lambda: C.distill_loss(x, idx, top).loss):
        plain, = torch.autograd.grad(loss(), x)
        g, = torch.autograd.grad(loss(), x, create_graph=True)
        assert torch.equal(g, plain)
        with pytest.raises(RuntimeError, match="once only"):
            torch.autograd.grad(g.sum(), x)
        with pytest.raises(RuntimeError, match="once only"):
            (g.square().sum() + x.sum()).backward()


def test_gradient_in_place_is_noticed(C):
    """Logits that another graph has saved, written over with their gradient."""
    h = torch.randn(3, 20, device="cuda")
    w = torch.ones(3, 20, device="cuda", requires_grad=True)
    z = (w * h).sum()
    a, old, adv, _, _ = ppo_inputs(3, 20, 62, h)
    C.ppo_loss_grad(h, a, old, adv, out=h)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.backward()


def test_autograd_is_refused_in_a_capture(C):
    x = torch.randn(3, 20, device="cuda", requires_grad=True)
    a, old, adv, _, _ = ppo_inputs(3, 20, 63, x.detach())
    idx, top, _ = teacher_inputs(3, 20, 4, 63)
    C.ppo_loss_grad(x.detach(), a, old, adv)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        with pytest.raises(RuntimeError, match="captured"):
            C.ppo_loss(x, a, old, adv)
        with pytest.raises(RuntimeError, match="captured"):
            C.distill_loss(x, idx, top)
        r, grad = C.ppo_loss_grad(x.detach(), a, old, adv)
    g.replay()
    want, wgrad = C.ppo_loss_grad(x.detach(), a, old, adv)
    assert torch.equal(grad, wgrad) and torch.equal(r.loss, want.loss)


@pytest.mark.parametrize("v", [11, 300, 2000, 60000])
def test_ppo_impossible_before(C, v):
    """An action that the old policy ruled out, or nearly: the ratio is infinite, the clipped side finite."""
    x = rows(4, v, torch.float32, 81)
    a, old, adv, w, _ = ppo_inputs(4, v, 81, x)
    adv = adv.abs() + 0.5
    old[1], old[2] = -INF, -1e30
    want = P.ppo(x, a, old, adv, w, low=0.2, high=0.3)
    rest = P.ppo(x[::3], a[::3], old[::3], adv[::3], w[::3], low=0.2, high=0.3)
    clipped = -(w[1:3] * adv[1:3]).double().sum() * 1.3
    for r, g in (C.ppo_loss_grad(x, a, old, adv, weights=w, clip_coef=0.2, clip_coef_high=0.3), (None, None)):
        if r is None:
            leaf = x.detach().requires_grad_()
            r = C.ppo_loss(leaf, a, old, adv, weights=w, clip_coef=0.2, clip_coef_high=0.3)
            g, = torch.autograd.grad(r.loss, leaf)
        near(r._asdict(), want, ("logprob", "entropy"))
        assert r.stats[3] == -INF and r.stats[4].isnan()  # sums of -inf, and of inf - inf, by their definition
        assert abs(float(r.loss.detach() - rest["loss"][0] - clipped)) <= float(rest["loss"][1]) + 2.0 ** -22 * float(clipped.abs())
        assert not g[1:3].any()
        near({"grad": g[::3]}, rest, ("grad",))
    r, g = C.ppo_loss_grad(x, a, old, -adv, weights=w)  # the other side is not clipped
    assert r.loss == INF and not g[::3].isnan().any()
    r = C.ppo_loss(x, a, old.clamp(max=0).abs() * INF, adv.nan_to_num(), weights=w)  # certain before: the ratio is 0
    assert r.loss == 0.0
    idx = torch.tensor([[0], [1]], device="cuda")  # a teacher's normaliser of nothing
    r = C.distill_loss(x[:2], idx, torch.zeros(2, 1, device="cuda"), teacher_lse=torch.tensor([0.0, -INF], device="cuda"))
    assert r.kl[0].isfinite() and r.kl[1] == INF


@pytest.mark.parametrize("v", [11, 300, 5000, 60000])
def test_gradient_between_the_rows(C, v):
    """Logits and gradient as columns of one buffer, that share no element."""
    a, old, adv, w, _ = ppo_inputs(5, v, 95, torch.zeros(5, v, device="cuda"))
    idx, top, _ = teacher_inputs(5, v, 4, 95)
    for dtype in DTYPES:
        for gap, first in ((0, False), (3, True)):
            wide = torch.full((5, 2 * v + 2 * gap), 5.0, dtype=dtype, device="cuda")
            left, right = wide[:, :v], wide[:, v + gap:2 * v + gap]
            x, out = (right, left) if first else (left, right)
            x.copy_(rows(5, v, dtype, 96))
            y = x.clone()
            r, g = C.ppo_loss_grad(x, a, old, adv, weights=w, out=out)
            assert g is out and torch.equal(x, y) and (wide[:, v:v + gap] == 5).all() and (wide[:, 2 * v + gap:] == 5).all()
            near(r._asdict() | {"grad": out}, P.ppo(y, a, old, adv, w), ("loss", "logprob", "entropy", "stats", "grad"))
            r, g = C.distill_loss_grad(x, idx, top, weights=w, out=out)
            assert torch.equal(x, y)
            near(r._asdict() | {"grad": out}, P.distill(y, idx, top, w), ("loss", "kl", "grad"))
    from ppo_radiotherapy_amd._lib import RtError

    wide = torch.randn(5, 2 * v, device="cuda")
    for at in (1, v - 1):
        with pytest.raises(RtError, match="overlaps"):
            C.ppo_loss_grad(wide[:, :v], a, old, adv, out=wide[:, at:at + v])
    flat = torch.randn(10 * v, device="cuda")
    for x, out in ((flat.as_strided((5, v), (2 * v, 1)), flat[5 * v:].view(5, v)), (flat[:5 * v].view(5, v), flat[4 * v:9 * v].view(5, v))):
        with pytest.raises(RtError, match="overlaps"):
            C.ppo_loss_grad(x, a, old, adv, out=out)


@pytest.mark.parametrize("v,n,n_loss", [(33, 2 ** 26 + 5, 2 ** 28 + 3), (577, 2 ** 24 + 3, 2 ** 26 + 5), (1025, 2 ** 24 + 3, 2 ** 26 + 5)])
def test_more_rows_than_one_launch_dimension_has(C, v, n, n_loss):
    """2^32 threads and more; one row of logits for all (stride 0), so that every row's result is known."""
    row = rows(1, v, torch.bfloat16, 71)
    x = row.expand(n, v)
    u = torch.zeros(n, device="cuda")
    few = torch.tensor([0.1, 0.5, 0.93], device="cuda")
    u[-3:] = few
    got, want = C.sample(x, u, top_p=0.9), C.sample(row.expand(3, v), few, top_p=0.9)
    zero = C.sample(row, u[:1], top_p=0.9)
    for p, q, z in zip(got, want, zero):
        assert torch.equal(p[-3:], q) and bool((p[:-3] == z).all())
    del got, u
    n = n_loss
    x = row.expand(n, v)
    a = torch.full((n,), -1, device="cuda")
    a[-2:] = torch.tensor([0, v - 1], device="cuda")
    f = torch.zeros(n, device="cuda")
    f[-2:] = torch.tensor([1.0, -2.0], device="cuda")
    r = C.ppo_loss(x, a, f, f, weights=torch.ones(1, device="cuda").expand(n))
    s = C.ppo_loss(x[-2:], a[-2:], f[-2:], f[-2:], weights=torch.ones(2, device="cuda"))
    assert torch.equal(r.logprob[-2:], s.logprob) and not r.logprob[:-2].any()
    assert torch.equal(r.loss, s.loss) and torch.equal(r.stats, s.stats)


def test_refusals(C):
    x = torch.randn(4, 10, device="cuda")
    v = torch.zeros(4, device="cuda")
    i = torch.zeros(4, dtype=torch.int64, device="cuda")
    bad = [
        (lambda: C.sample(x.double(), v), TypeError), (lambda: C.sample(x.cpu(), v), ValueError),
        (lambda: C.sample(x, v.cpu()), ValueError), (lambda: C.sample(x, v[:3]), ValueError),
        (lambda: C.sample(x, None), TypeError), (lambda: C.sample(x.t(), torch.zeros(10, device="cuda")), ValueError),
        (lambda: C.sample(x, v, temperature=-1.0), ValueError), (lambda: C.sample(x, v, temperature=NAN), ValueError),
        (lambda: C.sample(x, v, top_k=-1), ValueError), (lambda: C.sample(x, v, top_k=1.5), ValueError),
        (lambda: C.sample(x, v, top_p=NAN), ValueError), (lambda: C.sample(x, v, min_p=-0.1), ValueError),
        (lambda: C.sample(x, v, top_k=v), TypeError), (lambda: C.sample(x[:, :0], v), ValueError),
        (lambda: C.sample(torch.randn(4, 3, 10, device="cuda")[:, :2], torch.zeros(4, 2, device="cuda")), ValueError),
        (lambda: C.ppo_loss(x, i, v, v, temperature=0.0), ValueError), (lambda: C.ppo_loss(x, i, v, v, clip_coef=-1), ValueError),
        (lambda: C.ppo_loss(x, i, v, v, ent_coef=INF), ValueError), (lambda: C.ppo_loss(x, i, v, v, kl_coef=0.1), ValueError),
        (lambda: C.ppo_loss(x, v, v, v), TypeError), (lambda: C.ppo_loss(x, i, v, None), TypeError),
        (lambda: C.ppo_loss_grad(x, i, v, v, out=x.half()), ValueError),
        (lambda: C.ppo_loss_grad(x, i, v, v, out=x[:1].expand(4, 10)), ValueError),
        (lambda: C.distill_loss(x, i, v), ValueError),
        (lambda: C.distill_loss(x, i[:, None], v[:, None], temperature=INF), ValueError),
        (lambda: C.distill_loss(x, i[:, None].expand(4, 1025), v[:, None].expand(4, 1025)), ValueError),
        (lambda: C.distill_loss(x, i[:, None][:, :0], v[:, None][:, :0]), ValueError),
        (lambda: C.distill_loss(x, i[:, None], v[:, None], teacher_lse=i), TypeError),
    ]
    for k, (call, kind) in enumerate(bad):
        with pytest.raises(kind):
            call()
            pytest.fail(f"call {k} was not refused")
    import _rtpkg  # noqa: F401
    from ppo_radiotherapy_amd._lib import RtError

    wide = torch.randn(4, 20, device="cuda")
    with pytest.raises(RtError, match="overlaps"):
        C.ppo_loss_grad(wide[:, :10], i, v, v, out=wide[:, 5:15])


def test_documented_use(C):
    """README's and the module's own lines: of an unmoved policy the ratio is 1 throughout."""
    import os
    import re

    with open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "README.md")) as f:
        readme = re.search(r"```python\nfrom ppo_radiotherapy_amd import categorical\n(.*?)```", f.read(), re.S).group(1)
    module = "\n".join(re.findall(r"^    (\S.*)$", C.__doc__, re.M))
    for text in (readme, module):
        logits = rows(64, 50, torch.float32, 91).requires_grad_()
        lines = {"categorical": C, "logits": logits, "u": torch.rand(64, generator=gen(92), device="cuda"), "adv": torch.ones(64, device="cuda")}
        lines |= {k: getattr(C, k) for k in ("sample", "ppo_loss", "ppo_loss_grad", "distill_loss")}
        lines["top_logits"], lines["idx"] = lines["teacher_logits"], lines["teacher_idx"] = rows(64, 50, torch.float32, 93).topk(5)
        seen = []
        for line in text.splitlines():
            exec(line, lines)
            if "ppo_loss" in line:
                seen.append(lines["out"].stats)
        assert len(seen) >= 2
        for s in seen:
            assert s[5] == 0 and abs(float(s[3])) <= 2.0 ** -19 and abs(float(s[4])) <= 2.0 ** -30


def test_forward_mode_is_refused(C):
    """A tangent of the logits would be lost: nothing carries it on."""
    from torch.autograd import forward_ad

    x = torch.randn(3, 20, device="cuda")
    a, old, adv, _, _ = ppo_inputs(3, 20, 65, x)
    idx, top, _ = teacher_inputs(3, 20, 4, 65)
    want = C.ppo_loss(x, a, old, adv).loss
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for call in (lambda y: C.ppo_loss(y, a, old, adv), lambda y: C.distill_loss(y, idx, top)):
            for y in (dual, dual.bfloat16()):
                with pytest.raises(RuntimeError, match="forward"):
                    call(y)
        assert torch.equal(C.ppo_loss(x, a, old, adv).loss, want)  # no tangent, nothing lost


def test_what_the_backward_pass_does_not_read_may_change(C):
    """Weights and normalisers are in the row state: their buffers may be filled anew before the backward pass."""
    for v in (20, 3000):
        x = torch.randn(3, v, device="cuda", requires_grad=True)
        a, old, adv, w, ref = ppo_inputs(3, v, 66, x.detach())
        idx, top, _ = teacher_inputs(3, v, 4, 66)
        lse = torch.logsumexp(top, 1) + 0.1
        for loss, inputs in ((lambda: C.ppo_loss(x, a, old, adv, weights=w, ref_logprobs=ref, kl_coef=0.1).loss, (w, old, adv, ref)),
                             (lambda: C.distill_loss(x, idx, top, weights=w, teacher_lse=lse).loss, (w, lse))):
            want, = torch.autograd.grad(loss(), x)
            later, kept = loss(), [t.clone() for t in inputs]
            for t in inputs:
                t.fill_(5.0)
            got, = torch.autograd.grad(later, x)
            assert torch.equal(got, want)
            for t, k in zip(inputs, kept):
                t.copy_(k)
        later = C.distill_loss(x, idx, top, weights=w).loss
        top.add_(1.0)  # what it does read is noticed
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            later.backward()


def test_policy_iteration_together(C):
    """The operators as one iteration uses them: sample a rollout, GAE, a PPO update of a linear policy through
    autograd, then its distillation into another; each step against the definitions in 64 bits."""
    import _rtpkg  # noqa: F401
    from ppo_radiotherapy_amd import _lib

    L = _lib.load()
    T, N, D, V = 8, 32, 12, 44
    g = gen(77)
    W = (0.3 * torch.randn(D, V, generator=g, device="cuda")).requires_grad_()
    obs = torch.randn(T, N, D, generator=g, device="cuda")
    u = torch.rand(T, N, generator=g, device="cuda")
    with torch.no_grad():
        logits = obs.reshape(T * N, D).mm(W).reshape(T, N, V)
        s = C.sample(logits, u, temperature=1.1)
    reward = (s.action % 5 == 0).float()
    values, zero = torch.zeros(T, N, device="cuda"), torch.zeros(T, N, device="cuda")
    last = torch.zeros(N, device="cuda")
    adv, ret = torch.empty_like(values), torch.empty_like(values)
    _lib.check(L.rt_gae(T, N, reward.data_ptr(), values.data_ptr(), zero.data_ptr(), last.data_ptr(), last.data_ptr(),
                        0.99, 0.95, adv.data_ptr(), ret.data_ptr(), _lib.stream_handle()), "rt_gae")
    x = obs.reshape(T * N, D).mm(W)
    out = C.ppo_loss(x, s.action.reshape(-1), s.logprob.reshape(-1), adv.reshape(-1), temperature=1.1, ent_coef=0.01)
    # the policy has not moved: its log-probabilities are the rollout's, the ratio is 1
    assert float((out.logprob - s.logprob.reshape(-1)).abs().max()) <= 2.0 ** -19
    assert out.stats[5] == 0 and abs(float(out.stats[4])) <= 2.0 ** -30
    out.loss.backward()
    want = P.ppo(x.detach(), s.action.reshape(-1), s.logprob.reshape(-1), adv.reshape(-1), T=1.1, ent=0.01)
    gW = obs.reshape(T * N, D).double().t() @ want["grad"][0]
    room = obs.reshape(T * N, D).double().abs().t() @ (want["grad"][1] + want["grad"][0].abs() * 2.0 ** -20)
    assert ((W.grad.double() - gW).abs() <= room).all()
    with torch.no_grad():
        W -= 0.5 * W.grad
        x = obs.reshape(T * N, D).mm(W)
    top, idx = x.topk(6, dim=1)
    student = torch.zeros(T * N, V, device="cuda")
    r, grad = C.distill_loss_grad(student, idx, top, temperature=1.0)
    near(r._asdict() | {"grad": grad}, P.distill(student, idx, top), ("loss", "kl", "grad"))
