"""Operators on rows of vocabulary logits -- the k largest logits, token log-probability, distillation, policy and
preference losses -- through the package's functions against plain 64-bit restatements (oracle/token_ops_oracle.py).

Tolerances.  A term exp(c (x - m)) is computed in fp32: the rounded difference, the rounded c and the rounded product
each move the exponent by at most (D / tau) 2^-24 (D: the row's largest |x - m|), the exponential adds 2^-23, and it counts as 0
below 2^-126.  A sum of V such terms, in 64 threads at least, adds at most (V / 64 + 12) 2^-24 relative.  So a row's sum
and every probability are within  delta = (3 D / tau + 4 + V / 64 + 12) 2^-24  relative (`_delta`).  Log-probabilities and entropies are
within delta (times D / tau + 1 for the entropy, whose terms are weighted with log p) plus half a step of their own
rounding; a gradient sum_i a_i p_j b_i is within 4 delta sum |a_i b_i| plus half a step of its type, 2^-25 absolute
for fp16's subnormals."""
import math

import pytest
import torch

from oracle import token_ops_oracle as O

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
SIZES = [  # (T, B, V)
    (1, 1, 1), (1, 1, 2), (3, 2, 7), (1, 5, 64), (4, 3, 65), (2, 2, 513), (5, 4, 1000), (3, 3, 2049), (3, 2, 4099), (2, 3, 9001),
    (2, 2, 16387), (2, 2, 30522), (1, 2, 40001), (1, 2, 66001), (1, 2, 140003),
]


def _fn():
    from gtg_vae_amd import functional as Fn

    return Fn


def _logits(T, B, V, dtype, seed, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    x = spread * torch.randn((T, B, V), generator=g)
    x[..., :: max(1, V // 5)] += 4.0
    y = torch.randint(1, max(2, V), (T, B), generator=g).clamp_(max=V - 1)
    return x.to(dtype), y, g


def _delta(x, tau=1.0):
    z = x.double()
    z = z[torch.isfinite(z) & (z > -1e30)]
    D = float(z.max() - z.min()) if z.numel() else 0.0
    return (3 * D / tau + 16 + x.shape[-1] / 64) * 2.0 ** -24, D / tau


def _half(dtype):
    return torch.finfo(dtype).eps / 2


def _tiny(dtype):
    return 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -126


def _check_grad(got, want, scale, delta, what=""):
    got64 = got.double().cpu()
    allowed = _half(got.dtype) * want.abs() * 1.01 + 4 * delta * scale + _tiny(got.dtype)
    worst = ((got64 - want).abs() - allowed).max().item() if want.numel() else 0.0
    assert got.shape == want.shape and worst <= 0, f"{what}: off by {worst} more than allowed"


def _check_rows(got, want, tol, what=""):
    got, want = got.double().cpu(), want.double()
    assert got.shape == want.shape
    off = (got - want).abs() - (tol + want.abs() * 2.0 ** -23)
    assert not want.numel() or off.max().item() <= 0, f"{what}: {off.max().item()}"


# ---------------------------------------------------------------------------
# top_logits
# ---------------------------------------------------------------------------
def _nan_as(t, number):
    return torch.where(torch.isnan(t), number, t.double())


def _check_top(x, k, tau=1.0):
    v, i, tail = _fn().top_logits(x.cuda() if not x.is_cuda else x, k, tau)
    xc = x.cpu()
    wv, wi, wt = O.top_logits(xc, k, tau)
    assert v.dtype == x.dtype and i.dtype == torch.int32 and tail.dtype == torch.float32
    assert torch.equal(i.cpu(), wi)
    assert torch.equal(_nan_as(v.cpu(), 123.0), _nan_as(wv, 123.0))
    fin = torch.isfinite(wt)
    assert torch.equal(_nan_as(tail.cpu(), 7.0)[~fin], _nan_as(wt, 7.0)[~fin])
    delta, _ = _delta(xc.nan_to_num(nan=0.0), tau)
    _check_rows(tail.cpu()[fin], wt[fin], delta, "tail")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,B,V", SIZES)
def test_top_logits_matches_a_stable_sort(T, B, V, dtype):
    x, _, _ = _logits(T, B, V, dtype, seed=V)
    for k in sorted({1, min(V, 3), min(V, 64), min(V, 256)}):
        _check_top(x, k, 1.0 if k % 2 else 1.7)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [300, 5000, 30522])
def test_top_logits_ties_zeros_masks_and_nan(V, dtype):
    g = torch.Generator().manual_seed(V)
    rows = [
        torch.zeros(V),                                                     # all equal
        -torch.zeros(V),
        torch.where(torch.rand(V, generator=g) < 0.5, 0.0, -0.0),           # both zeros are one value
        torch.randint(0, 3, (V,), generator=g).float(),                     # few distinct values
        torch.full((V,), -math.inf),
        torch.full((V,), torch.finfo(dtype).min),
        torch.arange(V).float() / V, -torch.arange(V).float() / V,          # sorted either way
    ]
    r = torch.randn(V, generator=g)
    few = torch.full((V,), -math.inf)
    few[V // 3: V // 3 + 40] = r[:40]                                       # fewer finite ones than k
    inf = r.clone()
    inf[[5, V - 1, 77]] = math.inf
    nan = r.clone()
    nan[[9, V - 2]] = math.nan
    nan[3] = -math.nan
    many_inf = r.clone()
    many_inf[: V - 20] = math.inf
    many_nan = r.clone()
    many_nan[20:] = math.nan
    peak = torch.full((V,), -200.0)
    peak[V // 2] = 200.0                                                    # a tail 400 below
    x = torch.stack(rows + [few, inf, nan, many_inf, many_nan, peak]).to(dtype)
    for k in (1, 17, 64, 256):
        _check_top(x, k)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [200, 256, 257, 300, 511, 512, 1024, 2048, 4096, 8192])
def test_top_logits_of_many_out_of_few(V, dtype):
    """A k near the vocabulary's size, or beyond the number of parts whose maxima bound it, where the maxima are alike and the
    rest far below; and rows whose largest lie next to each other."""
    g = torch.Generator().manual_seed(V)
    low = torch.rand(V, generator=g) - 40
    low[::4] = 1 + torch.rand((V + 3) // 4, generator=g)
    run = torch.randn(V, generator=g)
    run[V // 3: V // 3 + 150] += 20
    x = torch.stack([low, low.flip(0), run, torch.randn(V, generator=g).sort()[0]]).to(dtype)
    for k in (min(V, 256), 199, 129, 128):
        _check_top(x, k)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [300, 1500, 9001, 30522, 140003])
def test_top_logits_of_masked_vocabularies(V, dtype):
    """Rows of which a mask leaves few classes: fewer than k, about as many, all in one place, or none."""
    g = torch.Generator().manual_seed(V)
    rows = []
    for mask in (-math.inf, torch.finfo(dtype).min, -1e4, 0.0):
        for keep in (torch.randperm(V, generator=g)[:10], torch.randperm(V, generator=g)[:100], torch.arange(V - 150, V), torch.arange(70, 90),
                     torch.arange(1)):
            r = torch.full((V,), mask)
            r[keep] = torch.randn(keep.numel(), generator=g).abs()
            rows.append(r)
        nan = rows[-1].clone()
        nan[V // 2] = math.nan
        rows.append(nan)
        both = rows[-5].clone()                  # two kinds of masked places
        both[: V // 2] = torch.where(both[: V // 2] == mask, -2e4, both[: V // 2])
        rows.append(both)
    x = torch.stack(rows).to(dtype)
    for k in (1, 20, 64, 256):
        _check_top(x, k)


def test_top_logits_takes_strides_and_other_shapes():
    Fn = _fn()
    x, _, _ = _logits(6, 5, 1003, torch.bfloat16, seed=1)
    wide = torch.empty((6, 5, 1100), dtype=torch.bfloat16, device="cuda").fill_(99.0)
    wide[..., 3:1006] = x.cuda()
    for view in (wide[..., 3:1006], x.cuda().transpose(0, 1), x.cuda()[1:4], x.cuda()[0], x.cuda()[0, 0],
                 x.cuda().transpose(1, 2).contiguous().transpose(1, 2), x.cuda()[:1].expand(4, 5, 1003)):
        v, i, t = Fn.top_logits(view, 20)
        wv, wi, wt = O.top_logits(view.cpu(), 20)
        assert torch.equal(i.cpu(), wi) and torch.equal(v.cpu(), wv) and torch.allclose(t.cpu().double(), wt, atol=1e-5)
    v, i, t = Fn.top_logits(x.cuda()[:0], 4)
    assert v.shape == (0, 5, 4) and i.shape == (0, 5, 4) and t.shape == (0, 5)


# ---------------------------------------------------------------------------
# token_logprob
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,B,V", SIZES)
def test_token_logprob_and_its_gradient(T, B, V, dtype):
    tau = 1.0 if V % 2 else 0.7
    x, y, g = _logits(T, B, V, dtype, seed=7 + V)
    if T * B > 3:
        y[-1, 0] = 0
    gl, gh = torch.randn((T, B), generator=g), torch.randn((T, B), generator=g)
    xg = x.cuda().requires_grad_(True)
    logp, ent = _fn().token_logprob(xg, y.cuda(), 0 if V > 1 else -1, temperature=tau)
    pad = 0 if V > 1 else -1
    x64 = x.double().requires_grad_(True)
    wl, we = O.token_logprob(x64, y, pad, tau)
    delta, D = _delta(x, tau)
    _check_rows(logp.detach(), wl.detach(), delta, "logp")
    _check_rows(ent.detach(), we.detach(), delta * (D + 2), "entropy")
    (want,) = torch.autograd.grad((wl * gl.double()).sum() + (we * gh.double()).sum(), x64)
    (got,) = torch.autograd.grad((logp, ent), (xg,), (gl.cuda(), gh.cuda()))
    assert got.dtype == dtype
    scale = ((gl.abs() + gh.abs() * (D + 12)) / tau)[..., None]
    _check_grad(got, want, scale, delta, "dlogits")
    # one output alone
    logp, ent = _fn().token_logprob(xg, y.cuda(), pad, temperature=tau)
    (got,) = torch.autograd.grad(ent.sum(), (xg,))
    x64 = x.double().requires_grad_(True)
    (want,) = torch.autograd.grad(O.token_logprob(x64, y, pad, tau)[1].sum(), x64)
    _check_grad(got, want, torch.full((T, B, 1), (D + 12) / tau), delta, "entropy alone")


@pytest.mark.parametrize("dtype", DTYPES)
def test_masked_logits_and_rows_that_do_not_count(dtype):
    T, B, V = 4, 6, 1201
    x, y, _ = _logits(T, B, V, dtype, seed=3)
    low = torch.finfo(dtype).min
    x[0, 0, 100:] = -math.inf
    x[0, 1, 100:] = low
    y[0, 0], y[0, 1] = 50, 60
    x[1, 0] = low                      # nothing but the lowest value: uniform
    x[1, 1] = math.nan                 # a row that does not count may hold anything
    y[1, 1] = 0
    x[1, 2] = math.inf
    y[1, 2] = 0
    y[2, 3] = 700
    x[2, 3, 700] = -math.inf           # the target itself is masked
    xg = x.cuda().requires_grad_(True)
    logp, ent = _fn().token_logprob(xg, y.cuda(), 0)
    x64 = torch.where((y == 0)[..., None], 0.0, x.double()).requires_grad_(True)
    wl, we = O.token_logprob(x64, y, 0)
    fin = torch.isfinite(wl)
    assert torch.equal(logp.detach().cpu()[~fin].double(), wl.detach()[~fin]) and (~fin).sum() == 1
    _check_rows(logp.detach().cpu()[fin], wl.detach()[fin], 1e-5)
    _check_rows(ent.detach(), we.detach(), 1e-4)
    (got,) = torch.autograd.grad(logp[logp > -1e30].sum(), (xg,))
    assert torch.isfinite(got).all() and (got[1, 1] == 0).all() and (got[1, 2] == 0).all()
    p = torch.softmax(x64.detach(), -1)
    onehot = torch.zeros_like(p).scatter_(-1, y[..., None], 1.0)
    want = torch.where(((y != 0) & fin)[..., None], onehot - p, 0.0)
    _check_grad(got, want, torch.ones(T, B, 1), _delta(x)[0])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [40, 1201, 9001, 140003])
def test_masked_logits_under_large_entropy_gradients(V, dtype):
    """Masked places, -inf or the type's lowest value, take no gradient however large what comes from above: a temperature
    below 1, the scale of a gradient scaler, a sum over rows."""
    T, B, tau, up = 2, 3, 0.5, 512.0
    x, y, _ = _logits(T, B, V, dtype, seed=V, spread=4.0)
    x[0, :, V // 3: V // 2] = -math.inf
    x[1, :, V // 3: V // 2] = torch.finfo(dtype).min
    x[1, 2, 1:] = -math.inf                # one class left
    y = y % (V // 3)
    delta, D = _delta(x, tau)
    logp = torch.log_softmax(x.double() / tau, -1)
    p = logp.exp()
    logp = torch.where(p > 0, logp, 0.0)
    want = -up / tau * p * (logp - (p * logp).sum(-1, keepdim=True))       # of up times the entropy
    scale = torch.full((T, B, 1), up * (D + 12) / tau)
    xg, yc, none = x.cuda().requires_grad_(True), y.cuda(), torch.zeros(T, B, device="cuda")
    (got,) = torch.autograd.grad(up * _fn().token_logprob(xg, yc, -1, tau)[1].sum(), (xg,))
    _check_grad(got, want, scale, delta, "entropy")
    for eager in (True, False):
        loss = _fn().policy_loss(xg, yc, -1, none, none, entropy_coef=0.25, temperature=tau, reduction="sum", eager_grad=eager)[0]
        (got,) = torch.autograd.grad(-4 * up * loss, (xg,))
        _check_grad(got, want, scale, delta, "policy")


@pytest.mark.parametrize("dtype", DTYPES)
def test_preference_with_masked_logits(dtype):
    T, P, V = 4, 2, 700
    x, y, g = _logits(T, 2 * P, V, dtype, seed=21)
    x[0, :, 300:] = -math.inf
    x[1, :, 300:] = torch.finfo(dtype).min
    y = y % 300
    seq = O.token_logprob(x.double(), y, 0)[0].sum(0)
    _check_prefer(x, y, (seq + torch.randn((2 * P,), generator=g)).float())


def test_rows_of_minus_infinity_bad_targets_and_nan_are_loud():
    x = torch.randn(5, 300).cuda()
    x[0] = -math.inf
    x[1, 7] = math.nan
    x[2, 7] = math.inf
    y = torch.tensor([3, 3, 3, 300, -2]).cuda()
    xg = x.clone().requires_grad_(True)
    logp, ent = _fn().token_logprob(xg, y, 0)
    assert torch.isnan(logp).all() and torch.isnan(ent[:3]).all()
    (got,) = torch.autograd.grad(logp.sum(), (xg,))
    assert torch.isnan(got).any(1).all()


def test_everything_is_pad_and_nothing_at_all():
    Fn = _fn()
    x = torch.randn(3, 4, 50, device="cuda", requires_grad=True)
    y = torch.zeros(3, 4, dtype=torch.long, device="cuda")
    f = torch.zeros(3, 4, device="cuda")
    v, i, t = Fn.top_logits(x, 5)
    for red, want in (("mean", ()), ("sum", ()), ("none", (3, 4))):
        for loss in (Fn.distill_loss(x, v, i, y, 0, t, reduction=red), Fn.policy_loss(x, y, 0, f, f, reduction=red)[0]):
            assert loss.shape == want and (loss == 0).all()
            (g,) = torch.autograd.grad(loss.sum(), (x,))
            assert (g == 0).all()
    loss, seq = Fn.preference_loss(x, y, 0, torch.zeros(4, device="cuda"))
    assert abs(loss.item() - math.log(2)) < 1e-6 and (seq == 0).all()
    (g,) = torch.autograd.grad(loss, (x,))
    assert (g == 0).all()
    for T, B in ((0, 4), (3, 0)):
        x = torch.randn(T, B, 50, device="cuda", requires_grad=True)
        y, f = torch.ones(T, B, dtype=torch.long, device="cuda"), torch.zeros(T, B, device="cuda")
        v, i, t = Fn.top_logits(x, 5)
        outs = [Fn.distill_loss(x, v, i, y, 0, t), Fn.policy_loss(x, y, 0, f, f)[0], Fn.token_logprob(x, y, 0)[0].sum()]
        loss, seq = Fn.preference_loss(x, y, 0, torch.zeros(B, device="cuda"))
        assert seq.shape == (B,) and abs(loss.item() - (math.log(2) if B else 0.0)) < 1e-6
        for o in outs + [loss]:
            (g,) = torch.autograd.grad(o, (x,))
            assert g.shape == x.shape
        assert all(o.item() == 0 for o in outs)


# ---------------------------------------------------------------------------
# distillation
# ---------------------------------------------------------------------------
def _teacher(x, k, tau, g, dtype):
    t = (x.float() + 0.8 * torch.randn(x.shape, generator=g)).to(dtype)
    return O.top_logits(t, k, tau)


def _check_distill(x, y, v, i, t, tau, a, reduction="mean", upstream=None, eager=True):
    xg = x.cuda().requires_grad_(True)
    loss = _fn().distill_loss(xg, v.cuda(), i.cuda(), y.cuda(), 0, None if t is None else t.float().cuda(), tau, a, reduction, eager)
    x64 = x.double().requires_grad_(True)
    keep = O.keep_rows(y, 0)
    rows = O.distill_rows(x64, v, i, y, 0, None if t is None else t.float(), tau, a)
    want = O.reduce(rows, keep, reduction)
    delta, D = _delta(x, tau)
    row_tol = 4 * delta * (tau * tau + 1) * (D + 4)
    _check_rows(loss.detach(), want.detach(), row_tol * (int(keep.sum()) if reduction == "sum" else 1), "loss")
    up = torch.ones(()) if upstream is None else upstream
    (wg,) = torch.autograd.grad(want, x64, up.double().expand(want.shape))
    (got,) = torch.autograd.grad(loss, (xg,), up.float().cuda().expand(loss.shape))
    w = up.double().abs().expand(want.shape) if reduction == "none" else up.double().abs()
    if reduction == "mean":
        w = w / max(1, int(keep.sum()))
    # 1 + q_t / p_t p_j: both parts of a class outside the list are at most 1
    scale = torch.as_tensor(w * (2 * tau + 1)).expand(y.shape)[..., None]
    _check_grad(got, wg, scale, delta, "dlogits")
    return got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,B,V", SIZES)
def test_distill_loss_and_its_gradient(T, B, V, dtype):
    x, y, g = _logits(T, B, V, dtype, seed=11 + V)
    if V == 1:
        return
    if T * B > 3:
        y[-1, 0] = 0
    for k, tau, a, tail in ((1, 1.0, 0.0, True), (min(V, 17), 2.0, 0.5, True), (min(V, 64), 1.0, 0.3, False),
                            (min(V, 256), 3.0, 0.0, False)):
        v, i, t = _teacher(x, k, tau, g, dtype)
        if k == V:
            t = None
        _check_distill(x, y, v, i, t if tail else None, tau, a)


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("eager", [True, False])
def test_distill_reductions_and_upstream_gradients(reduction, eager):
    T, B, V = 4, 3, 777
    x, y, g = _logits(T, B, V, torch.float16, seed=5)
    y[2, 1] = 0
    v, i, t = _teacher(x, 9, 1.5, g, torch.float32)
    up = torch.randn((T, B), generator=g) if reduction == "none" else torch.tensor(0.37)
    _check_distill(x, y, v, i, t, 1.5, 0.25, reduction, up, eager)


@pytest.mark.parametrize("dtype", DTYPES)
def test_distill_lists_with_gaps_repeats_and_masks(dtype):
    T, B, V, k = 3, 4, 515, 12
    x, y, g = _logits(T, B, V, dtype, seed=6)
    v, i, t = _teacher(x, k, 1.0, g, dtype)
    i = i.clone()
    v = v.clone()
    i[0, 0, 5:] = -1                        # a shorter list
    i[0, 1, 3] = i[0, 1, 7]                 # a class twice
    i[0, 2, :] = i[0, 2, :1]                # one class, k times
    v[0, 3, 4:] = -math.inf                 # teacher masks
    y[1, 0] = int(i[1, 0, 2])               # the target is on the list
    y[1, 1] = 510
    i[1, 1] = torch.arange(k)               # and is not
    x[1, 2, 100:200] = -math.inf            # masked classes of the student, off the list
    i[1, 2] = torch.arange(k)
    i[2, 0] = -1                            # the teacher lists nothing, but has a tail: nothing to learn
    x[2, 1] = torch.finfo(dtype).min
    for tail in (None, t):
        for a in (0.0, 0.4, 1.0):
            if tail is None:
                _check_distill(x, y, v, i, None, 1.0, a)
            else:
                _check_distill(x, y, v, i, tail, 2.0, a)
    # no list and no tail: the cross-entropy alone is left
    none = torch.full_like(i, -1)
    xg = x.cuda().requires_grad_(True)
    loss = _fn().distill_loss(xg, v.cuda(), none.cuda(), y.cuda(), 0)
    (got,) = torch.autograd.grad(loss, (xg,))
    assert loss.item() == 0 and (got == 0).all()
    _check_distill(x, y, v, none, None, 1.0, 0.5)
    # int64 indices, other value types, an index past the vocabulary
    one = _fn().distill_loss(xg, v.cuda(), i.cuda(), y.cuda(), 0)
    assert torch.equal(one, _fn().distill_loss(xg, v.cuda(), i.long().cuda(), y.cuda(), 0))
    far = i.long().clone()
    far[0, 0, 0] = 2 ** 32 + 1
    assert torch.isnan(_fn().distill_loss(xg, v.cuda(), far.cuda(), y.cuda(), 0))


@pytest.mark.parametrize("dtype", DTYPES)
def test_distill_at_the_largest_vocabulary(dtype):
    V, k = 400000, 256
    x, y, g = _logits(1, 2, V, dtype, seed=8)
    v, i, t = _teacher(x, k, 2.0, g, dtype)
    i = i.clone()
    i[0, 0, 0], i[0, 1, 255] = V - 1, 0
    y[0, 0], y[0, 1] = V - 1, int(i[0, 1, 3])
    _check_distill(x, y, v, i, t, 2.0, 0.5)


def test_distill_student_far_below_the_teachers_tail():
    # nearly all of the student's mass on the list, the rest 100 below: p_t is e^-100 and still has its relative precision
    V, k = 400, 4
    x = torch.full((1, 1, V), -100.0)
    x[0, 0, :k] = torch.tensor([0.0, 1.0, 2.0, 3.0])
    x[0, 0, k:] += torch.linspace(0, 1, V - k)
    i = torch.arange(k, dtype=torch.int32).view(1, 1, k)
    v = torch.tensor([3.0, 2.0, 1.0, 0.0]).view(1, 1, k)
    _check_distill(x, torch.ones(1, 1, dtype=torch.long), v, i, torch.tensor([[-2.0]]), 1.0, 0.0)


# ---------------------------------------------------------------------------
# policy
# ---------------------------------------------------------------------------
def _policy_case(T, B, V, dtype, seed, tau):
    x, y, g = _logits(T, B, V, dtype, seed)
    if T * B > 3:
        y[-1, 0] = 0
    now, _ = O.token_logprob(x.double(), y, 0, tau)
    old = (now + 0.3 * torch.randn((T, B), generator=g)).float()
    ref = (now + 0.5 * torch.randn((T, B), generator=g)).float()
    return x, y, old, ref, torch.randn((B,), generator=g), g


def _check_policy(x, y, old, adv, ref, reduction="mean", upstream=None, eager=True, mask=None, pad=0, **kw):
    xg = x.cuda().requires_grad_(True)
    cu = lambda t: None if t is None else t.cuda()  # noqa: E731
    loss, logp, ent = _fn().policy_loss(xg, y.cuda(), pad, old.cuda(), adv.cuda(), cu(ref), mask=cu(mask), reduction=reduction,
                                        eager_grad=eager, **kw)
    x64 = x.double().requires_grad_(True)
    rows, wl, we = O.policy_rows(x64, y, pad, old, adv, ref, mask=mask, **kw)
    keep = O.keep_rows(y, pad, mask)
    want = O.reduce(rows, keep, reduction)
    tau = kw.get("temperature", 1.0)
    delta, D = _delta(x, tau)
    _check_rows(logp, wl.detach(), delta, "logp")
    _check_rows(ent, we.detach(), delta * (D + 2), "entropy")
    assert not logp.requires_grad and not ent.requires_grad
    # d loss / d logp and d loss / d H are bounded by what the case allows
    with torch.no_grad():
        slope = torch.exp((wl - old.double()).clamp(max=20)) * adv.double().abs().expand(y.shape)
        if ref is not None:
            slope = slope + kw.get("kl_coef", 0.0) * (1 + torch.exp(ref.double() - wl))
        slope = torch.where(keep, slope + abs(kw.get("entropy_coef", 0.0)) * (D + 12), 0.0)
    n = int(keep.sum()) if reduction == "mean" else 1
    _check_rows(loss.detach(), want.detach(), 2 * delta * (slope if reduction == "none" else slope.sum() / max(1, n)), "loss")
    up = torch.ones(()) if upstream is None else upstream
    (wg,) = torch.autograd.grad(want, x64, up.double().expand(want.shape))
    (got,) = torch.autograd.grad(loss, (xg,), up.float().cuda().expand(loss.shape))
    scale = (slope * up.double().abs() / max(1, n) / tau)[..., None]
    _check_grad(got, wg, scale, delta, "dlogits")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,B,V", [s for s in SIZES if s[2] > 1])
def test_policy_loss_and_its_gradient(T, B, V, dtype):
    for tau, kl, ent in ((1.0, 0.0, 0.0), (0.8, 0.05, 0.0), (1.3, 0.1, 0.02)):
        x, y, old, ref, adv, g = _policy_case(T, B, V, dtype, 13 + V, tau)
        _check_policy(x, y, old, adv, ref if kl else None, clip_low=0.2, clip_high=0.28, kl_coef=kl, entropy_coef=ent, temperature=tau)


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("eager", [True, False])
def test_policy_reductions_masks_and_upstream_gradients(reduction, eager):
    T, B, V = 6, 5, 901
    x, y, old, ref, adv, g = _policy_case(T, B, V, torch.bfloat16, 4, 1.0)
    mask = torch.rand((T, B), generator=g) < 0.6
    up = torch.randn((T, B), generator=g) if reduction == "none" else torch.tensor(-2.5)
    per_token = torch.randn((T, B), generator=g)
    for m in (mask, mask.int() * 7):
        _check_policy(x, y, old, per_token, ref, reduction, up, eager, m, kl_coef=0.04, entropy_coef=0.01)
    _check_policy(x, y, old, adv, ref, reduction, up, eager, None, pad=-100, kl_coef=0.04)


def test_policy_clipping_border_cases():
    T, B, V = 1, 8, 64
    x, y, _ = _logits(T, B, V, torch.float32, 8)
    now, _ = O.token_logprob(x.double(), y, 0)
    shift = torch.tensor([[0.0, 3.0, -3.0, 3.0, -3.0, 200.0, -200.0, 0.1]])
    adv = torch.tensor([[1.0, 1.0, 1.0, -1.0, -1.0, 1.0, 1.0, 0.0]])
    _check_policy(x, y, (now - shift).float(), adv, None)


# ---------------------------------------------------------------------------
# preference
# ---------------------------------------------------------------------------
def _check_prefer(x, y, ref, reduction="mean", upstream=None, mask=None, batch_first=False, beta=0.1, eps=0.0):
    xg = x.cuda().requires_grad_(True)
    m = None if mask is None else mask.cuda()
    loss, seq = _fn().preference_loss(xg, y.cuda(), 0, ref.cuda(), beta, eps, m, batch_first, reduction)
    x64 = x.double().requires_grad_(True)
    pairs, wseq = O.preference(x64, y, 0, ref, beta, eps, mask, batch_first)
    want = pairs if reduction == "none" else pairs.sum() if reduction == "sum" else pairs.mean()
    delta, _ = _delta(x)
    T, P = y.shape[1 if batch_first else 0], ref.numel() // 2
    n = {"mean": 1, "none": 1, "sum": P}[reduction]
    _check_rows(seq, wseq.detach(), delta * T, "seq")
    _check_rows(loss.detach(), want.detach(), 2 * delta * T * beta * n, "loss")
    up = torch.ones(()) if upstream is None else upstream
    (wg,) = torch.autograd.grad(want, x64, up.double().expand(want.shape))
    (got,) = torch.autograd.grad(loss, (xg,), up.float().cuda().expand(loss.shape))
    # a sequence's weight is at most beta, and moves with the margin by beta / 4 of it
    scale = up.double().abs().max() * beta * (1 + beta * T) / (P if reduction == "mean" else 1)
    _check_grad(got, wg, scale, delta, "dlogits")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,P,V", [(1, 1, 2), (5, 3, 65), (7, 2, 1000), (3, 1, 4099), (40, 4, 2051), (2, 1, 30522), (700, 1, 130)])
def test_preference_loss_and_its_gradient(T, P, V, dtype):
    x, y, g = _logits(T, 2 * P, V, dtype, seed=17 + V)
    if T > 3:
        y[T // 2:, 0] = 0
    seq = O.token_logprob(x.double(), y, 0)[0].sum(0)
    ref = (seq + 2.0 * torch.randn((2 * P,), generator=g)).float()
    _check_prefer(x, y, ref)
    _check_prefer(x, y, ref, beta=0.4, eps=0.1)


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("batch_first", [False, True])
def test_preference_reductions_masks_and_layouts(reduction, batch_first):
    T, P, V = 9, 3, 333
    x, y, g = _logits(T, 2 * P, V, torch.float32, seed=2)
    mask = torch.rand((T, 2 * P), generator=g) < 0.7
    mask[:, 4] = False                      # a sequence of which nothing counts
    if batch_first:
        x, y, mask = x.transpose(0, 1).contiguous(), y.t().contiguous(), mask.t().contiguous()
    seq = O.token_logprob(x.double(), y, 0, mask=mask)[0].sum(1 if batch_first else 0)
    ref = (seq + torch.randn((2 * P,), generator=g)).float()
    up = torch.randn((P,), generator=g) if reduction == "none" else torch.tensor(1.7)
    _check_prefer(x, y, ref, reduction, up, mask, batch_first, 0.2, 0.05)


def test_preference_many_pairs_and_far_margins():
    T, P, V = 2, 700, 33                    # more sequences than the joining block has threads
    x, y, g = _logits(T, 2 * P, V, torch.float32, seed=3)
    seq = O.token_logprob(x.double(), y, 0)[0].sum(0)
    ref = (seq + 2 * torch.randn((2 * P,), generator=g)).float()
    _check_prefer(x, y, ref)
    ref[0], ref[1] = ref[0] + 1e4, ref[1] - 1e4
    _check_prefer(x, y, ref, reduction="none", upstream=torch.ones(P), eps=0.1)
    loss, _ = _fn().preference_loss(x.cuda(), y.cuda(), 0, (ref - 1e30).cuda())
    assert torch.isfinite(loss)


# ---------------------------------------------------------------------------
# gradients against differences
# ---------------------------------------------------------------------------
def test_gradients_against_differences():
    """Directional derivatives by central differences: with h = 2^-5 the loss's third derivative leaves h^2 / 6 of its
    scale (1.6e-4), the losses' fp32 rounding 2^-24 |loss| / h."""
    Fn = _fn()
    T, B, V = 5, 4, 257
    x, y, old, ref, adv, g = _policy_case(T, B, V, torch.float32, 9, 1.0)
    v, i, t = _teacher(x, 8, 1.5, g, torch.float32)
    old = (O.token_logprob(x.double(), y, 0)[0] + 0.05).float()     # every ratio well inside the clip's borders
    xc, yc = x.cuda(), y.cuda()
    seq = O.token_logprob(x.double(), y, 0)[0].sum(0).float().cuda()
    losses = {
        "logprob": lambda z: Fn.token_logprob(z, yc, 0, 1.2)[0].sum() + Fn.token_logprob(z, yc, 0, 1.2)[1].sum(),
        "distill": lambda z: Fn.distill_loss(z, v.cuda(), i.cuda(), yc, 0, t.float().cuda(), 1.5, 0.3),
        "policy": lambda z: Fn.policy_loss(z, yc, 0, old.cuda(), adv.cuda(), ref.cuda(), 0.9, 0.9, 0.1, 0.05)[0],
        "prefer": lambda z: Fn.preference_loss(z, yc, 0, seq + 1.0)[0],
    }
    h = 2.0 ** -5
    d = torch.randn(x.shape, generator=g).cuda()
    for name, f in losses.items():
        z = xc.clone().requires_grad_(True)
        loss = f(z)
        (grad,) = torch.autograd.grad(loss, (z,))
        along = (grad.double() * d.double()).sum().item()
        with torch.no_grad():
            diff = (f(xc + h * d).double() - f(xc - h * d).double()).item() / (2 * h)
        size = grad.double().norm().item() * d.double().norm().item()
        assert abs(along - diff) <= 1e-3 * size + abs(loss.item()) * 2.0 ** -23 / h, (name, along, diff)


# ---------------------------------------------------------------------------
# streams, graphs, determinism, retained graphs, far offsets, alignment
# ---------------------------------------------------------------------------
def _all_losses(x, st):
    Fn = _fn()
    return [Fn.distill_loss(x, st["v"], st["i"], st["y"], 0, st["t"], 2.0, 0.5), Fn.policy_loss(x, st["y"], 0, st["old"], st["adv"],
            st["ref"], kl_coef=0.1, entropy_coef=0.01)[0], Fn.preference_loss(x, st["y"], 0, st["seq"])[0],
            Fn.token_logprob(x, st["y"], 0)[0].sum()]


def _all_state(T, B, V, dtype, seed):
    x, y, old, ref, adv, g = _policy_case(T, B, V, dtype, seed, 1.0)
    v, i, t = _teacher(x, 16, 2.0, g, dtype)
    st = dict(y=y, old=old, ref=ref, adv=adv, v=v, i=i, t=t.float(), seq=old.sum(0))
    return x.cuda(), {k: s.cuda() for k, s in st.items()}


@pytest.mark.parametrize("dtype", DTYPES)
def test_same_inputs_same_bits_also_on_another_stream(dtype):
    x, st = _all_state(6, 4, 5003, dtype, 1)
    st["i"][0, 0, 3] = st["i"][0, 0, 9]

    def once():
        z = x.clone().requires_grad_(True)
        return [t for loss in _all_losses(z, st) for t in (loss.detach(), torch.autograd.grad(loss, (z,))[0])] + list(_fn().top_logits(x, 30))

    first = once()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = once()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for a, b, c in zip(first, once(), other):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_retained_graph_second_backward_and_other_scale():
    x, st = _all_state(3, 4, 700, torch.float32, 2)
    z = x.clone().requires_grad_(True)
    for loss in _all_losses(z, st):
        (a,) = torch.autograd.grad(loss, (z,), torch.tensor(0.5, device="cuda"), retain_graph=True)
        keep = a.clone()
        (b,) = torch.autograd.grad(loss, (z,), retain_graph=True)
        (c,) = torch.autograd.grad(loss, (z,), torch.tensor(0.5, device="cuda"))
        assert torch.equal(a, keep) and torch.equal(a, c) and torch.allclose(2 * a, b, rtol=1e-6, atol=0)


def test_a_large_loss_scale_reaches_small_half_precision_gradients():
    """At an upstream gradient of 2^14 the gradient is rounded once, after the scale: what would be below fp16's
    smallest number at scale 1 is not lost."""
    T, B, V = 16, 64, 1000
    x, y, g = _logits(T, B, V, torch.float16, 1, spread=0.1)
    v, i, t = _teacher(x, 8, 1.0, g, torch.float16)
    up = torch.tensor(2.0 ** 14)
    for eager in (True, False):
        _check_distill(x[:4, :4], y[:4, :4], v[:4, :4], i[:4, :4], t[:4, :4], 1.0, 0.0, "mean", up, eager)


def test_captured_and_replayed_beside_eager_work():
    x, st = _all_state(5, 4, 2050, torch.bfloat16, 3)
    static = x.clone()

    def step():
        # a leaf of the capture's own: an eager graph of the same leaf may live on
        z = static.detach().requires_grad_(True)
        return [t for loss in _all_losses(z, st) for t in (loss.detach(), torch.autograd.grad(loss, (z,))[0])] + list(_fn().top_logits(static, 30))

    from gtg_vae_amd.streams import owned_stream

    s = owned_stream(torch.device("cuda", torch.cuda.current_device()), "capture")
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s, capture_error_mode="thread_local"):
            out = step()
        graphs.append((g, out))
    for k in range(3):
        static.copy_(x + 0.25 * k)
        static[k, 0, :50] = 3.0
        want = step()
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            for a, b in zip(out, want):
                assert torch.equal(a, b)


def test_offsets_past_32_bits():
    """Rows behind the 2^32-th byte and the 2^31-th element; all but a few rows are padding."""
    V, R = 131072, 16640
    x = torch.zeros((R, V), dtype=torch.bfloat16, device="cuda")
    y = torch.zeros(R, dtype=torch.long, device="cuda")
    g = torch.Generator().manual_seed(1)
    rows = [3, 16384, R - 1]
    some = torch.randn((len(rows), V), generator=g).to(torch.bfloat16)
    for r, s in zip(rows, some):
        x[r] = s.cuda()
        y[r] = 77
    x.requires_grad_(True)
    f = torch.zeros(R, device="cuda")
    for loss, formula in ((_fn().policy_loss(x, y, 0, f - 12.0, f + 1.0, reduction="sum", clip_high=1e9)[0],
                           lambda lp: -torch.exp(lp + 12.0).sum()), (_fn().token_logprob(x, y, 0)[0].sum(), lambda lp: lp.sum())):
        (got,) = torch.autograd.grad(loss, (x,))
        s64 = some.double().requires_grad_(True)
        l64 = formula(torch.log_softmax(s64, -1)[:, 77])
        assert abs(loss.item() - l64.item()) <= 1e-4 * abs(l64.item())
        (w,) = torch.autograd.grad(l64, s64)
        for n, r in enumerate(rows):
            _check_grad(got[r], w[n], w[n].abs().max() * 2, _delta(some)[0])
        assert (got[16383] == 0).all() and (got[4] == 0).all()
        del got
    _, i, _ = _fn().top_logits(x.detach(), 8)
    assert torch.equal(i[rows].cpu(), O.top_logits(some, 8)[1])


def test_more_rows_than_one_launch_takes():
    """2^21 rows go into one launch; the rows behind them into the next."""
    R, V = (1 << 21) + 5000, 3
    g = torch.Generator().manual_seed(2)
    x = torch.randn((R, V), generator=g)
    y = torch.randint(0, 3, (R,), generator=g)
    f = 0.1 * torch.randn((R,), generator=g)
    xg = x.cuda().requires_grad_(True)
    x64 = x.double().requires_grad_(True)
    loss, logp, ent = _fn().policy_loss(xg, y.cuda(), 0, f.cuda() - 1.0, f.cuda(), entropy_coef=0.1)
    rows, wl, we = O.policy_rows(x64, y, 0, f - 1.0, f, entropy_coef=0.1)
    want = O.reduce(rows, y != 0, "mean")
    delta, D = _delta(x)
    _check_rows(logp, wl.detach(), delta)
    _check_rows(ent, we.detach(), delta * (D + 2))
    assert abs(loss.item() - want.item()) < 1e-6
    (got,) = torch.autograd.grad(loss, (xg,))
    (w,) = torch.autograd.grad(want, x64)
    _check_grad(got, w, torch.full((R, 1), 2.0 / int((y != 0).sum())) * (D + 2), delta)
    logp, _ = _fn().token_logprob(xg, y.cuda(), 0)
    (got,) = torch.autograd.grad(logp.sum(), (xg,))
    p = torch.softmax(x.double(), -1)
    want = torch.where((y != 0)[:, None], torch.nn.functional.one_hot(y, 3) - p, 0.0)
    _check_grad(got, want, torch.ones(R, 1), delta)
    v, i, t = _fn().top_logits(xg, 2)
    assert torch.equal(i.cpu().long(), torch.topk(x, 2).indices)
    loss = _fn().distill_loss(xg, v, i, y.cuda(), 0, t, reduction="none")
    assert loss.abs().max().item() < 1e-5 and loss.shape == (R,)


@pytest.mark.parametrize("dtype", DTYPES)
def test_strided_logits_and_a_gradient_of_another_alignment(dtype):
    Fn = _fn()
    T, B, V = 3, 4, 517
    x, y, old, ref, adv, g = _policy_case(T, B, V, dtype, 6, 1.0)
    y[T - 1, 0] = 0
    yc, f = y.cuda(), old.cuda()
    wide = torch.full((T, B, V + 20), 50.0, dtype=dtype, device="cuda")
    wide[..., 3:3 + V] = x.cuda()
    views = {"contiguous": x.cuda(), "inside a wider tensor": wide[..., 3:3 + V],
             "batch-major": x.transpose(0, 1).contiguous().cuda().transpose(0, 1),
             "vocabulary-major": x.permute(2, 0, 1).contiguous().cuda().permute(1, 2, 0)}
    x64 = x.double().requires_grad_(True)
    rows, wl, _ = O.policy_rows(x64, y, 0, old, adv, entropy_coef=0.01)
    keep = O.keep_rows(y, 0)
    wants = [torch.autograd.grad(O.reduce(rows, keep, "mean"), x64, retain_graph=True)[0], torch.autograd.grad(wl.sum(), x64)[0]]
    delta, D = _delta(x)
    slope = (torch.exp(wl.detach() - old.double()) * adv.double().abs() + 0.01 * (D + 12)) / int(keep.sum())
    for name, view in views.items():
        z = view.detach().requires_grad_(True)
        got = [torch.autograd.grad(Fn.policy_loss(z, yc, 0, f, adv.cuda(), entropy_coef=0.01)[0], (z,))[0],
               torch.autograd.grad(Fn.token_logprob(z, yc, 0)[0].sum(), (z,))[0]]
        _check_grad(got[0], wants[0], slope[..., None], delta, name)
        _check_grad(got[1], wants[1], torch.ones(T, B, 1), delta, name)
        if name == "contiguous":
            want = got
    assert (wide[..., :3] == 50).all() and (wide[..., 3 + V:] == 50).all()
    # through the C ABI: a gradient whose rows are aligned unlike the logits' own
    from gtg_vae_amd import _lib
    from gtg_vae_amd._lib import check, stream_ptr

    xc = x.cuda()
    logp, ent = Fn.token_logprob(xc, yc, 0)
    stats = torch.empty((T * B, 4), device="cuda")
    L = _lib.lib()
    code = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}[dtype]
    check(L.gtg_token_logprob_fwd(xc.data_ptr(), code, T * B, V, V, yc.data_ptr(), 0, 1.0, logp.data_ptr(), ent.data_ptr(),
                                  stats.data_ptr(), stream_ptr()))
    out = torch.full((T * B, V + 6), 7.0, dtype=dtype, device="cuda")
    one = torch.ones(T * B, device="cuda")
    check(L.gtg_token_logprob_bwd(xc.data_ptr(), code, T * B, V, V, yc.data_ptr(), 0, 1.0, stats.data_ptr(), one.data_ptr(), None,
                                  out[:, 1:].data_ptr(), V + 6, stream_ptr()))
    assert torch.equal(out[:, 1:V + 1].reshape(T, B, V), want[1]) and (out[:, 0] == 7).all() and (out[:, V + 1:] == 7).all()


# ---------------------------------------------------------------------------
# refusals
# ---------------------------------------------------------------------------
def test_refusals():
    Fn = _fn()
    from gtg_vae_amd._lib import GtgError

    x = torch.randn(2, 4, 40, device="cuda", requires_grad=True)
    y, f = torch.ones(2, 4, dtype=torch.long, device="cuda"), torch.zeros(2, 4, device="cuda")
    v, i, t = Fn.top_logits(x, 6)
    r = torch.zeros(4, device="cuda")
    bad = [
        lambda: Fn.top_logits(x, 0), lambda: Fn.top_logits(x, 41), lambda: Fn.top_logits(x, 2.0), lambda: Fn.top_logits(x, 3, 0.0),
        lambda: Fn.top_logits(torch.randn(2, 300, device="cuda"), 257), lambda: Fn.top_logits(x.double(), 3),
        lambda: Fn.top_logits(x.cpu(), 3), lambda: Fn.top_logits(x, 3, math.nan),
        lambda: Fn.token_logprob(x, y[:1], 0), lambda: Fn.token_logprob(x, f, 0), lambda: Fn.token_logprob(x, y.cpu(), 0),
        lambda: Fn.token_logprob(x, y, 0, -1.0), lambda: Fn.token_logprob(x.int(), y, 0),
        lambda: Fn.distill_loss(x, v[:, :2], i, y, 0), lambda: Fn.distill_loss(x, v, i[..., :3], y, 0),
        lambda: Fn.distill_loss(x, v, i.float(), y, 0), lambda: Fn.distill_loss(x, v, i, y, 0, t[:1]),
        lambda: Fn.distill_loss(x, v, i, y, 0, t, 0.0), lambda: Fn.distill_loss(x, v, i, y, 0, t, 1.0, 1.5),
        lambda: Fn.distill_loss(x, v, i, y, 0, t, reduction="avg"), lambda: Fn.distill_loss(x, v.cpu(), i, y, 0),
        lambda: Fn.distill_loss(torch.randn(1, 1, 400001, device="cuda"), v[:1, :1], i[:1, :1], y[:1, :1], 0),
        lambda: Fn.policy_loss(x, y, 0, f[:1], f), lambda: Fn.policy_loss(x, y, 0, f, f[:, :3]),
        lambda: Fn.policy_loss(x, y, 0, f, f, kl_coef=0.1), lambda: Fn.policy_loss(x, y, 0, f, f, clip_low=-0.1),
        lambda: Fn.policy_loss(x, y, 0, f, f, mask=f[:1]), lambda: Fn.policy_loss(x, y, 0, f, f, entropy_coef=math.inf),
        lambda: Fn.policy_loss(x, y, 0, f, 1.0), lambda: Fn.policy_loss(x, y, 0, f, f, reduction="batch"),
        lambda: Fn.preference_loss(x[:, :3], y[:, :3], 0, r[:3]), lambda: Fn.preference_loss(x, y, 0, r[:2]),
        lambda: Fn.preference_loss(x, y, 0, r, label_smoothing=1.0), lambda: Fn.preference_loss(x, y, 0, r, beta=math.nan),
        lambda: Fn.preference_loss(x[0], y[0], 0, r),
    ]
    for n, call in enumerate(bad):
        with pytest.raises(GtgError):
            call()
            pytest.fail(f"call {n} was accepted")
    # second derivatives are refused, not wrong
    loss = Fn.token_logprob(x, y, 0)[0].sum()
    (g,) = torch.autograd.grad(loss, (x,), create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
