"""What the entry points on rows of logits refuse on the host, before anything is launched: no GPU needed."""
import ctypes
import math

import pytest

from gtg_vae_amd import _lib

P = ctypes.c_void_p(4096)          # never read: every call below is refused first
F32, F16, BF16 = 0, 1, 2
NONE, SUM, MEAN = 0, 1, 2


def refused(name, *args, part=None):
    L = _lib.lib()
    rc = getattr(L, name)(*args)
    assert rc < 0, f"{name}{args} was accepted"
    msg = L.gtg_last_error().decode()
    assert name in msg and (part is None or part in msg), msg


BAD_LOGITS = [
    ((P, 3, 4, 50, 50), "dtype"), ((P, -1, 4, 50, 50), "dtype"), ((P, F32, -1, 50, 50), "size"), ((P, F32, 4, 0, 50), "size"),
    ((P, F32, 4, 50, 49), "stride"), ((None, F32, 4, 50, 50), "logits"), ((ctypes.c_void_p(4098), F32, 4, 50, 50), "logits"),
    ((ctypes.c_void_p(4097), BF16, 4, 50, 50), "logits"), ((P, F32, 1 << 31, 50, 50), "size"),
]


@pytest.mark.parametrize("logits,part", BAD_LOGITS)
def test_bad_logits_are_refused_by_every_entry_point(logits, part):
    refused("gtg_top_logits", *logits, 3, 1.0, P, P, P, None, part=part)
    refused("gtg_token_logprob_fwd", *logits, P, 0, 1.0, P, P, P, None, part=part)
    refused("gtg_token_logprob_bwd", *logits, P, 0, 1.0, P, P, P, P, 50, None, part=part)
    refused("gtg_distill_loss_fwd", *logits, P, 0, P, F32, P, 3, P, 1.0, 0.0, MEAN, P, P, P, None, 50, None, part=part)
    refused("gtg_distill_loss_bwd", *logits, P, 0, P, F32, P, 3, P, 1.0, 0.0, P, None, P, 0, P, 50, None, part=part)
    hyper = (0.2, 0.2, 0.0, 0.0, 1.0)
    refused("gtg_policy_loss_fwd", *logits, P, 0, None, P, P, 4, None, *hyper, MEAN, P, P, P, P, P, None, 50, None, part=part)
    refused("gtg_policy_loss_bwd", *logits, P, 0, None, P, P, 4, None, *hyper, P, None, P, 0, P, 50, None, part=part)


OK = (P, F32, 4, 50, 50)
Q = ctypes.c_void_p(8192)


def test_top_logits_refusals():
    for k in (0, -1, 51, 257):
        refused("gtg_top_logits", *OK, k, 1.0, P, P, P, None, part="k must")
    for t in (0.0, -1.0, math.inf, math.nan):
        refused("gtg_top_logits", *OK, 3, t, P, P, P, None, part="temperature")
    for n in range(3):
        outs = [P, P, P]
        outs[n] = None
        refused("gtg_top_logits", *OK, 3, 1.0, *outs, None, part="null")


def test_token_logprob_refusals():
    refused("gtg_token_logprob_fwd", *OK, None, 0, 1.0, P, P, P, None, part="null")
    refused("gtg_token_logprob_fwd", *OK, P, 0, 0.0, P, P, P, None, part="temperature")
    refused("gtg_token_logprob_fwd", *OK, P, 0, 1.0, P, P, ctypes.c_void_p(4100), None, part="stats")
    refused("gtg_token_logprob_bwd", *OK, P, 0, 1.0, None, P, P, Q, 50, None, part="null")
    refused("gtg_token_logprob_bwd", *OK, P, 0, 1.0, P, P, P, P, 50, None, part="overlap")
    refused("gtg_token_logprob_bwd", *OK, P, 0, 1.0, P, P, P, Q, 49, None, part="stride")
    refused("gtg_token_logprob_bwd", *OK, P, 0, 1.0, P, P, P, None, 50, None, part="dlogits")


def test_distill_refusals():
    def fwd(values=P, vt=F32, indices=P, k=3, temp=1.0, ce=0.0, red=MEAN, norm=P, row=P, loss=P, dx=None, ldg=50, logits=OK, **kw):
        refused("gtg_distill_loss_fwd", *logits, P, 0, values, vt, indices, k, P, temp, ce, red, norm, row, loss, dx, ldg, None, **kw)

    fwd(values=None, part="null")
    fwd(vt=5, part="value_dtype")
    fwd(indices=None, part="null")
    for k in (0, 257):
        fwd(k=k, part="k must")
    for t in (0.0, math.nan, math.inf):
        fwd(temp=t, part="temperature")
    for c in (-0.1, 1.1, math.nan):
        fwd(ce=c, part="ce_weight")
    for r in (-1, 3):
        fwd(red=r, part="reduction")
    fwd(norm=None, part="null")
    fwd(row=None, part="null")
    fwd(loss=None, red=SUM, part="null")
    fwd(dx=P, part="overlap")
    fwd(dx=Q, ldg=10, part="stride")
    fwd(logits=(P, BF16, 4, 400001, 400001), part="400 000")
    refused("gtg_distill_loss_bwd", *OK, P, 0, P, F32, P, 3, P, 1.0, 0.0, P, None, None, 1, Q, 50, None, part="unless_unit")


def test_policy_refusals():
    def fwd(old=P, adv=P, adv_rows=4, ref=None, lo=0.2, hi=0.2, kl=0.0, ent=0.0, temp=1.0, red=MEAN, norm=P, row=P, loss=P, **kw):
        refused("gtg_policy_loss_fwd", *OK, P, 0, None, old, adv, adv_rows, ref, lo, hi, kl, ent, temp, red, norm, row, loss, P, P, None,
                50, None, **kw)

    fwd(old=None, part="null")
    fwd(adv=None, part="null")
    fwd(adv_rows=0, part="adv_rows")
    fwd(kl=0.1, part="ref_logp")
    fwd(lo=-0.1, part="clip")
    fwd(hi=math.nan, part="clip")
    fwd(ent=math.inf, part="finite")
    fwd(temp=0.0, part="temperature")
    fwd(red=7, part="reduction")
    fwd(norm=None, part="null")
    fwd(row=None, part="null")
    fwd(loss=None, part="null")


def test_preference_refusals_and_workspace():
    L = _lib.lib()
    assert L.gtg_preference_workspace_bytes(5, 3) == (5 * 6 + 6) * 8
    assert L.gtg_preference_workspace_bytes(0, 2) == 4 * 8

    def fwd(T=2, pairs=2, ld=50, targets=P, ref=P, beta=0.1, eps=0.0, red=MEAN, stats=P, loss=P, ws=P, nbytes=1 << 20, **kw):
        refused("gtg_preference_fwd", P, F32, T, pairs, 50, ld, 0, targets, 0, None, ref, beta, eps, red, stats, P, P, P, loss, ws, nbytes,
                None, **kw)

    fwd(T=-1, part="size")
    fwd(pairs=-1, part="size")
    fwd(T=1 << 20, pairs=1 << 20, part="size")
    fwd(ld=49, part="stride")
    fwd(targets=None, part="null")
    fwd(ref=None, part="null")
    fwd(beta=math.inf, part="beta")
    for e in (-0.1, 1.0, math.nan):
        fwd(eps=e, part="label_smoothing")
    fwd(red=9, part="reduction")
    fwd(stats=None, part="null")
    fwd(loss=None, part="null")
    fwd(ws=None, part="workspace")
    fwd(nbytes=8, part="workspace")
    refused("gtg_preference_bwd", P, F32, 2, 2, 50, 50, 0, P, 0, None, P, None, P, None, Q, 50, None, part="null")
    refused("gtg_preference_bwd", P, F32, 2, 2, 50, 50, 0, P, 0, None, P, P, P, None, P, 50, None, part="overlap")


def test_nothing_to_do_is_not_an_error():
    L = _lib.lib()
    assert L.gtg_top_logits(None, F32, 0, 50, 50, 3, 1.0, None, None, None, None) == 0
    assert L.gtg_token_logprob_fwd(None, BF16, 0, 50, 50, None, 0, 1.0, None, None, None, None) == 0
    assert L.gtg_token_logprob_bwd(None, F16, 0, 50, 50, None, 0, 1.0, None, None, None, None, 50, None) == 0


def test_python_functions_refuse_cpu_tensors():
    import torch

    from gtg_vae_amd import functional as Fn

    x, y, f = torch.randn(2, 4, 30), torch.ones(2, 4, dtype=torch.long), torch.zeros(2, 4)
    i = torch.zeros(2, 4, 3, dtype=torch.int32)
    for call in (lambda: Fn.top_logits(x, 3), lambda: Fn.token_logprob(x, y, 0), lambda: Fn.distill_loss(x, x[..., :3], i, y, 0),
                 lambda: Fn.policy_loss(x, y, 0, f, f), lambda: Fn.preference_loss(x, y, 0, f[0])):
        with pytest.raises(_lib.GtgError):
            call()


def test_temperatures_out_of_range_are_refused():
    for t in (1e-7, 1e7, 1e-300, 1e300):
        refused("gtg_top_logits", *OK, 3, t, P, P, P, None, part="temperature")
        refused("gtg_token_logprob_fwd", *OK, P, 0, t, P, P, P, None, part="temperature")
        refused("gtg_token_logprob_bwd", *OK, P, 0, t, P, P, P, Q, 50, None, part="temperature")
