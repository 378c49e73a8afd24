"""Plain 64-bit restatements of the operators on rows of vocabulary logits (gtg_top_logits, gtg_token_logprob,
gtg_distill_loss, gtg_policy_loss, gtg_preference): test infrastructure only.  Losses are built from the definitions;
their gradients come from autograd on them."""
import math

import torch
import torch.nn.functional as F


def keep_rows(targets, padidx, mask=None):
    keep = targets != padidx
    return keep if mask is None else keep & mask.bool()


def top_logits(logits, k, temperature=1.0):
    x = logits.double() + 0.0                      # -0 and +0 are equal
    key = torch.where(torch.isnan(x), math.inf, x)
    nan_first = torch.isnan(x).int()
    # larger first, equal ones by index: a stable sort by value, then by "is a NaN"
    order = torch.argsort(key, dim=-1, descending=True, stable=True)
    order = order.gather(-1, torch.argsort(nan_first.gather(-1, order), dim=-1, descending=True, stable=True))
    idx = order[..., :k]
    rest = x.scatter(-1, idx, -math.inf) / temperature
    tail = torch.logsumexp(rest, -1)
    return logits.gather(-1, idx), idx.int(), tail


def _log_softmax(z):
    return torch.log_softmax(z, -1)


def token_logprob(logits, targets, padidx, temperature=1.0, mask=None):
    """logits float64 (autograd leaf or not)."""
    keep = keep_rows(targets, padidx, mask)
    lp = _log_softmax(logits / temperature)
    y = torch.where(keep, targets, 0)
    logp = lp.gather(-1, y[..., None])[..., 0]
    p = lp.exp()
    ent = -(p * torch.where(p > 0, lp, 0.0)).sum(-1)
    return torch.where(keep, logp, 0.0), torch.where(keep, ent, 0.0)


def reduce(rows, keep, reduction):
    rows = torch.where(keep, rows, 0.0)
    if reduction == "none":
        return rows
    n = keep.sum() if reduction == "mean" else 1
    return rows.sum() / max(int(n), 1)


def distill_rows(logits, values, indices, targets, padidx, tail=None, temperature=1.0, ce_weight=0.0):
    keep = keep_rows(targets, padidx)
    lead, V = targets.shape, logits.shape[-1]
    z = logits.reshape(-1, V)
    k = values.shape[-1]
    v, i = values.double().reshape(-1, k), indices.long().reshape(-1, k)
    t = None if tail is None else tail.double().reshape(-1)
    y, on = targets.reshape(-1), keep.reshape(-1)
    out = []
    for r in range(z.shape[0]):
        if not on[r]:
            out.append(z.new_zeros(()))
            continue
        lp = _log_softmax(z[r] / temperature)
        ok = i[r] >= 0
        loss = z.new_zeros(())
        u = v[r][ok] / temperature
        student = lp[i[r][ok]]
        if t is not None and t[r] > -math.inf:
            others = torch.ones(V, dtype=torch.bool, device=z.device)
            others[i[r][ok]] = False
            u = torch.cat((u, t[r][None]))
            student = torch.cat((student, torch.logsumexp(lp[others], 0)[None]))
        use = u > -math.inf
        if use.any() and ce_weight < 1:
            log_q = _log_softmax(u[use])
            loss = (1 - ce_weight) * temperature ** 2 * (log_q.exp() * (log_q - student[use])).sum()
        if ce_weight > 0:
            loss = loss - ce_weight * _log_softmax(z[r])[y[r]]
        out.append(loss)
    return (torch.stack(out) if out else z.new_zeros((0,))).view(lead)


def policy_rows(logits, targets, padidx, old_logp, advantages, ref_logp=None, clip_low=0.2, clip_high=0.2, kl_coef=0.0,
                entropy_coef=0.0, temperature=1.0, mask=None):
    logp, ent = token_logprob(logits, targets, padidx, temperature, mask)
    keep = keep_rows(targets, padidx, mask)
    adv = advantages.double().expand(targets.shape)
    rho = torch.exp(logp - torch.where(keep, old_logp.double(), 0.0))
    free, held = rho * adv, rho.clamp(1 - clip_low, 1 + clip_high) * adv
    rows = -torch.where(free <= held, free, held.detach())
    if ref_logp is not None and kl_coef:
        gap = torch.where(keep, ref_logp.double(), 0.0) - logp
        rows = rows + kl_coef * (torch.exp(gap) - gap - 1)
    return torch.where(keep, rows - entropy_coef * ent, 0.0), logp, ent


def preference(logits, targets, padidx, ref_logp, beta=0.1, label_smoothing=0.0, mask=None, batch_first=False):
    logp, _ = token_logprob(logits, targets, padidx, 1.0, mask)
    seq = logp.sum(1 if batch_first else 0)
    ratio = seq - ref_logp.double()
    P = seq.numel() // 2
    m = beta * (ratio[:P] - ratio[P:])
    return -(1 - label_smoothing) * F.logsigmoid(m) - label_smoothing * F.logsigmoid(-m), seq
