"""What the losses and read-outs on rows of vocabulary logits cost, as a user's program calls them.

Five operators on the text decoder's logits (T, B, V), time-major as the decoder returns them:

  top       a teacher's k largest logits per token and the log mass of the rest
  logprob   log-probability of the given tokens and the entropy of their distributions, without or with gradient
  distill   a student's loss against a teacher's top logits, and its gradient
  policy    the clipped policy loss with KL and entropy terms, and its gradient
  prefer    the preference loss over (chosen, rejected) pairs, and its gradient

``run`` computes them from elementary torch operations, or, where ``own`` is true, through the package's functions.
"""
import math

import torch

own = False

PAD = 0
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
# tokens x vocabulary of the largest case: 40 steps of 256 sentences over 30 522 words, the joint model's batch
LARGEST = 40 * 256 * 30522


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # scoring one new token of eight sentences while they are being generated: nothing but latency
        {"name": "logprob step", "op": "logprob", "grad": False, "dtype": "float32", "T": 1, "B": 8, "V": 30522, "tau": 1.0},
        # a whole joint batch with gradients through both outputs (log-probability and entropy)
        {"name": "logprob batch", "op": "logprob", "grad": True, "dtype": "float32", "T": 40, "B": 256, "V": 30522, "tau": 1.0},
        # a teacher answering one step of a few sentences
        {"name": "top step", "op": "top", "dtype": "float32", "T": 1, "B": 16, "V": 30522, "k": 16, "tau": 1.0},
        # a teacher's joint batch stored as its 64 largest logits at temperature 2
        {"name": "top batch", "op": "top", "dtype": "bfloat16", "T": 40, "B": 256, "V": 30522, "k": 64, "tau": 2.0},
        # a small student's step on a small vocabulary
        {"name": "distill small", "op": "distill", "dtype": "bfloat16", "T": 12, "B": 64, "V": 1000, "k": 8, "tau": 1.0,
         "alpha": 0.0, "tail": True},
        # the joint batch, softened, mixed half and half with the words themselves, with the teacher's rest mass
        {"name": "distill batch", "op": "distill", "dtype": "float32", "T": 40, "B": 256, "V": 30522, "k": 64, "tau": 2.0,
         "alpha": 0.5, "tail": True},
        # a wide vocabulary, sequences of odd length, the teacher's list taken as its whole distribution
        {"name": "distill wide", "op": "distill", "dtype": "bfloat16", "T": 73, "B": 21, "V": 131072, "k": 128, "tau": 1.0,
         "alpha": 0.1, "tail": False},
        # one policy update on a handful of short answers
        {"name": "policy small", "op": "policy", "dtype": "float32", "T": 16, "B": 8, "V": 4099, "tau": 1.0, "kl": 0.04,
         "ent": 0.0},
        # one policy update on a joint batch of answers, with KL and entropy terms
        {"name": "policy batch", "op": "policy", "dtype": "bfloat16", "T": 40, "B": 256, "V": 30522, "tau": 0.8, "kl": 0.04,
         "ent": 0.01},
        # a single pair of short answers
        {"name": "prefer pair", "op": "prefer", "dtype": "float16", "T": 24, "B": 2, "V": 30522, "beta": 0.1, "eps": 0.0},
        # 128 pairs, the joint batch's size
        {"name": "prefer batch", "op": "prefer", "dtype": "float32", "T": 40, "B": 256, "V": 30522, "beta": 0.1, "eps": 0.1},
        # long answers over an odd, wide vocabulary
        {"name": "prefer long", "op": "prefer", "dtype": "bfloat16", "T": 513, "B": 6, "V": 50021, "beta": 0.3, "eps": 0.0},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["top", "logprob", "distill", "policy", "prefer"])
    V = _log_int(rng, 300, 131072)
    rows = min(_log_int(rng, 1, 40 * 256), max(1, LARGEST // V))
    T = max(1, min(rows, _log_int(rng, 1, 640)))
    B = max(1, rows // T)
    if op == "prefer":
        B = max(2, B // 2 * 2)
        T = max(1, min(T, LARGEST // (V * B)))
    c = {"op": op, "dtype": rng.choice(sorted(DTYPES)), "T": T, "B": B, "V": V}
    if op in ("top", "distill"):
        c["k"] = _log_int(rng, 1, 256)
    if op != "prefer":
        c["tau"] = rng.choice([1.0, round(rng.uniform(0.5, 4.0), 3)])
    if op == "logprob":
        c["grad"] = rng.random() < 0.7
    elif op == "distill":
        c["alpha"] = rng.choice([0.0, round(rng.uniform(0.0, 1.0), 3)])
        c["tail"] = rng.random() < 0.6
    elif op == "policy":
        c["kl"] = rng.choice([0.0, round(rng.uniform(0.01, 0.2), 3)])
        c["ent"] = rng.choice([0.0, round(rng.uniform(0.001, 0.05), 4)])
    elif op == "prefer":
        c["beta"] = round(rng.uniform(0.05, 0.5), 3)
        c["eps"] = rng.choice([0.0, 0.1])
    return c


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _blocks(rows, V):
    """Row ranges of at most 64 M logits, so that the helpers' 32- and 64-bit copies stay small."""
    step = max(1, (64 << 20) // V)
    return [(a, min(rows, a + step)) for a in range(0, rows, step)]


def _make_logits(case, gen):
    """Rows as a trained decoder gives them: a spread of about 2, a few words well above it."""
    T, B, V = case["T"], case["B"], case["V"]
    rows, dt, dev = T * B, DTYPES[case["dtype"]], "cuda"
    x = torch.empty((rows, V), dtype=dt, device=dev)
    for a, b in _blocks(rows, V):
        x[a:b] = (2.0 * torch.randn((b - a, V), generator=gen, device=dev)).to(dt)
    top = torch.randint(1, V, (rows, 5), generator=gen, device=dev)
    lift = 4.0 + 5.0 * torch.rand((rows, 5), generator=gen, device=dev)
    x.scatter_(1, top, lift.to(dt))
    # the words that were said: mostly among the likely ones
    said = torch.where(torch.rand((rows,), generator=gen, device=dev) < 0.75, top[:, 0],
                       torch.randint(1, V, (rows,), generator=gen, device=dev)).view(T, B)
    # sentences end between a fifth of the longest and the longest (all of one length where there is one step)
    lengths = torch.randint(max(1, T // 5), T + 1, (B,), generator=gen, device=dev)
    lengths[0] = T
    targets = torch.where(torch.arange(T, device=dev)[:, None] < lengths[None, :], said, PAD)
    return x.view(T, B, V), targets


def _logp_of(x, targets, tau):
    """(T, B) float32 log-probabilities of the targets under x."""
    T, B, V = x.shape
    flat, y, out = x.view(T * B, V), targets.reshape(-1), torch.empty((T * B,), device=x.device)
    for a, b in _blocks(T * B, V):
        z = flat[a:b].float() / tau
        out[a:b] = z.gather(1, y[a:b, None])[:, 0] - torch.logsumexp(z, 1)
    return out.view(T, B)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(1000003 * seed + 17)
    x, targets = _make_logits(case, gen)
    T, B, V = x.shape
    st = {"case": case, "x": x, "targets": targets}
    op = case["op"]
    randn = lambda *s: torch.randn(s, generator=gen, device="cuda")  # noqa: E731
    if op == "distill":
        # the teacher: the student's logits and some, its k largest stored in the student's type
        k, rows, flat = case["k"], T * B, x.view(T * B, V)
        val = torch.empty((rows, k), dtype=x.dtype, device="cuda")
        idx = torch.empty((rows, k), dtype=torch.int32, device="cuda")
        tail = torch.empty((rows,), device="cuda")
        for a, b in _blocks(rows, V):
            t = flat[a:b].float() + 0.7 * randn(b - a, V)
            v, i = torch.topk(t, k, dim=1)
            val[a:b], idx[a:b] = v.to(x.dtype), i.int()
            tail[a:b] = torch.logsumexp(t.scatter(1, i, -math.inf) / case["tau"], 1)
        st.update(values=val.view(T, B, k), indices=idx.view(T, B, k), tail=tail.view(T, B) if case["tail"] else None)
    elif op == "policy":
        # the answers were sampled a few updates ago; the reference model is further away
        now = _logp_of(x, targets, case["tau"])
        st.update(old=now + 0.15 * randn(T, B), ref=now + 0.3 * randn(T, B), adv=randn(B))
    elif op == "prefer":
        seq = torch.where(targets != PAD, _logp_of(x, targets, 1.0), 0.0).sum(0)
        st.update(ref=seq + 3.0 * randn(B))
    elif op == "logprob" and case["grad"]:
        st.update(g_logp=randn(T, B), g_ent=0.1 * randn(T, B))
    if op in ("distill", "policy", "prefer") or case.get("grad"):
        x.requires_grad_(True)
    return st


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
CLIP_LOW, CLIP_HIGH = 0.2, 0.28


def run(st):
    c = st["case"]
    return _OWN[c["op"]](st, c) if own else _PLAIN[c["op"]](st, c)


def _own_top(st, c):
    from gtg_vae_amd import functional as Fn

    v, i, tail = Fn.top_logits(st["x"], c["k"], temperature=c["tau"])
    return {"values": v, "indices": i, "tail": tail}


def _own_logprob(st, c):
    from gtg_vae_amd import functional as Fn

    x = st["x"]
    logp, ent = Fn.token_logprob(x, st["targets"], PAD, temperature=c["tau"])
    out = {"logp": logp.detach(), "entropy": ent.detach()}
    if c["grad"]:
        (out["dlogits"],) = torch.autograd.grad((logp, ent), (x,), (st["g_logp"], st["g_ent"]))
    return out


def _own_distill(st, c):
    from gtg_vae_amd import functional as Fn

    x = st["x"]
    loss = Fn.distill_loss(x, st["values"], st["indices"], st["targets"], PAD, tail=st["tail"], temperature=c["tau"],
                           ce_weight=c["alpha"])
    (dx,) = torch.autograd.grad(loss, (x,))
    return {"loss": loss.detach(), "dlogits": dx}


def _own_policy(st, c):
    from gtg_vae_amd import functional as Fn

    x = st["x"]
    loss, logp, ent = Fn.policy_loss(x, st["targets"], PAD, st["old"], st["adv"], ref_logp=st["ref"], clip_low=CLIP_LOW,
                                     clip_high=CLIP_HIGH, kl_coef=c["kl"], entropy_coef=c["ent"], temperature=c["tau"])
    (dx,) = torch.autograd.grad(loss, (x,))
    return {"loss": loss.detach(), "logp": logp, "entropy": ent, "dlogits": dx}


def _own_prefer(st, c):
    from gtg_vae_amd import functional as Fn

    x = st["x"]
    loss, seq = Fn.preference_loss(x, st["targets"], PAD, st["ref"], beta=c["beta"], label_smoothing=c["eps"])
    (dx,) = torch.autograd.grad(loss, (x,))
    return {"loss": loss.detach(), "seq_logp": seq, "dlogits": dx}


_OWN = {"top": _own_top, "logprob": _own_logprob, "distill": _own_distill, "policy": _own_policy, "prefer": _own_prefer}


# ---- plain forms: elementary operations over the rows in 32 bits, what is one number per row in 64 ------------------
def _softmax_parts(z):
    """For z (T, B, V) float32: row maximum, exp(z - max) and its sum."""
    m = z.max(-1, keepdim=True).values
    e = torch.exp(z - m)
    return m, e, e.sum(-1, keepdim=True)


@torch.no_grad()
def _plain_top(st, c):
    x = st["x"]
    z = x.float() + 0.0
    bits = z.view(torch.int32)
    order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()          # integers in the order of the values
    V = x.shape[-1]
    order = (order << 32) | (V - 1 - torch.arange(V, device=x.device))     # among equals the lowest index is the largest
    key = torch.topk(order, c["k"], dim=-1).values
    idx = V - 1 - (key & 0xFFFFFFFF)
    val = x.gather(-1, idx)
    rest = z.scatter_(-1, idx, -math.inf) / c["tau"]
    m, _, s = _softmax_parts(rest)
    return {"values": val, "indices": idx.int(), "tail": (m.double() + s.double().log())[..., 0].float()}


def _logprob_rows(z, y):
    """p, its row maximum, and (T, B, 1) float64 rows: log sum exp(z - max), log-probability of y, entropy."""
    m, e, s = _softmax_parts(z)
    log_s = s.double().log()
    logp = (z.gather(-1, y[..., None]) - m).double() - log_s
    ent = log_s - ((e * (z - m)).sum(-1, keepdim=True).double() / s.double())
    return e / s, m, log_s, logp, ent


@torch.no_grad()
def _plain_logprob(st, c):
    x, y = st["x"], st["targets"]
    keep = (y != PAD)[..., None]
    z = x.float() / c["tau"]
    p, m, log_s, logp, ent = _logprob_rows(z, y)
    out = {"logp": torch.where(keep, logp, 0.0)[..., 0].float(), "entropy": torch.where(keep, ent, 0.0)[..., 0].float()}
    if c["grad"]:
        g_l, g_h = (torch.where(keep, st[k][..., None], 0.0) / c["tau"] for k in ("g_logp", "g_ent"))
        d = -p * (g_l + g_h * ((z - m) + (ent - log_s).float()))
        d.scatter_add_(-1, y[..., None], g_l)
        out["dlogits"] = d.to(x.dtype)
    return out


@torch.no_grad()
def _plain_distill(st, c):
    x, y, idx, tau, a = st["x"], st["targets"], st["indices"].long(), c["tau"], c["alpha"]
    keep = (y != PAD)[..., None]
    n = keep.sum()
    # the teacher's distribution over its list and the rest
    t = st["values"].double() / tau
    if st["tail"] is not None:
        t = torch.cat((t, st["tail"][..., None].double()), -1)
    t = t - t.max(-1, keepdim=True).values
    log_q = t - t.exp().sum(-1, keepdim=True).log()
    q = log_q.exp()
    # the student's
    z = x.float() / tau
    m, e, s = _softmax_parts(z)
    log_s = s.double().log()
    log_p = (z.gather(-1, idx) - m).double() - log_s
    d = e / s
    if st["tail"] is not None:
        s_rest = e.scatter(-1, idx, 0.0).sum(-1, keepdim=True)
        log_p = torch.cat((log_p, s_rest.double().log() - log_s), -1)
        d *= (1.0 - q[..., -1:] * s.double() / s_rest.double()).float()
        d.scatter_(-1, idx, log_p[..., :-1].exp().float() - q[..., :-1].float())
    else:
        d.scatter_add_(-1, idx, -q.float())
    loss = (1.0 - a) * tau * tau * (q * (log_q - log_p)).sum(-1, keepdim=True)
    d *= (1.0 - a) * tau
    if a > 0:
        x32 = x.float()
        m, e, s = _softmax_parts(x32)
        loss = loss + a * (s.double().log() - (x32.gather(-1, y[..., None]) - m).double())
        d += a * (e / s)
        d.scatter_add_(-1, y[..., None], torch.full(y.shape + (1,), -a, device=x.device))
    d *= torch.where(keep, 1.0 / n, 0.0).float()
    return {"loss": (torch.where(keep, loss, 0.0).sum() / n).float(), "dlogits": d.to(x.dtype)}


@torch.no_grad()
def _plain_policy(st, c):
    x, y, tau = st["x"], st["targets"], c["tau"]
    keep = (y != PAD)[..., None]
    n = keep.sum()
    z = x.float() / tau
    p, m, log_s, logp, ent = _logprob_rows(z, y)
    old, ref, adv = st["old"][..., None].double(), st["ref"][..., None].double(), st["adv"][None, :, None].double()
    r = torch.exp(logp - old)
    free, held = r * adv, r.clamp(1.0 - CLIP_LOW, 1.0 + CLIP_HIGH) * adv
    away = torch.exp(ref - logp)
    loss = -torch.minimum(free, held) + c["kl"] * (away - (ref - logp) - 1.0) - c["ent"] * ent
    w = torch.where(keep, 1.0 / n, 0.0).double()
    g = w / tau * (-torch.where(free <= held, free, 0.0) + c["kl"] * (1.0 - away))
    d = p * -g.float()
    if c["ent"] > 0:
        d += p * ((z - m) + (ent - log_s).float()) * (w * c["ent"] / tau).float()
    d.scatter_add_(-1, y[..., None], g.float())
    rows = lambda v: torch.where(keep, v, 0.0)[..., 0].float()  # noqa: E731
    return {"loss": (w * loss).sum().float(), "logp": rows(logp), "entropy": rows(ent), "dlogits": d.to(x.dtype)}


@torch.no_grad()
def _plain_prefer(st, c):
    x, y = st["x"], st["targets"]
    keep = (y != PAD)[..., None]
    P = y.shape[1] // 2
    z = x.float()
    m, e, s = _softmax_parts(z)
    logp = (z.gather(-1, y[..., None]) - m).double() - s.double().log()
    seq = torch.where(keep, logp, 0.0)[..., 0].sum(0)
    ratio = seq - st["ref"].double()
    margin = c["beta"] * (ratio[:P] - ratio[P:])
    softplus = lambda v: torch.log1p(torch.exp(-v.abs())) + v.clamp(min=0.0)  # noqa: E731
    loss = ((1.0 - c["eps"]) * softplus(-margin) + c["eps"] * softplus(margin)).mean()
    dm = (c["eps"] - 1.0 / (1.0 + torch.exp(margin))) * (c["beta"] / P)
    g = torch.where(keep, torch.cat((dm, -dm))[None, :, None], 0.0).float()
    d = e / s * -g
    d.scatter_add_(-1, y[..., None], g)
    return {"loss": loss.float(), "seq_logp": seq.float(), "dlogits": d.to(x.dtype)}


_PLAIN = {"top": _plain_top, "logprob": _plain_logprob, "distill": _plain_distill, "policy": _plain_policy,
          "prefer": _plain_prefer}


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    rows, V, s = case["T"] * case["B"], case["V"], DTYPES[case["dtype"]].itemsize
    op, k = case["op"], case.get("k", 0)
    grad = op in ("distill", "policy", "prefer") or case.get("grad", False)
    # the rows that count: a teacher answers every token, the losses leave out what lies behind a sentence's end (its
    # logits need not be read; its gradient is zero, and written)
    kept = rows if op == "top" else case["T"] + (case["B"] - 1) * (max(1, case["T"] // 5) + case["T"]) / 2
    row = {"top": k * (s + 4) + 4, "logprob": 8 + 8 + (8 if grad else 0), "distill": 8 + k * (s + 4) + 4,
           "policy": 8 + 8 + 8, "prefer": 8}[op]
    # a subtraction, a scaling, an exponential and an addition per logit; as much again for the gradient
    return {"bytes": kept * V * s + (rows * V * s if grad else 0) + rows * row, "flops": kept * V * (8 if grad else 4)}


# ---------------------------------------------------------------------------
# the same from the definitions in 64 bits
# ---------------------------------------------------------------------------
@torch.no_grad()
def exact(case, seed):
    st = prepare(case, seed)
    x, y = st["x"].detach(), st["targets"]
    T, B, V = x.shape
    rows, flat, yf = T * B, x.view(T * B, V), y.reshape(-1)
    on = yf != PAD
    op = case["op"]
    if op == "top":
        k = case["k"]
        val, idx, tail = [], [], []
        for a, b in _blocks(rows, V):
            srt, pos = torch.sort(flat[a:b].double(), dim=1, descending=True, stable=True)
            val.append(srt[:, :k])
            idx.append(pos[:, :k].int())
            tail.append(torch.logsumexp(srt[:, k:] / case["tau"], 1))
        return {"values": torch.cat(val).view(T, B, k), "indices": torch.cat(idx).view(T, B, k),
                "tail": torch.cat(tail).view(T, B)}
    tau = case.get("tau", 1.0)
    logp, ent = torch.zeros(rows, dtype=torch.float64, device=x.device), torch.zeros(rows, dtype=torch.float64, device=x.device)
    for a, b in _blocks(rows, V):
        lp = torch.log_softmax(flat[a:b].double() / tau, 1)
        logp[a:b] = lp.gather(1, yf[a:b, None])[:, 0]
        ent[a:b] = -(lp.exp() * lp).sum(1)
    logp, ent = torch.where(on, logp, 0.0), torch.where(on, ent, 0.0)
    n = on.sum().double()
    # per row: how the result changes with the row's log-probability and with its entropy
    zero = torch.zeros_like(logp)
    if op == "logprob":
        out = {"logp": logp.view(T, B), "entropy": ent.view(T, B)}
        if not case["grad"]:
            return out
        by_logp = torch.where(on, st["g_logp"].reshape(-1).double(), 0.0)
        by_ent = torch.where(on, st["g_ent"].reshape(-1).double(), 0.0)
    elif op == "policy":
        adv = st["adv"].double().repeat(T)
        lp = logp.clone().requires_grad_(True)
        h = ent.clone().requires_grad_(True)
        with torch.enable_grad():
            ratio = (lp - st["old"].reshape(-1).double()).exp()
            gap = st["ref"].reshape(-1).double() - lp
            each = -torch.minimum(ratio * adv, ratio.clamp(1 - CLIP_LOW, 1 + CLIP_HIGH) * adv) \
                + case["kl"] * (gap.exp() - gap - 1) - case["ent"] * h
            loss = each[on].sum() / n
            by_logp, by_ent = torch.autograd.grad(loss, (lp, h))
        out = {"loss": loss.detach(), "logp": logp.view(T, B), "entropy": ent.view(T, B)}
    elif op == "prefer":
        lp = logp.clone().requires_grad_(True)
        with torch.enable_grad():
            seq = lp.view(T, B).sum(0)
            ratio = seq - st["ref"].double()
            margin = case["beta"] * (ratio[: B // 2] - ratio[B // 2:])
            ls = torch.nn.functional.logsigmoid
            loss = (-(1 - case["eps"]) * ls(margin) - case["eps"] * ls(-margin)).mean()
            (by_logp,) = torch.autograd.grad(loss, (lp,))
        by_logp, by_ent = torch.where(on, by_logp, 0.0), zero
        out = {"loss": loss.detach(), "seq_logp": seq.detach()}
    grad = torch.empty((rows, V), dtype=torch.float64, device=x.device)
    if op == "distill":
        total = torch.zeros((), dtype=torch.float64, device=x.device)
        k, al = case["k"], case["alpha"]
        val, idx = st["values"].reshape(rows, k), st["indices"].reshape(rows, k).long()
        for a, b in _blocks(rows, V):
            z = flat[a:b].double().requires_grad_(True)
            with torch.enable_grad():
                lp = torch.log_softmax(z / tau, 1)
                student = lp.gather(1, idx[a:b])
                teacher = val[a:b].double() / tau
                if st["tail"] is not None:
                    rest = torch.logsumexp(lp.scatter(1, idx[a:b], -math.inf), 1)
                    student = torch.cat((student, rest[:, None]), 1)
                    teacher = torch.cat((teacher, st["tail"].reshape(-1)[a:b, None].double()), 1)
                teacher = torch.log_softmax(teacher, 1)
                each = (1 - al) * tau ** 2 * (teacher.exp() * (teacher - student)).sum(1)
                if al > 0:
                    each = each - al * torch.log_softmax(z, 1).gather(1, yf[a:b, None])[:, 0]
                part = torch.where(on[a:b], each, 0.0).sum() / n
                (grad[a:b],) = torch.autograd.grad(part, (z,))
            total += part.detach()
        return {"loss": total, "dlogits": grad.view(T, B, V)}
    for a, b in _blocks(rows, V):
        lp = torch.log_softmax(flat[a:b].double() / tau, 1)
        g = -lp.exp() * (by_logp[a:b, None] + by_ent[a:b, None] * (lp + ent[a:b, None]))
        g[torch.arange(b - a, device=x.device), yf[a:b]] += by_logp[a:b]
        grad[a:b] = g / tau
    out["dlogits"] = grad.view(T, B, V)
    return out
