"""The losses on vocabulary logits as a program uses them: text decoders (DAE) in the roles of teacher and student, of behaviour,
reference and trained model, and each loss's gradient through decoder and projection against autograd on the plain 64-bit
restatement of the same logits."""
import pytest
import torch

from oracle import token_ops_oracle as O

pytestmark = pytest.mark.gpu
T, B, V, LATENT = 7, 6, 1201, 8


def _model(seed, train=False):
    from gtg_vae_amd.text_vae import DAE

    torch.manual_seed(seed)
    return DAE(LATENT, V, 0).cuda().train(train)


def _batch(seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randint(3, V, (T + 1, B), generator=g)
    x[0] = 2
    for b in range(1, B):
        x[T + 1 - b:, b] = 0                  # sentences of several lengths
    return torch.randn((B, LATENT), generator=g).cuda(), x[:-1].cuda(), x[1:].cuda()


def _through_the_model(model, z, inputs, loss_of, oracle_of, tol):
    """One forward and backward of `model` with loss_of(logits); the gradient at the logits against oracle_of(float64
    logits), and the projection's weight gradient against the product of that with the decoder's output."""
    logits, _ = model.decode(z, inputs)
    logits.retain_grad()
    model.zero_grad(set_to_none=True)
    loss = loss_of(logits)
    loss.backward()
    x64 = logits.detach().double().cpu().requires_grad_(True)
    want = oracle_of(x64)
    (dx,) = torch.autograd.grad(want, x64)
    assert abs(loss.item() - want.item()) <= 1e-5 * (1 + abs(want.item()))
    scale = dx.abs().max().item()
    assert (logits.grad.double().cpu() - dx).abs().max().item() <= tol * scale
    db = dx.reshape(-1, V).sum(0)
    assert (model.proj.bias.grad.double().cpu() - db).abs().max().item() <= 10 * tol * db.abs().max().item()
    for name, p in model.named_parameters():
        if name.startswith(("proj", "G", "z2emb", "embed")):
            assert p.grad is not None and torch.isfinite(p.grad).all() and p.grad.abs().max() > 0, name
    return logits


# fp32 logits of a spread below 10: a probability is within (3 * 10 + 16 + V / 64) 2^-24 = 4e-6 (the row kernels' bound)
TOL = 4 * 4e-6


@pytest.mark.parametrize("with_tail", [True, False])
def test_teacher_to_student(with_tail):
    teacher, student = _model(1), _model(2)
    z, inputs, targets = _batch(3)
    with torch.no_grad():
        answer, _ = teacher.decode(z, inputs)
    values, indices, tail = teacher.top_logits(answer, 20, temperature=2.0)
    tail = tail if with_tail else None
    y = targets.cpu()

    def oracle(x64):
        rows = O.distill_rows(x64, values.cpu(), indices.cpu(), y, 0, None if tail is None else tail.cpu(), 2.0, 0.3)
        return O.reduce(rows, y != 0, "mean")

    _through_the_model(student, z, inputs, lambda l: student.loss_distill(l, targets, values, indices, tail, 2.0, 0.3), oracle, TOL)
    # a student that is the teacher has nothing to learn
    loss = teacher.loss_distill(answer, targets, values, indices, tail, 2.0)
    if with_tail:
        assert abs(loss.item()) < 1e-6


def test_sample_score_and_update():
    behaviour, reference = _model(1), _model(5)
    z, _, _ = _batch(3)
    with torch.no_grad():
        tokens = torch.cat(behaviour.generate(z, T + 1, "sample"))          # (T + 1, B), the first one the start symbol
        inputs, targets = tokens[:-1], tokens[1:].clone()
        targets[T - 2:, 1] = 0                                              # one answer ends early
        old, entropy = behaviour.token_logprob(behaviour.decode(z, inputs)[0], targets)
        ref, _ = reference.token_logprob(reference.decode(z, inputs)[0], targets)
    adv = torch.randn(B, device="cuda")
    y = targets.cpu()

    def oracle(x64):
        rows, _, _ = O.policy_rows(x64, y, 0, old.cpu(), adv.cpu(), ref.cpu(), kl_coef=0.05, entropy_coef=0.01)
        return O.reduce(rows, y != 0, "mean")

    seen = {}

    def loss_of(logits):
        loss, seen["logp"], seen["entropy"] = behaviour.loss_policy(logits, targets, old, adv, ref, kl_coef=0.05, entropy_coef=0.01)
        return loss

    _through_the_model(behaviour, z, inputs, loss_of, oracle, TOL)
    # nothing has changed since the answers were sampled: every ratio is 1
    assert torch.equal(seen["logp"], old) and torch.equal(seen["entropy"], entropy)


def test_pairs_of_answers():
    policy, reference = _model(1), _model(5)
    z, inputs, targets = _batch(4)
    z = torch.cat((z[: B // 2], z[: B // 2]))                               # the same sentences, two answers each
    with torch.no_grad():
        ref = reference.token_logprob(reference.decode(z, inputs)[0], targets)[0].sum(0)
    y = targets.cpu()
    _through_the_model(policy, z, inputs, lambda l: policy.loss_preference(l, targets, ref, beta=0.2, label_smoothing=0.05)[0],
                       lambda x64: O.preference(x64, y, 0, ref.cpu(), 0.2, 0.05)[0].mean(), TOL)


def test_losses_add_up_on_one_graph():
    """Two of the losses and the reference's cross-entropy on the same logits: gradients add."""
    model = _model(1)
    z, inputs, targets = _batch(3)
    with torch.no_grad():
        logits0, _ = model.decode(z, inputs)
    values, indices, tail = model.top_logits(logits0 + 0.1 * torch.randn_like(logits0), 9)
    parts = [lambda l: model.loss_distill(l, targets, values, indices, tail), lambda l: model.token_logprob(l, targets)[0].sum(),
             lambda l: model.loss_rec(l, targets).mean()]
    one = []
    for f in parts:
        x = logits0.clone().requires_grad_(True)
        one.append(torch.autograd.grad(f(x), x)[0])
    x = logits0.clone().requires_grad_(True)
    (both,) = torch.autograd.grad(sum(f(x) for f in parts), x)
    assert torch.allclose(both, sum(one), rtol=1e-5, atol=1e-7)
    # the log-probability is the cross-entropy's negative
    assert torch.allclose(one[1], -one[2] * B, rtol=1e-4, atol=1e-6)


def test_under_mixed_precision():
    """bf16 logits out of an autocast projection: gradients come back in bf16 and reach the fp32 weights."""
    model = _model(1)
    z, inputs, targets = _batch(3)
    emb = model._embed(inputs, model._linear(model.z2emb, z))
    output, _ = model.run_lstm(model.G, emb)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        logits = model.proj(output.reshape(-1, 1024)).view(T, B, V)
        assert logits.dtype == torch.bfloat16
        logits.retain_grad()
        loss, _, _ = model.loss_policy(logits, targets, torch.full((T, B), -7.0, device="cuda"), torch.ones(B, device="cuda"))
    loss.backward()
    x64 = logits.detach().double().cpu().requires_grad_(True)
    y = targets.cpu()
    rows, _, _ = O.policy_rows(x64, y, 0, torch.full((T, B), -7.0), torch.ones(B))
    (dx,) = torch.autograd.grad(O.reduce(rows, y != 0, "mean"), x64)
    assert logits.grad.dtype == torch.bfloat16 and model.proj.weight.grad.dtype == torch.float32
    off = (logits.grad.double().cpu() - dx).abs() - (2.0 ** -8 * dx.abs() + TOL * dx.abs().max())
    assert off.max().item() <= 0
